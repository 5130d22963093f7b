"""A long context in three places: what was just read, an 8-bit cache, and an index.

One attention layer of a language model (random weights, two key heads of four
query heads each) reads a prompt, answers token by token, and keeps only
`budget` tokens a head in its cache.  What the cache gives up is not lost: the
evicted keys become the rows of a graph index, every later query is searched
in it, and attention over the tokens found is joined with attention over the
cache.

    python examples/context_memory.py
"""
from __future__ import annotations

import os
import sys
from dataclasses import dataclass

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

import beam_search_collab_b200 as B  # noqa: E402
from beam_search_collab_b200 import memory  # noqa: E402

HEADS, GROUP, DIM, BLOCK = 2, 4, 64, 32


def rows_for_search(keys: np.ndarray) -> np.ndarray:
    """Keys with one more coordinate, so that the nearest row of a query with 0
    there is the key with the largest inner product: |q - k|^2 is then
    |q|^2 + m^2 - 2 <q, k> with m the largest key's length."""
    squares = (keys.astype(np.float64) ** 2).sum(1)
    return np.concatenate((keys, np.sqrt(squares.max() - squares)[:, None]), 1).astype(np.float32)


@dataclass
class Archive:
    """What one eviction gave up: an index a head over its keys, whose row i is
    position gone[head, i] of the `lens` tokens that `table`'s blocks held."""
    indexes: list[B.Index]
    gone: torch.Tensor
    table: torch.Tensor
    lens: torch.Tensor


class ContextMemory:
    """The tokens of one sequence: `table` and `tokens` say which of `cache`'s
    blocks hold the recent ones and those that got much attention, `archives`
    (one an eviction) where the others are."""

    def __init__(self, room: int):
        self.cache = memory.TokenCache.empty(-(-room // BLOCK), HEADS, DIM, BLOCK)
        self.free = list(range(self.cache.k.shape[0]))
        self.table = torch.empty((1, 0), dtype=torch.int32, device="cuda")
        self.tokens = 0
        self.mass = None
        self.archives: list[Archive] = []

    def blocks(self, tokens: int) -> torch.Tensor:
        n = -(-tokens // BLOCK)
        got, self.free = self.free[:n], self.free[n:]
        return torch.tensor([got], dtype=torch.int32, device="cuda")

    def append(self, k, v) -> None:
        """k, v [tokens, HEADS, DIM] behind what is there."""
        n = k.shape[0]
        room = self.table.shape[1] * BLOCK
        if self.tokens + n > room:
            self.table = torch.cat((self.table, self.blocks(self.tokens + n - room)), 1).contiguous()
        i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        self.cache.write(k, v, i32(0, n), self.table, i32(self.tokens))
        self.tokens += n
        if self.mass is not None:       # new tokens start without weight
            self.mass = torch.nn.functional.pad(self.mass, (0, n))
        else:
            self.mass = torch.zeros((1, HEADS, n), device="cuda")

    def attend(self, q):
        """Attention of the last token's q [HEADS * GROUP, DIM] over the cache."""
        lens = torch.tensor([self.tokens], dtype=torch.int32, device="cuda")
        out, lse, self.mass = self.cache.attention(q[None, None], self.table, lens, with_lse=True, mass=self.mass)
        return out[0, 0], lse[0, 0]

    def evict(self, budget: int, recent: int) -> None:
        """Down to `budget` tokens a head; the others become rows of an index of
        this eviction's own.  Nothing to do where there are no more tokens."""
        if self.tokens <= budget:
            return
        lens = torch.tensor([self.tokens], dtype=torch.int32, device="cuda")
        new_table = self.blocks(budget)
        kept, new_lens, new_mass = self.cache.evict(self.mass, self.table, lens, new_table, budget, sinks=4, recent=recent)
        gone = torch.ones((HEADS, self.tokens), dtype=torch.bool, device="cuda").scatter_(1, kept[0].long(), False)
        gone = torch.stack([g.nonzero()[:, 0] for g in gone]).to(torch.int32)
        keys, _ = self.cache.read(self.table, lens, gone[None], values=False)
        indexes = [B.Index.from_vectors(rows_for_search(keys[0, h].cpu().numpy()), degree=32) for h in range(HEADS)]
        for ix in indexes:
            ix.build_graph(beam_width=64)
        self.archives.append(Archive(indexes, gone, self.table, lens))
        self.table, self.mass, self.tokens = new_table, new_mass, budget

    def recall(self, q, k: int):
        """Attention of q over the evicted tokens: of each eviction the `k`
        nearest keys of each query head (every query head of a key head sees
        them all).  Nothing evicted: zeros, whose log-sum is -infinity."""
        if not self.archives:
            return torch.zeros_like(q), torch.full((HEADS * GROUP,), -torch.inf, device="cuda")
        queries = torch.nn.functional.pad(q.float().view(HEADS, GROUP, DIM), (0, 1))
        torch.cuda.current_stream().synchronize()      # the search runs on the default stream
        found = [([], []) for _ in range(HEADS)]       # of each head: keys, values
        for a in self.archives:
            places = []
            for h in range(HEADS):
                ids, _, _ = a.indexes[h].search(queries[h].contiguous(), mode="warp4", K=k, topk_size=max(64, 2 * k))
                places.append(a.gone[h][torch.unique(ids[ids >= 0].long())])
            n = [len(p) for p in places]
            table = torch.full((HEADS, max(n)), -1, dtype=torch.int32, device="cuda")
            for h in range(HEADS):
                table[h, :n[h]] = places[h]
            for x, into in zip(self.cache.read(a.table, a.lens, table[None], dtype=q.dtype), (0, 1)):
                for h in range(HEADS):
                    found[h][into].append(x[0, h, :n[h]])
        # one sequence for each key head: its query heads over what they found
        keys, values = (torch.cat([x for h in range(HEADS) for x in found[h][i]])[:, None] for i in (0, 1))
        n = [sum(map(len, found[h][0])) for h in range(HEADS)]
        at = lambda x: torch.tensor(np.cumsum([0] + x), dtype=torch.int32, device="cuda")  # noqa: E731
        out, lse = memory.prompt_attention(q.view(HEADS, GROUP, DIM), keys, values, at([1] * HEADS), at(n), causal=False,
                                           with_lse=True)
        return out.reshape(HEADS * GROUP, DIM), lse.reshape(-1)

    def close(self) -> None:
        for a in self.archives:
            for ix in a.indexes:
                ix.close()


def run(tokens: int = 6000, steps: int = 24, budget: int = 512, found: int = 32, seed: int = 0) -> dict:
    """Reads `tokens` tokens, answers `steps`, and compares attention over the
    cache alone, and over the cache and what the index finds, with attention
    over everything (mean relative error of the outputs)."""
    g = torch.Generator("cuda").manual_seed(seed)
    width = 128
    topics = torch.randn((40, width), generator=g, device="cuda")
    weights = [torch.randn((width, n * DIM), generator=g, device="cuda") / width ** 0.5 for n in (HEADS * GROUP, HEADS, HEADS)]
    weights[0] = weights[1].view(width, HEADS, 1, DIM).expand(-1, -1, GROUP, -1).reshape(width, -1) + 0.3 * weights[0]

    def project(topic):
        x = topics[topic] + 0.5 * torch.randn((len(topic), width), generator=g, device="cuda")
        return [(x @ w).to(torch.bfloat16).view(len(topic), -1, DIM) for w in weights]

    q, k, v = project(torch.randint(0, 40, (tokens,), generator=g, device="cuda"))
    cu = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
    prompt_out, _ = memory.prompt_attention(q, k, v, cu)
    m = ContextMemory(2 * tokens + 4 * budget + 64 * steps)
    m.append(k, v)
    # the weights of the prompt's last tokens say what is worth keeping
    for i in range(tokens - 32, tokens):
        m.attend(q[i])
    m.evict(budget, recent=64)
    all_k, all_v = [k], [v]
    errors = {"cache": 0.0, "cache and index": 0.0}
    for step in range(steps):
        topic = torch.randint(0, 40, (1,), generator=g, device="cuda")
        q1, k1, v1 = project(topic)
        all_k.append(k1), all_v.append(v1)
        m.append(k1, v1)
        near, near_lse = m.attend(q1[0])
        far, far_lse = m.recall(q1[0], found)
        out, _ = memory.merge((near, far), (near_lse, far_lse))
        # everything, in 32 bits
        keys, values = torch.cat(all_k).float(), torch.cat(all_v).float()
        s = torch.einsum("hgd,thd->hgt", q1[0].float().view(HEADS, GROUP, DIM), keys) * DIM ** -0.5
        want = torch.einsum("hgt,thd->hgd", torch.softmax(s, 2), values).reshape(HEADS * GROUP, DIM)
        for name, got in (("cache", near), ("cache and index", out)):
            errors[name] += float((got.float() - want).norm() / want.norm()) / steps
    flags = memory.take_errors()
    m.close()
    return {"prompt": prompt_out, "errors": errors, "evicted": sum(int(a.gone.shape[1]) for a in m.archives), "flags": flags}


if __name__ == "__main__":
    r = run()
    print(f"{r['evicted']} tokens a head evicted to the index; error of the attention's output against all tokens:")
    for name, e in r["errors"].items():
        print(f"  {name}: {e:.3f}")
