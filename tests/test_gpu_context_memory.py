"""GPU: the token-memory operators and the index together, as an example program uses them."""
import os
import sys

import pytest
import torch

from beam_search_collab_b200 import memory

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def test_evicted_tokens_are_found_again():
    import context_memory
    r = context_memory.run(tokens=3000, steps=8, budget=256, found=32)
    assert r["flags"] == 0 and r["evicted"] == 3000 - 256
    assert torch.isfinite(r["prompt"].float()).all()
    # the tokens found carry most of what the cache had lost
    assert r["errors"]["cache and index"] < 0.5 * r["errors"]["cache"], r["errors"]


def test_tokens_of_every_eviction_are_recalled():
    # a query that is one evicted key, eight times as long, gets that key's value: nothing else comes near its weight
    import context_memory as C
    g = torch.Generator("cuda").manual_seed(47)
    m = C.ContextMemory(4000)
    k, v = (torch.randn((1100, C.HEADS, C.DIM), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    m.append(k[:600], v[:600])
    for n in (600, 1100):
        if n == 1100:
            m.append(k[600:], v[600:])
        m.mass = torch.linspace(1, 0, m.tokens, device="cuda").repeat(1, C.HEADS, 1).contiguous()   # the first tokens stay
        m.evict(64, recent=8)
    for at in (400, 580, 700, 1050):
        q = (8 * k[at].float()).to(torch.bfloat16).repeat_interleave(C.GROUP, 0)
        out, _ = m.recall(q, 16)
        want = v[at].float().repeat_interleave(C.GROUP, 0)
        assert (out.float() - want).abs().max() < 0.1, at       # (steps of the 8-bit codes are 0.03)
    m.close()


@pytest.mark.parametrize("tokens", [40, 64])
def test_a_cache_within_its_budget_is_left_alone(tokens):
    import context_memory as C
    g = torch.Generator("cuda").manual_seed(48)
    m = C.ContextMemory(400)
    k, v = (torch.randn((tokens, C.HEADS, C.DIM), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    m.append(k, v)
    before = m.attend(k[0].repeat_interleave(C.GROUP, 0))
    m.evict(64, recent=8)
    assert m.tokens == tokens and not m.archives
    q = k[0].repeat_interleave(C.GROUP, 0)
    assert all(torch.equal(a, b) for a, b in zip(before, m.attend(q)))
    out, lse = memory.merge(*zip(before, m.recall(q, 16)))
    assert torch.equal(out, before[0]) and torch.allclose(lse, before[1])
    m.close()
