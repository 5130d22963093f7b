"""Token memory: attention of a language model whose context is searched.

Keys and values of the tokens a model has read live in an 8-bit cache on the
GPU (blocks of tokens, one scale per block and head).  Tokens that the cache
gives up are rows for an :class:`Index`, found again by its search.

    from beam_search_collab_b200 import memory
    out, _ = memory.prompt_attention(q, k, v, cu)             # a packed batch of prompts
    cache = memory.TokenCache.empty(num_blocks, kv_heads, dim, block=64)
    cache.write(k, v, cu, table, start)                       # its keys and values, quantised
    out, lse, mass = cache.attention(q1, table, lens, mass=mass, with_mass=True)   # one new token each
    kept, lens, mass = cache.evict(mass, table, lens, new_table, budget)
    keys, values = cache.read(old_table, old_lens, positions)  # float rows for Index.from_vectors

Everything is a CUDA tensor; calls are asynchronous on `stream` (default: the
current stream of the tensors' device) and never wait for the lengths, tables
and positions, which stay on the device.  What only the device can see to be
wrong is skipped and sets a bit that :func:`take_errors` returns.  There are no
gradients: a backward pass that reaches an output raises, and what is written
to a cache is cut off from the pass that made it.  C entries:
bs_prompt_attention, bs_cache_* of include/bsearch.h.
"""
from __future__ import annotations

import math
import os

import torch

from . import PKG, BSearchError, lib

if not os.path.exists(os.path.join(PKG, "_memory.so")):
    raise FileNotFoundError(f"{PKG}/_memory.so is missing: run `python -m beam_search_collab_b200.build`")
lib()
from . import _memory  # noqa: E402

_memory.set_error(BSearchError)


def prompt_attention(q, k, v, cu_q, cu_k=None, *, causal=True, scale=None, with_lse=False, stream=None):
    """Attention of a packed batch of prompts (bs_prompt_attention).

    q [total_q, q_heads, dim], k and v [total_k, kv_heads, dim], float16 or
    bfloat16, any token and head strides that are positive multiples of 8
    elements (no broadcast tensors).
    cu_q and cu_k (default: cu_q), int32 [sequences + 1]: where each sequence
    begins.  With `causal` a sequence's last query sees all its keys and each
    earlier query one fewer.  scale defaults to dim ** -0.5.  Returns (out,
    lse): out like q, contiguous; lse float32 [total_q, q_heads] or None."""
    return _memory.prompt_attention(q, k, v, cu_q, cu_k, causal, scale, with_lse, stream)


class TokenCache(_memory.Cache):
    """Keys and values in 8 bits: blocks of tokens, one scale per block and
    head.  Which blocks are whose is the caller's affair: every method takes a
    table int32 [sequences, width] whose row b lists sequence b's blocks in
    order (entries past its last block are not read).

    TokenCache(k, v, k_scale, v_scale) is a cache over tensors that exist: k, v
    int8 [blocks, kv_heads, block, dim], k_scale, v_scale float32 [blocks,
    kv_heads], all contiguous; they are its attributes."""

    @classmethod
    def empty(cls, num_blocks, kv_heads, dim, block=64, device=0):
        """A cache of zeros."""
        dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        codes = [torch.zeros((num_blocks, kv_heads, block, dim), dtype=torch.int8, device=dev) for _ in range(2)]
        scales = [torch.zeros((num_blocks, kv_heads), dtype=torch.float32, device=dev) for _ in range(2)]
        return cls(*codes, *scales)

    @property
    def block(self) -> int:
        return self.k.shape[2]

    def write(self, k, v, cu, table, start, *, stream=None):
        """Appends rows cu[b] .. cu[b + 1] of k and v [tokens, kv_heads, dim]
        to sequence b as positions start[b], start[b] + 1, ... (bs_cache_write:
        how scales come about)."""
        self._write(k, v, cu, table, start, stream)

    def read(self, table, lens, positions, *, dtype=torch.float32, keys=True, values=True, stream=None):
        """(keys, values) [sequences, kv_heads, n, dim] at positions int32
        [sequences, n], or [sequences, kv_heads, n] (any strides but the last);
        zeros where a position is negative or not below lens[b]."""
        return self._read(table, lens, positions, dtype, keys, values, stream)

    def attention(self, q, table, lens, *, scale=None, with_lse=False, mass=None, with_mass=False, out_mass=None,
                  stream=None):
        """Attention of each sequence's last tokens over its cached ones
        (bs_cache_attention).  q [sequences, queries, q_heads, dim]; the cache
        holds lens[b] tokens of sequence b, those of the queries included.

        Returns (out, lse, mass): out like q, contiguous; lse float32
        [sequences, queries, q_heads] or None; mass float32 [sequences,
        kv_heads, width]: the weight each token got, added to `mass` where that
        is given (into `out_mass` where that is given, which may be `mass`),
        or None without with_mass, mass and out_mass."""
        return self._attention(q, table, lens, scale, with_lse, mass, with_mass, out_mass, stream)

    def evict(self, mass, table, lens, new_table, budget, *, sinks=4, recent=0, stream=None):
        """Cuts every sequence down to `budget` tokens for each head: the first
        `sinks`, the last `recent` and of the rest those with the largest mass
        (bs_cache_evict).  They move into the blocks of new_table, none of them
        in use.  Returns (kept, new_lens, new_mass): kept int32 and new_mass
        float32 [sequences, kv_heads, budget], -1 and 0 past the end."""
        return self._evict(mass, table, lens, new_table, budget, sinks, recent, stream)


def take_errors(device=None, stream=None) -> int:
    """Error bits of the token-memory kernels on `device` (default: the
    current one) since the last call, then cleared (bs_memory_take_errors);
    waits for `stream`.  0: none; 1 a wait gave up, 2 a block id outside the
    cache, 4 lengths outside their buffers."""
    if not isinstance(device, int):
        device = None if device is None else torch.device(device).index
        device = torch.cuda.current_device() if device is None else device
    return _memory.take_errors(device, stream)


def merge(outs, lses):
    """Joins attentions of the same queries over disjoint sets of tokens: the
    outputs [..., dim] and their lse [...] as one (out, lse)."""
    top = torch.stack(list(lses)).amax(0)
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    weights = [torch.exp(x - base) for x in lses]
    total = sum(weights)
    out = sum(o.float() * w[..., None] for o, w in zip(outs, weights)) / torch.where(total > 0, total, torch.ones_like(total))[..., None]
    return out.to(outs[0].dtype), torch.log(total) + base
