"""Token memory: attention of a language model whose context is searched.

Keys and values of the tokens a model has read live in an 8-bit cache on the
GPU (blocks of tokens, one scale per block and head).  Tokens that the cache
gives up are rows for an :class:`Index`, found again by its search.

    from beam_search_collab_b200 import memory
    out, _ = memory.prompt_attention(q, k, v, cu)             # a packed batch of prompts
    cache = memory.TokenCache.empty(num_blocks, kv_heads, dim, block=64)
    cache.write(k, v, cu, table, start)                       # its keys and values, quantised
    q1, k1 = memory.norm_rotate(q1, k1, positions, freqs, q_weight=w, k_weight=w)  # of one new token each
    q1 = q1[:, None]                                           # [sequences, queries, heads, dim]
    out, lse, mass = cache.attention(q1, table, lens, mass=mass, with_mass=True)
    blocks = cache.choose_blocks(q1, cache.update_bounds(bounds, table, lens), table, lens, count)
    out, lse = cache.block_attention(q1, table, lens, blocks)                      # or over a part of its cache
    out, lse = cache.shared_attention(q1, shared_table, shared_lens, groups, table, lens)   # or with a shared beginning
    kept, lens, mass = cache.evict(mass, table, lens, new_table, budget)
    keys, values = cache.read(old_table, old_lens, found)      # float rows for Index.from_vectors

Everything is a CUDA tensor; calls are asynchronous on `stream` (default: the
current stream of the tensors' device) and never wait for the lengths, tables
and positions, which stay on the device.  What only the device can see to be
wrong is skipped and sets a bit that :func:`take_errors` returns.  There are no
gradients: a backward pass that reaches an output raises, and what is written
to a cache is cut off from the pass that made it.  C entries: from bs_dtype
on in include/bsearch.h.
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


def rotary_frequencies(rotary, base=10000.0, *, scaling=None, factor=1.0, trained=None, fast=32.0, slow=1.0, device=None):
    """(freqs, amplitude) for :func:`norm_rotate`: freqs float64 [rotary / 2],
    base ** (-2 j / rotary) radians a position, changed for contexts `factor`
    times as long as those of training:

    scaling None: not at all; "linear": positions count 1 / factor; "base":
    the base grows so that the slowest pair turns 1 / factor as fast and the
    fastest as before; "parts": pairs that turn more than `fast` times in
    `trained` positions stay, those that turn less than `slow` times count
    1 / factor, those between a mixture that is linear in their turns (a program
    that mixes linearly in the index j gets others there), and the amplitude is 0.1 log(factor) + 1."""
    if rotary < 0 or rotary % 2:
        raise ValueError("rotary must be even and not negative")
    if scaling not in (None, "linear", "base", "parts"):
        raise ValueError('scaling must be None, "linear", "base" or "parts"')
    if not factor >= 1 or not base > 1:
        raise ValueError("factor must be at least 1, base above 1")
    j = torch.arange(0, rotary, 2, dtype=torch.float64, device=device)
    if scaling == "base" and rotary > 2:
        base = base * factor ** (rotary / (rotary - 2))
    freqs = base ** (-j / max(rotary, 1))
    if scaling == "linear":
        return freqs / factor, 1.0
    if scaling != "parts":
        return freqs, 1.0
    if trained is None or not fast > slow:
        raise ValueError('"parts" needs `trained`, the positions of training, and fast above slow')
    stay = ((trained * freqs / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
    return freqs * (stay + (1 - stay) / factor), 0.1 * math.log(factor) + 1


def norm_rotate(q, k, positions=None, freqs=None, *, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, amplitude=1.0, stream=None):
    """Norm of queries and keys for each head, then their rotary position, in
    one pass (bs_norm_rotate).

    q [tokens, q_heads, dim] and k [tokens, kv_heads, dim] (or None), float16
    or bfloat16, any token and head strides that are multiples of 8 elements
    (slices of one projection's output, for instance).  A head is divided by
    the root of its mean square and multiplied by q_weight or k_weight [dim]
    where that is given.  Then its first 2 * len(freqs) dimensions are rotated
    by positions (int32 [tokens], any sign) times freqs (float64, radians a
    position; None: no rotation, and positions may be None): pairs are the first and second half's j-th
    dimensions, or with `interleaved` neighbours; `amplitude` multiplies sines
    and cosines (:func:`rotary_frequencies` gives both).  Returns (q, k),
    contiguous."""
    return _memory.norm_rotate(q, k, positions, freqs, q_weight, k_weight, eps, interleaved, amplitude, stream)


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

    def empty_bounds(self):
        """Bounds of this cache's blocks, int8 [blocks, kv_heads, 2, dim], none known yet."""
        blocks, heads, _, dim = self.k.shape
        return torch.zeros((blocks, heads, 2, dim), dtype=torch.int8, device=self.k.device)

    def update_bounds(self, bounds, table, lens, *, last=None, stream=None):
        """Largest and smallest key code of each dimension (bs_block_bounds), into
        `bounds`, for the blocks that hold any of the last `last` tokens of a
        sequence (None: all its blocks); to be called when they have changed.
        Returns bounds."""
        self._update_bounds(bounds, table, lens, last, stream)
        return bounds

    def choose_blocks(self, q, bounds, table, lens, count, *, sinks=1, recent=1, stream=None):
        """Which `count` blocks each query and key head attends to
        (bs_block_choice: the first `sinks`, the last `recent`, and those that
        may hold the largest scores by their bounds).  q [sequences, queries,
        q_heads, dim] as in :meth:`attention`.  Returns int32 [sequences,
        queries, kv_heads, count]: columns of the table, ascending, -1 past
        the end."""
        return self._choose_blocks(q, bounds, table, lens, count, sinks, recent, stream)

    def block_attention(self, q, table, lens, blocks, *, scale=None, with_lse=False, stream=None):
        """Attention of each sequence's last tokens over chosen blocks of its cache
        (bs_block_attention): blocks int32 [sequences, queries, kv_heads,
        count], columns of the table in any order, negative ones skipped.
        Returns (out, lse) like :meth:`attention`."""
        return self._block_attention(q, table, lens, blocks, scale, with_lse, stream)

    def shared_attention(self, q, shared_table, shared_lens, cu, table, lens, *, scale=None, with_lse=False, stream=None):
        """Attention of sequences that begin with the same tokens
        (bs_shared_attention).  Sequences cu[m] .. cu[m + 1] (int32 [groups +
        1]) begin with the shared_lens[m] tokens of shared_table[m] (int32
        [groups, width]), which are read once for many query rows where sequences
        and shared tokens are many, by each sequence where they are few; table
        and lens are of what each has beyond those.  Returns (out, lse) like
        :meth:`attention`, over both."""
        return self._shared_attention(q, shared_table, shared_lens, cu, table, lens, scale, with_lse, stream)

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
