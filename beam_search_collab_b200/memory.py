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
wrong is skipped and sets a bit that :func:`take_errors` returns.  C entries:
bs_prompt_attention, bs_cache_* of include/bsearch.h.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _check, lib

_vp, _i32, _u32, _i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_uint32, ctypes.c_int64
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class _Cache(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("num_blocks", _u32), ("kv_heads", _i32),
                ("block", _i32), ("dim", _i32)]


class _Prompt(ctypes.Structure):
    _fields_ = [("q", _vp), ("k", _vp), ("v", _vp), ("out", _vp), ("lse", _vp), ("q_stride", _i64 * 2),
                ("k_stride", _i64 * 2), ("v_stride", _i64 * 2), ("cu_q", _vp), ("cu_k", _vp), ("total_q", _u32),
                ("total_k", _u32), ("num_seqs", _u32), ("q_heads", _i32), ("kv_heads", _i32), ("dim", _i32),
                ("dtype", _i32), ("causal", _i32), ("scale", ctypes.c_float)]


class _Write(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("k_stride", _i64 * 2), ("v_stride", _i64 * 2), ("cu", _vp), ("table", _vp),
                ("start", _vp), ("total", _u32), ("num_seqs", _u32), ("table_width", _u32), ("dtype", _i32)]


class _Read(ctypes.Structure):
    _fields_ = [("table", _vp), ("lens", _vp), ("positions", _vp), ("position_seq_stride", _i64),
                ("position_head_stride", _i64), ("k", _vp), ("v", _vp), ("num_seqs", _u32), ("table_width", _u32),
                ("count", _u32), ("dtype", _i32)]


class _Attention(ctypes.Structure):
    _fields_ = [("q", _vp), ("q_stride", _i64 * 3), ("table", _vp), ("lens", _vp), ("out", _vp), ("lse", _vp),
                ("mass", _vp), ("out_mass", _vp), ("workspace", _vp), ("workspace_bytes", ctypes.c_size_t),
                ("num_seqs", _u32), ("table_width", _u32), ("mass_width", _u32), ("queries", _i32), ("q_heads", _i32),
                ("dtype", _i32), ("scale", ctypes.c_float)]


class _Evict(ctypes.Structure):
    _fields_ = [("mass", _vp), ("table", _vp), ("lens", _vp), ("new_table", _vp), ("kept", _vp), ("new_lens", _vp),
                ("new_mass", _vp), ("workspace", _vp), ("workspace_bytes", ctypes.c_size_t), ("num_seqs", _u32),
                ("table_width", _u32), ("new_table_width", _u32), ("mass_width", _u32), ("budget", _i32),
                ("sinks", _i32), ("recent", _i32)]


_ready = None


def _lib():
    """The library with the token-memory entries' argument types set (once)."""
    global _ready
    if _ready is None:
        L = lib()
        P = ctypes.POINTER
        for name, args in (("bs_prompt_attention", [P(_Prompt), _vp]),
                           ("bs_cache_write", [P(_Cache), P(_Write), _vp]),
                           ("bs_cache_read", [P(_Cache), P(_Read), _vp]),
                           ("bs_cache_attention", [P(_Cache), P(_Attention), _vp]),
                           ("bs_cache_attention_workspace", [P(_Cache), P(_Attention), P(ctypes.c_size_t)]),
                           ("bs_cache_evict", [P(_Cache), P(_Evict), _vp]),
                           ("bs_cache_evict_workspace", [P(_Cache), P(_Evict), P(ctypes.c_size_t)]),
                           ("bs_memory_take_errors", [_vp, P(_u32)])):
            f = getattr(L, name)
            f.argtypes, f.restype = args, ctypes.c_int
        _ready = L
    return _ready


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _call(device, stream, outputs, launch):
    """launch(stream handle) with `device` current; outputs made for the
    current stream are marked as used on `stream` when that is another one."""
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _call(device, stream, outputs, launch)
    here = torch._C._cuda_getCurrentRawStream(device.index)
    to = here if stream is None else int(stream)
    _check(launch(to))
    if to != here:
        s = torch.cuda.ExternalStream(to, device=device) if to else torch.cuda.default_stream(device)
        for t in outputs:
            if t is not None:
                t.record_stream(s)


def _index(t, shape, name, device):
    _need(t.dtype == torch.int32 and t.is_contiguous() and t.device == device and tuple(t.shape) == shape,
          f"{name} must be a contiguous int32 tensor of shape {list(shape)} on {device}")
    return t.data_ptr()


def _rows(t, name, like=None):
    """A [tokens, heads, dim] tensor whose last dimension is contiguous."""
    _need(t.is_cuda and t.dim() == 3 and t.stride(2) == 1, f"{name} must be a CUDA tensor [tokens, heads, dim], last dimension contiguous")
    _need(t.dtype in (torch.float16, torch.bfloat16), f"{name} must be float16 or bfloat16")
    if like is not None:
        _need(t.dtype == like.dtype and t.device == like.device and t.shape[2] == like.shape[2],
              f"{name} must have the type, device and last dimension of the others")
    return t.data_ptr()


def _strides(t):
    # a stride that is never multiplied by anything but 0 may be anything: 0
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]))


def prompt_attention(q, k, v, cu_q, cu_k=None, *, causal=True, scale=None, with_lse=False, stream=None):
    """Attention of a packed batch of prompts (bs_prompt_attention).

    q [total_q, q_heads, dim], k and v [total_k, kv_heads, dim], float16 or
    bfloat16, any token and head strides that are multiples of 8 elements.
    cu_q and cu_k (default: cu_q), int32 [sequences + 1]: where each sequence
    begins.  With `causal` a sequence's last query sees all its keys and each
    earlier query one fewer.  scale defaults to dim ** -0.5.  Returns (out,
    lse): out like q, contiguous; lse float32 [total_q, q_heads] or None."""
    qp, kp, vp = _rows(q, "q"), _rows(k, "k", q), _rows(v, "v", q)
    _need(k.shape == v.shape, "k and v must have the same shape")
    if cu_k is None:
        _need(q.shape[0] == k.shape[0], "cu_k is needed when q and k have different numbers of rows")
        cu_k = cu_q
    n = cu_q.numel() - 1
    _need(n >= 0, "cu_q must have at least one entry")
    d = _Prompt(qp, kp, vp, None, None, _strides(q), _strides(k), _strides(v), _index(cu_q, (n + 1,), "cu_q", q.device),
                _index(cu_k, (n + 1,), "cu_k", q.device), q.shape[0], k.shape[0], n, q.shape[1], k.shape[1], q.shape[2],
                _TYPES[q.dtype], bool(causal), q.shape[2] ** -0.5 if scale is None else scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if with_lse else None
    d.out, d.lse = out.data_ptr(), lse.data_ptr() if with_lse else None
    _call(q.device, stream, (out, lse), lambda s: _lib().bs_prompt_attention(d, s))
    return out, lse


class TokenCache:
    """Keys and values in 8 bits: blocks of tokens, one scale per block and
    head.  Which blocks are whose is the caller's affair: every method takes a
    table int32 [sequences, width] whose row b lists sequence b's blocks in
    order (entries past its last block are not read)."""

    def __init__(self, k, v, k_scale, v_scale):
        """A cache over tensors that exist: k, v int8 [blocks, kv_heads, block,
        dim], k_scale, v_scale float32 [blocks, kv_heads], all contiguous."""
        _need(k.is_cuda and k.dim() == 4 and k.dtype == torch.int8 and k.is_contiguous(),
              "k must be a contiguous CUDA int8 tensor [blocks, kv_heads, block, dim]")
        _need(v.shape == k.shape and v.dtype == k.dtype and v.device == k.device and v.is_contiguous(), "v must be like k")
        for s in (k_scale, v_scale):
            _need(s.shape == k.shape[:2] and s.dtype == torch.float32 and s.device == k.device and s.is_contiguous(),
                  "scales must be contiguous float32 tensors [blocks, kv_heads]")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self._c = _Cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *k.shape)

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
        kp, vp = _rows(k, "k"), _rows(v, "v", k)
        _need(k.shape == v.shape and k.shape[1:] == (self.k.shape[1], self.k.shape[3]) and k.device == self.k.device,
              "k and v must be [tokens, kv_heads, dim] of the cache, on its device")
        _need(table.dim() == 2, "table must be [sequences, width]")
        n, width = table.shape
        d = _Write(kp, vp, _strides(k), _strides(v), _index(cu, (n + 1,), "cu", k.device),
                   _index(table, (n, width), "table", k.device), _index(start, (n,), "start", k.device), k.shape[0], n, width,
                   _TYPES[k.dtype])
        _call(k.device, stream, (), lambda s: _lib().bs_cache_write(self._c, d, s))

    def read(self, table, lens, positions, *, dtype=torch.float32, keys=True, values=True, stream=None):
        """(keys, values) [sequences, kv_heads, n, dim] at positions int32
        [sequences, n], or [sequences, kv_heads, n] (any strides but the last);
        zeros where a position is negative or not below lens[b]."""
        dev = self.k.device
        n, width = table.shape
        heads = self.k.shape[1]
        _need(dtype in _TYPES, "dtype must be float32, float16 or bfloat16")
        _need(positions.dtype == torch.int32 and positions.device == dev and positions.dim() in (2, 3)
              and positions.shape[0] == n and (positions.dim() == 2 or positions.shape[1] == heads)
              and (positions.stride(-1) == 1 or positions.shape[-1] <= 1),
              "positions must be int32 [sequences, n] or [sequences, kv_heads, n]")
        count = positions.shape[-1]
        shape = (n, heads, count, self.k.shape[3])
        k = torch.empty(shape, dtype=dtype, device=dev) if keys else None
        v = torch.empty(shape, dtype=dtype, device=dev) if values else None
        d = _Read(_index(table, (n, width), "table", dev), _index(lens, (n,), "lens", dev), positions.data_ptr(),
                  positions.stride(0), positions.stride(1) if positions.dim() == 3 else 0,
                  k.data_ptr() if keys else None, v.data_ptr() if values else None, n, width, count, _TYPES[dtype])
        _call(dev, stream, (k, v), lambda s: _lib().bs_cache_read(self._c, d, s))
        return k, v

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
        dev = self.k.device
        _need(q.dim() == 4 and q.device == dev and q.stride(3) == 1 and q.dtype in (torch.float16, torch.bfloat16)
              and q.shape[3] == self.k.shape[3],
              "q must be float16 or bfloat16 [sequences, queries, q_heads, dim] on the cache's device, last dimension contiguous")
        n, width = table.shape
        _need(q.shape[0] == n, "q and table must have the same number of sequences")
        d = _Attention(q.data_ptr(), _strides(q), _index(table, (n, width), "table", dev), _index(lens, (n,), "lens", dev),
                       num_seqs=n, table_width=width, queries=q.shape[1], q_heads=q.shape[2], dtype=_TYPES[q.dtype],
                       scale=q.shape[3] ** -0.5 if scale is None else scale)
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device=dev) if with_lse else None
        if mass is None and out_mass is None and with_mass:
            out_mass = torch.empty((n, self.k.shape[1], width * self.block), dtype=torch.float32, device=dev)
        elif mass is not None and out_mass is None:
            out_mass = torch.empty_like(mass, memory_format=torch.contiguous_format)
        for m in (mass, out_mass):
            if m is not None:
                _need(m.dtype == torch.float32 and m.device == dev and m.dim() == 3 and m.is_contiguous()
                      and m.shape == out_mass.shape and m.shape[:2] == (n, self.k.shape[1]),
                      "mass must be contiguous float32 [sequences, kv_heads, width]")
        d.out, d.lse = out.data_ptr(), lse.data_ptr() if with_lse else None
        if out_mass is not None:
            d.out_mass, d.mass_width = out_mass.data_ptr(), out_mass.shape[2]
            d.mass = mass.data_ptr() if mass is not None else None
        work = self._workspace(_lib().bs_cache_attention_workspace, d)
        _call(dev, stream, (out, lse, out_mass, work), lambda s: _lib().bs_cache_attention(self._c, d, s))
        return out, lse, out_mass

    def evict(self, mass, table, lens, new_table, budget, *, sinks=4, recent=0, stream=None):
        """Cuts every sequence down to `budget` tokens for each head: the first
        `sinks`, the last `recent` and of the rest those with the largest mass
        (bs_cache_evict).  They move into the blocks of new_table, none of them
        in use.  Returns (kept, new_lens, new_mass): kept int32 and new_mass
        float32 [sequences, kv_heads, budget], -1 and 0 past the end."""
        dev = self.k.device
        n, width = table.shape
        heads = self.k.shape[1]
        _need(mass.dtype == torch.float32 and mass.device == dev and mass.is_contiguous() and mass.dim() == 3
              and mass.shape[:2] == (n, heads), "mass must be contiguous float32 [sequences, kv_heads, width]")
        _need(new_table.dim() == 2, "new_table must be [sequences, width]")
        _need(budget > 0, "budget must be positive")
        kept = torch.empty((n, heads, budget), dtype=torch.int32, device=dev)
        new_mass = torch.empty((n, heads, budget), dtype=torch.float32, device=dev)
        new_lens = torch.empty(n, dtype=torch.int32, device=dev)
        d = _Evict(mass.data_ptr(), _index(table, (n, width), "table", dev), _index(lens, (n,), "lens", dev),
                   _index(new_table, (n, new_table.shape[1]), "new_table", dev), kept.data_ptr(), new_lens.data_ptr(),
                   new_mass.data_ptr(), None, 0, n, width, new_table.shape[1], mass.shape[2], budget, sinks, recent)
        work = self._workspace(_lib().bs_cache_evict_workspace, d)
        _call(dev, stream, (kept, new_lens, new_mass, work), lambda s: _lib().bs_cache_evict(self._c, d, s))
        return kept, new_lens, new_mass

    def _workspace(self, size, d):
        bytes_ = ctypes.c_size_t()
        dev = self.k.device
        if torch.cuda.current_device() != dev.index:
            with torch.cuda.device(dev):
                _check(size(self._c, d, ctypes.byref(bytes_)))
        else:
            _check(size(self._c, d, ctypes.byref(bytes_)))
        if not bytes_.value:
            return None
        work = torch.empty(bytes_.value, dtype=torch.uint8, device=dev)
        d.workspace, d.workspace_bytes = work.data_ptr(), bytes_.value
        return work


def take_errors(device=None, stream=None) -> int:
    """Error bits of the token-memory kernels on `device` since the last call,
    then cleared (bs_memory_take_errors); waits for `stream`.  0: none; 1 a
    wait gave up, 2 a block id outside the cache, 4 lengths outside their
    buffers."""
    flags = _u32()
    with torch.cuda.device(device):
        s = torch.cuda.current_stream().cuda_stream if stream is None else int(stream)
        _check(_lib().bs_memory_take_errors(s, ctypes.byref(flags)))
    return flags.value


def merge(outs, lses):
    """Joins attentions of the same queries over disjoint sets of tokens: the
    outputs [..., dim] and their lse [...] as one (out, lse)."""
    top = torch.stack(list(lses)).amax(0)
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    weights = [torch.exp(x - base) for x in lses]
    total = sum(weights)
    out = sum(o.float() * w[..., None] for o, w in zip(outs, weights)) / torch.where(total > 0, total, torch.ones_like(total))[..., None]
    return out.to(outs[0].dtype), torch.log(total) + base
