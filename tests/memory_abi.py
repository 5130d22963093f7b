"""The token-memory entries of include/bsearch.h as ctypes sees them (the C
ABI without the Python binding)."""
import ctypes

from beam_search_collab_b200 import lib

_vp, _i32, _u32, _i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_uint32, ctypes.c_int64


class _Cache(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("num_blocks", _u32), ("kv_heads", _i32),
                ("block", _i32), ("dim", _i32)]


class _Prompt(ctypes.Structure):
    _fields_ = [("q", _vp), ("k", _vp), ("v", _vp), ("out", _vp), ("lse", _vp), ("q_stride", _i64 * 2),
                ("k_stride", _i64 * 2), ("v_stride", _i64 * 2), ("cu_q", _vp), ("cu_k", _vp),
                ("workspace", _vp), ("workspace_bytes", ctypes.c_size_t), ("total_q", _u32),
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


class _Rotate(ctypes.Structure):
    _fields_ = [("q", _vp), ("k", _vp), ("out_q", _vp), ("out_k", _vp), ("q_stride", _i64 * 2), ("k_stride", _i64 * 2),
                ("q_weight", _vp), ("k_weight", _vp), ("positions", _vp), ("freqs", _vp), ("total", _u32), ("q_heads", _i32),
                ("kv_heads", _i32), ("dim", _i32), ("rotary", _i32), ("interleaved", _i32), ("dtype", _i32),
                ("weight_dtype", _i32), ("eps", ctypes.c_float), ("amplitude", ctypes.c_float)]


class _Bounds(ctypes.Structure):
    _fields_ = [("bounds", _vp), ("table", _vp), ("lens", _vp), ("num_seqs", _u32), ("table_width", _u32), ("last", _i32)]


class _Choice(ctypes.Structure):
    _fields_ = [("q", _vp), ("q_stride", _i64 * 3), ("bounds", _vp), ("table", _vp), ("lens", _vp), ("blocks", _vp),
                ("num_seqs", _u32), ("table_width", _u32), ("queries", _i32), ("q_heads", _i32), ("count", _i32),
                ("sinks", _i32), ("recent", _i32), ("dtype", _i32)]


class _Blocks(ctypes.Structure):
    _fields_ = [("q", _vp), ("q_stride", _i64 * 3), ("table", _vp), ("lens", _vp), ("blocks", _vp), ("out", _vp), ("lse", _vp),
                ("num_seqs", _u32), ("table_width", _u32), ("queries", _i32), ("q_heads", _i32), ("count", _i32),
                ("dtype", _i32), ("scale", ctypes.c_float)]


class _Shared(ctypes.Structure):
    _fields_ = [("q", _vp), ("q_stride", _i64 * 3), ("shared_table", _vp), ("shared_lens", _vp), ("cu", _vp), ("table", _vp),
                ("lens", _vp), ("out", _vp), ("lse", _vp), ("workspace", _vp), ("workspace_bytes", ctypes.c_size_t),
                ("num_seqs", _u32), ("num_groups", _u32), ("shared_width", _u32), ("table_width", _u32), ("queries", _i32),
                ("q_heads", _i32), ("dtype", _i32), ("scale", ctypes.c_float)]


_ready = None


def _lib():
    """The library with the token-memory entries' argument types set (once)."""
    global _ready
    if _ready is None:
        L = lib()
        P = ctypes.POINTER
        for name, args in (("bs_prompt_attention", [P(_Prompt), _vp]),
                           ("bs_prompt_attention_workspace", [P(_Prompt), P(ctypes.c_size_t)]),
                           ("bs_cache_write", [P(_Cache), P(_Write), _vp]),
                           ("bs_cache_read", [P(_Cache), P(_Read), _vp]),
                           ("bs_cache_attention", [P(_Cache), P(_Attention), _vp]),
                           ("bs_cache_attention_workspace", [P(_Cache), P(_Attention), P(ctypes.c_size_t)]),
                           ("bs_cache_evict", [P(_Cache), P(_Evict), _vp]),
                           ("bs_cache_evict_workspace", [P(_Cache), P(_Evict), P(ctypes.c_size_t)]),
                           ("bs_norm_rotate", [P(_Rotate), _vp]),
                           ("bs_block_bounds", [P(_Cache), P(_Bounds), _vp]),
                           ("bs_block_choice", [P(_Cache), P(_Choice), _vp]),
                           ("bs_block_attention", [P(_Cache), P(_Blocks), _vp]),
                           ("bs_shared_attention", [P(_Cache), P(_Shared), _vp]),
                           ("bs_shared_attention_workspace", [P(_Cache), P(_Shared), P(ctypes.c_size_t)]),
                           ("bs_memory_take_errors", [_vp, P(_u32)])):
            f = getattr(L, name)
            f.argtypes, f.restype = args, ctypes.c_int
        _ready = L
    return _ready
