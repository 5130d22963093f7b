"""CPU: the token-memory entries' checks that need no GPU, and the 64-bit
definitions that the GPU tests go by against an independent formulation."""
import ctypes
import math

import pytest
import torch

import beam_search_collab_b200 as B
import memory_abi as A
import memory_ref as R
from beam_search_collab_b200 import memory as M


def cache(**kw):
    c = A._Cache(64, 64, 64, 64, 4, 2, 32, 64)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def status(name, *args):
    rc = getattr(A._lib(), name)(*args)
    return rc, B.lib().bs_last_error().decode()


def test_null_descriptors():
    c = cache()
    for name in ("bs_cache_write", "bs_cache_read", "bs_cache_attention", "bs_cache_evict"):
        assert status(name, c, None, None) == (1, "desc is NULL")
    assert status("bs_prompt_attention", None, None) == (1, "desc is NULL")
    assert status("bs_cache_read", None, A._Read(), None) == (1, "cache is NULL")
    assert status("bs_memory_take_errors", None, None)[0] == 1
    assert status("bs_cache_evict_workspace", c, A._Evict(), None)[0] == 1


@pytest.mark.parametrize("field,value,code,text", [
    ("dtype", 0, 1, "BS_F16 or BS_BF16"), ("dim", 0, 1, "positive"), ("dim", 24, 2, "multiple of 16"), ("dim", 144, 2, "up to 128"),
    ("q_heads", 3, 1, "multiple of kv_heads"), ("kv_heads", 0, 1, "multiple of kv_heads"), ("q_heads", 258, 2, "128 query heads"),
    ("scale", math.nan, 1, "NaN"), ("total_k", 1 << 30, 2, "2^30"), ("num_seqs", 65536, 2, "65535"), ("cu_q", None, 1, "NULL"),
    ("out", None, 1, "NULL"), ("k", 72, 1, "16-byte aligned"), ("q_stride", (4, 64), 1, "multiples of 8"),
    ("v_stride", (-8, 64), 1, "non-negative")])
def test_prompt_checks(field, value, code, text):
    d = A._Prompt(64, 64, 64, 64, 64, (128, 64), (128, 64), (128, 64), 64, 64, None, 0, 10, 10, 1, 2, 2, 64, 1, 1,
                  0.1)
    setattr(d, field, (ctypes.c_int64 * 2)(*value) if isinstance(value, tuple) else value)
    rc, why = status("bs_prompt_attention", d, None)
    assert rc == code and text in why, (rc, why)


@pytest.mark.parametrize("field,value,code,text", [("block", 24, 1, "16, 32, 64 or 128"), ("dim", 40, 2, "multiple of 16"),
                                                   ("kv_heads", 0, 1, "kv_heads"), ("kv_heads", 70000, 1, "kv_heads")])
def test_cache_checks(field, value, code, text):
    d = A._Read(64, 64, 64, 0, 0, 64, 64, 1, 1, 1, 0)
    rc, why = status("bs_cache_read", cache(**{field: value}), d, None)
    assert rc == code and text in why, (rc, why)


@pytest.mark.parametrize("field,value,code,text", [
    ("queries", 0, 1, "queries"), ("queries", 1025, 1, "queries"), ("q_heads", 5, 1, "multiple"), ("dtype", 0, 1, "BS_F16"),
    ("table_width", 1 << 26, 2, "2^30"), ("lens", None, 1, "NULL"), ("out_mass", None, 1, "mass without out_mass"),
    ("mass_width", 0, 1, "mass_width is 0"), ("scale", math.nan, 1, "NaN"), ("q", 65, 1, "aligned")])
def test_attention_checks(field, value, code, text):
    d = A._Attention(64, (256, 256, 64), 64, 64, 64, 64, 64, 64, None, 0, 1, 2, 64, 1, 4, 1, 0.1)
    setattr(d, field, value)
    rc, why = status("bs_cache_attention", cache(), d, None)
    assert rc == code and text in why, (rc, why)


@pytest.mark.parametrize("field,value,code,text", [
    ("budget", 0, 1, "budget"), ("sinks", -1, 1, "sinks"), ("recent", 30, 1, "sinks + recent"), ("new_table_width", 0, 1, "room"),
    ("mass_width", 1 << 30, 2, "mass_width"), ("kept", None, 1, "NULL")])
def test_evict_checks(field, value, code, text):
    d = A._Evict(64, 64, 64, 64, 64, 64, 64, None, 0, 1, 4, 1, 128, 32, 4, 8)
    setattr(d, field, value)
    rc, why = status("bs_cache_evict", cache(), d, None)
    assert rc == code and text in why, (rc, why)


def test_nothing_to_do_is_done_without_a_gpu():
    d = A._Prompt(None, None, None, None, None, (0, 0), (0, 0), (0, 0), None, None, None, 0, 0, 0, 0, 2, 2, 64, 1, 1, 0.1)
    assert status("bs_prompt_attention", d, None)[0] == 0
    assert status("bs_cache_write", cache(), A._Write(dtype=1), None)[0] == 0
    assert status("bs_cache_read", cache(), A._Read(dtype=1), None)[0] == 0
    assert status("bs_cache_attention", cache(), A._Attention(queries=1, q_heads=2, dtype=1, scale=1.0), None)[0] == 0


def test_host_tensors_are_refused():
    q = torch.zeros((4, 2, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        M.prompt_attention(q, q, q, torch.tensor([0, 4], dtype=torch.int32))
    codes, scales = torch.zeros((2, 2, 16, 64), dtype=torch.int8), torch.zeros((2, 2))
    with pytest.raises(ValueError, match="CUDA"):
        M.TokenCache(codes, codes, scales, scales)


def test_merge_is_the_attention_over_both_sets():
    g = torch.Generator().manual_seed(0)
    s, v = torch.randn((5, 9), generator=g, dtype=torch.float64), torch.randn((9, 4), generator=g, dtype=torch.float64)
    part = lambda a, b: (torch.softmax(s[:, a:b], 1) @ v[a:b], torch.logsumexp(s[:, a:b], 1))  # noqa: E731
    nothing = (torch.zeros((5, 4), dtype=torch.float64), torch.full((5,), -math.inf, dtype=torch.float64))
    out, lse = M.merge(*zip(part(0, 3), part(3, 9), nothing))
    assert torch.allclose(out, torch.softmax(s, 1) @ v, atol=1e-6) and torch.allclose(lse, torch.logsumexp(s, 1))
    out, lse = M.merge(*zip(nothing, nothing))
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("causal", [True, False])
def test_prompt_definition(causal):
    g = torch.Generator().manual_seed(1)
    lens_q, lens_k = [3, 0, 5], [4, 2, 2]
    q = torch.randn((8, 4, 16), generator=g, dtype=torch.float64)
    k, v = (torch.randn((8, 2, 16), generator=g, dtype=torch.float64) for _ in range(2))
    out, lse, weighted, _ = R.prompt(q, k, v, lens_q, lens_k, causal, 0.25)
    a = b = 0
    for nq, nk in zip(lens_q, lens_k):
        for i in range(nq):
            for h in range(4):
                n = max(0, nk - nq + 1 + i) if causal else nk
                s = (k[b:b + n, h // 2] * q[a + i, h]).sum(1) * 0.25
                w = torch.softmax(s, 0)
                want = (w[:, None] * v[b:b + n, h // 2]).sum(0) if n else torch.zeros(16, dtype=torch.float64)
                assert torch.allclose(out[a + i, h], want)
                assert torch.allclose(lse[a + i, h], torch.logsumexp(s, 0)) if n else lse[a + i, h] == -math.inf
        a, b = a + nq, b + nk
    assert (weighted >= out.abs() - 1e-12).all()


@pytest.mark.parametrize("device,index", [(None, 3), ("cuda", 3), (torch.device("cuda"), 3), ("cuda:1", 1), (2, 2), (torch.device("cuda", 0), 0)])
def test_take_errors_finds_its_device(device, index, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(M._memory, "take_errors", lambda device, stream: (device, stream))
    assert M.take_errors(device, 7) == (index, 7)


def test_rows_of_no_sequence_are_refused():
    # they would be left as the buffers were
    d = A._Prompt(64, 64, 64, 64, 64, (128, 64), (128, 64), (128, 64), 64, 64, None, 0, 10, 10, 0, 2, 2, 64, 1, 1, 0.1)
    rc, why = status("bs_prompt_attention", d, None)
    assert rc == 1 and "num_seqs is 0" in why
    d.total_q = 0
    assert status("bs_prompt_attention", d, None)[0] == 0


def test_kernels_wait_for_the_one_before_them_first():
    # launched under the end of the kernel before: its results, lengths among them, are not read and no
    # error bit is set before the wait
    import os
    import re
    kernels = 0
    for name in ("bs_prompt_attention.cu", "bs_cache_attention.cu", "bs_token_cache.cu"):
        with open(os.path.join(B.PKG, "csrc", name)) as f:
            text = f.read()
        for m in re.finditer(r"__global__ void[^;{]*?(k_\w+)\(", text):
            body = text[m.end():text.index("\n}\n", m.end())]
            before, wait, _ = body.partition("cudaGridDependencySynchronize();")
            assert wait, m[1]
            assert not re.search(r"held_tokens\(|count_cost\(|atomicOr\(|\bd\.\w+\[|mass\[|kept\[", before), m[1]
            kernels += 1
    assert kernels == 9


def calls():
    """A call of each entry that only lacks memory of a GPU."""
    return {"bs_prompt_attention": A._Prompt(64, 64, 64, 64, 64, (128, 64), (128, 64), (128, 64), 64, 64, None, 0, 10, 10, 1, 2, 2, 64, 1, 1, 0.1),
            "bs_cache_write": A._Write(64, 64, (128, 64), (128, 64), 64, 64, 64, 10, 1, 1, 1),
            "bs_cache_read": A._Read(64, 64, 64, 0, 0, 64, 64, 1, 1, 1, 0),
            "bs_cache_attention": A._Attention(64, (256, 256, 64), 64, 64, 64, 64, 64, 64, None, 0, 1, 2, 64, 1, 4, 1, 0.1),
            "bs_cache_evict": A._Evict(64, 64, 64, 64, 64, 64, 64, None, 0, 1, 4, 1, 128, 32, 4, 8)}


def call(name, d, **kw):
    return status(name, d, None) if name == "bs_prompt_attention" else status(name, cache(**kw), d, None)


@pytest.mark.parametrize("name,fields", [("bs_prompt_attention", "lse cu_q cu_k"), ("bs_cache_write", "cu table start"),
                                         ("bs_cache_read", "table lens positions"),
                                         ("bs_cache_attention", "table lens lse mass out_mass"),
                                         ("bs_cache_evict", "mass table lens new_table kept new_lens new_mass")])
def test_misaligned_32_bit_buffers_are_refused(name, fields):
    for field in fields.split():
        d = calls()[name]
        setattr(d, field, 66)
        rc, why = call(name, d)
        assert rc == 1 and "4-byte aligned" in why, (field, rc, why)


@pytest.mark.parametrize("name,field,value", [
    ("bs_prompt_attention", "q_stride", (1 << 36, 64)), ("bs_prompt_attention", "k_stride", (1 << 36, 64)),
    ("bs_prompt_attention", "v_stride", (1 << 36, 64)), ("bs_cache_write", "k_stride", (1 << 36, 64)),
    ("bs_cache_write", "v_stride", (1 << 36, 64)), ("bs_cache_read", "position_seq_stride", 1 << 58),
    ("bs_cache_read", "position_head_stride", 1 << 62)])
def test_strides_beyond_64_bit_addresses_are_refused(name, field, value):
    # legal by itself, but the last of 2^29 rows (or of 60,000 sequences) would be out of any address's reach
    d = calls()[name]
    for count, n in (("total_q", 1 << 29), ("total_k", 1 << 29), ("total", 1 << 29), ("num_seqs", 60000)):
        if hasattr(d, count):
            setattr(d, count, n)
    setattr(d, field, (ctypes.c_int64 * len(value))(*value) if isinstance(value, tuple) else value)
    rc, why = call(name, d)
    assert rc == 1 and "reach" in why, (rc, why)


def test_the_build_needs_no_pytorch(monkeypatch, capfd):
    import sys

    from beam_search_collab_b200 import build
    ran = []
    monkeypatch.setitem(sys.modules, "torch", None)              # import torch: ImportError
    monkeypatch.setattr(build, "_run", ran.append)
    monkeypatch.setattr(build, "_stale", lambda target, sources: target == build.MEMORY_PY)
    assert build.build() == build.LIB and not ran
    assert "memory" in capfd.readouterr().err
