"""CPU: the checks, without a GPU, of the token-memory entries for long and shared contexts (norm and rotary position,
block bounds, choice of blocks, attention over chosen blocks, shared attention), and the frequencies' definition."""
import math
import os
import re

import pytest
import torch

import beam_search_collab_b200 as B
import memory_abi as A
from beam_search_collab_b200 import memory as M


def cache(**kw):
    c = A._Cache(64, 64, 64, 64, 4, 2, 32, 64)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def calls():
    """A call of each entry that only lacks memory of a GPU."""
    return {"bs_norm_rotate": A._Rotate(64, 64, 64, 64, (256, 64), (128, 64), 64, 64, 64, 64, 10, 4, 2, 64, 32, 0, 1, 0, 1e-6, 1.0),
            "bs_block_bounds": A._Bounds(64, 64, 64, 2, 3, -1),
            "bs_block_choice": A._Choice(64, (256, 256, 64), 64, 64, 64, 64, 2, 3, 1, 4, 8, 1, 1, 1),
            "bs_block_attention": A._Blocks(64, (256, 256, 64), 64, 64, 64, 64, 64, 2, 3, 1, 4, 8, 1, 0.1),
            "bs_shared_attention": A._Shared(64, (256, 256, 64), 64, 64, 64, 64, 64, 64, 64, None, 0, 2, 1, 3, 3, 1, 4, 1, 0.1)}


def call(name, d, **kw):
    f = getattr(A._lib(), name)
    rc = f(d, None) if name == "bs_norm_rotate" else f(cache(**kw), d, None)
    return rc, B.lib().bs_last_error().decode()


def put(d, field, value):
    t = dict(d._fields_)[field]
    setattr(d, field, t(*value) if isinstance(value, tuple) else value)


def test_null_descriptors():
    for name in calls():
        assert call(name, None) == (1, "desc is NULL")
        if name != "bs_norm_rotate":
            f = getattr(A._lib(), name)
            assert f(None, calls()[name], None) == 1 and b"cache is NULL" in B.lib().bs_last_error()
    assert A._lib().bs_shared_attention_workspace(cache(), calls()["bs_shared_attention"], None) == 1


@pytest.mark.parametrize("field,value,code,text", [
    ("dtype", 0, 1, "BS_F16 or BS_BF16"), ("dim", 24, 2, "multiple of 16"), ("dim", 144, 2, "up to 128"), ("q_heads", -1, 1, "negative"),
    ("q_heads", 70000, 2, "65535"), ("total", 1 << 30, 2, "2^30"), ("rotary", 31, 1, "even"), ("rotary", 66, 1, "0 .. dim"),
    ("rotary", -2, 1, "0 .. dim"), ("weight_dtype", 3, 1, "weight_dtype"), ("eps", -1.0, 1, "eps"), ("eps", math.nan, 1, "eps"),
    ("amplitude", math.inf, 1, "amplitude"), ("q", None, 1, "NULL"), ("out_k", None, 1, "NULL"), ("freqs", None, 1, "NULL"),
    ("positions", None, 1, "NULL"), ("k", 72, 1, "16-byte aligned"), ("out_q", 72, 1, "16-byte aligned"),
    ("q_stride", (252, 64), 1, "multiples of 8"), ("k_stride", (-128, 64), 1, "non-negative"), ("freqs", 68, 1, "8-byte"),
    ("positions", 66, 1, "4-byte"), ("q_weight", 66, 1, "aligned to their type")])
def test_norm_rotate_checks(field, value, code, text):
    d = calls()["bs_norm_rotate"]
    put(d, field, value)
    rc, why = call("bs_norm_rotate", d)
    assert rc == code and text in why, (rc, why)


COMMON = [("queries", 0, 1, "queries"), ("queries", 1025, 1, "queries"), ("q_heads", 5, 1, "multiple"), ("dtype", 0, 1, "BS_F16"),
          ("table_width", 1 << 26, 2, "2^30"), ("num_seqs", 65536, 2, "65535"), ("lens", None, 1, "NULL"), ("table", None, 1, "NULL"),
          ("q", 72, 1, "16-byte aligned"), ("q_stride", (252, 256, 64), 1, "multiples of 8"),
          ("q_stride", (1 << 40, 256, 64), 1, "reach")]


@pytest.mark.parametrize("name", ["bs_block_choice", "bs_block_attention", "bs_shared_attention"])
@pytest.mark.parametrize("field,value,code,text", COMMON)
def test_common_checks(name, field, value, code, text):
    d = calls()[name]
    put(d, field, value)
    rc, why = call(name, d)
    assert rc == code and text in why, (rc, why)


@pytest.mark.parametrize("name,field,value,code,text", [
    ("bs_block_choice", "count", 0, 1, "count"), ("bs_block_choice", "count", 1 << 26, 1, "count"), ("bs_block_choice", "sinks", -1, 1, "sinks"),
    ("bs_block_choice", "recent", 8, 1, "sinks + recent"), ("bs_block_choice", "bounds", 72, 1, "bounds"), ("bs_block_choice", "blocks", None, 1, "NULL"),
    ("bs_block_attention", "count", -1, 1, "count"), ("bs_block_attention", "count", 1 << 25, 1, "2^30"), ("bs_block_attention", "scale", 0.0, 1, "scale"),
    ("bs_block_attention", "scale", math.nan, 1, "scale"), ("bs_block_attention", "blocks", None, 1, "NULL"), ("bs_block_attention", "out", None, 1, "NULL"),
    ("bs_shared_attention", "num_groups", 0, 1, "num_groups is 0"), ("bs_shared_attention", "shared_width", 1 << 26, 2, "2^30"),
    ("bs_shared_attention", "cu", None, 1, "NULL"), ("bs_shared_attention", "shared_table", None, 1, "NULL"),
    ("bs_shared_attention", "scale", -1.0, 1, "scale"), ("bs_shared_attention", "workspace", 72, 1, "aligned"),
    ("bs_block_bounds", "num_seqs", 65536, 2, "65535"), ("bs_block_bounds", "bounds", None, 1, "NULL"), ("bs_block_bounds", "bounds", 72, 1, "bounds")])
def test_own_checks(name, field, value, code, text):
    d = calls()[name]
    put(d, field, value)
    rc, why = call(name, d)
    assert rc == code and text in why, (rc, why)


@pytest.mark.parametrize("name", [n for n in calls() if n != "bs_norm_rotate"])
@pytest.mark.parametrize("field,value,code,text", [("block", 24, 1, "16, 32, 64 or 128"), ("dim", 40, 2, "multiple of 16"), ("kv_heads", 0, 1, "kv_heads")])
def test_cache_checks(name, field, value, code, text):
    rc, why = call(name, calls()[name], **{field: value})
    assert rc == code and text in why, (rc, why)


@pytest.mark.parametrize("name,fields", [("bs_norm_rotate", "positions"), ("bs_block_bounds", "table lens"), ("bs_block_choice", "table lens blocks"),
                                         ("bs_block_attention", "table lens blocks lse"),
                                         ("bs_shared_attention", "shared_table shared_lens cu table lens lse")])
def test_misaligned_32_bit_buffers_are_refused(name, fields):
    for field in fields.split():
        d = calls()[name]
        setattr(d, field, 66)
        rc, why = call(name, d)
        assert rc == 1 and "4-byte" in why, (field, rc, why)


def test_memory_that_is_no_gpus_is_refused():
    # (where there is no GPU the device query fails first)
    for name in calls():
        rc, why = call(name, calls()[name])
        assert rc != 0 and ("current device" in why or "device query" in why), (name, rc, why)


def test_nothing_to_do_is_done_without_a_gpu():
    assert call("bs_norm_rotate", A._Rotate(q_heads=2, kv_heads=1, dim=64, dtype=2, amplitude=1.0))[0] == 0
    assert call("bs_block_bounds", A._Bounds())[0] == 0
    assert call("bs_block_bounds", A._Bounds(64, 64, 64, 2, 3, 0))[0] == 0                 # the last 0 tokens
    assert call("bs_block_choice", A._Choice(queries=1, q_heads=2, dtype=1, count=1))[0] == 0
    assert call("bs_block_attention", A._Blocks(queries=1, q_heads=2, dtype=1, scale=1.0))[0] == 0
    assert call("bs_shared_attention", A._Shared(queries=1, q_heads=2, dtype=1, scale=1.0))[0] == 0


def test_host_tensors_are_refused():
    q = torch.zeros((4, 2, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        M.norm_rotate(q, q, torch.zeros(4, dtype=torch.int32))


def test_kernels_wait_for_the_one_before_them_first():
    # launched under the end of the kernel before: nothing of the caller's is read and no error bit set before the wait
    kernels = 0
    for name in ("bs_norm_rotate.cu", "bs_block_choice.cu", "bs_block_attention.cu", "bs_shared_attention.cu"):
        with open(os.path.join(B.PKG, "csrc", name)) as f:
            text = f.read()
        for m in re.finditer(r"__global__ void[^;{]*?(k_\w+)\(", text):
            body = text[m.end():text.index("\n}\n", m.end())]
            before, wait, _ = body.partition("cudaGridDependencySynchronize();")
            assert wait, m[1]
            assert not re.search(r"tokens_of\(|group_of\(|count_cost\(|atomicOr\(|\bd\.\w+\[|table\[", before), m[1]
            kernels += 1
    assert kernels >= 5


def test_frequencies():
    f, a = M.rotary_frequencies(64)
    assert a == 1.0 and f.dtype == torch.float64 and torch.allclose(f, 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32), rtol=1e-14)
    g, a = M.rotary_frequencies(64, scaling="linear", factor=4)
    assert a == 1.0 and torch.equal(g, f / 4)
    g, a = M.rotary_frequencies(64, scaling="base", factor=8)
    assert a == 1.0 and g[0] == 1 and abs(float(f[-1] / g[-1]) - 8) < 1e-9
    g, a = M.rotary_frequencies(128, 500000.0, scaling="parts", factor=16, trained=8192)
    f, _ = M.rotary_frequencies(128, 500000.0)
    turns = 8192 * f / (2 * math.pi)
    assert abs(a - (0.1 * math.log(16) + 1)) < 1e-12
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.allclose(g[turns <= 1], f[turns <= 1] / 16, rtol=1e-14)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and ((g < f) & (g > f / 16))[mid].all()
    assert M.rotary_frequencies(0)[0].shape == (0,) and M.rotary_frequencies(2, scaling="base", factor=2)[0].tolist() == [1.0]


@pytest.mark.parametrize("kw", [dict(rotary=3), dict(rotary=-2), dict(rotary=4, scaling="yes"), dict(rotary=4, factor=0.5), dict(rotary=4, base=1.0),
                                dict(rotary=4, scaling="parts", factor=2), dict(rotary=4, scaling="parts", trained=64, fast=1.0, slow=2.0)])
def test_frequencies_refusals(kw):
    with pytest.raises(ValueError):
        M.rotary_frequencies(**kw)


def test_angles_reduced_in_integers_are_right():
    # the kernel's reduction, in Python integers, against exact rational arithmetic
    from fractions import Fraction
    pi = Fraction(314159265358979323846264338327950288419716939937510, 10 ** 50)
    for freq in (1.0, 0.7498942093324559, 1e-4, 3.7):
        for position in (0, 1, -1, 12345, 2 ** 31 - 1, -2 ** 31):
            turn = freq * 0.15915494309189535
            fixed = int((turn - math.floor(turn)) * 2.0 ** 64) % 2 ** 64
            got = Fraction((fixed * position) % 2 ** 64 >> 32, 2 ** 32)
            want = Fraction(freq) / (2 * pi) * position % 1
            off = abs(got - want)
            off = float(min(off, 1 - off))
            assert off <= 2.0 ** -32 + abs(position) * (2.0 ** -64 + 2.0 ** -52 * abs(turn)), (freq, position, off)


@pytest.mark.parametrize("name", ["bs_prompt_attention.cu", "bs_cache_attention.cu", "bs_token_cache.cu", "bs_norm_rotate.cu", "bs_block_choice.cu",
                                  "bs_block_attention.cu", "bs_shared_attention.cu"])
def test_every_block_waits_whatever_the_call_is(name):
    # the wait is a statement of its own, under no condition, and alone: a kernel that begins without it would count on what a
    # kernel two before it wrote, which is promised to those alone that wait themselves
    with open(os.path.join(B.PKG, "csrc", name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    kernels = [(m[1], text[m.end():text.index("\n}\n", m.end())]) for m in re.finditer(r"__global__ void[^;{]*?(k_\w+)\(", text)]
    assert kernels
    for kernel, body in kernels:
        assert body.count("cudaGridDependencySynchronize()") == 1, kernel
        before, wait, _ = body.partition("\n    cudaGridDependencySynchronize();")        # (four spaces: the kernel's own block)
        assert wait and re.search(r"[;{}]\s*\Z", before), kernel
        assert not re.search(r"\breturn\b|atomicOr\(|\blens\b|\bd\.\w+\[", before.partition("{")[2]), kernel


def test_bounds_of_more_blocks_than_32_bits_count():
    # (the widest table of blocks of 16, and key heads: its product with them reaches 2^31)
    d = calls()["bs_block_bounds"]
    d.table_width = (1 << 26) - 1
    rc, why = call("bs_block_bounds", d, block=16, kv_heads=33)
    assert rc == 2 and "2^31" in why, (rc, why)
    for heads, last in ((32, -1), (65535, 1)):
        d.last = last
        rc, why = call("bs_block_bounds", d, block=16, kv_heads=heads)
        assert rc != 2 and ("current device" in why or "device query" in why), (rc, why)
