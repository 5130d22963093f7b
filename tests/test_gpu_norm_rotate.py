"""GPU: norm and rotary position of queries and keys (bs_norm_rotate) against the definition in 64 bits."""
import math

import pytest
import torch

import memory_ref as R
from beam_search_collab_b200 import BSearchError
from beam_search_collab_b200 import memory as M

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
FAR = 1 << 20


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def reference(x, positions, freqs, weight, eps, interleaved, amplitude):
    """(result, magnitude of the pair that each value is made of), 64 bits."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * weight.double()
    out, size = y.clone(), y.abs()
    half = 0 if freqs is None else len(freqs)
    if half:
        t = positions.double()[:, None, None] * freqs
        c, s = amplitude * torch.cos(t), amplitude * torch.sin(t)
        one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
        a, b = y[..., one], y[..., two]
        out[..., one], out[..., two] = a * c - b * s, b * c + a * s
        # (and what 53 bits lose of far angles, here and in the operator's frequencies, above 2^-17)
        size[..., one] = size[..., two] = abs(amplitude) * (a.abs() + b.abs()) * (1 + 2.0 ** 17 * 2.0 ** -51 * t.abs())
    return out, size


def check(got, x, positions, freqs, weight, eps, interleaved, amplitude):
    ref, size = reference(x, positions, freqs, weight, eps, interleaved, amplitude)
    assert got.dtype == x.dtype and got.shape == x.shape and got.is_contiguous()
    # one rounding to the type (in f16's subnormals half of 2^-24), and 32-bit arithmetic before it: a sum of 128
    # squares (2^-17 of itself at most, its root half of that), root, products, sine and cosine: 2^-17 of the pair
    off = (got.double() - ref).abs() - (R.UNIT[x.dtype] * ref.abs() + 2.0 ** -17 * size + (2.0 ** -25 if x.dtype == F16 else 1e-40))
    assert not off.numel() or off.max() <= 0, off.max()


def run_case(seed, tokens, hq, hkv, dim, rotary, interleaved, norm, dtype, weight_dtype=None, amplitude=1.0, spread=1.0, eps=1e-6):
    g = gen(seed)
    x = spread * torch.randn((tokens, hq + 2 * hkv, dim), generator=g, device="cuda")
    x = (x * torch.exp(torch.randn((tokens, hq + 2 * hkv, 1), generator=g, device="cuda"))).to(dtype)
    q, k = x[:, :hq], x[:, hq:hq + hkv]
    positions = torch.randint(-FAR, FAR, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    freqs = M.rotary_frequencies(rotary, device="cuda")[0] if rotary else None
    w = [(0.2 + torch.rand(dim, generator=g, device="cuda")).to(weight_dtype or dtype) if norm else None for _ in range(2)]
    out = M.norm_rotate(q, k, positions, freqs, q_weight=w[0], k_weight=w[1], eps=eps, interleaved=interleaved, amplitude=amplitude)
    for got, y, weight in zip(out, (q, k), w):
        check(got, y, positions, freqs, weight, eps, interleaved, amplitude)
    return q, k, positions, freqs, w, out


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_dimensions_and_parts(dim, interleaved, norm):
    for part in sorted({0, 2, 4, 6, 8, 10, 12, dim // 4 // 2 * 2, dim // 2, dim - 2, dim}):
        run_case(part, 5, 3, 2, dim, part, interleaved, norm, BF16 if part % 4 else F16)


@pytest.mark.parametrize("tokens,hq,hkv", [(1, 1, 1), (1, 40, 8), (3, 7, 5), (64, 12, 4), (2000, 32, 8), (5000, 5, 1), (3000, 1, 33)])
@pytest.mark.parametrize("dtype,interleaved", [(F16, True), (BF16, False)])
def test_sizes(tokens, hq, hkv, dtype, interleaved):
    run_case(1, tokens, hq, hkv, 128, 128, interleaved, True, dtype)
    run_case(2, tokens, hq, hkv, 80, 20, interleaved, False, dtype)


@pytest.mark.parametrize("weight_dtype", [F32, F16, BF16])
def test_weights_of_each_type(weight_dtype):
    run_case(3, 33, 8, 2, 64, 32, False, True, F16, weight_dtype)
    run_case(3, 33, 8, 2, 64, 32, True, True, BF16, weight_dtype)


def test_one_weight_alone_and_no_keys():
    q, k, positions, freqs, w, _ = run_case(4, 17, 6, 2, 96, 48, False, True, BF16)
    for qw, kw in ((w[0], None), (None, w[1])):
        out = M.norm_rotate(q, k, positions, freqs, q_weight=qw, k_weight=kw)
        check(out[0], q, positions, freqs, qw, 1e-6, False, 1.0)
        check(out[1], k, positions, freqs, kw, 1e-6, False, 1.0)
    out, none = M.norm_rotate(q, None, positions, freqs, q_weight=w[0])
    assert none is None
    check(out, q, positions, freqs, w[0], 1e-6, False, 1.0)


def test_without_rotation_and_norm_values_pass():
    q, k, positions, _, _, out = run_case(5, 40, 3, 3, 48, 0, False, False, F16)
    assert torch.equal(out[0], q) and torch.equal(out[1], k)


def test_amplitude_and_scaled_frequencies():
    g = gen(6)
    q, k = (torch.randn((300, h, 128), generator=g, device="cuda").to(BF16) for h in (8, 2))
    positions = torch.randint(0, 1 << 21, (300,), generator=g, device="cuda", dtype=torch.int32)
    for scaling in (None, "linear", "base", "parts"):
        freqs, amplitude = M.rotary_frequencies(128, 500000.0, scaling=scaling, factor=16.0, trained=8192, device="cuda")
        for got, x in zip(M.norm_rotate(q, k, positions, freqs, amplitude=amplitude), (q, k)):
            check(got, x, positions, freqs, None, 1e-6, False, amplitude)
    check(M.norm_rotate(q, None, positions, freqs, amplitude=-0.0)[0], q, positions, freqs, None, 1e-6, False, 0.0)


def test_the_farthest_positions_and_fast_frequencies():
    positions = torch.tensor([2 ** 31 - 1, -2 ** 31, -1, 0, 1, 123456789], dtype=torch.int32, device="cuda")
    freqs = torch.tensor([1.0, 3.1, -0.5, 1e-9, 0.0, 7.0, 1e-3, 100.0], dtype=torch.float64, device="cuda")
    # the reference's own product is rounded to 53 bits: 2^31 * 100 radians keep 2^-16 of a radian
    g = gen(7)
    q = torch.randn((6, 2, 16), generator=g, device="cuda").to(F16)
    check(M.norm_rotate(q, None, positions, freqs)[0], q, positions, freqs, None, 1e-6, False, 1.0)


def test_zeros_large_and_small_rows():
    positions = torch.arange(4, dtype=torch.int32, device="cuda")
    freqs = M.rotary_frequencies(64, device="cuda")[0]
    w = torch.ones(64, device="cuda")
    x = torch.zeros((4, 1, 64), dtype=BF16, device="cuda")
    out, _ = M.norm_rotate(x, None, positions, freqs, q_weight=w)
    assert (out == 0).all()
    out, _ = M.norm_rotate(x, None, positions, freqs, q_weight=w, eps=1e-30)
    assert (out == 0).all()
    for size in (2.0 ** 60, 2.0 ** -60):
        x = (size * torch.randn((4, 3, 64), generator=gen(8), device="cuda")).to(BF16)
        check(M.norm_rotate(x, None, positions, freqs, q_weight=w, eps=1e-38)[0], x, positions, freqs, w, 1e-38, False, 1.0)
    x = (60000 * torch.rand((4, 3, 64), generator=gen(9), device="cuda")).to(F16)
    check(M.norm_rotate(x, None, positions, freqs, q_weight=w)[0], x, positions, freqs, w, 1e-6, False, 1.0)


def test_a_row_that_is_not_finite_leaves_the_others():
    q, k, positions, freqs, w, out = run_case(10, 9, 4, 2, 128, 64, False, True, BF16)
    x = q.clone()
    x[3, 1, 5], x[4, 2, 7] = float("nan"), float("inf")
    got, _ = M.norm_rotate(x, None, positions, freqs, q_weight=w[0])
    rows = torch.ones((9, 4), dtype=torch.bool, device="cuda")
    rows[3, 1] = rows[4, 2] = False
    assert torch.equal(got[rows], out[0][rows]) and got[3, 1].isnan().all()


def test_strides_streams_graphs_and_no_tokens():
    q, k, positions, freqs, w, out = run_case(11, 200, 8, 2, 64, 64, True, True, F16)
    kw = dict(q_weight=w[0], k_weight=w[1], interleaved=True)
    for a, b in ((q.contiguous(), k.contiguous()), (q.transpose(0, 1).contiguous().transpose(0, 1), k)):
        got = M.norm_rotate(a, b, positions, freqs, **kw)
        assert torch.equal(got[0], out[0]) and torch.equal(got[1], out[1])
    one = q[:1].expand(200, -1, -1)                     # one token's heads at 200 positions
    got, _ = M.norm_rotate(one, None, positions, freqs, q_weight=w[0], interleaved=True)
    assert torch.equal(got, M.norm_rotate(one.contiguous(), None, positions, freqs, q_weight=w[0], interleaved=True)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = M.norm_rotate(q, k, positions, freqs, stream=side.cuda_stream, **kw)
    side.synchronize()
    assert torch.equal(got[0], out[0]) and torch.equal(got[1], out[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = M.norm_rotate(q, k, positions, freqs, **kw)
    positions.add_(7)
    graph.replay()
    want = M.norm_rotate(q, k, positions, freqs, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and not torch.equal(got[0], out[0])
    none = M.norm_rotate(q[:0], k[:0], positions[:0], freqs, **kw)
    assert none[0].shape == (0, 8, 64) and none[1].shape == (0, 2, 64)
    assert M.take_errors() == 0


def test_refusals():
    q, k, positions, freqs, w, _ = run_case(12, 4, 4, 2, 64, 32, False, True, F16)
    bad = [dict(k=k[:3]), dict(k=k.to(BF16)), dict(positions=positions.long()), dict(positions=positions[:3]), dict(freqs=freqs.float()),
           dict(freqs=freqs.cpu()), dict(q_weight=w[0][:32]), dict(q_weight=w[0].float()), dict(k_weight=w[1].cpu()), dict(k=None),
           dict(q_weight=w[0].to(torch.int32), k_weight=None), dict(q=q.float(), k=None, k_weight=None)]
    for change in bad:
        kw = dict(q=q, k=k, positions=positions, freqs=freqs, q_weight=w[0], k_weight=w[1]) | change
        with pytest.raises(ValueError):
            M.norm_rotate(kw.pop("q"), kw.pop("k"), kw.pop("positions"), kw.pop("freqs"), **kw)
    for kw in (dict(eps=-1.0), dict(amplitude=float("nan")), dict(freqs=torch.zeros(33, dtype=torch.float64, device="cuda"))):
        kw = dict(freqs=freqs) | kw
        with pytest.raises(BSearchError):
            M.norm_rotate(q, k, positions, kw.pop("freqs"), **kw)
    wide = torch.zeros((4, 4, 68), dtype=F16, device="cuda")
    with pytest.raises(BSearchError, match="multiples of 8"):
        M.norm_rotate(wide[:, :, :64], None, positions, freqs)


def test_gradients_are_refused():
    q, k, positions, freqs, w, _ = run_case(13, 4, 4, 2, 64, 32, False, True, F16)
    for need in ("q", "w"):
        a, b = q.clone().requires_grad_(need == "q"), w[0].clone().requires_grad_(need == "w")
        out, out_k = M.norm_rotate(a, k, positions, freqs, q_weight=b)
        assert out.requires_grad and not out_k.requires_grad
        with pytest.raises(RuntimeError, match="no gradient"):
            out.float().sum().backward()


def same(a, b):
    return torch.allclose(a, b, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 0), (16, 0), (128, 64), (96, 40), (80, 12), (48, 6), (128, 100), (64, 62)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_a_value_that_is_not_finite_stays_in_its_place(dim, rotary, value, interleaved):
    # token i has it in dimension i: past the rotated part it passes, in it the other of its pair alone is not finite either
    g = gen(14)
    x = torch.randn((dim, 3, dim), generator=g, device="cuda").to(F16 if rotary % 8 else BF16)
    positions = torch.randint(-9999, 9999, (dim,), generator=g, device="cuda", dtype=torch.int32)
    freqs = M.rotary_frequencies(rotary, device="cuda")[0] if rotary else None
    weight = torch.rand(dim, generator=g, device="cuda") + 0.5
    kw = dict(interleaved=interleaved, k_weight=weight)
    want, clean_k = M.norm_rotate(x, x[:, :1], positions, freqs, **kw)
    y, at = x.clone(), torch.arange(dim, device="cuda")
    y[at, 1, at] = value
    got, got_k = M.norm_rotate(y, x[:, :1], positions, freqs, **kw)
    want[at, 1, at] = value
    for d in range(rotary):
        for out in (want, got):
            out[d, 1, d] = out[d, 1, d ^ 1 if interleaved else (d + rotary // 2) % rotary] = 0
    assert same(got, want) and torch.equal(got_k, clean_k)


def test_positions_are_needed_for_a_rotation_alone():
    g = torch.Generator("cuda").manual_seed(15)
    q, k = (torch.randn((7, h, 64), generator=g, device="cuda").to(F16) for h in (4, 2))
    w = torch.rand(64, generator=g, device="cuda") + 0.5
    positions = torch.arange(7, dtype=torch.int32, device="cuda")
    want = M.norm_rotate(q, k, positions, q_weight=w)
    for got in (M.norm_rotate(q, k, q_weight=w), M.norm_rotate(q, k, None, None, q_weight=w)):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    none = M.rotary_frequencies(0, device="cuda")[0]
    assert torch.equal(M.norm_rotate(q, k, None, none, q_weight=w)[0], want[0])
    with pytest.raises(ValueError, match="positions"):
        M.norm_rotate(q, k, freqs=M.rotary_frequencies(32, device="cuda")[0])
    with pytest.raises(ValueError, match="positions"):
        M.norm_rotate(q, k, positions[:3])


@pytest.mark.parametrize("interleaved", [False, True])
def test_sines_and_cosines_of_far_positions(interleaved):
    # one dimension of a pair is 1: the pair becomes the cosine and the sine.  Off by one rounding (f16's below 2^-14: half of
    # 2^-24) and by 2^-19: the angle, a part of a turn, is reduced to 2^-32 turns (2^-29 radians), and in 32 bits rounded
    # three times, up to pi * 3 * 2^-24 = 2^-20.8; sine and cosine are off by 2^-21.2; in all 2^-19.9.  The angle itself
    # keeps 2^-52 of it, 2^-21 radians at 2^31, so the frequencies here are such that 2^53 holds the products exactly.
    g = torch.Generator("cuda").manual_seed(16)
    freqs = torch.tensor([1.0, 0.5, 3 * 2.0 ** -12, 2.0 ** -20, 5 * 2.0 ** -7, 1.5, 2.0 ** -16, 2.0 ** -9], dtype=torch.float64, device="cuda")
    positions = torch.randint(-(1 << 24), 1 << 24, (5000,), generator=g, device="cuda", dtype=torch.int32)
    x = torch.zeros((5000, 2, 16), dtype=F16, device="cuda")
    one, two = (slice(0, 16, 2), slice(1, 16, 2)) if interleaved else (slice(0, 8), slice(8, 16))
    x[:, 0, one] = x[:, 1, two] = 1
    out = M.norm_rotate(x, None, positions, freqs, interleaved=interleaved)[0].double()
    t = positions.double()[:, None] * freqs
    off = 2.0 ** -19 + 2.0 ** -25 + t.abs() * 2.0 ** -51
    for got, want in ((out[:, 0, one], t.cos()), (out[:, 0, two], t.sin()), (out[:, 1, two], t.cos()), (out[:, 1, one], -t.sin())):
        assert ((got - want).abs() <= 2.0 ** -11 * want.abs() + off).all()
