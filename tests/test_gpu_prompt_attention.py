"""GPU: attention of packed prompts against its definition in 64 bits."""
import math

import pytest
import torch

import memory_ref as R
from beam_search_collab_b200 import memory as M

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def inputs(seed, tq, tk, hq, hkv, d, dtype, spread=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    q = (torch.randn((tq, hq, d), generator=g, device="cuda") * spread).to(dtype)
    k, v = (torch.randn((tk, hkv, d), generator=g, device="cuda").to(dtype) for _ in range(2))
    return q, k, v


def check(q, k, v, lens_q, lens_k, causal=True, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out, lse = M.prompt_attention(q, k, v, R.cu(lens_q), R.cu(lens_k), causal=causal, scale=scale, with_lse=True)
    assert M.take_errors() == 0
    ref, ref_lse, weighted, big = R.prompt(q, k, v, lens_q, lens_k, causal, scale)
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    empty = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert (out[empty] == 0).all()
    off = (out.double() - ref).abs() - R.out_bound(ref, weighted, q.dtype, R.UNIT[q.dtype])
    assert off.max() <= 0, off.max()
    off = ((lse.double() - ref_lse).abs() - R.lse_bound(big))[~empty]
    assert not len(off) or off.max() <= 0, off.max()
    return out, lse


@pytest.mark.parametrize("lens", [[1], [2], [31], [127], [128], [129], [255, 257], [1, 1, 1], [5, 0, 300, 1, 0, 64],
                                  [640, 3, 1000]])
@pytest.mark.parametrize("dtype,hq,hkv,d", [(BF16, 4, 4, 128), (F16, 8, 2, 64), (BF16, 6, 2, 96)])
def test_lengths(lens, dtype, hq, hkv, d):
    q, k, v = inputs(1, sum(lens), sum(lens), hq, hkv, d, dtype)
    check(q, k, v, lens, lens)


@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_dimensions(d, dtype):
    lens = [200, 77]
    q, k, v = inputs(2, 277, 277, 6, 3, d, dtype)
    check(q, k, v, lens, lens)
    check(q, k, v, lens, lens, causal=False)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (5, 1), (7, 1), (16, 1), (12, 4), (40, 8), (100, 1), (128, 1)])
def test_groups(hq, hkv):
    lens = [150, 1, 33]
    q, k, v = inputs(3, 184, 184, hq, hkv, 64, BF16)
    check(q, k, v, lens, lens)


@pytest.mark.parametrize("lens_q,lens_k", [([1, 1], [500, 3]), ([100, 7], [356, 1000]), ([64], [64 + 4000]),
                                           ([130, 2, 1], [10, 2, 0]),     # more queries than keys: the first see none
                                           ([20, 5], [0, 0]), ([0, 3], [9, 3])])
@pytest.mark.parametrize("causal", [True, False])
def test_pieces_and_rows_that_see_nothing(lens_q, lens_k, causal):
    q, k, v = inputs(4, sum(lens_q), sum(lens_k), 4, 2, 128, BF16)
    check(q, k, v, lens_q, lens_k, causal=causal)


def test_many_sequences_of_all_lengths():
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 90, (300,), generator=g).tolist()
    q, k, v = inputs(5, sum(lens), sum(lens), 4, 2, 64, F16)
    check(q, k, v, lens, lens)


@pytest.mark.parametrize("spread", [0.0, 12.0])
def test_flat_and_peaked_scores(spread):
    # 0: every weight alike; 12: maxima that move far from tile to tile
    lens = [700]
    q, k, v = inputs(6, 700, 700, 4, 1, 128, BF16, spread)
    check(q, k, v, lens, lens)


def test_rising_scores_force_new_maxima():
    # each key's score is larger than the last by far: the running maximum moves at every tile
    n = 900
    q, k, v = inputs(7, n, n, 2, 1, 64, BF16)
    ramp = torch.linspace(0, 8, n, device="cuda")[:, None, None]
    q, k = torch.ones_like(q), (torch.ones_like(k).float() * ramp).to(BF16)
    check(q, k, v, [n], [n])


def test_fused_strides_and_unaligned_heads():
    # q, k, v as slices of one projection [tokens, (hq + 2 hkv) * d]
    lens, hq, hkv, d = [200, 57], 6, 2, 80
    g = torch.Generator("cuda").manual_seed(8)
    x = torch.randn((257, hq + 2 * hkv, d), generator=g, device="cuda").to(F16)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    one, lse = check(q, k, v, lens, lens)
    two, lse2 = M.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), R.cu(lens), with_lse=True)
    assert torch.equal(one, two) and torch.equal(lse, lse2)
    # heads outermost
    check(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, lens, lens)


def test_values_beyond_a_sequence_do_not_reach_it():
    # a neighbour's infinities and NaN sit in the rows a tile also covers
    lens = [50, 60, 70]
    q, k, v = inputs(9, 180, 180, 4, 2, 64, BF16)
    out, lse = check(q, k, v, lens, lens)
    k2, v2 = k.clone(), v.clone()
    k2[50:110], v2[50:110] = math.nan, math.inf
    q2 = q.clone()
    q2[50:110] = math.nan
    got, got_lse = M.prompt_attention(q2, k2, v2, R.cu(lens), with_lse=True)
    for rows in (slice(0, 50), slice(110, 180)):
        assert torch.equal(got[rows], out[rows]) and torch.equal(got_lse[rows], lse[rows])
    assert torch.isnan(got[50:110].float()).all()


def test_future_values_do_not_reach_a_query():
    q, k, v = inputs(10, 300, 300, 2, 1, 128, BF16)
    out, _ = check(q, k, v, [300], [300])
    k[200:], v[200:] = math.nan, math.nan
    got, _ = M.prompt_attention(q, k, v, R.cu([300]))
    assert torch.equal(got[:200], out[:200])


def test_repeats_and_streams():
    lens = [300, 411]
    q, k, v = inputs(11, 711, 711, 8, 2, 128, BF16)
    one, lse = M.prompt_attention(q, k, v, R.cu(lens), with_lse=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        two, lse2 = M.prompt_attention(q, k, v, R.cu(lens), with_lse=True)
    three, lse3 = M.prompt_attention(q, k, v, R.cu(lens), with_lse=True, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(one, two) and torch.equal(one, three) and torch.equal(lse, lse2) and torch.equal(lse, lse3)


def test_graph_capture():
    lens = [130, 60]
    q, k, v = inputs(12, 190, 190, 4, 2, 64, F16)
    at = R.cu(lens)
    M.prompt_attention(q, k, v, at)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = M.prompt_attention(q, k, v, at, with_lse=True)
    q2, k2, v2 = inputs(13, 190, 190, 4, 2, 64, F16)
    q.copy_(q2), k.copy_(k2), v.copy_(v2), at.copy_(R.cu([100, 90]))
    graph.replay()
    want, want_lse = M.prompt_attention(q2, k2, v2, R.cu([100, 90]), with_lse=True)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    del graph


def test_bad_lengths_set_an_error_bit_and_touch_nothing_else():
    q, k, v = inputs(14, 100, 100, 2, 1, 64, F16)
    good, _ = M.prompt_attention(q, k, v, R.cu([40, 60]))
    M.prompt_attention(q, k, v, R.i32([0, 40, 120]))          # beyond total_q
    assert M.take_errors() == 4
    M.prompt_attention(q, k, v, R.i32([0, 40, 100]), R.i32([0, -5, 100]))
    assert M.take_errors() == 4
    again, _ = M.prompt_attention(q, k, v, R.cu([40, 60]))
    assert M.take_errors() == 0 and torch.equal(good, again)


@pytest.mark.parametrize("d,lens", [(64, [300]), (128, [2000, 5]), (128, [1])])
def test_a_wait_that_gives_up_is_reported_and_the_gpu_stays_usable(d, lens, monkeypatch):
    # BSEARCH_WAIT_POLLS=0: the first wait of every block gives up at once
    q, k, v = inputs(16, sum(lens), sum(lens), 4, 2, d, BF16)
    good, _ = M.prompt_attention(q, k, v, R.cu(lens))
    assert M.take_errors() == 0
    monkeypatch.setenv("BSEARCH_WAIT_POLLS", "0")
    M.prompt_attention(q, k, v, R.cu(lens))
    assert M.take_errors() == 1 and M.take_errors() == 0
    monkeypatch.delenv("BSEARCH_WAIT_POLLS")
    again, _ = M.prompt_attention(q, k, v, R.cu(lens))
    assert M.take_errors() == 0 and torch.equal(good, again)


def test_few_queries_over_many_keys():
    # few tiles of queries: the keys are cut into chunks that a second kernel joins
    for lens_q, lens_k in (([1], [9000]), ([40, 3], [6000, 17]), ([128], [5000])):
        q, k, v = inputs(17, sum(lens_q), sum(lens_k), 4, 2, 96, F16)
        check(q, k, v, lens_q, lens_k)
        check(q, k, v, lens_q, lens_k, causal=False)


def test_values_that_are_not_finite_reach_those_who_see_them():
    q, k, v = inputs(18, 400, 400, 2, 1, 128, BF16)
    v[150, 0, 3], v[390, 0, 5] = math.inf, math.nan
    out, _ = M.prompt_attention(q, k, v, R.cu([400]))
    out = out.float()
    assert torch.isfinite(out[:150]).all()
    assert (out[150:, :, 3] == math.inf).all()
    assert torch.isnan(out[390:, :, 5]).all() and torch.isfinite(out[:390, :, 5]).all()
    rest = [i for i in range(128) if i not in (3, 5)]
    assert torch.isfinite(out[:, :, rest]).all()
    ref, _, weighted, _ = R.prompt(q, k, torch.nan_to_num(v, 0.0, 0.0, 0.0), [400], [400], True, 128 ** -0.5)
    off = (out.double() - ref)[:, :, rest].abs() - R.out_bound(ref, weighted, BF16, R.UNIT[BF16])[:, :, rest]
    assert off.max() <= 0


def test_refusals():
    q, k, v = inputs(15, 10, 10, 4, 2, 64, F16)
    at = R.cu([10])
    with pytest.raises(ValueError, match="type, device"):
        M.prompt_attention(q, k.to(BF16), v, at)
    with pytest.raises(ValueError, match="last dimension"):
        M.prompt_attention(q[:, :, ::2], k, v, at)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        M.prompt_attention(q.float(), k, v, at)
    with pytest.raises(ValueError, match="cu_q"):
        M.prompt_attention(q, k, v, at.long())
    with pytest.raises(ValueError, match="cu_k is needed"):
        M.prompt_attention(q, k[:5], v[:5], at)
    from beam_search_collab_b200 import BSearchError
    with pytest.raises(BSearchError, match="multiple of kv_heads"):
        M.prompt_attention(q[:, :3], k, v, at)
    wide = torch.zeros((10, 2, 200), dtype=F16, device="cuda")
    with pytest.raises(BSearchError, match="up to 128") as e:
        M.prompt_attention(wide[..., :144], wide[..., :144], wide[..., :144], at)
    assert e.value.status == 2
    odd = torch.zeros((10, 2, 65), dtype=F16, device="cuda")[..., :64]
    with pytest.raises(BSearchError, match="16-byte aligned"):
        M.prompt_attention(odd, odd, odd, at)
    shifted = torch.zeros(10 * 64 + 1, dtype=F16, device="cuda")[1:].view(10, 1, 64)
    with pytest.raises(BSearchError, match="16-byte aligned"):
        M.prompt_attention(shifted, shifted, shifted, at)
    with pytest.raises(BSearchError, match="NaN"):
        M.prompt_attention(q, k, v, at, scale=math.nan)
    assert M.take_errors() == 0


@pytest.mark.parametrize("heads,keys", [(4, 60), (1, 6000)])            # (6,000 keys of one head: several pieces)
def test_lists_that_begin_late_or_end_early_set_an_error_bit(heads, keys):
    q, k, v = inputs(43, 40, keys, heads, heads, 64, F16)
    whole_q, whole_k = R.cu([32, 8]), R.cu([keys - 10, 10])
    M.prompt_attention(q, k, v, whole_q, whole_k)
    assert M.take_errors() == 0
    for cu_q, cu_k in ((R.i32([10, 22, 40]), whole_k), (R.i32([0, 22, 30]), whole_k), (whole_q, R.i32([3, 5, keys])),
                       (whole_q, R.i32([0, 5, keys - 1]))):
        M.prompt_attention(q, k, v, cu_q, cu_k)
        assert M.take_errors() == 4
    # the rows that the lists do cover are right all the same
    out, lse = M.prompt_attention(q, k, v, R.i32([10, 22, 30]), R.i32([3, keys - 17, keys - 7]), with_lse=True)
    assert M.take_errors() == 4
    ref, ref_lse, weighted, big = R.prompt(q[10:30], k[3:-7], v[3:-7], [12, 8], [keys - 20, 10], True, 0.125)
    assert ((out[10:30].double() - ref).abs() <= R.out_bound(ref, weighted, F16, R.UNIT[F16])).all()
    assert ((lse[10:30].double() - ref_lse).abs() <= R.lse_bound(big)).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("nats", [8, 13, 14, 15])
def test_small_weights_beside_a_large_one(nats, dtype):
    # the first key has no value and most of the weight, all others e^-nats of its: what 16 bits lose of one they lose of all
    n, heads, d = 1024, 160, 64                    # (so many heads that the keys stay in one piece)
    q, k, v = inputs(41, 1, n, heads, heads, d, dtype)
    q, v = torch.ones_like(q), v.abs()
    k.zero_()
    k[0], v[0] = nats / 8, 0
    out, lse = M.prompt_attention(q, k, v, R.cu([1]), R.cu([n]), with_lse=True)
    ref, ref_lse, weighted, big = R.prompt(q, k, v, [1], [n], True, 0.125)
    # the result's rounding, a weight's and its score's, and (f16) half a step of the smallest numbers at 2^7 for the largest
    bound = R.UNIT[dtype] * ref.abs() + (R.UNIT[dtype] + 2.0 ** -12) * (1 + 2.0 ** -7) * weighted + 2.0 ** -32 * v.double().sum(0)
    assert ((out.double() - ref).abs() <= bound).all()
    assert ((lse.double() - ref_lse).abs() <= R.lse_bound(big)).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_whose_scores_are_far_below_zero_and_far_above(dtype):
    lens = [300, 70]
    q, k, v = inputs(42, 370, 370, 4, 2, 64, dtype)
    k[:, :, 0], q[:, :, 0] = 20.0, torch.linspace(-60, 60, 370, device="cuda")[:, None].to(dtype)
    check(q, k, v, lens, lens)


@pytest.mark.parametrize("value", ["", "many", "-1", "0x", "1e3", "0 ", "99999999999999999999999"])
def test_what_is_not_a_number_of_polls_is_ignored(value, monkeypatch):
    q, k, v = inputs(46, 40, 40, 4, 4, 64, F16)
    good, _ = M.prompt_attention(q, k, v, R.cu([40]))
    monkeypatch.setenv("BSEARCH_WAIT_POLLS", value)
    got, _ = M.prompt_attention(q, k, v, R.cu([40]))
    assert M.take_errors() == 0 and torch.equal(got, good)


def test_keys_and_values_with_heads_outermost():
    lens = [200, 57]
    q, k, v = inputs(51, 257, 257, 6, 2, 80, F16)
    one, lse = check(q, k, v, lens, lens)
    k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k, v))
    two, lse2 = M.prompt_attention(q, k, v, R.cu(lens), with_lse=True)
    assert torch.equal(one, two) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens_q,lens_k,at", [([100], [100], 20), ([300, 40], [300, 40], 20),          # in an item's first tile of keys
                                              ([64], [6000], 5950), ([64], [6000], 20)])               # keys in several pieces
def test_values_that_are_not_finite_in_first_tiles_and_pieces(dtype, lens_q, lens_k, at):
    q, k, v = inputs(52, sum(lens_q), sum(lens_k), 2, 1, 64, dtype)
    v[at, 0, 3], v[at + 5, 0, 7] = math.inf, math.nan
    out, _ = M.prompt_attention(q, k, v, R.cu(lens_q), R.cu(lens_k))
    assert M.take_errors() == 0
    first = out[:lens_q[0]].float()
    sees = torch.arange(lens_q[0], device="cuda") + lens_k[0] - lens_q[0]
    a, b = sees >= at, sees >= at + 5
    assert (first[a][:, :, 3] == math.inf).all() and torch.isfinite(first[~a]).all()
    assert torch.isnan(first[b][:, :, 7]).all() and torch.isfinite(first[~b][:, :, 7]).all()
    ref, _, weighted, _ = R.prompt(q, k, torch.nan_to_num(v, 0.0, 0.0, 0.0), lens_q, lens_k, True, 0.125)
    rest = [i for i in range(64) if i not in (3, 7)]
    off = (out.double() - ref)[:, :, rest].abs() - R.out_bound(ref, weighted, dtype, R.UNIT[dtype])[:, :, rest]
    assert off.max() <= 0
