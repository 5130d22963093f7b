"""GPU: attention of sequences that begin with the same tokens (bs_shared_attention) against its definition, and the
operators of a decoding step together."""
import math

import pytest
import torch

import memory_ref as R
from beam_search_collab_b200 import BSearchError
from beam_search_collab_b200 import memory as M

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def case(seed, groups, shared, lens, hq, hkv, block, dim, queries, dtype, spread=1.0):
    g = gen(seed)
    counts, shared_counts = ([-(-n // block) for n in x] for x in (lens, shared))
    ids = torch.randperm(sum(counts) + sum(shared_counts) + 1, generator=g, device="cuda").to(torch.int32)
    pool = R.random_pool(g, len(ids), hkv, block, dim)

    def table(n, first):
        t = torch.full((len(n), max(n)), -1, dtype=torch.int32, device="cuda")
        for b, x in enumerate(n):
            t[b, :x] = ids[first:first + x]
            first += x
        return t

    q = (spread * torch.randn((len(lens), queries, hq, dim), generator=g, device="cuda")).to(dtype)
    return pool, table(shared_counts, sum(counts)), table(counts, 0), q


def reference(pool, shared_table, table, q, groups, shared, lens, scale):
    n_seq, nq, hq, d = q.shape
    hkv = pool[0].shape[1]
    g = hq // hkv
    out, weighted = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    lse, big = (torch.zeros(q.shape[:3], dtype=torch.float64, device="cuda") for _ in range(2))
    b = 0
    for m, (size, p) in enumerate(zip(groups, shared)):
        for h in range(hkv):
            far = [R.held(pool, shared_table, m, p, h, i) for i in (0, 1)]
            for x in range(b, b + size):
                k, v = (torch.cat((far[i], R.held(pool, table, x, lens[x], h, i))) for i in (0, 1))
                limits = p + (torch.arange(nq, device="cuda") + lens[x] - nq + 1).clamp(min=0).repeat_interleave(g)
                o = R.attend(q[x, :, h * g:h * g + g].reshape(nq * g, d).double(), k, v, scale, limits)
                to = (x, slice(None), slice(h * g, h * g + g))
                out[to], lse[to], weighted[to], big[to] = o[0].view(nq, g, d), o[1].view(nq, g), o[3].view(nq, g, d), o[4].view(nq, g)
        b += size
    return out, lse, weighted, big


def check(pool, shared_table, table, q, groups, shared, lens, scale=None):
    scale = q.shape[3] ** -0.5 if scale is None else scale
    out, lse = M.TokenCache(*pool).shared_attention(q, shared_table, R.i32(shared), R.cu(groups), table, R.i32(lens), scale=scale, with_lse=True)
    assert M.take_errors() == 0
    ref, ref_lse, weighted, big = reference(pool, shared_table, table, q, groups, shared, lens, scale)
    empty = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert (out[empty] == 0).all()
    # weights rounded to f16, as in the attention over the whole cache
    off = (out.double() - ref).abs() - R.out_bound(ref, weighted, q.dtype, R.UNIT[F16])
    assert off.max() <= 0, off.max()
    off = ((lse.double() - ref_lse).abs() - R.lse_bound(big))[~empty]
    assert not len(off) or off.max() <= 0, off.max()
    return out, lse


@pytest.mark.parametrize("groups,shared,lens", [
    ([1], [1], [1]), ([1], [0], [5]), ([2], [17], [0, 3]), ([3], [128], [1, 16, 129]), ([1, 1, 1], [127, 0, 300], [10, 0, 5]),
    ([5, 2], [1000, 129], [1, 0, 33, 7, 200, 64, 65]), ([4, 0, 3], [256, 50, 384], [3] * 7), ([17], [2049], [1] * 17)])
@pytest.mark.parametrize("dtype,hq,hkv,block,dim,queries", [(F16, 8, 2, 16, 64, 1), (BF16, 8, 8, 64, 128, 1), (BF16, 12, 2, 32, 96, 3),
                                                            (F16, 4, 1, 128, 48, 2)])
def test_groups_and_lengths(groups, shared, lens, dtype, hq, hkv, block, dim, queries):
    check(*case(1, groups, shared, lens, hq, hkv, block, dim, queries, dtype), groups, shared, lens)


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_dimensions(dim, block, dtype):
    groups, shared, lens = [3, 1], [700, 55], [20, 1, 150, 9]
    check(*case(2, groups, shared, lens, 6, 3, block, dim, 1, dtype), groups, shared, lens)


@pytest.mark.parametrize("seqs,hq,hkv,queries", [(1, 1, 1, 1), (31, 4, 1, 1), (32, 4, 1, 1), (33, 4, 1, 1), (64, 4, 1, 1), (65, 4, 1, 1),
                                                 (9, 128, 1, 1), (3, 17, 1, 5), (150, 4, 2, 1), (20, 32, 2, 2)])
def test_rows(seqs, hq, hkv, queries):
    # less than a tile of rows, whole tiles, one more
    lens = [(7 * i) % 50 for i in range(seqs)]
    check(*case(3, [seqs], [901], lens, hq, hkv, 32, 128, queries, BF16), [seqs], [901], lens)


# Many sequences: what they share is multiplied for all of them at once.

@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_dimensions_of_many_sequences(dim, block, dtype):
    groups, shared, lens = [250, 50], [700, 1329], [(7 * i) % 20 for i in range(300)]
    check(*case(19, groups, shared, lens, 6, 3, block, dim, 1, dtype), groups, shared, lens)


@pytest.mark.parametrize("groups,shared", [([300], [1]), ([300], [128]), ([300], [129]), ([300], [2049]), ([31, 33, 32, 200], [513, 2000, 640, 5000]),
                                           ([1] * 10 + [290], [3000] * 10 + [777]), ([150, 0, 150], [999, 50, 0]), ([64, 65, 128, 129], [1500] * 4)])
@pytest.mark.parametrize("dtype,hq,hkv,block,dim,queries", [(F16, 4, 2, 16, 64, 1), (BF16, 8, 2, 64, 128, 1), (BF16, 6, 2, 128, 96, 2)])
def test_groups_of_many_sequences(groups, shared, dtype, hq, hkv, block, dim, queries):
    lens = [(11 * i) % 30 for i in range(sum(groups))]
    check(*case(20, groups, shared, lens, hq, hkv, block, dim, queries, dtype), groups, shared, lens)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_scales_and_maxima_of_many_sequences(dtype):
    # flat and peaked scores, scales of 0 and of all sizes, scores that grow from tile to tile, blocks that are not there
    groups, shared, lens = [200, 100], [2500, 3001], [(3 * i) % 10 for i in range(300)]
    for spread in (0.0, 1.0, 6.0):
        pool, shared_table, table, q = case(21, groups, shared, lens, 8, 2, 64, 128, 1, dtype, spread)
        for col, factor in ((3, 0), (5, 1e4), (6, 1e-6)):
            pool[3][shared_table[:, col].long()] *= factor
        pool[2][shared_table[0, 4].long()] = 0
        one = check(pool, shared_table, table, q, groups, shared, lens)
        two = check(pool, shared_table, table, q, groups, shared, lens)
        assert all(torch.equal(a, b) for a, b in zip(one, two))            # the same every time
    pool, shared_table, table, q = case(22, groups, shared, lens, 4, 1, 16, 64, 1, dtype)
    for col in range(shared_table.shape[1]):
        at = shared_table[:, col]
        pool[2][at[at >= 0].long()] = 1e-5 * 1.08 ** col
    check(pool, shared_table, table, q, groups, shared, lens)
    pool, shared_table, table, q = case(23, groups, shared, lens, 8, 2, 32, 64, 1, BF16)
    check(pool, shared_table, table, (q.float() * 2.0 ** 40).to(BF16), groups, shared, lens, scale=2.0 ** -43)
    check(pool, shared_table, table, (q.float() * 2.0 ** -60).to(BF16), groups, shared, lens, scale=2.0 ** 57)


def test_blocks_that_are_not_there_of_many_sequences():
    # as if their tokens were not there: the same as a table without them, where they are whole blocks
    groups, shared, lens = [300], [1500], [5] * 300
    pool, shared_table, table, q = case(24, groups, shared, lens, 8, 2, 16, 128, 1, BF16)
    cache = M.TokenCache(*pool)
    bad = shared_table.clone()
    bad[0, [0, 1, 2, 3, 4, 5, 6, 7, 9, 40]] = R.i32([-1, 99999, -7, 2 ** 31 - 1, -1, -1, -1, -1, 12345, -2 ** 31])
    keep = [i for i in range(94) if i not in (0, 1, 2, 3, 4, 5, 6, 7, 9, 40)]
    out, lse = cache.shared_attention(q, bad, R.i32(shared), R.cu(groups), table, R.i32(lens), with_lse=True)
    assert M.take_errors() == 2
    less = shared_table[:, keep].contiguous()
    ref, ref_lse, weighted, big = reference(pool, less, table, q, groups, [1500 - 160], lens, 128 ** -0.5)
    assert ((out.double() - ref).abs() <= R.out_bound(ref, weighted, BF16, R.UNIT[F16])).all()
    assert ((lse.double() - ref_lse).abs() <= R.lse_bound(big)).all()


@pytest.mark.parametrize("cu", [[1, 200, 300], [0, 200, 299], [0, 200, 301], [0, 300, 200], [0, -1, 300], [0, 1 << 30, 300], [-5, 200, 300], [0, 0, 0]])
def test_wrong_lists_of_many_sequences_set_a_bit(cu):
    groups, shared, lens = [200, 100], [2500, 3001], [2] * 300
    pool, shared_table, table, q = case(25, groups, shared, lens, 8, 2, 64, 64, 1, F16)
    M.TokenCache(*pool).shared_attention(q, shared_table, R.i32(shared), R.i32(cu), table, R.i32(lens))
    assert M.take_errors() & 4


def test_lengths_and_groups_that_change_in_a_graph_of_many_sequences():
    groups, shared, lens = [150, 150], [3000, 3000], [40] * 300
    pool, shared_table, table, q = case(26, groups, shared, lens, 8, 2, 32, 64, 1, F16)
    cache = M.TokenCache(*pool)
    far, near, cu = R.i32(shared), R.i32(lens), R.cu(groups)
    graph = torch.cuda.CUDAGraph()
    cache.shared_attention(q, shared_table, far, cu, table, near)
    with torch.cuda.graph(graph):
        got = cache.shared_attention(q, shared_table, far, cu, table, near, with_lse=True)
    for groups, shared in (([10, 290], [130, 2999]), ([300, 0], [2000, 17]), ([150, 150], [0, 0])):
        lens = [(13 * i) % 41 for i in range(300)]
        far.copy_(R.i32(shared)), near.copy_(R.i32(lens)), cu.copy_(R.cu(groups))
        graph.replay()
        want = check(pool, shared_table, table, q, groups, shared, lens)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_of_many_sequences():
    groups, shared, lens = [150, 150], [3000, 2000], [20] * 300
    pool, shared_table, table, q = case(27, groups, shared, lens, 8, 2, 32, 128, 1, BF16)
    cache = M.TokenCache(*pool)
    args = (shared_table, R.i32(shared), R.cu(groups), table, R.i32(lens))
    qs = [q, (q.float() * 0.5).to(BF16)]
    want = [cache.shared_attention(x, *args)[0] for x in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            got[i].append(cache.shared_attention(qs[i], *args, stream=s.cuda_stream)[0])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_many_groups_and_long_beginnings():
    groups = [1] * 40 + [7, 30, 2]
    shared = [(37 * i) % 400 for i in range(40)] + [9000, 5001, 12800]
    lens = [(11 * i) % 90 for i in range(sum(groups))]
    one = check(*case(4, groups, shared, lens, 8, 2, 64, 128, 1, BF16), groups, shared, lens)
    two = check(*case(4, groups, shared, lens, 8, 2, 64, 128, 1, BF16), groups, shared, lens)
    assert all(torch.equal(a, b) for a, b in zip(one, two))            # the same every time


def test_long_own_contexts():
    groups, shared, lens = [2, 1], [300, 10], [9000, 40, 3001]
    check(*case(5, groups, shared, lens, 8, 2, 16, 64, 1, F16), groups, shared, lens)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("spread", [0.0, 6.0])
def test_flat_and_peaked_with_scales_of_all_sizes(spread, dtype):
    groups, shared, lens = [40], [3000], [30] * 40
    pool, shared_table, table, q = case(6, groups, shared, lens, 8, 2, 64, 128, 1, dtype, spread)
    pool[2][shared_table[0, 3].long()] = 0               # keys of zeros: score 0
    pool[3][shared_table[0, 4].long()] = 0               # values of zeros keep their weight
    pool[3][shared_table[0, 5].long()] *= 1e4
    pool[3][shared_table[0, 6].long()] *= 1e-6
    pool[3][table[7, 0].long()] = 0
    check(pool, shared_table, table, q, groups, shared, lens)
    pool[3].zero_()
    check(pool, shared_table, table, q, groups, shared, lens)


def test_maxima_that_move_late():
    # scores that grow from tile to tile of the shared tokens, by far more than a weight may grow
    groups, shared, lens = [33], [2000], [5] * 33
    pool, shared_table, table, q = case(7, groups, shared, lens, 4, 1, 16, 64, 1, F16)
    for col in range(shared_table.shape[1]):
        pool[2][shared_table[0, col].long()] = 1e-5 * 1.1 ** col
    check(pool, shared_table, table, q, groups, shared, lens)
    check(pool, shared_table, table, q.to(BF16), groups, shared, lens)


def test_large_and_small_queries():
    groups, shared, lens = [20], [500], [10] * 20
    pool, shared_table, table, q = case(8, groups, shared, lens, 8, 2, 32, 64, 1, BF16)
    check(pool, shared_table, table, (q.float() * 2.0 ** 40).to(BF16), groups, shared, lens, scale=2.0 ** -43)
    check(pool, shared_table, table, (q.float() * 2.0 ** -60).to(BF16), groups, shared, lens, scale=2.0 ** 57)


def test_stale_slots_and_blocks_do_not_matter():
    groups, shared, lens = [5], [300], [20] * 5
    pool, shared_table, table, q = case(9, groups, shared, lens, 4, 2, 64, 64, 1, BF16)
    one = check(pool, shared_table, table, q, groups, shared, lens)
    last = shared_table[0, 4].long()
    pool[0][last, :, 44:], pool[1][last, :, 44:] = 127, -128
    used = set(shared_table[shared_table >= 0].tolist()) | set(table[table >= 0].tolist())
    spare = [i for i in range(pool[0].shape[0]) if i not in used]
    pool[2][spare], pool[3][spare] = math.nan, math.inf
    wide = torch.nn.functional.pad(shared_table, (0, 3), value=spare[0]).contiguous()
    two = check(pool, wide, table, q, groups, shared, lens)
    assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_equal_to_one_table_of_everything():
    # the same tokens, block by block, in tables of their own
    groups, shared, lens = [6], [512], [64, 1, 100, 0, 30, 64]
    pool, shared_table, table, q = case(10, groups, shared, lens, 8, 2, 32, 128, 1, BF16)
    out, lse = check(pool, shared_table, table, q, groups, shared, lens)
    whole = torch.cat((shared_table.expand(6, -1), table), 1).contiguous()
    want, want_lse, _ = M.TokenCache(*pool).attention(q, whole, R.i32([512 + n for n in lens]), with_lse=True)
    assert torch.allclose(out.float(), want.float(), atol=0.02, rtol=0.01) and torch.allclose(lse, want_lse, atol=1e-4)


def test_bad_tables_and_lengths():
    groups, shared, lens = [3, 2], [300, 200], [40] * 5
    pool, shared_table, table, q = case(11, groups, shared, lens, 4, 2, 32, 64, 1, F16)
    cache = M.TokenCache(*pool)
    args = [q, shared_table, R.i32(shared), R.cu(groups), table, R.i32(lens)]

    def run(**kw):
        a = list(args)
        for i, x in kw.items():
            a[int(i[1])] = x
        out, _ = cache.shared_attention(*a)
        return out, M.take_errors()

    good, flags = run()
    assert flags == 0
    bad = shared_table.clone()
    bad[0, 2] = 5000
    out, flags = run(_1=bad)
    assert flags == 2 and torch.equal(out[3:], good[3:]) and out.isfinite().all()
    bad = table.clone()
    bad[1, 0] = -3
    out, flags = run(_4=bad)
    rest = torch.tensor([0, 2, 3, 4], device="cuda")
    assert flags == 2 and torch.equal(out[rest], good[rest]) and out.isfinite().all()
    # (lengths past a table are cut to it: entries there may name no block, which sets bit 2 too)
    out, flags = run(_2=R.i32([300, 1 << 20]))
    assert flags & 4 and torch.equal(out[:3], good[:3])
    out, flags = run(_2=R.i32([-1, 200]))
    assert flags == 4 and torch.equal(out[3:], good[3:])
    out, flags = run(_5=R.i32([40, 40, 40, 40, 5000]))
    assert flags & 4 and torch.equal(out[:4], good[:4])


@pytest.mark.parametrize("cu", [[1, 3, 5], [0, 3, 4], [0, 3, 6], [0, 4, 3], [0, -1, 5], [0, 1 << 30, 5], [-5, 3, 5], [0, 0, 0]])
def test_lists_of_groups_that_are_wrong_set_a_bit(cu):
    groups, shared, lens = [3, 2], [300, 200], [40] * 5
    pool, shared_table, table, q = case(12, groups, shared, lens, 4, 2, 32, 64, 1, F16)
    M.TokenCache(*pool).shared_attention(q, shared_table, R.i32(shared), R.i32(cu), table, R.i32(lens))
    assert M.take_errors() & 4


def test_strides_streams_and_graphs():
    groups, shared, lens = [3, 4], [500, 1300], [40, 7, 0, 90, 1, 2, 3]
    pool, shared_table, table, q = case(13, groups, shared, [90] * 7, 8, 2, 32, 64, 2, F16)      # (blocks for lengths to come)
    cache = M.TokenCache(*pool)
    far, near, cu = R.i32(shared), R.i32(lens), R.cu(groups)

    def step(x, **kw):
        return cache.shared_attention(x, shared_table, far, cu, table, near, with_lse=True, **kw)

    want = step(q)
    wide = torch.zeros((7, 2, 12, 64), dtype=F16, device="cuda")
    wide[:, :, 2:10] = q
    for x in (wide[:, :, 2:10], q.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3), q.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)):
        assert all(torch.equal(a, b) for a, b in zip(step(x), want))
    one = q[:1].expand(7, -1, -1, -1)                    # one query for all
    assert all(torch.equal(a, b) for a, b in zip(step(one), step(one.contiguous())))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(q, stream=side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(q)
    far.copy_(R.i32([130, 900])), near.copy_(R.i32([1, 90, 30, 0, 0, 33, 64])), cu.copy_(R.cu([5, 2]))
    graph.replay()
    want = step(q)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    check(pool, shared_table, table, q, [5, 2], [130, 900], [1, 90, 30, 0, 0, 33, 64])
    assert M.take_errors() == 0


def test_two_streams_at_once():
    groups, shared, lens = [30, 30], [4000, 2000], [40] * 60
    pool, shared_table, table, q = case(14, groups, shared, lens, 8, 2, 32, 128, 1, BF16)
    cache = M.TokenCache(*pool)
    args = (shared_table, R.i32(shared), R.cu(groups), table, R.i32(lens))
    qs = [q, (q.float() * 0.5).to(BF16)]
    want = [cache.shared_attention(x, *args)[0] for x in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            got[i].append(cache.shared_attention(qs[i], *args, stream=s.cuda_stream)[0])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_a_wait_that_gives_up_sets_a_bit(monkeypatch):
    groups, shared, lens = [300], [3000], [3] * 300           # (few sequences have no wait in their kernel)
    pool, shared_table, table, q = case(18, groups, shared, lens, 8, 2, 32, 128, 1, BF16)
    good = check(pool, shared_table, table, q, groups, shared, lens)
    monkeypatch.setenv("BSEARCH_WAIT_POLLS", "0")
    M.TokenCache(*pool).shared_attention(q, shared_table, R.i32(shared), R.cu(groups), table, R.i32(lens))
    assert M.take_errors() & 1
    monkeypatch.delenv("BSEARCH_WAIT_POLLS")
    again = check(pool, shared_table, table, q, groups, shared, lens)
    assert all(torch.equal(a, b) for a, b in zip(good, again))


def test_refusals():
    groups, shared, lens = [3, 2], [300, 200], [40] * 5
    pool, shared_table, table, q = case(15, groups, shared, lens, 4, 2, 32, 64, 1, F16)
    cache = M.TokenCache(*pool)
    args = [q, shared_table, R.i32(shared), R.cu(groups), table, R.i32(lens)]
    bad = [(0, q.float()), (0, q[:4]), (0, q[..., :32]), (0, q.cpu()), (1, shared_table.long()), (1, shared_table[0]), (1, shared_table[:1]),
           (2, args[2][:1]), (2, args[2].cpu()), (3, args[3][:2]), (3, args[3].long()), (4, table[:4]), (4, table[:, ::2]), (5, args[5][:4])]
    for i, x in bad:
        with pytest.raises(ValueError):
            cache.shared_attention(*args[:i], x, *args[i + 1:])
    with pytest.raises(BSearchError, match="scale"):
        cache.shared_attention(*args, scale=-1.0)
    with pytest.raises(BSearchError, match="num_groups is 0"):
        cache.shared_attention(q, shared_table[:0], args[2][:0], args[3][:1], table, args[5])
    with pytest.raises(BSearchError, match="multiple"):
        cache.shared_attention(q[:, :, :3].contiguous(), *args[1:])
    none, _ = cache.shared_attention(q[:0], shared_table, args[2], R.i32([0, 0, 0]), table[:0], args[5][:0])
    assert none.shape == (0, 1, 4, 64)


def test_gradients_are_refused():
    groups, shared, lens = [2], [100], [10, 3]
    pool, shared_table, table, q = case(16, groups, shared, lens, 4, 2, 32, 64, 1, F16)
    q.requires_grad_()
    for x in M.TokenCache(*pool).shared_attention(q, shared_table, R.i32(shared), R.cu(groups), table, R.i32(lens), with_lse=True):
        with pytest.raises(RuntimeError, match="no gradient"):
            x.float().sum().backward()


# ---- the operators of a decoding step together --------------------------------

def test_a_decoding_step_of_conversations_about_one_document():
    # projections -> norm and rotary position -> cache -> attention with the shared document, and over chosen blocks of
    # the whole; against the same in 64 bits from the values that the cache holds
    g = gen(17)
    hq, hkv, dim, block, document, seqs = 8, 2, 64, 32, 1500, 6
    w = [0.5 + torch.rand(dim, generator=g, device="cuda") for _ in range(2)]
    freqs, amplitude = M.rotary_frequencies(dim, scaling="parts", factor=4.0, trained=512, device="cuda")
    kw = dict(q_weight=w[0], k_weight=w[1], amplitude=amplitude)

    def tokens(n):
        x = torch.randn((n, hq + 2 * hkv, dim), generator=g, device="cuda").to(BF16)
        return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]

    cache = M.TokenCache.empty(120, hkv, dim, block=block)
    free = torch.randperm(120, generator=g, device="cuda").to(torch.int32)
    shared_table, table = free[None, :47].contiguous(), free[47:47 + seqs * 4].view(seqs, 4).contiguous()
    q, k, v = tokens(document)
    _, k = M.norm_rotate(q, k, torch.arange(document, dtype=torch.int32, device="cuda"), freqs, **kw)
    cache.write(k, v, R.cu([document]), shared_table, R.i32([0]))
    lens = [0] * seqs
    for step in range(3):
        new = [20 + 7 * i if step == 0 else 1 for i in range(seqs)]
        q, k, v = tokens(sum(new))
        at = torch.cat([document + lens[i] + torch.arange(n, device="cuda") for i, n in enumerate(new)]).to(torch.int32)
        q, k = M.norm_rotate(q, k, at, freqs, **kw)
        cache.write(k, v, R.cu(new), table, R.i32(lens))
        lens = [a + n for a, n in zip(lens, new)]
        last = torch.tensor([sum(new[:i + 1]) - 1 for i in range(seqs)], device="cuda")
        q1 = q[last][:, None].contiguous()
        pool = [cache.k, cache.v, cache.k_scale, cache.v_scale]
        check(pool, shared_table, table, q1, [seqs], [document], lens)
        # the whole as one table: 1,500 tokens end inside a block, so the document's last block is left out here
        whole = torch.cat((shared_table[:, :46].expand(seqs, -1), table), 1).contiguous()
        total = R.i32([46 * block + n for n in lens])
        bounds = cache.update_bounds(cache.empty_bounds(), whole, total)
        blocks = cache.choose_blocks(q1, bounds, whole, total, 12, sinks=1, recent=2)
        out, lse = cache.block_attention(q1, whole, total, blocks, with_lse=True)
        for b in range(seqs):
            for h in range(hkv):
                cols = blocks[b, 0, h].long()
                assert (cols >= 0).all() and (cols[1:] > cols[:-1]).all()
                pos = (cols[:, None] * block + torch.arange(block, device="cuda")).reshape(-1)
                keys, values = (R.held(pool, whole, b, 50 * block, h, i)[pos][pos < total[b]] for i in (0, 1))
                rows = q1[b, 0, h * 4:h * 4 + 4].double()
                ref = R.attend(rows, keys, values, dim ** -0.5, torch.full((4,), len(keys), device="cuda"))
                off = (out[b, 0, h * 4:h * 4 + 4].double() - ref[0]).abs() - R.out_bound(ref[0], ref[3], BF16, R.UNIT[F16])
                assert off.max() <= 0
                assert ((lse[b, 0, h * 4:h * 4 + 4].double() - ref[1]).abs() <= R.lse_bound(ref[4])).all()
    assert M.take_errors() == 0


@pytest.mark.parametrize("seqs", [6, 300])
def test_lengths_of_shared_tokens_outside_their_table_set_a_bit(seqs):
    # a table without columns, and groups without sequences, have lengths too
    groups, shared, lens = [seqs - 1, 0, 1], [2000, 50, 300], [(7 * i) % 40 for i in range(seqs)]
    pool, shared_table, table, q = case(28, groups, shared, lens, 8, 2, 32, 64, 1, BF16)
    cache = M.TokenCache(*pool)

    def run(t, n):
        out, _ = cache.shared_attention(q, t, R.i32(n), R.cu(groups), table, R.i32(lens))
        return out, M.take_errors()

    good, flags = run(shared_table, shared)
    assert flags == 0
    for n in (1 << 20, -1):
        out, flags = run(shared_table, [2000, n, 300])
        assert flags == 4 and torch.equal(out, good)
    none = shared_table[:, :0].contiguous()
    own, flags = run(none, [0, 0, 0])
    assert flags == 0
    for n in ([5, 0, 0], [0, 0, -1], [0, 1, 0]):
        out, flags = run(none, n)
        assert flags == 4 and torch.equal(out, own)
