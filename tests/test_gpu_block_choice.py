"""GPU: bounds of the token cache's blocks, the choice of blocks by them, and attention over chosen blocks, against the
operators' definitions."""
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


def case(seed, lens, hq, hkv, block, dim, queries, dtype, spread=1.0, spare=1, width=0):
    g = gen(seed)
    counts = [-(-n // block) for n in lens]
    table, _ = R.random_table(g, counts, spare)
    if width > table.shape[1]:
        table = torch.nn.functional.pad(table, (0, width - table.shape[1]), value=-1)
    pool = R.random_pool(g, sum(counts) + spare, hkv, block, dim)
    q = (spread * torch.randn((len(lens), queries, hq, dim), generator=g, device="cuda")).to(dtype)
    return pool, table.contiguous(), q


# ---- bounds -----------------------------------------------------------------

def bounds_ref(pool, table, lens, last, old):
    bounds, block = old.clone(), pool[0].shape[2]
    for b, n in enumerate(lens):
        first = 0 if last is None or last >= n else (n - last) // block
        for col in range(first, -(-n // block) if last != 0 else 0):
            x = pool[0][table[b, col].long(), :, :min(block, n - col * block)]
            bounds[table[b, col].long()] = torch.stack((x.amax(1), x.amin(1)), 1)
    return bounds


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("last", [None, 0, 1, 17, 200, 5000])
def test_bounds(dim, block, last):
    lens = [260, 0, 1, block, block + 1, 77]
    pool, table, _ = case(1, lens, 3, 3, block, dim, 1, F16, width=20)
    cache = M.TokenCache(*pool)
    old = torch.randint(-128, 128, (pool[0].shape[0], 3, 2, dim), generator=gen(2), device="cuda", dtype=torch.int8)
    bounds = old.clone()
    assert cache.update_bounds(bounds, table, R.i32(lens), last=last) is bounds
    assert M.take_errors() == 0
    assert torch.equal(bounds, bounds_ref(pool, table, lens, last, old))


def test_bounds_of_extreme_codes():
    cache = M.TokenCache.empty(2, 2, 64, block=32)
    cache.k[0], cache.k[1] = -128, 127
    bounds = cache.update_bounds(cache.empty_bounds(), R.i32([[0], [1]]), R.i32([32, 5]))
    assert (bounds[0] == -128).all() and (bounds[1] == 127).all()


def test_bounds_of_bad_tables():
    pool, table, _ = case(3, [100, 40], 2, 2, 32, 64, 1, F16)
    cache, bounds = M.TokenCache(*pool), M.TokenCache(*pool).empty_bounds()
    bad = table.clone()
    bad[0, 1], bad[1, 0] = -7, 99
    cache.update_bounds(bounds, bad, R.i32([100, 40]))
    assert M.take_errors() == 2
    done = bounds.flatten(1).any(1)
    assert done.sum() == 4 and done[table[0, [0, 2, 3]].long()].all()
    cache.update_bounds(bounds, table, R.i32([129, -1]))
    assert M.take_errors() == 4


# ---- choice -----------------------------------------------------------------

def choice_ref(pool, bounds, table, q, lens, count, sinks, recent):
    n_seq, nq, hq, d = q.shape
    hkv, block = pool[0].shape[1], pool[0].shape[2]
    out = torch.full((n_seq, nq, hkv, count), -1, dtype=torch.int32, device="cuda")
    for b in range(n_seq):
        for i in range(nq):
            n = -(-max(0, lens[b] - nq + 1 + i) // block)
            for h in range(hkv):
                if n <= count:
                    out[b, i, h, :n] = torch.arange(n)
                    continue
                x = q[b, i, h * hq // hkv:(h + 1) * hq // hkv].float()
                top = x.abs().max()
                code = torch.round(x * (127 / top if top >= 1e-30 else torch.zeros_like(top))).long()
                ids = table[b, :n].long()
                hi, lo = bounds[ids, h, 0].long(), bounds[ids, h, 1].long()
                each = torch.maximum(code[:, None] * hi, code[:, None] * lo).sum((0, 2))
                score = each.float() * pool[2][ids, h]
                order = torch.argsort(score[sinks:n - recent], descending=True, stable=True)[:count - sinks - recent] + sinks
                at = torch.arange(n, device="cuda")
                out[b, i, h] = torch.cat((at[:sinks], order.sort().values, at[n - recent:])).to(torch.int32)
    return out


def check_choice(pool, table, q, lens, count, sinks=1, recent=1):
    cache = M.TokenCache(*pool)
    bounds = cache.update_bounds(cache.empty_bounds(), table, R.i32(lens))
    got = cache.choose_blocks(q, bounds, table, R.i32(lens), count, sinks=sinks, recent=recent)
    assert M.take_errors() == 0
    assert torch.equal(got, choice_ref(pool, bounds, table, q, lens, count, sinks, recent))
    return got


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("dtype,hq,hkv,queries", [(F16, 8, 2, 1), (BF16, 3, 3, 3)])
def test_choice_dimensions(dim, dtype, hq, hkv, queries):
    lens = [500, 0, 1, 33, 290]
    pool, table, q = case(4, lens, hq, hkv, 16, dim, queries, dtype)
    check_choice(pool, table, q, lens, 9)


@pytest.mark.parametrize("count,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (2, 1, 1), (4, 0, 0), (7, 2, 3), (30, 10, 20), (31, 1, 2), (200, 1, 1)])
def test_choice_counts(count, sinks, recent):
    lens = [1000, 481, 480, 15, 16, 17]
    pool, table, q = case(5, lens, 4, 2, 16, 64, 2, BF16)
    check_choice(pool, table, q, lens, count, sinks, recent)


@pytest.mark.parametrize("seqs,tokens,hkv", [(1, 40000, 1), (1, 70001, 2), (3, 20000, 8), (40, 5000, 8), (2, 140000, 4)])
def test_choice_of_long_contexts(seqs, tokens, hkv):
    # rows of one to eight thread blocks
    lens = [max(1, tokens - 997 * i) for i in range(seqs)]
    pool, table, q = case(6, lens, 2 * hkv, hkv, 16, 32, 1, F16)
    check_choice(pool, table, q, lens, 64, 1, 2)


def test_choice_of_more_blocks_than_shared_memory_holds():
    # 148 rows and more leave one thread block to each: 47,104 scores of a row stay in shared memory
    blocks, heads = 50000, 160
    table = torch.randint(0, 64, (1, blocks), generator=gen(7), device="cuda", dtype=torch.int32)
    pool = R.random_pool(gen(8), 64, heads, 16, 16)
    pool[2][:] = 0.01 + 0.01 * torch.rand((64, heads), generator=gen(9), device="cuda")
    q = torch.randn((1, 1, heads, 16), generator=gen(10), device="cuda").to(F16)
    check_choice(pool, table, q, [16 * blocks - 3], 1500, 1, 1)


def test_choice_ties_go_to_the_lower_column():
    pool, table, q = case(11, [1600], 2, 1, 16, 32, 1, F16)
    pool[0][:] = pool[0][:1]
    pool[2][:] = 0.5
    got = check_choice(pool, table, q, [1600], 10, 1, 2)
    assert got[0, 0, 0].tolist() == list(range(8)) + [98, 99]
    zero = check_choice(pool, table, torch.zeros_like(q), [1600], 10, 0, 0)
    assert zero[0, 0, 0].tolist() == list(range(10))
    tiny = (q.float() * 0 + 1e-36).to(BF16)                       # below the smallest that counts
    assert check_choice(pool, table, tiny, [1600], 10, 0, 0)[0, 0, 0].tolist() == list(range(10))


def test_choice_holds_the_blocks_of_the_largest_scores():
    # what the score is for: no token of a block that is left out scores higher than the bound of one that is chosen
    lens = [3000]
    pool, table, q = case(12, lens, 1, 1, 32, 64, 1, F16)
    cache = M.TokenCache(*pool)
    bounds = cache.update_bounds(cache.empty_bounds(), table, R.i32(lens))
    got = cache.choose_blocks(q, bounds, table, R.i32(lens), 20, sinks=0, recent=0)[0, 0, 0].long()
    x = q[0, 0, 0].double()
    up = x.abs().max() / 127
    code = torch.round(x / up)
    ids = table[0].long()
    scale = pool[2][ids, 0].double()
    allowed = torch.maximum(code * bounds[ids, 0, 0].double(), code * bounds[ids, 0, 1].double()).sum(1) * scale
    true = (R.held(pool, table, 0, 3000, 0, 0) @ code)
    true = torch.nn.functional.pad(true, (0, -3000 % 32), value=-math.inf).view(-1, 32).amax(1)
    assert (true <= allowed * (1 + 1e-6)).all()
    left = torch.ones(len(ids), dtype=torch.bool, device="cuda").index_fill_(0, got, False)
    assert true[left].max() <= allowed[got].min() * (1 + 1e-6)


def test_choice_of_queries_that_are_not_finite_is_some_choice():
    lens = [700]
    pool, table, q = case(13, lens, 2, 2, 16, 32, 1, F16)
    q[0, 0, 0, 3], q[0, 0, 1, 4] = math.nan, math.inf
    pool[2][table[0, 5].long(), 0] = math.nan                     # counts as the largest
    cache = M.TokenCache(*pool)
    bounds = cache.update_bounds(cache.empty_bounds(), table, R.i32(lens))
    got = cache.choose_blocks(q, bounds, table, R.i32(lens), 6, sinks=1, recent=1)
    assert 5 in got[0, 0, 0].tolist()
    for h in range(2):
        x = got[0, 0, h]
        assert (x[1:] > x[:-1]).all() and x[0] == 0 and x[-1] == 43


def test_choice_of_bad_tables_and_lengths():
    lens = [700]
    pool, table, q = case(14, lens, 2, 2, 16, 32, 1, F16)
    cache = M.TokenCache(*pool)
    bounds = cache.update_bounds(cache.empty_bounds(), table, R.i32(lens))
    bad = table.clone()
    bad[0, 7] = 1000
    got = cache.choose_blocks(q, bounds, bad, R.i32(lens), 6)
    assert M.take_errors() == 2 and (got >= 0).all() and (got < 44).all()
    got = cache.choose_blocks(q, bounds, table, R.i32([2000]), 6)
    assert M.take_errors() == 4 and (got >= 0).all() and (got < 44).all()
    got = cache.choose_blocks(q, bounds, table, R.i32([-5]), 6)
    assert M.take_errors() == 4 and (got == -1).all()
    none = cache.choose_blocks(q, bounds, table[:, :0].contiguous(), R.i32([0]), 6)
    assert M.take_errors() == 0 and (none == -1).all()


# ---- attention over chosen blocks -------------------------------------------

def attention_ref(pool, table, q, lens, blocks, scale):
    n_seq, nq, hq, d = q.shape
    hkv, block = pool[0].shape[1], pool[0].shape[2]
    g = hq // hkv
    out, weighted = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    lse, big = (torch.zeros(q.shape[:3], dtype=torch.float64, device="cuda") for _ in range(2))
    for b in range(n_seq):
        for i in range(nq):
            seen = max(0, lens[b] - nq + 1 + i)
            for h in range(hkv):
                cols = blocks[b, i, h].long()
                cols = cols[cols >= 0]
                at = (cols[:, None] * block + torch.arange(block, device="cuda")).reshape(-1)
                ids = table[b, cols].long()
                k, v = ((pool[x][ids, h].double() * pool[2 + x][ids, h].double()[:, None, None]).reshape(-1, d)[at < seen] for x in (0, 1))
                limits = torch.full((g,), len(k), device="cuda")
                o = R.attend(q[b, i, h * g:h * g + g].double(), k, v, scale, limits)
                to = (b, i, slice(h * g, h * g + g))
                out[to], lse[to], weighted[to], big[to] = o[0], o[1], o[3], o[4]
    return out, lse, weighted, big


def check_blocks(pool, table, q, lens, blocks, scale=None):
    scale = q.shape[3] ** -0.5 if scale is None else scale
    out, lse = M.TokenCache(*pool).block_attention(q, table, R.i32(lens), blocks, scale=scale, with_lse=True)
    assert M.take_errors() == 0
    ref, ref_lse, weighted, big = attention_ref(pool, table, q, lens, blocks, scale)
    empty = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert (out[empty] == 0).all()
    # weights rounded to f16, as in the attention over the whole cache
    off = (out.double() - ref).abs() - R.out_bound(ref, weighted, q.dtype, R.UNIT[F16])
    assert off.max() <= 0, off.max()
    off = ((lse.double() - ref_lse).abs() - R.lse_bound(big))[~empty]
    assert not len(off) or off.max() <= 0, off.max()
    return out, lse


def random_blocks(seed, lens, queries, hkv, count, block, any_order=False):
    g = gen(seed)
    out = torch.full((len(lens), queries, hkv, count), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):
        for i in range(queries):
            have = -(-max(0, n - queries + 1 + i) // block)
            for h in range(hkv):
                x = torch.randperm(have, generator=g, device="cuda")[:count]
                x = x if any_order else x.sort().values
                to = torch.randperm(count, generator=g, device="cuda")[:len(x)] if any_order else torch.arange(len(x), device="cuda")
                out[b, i, h, to] = x.to(torch.int32)
    return out


@pytest.mark.parametrize("lens", [[1], [15, 16, 17], [0, 5, 0], [300], [64, 1, 129, 2000], [6000, 31]])
@pytest.mark.parametrize("dtype,hq,hkv,block,dim,queries", [(F16, 8, 2, 16, 64, 1), (BF16, 8, 8, 64, 128, 2), (BF16, 12, 2, 32, 96, 1),
                                                            (F16, 4, 1, 128, 48, 3)])
@pytest.mark.parametrize("count", [1, 5, 24])
def test_attention_lengths(lens, dtype, hq, hkv, block, dim, queries, count):
    pool, table, q = case(15, lens, hq, hkv, block, dim, queries, dtype)
    check_blocks(pool, table, q, lens, random_blocks(16, lens, queries, hkv, count, block))


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_attention_dimensions_in_any_order(dim, block):
    lens = [1000, 77]
    pool, table, q = case(17, lens, 6, 3, block, dim, 1, F16)
    check_blocks(pool, table, q, lens, random_blocks(18, lens, 1, 3, 13, block, any_order=True))


@pytest.mark.parametrize("hq,hkv,queries", [(1, 1, 1), (9, 1, 2), (16, 1, 1), (17, 1, 1), (64, 2, 1), (128, 1, 1), (4, 4, 5)])
def test_attention_groups(hq, hkv, queries):
    lens = [700, 3, 97]
    pool, table, q = case(19, lens, hq, hkv, 32, 128, queries, BF16)
    check_blocks(pool, table, q, lens, random_blocks(20, lens, queries, hkv, 10, 32))


@pytest.mark.parametrize("count", [255, 256, 257, 700])
def test_attention_over_long_lists(count):
    # lists that are looked up in several turns, split over several thread blocks; twice the same, bit for bit
    lens = [16 * 900 - 5, 4000]
    pool, table, q = case(21, lens, 8, 2, 16, 64, 1, BF16)
    blocks = random_blocks(22, lens, 1, 2, count, 16, any_order=True)
    one = check_blocks(pool, table, q, lens, blocks)
    two = check_blocks(pool, table, q, lens, blocks)
    assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_attention_over_all_blocks_is_the_attention():
    lens = [900, 33, 0]
    pool, table, q = case(23, lens, 8, 2, 32, 128, 3, BF16)
    cache = M.TokenCache(*pool)
    every = torch.arange(table.shape[1], dtype=torch.int32, device="cuda").expand(3, 3, 2, -1).contiguous()
    out, lse = check_blocks(pool, table, q, lens, every)
    want, want_lse, _ = cache.attention(q, table, R.i32(lens), with_lse=True)
    assert torch.allclose(out.float(), want.float(), atol=0.02, rtol=0.01)
    assert torch.allclose(lse, want_lse, atol=1e-4)


def test_attention_counts_a_column_twice_and_leaves_others_out():
    lens = [200]
    pool, table, q = case(24, lens, 4, 2, 32, 64, 1, F16)
    # (column 6 ends inside; column 7 and what is past the table's width hold no tokens)
    table = torch.nn.functional.pad(table, (0, 2), value=-1).contiguous()
    blocks = R.i32([[[[3, 3, -1, 6, 8, -9], [7, 6, 1, 6, 1, 0]]]])
    check_blocks(pool, table, q, lens, blocks)
    out, lse = M.TokenCache(*pool).block_attention(q, table, R.i32(lens), torch.full_like(blocks, -1), with_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = M.TokenCache(*pool).block_attention(q, table, R.i32(lens), blocks[..., :0].contiguous(), with_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("spread", [0.0, 6.0])
def test_attention_flat_and_peaked_with_scales_of_all_sizes(spread):
    lens = [3000, 50]
    pool, table, q = case(25, lens, 8, 2, 64, 128, 1, BF16, spread)
    pool[2][table[0, 3].long()] = 0
    pool[3][table[0, 4].long()] = 0
    pool[3][table[0, 5].long()] *= 1e4
    pool[3][table[0, 6].long()] *= 1e-6
    check_blocks(pool, table, q, lens, random_blocks(26, lens, 1, 2, 40, 64))


def test_attention_stale_slots_do_not_matter():
    lens = [100, 33]
    pool, table, q = case(27, lens, 4, 2, 32, 64, 1, BF16)
    blocks = random_blocks(28, lens, 1, 2, 4, 32)
    one = check_blocks(pool, table, q, lens, blocks)
    pool[0][table[0, 3].long(), :, 4:] = 127
    pool[1][table[0, 3].long(), :, 4:] = -128
    used = set(table[table >= 0].tolist())
    spare = [i for i in range(pool[0].shape[0]) if i not in used]
    pool[2][spare], pool[3][spare] = math.nan, math.inf
    table[1, 2:] = -7
    two = check_blocks(pool, table, q, lens, blocks)
    assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_attention_of_bad_blocks_and_lengths():
    lens = [200]
    pool, table, q = case(29, lens, 4, 2, 32, 64, 1, F16)
    cache = M.TokenCache(*pool)
    good = R.i32([[[[0, 2, 5]] * 2]])
    bad = R.i32([[[[0, 2, 5, table.shape[1], 2 ** 31 - 1]] * 2]])
    want, _ = cache.block_attention(q, table, R.i32(lens), good)
    got, _ = cache.block_attention(q, table, R.i32(lens), bad)
    assert M.take_errors() == 4 and torch.equal(got, want)
    broken = table.clone()
    broken[0, 1] = 12345
    got, _ = cache.block_attention(q, broken, R.i32(lens), R.i32([[[[0, 1, 2, 5]] * 2]]))
    assert M.take_errors() == 2 and torch.allclose(got, want, atol=1e-3)
    cache.block_attention(q, table, R.i32([10000]), good)
    assert M.take_errors() == 4
    out, lse = cache.block_attention(q, table, R.i32([-1]), good, with_lse=True)
    assert M.take_errors() == 4 and (out == 0).all() and (lse == -math.inf).all()


def test_strides_streams_and_graphs():
    lens = [900, 500]
    pool, table, q = case(30, lens, 8, 2, 32, 64, 2, F16)
    cache, at = M.TokenCache(*pool), R.i32(lens)
    bounds = cache.update_bounds(cache.empty_bounds(), table, at)

    def step(x, **kw):
        blocks = cache.choose_blocks(x, cache.update_bounds(bounds, table, at, last=2, **kw), table, at, 8, **kw)
        return (blocks, *cache.block_attention(x, table, at, blocks, with_lse=True, **kw))

    want = step(q)
    wide = torch.zeros((2, 2, 12, 64), dtype=F16, device="cuda")
    wide[:, :, 2:10] = q
    for x in (wide[:, :, 2:10], q.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3)):
        assert all(torch.equal(a, b) for a, b in zip(step(x), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(q, stream=side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(q)
    at.copy_(R.i32([333, 20]))
    graph.replay()
    want = step(q)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert M.take_errors() == 0


def test_refusals():
    lens = [900, 500]
    pool, table, q = case(31, lens, 8, 2, 32, 64, 2, F16)
    cache, at = M.TokenCache(*pool), R.i32(lens)
    bounds = cache.empty_bounds()
    blocks = torch.zeros((2, 2, 2, 4), dtype=torch.int32, device="cuda")
    for bad in (bounds.float(), bounds[:, :1], bounds[:-1], bounds.cpu(), bounds.transpose(1, 2)):
        with pytest.raises(ValueError, match="bounds"):
            cache.update_bounds(bad, table, at)
        with pytest.raises(ValueError, match="bounds"):
            cache.choose_blocks(q, bad, table, at, 4)
    for args in ((bounds, table, at.long()), (bounds, table[:1], at), (bounds, table[0], at)):
        with pytest.raises(ValueError):
            cache.update_bounds(*args)
    with pytest.raises(ValueError, match="last"):
        cache.update_bounds(bounds, table, at, last=-1)
    for count, sinks, recent in ((0, 0, 0), (4, 5, 0), (4, -1, 0), (1 << 26, 0, 0)):
        with pytest.raises(ValueError):
            cache.choose_blocks(q, bounds, table, at, count, sinks=sinks, recent=recent)
    with pytest.raises(BSearchError, match="sinks"):
        cache.choose_blocks(q, bounds, table, at, 4, sinks=3, recent=2)
    for bad in (q.float(), q[:1], q[..., :32], q.cpu()):
        with pytest.raises(ValueError):
            cache.choose_blocks(bad, bounds, table, at, 4)
        with pytest.raises(ValueError):
            cache.block_attention(bad, table, at, blocks)
    for bad in (blocks.long(), blocks[:, :1], blocks[:, :, :1], blocks.cpu(), blocks[0], blocks.transpose(0, 1)[..., ::2]):
        with pytest.raises(ValueError, match="blocks"):
            cache.block_attention(q, table, at, bad)
    with pytest.raises(BSearchError, match="scale"):
        cache.block_attention(q, table, at, blocks, scale=0.0)
    with pytest.raises(BSearchError, match="multiple"):
        cache.block_attention(q[:, :, :3].contiguous(), table, at, blocks)


def test_gradients_are_refused():
    lens = [90]
    pool, table, q = case(32, lens, 4, 2, 32, 64, 1, F16)
    cache, at = M.TokenCache(*pool), R.i32(lens)
    q.requires_grad_()
    blocks = cache.choose_blocks(q, cache.update_bounds(cache.empty_bounds(), table, at), table, at, 2)
    assert not blocks.requires_grad
    for x in cache.block_attention(q, table, at, blocks, with_lse=True):
        with pytest.raises(RuntimeError, match="no gradient"):
            x.float().sum().backward()


def test_blocks_that_are_not_there_far_on_in_a_long_row_set_a_bit():
    # a row of which a thread block has more columns than it keeps: they count as score 0 there too
    g = torch.Generator("cuda").manual_seed(31)
    width, block, dim = 400000, 16, 16
    pool = R.random_pool(g, 9, 1, block, dim)
    pool[2][8] = 0
    table = torch.randint(0, 8, (1, width), generator=g, device="cuda", dtype=torch.int32)
    q = torch.randn((1, 1, 2, dim), generator=g, device="cuda").to(F16)
    cache = M.TokenCache(*pool)
    all_blocks = torch.arange(9, device="cuda", dtype=torch.int32)[None]
    bounds = cache.update_bounds(cache.empty_bounds(), all_blocks, R.i32([9 * block]))
    lens, far = R.i32([width * block]), 49000
    table[0, far] = 8
    want = cache.choose_blocks(q, bounds, table, lens, 1000)
    assert M.take_errors() == 0
    for bad in (9, -1, 2 ** 31 - 1):
        table[0, far] = bad
        got = cache.choose_blocks(q, bounds, table, lens, 1000)
        assert M.take_errors() == 2 and torch.equal(got, want)
