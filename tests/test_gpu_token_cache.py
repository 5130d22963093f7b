"""GPU: the 8-bit token cache (writing, reading, attention, eviction) against
the operators' definitions."""
import ctypes
import math
import threading
import time

import pytest
import torch

import memory_abi as A
import memory_ref as R
from beam_search_collab_b200 import BSearchError
from beam_search_collab_b200 import memory as M

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


# ---- write and read ---------------------------------------------------------

def write_ref(pool, x, i, lens, table, start):
    """bs_cache_write's rule for one of keys (i 0) and values (1), in 32 bits:
    (codes, scales) as they should be."""
    codes, scales = pool[i].clone(), pool[2 + i].clone()
    block, a = codes.shape[2], 0
    for b, n in enumerate(lens):
        s0, new = start[b], x[a:a + n].float().transpose(0, 1)      # [heads, n, dim]
        a += n
        for c in range(s0 // block, -(-(s0 + n) // block) if n else 0):
            lo, hi = max(c * block, s0), min((c + 1) * block, s0 + n)
            at = int(table[b, c])
            part = new[:, lo - s0:hi - s0]
            top = part.abs().amax((1, 2))
            s = torch.where(top < 1e-30, torch.zeros_like(top), top / 127)
            if lo > c * block:
                old = scales[at]
                s = torch.maximum(s, old)
                ratio = torch.where(s > old, old / s, torch.ones_like(s))
                keep = codes[at, :, :lo - c * block].float()
                codes[at, :, :lo - c * block] = torch.round(keep * ratio[:, None, None]).to(torch.int8)
            inv = torch.where(s > 0, 1 / s, torch.zeros_like(s))
            codes[at, :, lo - c * block:hi - c * block] = torch.round(part * inv[:, None, None]).clamp(-127, 127).to(torch.int8)
            scales[at] = s
    return codes, scales


@pytest.mark.parametrize("block,dim,heads,dtype", [(16, 64, 2, F16), (32, 128, 4, BF16), (64, 96, 3, F16), (128, 128, 1, BF16),
                                                   (64, 16, 8, BF16), (128, 48, 2, F16)])
@pytest.mark.parametrize("lens,start", [([1], [0]), ([300, 1, 65], [0, 0, 0]), ([1, 1, 1, 1], [15, 16, 17, 200]),
                                        ([100, 0, 7, 129], [60, 30, 127, 1])])
def test_write(block, dim, heads, dtype, lens, start):
    g = gen(1)
    counts = [-(-(n + s) // block) for n, s in zip(lens, start)]
    table, _ = R.random_table(g, counts, 2)
    pool = R.random_pool(g, sum(counts) + 2, heads, block, dim)
    k, v = (torch.randn((sum(lens), heads, dim), generator=g, device="cuda") for _ in range(2))
    k = (k * torch.exp(torch.randn((sum(lens), 1, 1), generator=g, device="cuda"))).to(dtype)      # scales that grow, and not
    v = (0.3 * v).to(dtype)
    want = [write_ref(pool, x, i, lens, table, start) for i, x in ((0, k), (1, v))]
    M.TokenCache(*pool).write(k, v, R.cu(lens), table, R.i32(start))
    assert M.take_errors() == 0
    own = torch.zeros(pool[0].shape[0], pool[0].shape[2], dtype=torch.bool, device="cuda")      # slots that hold tokens
    for b, (n, s) in enumerate(zip(lens, start)):
        for p in range(n + s if n else 0):
            own[table[b, p // block].long(), p % block] = True
    for i in (0, 1):
        assert torch.equal(pool[2 + i], want[i][1])
        mine, ref = pool[i].transpose(1, 2)[own], want[i][0].transpose(1, 2)[own]
        assert torch.equal(mine, ref)


def test_write_of_zeros_and_small_values():
    cache = M.TokenCache.empty(2, 1, 32, block=16)
    k = torch.zeros((3, 1, 32), dtype=BF16, device="cuda")
    v = torch.full((3, 1, 32), 1e-36, dtype=BF16, device="cuda")
    cache.write(k, v, R.cu([3]), R.i32([[1]]), R.i32([0]))
    assert cache.k_scale[1, 0] == 0 and cache.v_scale[1, 0] == 0 and (cache.k[1] == 0).all() and (cache.v[1] == 0).all()
    out, lse, _ = cache.attention(torch.ones((1, 1, 2, 32), dtype=BF16, device="cuda"), R.i32([[1]]), R.i32([3]), with_lse=True)
    assert (out == 0).all() and torch.allclose(lse, torch.full_like(lse, math.log(3)))
    # a block that starts anew forgets its old scale
    cache.k_scale.fill_(5.0)
    cache.write(torch.ones_like(k), v, R.cu([3]), R.i32([[1]]), R.i32([0]))
    assert cache.k_scale[1, 0] == torch.tensor(1.0) / 127


def test_written_values_come_back_within_half_a_step():
    g = gen(2)
    lens, block = [500, 37], 64
    table, _ = R.random_table(g, [8, 1])
    cache = M.TokenCache.empty(9, 4, 128, block=block)
    k, v = (torch.randn((537, 4, 128), generator=g, device="cuda").to(BF16) for _ in range(2))
    cache.write(k, v, R.cu(lens), table, R.i32([0, 0]))
    places = torch.arange(500, dtype=torch.int32, device="cuda").repeat(2, 1)
    for got, x, scale in zip(cache.read(table, R.i32(lens), places), (k, v), (cache.k_scale, cache.v_scale)):
        for b, (a, n) in enumerate(((0, 500), (500, 37))):
            step = scale[table[b, :-(-n // block)].long()].repeat_interleave(block, 0)[:n]        # [n, heads]
            off = (got[b, :, :n].transpose(0, 1) - x[a:a + n].float()).abs()
            assert (off <= 0.5001 * step[..., None]).all()
            assert (got[b, :, n:] == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_read_places(dtype):
    g = gen(3)
    pool = R.random_pool(g, 7, 3, 32, 48)
    table, _ = R.random_table(g, [4, 3])
    lens = [120, 70]
    cache = M.TokenCache(*pool)
    places = torch.randint(-3, 140, (2, 3, 50), generator=g, device="cuda", dtype=torch.int32)
    k, v = cache.read(table, R.i32(lens), places, dtype=dtype)
    assert M.take_errors() == 0
    for b in range(2):
        for h in range(3):
            for i, got in ((0, k), (1, v)):
                all_ = R.held(pool, table, b, lens[b], h, i).float()
                p = places[b, h].long()
                ok = (p >= 0) & (p < lens[b])
                want = torch.where(ok[:, None], all_[p.clamp(0, lens[b] - 1)], torch.zeros(()).cuda()).to(dtype)
                assert torch.equal(got[b, h], want)
    shared = places[:, 1]                                   # one list for all heads, rows apart
    k2, none = cache.read(table, R.i32(lens), shared, dtype=dtype, values=False)
    assert none is None and torch.equal(k2[:, 1], k[:, 1])


# ---- attention --------------------------------------------------------------

def attention_case(seed, lens, hq, hkv, block, dim, queries, dtype, spread=1.0):
    g = gen(seed)
    counts = [max(1, -(-n // block)) for n in lens]
    table, _ = R.random_table(g, counts, 1)
    pool = R.random_pool(g, sum(counts) + 1, hkv, block, dim)
    q = (spread * torch.randn((len(lens), queries, hq, dim), generator=g, device="cuda")).to(dtype)
    return pool, table, q


def check_attention(pool, table, q, lens, mass=None, scale=None):
    scale = q.shape[3] ** -0.5 if scale is None else scale
    out, lse, got = M.TokenCache(*pool).attention(q, table, R.i32(lens), scale=scale, with_lse=True, mass=mass, with_mass=True)
    assert M.take_errors() == 0
    ref, ref_lse, ref_mass, weighted, big = R.cache(pool, q, table, lens, scale)
    empty = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert (out[empty] == 0).all()
    off = (out.double() - ref).abs() - R.out_bound(ref, weighted, q.dtype, R.UNIT[F16])
    assert off.max() <= 0, off.max()
    off = ((lse.double() - ref_lse).abs() - R.lse_bound(big))[~empty]
    assert not len(off) or off.max() <= 0, off.max()
    width = got.shape[2]
    full = torch.zeros(got.shape, dtype=torch.float64, device="cuda")
    full[:, :, :min(width, ref_mass.shape[2])] = ref_mass[:, :, :width]
    if mass is not None:
        full += torch.where(torch.arange(width, device="cuda") < R.i32(lens)[:, None, None], mass.double(), 0.0)
    off = (got.double() - full).abs() - R.mass_bound(full, big.max())
    assert off.max() <= 0, off.max()
    return out, lse, got


@pytest.mark.parametrize("lens", [[1], [15, 16, 17], [0, 5, 0], [300], [64, 1, 129, 2000], [6000, 31]])
@pytest.mark.parametrize("dtype,hq,hkv,block,dim", [(F16, 8, 2, 16, 64), (BF16, 8, 8, 64, 128), (BF16, 12, 2, 32, 96),
                                                    (F16, 4, 1, 128, 48)])
def test_attention_lengths(lens, dtype, hq, hkv, block, dim):
    pool, table, q = attention_case(4, lens, hq, hkv, block, dim, 1, dtype)
    check_attention(pool, table, q, lens)


@pytest.mark.parametrize("hq,hkv,queries", [(1, 1, 1), (3, 1, 1), (16, 1, 1), (17, 1, 1), (64, 2, 1), (128, 1, 1), (4, 4, 2),
                                            (8, 2, 4), (6, 2, 5), (12, 4, 9), (8, 1, 33)])
def test_attention_groups_and_drafts(hq, hkv, queries):
    lens = [200, 3, 1, 97]
    pool, table, q = attention_case(5, lens, hq, hkv, 32, 128, queries, BF16)
    check_attention(pool, table, q, lens)


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_attention_dimensions(dim, block):
    lens = [260, 77]
    pool, table, q = attention_case(6, lens, 6, 3, block, dim, 1, F16)
    check_attention(pool, table, q, lens)


def test_attention_many_and_long():
    lens = [40000, 1, 12345, 0, 7, 640]
    pool, table, q = attention_case(7, lens, 8, 2, 64, 128, 1, BF16)
    mass = torch.rand((6, 2, 40000), device="cuda")
    one = check_attention(pool, table, q, lens, mass)
    two = check_attention(pool, table, q, lens, mass)
    assert all(torch.equal(a, b) for a, b in zip(one, two))          # the same every time


@pytest.mark.parametrize("spread", [0.0, 6.0])
def test_attention_flat_and_peaked(spread):
    lens = [3000, 50]
    pool, table, q = attention_case(8, lens, 8, 2, 64, 128, 1, BF16, spread)
    check_attention(pool, table, q, lens)


def test_attention_scales_of_zero_and_of_all_sizes():
    lens = [500]
    pool, table, q = attention_case(9, lens, 4, 2, 32, 64, 1, F16)
    pool[2][table[0, 3].long()] = 0                  # keys of zeros: score 0
    pool[3][table[0, 4].long()] = 0                  # values of zeros keep their weight
    pool[3][table[0, 5].long()] *= 1e4
    pool[3][table[0, 6].long()] *= 1e-6
    check_attention(pool, table, q, lens)


def test_attention_large_and_small_queries():
    lens = [400]
    pool, table, q = attention_case(10, lens, 4, 2, 32, 64, 1, BF16)
    check_attention(pool, table, (q.float() * 2.0 ** 40).to(BF16), lens, scale=2.0 ** -43)
    check_attention(pool, table, (q.float() * 2.0 ** -60).to(BF16), lens, scale=2.0 ** 57)


def test_attention_stale_blocks_and_slots_do_not_matter():
    lens = [100, 33]
    pool, table, q = attention_case(11, lens, 4, 2, 32, 64, 1, BF16)
    one = check_attention(pool, table, q, lens)
    pool[0][table[0, 3].long(), :, 4:] = 127          # behind the last token
    pool[1][table[0, 3].long(), :, 4:] = -128
    used = set(table[table >= 0].tolist())
    spare = [i for i in range(pool[0].shape[0]) if i not in used]
    pool[2][spare], pool[3][spare] = math.nan, math.inf
    table[1, 2:] = -7
    two = check_attention(pool, table, q, lens)
    assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_attention_strided_queries_in_place_mass_and_streams():
    lens = [300, 9]
    pool, table, q = attention_case(12, lens, 8, 2, 64, 64, 3, F16)
    wide = torch.zeros((2, 3, 12, 64), dtype=F16, device="cuda")
    wide[:, :, 2:10] = q
    mass = torch.rand((2, 2, 320), device="cuda")
    cache, at = M.TokenCache(*pool), R.i32(lens)
    a, la, ma = cache.attention(q, table, at, with_lse=True, mass=mass)
    b, lb, mb = cache.attention(wide[:, :, 2:10], table, at, with_lse=True, mass=mass)
    assert torch.equal(a, b) and torch.equal(la, lb) and torch.equal(ma, mb)
    c, none, mc = cache.attention(q.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3), table, at, mass=mass, out_mass=mass)
    assert none is None and mc is mass and torch.equal(mass, ma) and torch.equal(a, c)
    assert cache.attention(q, table, at)[1:] == (None, None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    d, ld, _ = cache.attention(q, table, at, with_lse=True, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(a, d) and torch.equal(la, ld)


def test_attention_in_a_graph_follows_the_lengths():
    lens = [300, 9, 64]
    pool, table, q = attention_case(13, [600, 600, 600], 8, 2, 64, 64, 1, F16)
    cache, at = M.TokenCache(*pool), R.i32(lens)
    cache.attention(q, table, at, with_lse=True, with_mass=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse, mass = cache.attention(q, table, at, with_lse=True, with_mass=True)
    for now in (lens, [1, 599, 0]):
        at.copy_(R.i32(now))
        graph.replay()
        want = cache.attention(q, table, R.i32(now), with_lse=True, with_mass=True)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((out, lse, mass), want))
    del graph


def test_offsets_past_32_bits():
    # a pool of 5 GB of keys: the blocks used lie at its end
    heads, block, dim = 8, 64, 128
    blocks = 5 * 2 ** 30 // (heads * block * dim)
    g = gen(14)
    small = R.random_pool(g, 4, heads, block, dim)
    pool = [torch.zeros((blocks, heads, block, dim), dtype=torch.int8, device="cuda") for _ in range(2)]
    pool += [torch.zeros((blocks, heads), device="cuda") for _ in range(2)]
    table = R.i32([[blocks - 1, 3, blocks - 4]])
    for j, at in enumerate(table[0].tolist()):
        for i in range(4):
            pool[i][at] = small[i][j]
    q = torch.randn((1, 1, 16, dim), generator=g, device="cuda").to(BF16)
    little = R.i32([[0, 1, 2]])
    big, cache = M.TokenCache(*pool), M.TokenCache(*small)
    a = big.attention(q, table, R.i32([170]), with_lse=True, with_mass=True)
    b = cache.attention(q, little, R.i32([170]), with_lse=True, with_mass=True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    k = torch.randn((5, heads, dim), generator=g, device="cuda").to(BF16)
    big.write(k, k, R.cu([5]), table, R.i32([170]))
    cache.write(k, k, R.cu([5]), little, R.i32([170]))
    places = torch.arange(175, dtype=torch.int32, device="cuda")[None]
    for x, y in zip(big.read(table, R.i32([175]), places), cache.read(little, R.i32([175]), places)):
        assert torch.equal(x, y)
    mass = torch.rand((1, heads, 175), generator=g, device="cuda")
    a = big.evict(mass, table, R.i32([175]), R.i32([[blocks - 7, blocks - 9]]), 100)
    b = cache.evict(mass, little, R.i32([175]), R.i32([[3, 2]])[:, :1].contiguous(), 64)
    assert M.take_errors() == 0 and torch.equal(a[0][0, :, :4], b[0][0, :, :4])
    got = big.read(R.i32([[blocks - 7, blocks - 9]]), a[1], a[0].new_zeros((1, 100)) + torch.arange(100, device="cuda", dtype=torch.int32))
    rows = big.read(table, R.i32([175]), a[0])
    step = big.k_scale.max()
    assert (got[0] - rows[0]).abs().max() <= 0.5001 * step


def test_bad_ids_and_lengths_set_error_bits():
    lens = [100, 33]
    pool, table, q = attention_case(15, lens, 4, 2, 32, 64, 1, BF16)
    cache, at = M.TokenCache(*pool), R.i32(lens)
    good = cache.attention(q, table, at, with_lse=True, with_mass=True)
    bad = table.clone()
    bad[0, 1] = pool[0].shape[0]
    cache.attention(q, bad, at, with_mass=True)
    assert M.take_errors() == 2
    cache.attention(q, table, R.i32([100, 100000]), with_mass=True)
    assert M.take_errors() & 4
    cache.attention(q, table, R.i32([-1, 33]))
    assert M.take_errors() == 4
    x = torch.zeros((2, 2, 64), dtype=BF16, device="cuda")
    before = [p.clone() for p in pool]
    cache.write(x, x, R.cu([1, 1]), bad[:, 1:2].contiguous(), R.i32([0, 64]))
    assert M.take_errors() & 2
    cache.write(x, x, R.i32([0, 3, 2]), table, R.i32([0, 0]))
    assert M.take_errors() & 4
    for p, b in zip(pool, before):
        p.copy_(b)
    cache.read(bad, at, R.i32([[40], [0]]))
    assert M.take_errors() == 2
    mass = torch.rand((2, 2, 128), device="cuda")
    cache.evict(mass, table, R.i32([4000, 3]), R.i32([[-1], [-1]]), 32)
    assert M.take_errors() == 6
    for p, b in zip(pool, before):
        assert torch.equal(p, b)
    again = cache.attention(q, table, at, with_lse=True, with_mass=True)
    assert M.take_errors() == 0 and all(torch.equal(x, y) for x, y in zip(good, again))


# ---- eviction ---------------------------------------------------------------

def evict_ref(mass, lens, budget, sinks, recent):
    kept = torch.full(mass.shape[:2] + (budget,), -1, dtype=torch.int32, device=mass.device)
    new = torch.zeros(mass.shape[:2] + (budget,), device=mass.device)
    for b, n in enumerate(lens):
        for h in range(mass.shape[1]):
            m = mass[b, h, :n].tolist()
            stay = range(n)
            if n > budget:
                free = range(sinks, n - recent)
                rank = sorted(free, key=lambda j: (not math.isnan(m[j]), -m[j] if not math.isnan(m[j]) else 0.0, j))
                stay = sorted([*range(sinks), *rank[:budget - sinks - recent], *range(n - recent, n)])
            at = R.i32(list(stay))
            kept[b, h, :len(at)], new[b, h, :len(at)] = at, mass[b, h, at.long()]
    return kept, R.i32([min(n, budget) for n in lens]), new


def check_evict(lens, budget, sinks, recent, block=32, dim=64, heads=2, mass=None, seed=20):
    g = gen(seed)
    counts = [max(1, -(-n // block)) for n in lens]
    width = -(-min(budget, max(max(lens), 1)) // block)
    table, free = R.random_table(g, counts, len(lens) * width)
    pool = R.random_pool(g, sum(counts) + len(lens) * width, heads, block, dim)
    new_table = free.view(len(lens), width).contiguous()
    if mass is None:
        mass = torch.rand((len(lens), heads, max(max(lens), 1)), generator=g, device="cuda") ** 6
    before = [p.clone() for p in pool]
    cache = M.TokenCache(*pool)
    kept, new_lens, new_mass = cache.evict(mass, table, R.i32(lens), new_table, budget, sinks=sinks, recent=recent)
    assert M.take_errors() == 0
    want = evict_ref(mass, lens, budget, sinks, recent)
    assert torch.equal(kept, want[0]) and torch.equal(new_lens, want[1])
    assert torch.equal(torch.nan_to_num(new_mass, 7.5), torch.nan_to_num(want[2], 7.5))
    for b, n in enumerate(new_lens.tolist()):
        for h in range(heads):
            at = kept[b, h, :n].long()
            src = table[b, at // block].long()
            for i in (0, 1):
                old = before[2 + i][src, h]
                top = torch.nn.functional.pad(old, (0, -n % block)).view(-1, block).amax(1)
                per = top.repeat_interleave(block)[:n]
                code = torch.round(before[i][src, h, at % block].float() * (old / per)[:, None])
                to = new_table[b, :-(-n // block)].long()
                assert torch.equal(pool[i][to, h].reshape(-1, dim)[:n].float(), code)
                assert torch.equal(pool[2 + i][to, h], top)
    used = torch.ones(pool[0].shape[0], dtype=torch.bool, device="cuda")
    used[new_table.flatten().long()] = False
    for p, q in zip(pool, before):
        assert torch.equal(p[used], q[used])                 # the old blocks are as they were


@pytest.mark.parametrize("lens", [[100, 64, 65, 63, 0, 1], [1000, 3000], [33]])
@pytest.mark.parametrize("budget,sinks,recent", [(64, 4, 16), (64, 0, 0), (64, 32, 32), (1, 0, 0), (1, 0, 1), (33, 1, 0)])
def test_evict(lens, budget, sinks, recent):
    check_evict(lens, budget, sinks, recent)


@pytest.mark.parametrize("block,dim,heads", [(16, 128, 1), (64, 96, 3), (128, 128, 2), (128, 16, 2)])
def test_evict_layouts(block, dim, heads):
    check_evict([700, 333], 200, 3, 10, block, dim, heads)


def test_evict_long():
    check_evict([70001, 20000], 9001, 4, 128)


def test_evict_ties_and_odd_weights():
    n = 3000
    g = gen(21)
    few = torch.randint(0, 3, (1, 2, n), generator=g, device="cuda").float()          # many equal
    check_evict([n], 1500, 4, 64, mass=few)
    check_evict([n], 1234, 0, 0, mass=torch.zeros((1, 2, n), device="cuda"))          # all equal
    odd = torch.randn((1, 2, n), generator=g, device="cuda")
    odd[0, 0, ::5], odd[0, 0, 1::7], odd[0, 1, ::3], odd[0, 1, 1::3] = math.inf, math.nan, -math.inf, -0.0
    odd[0, 1, 2::6] = 0.0
    check_evict([n], 700, 1, 1, mass=odd)
    check_evict([n], 2500, 1, 1, mass=odd)
    check_evict([n], 5, 0, 0, mass=-torch.rand((1, 2, n), generator=g, device="cuda"))


def test_cache_refusals():
    pool, table, q = attention_case(30, [50], 4, 2, 32, 64, 1, F16)
    cache, at = M.TokenCache(*pool), R.i32([50])
    with pytest.raises(ValueError, match="int8"):
        M.TokenCache(pool[0].float(), *pool[1:])
    with pytest.raises(ValueError, match="like k"):
        M.TokenCache(pool[0], pool[1][:1], *pool[2:])
    with pytest.raises(ValueError, match="scales"):
        M.TokenCache(pool[0], pool[1], pool[2].half(), pool[3])
    with pytest.raises(BSearchError, match="16, 32, 64 or 128"):
        M.TokenCache.empty(2, 2, 64, block=24).attention(q, table, at)
    with pytest.raises(ValueError, match="queries, q_heads, dim"):
        cache.attention(q[..., :32], table, at)
    with pytest.raises(ValueError, match="table"):
        cache.attention(q, table.long(), at)
    with pytest.raises(ValueError, match="mass"):
        cache.attention(q, table, at, mass=torch.zeros((1, 2, 64), device="cuda").half())
    with pytest.raises(BSearchError, match="multiple of kv_heads"):
        cache.attention(q[:, :, :3], table, at)
    x = torch.zeros((1, 2, 64), dtype=F16, device="cuda")
    with pytest.raises(ValueError, match="of the cache"):
        cache.write(x[:, :1], x[:, :1], R.cu([1]), table, at)
    with pytest.raises(ValueError, match="positions"):
        cache.read(table, at, torch.zeros((1, 3, 4), dtype=torch.int32, device="cuda"))
    mass = torch.zeros((1, 2, 64), device="cuda")
    with pytest.raises(BSearchError, match="sinks"):
        cache.evict(mass, table, at, table, 8, sinks=5, recent=4)
    with pytest.raises(BSearchError, match="room"):
        cache.evict(mass, table, at, torch.zeros((1, 0), dtype=torch.int32, device="cuda"), 8)
    with pytest.raises(ValueError, match="budget"):
        cache.evict(mass, table, at, table, 0)
    assert M.take_errors() == 0


def test_merge_joins_disjoint_sets():
    lens = [500]
    pool, table, q = attention_case(31, lens, 4, 2, 32, 64, 1, F16)
    cache = M.TokenCache(*pool)
    whole, lse, _ = cache.attention(q, table, R.i32([500]), with_lse=True)
    a = cache.attention(q, table[:, :5].contiguous(), R.i32([160]), with_lse=True)
    b = cache.attention(q, table[:, 5:].contiguous(), R.i32([340]), with_lse=True)
    c = cache.attention(q, table, R.i32([0]), with_lse=True)
    out, joined = M.merge([a[0], b[0], c[0]], [a[1], b[1], c[1]])
    assert (out - whole).abs().max() <= 4 * R.UNIT[F16] * whole.abs().max() and (joined - lse).abs().max() <= 1e-5


# ---- streams ----------------------------------------------------------------

def side_calls():
    """Calls by name: what to do on a stream, the cache's buffers it changes."""
    g = gen(60)
    pool, table, q = attention_case(60, [300, 90], 8, 2, 64, 64, 1, F16)
    cache, lens, new_table = M.TokenCache(*pool), R.i32([300, 90]), R.i32([[7, 8], [9, 10]])
    wide = M.TokenCache(*R.random_pool(g, 11, 2, 64, 64))
    x = torch.randn((711, 8, 64), generator=g, device="cuda").to(F16)
    cu, places, mass = R.cu([300, 411]), torch.arange(300, dtype=torch.int32, device="cuda").repeat(2, 1), torch.rand((2, 2, 300), device="cuda")
    cut_q, cut_k = R.cu([20]), R.cu([711])                   # several pieces of keys: a workspace
    torch.cuda.synchronize()
    return {"prompt": lambda s: M.prompt_attention(x, x[:, :2], x[:, 2:4], cu, with_lse=True, stream=s),
            "pieces": lambda s: M.prompt_attention(x[:20, :1], x[:, :1], x[:, 1:2], cut_q, cut_k, with_lse=True, stream=s),
            "read": lambda s: cache.read(table, lens, places, stream=s),
            "attention": lambda s: cache.attention(q, table, lens, with_lse=True, mass=mass, stream=s),
            "evict": lambda s: wide.evict(mass, table, lens, new_table, 100, stream=s)}


@pytest.mark.parametrize("name", ["prompt", "pieces", "read", "attention", "evict"])
def test_memory_of_a_call_on_a_side_stream_is_not_in_use_elsewhere(name):
    call = side_calls()[name]
    side = torch.cuda.Stream()
    want = call(side.cuda_stream)
    side.synchronize()
    want = [t.clone() for t in want]
    torch.cuda.synchronize()
    # freed on the current stream, which still has to write to it
    freed = [torch.empty_like(t).fill_(0) for t in want] + [torch.zeros(2 ** 21 * i, dtype=torch.uint8, device="cuda") for i in (1, 2, 4)]
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    for t in freed:
        t.fill_(7)
    del t, freed
    got = call(side.cuda_stream)                         # (the writes are still to come)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_inputs_of_a_call_on_a_side_stream_may_be_dropped_at_once():
    g = gen(61)
    side = torch.cuda.Stream()
    q, k, v = (torch.randn((500, 4, 64), generator=g, device="cuda").to(F16) for _ in range(3))
    want, _ = M.prompt_attention(q, k, v, R.cu([200, 300]))
    side.wait_stream(torch.cuda.current_stream())
    M.prompt_attention(q, k, v, R.cu([200, 300]), stream=side.cuda_stream)      # (what loads kernels or asks the driver for
    mine, at = [t.clone() for t in (q, k, v)], R.cu([200, 300])
    fill = lambda n: [torch.full_like(q, 3.0) for _ in range(n)] + [torch.full_like(at, 99) for _ in range(n)]  # noqa: E731
    keep = fill(12)                                                              # memory may wait for the GPU)
    del keep
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
    got, _ = M.prompt_attention(*mine, at, stream=side.cuda_stream)
    at = at.new_empty(3)                                 # (the first one is dropped)
    del mine
    again = fill(6)                                      # (what was dropped is still to be read)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and M.take_errors() == 0
    del again


def test_error_bits_of_another_stream_are_not_lost():
    # a kernel on a side stream sets a bit while the errors are taken: by this call or the next
    pool, table, q = attention_case(62, [40], 4, 2, 32, 64, 1, F16)
    cache, bad, lens, places = M.TokenCache(*pool), R.i32([[pool[0].shape[0], 0]]), R.i32([40]), R.i32([[3]])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(600):
        M.prompt_attention(q[0], q[0, :, :2], q[0, :, :2], R.cu([1]), R.i32([0, 2]))      # another bit: there is something to clear
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(1000 + 50 * i)             # the bit is set 1 to 16 us after the call, or a little later
        cache.read(bad, lens, places, stream=side.cuda_stream)
        first = M.take_errors()
        side.synchronize()
        assert first & 4 and first | M.take_errors() == 6, i


def test_other_threads_run_while_errors_are_waited_for():
    M.take_errors()
    at, done = [], threading.Event()

    def tick():
        while not done.wait(0.001):
            at.append(time.monotonic())
    thread = threading.Thread(target=tick)
    thread.start()
    torch.cuda._sleep(600_000_000)                       # 0.3 s
    began = time.monotonic()
    M.take_errors()
    ended = time.monotonic()
    done.set()
    thread.join()
    assert ended - began > 0.1 and sum(began < x < ended for x in at) >= 10


def test_weights_without_a_place_set_an_error_bit():
    lens = [100, 33]
    pool, table, q = attention_case(42, lens, 4, 2, 32, 64, 1, BF16)
    cache = M.TokenCache(*pool)
    mass = torch.rand((2, 2, 128), device="cuda")
    _, _, whole = cache.attention(q, table, R.i32(lens), mass=mass)
    assert M.take_errors() == 0
    for width, flags in ((100, 0), (99, 4), (64, 4)):
        _, _, got = cache.attention(q, table, R.i32(lens), mass=mass[:, :, :width].contiguous())
        assert M.take_errors() == flags and torch.equal(got, whole[:, :, :width])


# ---- small weights ----------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("nats", [8, 11, 14, 17])
def test_attention_small_weights_beside_a_large_one_and_a_large_scale(nats, dtype):
    # one token without values has most of the weight, all others e^-nats of its; one block has 50 times the others' value scale
    g = gen(40)
    pool = R.random_pool(g, 16, 2, 64, 64)
    table, _ = R.random_table(g, [16])
    at = table[0].long()
    pool[0].zero_(), pool[1].clamp_(min=0), pool[2].fill_(0.01), pool[3].fill_(0.01)
    pool[0][at[0], :, 0], pool[1][at[0], :, 0] = 100, 0
    pool[1][at[2]], pool[3][at[2]] = 0, 0.5
    q, scale = torch.ones((1, 1, 8, 64), dtype=dtype, device="cuda"), nats / 64.0
    out, _, _ = M.TokenCache(*pool).attention(q, table, R.i32([1024]), scale=scale)
    ref, _, _, weighted, _ = R.cache(pool, q, table, [1024], scale)
    # the result's rounding, a weight's and its score's, and half a step of f16's smallest numbers at 2^5 for the largest
    codes = pool[1][at].double().abs().sum((0, 2)).repeat_interleave(4, 0)
    bound = R.UNIT[dtype] * ref.abs() + (R.UNIT[F16] + 2.0 ** -12) * (1 + 2.0 ** -7) * weighted + 2.0 ** -30 * 0.5 * codes
    assert ((out.double() - ref).abs() <= bound).all()



def test_dimensions_past_32_bits_are_refused():
    cache, at = M.TokenCache.empty(2, 1, 16, block=16), R.i32([0])
    x = torch.zeros((1, 1, 16), dtype=F16, device="cuda").expand(2 ** 32 + 1, 1, 16)          # 1 row in 32 bits
    with pytest.raises(ValueError, match="2\\^31"):
        cache.write(x, x, R.cu([1]), R.i32([[0]]), at)
    with pytest.raises(ValueError, match="2\\^31"):
        M.prompt_attention(x[:1], x, x, R.cu([1]), R.cu([1]))
    many = torch.zeros((1, 2 ** 32 + 1), dtype=torch.int32, device="cuda")                    # (17 GB)
    with pytest.raises(ValueError, match="2\\^31"):
        cache.read(R.i32([[0]]), R.i32([1]), many, keys=False, values=False)
    with pytest.raises(ValueError, match="2\\^31"):
        cache.attention(x[:1, None], many, R.i32([1]))
    del many


def test_backward_through_an_output_raises():
    pool, table, q = attention_case(63, [50], 4, 2, 32, 64, 1, F16)
    cache, at, mass = M.TokenCache(*pool), R.i32([50]), torch.rand((1, 2, 64), device="cuda")
    k = torch.randn((5, 2, 64), device="cuda").to(F16)
    plain = [*M.prompt_attention(q[0], k, k, R.cu([1]), R.cu([5]), with_lse=True), *cache.attention(q, table, at, with_lse=True, mass=mass)]
    assert not any(t.requires_grad for t in plain)
    k.requires_grad_(), mass.requires_grad_()
    some = [*M.prompt_attention(q[0], k, k, R.cu([1]), R.cu([5]), with_lse=True), cache.attention(q, table, at, mass=mass)[2]]
    spare = ({0, 1, 2} - set(table[0].tolist())).pop()
    some.append(cache.evict(mass, table, at, R.i32([[spare]]), 32)[2])
    q.requires_grad_()
    some += cache.attention(q, table, at, with_lse=True, with_mass=True)
    for t in some:
        with pytest.raises(RuntimeError, match="no gradient"):
            (t.float().sum() + q.float().sum()).backward()
    same = [*M.prompt_attention(q[0], k, k, R.cu([1]), R.cu([5]), with_lse=True), *cache.attention(q, table, at, with_lse=True, mass=mass)]
    assert all(torch.equal(a, b) for a, b in zip(plain, same))
    with torch.no_grad():
        assert not any(t.requires_grad for t in cache.attention(q, table, at, with_lse=True, mass=mass))


# ---- workspaces -------------------------------------------------------------

def test_many_query_rows_need_little_workspace():
    c = A._Cache(None, None, None, None, 1000, 1, 64, 128)
    for queries, q_heads in ((1024, 128), (1024, 1), (16, 128), (3, 128)):
        d, n = A._Attention(queries=queries, q_heads=q_heads, num_seqs=4, table_width=2048, dtype=1, scale=1.0), ctypes.c_size_t()
        assert A._lib().bs_cache_attention_workspace(c, d, n) == 0
        assert n.value < 160e6, (queries, q_heads, n.value)


@pytest.mark.parametrize("queries,hq", [(64, 128), (300, 128), (1000, 3)])
def test_attention_many_query_rows(queries, hq):
    lens = [1100, 2000, 30]
    pool, table, q = attention_case(64, lens, hq, 1, 64, 64, queries, BF16)
    check_attention(pool, table, q, lens)


# ---- branches that other sizes do not reach ---------------------------------

@pytest.mark.parametrize("block,dim", [(16, 64), (64, 128), (128, 96)])
def test_write_of_strided_rows(block, dim):
    # slices of a fused projection, heads outermost, one row or head for all
    g = gen(50)
    lens, start, heads = [100, 0, 7, 129], [60, 30, 127, 1], 3
    counts = [-(-(n + s) // block) for n, s in zip(lens, start)]
    table, _ = R.random_table(g, counts, 2)
    pool = R.random_pool(g, sum(counts) + 2, heads, block, dim)
    x = torch.randn((236, 12, dim), generator=g, device="cuda").to(BF16)
    fused = x[:, 6:9], x[:, 9:]
    outermost = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in fused]
    same = x[:, 6:7].expand(-1, 3, -1), x[:1, 9:].expand(236, -1, -1)
    for k, v in (fused, outermost, same):
        one, two = [p.clone() for p in pool], [p.clone() for p in pool]
        M.TokenCache(*one).write(k, v, R.cu(lens), table, R.i32(start))
        M.TokenCache(*two).write(k.contiguous(), v.contiguous(), R.cu(lens), table, R.i32(start))
        assert M.take_errors() == 0 and all(torch.equal(a, b) for a, b in zip(one, two))


@pytest.mark.parametrize("n_seqs,heads,n", [(1, 1, 400000), (20, 8, 50001)])
def test_evict_rows_that_shared_memory_does_not_hold(n_seqs, heads, n):
    # more than 47,104 keys for a block: one row over a cluster of 8, and so many rows that each has one block
    g = gen(53)
    budget, sinks, recent, block, dim = 777, 4, 100, 128, 16
    mass = torch.rand((n_seqs, heads, n), generator=g, device="cuda")
    mass[:, 0] = torch.round(mass[:, 0] * 1000)              # equal ones at the threshold
    lens = [n - 13 * i for i in range(n_seqs)]
    table = torch.randint(0, 50, (n_seqs, -(-n // block)), generator=g, device="cuda").to(torch.int32)
    new_table = (50 + torch.arange(n_seqs * 7, device="cuda")).view(n_seqs, 7).to(torch.int32)
    cache = M.TokenCache(*R.random_pool(g, 50 + n_seqs * 7, heads, block, dim))
    kept, new_lens, new_mass = cache.evict(mass, table, R.i32(lens), new_table, budget, sinks=sinks, recent=recent)
    assert M.take_errors() == 0 and (new_lens == budget).all()
    for b, m in enumerate(lens):
        best = torch.sort(mass[b, :, sinks:m - recent], dim=1, descending=True, stable=True).indices
        ends = torch.cat((torch.arange(sinks, device="cuda"), torch.arange(m - recent, m, device="cuda"))).repeat(heads, 1)
        want = torch.cat((best[:, :budget - sinks - recent] + sinks, ends), 1).sort(1).values
        assert torch.equal(kept[b].long(), want) and torch.equal(new_mass[b], mass[b].gather(1, want))
