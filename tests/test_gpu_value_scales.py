"""GPU: value scales of all sizes in one cache.  Blocks whose value scale is far below another's keep their bits where that
other one gets no weight, in every attention over the cache."""
import pytest
import torch

import memory_ref as R
import test_gpu_shared_attention as S
from beam_search_collab_b200 import memory as M

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def prepare(pool, q, outliers, ratio, spread):
    """The blocks `outliers` have values `ratio` times the others' and scores of about -250, the others' are `spread` and less."""
    pool[0][..., 0] = 0
    pool[0][outliers, :, :, 0] = -127
    pool[2][:] = 0.01
    pool[3][:] = 0.01
    pool[3][outliers] = 0.01 * ratio
    q *= spread * (16 / q.shape[-1]) ** 0.5 / 2
    q[..., 0] = 200


def reference(pool, q, rows):
    """(out, what its elements are sums of, what f16 takes of that) in 64 bits; rows[b]: the blocks of sequence b's tokens and how
    many of each, in order.  f16 holds a weight times its value scale to half of 2^-24 where the largest such product of the row
    counts 2^5 and more: to 2^-30 of that one (2^-29 here), or it is lost whole."""
    n, _, hq, dim = q.shape
    hkv = pool[0].shape[1]
    g = hq // hkv
    out, weighted, lost = (torch.zeros((n, 1, hq, dim), dtype=torch.float64, device="cuda") for _ in range(3))
    for b, (ids, held) in enumerate(rows):
        for h in range(hkv):
            k, v = ((pool[i][ids, h].double() * pool[2 + i][ids, h].double()[:, None, None])[held] for i in (0, 1))
            s = pool[3][ids, h].double()[:, None].expand(held.shape)[held]
            s = s.clamp(min=2.0 ** -60 * s.max())                # (as far down as scales count; of 0 too)
            at = (b, 0, slice(h * g, h * g + g))
            out[at], _, w, weighted[at], _ = R.attend(q[at].double(), k, v, 1.0, torch.full((g,), len(k), device="cuda"))
            lost[at] = torch.minimum(w, 2.0 ** -29 * (w * s).amax(1, keepdim=True) / s) @ v.abs()
    return out, weighted, lost


def tokens(table, n, block):
    ids = table[:-(-n // block)].long()
    return ids, torch.arange(len(ids) * block, device="cuda").view(-1, block) < n


def check(out, ref, weighted, lost):
    # no more than each element's own: the output's rounding, the weights' to f16 and 2^-12 for exponentials and scores, of what the
    # element is a sum of, and what f16 loses of it (no part of the others' size, but half of f16's smallest step)
    size = (R.UNIT[out.dtype] * ref.abs() + (R.UNIT[F16] + 2.0 ** -12) * weighted * (1 + 2.0 ** -7) + lost +
            (2.0 ** -25 if out.dtype == F16 else 0))
    # (f16 rounds to infinity from 65520 on: one is right where the element is as large within its bound)
    right = torch.isinf(out) & (ref.sign() == out.sign()) & (ref.abs() + size >= 65520) & (out.dtype == F16)
    off = torch.where(right, -size, (out.double() - ref).abs() - size)
    assert off.max() <= 0, off.max()


SIZES = [(64, 32, 8, 2), (128, 16, 8, 8), (48, 128, 20, 1), (128, 64, 32, 2)]


@pytest.mark.parametrize("place", [0, 1, -1])
@pytest.mark.parametrize("ratio,spread", [(1e3, 0.5), (1e5, 8.0), (1e9, 0.5), (1e14, 0.5)])
@pytest.mark.parametrize("dtype,size", [(BF16, 0), (F16, 1), (BF16, 2), (F16, 3)])
def test_whole_and_chosen_blocks(place, ratio, spread, dtype, size):
    dim, block, hq, hkv = SIZES[size]
    g = torch.Generator("cuda").manual_seed(41)
    lens = [2000, 5 * block, 700]
    counts = [-(-n // block) for n in lens]
    pool = R.random_pool(g, sum(counts) + 3, hkv, block, dim)
    table, _ = R.random_table(g, counts, 3)
    q = torch.randn((3, 1, hq, dim), generator=g, device="cuda")
    prepare(pool, q, table[range(3), [place % n for n in counts]].long(), ratio, spread)
    q = q.to(dtype)
    cache = M.TokenCache(*pool)
    want = reference(pool, q, [tokens(table[b], n, block) for b, n in enumerate(lens)])
    check(cache.attention(q, table, R.i32(lens), scale=1.0)[0], *want)
    every = torch.arange(table.shape[1], device="cuda", dtype=torch.int32).expand(3, 1, hkv, -1).contiguous()
    check(cache.block_attention(q, table, R.i32(lens), every, scale=1.0)[0], *want)
    assert M.take_errors() == 0


@pytest.mark.parametrize("seqs", [3, 300])
@pytest.mark.parametrize("place", [0, 1, -1])
@pytest.mark.parametrize("ratio,spread", [(1e3, 0.5), (1e5, 8.0), (1e9, 0.5), (1e14, 0.5)])
@pytest.mark.parametrize("dtype,size", [(BF16, 0), (F16, 1), (BF16, 2), (F16, 3)])
def test_shared_tokens(seqs, place, ratio, spread, dtype, size):
    dim, block, hq, hkv = SIZES[size]
    groups, shared, lens = [seqs - 1, 1], [2301, 900], [(7 * i) % 40 for i in range(seqs)]
    pool, shared_table, table, q = S.case(42, groups, shared, lens, hq, hkv, block, dim, 1, torch.float32)
    prepare(pool, q, torch.stack([shared_table[m, place % -(-n // block)] for m, n in enumerate(shared)] + [table[2, 0]]).long(), ratio, spread)
    q = q.to(dtype)
    out, _ = M.TokenCache(*pool).shared_attention(q, shared_table, R.i32(shared), R.cu(groups), table, R.i32(lens), scale=1.0)
    rows = []
    for b, n in enumerate(lens):
        far, near = tokens(shared_table[b // (seqs - 1)], shared[b // (seqs - 1)], block), tokens(table[b], n, block)
        rows.append([torch.cat(x) for x in zip(far, near)])
    check(out, *reference(pool, q, rows))
    assert M.take_errors() == 0


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("seqs", [2, 300])
@pytest.mark.parametrize("dtype,size", [(BF16, 0), (F16, 1), (BF16, 3)])
def test_every_block_at_a_scale_of_its_own(seed, seqs, dtype, size):
    # 10^-8 to 10^8 (10^-4 to 10^3 for f16 outputs), and 0; scores that favour one or the other block
    dim, block, hq, hkv = SIZES[size]
    groups, shared, lens = [seqs], [1700], [(37 * i + 11) % 150 for i in range(seqs)]
    pool, shared_table, table, q = S.case(50 + seed, groups, shared, lens, hq, hkv, block, dim, 1, dtype, 1 + seed)
    g = torch.Generator("cuda").manual_seed(60 + seed)
    low, high = (-4, 3) if dtype == F16 else (-8, 8)
    pool[3][:] = 10.0 ** (low + (high - low) * torch.rand(pool[3].shape, generator=g, device="cuda"))
    pool[3][torch.rand(pool[3].shape, generator=g, device="cuda") < 0.05] = 0
    pool[2] *= dim ** -0.5
    cache = M.TokenCache(*pool)
    rows = []
    for b, n in enumerate(lens):
        rows.append([torch.cat(x) for x in zip(tokens(shared_table[0], shared[0], block), tokens(table[b], n, block))])
    out, _ = cache.shared_attention(q, shared_table, R.i32(shared), R.cu(groups), table, R.i32(lens), scale=1.0)
    check(out, *reference(pool, q, rows))
    own = [tokens(shared_table[0], 1700 - 13 * b, block) for b in range(2)]
    both, length = shared_table.expand(2, -1).contiguous(), R.i32([1700, 1687])
    want = reference(pool, q[:2], own)
    check(cache.attention(q[:2], both, length, scale=1.0)[0], *want)
    order = torch.randperm(both.shape[1], generator=g, device="cuda").to(torch.int32).expand(2, 1, hkv, -1).contiguous()
    check(cache.block_attention(q[:2], both, length, order, scale=1.0)[0], *want)
    assert M.take_errors() == 0
