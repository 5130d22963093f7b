"""GPU: the operators for long and shared contexts at their far ends: caches and rows past 32-bit offsets, empty tables,
the most queries, many groups, outputs over their inputs, graphs that run at once."""
import ctypes
import math
import re

import pytest
import torch

import memory_ref as R
import test_gpu_block_choice as C
import test_gpu_shared_attention as S
from beam_search_collab_b200 import memory as M
from memory_abi import _Cache, _lib, _Rotate, _Shared

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def test_blocks_past_32_bit_offsets():
    """The same blocks at the end of a cache whose codes pass 2^32 bytes, and in a small one."""
    hkv, block, dim, many = 8, 128, 128, 35000
    lens = [1000, 1, 0, 129, 700] + [(7 * i) % 40 for i in range(295)]
    groups, shared = [100, 200], [2500, 900]
    pool, shared_table, table, q = S.case(1, groups, shared, lens, 16, hkv, block, dim, 1, BF16)
    few = pool[0].shape[0]
    first = many - few
    assert first * hkv * block * dim > 1 << 32
    far = [torch.empty((many,) + tuple(x.shape[1:]), dtype=x.dtype, device="cuda") for x in pool]
    for a, b in zip(far, pool):
        a[first:] = b
    small, large = M.TokenCache(*pool), M.TokenCache(*far)
    n = R.i32(lens)
    far_table, far_shared = (torch.where(x >= 0, x + first, x) for x in (table, shared_table))
    bounds, far_bounds = small.empty_bounds(), large.empty_bounds()
    small.update_bounds(bounds, table, n)
    large.update_bounds(far_bounds, far_table, n)
    assert torch.equal(far_bounds[first:], bounds) and not far_bounds[:first].any()
    for count in (3, 8):
        blocks = small.choose_blocks(q, bounds, table, n, count)
        assert torch.equal(large.choose_blocks(q, far_bounds, far_table, n, count), blocks)
        want, got = small.block_attention(q, table, n, blocks), large.block_attention(q, far_table, n, blocks)
        assert torch.equal(got[0], want[0])
    sequences = slice(0, 4)
    for x, sizes in ((slice(None), groups), (sequences, [2, 2])):       # by the many sequences' way, and by themselves
        args = R.i32(shared), R.cu(sizes)
        want = small.shared_attention(q[x], shared_table, *args, table[x], n[x], with_lse=True)
        got = large.shared_attention(q[x], far_shared, *args, far_table[x], n[x], with_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert M.take_errors() == 0


def test_rows_past_32_bit_offsets():
    tokens, heads, dim, last = 1_060_000, 32, 128, 3000
    assert (tokens - last) * heads * dim > 1 << 32
    q = torch.zeros((tokens, heads, dim), dtype=BF16, device="cuda")
    q[-last:] = torch.randn((last, heads, dim), generator=S.gen(2), device="cuda").to(BF16)
    positions = torch.arange(tokens, device="cuda", dtype=torch.int32)
    freqs, _ = M.rotary_frequencies(dim, device="cuda")
    got, _ = M.norm_rotate(q, None, positions, freqs)
    want, _ = M.norm_rotate(q[-last:].clone(), None, positions[-last:].clone(), freqs)
    assert torch.equal(got[-last:], want) and not got[:-last].any()


@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rotary", [(3, 5, 1, 64, 48), (4000, 8, 2, 128, 128), (900, 3, 3, 96, 4)])
def test_rotation_over_its_own_input(tokens, hq, hkv, dim, rotary, interleaved):
    g = S.gen(3)
    q, k = (torch.randn((tokens, h, dim), generator=g, device="cuda").to(F16) for h in (hq, hkv))
    positions = torch.randint(-5000, 5000, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    freqs, _ = M.rotary_frequencies(rotary, device="cuda")
    weight = torch.rand(dim, generator=g, device="cuda")
    want = M.norm_rotate(q, k, positions, freqs, q_weight=weight, k_weight=weight, interleaved=bool(interleaved))
    d = _Rotate(q=q.data_ptr(), k=k.data_ptr(), out_q=q.data_ptr(), out_k=k.data_ptr(), q_weight=weight.data_ptr(), k_weight=weight.data_ptr(),
                positions=positions.data_ptr(), freqs=freqs.data_ptr(), total=tokens, q_heads=hq, kv_heads=hkv, dim=dim, rotary=rotary,
                interleaved=interleaved, dtype=_dtype(F16), weight_dtype=_dtype(torch.float32), eps=1e-6, amplitude=1.0)
    d.q_stride[:] = [hq * dim, dim]
    d.k_stride[:] = [hkv * dim, dim]
    assert _lib().bs_norm_rotate(ctypes.byref(d), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def _dtype(t):
    return {torch.float32: 0, F16: 1, BF16: 2}[t]


@pytest.mark.parametrize("seqs,hkv,queries", [(1, 1, 1), (2, 2, 2), (3, 8, 1), (5, 8, 2), (21, 8, 1)])
@pytest.mark.parametrize("width", [64, 65, 256, 257, 513, 1025, 2049, 4095, 4096, 4097, 8192, 8193])
def test_choice_by_one_block_and_by_several(seqs, hkv, queries, width):
    """Rows of all the ways that a table's width and the number of rows lead to, some of them short in a wide table."""
    lens = [width * 16 - 16 * (i % 3) - i % 16 if i % 4 < 2 else (i * 977) % (width * 16) for i in range(seqs)]
    pool, table, q = C.case(9, lens, 2 * hkv, hkv, 16, 16, queries, BF16, width=width)
    C.check_choice(pool, table, q, lens, 33, 2, 5)
    assert M.take_errors() == 0


def test_tables_without_columns():
    pool, shared_table, table, q = S.case(4, [2, 1], [300, 40], [50, 0, 9], 8, 2, 32, 64, 2, F16)
    cache = M.TokenCache(*pool)
    none, zeros = table[:, :0].contiguous(), R.i32([0] * 3)
    # nothing at all
    empty = shared_table[:, :0].contiguous()
    for out, lse in (cache.shared_attention(q, empty, R.i32([0, 0]), R.cu([2, 1]), none, zeros, with_lse=True),
                     cache.block_attention(q, none, zeros, torch.zeros((3, 2, 2, 5), dtype=torch.int32, device="cuda") - 1, with_lse=True),
                     cache.block_attention(q, table, R.i32([50, 0, 9]), torch.zeros((3, 2, 2, 0), dtype=torch.int32, device="cuda"), with_lse=True)):
        assert (out == 0).all() and (lse == -float("inf")).all()
    bounds = cache.empty_bounds()
    assert not cache.update_bounds(bounds, none, zeros).any()
    assert (cache.choose_blocks(q, bounds, none, zeros, 4) == -1).all()
    assert M.take_errors() == 0
    # one of the two
    S.check(pool, shared_table, none, q, [2, 1], [300, 40], [0] * 3)
    S.check(pool, empty, table, q, [2, 1], [0, 0], [50, 0, 9])


def test_the_most_queries():
    """1,024 query tokens: those before the sequence's first token see what is shared alone."""
    lens = [1100, 700, 0]
    pool, shared_table, table, q = S.case(5, [3], [200], lens, 4, 2, 64, 32, 1024, F16)
    S.check(pool, shared_table, table, q, [3], [200], lens)
    bounds = M.TokenCache(*pool).empty_bounds()
    M.TokenCache(*pool).update_bounds(bounds, table, R.i32(lens))
    blocks = M.TokenCache(*pool).choose_blocks(q, bounds, table, R.i32(lens), 5)
    few = [0, 1, 300, 323, 324, 325, 900, 1022, 1023]
    for i in few:                           # a query by itself is the last of a shorter sequence
        n = [max(0, x - 1023 + i) for x in lens]
        one = M.TokenCache(*pool).choose_blocks(q[:, i:i + 1], bounds, table, R.i32(n), 5)
        assert torch.equal(one, blocks[:, i:i + 1])
    out, lse = M.TokenCache(*pool).block_attention(q, table, R.i32(lens), blocks, with_lse=True)
    for i in few:
        n = [max(0, x - 1023 + i) for x in lens]
        ref, ref_lse, weighted, big = C.attention_ref(pool, table, q[:, i:i + 1], n, blocks[:, i:i + 1], 32 ** -0.5)
        off = (out[:, i:i + 1].double() - ref).abs() - R.out_bound(ref, weighted, F16, R.UNIT[F16])
        assert off.max() <= 0, off.max()
        empty = ref_lse == -float("inf")
        assert torch.equal(lse[:, i:i + 1] == -float("inf"), empty)
        off = ((lse[:, i:i + 1].double() - ref_lse).abs() - R.lse_bound(big))[~empty]
        assert off.max() <= 0, off.max()


@pytest.mark.parametrize("count,size", [(33, 60), (470, 9)])
def test_many_groups_of_many_sequences(count, size):
    """More groups than a warp has lanes, and than a block has threads; some of them empty or without shared tokens."""
    groups = [0 if i % 9 == 4 else size for i in range(count)]
    shared = [0 if i % 7 == 3 else 1 + (97 * i) % 640 for i in range(count)]
    shared[1] = 640
    lens = [(5 * i) % 17 for i in range(sum(groups))]
    dim, hq = 16, 128
    case = S.case(6, groups, shared, lens, hq, 1, 16, dim, 1, F16)
    pool, shared_table, table, q = case
    c = _Cache(num_blocks=pool[0].shape[0], kv_heads=1, block=16, dim=dim)
    d = _Shared(num_seqs=len(lens), num_groups=count, shared_width=shared_table.shape[1], table_width=table.shape[1], queries=1, q_heads=hq,
                dtype=_dtype(F16), scale=0.25)
    work = ctypes.c_size_t()
    assert _lib().bs_shared_attention_workspace(ctypes.byref(c), ctypes.byref(d), ctypes.byref(work)) == 0
    assert work.value > 0                   # by the way for many sequences
    S.check(*case, groups, shared, lens)


def test_groups_with_the_same_beginning():
    """One row of blocks for two groups, and a sequence's own blocks among those that are shared."""
    groups, shared, lens = [3, 4], [500, 500], [64, 1, 0, 30, 64, 2, 5]
    pool, shared_table, table, q = S.case(7, groups, shared, lens, 8, 2, 32, 64, 1, BF16)
    shared_table[1] = shared_table[0]
    table[4] = shared_table[0, 3:3 + table.shape[1]]
    S.check(pool, shared_table, table, q, groups, shared, lens)


def test_graphs_that_run_at_once():
    """Two captured steps, each with its own workspaces and outputs, replayed on two streams."""
    groups, shared, lens = [150, 150], [1500, 2000], [70] * 300
    pool, shared_table, table, q = S.case(8, groups, shared, lens, 8, 2, 32, 128, 1, BF16)
    cache = M.TokenCache(*pool)
    n, args = R.i32(lens), (shared_table, R.i32(shared), R.cu(groups))
    positions, (freqs, _) = R.i32([3] * 300), M.rotary_frequencies(64, device="cuda")
    qs = [q, (q.float() * 0.5).to(BF16)]

    def step(x):
        x = M.norm_rotate(x[:, 0], None, positions, freqs)[0][:, None]
        bounds = cache.update_bounds(cache.empty_bounds(), table, n)
        blocks = cache.choose_blocks(x, bounds, table, n, 2)
        return (*cache.block_attention(x, table, n, blocks, with_lse=True), *cache.shared_attention(x, *args, table, n, with_lse=True))

    want = [step(x) for x in qs]
    graphs, got, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for x in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(step(x))
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(4):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert M.take_errors() == 0


def test_the_modules_example_runs():
    # (its lines from the documentation, two conversations of an instruction and a few tokens each)
    g = torch.Generator("cuda").manual_seed(18)
    hq, kv_heads, dim, block, count, budget = 8, 2, 64, 64, 2, 100
    code = re.search(r"\n\n((?:    .*\n)+)", M.__doc__)[1]
    lines = [x[4:] for x in code.splitlines() if "import" not in x]
    lengths, num_blocks = [300, 150], 40

    def rows(n, heads):
        return torch.randn((n, heads, dim), generator=g, device="cuda").to(BF16)

    ids = torch.randperm(num_blocks, generator=g, device="cuda").to(torch.int32)
    w = torch.ones(dim, device="cuda")
    names = dict(memory=M, q=rows(450, hq), k=rows(450, kv_heads), v=rows(450, kv_heads), cu=R.cu(lengths), num_blocks=num_blocks,
                 kv_heads=kv_heads, dim=dim, table=ids[:16].view(2, 8), start=R.i32([0, 0]), lens=R.i32(lengths), w=w, count=count, budget=budget,
                 q1=rows(2, hq), k1=rows(2, kv_heads), positions=R.i32(lengths), freqs=M.rotary_frequencies(dim, device="cuda")[0],
                 mass=torch.zeros((2, kv_heads, 512), device="cuda"), bounds=torch.zeros((num_blocks, kv_heads, 2, dim), dtype=torch.int8, device="cuda"),
                 shared_table=ids[16:18][None].contiguous(), shared_lens=R.i32([128]), groups=R.cu([2]), new_table=ids[20:24].view(2, 2).contiguous(),
                 old_table=ids[:16].view(2, 8), old_lens=R.i32(lengths))
    names["found"] = R.i32([[3, 7], [1, 149]])
    exec("\n".join(lines), names)
    assert M.take_errors() == 0
    assert names["blocks"].shape == (2, 1, kv_heads, count) and names["keys"].shape[:2] == (2, kv_heads)


def test_as_many_shared_tokens_as_there_can_be():
    # 2^30 - 16 tokens that each sequence reads by itself, and no own ones: the queries see the last shared tokens too
    heads, queries, block, dim, width = 9, 32, 16, 16, (1 << 26) - 1
    pool = [torch.zeros((2, heads, block, dim), dtype=torch.int8, device="cuda") for _ in range(2)] + [torch.zeros((2, heads), device="cuda") for _ in range(2)]
    pool[0][1], pool[1][1], pool[2][1], pool[3][1] = 100, 50, 0.03, 0.02        # scores of 100 * 0.03 * 16 = 48 against 0
    shared_table = torch.zeros((1, width), dtype=torch.int32, device="cuda")
    shared_table[0, -1] = 1
    q = torch.ones((1, queries, heads, dim), dtype=F16, device="cuda")
    table = torch.zeros((1, 0), dtype=torch.int32, device="cuda")
    out, lse = M.TokenCache(*pool).shared_attention(q, shared_table, R.i32([width * block]), R.cu([1]), table, R.i32([0]), scale=1.0, with_lse=True)
    assert M.take_errors() == 0
    n, top = (width - 1) * block, torch.tensor(0.03).item() * 1600
    far = math.log(n * math.exp(-top) + 16)
    # (16 of e^48 against 2^30 of 1: sums of 2^30 ones in 32 bits may lose all of them, e^-48 * 2^30 / 16 = 1e-13 of the whole)
    assert (lse.double() - (top + far)).abs().max() <= 2.0 ** -17 * top + 2.0 ** -17
    assert (out.double() - 1.0).abs().max() <= 2.0 ** -10
