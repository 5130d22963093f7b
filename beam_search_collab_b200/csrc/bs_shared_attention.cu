// bs_shared_attention.cu -- attention of many query rows over tokens of the
// 8-bit cache that they share (include/bsearch.h, bs_shared_attention; the
// shared tokens' part of it).
//
// The rows of a key head over all sequences of a group are a matrix, so this is
// work for the tensor cores, as in bs_prompt_attention.cu: two tiles of 128 rows
// a thread block, 128 tokens at a time, scores, weights and outputs in TMEM.
// What differs: keys and values are codes, which warps of their own load,
// convert and leave in shared memory in the products' swizzled layout, once for
// both tiles of rows; scales belong to blocks of tokens, so the scores are
// multiplied by theirs 16 columns at a time, and the weights by the values'.
// Every row sees every token, but for the end of the last tile.
//
// Warps 0-3 and 4-7 are the softmax of tile 0 and 1 (a thread has one row),
// 8-11 convert keys and values, 12 issues the matrix instructions, 13 finds the
// pieces of the share and copies codes (a bulk copy for each block) and scales to
// shared memory:
//   S_t = Q_t K^T     codes of K exact in f16, as are bf16 queries times a power
//                     of two of each row's own (elements below 2^-29 of the
//                     row's largest lose bits); bf16 keys took twice the
//                     instructions to convert
//   O_t += P_t V      codes of V exact in f16, P_t f16: a weight times its values'
//                     scale, over the largest of the piece, rounded to 2^-11 of
//                     itself or, where that is more, 2^-29 of the row's largest
//                     such product (they count in 2^-kLift, the room that a
//                     maximum moved at 2^10 leaves)
// So the maximum that weights count from is that of a score plus log2 of its value
// scale over the piece's largest (at least -kDeep): counted from the largest score
// alone, weights of 1 at a scale 10^-7 of another's had few bits left, whatever weight
// that other one got.  It is moved only when 16 weights times their scale pass 2^10
// together (no maximum is taken before the exponentials); sums are 32-bit, of the
// unrounded weights.
//
// 512 rows of each of 8 key heads over 32,768 tokens take 106 us here: 28 times 128 tokens
// a block, 4,100 to 4,700 clocks each, and 12,000 to the first scores and 5,500 for the
// outputs.  128 tokens need 2,048 clocks of the tensor cores and 2,560 of shared memory
// (operands 192 KB, codes in and out 64, converted 64, at 128 bytes a clock); the rest
// is each tile's chain of scores, weights and products, which the other tile alone
// hides.  Scores in halves of 64 tokens, the next ones under the last ones' products,
// hide more of it, but read the queries twice as often from shared memory (135 us of
// the whole call against 129).  One lane of a warp that waits for all of them: 207
// against 136.  More registers for the softmax and fewer for the others: spills, slower.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bs_device.cuh"
#include "bs_f32x2.cuh"
#include "bs_memory.h"
#include "bs_shared.cuh"
#include "bs_tcgen05.cuh"

namespace bsb {

using namespace dev;
using namespace shared;
using namespace tc;

namespace {

constexpr int kConverters = 4;         // warps
constexpr int kIssuer = 8 + kConverters;
constexpr int kCopier = kIssuer + 1;
constexpr int kThreads = 32 * (kCopier + 1);
// Rings of converted tiles (keys and values in turn: a tile's values and the next
// one's keys are in use together, meanwhile the next ones are converted) and of
// quarters of tiles of codes.  A quarter is one warp's, the same of every tile (a
// barrier's parity tells a phase from the one before it, not from the one before
// that, so whoever waits for one has to wait for each): with all warps on each part
// of a tile their barriers took a third of the time.
constexpr uint32_t kRing = 4;
constexpr uint32_t kQuarter = kRows / 4;
template <int BOXES>
constexpr uint32_t kRawRing = BOXES == 2 ? 8 : 16;
// Up to so many groups the warp that finds the pieces counts their cost too, a group
// to a lane, meanwhile the other warps get ready; more are counted by all warps first.
constexpr uint32_t kFewGroups = 32;
constexpr float kLift = 5.f;
constexpr float kMost = 32768.f;       // of 16 lifted weights times their scale together, and so of each: below f16's 65504
constexpr float kDeep = 60.f;          // value scales count down to 2^-kDeep of the piece's largest
constexpr float kDeepest = 0x1p-60f;
// Tiles whose scales are in shared memory.  Those of tile n are written when
// codes of tile n - kRawRing / 8 have been converted, into the place of keys that
// were multiplied two tiles before; those products are issued when the weights of
// the tile before that are made, and its scales read no more.
constexpr int kScales = 8;
static_assert(kConverters * kQuarter == kRows, "a quarter for each warp");
static_assert(kRawRing<1> / 8 + 3 <= kScales && kRawRing<2> / 8 + 3 <= kScales, "scales are overwritten while they are read");

// Eight codes in f16: 0x6400 | u is 1024 + u, minus 1152.
__device__ __forceinline__ uint4 codes_to_halves(uint2 x) {
    uint4 r;
    uint32_t* const w = reinterpret_cast<uint32_t*>(&r);
    x.x ^= 0x80808080u;
    x.y ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = __byte_perm(i < 2 ? x.x : x.y, 0x64646464u, i & 1 ? 0x4342 : 0x4140);
        const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __float2half2_rn(1152.f));
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return r;
}

// 16-byte aligned bytes of memory into shared memory.
__device__ __forceinline__ void copy_bulk(void* dst, const void* src, unsigned bytes, uint64_t* bar) {
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");     // after what was read there before
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(smem_addr(dst)), "l"(src),
                 "r"(bytes), "r"(smem_addr(bar))
                 : "memory");
}

// Whether a phase is over, without a wait (lanes may ask of barriers of their own).
__device__ __forceinline__ bool barrier_done(uint64_t* b, unsigned phase) {
    unsigned ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok)
                 : "r"(smem_addr(b)), "r"(phase)
                 : "memory");
    return ok != 0;
}

// Where a block is in its share: tiles t .. end of a segment (group m, key
// head h, pair of row tiles).
struct Piece {
    uint32_t m, segment;       // segment: h * pairs + pair
    uint32_t t, end;
    uint64_t left;             // units of the share after this piece
    uint64_t at, begin;        // units: of the piece's end, of the segment's begin
    Group g;
    uint32_t slot;             // 0: the share's first piece
};

// What the block works on: a piece, as the warp that finds them leaves it to
// the others.
struct Item {
    uint32_t valid;                     // 0: there is no more
    uint32_t m, h;                      // group, key head
    uint32_t row0, rows, first;         // first row of the pair in the group, rows from there on; the group's first sequence
    uint32_t tokens, t, end;
    uint32_t slot, whole;
};

struct Control {
    uint64_t q_full[2], s_full[2], p_full[2], o_full[2], done;
    uint64_t full[kRing], empty[kRing], raw_full[16], raw_empty[16];
    uint64_t item_full[2], item_empty[2];
    Item item[2];
    uint64_t sums[kCopier + 1];
    uint32_t missing[kScales];          // by tile: bits of 16 tokens whose block is not there
    __align__(16) float2 scales[kScales][8];      // by tile and 16 tokens: of keys, of values
    uint32_t tmem;
    uint32_t gave_up;
};

template <int BOXES>
constexpr size_t kSmem = 1024 + (2 + kRing) * BOXES * kBoxBytes + kRawRing<BOXES> * (BOXES * kBoxBytes / 8) + sizeof(Control);

// The piece of a segment from its unit `from` on; its first kStart units
// stand for no tiles.
__device__ __forceinline__ void cut_piece(Piece& p, uint32_t from) {
    const uint32_t cost = p.g.tiles + kStart, take = p.left < cost - from ? static_cast<uint32_t>(p.left) : cost - from;
    p.t = from > kStart ? from - kStart : 0;
    p.end = from + take > kStart ? from + take - kStart : 0;
    p.left -= take;
    p.begin = p.at - from;
    p.at += take;
}

// To the next piece; false: there is none.
__device__ __forceinline__ bool next_piece(const SharedArgs& a, Piece& p) {
    if (p.left == 0) return false;
    if (++p.segment == p.g.pairs * a.c.kv_heads) {
        p.segment = 0;
        do {
            if (++p.m >= a.d.num_groups) return false;         // (not with lists that stay as they are)
            p.g = group_of(a, p.m);
        } while (p.g.tiles == 0);
    }
    p.slot = 1;
    cut_piece(p, 0);
    return true;
}

// The first piece of the block's share (by one warp); none: p.left and its tiles
// are 0.  w, n: cost of all pieces and shares in use, found here too if the groups
// are few.
__device__ __forceinline__ void find_piece(const SharedArgs& a, Piece& p, uint64_t& w, uint32_t& n) {
    const uint32_t lane = threadIdx.x & 31, groups = a.d.num_groups;
    uint64_t seen = 0, first = 0;
    p.left = p.t = p.end = p.segment = p.slot = 0;
    p.m = groups - 1;
    p.g = Group{};
    for (uint32_t m0 = 0; m0 < groups; m0 += 32) {       // 32 at a time
        Group g{};
        if (m0 + lane < groups) g = group_of(a, m0 + lane);
        const uint64_t mine = cost_of(g) * a.c.kv_heads;
        uint64_t sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t up = __shfl_up_sync(kFull, sum, o);
            if (lane >= static_cast<uint32_t>(o)) sum += up;
        }
        const uint64_t together = __shfl_sync(kFull, sum, 31);
        if (m0 == 0) {
            if (groups <= kFewGroups) {
                w = together;
                n = used_shares(w, a.shares);
            }
            if (blockIdx.x >= n) return;
            first = share_first(w, n, blockIdx.x);
            p.left = share_first(w, n, blockIdx.x + 1) - first;
        }
        const unsigned past = __ballot_sync(kFull, seen + sum > first);
        if (past) {
            const int l = __ffs(past) - 1;
            seen += __shfl_sync(kFull, sum - mine, l);
            p.m = m0 + l;
            p.g.first = __shfl_sync(kFull, g.first, l);
            p.g.rows = __shfl_sync(kFull, g.rows, l);
            p.g.pairs = __shfl_sync(kFull, g.pairs, l);
            p.g.tokens = __shfl_sync(kFull, g.tokens, l);
            p.g.tiles = __shfl_sync(kFull, g.tiles, l);
            break;
        }
        seen += together;
    }
    if (p.g.tiles == 0) {                                // (not with lists that stay as they are)
        p.left = 0;
        return;
    }
    const uint32_t cost = p.g.tiles + kStart;
    p.segment = static_cast<uint32_t>((first - seen) / cost);
    p.at = first;
    cut_piece(p, static_cast<uint32_t>((first - seen) % cost));
}

// The warp's rows times `shrink`: the first `quarters` of their weights of a
// tile and `dim` columns of outputs.
__device__ __forceinline__ void rescale(uint32_t p_at, uint32_t o_at, int quarters, int dim, float shrink) {
    wait_stores();
#pragma unroll 1
    for (int c = 0; c < quarters; ++c) {
        uint32_t p[16];
        tmem_load16(p_at + 16 * c, p);
        wait_loads16(p);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const float2 f = Type16<__half>::unpack(p[k]);
            p[k] = Type16<__half>::pack(f.x * shrink, f.y * shrink);
        }
        tmem_store16(p_at + 16 * c, p);
    }
#pragma unroll 1
    for (int x = 0; x < dim; x += 16) {
        uint32_t o[16];
        tmem_load16(o_at + x, o);
        wait_loads16(o);
#pragma unroll
        for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * shrink);
        tmem_store16(o_at + x, o);
    }
    wait_stores();
}

// log2 of a value scale (v_by: 1 over the piece's largest), what a score counts for besides its weight.
__device__ __forceinline__ float scale_log2(float v_scale, float v_by) { return __log2f(fmaxf(v_scale * v_by, kDeepest)); }

// 64 scores of a row that are all seen, 32 at a time; s[0] is on its way, the
// next 32 follow (`more`: those after these too): weights 2^(key scale * s +
// base), their sum returned, times their value scale packed in p.  scales: of 16
// tokens each; k_by and v_by are what they are multiplied by besides.  `most`: the
// largest of 16 weights together times their scale.  (Unrolled: at 32 a turn the
// special-function pipe runs dry at each, 2,400 clocks a tile.)
__device__ __forceinline__ float weights64(uint32_t s_at, bool more, float (&s)[2][32], const float2* scales, float k_by, float v_by, float base,
                                           uint32_t (&p)[32], float& most) {
    const float2 base2 = make_float2(base, base);
    float sum = 0.f;
    most = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        wait_loads32(s[c]);
        if (c == 0 || more) tmem_load32(s_at + 32 * (c + 1), s[c ^ 1]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const float2 scale = scales[2 * c + half];
            const float2 k = make_float2(scale.x * k_by, scale.x * k_by), v = make_float2(scale.y * v_by, scale.y * v_by);
            float2 add[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int i = 8 * half; i < 8 * half + 8; ++i) {
                float2 x = fma2(make_float2(s[c][2 * i], s[c][2 * i + 1]), k, base2);
                x.x = exp2_fast(x.x);
                x.y = exp2_fast(x.y);
                add[i & 1] = add2(add[i & 1], x);
                x = mul2(x, v);
                p[16 * c + i] = Type16<__half>::pack(x.x, x.y);
            }
            add[0] = add2(add[0], add[1]);
            const float together = add[0].x + add[0].y;
            sum += together;
            most = fmaxf(most, together * fmaxf(v.x, kDeepest));
        }
    }
    return sum;
}

// The largest of a row's 128 scores, in log2 units, each plus its value scale's.
__device__ __noinline__ float largest_score(uint32_t s_at, const float2* scales, float k_by, float v_by) {
    float most = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        float s[32];
        tmem_load32(s_at + 32 * c, s);
        wait_loads32(s);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float high = s[16 * half];
#pragma unroll
            for (int i = 1; i < 16; ++i) high = fmaxf(high, s[16 * half + i]);
            most = fmaxf(most, fmaf(high, scales[2 * c + half].x * k_by, scale_log2(scales[2 * c + half].y, v_by)));
        }
    }
    return most;
}

// The last tile where the tokens end inside it, tiles with blocks that are not
// there, and where the maximum moves: the largest first, then the weights.  From
// the quarter `from` on; `left` tokens of the tile are there, `missing` has a bit
// for each 16 that are not.  `state` is the row's maximum (log2, of scores and value
// scales) and sum, returned as they become.
__device__ __noinline__ float2 weights_with_care(uint32_t s_at, uint32_t o_at, int from, int quarters, int32_t left, uint32_t missing,
                                                 const float2* scales, float k_by, float v_by, int dim, float2 state) {
    float next = state.x;
    float z[32];
    auto scores = [&](int c) {             // in log2 units, -infinity where there is no token
        tmem_load32(s_at + 32 * c, z);
        wait_loads32(z);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const float k = scales[2 * c + half].x * k_by;
            const int32_t there = missing >> (2 * c + half) & 1 ? 0 : left - 32 * c;
#pragma unroll
            for (int i = 16 * half; i < 16 * half + 16; ++i) z[i] = i < there ? z[i] * k : -INFINITY;
        }
    };
#pragma unroll 1
    for (int c = from; c < quarters; ++c) {
        scores(c);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float high = z[16 * half];
#pragma unroll
            for (int i = 1; i < 16; ++i) high = fmaxf(high, z[16 * half + i]);
            next = fmaxf(next, high + scale_log2(scales[2 * c + half].y, v_by));
        }
    }
    if (__any_sync(kFull, next > state.x)) {
        // the maximum moves, what was summed is rescaled
        const float shrink = state.x == -INFINITY ? 0.f : exp2_fast(state.x - next);
        state.y *= shrink;
        if (from || dim) rescale(s_at, o_at, from, dim, next == -INFINITY ? 1.f : shrink);
    }
    const float base = next == -INFINITY ? 0.f : kLift - next;
#pragma unroll 1
    for (int c = from; c < quarters; ++c) {
        scores(c);
        uint32_t p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float v = scales[2 * c + i / 8].y * v_by;
            const float x = exp2_fast(z[2 * i] + base), y = exp2_fast(z[2 * i + 1] + base);
            state.y += x + y;
            p[i] = Type16<__half>::pack(x * v, y * v);
        }
        tmem_store16(s_at + 16 * c, p);
    }
    return make_float2(next, state.y);
}

template <int BOXES>
__global__ void __launch_bounds__(kThreads, 1) k_shared(const __grid_constant__ SharedArgs a) {
    extern __shared__ unsigned char raw_smem[];
    unsigned char* const smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t{1023});
    constexpr int kTileBytes = BOXES * kBoxBytes, kRawBytes = kTileBytes / 8;
    constexpr uint32_t kRaw = kRawRing<BOXES>;
    unsigned char* const ring = smem + 2 * kTileBytes;
    unsigned char* const raw = ring + kRing * kTileBytes;             // codes
    Control& ctl = *reinterpret_cast<Control*>(raw + kRaw * kRawBytes);
    const bs_shared_attention_desc& d = a.d;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hkv = a.c.kv_heads, dim = a.c.dim, block = a.c.block;

    cudaGridDependencySynchronize();       // in every block, before anything of the caller's
    cudaTriggerProgrammaticLaunchCompletion();       // the kernel after this one is launched meanwhile, and waits
    uint64_t w = 0;                        // cost of all pieces
    uint32_t n = 0;                        // shares in use
    if (d.num_groups > kFewGroups) {
        w = count_cost(a, ctl.sums) * hkv;
        n = used_shares(w, a.shares);
        if (blockIdx.x >= n) return;
    }
    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            barrier_init(&ctl.q_full[t], 4);
            barrier_init(&ctl.s_full[t], 1);
            barrier_init(&ctl.p_full[t], 4);
            barrier_init(&ctl.o_full[t], 1);
            barrier_init(&ctl.item_full[t], 1);
            barrier_init(&ctl.item_empty[t], kCopier);       // (all other warps)
        }
        barrier_init(&ctl.done, 1);
        for (uint32_t s = 0; s < kRing; ++s) {
            barrier_init(&ctl.full[s], 4);
            barrier_init(&ctl.empty[s], 1);
        }
        for (uint32_t s = 0; s < kRaw; ++s) {
            barrier_init(&ctl.raw_full[s], 1);
            barrier_init(&ctl.raw_empty[s], 1);
        }
        ctl.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == kIssuer) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_addr(&ctl.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = ctl.tmem;

    // A bounded wait.  Once one has given up none waits any more: the warps
    // leave their loops together and nothing is stored.
    volatile uint32_t* const gave_up = &ctl.gave_up;
    auto wait = [&](uint64_t* bar, unsigned phase) {
        for (unsigned i = 0; i < a.polls && !*gave_up; ++i)
            if (barrier_test(bar, phase)) return;
        if (!*gave_up) {
            *gave_up = 1;
            atomicOr(a.errors, kMemErrWait);
        }
    };
    auto stopped = [&]() { return __any_sync(kFull, *gave_up != 0); };
    // The next item for a warp that does not find them (not valid: the end), and
    // that it has read it.  (What a loop does not need every time stays in shared
    // memory: a register that is put aside costs more than its time, since what
    // comes back from local memory waits behind the copies on their way.)
    auto next_item = [&](uint32_t i) -> const Item& {
        wait(&ctl.item_full[i & 1], i >> 1 & 1);
        return ctl.item[i & 1];
    };
    auto item_read = [&](uint32_t i) {
        __syncwarp();
        if (lane == 0) barrier_arrive(&ctl.item_empty[i & 1]);
    };
    // columns of tile j that hold tokens, to a multiple of 16
    auto columns = [&](uint32_t tokens, uint32_t j) {
        const uint32_t left = tokens - j * kTileTokens;
        return left >= kTileTokens ? kTileTokens : (left + 15) & ~15u;
    };

    if (warp == kIssuer) {
        // ---------------------------------------------------- matrix products
        // (the whole warp runs the loop, one elected lane issues)
        constexpr uint32_t kCommon = 1u << 4 | static_cast<uint32_t>(kRows >> 4) << 24;
        const uint32_t what_o = kCommon | 1u << 16 | (dim >> 3) << 17;         // (values do not lie along the contraction)
        const int steps = dim / 16;
        const uint64_t q_base = operand(smem_addr(smem), 16, 1024), k_base = operand(smem_addr(ring), 16, 1024);
        const uint64_t v_base = operand(smem_addr(ring), kBoxBytes, 1024);
        constexpr uint32_t kTileUnits = kTileBytes / 16, kBoxUnits = kBoxBytes / 16;
        auto scores = [&](int t, uint32_t stage, uint32_t cols) {
            const uint64_t q = q_base + t * kTileUnits, k = k_base + stage * kTileUnits;
            const uint32_t what = kCommon | (cols >> 3) << 17;
#pragma unroll
            for (int i = 0; i < 4 * BOXES; ++i) {
                const uint32_t off = (i >> 2) * kBoxUnits + (i & 3) * 2;
                if (i < steps) mma_shared(tmem + t * 128, q + off, k + off, what, i > 0);
            }
            mma_commit(&ctl.s_full[t]);
        };
        auto products = [&](int t, uint32_t stage, bool add, uint32_t cols) {
            const uint64_t v = v_base + stage * kTileUnits;
#pragma unroll
            for (int i = 0; i < kRows / 16; ++i) {
                if (16u * i >= cols) break;
                mma_tmem(tmem + 256 + t * 128, tmem + t * 128 + i * 8, v + i * 128, what_o, add || i > 0);
            }
        };
        uint32_t tiles = 0, q_used[2] = {0, 0}, p_used[2] = {0, 0};      // tile i's keys are the ring's 2 i, its values 2 i + 1
        bool issued = false;
        auto full = [&](uint32_t i) { wait(&ctl.full[i % kRing], i / kRing & 1); };
        for (uint32_t it = 0;; ++it) {
            const Item& m = next_item(it);
            if (stopped() || !m.valid) break;
            const uint32_t first = m.t, end = m.end, tokens = m.tokens;
            const bool both = m.rows > kRows;
            item_read(it);
            full(2 * tiles);
            for (int t = 0; t <= both; ++t) wait(&ctl.q_full[t], q_used[t]++ & 1);
            if (stopped()) break;
            issued = true;
            fence_after();
            if (elected()) {
                for (int t = 0; t <= both; ++t) scores(t, 2 * tiles % kRing, columns(tokens, first));
                mma_commit(&ctl.empty[2 * tiles % kRing]);
            }
            __syncwarp();
            for (uint32_t j = first; j < end; ++j, ++tiles) {
                const uint32_t stage = (2 * tiles + 1) % kRing, next = (2 * tiles + 2) % kRing;
                const bool last = j + 1 == end;
                if (stopped()) break;
                full(2 * tiles + 1);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (t && !both) break;
                    wait(&ctl.p_full[t], p_used[t]++ & 1);
                    fence_after();
                    if (elected()) {
                        products(t, stage, j > first, columns(tokens, j));
                        if (last) mma_commit(&ctl.o_full[t]);
                    }
                    __syncwarp();
                    if (last) continue;
                    if (t == 0) {
                        full(2 * tiles + 2);
                        fence_after();
                    }
                    if (elected()) scores(t, next, columns(tokens, j + 1));
                    __syncwarp();
                }
                if (elected()) {
                    mma_commit(&ctl.empty[stage]);
                    if (!last) mma_commit(&ctl.empty[next]);
                }
                __syncwarp();
            }
        }
        // TMEM and the stages are in use until this
        if (issued) {
            if (elected()) mma_commit(&ctl.done);
            __syncwarp();
            for (unsigned i = 0; i < kPolls && !barrier_test(&ctl.done, 0); ++i) {}
        }
        __syncwarp();
    } else if (warp == kCopier) {
        // ------------------------------------------------------------ copies
        // (lanes 0-7 look up every 16 tokens of a tile, and copy its quarters of keys
        // and of values, each when there is room for it: one after the other, with
        // the whole warp, took 700 clocks each)
        const uint32_t run = block < kQuarter ? block : kQuarter, bytes = run * dim, quarter = lane & 3;
        uint32_t tiles = 0, items = 0, copied = 0;     // copied: quarters by this lane
        Piece p;
        find_piece(a, p, w, n);
        for (bool more = true; more && !stopped(); more = next_piece(a, p)) {
            if (p.t == p.end) continue;            // (a share that ends before a segment's first tile)
            const uint32_t h = p.segment / p.g.pairs, row0 = p.segment % p.g.pairs * kPairRows;
            wait(&ctl.item_empty[items & 1], (items >> 1 & 1) ^ 1);
            if (lane == 0) {
                ctl.item[items & 1] = Item{1, p.m, h, row0, p.g.rows - row0, p.g.first, p.g.tokens, p.t, p.end, p.slot, p.t == 0 && p.end == p.g.tiles};
                barrier_arrive(&ctl.item_full[items & 1]);
                if (p.t == 0)                      // where the segment's pieces are
                    a.far[output_row(a, p.g, h, row0)] =
                        FarRow{share_of(w, n, p.begin + kStart + p.g.tiles - 1) - blockIdx.x + 1, blockIdx.x, p.slot, 0};
            }
            __syncwarp();
            ++items;
            const int32_t* const table = d.shared_table + static_cast<uint64_t>(p.m) * d.shared_width;
            auto there = [&](uint32_t j) { return lane < 8 && j * kTileTokens + lane * 16 < p.g.tokens; };
            auto id_at = [&](uint32_t j) { return there(j) ? static_cast<uint32_t>(table[(j * kTileTokens + lane * 16) >> a.block_log2]) : kNoNode; };
            auto scale_of = [&](uint32_t id) {
                const uint64_t slab = static_cast<uint64_t>(id) * hkv + h;
                return id < a.c.num_blocks ? make_float2(a.c.k_scale[slab], a.c.v_scale[slab]) : make_float2(0.f, 0.f);
            };
            // (asked for ahead: ids two tiles, scales one)
            uint32_t next = id_at(p.t), later = p.t + 1 < p.end ? id_at(p.t + 1) : kNoNode;
            float2 next_scale = scale_of(next);
            for (uint32_t j = p.t; j < p.end && !stopped(); ++j, ++tiles) {
                const uint32_t id = next;
                const float2 scale = next_scale;
                next = later;
                next_scale = scale_of(next);
                later = j + 2 < p.end ? id_at(j + 2) : kNoNode;
                const bool ok = id < a.c.num_blocks;
                const uint32_t missing = __ballot_sync(kFull, there(j) && !ok);
                if (missing && lane == 0) atomicOr(a.errors, kMemErrBlock);
                // this lane's quarter: a run of a block, or two blocks of 16
                const uint32_t one = __shfl_sync(kFull, id, 2 * quarter), two = run < kQuarter ? __shfl_sync(kFull, id, 2 * quarter + 1) : kNoNode;
                const uint32_t load = 8 * tiles + lane, stage = load % kRaw;
                wait(&ctl.raw_empty[8 * tiles % kRaw], (8 * tiles / kRaw & 1) ^ 1);
                if (stopped()) break;
                if (lane < 8) ctl.scales[tiles % kScales][lane] = scale;
                if (lane == 0) ctl.missing[tiles % kScales] = missing;
                __syncwarp();
                bool waits = lane < 8;
                for (unsigned i = 0; i < a.polls && __any_sync(kFull, waits); ++i) {
                    if (waits && barrier_done(&ctl.raw_empty[stage], (load / kRaw & 1) ^ 1)) {
                        waits = false;
                        const bool first = one < a.c.num_blocks, second = two < a.c.num_blocks;
                        barrier_expect(&ctl.raw_full[stage], (first + second) * bytes);
                        const int8_t* const codes = lane < 4 ? a.c.k : a.c.v;
                        unsigned char* const to = raw + stage * kRawBytes;
                        auto from = [&](uint32_t x) { return codes + ((static_cast<uint64_t>(x) * hkv + h) * block + (quarter * kQuarter & (block - 1))) * dim; };
                        if (first) copy_bulk(to, from(one), bytes, &ctl.raw_full[stage]);
                        if (second) copy_bulk(to + 16 * dim, codes + (static_cast<uint64_t>(two) * hkv + h) * bytes, bytes, &ctl.raw_full[stage]);
                        copied += 1;
                    }
                    if (i % 64 == 63 && stopped()) break;
                }
                if (__any_sync(kFull, waits)) {            // (the others' wait has given up, or this one does)
                    if (lane == 0 && !*gave_up) {
                        *gave_up = 1;
                        atomicOr(a.errors, kMemErrWait);
                    }
                    __syncwarp();
                    break;
                }
            }
        }
        wait(&ctl.item_empty[items & 1], (items >> 1 & 1) ^ 1);
        if (lane == 0) {
            ctl.item[items & 1].valid = 0;
            barrier_arrive(&ctl.item_full[items & 1]);
        }
        // no copy may be in flight when the block ends: this lane's last ones
        for (uint32_t i = copied > kRaw / 8 ? copied - kRaw / 8 : 0; i < copied; ++i) {
            const uint32_t load = 8 * i + lane;
            for (unsigned x = 0; x < kPolls && !barrier_test(&ctl.raw_full[load % kRaw], load / kRaw & 1); ++x) {}
        }
        __syncwarp();
    } else if (warp >= 8) {
        // --------------------------------------------------------- conversion
        // (a warp has a quarter; 16 codes side by side to a lane, the next
        // 16 to the next; of a row of 128, lanes of the upper half take their second
        // eight first, so that the units that eight lanes store fall on all banks)
        const uint32_t nw = dim / 16;
        constexpr int kEach = 4 * BOXES;                     // 16 codes of a lane, of a quarter
        uint32_t from[kEach], to[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint32_t u = lane + 32 * i, r = u / nw, x = u % nw, later = x >> 2;      // of 32 * nw
            from[i] = u * 16 + later * 8;
            to[i] = later * kBoxBytes + r * 128 + (((2 * (x & 3)) ^ (r & 7)) ^ later) * 16;
        }
        // load 8 i + u: tile i's quarters of keys (u < 4) and of values
        const uint32_t quarter = warp - 8;
        auto convert = [&](uint32_t load) {
            const uint32_t at = load % kRaw, stage = load / 4 % kRing;
            const unsigned char* const codes = raw + at * kRawBytes;
            unsigned char* const tile = ring + stage * kTileBytes + quarter * (kQuarter * 128);
            wait(&ctl.empty[stage], (load / 4 / kRing & 1) ^ 1);
            wait(&ctl.raw_full[at], load / kRaw & 1);
            if (stopped()) return false;
            const uint32_t missing = ctl.missing[load / 8 % kScales] >> 2 * quarter & 3;
            uint2 x[kEach][2];
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (i < static_cast<int>(nw)) {
                    x[i][0] = *reinterpret_cast<const uint2*>(codes + from[i]);
                    x[i][1] = *reinterpret_cast<const uint2*>(codes + (from[i] ^ 8));
                }
            if (missing) {
#pragma unroll
                for (int i = 0; i < kEach; ++i)
                    if (missing >> ((lane + 32 * i) / nw / 16) & 1) x[i][0] = x[i][1] = make_uint2(0, 0);
            }
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (i < static_cast<int>(nw)) {
                    *reinterpret_cast<uint4*>(tile + to[i]) = codes_to_halves(x[i][0]);
                    *reinterpret_cast<uint4*>(tile + (to[i] ^ 16)) = codes_to_halves(x[i][1]);
                }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                barrier_arrive(&ctl.raw_empty[at]);
                barrier_arrive(&ctl.full[stage]);
            }
            return true;
        };
        uint32_t load = quarter, past = 0;
        for (uint32_t it = 0;; ++it) {
            const Item& m = next_item(it);
            if (stopped() || !m.valid) break;
            past += 8 * (m.end - m.t);
            item_read(it);
            while (load < past && convert(load)) load += 4;
            if (load < past) break;
        }
    } else {
        // ----------------------------------------------------------- softmax
        const uint32_t t = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (warp & 3) * 32 << 16;                  // this warp's TMEM lanes
        const uint32_t s_at = tmem + t * 128 + lanes, o_at = tmem + 256 + t * 128 + lanes;
        unsigned char* const tile = smem + t * kTileBytes;
        unsigned char* const staging = tile + (warp & 3) * 4096;       // the queries' place, once they are done with
        uint32_t s_used = 0, o_used = 0, tiles = 0;
        for (uint32_t it = 0;; ++it) {
            const Item& m = next_item(it);
            if (stopped() || !m.valid) break;
            const uint32_t first = m.t, end = m.end;
            if (m.rows <= t * kRows) {
                tiles += end - first;
                item_read(it);
                continue;
            }
            const bool real = t * kRows + row < m.rows;
            // this row's place in the outputs and in the queries
            auto place = [&](uint32_t& b, uint32_t& i, uint32_t& head) {
                const uint32_t r = m.row0 + t * kRows + row, in = r % a.rows;
                b = m.first + r / a.rows;
                i = in / a.group;
                head = m.h * a.group + in % a.group;
            };
            // The warp's queries, a row's units to lanes side by side.  (As little code
            // as can be: what a warp executes for the first time takes 230 clocks for
            // eight instructions.)
            float row_scale = 1.f;
            {
                constexpr uint32_t kLanes = 8 * BOXES, kAtOnce = 32 / kLanes;
                const uint32_t c = lane % kLanes;
                uint32_t b, i, head;
                place(b, i, head);
                const uint16_t* const mine = static_cast<const uint16_t*>(d.q) + (real ? b * d.q_stride[0] + i * d.q_stride[1] + head * d.q_stride[2] : 0);
#pragma unroll 1
                for (uint32_t y = lane / kLanes; y < 32; y += kAtOnce) {
                    const uint16_t* const q = reinterpret_cast<const uint16_t*>(__shfl_sync(kFull, reinterpret_cast<uintptr_t>(mine), y));
                    const uint32_t there = __shfl_sync(kFull, real, y) && c < dim / 8 ? 16 : 0, to = (warp & 3) * 32 + y;      // (else zeros)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(
                                     smem_addr(tile + (c >> 3) * kBoxBytes + to * 128 + ((c ^ to) & 7) * 16)),
                                 "l"(there ? q + c * 8 : q), "r"(there)
                                 : "memory");
                }
                asm volatile("cp.async.wait_all;\n" ::: "memory");
                __syncwarp();
                if (d.dtype != BS_F16) {
                    // a lane's own row times 2^e with its largest in [2^12, 2^13); rows of zeros, infinities and NaN as they are
                    auto unit_at = [&](uint32_t x) { return reinterpret_cast<uint4*>(tile + (x >> 3) * kBoxBytes + row * 128 + ((x ^ row) & 7) * 16); };
                    uint32_t high = 0;       // magnitudes of bf16 order as integers
#pragma unroll 2
                    for (uint32_t x = 0; x < dim / 8; ++x) {
                        const uint4 w = *unit_at(x);
                        high = __vmaxu2(high, __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
                    }
                    high = max(high >> 16, high & 0xffffu);
                    uint32_t e = high >> 7;  // biased exponent
                    e = high == 0 || e == 255 ? 139 : e < 13 ? 13 : e;
                    const float up = __uint_as_float((266 - e) << 23);
                    row_scale = __uint_as_float((e - 12) << 23);
#pragma unroll 2
                    for (uint32_t x = 0; x < dim / 8; ++x) {
                        uint4 u = *unit_at(x);
                        uint32_t* const w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
                        for (int k = 0; k < 4; ++k) w[k] = Type16<__half>::pack(__uint_as_float(w[k] << 16) * up, __uint_as_float(w[k] & 0xffff0000u) * up);
                        *unit_at(x) = u;
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                __syncwarp();
                if (lane == 0) barrier_arrive(&ctl.q_full[t]);
            }
            // the largest value scale of the piece
            float unit = 0.f;
            {
                const int32_t* const table = d.shared_table + static_cast<uint64_t>(m.m) * d.shared_width;
                const uint32_t past = min(end * kTileTokens, m.tokens);
                for (uint32_t col = (first * kTileTokens >> a.block_log2) + lane; col << a.block_log2 < past; col += 32) {
                    const uint32_t id = table[col];
                    if (id < a.c.num_blocks) unit = fmaxf(unit, a.c.v_scale[static_cast<uint64_t>(id) * hkv + m.h]);
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) unit = fmaxf(unit, __shfl_xor_sync(kFull, unit, o));
            if (!(unit > 0.f)) unit = 1.f;
            const float k_by = d.scale * 1.4426950408889634f * row_scale, v_by = 1.f / unit;
            float top = -INFINITY, sum = 0.f;       // top: in log2 units
            for (uint32_t j = first; j < end; ++j, ++tiles) {
                wait(&ctl.s_full[t], s_used++ & 1);        // and the value product before it is done
                if (stopped()) break;
                fence_after();
                const uint32_t left = m.tokens - j * kTileTokens;
                int done = 0;           // quarters of the tile whose weights are made
                const float2* const scales = ctl.scales[tiles % kScales];
                const uint32_t missing = ctl.missing[tiles % kScales];
                if (left >= kTileTokens && !missing) {
                    if (j == first) top = largest_score(s_at, scales, k_by, v_by);
                    float s[2][32];
                    tmem_load32(s_at, s[0]);
#pragma unroll 1
                    for (; done < 4; done += 2) {
                        uint32_t w16[32];
                        float most;
                        const float part = weights64(s_at + 32 * done, done == 0, s, scales + 2 * done, k_by, v_by, kLift - top, w16, most);
                        if (__any_sync(kFull, real && most > kMost)) break;       // (rows that are none hold anything)
                        sum += part;
                        tmem_store16(s_at + 16 * done, w16);
                        tmem_store16(s_at + 16 * done + 16, w16 + 16);
                    }
                    if (done == 0) wait_loads32(s[0]);
                }
                if (done < 4) {
                    const int quarters = (static_cast<int>(columns(m.tokens, j)) + 31) / 32;
                    const float2 state = weights_with_care(s_at, o_at, done, quarters, left < kTileTokens ? left : kTileTokens, missing, scales, k_by,
                                                           v_by, j > first ? dim : 0, make_float2(top, sum));
                    top = state.x;
                    sum = state.y;
                }
                wait_stores();
                fence_before();
                __syncwarp();
                if (lane == 0) barrier_arrive(&ctl.p_full[t]);
            }
            wait(&ctl.o_full[t], o_used++ & 1);
            if (stopped()) break;
            fence_after();
            // unnormalised outputs, to be joined with those over the sequences' own tokens
            uint32_t b, i, head;
            place(b, i, head);
            const uint64_t at = m.whole ? (static_cast<uint64_t>(b) * d.queries + i) * d.q_heads + head
                                        : (static_cast<uint64_t>(blockIdx.x) * 2 + m.slot) * kPairRows + t * kRows + row;
            float* const out = real ? (m.whole ? a.whole_o : a.part_o) + at * dim : nullptr;
            if (real) (m.whole ? a.whole_ml : a.part_ml)[at] = make_float2(top - kLift, sum);
#pragma unroll 1
            for (uint32_t x = 0; x < dim; x += 32) {
                float o[32];
                tmem_load32(o_at + x, o);
                wait_loads32(o);
                uint32_t u[32];
#pragma unroll
                for (int k = 0; k < 32; ++k) u[k] = __float_as_uint(o[k] * unit);
                store_rows(u, staging, out, x * 4, dim * 4);
            }
            item_read(it);
            // the next item's first value product overwrites the outputs: it
            // waits for weights that this warp makes after these loads
            fence_before();
        }
    }
    fence_before();
    __syncthreads();
    if (warp == kIssuer) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
}

template <int BOXES>
cudaError_t launch(const SharedArgs& a, cudaStream_t stream) {
    const cudaError_t e = cudaFuncSetAttribute(k_shared<BOXES>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem<BOXES>);
    if (e != cudaSuccess) return e;
    return launch_after(k_shared<BOXES>, dim3(a.shares), kThreads, kSmem<BOXES>, stream, a);
}

}  // namespace

cudaError_t launch_shared_part(const SharedArgs& given, cudaStream_t stream) {
    SharedArgs a = given;
    a.polls = wait_polls();
    return a.c.dim <= 64 ? launch<1>(a, stream) : launch<2>(a, stream);
}

}  // namespace bsb
