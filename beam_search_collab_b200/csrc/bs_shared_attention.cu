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
// 8-11 load and convert keys and values, 12 issues the matrix instructions:
//   S_t = Q_t K^T     codes of K exact in the queries' 16-bit type
//   O_t += P_t V      codes of V exact in f16, P_t f16: a weight times its values'
//                     scale, over the largest of the piece, rounded to 2^-11 of
//                     itself or, where that is more, 2^-31 of a weight of 1 at
//                     the largest scale (weights count in 2^-kLift, the room
//                     that a maximum moved at 2^8 leaves)
// The maximum is moved only when a sum of 32 weights passes 2^8 (no maximum is
// taken before the exponentials); sums are 32-bit, of the unrounded weights.
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
constexpr int kThreads = 32 * (kIssuer + 1);
constexpr int kStages = 2;             // of keys, and of values
constexpr float kLift = 7.f, kLifted = 128.f;
constexpr float kMost = 256.f * kLifted;      // of a sum of 32 weights, and so of each: below f16's 65504

template <typename T>
__device__ __forceinline__ uint4 codes_to_16(uint32_t a, uint32_t b);
// Four codes to a word: 0x6400 | u is 1024 + u in f16, minus 1152.
template <>
__device__ __forceinline__ uint4 codes_to_16<__half>(uint32_t a, uint32_t b) {
    uint4 r;
    uint32_t* const w = reinterpret_cast<uint32_t*>(&r);
    a ^= 0x80808080u;
    b ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = __byte_perm(i < 2 ? a : b, 0x64646464u, i & 1 ? 0x4342 : 0x4140);
        const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __float2half2_rn(1152.f));
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return r;
}
// In bf16 0x4300 | x is 128 + x for x < 128: the code's low seven bits, minus
// 128, or 256 where its sign is set.
template <>
__device__ __forceinline__ uint4 codes_to_16<__nv_bfloat16>(uint32_t a, uint32_t b) {
    uint4 r;
    uint32_t* const w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = __byte_perm(i < 2 ? a : b, 0x43434343u, i & 1 ? 0x4342 : 0x4140);
        const uint32_t x = u & 0xff7fff7fu, y = u & 0xff80ff80u;
        const __nv_bfloat162 h = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return r;
}

// 16 codes of row r, two 16-byte units of it.
template <typename T>
__device__ __forceinline__ void put_codes(unsigned char* row, uint32_t unit, uint32_t r, const uint4& x) {
    *reinterpret_cast<uint4*>(row + ((unit ^ r) * 16)) = codes_to_16<T>(x.x, x.y);
    *reinterpret_cast<uint4*>(row + (((unit + 1) ^ r) * 16)) = codes_to_16<T>(x.z, x.w);
}

// Where a block is in its share: tiles t .. end of a segment (group m, key
// head h, pair of row tiles).
struct Piece {
    uint32_t m, segment;       // segment: h * pairs + pair
    uint32_t t, end;
    uint64_t left;             // units of the share after this piece
    Group g;
    uint32_t slot;             // 0: the share's first piece
};

struct Control {
    uint64_t q_full[2], s_full[2], p_full[2], o_full[2], done;
    uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    uint64_t sums[2 * (kIssuer + 1)];
    Piece start;
    uint32_t tmem;
    uint32_t gave_up;
};

template <int BOXES>
constexpr size_t kSmem = 1024 + (2 + 2 * kStages) * BOXES * kBoxBytes + sizeof(Control);

// The piece of a segment from its unit `from` on; its first kStart units
// stand for no tiles.
__device__ __forceinline__ void cut_piece(Piece& p, uint32_t from) {
    const uint32_t cost = p.g.tiles + kStart, take = p.left < cost - from ? static_cast<uint32_t>(p.left) : cost - from;
    p.t = from > kStart ? from - kStart : 0;
    p.end = from + take > kStart ? from + take - kStart : 0;
    p.left -= take;
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

// The first piece of the share that begins at unit `first` (by one warp).
__device__ __forceinline__ void find_piece(const SharedArgs& a, Piece& p, uint64_t first) {
    const uint32_t lane = threadIdx.x & 31;
    uint64_t seen = 0;
    p.m = a.d.num_groups - 1;
    for (uint32_t m0 = 0; m0 < a.d.num_groups; m0 += 32) {       // 32 at a time
        Group g{};
        if (m0 + lane < a.d.num_groups) g = group_of(a, m0 + lane);
        const uint64_t mine = cost_of(g) * a.c.kv_heads;
        uint64_t sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t up = __shfl_up_sync(kFull, sum, o);
            if (lane >= static_cast<uint32_t>(o)) sum += up;
        }
        const unsigned past = __ballot_sync(kFull, seen + sum > first);
        if (past) {
            const int l = __ffs(past) - 1;
            seen += __shfl_sync(kFull, sum - mine, l);
            p.m = m0 + l;
            break;
        }
        seen += __shfl_sync(kFull, sum, 31);
    }
    p.g = group_of(a, p.m);
    if (p.g.tiles == 0) {                                        // (not with lists that stay as they are)
        p.left = p.t = p.end = p.segment = p.slot = 0;
        return;
    }
    const uint32_t cost = p.g.tiles + kStart;
    p.segment = static_cast<uint32_t>((first - seen) / cost);
    p.slot = 0;
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

// 32 scores of a row: weights 2^(key scale * s + base) added to `part`, and
// times their value scale packed in p.  `scales`: a lane below 8 has the tile's
// block's key scale (log2 units), the next 8 lanes the value scales.
__device__ __forceinline__ void weights32(const float* s, float scales, uint32_t col, uint32_t block_log2, float base, uint32_t* p, float& part) {
    const float2 base2 = make_float2(base, base);
    float2 add[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const uint32_t e = (col + 16 * half) >> block_log2;
        const float k = __shfl_sync(kFull, scales, e), v = __shfl_sync(kFull, scales, 8 + e);
#pragma unroll
        for (int i = 8 * half; i < 8 * half + 8; ++i) {
            float2 x = fma2(make_float2(s[2 * i], s[2 * i + 1]), make_float2(k, k), base2);
            x.x = exp2_fast(x.x);
            x.y = exp2_fast(x.y);
            add[i & 1] = add2(add[i & 1], x);
            x = mul2(x, make_float2(v, v));
            p[i] = Type16<__half>::pack(x.x, x.y);
        }
    }
    add[0] = add2(add[0], add[1]);
    part = add[0].x + add[0].y;
}

// The first tile, the last one where the tokens end inside it, tiles with
// blocks that are not there, and where the maximum moves.  From the quarter
// `from` on; `left` tokens of the tile are there, `bad` has a bit for each 16
// that are not.  `state` is the row's maximum (log2) and sum, returned as they
// become.
__device__ __noinline__ float2 weights_with_care(uint32_t s_at, uint32_t o_at, int from, int quarters, int32_t left, uint32_t bad, bool real,
                                                 float scales, uint32_t block_log2, int dim, float2 state) {
    float top = state.x, sum = state.y;
#pragma unroll 1
    for (int c = from; c < quarters; ++c) {
        float s[32];
        tmem_load32(s_at + 32 * c, s);
        wait_loads32(s);
        float z[32];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const float k = __shfl_sync(kFull, scales, (32 * c + 16 * half) >> block_log2);
            const bool gone = bad >> (2 * c + half) & 1;
#pragma unroll
            for (int i = 16 * half; i < 16 * half + 16; ++i) z[i] = gone || 32 * c + i >= left ? -INFINITY : s[i] * k;
        }
        auto make = [&](uint32_t (&p)[16], float& part) {
            const float base = top == -INFINITY ? 0.f : kLift - top;
            part = 0.f;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float v = __shfl_sync(kFull, scales, 8 + ((32 * c + 16 * half) >> block_log2));
#pragma unroll
                for (int i = 8 * half; i < 8 * half + 8; ++i) {
                    const float x = exp2_fast(z[2 * i] + base), y = exp2_fast(z[2 * i + 1] + base);
                    part += x + y;
                    p[i] = Type16<__half>::pack(x * v, y * v);
                }
            }
        };
        uint32_t p[16];
        float part;
        make(p, part);
        if (__any_sync(kFull, real && (part > kMost || top == -INFINITY))) {
            // the maximum moves, what was summed is rescaled
            float next = top;
#pragma unroll
            for (int i = 0; i < 32; ++i) next = fmaxf(next, z[i]);
            const float shrink = next == -INFINITY || top == -INFINITY ? (next == top ? 1.f : 0.f) : exp2_fast(top - next);
            top = next;
            sum *= shrink;
            rescale(s_at, o_at, c, dim, shrink);
            make(p, part);
        }
        sum += part;
        tmem_store16(s_at + 16 * c, p);
    }
    return make_float2(top, sum);
}

template <typename T, int BOXES>
__global__ void __launch_bounds__(kThreads, 1) k_shared(const __grid_constant__ SharedArgs a) {
    extern __shared__ unsigned char raw_smem[];
    unsigned char* const smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t{1023});
    constexpr int kTileBytes = BOXES * kBoxBytes;
    unsigned char* const keys = smem + 2 * kTileBytes;
    unsigned char* const values = keys + kStages * kTileBytes;
    Control& ctl = *reinterpret_cast<Control*>(values + kStages * kTileBytes);
    const bs_shared_attention_desc& d = a.d;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hkv = a.c.kv_heads, dim = a.c.dim, block = a.c.block;

    cudaGridDependencySynchronize();       // in every block, before anything of the caller's
    uint64_t before, all;
    count_cost(a, 0, before, all, ctl.sums);
    const uint64_t w = all * hkv;
    const uint32_t n = used_shares(w, a.shares);
    if (blockIdx.x >= n) return;
    if (warp == 0) {
        const uint64_t first = share_first(w, n, blockIdx.x);
        Piece p;
        p.left = share_first(w, n, blockIdx.x + 1) - first;
        find_piece(a, p, first);
        if (lane == 0) {
            ctl.start = p;
            for (int t = 0; t < 2; ++t) {
                barrier_init(&ctl.q_full[t], 4);
                barrier_init(&ctl.s_full[t], 1);
                barrier_init(&ctl.p_full[t], 4);
                barrier_init(&ctl.o_full[t], 1);
            }
            barrier_init(&ctl.done, 1);
            for (int s = 0; s < kStages; ++s) {
                barrier_init(&ctl.k_full[s], kConverters);
                barrier_init(&ctl.v_full[s], kConverters);
                barrier_init(&ctl.k_empty[s], 1);
                barrier_init(&ctl.v_empty[s], 1);
            }
            ctl.gave_up = 0;
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        }
        __syncwarp();
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
    auto rows_left = [&](const Piece& p) { return p.g.rows - p.segment % p.g.pairs * kPairRows; };     // of the segment, from its first on
    auto pieces = [&](auto&& work) {           // every piece of the share, till `work` says no
        Piece p = ctl.start;
        do {
            if (p.t == p.end) continue;        // (a share that ends before a segment's first tile)
            if (!work(p)) return;
        } while (next_piece(a, p));
    };
    // columns of tile j that hold tokens, to a multiple of 16
    auto columns = [&](const Piece& p, uint32_t j) {
        const uint32_t left = p.g.tokens - j * kTileTokens;
        return left >= kTileTokens ? kTileTokens : (left + 15) & ~15u;
    };

    if (warp == kIssuer) {
        // ---------------------------------------------------- matrix products
        // (the whole warp runs the loop, one elected lane issues)
        constexpr uint32_t kCommon = 1u << 4 | static_cast<uint32_t>(kRows >> 4) << 24;
        constexpr uint32_t kScores = kCommon | Type16<T>::kFormat << 7 | Type16<T>::kFormat << 10;
        const uint32_t what_o = kCommon | 1u << 16 | (dim >> 3) << 17;         // f16 by f16, values not along the contraction
        const int steps = dim / 16;
        const uint64_t q_base = operand(smem_addr(smem), 16, 1024), k_base = operand(smem_addr(keys), 16, 1024);
        const uint64_t v_base = operand(smem_addr(values), kBoxBytes, 1024);
        constexpr uint32_t kTileUnits = kTileBytes / 16, kBoxUnits = kBoxBytes / 16;
        auto scores = [&](int t, uint32_t stage, uint32_t cols) {
            const uint64_t q = q_base + t * kTileUnits, k = k_base + stage * kTileUnits;
            const uint32_t what = kScores | (cols >> 3) << 17;
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
        uint32_t loads = 0, q_used[2] = {0, 0}, p_used[2] = {0, 0};
        bool issued = false;
        pieces([&](const Piece& p) {
            const bool both = rows_left(p) > kRows;
            wait(&ctl.k_full[loads % kStages], loads / kStages & 1);
            for (int t = 0; t <= both; ++t) wait(&ctl.q_full[t], q_used[t]++ & 1);
            if (stopped()) return false;
            issued = true;
            fence_after();
            if (elected()) {
                for (int t = 0; t <= both; ++t) scores(t, loads % kStages, columns(p, p.t));
                mma_commit(&ctl.k_empty[loads % kStages]);
            }
            __syncwarp();
            for (uint32_t j = p.t; j < p.end; ++j, ++loads) {
                const uint32_t stage = loads % kStages, next = (loads + 1) % kStages;
                const bool last = j + 1 == p.end;
                wait(&ctl.v_full[stage], loads / kStages & 1);
                if (!last) wait(&ctl.k_full[next], (loads + 1) / kStages & 1);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (t && !both) break;
                    wait(&ctl.p_full[t], p_used[t]++ & 1);
                    if (stopped()) return false;
                    fence_after();
                    if (elected()) {
                        products(t, stage, j > p.t, columns(p, j));
                        if (last) mma_commit(&ctl.o_full[t]);
                        else scores(t, next, columns(p, j + 1));
                    }
                    __syncwarp();
                }
                if (elected()) {
                    mma_commit(&ctl.v_empty[stage]);
                    if (!last) mma_commit(&ctl.k_empty[next]);
                }
                __syncwarp();
            }
            return true;
        });
        // TMEM and the stages are in use until this
        if (issued) {
            if (elected()) mma_commit(&ctl.done);
            __syncwarp();
            for (unsigned i = 0; i < kPolls && !barrier_test(&ctl.done, 0); ++i) {}
        }
        __syncwarp();
    } else if (warp >= 8) {
        // --------------------------------------------------------- conversion
        // (eight lanes: one 16-byte chunk of eight tokens side by side, so that
        // the swizzled stores fall on all banks; four such for 64 bytes of a row)
        const uint32_t who = threadIdx.x - 256, sub = who >> 3, nw = dim / 16;
        constexpr int kEach = 4 * BOXES;                     // chunks of a thread, of keys and of values
        uint32_t row_of[kEach], chunk_of[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint32_t u = sub + 16 * i;                 // of 16 * nw
            row_of[i] = u / nw * 8 + (who & 7);
            chunk_of[i] = u % nw;
        }
        // chunk i's place in the codes, in 16 bytes; kNothing: there are none
        constexpr uint64_t kNothing = ~0ull;
        auto find = [&](const Piece& p, uint32_t j, uint64_t (&place)[kEach]) {
            const int32_t* const table = d.shared_table + static_cast<uint64_t>(p.m) * d.shared_width;
            const uint32_t first = j * kTileTokens, h = p.segment / p.g.pairs;
            uint32_t id[kEach];
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const uint32_t pos = first + row_of[i];
                id[i] = i < static_cast<int>(nw) && (pos & ~15u) < p.g.tokens ? static_cast<uint32_t>(table[pos >> a.block_log2]) : kNoNode;
            }
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const uint32_t pos = first + row_of[i];
                place[i] = (((static_cast<uint64_t>(id[i]) * hkv + h) << a.block_log2) + (pos & (block - 1))) * nw + chunk_of[i];
                if (id[i] >= a.c.num_blocks) {
                    if (i < static_cast<int>(nw) && (pos & ~15u) < p.g.tokens) atomicOr(a.errors, kMemErrBlock);
                    place[i] = kNothing;
                }
            }
        };
        auto load = [&](const int8_t* codes, const uint64_t (&place)[kEach], uint4 (&x)[kEach]) {
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                x[i] = place[i] != kNothing ? reinterpret_cast<const uint4*>(codes)[place[i]] : make_uint4(0, 0, 0, 0);
        };
        uint32_t loads = 0;
        auto leave = [&](const uint4 (&x)[kEach], bool is_v) {
            const uint32_t stage = loads % kStages;
            wait(&(is_v ? ctl.v_empty : ctl.k_empty)[stage], (loads / kStages & 1) ^ 1);
            if (stopped()) return false;
            unsigned char* const to = (is_v ? values : keys) + stage * kTileBytes;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                if (i >= static_cast<int>(nw)) break;
                unsigned char* const row = to + (chunk_of[i] >> 2) * kBoxBytes + row_of[i] * 128;
                const uint32_t unit = (chunk_of[i] & 3) * 2, r = row_of[i] & 7;
                if (is_v) put_codes<__half>(row, unit, r, x[i]);
                else put_codes<T>(row, unit, r, x[i]);
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) barrier_arrive(&(is_v ? ctl.v_full : ctl.k_full)[stage]);
            return true;
        };
        // each tile's codes are on their way while the one before is converted
        Piece p = ctl.start;
        bool more = true;
        auto skip = [&]() {
            while (more && p.t == p.end) more = next_piece(a, p);
        };
        skip();
        uint32_t j = p.t;
        uint64_t place[kEach];
        uint4 k[kEach], v[kEach];
        if (more) {
            find(p, j, place);
            load(a.c.k, place, k);
            load(a.c.v, place, v);
        }
        while (more) {
            if (++j == p.end) {
                more = next_piece(a, p);
                skip();
                j = p.t;
            }
            if (more) find(p, j, place);
            if (!leave(k, false)) break;
            if (more) load(a.c.k, place, k);
            if (!leave(v, true)) break;
            if (more) load(a.c.v, place, v);
            ++loads;
        }
    } else {
        // ----------------------------------------------------------- softmax
        const uint32_t t = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (warp & 3) * 32 << 16;                  // this warp's TMEM lanes
        const uint32_t s_at = tmem + t * 128 + lanes, o_at = tmem + 256 + t * 128 + lanes;
        unsigned char* const tile = smem + t * kTileBytes;
        unsigned char* const staging = tile + (warp & 3) * 4096;       // the queries' place, once they are done with
        const float score_scale = d.scale * 1.4426950408889634f;
        const uint32_t per_tile = kTileTokens >> a.block_log2, e = lane & 7;
        const bool has_scale = lane < 16 && e < per_tile;
        uint32_t s_used = 0, o_used = 0;
        pieces([&](const Piece& p) {
            if (rows_left(p) <= t * kRows) return true;
            const uint32_t h = p.segment / p.g.pairs, r = p.segment % p.g.pairs * kPairRows + t * kRows + row;
            const bool real = r < p.g.rows;
            const uint32_t b = p.g.first + r / a.rows, i = r % a.rows / a.group, head = h * a.group + r % a.rows % a.group;
            // this row's query
            {
                const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(d.q) + b * d.q_stride[0] + i * d.q_stride[1] +
                                                                head * d.q_stride[2]);
#pragma unroll
                for (int c0 = 0; c0 < 8 * BOXES; c0 += 8) {
                    uint4 x[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c) x[c] = real && c0 + c < static_cast<int>(dim / 8) ? q[c0 + c] : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        *reinterpret_cast<uint4*>(tile + (c0 >> 3) * kBoxBytes + row * 128 + ((c ^ row) & 7) * 16) = x[c];
                }
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                __syncwarp();
                if (lane == 0) barrier_arrive(&ctl.q_full[t]);
            }
            const int32_t* const table = d.shared_table + static_cast<uint64_t>(p.m) * d.shared_width;
            const uint32_t blocks = (p.g.tokens + block - 1) >> a.block_log2;
            auto id_at = [&](uint32_t col) { return col < blocks ? static_cast<uint32_t>(table[col]) : 0u; };
            // the largest value scale of the piece
            float unit = 0.f;
            for (uint32_t col = p.t * per_tile + lane; col < min(p.end * per_tile, blocks); col += 32) {
                const uint32_t id = table[col];
                if (id < a.c.num_blocks) unit = fmaxf(unit, a.c.v_scale[static_cast<uint64_t>(id) * hkv + h]);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) unit = fmaxf(unit, __shfl_xor_sync(kFull, unit, o));
            if (!(unit > 0.f)) unit = 1.f;
            const float factor = lane < 8 ? score_scale : 1.f / unit;
            auto scale_of = [&](uint32_t id, bool& missing) {          // of block e of a tile: lanes below 8 keys', the next 8 values'
                missing = has_scale && id >= a.c.num_blocks;
                if (!has_scale || missing) return 0.f;
                return (lane < 8 ? a.c.k_scale : a.c.v_scale)[static_cast<uint64_t>(id) * hkv + h] * factor;
            };
            bool missing;
            float next_scales = scale_of(id_at(p.t * per_tile + e), missing);
            uint32_t next_bad = __ballot_sync(kFull, missing), next_id = id_at((p.t + 1) * per_tile + e);
            float top = -INFINITY, sum = 0.f;       // top: in log2 units, moved when weights are past 2^8
            for (uint32_t j = p.t; j < p.end; ++j) {
                const float scales = next_scales;
                const uint32_t bad_blocks = next_bad & 255u;
                if (j + 1 < p.end) {
                    next_scales = scale_of(next_id, missing);
                    next_bad = __ballot_sync(kFull, missing);
                    next_id = id_at((j + 2) * per_tile + e);
                }
                wait(&ctl.s_full[t], s_used++ & 1);        // and the value product before it is done
                if (stopped()) return false;
                fence_after();
                const uint32_t left = p.g.tokens - j * kTileTokens;
                int done = 0;           // quarters of the tile whose weights are made
                if (j > p.t && left >= kTileTokens && !bad_blocks) {
                    float s[2][32];
                    tmem_load32(s_at, s[0]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        wait_loads32(s[c & 1]);
                        if (c < 3) tmem_load32(s_at + 32 * (c + 1), s[(c + 1) & 1]);
                        uint32_t w16[16];
                        float part;
                        weights32(s[c & 1], scales, 32 * c, a.block_log2, kLift - top, w16, part);
                        if (__any_sync(kFull, real && part > kMost)) break;       // (rows that are none hold zeros)
                        sum += part;
                        tmem_store16(s_at + 16 * c, w16);
                        done = c + 1;
                    }
                    if (done < 4) {
                        wait_loads32(s[0]);
                        wait_loads32(s[1]);
                    }
                }
                if (done < 4) {
                    uint32_t bad = 0;       // by 16 columns
                    for (uint32_t x = 0; bad_blocks && x < 8; ++x) bad |= (bad_blocks >> ((16 * x) >> a.block_log2) & 1) << x;
                    const int quarters = (static_cast<int>(columns(p, j)) + 31) / 32;
                    const float2 state = weights_with_care(s_at, o_at, done, quarters, left < kTileTokens ? left : kTileTokens, bad, real, scales,
                                                           a.block_log2, j > p.t ? dim : 0, make_float2(top, sum));
                    top = state.x;
                    sum = state.y;
                }
                wait_stores();
                fence_before();
                __syncwarp();
                if (lane == 0) barrier_arrive(&ctl.p_full[t]);
            }
            wait(&ctl.o_full[t], o_used++ & 1);
            if (stopped()) return false;
            fence_after();
            // unnormalised outputs, to be joined with those over the sequences' own tokens
            const bool whole = p.t == 0 && p.end == p.g.tiles;
            const uint64_t at = whole ? (static_cast<uint64_t>(b) * d.queries + i) * d.q_heads + head
                                      : (static_cast<uint64_t>(blockIdx.x) * 2 + p.slot) * kPairRows + t * kRows + row;
            float* const out = real ? (whole ? a.whole_o : a.part_o) + at * dim : nullptr;
            for (uint32_t x = 0; x < dim; x += 32) {
                float o[32];
                tmem_load32(o_at + x, o);
                wait_loads32(o);
                uint32_t u[32];
#pragma unroll
                for (int k = 0; k < 32; ++k) u[k] = __float_as_uint(o[k] * unit);
                store_rows(u, staging, out, x * 4, dim * 4);
            }
            if (real) (whole ? a.whole_ml : a.part_ml)[at] = make_float2(top - kLift, sum);
            // the next piece's first value product overwrites the outputs: it
            // waits for weights that this warp makes after these loads
            fence_before();
            return true;
        });
    }
    fence_before();
    __syncthreads();
    if (warp == kIssuer) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
}

template <typename T, int BOXES>
cudaError_t launch(const SharedArgs& a, cudaStream_t stream) {
    const cudaError_t e = cudaFuncSetAttribute(k_shared<T, BOXES>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem<BOXES>);
    if (e != cudaSuccess) return e;
    return launch_after(k_shared<T, BOXES>, dim3(a.shares), kThreads, kSmem<BOXES>, stream, a);
}

}  // namespace

cudaError_t launch_shared_part(const SharedArgs& given, cudaStream_t stream) {
    SharedArgs a = given;
    a.polls = wait_polls();
    if (a.d.dtype == BS_F16) return a.c.dim <= 64 ? launch<__half, 1>(a, stream) : launch<__half, 2>(a, stream);
    return a.c.dim <= 64 ? launch<__nv_bfloat16, 1>(a, stream) : launch<__nv_bfloat16, 2>(a, stream);
}

}  // namespace bsb
