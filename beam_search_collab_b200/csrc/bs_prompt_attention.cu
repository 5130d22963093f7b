// bs_prompt_attention.cu -- attention of packed prompts (include/bsearch.h,
// bs_prompt_attention).
//
// One thread block computes two tiles of 128 query rows against the keys they
// see, 128 at a time, with a running maximum and sum per row.  The rows of a
// tile are consecutive tokens times the query heads that share a key head, so
// a tile's keys and values are loaded once for all those heads.
//
// Warps 0-3 and 4-7 are the softmax of tile 0 and 1 (a thread has one row),
// warp 8 issues the matrix instructions, warp 9 the copies:
//   copies    query tiles, then keys and values through one ring of stages
//             (tiled TMA, 128-byte swizzle, 64 columns of a row at a time)
//   matrix    S_t = Q_t K^T    (both K-major in shared memory, S_t in TMEM)
//             O_t += P_t V     (P_t in TMEM over S_t's columns, V MN-major)
//             in the order S0 S1 | P0V S0' P1V S1' | ...: while one tile's
//             softmax runs, the tensor pipe has the other tile's work
//   softmax   S_t to registers, P_t = 2^(scale' S_t - m) back to TMEM in the
//             inputs' 16-bit type.  m is moved only when a row's maximum has
//             grown by more than 2^8 (then O_t, in TMEM, is rescaled), so most
//             tiles touch O_t not at all; sums are 32-bit of the unrounded P.
// TMEM (512 columns): S0 S1 O0 O1, 128 columns each.
//
// Keys of other sequences or of the future that a tile also covers are set to
// -infinity in S.  A zero weight would still pass an infinity or NaN of a
// hidden VALUE on, so in tiles with hidden keys the copying warp clears value
// rows past the sequence, and rows that are not finite and not seen by all;
// the softmax adds the latter for the rows that see them (never taken with
// finite inputs).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bs_device.cuh"
#include "bs_memory.h"

namespace bsb {

using namespace dev;

namespace {

constexpr int kRows = 128;             // query rows of a tile, keys of a tile
constexpr int kThreads = 320;
constexpr int kBoxBytes = kRows * 128; // 128 rows of 64 elements
constexpr unsigned kPolls = 1u << 22;
constexpr float kMost = 256.f;         // weights may grow to this before the maximum is moved

struct PromptArgs {
    bs_prompt_attention_desc d;
    unsigned int* errors;
    uint32_t group;            // query heads per key head
    uint32_t tile_tokens;      // tokens of a tile: group * tile_tokens <= 128 rows
    CUtensorMap q, k, v;
};

__device__ __forceinline__ unsigned smem_addr(const void* p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void barrier_init(uint64_t* b, unsigned count) {
    asm volatile("mbarrier.init.shared.b64 [%0], %1;\n" ::"r"(smem_addr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared.b64 _, [%0];\n" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint64_t* b, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;\n" ::"r"(smem_addr(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_test(uint64_t* b, unsigned phase) {
    unsigned ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok)
                 : "r"(smem_addr(b)), "r"(phase)
                 : "memory");
    return ok != 0;
}

// 64 columns x rows x 1 of a tensor (dim, heads, tokens) into shared memory.
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
            smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
        : "memory");
}

// Shared-memory operand: 128-byte swizzled rows, groups of 8 rows `sbo` bytes
// apart; `lbo`: from 64 columns to the next, where the columns are not the
// contraction's.
__device__ __forceinline__ uint64_t operand(unsigned addr, unsigned lbo, unsigned sbo) {
    return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | static_cast<uint64_t>(lbo >> 4) << 16 |
           static_cast<uint64_t>(sbo >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t what, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(what), "r"(static_cast<unsigned>(add))
                 : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t what, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(what), "r"(static_cast<unsigned>(add))
                 : "memory");
}
__device__ __forceinline__ bool elected() {
    unsigned yes;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(yes));
    return yes != 0;
}
// The barrier completes when every matrix instruction issued so far has.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
// (The registers are named so that nothing computed from them moves ahead.)
__device__ __forceinline__ void wait_loads32(float* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]),
                   "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]),
                   "+f"(r[14]), "+f"(r[15]), "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]),
                   "+f"(r[21]), "+f"(r[22]), "+f"(r[23]), "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]),
                   "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void wait_loads16(float* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]),
                   "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]),
                   "+f"(r[14]), "+f"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// 32, 16 or 1 columns of the warp's 32 TMEM lanes: a register each.
__device__ __forceinline__ void tmem_load32(uint32_t at, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]),
          "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]),
          "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]),
          "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t* u) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};\n" ::"r"(u[0]),
        "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]),
        "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]),
        "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31]), "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t at, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]),
          "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const float* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n" ::"f"(r[0]),
        "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]), "f"(r[8]), "f"(r[9]), "f"(r[10]), "f"(r[11]),
        "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15]), "r"(at)
        : "memory");
}
__device__ __forceinline__ uint32_t tmem_load1(uint32_t at) {
    uint32_t u;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\ntcgen05.wait::ld.sync.aligned;\n" : "=r"(u) : "r"(at) : "memory");
    return u;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n .reg .b64 a, b, c, r;\n mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 c, {%6, %7}; fma.rn.f32x2 r, a, b, c; mov.b64 {%0, %1}, r;\n}\n"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n .reg .b64 a, b, r;\n mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; add.rn.f32x2 r, a, b; mov.b64 {%0, %1}, r;\n}\n"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

template <typename T>
struct Type16;
template <>
struct Type16<__half> {
    static constexpr uint32_t kFormat = 0, kExponent = 0x7c007c00u;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
    static __device__ __forceinline__ uint32_t larger(uint32_t x, uint32_t y) {
        const __half2 h = __hmax2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&y));
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <>
struct Type16<__nv_bfloat16> {
    static constexpr uint32_t kFormat = 1, kExponent = 0x7f807f80u;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u)); }
    static __device__ __forceinline__ uint32_t larger(uint32_t x, uint32_t y) {
        const __nv_bfloat162 h = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};

// Stages of keys or values that fit beside the query tiles.
template <int BOXES>
constexpr int kStagesOf = BOXES == 2 ? 5 : 8;

// The row's largest score among the `left` first of a tile.
__device__ __forceinline__ float largest(uint32_t s_at, int32_t left) {
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < kRows / 32; ++c) {
        float s[32];
        tmem_load32(s_at + 32 * c, s);
        wait_loads32(s);
#pragma unroll
        for (int i = 0; i < 32; ++i) m[i & 3] = fmaxf(m[i & 3], 32 * c + i < left ? s[i] : -INFINITY);
    }
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// One row of a tile: weights 2^(scale * s + base), packed in p, their sum in
// `part`; returns the largest weight.  Scores come from TMEM 32 at a time, the
// next 32 on their way meanwhile.
template <typename T, bool HIDES>
__device__ __forceinline__ float weights(uint32_t s_at, int32_t left, float scale, float base, uint32_t (&p)[kRows / 2], float& part) {
    const float2 scale2 = make_float2(scale, scale), base2 = make_float2(base, base);
    float2 add[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    uint32_t high[2] = {0, 0};
    float s[2][32];
    tmem_load32(s_at, s[0]);
#pragma unroll
    for (int c = 0; c < kRows / 32; ++c) {
        float* now = s[c & 1];
        wait_loads32(now);
        if (c + 1 < kRows / 32) tmem_load32(s_at + 32 * (c + 1), s[(c + 1) & 1]);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float2 x = make_float2(now[2 * i], now[2 * i + 1]);
            if (HIDES) {
                x.x = 32 * c + 2 * i < left ? x.x : -INFINITY;
                x.y = 32 * c + 2 * i + 1 < left ? x.y : -INFINITY;
            }
            x = fma2(x, scale2, base2);
            x.x = exp2_fast(x.x);
            x.y = exp2_fast(x.y);
            add[i & 1] = add2(add[i & 1], x);
            p[16 * c + i] = Type16<T>::pack(x.x, x.y);
            high[i & 1] = Type16<T>::larger(high[i & 1], p[16 * c + i]);
        }
    }
    add[0] = add2(add[0], add[1]);
    part = add[0].x + add[0].y;
    const float2 h = Type16<T>::unpack(Type16<T>::larger(high[0], high[1]));
    return fmaxf(h.x, h.y);
}

struct Control {
    uint64_t q_full[2], s_full[2], p_full[2], o_full[2], done, raw;
    uint64_t full[8], empty[8];
    uint32_t not_finite[8][4];      // by stage: value rows cleared because they are not finite
    uint32_t keep[2];               // outputs hold something before the first value product
    uint32_t tmem;
    uint32_t gave_up;
};

template <int BOXES>
constexpr size_t kSmem = 1024 + (2 + kStagesOf<BOXES>) * BOXES * kBoxBytes + sizeof(Control);

// BOXES: 64-column boxes of a row (1: dim <= 64, 2: dim <= 128).
template <typename T, int BOXES>
__global__ void __launch_bounds__(kThreads, 1) k_prompt(const __grid_constant__ PromptArgs a) {
    extern __shared__ unsigned char raw_smem[];
    unsigned char* const smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t{1023});
    constexpr int kStages = kStagesOf<BOXES>, kTileBytes = BOXES * kBoxBytes;
    unsigned char* const ring = smem + 2 * kTileBytes;
    Control& ctl = *reinterpret_cast<Control*>(smem + (2 + kStages) * kTileBytes);
    const bs_prompt_attention_desc& d = a.d;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // which sequence, tokens and key head: sequence b has the blocks
    // base(b) .. base(b + 1), base(b) = cu_q[b] / pair + b, enough for its
    // ceil(len / pair) pairs of tiles; the last pair, with the most keys, first
    const uint32_t pair = 2 * a.tile_tokens, kv_head = blockIdx.x % d.kv_heads, place = blockIdx.x / d.kv_heads;
    uint32_t b = 0;
    if (d.num_seqs > 1) {
        uint32_t at_or_below = 0;
        for (uint32_t b0 = 0; b0 < d.num_seqs; b0 += kThreads) {
            const uint32_t i = b0 + threadIdx.x;
            const uint32_t n = __syncthreads_count(i < d.num_seqs && static_cast<uint32_t>(d.cu_q[i]) / pair + i <= place);
            at_or_below += n;
            if (n < kThreads) break;
        }
        if (at_or_below == 0) return;
        b = at_or_below - 1;
    }
    const int32_t q0 = d.cu_q[b], q1 = d.cu_q[b + 1], k0 = d.cu_k[b], k1 = d.cu_k[b + 1];
    if (q0 < 0 || q1 < q0 || static_cast<uint32_t>(q1) > d.total_q || k0 < 0 || k1 < k0 || static_cast<uint32_t>(k1) > d.total_k) {
        if (threadIdx.x == 0) atomicOr(a.errors, kMemErrLength);
        return;
    }
    const int32_t lq = q1 - q0, lk = k1 - k0;
    const uint32_t pairs = (lq + pair - 1) / pair, local = place - (static_cast<uint32_t>(q0) / pair + b);
    if (local >= pairs) return;
    const int32_t token0 = (pairs - 1 - local) * pair;
    // keys a token sees, and tiles of keys of each tile of queries
    const int32_t ahead = lk - lq + 1;
    auto seen = [&](int32_t token) { return d.causal ? max(0, min(lk, token + ahead)) : lk; };
    int32_t tiles[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int32_t first = token0 + t * static_cast<int32_t>(a.tile_tokens);
        const int32_t last = min(first + static_cast<int32_t>(a.tile_tokens), lq) - 1;
        tiles[t] = last < first ? 0 : (seen(last) + kRows - 1) / kRows;
    }
    const int32_t n = max(tiles[0], tiles[1]);
    const int32_t all_see = seen(token0);        // keys that every row of the pair sees

    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_addr(&ctl.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            barrier_init(&ctl.q_full[t], 1);
            barrier_init(&ctl.s_full[t], 1);
            barrier_init(&ctl.p_full[t], 4);
            barrier_init(&ctl.o_full[t], 1);
        }
        barrier_init(&ctl.done, 1);
        barrier_init(&ctl.raw, 1);
        for (int s = 0; s < kStages; ++s) {
            barrier_init(&ctl.full[s], 1);
            barrier_init(&ctl.empty[s], 1);
        }
        ctl.keep[0] = ctl.keep[1] = ctl.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = ctl.tmem;

    // A bounded wait.  Once one has given up none waits any more: the warps
    // leave their loops, what is in flight is waited for (bounded too), and
    // nothing is stored.
    volatile uint32_t* const gave_up = &ctl.gave_up;
    auto wait = [&](uint64_t* bar, unsigned phase) {
        for (unsigned i = 0; i < kPolls && !*gave_up; ++i)
            if (barrier_test(bar, phase)) return;
        if (!*gave_up) {
            *gave_up = 1;
            atomicOr(a.errors, kMemErrWait);
        }
    };

    if (warp == 9) {
        // ------------------------------------------------------------ copies
        uint32_t stage = 0, phase = 0;
        if (lane == 0) {
            for (int t = 0; t < 2; ++t) {
                if (!tiles[t]) continue;
                barrier_expect(&ctl.q_full[t], BOXES * 128 * a.group * a.tile_tokens);
                for (int x = 0; x < BOXES; ++x)
                    load_box(smem + t * kTileBytes + x * kBoxBytes, &a.q, 64 * x, kv_head * a.group,
                             q0 + token0 + t * static_cast<int32_t>(a.tile_tokens), &ctl.q_full[t]);
            }
        }
        uint32_t raw_phase = 0;
        int32_t loads = 0;
        bool stop = false;
        for (int32_t j = 0; j < n && !stop; ++j) {
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                unsigned char* const dst = ring + stage * kTileBytes;
                // value rows of this tile that not all rows see, and rows past the sequence
                const int32_t hidden = max(0, all_see - j * kRows), past = lk - j * kRows;
                const bool look = kv == 1 && hidden < kRows;
                if (lane == 0) wait(&ctl.empty[stage], phase ^ 1);
                stop = __shfl_sync(kFull, *gave_up, 0) != 0;
                if (stop) break;
                ++loads;
                if (lane == 0) {
                    uint64_t* const bar = look ? &ctl.raw : &ctl.full[stage];
                    barrier_expect(bar, kTileBytes);
                    for (int x = 0; x < BOXES; ++x)
                        load_box(dst + x * kBoxBytes, kv ? &a.v : &a.k, 64 * x, kv_head, k0 + j * kRows, bar);
                    if (look)
                        for (unsigned i = 0; i < kPolls && !barrier_test(&ctl.raw, raw_phase); ++i) {}
                }
                __syncwarp();
                if (look) {
                    raw_phase ^= 1;
#pragma unroll 1
                    for (int i = 0; i < kRows / 32; ++i) {
                        const int32_t r = 32 * i + lane;
                        bool odd = false;
                        if (r >= hidden && r < past) {
#pragma unroll 1
                            for (int x = 0; x < BOXES; ++x)
                                for (int u = 0; u < 8; ++u) {
                                    const uint4 w = *reinterpret_cast<const uint4*>(dst + x * kBoxBytes + r * 128 + ((u + lane) & 7) * 16);
                                    constexpr uint32_t e = Type16<T>::kExponent;
                                    odd |= (__vcmpeq2(w.x & e, e) | __vcmpeq2(w.y & e, e) | __vcmpeq2(w.z & e, e) | __vcmpeq2(w.w & e, e)) != 0;
                                }
                        }
                        const uint32_t rows = __ballot_sync(kFull, odd);
                        if (lane == 0) ctl.not_finite[stage][i] = rows;
                        if (odd || r >= past) {
#pragma unroll 1
                            for (int x = 0; x < BOXES; ++x)
                                for (int u = 0; u < 8; ++u)
                                    *reinterpret_cast<uint4*>(dst + x * kBoxBytes + r * 128 + ((u + lane) & 7) * 16) = make_uint4(0, 0, 0, 0);
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    __syncwarp();
                    if (lane == 0) barrier_arrive(&ctl.full[stage]);
                }
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
        // no copy may be in flight when the block ends
        if (lane == 0) {
            for (int t = 0; t < 2; ++t)
                for (unsigned i = 0; tiles[t] && i < kPolls && !barrier_test(&ctl.q_full[t], 0); ++i) {}
            for (int32_t i = max(0, loads - kStages); i < loads; ++i)
                for (unsigned x = 0; x < kPolls && !barrier_test(&ctl.full[i % kStages], (i / kStages) & 1); ++x) {}
        }
        __syncwarp();
    } else if (warp == 8) {
        // ---------------------------------------------------- matrix products
        // (the whole warp runs the loop, one elected lane issues)
        if (n > 0) {
            constexpr uint32_t kCommon = 1u << 4 | Type16<T>::kFormat << 7 | Type16<T>::kFormat << 10 | (kRows >> 4) << 24;
            const uint32_t what_s = kCommon | (kRows >> 3) << 17;
            const uint32_t what_o = kCommon | 1u << 16 | static_cast<uint32_t>(d.dim >> 3) << 17;
            // what the lane does per instruction counts: operands are a base
            // and constants (16-byte units)
            const int steps = d.dim / 16;
            const uint64_t q_base = operand(smem_addr(smem), 16, 1024), k_base = operand(smem_addr(ring), 16, 1024);
            const uint64_t v_base = operand(smem_addr(ring), kBoxBytes, 1024);
            constexpr uint32_t kTileUnits = kTileBytes / 16, kBoxUnits = kBoxBytes / 16;
            auto scores = [&](int t, uint32_t stage) {
                const uint64_t q = q_base + t * kTileUnits, k = k_base + stage * kTileUnits;
                if (elected()) {
#pragma unroll
                    for (int i = 0; i < 4 * BOXES; ++i) {
                        const uint32_t off = (i >> 2) * kBoxUnits + (i & 3) * 2;
                        if (i < steps) mma_shared(tmem + t * 128, q + off, k + off, what_s, i > 0);
                    }
                    mma_commit(&ctl.s_full[t]);
                }
                __syncwarp();
            };
            auto values = [&](int t, uint32_t stage, bool add) {
                const uint64_t v = v_base + stage * kTileUnits;
                if (elected()) {
#pragma unroll
                    for (int i = 0; i < kRows / 16; ++i)
                        mma_tmem(tmem + 256 + t * 128, tmem + t * 128 + i * 8, v + i * 128, what_o, add || i > 0);
                }
                __syncwarp();
            };
            auto commit = [&](uint64_t* bar) {
                if (elected()) mma_commit(bar);
                __syncwarp();
            };
            auto full = [&](int32_t i) { wait(&ctl.full[i % kStages], (i / kStages) & 1); };
            full(0);
            for (int t = 0; t < 2; ++t) {
                if (!tiles[t]) continue;
                wait(&ctl.q_full[t], 0);
                fence_after();
                scores(t, 0);
            }
            commit(&ctl.empty[0]);
            for (int32_t j = 0; j < n; ++j) {
                if (__any_sync(kFull, *gave_up != 0)) break;
                const int32_t v_load = 2 * j + 1, k_load = 2 * j + 2;
                full(v_load);
                if (j + 1 < n) full(k_load);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (j >= tiles[t]) continue;
                    wait(&ctl.p_full[t], j & 1);
                    fence_after();
                    values(t, v_load % kStages, j > 0 || ctl.keep[t]);
                    if (j + 1 == tiles[t]) commit(&ctl.o_full[t]);
                    else scores(t, k_load % kStages);
                }
                commit(&ctl.empty[v_load % kStages]);
                if (j + 1 < n) commit(&ctl.empty[k_load % kStages]);
            }
            // TMEM and the stages are in use until this
            commit(&ctl.done);
            for (unsigned i = 0; i < kPolls && !barrier_test(&ctl.done, 0); ++i) {}
        }
        __syncwarp();
    } else {
        // ----------------------------------------------------------- softmax
        const uint32_t t = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (warp & 3) * 32 << 16;                  // this warp's TMEM lanes
        const uint32_t s_at = tmem + t * 128 + lanes, o_at = tmem + 256 + t * 128 + lanes;
        const int32_t token = token0 + static_cast<int32_t>(t * a.tile_tokens + row / a.group);
        const bool real = row < a.group * a.tile_tokens && token < lq;
        const int32_t limit = real ? seen(token) : 0;
        const int32_t mine = t ? tiles[1] : tiles[0];
        const float scale = d.scale * 1.4426950408889634f;
        float top = -INFINITY, sum = 0.f;       // top: of the unscaled scores
        for (int32_t j = 0; j < mine && !*gave_up; ++j) {
            wait(&ctl.s_full[t], j & 1);        // and the value product before it is done
            fence_after();
            const bool hides = (j + 1) * kRows > all_see;
            const int32_t left = limit - j * kRows;         // keys of this tile that the row sees
            if (j == 0) top = largest(s_at, left);
            uint32_t p[kRows / 2];
            float part;
            for (bool again = false;; again = true) {
                const float base = top == -INFINITY ? 0.f : -top * scale;
                const float high = hides ? weights<T, true>(s_at, left, scale, base, p, part) : weights<T, false>(s_at, left, scale, base, p, part);
                if (again || !__any_sync(kFull, real && high > kMost)) break;     // (other rows hold anything)
                // rare: the maximum moves, what was summed is rescaled
                const float next = fmaxf(top, largest(s_at, left));
                const float shrink = next == -INFINITY ? 1.f : exp2_fast((top - next) * scale);
                sum *= shrink;
                for (int x = 0; x < d.dim; x += 16) {
                    float o[16];
                    tmem_load16(o_at + x, o);
                    wait_loads16(o);
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] *= shrink;
                    tmem_store16(o_at + x, o);
                }
                top = next;
            }
            sum += part;
            tmem_store32(s_at, p);
            tmem_store32(s_at + 32, p + 32);
            wait_stores();
            if (hides) {
                // value rows that were cleared because they are not finite,
                // for the query rows that see them
                const uint32_t stage = (2 * j + 1) % kStages;
                wait(&ctl.full[stage], ((2 * j + 1) / kStages) & 1);
                const uint32_t* odd = ctl.not_finite[stage];
                if (j == 0 && (odd[0] | odd[1] | odd[2] | odd[3])) {
                    const float zeros[16] = {};
                    for (int x = 0; x < d.dim; x += 16) tmem_store16(o_at + x, zeros);
                    wait_stores();
                    ctl.keep[t] = 1;
                }
                for (int w = 0; w < 4; ++w)
                    for (uint32_t left = odd[w]; left; left &= left - 1) {
                        const int r = 32 * w + __ffs(left) - 1;
                        const uint32_t two = tmem_load1(s_at + r / 2);
                        const float2 f = Type16<T>::unpack(two);
                        const float weight = r & 1 ? f.y : f.x;
                        const T* v = static_cast<const T*>(d.v) + (k0 + j * kRows + r) * d.v_stride[0] + kv_head * d.v_stride[1];
                        for (int x = 0; x < d.dim; x += 16) {
                            float o[16];
                            tmem_load16(o_at + x, o);
                            wait_loads16(o);
                            if (j * kRows + r < limit)
                                for (int i = 0; i < 16; ++i) o[i] += weight * static_cast<float>(v[x + i]);
                            __syncwarp();
                            tmem_store16(o_at + x, o);
                            wait_stores();
                        }
                    }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) barrier_arrive(&ctl.p_full[t]);
        }
        if (mine > 0) {
            wait(&ctl.o_full[t], 0);
            fence_after();
        }
        const bool ok = real && !*gave_up;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const uint64_t at = (static_cast<uint64_t>(q0) + token) * d.q_heads + kv_head * a.group + row % a.group;
        T* out = static_cast<T*>(d.out) + at * d.dim;
        for (int x = 0; x < d.dim; x += 16) {
            float o[16];
            if (mine > 0) {
                tmem_load16(o_at + x, o);
                wait_loads16(o);
            }
            uint32_t u[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = mine > 0 && sum != 0.f ? Type16<T>::pack(o[2 * i] * inv, o[2 * i + 1] * inv) : 0;
            if (ok) {
                reinterpret_cast<uint4*>(out + x)[0] = make_uint4(u[0], u[1], u[2], u[3]);
                reinterpret_cast<uint4*>(out + x)[1] = make_uint4(u[4], u[5], u[6], u[7]);
            }
        }
        if (ok && d.lse) d.lse[at] = sum == 0.f ? -INFINITY : top * d.scale + logf(sum);
    }
    fence_before();
    __syncthreads();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                              CUtensorMapFloatOOBfill);

cudaError_t encoder(EncodeFn& out) {
    static EncodeFn fn = nullptr;
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r);
        if (e != cudaSuccess) return e;
        if (r != cudaDriverEntryPointSuccess || !p) return cudaErrorNotSupported;
        fn = reinterpret_cast<EncodeFn>(p);
    }
    out = fn;
    return cudaSuccess;
}

// [tokens][heads][dim] with strides, read in boxes of 64 x heads x tokens.
cudaError_t tensor_map(CUtensorMap* map, const void* p, int32_t dtype, int32_t dim, uint32_t heads, uint32_t tokens,
                       const int64_t* stride, uint32_t box_heads, uint32_t box_tokens) {
    EncodeFn encode;
    cudaError_t e = encoder(encode);
    if (e != cudaSuccess) return e;
    const cuuint64_t extent[3] = {static_cast<cuuint64_t>(dim), heads, tokens};
    // a stride that only ever meets coordinate 0 may be any
    const cuuint64_t bytes[2] = {static_cast<cuuint64_t>(heads > 1 ? stride[1] * 2 : dim * 2),
                                 static_cast<cuuint64_t>(tokens > 1 ? stride[0] * 2 : dim * 2)};
    const cuuint32_t box[3] = {64, box_heads, box_tokens}, step[3] = {1, 1, 1};
    const CUresult r = encode(map, dtype == BS_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                              const_cast<void*>(p), extent, bytes, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <typename T, int BOXES>
cudaError_t launch(const PromptArgs& a, cudaStream_t stream) {
    cudaError_t e = cudaFuncSetAttribute(k_prompt<T, BOXES>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem<BOXES>);
    if (e != cudaSuccess) return e;
    const uint64_t blocks = (a.d.total_q / (2 * a.tile_tokens) + static_cast<uint64_t>(a.d.num_seqs)) * a.d.kv_heads;
    if (blocks > 0x7fffffffu) return cudaErrorInvalidConfiguration;
    k_prompt<T, BOXES><<<static_cast<unsigned>(blocks), kThreads, kSmem<BOXES>, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_prompt_attention(const bs_prompt_attention_desc& d, const MemoryDevice& dev, cudaStream_t stream) {
    PromptArgs a{};
    a.d = d;
    a.errors = dev.errors;
    a.group = d.q_heads / d.kv_heads;
    a.tile_tokens = kRows / a.group;
    cudaError_t e = tensor_map(&a.q, d.q, d.dtype, d.dim, d.q_heads, d.total_q, d.q_stride, a.group, a.tile_tokens);
    // (no keys: nothing is read through the maps)
    if (e == cudaSuccess && d.total_k) e = tensor_map(&a.k, d.k, d.dtype, d.dim, d.kv_heads, d.total_k, d.k_stride, 1, kRows);
    if (e == cudaSuccess && d.total_k) e = tensor_map(&a.v, d.v, d.dtype, d.dim, d.kv_heads, d.total_k, d.v_stride, 1, kRows);
    if (e != cudaSuccess) return e;
    if (d.dtype == BS_F16) return d.dim <= 64 ? launch<__half, 1>(a, stream) : launch<__half, 2>(a, stream);
    return d.dim <= 64 ? launch<__nv_bfloat16, 1>(a, stream) : launch<__nv_bfloat16, 2>(a, stream);
}

}  // namespace bsb
