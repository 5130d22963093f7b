// bs_cache_tile.cuh -- a warp's work on a tile of 32 tokens of the 8-bit token
// cache in shared memory: scores, weights and values of 8 * NT query rows.
// Shared by the kernels of bs_cache_attention.cu (where the layout of the
// products and their roundings are explained) and bs_block_attention.cu.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bs_device.cuh"

namespace bsb {
namespace tile {

using namespace dev;

constexpr int kWarps = 4;              // per block; they take a segment's tiles in turn
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;              // tokens: two halves of 16, independent chains of instructions
constexpr float kNoScore = -1e30f;     // running maximum before the first score
constexpr float kSlack = 8.f;          // weights may grow to 2^kSlack before the maximum is moved
constexpr float kFold = 32.f;          // a weight of 2^top at the largest value scale in f16; 2^kSlack * 4 * kFold is below 65504
constexpr float kDeep = 60.f;          // value scales count down to 2^-kDeep of the largest
constexpr float kMostSum = 80.f;       // the maximum is moved down only as far as sums stay below 2^kMostSum

__device__ __forceinline__ unsigned smem_addr(const void* p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}

__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transposed8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// The maximum that weights count from is that of a score and this: log2 of its
// value scale in units of the warp's largest (a scale below zero, of tokens that
// are not seen, is NaN there and counts as the least).  What is rounded to f16 is a
// weight times its value scale: counted from the largest score alone, weights of
// 1 at a value scale 10^-7 of another's had two bits left, whatever weight that
// other one got.
__device__ __forceinline__ float scale_log2(float v_scale, float inv_unit) { return fmaxf(log2_fast(v_scale * inv_unit) - 5.f, -kDeep); }
static_assert(kFold == 32.f, "log2 of it is above");

// Bytes [x, y] (in bits 0-7 and 8-15, or 16-23 and 24-31) biased by 128 ->
// two f16 of the codes: 0x6400 | u is 1024 + u, minus 1152.
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t biased, uint32_t selector) {
    const uint32_t u = __byte_perm(biased, 0x64646464u, selector);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __float2half2_rn(1152.f));
    return *reinterpret_cast<const uint32_t*>(&h);
}
constexpr uint32_t kLow = 0x4140u, kHigh = 0x4342u;

// Rows of a stage are an odd number of 16-byte units apart, so that the lanes
// of a shared-memory access fall on different banks; rows of 128 bytes have no
// gap (two blocks would not fit an SM) but their units permuted: unit x of row
// r lies at x ^ (r & 7).
template <int NW>
constexpr int kPitch = NW == 8 ? 128 : 16 * (NW | 1);
template <int NW>
__device__ __forceinline__ uint32_t unit_at(uint32_t x, uint32_t row) {
    return 16 * (NW == 8 ? x ^ (row & 7) : x);
}
// NW words (of 4 codes) per lane of a key row: the lane's quarter of it.
template <int NW>
__device__ __forceinline__ void load_key_words(uint32_t (&w)[NW], const unsigned char* tile, uint32_t r, uint32_t c) {
    const unsigned char* p = tile + r * kPitch<NW> + c * (NW * 4);
    if constexpr (NW % 4 == 0) {
#pragma unroll
        for (int i = 0; i < NW / 4; ++i)
            *reinterpret_cast<uint4*>(&w[4 * i]) =
                *reinterpret_cast<const uint4*>(tile + r * kPitch<NW> + unit_at<NW>(c * (NW / 4) + i, r));
    } else if constexpr (NW % 2 == 0) {
#pragma unroll
        for (int i = 0; i < NW / 2; ++i) *reinterpret_cast<uint2*>(&w[2 * i]) = reinterpret_cast<const uint2*>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < NW; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
}

// The lane's codes of one value row: output row tile t (16 dimensions) takes
// the bytes 2t (tile row g) and 2t + 1 (row g + 8) of these words.  In memory
// they are 16 g + 2t, 8 g + 2t, or, by pairs of tiles, 32 (t / 2) + 4 g + 2 (t % 2)
// (a last single tile: 16 t + 2 g); value_dim gives the dimension.
template <int NW>
__device__ __forceinline__ void load_value_words(uint32_t (&w)[(NW + 1) / 2], const unsigned char* tile, uint32_t r, uint32_t g) {
    const unsigned char* row = tile + r * kPitch<NW>;
    if constexpr (NW == 8) {
        *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(row + unit_at<NW>(g, r));
    } else if constexpr (NW == 4) {
        *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(row + 8 * g);
    } else {
#pragma unroll
        for (int i = 0; i < NW / 2; ++i) w[i] = *reinterpret_cast<const uint32_t*>(row + 32 * i + 4 * g);
        if constexpr (NW % 2) w[NW / 2] = *reinterpret_cast<const uint16_t*>(row + 16 * (NW - 1) + 2 * g);
    }
}
template <int NW>
__device__ __forceinline__ constexpr uint32_t value_dim(int t, uint32_t g) {
    if (NW == 8) return 16 * g + 2 * t;
    if (NW == 4) return 8 * g + 2 * t;
    if (NW % 2 && t == NW - 1) return 16 * t + 2 * g;
    return 32 * (t / 2) + 4 * g + 2 * (t % 2);
}

// One query row as column g of the products; `scale` times what its scaling
// by a power of two took off is returned for columns 2c and 2c + 1.
template <int NW>
__device__ __forceinline__ void fetch_query_row(uint32_t (&q)[NW][2], const uint16_t* row, bool real) {
#pragma unroll
    for (int j = 0; j < NW; ++j) {
        const uint2 u = real ? *reinterpret_cast<const uint2*>(row + 4 * j) : make_uint2(0, 0);
        q[j][0] = u.x;
        q[j][1] = u.y;
    }
}
template <int NW>
__device__ __forceinline__ void scale_query_row(uint32_t (&q)[NW][2], float (&row_scale)[2], bool bf16, float scale, uint32_t c) {
    if (bf16) {
        // times 2^e with the row's largest in [2^12, 2^13); rows of zeros, infinities and NaN as they are
        uint32_t top = 0;        // magnitudes of bf16 order as integers
#pragma unroll
        for (int j = 0; j < NW; ++j) top = __vmaxu2(top, __vmaxu2(q[j][0] & 0x7fff7fffu, q[j][1] & 0x7fff7fffu));
        top = max(top >> 16, top & 0xffffu);
        top = max(top, __shfl_xor_sync(kFull, top, 1));
        top = max(top, __shfl_xor_sync(kFull, top, 2));
        uint32_t e = top >> 7;   // biased exponent
        e = top == 0 || e == 255 ? 139 : e < 13 ? 13 : e;
        const float up = __uint_as_float((266 - e) << 23), down = __uint_as_float((e - 12) << 23);
#pragma unroll
        for (int j = 0; j < NW; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const __half2 h = __floats2half2_rn(__uint_as_float(q[j][i] << 16) * up, __uint_as_float(q[j][i] & 0xffff0000u) * up);
                q[j][i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        scale *= down;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) row_scale[i] = __shfl_sync(kFull, scale, (2 * c + i) * 4);
}
template <int NW>
__device__ __forceinline__ void load_query_row(uint32_t (&q)[NW][2], float (&row_scale)[2], const uint16_t* row, bool real, bool bf16,
                                               float scale, uint32_t c) {
    fetch_query_row<NW>(q, row, real);
    scale_query_row<NW>(q, row_scale, bf16, scale, c);
}

// Products of the tile's key codes with the queries: z[half] has tokens g and
// g + 8 (+ 16 half), columns 2c and 2c + 1.
template <int NW, int NT>
__device__ __forceinline__ void tile_scores(float (&z)[2][NT][4], const unsigned char* s, const uint32_t (&q)[NT][NW][2], uint32_t g, uint32_t c) {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) z[half][nt][0] = z[half][nt][1] = z[half][nt][2] = z[half][nt][3] = 0.f;
    uint32_t k[2][2][NW];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        load_key_words<NW>(k[half][0], s, 16 * half + g, c);
        load_key_words<NW>(k[half][1], s, 16 * half + g + 8, c);
    }
#pragma unroll
    for (int j = 0; j < NW; ++j)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t u0 = k[half][0][j] ^ 0x80808080u, u1 = k[half][1][j] ^ 0x80808080u;
            const uint32_t a0 = codes_to_half2(u0, kLow), a1 = codes_to_half2(u1, kLow);
            const uint32_t a2 = codes_to_half2(u0, kHigh), a3 = codes_to_half2(u1, kHigh);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16(z[half][nt], a0, a1, a2, a3, q[nt][j][0], q[nt][j][1]);
        }
}

// Rare: the maxima move, what was summed is rescaled.  Where a larger value scale
// than before becomes the unit, they move down by as much, so that weights at the
// old scales keep their bits.
template <int NW, int NT>
__device__ __forceinline__ void move_maxima(const float (&z)[2][NT][4], const float (&v_scale)[2], float (&top)[NT][2], float (&sum)[NT][2],
                                            float (&o)[NT][NW][4], float& unit, float& inv_unit) {
    const float new_unit = fmaxf(unit, fmaxf(v_scale[0], v_scale[1]));
    const float by_unit = unit / new_unit, less = log2_fast(by_unit);
    unit = new_unit;
    inv_unit = kFold / unit;
    const float deep[2] = {scale_log2(v_scale[0], inv_unit), scale_log2(v_scale[1], inv_unit)};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float m = fmaxf(fmaxf(z[0][nt][i], z[0][nt][2 + i]) + deep[0], fmaxf(z[1][nt][i], z[1][nt][2 + i]) + deep[1]);
            m = fmaxf(m, top[nt][i] + fmaxf(less, log2_fast(sum[nt][i]) - kMostSum));
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, x));
            m = fmaxf(m, kNoScore);
            const float shrink = exp2_fast(top[nt][i] - m);
            top[nt][i] = m;
            sum[nt][i] *= shrink;
#pragma unroll
            for (int j = 0; j < NW; ++j) {
                o[nt][j][i] *= shrink * by_unit;
                o[nt][j][2 + i] *= shrink * by_unit;
            }
        }
}

// Weights of the tile's scores (log2 units, -infinity: not seen), and their
// products with its values.
template <int NW, int NT>
__device__ __forceinline__ void tile_values(const float (&z)[2][NT][4], const unsigned char* s, const float (&v_scale)[2], float inv_unit,
                                            const float (&top)[NT][2], float (&sum)[NT][2], float (&o)[NT][NW][4], uint32_t g, uint32_t c) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const float by = v_scale[half] * inv_unit;
        uint32_t p[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = exp2_fast(z[half][nt][i] - top[nt][i & 1]);
                sum[nt][i & 1] += w[i];
                w[i] *= by;
            }
            const __half2 lo = __floats2half2_rn(w[0], w[1]), hi = __floats2half2_rn(w[2], w[3]);
            p[nt][0] = transposed8x8(*reinterpret_cast<const uint32_t*>(&lo));
            p[nt][1] = transposed8x8(*reinterpret_cast<const uint32_t*>(&hi));
        }
        const unsigned char* v = s + kTile * kPitch<NW>;
        constexpr int kWords = (NW + 1) / 2;
        uint32_t v0[kWords], v1[kWords], v2[kWords], v3[kWords];
        load_value_words<NW>(v0, v, 16 * half + 2 * c, g);
        load_value_words<NW>(v1, v, 16 * half + 2 * c + 1, g);
        load_value_words<NW>(v2, v, 16 * half + 2 * c + 8, g);
        load_value_words<NW>(v3, v, 16 * half + 2 * c + 9, g);
#pragma unroll
        for (int j = 0; j < NW; ++j) {
            const uint32_t pick = j % 2 ? 0x7362u : 0x5140u;      // the two tokens' bytes side by side
            const uint32_t x = __byte_perm(v0[j / 2], v1[j / 2], pick) ^ 0x80808080u;
            const uint32_t y = __byte_perm(v2[j / 2], v3[j / 2], pick) ^ 0x80808080u;
            const uint32_t a0 = codes_to_half2(x, kLow), a1 = codes_to_half2(x, kHigh);
            const uint32_t a2 = codes_to_half2(y, kLow), a3 = codes_to_half2(y, kHigh);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16(o[nt][j], a0, a1, a2, a3, p[nt][0], p[nt][1]);
        }
    }
}

// The block's warps' maxima, then their sums and outputs as one: warp 0 has
// the outputs, every warp maxima and sums.  join_o: two warps' outputs,
// join_ml: [warps][8 * NT][2].
template <int NW, int NT>
__device__ __forceinline__ void join_warps(float (&o)[NT][NW][4], const float (&top)[NT][2], float (&sum)[NT][2], float unit,
                                           float (&all_top)[NT][2], float (&all_sum)[NT][2], float* join_o, float* join_ml, uint32_t warp,
                                           uint32_t lane) {
    constexpr int kDim = NW * 16, kRows = 8 * NT;
    const uint32_t g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) sum[nt][i] += __shfl_xor_sync(kFull, sum[nt][i], x);
            if (g == 0) {
                float* ml = join_ml + (warp * kRows + 8 * nt + 2 * c + i) * 2;
                ml[0] = top[nt][i];
                ml[1] = sum[nt][i];
            }
        }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float* ml = join_ml + (8 * nt + 2 * c + i) * 2;
            float m = kNoScore, l = 0.f;
#pragma unroll
            for (int x = 0; x < kWarps; ++x) m = fmaxf(m, ml[x * kRows * 2]);
#pragma unroll
            for (int x = 0; x < kWarps; ++x) l += ml[x * kRows * 2 + 1] * exp2_fast(ml[x * kRows * 2] - m);
            const float f = exp2_fast(top[nt][i] - m) * (unit * (1.f / kFold));
            all_top[nt][i] = m;
            all_sum[nt][i] = l;
#pragma unroll
            for (int j = 0; j < NW; ++j) {
                o[nt][j][i] *= f;
                o[nt][j][2 + i] *= f;
            }
        }
    auto put = [&](float* to) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < NW; ++j) *reinterpret_cast<float4*>(to + ((nt * NW + j) * 32 + lane) * 4) = *reinterpret_cast<float4*>(o[nt][j]);
    };
    auto add = [&](const float* from) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < NW; ++j) {
                const float4 x = *reinterpret_cast<const float4*>(from + ((nt * NW + j) * 32 + lane) * 4);
                o[nt][j][0] += x.x, o[nt][j][1] += x.y, o[nt][j][2] += x.z, o[nt][j][3] += x.w;
            }
    };
    if (warp >= 2) put(join_o + (warp - 2) * kRows * kDim);
    __syncthreads();
    if (warp < 2) add(join_o + warp * kRows * kDim);
    __syncthreads();
    if (warp == 1) put(join_o);
    __syncthreads();
    if (warp == 0) add(join_o);
}

template <int NW>
constexpr int kStageBytes = 2 * kTile * kPitch<NW> + 16;      // keys, values, (key, value) scales of the halves
template <int NW, int NT>
constexpr int kJoinBytes = 2 * 8 * NT * NW * 16 * 4;           // two warps' outputs

}  // namespace tile
}  // namespace bsb
