// bs_norm_rotate.cu -- norm of queries and keys for each head and the rotary
// position in one pass (include/bsearch.h, bs_norm_rotate).
//
// The time is that of reading and writing every value once, so a value is in
// registers from its load to its store.  A lane has V values and the V that
// they are rotated with: 16 bytes of each where half the rotated part is a
// multiple of 8 dimensions (and in the interleaved layout always), fewer where
// it is not.  The lanes of a row add their squares by shuffles.  A warp takes
// one token, so that the sines and cosines of its position are computed once
// for all its heads, or for as many as it has where tokens are few.
//
// Angles: freqs / 2 pi is taken as a 64-bit fraction of a turn; its product
// with the position, modulo 2^64, is the angle's fraction of a turn, of which
// the upper 32 bits are kept.  A product in 32-bit floats would be off by 0.06
// radians at position 10^6.  As a float those bits and the radians made of them
// are off by up to 2^-20.8 near half a turn, the fast sine and cosine by 2^-21
// more: 2^-19.9 in all, 2^-8 of f16's rounding of 1 (bf16's: 2^-11).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bs_device.cuh"
#include "bs_memory.h"

namespace bsb {

using namespace dev;

namespace {

constexpr int kThreads = 128;
constexpr int kMostDim = 128;
constexpr int kBatch = 2;             // rows of a lane whose loads are on their way together
constexpr int kBlocks = 5;            // resident on an SM

struct RotateArgs {
    bs_norm_rotate_desc d;
    uint32_t lanes;       // of a row, a power of two
    uint32_t parts;       // warps that share a token
    uint32_t part_rows;   // rows (heads) of a part
};

template <int V>
struct Words;
template <>
struct Words<8> {
    using type = uint4;
};
template <>
struct Words<4> {
    using type = uint2;
};
template <>
struct Words<2> {
    using type = uint32_t;
};
template <>
struct Words<1> {
    using type = uint16_t;
};

__device__ __forceinline__ float2 two_floats(uint32_t u, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
__device__ __forceinline__ float2 two_floats(uint32_t u, __nv_bfloat16) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ uint32_t two_rounded(float x, float y, __half) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t two_rounded(float x, float y, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, int V>
__device__ __forceinline__ void to_floats(float (&x)[V], const typename Words<V>::type& w) {
    if constexpr (V == 1) {
        x[0] = two_floats(w, T()).x;
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 f = two_floats(reinterpret_cast<const uint32_t*>(&w)[i], T());
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}
template <typename T, int V>
__device__ __forceinline__ void rounded(typename Words<V>::type& w, const float (&x)[V]) {
    if constexpr (V == 1) {
        w = static_cast<uint16_t>(two_rounded(x[0], 0.f, T()));
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) reinterpret_cast<uint32_t*>(&w)[i] = two_rounded(x[2 * i], x[2 * i + 1], T());
    }
}

// A chunk's V values times `by` and its weights (a chunk begins at a multiple of V).
template <int V>
__device__ __forceinline__ void weighted(float (&x)[V], const float* w, float by) {
    using Some = typename Words<V >= 4 ? 8 : V >= 2 ? 4 : 2>::type;      // 4, 2 or 1 floats
    constexpr int kSome = sizeof(Some) / 4;
#pragma unroll
    for (int i = 0; i < V; i += kSome) {
        const Some f = *reinterpret_cast<const Some*>(w + i);
#pragma unroll
        for (int j = 0; j < kSome; ++j) x[i + j] *= by * __uint_as_float(reinterpret_cast<const uint32_t*>(&f)[j]);
    }
}

__device__ __forceinline__ float weight_at(const void* w, int32_t dtype, uint32_t i) {
    if (dtype == BS_F32) return static_cast<const float*>(w)[i];
    if (dtype == BS_F16) return __half2float(static_cast<const __half*>(w)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// Every block takes tokens (or parts of them) in turn, and a warp asks for its
// next rows before it works on the last ones: with a block for each four tokens the
// loads stood still while angles were computed (50 us against 30 for 7,196 tokens of
// 40 heads of 128: 147 MB, 4.8 TB/s, where the copies alone are 22.5 us).  What is left
// is instructions, 2.6 of 4 a cycle; DRAM is at a third of its rate.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, kBlocks) k_norm_rotate(const __grid_constant__ RotateArgs a) {
    constexpr int kEach = V == 1 ? 2 : 1;              // pairs of chunks of a lane: 128 dimensions are 64 of them
    constexpr int kPairs = INTERLEAVED ? 8 : V;        // of values that are rotated with each other
    using Word = typename Words<V>::type;
    __shared__ __align__(16) float weights[2][kMostDim];
    __shared__ uint64_t turns[kMostDim / 2];
    const bs_norm_rotate_desc& d = a.d;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dim = d.dim, half = d.rotary / 2;
    const uint32_t q_heads = d.q_heads, heads = q_heads + d.kv_heads, slots = dim / (2 * V);
    cudaGridDependencySynchronize();       // in every block, before anything of the caller's

    const uint32_t sub = lane / a.lanes, at = lane % a.lanes, step = 32 / a.lanes;
    // where the lane's chunks lie in a row
    uint32_t lo[kEach], hi[kEach];
    bool mine[kEach];
    int turned[kEach];                                 // pairs that are rotated, the first ones
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const uint32_t u = at + e * a.lanes;
        mine[e] = u < slots;
        turned[e] = V * u < half ? static_cast<int>(min(half - V * u, static_cast<uint32_t>(kPairs))) : 0;
        if (INTERLEAVED || u >= half / V) {
            lo[e] = INTERLEAVED ? 2 * V * u : 2 * half + 2 * V * (u - half / V);
            hi[e] = lo[e] + V;
        } else {
            lo[e] = u * V;
            hi[e] = half + u * V;
        }
    }
    // a batch: rows r .. end of a token's queries or keys
    struct Batch {
        uint64_t item;
        uint32_t token, r, end;
        bool keys;
    };
    const uint64_t items = static_cast<uint64_t>(d.total) * a.parts, all_warps = static_cast<uint64_t>(gridDim.x) * (kThreads / 32);
    auto begin = [&](Batch& b) {           // an item's first
        b.token = static_cast<uint32_t>(b.item / a.parts);
        const uint32_t first = static_cast<uint32_t>(b.item % a.parts) * a.part_rows, end = min(heads, first + a.part_rows);
        b.keys = first >= q_heads;
        b.r = b.keys ? first - q_heads : first;
        b.end = b.keys ? end - q_heads : min(end, q_heads);
    };
    auto advance = [&](Batch& b) {
        b.r += kBatch * step;
        if (b.r < b.end) return;
        const uint32_t past = min(heads, (static_cast<uint32_t>(b.item % a.parts) + 1) * a.part_rows);
        if (!b.keys && past > q_heads) {   // the token's keys
            b.keys = true;
            b.r = 0;
            b.end = past - q_heads;
            return;
        }
        b.item += all_warps;
        begin(b);
    };
    Word x[kBatch][kEach][2];
    int64_t position = 0;
    auto request = [&](const Batch& b) {
        const int64_t* const stride = b.keys ? d.k_stride : d.q_stride;
        const T* const rows = static_cast<const T*>(b.keys ? d.k : d.q) + b.token * stride[0];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const uint32_t r = b.r + u * step + sub;
            const T* const row = rows + r * stride[1];
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                x[u][e][0] = x[u][e][1] = Word{};
                if (mine[e] && r < b.end) {
                    x[u][e][0] = *reinterpret_cast<const Word*>(row + lo[e]);
                    x[u][e][1] = *reinterpret_cast<const Word*>(row + hi[e]);
                }
            }
        }
        if (half) position = d.positions[b.token];
    };
    Batch b;
    b.item = static_cast<uint64_t>(blockIdx.x) * (kThreads / 32) + warp;
    begin(b);
    if (b.item < items) request(b);

    for (uint32_t i = threadIdx.x; i < half; i += kThreads) {
        const double turn = d.freqs[i] * 0.15915494309189535;
        turns[i] = __double2ull_rd((turn - floor(turn)) * 18446744073709551616.);
    }
    for (uint32_t i = threadIdx.x; i < 2 * kMostDim; i += kThreads) {
        const void* const w = i < kMostDim ? d.q_weight : d.k_weight;
        weights[i / kMostDim][i % kMostDim] = w && i % kMostDim < dim ? weight_at(w, d.weight_dtype, i % kMostDim) : 1.f;
    }
    __syncthreads();
    float cosine[kEach][kPairs], sine[kEach][kPairs];
    uint64_t known = ~0ull;                // item whose angles those are
    const float one_of_dim = 1.f / dim;
    while (b.item < items) {
        Word now[kBatch][kEach][2];
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                now[u][e][0] = x[u][e][0];
                now[u][e][1] = x[u][e][1];
            }
        const int64_t here = position;
        const Batch c = b;
        advance(b);
        if (b.item < items) request(b);
        if (known != c.item) {
            known = c.item;
#pragma unroll
            for (int e = 0; e < kEach; ++e)
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    const uint32_t p = INTERLEAVED ? V * (at + e * a.lanes) + j : lo[e] + j;
                    cosine[e][j] = 1.f;
                    sine[e][j] = 0.f;
                    if (p < half) {
                        // (a part of a turn between -1/2 and 1/2, where the fast functions are good)
                        const uint64_t angle = turns[p] * static_cast<uint64_t>(here);
                        __sincosf(static_cast<float>(static_cast<int32_t>(angle >> 32)) * 1.4629180792671596e-09f, &sine[e][j], &cosine[e][j]);
                        cosine[e][j] *= d.amplitude;
                        sine[e][j] *= d.amplitude;
                    }
                }
        }
        const bool norm = c.keys ? d.k_weight != nullptr : d.q_weight != nullptr;
        const float* const weight = weights[c.keys];
        T* const out = static_cast<T*>(c.keys ? d.out_k : d.out_q) + static_cast<uint64_t>(c.token) * (c.keys ? d.kv_heads : q_heads) * dim;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if (c.r + u * step >= c.end) break;                     // (all lanes)
            const uint32_t r = c.r + u * step + sub;
            float y[kEach][2][V];
            float squares = 0.f;
#pragma unroll
            for (int e = 0; e < kEach; ++e)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    to_floats<T, V>(y[e][s], now[u][e][s]);
#pragma unroll
                    for (int i = 0; i < V; ++i) squares = fmaf(y[e][s][i], y[e][s][i], squares);
                }
            if (norm) {                                             // (all lanes)
                for (uint32_t o = a.lanes / 2; o > 0; o >>= 1) squares += __shfl_xor_sync(kFull, squares, o);
                const float by = rsqrtf(fmaf(squares, one_of_dim, d.eps));
#pragma unroll
                for (int e = 0; e < kEach; ++e)
#pragma unroll
                    for (int s = 0; s < 2; ++s) weighted<V>(y[e][s], weight + (!mine[e] ? 0 : s ? hi[e] : lo[e]), by);
            }
            if (r >= c.end) continue;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                if (!mine[e]) continue;
                // past the rotated part values pass as they are (by a cosine of 1 and a sine of
                // 0 an infinity would make its partner NaN): `only` says of some pairs which
                float z[2][V];
                auto rotate = [&](auto only) {
#pragma unroll
                    for (int j = 0; j < kPairs; ++j) {
                        const int s = INTERLEAVED ? j / (V / 2) : 0, i = INTERLEAVED ? 2 * (j % (V / 2)) : j;
                        const int s2 = INTERLEAVED ? s : 1, i2 = INTERLEAVED ? i + 1 : i;
                        const float p = y[e][s][i], q = y[e][s2][i2];
                        const bool turn = only(j);
                        z[s][i] = turn ? fmaf(cosine[e][j], p, -sine[e][j] * q) : p;
                        z[s2][i2] = turn ? fmaf(cosine[e][j], q, sine[e][j] * p) : q;
                    }
                };
                if (turned[e] == kPairs) rotate([](int) { return true; });
                else if (INTERLEAVED) rotate([&](int j) { return j < turned[e]; });
                else rotate([](int) { return false; });             // (half is a multiple of V: a chunk is in or out)
                Word w[2];
                rounded<T, V>(w[0], z[0]);
                rounded<T, V>(w[1], z[1]);
                T* const row = out + static_cast<uint64_t>(r) * dim;
                *reinterpret_cast<Word*>(row + lo[e]) = w[0];
                *reinterpret_cast<Word*>(row + hi[e]) = w[1];
            }
        }
    }
}

template <typename T, int V, bool INTERLEAVED>
cudaError_t launch(const bs_norm_rotate_desc& d, const MemoryDevice& dev, cudaStream_t stream) {
    RotateArgs a{d};
    const uint32_t slots = d.dim / (2 * V), heads = d.q_heads + d.kv_heads;
    a.lanes = 1;
    while (a.lanes < 32 && a.lanes < slots) a.lanes *= 2;
    // A warp has a token's heads, or, where that leaves over half of the GPU's warps
    // idle, as many as it reads at once (tokens of 32 and 8 heads of 128: 64 of them
    // 7.8 us by whole tokens and 3.9 in parts, 700 8.8 and 6.8, 2,000 10.9 and 12.4,
    // 7,196 30 and 39).
    const uint32_t at_once = 32 / a.lanes * kBatch;
    const uint64_t resident = static_cast<uint64_t>(dev.num_sms) * kBlocks * (kThreads / 32);
    a.parts = 2ull * d.total < resident ? (heads + at_once - 1) / at_once : 1;
    a.part_rows = a.parts > 1 ? at_once : heads;
    const uint64_t items = static_cast<uint64_t>(d.total) * a.parts, blocks = ((items < resident ? items : resident) + kThreads / 32 - 1) / (kThreads / 32);
    return launch_after(k_norm_rotate<T, V, INTERLEAVED>, dim3(static_cast<unsigned>(blocks)), kThreads, 0, stream, a);
}

template <typename T>
cudaError_t launch_typed(const bs_norm_rotate_desc& d, const MemoryDevice& dev, cudaStream_t stream) {
    if (d.interleaved) return launch<T, 8, true>(d, dev, stream);
    // the largest chunk that both halves of the rotated part are made of
    const int32_t half = d.rotary / 2;
    if (half % 8 == 0) return launch<T, 8, false>(d, dev, stream);
    if (half % 4 == 0) return launch<T, 4, false>(d, dev, stream);
    if (half % 2 == 0) return launch<T, 2, false>(d, dev, stream);
    return launch<T, 1, false>(d, dev, stream);
}

}  // namespace

cudaError_t launch_norm_rotate(const bs_norm_rotate_desc& d, const MemoryDevice& dev, cudaStream_t stream) {
    return d.dtype == BS_F16 ? launch_typed<__half>(d, dev, stream) : launch_typed<__nv_bfloat16>(d, dev, stream);
}

}  // namespace bsb
