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
// radians at position 10^6.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bs_device.cuh"
#include "bs_memory.h"

namespace bsb {

using namespace dev;

namespace {

constexpr int kThreads = 128;
constexpr int kMostDim = 128;

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

template <typename T, int V>
__device__ __forceinline__ void to_floats(float (&x)[V], const typename Words<V>::type& w) {
    const T* p = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = static_cast<float>(p[i]);
}
__device__ __forceinline__ void round_to(__half& to, float x) { to = __float2half_rn(x); }
__device__ __forceinline__ void round_to(__nv_bfloat16& to, float x) { to = __float2bfloat16_rn(x); }

__device__ __forceinline__ float weight_at(const void* w, int32_t dtype, uint32_t i) {
    if (dtype == BS_F32) return static_cast<const float*>(w)[i];
    if (dtype == BS_F16) return __half2float(static_cast<const __half*>(w)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) k_norm_rotate(const __grid_constant__ RotateArgs a) {
    constexpr int kEach = V == 1 ? 2 : 1;              // pairs of chunks of a lane: 128 dimensions are 64 of them
    constexpr int kBatch = V == 8 ? 4 : 2;             // rows of a lane whose loads are on their way together
    constexpr int kPairs = INTERLEAVED ? 8 : V;
    using Word = typename Words<V>::type;
    __shared__ __align__(16) float weights[2][kMostDim];
    __shared__ uint64_t turns[kMostDim / 2];
    const bs_norm_rotate_desc& d = a.d;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dim = d.dim, half = d.rotary / 2;
    const uint32_t heads = d.q_heads + d.kv_heads, slots = dim / (2 * V);
    cudaGridDependencySynchronize();       // in every block, before anything of the caller's

    const uint64_t item = static_cast<uint64_t>(blockIdx.x) * (kThreads / 32) + warp;
    const uint32_t token = static_cast<uint32_t>(item / a.parts), r_first = static_cast<uint32_t>(item % a.parts) * a.part_rows;
    const uint32_t r_end = token < d.total ? min(heads, r_first + a.part_rows) : r_first;
    const uint32_t sub = lane / a.lanes, at = lane % a.lanes, step = 32 / a.lanes;
    // where the lane's chunks lie in a row
    uint32_t lo[kEach], hi[kEach];
    bool mine[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const uint32_t u = at + e * a.lanes;
        mine[e] = u < slots;
        if (INTERLEAVED || u >= half / V) {
            lo[e] = INTERLEAVED ? 2 * V * u : 2 * half + 2 * V * (u - half / V);
            hi[e] = lo[e] + V;
        } else {
            lo[e] = u * V;
            hi[e] = half + u * V;
        }
    }
    auto row_of = [&](uint32_t r) {
        const bool q = r < static_cast<uint32_t>(d.q_heads);
        return static_cast<const T*>(q ? d.q : d.k) + token * (q ? d.q_stride : d.k_stride)[0] +
               (q ? r : r - d.q_heads) * (q ? d.q_stride : d.k_stride)[1];
    };
    Word x[kBatch][kEach][2];
    auto request = [&](uint32_t r0) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const uint32_t r = r0 + u * step + sub;
            if (r >= r_end) continue;
            const T* row = row_of(r);
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                if (mine[e]) {
                    x[u][e][0] = *reinterpret_cast<const Word*>(row + lo[e]);
                    x[u][e][1] = *reinterpret_cast<const Word*>(row + hi[e]);
                }
        }
    };
    request(r_first);

    const int64_t position = d.rotary && token < d.total ? d.positions[token] : 0;
    for (uint32_t i = threadIdx.x; i < half; i += kThreads) {
        const double turn = d.freqs[i] * 0.15915494309189535;
        turns[i] = __double2ull_rd((turn - floor(turn)) * 18446744073709551616.);
    }
    for (uint32_t i = threadIdx.x; i < 2 * dim; i += kThreads) {
        const void* w = i < dim ? d.q_weight : d.k_weight;
        weights[i >= dim][i < dim ? i : i - dim] = w ? weight_at(w, d.weight_dtype, i < dim ? i : i - dim) : 1.f;
    }
    __syncthreads();
    float cosine[kEach][kPairs], sine[kEach][kPairs];
#pragma unroll
    for (int e = 0; e < kEach; ++e)
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
            const uint32_t p = INTERLEAVED ? V * (at + e * a.lanes) + j : lo[e] + j;
            cosine[e][j] = 1.f;
            sine[e][j] = 0.f;
            if (p < half) {
                const uint64_t angle = turns[p] * static_cast<uint64_t>(position);
                sincospif(static_cast<float>(static_cast<int32_t>(angle >> 32)) * 4.656612873077393e-10f, &sine[e][j], &cosine[e][j]);
                cosine[e][j] *= d.amplitude;
                sine[e][j] *= d.amplitude;
            }
        }

    for (uint32_t r0 = r_first; r0 < r_end; r0 += kBatch * step) {
        if (r0 != r_first) request(r0);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const uint32_t r = r0 + u * step + sub;
            if (r0 + u * step >= r_end) break;                  // (all lanes)
            const bool q = r < static_cast<uint32_t>(d.q_heads);
            float y[kEach][2][V];
            float squares = 0.f;
#pragma unroll
            for (int e = 0; e < kEach; ++e)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    to_floats<T, V>(y[e][s], x[u][e][s]);
#pragma unroll
                    for (int i = 0; i < V; ++i) squares += mine[e] && r < r_end ? y[e][s][i] * y[e][s][i] : 0.f;
                }
            if (d.q_weight || d.k_weight)           // (all lanes)
                for (uint32_t o = a.lanes / 2; o > 0; o >>= 1) squares += __shfl_xor_sync(kFull, squares, o);
            if (q ? d.q_weight != nullptr : d.k_weight != nullptr) {
                const float by = rsqrtf(squares / dim + d.eps);
#pragma unroll
                for (int e = 0; e < kEach; ++e)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        y[e][0][i] *= by * weights[!q][(lo[e] + i) % kMostDim];
                        y[e][1][i] *= by * weights[!q][(hi[e] + i) % kMostDim];
                    }
            }
            if (r >= r_end) continue;
            T* const out = static_cast<T*>(q ? d.out_q : d.out_k) +
                           (static_cast<uint64_t>(token) * (q ? d.q_heads : d.kv_heads) + (q ? r : r - d.q_heads)) * dim;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                if (!mine[e]) continue;
                Word w[2];
                T* const to[2] = {reinterpret_cast<T*>(&w[0]), reinterpret_cast<T*>(&w[1])};
                if constexpr (INTERLEAVED) {
#pragma unroll
                    for (int j = 0; j < kPairs; ++j) {
                        const int s = j / (V / 2), i = 2 * (j % (V / 2));
                        const float c = cosine[e][j], n = sine[e][j];
                        round_to(to[s][i], y[e][s][i] * c - y[e][s][i + 1] * n);
                        round_to(to[s][i + 1], y[e][s][i + 1] * c + y[e][s][i] * n);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float c = cosine[e][i], n = sine[e][i];
                        round_to(to[0][i], y[e][0][i] * c - y[e][1][i] * n);
                        round_to(to[1][i], y[e][1][i] * c + y[e][0][i] * n);
                    }
                }
                *reinterpret_cast<Word*>(out + lo[e]) = w[0];
                *reinterpret_cast<Word*>(out + hi[e]) = w[1];
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
    // a warp has a token's heads, or, where that leaves the GPU idle, as many as it
    // reads at once
    const uint32_t at_once = 32 / a.lanes * (V == 8 ? 4 : 2);
    a.parts = d.total < 16u * dev.num_sms ? (heads + at_once - 1) / at_once : 1;
    a.part_rows = a.parts > 1 ? at_once : heads;
    const uint64_t blocks = (static_cast<uint64_t>(d.total) * a.parts + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > 0x7fffffffu) return cudaErrorInvalidConfiguration;
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
