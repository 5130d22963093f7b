// bs_cache_attention.cu -- attention over the 8-bit token cache
// (include/bsearch.h, bs_cache_attention).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bs_device.cuh"
#include "bs_memory.h"

namespace bsb {

using namespace dev;

namespace {

struct CacheArgs {
    bs_token_cache c;
    bs_cache_attention_desc d;
    unsigned int* errors;
    float* lse;        // [num_seqs][queries][q_heads]
};

template <typename T>
__device__ __forceinline__ const T* query_row(const CacheArgs& a, uint32_t b, uint32_t i, uint32_t h) {
    return static_cast<const T*>(a.d.q) + b * a.d.q_stride[0] + i * a.d.q_stride[1] + h * a.d.q_stride[2];
}

__device__ __forceinline__ uint32_t held_tokens(const CacheArgs& a, uint32_t b) {
    const int32_t len = a.d.lens[b];
    const int64_t most = static_cast<int64_t>(a.d.table_width) * a.c.block;
    if (len >= 0 && len <= most) return len;
    if (threadIdx.x == 0) atomicOr(a.errors, kMemErrLength);
    return len < 0 ? 0 : static_cast<uint32_t>(most);
}

// The block of a position, or one past the cache's last where there is none.
__device__ __forceinline__ uint32_t block_of(const CacheArgs& a, uint32_t b, uint32_t pos) {
    const uint32_t id = a.d.table[static_cast<uint64_t>(b) * a.d.table_width + pos / a.c.block];
    if (id < a.c.num_blocks) return id;
    atomicOr(a.errors, kMemErrBlock);
    return a.c.num_blocks;
}

template <typename T>
__device__ __forceinline__ float score(const CacheArgs& a, const T* q, uint32_t b, uint32_t g, uint32_t pos) {
    const uint32_t id = block_of(a, b, pos);
    if (id == a.c.num_blocks) return -INFINITY;
    const uint64_t slab = static_cast<uint64_t>(id) * a.c.kv_heads + g;
    const int8_t* k = a.c.k + (slab * a.c.block + pos % a.c.block) * a.c.dim;
    float dot = 0.f;
    for (int32_t x = 0; x < a.c.dim; ++x) dot += static_cast<float>(q[x]) * k[x];
    return dot * (a.c.k_scale[slab] * a.d.scale);
}

// One warp per query and head.
template <typename T>
__global__ void __launch_bounds__(32) k_cache_rows(const CacheArgs a) {
    const uint32_t lane = threadIdx.x, h = blockIdx.x, i = blockIdx.y, b = blockIdx.z;
    const uint32_t g = h / (a.d.q_heads / a.c.kv_heads), dim = a.c.dim, block = a.c.block;
    const int64_t n = static_cast<int64_t>(held_tokens(a, b)) - a.d.queries + 1 + i;
    const T* q = query_row<T>(a, b, i, h);
    float top = -INFINITY, sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t j0 = 0; j0 < n; j0 += 32) {
        const float s = j0 + lane < n ? score<T>(a, q, b, g, static_cast<uint32_t>(j0 + lane)) : -INFINITY;
        float m = s;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
        const float next = fmaxf(top, m);
        const float safe = next == -INFINITY ? 0.f : next;
        const float shrink = expf(top - safe), p = expf(s - safe);
        sum = sum * shrink + p;
        top = next;
        for (int x = 0; x < 4; ++x) acc[x] *= shrink;
        for (int64_t j = j0; j < j0 + 32 && j < n; ++j) {
            const float w = __shfl_sync(kFull, p, static_cast<int>(j - j0));
            const uint32_t id = block_of(a, b, static_cast<uint32_t>(j));
            if (id == a.c.num_blocks) continue;
            const uint64_t slab = static_cast<uint64_t>(id) * a.c.kv_heads + g;
            const int8_t* v = a.c.v + (slab * block + j % block) * dim;
            const float ws = w * a.c.v_scale[slab];
            for (int x = 0; x < 4; ++x)
                if (lane + 32 * x < dim) acc[x] += ws * v[lane + 32 * x];
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
    const uint64_t row = (static_cast<uint64_t>(b) * a.d.queries + i) * a.d.q_heads + h;
    T* out = static_cast<T*>(a.d.out) + row * dim;
    for (int x = 0; x < 4; ++x)
        if (lane + 32 * x < dim) out[lane + 32 * x] = static_cast<T>(acc[x] * inv);
    if (lane == 0) a.lse[row] = sum == 0.f ? -INFINITY : top + logf(sum);
}

// One thread per token and key head: its weight over all queries and heads.
template <typename T>
__global__ void __launch_bounds__(256) k_cache_mass(const CacheArgs a) {
    const uint32_t j = blockIdx.x * 256 + threadIdx.x, g = blockIdx.y, b = blockIdx.z;
    const uint32_t len = held_tokens(a, b);
    if (j >= a.d.mass_width) return;
    const uint32_t group = a.d.q_heads / a.c.kv_heads;
    const uint64_t at = (static_cast<uint64_t>(b) * a.c.kv_heads + g) * a.d.mass_width + j;
    float w = 0.f;
    if (j < len) {
        w = a.d.mass ? a.d.mass[at] : 0.f;
        for (int32_t i = 0; i < a.d.queries; ++i) {
            if (static_cast<int64_t>(j) >= static_cast<int64_t>(len) - a.d.queries + 1 + i) continue;
            for (uint32_t h = g * group; h < (g + 1) * group; ++h) {
                const float lse = a.lse[(static_cast<uint64_t>(b) * a.d.queries + i) * a.d.q_heads + h];
                w += expf(score<T>(a, query_row<T>(a, b, i, h), b, g, j) - lse);
            }
        }
    }
    a.d.out_mass[at] = w;
}

template <typename T>
cudaError_t attention_typed(const CacheArgs& a, cudaStream_t stream) {
    k_cache_rows<T><<<dim3(a.d.q_heads, a.d.queries, a.d.num_seqs), 32, 0, stream>>>(a);
    if (a.d.out_mass)
        k_cache_mass<T><<<dim3((a.d.mass_width + 255) / 256, a.c.kv_heads, a.d.num_seqs), 256, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

size_t cache_attention_scratch(const bs_token_cache&, const bs_cache_attention_desc& d, const MemoryDevice&) {
    return d.lse ? 0 : static_cast<size_t>(d.num_seqs) * d.queries * d.q_heads * 4;
}

cudaError_t launch_cache_attention(const bs_token_cache& c, const bs_cache_attention_desc& d, const MemoryDevice& dev,
                                   cudaStream_t stream) {
    const CacheArgs a{c, d, dev.errors, d.lse ? d.lse : static_cast<float*>(d.workspace)};
    return d.dtype == BS_F16 ? attention_typed<__half>(a, stream) : attention_typed<__nv_bfloat16>(a, stream);
}

}  // namespace bsb
