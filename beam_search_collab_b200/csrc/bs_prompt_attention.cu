// bs_prompt_attention.cu -- attention of packed prompts (include/bsearch.h,
// bs_prompt_attention).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bs_device.cuh"
#include "bs_memory.h"

namespace bsb {

using namespace dev;

namespace {

struct PromptArgs {
    bs_prompt_attention_desc d;
    unsigned int* errors;
};

// One warp per query and head: each lane takes every 32nd key for the scores,
// then every 32nd dimension of the values; running maximum and sum in 32 bits.
template <typename T>
__global__ void __launch_bounds__(128) k_prompt_rows(const PromptArgs a) {
    const bs_prompt_attention_desc& d = a.d;
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t unit = static_cast<uint64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    if (unit >= static_cast<uint64_t>(d.total_q) * d.q_heads) return;
    const uint32_t row = static_cast<uint32_t>(unit / d.q_heads), h = static_cast<uint32_t>(unit % d.q_heads);
    uint32_t b = 0;
    while (b + 1 < d.num_seqs && static_cast<uint32_t>(d.cu_q[b + 1]) <= row) ++b;
    const int32_t q0 = d.cu_q[b], q1 = d.cu_q[b + 1], k0 = d.cu_k[b], k1 = d.cu_k[b + 1];
    const uint32_t g = h / (d.q_heads / d.kv_heads);
    int32_t n = k1 - k0;
    if (q0 < 0 || q1 < q0 || static_cast<uint32_t>(q1) > d.total_q || k0 < 0 || n < 0 || static_cast<uint32_t>(k1) > d.total_k) {
        if (lane == 0) atomicOr(a.errors, kMemErrLength);
        n = 0;
    }
    if (d.causal) n = min(n, static_cast<int32_t>(row) - q0 + n - (q1 - q0) + 1);
    const T* q = static_cast<const T*>(d.q) + row * d.q_stride[0] + h * d.q_stride[1];
    const T* k = static_cast<const T*>(d.k) + k0 * d.k_stride[0] + g * d.k_stride[1];
    const T* v = static_cast<const T*>(d.v) + k0 * d.v_stride[0] + g * d.v_stride[1];
    float top = -INFINITY, sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int32_t j0 = 0; j0 < n; j0 += 32) {
        float s = -INFINITY;
        if (j0 + static_cast<int32_t>(lane) < n) {
            float dot = 0.f;
            for (int32_t x = 0; x < d.dim; ++x)
                dot += static_cast<float>(q[x]) * static_cast<float>(k[(j0 + lane) * d.k_stride[0] + x]);
            s = dot * d.scale;
        }
        float m = s;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
        const float next = fmaxf(top, m);
        const float safe = next == -INFINITY ? 0.f : next;
        const float shrink = expf(top - safe), p = expf(s - safe);
        sum = sum * shrink + p;
        top = next;
        for (int i = 0; i < 4; ++i) acc[i] *= shrink;
        for (int32_t j = 0; j < 32 && j0 + j < n; ++j) {
            const float w = __shfl_sync(kFull, p, j);
            for (int i = 0; i < 4; ++i) {
                const int32_t x = lane + 32 * i;
                if (x < d.dim) acc[i] += w * static_cast<float>(v[(j0 + j) * d.v_stride[0] + x]);
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
    T* out = static_cast<T*>(d.out) + unit * d.dim;
    for (int i = 0; i < 4; ++i) {
        const int32_t x = lane + 32 * i;
        if (x < d.dim) out[x] = static_cast<T>(acc[i] * inv);
    }
    if (lane == 0 && d.lse) d.lse[unit] = sum == 0.f ? -INFINITY : top + logf(sum);
}

}  // namespace

cudaError_t launch_prompt_attention(const bs_prompt_attention_desc& d, const MemoryDevice& dev, cudaStream_t stream) {
    const PromptArgs a{d, dev.errors};
    const unsigned blocks = static_cast<unsigned>((static_cast<uint64_t>(d.total_q) * d.q_heads + 3) / 4);
    if (d.dtype == BS_F16) k_prompt_rows<__half><<<blocks, 128, 0, stream>>>(a);
    else k_prompt_rows<__nv_bfloat16><<<blocks, 128, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace bsb
