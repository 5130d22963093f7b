// bs_token_cache.cu -- writing to, reading from and evicting from the 8-bit
// token cache (include/bsearch.h, bs_token_cache).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bs_device.cuh"
#include "bs_memory.h"

namespace bsb {

using namespace dev;

namespace {

template <typename T>
__device__ __forceinline__ float2 pair_to_float(uint32_t u);
template <>
__device__ __forceinline__ float2 pair_to_float<__half>(uint32_t u) {
    return __half22float2(*reinterpret_cast<__half2*>(&u));
}
template <>
__device__ __forceinline__ float2 pair_to_float<__nv_bfloat16>(uint32_t u) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
}

__device__ __forceinline__ uint4 ldg_stream(const void* p) { return __ldcs(static_cast<const uint4*>(p)); }

// ------------------------------------------------------------------- write

struct WriteArgs {
    bs_token_cache c;
    bs_cache_write_desc d;
    unsigned int* errors;
};

constexpr int kWriteThreads = 128;

// One CTA writes one head's part of one block, keys (z = 0) or values (z = 1).
// Sequence b touches at most n / block + 2 blocks for its n tokens, so with
// base(b) = cu[b] / block + 2 b the CTAs base(b) .. base(b + 1) are enough for
// it, and a CTA finds its sequence by counting the bases at or below its index.
template <typename T, int CHUNKS>
__global__ void __launch_bounds__(kWriteThreads) k_cache_write(const WriteArgs a) {
    __shared__ float warp_max[kWriteThreads / 32];
    const bs_cache_write_desc& d = a.d;
    const uint32_t block = a.c.block, dim = a.c.dim, per_row = dim / 8;
    const uint32_t h = blockIdx.y;

    uint32_t at_or_below = 0;
    for (uint32_t b0 = 0; b0 < d.num_seqs; b0 += kWriteThreads) {
        const uint32_t b = b0 + threadIdx.x;
        const bool below = b < d.num_seqs && static_cast<uint32_t>(d.cu[b]) / block + 2 * b <= blockIdx.x;
        const uint32_t n = __syncthreads_count(below);
        at_or_below += n;
        if (n < kWriteThreads) break;
    }
    if (at_or_below == 0) return;
    const uint32_t b = at_or_below - 1;
    const int32_t first = d.cu[b], past = d.cu[b + 1], start = d.start[b];
    if (first < 0 || past < first || static_cast<uint32_t>(past) > d.total || start < 0) {
        if (threadIdx.x == 0) atomicOr(a.errors, kMemErrLength);
        return;
    }
    const uint32_t n = past - first;
    const uint32_t col = static_cast<uint32_t>(start) / block + (blockIdx.x - (static_cast<uint32_t>(first) / block + 2 * b));
    const int64_t end = static_cast<int64_t>(start) + n;
    const int64_t lo = static_cast<int64_t>(col) * block;      // position of the block's first token
    if (n == 0 || lo >= end) return;
    if (col >= d.table_width) {
        if (threadIdx.x == 0) atomicOr(a.errors, kMemErrLength);
        return;
    }
    const uint32_t id = d.table[static_cast<uint64_t>(b) * d.table_width + col];
    if (id >= a.c.num_blocks) {
        if (threadIdx.x == 0) atomicOr(a.errors, kMemErrBlock);
        return;
    }
    const uint32_t held = lo < start ? static_cast<uint32_t>(start - lo) : 0;   // earlier tokens in the block
    const uint32_t stop = end - lo < block ? static_cast<uint32_t>(end - lo) : block;
    const uint64_t slab = static_cast<uint64_t>(id) * a.c.kv_heads + h;
    int8_t* codes = (blockIdx.z ? a.c.v : a.c.k) + slab * block * dim;
    float* scale_at = (blockIdx.z ? a.c.v_scale : a.c.k_scale) + slab;
    const int64_t* stride = blockIdx.z ? d.v_stride : d.k_stride;
    // the block's slot s holds row first + (lo + s - start)
    const T* src = static_cast<const T*>(blockIdx.z ? d.v : d.k) + (first + lo - start) * stride[0] + h * stride[1];

    uint4 x[CHUNKS];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        const uint32_t chunk = held * per_row + i * kWriteThreads + threadIdx.x;
        x[i] = make_uint4(0, 0, 0, 0);
        if (chunk < stop * per_row) x[i] = ldg_stream(src + (chunk / per_row) * stride[0] + (chunk % per_row) * 8);
    }
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = pair_to_float<T>(w[j]);
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = top;
    const float old = held ? *scale_at : 0.f;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWriteThreads / 32; ++i) top = fmaxf(top, warp_max[i]);
    const float fresh = top < 1e-30f ? 0.f : top * (1.f / 127.f);
    const float scale = fmaxf(fresh, old);
    const float inv = scale > 0.f ? __frcp_rn(scale) : 0.f;

    if (scale > old && held) {      // the earlier tokens' codes at the larger scale
        const float ratio = __fdiv_rn(old, scale);
        for (uint32_t chunk = threadIdx.x; chunk < held * per_row; chunk += kWriteThreads) {
            uint2* p = reinterpret_cast<uint2*>(codes) + chunk;
            uint2 u = *p;
            int8_t* c = reinterpret_cast<int8_t*>(&u);
#pragma unroll
            for (int j = 0; j < 8; ++j) c[j] = static_cast<int8_t>(__float2int_rn(c[j] * ratio));
            *p = u;
        }
    }
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        const uint32_t chunk = held * per_row + i * kWriteThreads + threadIdx.x;
        if (chunk >= stop * per_row) continue;
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        uint2 u;
        int8_t* c = reinterpret_cast<int8_t*>(&u);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = pair_to_float<T>(w[j]);
            c[2 * j] = static_cast<int8_t>(max(-127, min(127, __float2int_rn(f.x * inv))));
            c[2 * j + 1] = static_cast<int8_t>(max(-127, min(127, __float2int_rn(f.y * inv))));
        }
        reinterpret_cast<uint2*>(codes)[chunk] = u;
    }
    if (threadIdx.x == 0) *scale_at = scale;
}

template <typename T>
cudaError_t write_typed(const WriteArgs& a, cudaStream_t stream) {
    const uint32_t chunks = a.c.block * a.c.dim / 8;      // of 8 values, per block and head
    const uint64_t blocks = a.d.total / a.c.block + 2ull * a.d.num_seqs + 1;
    const dim3 grid(static_cast<unsigned>(blocks), a.c.kv_heads, 2);
    if (chunks <= kWriteThreads) k_cache_write<T, 1><<<grid, kWriteThreads, 0, stream>>>(a);
    else if (chunks <= 2 * kWriteThreads) k_cache_write<T, 2><<<grid, kWriteThreads, 0, stream>>>(a);
    else if (chunks <= 4 * kWriteThreads) k_cache_write<T, 4><<<grid, kWriteThreads, 0, stream>>>(a);
    else if (chunks <= 8 * kWriteThreads) k_cache_write<T, 8><<<grid, kWriteThreads, 0, stream>>>(a);
    else k_cache_write<T, 16><<<grid, kWriteThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

// -------------------------------------------------------------------- read

struct ReadArgs {
    bs_token_cache c;
    bs_cache_read_desc d;
    unsigned int* errors;
};

template <typename T>
__device__ __forceinline__ void store_values(void* out, uint64_t at, uint4 codes, float scale) {
    const int8_t* c = reinterpret_cast<const int8_t*>(&codes);
    __align__(16) T v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = static_cast<T>(c[j] * scale);
    uint4* p = reinterpret_cast<uint4*>(static_cast<T*>(out) + at);
#pragma unroll
    for (unsigned j = 0; j < sizeof(v) / 16; ++j) __stcs(p + j, reinterpret_cast<const uint4*>(v)[j]);
}

// One thread: 16 codes of one position's key and value.
template <typename T>
__global__ void __launch_bounds__(256) k_cache_read(const ReadArgs a) {
    const bs_cache_read_desc& d = a.d;
    const uint32_t per_row = a.c.dim / 16, h = blockIdx.y, b = blockIdx.z;
    const uint64_t unit = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (unit >= static_cast<uint64_t>(d.count) * per_row) return;
    const uint32_t i = static_cast<uint32_t>(unit / per_row), chunk = static_cast<uint32_t>(unit % per_row);
    const int32_t pos = d.positions[b * d.position_seq_stride + h * d.position_head_stride + i];
    uint4 kc = make_uint4(0, 0, 0, 0), vc = kc;
    float ks = 0.f, vs = 0.f;
    if (pos >= 0 && pos < d.lens[b]) {
        const uint32_t col = static_cast<uint32_t>(pos) / a.c.block;
        const uint32_t id = col < d.table_width ? d.table[static_cast<uint64_t>(b) * d.table_width + col] : kNoNode;
        if (id < a.c.num_blocks) {
            const uint64_t slab = static_cast<uint64_t>(id) * a.c.kv_heads + h;
            const uint64_t row = (slab * a.c.block + pos % a.c.block) * a.c.dim + chunk * 16;
            if (d.k) {
                kc = ldg_stream(a.c.k + row);
                ks = a.c.k_scale[slab];
            }
            if (d.v) {
                vc = ldg_stream(a.c.v + row);
                vs = a.c.v_scale[slab];
            }
        } else if (chunk == 0) {
            atomicOr(a.errors, col < d.table_width ? kMemErrBlock : kMemErrLength);
        }
    }
    const uint64_t at = ((static_cast<uint64_t>(b) * a.c.kv_heads + h) * d.count + i) * a.c.dim + chunk * 16;
    if (d.k) store_values<T>(d.k, at, kc, ks);
    if (d.v) store_values<T>(d.v, at, vc, vs);
}

// ---------------------------------------------------------------- eviction

struct EvictArgs {
    bs_token_cache c;
    bs_cache_evict_desc d;
    unsigned int* errors;
};

// Order of weights as integers: larger weight, larger key; NaN above all.
__device__ __forceinline__ uint32_t mass_key(float f) { return isnan(f) ? 0xffffffffu : f2ord(f); }

constexpr int kSelectThreads = 1024;

// One CTA: which tokens of one sequence stay for one head.  The m-th largest
// key among the free tokens is found digit by digit (8 bits at a time, counted
// in shared memory); then one ordered pass numbers the tokens that stay.
__global__ void __launch_bounds__(kSelectThreads) k_evict_select(const EvictArgs a) {
    __shared__ uint32_t count[256];
    __shared__ uint32_t chosen[2];
    __shared__ uint32_t warp_sum[2][32];
    const bs_cache_evict_desc& d = a.d;
    const uint32_t h = blockIdx.x, b = blockIdx.y, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const uint64_t row = static_cast<uint64_t>(b) * a.c.kv_heads + h;
    const float* mass = d.mass + row * d.mass_width;
    int32_t* kept = d.kept + row * d.budget;
    float* new_mass = d.new_mass + row * d.budget;
    int32_t len = d.lens[b];
    const uint64_t most = min(static_cast<uint64_t>(d.table_width) * a.c.block, static_cast<uint64_t>(d.mass_width));
    if (len < 0 || static_cast<uint64_t>(len) > most) {
        if (t == 0) atomicOr(a.errors, kMemErrLength);
        len = len < 0 ? 0 : static_cast<int32_t>(most);
    }
    const uint32_t n = len, budget = d.budget, stay = n < budget ? n : budget;
    if (h == 0 && t == 0) d.new_lens[b] = stay;
    for (uint32_t i = stay + t; i < budget; i += kSelectThreads) {
        kept[i] = -1;
        new_mass[i] = 0.f;
    }
    if (n <= budget) {
        for (uint32_t i = t; i < n; i += kSelectThreads) {
            kept[i] = i;
            new_mass[i] = mass[i];
        }
        return;
    }
    const uint32_t lo = d.sinks, hi = n - d.recent;
    uint32_t need = budget - d.sinks - d.recent;      // of the free tokens [lo, hi); fewer than there are
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0 && need; shift -= 8) {
        for (uint32_t i = t; i < 256; i += kSelectThreads) count[i] = 0;
        __syncthreads();
        for (uint32_t i = lo + t; i < hi; i += kSelectThreads) {
            const uint32_t key = mass_key(mass[i]);
            if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&count[(key >> shift) & 255], 1u);
        }
        __syncthreads();
        if (t == 0) {
            uint32_t left = need, digit = 255;
            while (count[digit] < left) left -= count[digit--];
            chosen[0] = prefix | (digit << shift);
            chosen[1] = left;
        }
        __syncthreads();
        prefix = chosen[0];
        need = chosen[1];
    }
    // stays: forced, above the threshold, or one of the first `need` equal to it
    const bool any = budget > static_cast<uint32_t>(d.sinks) + d.recent;
    uint32_t base = 0, base_eq = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += kSelectThreads) {
        const uint32_t i = i0 + t;
        const float w = i < n ? mass[i] : 0.f;
        const bool is_free = i >= lo && i < hi;
        const uint32_t key = mass_key(w);
        const bool eq = is_free && any && key == prefix;
        const unsigned eq_mask = __ballot_sync(kFull, eq);
        if (lane == 0) warp_sum[0][warp] = __popc(eq_mask);
        __syncthreads();
        uint32_t before = base_eq, total_eq = 0;
        for (uint32_t k = 0; k < 32; ++k) {
            before += k < warp ? warp_sum[0][k] : 0;
            total_eq += warp_sum[0][k];
        }
        before += __popc(eq_mask & ((1u << lane) - 1));
        const bool in = i < n && (!is_free || (any && key > prefix) || (eq && before < need));
        const unsigned in_mask = __ballot_sync(kFull, in);
        if (lane == 0) warp_sum[1][warp] = __popc(in_mask);
        __syncthreads();
        uint32_t to = base, total = 0;
        for (uint32_t k = 0; k < 32; ++k) {
            to += k < warp ? warp_sum[1][k] : 0;
            total += warp_sum[1][k];
        }
        to += __popc(in_mask & ((1u << lane) - 1));
        if (in) {
            kept[to] = i;
            new_mass[to] = w;
        }
        base += total;
        base_eq += total_eq;
        __syncthreads();
    }
}

constexpr int kMoveThreads = 256;

// One CTA: one new block of one head, keys and values.
__global__ void __launch_bounds__(kMoveThreads) k_evict_move(const EvictArgs a) {
    __shared__ int64_t from[128];          // row of each token in the codes, -1: none
    __shared__ float scale[2][128];
    __shared__ float top[2];
    const bs_cache_evict_desc& d = a.d;
    const uint32_t col = blockIdx.x, h = blockIdx.y, b = blockIdx.z, t = threadIdx.x, block = a.c.block;
    const uint64_t row = static_cast<uint64_t>(b) * a.c.kv_heads + h;
    const uint32_t i0 = col * block;
    const uint32_t most = min(d.new_lens[b], d.budget);
    if (i0 >= most) return;
    const uint32_t id = d.new_table[static_cast<uint64_t>(b) * d.new_table_width + col];
    if (id >= a.c.num_blocks) {
        if (t == 0) atomicOr(a.errors, kMemErrBlock);
        return;
    }
    if (t < block) {
        int64_t r = -1;
        float ks = 0.f, vs = 0.f;
        if (i0 + t < most) {
            const uint32_t pos = d.kept[row * d.budget + i0 + t];
            const uint32_t src = d.table[static_cast<uint64_t>(b) * d.table_width + pos / block];
            if (src < a.c.num_blocks) {
                const uint64_t slab = static_cast<uint64_t>(src) * a.c.kv_heads + h;
                r = slab * block + pos % block;
                ks = a.c.k_scale[slab];
                vs = a.c.v_scale[slab];
            } else {
                atomicOr(a.errors, kMemErrBlock);
            }
        }
        from[t] = r;
        scale[0][t] = ks;
        scale[1][t] = vs;
    }
    __syncthreads();
    const uint64_t slab = static_cast<uint64_t>(id) * a.c.kv_heads + h;
    if (t < 64) {
        float m = 0.f;
        for (uint32_t i = t & 31; i < block; i += 32) m = fmaxf(m, scale[t >> 5][i]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
        if ((t & 31) == 0) {
            top[t >> 5] = m;
            (t >> 5 ? a.c.v_scale : a.c.k_scale)[slab] = m;
        }
    }
    __syncthreads();
    const uint32_t per_row = a.c.dim / 16;
    for (uint32_t u = t; u < 2 * block * per_row; u += kMoveThreads) {
        const uint32_t kv = u >= block * per_row, w = u - kv * block * per_row, i = w / per_row, chunk = w % per_row;
        uint4 codes = make_uint4(0, 0, 0, 0);
        if (from[i] >= 0) {
            const int8_t* src = kv ? a.c.v : a.c.k;
            codes = ldg_stream(src + from[i] * a.c.dim + chunk * 16);
            const float ratio = top[kv] > 0.f ? __fdiv_rn(scale[kv][i], top[kv]) : 0.f;
            if (ratio != 1.f) {
                int8_t* c = reinterpret_cast<int8_t*>(&codes);
#pragma unroll
                for (int j = 0; j < 16; ++j) c[j] = static_cast<int8_t>(__float2int_rn(c[j] * ratio));
            }
        }
        int8_t* dst = (kv ? a.c.v : a.c.k) + (slab * block + i) * a.c.dim + chunk * 16;
        *reinterpret_cast<uint4*>(dst) = codes;
    }
}

}  // namespace

cudaError_t launch_cache_write(const bs_token_cache& c, const bs_cache_write_desc& d, const MemoryDevice& dev,
                               cudaStream_t stream) {
    const WriteArgs a{c, d, dev.errors};
    return d.dtype == BS_F16 ? write_typed<__half>(a, stream) : write_typed<__nv_bfloat16>(a, stream);
}

cudaError_t launch_cache_read(const bs_token_cache& c, const bs_cache_read_desc& d, const MemoryDevice& dev,
                              cudaStream_t stream) {
    const ReadArgs a{c, d, dev.errors};
    const uint64_t units = static_cast<uint64_t>(d.count) * (c.dim / 16);
    const dim3 grid(static_cast<unsigned>((units + 255) / 256), c.kv_heads, d.num_seqs);
    if (d.dtype == BS_F32) k_cache_read<float><<<grid, 256, 0, stream>>>(a);
    else if (d.dtype == BS_F16) k_cache_read<__half><<<grid, 256, 0, stream>>>(a);
    else k_cache_read<__nv_bfloat16><<<grid, 256, 0, stream>>>(a);
    return cudaGetLastError();
}

size_t cache_evict_scratch(const bs_token_cache&, const bs_cache_evict_desc&, const MemoryDevice&) { return 0; }

cudaError_t launch_cache_evict(const bs_token_cache& c, const bs_cache_evict_desc& d, const MemoryDevice& dev,
                               cudaStream_t stream) {
    const EvictArgs a{c, d, dev.errors};
    k_evict_select<<<dim3(c.kv_heads, d.num_seqs), kSelectThreads, 0, stream>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const uint32_t cols = (d.budget + c.block - 1) / c.block;
    const uint32_t used = cols < d.new_table_width ? cols : d.new_table_width;
    if (used) k_evict_move<<<dim3(used, c.kv_heads, d.num_seqs), kMoveThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace bsb
