// bs_token_cache.cu -- writing to, reading from and evicting from the 8-bit
// token cache (include/bsearch.h, bs_token_cache).
//
// All of them are bound by memory, provided the conversions stay off the
// special-function pipe (16 int <-> float conversions a clock and SM: the
// eviction's move took 60 us through it, as long as all its traffic), so
// integers are made and read through a float's low bits.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bs_device.cuh"
#include "bs_f32x2.cuh"
#include "bs_memory.h"

namespace bsb {

using namespace dev;

namespace {

// Two 16-bit values of a word: as floats, and the larger magnitudes of two
// words' (exact in 16 bits).
template <typename T>
__device__ __forceinline__ float2 pair_to_float(uint32_t u);
template <typename T>
__device__ __forceinline__ uint32_t larger_magnitudes(uint32_t top, uint32_t u);
template <>
__device__ __forceinline__ float2 pair_to_float<__half>(uint32_t u) {
    return __half22float2(*reinterpret_cast<__half2*>(&u));
}
template <>
__device__ __forceinline__ uint32_t larger_magnitudes<__half>(uint32_t top, uint32_t u) {
    const __half2 h = __hmax2(*reinterpret_cast<__half2*>(&top), __habs2(*reinterpret_cast<__half2*>(&u)));
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ float2 pair_to_float<__nv_bfloat16>(uint32_t u) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
}
template <>
__device__ __forceinline__ uint32_t larger_magnitudes<__nv_bfloat16>(uint32_t top, uint32_t u) {
    const __nv_bfloat162 h = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&top), __habs2(*reinterpret_cast<__nv_bfloat162*>(&u)));
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint4 ldg_stream(const void* p) { return __ldcs(static_cast<const uint4*>(p)); }

struct Four {
    float2 lo, hi;
};

// Four codes of a word as floats: 0x4b000000 | u is 2^23 + u.
__device__ __forceinline__ Four codes_to_floats(uint32_t w) {
    const uint32_t u = w ^ 0x80808080u;
    const float2 bias = make_float2(-(8388608.f + 128.f), -(8388608.f + 128.f));
    return {add2(make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7541))), bias),
            add2(make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7542)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7543))), bias)};
}

// Four values times `by` (rounded to 32 bits), rint, their low bytes as a word:
// a sum with 1.5 * 2^23 rounds to the nearest integer, ties to even.  The
// products are below 2^22 in magnitude.  (One at a time: a packed product and
// sum were contracted to one rounding.)
__device__ __forceinline__ uint32_t floats_to_codes(Four x, float by) {
    const float2 magic = make_float2(12582912.f, 12582912.f);
    const float2 a = add2(make_float2(__fmul_rn(x.lo.x, by), __fmul_rn(x.lo.y, by)), magic);
    const float2 b = add2(make_float2(__fmul_rn(x.hi.x, by), __fmul_rn(x.hi.y, by)), magic);
    const uint32_t lo = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
}

// Codes times a ratio of at most 1, rounded.
__device__ __forceinline__ uint32_t rescaled(uint32_t w, float ratio) { return floats_to_codes(codes_to_floats(w), ratio); }

// x / d for x < 2048 and d <= 16, from reciprocal(d): off by less than x / 2^16.
__device__ __forceinline__ uint32_t reciprocal(uint32_t d) { return 65536u / d + 1; }
__device__ __forceinline__ uint32_t divided(uint32_t x, uint32_t by) { return (x * by) >> 16; }

// ------------------------------------------------------------------- write

struct WriteArgs {
    bs_token_cache c;
    bs_cache_write_desc d;
    unsigned int* errors;
};

constexpr int kWriteThreads = 256;

// One block writes one head's part of one cache block, keys and values.
// Sequence b touches at most n / block + 2 blocks for its n tokens, so with
// base(b) = cu[b] / block + 2 b the thread blocks base(b) .. base(b + 1) are
// enough for it, and one finds its sequence by counting the bases at or below
// its index.  Bound by the chain of loads before the values (lengths, table,
// values) rather than by bytes, so both tensors' values are requested at once.
// Measured: 15,868 tokens, 8 heads of 128 (97 MB) 22.6 us (4.3 TB/s); one token
// of each of 64 sequences 5.7 us.
template <typename T, int CHUNKS>
__global__ void __launch_bounds__(kWriteThreads, CHUNKS <= 2 ? 4 : CHUNKS == 4 ? 3 : 2) k_cache_write(const __grid_constant__ WriteArgs a) {
    __shared__ float warp_max[2][kWriteThreads / 32];
    __shared__ int32_t found[3];               // cu[b], cu[b + 1], start[b]
    const bs_cache_write_desc& d = a.d;
    const uint32_t block = a.c.block, dim = a.c.dim, per_row = dim / 8;
    // heads side by side: their rows are side by side in k and v
    const uint32_t h = blockIdx.x % a.c.kv_heads, place = blockIdx.x / a.c.kv_heads;

    cudaGridDependencySynchronize();       // in every block, before anything of the caller's
    uint32_t at_or_below = 0;
    for (uint32_t b0 = 0; b0 < d.num_seqs; b0 += kWriteThreads) {
        const uint32_t i = b0 + threadIdx.x;
        const int32_t first = i < d.num_seqs ? d.cu[i] : 0, past = i < d.num_seqs ? d.cu[i + 1] : 0;
        const int32_t start = i < d.num_seqs ? d.start[i] : 0;
        const uint32_t n = __syncthreads_count(i < d.num_seqs && static_cast<uint32_t>(first) / block + 2 * i <= place);
        if (n && threadIdx.x == n - 1) {
            found[0] = first;
            found[1] = past;
            found[2] = start;
        }
        at_or_below += n;
        if (n < kWriteThreads) break;
    }
    __syncthreads();
    if (at_or_below == 0) return;
    const uint32_t b = at_or_below - 1;
    const int32_t first = found[0], past = found[1], start = found[2];
    if (first < 0 || past < first || static_cast<uint32_t>(past) > d.total || start < 0) {
        if (threadIdx.x == 0) atomicOr(a.errors, kMemErrLength);
        return;
    }
    const uint32_t n = past - first;
    const uint32_t col = static_cast<uint32_t>(start) / block + (place - (static_cast<uint32_t>(first) / block + 2 * b));
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

    uint4 x[2][CHUNKS];
    float top[2] = {0.f, 0.f}, old[2];
    const uint32_t by_row = reciprocal(per_row);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        const int64_t* stride = kv ? d.v_stride : d.k_stride;
        // the block's slot s holds row first + (lo + s - start)
        const T* src = static_cast<const T*>(kv ? d.v : d.k) + (first + lo - start) * stride[0] + h * stride[1];
        old[kv] = held ? (kv ? a.c.v_scale : a.c.k_scale)[slab] : 0.f;
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const uint32_t chunk = held * per_row + i * kWriteThreads + threadIdx.x;
            x[kv][i] = make_uint4(0, 0, 0, 0);
            const uint32_t r = divided(chunk, by_row);
            if (chunk < stop * per_row) x[kv][i] = ldg_stream(src + r * stride[0] + (chunk - r * per_row) * 8);
        }
    }
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            most = larger_magnitudes<T>(larger_magnitudes<T>(most, x[kv][i].x), x[kv][i].y);
            most = larger_magnitudes<T>(larger_magnitudes<T>(most, x[kv][i].z), x[kv][i].w);
        }
        const float2 two = pair_to_float<T>(most);
        top[kv] = fmaxf(two.x, two.y);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top[kv] = fmaxf(top[kv], __shfl_xor_sync(kFull, top[kv], o));
        if ((threadIdx.x & 31) == 0) warp_max[kv][threadIdx.x >> 5] = top[kv];
    }
    __syncthreads();
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        int8_t* codes = (kv ? a.c.v : a.c.k) + slab * block * dim;
#pragma unroll
        for (int i = 0; i < kWriteThreads / 32; ++i) top[kv] = fmaxf(top[kv], warp_max[kv][i]);
        const float fresh = top[kv] < 1e-30f ? 0.f : top[kv] * (1.f / 127.f);
        const float scale = fmaxf(fresh, old[kv]);
        const float inv = scale > 0.f ? __frcp_rn(scale) : 0.f;

        if (scale > old[kv] && held) {      // the earlier tokens' codes at the larger scale
            const float ratio = __fdiv_rn(old[kv], scale);
            for (uint32_t chunk = threadIdx.x; chunk < held * per_row; chunk += kWriteThreads) {
                uint2* p = reinterpret_cast<uint2*>(codes) + chunk;
                const uint2 u = *p;
                *p = make_uint2(rescaled(u.x, ratio), rescaled(u.y, ratio));
            }
        }
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const uint32_t chunk = held * per_row + i * kWriteThreads + threadIdx.x;
            if (chunk >= stop * per_row) continue;
            const uint32_t w[4] = {x[kv][i].x, x[kv][i].y, x[kv][i].z, x[kv][i].w};
            // (|x| * inv is at most 127 and a rounding: no clamp)
            const uint32_t lo = floats_to_codes({pair_to_float<T>(w[0]), pair_to_float<T>(w[1])}, inv);
            const uint32_t hi = floats_to_codes({pair_to_float<T>(w[2]), pair_to_float<T>(w[3])}, inv);
            reinterpret_cast<uint2*>(codes)[chunk] = make_uint2(lo, hi);
        }
        if (threadIdx.x == 0) (kv ? a.c.v_scale : a.c.k_scale)[slab] = scale;
    }
}

template <typename T>
cudaError_t write_typed(const WriteArgs& a, cudaStream_t stream) {
    const uint32_t chunks = a.c.block * a.c.dim / 8;      // of 8 values, per block, head and tensor
    const uint64_t blocks = (a.d.total / a.c.block + 2ull * a.d.num_seqs + 1) * a.c.kv_heads;
    if (blocks > 0x7fffffffu) return cudaErrorInvalidConfiguration;
    const unsigned grid = static_cast<unsigned>(blocks);
    if (chunks <= kWriteThreads) return launch_after(k_cache_write<T, 1>, dim3(grid), kWriteThreads, 0, stream, a);
    if (chunks <= 2 * kWriteThreads) return launch_after(k_cache_write<T, 2>, dim3(grid), kWriteThreads, 0, stream, a);
    if (chunks <= 4 * kWriteThreads) return launch_after(k_cache_write<T, 4>, dim3(grid), kWriteThreads, 0, stream, a);
    return launch_after(k_cache_write<T, 8>, dim3(grid), kWriteThreads, 0, stream, a);
}

// -------------------------------------------------------------------- read

struct ReadArgs {
    bs_token_cache c;
    bs_cache_read_desc d;
    unsigned int* errors;
};

template <typename T>
__device__ __forceinline__ T rounded(float x);
template <>
__device__ __forceinline__ float rounded<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ __half rounded<__half>(float x) {
    return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}

template <typename T>
__device__ __forceinline__ void store_values(void* out, uint64_t at, uint4 codes, float scale) {
    const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
    __align__(16) T v[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const Four f = codes_to_floats(w[j]);
        const float2 lo = mul2(f.lo, make_float2(scale, scale)), hi = mul2(f.hi, make_float2(scale, scale));
        v[4 * j] = rounded<T>(lo.x);
        v[4 * j + 1] = rounded<T>(lo.y);
        v[4 * j + 2] = rounded<T>(hi.x);
        v[4 * j + 3] = rounded<T>(hi.y);
    }
    uint4* p = reinterpret_cast<uint4*>(static_cast<T*>(out) + at);
#pragma unroll
    for (unsigned j = 0; j < sizeof(v) / 16; ++j) __stcs(p + j, reinterpret_cast<const uint4*>(v)[j]);
}

// One thread: 16 codes of one position's key and value.  (Two or four
// positions a thread were slower: 62 and 66 us against 56 where 267 MB move.)
// Bound by DRAM: 4.6 TB/s there, 6.0 where 385 MB are read and written.
constexpr int kReadThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kReadThreads) k_cache_read(const __grid_constant__ ReadArgs a) {
    const bs_cache_read_desc& d = a.d;
    const uint32_t per_row = a.c.dim / 16, h = blockIdx.y, b = blockIdx.z;
    const uint32_t rows = kReadThreads / per_row, r = divided(threadIdx.x, reciprocal(per_row)), chunk = threadIdx.x - r * per_row;
    const uint32_t i = blockIdx.x * rows + r;
    cudaGridDependencySynchronize();       // in every block, before anything of the caller's
    if (r >= rows || i >= d.count) return;
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

// Which tokens of one sequence stay for one head: a cluster of blocks holds
// the row's keys in shared memory, a slice each (what does not fit is read
// again from L2).  The m-th largest key among the free tokens is found by its
// digits of 11, 11 and 10 bits, counted by every block and added up through
// distributed shared memory; then each block numbers the tokens of its slice
// that stay, in order, from what the blocks before it have.
//   measured, 32 rows of 8,000 to 65,536 tokens: 26 us (one block a row, 8-bit
//   digits from L2: 219).  4.7 MB come from DRAM; bound by counting in shared
//   memory and the barriers between the digits.  16 rows of 18,000 and 868,000
//   tokens, where most keys are read again from L2, take 168 us.
constexpr uint32_t kBins = 2048;
constexpr uint32_t kMostCached = 46 * 1024;       // keys of a slice in shared memory
constexpr uint32_t kMostCluster = 8;

// Exclusive prefix over the block of one number per thread, and the total.
template <int THREADS>
__device__ __forceinline__ uint32_t block_prefix(uint32_t x, uint32_t* warp_sums, uint32_t& total) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t sum = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(kFull, sum, o);
        if (lane >= static_cast<uint32_t>(o)) sum += up;
    }
    __syncthreads();                 // the last use of warp_sums is over
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    const uint32_t mine = lane < THREADS / 32 ? warp_sums[lane] : 0;
    uint32_t before = lane < warp ? mine : 0, all = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        before += __shfl_xor_sync(kFull, before, o);
        all += __shfl_xor_sync(kFull, all, o);
    }
    total = all;
    return before + sum - x;
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) k_evict_select(const __grid_constant__ EvictArgs a, uint32_t cached) {
    namespace cg = cooperative_groups;
    extern __shared__ uint32_t keys[];             // [cached]
    __shared__ __align__(16) uint32_t count[3][kBins];
    __shared__ uint32_t warp_sums[32];
    __shared__ uint32_t slice_counts[2];           // tokens that stay for certain, tokens equal to the threshold
    __shared__ uint32_t chosen[2];
    cudaGridDependencySynchronize();       // in every block, before anything of the caller's
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank(), blocks = cluster.num_blocks();
    const bs_cache_evict_desc& d = a.d;
    const uint32_t h = blockIdx.x / blocks, b = blockIdx.y, t = threadIdx.x, lane = t & 31;
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
    if (blockIdx.x == 0 && t == 0) d.new_lens[b] = stay;
    for (uint32_t i = stay + rank * THREADS + t; i < budget; i += blocks * THREADS) {
        kept[i] = -1;
        new_mass[i] = 0.f;
    }
    if (n <= budget) {                             // (the whole cluster)
        for (uint32_t i = rank * THREADS + t; i < n; i += blocks * THREADS) {
            kept[i] = i;
            new_mass[i] = mass[i];
        }
        return;
    }
    // this block's slice of the row
    const uint32_t width = ((n + blocks - 1) / blocks + 3) & ~3u;
    const uint32_t first = min(rank * width, n), size = min(width, n - first);
    const uint32_t lo = d.sinks, hi = n - d.recent;              // free tokens
    auto key_of = [&](uint32_t i) { return i < cached ? keys[i] : mass_key(mass[first + i]); };
    auto sync = [&]() {
        if (blocks > 1) cluster.sync();
        else __syncthreads();
    };
#pragma unroll
    for (uint32_t i = t; i < 3 * kBins / 4; i += THREADS) reinterpret_cast<uint4*>(&count[0][0])[i] = make_uint4(0, 0, 0, 0);
    for (uint32_t i0 = t; i0 < min(size, cached); i0 += 8 * THREADS) {
        float x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = i0 + u * THREADS < size ? mass[first + i0 + u * THREADS] : 0.f;
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (i0 + u * THREADS < min(size, cached)) keys[i0 + u * THREADS] = mass_key(x[u]);
    }
    __syncthreads();

    uint32_t need = budget - d.sinks - d.recent;   // of the free tokens; fewer than there are
    const bool any = need > 0;
    uint32_t prefix = 0;
    const uint32_t free0 = max(lo, first) - first, free1 = max(min(hi, first + size), first + free0) - first;   // of the slice
    uint32_t above = 0;                            // free tokens of the slice above the threshold
    if (any) {
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, known = pass == 1 ? 21 : 10;
            const uint32_t mask = pass == 2 ? 1023 : 2047;
            for (uint32_t i0 = free0; i0 < free1; i0 += 4 * THREADS) {    // (all lanes together)
                uint32_t key[4];
                bool in[4];
#pragma unroll
                for (uint32_t u = 0; u < 4; ++u) {
                    const uint32_t i = i0 + u * THREADS + t;
                    in[u] = i < free1;
                    key[u] = in[u] ? key_of(i) : 0;
                    if (pass) in[u] = in[u] && (key[u] ^ prefix) >> known == 0;
                }
#pragma unroll
                for (uint32_t u = 0; u < 4; ++u) {
                    const uint32_t digit = (key[u] >> shift) & mask;
                    // a warp whose tokens all agree counts once: rows of equal weights do not queue up
                    const uint32_t lead = __shfl_sync(kFull, digit, 0);
                    if (__all_sync(kFull, in[u] && digit == lead)) {
                        if (lane == 0) atomicAdd(&count[pass][digit], 32u);
                    } else if (in[u]) {
                        atomicAdd(&count[pass][digit], 1u);
                    }
                }
            }
            __syncwarp();
            sync();
            // bins from the largest digit down, kBins / THREADS to a thread
            constexpr int kEach = kBins / THREADS;
            uint32_t mine[kEach] = {}, sum = 0;
            const uint32_t top_bin = kBins - (t + 1) * kEach;
#pragma unroll
            for (uint32_t x = 0; x < kMostCluster; ++x) {
                if (x >= blocks) break;
                const uint2* from = reinterpret_cast<const uint2*>(cluster.map_shared_rank(&count[pass][0], x) + top_bin);
#pragma unroll
                for (int u = 0; u < kEach / 2; ++u) {
                    const uint2 c = from[u];
                    mine[kEach - 1 - 2 * u] += c.x;
                    mine[kEach - 2 - 2 * u] += c.y;
                }
            }
#pragma unroll
            for (int u = 0; u < kEach; ++u) sum += mine[u];
            uint32_t total;
            uint32_t before = block_prefix<THREADS>(sum, warp_sums, total);
#pragma unroll
            for (int u = 0; u < kEach; ++u) {
                if (before < need && need <= before + mine[u]) {
                    chosen[0] = prefix | (kBins - 1 - (t * kEach + u)) << shift;
                    chosen[1] = need - before;
                }
                before += mine[u];
            }
            __syncthreads();
            prefix = chosen[0];
            need = chosen[1];
            const uint32_t digit = (prefix >> shift) & mask;
#pragma unroll
            for (int u = 0; u < kEach; ++u)
                if (top_bin + u > digit) above += count[pass][top_bin + u];
        }
    }
    // a token stays if it is not free, above the threshold, or one of the
    // first `need` equal to it; both kinds are counted in one number
    auto kind = [&](uint32_t i) -> uint32_t {      // 1: stays for certain, 65536: equal
        const uint32_t at = first + i;
        if (i >= size) return 0;
        if (at < lo || at >= hi) return 1;
        if (!any) return 0;
        const uint32_t key = key_of(i);
        return key > prefix ? 1 : key == prefix ? 65536u : 0;
    };
    uint32_t total_above;
    block_prefix<THREADS>(above, warp_sums, total_above);
    const uint32_t total_sure = total_above + size - (free1 - free0), total_equal = any ? count[2][prefix & 1023] : 0;
    if (t == 0) {
        slice_counts[0] = total_sure;
        slice_counts[1] = total_equal;
    }
    sync();
    uint32_t base = 0, base_equal = 0;
    for (uint32_t x = 0; x < rank; ++x) {
        base += cluster.map_shared_rank(&slice_counts[0], x)[0];
        base_equal += cluster.map_shared_rank(&slice_counts[0], x)[1];
    }
    if (blocks > 1) cluster.sync();                // no block ends while another reads it
    constexpr uint32_t kRun = 4;                   // tokens of a thread, side by side
    for (uint32_t i0 = 0; i0 < size; i0 += kRun * THREADS) {
        uint32_t k[kRun], sum = 0, total;
#pragma unroll
        for (uint32_t u = 0; u < kRun; ++u) {
            k[u] = kind(i0 + t * kRun + u);
            sum += k[u];                           // (at most 4096 of each kind in the block)
        }
        const uint32_t before = block_prefix<THREADS>(sum, warp_sums, total);
        uint32_t to = base + (before & 0xffffu), eq = base_equal + (before >> 16);
#pragma unroll
        for (uint32_t u = 0; u < kRun; ++u) {
            const uint32_t i = first + i0 + t * kRun + u;
            if (k[u] == 1 || (k[u] && eq < need)) {
                kept[to + min(eq, need)] = i;
                new_mass[to + min(eq, need)] = mass[i];
            }
            to += k[u] & 1;
            eq += k[u] >> 16;
        }
        base += total & 0xffffu;
        base_equal += total >> 16;
    }
}

constexpr int kMoveThreads = 128;      // (256: 53 us for the 234 MB that four long contexts move, 128: 48, now 45)

// One CTA: one new block of one head, keys and values.  Bound by DRAM: 234 MB
// in 45 us (5.2 TB/s).
__global__ void __launch_bounds__(kMoveThreads) k_evict_move(const __grid_constant__ EvictArgs a) {
    __shared__ int64_t from[128];          // row of each token in the codes, -1: none
    __shared__ float scale[2][128];
    __shared__ float top[2];
    const bs_cache_evict_desc& d = a.d;
    const uint32_t col = blockIdx.x, h = blockIdx.y, b = blockIdx.z, t = threadIdx.x, block = a.c.block;
    const uint64_t row = static_cast<uint64_t>(b) * a.c.kv_heads + h;
    const uint32_t i0 = col * block;
    cudaGridDependencySynchronize();       // launched while the selection still runs; in every block
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
    for (uint32_t i = t; i < 2 * block; i += kMoveThreads) {       // scales become the ratios of the codes
        const uint32_t kv = i >= block, x = i - kv * block;
        scale[kv][x] = top[kv] > 0.f ? __fdiv_rn(scale[kv][x], top[kv]) : 0.f;
    }
    __syncthreads();
    const uint32_t per_row = a.c.dim / 16, units = block * per_row, by_row = reciprocal(per_row);
    constexpr int kBatch = 4;              // loads of a thread in flight
#pragma unroll
    for (uint32_t kv = 0; kv < 2; ++kv) {
        int8_t* const base = kv ? a.c.v : a.c.k;
        int8_t* const to = base + slab * block * a.c.dim;
        for (uint32_t u0 = t; u0 < units; u0 += kBatch * kMoveThreads) {
            uint4 codes[kBatch];
            float ratio[kBatch];
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                const uint32_t u = u0 + x * kMoveThreads, i = divided(u, by_row);
                codes[x] = make_uint4(0, 0, 0, 0);
                ratio[x] = 1.f;
                if (u < units && from[i] >= 0) {
                    codes[x] = ldg_stream(base + from[i] * a.c.dim + (u - i * per_row) * 16);
                    ratio[x] = scale[kv][i];
                }
            }
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                const uint32_t u = u0 + x * kMoveThreads;
                if (u >= units) break;
                if (ratio[x] != 1.f)
                    codes[x] = make_uint4(rescaled(codes[x].x, ratio[x]), rescaled(codes[x].y, ratio[x]), rescaled(codes[x].z, ratio[x]),
                                          rescaled(codes[x].w, ratio[x]));
                *reinterpret_cast<uint4*>(to + u * 16) = codes[x];
            }
        }
    }
}

template <int THREADS>
cudaError_t launch_select(const EvictArgs& a, uint32_t cluster, cudaStream_t stream) {
    const uint32_t slice = ((a.d.mass_width + cluster - 1) / cluster + 3) & ~3u, cached = slice < kMostCached ? slice : kMostCached;
    cudaError_t e = cudaFuncSetAttribute(k_evict_select<THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostCached * 4);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(a.c.kv_heads * cluster, a.d.num_seqs);
    config.blockDim = dim3(THREADS);
    config.dynamicSmemBytes = cached * 4;
    config.stream = stream;
    config.attrs = attr;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, k_evict_select<THREADS>, a, cached);
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
    const uint32_t rows = kReadThreads / (c.dim / 16);       // of a block
    const dim3 grid((d.count + rows - 1) / rows, c.kv_heads, d.num_seqs);
    if (d.dtype == BS_F32) return launch_after(k_cache_read<float>, grid, kReadThreads, 0, stream, a);
    if (d.dtype == BS_F16) return launch_after(k_cache_read<__half>, grid, kReadThreads, 0, stream, a);
    return launch_after(k_cache_read<__nv_bfloat16>, grid, kReadThreads, 0, stream, a);
}

size_t cache_evict_scratch(const bs_token_cache&, const bs_cache_evict_desc&, const MemoryDevice&) { return 0; }

cudaError_t launch_cache_evict(const bs_token_cache& c, const bs_cache_evict_desc& d, const MemoryDevice& dev,
                               cudaStream_t stream) {
    const EvictArgs a{c, d, dev.errors};
    // a row goes to more blocks while they would have over 4,096 tokens each
    // and the rows alone do not fill the GPU
    uint32_t cluster = 1;
    while (cluster < kMostCluster && d.mass_width / cluster > 4096 &&
           static_cast<uint64_t>(c.kv_heads) * d.num_seqs * cluster * 2 <= static_cast<uint64_t>(dev.num_sms))
        cluster *= 2;
    const cudaError_t e = d.mass_width <= 4096 ? launch_select<256>(a, cluster, stream) : launch_select<1024>(a, cluster, stream);
    if (e != cudaSuccess) return e;
    const uint32_t cols = (d.budget + c.block - 1) / c.block;
    const uint32_t used = cols < d.new_table_width ? cols : d.new_table_width;
    return used ? launch_after(k_evict_move, dim3(used, c.kv_heads, d.num_seqs), kMoveThreads, 0, stream, a) : cudaSuccess;
}

}  // namespace bsb
