// bs_block_choice.cu -- bounds of the token cache's key blocks, and which
// blocks a query attends to by them (include/bsearch.h, bs_block_bounds,
// bs_block_choice).
//
// For any key k of a block, of codes between `lower` and `upper` in every
// dimension, <q, k> <= k_scale * sum over d of max(q_d * upper_d, q_d * lower_d),
// which splits q into its positive and negative part: the sum is the product
// of (q+, q-) with (upper, lower).  So the query heads of a key head choose
// together at the cost of one: their parts add up before the product.  q counts
// in 127ths of its largest element, which makes every score an exact integer
// times the block's scale, the same in any order of summation.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "bs_device.cuh"
#include "bs_memory.h"
#include "bs_select.cuh"

namespace bsb {

using namespace dev;
using namespace select;

namespace {

// ------------------------------------------------------------------ bounds

struct BoundsArgs {
    bs_token_cache c;
    bs_block_bounds_desc d;
    unsigned int* errors;
    uint32_t cols;        // blocks of a sequence that may have changed, at most
};

constexpr int kBoundsWarps = 4;

// Larger and smaller of signed 16-bit halves whose upper bytes count; the
// lower bytes only decide between equal ones.
__device__ __forceinline__ void widen(uint32_t (&hi)[8], uint32_t (&lo)[8], uint4 x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t even = w[i] << 8;             // bytes 0 and 2 into the upper places
        hi[2 * i] = __vmaxs2(hi[2 * i], even);
        lo[2 * i] = __vmins2(lo[2 * i], even);
        hi[2 * i + 1] = __vmaxs2(hi[2 * i + 1], w[i]);
        lo[2 * i + 1] = __vmins2(lo[2 * i + 1], w[i]);
    }
}

// A warp: one block's keys of one head.  A lane has 16 dimensions of every
// (32 / per_row)-th token.  (2,287 blocks of 64 tokens, 8 heads of 128: 29 us, 5.4
// TB/s of the 155 MB that are read and written.)
__global__ void __launch_bounds__(32 * kBoundsWarps) k_block_bounds(const __grid_constant__ BoundsArgs a) {
    const bs_block_bounds_desc& d = a.d;
    const uint32_t hkv = a.c.kv_heads, block = a.c.block, per_row = a.c.dim / 16, lane = threadIdx.x & 31, b = blockIdx.y;
    const uint32_t unit = blockIdx.x * kBoundsWarps + (threadIdx.x >> 5), h = unit % hkv;
    cudaGridDependencySynchronize();       // in every block, before anything of the caller's
    int64_t len = d.lens[b];
    const int64_t most = static_cast<int64_t>(d.table_width) * block;
    if (len < 0 || len > most) {
        if (unit == 0 && lane == 0) atomicOr(a.errors, kMemErrLength);
        len = len < 0 ? 0 : most;
    }
    const int64_t from = d.last < 0 || d.last >= len ? 0 : (len - d.last) / block;
    const int64_t col = from + unit / hkv, left = len - col * block;      // tokens from the block's first on
    if (unit / hkv >= a.cols || left <= 0) return;
    const uint32_t id = d.table[static_cast<uint64_t>(b) * d.table_width + col];
    if (id >= a.c.num_blocks) {
        if (lane == 0) atomicOr(a.errors, kMemErrBlock);
        return;
    }
    const uint64_t slab = static_cast<uint64_t>(id) * hkv + h;
    const uint32_t rows = 32 / per_row, row = lane / per_row, tokens = left < block ? static_cast<uint32_t>(left) : block;
    uint32_t hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        hi[i] = 0x80008000u;
        lo[i] = 0x7fff7fffu;
    }
    if (row < rows) {
        const uint4* codes = reinterpret_cast<const uint4*>(a.c.k + slab * block * a.c.dim) + lane;
        constexpr uint32_t kBatch = 8;                 // loads on their way together
        for (uint32_t r0 = row; r0 < tokens; r0 += kBatch * rows) {
            uint4 x[kBatch];
#pragma unroll
            for (uint32_t u = 0; u < kBatch; ++u)      // (past the last token: this batch's first again)
                x[u] = __ldcs(codes + (r0 - row + (r0 + u * rows < tokens ? u * rows : 0)) * per_row);
#pragma unroll
            for (uint32_t u = 0; u < kBatch; ++u) widen(hi, lo, x[u]);
        }
    }
    for (uint32_t s = 16; s > 0; s >>= 1) {            // over the lanes of a chunk; rows of a lane past the others have none
        if (s >= rows) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t x = __shfl_down_sync(kFull, hi[i], s * per_row), y = __shfl_down_sync(kFull, lo[i], s * per_row);
            if (row + s < rows) {
                hi[i] = __vmaxs2(hi[i], x);
                lo[i] = __vmins2(lo[i], y);
            }
        }
    }
    if (row != 0) return;
    uint4 out[2];
    uint32_t* const w = reinterpret_cast<uint32_t*>(out);
#pragma unroll
    for (int i = 0; i < 4; ++i) {                      // the upper bytes, in order
        w[i] = __byte_perm(hi[2 * i], hi[2 * i + 1], 0x7351);
        w[4 + i] = __byte_perm(lo[2 * i], lo[2 * i + 1], 0x7351);
    }
    uint4* const to = reinterpret_cast<uint4*>(d.bounds + slab * 2 * a.c.dim) + lane;
    to[0] = out[0];
    to[per_row] = out[1];
}

// ------------------------------------------------------------------ choice

struct ChoiceArgs {
    bs_token_cache c;
    bs_block_choice_desc d;
    unsigned int* errors;
};

constexpr uint32_t kMostHeld = 8;      // scores of a thread where one block has a row

// Which of a row's n > count scores stay, by one block with kMostHeld of them in
// a thread's registers: the m-th largest of the free ones by its digits of 8 bits,
// then their places by prefix sums.  A row of 1,024 takes 2 us; the cluster's way
// (bs_select.cuh), with digits of 11 bits for longer rows, 6 and more (8 rows of
// 1,024 columns 24.6 us in all, against 8.8).
struct SmallShared {
    uint32_t count[4][256];
    uint32_t chosen[2];
};
template <int THREADS, typename Keep>
__device__ __forceinline__ void select_small(SmallShared& shared, uint32_t* warp_sums, const uint32_t* keys, uint32_t n, uint32_t sinks,
                                             uint32_t recent, uint32_t budget, Keep keep) {
    const uint32_t t = threadIdx.x, lane = t & 31, hi = n - recent;
    // places side by side: t * each and on
    const uint32_t each = (n + THREADS - 1) / THREADS;
    uint32_t key[kMostHeld];
#pragma unroll
    for (uint32_t u = 0; u < kMostHeld; ++u) key[u] = u < each && t * each + u < n ? keys[t * each + u] : 0;
    auto is_free = [&](uint32_t u) { return u < each && t * each + u >= sinks && t * each + u < hi; };
    for (uint32_t i = t; i < 4 * 256; i += THREADS) (&shared.count[0][0])[i] = 0;
    __syncthreads();
    uint32_t need = budget - sinks - recent, prefix = 0;
    const bool any = need > 0;
#pragma unroll 1
    for (int pass = 0; any && pass < 4; ++pass) {
        const int shift = 24 - 8 * pass;
#pragma unroll
        for (uint32_t u = 0; u < kMostHeld; ++u)
            if (is_free(u) && (pass == 0 || (key[u] ^ prefix) >> (shift + 8) == 0)) atomicAdd(&shared.count[pass][key[u] >> shift & 255], 1u);
        __syncthreads();
        if (t < 32) {                                  // eight bins to a lane, from the largest down
            uint32_t c[8], sum = 0;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                c[u] = shared.count[pass][255 - (lane * 8 + u)];
                sum += c[u];
            }
            uint32_t up_to = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(kFull, up_to, o);
                if (lane >= static_cast<uint32_t>(o)) up_to += up;
            }
            uint32_t before = up_to - sum;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                if (before < need && need <= before + c[u]) {
                    shared.chosen[0] = prefix | (255 - (lane * 8 + u)) << shift;
                    shared.chosen[1] = need - before;
                }
                before += c[u];
            }
        }
        __syncthreads();
        prefix = shared.chosen[0];
        need = shared.chosen[1];
    }
    // of those equal to the threshold the first `need`
    uint32_t kind[kMostHeld], sum = 0, total;          // 1: stays for certain, 65536: equal
#pragma unroll
    for (uint32_t u = 0; u < kMostHeld; ++u) {
        const uint32_t at = t * each + u;
        kind[u] = u >= each || at >= n ? 0 : !is_free(u) ? 1 : !any ? 0 : key[u] > prefix ? 1 : key[u] == prefix ? 65536u : 0;
        sum += kind[u];
    }
    const uint32_t before = block_prefix<THREADS>(sum, warp_sums, total);
    uint32_t to = before & 0xffffu, equal = before >> 16;
#pragma unroll
    for (uint32_t u = 0; u < kMostHeld; ++u) {
        if (kind[u] == 1 || (kind[u] && equal < need)) keep(to + min(equal, need), t * each + u);
        to += kind[u] & 1;
        equal += kind[u] >> 16;
    }
}

// A cluster of blocks has one row: a query and a key head.  Each block scores
// its slice of the table's columns, then the row's largest are found among the
// scores in shared memory.  SMALL: by the first block alone, for rows of at most
// kMostHeld columns a thread; the others leave their scores with it.
template <typename T, int THREADS, bool SMALL>
__global__ void __launch_bounds__(THREADS) k_block_choice(const __grid_constant__ ChoiceArgs a, uint32_t cached) {
    extern __shared__ uint32_t keys[];                     // [cached]: the columns' blocks, then their keys
    using Shared = std::conditional_t<SMALL, SmallShared, SelectShared>;
    __shared__ __align__(16) Shared shared;
    __shared__ __align__(16) int16_t parts[2][128];        // positive and negative part of the heads' codes
    __shared__ float warp_max[THREADS / 32];
    __shared__ uint32_t warp_sums[32];
    constexpr uint32_t kWarps = THREADS / 32;
    cudaGridDependencySynchronize();       // in every block, before anything of the caller's
    const cg::cluster_group cluster = cg::this_cluster();
    constexpr bool kAlone = SMALL && THREADS == 128;       // no cluster
    const uint32_t rank = kAlone ? 0 : cluster.block_rank(), blocks = kAlone ? 1 : cluster.num_blocks();
    const bs_block_choice_desc& d = a.d;
    const uint32_t hkv = a.c.kv_heads, group = d.q_heads / hkv, dim = a.c.dim, block = a.c.block;
    const uint32_t h = blockIdx.x / blocks, i = blockIdx.y, b = blockIdx.z, t = threadIdx.x, warp = t >> 5, lane = t & 31;
    // the heads' elements as codes, added up by sign (asked for with the length)
    const T* const q = static_cast<const T*>(d.q) + b * d.q_stride[0] + i * d.q_stride[1] + static_cast<int64_t>(h) * group * d.q_stride[2];
    constexpr uint32_t kHeads = 8;                         // of which a thread keeps the elements
    float x[kHeads];
#pragma unroll
    for (uint32_t g = 0; g < kHeads; ++g) x[g] = t < dim && g < group ? static_cast<float>(q[g * d.q_stride[2] + t]) : 0.f;
    int64_t len = d.lens[b];
    const int64_t most = static_cast<int64_t>(d.table_width) * block;
    if (len < 0 || len > most) {
        if (t == 0) atomicOr(a.errors, kMemErrLength);
        len = len < 0 ? 0 : most;
    }
    const int64_t seen = len - d.queries + 1 + i;
    const uint32_t n = seen > 0 ? static_cast<uint32_t>((seen + block - 1) / block) : 0, count = d.count;
    int32_t* const out = d.blocks + ((static_cast<uint64_t>(b) * d.queries + i) * hkv + h) * count;
    if (n <= count) {                                      // (the whole cluster)
        for (uint32_t y = rank * THREADS + t; y < count; y += blocks * THREADS) out[y] = y < n ? static_cast<int32_t>(y) : -1;
        return;
    }
    if (SMALL && !kAlone && blocks > 1) asm volatile("barrier.cluster.arrive.relaxed;\n" ::: "memory");     // this block has begun
    uint32_t first, size;
    select_slice(n, blocks, rank, first, size);
    const int32_t* const table = d.table + static_cast<uint64_t>(b) * d.table_width + first;
    const uint32_t held = min(size, cached);
    for (uint32_t col = t; col < held; col += THREADS) {
        const uint32_t id = table[col];
        if (id >= a.c.num_blocks) atomicOr(a.errors, kMemErrBlock);
        keys[col] = id < a.c.num_blocks ? id : kNoNode;
    }
    if constexpr (!SMALL) clear_counts<THREADS>(shared);
    float top = 0.f;
#pragma unroll
    for (uint32_t g = 0; g < kHeads; ++g) top = fmaxf(top, fabsf(x[g]));
    if (t < dim)
        for (uint32_t g = kHeads; g < group; ++g) top = fmaxf(top, fabsf(static_cast<float>(q[g * d.q_stride[2] + t])));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
    if (lane == 0) warp_max[warp] = top;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) top = fmaxf(top, warp_max[w]);
    const float by = top < 1e-30f ? 0.f : __fmul_rn(__frcp_rn(top), 127.f);
    if (t < dim) {
        int32_t positive = 0, negative = 0;
        auto add = [&](float y) {
            const int32_t c = __float2int_rn(__fmul_rn(y, by));
            positive += max(c, 0);
            negative += min(c, 0);
        };
#pragma unroll
        for (uint32_t g = 0; g < kHeads; ++g) add(x[g]);
        for (uint32_t g = kHeads; g < group; ++g) add(static_cast<float>(q[g * d.q_stride[2] + t]));
        parts[0][t] = static_cast<int16_t>(positive);      // (at most 128 heads of 127)
        parts[1][t] = static_cast<int16_t>(negative);
    }
    __syncthreads();

    // a column's 2 * dim bounds lie side by side: 16 to a lane
    const uint32_t per_col = dim / 8, cols = 32 / per_col, sub = lane / per_col, chunk = lane % per_col;
    int32_t weights[8] = {};
    if (sub < cols) {
#pragma unroll
        for (int y = 0; y < 8; ++y) weights[y] = reinterpret_cast<const int32_t*>(&parts[0][0] + (chunk * 16 < dim ? 0 : 128 - dim) + chunk * 16)[y];
    }
    auto product = [&](const uint4& y) {
        const int32_t w[4] = {static_cast<int32_t>(y.x), static_cast<int32_t>(y.y), static_cast<int32_t>(y.z), static_cast<int32_t>(y.w)};
        int32_t sum = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) sum = __dp2a_hi(weights[2 * u + 1], w[u], __dp2a_lo(weights[2 * u], w[u], sum));
        return sum;
    };
    auto key = [&](int32_t sum, float scale) { return select_key(__fmul_rn(__int2float_rn(sum), scale)); };
    uint32_t* scores = keys;                               // of this block's columns
    if (SMALL && !kAlone && blocks > 1) {
        asm volatile("barrier.cluster.wait;\n" ::: "memory");
        scores = cluster.map_shared_rank(keys, 0) + first;
    }
    // columns of a lane whose bounds are on their way together (128 rows of 1,024: 14.9 us
    // with 8, 15.7 with 4, 16.5 with 12; 1,024 threads have room for 4 alone)
    constexpr uint32_t kBatch = THREADS == 1024 ? 4 : 8;
    for (uint32_t x0 = warp * cols * kBatch; x0 < held; x0 += kWarps * cols * kBatch) {
        uint4 y[kBatch];
        float scale[kBatch];
#pragma unroll
        for (uint32_t u = 0; u < kBatch; ++u) {
            const uint32_t col = x0 + u * cols + sub, id = sub < cols && col < held ? keys[col] : kNoNode;
            const uint64_t slab = static_cast<uint64_t>(id) * hkv + h;
            y[u] = id != kNoNode ? __ldg(reinterpret_cast<const uint4*>(d.bounds + slab * 2 * dim) + chunk) : make_uint4(0, 0, 0, 0);
            scale[u] = id != kNoNode && chunk == 0 ? a.c.k_scale[slab] : 0.f;
        }
        __syncwarp();                                      // (the blocks are read: keys take their place)
#pragma unroll
        for (uint32_t u = 0; u < kBatch; ++u) {
            int32_t sum = product(y[u]);
#pragma unroll
            for (uint32_t s = 8; s > 0; s >>= 1) {
                const int32_t z = __shfl_down_sync(kFull, sum, s);
                if (chunk + s < per_col) sum += z;
            }
            const uint32_t col = x0 + u * cols + sub;
            if (chunk == 0 && sub < cols && col < held) scores[col] = key(sum, scale[u]);
        }
    }
    if (SMALL && !kAlone && blocks > 1) {
        cluster.sync();
        if (rank != 0) return;
    } else {
        __syncthreads();
    }
    auto keep = [&](uint32_t slot, uint32_t col) { out[slot] = col; };
    if constexpr (SMALL) {
        select_small<THREADS>(shared, warp_sums, keys, n, d.sinks, d.recent, count, keep);
    } else {
        select_row<THREADS>(
            cluster, shared, n, first, size, d.sinks, d.recent, count,
            [&](uint32_t col) -> uint32_t {
                if (col < cached) return keys[col];
                // a row too long for shared memory: scored again, by one thread
                const uint32_t id = table[col];
                if (id >= a.c.num_blocks) {
                    atomicOr(a.errors, kMemErrBlock);
                    return key(0, 0.f);
                }
                const uint64_t slab = static_cast<uint64_t>(id) * hkv + h;
                int32_t sum = 0;
                for (uint32_t y = 0; y < 2 * dim; ++y) sum += parts[y >= dim][y < dim ? y : y - dim] * d.bounds[slab * 2 * dim + y];
                return key(sum, a.c.k_scale[slab]);
            },
            keep);
    }
}

template <typename T, int THREADS, bool SMALL>
cudaError_t launch_choice(const ChoiceArgs& a, uint32_t cluster, cudaStream_t stream) {
    const uint32_t slice = ((a.d.table_width + (SMALL ? 0 : cluster - 1)) / (SMALL ? 1 : cluster) + 3) & ~3u, cached = slice < kMostCached ? slice : kMostCached;
    cudaError_t e = cudaFuncSetAttribute(k_block_choice<T, THREADS, SMALL>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostCached * 4);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(a.c.kv_heads * cluster, a.d.queries, a.d.num_seqs);
    config.blockDim = dim3(THREADS);
    config.dynamicSmemBytes = cached * 4;
    config.stream = stream;
    config.attrs = attr;
    config.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&config, k_block_choice<T, THREADS, SMALL>, a, cached);
}

template <typename T>
cudaError_t launch_choice(const bs_token_cache& c, const bs_block_choice_desc& d, const MemoryDevice& dev, cudaStream_t stream) {
    const ChoiceArgs a{c, d, dev.errors};
    const uint64_t rows = static_cast<uint64_t>(c.kv_heads) * d.queries * d.num_seqs;
    // Rows that one block's registers hold: more blocks score them while they would have
    // over 256 columns each and all are resident at once, one to an SM (clusters of 8
    // fit only half of the SMs, as they must not cross a group of SMs).  8 rows of
    // 1,024 columns take 8.8 us by 4 blocks and 14.2 by one; 16 rows 9.2 by 4, 13.6 by
    // 8; 64 rows 11.2 by 2, 14.4 by one and 17.7 by 4; 128 rows 14.6 by one, 21.6 by 2.
    // Small blocks are for many short rows (256 rows of 200 columns 11.2 against
    // 15.6 us, 96 rows 10.6 against 8.5) and for rows that they read at once (8 rows
    // of 40 columns 6.1 against 7.9).
    const uint64_t sms = dev.num_sms;
    if (d.table_width <= 64 || (d.table_width <= 256 && rows > sms)) return launch_choice<T, 128, true>(a, 1, stream);
    uint32_t cluster = 1;
    if (d.table_width <= 1024 * kMostHeld) {
        while (cluster < kMostCluster && d.table_width / cluster > 256 && rows * cluster * (cluster < 4 ? 2 : 4) <= sms) cluster *= 2;
        // (64 registers a thread with 1,024 of them: 8 rows of 1,024 columns 12.4 us)
        return d.table_width <= 512 * kMostHeld ? launch_choice<T, 512, true>(a, cluster, stream) : launch_choice<T, 1024, true>(a, cluster, stream);
    }
    // longer rows: counted by all blocks of a cluster (8 rows of 6,000 columns would take
    // 59 us, against 15)
    while (cluster < kMostCluster && d.table_width / cluster > 256 && rows * cluster * 2 <= 2u * dev.num_sms) cluster *= 2;
    return launch_choice<T, 256, false>(a, cluster, stream);
}

}  // namespace

cudaError_t launch_block_bounds(const bs_token_cache& c, const bs_block_bounds_desc& d, const MemoryDevice& dev, cudaStream_t stream) {
    BoundsArgs a{c, d, dev.errors};
    a.cols = bounds_columns(c, d);
    const uint64_t blocks = (static_cast<uint64_t>(a.cols) * c.kv_heads + kBoundsWarps - 1) / kBoundsWarps;
    return launch_after(k_block_bounds, dim3(static_cast<unsigned>(blocks), d.num_seqs), 32 * kBoundsWarps, 0, stream, a);
}

cudaError_t launch_block_choice(const bs_token_cache& c, const bs_block_choice_desc& d, const MemoryDevice& dev, cudaStream_t stream) {
    return d.dtype == BS_F16 ? launch_choice<__half>(c, d, dev, stream) : launch_choice<__nv_bfloat16>(c, d, dev, stream);
}

}  // namespace bsb
