// bs_select.cuh -- which elements of a row stay: the first, the last, and of
// the others those with the largest keys (ties: the lower place), in order.
// Shared by the eviction from the token cache (bs_token_cache.cu) and the
// choice of blocks (bs_block_choice.cu).
//
// A cluster of blocks has a slice of the row each.  The m-th largest key among
// the free elements is found by its digits of 11, 11 and 10 bits, counted by
// every block and added up through distributed shared memory; then each block
// numbers the elements of its slice that stay, in order, from what the blocks
// before it have.
#pragma once

#include <cooperative_groups.h>

#include "bs_device.cuh"

namespace bsb {
namespace select {

using namespace dev;
namespace cg = cooperative_groups;

constexpr uint32_t kBins = 2048;
constexpr uint32_t kMostCached = 46 * 1024;       // keys of a slice in shared memory
constexpr uint32_t kMostCluster = 8;

struct SelectShared {
    uint32_t count[3][kBins];
    uint32_t warp_sums[32];
    uint32_t slice_counts[2];      // elements that stay for certain, elements equal to the threshold
    uint32_t chosen[2];
};

// Order of floats as integers: the larger the larger; NaN above all.
__device__ __forceinline__ uint32_t select_key(float f) { return isnan(f) ? 0xffffffffu : f2ord(f); }

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

// The slice of a row of n elements that block `rank` of `blocks` has.
__device__ __forceinline__ void select_slice(uint32_t n, uint32_t blocks, uint32_t rank, uint32_t& first, uint32_t& size) {
    const uint32_t width = ((n + blocks - 1) / blocks + 3) & ~3u;
    first = min(rank * width, n);
    size = min(width, n - first);
}

template <int THREADS>
__device__ __forceinline__ void clear_counts(SelectShared& shared) {
#pragma unroll
    for (uint32_t i = threadIdx.x; i < 3 * kBins / 4; i += THREADS) reinterpret_cast<uint4*>(&shared.count[0][0])[i] = make_uint4(0, 0, 0, 0);
}

// Of n elements more than `budget`: keep(slot, place) for each that stays.
// key_of(i): key of the slice's element i.  All threads of the cluster call it,
// after clear_counts and a barrier.
template <int THREADS, typename KeyOf, typename Keep>
__device__ __forceinline__ void select_row(const cg::cluster_group& cluster, SelectShared& shared, uint32_t n, uint32_t first, uint32_t size,
                                           uint32_t sinks, uint32_t recent, uint32_t budget, KeyOf key_of, Keep keep) {
    const uint32_t rank = cluster.block_rank(), blocks = cluster.num_blocks(), t = threadIdx.x, lane = t & 31;
    const uint32_t lo = sinks, hi = n - recent;                  // free elements
    auto sync = [&]() {
        if (blocks > 1) cluster.sync();
        else __syncthreads();
    };
    uint32_t need = budget - sinks - recent;   // of the free elements; fewer than there are
    const bool any = need > 0;
    uint32_t prefix = 0;
    const uint32_t free0 = max(lo, first) - first, free1 = max(min(hi, first + size), first + free0) - first;   // of the slice
    uint32_t above = 0;                            // free elements of the slice above the threshold
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
                    // a warp whose elements all agree counts once: rows of equal weights do not queue up
                    const uint32_t lead = __shfl_sync(kFull, digit, 0);
                    if (__all_sync(kFull, in[u] && digit == lead)) {
                        if (lane == 0) atomicAdd(&shared.count[pass][digit], 32u);
                    } else if (in[u]) {
                        atomicAdd(&shared.count[pass][digit], 1u);
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
                const uint2* from = reinterpret_cast<const uint2*>(cluster.map_shared_rank(&shared.count[pass][0], x) + top_bin);
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
            uint32_t before = block_prefix<THREADS>(sum, shared.warp_sums, total);
#pragma unroll
            for (int u = 0; u < kEach; ++u) {
                if (before < need && need <= before + mine[u]) {
                    shared.chosen[0] = prefix | (kBins - 1 - (t * kEach + u)) << shift;
                    shared.chosen[1] = need - before;
                }
                before += mine[u];
            }
            __syncthreads();
            prefix = shared.chosen[0];
            need = shared.chosen[1];
            const uint32_t digit = (prefix >> shift) & mask;
#pragma unroll
            for (int u = 0; u < kEach; ++u)
                if (top_bin + u > digit) above += shared.count[pass][top_bin + u];
        }
    }
    // an element stays if it is not free, above the threshold, or one of the
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
    block_prefix<THREADS>(above, shared.warp_sums, total_above);
    const uint32_t total_sure = total_above + size - (free1 - free0), total_equal = any ? shared.count[2][prefix & 1023] : 0;
    if (t == 0) {
        shared.slice_counts[0] = total_sure;
        shared.slice_counts[1] = total_equal;
    }
    sync();
    uint32_t base = 0, base_equal = 0;
    for (uint32_t x = 0; x < rank; ++x) {
        base += cluster.map_shared_rank(&shared.slice_counts[0], x)[0];
        base_equal += cluster.map_shared_rank(&shared.slice_counts[0], x)[1];
    }
    if (blocks > 1) cluster.sync();                // no block ends while another reads it
    constexpr uint32_t kRun = 4;                   // elements of a thread, side by side
    for (uint32_t i0 = 0; i0 < size; i0 += kRun * THREADS) {
        uint32_t k[kRun], sum = 0, total;
#pragma unroll
        for (uint32_t u = 0; u < kRun; ++u) {
            k[u] = kind(i0 + t * kRun + u);
            sum += k[u];                           // (at most 4096 of each kind in the block)
        }
        const uint32_t before = block_prefix<THREADS>(sum, shared.warp_sums, total);
        uint32_t to = base + (before & 0xffffu), eq = base_equal + (before >> 16);
#pragma unroll
        for (uint32_t u = 0; u < kRun; ++u) {
            const uint32_t i = first + i0 + t * kRun + u;
            if (k[u] == 1 || (k[u] && eq < need)) keep(to + min(eq, need), i);
            to += k[u] & 1;
            eq += k[u] >> 16;
        }
        base += total & 0xffffu;
        base_equal += total >> 16;
    }
}

}  // namespace select
}  // namespace bsb
