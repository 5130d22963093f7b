// bs_shared.cuh -- how the work of attention over shared tokens is cut
// (bs_shared_attention.cu), and where its outputs wait for those over each
// sequence's own tokens (bs_block_attention.cu).
//
// A group's query rows of one key head (sequences x queries x heads) against
// its shared tokens are a segment for each pair of row tiles.  All segments, a
// group's heads side by side and a head's pairs, laid end to end, are cut into
// one share of equal cost per thread block.  A segment that one share has whole
// leaves its unnormalised outputs by row of the call's outputs, a piece of one
// in a slot of its share: 0 if it is the share's first piece, 1 if its last.
#pragma once

#include "bs_device.cuh"
#include "bs_memory.h"

namespace bsb {
namespace shared {

using namespace dev;

constexpr uint32_t kTileTokens = 128;
constexpr uint32_t kPairRows = 256;
// A piece costs its tiles and this many more: its queries, its first and last
// products, its outputs.
constexpr uint32_t kStart = 2;

// Where the outputs of a segment's rows are: by row of the outputs if there is
// one piece, else from slot `slot` of the share on (row `row` there).
struct FarRow {
    uint32_t pieces, share, slot, row;
};

struct SharedArgs {
    bs_token_cache c;
    bs_shared_attention_desc d;
    unsigned int* errors;
    FarRow* far;           // [rows of the outputs]: at a segment's first row, what the segment's rows have in common
    float* whole_o;        // [rows of the outputs][dim]
    float2* whole_ml;      // [rows of the outputs]: maximum (log2), sum
    float* part_o;         // [shares][2][256][dim]
    float2* part_ml;       // [shares][2][256]
    uint32_t group;        // query heads per key head
    uint32_t rows;         // of a sequence and key head
    uint32_t shares;       // thread blocks; 0: nothing is shared
    uint32_t block_log2;
    uint32_t polls;        // of a wait before it gives up (BSEARCH_WAIT_POLLS: a test sets 0)
};

struct Group {
    uint32_t first;        // sequence
    uint32_t rows, pairs;  // of a key head
    uint32_t tokens, tiles;
};

__device__ __forceinline__ Group group_of(const SharedArgs& a, uint32_t m) {
    Group g{};
    const int32_t first = a.d.cu[m], past = a.d.cu[m + 1];
    if (first < 0 || past <= first || static_cast<uint32_t>(past) > a.d.num_seqs) return g;
    g.first = first;
    int64_t tokens = a.d.shared_lens[m];
    const int64_t most = static_cast<int64_t>(a.d.shared_width) * a.c.block;
    if (tokens < 0 || tokens > most) {
        atomicOr(a.errors, kMemErrLength);
        tokens = tokens < 0 ? 0 : most;
    }
    if (tokens == 0) return g;
    g.rows = (past - first) * a.rows;
    g.pairs = (g.rows + kPairRows - 1) / kPairRows;
    g.tokens = static_cast<uint32_t>(tokens);
    g.tiles = (g.tokens + kTileTokens - 1) / kTileTokens;
    return g;
}

// Cost of a key head's part of a group, and of one segment.
__device__ __forceinline__ uint64_t cost_of(const Group& g) { return g.tiles ? static_cast<uint64_t>(g.pairs) * (g.tiles + kStart) : 0; }

__device__ __forceinline__ uint32_t used_shares(uint64_t w, uint32_t n) {
    const uint64_t most = (w + 2 * kStart - 1) / (2 * kStart);       // as many tiles as a piece costs besides
    return most < n ? static_cast<uint32_t>(most) : n;
}
__device__ __forceinline__ uint64_t share_first(uint64_t w, uint32_t n, uint32_t i) {
    return w / n * i + min(static_cast<uint64_t>(i), w % n);
}
// The share that holds unit x.
__device__ __forceinline__ uint32_t share_of(uint64_t w, uint32_t n, uint64_t x) {
    const uint64_t q = w / n, r = w % n, wide = r * (q + 1);
    return static_cast<uint32_t>(x < wide ? x / (q + 1) : r + (x - wide) / q);
}

// Cost of a key head's segments of all groups, for every thread of the block (a
// multiple of 32 threads).  sums: [warps].
__device__ __forceinline__ uint64_t count_cost(const SharedArgs& a, uint64_t* sums) {
    uint64_t total = 0;
    for (uint32_t i = threadIdx.x; i < a.d.num_groups; i += blockDim.x) total += cost_of(group_of(a, i));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(kFull, total, o);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = total;
    __syncthreads();
    total = 0;
    for (uint32_t i = 0; i < blockDim.x / 32; ++i) total += sums[i];
    __syncthreads();
    return total;
}

// Row of the outputs of a group's row r (of key head h).
__device__ __forceinline__ uint64_t output_row(const SharedArgs& a, const Group& g, uint32_t h, uint32_t r) {
    const uint32_t b = g.first + r / a.rows, i = r % a.rows / a.group, head = h * a.group + r % a.rows % a.group;
    return (static_cast<uint64_t>(b) * a.d.queries + i) * a.d.q_heads + head;
}

// Of sequence b's row r of key head h, b one of group g.
__device__ __forceinline__ FarRow far_row(const SharedArgs& a, const Group& g, uint32_t b, uint32_t h, uint32_t r) {
    const uint32_t in_group = (b - g.first) * a.rows + r;
    FarRow f = a.far[output_row(a, g, h, in_group / kPairRows * kPairRows)];
    f.row = in_group % kPairRows;
    // (anything may be there after a wait that gave up)
    if (f.share >= a.shares || f.pieces > a.shares - f.share || f.slot > 1) f.pieces = 0;
    return f;
}

}  // namespace shared

// Attention over the shared tokens alone, into whole_* and part_* (launched
// first), and over each sequence's own tokens, joined with it.
cudaError_t launch_shared_part(const shared::SharedArgs& a, cudaStream_t stream);

}  // namespace bsb
