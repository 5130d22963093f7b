// bs_block_attention.cu -- attention over chosen blocks of the 8-bit token
// cache, and the joint attention over shared and own tokens
// (include/bsearch.h, bs_block_attention, bs_shared_attention).
//
// The products, their layout and their roundings are those of
// bs_cache_attention.cu (bs_cache_tile.cuh).  What differs is where a tile's
// tokens come from: a list of table columns for each query and key head.  A
// cluster of blocks takes a segment (a query and a key head), a part of its
// list each; the list's entries are looked up in the table once, into shared
// memory (one without a visible token gets a position past all of them), so that
// the copies of tiles wait for no chain of loads.  The blocks of a cluster join
// their outputs through distributed shared memory: no second kernel, no workspace.
// 128 segments of 4,096 tokens (134 MB of codes) take 31 us, 4.3 TB/s, where the
// bytes alone are 20: three blocks to an SM, each with two tiles a warp on their way,
// and their ends; 128 of 2,048 whose tokens four have in common 17.5 us, most of
// it the 67 MB that they copy from the second-level cache.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "bs_cache_tile.cuh"
#include "bs_device.cuh"
#include "bs_memory.h"
#include "bs_shared.cuh"

namespace bsb {

using namespace dev;
using namespace tile;
using shared::FarRow;
using shared::Group;
using shared::SharedArgs;
namespace cg = cooperative_groups;

namespace {

constexpr uint32_t kMostIds = 256;     // entries looked up at a time
constexpr int32_t kHidden = 0x40000000;     // a position past all that are seen
constexpr int32_t kShared = -0x40000000;    // and where those of shared tokens begin
constexpr uint32_t kMostCluster = 8;
constexpr uint32_t kBatch = 8;          // pieces of the shared tokens' outputs on their way together
template <int NT>
constexpr int kStagesOf = NT == 1 ? 2 : 3;
constexpr int blocks_per_sm(int nt) { return nt == 1 ? 3 : 2; }

struct RowsArgs {
    SharedArgs s;                      // of a list of blocks: what both have
    const int32_t* blocks;             // [num_seqs][queries][kv_heads][count]
    uint32_t count;
    uint32_t rows;                     // of a segment
    uint32_t direct;                   // 1: the shared tokens are this kernel's too
};

template <int NW>
constexpr int kListStage = kStageBytes<NW> + 16;               // and the halves' first positions
constexpr int kIdBytes = kMostIds * 8;
// (the entries lie where the outputs are joined later: with 16 query rows two blocks just fit an SM)
template <int NW, int NT>
constexpr int kJoinOrIds = kJoinBytes<NW, NT> > kIdBytes ? kJoinBytes<NW, NT> : kIdBytes;
template <int NW, int NT>
constexpr size_t kRowsSmem = kWarps * kStagesOf<NT> * kListStage<NW> + (kWarps + 1) * 8 * NT * 2 * 4 + kJoinOrIds<NW, NT>;

__device__ __forceinline__ uint32_t tokens_of(const SharedArgs& a, const int32_t* lens, uint32_t i, uint32_t width) {
    const int32_t len = lens[i];
    const int64_t most = static_cast<int64_t>(width) * a.c.block;
    if (len >= 0 && len <= most) return len;
    atomicOr(a.errors, kMemErrLength);
    return len < 0 ? 0 : static_cast<uint32_t>(most);
}

template <int NW, int NT, bool LIST>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(NT)) k_rows(const __grid_constant__ RowsArgs given) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int kDim = NW * 16, kRows = 8 * NT, kStages = kStagesOf<NT>;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    unsigned char* const ring = smem + warp * kStages * kListStage<NW>;
    float* const join_ml = reinterpret_cast<float*>(smem + kWarps * kStages * kListStage<NW>);     // [warps + 1][kRows][2]
    float* const join_o = join_ml + (kWarps + 1) * kRows * 2;
    int2* const ids = reinterpret_cast<int2*>(join_o);          // block, first position; till the outputs are joined

    const SharedArgs& a = given.s;
    // In every block, before anything of the caller's.  (After the shared tokens' kernel
    // too: what the kernels before that one wrote is promised to this one by its own wait
    // alone.  Begun before it, its own tokens hid under that kernel's end.)
    cudaGridDependencySynchronize();
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank(), parts = cluster.num_blocks();
    const bs_shared_attention_desc& d = a.d;
    const uint32_t hkv = a.c.kv_heads, b = blockIdx.z, segment = blockIdx.x / parts, row0 = blockIdx.y * kRows;
    const uint32_t h = LIST ? segment % hkv : segment, query = LIST ? segment / hkv : 0, block = a.c.block;
    // what is known from the start is asked for at once: the queries, as columns of
    // K Q^T (column j is row row0 + j), the list's first entries, the length
    uint32_t q[NT][NW][2];
    float row_scale[NT][2];          // of columns 2c and 2c + 1
    int32_t limit[NT][2];            // tokens of its own that row sees
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const uint32_t r = row0 + 8 * nt + g;
        const uint16_t* row = static_cast<const uint16_t*>(d.q) + b * d.q_stride[0] + static_cast<int64_t>(LIST ? query : r / a.group) * d.q_stride[1] +
                              (static_cast<int64_t>(h) * a.group + r % a.group) * d.q_stride[2] + c * (NW * 4);
        fetch_query_row<NW>(q[nt], row, r < given.rows);
    }
    const int32_t* const list = given.blocks + ((static_cast<uint64_t>(b) * d.queries + query) * hkv + h) * given.count;
    int32_t ahead[kMostIds / kThreads];
    if (LIST) {
        const uint32_t from = static_cast<uint32_t>(static_cast<uint64_t>(given.count) * rank / parts) + threadIdx.x;
#pragma unroll
        for (uint32_t i = 0; i < kMostIds / kThreads; ++i) ahead[i] = from + i * kThreads < given.count ? list[from + i * kThreads] : -1;
    }
    const uint32_t len = tokens_of(a, d.lens, b, d.table_width);
    auto scale_queries = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            scale_query_row<NW>(q[nt], row_scale[nt], d.dtype != BS_F16, d.scale * 1.4426950408889634f, c);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                limit[nt][i] = static_cast<int32_t>(len) - d.queries + 1 + static_cast<int32_t>(LIST ? query : (row0 + 8 * nt + 2 * c + i) / a.group);
                if (!LIST) limit[nt][i] = max(limit[nt][i], 0);       // (below 0 are the shared tokens, which it sees)
            }
        }
    };
    Group group{};                   // what the sequence shares (none: no tokens)
    uint32_t m = 0;
    auto find_group = [&]() {
        for (uint32_t past = d.num_groups; past - m > 1;) {    // the last group that begins at b or before
            const uint32_t mid = (m + past) / 2;
            (d.cu[mid] <= static_cast<int32_t>(b) ? m : past) = mid;
        }
        group = shared::group_of(a, m);
        if (b < group.first || static_cast<int32_t>(b) >= d.cu[m + 1]) group = Group{};
    };
    float o[NT][NW][4];
    float top[NT][2], sum[NT][2], unit = kFold / -kNoScore, inv_unit = -kNoScore;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        top[nt][0] = top[nt][1] = kNoScore;
        sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
        for (int j = 0; j < NW; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
    }

    // the entries: the list's, or every block of what it shares, where that is done
    // here, and of its own.  Positions of shared tokens count from kShared.
    if (!LIST && given.direct) find_group();
    const uint32_t shared_entries = !LIST && given.direct ? (group.tokens + block - 1) / block : 0;
    const int32_t* const table = d.table + static_cast<uint64_t>(b) * d.table_width;
    const int32_t most = static_cast<int32_t>(len) - (LIST ? d.queries - 1 - static_cast<int32_t>(query) : 0);
    const uint32_t width = d.table_width, tokens = most > 0 ? most : 0;           // some row sees the tokens below
    const uint32_t entries = LIST ? given.count : shared_entries + (tokens + block - 1) / block;
    // this block's part of the entries
    const uint32_t end = static_cast<uint32_t>(static_cast<uint64_t>(entries) * (rank + 1) / parts);
    const uint32_t begin = static_cast<uint32_t>(static_cast<uint64_t>(entries) * rank / parts);
    for (uint32_t from = begin; from < end; from += kMostIds) {
        // look them up; one without a token that is seen begins past all of them
        const uint32_t held = min(end - from, kMostIds);
#pragma unroll
        for (uint32_t i = 0; i < kMostIds / kThreads; ++i) {
            const uint32_t e = threadIdx.x + i * kThreads;
            if (e >= held) break;
            int2 entry = make_int2(0, kHidden);
            if (!LIST && from + e < shared_entries) {
                const uint32_t id = d.shared_table[static_cast<uint64_t>(m) * d.shared_width + from + e];
                if (id < a.c.num_blocks) entry = make_int2(id, kShared + static_cast<int32_t>((from + e) * block));
                else atomicOr(a.errors, kMemErrBlock);
                ids[e] = entry;
                continue;
            }
            const int32_t col = !LIST ? static_cast<int32_t>(from + e - shared_entries) : from == begin ? ahead[i] : list[from + e];
            if (col >= 0 && static_cast<uint32_t>(col) < width && static_cast<int64_t>(col) * block < tokens) {
                const uint32_t id = table[col];
                if (id < a.c.num_blocks) entry = make_int2(id, static_cast<int32_t>(col * block));
                else atomicOr(a.errors, kMemErrBlock);
            } else if (LIST && col >= 0 && static_cast<uint32_t>(col) >= width) {
                atomicOr(a.errors, kMemErrLength);
            }
            ids[e] = entry;
        }
        __syncthreads();
        const uint32_t tiles = ((held << a.block_log2) + kTile - 1) / kTile;
        auto request = [&](uint32_t t, uint32_t stage) {
            if (t < tiles) {
                unsigned char* s = ring + stage * kListStage<NW>;
                float* scales = reinterpret_cast<float*>(s + 2 * kTile * kPitch<NW>);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t at = t * kTile + 16 * half, e = at >> a.block_log2, in = at & (block - 1);
                    const int2 entry = e < held ? ids[e] : make_int2(0, kHidden);
                    const int32_t pos = entry.y + static_cast<int32_t>(in);
                    const int32_t left = (pos < 0 ? kShared + static_cast<int32_t>(group.tokens) : static_cast<int32_t>(tokens)) - pos;
                    if (left > 0) {
                        const uint64_t slab = static_cast<uint64_t>(static_cast<uint32_t>(entry.x)) * hkv + h;
                        const uint64_t row = ((slab << a.block_log2) + in) * kDim + lane * 16;
                        const int8_t* k = a.c.k + row;
                        const int8_t* v = a.c.v + row;
#pragma unroll
                        for (int j = 0; j < (NW + 1) / 2; ++j) {
                            const uint32_t i = lane + 32 * j, r = i / NW + 16 * half, x = i % NW;
                            if (NW % 2 && i >= 16 * NW) break;
                            copy16(s + r * kPitch<NW> + unit_at<NW>(x, r), k + j * 512);
                            copy16(s + (kTile + r) * kPitch<NW> + unit_at<NW>(x, r), v + j * 512);
                        }
                        if (lane < 2) copy4(scales + 2 * half + lane, (lane ? a.c.v_scale : a.c.k_scale) + slab);
                    } else if (lane == 0) {       // no tokens to see: a value scale below zero says so
                        scales[2 * half] = 0.f;
                        scales[2 * half + 1] = -1.f;
                    }
                    if (lane == 2) *reinterpret_cast<int2*>(scales + 4 + 2 * half) = make_int2(pos, left);
                }
            }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < kStages; ++i) request(warp + i * kWarps, i);
        if (from == begin) {                           // (under the first copies)
            scale_queries();
            if (!LIST && a.shares) find_group();
        }
        uint32_t stage = 0;
        for (uint32_t t = warp; t < tiles; t += kWarps) {
            asm volatile("cp.async.wait_group %0;\n" ::"n"(kStages - 1) : "memory");
            __syncwarp();
            const unsigned char* s = ring + stage * kListStage<NW>;
            const float4 sc = *reinterpret_cast<const float4*>(s + 2 * kTile * kPitch<NW>);
            const int4 first = *reinterpret_cast<const int4*>(s + 2 * kTile * kPitch<NW> + 16);
            const float k_scale[2] = {sc.x, sc.z}, v_scale[2] = {sc.y, sc.w};
            const int32_t pos[2] = {first.x, first.z}, left[2] = {first.y, first.w};
            if (fmaxf(v_scale[0], v_scale[1]) < 0.f) {      // none to see
                __syncwarp();
                request(t + kStages * kWarps, stage);
                stage = stage + 1 == kStages ? 0 : stage + 1;
                continue;
            }
            float z[2][NT][4];           // [half]: tokens g and g + 8 (+ 16 half), columns 2c and 2c + 1
            tile_scores<NW, NT>(z, s, q, g, c);
            const bool edge = min(left[0], left[1]) < 16 || (!LIST && max(pos[0], pos[1]) + 16 > static_cast<int32_t>(tokens) - d.queries + 1);
            bool move = fmaxf(v_scale[0], v_scale[1]) > 4.f * unit;
            const float room[2] = {kSlack - scale_log2(v_scale[0], inv_unit), kSlack - scale_log2(v_scale[1], inv_unit)};
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        z[half][nt][i] *= row_scale[nt][i & 1] * k_scale[half];
                        const int32_t in = static_cast<int32_t>(g) + (i & 2) * 4;
                        if (edge && (in >= left[half] || pos[half] + in >= limit[nt][i & 1])) z[half][nt][i] = -INFINITY;
                        move |= z[half][nt][i] > top[nt][i & 1] + room[half];
                    }
            if (__any_sync(kFull, move)) move_maxima<NW, NT>(z, v_scale, top, sum, o, unit, inv_unit);
            tile_values<NW, NT>(z, s, v_scale, inv_unit, top, sum, o, g, c);
            __syncwarp();
            request(t + kStages * kWarps, stage);          // where this tile was
            stage = stage + 1 == kStages ? 0 : stage + 1;
        }
        __syncthreads();               // `ids` is done with
    }

    if (!LIST && a.shares && begin == end) find_group();
    FarRow far{};                    // a thread below kRows: where that row's outputs over the shared tokens are
    if (!LIST && a.shares && group.tiles && threadIdx.x < kRows && row0 + threadIdx.x < given.rows)
        far = shared::far_row(a, group, b, h, row0 + threadIdx.x);
    float all_top[NT][2], all_sum[NT][2];
    join_warps<NW, NT>(o, top, sum, unit, all_top, all_sum, join_o, join_ml, warp, lane);
    auto row_at = [&](uint32_t r) {        // row of the outputs
        const uint32_t i = LIST ? query : r / a.group;
        return (static_cast<uint64_t>(b) * d.queries + i) * d.q_heads + h * a.group + (LIST ? r : r - i * a.group);
    };
    if (LIST && parts == 1) {
        if (warp != 0) return;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t r = row0 + 8 * nt + 2 * c + i;
                if (r >= given.rows) continue;
                const float l = all_sum[nt][i], inv = l == 0.f ? 0.f : 1.f / l;
                const uint64_t row = row_at(r);
                if (g == 0 && d.lse) d.lse[row] = l == 0.f ? -INFINITY : (all_top[nt][i] + log2f(l)) * 0.6931471805599453f;
#pragma unroll
                for (int j = 0; j < NW; ++j) {
                    const float x = o[nt][j][i] * inv, y = o[nt][j][2 + i] * inv;
                    const uint64_t e = row * kDim + value_dim<NW>(j, g);
                    if (d.dtype == BS_F16) *reinterpret_cast<__half2*>(static_cast<__half*>(d.out) + e) = __floats2half2_rn(x, y);
                    else *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(d.out) + e) = __floats2bfloat162_rn(x, y);
                }
            }
        return;
    }
    // the cluster's outputs as one, and those over the shared tokens: a thread
    // has four dimensions of a row
    float* const part_o = join_o + kRows * kDim;               // (read by warp 1 alone, a barrier ago)
    float* const part_ml = join_ml + kWarps * kRows * 2;
    if (warp == 0)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t r = 8 * nt + 2 * c + i;
                if (g == 0) *reinterpret_cast<float2*>(part_ml + r * 2) = make_float2(all_top[nt][i], all_sum[nt][i]);
#pragma unroll
                for (int j = 0; j < NW; ++j)
                    *reinterpret_cast<float2*>(part_o + r * kDim + value_dim<NW>(j, g)) = make_float2(o[nt][j][i], o[nt][j][2 + i]);
            }
    FarRow* const far_rows = reinterpret_cast<FarRow*>(smem);  // (over the ring)
    if (!LIST && threadIdx.x < kRows) far_rows[threadIdx.x] = far;
    if (!LIST && blockIdx.x == 0 && blockIdx.y == 0 && b == 0)
        for (uint32_t i = threadIdx.x; i <= d.num_groups; i += kThreads) {
            const int32_t x = d.cu[i];
            if (i == 0 ? x != 0 : x < d.cu[i - 1] || (i == d.num_groups && static_cast<uint32_t>(x) != d.num_seqs))
                atomicOr(a.errors, kMemErrLength);
            // (groups without sequences and tables without columns are looked up nowhere else)
            if (i < d.num_groups) tokens_of(a, d.shared_lens, i, d.shared_width);
        }
    if (parts > 1) cluster.sync();
    else __syncthreads();
    for (uint32_t x = rank * kThreads + threadIdx.x; x < kRows * kDim / 4; x += parts * kThreads) {
        const uint32_t r = x / (kDim / 4), at = x % (kDim / 4) * 4;
        if (row0 + r >= given.rows) break;
        float2 ml[kMostCluster];
        float m = kNoScore, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (uint32_t p = 0; p < kMostCluster; ++p) {
            ml[p] = p < parts ? *reinterpret_cast<const float2*>(cluster.map_shared_rank(part_ml, p) + r * 2) : make_float2(kNoScore, 0.f);
            m = fmaxf(m, ml[p].x);
        }
#pragma unroll
        for (uint32_t p = 0; p < kMostCluster; ++p) {
            if (p >= parts) break;
            const float4 y = *reinterpret_cast<const float4*>(cluster.map_shared_rank(part_o, p) + r * kDim + at);
            const float w = exp2_fast(ml[p].x - m);
            l += ml[p].y * w;
            acc.x += y.x * w, acc.y += y.y * w, acc.z += y.z * w, acc.w += y.w * w;
        }
        const uint64_t row = row_at(row0 + r);
        const FarRow at_far = LIST ? FarRow{} : far_rows[r];
        for (uint32_t p0 = 0; p0 < at_far.pieces; p0 += kBatch) {
            float2 far_ml[kBatch];
            float4 y[kBatch];
            float high = m;
#pragma unroll
            for (uint32_t u = 0; u < kBatch; ++u) {
                const uint32_t p = min(p0 + u, at_far.pieces - 1);
                const uint64_t slot = ((static_cast<uint64_t>(at_far.share) + p) * 2 + (p == 0 ? at_far.slot : 0)) * shared::kPairRows + at_far.row;
                far_ml[u] = at_far.pieces == 1 ? a.whole_ml[row] : a.part_ml[slot];
                y[u] = *reinterpret_cast<const float4*>(at_far.pieces == 1 ? a.whole_o + row * kDim + at : a.part_o + slot * kDim + at);
                if (p0 + u >= at_far.pieces) far_ml[u] = make_float2(kNoScore, 0.f);
                high = fmaxf(high, far_ml[u].x);
            }
            const float shrink = exp2_fast(m - high);
            m = high;
            l *= shrink;
            acc.x *= shrink, acc.y *= shrink, acc.z *= shrink, acc.w *= shrink;
#pragma unroll
            for (uint32_t u = 0; u < kBatch; ++u) {
                if (p0 + u >= at_far.pieces) break;
                const float w = exp2_fast(far_ml[u].x - m);
                l += far_ml[u].y * w;
                acc.x += y[u].x * w, acc.y += y[u].y * w, acc.z += y[u].z * w, acc.w += y[u].w * w;
            }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (at == 0 && d.lse) d.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        uint2 u;
        if (d.dtype == BS_F16) {
            const __half2 lo = __floats2half2_rn(acc.x * inv, acc.y * inv), hi = __floats2half2_rn(acc.z * inv, acc.w * inv);
            u = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        } else {
            const __nv_bfloat162 lo = __floats2bfloat162_rn(acc.x * inv, acc.y * inv), hi = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
            u = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        }
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(d.out) + row * kDim + at) = u;
    }
    if (parts > 1) cluster.sync();         // no block ends while another reads it
}

// Blocks of a segment, by the time that they were measured to take, in us: a block
// with one, two or three to an SM 3.7, 4.9 or 6.0 to begin and end and 0.29, 0.38 or
// 0.47 for a tile of 32 tokens, a cluster of n 0.8 + n / 10 more.  Lists are as long
// as one another, so the blocks go in waves.  Sequences are taken to have half the
// tokens that their table has room for, those with all of them in the last wave.
// (64 segments of 4 blocks of 64 tokens: 6.3 us by 2, 14.0 by 8; 8 segments of 64:
// 39.9 by 1, 10.3 by 8; 128 of 2,000 own tokens: 23.7 by 1, 19.1 by 2, 24.2 by 4.)
// `shared` and `own`: tiles of a segment.
uint32_t parts_of(uint64_t segments, double shared, double own, uint32_t num_sms, uint32_t per_sm, bool lists, double& time) {
    uint32_t best = 1;
    for (uint32_t n = 1; n <= kMostCluster; ++n) {
        const uint64_t blocks = segments * n, resident = static_cast<uint64_t>(num_sms) * per_sm;
        auto wave = [&](uint64_t on_sm, double tiles) {
            return 3.7 + 1.15 * (on_sm - 1) + (n > 1 ? 0.8 + 0.1 * n : 0.) + (0.285 + 0.09 * (on_sm - 1)) * tiles / n;
        };
        const uint64_t rest = blocks % resident;
        const double t = blocks / resident * wave(per_sm, shared + (lists ? own : own / 2)) +
                         (rest ? wave((rest + num_sms - 1) / num_sms, shared + own) : 0.);
        if (n == 1 || t < time) {
            time = t;
            best = n;
        }
    }
    return best;
}

double tiles_of(const bs_token_cache& c, uint64_t blocks) { return static_cast<double>(blocks * c.block) / kTile; }

// The segments of attention over own tokens, as many as row tiles of key heads.
uint64_t own_segments(const bs_token_cache& c, const bs_shared_attention_desc& d, uint32_t rows) {
    const uint32_t tile = rows <= 8 ? 8 : 16;
    return static_cast<uint64_t>(c.kv_heads) * d.num_seqs * ((rows + tile - 1) / tile);
}

template <int NW, int NT, bool LIST>
cudaError_t launch_rows(const RowsArgs& a, const MemoryDevice& dev, cudaStream_t stream) {
    const cudaError_t e = cudaFuncSetAttribute(k_rows<NW, NT, LIST>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem<NW, NT>);
    if (e != cudaSuccess) return e;
    const uint32_t row_tiles = (a.rows + 8 * NT - 1) / (8 * NT);
    const uint64_t segments = static_cast<uint64_t>(a.s.c.kv_heads) * (LIST ? a.s.d.queries : 1);
    double time = 0;
    const uint32_t parts = parts_of(segments * row_tiles * a.s.d.num_seqs, a.direct ? tiles_of(a.s.c, a.s.d.shared_width) : 0.,
                                    tiles_of(a.s.c, LIST ? a.count : a.s.d.table_width), dev.num_sms, blocks_per_sm(NT), LIST, time);
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(segments * parts), row_tiles, a.s.d.num_seqs);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = kRowsSmem<NW, NT>;
    config.stream = stream;
    config.attrs = attr;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, k_rows<NW, NT, LIST>, a);
}

template <int NT, bool LIST>
cudaError_t launch_rows(const RowsArgs& a, const MemoryDevice& dev, cudaStream_t stream) {
    switch (a.s.c.dim / 16) {
        case 1: return launch_rows<1, NT, LIST>(a, dev, stream);
        case 2: return launch_rows<2, NT, LIST>(a, dev, stream);
        case 3: return launch_rows<3, NT, LIST>(a, dev, stream);
        case 4: return launch_rows<4, NT, LIST>(a, dev, stream);
        case 5: return launch_rows<5, NT, LIST>(a, dev, stream);
        case 6: return launch_rows<6, NT, LIST>(a, dev, stream);
        case 7: return launch_rows<7, NT, LIST>(a, dev, stream);
        default: return launch_rows<8, NT, LIST>(a, dev, stream);
    }
}

uint32_t log2_of(int32_t block) { return block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7; }

struct Layout {
    uint32_t shares;
    size_t far, whole_ml, whole_o, part_ml, part_o, total;
};

Layout plan(const bs_token_cache& c, const bs_shared_attention_desc& d, const MemoryDevice& dev) {
    Layout l{};
    // Few shared tokens or few sequences: each sequence reads them by itself, in
    // the kernel for its own.  The times of both ways, in us: the other one takes
    // 14 for its start, its end and the join, and 2.6 for 256 rows over 128 tokens.
    // (Of 32 query and 8 key heads of 128: 8 sequences over 1,000 tokens 11 us this
    // way and 27 that way; 64 over 1,000 38 and 39; 128 over 4,000 173 and 52.  Of 64
    // dimensions 9 and 23, 31 and 33, 132 and 43.  Each with 200 tokens of its own.
    // The constants are those of 128 dimensions, and the table's width stands for
    // the tokens; over 175 combinations of 32, 64 and 128 dimensions, 2 and 8 key heads,
    // 4 to 256 sequences and 256 to 16,000 tokens in tables of their width the way
    // taken was the slower one by more than 10% in three, 14% at most.)
    const uint32_t in_sequence = static_cast<uint32_t>(d.q_heads / c.kv_heads) * d.queries;
    const uint64_t segments = own_segments(c, d, in_sequence);
    const uint32_t per_sm = blocks_per_sm(in_sequence <= 8 ? 1 : 2);
    const double own = tiles_of(c, d.table_width);
    double here = 0, there = 0;
    parts_of(segments, tiles_of(c, d.shared_width), own, dev.num_sms, per_sm, false, here);
    parts_of(segments, 0., own, dev.num_sms, per_sm, false, there);
    const uint64_t tiles = (static_cast<uint64_t>(d.shared_width) * c.block + shared::kTileTokens - 1) / shared::kTileTokens;
    if (tiles == 0) return l;
    const uint64_t rows = static_cast<uint64_t>(d.num_seqs) * d.queries * d.q_heads;
    // pairs of row tiles: those that the rows fill, and one more for each group
    const uint64_t pairs = rows / c.kv_heads / shared::kPairRows + std::min(d.num_groups, d.num_seqs);
    const uint64_t units = pairs * c.kv_heads * (tiles + shared::kStart), most = (units + 2 * shared::kStart - 1) / (2 * shared::kStart);
    l.shares = static_cast<uint32_t>(most < static_cast<uint64_t>(dev.num_sms) ? most : dev.num_sms);
    there += 14 + 2.6 * static_cast<double>(units) / l.shares;
    if (here <= there) {
        l.shares = 0;
        return l;
    }
    auto take = [&l](size_t bytes) {
        const size_t at = l.total;
        l.total += (bytes + 255) & ~static_cast<size_t>(255);
        return at;
    };
    const size_t slots = static_cast<size_t>(l.shares) * 2 * shared::kPairRows;
    l.far = take(rows * sizeof(FarRow));
    l.whole_ml = take(rows * 8);
    l.whole_o = take(rows * c.dim * 4);
    l.part_ml = take(slots * 8);
    l.part_o = take(slots * c.dim * 4);
    return l;
}

}  // namespace

cudaError_t launch_block_attention(const bs_token_cache& c, const bs_block_attention_desc& d, const MemoryDevice& dev, cudaStream_t stream) {
    RowsArgs a{};
    a.s.c = c;
    a.s.errors = dev.errors;
    a.s.d.q = d.q;
    for (int i = 0; i < 3; ++i) a.s.d.q_stride[i] = d.q_stride[i];
    a.s.d.table = d.table;
    a.s.d.lens = d.lens;
    a.s.d.out = d.out;
    a.s.d.lse = d.lse;
    a.s.d.num_seqs = d.num_seqs;
    a.s.d.table_width = d.table_width;
    a.s.d.queries = d.queries;
    a.s.d.q_heads = d.q_heads;
    a.s.d.dtype = d.dtype;
    a.s.d.scale = d.scale;
    a.s.group = d.q_heads / c.kv_heads;
    a.s.block_log2 = log2_of(c.block);
    a.blocks = d.blocks;
    a.count = d.count;
    a.rows = a.s.group;
    return a.rows <= 8 ? launch_rows<1, true>(a, dev, stream) : launch_rows<2, true>(a, dev, stream);
}

size_t shared_attention_scratch(const bs_token_cache& c, const bs_shared_attention_desc& d, const MemoryDevice& dev) {
    return plan(c, d, dev).total;
}

cudaError_t launch_shared_attention(const bs_token_cache& c, const bs_shared_attention_desc& d, const MemoryDevice& dev, cudaStream_t stream) {
    const Layout l = plan(c, d, dev);
    unsigned char* const work = static_cast<unsigned char*>(d.workspace);
    RowsArgs a{};
    a.s.c = c;
    a.s.d = d;
    a.s.errors = dev.errors;
    a.s.far = reinterpret_cast<FarRow*>(work + l.far);
    a.s.whole_ml = reinterpret_cast<float2*>(work + l.whole_ml);
    a.s.whole_o = reinterpret_cast<float*>(work + l.whole_o);
    a.s.part_ml = reinterpret_cast<float2*>(work + l.part_ml);
    a.s.part_o = reinterpret_cast<float*>(work + l.part_o);
    a.s.group = d.q_heads / c.kv_heads;
    a.s.rows = a.rows = a.s.group * d.queries;
    a.s.shares = l.shares;
    a.direct = l.shares == 0 && d.shared_width > 0;
    a.s.block_log2 = log2_of(c.block);
    const cudaError_t e = l.shares ? launch_shared_part(a.s, stream) : cudaSuccess;
    if (e != cudaSuccess) return e;
    return a.rows <= 8 ? launch_rows<1, false>(a, dev, stream) : launch_rows<2, false>(a, dev, stream);
}

}  // namespace bsb
