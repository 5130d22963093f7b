// bs_cache_attention.cu -- attention over the 8-bit token cache
// (include/bsearch.h, bs_cache_attention).
//
// A few query rows (the heads that share a key head, times the query tokens)
// meet a long cache once, so the time is the cache's bytes.  Every (sequence,
// key head) is a segment of tiles of 32 tokens, and all segments, end to end,
// are cut into shares of equal cost, one per thread block, whatever the
// lengths are.  A share can end inside a segment; the pieces are joined by a
// second kernel.  A half of a tile (16 tokens) never spans two blocks, so it
// has one scale.
//
// The matrix instructions are m16n8k16 with the TOKENS as the 16 rows of the
// scores and the DIMENSIONS as the 16 rows of the outputs; the query rows are
// the 8 columns.  So a code is converted once for 8 * NT query rows and few
// rows waste little:
//   S^T[token][row] = K[token][dim] Q^T[dim][row]
//   O^T[dim][row]  += V^T[dim][token] P^T[token][row]
// A sum over dimensions or tokens may take them in any order, so each lane's
// share of a fragment is what lies side by side in memory.
//
// Codes become f16 exactly (|code| <= 128); bf16 queries become f16 exactly
// too, each row scaled by a power of two (elements below 2^-29 of the row's
// largest lose bits, far under a 32-bit sum's rounding).  Scores, weights' sums
// and outputs are 32-bit.  Where a weight meets the values, its
// product with their scale is rounded to f16: by 2^-11 of itself, as much as
// an f16 output's own rounding, or, where that is more (f16 has no exponents
// below), by 2^-30 of the largest such product that the warp has met (value
// scales count down to 2^-60 of the largest).  A fold of 2^5 (kFold) in those
// units uses the exponents that f16 has above 2^kSlack; without it the second
// figure is 2^-25, and weights e^-14 of the largest beside a scale 50 times
// theirs vanished.  The sum of weights takes them unrounded.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bs_cache_tile.cuh"
#include "bs_device.cuh"
#include "bs_memory.h"

namespace bsb {

using namespace dev;
using namespace tile;

namespace {

// Tiles a warp has in flight or in use, and resident blocks: 8 query rows fit
// three blocks with two stages each (35 us for a batch of 74 k tokens and 8
// key heads, 37 with two blocks of three stages), 16 rows only two (at three
// they spill: 56 us against 41).
template <int NT>
constexpr int kStagesOf = NT == 1 ? 2 : 3;
constexpr int blocks_per_sm(int nt) { return nt == 1 ? 3 : 2; }

struct CacheArgs {
    bs_token_cache c;
    bs_cache_attention_desc d;
    unsigned int* errors;
    float* lse;          // [num_seqs][queries][q_heads]
    float* part_o;       // [row tiles][blocks][2][8 * NT][dim]: unfinished outputs
    float* part_ml;      // [row tiles][blocks][2][8 * NT][2]: their maximum (log2) and sum
    float* scores;       // [num_seqs][kv_heads][rows][score_width], log2 units, or null
    uint32_t group;      // query heads per key head
    uint32_t rows;       // group * queries
    uint32_t score_width;
    uint32_t shares;     // thread blocks per row tile
    uint32_t block_log2;
    uint32_t direct;     // 1: a thread block per segment, nothing to join
};

__device__ __forceinline__ uint32_t held_tokens(const CacheArgs& a, uint32_t b) {
    const int32_t len = a.d.lens[b];
    const int64_t most = static_cast<int64_t>(a.d.table_width) * a.c.block;
    if (len >= 0 && len <= most) return len;
    atomicOr(a.errors, kMemErrLength);
    return len < 0 ? 0 : static_cast<uint32_t>(most);
}

__device__ __forceinline__ uint32_t tiles_of(uint32_t len) { return (len + kTile - 1) / kTile; }

// Shares.  A segment costs its tiles and kStart more for its queries and its
// last reduction (measured: about 3 us against 0.45 us a tile of one block);
// of W such units over n blocks, block i has first(i) .. first(i + 1).  A
// segment's first kStart units stand for no tiles.
constexpr uint32_t kStart = 6;
__device__ __forceinline__ uint32_t cost_of(uint32_t len) { return len ? tiles_of(len) + kStart : 0; }
__device__ __forceinline__ uint32_t used_shares(uint64_t w, uint32_t n) {
    const uint64_t most = (w + kStart + kWarps - 1) / (kStart + kWarps);      // a tile for each warp at least
    return most < n ? static_cast<uint32_t>(most) : n;
}
__device__ __forceinline__ uint64_t share_first(uint64_t w, uint32_t n, uint32_t i) {
    return w / n * i + min(static_cast<uint64_t>(i), w % n);
}
// The block whose share holds unit x.
__device__ __forceinline__ uint32_t share_of(uint64_t w, uint32_t n, uint64_t x) {
    const uint64_t q = w / n, r = w % n, wide = r * (q + 1);
    return static_cast<uint32_t>(x < wide ? x / (q + 1) : r + (x - wide) / q);
}

// Cost of one key head's segments before sequence b, and of all sequences;
// every thread of the block (a multiple of 32 threads) gets both.
__device__ __forceinline__ void count_cost(const CacheArgs& a, uint32_t b, uint64_t& before, uint64_t& all, uint64_t* warp_sums) {
    uint64_t mine = 0, total = 0;
    for (uint32_t i = threadIdx.x; i < a.d.num_seqs; i += blockDim.x) {
        const uint32_t t = cost_of(held_tokens(a, i));
        total += t;
        mine += i < b ? t : 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        mine += __shfl_xor_sync(kFull, mine, o);
        total += __shfl_xor_sync(kFull, total, o);
    }
    const uint32_t warps = blockDim.x / 32, warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) {
        warp_sums[warp] = mine;
        warp_sums[warps + warp] = total;
    }
    __syncthreads();
    before = all = 0;
    for (uint32_t i = 0; i < warps; ++i) {
        before += warp_sums[i];
        all += warp_sums[warps + i];
    }
    __syncthreads();
}

// Where a block is in its share: a piece is a run of tiles of one segment.
struct Piece {
    uint32_t b, h, len;
    uint32_t t, end;        // tiles of the segment
    uint64_t left;          // units of the share after this piece
};

// The piece of segment (b, h) from its unit `from` on.
__device__ __forceinline__ void cut_piece(Piece& p, uint32_t from) {
    const uint32_t cost = cost_of(p.len), take = p.left < cost - from ? static_cast<uint32_t>(p.left) : cost - from;
    p.t = from > kStart ? from - kStart : 0;
    p.end = from + take > kStart ? from + take - kStart : 0;
    p.left -= take;
}

__device__ __forceinline__ void next_piece(const CacheArgs& a, Piece& p) {
    if (p.left == 0) {
        p.t = p.end = 0;
        p.b = a.d.num_seqs;
        return;
    }
    if (++p.h == static_cast<uint32_t>(a.c.kv_heads)) {
        p.h = 0;
        do {
            ++p.b;
            p.len = held_tokens(a, p.b);
        } while (p.len == 0);
    }
    cut_piece(p, 0);
}

template <int NW, int NT>
constexpr size_t kSplitSmem = kWarps * kStagesOf<NT> * kStageBytes<NW> + kJoinBytes<NW, NT> + kWarps * (8 * NT * 2 + 4) * 4 + 128;

// One share of the tiles for one row tile of 8 * NT query rows.
// Measured (without | with the weights' scores): 16 x 65,536 tokens, 8 key
// heads of 128, 2.15 GB: 365 | 400 us (copies alone: 344); 32 sequences of 74 k
// tokens in all 35 us with them; 4 of 54 k in all, 4 drafted tokens each, 41 us
// without.  Long caches are
// bound by DRAM (5.4 to 5.9 TB/s); the others by the first and last tiles of
// the shares and, with 16 query rows, by the instructions of 8 warps an SM.
// Registers: outputs NW * NT * 4, queries NW * NT * 2, and about 60.
template <int NW, int NT>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(NT)) k_cache_split(const __grid_constant__ CacheArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int kDim = NW * 16, kRows = 8 * NT, kStages = kStagesOf<NT>;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    unsigned char* ring = smem + warp * kStages * kStageBytes<NW>;
    float* join_o = reinterpret_cast<float*>(smem + kWarps * kStages * kStageBytes<NW>);
    float* join_ml = join_o + 2 * kRows * kDim;                 // [warps][kRows][2]
    uint64_t* sums = reinterpret_cast<uint64_t*>(smem);         // before the ring is used

    cudaGridDependencySynchronize();       // in every block, before anything of the caller's
    // this block's share, and the piece it begins with
    const uint32_t hkv = a.c.kv_heads, row0 = blockIdx.y * kRows;
    Piece at;
    if (a.direct) {
        at.b = blockIdx.x / hkv;
        at.h = blockIdx.x % hkv;
        at.len = held_tokens(a, at.b);
        at.left = cost_of(at.len);
        if (at.len) cut_piece(at, 0);
        else at.t = at.end = 0;
    } else {
        uint64_t before, all;
        count_cost(a, 0, before, all, sums);
        const uint64_t w_all = all * hkv;
        const uint32_t n = used_shares(w_all, a.shares);
        if (blockIdx.x >= n) return;
        const uint64_t first = share_first(w_all, n, blockIdx.x);
        uint64_t seen = 0;
        uint32_t b = 0;
        for (uint32_t b0 = 0;; b0 += 32) {                       // 32 sequences at a time
            const uint32_t len = b0 + lane < a.d.num_seqs ? held_tokens(a, b0 + lane) : 0;
            const uint64_t mine = static_cast<uint64_t>(cost_of(len)) * hkv;
            uint64_t sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t up = __shfl_up_sync(kFull, sum, o);
                if (lane >= static_cast<uint32_t>(o)) sum += up;
            }
            const unsigned past = __ballot_sync(kFull, seen + sum > first);
            if (past) {
                const int l = __ffs(past) - 1;
                b = b0 + l;
                at.len = __shfl_sync(kFull, len, l);
                seen += __shfl_sync(kFull, sum - mine, l);
                break;
            }
            seen += __shfl_sync(kFull, sum, 31);
        }
        const uint32_t cost = cost_of(at.len);
        at.b = b;
        at.h = static_cast<uint32_t>((first - seen) / cost);
        at.left = share_first(w_all, n, blockIdx.x + 1) - first;
        cut_piece(at, static_cast<uint32_t>((first - seen) % cost));
    }

    // the copies run ahead of the arithmetic: `ahead` is the piece whose
    // tiles are being requested, ahead_t the next tile of this warp in it
    Piece ahead = at;
    uint32_t ahead_t = at.t + warp;
    uint32_t next_id[2];
    bool have_next;
    auto find_next = [&]() {            // to this warp's next tile, and its halves' block ids
        while (ahead_t >= ahead.end && ahead.b < a.d.num_seqs) {
            next_piece(a, ahead);
            ahead_t = ahead.t + warp;
        }
        have_next = ahead.b < a.d.num_seqs;
        if (have_next) {
            const int32_t* row = a.d.table + static_cast<uint64_t>(ahead.b) * a.d.table_width;
            next_id[0] = row[ahead_t * kTile >> a.block_log2];
            next_id[1] = next_id[0];
            if (a.block_log2 == 4 && ahead_t * kTile + 16 < ahead.len) next_id[1] = row[ahead_t * 2 + 1];
        }
    };
    auto request = [&](uint32_t stage) {
        if (have_next) {
            unsigned char* s = ring + stage * kStageBytes<NW>;
            float* scales = reinterpret_cast<float*>(s + 2 * kTile * kPitch<NW>);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t id = next_id[half], pos = ahead_t * kTile + 16 * half;
                if (id < a.c.num_blocks && pos < ahead.len) {
                    const uint64_t slab = static_cast<uint64_t>(id) * hkv + ahead.h;
                    const uint64_t row = ((slab << a.block_log2) + (pos & (a.c.block - 1))) * kDim + lane * 16;
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
                    if (pos < ahead.len) atomicOr(a.errors, kMemErrBlock);
                }
            }
            ahead_t += kWarps;
            find_next();
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    find_next();
    __syncthreads();                         // `sums` is done with
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) request(i);
    uint32_t stage = 0, fill = kStages - 1;

    // where this lane's query rows (columns of the products) lie within a
    // sequence and key head, and which query its columns 2c and 2c + 1 are
    int64_t row_off[NT];
    int32_t col_query[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const uint32_t r = row0 + 8 * nt + g, col = row0 + 8 * nt + 2 * c;
        row_off[nt] = (r / a.group) * a.d.q_stride[1] + (r % a.group) * a.d.q_stride[2] + c * (NW * 4);
        col_query[nt][0] = static_cast<int32_t>(col / a.group);
        col_query[nt][1] = static_cast<int32_t>((col + 1) / a.group);
    }

    for (bool first_piece = true; at.b < a.d.num_seqs; next_piece(a, at), first_piece = false) {
        if (at.t == at.end && !a.direct) continue;      // a share that ends before a segment's first tile
        // this piece's query rows as the columns of K Q^T: column j is row row0 + j
        uint32_t q[NT][NW][2];
        float row_scale[NT][2];          // of columns 2c and 2c + 1
        int32_t limit[NT][2];            // tokens that row sees
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint16_t* row = static_cast<const uint16_t*>(a.d.q) + at.b * a.d.q_stride[0] +
                                  static_cast<int64_t>(at.h) * a.group * a.d.q_stride[2] + row_off[nt];
            load_query_row<NW>(q[nt], row_scale[nt], row, row0 + 8 * nt + g < a.rows, a.d.dtype != BS_F16, a.d.scale * 1.4426950408889634f, c);
#pragma unroll
            for (int i = 0; i < 2; ++i) limit[nt][i] = static_cast<int32_t>(at.len) - a.d.queries + 1 + col_query[nt][i];
        }
        float o[NT][NW][4];
        // outputs count in 2^top * unit / kFold.  (Begun with another constant than
        // kNoScore's, drafts take 47.0 us, not 45.1.)
        float top[NT][2], sum[NT][2], unit = kFold / -kNoScore, inv_unit = -kNoScore;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            top[nt][0] = top[nt][1] = kNoScore;
            sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
            for (int j = 0; j < NW; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
        }
        float* score_at = a.scores ? a.scores + ((static_cast<uint64_t>(at.b) * hkv + at.h) * a.rows + row0 + 2 * c) * a.score_width + g : nullptr;

        for (uint32_t t = at.t + warp; t < at.end; t += kWarps) {
            asm volatile("cp.async.wait_group %0;\n" ::"n"(kStages - 2) : "memory");
            __syncwarp();
            request(fill);               // the stage that the last tile used
            fill = fill + 1 == kStages ? 0 : fill + 1;
            const unsigned char* s = ring + stage * kStageBytes<NW>;
            stage = stage + 1 == kStages ? 0 : stage + 1;
            const float4 sc = *reinterpret_cast<const float4*>(s + 2 * kTile * kPitch<NW>);
            const float k_scale[2] = {sc.x, sc.z}, v_scale[2] = {sc.y, sc.w};

            float z[2][NT][4];           // [half]: tokens g and g + 8 (+ 16 half), columns 2c and 2c + 1
            tile_scores<NW, NT>(z, s, q, g, c);
            const bool edge = static_cast<int32_t>((t + 1) * kTile) > static_cast<int32_t>(at.len) - a.d.queries + 1 ||
                              fminf(v_scale[0], v_scale[1]) < 0.f;
            bool move = fmaxf(v_scale[0], v_scale[1]) > 4.f * unit;
            const float room[2] = {kSlack - scale_log2(v_scale[0], inv_unit), kSlack - scale_log2(v_scale[1], inv_unit)};
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        z[half][nt][i] *= row_scale[nt][i & 1] * k_scale[half];
                        if (edge) {
                            const int32_t pos = static_cast<int32_t>(t * kTile + 16 * half + g) + (i & 2) * 4;
                            if (pos >= limit[nt][i & 1] || v_scale[half] < 0.f) z[half][nt][i] = -INFINITY;
                        }
                        move |= z[half][nt][i] > top[nt][i & 1] + room[half];
                    }
            if (score_at) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (row0 + 8 * nt + 2 * c + i < a.rows) {
                            float* p = score_at + static_cast<uint64_t>(8 * nt + i) * a.score_width + t * kTile;
                            p[0] = z[0][nt][i];
                            p[8] = z[0][nt][2 + i];
                            if (t * kTile + 16 < at.len) {
                                p[16] = z[1][nt][i];
                                p[24] = z[1][nt][2 + i];
                            }
                        }
            }
            if (__any_sync(kFull, move)) move_maxima<NW, NT>(z, v_scale, top, sum, o, unit, inv_unit);
            tile_values<NW, NT>(z, s, v_scale, inv_unit, top, sum, o, g, c);
            __syncwarp();
        }

        float all_top[NT][2], all_sum[NT][2];
        join_warps<NW, NT>(o, top, sum, unit, all_top, all_sum, join_o, join_ml, warp, lane);
        if (warp == 0) {
            const bool whole = at.t == 0 && at.end == tiles_of(at.len);
            const uint64_t slot = (static_cast<uint64_t>(blockIdx.y) * a.shares + blockIdx.x) * 2 + (first_piece ? 0 : 1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t r = 8 * nt + 2 * c + i, col = row0 + r;
                    if (col >= a.rows) continue;
                    const float l = all_sum[nt][i];
                    if (whole) {
                        const uint32_t query = col_query[nt][i];
                        const uint64_t row = (static_cast<uint64_t>(at.b) * a.d.queries + query) * a.d.q_heads + at.h * a.group +
                                             (col - query * a.group);
                        const float inv = l == 0.f ? 0.f : 1.f / l;
                        if (g == 0) a.lse[row] = l == 0.f ? -INFINITY : (all_top[nt][i] + log2f(l)) * 0.6931471805599453f;
#pragma unroll
                        for (int j = 0; j < NW; ++j) {
                            const float x = o[nt][j][i] * inv, y = o[nt][j][2 + i] * inv;
                            const uint64_t e = row * kDim + value_dim<NW>(j, g);
                            if (a.d.dtype == BS_F16) *reinterpret_cast<__half2*>(static_cast<__half*>(a.d.out) + e) = __floats2half2_rn(x, y);
                            else *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(a.d.out) + e) = __floats2bfloat162_rn(x, y);
                        }
                    } else {
                        if (g == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * kRows + r) * 2) = make_float2(all_top[nt][i], l);
#pragma unroll
                        for (int j = 0; j < NW; ++j)
                            *reinterpret_cast<float2*>(a.part_o + (slot * kRows + r) * kDim + value_dim<NW>(j, g)) =
                                make_float2(o[nt][j][i], o[nt][j][2 + i]);
                    }
                }
        }
    }
}

// One block per row: joins the pieces of a segment that lies in several
// shares, writes zeros for an empty one.  A lane has four dimensions, the
// warps take the pieces in turn.  Always the same order of additions.
// Launched while the first kernel still runs; waits for it before it reads.
// 5.7 us, most of it a launch and the chain of dependent loads.  Joining inside
// k_cache_mass instead was not faster: 14.3 us against 5.5 + 8.3 for 32
// sequences of 74 k tokens, 62 against 51 + 5 for 16 x 65,536.
constexpr int kJoinThreads = 128;
__global__ void __launch_bounds__(kJoinThreads) k_cache_join(const __grid_constant__ CacheArgs a, uint32_t tile_rows, uint32_t used_rows) {
    constexpr uint32_t kJoinWarps = kJoinThreads / 32;
    __shared__ uint64_t sums[2 * kJoinWarps];
    __shared__ float4 parts[kJoinWarps][32];
    const uint32_t h = blockIdx.x / used_rows, r = blockIdx.x % used_rows, rt = blockIdx.y, b = blockIdx.z;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hkv = a.c.kv_heads, dim = a.c.dim, col = rt * tile_rows + r;
    cudaGridDependencySynchronize();       // in every block, before anything of the caller's
    uint64_t before, all;
    count_cost(a, b, before, all, sums);
    const uint32_t tiles = tiles_of(held_tokens(a, b));
    if (col >= a.rows) return;
    const uint64_t w_all = all * hkv, s0 = before * hkv + static_cast<uint64_t>(h) * (tiles + kStart);
    uint32_t i0 = 0, pieces = 0, slot0 = 0;
    if (tiles) {
        const uint32_t n = used_shares(w_all, a.shares);
        i0 = share_of(w_all, n, s0 + kStart);                   // the segment's first and last tile
        pieces = share_of(w_all, n, s0 + kStart + tiles - 1) - i0 + 1;
        if (pieces == 1) return;                                // done by that share
        slot0 = share_first(w_all, n, i0) >= s0 ? 0 : 1;        // later shares begin inside the segment: slot 0
    }
    auto slot = [&](uint32_t i) { return ((static_cast<uint64_t>(rt) * a.shares + i0 + i) * 2 + (i == 0 ? slot0 : 0)) * tile_rows + r; };
    float m = kNoScore, l = 0.f;
    for (uint32_t i = lane; i < pieces; i += 32) m = fmaxf(m, a.part_ml[slot(i) * 2]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
    for (uint32_t i = lane; i < pieces; i += 32) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + slot(i) * 2);
        l += ml.y * exp2_fast(ml.x - m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(kFull, l, o);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (lane * 4 < dim) {
        constexpr uint32_t kBatch = 4;                          // loads in flight
        for (uint32_t i = warp; i < pieces; i += kJoinWarps * kBatch) {
            float4 o[kBatch];
            float f[kBatch];
#pragma unroll
            for (uint32_t u = 0; u < kBatch; ++u) {
                const uint32_t x = i + u * kJoinWarps, at = x < pieces ? x : i;
                f[u] = a.part_ml[slot(at) * 2];
                o[u] = *reinterpret_cast<const float4*>(a.part_o + slot(at) * dim + lane * 4);
            }
#pragma unroll
            for (uint32_t u = 0; u < kBatch; ++u) {
                if (i + u * kJoinWarps >= pieces) break;
                const float w = exp2_fast(f[u] - m);
                acc.x += o[u].x * w, acc.y += o[u].y * w, acc.z += o[u].z * w, acc.w += o[u].w * w;
            }
        }
    }
    parts[warp][lane] = acc;
    __syncthreads();
    if (warp != 0 || lane * 4 >= dim) return;
#pragma unroll
    for (uint32_t x = 1; x < kJoinWarps; ++x) {
        const float4 o = parts[x][lane];
        acc.x += o.x, acc.y += o.y, acc.z += o.z, acc.w += o.w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const uint64_t row = (static_cast<uint64_t>(b) * a.d.queries + col / a.group) * a.d.q_heads + h * a.group + col % a.group;
    if (lane == 0) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    const uint64_t at = row * dim + lane * 4;
    if (a.d.dtype == BS_F16) {
        __half2* p = reinterpret_cast<__half2*>(static_cast<__half*>(a.d.out) + at);
        p[0] = __floats2half2_rn(acc.x * inv, acc.y * inv);
        p[1] = __floats2half2_rn(acc.z * inv, acc.w * inv);
    } else {
        __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(a.d.out) + at);
        p[0] = __floats2bfloat162_rn(acc.x * inv, acc.y * inv);
        p[1] = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
    }
}

// One thread per four tokens of a key head: their weights over all query
// rows, from the scores that the first kernel left and the rows' lse.  Bound
// by reading the scores: 45 us for 16 x 65,536 tokens of 32 heads (134 MB of
// scores, 67 of sums: 4.5 TB/s), 8 us for 74 k tokens.
constexpr int kMassThreads = 128;
__global__ void __launch_bounds__(kMassThreads) k_cache_mass(const __grid_constant__ CacheArgs a) {
    const uint32_t j = (blockIdx.x * kMassThreads + threadIdx.x) * 4, h = blockIdx.y, b = blockIdx.z;
    const uint32_t width = a.d.mass_width;
    cudaGridDependencySynchronize();       // in every block, before anything of the caller's
    const uint32_t len = held_tokens(a, b);
    if (j == 0 && len > width) atomicOr(a.errors, kMemErrLength);      // tokens whose weights have no place
    if (j >= width) return;
    const uint64_t seg = static_cast<uint64_t>(b) * a.c.kv_heads + h, at = seg * width + j;
    const uint32_t n = j < len ? min(len - j, 4u) : 0;
    // four at once where their place is a multiple of 16 bytes
    const bool whole = j + 4 <= width && width % 4 == 0 &&
                       ((reinterpret_cast<uintptr_t>(a.d.mass) | reinterpret_cast<uintptr_t>(a.d.out_mass)) & 15) == 0;
    float w[4] = {0.f, 0.f, 0.f, 0.f};
    if (n && a.d.mass) {
        if (whole) *reinterpret_cast<float4*>(w) = *reinterpret_cast<const float4*>(a.d.mass + at);
        else
            for (uint32_t i = 0; i < n && j + i < width; ++i) w[i] = a.d.mass[at + i];
    }
    if (n) {
        const float* s = a.scores + seg * a.rows * a.score_width + j;
        constexpr uint32_t kBatch = 4;             // rows whose scores are on their way together
        for (uint32_t r0 = 0; r0 < a.rows; r0 += kBatch) {
            float4 z[kBatch];
            float lse[kBatch];
#pragma unroll
            for (uint32_t u = 0; u < kBatch; ++u) {
                const uint32_t r = min(r0 + u, a.rows - 1);
                z[u] = __ldcs(reinterpret_cast<const float4*>(s + static_cast<uint64_t>(r) * a.score_width));
                lse[u] = a.lse[(static_cast<uint64_t>(b) * a.d.queries + r / a.group) * a.d.q_heads + h * a.group + r % a.group];
            }
#pragma unroll
            for (uint32_t u = 0; u < kBatch; ++u) {
                if (r0 + u >= a.rows) break;
                const float l = lse[u] * 1.4426950408889634f;
                if (z[u].x != -INFINITY) w[0] += exp2_fast(z[u].x - l);
                if (z[u].y != -INFINITY) w[1] += exp2_fast(z[u].y - l);
                if (z[u].z != -INFINITY) w[2] += exp2_fast(z[u].z - l);
                if (z[u].w != -INFINITY) w[3] += exp2_fast(z[u].w - l);
            }
        }
    }
    for (uint32_t i = n; i < 4; ++i) w[i] = 0.f;
    if (whole) *reinterpret_cast<float4*>(a.d.out_mass + at) = *reinterpret_cast<const float4*>(w);
    else
        for (uint32_t i = 0; i < 4 && j + i < width; ++i) a.d.out_mass[at + i] = w[i];
}

constexpr uint32_t kWaves = 8;

struct Layout {
    uint32_t nt, row_tiles, shares, score_width, direct;
    size_t lse, part_o, part_ml, scores, total;
};

Layout plan(const bs_token_cache& c, const bs_cache_attention_desc& d, const MemoryDevice& dev) {
    Layout l{};
    const uint32_t rows = static_cast<uint32_t>(d.q_heads / c.kv_heads) * d.queries;
    l.nt = rows <= 8 ? 1 : 2;
    l.row_tiles = (rows + 8 * l.nt - 1) / (8 * l.nt);
    const uint64_t tokens = static_cast<uint64_t>(d.table_width) * c.block;
    const uint64_t most = (static_cast<uint64_t>(d.num_seqs) * c.kv_heads * ((tokens + kTile - 1) / kTile + kStart) + kStart + kWarps - 1) /
                          (kStart + kWarps);
    const uint64_t cap = static_cast<uint64_t>(dev.num_sms) * blocks_per_sm(l.nt);
    l.shares = static_cast<uint32_t>(most < cap ? most : cap);
    // many row tiles fill the GPU by themselves: eight waves of blocks are cut
    // fine enough (33 queries of 8 heads a key head 162 -> 130 us, 64 of 128 780
    // -> 417), and the pieces (two a share) stay below 140 MB where 1,024 queries
    // of 128 heads would have 40 GB
    const uint32_t enough = static_cast<uint32_t>((kWaves * cap + l.row_tiles - 1) / l.row_tiles);
    if (l.shares > enough) l.shares = enough;
    // short sequences: a thread block for each segment costs less than a
    // second kernel (300 tokens: 6 us against 5 + 4)
    l.direct = tokens <= 1024;
    if (l.direct) l.shares = d.num_seqs * static_cast<uint32_t>(c.kv_heads);
    l.score_width = static_cast<uint32_t>(tokens);
    auto take = [&l](size_t bytes) {
        const size_t at = l.total;
        l.total += (bytes + 255) & ~static_cast<size_t>(255);
        return at;
    };
    const size_t slots = l.direct ? 0 : static_cast<size_t>(l.row_tiles) * l.shares * 2 * 8 * l.nt;
    l.lse = take(d.lse ? 0 : static_cast<size_t>(d.num_seqs) * d.queries * d.q_heads * 4);
    l.part_ml = take(slots * 8);
    l.part_o = take(slots * c.dim * 4);
    l.scores = take(d.out_mass ? static_cast<size_t>(d.num_seqs) * c.kv_heads * rows * tokens * 4 : 0);
    return l;
}

template <int NW, int NT>
cudaError_t launch_split(const CacheArgs& a, uint32_t row_tiles, cudaStream_t stream) {
    const cudaError_t e = cudaFuncSetAttribute(k_cache_split<NW, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSplitSmem<NW, NT>);
    if (e != cudaSuccess) return e;
    return launch_after(k_cache_split<NW, NT>, dim3(a.shares, row_tiles), kThreads, kSplitSmem<NW, NT>, stream, a);
}

template <int NT>
cudaError_t launch_split(const CacheArgs& a, uint32_t row_tiles, cudaStream_t stream) {
    switch (a.c.dim / 16) {
        case 1: return launch_split<1, NT>(a, row_tiles, stream);
        case 2: return launch_split<2, NT>(a, row_tiles, stream);
        case 3: return launch_split<3, NT>(a, row_tiles, stream);
        case 4: return launch_split<4, NT>(a, row_tiles, stream);
        case 5: return launch_split<5, NT>(a, row_tiles, stream);
        case 6: return launch_split<6, NT>(a, row_tiles, stream);
        case 7: return launch_split<7, NT>(a, row_tiles, stream);
        default: return launch_split<8, NT>(a, row_tiles, stream);
    }
}

}  // namespace

size_t cache_attention_scratch(const bs_token_cache& c, const bs_cache_attention_desc& d, const MemoryDevice& dev) {
    return plan(c, d, dev).total;
}

cudaError_t launch_cache_attention(const bs_token_cache& c, const bs_cache_attention_desc& d, const MemoryDevice& dev,
                                   cudaStream_t stream) {
    const Layout l = plan(c, d, dev);
    unsigned char* work = static_cast<unsigned char*>(d.workspace);
    CacheArgs a{c, d, dev.errors};
    a.lse = d.lse ? d.lse : reinterpret_cast<float*>(work + l.lse);
    a.part_o = reinterpret_cast<float*>(work + l.part_o);
    a.part_ml = reinterpret_cast<float*>(work + l.part_ml);
    a.scores = d.out_mass ? reinterpret_cast<float*>(work + l.scores) : nullptr;
    a.group = d.q_heads / c.kv_heads;
    a.rows = a.group * d.queries;
    a.score_width = l.score_width;
    a.shares = l.shares;
    a.block_log2 = c.block == 16 ? 4 : c.block == 32 ? 5 : c.block == 64 ? 6 : 7;
    cudaError_t e = cudaSuccess;
    a.direct = l.direct;
    if (l.shares) e = l.nt == 1 ? launch_split<1>(a, l.row_tiles, stream) : launch_split<2>(a, l.row_tiles, stream);
    if (e != cudaSuccess) return e;
    const uint32_t tile_rows = 8 * l.nt, used_rows = a.rows < tile_rows ? a.rows : tile_rows;
    if (!l.direct) e = launch_after(k_cache_join, dim3(c.kv_heads * used_rows, l.row_tiles, d.num_seqs), kJoinThreads, 0, stream, a, tile_rows, used_rows);
    if (e == cudaSuccess && d.out_mass)
        e = launch_after(k_cache_mass, dim3((d.mass_width + 4 * kMassThreads - 1) / (4 * kMassThreads), c.kv_heads, d.num_seqs),
                         kMassThreads, 0, stream, a);
    return e;
}

}  // namespace bsb
