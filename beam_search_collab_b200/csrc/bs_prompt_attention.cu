// bs_prompt_attention.cu -- attention of packed prompts (include/bsearch.h,
// bs_prompt_attention).
//
// One thread block computes two tiles of 128 query rows against the keys they
// see, 128 at a time, with a running maximum and sum per row.  The rows of a
// tile are consecutive tokens times the query heads that share a key head, so
// a tile's keys and values are loaded once for all those heads.  A block that
// is done takes over the next one of the grid that has not started (cluster
// launch control), its copies and first products under the last one's
// epilogue.  Where there are few tiles of queries and many of keys, the keys
// are cut into chunks and a second kernel joins them.
//
// Warps 0-3 and 4-7 are the softmax of tile 0 and 1 (a thread has one row),
// warp 8 issues the matrix instructions, warp 9 the copies, warp 10 looks at
// hidden values, warp 11 finds the next item:
//   copies    query tiles, then keys and values through one ring of stages
//             (tiled TMA, 128-byte swizzle, 64 columns of a row at a time)
//   matrix    S_t = Q_t K^T    (both K-major in shared memory, S_t in TMEM)
//             O_t += P_t V     (P_t in TMEM over S_t's columns, V MN-major)
//             in the order S0 S1 | P0V S0' P1V S1' | ...: while one tile's
//             softmax runs, the tensor pipe has the other tile's work
//   softmax   S_t to registers, P_t = 2^(scale' S_t - m) back to TMEM in the
//             inputs' 16-bit type.  m is moved only when a weight would be
//             over 2^8 (then O_t, in TMEM, is rescaled, and so are the tile's
//             weights that are there already, rounded a second time), so most
//             tiles touch O_t not at all and no maximum is taken before the
//             exponentials; sums are 32-bit of the unrounded P.
// TMEM (512 columns): S0 S1 O0 O1, 128 columns each.
//
// Keys of other sequences or of the future that a tile also covers are set to
// -infinity in S.  A zero weight would still pass an infinity or NaN of a
// hidden VALUE on, so in tiles with hidden keys warp 10 clears value
// rows past the sequence, and rows that are not finite and not seen by all;
// the softmax adds the latter for the rows that see them (never taken with
// finite inputs).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "bs_device.cuh"
#include "bs_f32x2.cuh"
#include "bs_memory.h"
#include "bs_tcgen05.cuh"

namespace bsb {

using namespace dev;
using namespace tc;

namespace {

constexpr int kThreads = 384;
constexpr uint32_t kMostChunks = 8;
constexpr float kMost = 256.f;         // weights may grow to this before the maximum is moved
// Weights count in 2^-kLift: in f16 the room that kMost leaves above is room
// for small ones (2^-21 of the largest with all bits; without it 2^-14, and
// keys e^-15 of the first one's weight were 3% off).  bf16 has exponents enough.
template <typename T>
constexpr float kLift = 0.f;
template <>
constexpr float kLift<__half> = 7.f;
template <typename T>
constexpr float kLifted = 1.f;
template <>
constexpr float kLifted<__half> = 128.f;     // 2^kLift

struct PromptArgs {
    bs_prompt_attention_desc d;
    unsigned int* errors;
    uint32_t group;            // query heads per key head
    uint32_t tile_tokens;      // tokens of a tile: group * tile_tokens <= 128 rows
    uint32_t polls;            // of a wait before it gives up (BSEARCH_WAIT_POLLS: a test sets 0)
    uint32_t chunks;           // pieces that the keys are cut into
    float* part_o;             // [chunks][rows][dim], where there are several
    float2* part_ml;           // [chunks][rows]: maximum (log2), sum
    CUtensorMap q, k, v;
};

// 64 columns x rows x 1 of a tensor (dim, heads, tokens) into shared memory.
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
            smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
        : "memory");
}

// Stages of keys or values that fit beside the query tiles and the softmax
// warps' 4 KB each for outputs.
template <int BOXES>
constexpr int kStagesOf = BOXES == 2 ? 4 : 8;
constexpr int kStagingBytes = 8 * 4096;

// 32 scores of a row: weights 2^(scale * s + base), packed in p; adds to two
// pairs of sums and of largest weights.
template <typename T>
__device__ __forceinline__ void weights32(const float* s, float2 scale, float2 base, uint32_t* p, float2 (&add)[2], uint32_t (&high)[2]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float2 x = fma2(make_float2(s[2 * i], s[2 * i + 1]), scale, base);
        x.x = exp2_fast(x.x);
        x.y = exp2_fast(x.y);
        add[i & 1] = add2(add[i & 1], x);
        p[i] = Type16<T>::pack(x.x, x.y);
        high[i & 1] = Type16<T>::larger(high[i & 1], p[i]);
    }
}

// 64 scores of a row that sees them all, 32 at a time; s[0] is on its way, the
// next 32 follow (`more`: those after these too).  Returns the largest
// weight, their sum in `part`.  (Unrolled: in a loop of 32 the
// special-function pipe runs dry at each turn, 2,650 clocks a tile against
// 1,650.)
template <typename T>
__device__ __forceinline__ float weights64(uint32_t s_at, bool more, float (&s)[2][32], float scale, float base, uint32_t (&p)[kRows / 4],
                                           float& part) {
    const float2 scale2 = make_float2(scale, scale), base2 = make_float2(base, base);
    float2 add[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    uint32_t high[2] = {0, 0};
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        wait_loads32(s[c]);
        if (c == 0 || more) tmem_load32(s_at + 32 * (c + 1), s[c ^ 1]);
        weights32<T>(s[c], scale2, base2, p + 16 * c, add, high);
    }
    add[0] = add2(add[0], add[1]);
    part = add[0].x + add[0].y;
    const float2 h = Type16<T>::unpack(Type16<T>::larger(high[0], high[1]));
    return fmaxf(h.x, h.y);
}

// The same for 32 scores in registers.
template <typename T>
__device__ __forceinline__ float weights(const float (&s)[32], float scale, float base, uint32_t (&p)[16], float& part) {
    float2 add[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    uint32_t high[2] = {0, 0};
    weights32<T>(s, make_float2(scale, scale), make_float2(base, base), p, add, high);
    add[0] = add2(add[0], add[1]);
    part = add[0].x + add[0].y;
    const float2 h = Type16<T>::unpack(Type16<T>::larger(high[0], high[1]));
    return fmaxf(h.x, h.y);
}

// The warp's rows times `shrink`: the first `quarters` of their weights of a tile
// and `dim` columns of outputs.
template <typename T>
__device__ __forceinline__ void rescale(uint32_t p_at, uint32_t o_at, int quarters, int dim, float shrink) {
    wait_stores();
#pragma unroll 1
    for (int c = 0; c < quarters; ++c) {
        uint32_t p[16];
        tmem_load16(p_at + 16 * c, p);
        wait_loads16(p);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const float2 f = Type16<T>::unpack(p[k]);
            p[k] = Type16<T>::pack(f.x * shrink, f.y * shrink);
        }
        tmem_store16(p_at + 16 * c, p);
    }
#pragma unroll 1
    for (int x = 0; x < dim; x += 16) {
        uint32_t o[16];
        tmem_load16(o_at + x, o);
        wait_loads16(o);
#pragma unroll
        for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * shrink);
        tmem_store16(o_at + x, o);
    }
    wait_stores();
}

// The first tile, tiles with hidden keys, and where the maximum moves: 32
// scores at a time, so that the weights can go to columns whose scores have
// been read.  From the quarter `from` on (0, or 2 where the first half's weights
// are made).  `state` is the row's maximum and sum, returned as they become.
template <typename T>
__device__ __noinline__ float2 weights_with_care(uint32_t s_at, uint32_t o_at, int from, int chunks, int32_t left, bool real, float scale,
                                                 int dim, float2 state) {
    float top = state.x, sum = state.y;
    float s[2][32];
    tmem_load32(s_at + 32 * from, s[0]);
#pragma unroll 1
    for (int c = from; c < chunks; c += 2) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int at = c + x;
            if (at >= chunks) break;
            wait_loads32(s[x]);
            if (at + 1 < chunks) tmem_load32(s_at + 32 * (at + 1), s[x ^ 1]);
#pragma unroll
            for (int k = 0; k < 32; ++k) s[x][k] = 32 * at + k < left ? s[x][k] : -INFINITY;
            uint32_t p[16];
            float part;
            const float high = weights<T>(s[x], scale, top == -INFINITY ? 0.f : kLift<T> - top * scale, p, part);
            if (__any_sync(kFull, real && (high > kMost * kLifted<T> || top == -INFINITY))) {
                // the maximum moves, what was summed is rescaled
                float next = top;
#pragma unroll
                for (int k = 0; k < 32; ++k) next = fmaxf(next, s[x][k]);
                const float shrink = next == -INFINITY ? 1.f : exp2_fast((top - next) * scale);
                top = next;
                sum *= shrink;
                if (at + 1 < chunks) wait_loads32(s[x ^ 1]);
                rescale<T>(s_at, o_at, at, dim, shrink);
                weights<T>(s[x], scale, top == -INFINITY ? 0.f : kLift<T> - top * scale, p, part);
            }
            sum += part;
            tmem_store16(s_at + 16 * at, p);
        }
    }
    return make_float2(top, sum);
}

// What a block works on: a pair of tiles and a run of key tiles.
struct Item {
    int32_t valid;              // 0: there is no more
    int32_t q0, k0, lq, lk;     // the sequence's rows
    int32_t token0;             // first token of the pair
    int32_t kv_head, chunk;
    int32_t first, end[2];      // key tiles of each tile of queries: first .. end[t]
    int32_t all_see;            // keys that every row of the pair sees
    int32_t most_see[2];        // keys that any row of a tile sees
};

struct Control {
    uint64_t q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2], done, asked;
    uint64_t item_full[2], item_empty[2], next_full;
    uint64_t full[8], empty[8], raw[8];      // raw: values that warp 10 looks at before they are full
    __align__(16) uint32_t next[4]; // the launch control's answer
    Item item[2];
    uint32_t not_finite[8][4];      // by stage: value rows cleared because they are not finite
    uint32_t keep[2];               // outputs hold something before the first value product
    uint32_t tmem;
    uint32_t gave_up;
};

template <int BOXES>
constexpr size_t kSmem = 1024 + (2 + kStagesOf<BOXES>) * BOXES * kBoxBytes + kStagingBytes + sizeof(Control);

// Asks for the next block of the grid that has not started; the answer
// arrives at `bar`.
__device__ __forceinline__ void ask_next(void* answer, uint64_t* bar) {
    barrier_expect(bar, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];\n" ::"r"(smem_addr(answer)),
                 "r"(smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ bool read_next(const void* answer, uint32_t& block) {
    uint32_t ok, x;
    asm volatile(
        "{\n .reg .pred p;\n .reg .b128 h;\n ld.shared.b128 h, [%2];\n"
        " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n selp.u32 %0, 1, 0, p;\n mov.u32 %1, 0;\n"
        " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n}\n"
        : "=r"(ok), "=r"(x)
        : "r"(smem_addr(answer))
        : "memory");
    block = x;
    return ok != 0;
}

// BOXES: 64-column boxes of a row (1: dim <= 64, 2: dim <= 128).
// Work: 4 * dim operations per query head and visible pair.  Measured: one
// prompt of 16,384 tokens, 16/4 heads of 128, 1.02 to 1.05 ms run after run
// under the power cap (1.05 to 1.08 PFLOP/s; a large matrix product reaches 1.38
// there), 0.89 ms in a burst (1.24 of 1.65); 13 prompts of 7,196 tokens in all,
// 32/8 heads, 109 us (0.62); 24 tokens 7 us.  On long prompts the tensor pipe is
// busy 53% of the cycles and the exponentials' pipe 53%: at 8,192 tokens a pair
// of tiles takes 3,820 clocks with all that goes with it, its products 2,048
// and its exponentials, 32,768 at 16 a clock, 2,048 as well.  What bounds it is
// the chain S -> weights -> P V of each tile, which only the other tile hides.
// On short ones it is also each item's last tile, with hidden keys (3,800
// clocks), and its outputs (3,700).  Not kept, at 16,384 tokens (bursts) and
// the 13 prompts: two blocks of one tile an SM 1.12 ms and 130 us; weights
// handed over in halves 1.03 ms; scores in halves too, the next ones made
// meanwhile, 1.16 ms and 120 us; part of the exponentials as a polynomial,
// slower at every share; outputs by tensor copies 115 us.  With the copying
// warp also finding items and looking at hidden values, and items taken one
// ahead, the 13 prompts took 117 us and 11 of 3,888 tokens 39 (now 29).
template <typename T, int BOXES>
__global__ void __launch_bounds__(kThreads, 1) k_prompt(const __grid_constant__ PromptArgs a) {
    extern __shared__ unsigned char raw_smem[];
    unsigned char* const smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t{1023});
    constexpr int kStages = kStagesOf<BOXES>, kTileBytes = BOXES * kBoxBytes;
    unsigned char* const ring = smem + 2 * kTileBytes;
    unsigned char* const staging = smem + (2 + kStages) * kTileBytes;
    Control& ctl = *reinterpret_cast<Control*>(staging + kStagingBytes);
    const bs_prompt_attention_desc& d = a.d;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == 9 && lane < 3) {
        const CUtensorMap* map = lane == 0 ? &a.q : lane == 1 ? &a.k : &a.v;
        if (lane == 0 || d.total_k) asm volatile("prefetch.tensormap [%0];\n" ::"l"(map) : "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_addr(&ctl.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            barrier_init(&ctl.q_full[t], 1);
            barrier_init(&ctl.q_empty[t], 1);
            barrier_init(&ctl.s_full[t], 1);
            barrier_init(&ctl.p_full[t], 4);
            barrier_init(&ctl.o_full[t], 1);
            barrier_init(&ctl.item_full[t], 1);
            barrier_init(&ctl.item_empty[t], 11);
        }
        barrier_init(&ctl.done, 1);
        barrier_init(&ctl.next_full, 1);
        barrier_init(&ctl.asked, 1);
        for (int s = 0; s < kStages; ++s) {
            barrier_init(&ctl.full[s], 1);
            barrier_init(&ctl.empty[s], 1);
            barrier_init(&ctl.raw[s], 1);
        }
        ctl.keep[0] = ctl.keep[1] = ctl.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = ctl.tmem;
    cudaGridDependencySynchronize();       // nothing before this reads or writes a caller's memory

    // A bounded wait.  Once one has given up none waits any more: the warps
    // leave their loops together, what is in flight is waited for (`drain`,
    // bounded too), and nothing is stored.
    volatile uint32_t* const gave_up = &ctl.gave_up;
    auto wait = [&](uint64_t* bar, unsigned phase) {
        for (unsigned i = 0; i < a.polls && !*gave_up; ++i)
            if (barrier_test(bar, phase)) return;
        if (!*gave_up) {
            *gave_up = 1;
            atomicOr(a.errors, kMemErrWait);
        }
    };
    auto drain = [&](uint64_t* bar, unsigned phase) {
        for (unsigned i = 0; i < kPolls && !barrier_test(bar, phase); ++i) {}
    };
    // the next item for a warp that does not copy (not valid: the end), and
    // that it has read it
    auto next_item = [&](uint32_t i) -> const Item& {
        wait(&ctl.item_full[i & 1], (i >> 1) & 1);
        return ctl.item[i & 1];
    };
    auto item_read = [&](uint32_t i) {
        __syncwarp();
        if (lane == 0) barrier_arrive(&ctl.item_empty[i & 1]);
    };
    // keys that a token sees
    auto seen = [&](int32_t lq, int32_t lk, int32_t token) { return d.causal ? max(0, min(lk, token + lk - lq + 1)) : lk; };
    // columns of key tile j that a row seeing `most` keys sees, to a multiple of 16
    auto columns = [&](int32_t most, int32_t j) { return min(kRows, (most - j * kRows + 15) & ~15); };

    // value rows that a tile of keys has in sight of not all rows of an item
    auto look = [&](const Item& m, int32_t j) { return m.all_see - j * kRows < kRows; };

    if (warp == 11) {
        // ------------------------------------------------------------- items
        // Which sequence, tokens and key head a block of the grid stands for:
        // sequence b has the places base(b) .. base(b + 1), base(b) =
        // cu_q[b] / pair + b, enough for its ceil(len / pair) pairs of tiles;
        // the last pair, with the most keys, first.  A place is all key heads,
        // each all chunks.
        const uint32_t pair = 2 * a.tile_tokens;
        uint32_t block = blockIdx.x, next_phase = 0;
        bool more = true;
        for (uint32_t items = 0; more; ++items) {
            // The next block of the grid is asked for when all of this one's
            // copies are, not before: others may have nothing left to do.
            const uint32_t slot = items & 1;
            if (lane == 0) {
                wait(&ctl.item_empty[slot], ((items >> 1) & 1) ^ 1);
                if (items) wait(&ctl.asked, (items - 1) & 1);
            }
            __syncwarp();
            Item m;
            m.valid = 0;
            for (bool own = items == 0; more && !m.valid; own = false) {
                if (__any_sync(kFull, *gave_up != 0)) more = false;
                if (more && !own) {
                    // (only this block's own place and those not yet started are asked for)
                    if (lane == 0) {
                        ask_next(ctl.next, &ctl.next_full);
                        drain(&ctl.next_full, next_phase);
                    }
                    __syncwarp();
                    next_phase ^= 1;
                    more = read_next(ctl.next, block);
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    __syncwarp();
                }
                if (!more) break;
                m.chunk = block % a.chunks;
                m.kv_head = block / a.chunks % d.kv_heads;
                const uint32_t place = block / a.chunks / d.kv_heads;
                uint32_t lo = 0, hi = d.num_seqs;              // base(lo) <= place, the answer is in [lo, hi)
                while (hi - lo > 1) {                          // 32 probes at a time
                    const uint32_t step = (hi - lo + 31) / 32, at = lo + lane * step;
                    const bool below = at < hi && (at == 0 || static_cast<uint32_t>(d.cu_q[at]) / pair + at <= place);
                    const int last = 31 - __clz(__ballot_sync(kFull, below) | 1u);
                    hi = min(hi, lo + (last + 1) * step);
                    lo = lo + last * step;
                }
                const int32_t q1 = d.cu_q[lo + 1], k1 = d.cu_k[lo + 1];
                m.q0 = d.cu_q[lo];
                m.k0 = d.cu_k[lo];
                m.lq = q1 - m.q0;
                m.lk = k1 - m.k0;
                bool work = true;
                if (m.q0 < 0 || m.lq < 0 || static_cast<uint32_t>(q1) > d.total_q || m.k0 < 0 || m.lk < 0 || static_cast<uint32_t>(k1) > d.total_k) {
                    if (lane == 0) atomicOr(a.errors, kMemErrLength);
                    work = false;
                }
                const uint32_t pairs = work ? (m.lq + pair - 1) / pair : 0, local = place - (static_cast<uint32_t>(m.q0) / pair + lo);
                if (local >= pairs) continue;
                m.valid = 1;
                m.token0 = (pairs - 1 - local) * pair;
                m.all_see = seen(m.lq, m.lk, m.token0);
                int32_t tiles[2];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int32_t from = m.token0 + t * static_cast<int32_t>(a.tile_tokens);
                    const int32_t last = min(from + static_cast<int32_t>(a.tile_tokens), m.lq) - 1;
                    m.most_see[t] = last < from ? 0 : seen(m.lq, m.lk, last);
                    tiles[t] = (m.most_see[t] + kRows - 1) / kRows;
                }
                const int32_t n = max(tiles[0], tiles[1]), chunks = static_cast<int32_t>(a.chunks);
                m.first = static_cast<int32_t>(static_cast<int64_t>(n) * m.chunk / chunks);
                const int32_t end = static_cast<int32_t>(static_cast<int64_t>(n) * (m.chunk + 1) / chunks);
                m.end[0] = max(m.first, min(end, tiles[0]));
                m.end[1] = max(m.first, min(end, tiles[1]));
            }
            if (lane == 0 && !*gave_up) {
                ctl.item[slot] = m;
                barrier_arrive(&ctl.item_full[slot]);
            }
            __syncwarp();
        }
    } else if (warp == 10) {
        // ----------------------------------------- value rows that are hidden
        uint32_t loads = 0, raw_phases = 0;
        for (uint32_t i = 0;; ++i) {
            const Item m = next_item(i);
            if (__any_sync(kFull, *gave_up != 0) || !m.valid) break;
            item_read(i);
            const int32_t end = max(m.end[0], m.end[1]);
#pragma unroll 1
            for (int32_t j = max(m.first, m.all_see / kRows); j < end; ++j) {
                // value rows of this tile that not all rows see, and rows past the sequence
                const int32_t hidden = max(0, m.all_see - j * kRows), past = m.lk - j * kRows;
                const uint32_t stage = (loads + 2 * (j - m.first) + 1) % kStages;
                unsigned char* const dst = ring + stage * kTileBytes;
                wait(&ctl.raw[stage], (raw_phases >> stage) & 1);
                if (__any_sync(kFull, *gave_up != 0)) break;
                raw_phases ^= 1u << stage;
#pragma unroll 1
                for (int x = 0; x < kRows / 32; ++x) {
                    const int32_t r = 32 * x + lane;
                    uint32_t carry = 0;          // an exponent of all ones plus one carries over
                    if (32 * x + 31 >= hidden && 32 * x < past) {
#pragma unroll 1
                        for (int box = 0; box < BOXES; ++box)
#pragma unroll
                            for (int u = 0; u < 8; ++u) {
                                const uint4 w = *reinterpret_cast<const uint4*>(dst + box * kBoxBytes + r * 128 + ((u + lane) & 7) * 16);
                                constexpr uint32_t e = Type16<T>::kExponent, one = Type16<T>::kExponentOne;
                                carry |= ((w.x & e) + one) | ((w.y & e) + one) | ((w.z & e) + one) | ((w.w & e) + one);
                            }
                    }
                    const bool odd = (carry & 0x80008000u) && r >= hidden && r < past;
                    const uint32_t rows = __ballot_sync(kFull, odd);
                    if (lane == 0) ctl.not_finite[stage][x] = rows;
                    if (odd || r >= past) {
#pragma unroll 1
                        for (int box = 0; box < BOXES; ++box)
#pragma unroll
                            for (int u = 0; u < 8; ++u)
                                *reinterpret_cast<uint4*>(dst + box * kBoxBytes + r * 128 + ((u + lane) & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                __syncwarp();
                if (lane == 0) barrier_arrive(&ctl.full[stage]);
            }
            loads += 2 * (end - m.first);
        }
        // and, under the last item's epilogue, the ends of the lists (in every
        // block that runs; at its start this held up pieces of prompts by 1 us)
        if (lane < 4) {
            const int32_t end = (lane & 1 ? d.cu_k : d.cu_q)[lane < 2 ? 0 : d.num_seqs];
            if (static_cast<uint32_t>(end) != (lane < 2 ? 0 : lane & 1 ? d.total_k : d.total_q)) atomicOr(a.errors, kMemErrLength);
        }
        __syncwarp();
    } else if (warp == 9) {
        // ------------------------------------------------------------ copies
        // (by lane 0)
        uint32_t stage = 0, phase = 0, loads = 0, q_used[2] = {0, 0};
        uint32_t raw = 0, raw_phases = 0;      // a bit a stage: its last load is warp 10's, of which phase
        for (uint32_t i = 0;; ++i) {
            const Item m = next_item(i);
            if (__any_sync(kFull, *gave_up != 0) || !m.valid) break;
            item_read(i);
            const int32_t end = max(m.end[0], m.end[1]);
            if (lane == 0) {
                for (int32_t u = 0; u < 2 * (end - m.first); ++u) {          // keys, values of a tile
                    const int32_t j = m.first + (u >> 1);
                    wait(&ctl.empty[stage], phase ^ 1);
                    if (*gave_up) break;
                    uint64_t* bar = &ctl.full[stage];
                    raw &= ~(1u << stage);
                    if ((u & 1) && look(m, j)) {
                        bar = &ctl.raw[stage];
                        raw |= 1u << stage;
                        raw_phases ^= 1u << stage;
                    }
                    ++loads;
                    barrier_expect(bar, kTileBytes);
                    unsigned char* const dst = ring + stage * kTileBytes;
                    for (int x = 0; x < BOXES; ++x) load_box(dst + x * kBoxBytes, u & 1 ? &a.v : &a.k, 64 * x, m.kv_head, m.k0 + j * kRows, bar);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                    if (u) continue;
                    for (int t = 0; t < 2; ++t) {
                        if (m.end[t] == m.first) continue;
                        wait(&ctl.q_empty[t], (q_used[t] & 1) ^ 1);
                        if (*gave_up) break;
                        ++q_used[t];
                        barrier_expect(&ctl.q_full[t], BOXES * 128 * a.group * a.tile_tokens);
                        for (int x = 0; x < BOXES; ++x)
                            load_box(smem + t * kTileBytes + x * kBoxBytes, &a.q, 64 * x, m.kv_head * a.group,
                                     m.q0 + m.token0 + t * static_cast<int32_t>(a.tile_tokens), &ctl.q_full[t]);
                    }
                }
                barrier_arrive(&ctl.asked);
            }
            __syncwarp();
        }
        if (lane == 0) {
            // no copy may be in flight when the block ends
            for (int t = 0; t < 2; ++t)
                if (q_used[t]) drain(&ctl.q_full[t], (q_used[t] - 1) & 1);
            for (uint32_t i = loads > kStages ? loads - kStages : 0; i < loads; ++i) {
                const uint32_t s = i % kStages;
                if ((raw >> s) & 1) drain(&ctl.raw[s], ((raw_phases >> s) & 1) ^ 1);
                else drain(&ctl.full[s], (i / kStages) & 1);
            }
        }
        __syncwarp();
    } else if (warp == 8) {
        // ---------------------------------------------------- matrix products
        // (the whole warp runs the loop, one elected lane issues)
        constexpr uint32_t kCommon = 1u << 4 | Type16<T>::kFormat << 7 | Type16<T>::kFormat << 10 | (kRows >> 4) << 24;
        const uint32_t what_o = kCommon | 1u << 16 | static_cast<uint32_t>(d.dim >> 3) << 17;
        // what the lane does per instruction counts: operands are a base
        // and constants (16-byte units)
        const int steps = d.dim / 16;
        const uint64_t q_base = operand(smem_addr(smem), 16, 1024), k_base = operand(smem_addr(ring), 16, 1024);
        const uint64_t v_base = operand(smem_addr(ring), kBoxBytes, 1024);
        constexpr uint32_t kTileUnits = kTileBytes / 16, kBoxUnits = kBoxBytes / 16;
        // (by the elected lane)
        auto scores = [&](int t, uint32_t stage, int32_t cols) {
            const uint64_t q = q_base + t * kTileUnits, k = k_base + stage * kTileUnits;
            const uint32_t what_s = kCommon | static_cast<uint32_t>(cols >> 3) << 17;
#pragma unroll
            for (int i = 0; i < 4 * BOXES; ++i) {
                const uint32_t off = (i >> 2) * kBoxUnits + (i & 3) * 2;
                if (i < steps) mma_shared(tmem + t * 128, q + off, k + off, what_s, i > 0);
            }
            mma_commit(&ctl.s_full[t]);
        };
        auto values = [&](int t, uint32_t stage, bool add, int32_t cols) {
            const uint64_t v = v_base + stage * kTileUnits;
#pragma unroll
            for (int i = 0; i < kRows / 16; ++i) {
                if (16 * i >= cols) break;
                mma_tmem(tmem + 256 + t * 128, tmem + t * 128 + i * 8, v + i * 128, what_o, add || i > 0);
            }
        };
        auto full = [&](uint32_t i) { wait(&ctl.full[i % kStages], (i / kStages) & 1); };
        uint32_t loads = 0, q_used[2] = {0, 0}, p_used[2] = {0, 0};
        bool issued = false;
        for (uint32_t i = 0;; ++i) {
            const Item m = next_item(i);
            if (__any_sync(kFull, *gave_up != 0) || !m.valid) break;
            item_read(i);
            const int32_t end = max(m.end[0], m.end[1]);
            if (end == m.first) continue;
            issued = true;
            full(loads);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (m.end[t] == m.first) continue;
                wait(&ctl.q_full[t], q_used[t]++ & 1);
                fence_after();
                const int32_t cols = columns(m.most_see[t], m.first);
                if (elected()) {
                    scores(t, loads % kStages, cols);
                    if (m.end[t] == m.first + 1) mma_commit(&ctl.q_empty[t]);
                }
                __syncwarp();
            }
            if (elected()) mma_commit(&ctl.empty[loads % kStages]);
            __syncwarp();
            for (int32_t j = m.first; j < end; ++j) {
                if (__any_sync(kFull, *gave_up != 0)) break;
                const uint32_t v_load = loads + 1, k_load = loads + 2;
                const uint32_t v_stage = v_load % kStages, k_stage = k_load % kStages;
                loads += 2;
                full(v_load);
                if (j + 1 < end) full(k_load);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (j >= m.end[t]) continue;
                    const int32_t cols = columns(m.most_see[t], j), next_cols = columns(m.most_see[t], j + 1);
                    const bool last = j + 1 == m.end[t];
                    wait(&ctl.p_full[t], p_used[t]++ & 1);
                    fence_after();
                    const bool add = j > m.first || ctl.keep[t];
                    if (elected()) {
                        values(t, v_stage, add, cols);
                        if (last) {
                            mma_commit(&ctl.o_full[t]);
                        } else {
                            scores(t, k_stage, next_cols);
                            if (j + 2 == m.end[t]) mma_commit(&ctl.q_empty[t]);
                        }
                    }
                    __syncwarp();
                }
                if (elected()) {
                    mma_commit(&ctl.empty[v_stage]);
                    if (j + 1 < end) mma_commit(&ctl.empty[k_stage]);
                }
                __syncwarp();
            }
        }
        // TMEM and the stages are in use until this
        if (issued) {
            if (elected()) mma_commit(&ctl.done);
            __syncwarp();
            drain(&ctl.done, 0);
        }
        __syncwarp();
    } else {
        // ----------------------------------------------------------- softmax
        const uint32_t t = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (warp & 3) * 32 << 16;                  // this warp's TMEM lanes
        const uint32_t s_at = tmem + t * 128 + lanes, o_at = tmem + 256 + t * 128 + lanes;
        const int32_t row_token = static_cast<int32_t>(t * a.tile_tokens + row / a.group);
        const bool in_tile = row < a.group * a.tile_tokens;
        const float scale = d.scale * 1.4426950408889634f;
        uint32_t s_used = 0, o_used = 0, loads = 0;
        for (uint32_t i = 0;; ++i) {
            // (what the loop does not need every time stays in shared memory
            // till the item is done: registers)
            const Item& item = next_item(i);
            if (__any_sync(kFull, *gave_up != 0) || !item.valid) break;
            const int32_t first = item.first, end = item.end[t], all_see = item.all_see;
            const bool real = in_tile && item.token0 + row_token < item.lq;
            const int32_t limit = real ? seen(item.lq, item.lk, item.token0 + row_token) : 0;
            float top = -INFINITY, sum = 0.f;       // top: of the unscaled scores, moved when a weight is past 2^8
            for (int32_t j = first; j < end; ++j) {
                wait(&ctl.s_full[t], s_used++ & 1);        // and the value product before it is done
                if (__any_sync(kFull, *gave_up != 0)) break;
                fence_after();
                const bool hides = (j + 1) * kRows > all_see;
                const int32_t left = limit - j * kRows;         // keys of this tile that the row sees
                const int chunks = hides ? (columns(item.most_see[t], j) + 31) / 32 : kRows / 32;
                int done = 0;           // quarters of the tile whose weights are made
                if (!hides && j > first) {
                    float s[2][32];
                    tmem_load32(s_at, s[0]);
#pragma unroll 1
                    for (; done < 4; done += 2) {
                        uint32_t p[kRows / 4];
                        float part;
                        const float high = weights64<T>(s_at + 32 * done, done == 0, s, scale, kLift<T> - top * scale, p, part);
                        if (__any_sync(kFull, real && high > kMost * kLifted<T>)) break;       // (rows that are none of the tile's hold anything)
                        sum += part;
                        tmem_store16(s_at + 16 * done, p);
                        tmem_store16(s_at + 16 * done + 16, p + 16);
                    }
                    if (done == 0) wait_loads32(s[0]);
                }
                if (done < 4) {
                    const float2 r = weights_with_care<T>(s_at, o_at, done, chunks, hides ? left : kRows, real, scale, j > first ? d.dim : 0,
                                                          make_float2(top, sum));
                    top = r.x;
                    sum = r.y;
                }
                wait_stores();
                bool keep = false;
                if (hides) {
                    // value rows that were cleared because they are not finite,
                    // for the query rows that see them
                    const uint32_t load = loads + 2 * (j - first) + 1, stage = load % kStages;
                    wait(&ctl.full[stage], (load / kStages) & 1);
                    if (__any_sync(kFull, *gave_up != 0)) break;
                    const uint32_t* odd = ctl.not_finite[stage];
                    keep = j == first && (odd[0] | odd[1] | odd[2] | odd[3]);
                    if (keep) {
                        const uint32_t zeros[16] = {};
                        for (int x = 0; x < d.dim; x += 16) tmem_store16(o_at + x, zeros);
                        wait_stores();
                    }
                    for (int w = 0; w < 4; ++w)
                        for (uint32_t rest = odd[w]; rest; rest &= rest - 1) {
                            const int r = 32 * w + __ffs(rest) - 1;
                            if (r >= 32 * chunks) break;       // seen by none of this tile
                            const float2 f = Type16<T>::unpack(tmem_load1(s_at + r / 2));
                            const float weight = r & 1 ? f.y : f.x;
                            const T* v = static_cast<const T*>(d.v) + (item.k0 + j * kRows + r) * d.v_stride[0] + item.kv_head * d.v_stride[1];
                            for (int x = 0; x < d.dim; x += 16) {
                                uint32_t o[16];
                                tmem_load16(o_at + x, o);
                                wait_loads16(o);
                                if (r < left)
#pragma unroll
                                    for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) + weight * static_cast<float>(v[x + k]));
                                __syncwarp();
                                tmem_store16(o_at + x, o);
                                wait_stores();
                            }
                        }
                }
                if (j == first && lane == 0) ctl.keep[t] = keep;
                fence_before();
                __syncwarp();
                if (lane == 0) barrier_arrive(&ctl.p_full[t]);
            }
            loads += 2 * (max(item.end[0], item.end[1]) - first);
            const bool any = end > first;
            if (any) {
                wait(&ctl.o_full[t], o_used++ & 1);
                fence_after();
            }
            const bool ok = !__any_sync(kFull, *gave_up != 0) && real;
            const uint64_t at = (static_cast<uint64_t>(item.q0) + item.token0 + row_token) * d.q_heads + item.kv_head * a.group + row % a.group;
            if (a.chunks > 1) {
                // a piece of the keys: unnormalised, to be joined
                const uint64_t slot = item.chunk * (static_cast<uint64_t>(d.total_q) * d.q_heads) + at;
                float* const out = ok ? a.part_o + slot * d.dim : nullptr;
                for (int x = 0; any && x < d.dim; x += 32) {
                    float o[32];
                    tmem_load32(o_at + x, o);
                    wait_loads32(o);
                    uint32_t u[32];
#pragma unroll
                    for (int k = 0; k < 32; ++k) u[k] = __float_as_uint(o[k]);
                    store_rows(u, staging + warp * 4096, out, x * 4, d.dim * 4);
                }
                if (ok) a.part_ml[slot] = make_float2(top * scale - kLift<T>, sum);
            } else {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                T* const out = ok ? static_cast<T*>(d.out) + at * d.dim : nullptr;
                for (int x = 0; x < d.dim; x += 64) {
                    uint32_t u[32];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float o[32];
                        tmem_load32(o_at + x + 32 * half, o);
                        wait_loads32(o);
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            u[16 * half + k] = any && sum != 0.f ? Type16<T>::pack(o[2 * k] * inv, o[2 * k + 1] * inv) : 0;
                    }
                    store_rows(u, staging + warp * 4096, out, x * 2, d.dim * 2);
                }
                if (ok && d.lse) d.lse[at] = sum == 0.f ? -INFINITY : top * d.scale + logf(sum * (1.f / kLifted<T>));
            }
            item_read(i);
            // the next item's first value product overwrites the outputs: it
            // waits for weights that this warp makes after these loads
            fence_before();
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
}

// One warp per row: joins the pieces of its keys, always in the same order.
// Bound by its traffic: four pieces of 15,900 rows of 96 in 9 us (2.7 TB/s).
__global__ void __launch_bounds__(128) k_prompt_join(const __grid_constant__ PromptArgs a) {
    const bs_prompt_attention_desc& d = a.d;
    const uint64_t rows = static_cast<uint64_t>(d.total_q) * d.q_heads, row = static_cast<uint64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const uint32_t lane = threadIdx.x & 31;
    cudaGridDependencySynchronize();       // in every block: what follows this kernel may count on both being done
    if (row >= rows) return;
    float2 ml[kMostChunks];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (uint32_t c = 0; c < kMostChunks; ++c) {
        ml[c] = c < a.chunks ? a.part_ml[c * rows + row] : make_float2(-INFINITY, 0.f);
        m = fmaxf(m, ml[c].x);
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float4 o[kMostChunks];
    const bool mine = lane * 4 < static_cast<uint32_t>(d.dim);
#pragma unroll
    for (uint32_t c = 0; c < kMostChunks; ++c)          // (a piece that saw nothing was not written)
        if (ml[c].y != 0.f && mine) o[c] = *reinterpret_cast<const float4*>(a.part_o + (c * rows + row) * d.dim + lane * 4);
#pragma unroll
    for (uint32_t c = 0; c < kMostChunks; ++c) {
        if (ml[c].y == 0.f || !mine) continue;
        const float w = exp2_fast(ml[c].x - m);
        acc.x += o[c].x * w, acc.y += o[c].y * w, acc.z += o[c].z * w, acc.w += o[c].w * w;
    }
#pragma unroll
    for (uint32_t c = 0; c < kMostChunks; ++c)
        if (ml[c].y != 0.f) l += ml[c].y * exp2_fast(ml[c].x - m);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (lane == 0 && d.lse) d.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    if (!mine) return;
    uint2 u;
    if (d.dtype == BS_F16) u = make_uint2(Type16<__half>::pack(acc.x * inv, acc.y * inv), Type16<__half>::pack(acc.z * inv, acc.w * inv));
    else u = make_uint2(Type16<__nv_bfloat16>::pack(acc.x * inv, acc.y * inv), Type16<__nv_bfloat16>::pack(acc.z * inv, acc.w * inv));
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(d.out) + row * d.dim + lane * 4) = u;
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                              CUtensorMapFloatOOBfill);

cudaError_t encoder(EncodeFn& out) {
    static std::atomic<EncodeFn> known{nullptr};       // (threads may look it up at once)
    EncodeFn fn = known.load();
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r);
        if (e != cudaSuccess) return e;
        if (r != cudaDriverEntryPointSuccess || !p) return cudaErrorNotSupported;
        known.store(fn = reinterpret_cast<EncodeFn>(p));
    }
    out = fn;
    return cudaSuccess;
}

// [tokens][heads][dim] with strides, read in boxes of 64 x heads x tokens.
cudaError_t tensor_map(CUtensorMap* map, const void* p, int32_t dtype, int32_t dim, uint32_t heads, uint32_t tokens,
                       const int64_t* stride, uint32_t box_heads, uint32_t box_tokens) {
    EncodeFn encode;
    cudaError_t e = encoder(encode);
    if (e != cudaSuccess) return e;
    const cuuint64_t extent[3] = {static_cast<cuuint64_t>(dim), heads, tokens};
    // a stride that only ever meets coordinate 0 may be any
    const cuuint64_t bytes[2] = {static_cast<cuuint64_t>(heads > 1 ? stride[1] * 2 : dim * 2),
                                 static_cast<cuuint64_t>(tokens > 1 ? stride[0] * 2 : dim * 2)};
    const cuuint32_t box[3] = {64, box_heads, box_tokens}, step[3] = {1, 1, 1};
    const CUresult r = encode(map, dtype == BS_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                              const_cast<void*>(p), extent, bytes, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

uint32_t tile_tokens(const bs_prompt_attention_desc& d) { return kRows / static_cast<uint32_t>(d.q_heads / d.kv_heads); }

// Pairs of tiles times key heads, at most.
uint64_t most_items(const bs_prompt_attention_desc& d) {
    return (d.total_q / (2 * tile_tokens(d)) + static_cast<uint64_t>(d.num_seqs)) * d.kv_heads;
}

// Pieces that the keys are cut into, by what was measured: a block is busy
// about 4 us an item and 2 us a tile of keys, a join takes 4 us and its
// traffic (4 TB/s); the time is that of the longest item, or of all of them
// over the SMs.  Lengths are not known here: the longest sequence is taken to
// have twice the average's keys, a query half of its own piece of prompt.
// Measured, in 1, 2, 4, 8 pieces (when items were still taken one ahead): 3
// sequences of 12/4 heads, 8,000 keys 77, 58, 55, 56 us (4 taken); 8 of one key
// head, 5,800 keys 72, 46, 32, 30 (4); 16 short ones over 6,500 keys 39, 27, 21,
// 23 (4); 1,109 tokens of 18/3 heads 28, 36, 37, 44 (1).
uint32_t chunks_of(const bs_prompt_attention_desc& d, const MemoryDevice& dev) {
    const double items = static_cast<double>(most_items(d)), seqs = d.num_seqs ? d.num_seqs : 1;
    const double total = d.total_k / static_cast<double>(kRows), most = std::min(total, 2 * total / seqs) + 1;
    const double mean = (d.total_k - d.total_q / 2.) / (kRows * seqs) + 1;
    const double traffic = 2. * d.total_q * d.q_heads * (d.dim * 4 + 8) / 4e6;      // us a piece
    uint32_t best = 1;
    double least = 0;
    for (uint32_t n = 1; n <= kMostChunks; n *= 2) {
        const double time = std::max(4 + 2 * most / n, items * n / dev.num_sms * (4 + 2 * mean / n)) + (n > 1 ? 4 + traffic * n : 0);
        if (n == 1 || time < least) {
            least = time;
            best = n;
        }
    }
    return best;
}

template <typename T, int BOXES>
cudaError_t launch(const PromptArgs& a, cudaStream_t stream) {
    cudaError_t e = cudaFuncSetAttribute(k_prompt<T, BOXES>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem<BOXES>);
    if (e != cudaSuccess) return e;
    const uint64_t blocks = most_items(a.d) * a.chunks;
    if (blocks > 0x7fffffffu) return cudaErrorInvalidConfiguration;
    e = launch_after(k_prompt<T, BOXES>, dim3(static_cast<unsigned>(blocks)), kThreads, kSmem<BOXES>, stream, a);
    if (e != cudaSuccess || a.chunks == 1) return e;
    const uint64_t rows = static_cast<uint64_t>(a.d.total_q) * a.d.q_heads;
    return launch_after(k_prompt_join, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, stream, a);
}

}  // namespace

size_t prompt_attention_scratch(const bs_prompt_attention_desc& d, const MemoryDevice& dev) {
    const uint32_t chunks = chunks_of(d, dev);
    return chunks == 1 ? 0 : static_cast<size_t>(chunks) * d.total_q * d.q_heads * (d.dim * 4 + 8);
}

cudaError_t launch_prompt_attention(const bs_prompt_attention_desc& d, const MemoryDevice& dev, cudaStream_t stream) {
    PromptArgs a{};
    a.d = d;
    a.errors = dev.errors;
    a.polls = wait_polls();
    a.group = d.q_heads / d.kv_heads;
    a.tile_tokens = tile_tokens(d);
    a.chunks = chunks_of(d, dev);
    a.part_o = static_cast<float*>(d.workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + static_cast<size_t>(a.chunks) * d.total_q * d.q_heads * d.dim);
    cudaError_t e = tensor_map(&a.q, d.q, d.dtype, d.dim, d.q_heads, d.total_q, d.q_stride, a.group, a.tile_tokens);
    // (no keys: nothing is read through the maps)
    if (e == cudaSuccess && d.total_k) e = tensor_map(&a.k, d.k, d.dtype, d.dim, d.kv_heads, d.total_k, d.k_stride, 1, kRows);
    if (e == cudaSuccess && d.total_k) e = tensor_map(&a.v, d.v, d.dtype, d.dim, d.kv_heads, d.total_k, d.v_stride, 1, kRows);
    if (e != cudaSuccess) return e;
    if (d.dtype == BS_F16) return d.dim <= 64 ? launch<__half, 1>(a, stream) : launch<__half, 2>(a, stream);
    return d.dim <= 64 ? launch<__nv_bfloat16, 1>(a, stream) : launch<__nv_bfloat16, 2>(a, stream);
}

}  // namespace bsb
