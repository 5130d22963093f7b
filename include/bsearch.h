/*
 * bsearch.h -- C ABI of the B200 graph beam-search library
 * (libbsearch_b200.so).  Plain C types only: pointers, sizes, status codes.
 *
 * The reference (SophiaSun18/beam_search_collab) has no library boundary: its
 * gpu_cli main() builds device copies of the graph and codebook and calls
 * templated launchers directly.  Each entry point below names the reference
 * piece it replaces (reference-relative file:line), so a host program written
 * against the reference structure can bind this library one to one.
 *
 * Threading: an index is bound to one CUDA device.  bs_search may run
 * concurrently on different streams; each call uses its own scratch.
 * Errors: every call returns a bs_status; bs_last_error() gives the message
 * of the calling thread's last failure.  The library never exits the process.
 */
#ifndef BSEARCH_H
#define BSEARCH_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define BS_API __attribute__((visibility("default")))
#else
#define BS_API
#endif

#define BS_NO_NODE 0xFFFFFFFFu

typedef enum bs_status {
    BS_OK = 0,
    BS_ERR_INVALID_ARGUMENT = 1, /* bad pointer, size, mode or config        */
    BS_ERR_UNSUPPORTED = 2,      /* valid but outside this build's limits     */
    BS_ERR_IO = 3,               /* file missing, short or malformed          */
    BS_ERR_OUT_OF_MEMORY = 4,    /* host or device allocation failed          */
    BS_ERR_CUDA = 5,             /* CUDA runtime error                        */
    BS_ERR_KERNEL = 6            /* a kernel reported an internal error flag  */
} bs_status;

typedef struct bs_index bs_index;

/* Host-resident graph: num_nodes rows of dim floats and of degree node ids
 * (the CPUGraph fields of reference include/cpu_graph.hpp:24-28). */
typedef struct bs_graph_desc {
    uint64_t num_nodes;
    int32_t dim;
    int32_t degree;
    const float* vectors;     /* [num_nodes][dim]    */
    const uint32_t* edges;    /* [num_nodes][degree]; NULL: no graph yet (for
                                 bs_index_build_graph)                        */
} bs_graph_desc;

/* Host-resident RaBitQ data (CPURabitqData, reference include/rabitq.hpp:25-35).
 * padded_dim = next power of two >= dim; words_per_plane = padded_dim/32. */
typedef struct bs_rabitq_desc {
    uint32_t entry_point;     /* BS_NO_NODE: none stored                      */
    int32_t padded_dim;
    const uint32_t* codes;    /* [num_nodes][degree][padded_dim/32]            */
    const float* factors;     /* [num_nodes][3][degree] triple_x|factor_dq|factor_vq */
    const float* signs;       /* [padded_dim]                                 */
} bs_rabitq_desc;

/* Search configuration: the "search" object of the reference JSON config
 * (src/gpu_cli.cu:414-452).  mode is one of "base", "warp1", "warp2",
 * "warp4", "warp8", "bwarp1", "bwarp2", "bwarp4", "bwarp8", "rabitq". */
typedef struct bs_search_params {
    const char* mode;
    int32_t K;
    uint32_t topk_size;
    uint32_t filter_capacity;
    int32_t max_iterations;
    int32_t reset_interval;
    uint32_t entry_point;     /* BS_NO_NODE: the index's default entry        */
} bs_search_params;

typedef struct bs_stats {
    uint64_t expansions;      /* nodes expanded, all queries                  */
    uint64_t distances;       /* exact L2 distances computed                  */
    uint64_t estimates;       /* RaBitQ estimates computed                    */
    uint64_t rerank;          /* exact distances in the RaBitQ final rerank   */
    uint32_t error_flags;     /* kernel-side error bits (0 = none)            */
    uint32_t entry_point;     /* entry node the search used                   */
    uint32_t integer_exact;   /* 1: integer-exact distance path was used       */
    uint32_t row_bytes;       /* bytes per base row as stored on the device   */
    uint32_t block_bytes;     /* bytes per node block copied per expansion
                                 (neighbourhood block, or the RaBitQ node
                                 block; 0: the gather layout was used)       */
    uint32_t warps_per_query; /* warps that worked on each query: 1 for the
                                 warp-per-query kernels, 2 or 4 for mode base
                                 over neighbourhood blocks (one thread block
                                 per query)                                  */
} bs_stats;

/* Fills the reference defaults: mode "base", K 100, topk_size 256,
 * filter_capacity 1024, max_iterations 1024, reset_interval 16
 * (src/gpu_cli.cu:415-452). */
BS_API void bs_search_params_default(bs_search_params* p);

/* Replaces GPUGraph::GPUGraph(const CPUGraph&) (include/gpu_graph.cuh:126-141):
 * copies vectors and edges to `device`.  The caller keeps its host arrays. */
BS_API bs_status bs_index_create(const bs_graph_desc* desc, int device, bs_index** out);

/* Replaces CPUGraph::load (include/cpu_graph.hpp:125-173) + GPUGraph: reads
 * graph.bin (int32 n, int32 degree, uint32[n*degree]) and base .fvecs. */
BS_API bs_status bs_index_load(const char* graph_bin, const char* base_fvecs, int device,
                               bs_index** out);

/* Replaces GPURabitq::GPURabitq(const CPURabitqData&) (include/rabitq.cuh:84-104). */
BS_API bs_status bs_index_attach_rabitq(bs_index* index, const bs_rabitq_desc* desc);

/* Replaces load_rabitq_codebook (include/rabitq.hpp:49-97) + GPURabitq. */
BS_API bs_status bs_index_load_codebook(bs_index* index, const char* codebook_path);

/* Replaces the reference codebook builder (src/build_rabitq.cpp:120-285),
 * on the GPU over the index's own rows and graph: sign table from
 * std::mt19937_64(seed) as build_rabitq -seed, medoid entry point, per-edge
 * codes and factors with the same arithmetic (bit-identical).  The result is
 * attached to the index as bs_index_load_codebook would attach it; when
 * out_path is non-NULL it is also written there in the codebook.bin format,
 * byte-identical to the reference tool's file.  entry_out (nullable)
 * receives the medoid.  Needs padded_dim >= 32 (dim > 16). */
BS_API bs_status bs_index_build_codebook(bs_index* index, uint32_t seed, const char* out_path,
                                         uint32_t* entry_out);

BS_API bs_status bs_index_info(const bs_index* index, uint64_t* num_nodes, int32_t* dim,
                               int32_t* degree);

/* Parameters of the graph builder (the reference build_graph's options,
 * src/build_graph.cpp:22-31; --metric ip is not supported). */
typedef struct bs_graph_build_params {
    int32_t beam_width;       /* build beam width L (reference default 128)  */
    float alpha;              /* pruning alpha >= 1 (reference default 2.0)  */
    uint32_t seed;            /* insertion-order shuffle seed (default 1234) */
} bs_graph_build_params;

/* Replaces the reference Vamana builder build_graph (src/build_graph.cpp:
 * 255-397), on the GPU over the index's own rows: the same insertion order
 * (std::mt19937(seed) + std::shuffle from the same standard library), batch
 * schedule, greedy searches, robust prune and reverse edges, so the result is
 * the reference's graph.bin.  The index's degree is the out-degree R (<= 64);
 * create the index with edges == NULL.  The new adjacency replaces the
 * index's; a codebook and the neighbourhood blocks built for the old one are
 * dropped.  edges_out (host, nullable) receives [num_nodes][degree]. */
BS_API bs_status bs_index_build_graph(bs_index* index, const bs_graph_build_params* params, uint32_t* edges_out);

/* Replaces compute_entry_point (src/gpu_cli.cu:55-83): row nearest to the
 * float centroid, same arithmetic, computed on the GPU and cached. */
BS_API bs_status bs_index_entry_point(bs_index* index, uint32_t* entry);

/* The codebook's stored entry (medoid), BS_NO_NODE when absent or when no
 * codebook is attached (reference src/gpu_cli.cu:436-437). */
BS_API bs_status bs_index_rabitq_entry(const bs_index* index, uint32_t* entry);

/* Replaces the ground-truth files the reference reads (src/gpu_cli.cu:379-381,
 * made offline by script/unpack.py): the exact k nearest rows of every query
 * by brute force over all the index's rows, ordered by (distance, id), with
 * the search's own distances (the reference's sequential fp32 sums, or exact
 * integer sums for byte rows and integer queries).  k <= 256.  queries
 * [nq][dim], ids [nq][k] and dists [nq][k] (nullable) may be host or device
 * pointers; with any host buffer the call returns when the results are in
 * place, otherwise it is asynchronous on `stream`. */
BS_API bs_status bs_ground_truth(bs_index* index, const float* queries, uint32_t nq, uint32_t k, uint32_t* ids,
                                 float* dists, void* stream);

/* No counterpart in the reference.  Builds the device layout the exact and
 * Bloom modes search fastest on (one contiguous neighbourhood block per node:
 * its adjacency row and its neighbours' rows, one bulk copy per expansion;
 * C2: 4.2 KB per node), when it fits in 40% of the free device memory.
 * bs_search does this on its first exact or Bloom search; call it at set-up
 * to take that cost out of the first search, or before bs_search_no_alloc,
 * which never builds it (until then it searches the plain layout, with the
 * same results).  A RaBitQ-only index never needs it.  "rabitq" checks that
 * a codebook is attached (its node blocks are built when it is attached). */
BS_API bs_status bs_index_prepare(bs_index* index, const char* mode);

/* No counterpart in the reference, whose kernels have no error channel.
 * Every search kernel on this index also ORs its error bits (the ones
 * bs_search reports as BS_ERR_KERNEL) into a word held by the index, so that a
 * caller of asynchronous searches -- bs_search with device buffers and no
 * stats, or bs_search_no_alloc -- can collect them later: this call copies
 * the word to *flags and clears it, ordered after the work already queued on
 * `stream`, and synchronises `stream`.  Bits: 1 a visited-table probe ran the
 * whole table, 2 a RaBitQ visited table overflowed, 4 a block copy's wait
 * gave up, 8 that copy never landed.  0 means no kernel reported an error. */
BS_API bs_status bs_index_take_errors(bs_index* index, void* stream, uint32_t* flags);

BS_API void bs_index_destroy(bs_index* index);

/* Replaces run_base / run_warp / run_rabitq and their kernels
 * (src/gpu_cli.cu:87-349): searches nq queries ([nq][dim] floats), writes
 * ids [nq][K] (BS_NO_NODE past the end of the beam) and, when `dists` is not
 * NULL, the matching squared L2 distances.  `queries`, `ids` and `dists` may
 * each be host or device pointers.  Pageable host buffers are copied inside
 * the call; page-locked host buffers mapped into the index's device (e.g.
 * cudaHostAlloc / cudaMallocHost on that device) are read and written in
 * place by the search kernel, so their transfers overlap the search.  With
 * any host buffer the call returns only when the results are in place.  With device
 * buffers only and stats == NULL the call is asynchronous on `stream`
 * (a cudaStream_t; NULL = legacy default stream). */
BS_API bs_status bs_search(bs_index* index, const bs_search_params* params, const float* queries,
                           uint32_t nq, uint32_t* ids, float* dists, bs_stats* stats,
                           void* stream);

/* No counterpart in the reference.  The same search as bs_search for the
 * exact and Bloom modes (every mode but "rabitq"), for callers that cannot
 * allocate device memory while they run -- a process that reserves the GPU's
 * memory at start-up and forbids later allocations (fixed-budget serving, a
 * plugin inside a runtime that owns all device memory), or a loop where an
 * allocation's possible blocking or failure is not acceptable.  It calls no
 * cudaMalloc/cudaFree or allocating routine: the kernel's scratch (work
 * counter, statistics, error flags; the centroid when the entry point is
 * first computed) lives in one 16 KiB file-scope device array that every GPU
 * loading the library holds until the process exits.
 *   - queries, ids and dists (NULL allowed) must be device pointers;
 *   - nq <= 2^31; "rabitq" is rejected (its never-forgetting visited sets
 *     need a bitmap over all node ids per resident warp, far more than the
 *     fixed scratch), as is computing the entry point for dim > 4028 (pass
 *     entry_point or call bs_index_entry_point first);
 *   - it searches the layout the index already has: the neighbourhood blocks
 *     once bs_index_prepare (or an exact or Bloom bs_search) built them, else
 *     the plain layout, with the same results;
 *   - the first call on a device looks up the array's device address, and if
 *     neither entry_point nor a cached entry is available it computes the
 *     entry point and synchronises `stream`; make that first call before any
 *     stream capture;
 *   - all calls share the one array, which keeps the last call's contents
 *     (the counters are cleared at the start of every call): calls that
 *     overlap on the GPU race, so serialise them (one stream, or events);
 *   - asynchronous on `stream`; no statistics are returned (kernel error
 *     bits reach the index's error word: bs_index_take_errors). */
BS_API bs_status bs_search_no_alloc(bs_index* index, const bs_search_params* params, const float* queries,
                                    uint32_t nq, uint32_t* ids, float* dists, void* stream);

/* No counterpart in the reference, which searches one index on one GPU: the
 * merge step of a sharded index (one shard per GPU, each with its own graph
 * over its own rows; every query searched on every shard).  Input: the
 * shards' result lists gathered into dists[shards][nq][K] and
 * ids[shards][nq][K] (shard-local ids, BS_NO_NODE past the end, each list
 * ascending by (distance, id) as bs_search returns it), device pointers on
 * the current device.  Output: out_ids[nq][K_out] (and out_dists when not
 * NULL), the K_out smallest (distance, global id) entries over all shards,
 * global id = local id + id_offsets[shard] (a host array of `shards` values;
 * global ids must stay below 0xffffffff), BS_NO_NODE / FLT_MAX past the end.
 * shards <= 32, K_out <= shards * K.  Asynchronous on `stream`. */
BS_API bs_status bs_merge_shards(const float* dists, const uint32_t* ids, uint32_t shards, uint32_t nq,
                                 uint32_t K, const uint32_t* id_offsets, uint32_t K_out, uint32_t* out_ids,
                                 float* out_dists, void* stream);

/* ---------------------------------------------------------------------------
 * Token memory: the attention of a language model whose context is searched.
 * No counterpart in the reference.  Keys and values of the tokens a model has
 * read live in an 8-bit cache; tokens that the cache gives up are rows for an
 * index (bs_index_create), found again by bs_search.
 *
 * All pointers are device pointers on the current device; every call is
 * asynchronous on `stream` and allocates nothing: scratch is the caller's, of
 * the size the matching *_workspace call gives (0 bytes: NULL is fine).
 * Lengths, tables and positions are read on the device, so none of the calls
 * waits for them and all can be captured in a CUDA graph.  What only the
 * device can see to be wrong (a block id outside the cache, lengths outside
 * their buffers) is not read or written; it sets an error bit that
 * bs_memory_take_errors returns.
 *
 * dim is a multiple of 16 up to 128.  q, k and v have strides in elements
 * between tokens and between heads; they and the base address are multiples
 * of 16 bytes (0, a row or head for all, too, but not in bs_prompt_attention),
 * the last dimension is contiguous.  Outputs are contiguous; out, the values
 * that bs_cache_read writes and workspaces are 16-byte aligned, other 32-bit
 * buffers 4-byte.  scale is positive and finite. */
typedef enum bs_dtype { BS_F32 = 0, BS_F16 = 1, BS_BF16 = 2 } bs_dtype;

/* The 8-bit cache: blocks of `block` tokens (16, 32, 64 or 128).  A value is
 * code * scale, one scale per block and head. */
typedef struct bs_token_cache {
    int8_t* k;                /* [num_blocks][kv_heads][block][dim], 16-byte aligned */
    int8_t* v;
    float* k_scale;           /* [num_blocks][kv_heads]                       */
    float* v_scale;
    uint32_t num_blocks;
    int32_t kv_heads;
    int32_t block;
    int32_t dim;
} bs_token_cache;

/* Attention of packed prompts.  Sequence b's queries are rows cu_q[b] ..
 * cu_q[b+1] of q and its keys rows cu_k[b] .. cu_k[b+1] of k and v; both lists
 * start at 0, ascend and end at total_q and total_k (else error bit 4 is set,
 * and the rows of out and lse that no sequence has, or one whose lists are
 * wrong, hold anything).  With `causal`, query i
 * of Lq sees the keys j <= i + Lk - Lq (the last query sees all), else all.
 * Query head h goes with key head h / (q_heads / kv_heads).
 *   s_j = scale * <q, k_j>,  lse = log sum_j exp(s_j),  out = sum_j exp(s_j - lse) v_j
 * A query that sees no key gives out = 0, lse = -infinity.
 * Every wait inside the kernel is bounded; one that gives up stores nothing and
 * sets error bit 1.  The environment variable BSEARCH_WAIT_POLLS, read at each
 * call, is the bound as a number of polls (default 4194304; 0, for tests of
 * this path: the first wait gives up; what is not a number is ignored). */
typedef struct bs_prompt_attention_desc {
    const void* q;            /* [total_q][q_heads][dim]                      */
    const void* k;            /* [total_k][kv_heads][dim]                     */
    const void* v;
    void* out;                /* [total_q][q_heads][dim], type dtype          */
    float* lse;               /* [total_q][q_heads], or NULL                  */
    int64_t q_stride[2];      /* elements from token to token, head to head   */
    int64_t k_stride[2];
    int64_t v_stride[2];
    const int32_t* cu_q;      /* [num_seqs + 1]                               */
    const int32_t* cu_k;
    void* workspace;
    size_t workspace_bytes;
    uint32_t total_q, total_k, num_seqs;
    int32_t q_heads, kv_heads, dim;
    int32_t dtype;            /* BS_F16 or BS_BF16                            */
    int32_t causal;
    float scale;
} bs_prompt_attention_desc;

BS_API bs_status bs_prompt_attention(const bs_prompt_attention_desc* desc, void* stream);
BS_API bs_status bs_prompt_attention_workspace(const bs_prompt_attention_desc* desc, size_t* bytes);

/* Appends tokens: rows cu[b] .. cu[b+1] of k and v become positions start[b],
 * start[b] + 1, ... of sequence b, whose position p lies in block
 * table[b][p / block].  A block's scale is max|x| * (1 / 127) over its new tokens
 * (0 when that maximum is below 1e-30), and where it holds earlier tokens
 * (positions below start[b]) at least the scale it has; those tokens' codes
 * are rounded anew when the scale grows.  code = rint(x * (1 / scale))
 * (+-127 at most).  Values must be finite.  A block is written by one
 * sequence of a call only. */
typedef struct bs_cache_write_desc {
    const void* k;            /* [total][kv_heads][dim]                       */
    const void* v;
    int64_t k_stride[2];
    int64_t v_stride[2];
    const int32_t* cu;        /* [num_seqs + 1]                               */
    const int32_t* table;     /* [num_seqs][table_width]                      */
    const int32_t* start;     /* [num_seqs]                                   */
    uint32_t total, num_seqs, table_width;
    int32_t dtype;
} bs_cache_write_desc;

BS_API bs_status bs_cache_write(const bs_token_cache* cache, const bs_cache_write_desc* desc, void* stream);

/* Reads values back (as rows for an index, for instance): out[b][h][i] is the
 * value at position positions[b][h][i] of sequence b (position_head_stride 0:
 * the same positions for every head).  Zeros where the position is negative
 * or not below lens[b]. */
typedef struct bs_cache_read_desc {
    const int32_t* table;     /* [num_seqs][table_width]                      */
    const int32_t* lens;      /* [num_seqs]                                   */
    const int32_t* positions; /* [num_seqs][heads or 1][count]                */
    int64_t position_seq_stride, position_head_stride;
    void* k;                  /* [num_seqs][kv_heads][count][dim], or NULL    */
    void* v;                  /* or NULL                                      */
    uint32_t num_seqs, table_width, count;
    int32_t dtype;            /* BS_F32, BS_F16 or BS_BF16                    */
} bs_cache_read_desc;

BS_API bs_status bs_cache_read(const bs_token_cache* cache, const bs_cache_read_desc* desc, void* stream);

/* Attention over the cache, over chosen blocks of it and over shared tokens
 * (bs_cache_attention, bs_block_attention, bs_shared_attention) rounds twice
 * before its output: elements of a bf16 query below 2^-29 of its row's largest
 * lose bits (f16 queries are exact), and a weight times its value scale meets the
 * codes as f16, off by 2^-11 of itself or, where that is more, by 2^-29 of the
 * row's largest such product (value scales count down to 2^-60 of the largest).
 * Scores, sums of weights, lse and mass are 32-bit, of weights not rounded. */

/* Attention over the cache.  Sequence b holds lens[b] tokens, the last
 * `queries` of which are the query tokens: query i sees the positions below
 * lens[b] - queries + 1 + i (one query: all).  out, lse as in
 * bs_prompt_attention.  With out_mass, the weight that each cached token got,
 *   out_mass[b][h][j] = mass[b][h][j] + sum over the queries and the heads of
 *                       key head h of exp(s_j - lse)        (j < lens[b])
 * and 0 for lens[b] <= j < mass_width; mass may be NULL (zeros) or out_mass.
 * Weights of tokens at and past mass_width have no place: they are left out,
 * and error bit 4 is set.  With out_mass the workspace holds a score of every
 * query row and place of the tables, in use or not: 4 * num_seqs * queries *
 * q_heads * table_width * block bytes (32 sequences of 32 heads over tables of
 * 131,072 tokens: 0.54 GB). */
typedef struct bs_cache_attention_desc {
    const void* q;            /* [num_seqs][queries][q_heads][dim]            */
    int64_t q_stride[3];      /* elements from sequence to sequence, token to token, head to head */
    const int32_t* table;     /* [num_seqs][table_width]                      */
    const int32_t* lens;      /* [num_seqs], at most table_width * block      */
    void* out;                /* [num_seqs][queries][q_heads][dim], type dtype */
    float* lse;               /* [num_seqs][queries][q_heads], or NULL        */
    const float* mass;        /* [num_seqs][kv_heads][mass_width], or NULL    */
    float* out_mass;          /* the same shape, or NULL                      */
    void* workspace;
    size_t workspace_bytes;
    uint32_t num_seqs, table_width, mass_width;
    int32_t queries, q_heads;
    int32_t dtype;            /* BS_F16 or BS_BF16                            */
    float scale;
} bs_cache_attention_desc;

BS_API bs_status bs_cache_attention(const bs_token_cache* cache, const bs_cache_attention_desc* desc, void* stream);
BS_API bs_status bs_cache_attention_workspace(const bs_token_cache* cache, const bs_cache_attention_desc* desc,
                                              size_t* bytes);

/* Eviction by accumulated attention weight.  Of a sequence of n = lens[b] >
 * budget tokens stay, for each head apart: the first `sinks`, the last
 * `recent`, and of the others the budget - sinks - recent with the largest
 * mass (ties: the lower position; NaN counts as largest); of a shorter one
 * all.  The tokens that stay move, in order, into the blocks of new_table,
 * which must not be blocks of any sequence of `table`.  kept[b][h][i] is the
 * old position of new position i (-1 past the end), new_mass its mass (0 past
 * the end), new_lens[b] = min(lens[b], budget).  A new block's scale is the
 * largest of its tokens' old scales; codes become rint(code * (old / new)).
 * The workspace is not used yet: bs_cache_evict_workspace gives 0. */
typedef struct bs_cache_evict_desc {
    const float* mass;        /* [num_seqs][kv_heads][mass_width]             */
    const int32_t* table;     /* [num_seqs][table_width]                      */
    const int32_t* lens;      /* [num_seqs], at most mass_width               */
    const int32_t* new_table; /* [num_seqs][new_table_width]                  */
    int32_t* kept;            /* [num_seqs][kv_heads][budget]                 */
    int32_t* new_lens;        /* [num_seqs]                                   */
    float* new_mass;          /* [num_seqs][kv_heads][budget]                 */
    void* workspace;
    size_t workspace_bytes;
    uint32_t num_seqs, table_width, new_table_width, mass_width;
    int32_t budget, sinks, recent;
} bs_cache_evict_desc;

BS_API bs_status bs_cache_evict(const bs_token_cache* cache, const bs_cache_evict_desc* desc, void* stream);
BS_API bs_status bs_cache_evict_workspace(const bs_token_cache* cache, const bs_cache_evict_desc* desc, size_t* bytes);

/* Norm and rotary position of queries and keys in one pass.  Each head's row x
 * of q (and of k, with its own weight) becomes
 *   y = x * w / sqrt(mean(x^2) + eps)        (no weight: y = x)
 * and of its first `rotary` dimensions the pairs j < rotary / 2, (a, b) =
 * (y[j], y[j + rotary / 2]) or, interleaved, (y[2 j], y[2 j + 1]), become
 *   amplitude * (a cos t - b sin t, b cos t + a sin t),  t = position * freqs[j],
 * rounded once, at the end, from 32-bit floats.  An angle keeps its accuracy at
 * any position: it is reduced to a part of a turn in integers, off by at most
 * 2^-32 turns and 2^-52 of itself; its sine and cosine, from a 32-bit float, are
 * off by at most 2^-19 (not of themselves).  The sum of squares is finite for
 * |x| below 2^60.  freqs are finite, positions any.
 * Outputs are contiguous; an output may be its own contiguous input. */
typedef struct bs_norm_rotate_desc {
    const void* q;            /* [total][q_heads][dim]                        */
    const void* k;            /* [total][kv_heads][dim]; kv_heads 0: none     */
    void* out_q;
    void* out_k;
    int64_t q_stride[2];      /* elements from token to token, head to head   */
    int64_t k_stride[2];
    const void* q_weight;     /* [dim], type weight_dtype, or NULL: no norm of q */
    const void* k_weight;
    const int32_t* positions; /* [total]; not read when rotary is 0           */
    const double* freqs;      /* [rotary / 2], radians a position, 8-byte aligned */
    uint32_t total;
    int32_t q_heads, kv_heads, dim;
    int32_t rotary;           /* even, at most dim; 0: norm alone             */
    int32_t interleaved;
    int32_t dtype;            /* BS_F16 or BS_BF16                            */
    int32_t weight_dtype;     /* BS_F32, BS_F16 or BS_BF16                    */
    float eps, amplitude;     /* eps finite and not negative, amplitude finite */
} bs_norm_rotate_desc;

BS_API bs_status bs_norm_rotate(const bs_norm_rotate_desc* desc, void* stream);

/* Bounds of the key codes of a block: bounds[id][h][0][x] is the largest and
 * [1][x] the smallest code of dimension x among the block's tokens at positions
 * below lens[b].  Written are the blocks that hold any of the last `last` tokens
 * of a sequence (last < 0: all its blocks), others stay as they are.  A block
 * that is in the tables of several sequences gets, value by value, the bounds of
 * any of them (so all should have the same of its tokens).
 * To be called when codes have changed: after bs_cache_write with the number of
 * new tokens, after bs_cache_evict with last < 0 on the new tables. */
typedef struct bs_block_bounds_desc {
    int8_t* bounds;           /* [num_blocks][kv_heads][2][dim], 16-byte aligned */
    const int32_t* table;     /* [num_seqs][table_width]                      */
    const int32_t* lens;      /* [num_seqs], at most table_width * block      */
    uint32_t num_seqs, table_width;
    int32_t last;
} bs_block_bounds_desc;

BS_API bs_status bs_block_bounds(const bs_token_cache* cache, const bs_block_bounds_desc* desc, void* stream);

/* Which blocks a query attends to, by what their bounds allow.  Query i of
 * sequence b sees the positions below n = lens[b] - queries + 1 + i, so the
 * first ceil(n / block) columns of its table.  If they are at most `count`, all
 * are chosen; else the first `sinks`, the last `recent`, and of the others the
 * count - sinks - recent of the largest score (ties: the lower column; NaN
 * counts as largest).  A key head's query heads choose together:
 *   m = max |q| over their elements,  c = rint(q * (127 * (1 / m)))  (0 if
 *   m < 1e-30; each step rounded to 32 bits)
 *   score = k_scale * sum over heads and dimensions of max(c * upper, c * lower),
 * the sum exact in integers, then rounded to 32 bits, then the product: no sum
 * of those heads' scores with a token of the block, in units of m / 127, is
 * larger, but for the rounding of q.  blocks[b][i][h]: columns in ascending order, -1 past the end. */
typedef struct bs_block_choice_desc {
    const void* q;            /* [num_seqs][queries][q_heads][dim]            */
    int64_t q_stride[3];      /* elements from sequence to sequence, token to token, head to head */
    const int8_t* bounds;     /* [num_blocks][kv_heads][2][dim], 16-byte aligned */
    const int32_t* table;     /* [num_seqs][table_width]                      */
    const int32_t* lens;      /* [num_seqs], at most table_width * block      */
    int32_t* blocks;          /* [num_seqs][queries][kv_heads][count]         */
    uint32_t num_seqs, table_width;
    int32_t queries, q_heads, count, sinks, recent;
    int32_t dtype;            /* BS_F16 or BS_BF16                            */
} bs_block_choice_desc;

BS_API bs_status bs_block_choice(const bs_token_cache* cache, const bs_block_choice_desc* desc, void* stream);

/* Attention over chosen blocks: query i of sequence b and the heads of key head
 * h see the tokens of the columns blocks[b][i][h][...] of the sequence's table
 * at positions below lens[b] - queries + 1 + i.  Negative entries are skipped;
 * a column twice in a list counts twice.  out, lse as in bs_prompt_attention. */
typedef struct bs_block_attention_desc {
    const void* q;            /* [num_seqs][queries][q_heads][dim]            */
    int64_t q_stride[3];
    const int32_t* table;     /* [num_seqs][table_width]                      */
    const int32_t* lens;      /* [num_seqs], at most table_width * block      */
    const int32_t* blocks;    /* [num_seqs][queries][kv_heads][count], in any order */
    void* out;                /* [num_seqs][queries][q_heads][dim], type dtype */
    float* lse;               /* [num_seqs][queries][q_heads], or NULL        */
    uint32_t num_seqs, table_width;
    int32_t queries, q_heads, count;
    int32_t dtype;            /* BS_F16 or BS_BF16                            */
    float scale;
} bs_block_attention_desc;

BS_API bs_status bs_block_attention(const bs_token_cache* cache, const bs_block_attention_desc* desc, void* stream);

/* Attention of sequences that begin with the same tokens.  Sequences cu[m] ..
 * cu[m+1] are group m, whose tokens' first shared_lens[m] are the positions of
 * row m of shared_table; what a sequence has beyond them is in its own table,
 * lens[b] tokens, the last `queries` of which are the query tokens: query i
 * sees all shared tokens of its group and its own positions below
 * lens[b] - queries + 1 + i.  cu starts at 0, ascends and ends at num_seqs
 * (else error bit 4 is set and outputs may hold anything).  Where sequences and
 * shared tokens are many, the shared keys and values are read once for up to 256
 * query rows of a group (sequences x queries x heads of a key head); where they
 * are few, by each sequence.  Which way is taken goes by the numbers of
 * sequences, heads and columns of the tables.  out, lse as in
 * bs_prompt_attention, over both sets of tokens.  Waits inside are bounded as
 * there; after one that gave up (error bit 1) outputs hold anything. */
typedef struct bs_shared_attention_desc {
    const void* q;            /* [num_seqs][queries][q_heads][dim]            */
    int64_t q_stride[3];
    const int32_t* shared_table; /* [num_groups][shared_width]                */
    const int32_t* shared_lens;  /* [num_groups], at most shared_width * block */
    const int32_t* cu;        /* [num_groups + 1]                             */
    const int32_t* table;     /* [num_seqs][table_width]                      */
    const int32_t* lens;      /* [num_seqs], at most table_width * block      */
    void* out;                /* [num_seqs][queries][q_heads][dim], type dtype */
    float* lse;               /* [num_seqs][queries][q_heads], or NULL        */
    void* workspace;
    size_t workspace_bytes;
    uint32_t num_seqs, num_groups, shared_width, table_width;
    int32_t queries, q_heads;
    int32_t dtype;            /* BS_F16 or BS_BF16                            */
    float scale;
} bs_shared_attention_desc;

BS_API bs_status bs_shared_attention(const bs_token_cache* cache, const bs_shared_attention_desc* desc, void* stream);
BS_API bs_status bs_shared_attention_workspace(const bs_token_cache* cache, const bs_shared_attention_desc* desc, size_t* bytes);

/* Error bits that token-memory kernels have set on the current device since
 * the last call, ordered after the work queued on `stream`; synchronises
 * `stream`.  The bits returned are cleared, others that kernels on other
 * streams set meanwhile stay for the next call.  The bits are the device's,
 * not a stream's or a caller's: who takes them takes everyone's, and of two
 * calls at once both may return the same bit.  Bits: 1 a wait inside a kernel
 * gave up, 2 a block id outside the cache, 4 lengths outside their buffers. */
BS_API bs_status bs_memory_take_errors(void* stream, uint32_t* flags);

/* Device buffers on the index's device (for callers that stage queries once
 * and search many times, like the reference CLI's timed loop,
 * src/gpu_cli.cu:400-421). */
BS_API bs_status bs_device_alloc(const bs_index* index, size_t bytes, void** dptr);
BS_API bs_status bs_device_free(const bs_index* index, void* dptr);
BS_API bs_status bs_copy_to_device(const bs_index* index, void* dst, const void* src, size_t bytes);
BS_API bs_status bs_copy_to_host(const bs_index* index, void* dst, const void* src, size_t bytes);
BS_API bs_status bs_device_fill(const bs_index* index, void* dptr, int byte_value, size_t bytes);
BS_API bs_status bs_synchronize(const bs_index* index, void* stream);

BS_API const char* bs_last_error(void);
BS_API const char* bs_version(void);

#ifdef __cplusplus
}
#endif
#endif /* BSEARCH_H */
