// bs_memory_capi.cu -- C entries of the token-memory operators
// (include/bsearch.h): argument checks, then one launcher each.
#include <cuda_runtime.h>

#include <cmath>
#include <initializer_list>
#include <mutex>

#include "bsearch.h"
#include "bs_memory.h"

// One word per GPU that holds the library; the kernels OR their error bits
// into it, bs_memory_take_errors reads it and clears the bits it has read.
static __device__ unsigned int g_memory_errors;

static __global__ void k_clear_errors(unsigned int bits) { atomicAnd(&g_memory_errors, ~bits); }

namespace bsb {

namespace {

constexpr int kMaxDevices = 64;
std::mutex g_mu;
MemoryDevice g_devices[kMaxDevices];
bool g_known[kMaxDevices];

bs_status cuda_error(cudaError_t e, const char* what) {
    return report_error(e == cudaErrorMemoryAllocation ? BS_ERR_OUT_OF_MEMORY : BS_ERR_CUDA, "%s: %s", what,
                        cudaGetErrorString(e));
}

// Every pointer is NULL or memory that kernels on `device` can use.
bool on_device(int device, std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs) {
        if (!p) continue;
        cudaPointerAttributes a;
        if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
            cudaGetLastError();
            return false;
        }
        if (a.type != cudaMemoryTypeManaged && (a.type != cudaMemoryTypeDevice || a.device != device)) return false;
    }
    return true;
}

bool any_null(std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs)
        if (!p) return true;
    return false;
}

bool aligned16(std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) & 15) return false;
    return true;
}

// Lists, lengths, scales and masses: read and written 4 bytes at a time.
bool aligned4(std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) & 3) return false;
    return true;
}

// Strides between `extents` places: not negative, and no place so far away
// that address arithmetic could overflow.
bool within_reach(const int64_t* s, std::initializer_list<uint32_t> extents) {
    int64_t left = int64_t{1} << 59;
    int i = 0;
    for (uint32_t extent : extents) {
        const int64_t steps = extent > 1 ? extent - 1 : 1;
        if (s[i] < 0 || s[i] > left / steps) return false;
        left -= s[i++] * steps;
    }
    return true;
}

// Of 16-bit elements: multiples of 16 bytes too, below the 2^40 bytes of a
// tensor map.
bool strides_ok(const int64_t* s, std::initializer_list<uint32_t> extents) {
    for (size_t i = 0; i < extents.size(); ++i)
        if ((s[i] & 7) || s[i] >= (int64_t{1} << 37)) return false;
    return within_reach(s, extents);
}

const char* const kWhere = "pointers must be memory of the current device";
const char* const kAlign4 = "32-bit buffers must be 4-byte aligned";
const char* const kAlign = "q, k, v and outputs must be 16-byte aligned, their strides non-negative multiples of 8 elements within a buffer's reach";

bs_status check_dim(int32_t dim) {
    if (dim <= 0) return report_error(BS_ERR_INVALID_ARGUMENT, "dim must be positive");
    if (dim % 16 || dim > 128) return report_error(BS_ERR_UNSUPPORTED, "dim %d: a multiple of 16 up to 128 is supported", dim);
    return BS_OK;
}

bs_status check_heads(int32_t q_heads, int32_t kv_heads) {
    if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads)
        return report_error(BS_ERR_INVALID_ARGUMENT, "q_heads (%d) must be a positive multiple of kv_heads (%d)", q_heads,
                            kv_heads);
    if (q_heads / kv_heads > 128 || kv_heads > 65535)
        return report_error(BS_ERR_UNSUPPORTED, "at most 128 query heads per key head and 65535 key heads are supported");
    return BS_OK;
}

bs_status check_dtype16(int32_t dtype) {
    if (dtype == BS_F16 || dtype == BS_BF16) return BS_OK;
    return report_error(BS_ERR_INVALID_ARGUMENT, "dtype must be BS_F16 or BS_BF16");
}

bs_status check_cache(const bs_token_cache* c, int device, bool pointers) {
    if (!c) return report_error(BS_ERR_INVALID_ARGUMENT, "cache is NULL");
    if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128)
        return report_error(BS_ERR_INVALID_ARGUMENT, "block must be 16, 32, 64 or 128 tokens");
    if (bs_status s = check_dim(c->dim)) return s;
    if (c->kv_heads <= 0 || c->kv_heads > 65535) return report_error(BS_ERR_INVALID_ARGUMENT, "kv_heads must be in 1..65535");
    if (!pointers) return BS_OK;
    if (any_null({c->k, c->v, c->k_scale, c->v_scale})) return report_error(BS_ERR_INVALID_ARGUMENT, "a cache buffer is NULL");
    if (!aligned16({c->k, c->v})) return report_error(BS_ERR_INVALID_ARGUMENT, "the cache's codes must be 16-byte aligned");
    if (!aligned4({c->k_scale, c->v_scale})) return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kAlign4);
    if (!on_device(device, {c->k, c->v, c->k_scale, c->v_scale}))
        return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kWhere);
    return BS_OK;
}

// Counts that kernels keep in 32 bits.
bs_status check_table(const bs_token_cache* c, uint32_t num_seqs, uint32_t width) {
    if (static_cast<uint64_t>(width) * c->block >= (1u << 30) || num_seqs > 65535)
        return report_error(BS_ERR_UNSUPPORTED, "at most 65535 sequences of fewer than 2^30 tokens are supported");
    return BS_OK;
}

}  // namespace

bs_status memory_device(MemoryDevice& out) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_error(e, "device query");
    if (dev < 0 || dev >= kMaxDevices) return report_error(BS_ERR_UNSUPPORTED, "device %d is beyond the %d tracked", dev, kMaxDevices);
    std::lock_guard<std::mutex> lk(g_mu);
    if (!g_known[dev]) {
        MemoryDevice d{};
        d.device = dev;
        void* word = nullptr;
        e = cudaDeviceGetAttribute(&d.num_sms, cudaDevAttrMultiProcessorCount, dev);
        if (e == cudaSuccess) e = cudaGetSymbolAddress(&word, g_memory_errors);
        if (e != cudaSuccess) return cuda_error(e, "device query");
        d.errors = static_cast<unsigned int*>(word);
        g_devices[dev] = d;
        g_known[dev] = true;
    }
    out = g_devices[dev];
    return BS_OK;
}

}  // namespace bsb

using namespace bsb;

extern "C" {

static bs_status check_prompt(const bs_prompt_attention_desc* d) {
    if (!d) return report_error(BS_ERR_INVALID_ARGUMENT, "desc is NULL");
    if (bs_status s = check_dtype16(d->dtype)) return s;
    if (bs_status s = check_dim(d->dim)) return s;
    if (bs_status s = check_heads(d->q_heads, d->kv_heads)) return s;
    if (!(d->scale > 0.f) || std::isinf(d->scale))
        return report_error(BS_ERR_INVALID_ARGUMENT, "scale must be positive and finite (not 0, negative, infinite or NaN)");
    if (d->total_q >= (1u << 30) || d->total_k >= (1u << 30) || d->num_seqs > 65535)
        return report_error(BS_ERR_UNSUPPORTED, "at most 65535 sequences of fewer than 2^30 tokens in all are supported");
    return BS_OK;
}

BS_API bs_status bs_prompt_attention_workspace(const bs_prompt_attention_desc* d, size_t* bytes) {
    if (!bytes) return report_error(BS_ERR_INVALID_ARGUMENT, "bytes is NULL");
    if (bs_status s = check_prompt(d)) return s;
    MemoryDevice dev;
    if (bs_status s = memory_device(dev)) return s;
    *bytes = prompt_attention_scratch(*d, dev);
    return BS_OK;
}

BS_API bs_status bs_prompt_attention(const bs_prompt_attention_desc* d, void* stream) {
    if (bs_status s = check_prompt(d)) return s;
    if (d->total_q == 0) return BS_OK;
    if (d->num_seqs == 0)
        return report_error(BS_ERR_INVALID_ARGUMENT, "num_seqs is 0, but q has %u rows", static_cast<unsigned>(d->total_q));
    const uint32_t q_heads = d->q_heads, kv_heads = d->kv_heads;
    if (any_null({d->q, d->out, d->cu_q, d->cu_k}) || (d->total_k && any_null({d->k, d->v})))
        return report_error(BS_ERR_INVALID_ARGUMENT, "a buffer is NULL");
    if (!aligned16({d->q, d->k, d->v, d->out, d->workspace}) || !strides_ok(d->q_stride, {d->total_q, q_heads}) ||
        !strides_ok(d->k_stride, {d->total_k, kv_heads}) || !strides_ok(d->v_stride, {d->total_k, kv_heads}))
        return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kAlign);
    if (!aligned4({d->lse, d->cu_q, d->cu_k})) return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kAlign4);
    // one head or token for many (a stride of 0) has no tensor map
    if ((d->total_q > 1 && d->q_stride[0] == 0) || (d->q_heads > 1 && d->q_stride[1] == 0) ||
        (d->total_k > 1 && (d->k_stride[0] == 0 || d->v_stride[0] == 0)) || (d->kv_heads > 1 && (d->k_stride[1] == 0 || d->v_stride[1] == 0)))
        return report_error(BS_ERR_UNSUPPORTED, "a stride of 0 (a broadcast tensor) is not supported: make it contiguous");
    MemoryDevice dev;
    if (bs_status s = memory_device(dev)) return s;
    if (!on_device(dev.device, {d->q, d->k, d->v, d->out, d->lse, d->cu_q, d->cu_k, d->workspace}))
        return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kWhere);
    const size_t need = prompt_attention_scratch(*d, dev);
    if (need > (d->workspace ? d->workspace_bytes : 0))
        return report_error(BS_ERR_INVALID_ARGUMENT, "workspace of %zu bytes, %zu are needed", d->workspace ? d->workspace_bytes : 0,
                            need);
    const cudaError_t e = launch_prompt_attention(*d, dev, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? BS_OK : cuda_error(e, "prompt attention launch");
}

BS_API bs_status bs_cache_write(const bs_token_cache* c, const bs_cache_write_desc* d, void* stream) {
    if (!d) return report_error(BS_ERR_INVALID_ARGUMENT, "desc is NULL");
    MemoryDevice dev;
    if (bs_status s = check_cache(c, 0, false)) return s;
    if (bs_status s = check_dtype16(d->dtype)) return s;
    if (bs_status s = check_table(c, d->num_seqs, d->table_width)) return s;
    if (d->total >= (1u << 30)) return report_error(BS_ERR_UNSUPPORTED, "at most 2^30 tokens a call are supported");
    if (d->total == 0 || d->num_seqs == 0) return BS_OK;
    if (any_null({d->k, d->v, d->cu, d->table, d->start})) return report_error(BS_ERR_INVALID_ARGUMENT, "a buffer is NULL");
    const uint32_t heads = c->kv_heads;
    if (!aligned16({d->k, d->v}) || !strides_ok(d->k_stride, {d->total, heads}) || !strides_ok(d->v_stride, {d->total, heads}))
        return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kAlign);
    if (!aligned4({d->cu, d->table, d->start})) return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kAlign4);
    if (bs_status s = memory_device(dev)) return s;
    if (bs_status s = check_cache(c, dev.device, true)) return s;
    if (!on_device(dev.device, {d->k, d->v, d->cu, d->table, d->start})) return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kWhere);
    const cudaError_t e = launch_cache_write(*c, *d, dev, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? BS_OK : cuda_error(e, "cache write launch");
}

BS_API bs_status bs_cache_read(const bs_token_cache* c, const bs_cache_read_desc* d, void* stream) {
    if (!d) return report_error(BS_ERR_INVALID_ARGUMENT, "desc is NULL");
    MemoryDevice dev;
    if (bs_status s = check_cache(c, 0, false)) return s;
    if (d->dtype != BS_F32 && d->dtype != BS_F16 && d->dtype != BS_BF16)
        return report_error(BS_ERR_INVALID_ARGUMENT, "dtype must be BS_F32, BS_F16 or BS_BF16");
    if (bs_status s = check_table(c, d->num_seqs, d->table_width)) return s;
    if (d->count >= (1u << 30)) return report_error(BS_ERR_UNSUPPORTED, "at most 2^30 positions are supported");
    const int64_t steps[2] = {d->position_seq_stride, d->position_head_stride};
    if (!within_reach(steps, {d->num_seqs, static_cast<uint32_t>(c->kv_heads)}))
        return report_error(BS_ERR_INVALID_ARGUMENT, "strides of positions must not be negative or out of any buffer's reach");
    if (d->count == 0 || d->num_seqs == 0 || (!d->k && !d->v)) return BS_OK;
    if (any_null({d->lens, d->positions}) || (d->table_width && !d->table))
        return report_error(BS_ERR_INVALID_ARGUMENT, "a buffer is NULL");
    if (!aligned16({d->k, d->v})) return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kAlign);
    if (!aligned4({d->table, d->lens, d->positions})) return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kAlign4);
    if (bs_status s = memory_device(dev)) return s;
    if (bs_status s = check_cache(c, dev.device, true)) return s;
    if (!on_device(dev.device, {d->table, d->lens, d->positions, d->k, d->v}))
        return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kWhere);
    const cudaError_t e = launch_cache_read(*c, *d, dev, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? BS_OK : cuda_error(e, "cache read launch");
}

static bs_status check_attention(const bs_token_cache* c, const bs_cache_attention_desc* d) {
    if (!d) return report_error(BS_ERR_INVALID_ARGUMENT, "desc is NULL");
    if (bs_status s = check_cache(c, 0, false)) return s;
    if (bs_status s = check_dtype16(d->dtype)) return s;
    if (bs_status s = check_heads(d->q_heads, c->kv_heads)) return s;
    if (bs_status s = check_table(c, d->num_seqs, d->table_width)) return s;
    if (d->queries <= 0 || d->queries > 1024) return report_error(BS_ERR_INVALID_ARGUMENT, "queries must be in 1..1024");
    if (!(d->scale > 0.f) || std::isinf(d->scale))
        return report_error(BS_ERR_INVALID_ARGUMENT, "scale must be positive and finite (not 0, negative, infinite or NaN)");
    if (d->out_mass && d->mass_width >= (1u << 30)) return report_error(BS_ERR_UNSUPPORTED, "mass_width must be below 2^30");
    return BS_OK;
}

BS_API bs_status bs_cache_attention_workspace(const bs_token_cache* c, const bs_cache_attention_desc* d, size_t* bytes) {
    if (!bytes) return report_error(BS_ERR_INVALID_ARGUMENT, "bytes is NULL");
    if (bs_status s = check_attention(c, d)) return s;
    MemoryDevice dev;
    if (bs_status s = memory_device(dev)) return s;
    *bytes = cache_attention_scratch(*c, *d, dev);
    return BS_OK;
}

BS_API bs_status bs_cache_attention(const bs_token_cache* c, const bs_cache_attention_desc* d, void* stream) {
    if (bs_status s = check_attention(c, d)) return s;
    if (d->num_seqs == 0) return BS_OK;
    if (any_null({d->q, d->lens, d->out}) || (d->table_width && !d->table))
        return report_error(BS_ERR_INVALID_ARGUMENT, "a buffer is NULL");
    if (d->mass && !d->out_mass) return report_error(BS_ERR_INVALID_ARGUMENT, "mass without out_mass");
    if (d->out_mass && d->mass_width == 0) return report_error(BS_ERR_INVALID_ARGUMENT, "mass_width is 0");
    if (!aligned16({d->q, d->out, d->workspace}) || !strides_ok(d->q_stride, {d->num_seqs, static_cast<uint32_t>(d->queries), static_cast<uint32_t>(d->q_heads)}))
        return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kAlign);
    if (!aligned4({d->table, d->lens, d->lse, d->mass, d->out_mass})) return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kAlign4);
    MemoryDevice dev;
    if (bs_status s = memory_device(dev)) return s;
    if (bs_status s = check_cache(c, dev.device, true)) return s;
    if (!on_device(dev.device, {d->q, d->table, d->lens, d->out, d->lse, d->mass, d->out_mass, d->workspace}))
        return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kWhere);
    const size_t need = cache_attention_scratch(*c, *d, dev);
    if (need > (d->workspace ? d->workspace_bytes : 0))
        return report_error(BS_ERR_INVALID_ARGUMENT, "workspace of %zu bytes, %zu are needed", d->workspace ? d->workspace_bytes : 0,
                            need);
    const cudaError_t e = launch_cache_attention(*c, *d, dev, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? BS_OK : cuda_error(e, "cache attention launch");
}

static bs_status check_evict(const bs_token_cache* c, const bs_cache_evict_desc* d) {
    if (!d) return report_error(BS_ERR_INVALID_ARGUMENT, "desc is NULL");
    if (bs_status s = check_cache(c, 0, false)) return s;
    if (bs_status s = check_table(c, d->num_seqs, d->table_width)) return s;
    if (bs_status s = check_table(c, d->num_seqs, d->new_table_width)) return s;
    if (d->mass_width >= (1u << 30)) return report_error(BS_ERR_UNSUPPORTED, "mass_width must be below 2^30");
    if (d->budget <= 0 || d->budget >= (1 << 30) || d->sinks < 0 || d->recent < 0 ||
        static_cast<int64_t>(d->sinks) + d->recent > d->budget)
        return report_error(BS_ERR_INVALID_ARGUMENT, "need 0 < budget < 2^30 and sinks + recent <= budget, none negative");
    const uint64_t held = static_cast<uint64_t>(d->table_width) * c->block, room = static_cast<uint64_t>(d->new_table_width) * c->block;
    const uint64_t most = held < d->mass_width ? held : d->mass_width;
    if (room < (most < static_cast<uint64_t>(d->budget) ? most : static_cast<uint64_t>(d->budget)))
        return report_error(BS_ERR_INVALID_ARGUMENT, "new_table has room for %llu tokens of a sequence, %d may stay",
                            static_cast<unsigned long long>(room), d->budget);
    return BS_OK;
}

BS_API bs_status bs_cache_evict_workspace(const bs_token_cache* c, const bs_cache_evict_desc* d, size_t* bytes) {
    if (!bytes) return report_error(BS_ERR_INVALID_ARGUMENT, "bytes is NULL");
    if (bs_status s = check_evict(c, d)) return s;
    MemoryDevice dev;
    if (bs_status s = memory_device(dev)) return s;
    *bytes = cache_evict_scratch(*c, *d, dev);
    return BS_OK;
}

BS_API bs_status bs_cache_evict(const bs_token_cache* c, const bs_cache_evict_desc* d, void* stream) {
    if (bs_status s = check_evict(c, d)) return s;
    if (d->num_seqs == 0) return BS_OK;
    if (any_null({d->lens, d->kept, d->new_lens, d->new_mass}) || (d->table_width && !d->table) ||
        (d->new_table_width && !d->new_table) || (d->mass_width && !d->mass))
        return report_error(BS_ERR_INVALID_ARGUMENT, "a buffer is NULL");
    if (!aligned16({d->workspace})) return report_error(BS_ERR_INVALID_ARGUMENT, "the workspace must be 16-byte aligned");
    if (!aligned4({d->mass, d->table, d->lens, d->new_table, d->kept, d->new_lens, d->new_mass})) return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kAlign4);
    MemoryDevice dev;
    if (bs_status s = memory_device(dev)) return s;
    if (bs_status s = check_cache(c, dev.device, true)) return s;
    if (!on_device(dev.device, {d->mass, d->table, d->lens, d->new_table, d->kept, d->new_lens, d->new_mass, d->workspace}))
        return report_error(BS_ERR_INVALID_ARGUMENT, "%s", kWhere);
    const size_t need = cache_evict_scratch(*c, *d, dev);
    if (need > (d->workspace ? d->workspace_bytes : 0))
        return report_error(BS_ERR_INVALID_ARGUMENT, "workspace of %zu bytes, %zu are needed", d->workspace ? d->workspace_bytes : 0,
                            need);
    const cudaError_t e = launch_cache_evict(*c, *d, dev, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? BS_OK : cuda_error(e, "cache eviction launch");
}

BS_API bs_status bs_memory_take_errors(void* stream_, uint32_t* flags) {
    if (!flags) return report_error(BS_ERR_INVALID_ARGUMENT, "flags is NULL");
    MemoryDevice dev;
    if (bs_status s = memory_device(dev)) return s;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    uint32_t h = 0;
    cudaError_t e = cudaMemcpyAsync(&h, dev.errors, 4, cudaMemcpyDeviceToHost, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    if (e == cudaSuccess && h) {       // bits set meanwhile by another stream's kernels stay for the next call
        k_clear_errors<<<1, 1, 0, stream>>>(h);
        e = cudaGetLastError();
        if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    }
    if (e != cudaSuccess) return cuda_error(e, "error word");
    *flags = h;
    return BS_OK;
}

}  // extern "C"
