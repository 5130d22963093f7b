// bs_memory.h -- launch-level interface of the token-memory operators
// (prompt attention, 8-bit token cache), shared by their C entries
// (bs_memory_capi.cu) and their kernels.  Not part of the public ABI.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "bsearch.h"

namespace bsb {

// Error bits of the token-memory kernels (bs_memory_take_errors).
enum MemoryError : unsigned int {
    kMemErrWait = 1u,      // a bounded wait gave up
    kMemErrBlock = 2u,     // a block id outside the cache
    kMemErrLength = 4u,    // lengths outside their buffers
};

// Records `status` and its message as the calling thread's last error
// (bs_capi.cu) and returns it.
bs_status report_error(bs_status status, const char* fmt, ...);

// The device a launch goes to: error word and sizes, looked up once per device.
struct MemoryDevice {
    int device;
    int num_sms;
    unsigned int* errors;   // device word the kernels OR their error bits into
};
bs_status memory_device(MemoryDevice& out);

size_t prompt_attention_scratch(const bs_prompt_attention_desc& d, const MemoryDevice& dev);
cudaError_t launch_prompt_attention(const bs_prompt_attention_desc& d, const MemoryDevice& dev, cudaStream_t stream);
cudaError_t launch_cache_write(const bs_token_cache& c, const bs_cache_write_desc& d, const MemoryDevice& dev,
                               cudaStream_t stream);
cudaError_t launch_cache_read(const bs_token_cache& c, const bs_cache_read_desc& d, const MemoryDevice& dev,
                              cudaStream_t stream);
size_t cache_attention_scratch(const bs_token_cache& c, const bs_cache_attention_desc& d, const MemoryDevice& dev);
cudaError_t launch_cache_attention(const bs_token_cache& c, const bs_cache_attention_desc& d, const MemoryDevice& dev,
                                   cudaStream_t stream);
size_t cache_evict_scratch(const bs_token_cache& c, const bs_cache_evict_desc& d, const MemoryDevice& dev);
cudaError_t launch_cache_evict(const bs_token_cache& c, const bs_cache_evict_desc& d, const MemoryDevice& dev,
                               cudaStream_t stream);

cudaError_t launch_norm_rotate(const bs_norm_rotate_desc& d, const MemoryDevice& dev, cudaStream_t stream);
// Blocks of a sequence that hold any of its last tokens, at most (these may begin
// and end inside a block).
inline uint32_t bounds_columns(const bs_token_cache& c, const bs_block_bounds_desc& d) {
    const uint64_t touched = d.last < 0 ? d.table_width : d.last == 0 ? 0 : (static_cast<uint64_t>(d.last) + c.block - 2) / c.block + 1;
    return touched < d.table_width ? static_cast<uint32_t>(touched) : d.table_width;
}
cudaError_t launch_block_bounds(const bs_token_cache& c, const bs_block_bounds_desc& d, const MemoryDevice& dev, cudaStream_t stream);
cudaError_t launch_block_choice(const bs_token_cache& c, const bs_block_choice_desc& d, const MemoryDevice& dev, cudaStream_t stream);
cudaError_t launch_block_attention(const bs_token_cache& c, const bs_block_attention_desc& d, const MemoryDevice& dev,
                                   cudaStream_t stream);
size_t shared_attention_scratch(const bs_token_cache& c, const bs_shared_attention_desc& d, const MemoryDevice& dev);
cudaError_t launch_shared_attention(const bs_token_cache& c, const bs_shared_attention_desc& d, const MemoryDevice& dev,
                                    cudaStream_t stream);

#ifdef __CUDACC__
// A kernel that may start while the one before it on the stream still runs,
// whosever that is, and waits for it by itself, in every block, before it reads
// or writes anything.
template <typename... Params, typename... Given>
cudaError_t launch_after(void (*kernel)(Params...), dim3 grid, int threads, size_t shared, cudaStream_t stream, Given... given) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    config.attrs = &attr;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, Params(given)...);
}
#endif

}  // namespace bsb
