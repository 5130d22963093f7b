// bs_tcgen05.cuh -- what the attention kernels on the tensor cores with tensor
// memory share (bs_prompt_attention.cu, bs_shared_attention.cu): barriers,
// products of shared and tensor memory, loads and stores of tensor memory, the
// 16-bit types, outputs' way to memory.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdlib>

#include "bs_device.cuh"

namespace bsb {
namespace tc {

using namespace dev;

constexpr int kRows = 128;             // query rows of a tile, keys of a tile
constexpr int kBoxBytes = kRows * 128; // 128 rows of 64 elements
constexpr unsigned kPolls = 1u << 22;

__device__ __forceinline__ unsigned smem_addr(const void* p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void barrier_init(uint64_t* b, unsigned count) {
    asm volatile("mbarrier.init.shared.b64 [%0], %1;\n" ::"r"(smem_addr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared.b64 _, [%0];\n" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint64_t* b, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;\n" ::"r"(smem_addr(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_test(uint64_t* b, unsigned phase) {
    unsigned ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok)
                 : "r"(smem_addr(b)), "r"(phase)
                 : "memory");
    return ok != 0;
}

// Shared-memory operand: 128-byte swizzled rows, groups of 8 rows `sbo` bytes
// apart; `lbo`: from 64 columns to the next, where the columns are not the
// contraction's.
__device__ __forceinline__ uint64_t operand(unsigned addr, unsigned lbo, unsigned sbo) {
    return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | static_cast<uint64_t>(lbo >> 4) << 16 |
           static_cast<uint64_t>(sbo >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t what, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(what), "r"(static_cast<unsigned>(add))
                 : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t what, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(what), "r"(static_cast<unsigned>(add))
                 : "memory");
}
__device__ __forceinline__ bool elected() {
    unsigned yes;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(yes));
    return yes != 0;
}
// The barrier completes when every matrix instruction issued so far has.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
// (The registers are named so that nothing computed from them moves ahead.)
__device__ __forceinline__ void wait_loads32(float* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]),
                   "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]),
                   "+f"(r[14]), "+f"(r[15]), "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]),
                   "+f"(r[21]), "+f"(r[22]), "+f"(r[23]), "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]),
                   "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void wait_loads16(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                   "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
                   "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// 32, 16 or 1 columns of the warp's 32 TMEM lanes: a register each.
__device__ __forceinline__ void tmem_load32(uint32_t at, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]),
          "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]),
          "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]),
          "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(at)
        : "memory");
}
__device__ __forceinline__ uint32_t tmem_load1(uint32_t at) {
    uint32_t u;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\ntcgen05.wait::ld.sync.aligned;\n" : "=r"(u) : "r"(at) : "memory");
    return u;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
template <typename T>
struct Type16;
template <>
struct Type16<__half> {
    static constexpr uint32_t kFormat = 0, kExponent = 0x7c007c00u, kExponentOne = 0x04000400u;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
    static __device__ __forceinline__ uint32_t larger(uint32_t x, uint32_t y) {
        const __half2 h = __hmax2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&y));
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <>
struct Type16<__nv_bfloat16> {
    static constexpr uint32_t kFormat = 1, kExponent = 0x7f807f80u, kExponentOne = 0x00800080u;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u)); }
    static __device__ __forceinline__ uint32_t larger(uint32_t x, uint32_t y) {
        const __nv_bfloat162 h = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};

// A warp's 32 rows, 128 bytes of each (a lane has its own row's), to memory: by
// way of shared memory, so that 8 lanes write a row's 128 bytes together
// (16 bytes of 32 rows at a time took 7,700 clocks for two tiles).  `row` is
// the lane's row in memory, null if it has none; `at` the first byte's place
// in it, `bytes` the row's length.
__device__ __forceinline__ void store_rows(const uint32_t (&u)[32], unsigned char* staging, void* row, uint32_t at, uint32_t bytes) {
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k)
        *reinterpret_cast<uint4*>(staging + lane * 128 + ((k ^ lane) & 7) * 16) = make_uint4(u[4 * k], u[4 * k + 1], u[4 * k + 2], u[4 * k + 3]);
    __syncwarp();
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) {
        const uint32_t r = 4 * k + lane / 8, unit = lane & 7;
        const uint4 w = *reinterpret_cast<const uint4*>(staging + r * 128 + ((unit ^ r) & 7) * 16);
        unsigned char* to = reinterpret_cast<unsigned char*>(__shfl_sync(kFull, reinterpret_cast<uintptr_t>(row), r));
        if (to && at + unit * 16 < bytes) *reinterpret_cast<uint4*>(to + at + unit * 16) = w;
    }
    __syncwarp();
}

// Polls of a wait before it gives up: BSEARCH_WAIT_POLLS where that is a number
// and nothing else.
inline uint32_t wait_polls() {
    const char* s = std::getenv("BSEARCH_WAIT_POLLS");
    if (!s || *s < '0' || *s > '9') return kPolls;
    char* end = nullptr;
    const unsigned long n = std::strtoul(s, &end, 10);
    return *end || n > 0xffffffffu ? kPolls : static_cast<uint32_t>(n);
}

}  // namespace tc
}  // namespace bsb
