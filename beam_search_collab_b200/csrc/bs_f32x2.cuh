// bs_f32x2.cuh -- two 32-bit sums or products at a time (one instruction on
// sm_100a), each rounded to nearest.  The compiler may contract a mul2 that
// feeds an add2 to one rounding: not where both roundings are wanted.
#pragma once

#include <cuda_runtime.h>

namespace bsb {
namespace dev {

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n .reg .b64 a, b, c, r;\n mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 c, {%6, %7}; fma.rn.f32x2 r, a, b, c; mov.b64 {%0, %1}, r;\n}\n"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n .reg .b64 a, b, r;\n mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; add.rn.f32x2 r, a, b; mov.b64 {%0, %1}, r;\n}\n"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n .reg .b64 a, b, r;\n mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mul.rn.f32x2 r, a, b; mov.b64 {%0, %1}, r;\n}\n"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

}  // namespace dev
}  // namespace bsb
