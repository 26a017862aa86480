// Packed binary32 arithmetic of sm_100: two values in one register pair, each rounded
// as by the scalar instruction, in half the instructions.
#pragma once

#include "qsml_internal.cuh"

namespace qsml {

struct P2 {
    uint64_t v;
};
__device__ __forceinline__ P2 pack(float a, float b) {
    P2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack(P2 p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
    return f;
}
__device__ __forceinline__ P2 add2(P2 a, P2 b) {
    P2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ P2 mul2(P2 a, P2 b) {
    P2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ P2 fma2(P2 a, P2 b, P2 c) {
    P2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ float sum2(P2 p) {
    const float2 f = unpack(p);
    return __fadd_rn(f.x, f.y);
}

__device__ __forceinline__ P2 both(float a) { return pack(a, a); }

}  // namespace qsml
