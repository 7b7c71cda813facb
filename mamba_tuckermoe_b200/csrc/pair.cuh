// Paired fp32 arithmetic (sm_100 f32x2 instructions) and approximate exponential / reciprocal shared by the row kernels.
#pragma once

#include "common.cuh"

namespace tmoe {

// Two fp32 values worked on by one instruction.  The row kernels around the layer are bound by the instructions they issue as much as by
// memory, and sm_100 multiplies and adds pairs at the price of one.
using f2 = unsigned long long;
__device__ __forceinline__ f2 pair(float lo, float hi) { f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi)); return r; }
__device__ __forceinline__ f2 both(float v) { return pair(v, v); }
__device__ __forceinline__ void split(f2 v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) { f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ float sum2(f2 v) { float a, b; split(v, a, b); return a + b; }


// 2^x and 1/x to about an ulp of 2^-22; results below the normal range are 0
__device__ __forceinline__ float fast_exp2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float fast_rcp(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
constexpr float kLog2e = 1.4426950408889634f;

}  // namespace tmoe
