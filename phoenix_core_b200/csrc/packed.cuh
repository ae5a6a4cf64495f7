// Two fp32 values in one 64-bit register pair: the packed additions, products and fused products of sm_100 (one issue slot for two values, each rounded as
// the single instruction rounds it).
#pragma once

namespace pcb {

struct Pair { unsigned long long v; };
__device__ __forceinline__ Pair pair(float a, float b) { Pair r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ Pair pair(float a) { return pair(a, a); }
__device__ __forceinline__ void halves(Pair p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ float sum(Pair p) { float a, b; halves(p, a, b); return a + b; }
__device__ __forceinline__ Pair operator+(Pair a, Pair b) { Pair r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ Pair operator*(Pair a, Pair b) { Pair r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) { Pair r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }

}  // namespace pcb
