// Rounding to e4m3 with a power-of-two scale per block (formulas: dense8_quant.cu), shared by the kernels that quantise.
#pragma once

#include <stdint.h>

namespace pcb {

__device__ __forceinline__ int scale_byte(uint32_t amax_bits) {            // e + 127 of a block with that fp32 maximum (finite)
    if (amax_bits == 0) return 127;
    int p = (int)(amax_bits >> 23);
    uint32_t m = amax_bits & 0x7fffffu;
    if (p == 0) return 1;                                                  // below 2^-126: e = -126
    const int e = p - 8 + (m > 0x600000u ? 1 : 0);                         // p is biased by 127 already
    return e < 1 ? 1 : e;
}
__device__ __forceinline__ float inverse_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }   // 2^-e, byte in [1, 247]

// two values times their scales, rounded
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b, float2 s) {
    unsigned long long v, f;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    asm("mov.b64 %0, {%1, %2};" : "=l"(f) : "f"(s.x), "f"(s.y));
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(v) : "l"(f));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
    uint16_t q;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(q) : "f"(b), "f"(a));
    return q;
}

}  // namespace pcb
