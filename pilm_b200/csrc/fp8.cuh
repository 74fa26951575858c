// e4m3 conversions of the 8-bit KV cache kernels.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"

namespace pilm {

constexpr int kKv8HD = 128;   // head_dim of the 8-bit cache kernels
constexpr int kKv8Page = 16;  // tokens per page

// Two floats to e4m3 (nearest even, saturating at +-448), lo in the low byte.
__device__ __forceinline__ uint32_t f32x2_to_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t f32x4_to_e4m3x4(float a, float b, float c, float d) {
    return f32x2_to_e4m3x2(a, b) | (f32x2_to_e4m3x2(c, d) << 16);
}
// Two e4m3 codes (low 16 bits) to f16x2: exact, every e4m3 value is an f16 value.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t v) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2hi_to_f16x2(uint32_t v) {  // the upper two codes
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float2 f16x2_to_f32x2(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}

}  // namespace pilm
