// Row codec arithmetic shared by the kernels that encode cache rows
// (reference state.h:326-629): fp32 to fp16 by truncation, and the clamps'
// order of comparison.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace kvc {

__device__ __forceinline__ uint16_t f32_to_f16_ref(float val) {
    const uint32_t f = __float_as_uint(val);
    const uint32_t sign = (f >> 16) & 0x8000;
    const int32_t e = (int32_t)((f >> 23) & 0xFF) - 127 + 15;
    uint32_t m = (f >> 13) & 0x3FF;
    if (e <= 0) {
        if (e < -10) return (uint16_t)sign;
        m = (m | 0x400) >> (1 - e);
        return (uint16_t)(sign | m);
    } else if (e >= 31) {
        return (uint16_t)(sign | 0x7C00);
    }
    return (uint16_t)(sign | ((uint32_t)e << 10) | m);
}

__device__ __forceinline__ float fmax_std(float a, float b) { return (a < b) ? b : a; }
__device__ __forceinline__ float fmin_std(float a, float b) { return (b < a) ? b : a; }

}  // namespace kvc
