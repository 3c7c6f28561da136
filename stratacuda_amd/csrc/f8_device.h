// Device-side pieces of the 8-bit floating-point operators (f8_convert.hip,
// f8_project.hip): e4m3 codes (OCP: 4 significant bits, largest 448, no
// infinities) with one power-of-two scale for each block of 128 columns, held
// as its e8m0 byte (2^(byte - 127)).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "internal.h"

namespace f8 {

// The byte of the smallest power of two 2^e with amax <= 448 * 2^e, e >= -127;
// amax is finite and not negative, 0 takes the scale 1. From the bits: amax =
// m * 2^x with 1 <= m < 2 and 448 = 1.75 * 2^8, so e = x - 8, one more where
// m > 1.75. A subnormal amax (x < -126) lies below 448 * 2^-127.
__device__ __forceinline__ uint32_t scale_byte(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int b = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u);
    return u == 0 ? 127u : (uint32_t)max(b, 0);
}
// 2^-e of a scale byte that scale_byte gave (e <= 120): exact, normal.
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

__device__ __forceinline__ float finite_magnitude(float v) {
    const float a = fabsf(v);
    return a < INFINITY ? a : 0.0f;  // 0 for NaN too
}
// v * 2^-e is exact (or below e4m3's smallest step); the conversion rounds to
// nearest, ties to even. A value that is not finite becomes NaN (v + 0 v is v,
// or NaN): e4m3 has no infinity, and a saturated one would pass as a number.
template <typename V>
__device__ __forceinline__ uint32_t codes4(const V &v, float inverse) {
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; i++) s[i] = fmaf(v[i], inverse, v[i] * 0.0f);
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], w, true);
}

// The lane's value combined with that of the lanes 1, 2, 4, 8 and 16 (and 32)
// away, by data-parallel moves: two swaps in quads, then mirrors of 8 and 16,
// which give any lane of the other half since the halves are equal by then.
template <int CTRL>
__device__ __forceinline__ float moved(float v) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ double moved(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
constexpr int kSwap1 = 0xb1, kSwap2 = 0x4e, kMirror8 = 0x141, kMirror16 = 0x140;
__device__ __forceinline__ float max_of_16(float v) {
    v = fmaxf(v, moved<kSwap1>(v));
    v = fmaxf(v, moved<kSwap2>(v));
    v = fmaxf(v, moved<kMirror8>(v));
    return fmaxf(v, moved<kMirror16>(v));
}
// Largest of the 32 lanes of each half of a wave, in all of them.
__device__ __forceinline__ float half_wave_max(float v) {
    v = max_of_16(v);
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
// Sum over a wave, in all lanes.
__device__ __forceinline__ double wave_sum(double v) {
    v += moved<kSwap1>(v);
    v += moved<kSwap2>(v);
    v += moved<kMirror8>(v);
    v += moved<kMirror16>(v);
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

__device__ __forceinline__ float bf16_value(uint32_t bits16) { return __uint_as_float(bits16 << 16); }

// Four consecutive columns of a row, 0 past `cols`; `vec`: cols is a multiple
// of 4, so that every four lie whole and aligned in the row.
template <typename T>
__device__ __forceinline__ void load4(const T *row, int col, int cols, bool vec, float v[4]) {
    if (vec) {
        if (col < cols) {
            if constexpr (sizeof(T) == 4) {
                const float4 q = *(const float4 *)(row + col);
                v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
            } else {
                const uint2 q = *(const uint2 *)(row + col);
                v[0] = bf16_value(q.x & 0xffffu), v[1] = __uint_as_float(q.x & 0xffff0000u);
                v[2] = bf16_value(q.y & 0xffffu), v[3] = __uint_as_float(q.y & 0xffff0000u);
            }
        } else {
            v[0] = v[1] = v[2] = v[3] = 0.0f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[i] = 0.0f;
            if (col + i < cols) {
                if constexpr (sizeof(T) == 4) v[i] = row[col + i];
                else v[i] = bf16_value(row[col + i]);
            }
        }
    }
}

}  // namespace f8
