// Device-side pieces of the operators over a 4-bit key-value cache
// (kv4_cache.hip, kv4_attention.hip): the layout of a page's tiles, the
// sequences of a call, and the conversions.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "f8_device.h"
#include "internal.h"

namespace kv4 {

using smi::Kv4Sequences;
using smi::Kv4View;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using f32x2 = __attribute__((ext_vector_type(2))) float;

constexpr int kPage = SM_KV4_PAGE;
constexpr int kMostPages = 1 << 24;  // of a sequence

// Byte offsets of a tile's parts.
__device__ __forceinline__ int value_codes(int pitch) { return 32 * pitch; }
__device__ __forceinline__ int key_scales(int pitch) { return 64 * pitch; }
__device__ __forceinline__ int value_scales(int pitch) { return 66 * pitch; }

// One sequence of a call: its `n` rows from `row` on, the last of its `length`
// positions. n = 0 where the device's numbers are none that the call may use.
struct Span {
    int row, n, length;
};
__device__ __forceinline__ Span span(const Kv4Sequences &q, int s) {
    const int a = q.starts[s], b = q.starts[s + 1], length = q.lengths[s];
    const bool fits = a >= 0 && b >= a && b <= q.tokens && b - a <= q.longest && length >= 0 &&
                      length <= q.table_pages * kPage;
    return {a, fits ? b - a : 0, length};
}
// The page that holds positions 64 at .. 64 at + 63 of sequence s; -1 for none.
__device__ __forceinline__ int page_of(const Kv4Sequences &q, int s, int at, int pages) {
    if (at < 0 || at >= q.table_pages) return -1;
    const int id = q.table[(int64_t)s * q.table_pages + at];
    return id >= 0 && id < pages ? id : -1;
}

// The byte of the smallest power of two 2^e with amax <= 6 * 2^e, -125 <= e <=
// 125 (so that every value that a code stands for is a normal f32 and bf16
// number, or 0); 0 takes the scale 1, a value that is not finite 255. From the
// bits: amax = m * 2^x with 1 <= m < 2 and 6 = 1.5 * 2^2, so e = x - 2, one
// more where m > 1.5. `all`: the largest of the block's bit patterns without
// their signs, which order as the magnitudes do, NaN last.
__device__ __forceinline__ uint32_t scale_byte(uint32_t all) {
    const int b = (int)(all >> 23) - 2 + ((all & 0x7fffffu) > 0x400000u);
    return all >= 0x7f800000u ? 255u : all == 0 ? 127u : (uint32_t)min(max(b, 2), 252);
}
// The scale as the f32 operand of the conversions below, which take its
// exponent field.
__device__ __forceinline__ float scale_value(uint32_t byte) { return __uint_as_float(byte << 23); }
// The scale of codes: 1 for a block that is marked as not finite, whose codes
// are 0.
__device__ __forceinline__ float code_scale(uint32_t byte) { return scale_value(byte == 255u ? 127u : byte); }
__device__ __forceinline__ float code_value(float v, uint32_t byte) { return byte == 255u ? 0.0f : v; }

__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <typename T>
__device__ __forceinline__ float value(T v) {
    if constexpr (sizeof(T) == 4) return v;
    else return f8::bf16_value(v);
}
// Eight neighbours of a row; `vec`: they lie aligned to 16 bytes (two loads of
// f32, one of bf16).
template <typename T>
__device__ __forceinline__ void load8(const T *p, bool vec, float v[8]) {
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = value(p[i]);
    } else if constexpr (sizeof(T) == 4) {
        const float4 a = ((const float4 *)p)[0], b = ((const float4 *)p)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 q = *(const uint4 *)p;
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; i++) v[2 * i] = f8::bf16_value(w[i] & 0xffffu), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, bf16x2));
}
// 16 bytes of neighbours, kPer values, as they are and as numbers: a load apart
// from what needs it, so that others follow before it is waited for. Without
// `vec` value by value.
template <typename T>
struct Piece16 {
    static constexpr int kPer = 16 / sizeof(T);
    T v[kPer];
    template <bool vec>
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (vec) {
            *(uint4 *)v = *(const uint4 *)p;
        } else {
#pragma unroll
            for (int i = 0; i < kPer; i++) v[i] = p[i];
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kPer; i++) v[i] = 0;
    }
    __device__ __forceinline__ float at(int i) const { return value(v[i]); }
};
template <bool vec, typename T>
__device__ __forceinline__ void store16(T *p, const float *v) {
    constexpr int kPer = 16 / sizeof(T);
    if constexpr (sizeof(T) == 4) {
        if constexpr (vec) {
            *(float4 *)p = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int i = 0; i < kPer; i++) p[i] = v[i];
        }
    } else {
        const uint32_t w[4] = {bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])};
        if constexpr (vec) {
            *(uint4 *)p = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) p[2 * i] = (T)w[i], p[2 * i + 1] = (T)(w[i] >> 16);
        }
    }
}
template <typename T>
__device__ __forceinline__ void store1(T *p, float v) {
    if constexpr (sizeof(T) == 4) *p = v;
    else *p = (T)bf16_pair(v, 0.0f);
}

}  // namespace kv4
