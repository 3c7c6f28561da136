// The key-value cache in 4 bits: positions written and read back, and the
// pass before it, the norm and rotation of each head's query and key.
//
// All three read each value once and write it once: bound by memory.
#include "kv4_device.h"

namespace {
using namespace smi;

// ------------------------------------------------------------------- write
// One workgroup a page and head. Keys: eight neighbouring dimensions a thread,
// so that four threads hold a block of 32 and a position's codes are stored in
// one piece. Values: a wave takes a block of 32 dimensions of all 64
// positions, a thread two dimensions (one byte of codes) of 16 of them, whose
// bytes lie together: 16 bytes a store where all are written.
template <typename T>
__global__ void __launch_bounds__(256) k_kv4_write(const T *K, Kv4View kv, const T *V, Kv4View vv, Kv4Sequences q, int run,
                                                   int dim, int pitch, uint8_t *pool, int pages, int heads, bool vec) {
    const int s = blockIdx.y, h = blockIdx.x / run, tid = threadIdx.x;
    const kv4::Span a = kv4::span(q, s);
    if (a.n == 0) return;
    const int first = a.length - a.n, at = (first >> 6) + (int)(blockIdx.x % run);  // first may lie before 0
    if (at * 64 >= a.length) return;
    const int page = kv4::page_of(q, s, at, pages);
    if (page < 0) return;
    // positions lo .. hi - 1 of the page are written; position p is row `base` + p
    const int lo = max(first - at * 64, 0), hi = min(a.length - at * 64, 64);
    const int64_t base = (int64_t)a.row + at * 64 - first;
    uint8_t *tile = pool + ((int64_t)page * heads + h) * (68 * pitch);
    const int nb = pitch / 32, wide = pitch / 8;
    for (int e = tid + lo * wide; e < hi * wide; e += 256) {
        const int p = e / wide, d = e % wide * 8;
        float v[8] = {};
        if (d < dim) kv4::load8(K + (base + p) * kv.stride + h * kv.head + kv.offset + d, vec, v);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) m = max(m, kv4::magnitude_bits(v[i]));
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, f8::kSwap1, 0xf, 0xf, true));
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, f8::kSwap2, 0xf, 0xf, true));
        const uint32_t byte = kv4::scale_byte(m);
        const float scale = kv4::code_scale(byte);
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = kv4::code_value(v[i], byte);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
        *(uint32_t *)(tile + p * (pitch / 2) + d / 2) = w;
        if (d % 32 == 0) tile[kv4::key_scales(pitch) + d / 32 * 64 + p % 16 * 4 + p / 16] = (uint8_t)byte;
    }
    const int lane = tid % 64, r = lane % 16, k = lane / 16;
    for (int b = tid / 64; b < nb; b += 4) {
        uint32_t w[4] = {}, scales[4] = {};
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int p = 16 * g + 4 * k + i, d = 32 * b + r;
                float x = 0.0f, y = 0.0f;
                if (p >= lo && p < hi) {
                    const T *row = V + (base + p) * vv.stride + h * vv.head + vv.offset;
                    if (d < dim) x = kv4::value(row[d]);
                    if (d + 16 < dim) y = kv4::value(row[d + 16]);
                }
                uint32_t m = max(kv4::magnitude_bits(x), kv4::magnitude_bits(y));
                m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, f8::kSwap1, 0xf, 0xf, true));
                m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, f8::kSwap2, 0xf, 0xf, true));
                m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, f8::kMirror8, 0xf, 0xf, true));
                m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, f8::kMirror16, 0xf, 0xf, true));
                const uint32_t byte = kv4::scale_byte(m);
                const float scale = kv4::code_scale(byte);
                x = kv4::code_value(x, byte), y = kv4::code_value(y, byte);
                if (i == 0) w[g] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[g], x, y, scale, 0);
                if (i == 1) w[g] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[g], x, y, scale, 1);
                if (i == 2) w[g] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[g], x, y, scale, 2);
                if (i == 3) w[g] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[g], x, y, scale, 3);
                scales[g] |= byte << (8 * i);
            }
        uint8_t *codes = tile + kv4::value_codes(pitch) + b * 1024 + lane * 16;
        uint8_t *bytes = tile + kv4::value_scales(pitch) + b * 64 + k * 16;
        if (lo == 0 && hi == 64) {
            *(uint4 *)codes = make_uint4(w[0], w[1], w[2], w[3]);
            if (r == 0) *(uint4 *)bytes = make_uint4(scales[0], scales[1], scales[2], scales[3]);
        } else {
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int p = 16 * g + 4 * k + i;
                    if (p < lo || p >= hi) continue;
                    codes[4 * g + i] = (uint8_t)(w[g] >> (8 * i));
                    if (r == 0) bytes[4 * g + i] = (uint8_t)(scales[g] >> (8 * i));
                }
        }
    }
}

// -------------------------------------------------------------------- read
// The same shares. What a code stands for is exact in bf16.
__device__ __forceinline__ void values_of(uint32_t w, float scale, float v[8]) {
    const kv4::f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1),
                     c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = c[0], v[5] = c[1], v[6] = d[0], v[7] = d[1];
}

template <typename T>
__global__ void __launch_bounds__(256) k_kv4_read(const uint8_t *pool, int pages, int heads, int dim, int pitch, Kv4Sequences q,
                                                  int run, T *K, Kv4View kv, T *V, Kv4View vv, bool vec) {
    const int s = blockIdx.y, h = blockIdx.x / run, tid = threadIdx.x;
    const kv4::Span a = kv4::span(q, s);
    if (a.n == 0) return;
    const int first = a.length - a.n, at = (first >> 6) + (int)(blockIdx.x % run);
    if (at * 64 >= a.length) return;
    const int page = kv4::page_of(q, s, at, pages);
    // positions lo .. hi - 1 of the page have rows; those of no page are zeros
    const int lo = max(first - at * 64, 0), hi = min(a.length - at * 64, 64);
    const int64_t base = (int64_t)a.row + at * 64 - first;
    const uint8_t *tile = pool + ((int64_t)max(page, 0) * heads + h) * (68 * pitch);
    const int nb = pitch / 32, wide = pitch / 8;
    for (int e = tid + lo * wide; e < hi * wide; e += 256) {
        const int p = e / wide, d = e % wide * 8;
        if (d >= dim) continue;
        float v[8] = {};
        if (page >= 0) {
            const uint32_t byte = tile[kv4::key_scales(pitch) + d / 32 * 64 + p % 16 * 4 + p / 16];
            values_of(*(const uint32_t *)(tile + p * (pitch / 2) + d / 2), kv4::scale_value(byte), v);
        }
        kv4::store8(K + (base + p) * kv.stride + h * kv.head + kv.offset + d, vec, v);
    }
    const int lane = tid % 64, r = lane % 16, k = lane / 16;
    for (int b = tid / 64; b < nb; b += 4) {
        const uint4 w4 = *(const uint4 *)(tile + kv4::value_codes(pitch) + b * 1024 + lane * 16);
        const uint4 s4 = *(const uint4 *)(tile + kv4::value_scales(pitch) + b * 64 + k * 16);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w}, scales[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int p = 16 * g + 4 * k + i, d = 32 * b + r;
                if (p < lo || p >= hi) continue;
                kv4::f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[g] >> (8 * i),
                                                                        kv4::scale_value(scales[g] >> (8 * i) & 255u), 0);
                if (page < 0) v[0] = v[1] = 0.0f;
                T *row = V + (base + p) * vv.stride + h * vv.head + vv.offset;
                if (d < dim) kv4::store1(row + d, v[0]);
                if (d + 16 < dim) kv4::store1(row + d + 16, v[1]);
            }
    }
}

// ----------------------------------------------------------- norm and rotate
// `lanes` lanes (a power of two, 32 at most) a head, eight dimensions each.
// The dimension that another is turned with lies half the rotated ones away:
// its value is read again (from the caches) rather than exchanged. The squares
// are summed in f64 and the power of two of 1 / sqrt(mean) is applied apart: a
// row of large values does not overflow, one of subnormal ones does not pass
// f32's range.
template <typename T>
__global__ void __launch_bounds__(256) k_qk_norm_rope(QkNormRope a, const T *Q, const T *K, T *Yq, T *Yk, int lanes, int items,
                                                      bool vec) {
    const int item = (int)((blockIdx.x * 256u + threadIdx.x) / (unsigned)lanes), lane = threadIdx.x % lanes, d = 8 * lane;
    const bool there = item < items && d < a.dim;
    const int all = a.heads + a.kv_heads, t = min(item, items - 1) / all, head = min(item, items - 1) % all;
    const bool is_q = head < a.heads;
    const int h = is_q ? head : head - a.heads;
    const Kv4View view = is_q ? a.q_view : a.k_view;
    const T *x = (is_q ? Q : K) + t * view.stride + h * view.head + view.offset;
    const float *gamma = is_q ? a.q_gamma : a.k_gamma;
    const int half = a.rotary / 2, position = a.positions[t];
    float v[8] = {}, g[8] = {};
    if (there) {
        kv4::load8(x + d, vec, v);
        kv4::load8(gamma + d, true, g);
    }
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 8; i++) sum += (double)v[i] * (double)v[i];
    if (lanes > 1) sum += f8::moved<f8::kSwap1>(sum);
    if (lanes > 2) sum += f8::moved<f8::kSwap2>(sum);
    if (lanes > 4) sum += f8::moved<f8::kMirror8>(sum);
    if (lanes > 8) sum += f8::moved<f8::kMirror16>(sum);
    if (lanes > 16) sum += __shfl_xor(sum, 16, 64);
    if (!there) return;
    const double root = 1.0 / sqrt(sum / (double)a.dim + (double)a.eps);
    const float inv = (float)__builtin_amdgcn_frexp_mant(root);
    const int inv_exp = __builtin_amdgcn_frexp_exp(root);
    const auto normed = [&](float value, float weight) { return __builtin_amdgcn_ldexpf(value, inv_exp) * inv * weight; };
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = normed(v[i], g[i]);
    if (d < a.rotary) {
        const bool inside = position >= 0 && position < a.context;
        const int64_t angle = (int64_t)(inside ? position : 0) * half;
        float o[8], og[8], c[8], s[8];
        if (half % 8 == 0) {  // all eight on one side
            const int other = d < half ? d + half : d - half, pair = d < half ? d : d - half;
            kv4::load8(x + other, vec, o);
            kv4::load8(gamma + other, true, og);
            kv4::load8(a.cos + angle + pair, true, c);
            kv4::load8(a.sin + angle + pair, true, s);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const bool turned = d + i < a.rotary;
                const int other = d + i < half ? d + i + half : d + i - half, pair = d + i < half ? d + i : d + i - half;
                o[i] = turned ? kv4::value(x[other]) : 0.0f, og[i] = turned ? gamma[other] : 0.0f;
                c[i] = turned ? a.cos[angle + pair] : 1.0f, s[i] = turned ? a.sin[angle + pair] : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (d + i >= a.rotary) continue;
            const float b = normed(o[i], og[i]);
            y[i] = inside ? (d + i < half ? y[i] * c[i] - b * s[i] : y[i] * c[i] + b * s[i]) : NAN;
        }
    }
    T *to = is_q ? Yq + ((int64_t)t * a.heads + h) * a.dim : Yk + ((int64_t)t * a.kv_heads + h) * a.dim;
    kv4::store8(to + d, true, y);
}

int run_of(int longest) { return (longest + 62) / 64 + 1; }  // pages that as many positions can touch

}  // namespace

namespace smi {

int kv4_write_launch(sm_ctx *ctx, const void *K, const Kv4View &kv, const void *V, const Kv4View &vv, bool bf16,
                     const Kv4Sequences &q, int heads, int dim, uint8_t *pool, int pages) {
    const int run = run_of(q.longest);
    const bool vec = kv.multiple_of(8);
    const dim3 grid((uint32_t)(run * heads), q.count);
    if (bf16)
        k_kv4_write<<<grid, 256, 0, ctx->stream>>>((const uint16_t *)K, kv, (const uint16_t *)V, vv, q, run, dim,
                                                   kv4_pitch(dim), pool, pages, heads, vec);
    else
        k_kv4_write<<<grid, 256, 0, ctx->stream>>>((const float *)K, kv, (const float *)V, vv, q, run, dim, kv4_pitch(dim), pool,
                                                   pages, heads, vec);
    return launched(ctx);
}

int kv4_read_launch(sm_ctx *ctx, const uint8_t *pool, int pages, int heads, int dim, const Kv4Sequences &q, void *K,
                    const Kv4View &kv, void *V, const Kv4View &vv, bool bf16) {
    const int run = run_of(q.longest);
    const bool vec = kv.multiple_of(8);
    const dim3 grid((uint32_t)(run * heads), q.count);
    if (bf16)
        k_kv4_read<<<grid, 256, 0, ctx->stream>>>(pool, pages, heads, dim, kv4_pitch(dim), q, run, (uint16_t *)K, kv,
                                                  (uint16_t *)V, vv, vec);
    else
        k_kv4_read<<<grid, 256, 0, ctx->stream>>>(pool, pages, heads, dim, kv4_pitch(dim), q, run, (float *)K, kv, (float *)V, vv,
                                                  vec);
    return launched(ctx);
}

int qk_norm_rope_launch(sm_ctx *ctx, const QkNormRope &a, const void *Q, const void *K, void *Yq, void *Yk, bool bf16) {
    int lanes = 1;
    while (8 * lanes < a.dim) lanes *= 2;
    const int items = a.tokens * (a.heads + a.kv_heads);
    const bool vec = a.q_view.multiple_of(8) && a.k_view.multiple_of(8);
    const uint32_t grid = (uint32_t)(((int64_t)items * lanes + 255) / 256);
    if (bf16)
        k_qk_norm_rope<<<grid, 256, 0, ctx->stream>>>(a, (const uint16_t *)Q, (const uint16_t *)K, (uint16_t *)Yq, (uint16_t *)Yk,
                                                      lanes, items, vec);
    else
        k_qk_norm_rope<<<grid, 256, 0, ctx->stream>>>(a, (const float *)Q, (const float *)K, (float *)Yq, (float *)Yk, lanes,
                                                      items, vec);
    return launched(ctx);
}

}  // namespace smi
