// The key-value cache in 4 bits: positions written and read back, and the
// pass before it, the norm and rotation of each head's query and key.
//
// All three read each value once and write it once: bound by memory.
#include "kv4_device.h"

namespace {
using namespace smi;

// Write and read: a workgroup takes 64 dimensions of a page and head, of its
// keys or of its values; a thread 16 bytes of neighbouring dimensions of some
// positions, four threads (bf16) or eight a block of 32, so that a wave's loads
// and stores are without gaps (with 32 bytes a thread f32 values took 147 us
// where they take 58: 4 sequences of up to 16384 positions, 2 heads of 256
// dimensions). Keys' codes lie in memory as the threads have them;
// values' (whose bytes are two dimensions of a position, 16 positions together)
// pass through LDS on their way, so that both sides are read and written in
// pieces of 16 bytes. 64 dimensions of one kind a workgroup: enough of them for
// one token each of 32 sequences of 8 heads of 128, 5 us to write and 4 to
// read. The 4 sequences are read into bf16 in 38 us, 3.9 TB/s.
struct Share {
    int head, part, page;  // `part`: which 64 dimensions; page -1: none
    int lo, hi;            // the page's positions that have rows; none: lo = hi
    int64_t row;           // position 0's
};
// run > 0: sequence blockIdx.y, the blockIdx.x % run-th page that its rows
// touch. run = 0: the pages of all sequences' rows lie in blockIdx.x one after
// another, and a workgroup looks for its own.
__device__ __forceinline__ Share share_of(const Kv4Sequences &q, int run, int heads, int pages) {
    int s = blockIdx.y, h, number;
    kv4::Span a;
    if (run > 0) {
        h = blockIdx.x / run, number = blockIdx.x % run;
        a = kv4::span(q, s);
    } else {
        const int unit = blockIdx.x / heads, lane = threadIdx.x % 64;
        h = blockIdx.x % heads, number = 0, a = {0, 0, 0};
        for (int at = 0, before = 0; at < q.count; at += 64) {
            const kv4::Span b = at + lane < q.count ? kv4::span(q, at + lane) : kv4::Span{0, 0, 0};
            const int mine = b.n > 0 ? ((b.length - 1) >> 6) - ((b.length - b.n) >> 6) + 1 : 0;
            int upto = mine;
#pragma unroll
            for (int i = 1; i < 64; i *= 2) {
                const int other = __shfl_up(upto, i, 64);
                if (lane >= i) upto += other;
            }
            const uint64_t past = __ballot(before + upto > unit && mine > 0);
            if (past) {
                const int who = __ffsll((unsigned long long)past) - 1;
                const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, who); };
                s = at + who, number = unit - before - (of(upto) - of(mine)), a = {of(b.row), of(b.n), of(b.length)};
                break;
            }
            before += __builtin_amdgcn_readlane(upto, 63);
        }
    }
    const int first = a.length - a.n, at = (first >> 6) + number, parts = gridDim.z / 2;  // first may lie before 0
    if (a.n == 0 || at * 64 >= a.length) return {h, 0, -1, 0, 0, 0};
    return {h, (int)blockIdx.z % parts, kv4::page_of(q, s, at, pages), max(first - at * 64, 0), min(a.length - at * 64, 64),
            (int64_t)a.row + at * 64 - first};
}

// How a thread's values lie: kPer of position tid / kWide + kStep * j.
template <typename T>
struct Lanes {
    static constexpr int kPer = 16 / sizeof(T), kWide = 64 / kPer, kStep = 256 / kWide, kTurns = 64 / kStep, kBlock = 32 / kPer;
};

template <typename T, bool vec>
__global__ void __launch_bounds__(256) k_kv4_write(const T *K, Kv4View kv, const T *V, Kv4View vv, Kv4Sequences q, int run,
                                                   int dim, int pitch, uint8_t *pool, int pages, int heads) {
    using L = Lanes<T>;
    __shared__ __attribute__((aligned(16))) uint8_t s_codes[2048], s_scales[128];
    const Share a = share_of(q, run, heads, pages);
    if (a.page < 0) return;
    const bool values = blockIdx.z >= gridDim.z / 2;
    const int tid = threadIdx.x, at = tid % L::kWide * L::kPer, d = 64 * a.part + at, b = at / 32, r0 = at % 16;
    const bool first = at % 32 == 0, upper = at % 32 >= 16;
    uint8_t *tile = pool + ((int64_t)a.page * heads + a.head) * (68 * pitch);
    const T *x = values ? V : K;
    const Kv4View view = values ? vv : kv;
    kv4::Piece16<T> in[L::kTurns];
#pragma unroll
    for (int j = 0; j < L::kTurns; j++) {
        const int p = tid / L::kWide + L::kStep * j;
        in[j].clear();
        if (p >= a.lo && p < a.hi && d < dim) in[j].template load<vec>(x + (a.row + p) * view.stride + a.head * view.head + view.offset + d);
    }
#pragma unroll
    for (int j = 0; j < L::kTurns; j++) {
        const int p = tid / L::kWide + L::kStep * j;
        float v[8];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < L::kPer; i++) v[i] = in[j].at(i), m = max(m, kv4::magnitude_bits(v[i]));
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, f8::kSwap1, 0xf, 0xf, true));
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, f8::kSwap2, 0xf, 0xf, true));
        if (L::kBlock > 4) m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, f8::kMirror8, 0xf, 0xf, true));
        const uint32_t byte = kv4::scale_byte(m);
        const float scale = kv4::code_scale(byte);
#pragma unroll
        for (int i = 0; i < L::kPer; i++) v[i] = kv4::code_value(v[i], byte);
        uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, v[0], v[1], scale, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
        if constexpr (L::kPer == 8) {
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
        }
        if (!values) {
            if (p < a.lo || p >= a.hi) continue;
            uint8_t *to = tile + p * (pitch / 2) + d / 2;
            if constexpr (L::kPer == 8) *(uint32_t *)to = w;
            else *(uint16_t *)to = (uint16_t)w;
            if (first) tile[kv4::key_scales(pitch) + d / 32 * 64 + p % 16 * 4 + p / 16] = (uint8_t)byte;
        } else {
            // dimensions r and r + 16 in a byte: the thread half a block further has the other ones; half of the bytes each
            const uint32_t other = L::kBlock == 4 ? (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, f8::kSwap2, 0xf, 0xf, true)
                                                  : (uint32_t)__shfl_xor((int)w, 4, 64);
            constexpr int kHalf = L::kPer / 2;
            const uint32_t low = upper ? other >> (4 * kHalf) : w, high = upper ? w >> (4 * kHalf) : other;
            const int r = r0 + (upper ? kHalf : 0), place = 16 * ((b * 4 + p / 4 % 4) * 16 + r) + p / 16 * 4 + p % 4;
#pragma unroll
            for (int i = 0; i < kHalf; i++) s_codes[place + 16 * i] = (uint8_t)((low >> (4 * i) & 15u) | (high >> (4 * i) & 15u) << 4);
            if (first) s_scales[b * 64 + p / 4 % 4 * 16 + p / 16 * 4 + p % 4] = (uint8_t)byte;
        }
    }
    if (!values) return;
    __syncthreads();
    // 16 bytes each: block, quarter k and (codes) dimension; byte 4 g + i is position 16 g + 4 k + i
    if (tid >= 136) return;
    const bool codes = tid < 128;
    const int u = codes ? tid : tid - 128, k = codes ? u / 16 % 4 : u % 4;
    const uint4 w4 = codes ? ((const uint4 *)s_codes)[u] : ((const uint4 *)s_scales)[u];
    uint8_t *to = codes ? tile + kv4::value_codes(pitch) + 2048 * a.part + 16 * u : tile + kv4::value_scales(pitch) + 128 * a.part + 16 * u;
    if (a.lo == 0 && a.hi == 64) {
        *(uint4 *)to = w4;
        return;
    }
    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
    for (int g = 0; g < 4; g++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (16 * g + 4 * k + i >= a.lo && 16 * g + 4 * k + i < a.hi) to[4 * g + i] = (uint8_t)(w[g] >> (8 * i));
}

// What a code stands for is exact in bf16.
template <typename T, bool vec>
__global__ void __launch_bounds__(256) k_kv4_read(const uint8_t *pool, int pages, int heads, int dim, int pitch, Kv4Sequences q,
                                                  int run, T *K, Kv4View kv, T *V, Kv4View vv) {
    using L = Lanes<T>;
    __shared__ __attribute__((aligned(8))) uint8_t s_codes[64][40];  // of a position: bytes 16 b + r; rows of 8 more for the banks
    const Share a = share_of(q, run, heads, pages);
    if (a.lo == a.hi) return;
    const bool values = blockIdx.z >= gridDim.z / 2;
    const int tid = threadIdx.x, at = tid % L::kWide * L::kPer, d = 64 * a.part + at, b = at / 32, r0 = at % 16;
    const bool upper = at % 32 >= 16;
    // positions of no page are zeros
    const uint8_t *tile = pool + ((int64_t)max(a.page, 0) * heads + a.head) * (68 * pitch);
    uint32_t bytes[L::kTurns], w[L::kTurns];
#pragma unroll
    for (int j = 0; j < L::kTurns; j++) {
        const int p = tid / L::kWide + L::kStep * j;
        bytes[j] = tile[values ? kv4::value_scales(pitch) + d / 32 * 64 + p / 4 % 4 * 16 + p / 16 * 4 + p % 4
                               : kv4::key_scales(pitch) + d / 32 * 64 + p % 16 * 4 + p / 16];
        const uint8_t *from = tile + p * (pitch / 2) + d / 2;
        if (!values) w[j] = L::kPer == 8 ? *(const uint32_t *)from : *(const uint16_t *)from;
    }
    if (values) {
        // half of 16 bytes each: block, quarter k, dimension; byte 4 g + i is position 16 g + 4 k + i
        const int u = tid / 2, k = u / 16 % 4, g0 = tid % 2 * 2;
        const uint2 two = *(const uint2 *)(tile + kv4::value_codes(pitch) + 2048 * a.part + 8 * tid);
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                s_codes[16 * (g0 + g) + 4 * k + i][u / 64 * 16 + u % 16] = (uint8_t)((g == 0 ? two.x : two.y) >> (8 * i));
        __syncthreads();
    }
    const Kv4View view = values ? vv : kv;
    T *x = values ? V : K;
#pragma unroll
    for (int j = 0; j < L::kTurns; j++) {
        const int p = tid / L::kWide + L::kStep * j;
        if (p < a.lo || p >= a.hi || d >= dim) continue;
        const float scale = kv4::scale_value(bytes[j]);
        float v[8];
        if (values) {
            uint32_t some[2];
            some[0] = *(const uint32_t *)&s_codes[p][16 * b + r0];
            if (L::kPer == 8) some[1] = *(const uint32_t *)&s_codes[p][16 * b + r0 + 4];
#pragma unroll
            for (int i = 0; i < L::kPer; i++) {
                const kv4::f32x2 f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(some[i / 4] >> (8 * (i % 4)), scale, 0);
                v[i] = upper ? f[1] : f[0];
            }
        } else {
            const kv4::f32x2 f0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], scale, 0), f1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], scale, 1);
            v[0] = f0[0], v[1] = f0[1], v[2] = f1[0], v[3] = f1[1];
            if constexpr (L::kPer == 8) {
                const kv4::f32x2 f2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], scale, 2), f3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], scale, 3);
                v[4] = f2[0], v[5] = f2[1], v[6] = f3[0], v[7] = f3[1];
            }
        }
        if (a.page < 0)
#pragma unroll
            for (int i = 0; i < L::kPer; i++) v[i] = 0.0f;
        kv4::store16<vec>(x + (a.row + p) * view.stride + a.head * view.head + view.offset + d, v);
    }
}

// ----------------------------------------------------------- norm and rotate
// kLanes lanes (a power of two, 16 at most) a head, 16 dimensions each in
// pieces of 16 bytes. The dimension that another is turned with lies half the
// rotated ones away: its value is read again (from the caches) rather than
// exchanged, and every load is under way before any is waited for. 4096 tokens
// of 24 and 2 heads of 256 dimensions, queries beside their gates: 33 us, 3.3
// TB/s, three quarters of it waiting for memory. The squares
// are summed in f64 and the power of two of 1 / sqrt(mean) is applied apart: a
// row of large values does not overflow, one of subnormal ones does not pass
// f32's range. kFast: everything lies aligned to 16 bytes, and half the rotated
// dimensions are a multiple of a piece's, so that a piece lies on one side.
template <typename T, int kLanes, bool kFast>
__global__ void __launch_bounds__(256) k_qk_norm_rope(QkNormRope a, const T *Q, const T *K, T *Yq, T *Yk, uint32_t items) {
    constexpr int kPer = 16 / sizeof(T), kPieces = 16 / kPer;
    const uint32_t all = a.heads + a.kv_heads, first = blockIdx.x * (256 / kLanes), t0 = first / all, own = threadIdx.x / kLanes;
    const int lane = threadIdx.x % kLanes;
    const uint32_t place = first - t0 * all + min(own, items - 1 - first);
    const uint32_t more = (uint32_t)(((float)place + 0.5f) / (float)all);  // place < 2^11 + 256: half a step off any border
    const uint32_t t = t0 + more, head = place - more * all;
    const bool is_q = head < (uint32_t)a.heads;
    const uint32_t h = is_q ? head : head - a.heads;
    const Kv4View view = is_q ? a.q_view : a.k_view;
    const T *x = (is_q ? Q : K) + t * view.stride + h * view.head + view.offset;
    const float *gamma = is_q ? a.q_gamma : a.k_gamma;
    const int half = a.rotary / 2, position = a.positions[t];
    const bool inside = position >= 0 && position < a.context;
    const int64_t angle = (int64_t)(inside ? position : 0) * half;
    kv4::Piece16<T> v[kPieces], o[kPieces];
    kv4::Piece16<float> g[kPieces][kPer / 4], og[kPieces][kPer / 4], c[kPieces][kPer / 4], s[kPieces][kPer / 4];
#pragma unroll
    for (int e = 0; e < kPieces; e++) {
        const int d = kPer * (lane + e * kLanes);
        v[e].clear();
        if (d < a.dim) {
            v[e].template load<kFast>(x + d);
#pragma unroll
            for (int n = 0; n < kPer / 4; n++) g[e][n].template load<true>(gamma + d + 4 * n);
        }
        if (d >= a.rotary) continue;
        if constexpr (kFast) {
            const int other = d < half ? d + half : d - half, pair = d < half ? d : d - half;
            o[e].template load<true>(x + other);
#pragma unroll
            for (int n = 0; n < kPer / 4; n++) {
                og[e][n].template load<true>(gamma + other + 4 * n);
                c[e][n].template load<true>(a.cos + angle + pair + 4 * n);
                s[e][n].template load<true>(a.sin + angle + pair + 4 * n);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                const int at = min(d + i, a.rotary - 1);
                const int other = at < half ? at + half : at - half, pair = at < half ? at : at - half;
                o[e].v[i] = x[other], og[e][i / 4].v[i % 4] = gamma[other];
                c[e][i / 4].v[i % 4] = a.cos[angle + pair], s[e][i / 4].v[i % 4] = a.sin[angle + pair];
            }
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < kPieces; e++)
#pragma unroll
        for (int i = 0; i < kPer; i++) sum = fma((double)v[e].at(i), (double)v[e].at(i), sum);
    if (kLanes > 1) sum += f8::moved<f8::kSwap1>(sum);
    if (kLanes > 2) sum += f8::moved<f8::kSwap2>(sum);
    if (kLanes > 4) sum += f8::moved<f8::kMirror8>(sum);
    if (kLanes > 8) sum += f8::moved<f8::kMirror16>(sum);
    if (first + own >= items) return;
    // 1 / sqrt: the unit's (2^-26 or better), one step of Newton's beyond what f32 shows
    const double mean = sum * (1.0 / a.dim) + (double)a.eps, guess = __builtin_amdgcn_rsq(mean);
    const double root = mean > 0.0 && mean < INFINITY ? guess * (1.5 - 0.5 * mean * guess * guess) : guess;
    const float inv = (float)__builtin_amdgcn_frexp_mant(root);
    const int inv_exp = __builtin_amdgcn_frexp_exp(root);
    const auto normed = [&](float value, float weight) { return __builtin_amdgcn_ldexpf(value, inv_exp) * inv * weight; };
    T *to = is_q ? Yq + ((int64_t)t * a.heads + h) * a.dim : Yk + ((int64_t)t * a.kv_heads + h) * a.dim;
#pragma unroll
    for (int e = 0; e < kPieces; e++) {
        const int d = kPer * (lane + e * kLanes);
        if (d >= a.dim) continue;
        float y[8];
#pragma unroll
        for (int i = 0; i < kPer; i++) y[i] = normed(v[e].at(i), g[e][i / 4].v[i % 4]);
        if (d < a.rotary) {
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                if (!kFast && d + i >= a.rotary) continue;
                const float b = normed(o[e].at(i), og[e][i / 4].v[i % 4]), turned = d + i < half ? -b : b;
                const float moved = y[i] * c[e][i / 4].v[i % 4] + turned * s[e][i / 4].v[i % 4];
                y[i] = inside ? moved : NAN;
            }
        }
        kv4::store16<true>(to + d, y);
    }
}

// A launch's first two dimensions, and the share_of()'s run: each sequence as many pages as the longest one's rows can
// touch, or, where fewer than half of these can be there, all sequences' together. 255 sequences' single tokens and a prompt
// of 2048, 8 heads of 128 dimensions, are written in 36 us, and in 135 by the first; where all have as many rows the search
// costs more (4 sequences of up to 16384 positions read in 44 us, in 38 without it).
struct Pages {
    int run;
    uint32_t x, y;
};
Pages pages_of(const Kv4Sequences &q, int heads) {
    const int run = (q.longest + 62) / 64 + 1;
    const int64_t all = q.tokens / 64 + 2 * (int64_t)q.count;
    if ((int64_t)run * q.count > 2 * all) return {0, (uint32_t)(all * heads), 1};
    return {run, (uint32_t)(run * heads), (uint32_t)q.count};
}

template <typename T, int kLanes>
void norm_rope(sm_ctx *ctx, const QkNormRope &a, const T *Q, const T *K, T *Yq, T *Yk) {
    constexpr int kPer = 16 / sizeof(T);
    const uint32_t items = (uint32_t)a.tokens * (a.heads + a.kv_heads), grid = (items + 256 / kLanes - 1) / (256 / kLanes);
    if (a.rotary % (2 * kPer) == 0 && a.q_view.multiple_of(kPer) && a.k_view.multiple_of(kPer))
        k_qk_norm_rope<T, kLanes, true><<<grid, 256, 0, ctx->stream>>>(a, Q, K, Yq, Yk, items);
    else
        k_qk_norm_rope<T, kLanes, false><<<grid, 256, 0, ctx->stream>>>(a, Q, K, Yq, Yk, items);
}
template <typename T>
void norm_rope(sm_ctx *ctx, const QkNormRope &a, const T *Q, const T *K, T *Yq, T *Yk) {
    if (a.dim <= 16) norm_rope<T, 1>(ctx, a, Q, K, Yq, Yk);
    else if (a.dim <= 32) norm_rope<T, 2>(ctx, a, Q, K, Yq, Yk);
    else if (a.dim <= 64) norm_rope<T, 4>(ctx, a, Q, K, Yq, Yk);
    else if (a.dim <= 128) norm_rope<T, 8>(ctx, a, Q, K, Yq, Yk);
    else norm_rope<T, 16>(ctx, a, Q, K, Yq, Yk);
}

}  // namespace

namespace smi {

int kv4_write_launch(sm_ctx *ctx, const void *K, const Kv4View &kv, const void *V, const Kv4View &vv, bool bf16,
                     const Kv4Sequences &q, int heads, int dim, uint8_t *pool, int pages) {
    const int pitch = kv4_pitch(dim), per = bf16 ? 8 : 4;
    const auto [run, x, y] = pages_of(q, heads);
    const bool vec = kv.multiple_of(per) && vv.multiple_of(per);
    const dim3 grid(x, y, 2 * (pitch / 64));
#define SM_WRITE(T, VEC) \
    k_kv4_write<T, VEC><<<grid, 256, 0, ctx->stream>>>((const T *)K, kv, (const T *)V, vv, q, run, dim, pitch, pool, pages, heads)
    if (bf16 && vec) SM_WRITE(uint16_t, true);
    else if (bf16) SM_WRITE(uint16_t, false);
    else if (vec) SM_WRITE(float, true);
    else SM_WRITE(float, false);
#undef SM_WRITE
    return launched(ctx);
}

int kv4_read_launch(sm_ctx *ctx, const uint8_t *pool, int pages, int heads, int dim, const Kv4Sequences &q, void *K,
                    const Kv4View &kv, void *V, const Kv4View &vv, bool bf16) {
    const int pitch = kv4_pitch(dim), per = bf16 ? 8 : 4;
    const auto [run, x, y] = pages_of(q, heads);
    const bool vec = kv.multiple_of(per) && vv.multiple_of(per);
    const dim3 grid(x, y, 2 * (pitch / 64));
#define SM_READ(T, VEC) \
    k_kv4_read<T, VEC><<<grid, 256, 0, ctx->stream>>>(pool, pages, heads, dim, pitch, q, run, (T *)K, kv, (T *)V, vv)
    if (bf16 && vec) SM_READ(uint16_t, true);
    else if (bf16) SM_READ(uint16_t, false);
    else if (vec) SM_READ(float, true);
    else SM_READ(float, false);
#undef SM_READ
    return launched(ctx);
}

int qk_norm_rope_launch(sm_ctx *ctx, const QkNormRope &a, const void *Q, const void *K, void *Yq, void *Yk, bool bf16) {
    if (bf16) norm_rope(ctx, a, (const uint16_t *)Q, (const uint16_t *)K, (uint16_t *)Yq, (uint16_t *)Yk);
    else norm_rope(ctx, a, (const float *)Q, (const float *)K, (float *)Yq, (float *)Yk);
    return launched(ctx);
}

}  // namespace smi
