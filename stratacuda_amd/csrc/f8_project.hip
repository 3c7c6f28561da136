// Products of 8-bit matrices: project (f32 or bf16 out, a residual added) and
// gate_up (SiLU-gated pair, 8-bit out).
//
//   Y[t, n] = sum_b 2^(ex[t, b] + ew[n / 128, b]) * sum_{k in block b} x[t, k] w[n, k]
//
// Two ways to multiply:
//   f32 and gated outputs: code times scale as bf16 (exact: 4 significant bits in
//     8, the exponent of f32) in v_mfma_f32_16x16x32_bf16, whose sums are f32's
//     (1e-7 measured).
//   bf16 outputs: v_mfma_scale_f32_16x16x128_f8f6f4, one instruction a block of
//     128, which takes the two scales as operands, at twice the rate. It aligns
//     the products of each eight neighbours to the largest of them and cuts them
//     off 13 bits below its leading bit before it adds the eights in f32: off by
//     7 * 2^-13 of the sum of magnitudes at most (measured on one MI355X: 1.3e-5
//     of the result for normal values, where rounding to bf16 costs 1.7e-3).
// A gated pair takes f32 sums at every size: a block's scale is a decision on the
// largest of its 128 columns, and a code keeps four bits of a column however much
// of its sums has cancelled.
#include "f8_device.h"
#include "f8_shapes.h"

namespace {
using namespace smi;

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

using namespace f8;

// An operand of one block of 128 columns: the codes with their scale, or
// (EXACT) their values in bf16, 32 columns an instruction. Which 32 columns
// lie in which instruction and lane is one order for both matrices.
struct Codes {
    v8i v;
    int scale;
};
struct Values {
    v8b q[4];
};
template <bool EXACT>
__device__ __forceinline__ auto operand(v8i c, uint32_t scale) {
    if constexpr (EXACT) {
        Values r;
        const float s = __uint_as_float(scale << 23);  // its exponent alone is used
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const v2b lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], s, false);
            const v2b hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], s, true);
            r.q[i / 2][4 * (i % 2)] = lo[0], r.q[i / 2][4 * (i % 2) + 1] = lo[1];
            r.q[i / 2][4 * (i % 2) + 2] = hi[0], r.q[i / 2][4 * (i % 2) + 3] = hi[1];
        }
        return r;
    } else {
        return Codes{c, (int)scale};
    }
}
// acc[i] += w[i] . x, each 16 weight rows x 16 tokens: lane l holds token
// l % 16, rows 4 (l / 16) on.
template <int N>
__device__ __forceinline__ void multiply(const Codes (&w)[N], const Codes &x, v4f *const (&acc)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++)
        *acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[i].v, x.v, *acc[i], 0, 0, 0, w[i].scale, 0, x.scale);
}
template <int N>
__device__ __forceinline__ void multiply(const Values (&w)[N], const Values &x, v4f *const (&acc)[N]) {
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
        for (int i = 0; i < N; i++) *acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[i].q[q], x.q[q], *acc[i], 0, 0, 0);
}

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {  // nearest, ties to even; NaN stays NaN
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2b));
}
// g / (1 + exp(-g)) * u, with t = exp(-|g|) <= 1: silu(g) = g / (1 + t), or
// g t / (1 + t) below 0, so that nothing overflows and 1 + t lies in [1, 2].
// |g| log2(e) in two parts (the second corrects t to first order), one Newton
// step on the reciprocal: eight half steps of f32 at most. Powers of two come last: t is 2^-n times e in [0.7, 1.5]
// and u its fraction times 2^k, so that a gate whose exp(-|g|) lies below f32's
// range (|g| > 87) keeps its bits until u has brought the product back into it.
__device__ __forceinline__ float silu_times(float g, float u) {
    const float a = fabsf(g), p = a * 1.44269502f;  // log2(e) = 1.44269502 + 1.92596303e-8
    const float r = fmaf(a, 1.92596303e-8f, fmaf(a, 1.44269502f, -p));
    const float q = fminf(p, 1024.0f), whole = rintf(q);  // 2^-1024 brings the largest g and u to 0
    const float near = __builtin_amdgcn_exp2f(whole - q);
    const float e = fmaf(near, fmaxf(fminf(r * -0.693147182f, 1e-3f), -1e-3f), near);  // the bounds are for infinities alone
    const int n = -(int)whole;
    const float d = 1.0f + __builtin_amdgcn_ldexpf(e, n), y0 = __builtin_amdgcn_rcpf(d), y = fmaf(fmaf(-d, y0, 1.0f), y0, y0);
    const bool below = !(g >= 0.0f);
    const float h = g * (below ? e * y : y) * __builtin_amdgcn_frexp_mantf(u);
    return __builtin_amdgcn_ldexpf(h, __builtin_amdgcn_frexp_expf(u) + (below ? n : 0));
}

struct Product {
    const uint8_t *X, *Xs, *W, *Ws, *Wu, *Wus;  // Wu, Wus: the second matrix of a gated pair
    const float *R;
    void *Y;
    int tokens, rows, kb;  // rows: of one matrix
    uint64_t pitch, spitch;
    int64_t stride, offset;
    uint8_t *codes, *scales;  // kCodes: the outputs, and their rows' bytes
    uint64_t codes_pitch, scales_pitch;
};

// 16 bytes of a token's outputs, aligned: eight in bf16, or four to which R is added.
template <Out OUT>
__device__ __forceinline__ void store16(const Product &a, int64_t at, v4i v) {
    if constexpr (OUT == kBf16) {
        *(v4i *)((uint16_t *)a.Y + at) = v;
    } else {
        v4f y = __builtin_bit_cast(v4f, v);
        if (a.R) {
            const v4f o = *(const v4f *)(a.R + at);
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = o[i] + y[i];
        }
        *(v4f *)((float *)a.Y + at) = y;
    }
}
// The first `n` of four, anywhere.
template <Out OUT>
__device__ __forceinline__ void store_some(const Product &a, int64_t at, int n, v4f v) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (i >= n) break;
        if constexpr (OUT == kBf16) ((uint16_t *)a.Y)[at + i] = (uint16_t)bf16_pair(v[i], v[i]);
        else ((float *)a.Y)[at + i] = a.R ? a.R[at + i] + v[i] : v[i];
    }
}

// A wave's sums: 16 NT tokens from `first_token` on, 16 NR rows from `row` on;
// `whole`: all of the rows are there, and aligned.
template <Out OUT, int M, int NR, int NT>
__device__ __forceinline__ void store_tile(const Product &a, int first_token, int row, const v4f (&acc)[M][NR][NT], bool whole,
                                           int in, int part) {
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int token = first_token + t * 16;
        v4f h[NR];
#pragma unroll
        for (int r = 0; r < NR; r++) {
            h[r] = acc[0][r][t];
        }
        if (!whole) {
            if (token + in < a.tokens)
#pragma unroll
                for (int r = 0; r < NR; r++)
                    store_some<OUT>(a, (token + in) * a.stride + a.offset + row + 16 * r + 4 * part,
                                    a.rows - row - 16 * r - 4 * part, h[r]);
            continue;
        }
        // 16 bytes a lane at its token's row + `mine` and as much again at
        // `mine` + `more`
        v4i v[OUT == kBf16 ? NR / 2 : NR];
        if constexpr (OUT == kBf16) {
            // lanes 16 apart hold rows 4 on: of two sets of 16 rows one
            // lane takes the first's eight rows, the other the second's
#pragma unroll
            for (int r = 0; r < NR; r += 2) {
                const auto lo = __builtin_amdgcn_permlane16_swap(bf16_pair(h[r][0], h[r][1]), bf16_pair(h[r + 1][0], h[r + 1][1]), false, false);
                const auto hi = __builtin_amdgcn_permlane16_swap(bf16_pair(h[r][2], h[r][3]), bf16_pair(h[r + 1][2], h[r + 1][3]), false, false);
                v[r / 2] = v4i{(int)lo[0], (int)hi[0], (int)lo[1], (int)hi[1]};
            }
        } else {
#pragma unroll
            for (int r = 0; r < NR; r++) v[r] = __builtin_bit_cast(v4i, h[r]);
        }
        constexpr int kMore = OUT == kBf16 ? 32 : 16;
        const int mine = OUT == kBf16 ? 16 * (part % 2) + part / 2 * 8 : 4 * part;
        constexpr int kSets = sizeof(v) / sizeof(v[0]);
#pragma unroll
        for (int k = 0; k + 1 < kSets; k += 2) {
            // 128 bytes of a token in one store: the first stores the
            // first eight tokens of both, the second the other eight
            const bool low = in < 8;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int got = __builtin_amdgcn_update_dpp(0, low ? v[k + 1][i] : v[k][i], 0x128, 0xf, 0xf, true);  // of lane ^ 8
                v[k][i] = low ? v[k][i] : got;
                v[k + 1][i] = low ? got : v[k + 1][i];
            }
            const int64_t at = (token + in % 8) * a.stride + a.offset + row + mine + k * kMore + (low ? 0 : kMore);
            if (token + in % 8 < a.tokens) store16<OUT>(a, at, v[k]);
            if (token + in % 8 + 8 < a.tokens) store16<OUT>(a, at + 8 * a.stride, v[k + 1]);
        }
        if constexpr (kSets % 2)
            if (token + in < a.tokens) store16<OUT>(a, (token + in) * a.stride + a.offset + row + mine, v[kSets - 1]);
    }
}

// The sums of 16 rows from r0 on for one token a lane group.
template <Out OUT, int M>
__device__ __forceinline__ void store_few(const Product &a, v4f (&v)[M], int t, int r0, int part, bool vec) {
    if constexpr (OUT == kHidden)
#pragma unroll
        for (int i = 0; i < 4; i++) v[0][i] = silu_times(v[0][i], v[M - 1][i]);
    if (t >= a.tokens) return;
    const int64_t at = t * a.stride + a.offset + r0 + 4 * part;
    if (vec && r0 + 16 <= a.rows) {
        if constexpr (OUT == kBf16)
            *(uint2 *)((uint16_t *)a.Y + at) = make_uint2(bf16_pair(v[0][0], v[0][1]), bf16_pair(v[0][2], v[0][3]));
        else
            store16<OUT>(a, at, __builtin_bit_cast(v4i, v[0]));
    } else {
        store_some<OUT>(a, at, a.rows - r0 - 4 * part, v[0]);
    }
}

// Whether every n-th output of a token starts n aligned ones (buffers start aligned).
bool aligned(const Product &a, int n) { return a.stride % n == 0 && a.offset % n == 0; }

// ------------------------------------------------------ many tokens: tiles
// A workgroup of WT x WR waves makes BT tokens x BR weight rows (a gated pair:
// BR / 2 rows of each matrix). Each step brings one block of 128 columns of
// both into LDS by DMA (16 bytes a lane) while the step before is multiplied:
// two buffers, one barrier a step. A row's 128 bytes lie in eight slots of 16
// whose order goes by the row's number, so that the 16 lanes that read one
// column of 16 rows meet all banks. 256 x 256 takes all 256 registers: a gated
// tile spills 17, one to f32 4, none of them in the steps. 8192 tokens, 2560
// columns to 10,240 rows, to bf16: 204 us, 2.1 PFLOP/s, matrix units busy 0.51 of
// the cycles; gated, 4096 tokens, 4096 to 8192: 403 us, 1.37 PFLOP/s, as much as
// a library's bf16 product reaches.
typedef __attribute__((address_space(3))) void lds_void;
// Rows of codes as a buffer: a load of other rows gives zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t piece_buffer(const uint8_t *m, int first, int left, int rows, int most, uint64_t pitch) {
    const F8Piece p = f8_piece(first, left, rows, most);
    const uint32_t at = __builtin_amdgcn_readfirstlane(p.first), count = __builtin_amdgcn_readfirstlane(p.count);
    return __builtin_amdgcn_make_buffer_rsrc((void *)(m + at * pitch), 0, count * (uint32_t)pitch, 0x00027000);
}
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t from, uint32_t lane_offset, uint32_t offset, void *lds) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_void *)lds, 16, lane_offset, offset, 0, 0);
}
__device__ __forceinline__ void dma4(const uint8_t *src, void *lds) {
    __builtin_amdgcn_global_load_lds(src, (lds_void *)lds, 4, 0, 0);
}
// The waves' barrier alone (the waits are the callers'); the compiler moves no memory access over it.
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void *p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p;
}
__device__ __forceinline__ int swizzle(int row) { return row & 7; }

// The tiles in the order of the eight XCDs that workgroups go round: each XCD
// takes neighbouring tiles, four of tokens by as many of rows, so that its L2
// holds what they share.
struct Tiles {
    int tokens, rows, per_xcd;  // tiles; workgroups of an XCD (grid / 8, all of them if they are fewer than 8)
    __device__ __forceinline__ void locate(int at, int &t, int &r) const {
        const int panel = at / (4 * rows), width = min(4, tokens - 4 * panel), in_panel = at - panel * 4 * rows;
        const int across = in_panel / width;
        t = __builtin_amdgcn_readfirstlane(4 * panel + in_panel - across * width), r = __builtin_amdgcn_readfirstlane(across);
    }
};

template <int BT, int BR, int WT, int WR, bool EXACT, Out OUT>
__global__ void __launch_bounds__(64 * WT * WR) k_f8_tile(Product a, Tiles tiles, bool vec) {
    constexpr int kThreads = 64 * WT * WR, NT = BT / WT / 16, M = OUT == kCodes ? 2 : 1, NR = BR / WR / 16 / M;
    constexpr int kStage = (BT + BR) * 128, kRows = kThreads / 8;  // rows that the threads bring at a time
    static_assert(BT % kRows == 0 && BR / M % kRows == 0 && kRows % 8 == 0 && BT % 64 == 0 && BT / 64 < WT * WR && NT >= 2, "");
    // two variables, so that reads of one need not wait for the DMA into the other
    __shared__ __attribute__((aligned(16))) uint8_t s_even[kStage], s_odd[kStage];
    __shared__ uint32_t s_even_scale[BT + 64], s_odd_scale[BT + 64];
    const int lane = threadIdx.x % 64, in = lane % 16, part = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int wt = wave / WR, wr = wave % WR;
    const int xcd = blockIdx.x % 8, n = tiles.tokens * tiles.rows;
    const int first = xcd * (n / 8) + min(xcd, n % 8) + blockIdx.x / 8, end = (xcd + 1) * (n / 8) + min(xcd + 1, n % 8);
    if (first >= end) return;

    // ---- bringing steps, two ahead: past a tile's last they are the next tile's
    // A thread brings 16 bytes of every kRows-th row: of row threadIdx.x / 8 on.
    const uint32_t from = threadIdx.x / 8 * (uint32_t)a.pitch + ((threadIdx.x ^ swizzle(threadIdx.x / 8)) & 7) * 16;
    const int slot = min(wave, BT / 64);
    struct Place {
        int t0, r0, x_rows, w_rows;  // rows of the matrices that are left from there; 0 past the last tile
        const uint8_t *scale;
    };
    auto place = [&](int at) __attribute__((always_inline)) {
        Place p;
        tiles.locate(min(at, end - 1), p.t0, p.r0);
        p.t0 *= BT, p.r0 *= BR / M;
        p.x_rows = at < end ? a.tokens - p.t0 : 0, p.w_rows = at < end ? a.rows - p.r0 : 0;
        // four blocks' scales of a token, or (the waves behind those) of a wave's weight rows, lane WR m + wr
        p.scale = slot < BT / 64 ? a.Xs + (uint64_t)min(p.t0 + slot * 64 + lane, a.tokens - 1) * a.spitch
                                 : (M == 2 && lane / WR % M ? a.Wus : a.Ws) +
                                       (uint64_t)(min(p.r0 + lane % WR * NR * 16, a.rows - 1) / 128) * a.spitch;
        return p;
    };
    // A step's loads one by one, [first, last) of them: kPieces - 1 times
    // kRows rows, then the scales.
    constexpr int kPieces = (BT + BR) / kRows + 1;
    auto fetch = [&](const Place &p, int b, uint8_t *to, uint32_t *to_scale, int first_piece, int last_piece) __attribute__((always_inline)) {
#pragma unroll
        for (int i = first_piece; i < last_piece; i++) {
            const int j = i * kRows;  // of the stage's rows
            if (j == BT + BR) {
                dma4(p.scale + (b & ~3), to_scale + slot * 64);
                continue;
            }
            const int in_w = j - BT, row = in_w < 0 ? j : in_w % (BR / M);
            const auto buffer = in_w < 0 ? piece_buffer(a.X, p.t0 + row, p.x_rows - row, a.tokens, kRows, a.pitch)
                                         : piece_buffer(in_w < BR / M ? a.W : a.Wu, p.r0 + row, p.w_rows - row, a.rows, kRows, a.pitch);
            dma16(buffer, from, b * 128, to + wave * 1024 + j * 128);
        }
    };

    // ---- multiplying them
    v4f acc[M][NR][NT];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < M; m++)
#pragma unroll
            for (int r = 0; r < NR; r++)
#pragma unroll
                for (int t = 0; t < NT; t++) acc[m][r][t] = v4f{0, 0, 0, 0};
    };
    const int s0 = in * 128 + (part ^ swizzle(in)) * 16, s1 = in * 128 + ((part + 4) ^ swizzle(in)) * 16;
    auto frag = [&](const uint8_t *q) __attribute__((always_inline)) {
        const v4i lo = *(const v4i *)(q + s0), hi = *(const v4i *)(q + s1);
        return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    // A step's weights, its first 32 tokens and its scales are read while the
    // step before still multiplies, later tokens 32 ahead.
    decltype(operand<EXACT>(v8i{}, 0)) wf[M * NR];
    v8i xf[2];
    uint32_t sx[NT], sw[M];
    auto weights = [&](const uint8_t *cur, int i) __attribute__((always_inline)) {
        return operand<EXACT>(frag(cur + (BT + i / NR * (BR / 2)) * 128 + (wr * NR + i % NR) * 2048), sw[i / NR]);
    };
    auto scales = [&](int b, const uint32_t *scale) __attribute__((always_inline)) {
        const int shift = 8 * (b & 3);
#pragma unroll
        for (int m = 0; m < M; m++) sw[m] = scale[BT + m * WR + wr] >> shift & 255u;
#pragma unroll
        for (int t = 0; t < NT; t++) sx[t] = scale[(wt * NT + t) * 16 + in] >> shift & 255u;
    };
    // 8-bit outputs: a tile's 128 columns are one block of scales. A wave has 32
    // of them, so the largest magnitudes meet in LDS.
    __shared__ float s_most[OUT == kCodes ? WR : 1][OUT == kCodes ? BT : 1];
    auto finish_codes = [&](int t0, int r0) __attribute__((always_inline)) {
        static_assert(OUT != kCodes || (NR == 2 && BR == 256), "");
        const int col = wr * 32 + 4 * part;  // of the block
        const bool whole = r0 + BR / M <= a.rows;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float most = 0.0f;
#pragma unroll
            for (int r = 0; r < NR; r++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float h = silu_times(acc[0][r][t][i], acc[M - 1][r][t][i]);
                    acc[0][r][t][i] = whole || r0 + col + 16 * r + i < a.rows ? h : 0.0f;
                    most = fmaxf(most, f8::finite_magnitude(acc[0][r][t][i]));
                }
            most = fmaxf(most, __shfl_xor(most, 16, 64));
            most = fmaxf(most, __shfl_xor(most, 32, 64));
            if (part == 0) s_most[wr][(wt * NT + t) * 16 + in] = most;
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
        barrier();
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int token = t0 + (wt * NT + t) * 16 + in;
            float most = s_most[0][(wt * NT + t) * 16 + in];
#pragma unroll
            for (int k = 1; k < WR; k++) most = fmaxf(most, s_most[k][(wt * NT + t) * 16 + in]);
            const uint32_t byte = f8::scale_byte(most);
            const float inverse = f8::inverse_scale(byte);
            // of two sets of 16 columns one lane takes eight of the first, the other eight of the second
            const auto v = __builtin_amdgcn_permlane16_swap(f8::codes4(acc[0][0][t], inverse), f8::codes4(acc[0][NR - 1][t], inverse), false, false);
            if (token < a.tokens) {
                *(uint2 *)(a.codes + token * a.codes_pitch + r0 + wr * 32 + 16 * (part % 2) + part / 2 * 8) = make_uint2(v[0], v[1]);
                if (wr == 0 && part == 0) {
                    uint8_t *to = a.scales + token * a.scales_pitch;
                    to[r0 / 128] = (uint8_t)byte;
                    if (r0 + 128 >= a.rows)
                        for (uint32_t k = r0 / 128 + 1; k < a.scales_pitch; k++) to[k] = 127;
                }
            }
        }
    };
    auto part_of = [&](int t) __attribute__((always_inline)) {
        v4f *to[M * NR];
#pragma unroll
        for (int i = 0; i < M * NR; i++) to[i] = &acc[i / NR][i % NR][t];
        multiply<M * NR>(wf, operand<EXACT>(xf[t & 1], sx[t]), to);
    };
    auto load_first = [&](const uint8_t *cur, const uint32_t *scale) __attribute__((always_inline)) {
        scales(0, scale);
        xf[0] = frag(cur + wt * NT * 2048), xf[1] = frag(cur + (wt * NT + 1) * 2048);
#pragma unroll
        for (int i = 0; i < M * NR; i++) wf[i] = weights(cur, i);
    };
    static_assert(NT % 2 == 0, "");
    int at = first;
    Place here = place(at), then = place(at + tiles.per_xcd);
    // The loads of the step after next begin when this one has been read, and
    // go on between the next one's first products, so that no wave waits to
    // issue them.
    constexpr int kSpread = NT - 2 < 2 ? NT - 2 : 2, kTail = kSpread ? (kPieces + 1) / 2 : kPieces;
    constexpr int kEach = kSpread ? (kPieces - kTail + kSpread - 1) / kSpread : 0;
    auto fetch_step = [&](int b, uint8_t *to, uint32_t *to_scale, int first_piece, int last_piece) __attribute__((always_inline)) {
        const bool over = b >= a.kb;
        const Place p = {over ? then.t0 : here.t0, over ? then.r0 : here.r0, over ? then.x_rows : here.x_rows,
                         over ? then.w_rows : here.w_rows, over ? then.scale : here.scale};
        fetch(p, over ? b - a.kb : b, to, to_scale, first_piece, last_piece);
    };
    auto step = [&](int b, uint8_t *cur, uint32_t *scale, uint8_t *next, uint32_t *next_scale) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t + 2 < NT; t++) {
            if (t < kSpread) fetch_step(b + 1, next, next_scale, min(kTail + t * kEach, kPieces), min(kTail + (t + 1) * kEach, kPieces));
            part_of(t);
            xf[t & 1] = frag(cur + (wt * NT + t + 2) * 2048);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0): the next step is in LDS, this one is read
        barrier();
        fetch_step(b + 2, cur, scale, 0, kTail);
        part_of(NT - 2);
        xf[0] = frag(next + wt * NT * 2048);
        part_of(NT - 1);
        scales(b + 1, next_scale);
#pragma unroll
        for (int i = 0; i < M * NR; i++) wf[i] = weights(next, i);
        xf[1] = frag(next + (wt * NT + 1) * 2048);
        __builtin_amdgcn_sched_barrier(0);
    };
    // One tile whose first step lies in `one`; its last steps bring the next
    // tile's first, so that its outputs are stored while those arrive.
    auto tile = [&](uint8_t *one, uint32_t *one_scale, uint8_t *two, uint32_t *two_scale) __attribute__((always_inline)) {
        load_first(one, one_scale);
        clear();
        int b = 0;
        for (; b + 1 < a.kb; b += 2) {
            step(b, one, one_scale, two, two_scale);
            step(b + 1, two, two_scale, one, one_scale);
        }
        if (b < a.kb) step(b, one, one_scale, two, two_scale);
        if constexpr (OUT == kCodes) finish_codes(here.t0, here.r0);
        else store_tile<OUT>(a, here.t0 + wt * NT * 16, here.r0 + wr * NR * 16, acc, here.r0 + BR / M <= a.rows && vec, in, part);
        at += tiles.per_xcd;
        here = then;
        then = place(at + tiles.per_xcd);
    };
    fetch(here, 0, s_even, s_even_scale, 0, kPieces);
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();
    fetch_step(1, s_odd, s_odd_scale, 0, kTail);
    while (true) {
        tile(s_even, s_even_scale, s_odd, s_odd_scale);
        if (at >= end) break;
        if (a.kb & 1) {
            tile(s_odd, s_odd_scale, s_even, s_even_scale);
            if (at >= end) break;
        }
    }
}

// ------------------------------------------------------ few tokens: streams
// A workgroup's W waves share 16 RR weight rows (of a gated pair: of both
// matrices) and 16 TT tokens and take the blocks of 128 columns in turn. A wave
// brings its block into its own part of LDS by DMA, eight lanes to a row's 128
// bytes, reads it into the matrix instructions' order, and has the next one under
// way while it multiplies; it waits for no other wave. Their sums meet in LDS,
// added in the waves' order. Bound by what L2 gives (16 TB/s) and, for one token,
// by a step's latency, which many small workgroups on a CU hide better than two or
// three blocks a wave under way (4 waves, 32 tokens, 2560 columns to 10,240 rows:
// 8.2 us with two, 7.6 with one; 32 tokens, 6144 to 2560 7.2 and 6.6, with eight
// waves 6.1). Fragments straight from memory, where every lane of an instruction
// is in another line, take 11.8.
struct Pair {
    v4i v[4];
};
// Two fragments of 16 rows from LDS: lane part's chunks {part, part + 4} of each.
template <int F, int G>
__device__ __forceinline__ Pair read_pair(uint32_t first, uint32_t second) {
    Pair p;
    asm volatile(
        "ds_read_b128 %0, %4 offset:%6\n\tds_read_b128 %1, %5 offset:%6\n\t"
        "ds_read_b128 %2, %4 offset:%7\n\tds_read_b128 %3, %5 offset:%7\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(p.v[0]), "=&v"(p.v[1]), "=&v"(p.v[2]), "=&v"(p.v[3])
        : "v"(first), "v"(second), "i"(2048 * F), "i"(2048 * G)
        : "memory");
    return p;
}
__device__ __forceinline__ v8i join(v4i a, v4i b) { return v8i{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}; }

template <int W, int RR, int TT, bool EXACT, Out OUT>
__global__ void __launch_bounds__(64 * W) k_f8_stream(Product a, int row_tiles, int token_tiles, bool vec) {
    constexpr int M = OUT == kHidden ? 2 : 1, kW = M * RR, kFrags = kW + TT, kStage = kFrags * 2048 + 512;
    constexpr int kSums = kW * TT * 1024, kPart = kStage > kSums ? kStage : kSums;
    static_assert(kFrags <= 8 && TT <= 4, "");
    __shared__ __attribute__((aligned(16))) uint8_t s_lds[W * kPart];
    const int lane = threadIdx.x % 64, in = lane % 16, part = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    // An XCD's workgroups take tiles that follow each other, eight token tiles of a weight tile first, so that those
    // that run together need few rows of both from its L2 (2048 tokens, 6144 columns to 2560 rows, f32, the same call again
    // and again: 87 us with all of them first, 78 so).
    const int xcd = blockIdx.x % 8, n = row_tiles * token_tiles, at = xcd * (n / 8) + min(xcd, n % 8) + blockIdx.x / 8;
    if ((int)(blockIdx.x / 8) >= n / 8 + (xcd < n % 8)) return;
    const int panel = at / (8 * row_tiles), width = min(8, token_tiles - 8 * panel), in_panel = at - panel * 8 * row_tiles;
    const int r0 = in_panel / width * 16 * RR, t0 = (8 * panel + in_panel % width) * 16 * TT;
    uint8_t *mine = s_lds + wave * kStage;
    const uint32_t from = lane / 8 * (uint32_t)a.pitch + ((lane ^ (lane / 8)) & 7) * 16, from8 = from + 8 * (uint32_t)a.pitch;
    const uint8_t *xs = a.Xs + (uint64_t)min(t0 + lane % (16 * TT), a.tokens - 1) * a.spitch;
    const uint8_t *ws = (M == 2 && lane % 2 ? a.Wus : a.Ws) + (uint64_t)(r0 / 128) * a.spitch;
    auto fetch = [&](int b) __attribute__((always_inline)) {
        if (b >= a.kb) return;
#pragma unroll
        for (int f = 0; f < kFrags; f++) {
            const int m = f / RR, first = f < kW ? r0 + f % RR * 16 : t0 + 16 * (f - kW);
            const uint8_t *src = f >= kW ? a.X : m ? a.Wu : a.W;
            const int rows = f < kW ? a.rows : a.tokens;
            const auto buffer = piece_buffer(src, first, rows - first, rows, 16, a.pitch);
            dma16(buffer, from, b * 128, mine + f * 2048);
            dma16(buffer, from8, b * 128, mine + f * 2048 + 1024);
        }
        dma4(xs + (b & ~3), mine + kFrags * 2048);
        dma4(ws + (b & ~3), mine + kFrags * 2048 + 256);
    };
    v4f acc[kW][TT];
#pragma unroll
    for (int m = 0; m < kW; m++)
#pragma unroll
        for (int t = 0; t < TT; t++) acc[m][t] = v4f{0, 0, 0, 0};
    fetch(wave);
    const uint32_t base = lds_address(mine);
    const uint32_t s0 = base + in * 128 + (part ^ swizzle(in)) * 16, s1 = base + in * 128 + ((part + 4) ^ swizzle(in)) * 16;
    for (int b = wave; b < a.kb; b += W) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this block is in LDS
        const uint32_t sc = base + kFrags * 2048;
        uint32_t c[6];
        asm volatile(
            "ds_read_b32 %0, %6\n\tds_read_b32 %1, %6 offset:64\n\tds_read_b32 %2, %6 offset:128\n\t"
            "ds_read_b32 %3, %6 offset:192\n\tds_read_b32 %4, %7\n\tds_read_b32 %5, %7 offset:4\n\ts_waitcnt lgkmcnt(0)"
            : "=&v"(c[0]), "=&v"(c[1]), "=&v"(c[2]), "=&v"(c[3]), "=&v"(c[4]), "=&v"(c[5])
            : "v"(sc + in * 4), "v"(sc + 256)
            : "memory");
        Pair p[4];
        p[0] = read_pair<0, 1>(s0, s1);
        if constexpr (kFrags > 2) p[1] = read_pair<2, kFrags == 3 ? 2 : 3>(s0, s1);
        if constexpr (kFrags > 4) p[2] = read_pair<4, kFrags == 5 ? 4 : 5>(s0, s1);
        if constexpr (kFrags > 6) p[3] = read_pair<6, kFrags == 7 ? 6 : 7>(s0, s1);
        fetch(b + W);  // it has been read
        const int shift = 8 * (b & 3);
        auto pair = [&](int f) __attribute__((always_inline)) { return join(p[f / 2].v[f % 2 * 2], p[f / 2].v[f % 2 * 2 + 1]); };
        decltype(operand<EXACT>(v8i{}, 0)) w[kW];
#pragma unroll
        for (int m = 0; m < kW; m++) w[m] = operand<EXACT>(pair(m), c[4 + m / RR] >> shift & 255u);
#pragma unroll
        for (int t = 0; t < TT; t++) {
            const auto x = operand<EXACT>(pair(kW + t), c[t] >> shift & 255u);
            if constexpr (kW == 4) multiply(w, x, {&acc[0][t], &acc[kW - 3][t], &acc[kW - 2][t], &acc[kW - 1][t]});
            else if constexpr (kW == 2) multiply(w, x, {&acc[0][t], &acc[kW - 1][t]});
            else multiply(w, x, {&acc[0][t]});
        }
    }
    barrier();  // every wave has read its blocks
    v4f *sums = (v4f *)s_lds;
#pragma unroll
    for (int m = 0; m < kW; m++)
#pragma unroll
        for (int t = 0; t < TT; t++) sums[((wave * kW + m) * TT + t) * 64 + lane] = acc[m][t];
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    barrier();
    for (int i = wave; i < RR * TT; i += W) {
        v4f v[M];
#pragma unroll
        for (int m = 0; m < M; m++) {
            v[m] = sums[(m * RR * TT + i) * 64 + lane];
            for (int k = 1; k < W; k++) {
                const v4f o = sums[((k * M + m) * RR * TT + i) * 64 + lane];
#pragma unroll
                for (int j = 0; j < 4; j++) v[m][j] = v[m][j] + o[j];
            }
        }
        store_few<OUT>(a, v, t0 + 16 * (i % TT) + in, r0 + 16 * (i / TT), part, vec);
    }
}

template <int W, int RR, int TT, bool EXACT, Out OUT>
void stream(sm_ctx *ctx, const Product &a) {
    const int row_tiles = (a.rows + 16 * RR - 1) / (16 * RR), token_tiles = (a.tokens + 16 * TT - 1) / (16 * TT);
    k_f8_stream<W, RR, TT, EXACT, OUT><<<(row_tiles * token_tiles + 7) / 8 * 8, 64 * W, 0, ctx->stream>>>(a, row_tiles, token_tiles, aligned(a, 4));
}
template <int BT, int BR, int WT, int WR, bool EXACT, Out OUT>
void tiles(sm_ctx *ctx, const Product &a, int cus, int resident) {
    const int m = OUT == kCodes ? 2 : 1;
    Tiles t = {(a.tokens + BT - 1) / BT, (a.rows + BR / m - 1) / (BR / m), 0};
    const int grid = tile_grid(t.tokens * t.rows, a.kb, cus, resident);
    t.per_xcd = grid / 8;
    k_f8_tile<BT, BR, WT, WR, EXACT, OUT><<<grid, 64 * WT * WR, 0, ctx->stream>>>(a, t, aligned(a, OUT == kBf16 ? 8 : 4));
}

int compute_units(sm_ctx *ctx) {
    int cus = 0;
    return hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, ctx->device) == hipSuccess && cus > 0 ? cus : 256;
}

template <bool EXACT, Out OUT>
void multiply_by_size(sm_ctx *ctx, const Product &a, int cus) {
    float us = 0.0f;
    const int best = best_shape(a.tokens, a.rows, a.kb, OUT, cus, &us), resident = kShapes[OUT][best].resident;
    if (best == 0) return stream<8, 1, 1, EXACT, OUT>(ctx, a);
    if (best == 1) return stream<8, 1, 2, EXACT, OUT>(ctx, a);
    if (best == 2) return stream<8, 2, 2, EXACT, OUT>(ctx, a);
    if constexpr (OUT == kHidden) {
        stream<4, 2, 4, EXACT, OUT>(ctx, a);
    } else {
        if (best == 3) return stream<8, 2, 4, EXACT, OUT>(ctx, a);
        if (best == 4) return stream<4, 4, 2, EXACT, OUT>(ctx, a);
        if (best == 5) return stream<4, 4, 4, EXACT, OUT>(ctx, a);
        if (best == 6) return tiles<128, 128, 2, 2, EXACT, OUT>(ctx, a, cus, resident);
        if (best == 7) return tiles<256, 128, 4, 2, EXACT, OUT>(ctx, a, cus, resident);
        if (best == 8) return tiles<256, 256, 2, 4, EXACT, OUT>(ctx, a, cus, resident);
        if constexpr (OUT == kBf16) tiles<64, 64, 2, 2, EXACT, OUT>(ctx, a, cus, resident);
    }
}

// A gated pair, in one kernel or two (f8_shapes.h).
int gate_up(sm_ctx *ctx, Product &a, uint8_t *codes, uint8_t *scales, void *workspace) {
    const int cus = compute_units(ctx);
    const F8Layout L = f8_layout(a.tokens, a.rows, 1);
    a.codes = codes, a.scales = scales, a.codes_pitch = L.pitch, a.scales_pitch = L.spitch;
    const int tile = gated_tile(a.tokens, a.rows, a.kb, cus);
    if (tile == 256) return tiles<256, 256, 2, 4, true, kCodes>(ctx, a, cus, 1), launched(ctx);
    if (tile == 128) return tiles<128, 256, 2, 4, true, kCodes>(ctx, a, cus, 1), launched(ctx);
    a.Y = workspace, a.stride = a.rows;
    multiply_by_size<true, kHidden>(ctx, a, cus);
    if (int rc = launched(ctx)) return rc;
    return f8_quantize_launch(ctx, workspace, false, a.tokens, a.rows, 1, codes, scales);
}

Product product_of(const F8Operand &X, const F8Operand &W, int tokens, int cols, int rows) {
    const F8Layout L = f8_layout(tokens, cols, 1);
    Product a = {};
    a.X = X.codes, a.Xs = X.scales, a.W = W.codes, a.Ws = W.scales;
    a.tokens = tokens, a.rows = rows, a.kb = (int)(L.pitch / 128);
    a.pitch = L.pitch, a.spitch = L.spitch;
    return a;
}

}  // namespace

namespace smi {

int f8_project_launch(sm_ctx *ctx, const F8Operand &X, int tokens, int cols, const F8Operand &W, int rows, const float *R,
                      void *Y, bool bf16, int64_t stride, int64_t offset) {
    Product a = product_of(X, W, tokens, cols, rows);
    a.R = R, a.Y = Y, a.stride = stride, a.offset = offset;
    if (bf16) multiply_by_size<false, kBf16>(ctx, a, compute_units(ctx));
    else multiply_by_size<true, kF32>(ctx, a, compute_units(ctx));
    return launched(ctx);
}

uint64_t f8_gate_up_workspace(int tokens, int ff) { return (uint64_t)tokens * ff * 4; }

int f8_gate_up_launch(sm_ctx *ctx, const F8Operand &X, int tokens, int cols, const F8Operand &Wg, const F8Operand &Wu, int ff,
                      uint8_t *codes, uint8_t *scales, void *workspace) {
    Product a = product_of(X, Wg, tokens, cols, ff);
    a.Wu = Wu.codes, a.Wus = Wu.scales;
    return gate_up(ctx, a, codes, scales, workspace);
}

}  // namespace smi
