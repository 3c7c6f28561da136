// Matrices into 8-bit floating point: the conversion (activations with a
// scale for each row, weights with a scale for each 128 rows) and the
// root-mean-square norm with the residual's addition.
//
// Both read each value once and write one byte for it: bound by memory. Half
// a wave holds one row's 128-column block, four columns a lane, so that a
// block's largest magnitude is five exchanges between lanes and its codes
// are one 128-byte line.
#include "f8_device.h"

namespace {
using namespace smi;

// ------------------------------------------------- a scale for each row
template <typename T>
__global__ void __launch_bounds__(256) k_f8_rows(const T *X, uint8_t *codes, uint8_t *scales, uint32_t blocks, int cols,
                                                 uint32_t kb, uint64_t pitch, uint32_t spitch, bool vec) {
    const uint32_t at = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
    if (at >= blocks) return;
    const uint32_t row = at / kb, b = at % kb;
    float v[4];
    f8::load4(X + (uint64_t)row * cols, b * 128 + 4 * lane, cols, vec, v);
    float m = fmaxf(fmaxf(f8::finite_magnitude(v[0]), f8::finite_magnitude(v[1])),
                    fmaxf(f8::finite_magnitude(v[2]), f8::finite_magnitude(v[3])));
    const uint32_t byte = f8::scale_byte(f8::half_wave_max(m));
    *(uint32_t *)(codes + row * pitch + b * 128 + 4 * lane) = f8::codes4(v, f8::inverse_scale(byte));
    if (lane == 0) scales[(uint64_t)row * spitch + b] = (uint8_t)byte;
    if (b == kb - 1 && lane >= 1 && b + lane < spitch) scales[(uint64_t)row * spitch + b + lane] = 127;
}

// --------------------------------------------- a scale for each 128 rows
// One workgroup a 128 x 128 block, held in registers between the maximum and
// the codes; 16 bytes a lane and load: half a wave a row in f32, a quarter in
// bf16 (10240 x 2560 from bf16: 19.6 us with 8 bytes a load, 18.7 with 16).
template <typename T>
__global__ void __launch_bounds__(256) k_f8_blocks(const T *X, uint8_t *codes, uint8_t *scales, int rows, int cols,
                                                   uint32_t kb, uint64_t pitch, uint32_t spitch, bool vec) {
    constexpr int kLanes = 8 * sizeof(T), kFours = 32 / kLanes, kRows = 256 / kLanes, N = 128 / kRows;  // kRows rows at a time
    const uint32_t br = blockIdx.x / kb, b = blockIdx.x % kb, lane = threadIdx.x % kLanes, first = threadIdx.x / kLanes;
    const int col = b * 128 + 4 * kFours * lane;
    __shared__ float s_max[4];
    float v[N][kFours][4], m = 0.0f;
#pragma unroll
    for (int j = 0; j < N; j++) {  // a row past the last repeats that one
        const T *row = X + (uint64_t)min((int)(br * 128 + j * kRows + first), rows - 1) * cols;
#pragma unroll
        for (int f = 0; f < kFours; f++) f8::load4(row, col + 4 * f, cols, vec, v[j][f]);
    }
#pragma unroll
    for (int j = 0; j < N; j++)
#pragma unroll
        for (int f = 0; f < kFours; f++)
#pragma unroll
            for (int i = 0; i < 4; i++) m = fmaxf(m, f8::finite_magnitude(v[j][f][i]));
    m = f8::half_wave_max(m);
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    if (threadIdx.x % 64 == 0) s_max[threadIdx.x / 64] = m;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; j++) m = fmaxf(m, s_max[j]);
    const uint32_t byte = f8::scale_byte(m);
    const float inverse = f8::inverse_scale(byte);
#pragma unroll
    for (int j = 0; j < N; j++) {
        const int row = br * 128 + j * kRows + first;
        if (row >= rows) break;
        uint8_t *to = codes + row * pitch + col;
        if constexpr (kFours == 2) *(uint2 *)to = make_uint2(f8::codes4(v[j][0], inverse), f8::codes4(v[j][kFours - 1], inverse));
        else *(uint32_t *)to = f8::codes4(v[j][0], inverse);
    }
    if (threadIdx.x == 0) scales[(uint64_t)br * spitch + b] = (uint8_t)byte;
    if (b == kb - 1 && threadIdx.x >= 1 && b + threadIdx.x < spitch)
        scales[(uint64_t)br * spitch + b + threadIdx.x] = 127;
}

// ------------------------------------------------------------------ norm
// One workgroup of `waves` waves a row; a wave takes 256 columns (two blocks)
// at a time. NI > 0: a lane's share of the row, up to 4 NI values, stays in
// registers between the sum of squares and the codes. NI = 0: rows of any
// length; the second pass reads the row again (H where it was written, so
// that H may be X or R itself).
// The squares are summed in f64: a row of large values does not overflow, and
// the order of the sum does not show in the codes.
template <typename T, int NI>
__global__ void __launch_bounds__(1024) k_f8_norm(const T *X, const float *R, const float *gamma, float eps, float *H,
                                                  uint8_t *codes, uint8_t *scales, int cols, uint32_t kb, uint64_t pitch,
                                                  uint32_t spitch, bool vec) {
    const uint64_t row = blockIdx.x;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, waves = blockDim.x / 64;
    const T *x = X + row * cols;
    const float *r = R ? R + row * cols : nullptr;
    float *h = H ? H + row * cols : nullptr;
    __shared__ double s_sum[16];
    constexpr int N = NI > 0 ? NI : 1;
    float v[N][4], t[N][4];
    double sum = 0.0;
    const int steps = NI > 0 ? 1 : (int)((pitch + 256 * waves - 1) / (256 * waves));
    for (int s = 0; s < steps; s++) {
        const int first = (s * waves + wave) * 256 + 4 * lane;
#pragma unroll
        for (int i = 0; i < N; i++) f8::load4(x, first + i * waves * 256, cols, vec, v[i]);
        if (r) {
#pragma unroll
            for (int i = 0; i < N; i++) f8::load4(r, first + i * waves * 256, cols, vec, t[i]);
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) v[i][j] = v[i][j] + t[i][j];
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int col = first + i * waves * 256;
#pragma unroll
            for (int j = 0; j < 4; j++) sum += (double)v[i][j] * (double)v[i][j];
            if (h) {
                if (vec) {
                    if (col < cols) *(float4 *)(h + col) = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (col + j < cols) h[col + j] = v[i][j];
                }
            }
        }
    }
    // gamma is under way while the sum is made
    float g[N][4];
    if (NI > 0)
#pragma unroll
        for (int i = 0; i < N; i++) f8::load4(gamma, (i * waves + wave) * 256 + 4 * lane, cols, vec, g[i]);
    sum = f8::wave_sum(sum);
    if (waves > 1) {
        if (lane == 0) s_sum[wave] = sum;
        __syncthreads();
        sum = 0.0;
        for (int i = 0; i < waves; i++) sum += s_sum[i];
    }
    // its power of two apart: 1 / sqrt of a row of subnormal values passes f32's range
    const double root = 1.0 / sqrt(sum / (double)cols + (double)eps);
    const float inv = (float)__builtin_amdgcn_frexp_mant(root);
    const int inv_exp = __builtin_amdgcn_frexp_exp(root);
    for (int s = 0; s < steps; s++) {
        const int first = (s * waves + wave) * 256 + 4 * lane;
        if (NI == 0) {
            if (h) {
                f8::load4(h, first, cols, vec, v[0]);
            } else {
                f8::load4(x, first, cols, vec, v[0]);
                if (r) {
                    f8::load4(r, first, cols, vec, t[0]);
#pragma unroll
                    for (int j = 0; j < 4; j++) v[0][j] = v[0][j] + t[0][j];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int col = first + i * waves * 256;
            float m = 0.0f;
            if (NI == 0) f8::load4(gamma, col, cols, vec, g[i]);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[i][j] = col + j < cols ? __builtin_amdgcn_ldexpf(v[i][j], inv_exp) * inv * g[i][j] : 0.0f;
                m = fmaxf(m, f8::finite_magnitude(v[i][j]));
            }
            const uint32_t byte = f8::scale_byte(f8::half_wave_max(m));
            if (col < (int64_t)pitch) {
                *(uint32_t *)(codes + row * pitch + col) = f8::codes4(v[i], f8::inverse_scale(byte));
                if (lane % 32 == 0) scales[row * spitch + col / 128] = (uint8_t)byte;
            }
        }
    }
    if (wave == 0 && lane < 3 && kb + lane < spitch) scales[row * spitch + kb + lane] = 127;
}

template <typename T>
void norm_kernel(sm_ctx *ctx, const T *X, const float *R, const float *gamma, float eps, uint32_t rows, int cols, float *H,
                 uint8_t *codes, uint8_t *scales) {
    const F8Layout L = f8_layout(rows, cols, 1);
    const uint32_t kb = (uint32_t)(L.pitch / 128);
    const bool vec = cols % 4 == 0;
    const int groups = (int)((L.pitch + 255) / 256);  // of 256 columns, one wave's step
    int waves = 1;
    while (waves < 16 && groups > 3 * waves) waves *= 2;
    const int ni = (groups + waves - 1) / waves;
#define SM_NORM(NI)                                                                                                      \
    k_f8_norm<T, NI><<<rows, 64 * waves, 0, ctx->stream>>>(X, R, gamma, eps, H, codes, scales, cols, kb, L.pitch,        \
                                                           (uint32_t)L.spitch, vec)
    if (ni <= 1) SM_NORM(1);
    else if (ni <= 2) SM_NORM(2);
    else if (ni <= 3) SM_NORM(3);
    else if (ni <= 6) SM_NORM(6);
    else SM_NORM(0);
#undef SM_NORM
}

}  // namespace

namespace smi {

int f8_quantize_launch(sm_ctx *ctx, const void *X, bool bf16, int rows, int cols, int block_rows, uint8_t *codes,
                       uint8_t *scales) {
    const F8Layout L = f8_layout(rows, cols, block_rows);
    const uint32_t kb = (uint32_t)(L.pitch / 128);
    const bool vec = cols % 4 == 0;
    if (block_rows == 1) {
        const uint32_t blocks = (uint32_t)rows * kb, grid = (blocks + 7) / 8;
        if (bf16)
            k_f8_rows<<<grid, 256, 0, ctx->stream>>>((const uint16_t *)X, codes, scales, blocks, cols, kb, L.pitch,
                                                     (uint32_t)L.spitch, vec);
        else
            k_f8_rows<<<grid, 256, 0, ctx->stream>>>((const float *)X, codes, scales, blocks, cols, kb, L.pitch,
                                                     (uint32_t)L.spitch, vec);
    } else {
        const uint32_t grid = (uint32_t)((rows + 127) / 128) * kb;
        if (bf16)
            k_f8_blocks<<<grid, 256, 0, ctx->stream>>>((const uint16_t *)X, codes, scales, rows, cols, kb, L.pitch,
                                                       (uint32_t)L.spitch, vec);
        else
            k_f8_blocks<<<grid, 256, 0, ctx->stream>>>((const float *)X, codes, scales, rows, cols, kb, L.pitch,
                                                       (uint32_t)L.spitch, vec);
    }
    return launched(ctx);
}

int f8_norm_launch(sm_ctx *ctx, const void *X, bool bf16, const float *R, const float *gamma, float eps, int rows, int cols,
                   float *H, uint8_t *codes, uint8_t *scales) {
    if (bf16) norm_kernel(ctx, (const uint16_t *)X, R, gamma, eps, (uint32_t)rows, cols, H, codes, scales);
    else norm_kernel(ctx, (const float *)X, R, gamma, eps, (uint32_t)rows, cols, H, codes, scales);
    return launched(ctx);
}

}  // namespace smi
