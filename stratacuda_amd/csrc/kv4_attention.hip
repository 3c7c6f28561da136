// Attention over a key-value cache held in 4 bits.
//
// For a query q of the sequence's position p and the positions t in
// (p - window, p]: s_t = scale q . k_t, y = sum_t e^(s_t - m) v_t / sum_t
// e^(s_t - m), one pass with the running maximum m; y * sigmoid(gate) where
// there is a gate. A row with no position gives 0.
//
// What a code and its scale stand for has two significant bits, so it is exact
// in bf16: keys and values go to the bf16 matrix units without a rounding.
// Queries of bf16 do too; those of f32 and their probabilities are taken as
// the sum of three bf16 numbers (8 significant bits each, so all 24) and cost
// three matrix instructions. For bf16 the probabilities are rounded to bf16,
// half a step of 2^-8 relative, like the result; sums are f32's.
#include <type_traits>

#include "kv4_device.h"
#include "kv4_shapes.h"
#include "strata_device.h"

namespace {
using namespace smi;
using kv4::bf16x2;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using i32x8 = __attribute__((ext_vector_type(8))) int;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

constexpr float kNone = -INFINITY;

__device__ __forceinline__ bf16x8 as_bf16(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }
__device__ __forceinline__ uint32_t bits(bf16x2 v) { return __builtin_bit_cast(uint32_t, v); }

// Three bf16 numbers whose sum is v: each the rounding of what is left, which
// the subtraction gives exactly.
__device__ __forceinline__ void three_parts(float a, float b, uint32_t part[3]) {
    part[0] = kv4::bf16_pair(a, b);
    const float a1 = a - __uint_as_float(part[0] << 16), b1 = b - __uint_as_float(part[0] & 0xffff0000u);
    part[1] = kv4::bf16_pair(a1, b1);
    part[2] = kv4::bf16_pair(a1 - __uint_as_float(part[1] << 16), b1 - __uint_as_float(part[1] & 0xffff0000u));
}

__device__ __forceinline__ float gated(float y, float g) { return y / (1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * g)); }

// v, of which nothing is known: what a loop makes of it is made in each turn instead of being held in registers.
__device__ __forceinline__ uint32_t here(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}

// Exponents past 2^30. A row's maximum is a rounded product there, off by 2^6 and more from its own scores' exact ones: the
// difference could leave f32 where there is none. So these rows take their scores times the power of two at or above the
// scale: exact, and numbers that differ do so by 2^6 at least, in powers of two, of which nothing is left in f32. A score of
// the maximum counts 1, any other 0.
constexpr float kFar = 0x1p30f;
__device__ __forceinline__ float far_scale(float scale_log2) {
    return __uint_as_float((__float_as_uint(scale_log2) + 0x7fffffu) & 0x7f800000u);
}
// Whether one of the exponents is far, or -infinity: no score.
__device__ __forceinline__ bool special(float a, float b) { return fmaxf(fabsf(a), fabsf(b)) >= kFar; }
// The score of a row with such a maximum m: what e to the power of it is, 1 or 0; NaN stays.
__device__ __forceinline__ float far_score(float s, float scale, float m) {
    const float d = m == kNone ? s : fmaf(s, scale, -m);
    return d < 0.0f ? kNone : d;
}

// The larger of a lane's value and those of the lanes 16, 32 and 48 away.
__device__ __forceinline__ float max_of_quarters(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_of_quarters(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ float max_of_halves(float v) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_of_halves(float v) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// ---------------------------------------------------------------- the shares
// A workgroup takes a tile of a sequence's rows for one key-value head and a
// piece of its pages. Where no sequence is cut, the tiles of all sequences lie
// in blockIdx.x one after another: a batch of one long prompt and many single
// tokens has no more workgroups than it has tiles. Else blockIdx.y is the piece
// of all sequences', of equally many pages; a sequence with rows has one at
// least. Small pieces are whole turns of a workgroup's kTurn pages: 2
// sequences of 8192 positions, 32 heads on 8 of dimension 128, take 13.5 us in
// pieces of 8 pages and 14.8 in pieces of 6. Larger ones are as equal as they
// can be (32 such sequences 42.3 and 42.9).
struct Piece {
    int s, first, end;  // the sequence and the pages; s = -1: there is no such piece
    int number, count;  // which of the sequence's pieces it is
    int tile;           // of the sequence's rows
    kv4::Span span;
    int at;             // where the piece's results go: the place of its first tile's first head
};
// The pages that the sequence's rows reach.
__device__ __forceinline__ int2 pages_of(const kv4::Span &a, int window) {
    const int first = a.length - a.n;
    const int lo = window > 0 ? max(first - window + 1, 0) / 64 : 0;
    return make_int2(lo, max((a.length + 63) / 64, lo));
}
__device__ __forceinline__ int pieces_in(const int2 &p, int n, int each) { return n > 0 ? max((p.y - p.x + each - 1) / each, 1) : 0; }
template <int kTileRows, int kTurn>
__device__ Piece piece_of(const Kv4Attention &a) {
    const Kv4Sequences &q = a.q;
    const int lane = threadIdx.x % 64, at_x = blockIdx.x / a.kv_heads, group = a.heads / a.kv_heads;
    const auto sequence = [&](int s) { return s < q.count ? kv4::span(q, s) : kv4::Span{0, 0, 0}; };
    const kv4::Span a0 = sequence(lane);
    const bool whole = a.pieces == 1;
    const int slot = whole ? at_x : blockIdx.y;
    int each = 0;
    if (!whole) {
        int total = 0;
        for (int at = 0; at < q.count; at += 64) {
            const kv4::Span b = at == 0 ? a0 : sequence(at + lane);
            const int2 p = pages_of(b, a.window);
            int some = b.n > 0 ? p.y - p.x : 0;
            if (q.count > 1)
#pragma unroll
                for (int i = 1; i < 64; i *= 2) some += __shfl_xor(some, i, 64);
            total += __builtin_amdgcn_readfirstlane(some);
        }
        each = max(a.least, (total + a.pieces - 1) / a.pieces);
        if (each < 4 * kTurn) each = (each + kTurn - 1) / kTurn * kTurn;
    }
    int before = 0;
    for (int at = 0; at < q.count; at += 64) {
        const kv4::Span b = at == 0 ? a0 : sequence(at + lane);
        const int2 p = pages_of(b, a.window);
        const int mine = whole ? (b.n * group + kTileRows - 1) / kTileRows : pieces_in(p, b.n, each);
        int upto = mine;  // with this lane's
        if (q.count > 1)
#pragma unroll
            for (int i = 1; i < 64; i *= 2) {
                const int other = __shfl_up(upto, i, 64);
                if (lane >= i) upto += other;
            }
        const uint64_t past = __ballot(before + upto > slot && mine > 0);
        if (past) {
            const int who = __ffsll((unsigned long long)past) - 1;
            // the same in all lanes: kept, and what it leads to, in scalar registers
            const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, who); };
            const int count = of(mine), number = slot - before - (of(upto) - count), first = of(p.x), end = of(p.y);
            const kv4::Span span = {of(b.row), of(b.n), of(b.length)};
            if (whole) return {at + who, first, end, 0, 1, number, span, 0};
            return {at + who, first + number * each, min(first + (number + 1) * each, end), number, count, at_x, span, (int)(blockIdx.y * gridDim.x)};
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return {-1, 0, 0, 0, 0, 0, {0, 0, 0}, 0};
}
// The same where rows differ and contexts are long: tiles and pieces of all sequences in blockIdx.x, a sequence's pieces one
// after another, in each all its tiles. Pieces are of equally many pages, so many that all tiles' pages make a.budget pieces
// and each tile's last one a part of one more. Where starts that go back make more tiles than the launch was sized for, no
// sequence is cut, and nothing is left in the workspace. Block 0 says where each sequence's pieces begin.
template <int kTileRows>
__device__ Piece piece_by_rows(const Kv4Attention &a) {
    const Kv4Sequences &q = a.q;
    const int lane = threadIdx.x % 64, slot = blockIdx.x / a.kv_heads, group = a.heads / a.kv_heads;
    const auto sequence = [&](int s) { return s < q.count ? kv4::span(q, s) : kv4::Span{0, 0, 0}; };
    const auto tiles_of = [&](const kv4::Span &b) { return (b.n * group + kTileRows - 1) / kTileRows; };
    int64_t pages = 0;
    int tiles = 0;
    for (int at = 0; at < q.count; at += 64) {
        const kv4::Span b = sequence(at + lane);
        const int2 p = pages_of(b, a.window);
        pages += (int64_t)tiles_of(b) * (p.y - p.x), tiles += tiles_of(b);
    }
#pragma unroll
    for (int i = 1; i < 64; i *= 2) pages += __shfl_xor(pages, i, 64), tiles += __shfl_xor(tiles, i, 64);
    int each = kv4::kMostPages;
    if (tiles <= a.units) each = (int)min(max((pages + a.budget - 1) / a.budget, (int64_t)a.least), (int64_t)kv4::kMostPages);
    each = __builtin_amdgcn_readfirstlane(each);
    Piece found = {-1, 0, 0, 0, 0, 0, {0, 0, 0}, 0};
    for (int at = 0, before = 0; at < q.count; at += 64) {
        const kv4::Span b = sequence(at + lane);
        const int2 p = pages_of(b, a.window);
        const int many = pieces_in(p, b.n, each), mine = many * tiles_of(b);
        int upto = mine;
#pragma unroll
        for (int i = 1; i < 64; i *= 2) {
            const int other = __shfl_up(upto, i, 64);
            if (lane >= i) upto += other;
        }
        if (blockIdx.x == 0 && threadIdx.x < 64 && at + lane < q.count) a.info[at + lane] = make_int2(before + upto - mine, many);
        const uint64_t past = __ballot(before + upto > slot && mine > 0);
        if (past && found.s < 0) {
            const int who = __ffsll((unsigned long long)past) - 1;
            const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, who); };
            const kv4::Span span = {of(b.row), of(b.n), of(b.length)};
            const int step = tiles_of(span), local = slot - before - (of(upto) - of(mine)), number = local / step, first = of(p.x);
            found = {at + who, first + number * each, min(first + (number + 1) * each, of(p.y)), number, of(many), local - number * step,
                     span, (slot - (local - number * step)) * a.kv_heads};
            if (blockIdx.x > 0) break;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return found;
}

// Either by the kernel's type: the second beside the first would cost one token over 2048 positions 0.5 us of 16.7.
template <int kTileRows, int kTurn, bool kByRows>
__device__ __forceinline__ Piece share(const Kv4Attention &a) {
    if constexpr (kByRows) return piece_by_rows<kTileRows>(a);
    else return piece_of<kTileRows, kTurn>(a);
}

// ------------------------------------------------------------------ 16 rows
// One workgroup: 16 rows (a token's heads of one key-value head, then the next
// token's) over one piece of the sequence, whose pages its four waves take in
// turn. Both products are transposed, S^T = K Q^T and O^T = V^T P^T: a lane
// holds one row's scores of 4 positions out of 16, which is what it brings to
// the second product, and every row's maximum and sum lie in its own lanes.
// Codes go from memory into registers: 16 bytes a lane are 32 dimensions of
// one key (its block: one scale), or two dimensions of 16 positions' values.
// The next page's keys are on their way while this one's probabilities are
// made, its values during the products.
//
// Long contexts are bound by memory (24 heads on 2 of dimension 256, bf16, one
// token over 131072 positions: 71 MB in 20 us and 6.7 to join them; 32
// sequences of 32 heads on 8 of 128: 161 MB in 37 us, 4.4 TB/s, and 4.2), short
// ones by what follows one another: the sequences' numbers, page numbers, keys,
// values (2048 positions, f32: 12 us and 4.3).
template <int NC, bool F32>
struct Rows16 {
    static constexpr int kPitch = 64 * NC, kBlocks = 2 * NC;
    static constexpr bool kWide = NC % 2 == 0;            // 16 bytes of a key a load; else 8
    static constexpr int kChunks = kWide ? NC / 2 : NC;   // loads of a key
    static constexpr int kSteps = kWide ? 4 : 2;          // matrix steps of 32 dimensions of each
    static constexpr int kParts = F32 ? 3 : 1;
    static constexpr int kWavesOfSimd = F32 && NC > 2 ? 1 : 2;  // at least: what their registers leave

    struct Keys {
        uint32_t codes[4][kChunks][kSteps];  // of positions 16 g + lane % 16
        uint32_t scales[kChunks];            // a byte for each g
    };
    struct Values {
        u32x4 codes[kBlocks], scales[kBlocks];
    };
    static __device__ __forceinline__ void load(Keys &k, const uint8_t *tile, int lane) {
        const int n = lane % 16, kq = lane / 16;
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
            const int block = kWide ? 4 * c + kq : 2 * c + kq / 2;
            k.scales[c] = *(const uint32_t *)(tile + kv4::key_scales(kPitch) + block * 64 + n * 4);
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const uint8_t *p = tile + (16 * g + n) * (kPitch / 2) + (4 * kSteps) * (4 * c + kq);
                if constexpr (kWide) {
                    const u32x4 v = *(const u32x4 *)p;
                    k.codes[g][c][0] = v[0], k.codes[g][c][1] = v[1], k.codes[g][c][2] = v[2], k.codes[g][c][3] = v[3];
                } else {
                    const uint2 v = *(const uint2 *)p;
                    k.codes[g][c][0] = v.x, k.codes[g][c][1] = v.y;
                }
            }
        }
    }
    static __device__ __forceinline__ void load(Values &v, const uint8_t *tile, int lane) {
#pragma unroll
        for (int b = 0; b < kBlocks; b++) {
            v.codes[b] = *(const u32x4 *)(tile + kv4::value_codes(kPitch) + b * 1024 + lane * 16);
            v.scales[b] = *(const u32x4 *)(tile + kv4::value_scales(kPitch) + b * 64 + lane / 16 * 16);
        }
    }
    // The query's part of step (c, s): dimensions as the keys' loads have them.
    static __device__ __forceinline__ int dimension(int c, int s, int kq) { return 8 * kSteps * (4 * c + kq) + 8 * s; }
};

// The byte i of w as a scale operand: the conversions take the exponent field
// alone, so what else the word brings along does not count.
__device__ __forceinline__ float scale_at(uint32_t w, int i) {
    return __uint_as_float(i == 0 ? w << 23 : i == 1 ? w << 15 : i == 2 ? w << 7 : w >> 1);
}
// Eight codes, of dimension 2 j and 2 j + 1 in byte j, as bf16.
__device__ __forceinline__ u32x4 eight(uint32_t w, float scale) {
    return u32x4{bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)), bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                 bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)), bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
}
// Four positions of two dimensions (a byte each, with its scale) as two
// registers of the lower dimension and two of the upper one.
__device__ __forceinline__ void four(uint32_t w, uint32_t scales, uint32_t low[2], uint32_t high[2]) {
    const uint32_t a = bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale_at(scales, 0), 0));
    const uint32_t b = bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale_at(scales, 1), 1));
    const uint32_t c = bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale_at(scales, 2), 2));
    const uint32_t d = bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale_at(scales, 3), 3));
    low[0] = __builtin_amdgcn_perm(b, a, 0x05040100u), low[1] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    high[0] = __builtin_amdgcn_perm(b, a, 0x07060302u), high[1] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

template <int NC, typename T, bool kByRows>
__global__ void __launch_bounds__(256, (Rows16<NC, sizeof(T) == 4>::kWavesOfSimd)) k_kv4_rows(Kv4Attention a, const T *Q, const uint8_t *pool,
                                                                                            const T *G, T *Y, float *parts, float2 *stats) {
    constexpr bool F32 = sizeof(T) == 4;
    using R = Rows16<NC, F32>;
    constexpr int kPitch = R::kPitch, kTiles = kPitch / 16, kLine = kPitch + 4;
    const uint32_t lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const Piece piece = share<16, 4, kByRows>(a);
    if (piece.s < 0) return;
    if (a.info && piece.number == 0 && blockIdx.x == 0 && threadIdx.x == 0) a.info[piece.s] = make_int2(blockIdx.y, piece.count);
    const kv4::Span span = piece.span;
    const int head = blockIdx.x % a.kv_heads, tile = piece.tile, group = a.heads / a.kv_heads;
    const int rows = span.n * group - 16 * tile;  // of the sequence, from this tile's first on
    if (rows <= 0) return;
    const int first = span.length - span.n;       // the first new token's position

    // the tile's rows: the first and last one's position, the lowest position of any, of all
    const int last = first + (16 * tile + min(15, rows - 1)) / group, early = first + 16 * tile / group;
    const int any_lo = a.window > 0 ? max(early - a.window + 1, 0) : 0, all_lo = a.window > 0 ? max(last - a.window + 1, 0) : 0;
    const int begin = max(piece.first, any_lo / 64), end = min(piece.end, (last >> 6) + 1);
    // this wave's pages: begin + wave + 4 i; their numbers, a lane's each, of 64
    const int mine = (end - begin - wave + 3) / 4, start = begin + wave;
    int ids = -1;
    const auto id_of = [&](int i) {
        if (i % 64 == 0) {
            const int at = start + 4 * (i + (int)lane);
            ids = at < end ? kv4::page_of(a.q, piece.s, at, a.pages) : -1;
        }
        return __builtin_amdgcn_readlane(ids, i % 64);
    };
    int page = mine > 0 ? id_of(0) : -1;

    // this lane's row, the last one's once more past it; its positions lo .. hi
    const int row = 16 * tile + min((int)(lane % 16), rows - 1), token = row / group, hq = head * group + row % group;
    const int hi = first + token, lo = a.window > 0 ? max(hi - a.window + 1, 0) : 0;
    uint32_t q[R::kParts][R::kChunks][R::kSteps][4];
    {
        const T *x = Q + (int64_t)(span.row + token) * a.q_view.stride + hq * a.q_view.head + a.q_view.offset;
#pragma unroll
        for (int c = 0; c < R::kChunks; c++)
#pragma unroll
            for (int s = 0; s < R::kSteps; s++) {
                const int d = R::dimension(c, s, lane / 16);
                float v[8] = {};
                if (d < a.dim) kv4::load8(x + d, a.vec, v);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if constexpr (F32) {
                        uint32_t part[3];
                        three_parts(v[2 * j], v[2 * j + 1], part);
#pragma unroll
                        for (int t = 0; t < 3; t++) q[t][c][s][j] = part[t];
                    } else {
                        q[0][c][s][j] = kv4::bf16_pair(v[2 * j], v[2 * j + 1]);
                    }
                }
            }
    }

    f32x4 o[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; t++) o[t] = f32x4{0, 0, 0, 0};
    float m = kNone, sum = 0.0f;  // the row's maximum (times scale_log2); this lane's share of its sum

    typename R::Keys keys;
    typename R::Values values;
    const int64_t step = (int64_t)a.kv_heads * (68 * kPitch);
    const uint8_t *base = pool + (int64_t)head * (68 * kPitch);
    const auto tile_of = [&](int id) { return base + max(id, 0) * step; };
    // page i of the wave; `whole`: every row has all its positions, and another page follows
    const auto turn = [&](int i, auto whole) {
        // S^T: positions 16 g + 4 kq + i of row lane % 16
        f32x4 s[4];
#pragma unroll
        for (int g = 0; g < 4; g++) {
            s[g] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < R::kChunks; c++) {
                const float scale = scale_at(keys.scales[c], g);
#pragma unroll
                for (int t = 0; t < R::kSteps; t++) {
                    const bf16x8 k = as_bf16(eight(keys.codes[g][c][t], scale));
#pragma unroll
                    for (int p = R::kParts - 1; p >= 0; p--)
                        s[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            k, as_bf16(u32x4{q[p][c][t][0], q[p][c][t][1], q[p][c][t][2], q[p][c][t][3]}), s[g], 0, 0, 0);
                }
            }
        }
        const int now = page, p0 = 64 * (start + 4 * i);
        const bool more = whole || i + 1 < mine;
        if (more) {
            page = id_of(i + 1);
            R::load(keys, tile_of(page), here(lane));
        }
        const bool edge = !whole && (now < 0 || p0 < all_lo || p0 + 63 > early);  // a position that some row does not have
        bool poisoned = false;
        if (edge) {
            const int kq = here(lane) / 16;
#pragma unroll
            for (int g = 0; g < 4; g++) {
                uint32_t kept = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int t = p0 + 16 * g + 4 * kq + i;
                    if (now < 0 || t < lo || t > hi) s[g][i] = kNone;
                    if (now >= 0 && t >= any_lo && t <= last) kept |= 255u << (8 * i);
                }
                // values that no row has may be anything: their scales count as 1, and 0 times their codes is 0
#pragma unroll
                for (int b = 0; b < R::kBlocks; b++) values.scales[b][g] = (values.scales[b][g] & kept) | (0x7f7f7f7fu & ~kept);
            }
            // a block of NaN that some rows have and others do not
#pragma unroll
            for (int b = 0; b < R::kBlocks; b++)
#pragma unroll
                for (int g = 0; g < 4; g++)
#pragma unroll
                    for (int i = 0; i < 4; i++) poisoned |= (values.scales[b][g] >> (8 * i) & 255u) == 255u;
            poisoned = __any(poisoned);
        }
        float top = kNone;
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int i = 0; i < 4; i++) top = fmaxf(top, s[g][i]);
        const float best = max_of_quarters(top);
        top = best * a.scale_log2;
        float from = m;
        // the maximum is raised once scores pass it by 2^8: any number near it does
        if (__any(top > m + 8.0f || special(top, m))) {
            if (fabsf(top) >= kFar) top = best * far_scale(a.scale_log2);
            const float to = __any(top > m + 8.0f) ? fmaxf(m, top) : m, by = m == kNone ? 0.0f : __builtin_amdgcn_exp2f(m - to);
            m = from = to;
            sum *= by;
#pragma unroll
            for (int t = 0; t < kTiles; t++) o[t] *= by;
            if (special(m, 0.0f)) {
                from = 0.0f;
#pragma unroll
                for (int g = 0; g < 4; g++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[g][i] = far_score(s[g][i], far_scale(a.scale_log2), m);
            }
        }
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[g][i] = __builtin_amdgcn_exp2f(fmaf(s[g][i], a.scale_log2, -from));
                sum += s[g][i];
            }
        uint32_t poison = 0;  // bit b: a block b of NaN at a position that the row has
        if (poisoned) {
            const int kq = here(lane) / 16;
#pragma unroll
            for (int b = 0; b < R::kBlocks; b++)
#pragma unroll
                for (int g = 0; g < 4; g++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int t = p0 + 16 * g + 4 * kq + i;
                        if ((values.scales[b][g] >> (8 * i) & 255u) != 255u) continue;
                        values.scales[b][g] ^= 0x80u << (8 * i);
                        // the scales are those of this quarter's positions, the same in its 16 lanes: each its own row
                        if (t >= lo && t <= hi) poison |= 1u << b;
                    }
            poison |= __shfl_xor(poison, 16, 64);
            poison |= __shfl_xor(poison, 32, 64);
        }
        // O^T: dimensions 16 t + 4 kq + i of row lane % 16
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            u32x4 p[R::kParts];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float x = s[2 * ks + j / 2][2 * (j % 2)], y = s[2 * ks + j / 2][2 * (j % 2) + 1];
                if constexpr (F32) {
                    uint32_t part[3];
                    three_parts(x, y, part);
#pragma unroll
                    for (int t = 0; t < 3; t++) p[t][j] = part[t];
                } else {
                    p[0][j] = kv4::bf16_pair(x, y);
                }
            }
#pragma unroll
            for (int b = 0; b < R::kBlocks; b++) {
                uint32_t low[4], high[4];
                four(values.codes[b][2 * ks], values.scales[b][2 * ks], low, high);
                four(values.codes[b][2 * ks + 1], values.scales[b][2 * ks + 1], low + 2, high + 2);
                const bf16x8 vl = as_bf16(u32x4{low[0], low[1], low[2], low[3]}),
                             vh = as_bf16(u32x4{high[0], high[1], high[2], high[3]});
#pragma unroll
                for (int t = R::kParts - 1; t >= 0; t--) {
                    o[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vl, as_bf16(p[t]), o[2 * b], 0, 0, 0);
                    o[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vh, as_bf16(p[t]), o[2 * b + 1], 0, 0, 0);
                }
            }
        }
        if (!whole && poison) {
#pragma unroll
            for (int b = 0; b < R::kBlocks; b++)
                if (poison >> b & 1) o[2 * b] = o[2 * b + 1] = f32x4{NAN, NAN, NAN, NAN};
        }
        if (more) R::load(values, tile_of(page), here(lane));
    };
    if (mine > 0) {
        R::load(keys, tile_of(page), lane);
        R::load(values, tile_of(page), lane);
    }
    // the wave's pages that are whole: from the first at or past all_lo to the last that ends at or before `early`, and not its last
    const int whole_from = max((all_lo + 63) / 64 - start + 3, 0) / 4, whole_to = min(((early + 1) / 64 - start + 3) / 4, mine - 1);
    int i = 0, from = whole_from < whole_to ? whole_from : mine;
    while (i < mine) {
        for (; i < from; i++) turn(i, std::false_type());
        from = mine;
        for (; i < whole_to && page >= 0; i++) turn(i, std::true_type());
    }

    // the four waves' sums meet
    __shared__ float s_o[4][16][kLine], s_m[4][16], s_sum[4][16];
    sum = sum_of_quarters(sum);
#pragma unroll
    for (int t = 0; t < kTiles; t++) *(f32x4 *)&s_o[wave][lane % 16][16 * t + lane / 16 * 4] = o[t];
    if (lane < 16) s_m[wave][lane] = m, s_sum[wave][lane] = sum;
    __syncthreads();
    const int r = threadIdx.x / 16, d0 = threadIdx.x % 16 * 4;
    if (r >= rows) return;
    float by[4], top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r])), all = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        by[w] = s_m[w][r] == kNone ? 0.0f : __builtin_amdgcn_exp2f(s_m[w][r] - top);
        // a sum that is not a number, of scores that are none, stays one
        all += s_m[w][r] == kNone ? (s_sum[w][r] == 0.0f ? 0.0f : NAN) : s_sum[w][r] * by[w];
    }
    const int64_t part = (int64_t)(piece.at + tile * a.kv_heads + head) * 16 + r;
    const int tok = (16 * tile + r) / group, h = head * group + (16 * tile + r) % group;
    const int64_t out = ((int64_t)(span.row + tok) * a.heads + h) * a.dim;
    const T *g = G ? G + (int64_t)(span.row + tok) * a.g_view.stride + h * a.g_view.head + a.g_view.offset : nullptr;
#pragma unroll
    for (int d = d0; d < kPitch; d += 64) {
        f32x4 v = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; w++) v += *(f32x4 *)&s_o[w][r][d] * by[w];
        if (piece.count > 1) {
            *(f32x4 *)(parts + part * kPitch + d) = v;
        } else {
            const float inv = all == 0.0f ? 0.0f : 1.0f / all;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (d + i < a.dim) {
                    float y = all == 0.0f ? 0.0f : v[i] * inv;
                    if (g) y = gated(y, kv4::value(g[d + i]));
                    kv4::store1(Y + out + d + i, y);
                }
        }
    }
    if (piece.count > 1 && d0 == 0) stats[part] = make_float2(top, all);
}

// ------------------------------------------------------------------ prompts
// One workgroup: 32 rows a wave, all of one key-value head, over one piece of
// the sequence, in units of 32 or 64 positions. The products are transposed as
// above, on 32 x 32 tiles: a lane holds one row's scores of half of a unit's
// positions, and brings them to the second product as they are.
//
// A wave alternates between the matrix unit (a unit's scores, the unit
// before's values) and vector instructions (its softmax, its share of the
// units that are staged next); of the two waves of a SIMD one is half a turn
// ahead, so that both are busy. Turns end at barriers. Keys are staged in LDS
// as codes, values as bf16, converted once; both twice, the next unit's on
// their way in registers.
//
// Scores of bf16 queries: codes go into the matrix unit as they are, with
// their scales. The query is the sum of two e4m3 numbers of 4 significant bits
// each, with one power of two for the row: all 8 bits of a bf16 number from
// 2^-13 of the row's largest up, 2^-22 of that largest otherwise. That unit
// cuts products 2^13 below the largest of eight neighbours: at most 7 * 2^-13
// of a score's products' magnitudes are lost, 1e-5 for ordinary ones, where
// probabilities are rounded by 2^-8. Queries of f32 take bf16's unit.
//
// From some thousand tokens on bound by the matrix units and by what their clock allows: 8192 tokens, 32 heads on 8 of
// dimension 128, bf16, 481 to 521 us, 1.06 to 1.14 PFLOP/s (520 to 585 where calls follow without a pause); 512 tokens
// behind 32256 positions, 24 heads on 2 of 256, 348 to 376 us, 1.09 to 1.18 (a library's product of 16384^3 reaches 1.35).
// Fewer are not: each workgroup takes 14 us to begin and end, and those of a prompt's first rows end long before the last.
template <int NC, typename T>
struct Prompt {
    static constexpr bool kF32 = sizeof(T) == 4;
    static constexpr int kPitch = 64 * NC, kBlocks = 2 * NC, kParts = kF32 ? 3 : 1;
    // f32 queries of more than 128 dimensions would take, in this shape, more registers than two waves of a SIMD have: sixteen
    // rows a workgroup then
    static constexpr bool kThere = !kF32 || NC < 3;
    static constexpr int kWaves = 8, kThreads = 64 * kWaves, kRows = 32 * kWaves;
    static_assert(kRows == kKv4PromptRows, "the shapes count on it");
    static constexpr int kHalves = NC > 2 || (kF32 && NC > 1) ? 1 : 2;  // of a page in a unit: what registers hold
    static constexpr int kUnit = 32 * kHalves, kTurns = 64 / kUnit;
    static constexpr int kPieces = 2 * NC;  // of 16 bytes, of a key's codes
    static constexpr bool kScoresFirst = NC < 3;
    // words of codes that are staged in a turn, and a thread's
    static constexpr int kKeyWords = kUnit * 4 * kPieces, kKeys = (kKeyWords + kThreads - 1) / kThreads;
    static constexpr int kValueWords = kBlocks * 128 * kHalves, kValues = (kValueWords + kThreads - 1) / kThreads;
    // Where piece `p` of position t lies: any eight neighbouring positions' same piece in other banks.
    static __device__ __forceinline__ int slot(int t, int p) {
        const int turned = NC == 1 ? p ^ (t >> 2 & 1) : NC == 2 ? p ^ (t >> 1 & 3) : NC == 4 ? p ^ (t & 7) : (p + (t >> 2 & 1)) % kPieces;
        return (t * kPieces + turned) * 16;
    }
};

template <int NC, typename T, bool kByRows>
__global__ void __launch_bounds__((Prompt<NC, T>::kThreads)) k_kv4_prompt(Kv4Attention a, const T *Q, const uint8_t *pool, const T *G,
                                                                          T *Y, float *parts, float2 *stats, int tiles) {
    using R = Prompt<NC, T>;
    constexpr int kPitch = R::kPitch, kBlocks = R::kBlocks, kUnit = R::kUnit, kHalves = R::kHalves, kTurns = R::kTurns;
    constexpr int kGroups = kUnit / 16;  // of 16 positions
    __shared__ __attribute__((aligned(16))) uint8_t s_keys[2][kUnit * R::kPieces * 16];
    __shared__ __attribute__((aligned(16))) uint8_t s_values[2][kBlocks * kGroups * 1024];
    __shared__ uint32_t s_scales[2][kBlocks][16];  // of the keys: a byte for each 16 positions of the page
    __shared__ uint64_t s_nan[4][kBlocks];         // values that are NaN for some rows and not there for others
    const uint32_t lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const Piece piece = share<R::kRows, 1, kByRows>(a);
    if (piece.s < 0) return;
    if (a.info && piece.number == 0 && blockIdx.x == 0 && threadIdx.x == 0) a.info[piece.s] = make_int2(blockIdx.y, piece.count);
    const kv4::Span span = piece.span;
    const int head = blockIdx.x % a.kv_heads, group = a.heads / a.kv_heads;
    // a sequence's longest rows first
    const int tile = (a.pieces == 1 ? (span.n * group + R::kRows - 1) / R::kRows : tiles) - 1 - piece.tile;
    const int rows = span.n * group - R::kRows * tile;
    if (rows <= 0) return;
    const int first = span.length - span.n;
    const auto token_of = [&](int r) { return (R::kRows * tile + min(r, rows - 1)) / group; };

    const int row = R::kRows * tile + min(32 * wave + (int)(lane % 32), rows - 1), token = row / group, hq = head * group + row % group;
    const int hi = first + token, lo = a.window > 0 ? max(hi - a.window + 1, 0) : 0;
    const auto low = [&](int position) { return a.window > 0 ? max(position - a.window + 1, 0) : 0; };
    // the workgroup's rows and the wave's: the first and last one's position, the lowest position of any, of all
    const int last = first + token_of(R::kRows - 1), early = first + token_of(0), any_lo = low(early), all_lo = low(last);
    const int w_last = first + token_of(32 * wave + 31), w_early = first + token_of(32 * wave), w_any = low(w_early), w_all = low(w_last);
    const bool works = 32 * wave < rows;
    const int begin = max(piece.first, any_lo / 64), end = min(piece.end, (last >> 6) + 1), units = max(end - begin, 0) * kTurns;
    const auto position_of = [&](int u) { return 64 * begin + kUnit * u; };
    // page numbers, a lane's each, of 64 pages; asked for in order
    int ids = -1;
    bool holes = false;  // a page that is none was among them
    const auto id_of = [&](int u) {
        const int at = u / kTurns;
        if (at >= end - begin) return -1;
        if (u % (64 * kTurns) == 0) {
            ids = kv4::page_of(a.q, piece.s, min(begin + at + (int)lane, end - 1), a.pages);
            holes = holes || __any(ids < 0);
        }
        return __builtin_amdgcn_readlane(ids, at % 64);
    };
    const auto is_edge = [&](int p0, int id) { return id < 0 || p0 < all_lo || p0 + kUnit - 1 > early; };
    // units all of whose positions every row of the workgroup has
    const int whole_from = (max(all_lo - 64 * begin, 0) + kUnit - 1) / kUnit, whole_to = min(max(early + 1 - 64 * begin, 0) / kUnit, units);
    const auto is_live = [&](int p0) { return works && p0 <= w_last && p0 + kUnit - 1 >= w_any; };

    // queries: for f32 three bf16 numbers, dimensions 64 c + 32 kq + 8 s of step (c, s) a lane; else two e4m3 ones,
    // 64 c + 32 i + 16 kq of half i of step c
    uint32_t q[R::kParts][NC][16];
    int q_scale = 0;
    {
        const T *x = Q + (int64_t)(span.row + token) * a.q_view.stride + hq * a.q_view.head + a.q_view.offset;
        const int kq = lane / 32;
        if constexpr (R::kF32) {
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const int d = 64 * c + 32 * kq + 8 * s;
                    float v[8] = {};
                    if (d < a.dim) kv4::load8(x + d, a.vec, v);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        uint32_t part[3];
                        three_parts(v[2 * j], v[2 * j + 1], part);
#pragma unroll
                        for (int t = 0; t < 3; t++) q[t][c][4 * s + j] = part[t];
                    }
                }
        } else {
            float amax = 0.0f;
#pragma unroll
            for (int turn = 0; turn < 2; turn++) {  // the row's largest magnitude, then its parts
                float by = 0.0f;
                if (turn == 1) {
                    // at least 2^-123, so that the lower part's scale is one
                    const int byte = max((int)f8::scale_byte(max_of_halves(amax)), 4);
                    q_scale = byte | (byte - 4) << 8, by = f8::inverse_scale(byte);  // byte 0 for the higher part, 1 for the lower
                }
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int s = 0; s < 4; s++) {
                        const int d = 64 * c + 32 * (s / 2) + 16 * kq + 8 * (s % 2);
                        float v[8] = {};
                        if (d < a.dim) kv4::load8(x + d, a.vec, v);
                        if (turn == 0) {
#pragma unroll
                            for (int j = 0; j < 8; j++) amax = fmaxf(amax, f8::finite_magnitude(v[j]));
                            continue;
                        }
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const float *w = v + 4 * j;
                            const uint32_t high = f8::codes4((float4){w[0], w[1], w[2], w[3]}, by);
                            const kv4::f32x2 h0 = __builtin_amdgcn_cvt_pk_f32_fp8(high, false), h1 = __builtin_amdgcn_cvt_pk_f32_fp8(high, true);
                            const float4 rest = {w[0] * by - h0[0], w[1] * by - h0[1], w[2] * by - h1[0], w[3] * by - h1[1]};
                            q[0][c][2 * s + j] = high;
                            q[0][c][8 + 2 * s + j] = f8::codes4(rest, 16.0f);  // at most 16, half a step of 448
                        }
                    }
            }
        }
    }

    f32x16 o[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; b++) o[b] = f32x16{};
    float m = kNone, sum = 0.0f;

    // ------------------------------------------------------------- staging
    const int64_t step = (int64_t)a.kv_heads * (68 * kPitch);
    const uint8_t *base = pool + (int64_t)head * (68 * kPitch);
    uint32_t key[R::kKeys], key_scale = 0, value[R::kValues], scale[R::kValues];
    // word w of a unit's values: block, quarter of the positions, dimension, group of 16 positions
    struct Word {
        uint32_t b, k, r, g;
    };
    const auto word_of = [&](uint32_t w) { return Word{w / kGroups / 64, w / kGroups / 16 % 4, w / kGroups % 16, w % kGroups}; };
    const auto codes_of = [](const Word &w) { return kv4::value_codes(kPitch) + ((w.b * 4 + w.k) * 16 + w.r) * 16 + w.g * 4; };
    const auto scales_of = [](const Word &w) { return kv4::value_scales(kPitch) + (w.b * 4 + w.k) * 16 + w.g * 4; };
    constexpr int kRun = R::kValues % 2 == 0 ? 2 : 1;  // a thread's words that lie together
    // Every load is sent, also those that nothing follows (threads and units past the last take one that is there): so
    // the ones under way are known where others are waited for. Offsets in 32 bits, opened in each turn: beside a
    // scalar base they need no registers of their own.
    const bool has_keys = R::kKeyWords % R::kThreads == 0 || threadIdx.x * R::kKeys < R::kKeyWords;
    const bool has_values = R::kValueWords % R::kThreads == 0 || threadIdx.x * R::kValues < R::kValueWords;
    const uint32_t key_at = has_keys ? threadIdx.x * (4 * R::kKeys) : 0, key_scale_at = min(threadIdx.x, 16u * kBlocks - 1) * 4;
    const uint32_t value_word = has_values ? threadIdx.x * R::kValues : 0;
    uint32_t value_at[R::kValues / kRun], scale_at_[R::kValues / kRun];
#pragma unroll
    for (int j = 0; j < R::kValues; j += kRun)
        value_at[j / kRun] = codes_of(word_of(value_word + j)), scale_at_[j / kRun] = scales_of(word_of(value_word + j));
    const auto tile_of = [&](int id) { return base + max(id, 0) * step; };
    const auto fetch_keys = [&](int u, const uint8_t *t) {
        const uint8_t *from = t + u % kTurns * (4 * R::kKeyWords);
        const uint32_t at = here(key_at);
        if constexpr (R::kKeys == 4) {
            const u32x4 v = *(const u32x4 *)(from + at);
            key[0] = v[0], key[1] = v[1], key[2] = v[2], key[3] = v[3];
        } else if constexpr (R::kKeys == 2) {
            const uint2 v = *(const uint2 *)(from + at);
            key[0] = v.x, key[1] = v.y;
        } else {
#pragma unroll
            for (int j = 0; j < R::kKeys; j++) key[j] = *(const uint32_t *)(from + at + 4 * j);
        }
        key_scale = *(const uint32_t *)(t + kv4::key_scales(kPitch) + here(key_scale_at));
    };
    const auto fetch_values = [&](int u, const uint8_t *t) {
        t += u % kTurns * 8;
#pragma unroll
        for (int j = 0; j < R::kValues; j += kRun) {
            const uint8_t *v = t + here(value_at[j / kRun]), *f = t + here(scale_at_[j / kRun]);
            if constexpr (kRun == 2) {
                const uint2 x = *(const uint2 *)v, y = *(const uint2 *)f;
                value[j] = x.x, value[j + 1] = x.y, scale[j] = y.x, scale[j + 1] = y.y;
            } else {
                value[j] = *(const uint32_t *)v, scale[j] = *(const uint32_t *)f;
            }
        }
    };
    const auto stage_keys = [&](int u) {
        const uint32_t tid = threadIdx.x, word = tid * R::kKeys;
        const int buffer = u & 1;
        if (has_keys) {
            const auto place = [&](uint32_t w) { return s_keys[buffer] + R::slot(w / (4 * R::kPieces), w / 4 % R::kPieces) + w % 4 * 4; };
            if constexpr (R::kKeys == 4) {
                *(u32x4 *)place(word) = u32x4{key[0], key[1], key[2], key[3]};
            } else if constexpr (R::kKeys == 2) {
                *(uint2 *)place(word) = make_uint2(key[0], key[1]);
            } else {
#pragma unroll
                for (int j = 0; j < R::kKeys; j++) *(uint32_t *)place(word + j) = key[j];
            }
        }
        *(uint32_t *)((uint8_t *)s_scales[buffer] + key_scale_at) = key_scale;  // threads past the last write the same
    };
    const auto stage_values = [&](int u, int id, auto whole) {
        const int p0 = position_of(u);
        if (!has_values) return;
        if (!whole && u < units && is_edge(p0, id)) {
            // values that no row has may be anything: their scales count as 1, and 0 times their codes is 0;
            // NaN that some rows have and others do not is told apart afterwards
            const uint32_t tid = here(threadIdx.x);
#pragma unroll
            for (int j = 0; j < R::kValues; j++) {
                const Word w = word_of(tid * R::kValues + j);
                const int t0 = 16 * w.g + 4 * w.k;
                for (int i = 0; i < 4; i++) {
                    const int t = p0 + t0 + i;
                    const bool has = id >= 0 && t >= any_lo && t <= last, nan = (scale[j] >> (8 * i) & 255u) == 255u;
                    if (has && nan) atomicOr((unsigned long long *)&s_nan[u & 3][w.b], 1ull << (t0 + i));
                    if (!has || nan) scale[j] = (scale[j] & ~(255u << (8 * i))) | 127u << (8 * i);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < R::kValues; j++) {
            const Word w = word_of(threadIdx.x * R::kValues + j);
            uint32_t v[2][2];
            four(value[j], scale[j], v[0], v[1]);
            uint8_t *to = s_values[u & 1] + ((w.b * kGroups + w.g) * 2 + (w.k & 1)) * 512 + w.r * 16 + (w.k >> 1) * 8;
            *(uint2 *)to = make_uint2(v[0][0], v[0][1]);
            *(uint2 *)(to + 256) = make_uint2(v[1][0], v[1][1]);
        }
    };
    // unit u's turn brings in unit u + 1's keys and its own values, and sends for the next ones; past the last unit it
    // writes where nobody reads any more
    int id_now = -1, id_0 = id_of(0), id_1 = id_of(1), id_2 = id_of(2);  // pages of the unit at hand and of the next ones
    const uint8_t *tile_values = tile_of(id_1), *tile_keys = tile_of(id_2);
    const auto stage = [&](int u, auto whole) {
        stage_keys(u + 1);
        stage_values(u, id_0, whole);
        fetch_keys(u + 2, tile_keys);
        fetch_values(u + 1, tile_values);
    };
    const auto advance = [&](int u) {  // to the turn after unit u's
        id_now = id_0, id_0 = id_1, id_1 = id_2, id_2 = id_of(u + 3);
        tile_values = tile_keys, tile_keys = tile_of(id_2);
    };
    if (threadIdx.x < 4 * kBlocks) s_nan[threadIdx.x / kBlocks][threadIdx.x % kBlocks] = 0;
    if (units > 0) {
        fetch_keys(0, tile_of(id_0));
        fetch_values(0, tile_of(id_0));
        stage_keys(0);
        fetch_keys(1, tile_of(id_1));
    }

    // ----------------------------------------------------------------- turns
    f32x16 s[kHalves];                         // S^T: positions 32 h + 8 (i / 4) + 4 kq + i % 4 of row n32
    uint32_t p[R::kParts][kHalves][2][4] = {};  // the same positions' probabilities, as the second product takes them
    const auto scores = [&](int u) {
        const uint32_t l = here(lane);
        const int n32 = l % 32, kq = l / 32, buffer = u & 1;
        const int shift = n32 / 16 * 8 + (kTurns == 2 ? u % 2 * 16 : 0);
#pragma unroll
        for (int h = 0; h < kHalves; h++) {
            s[h] = f32x16{};
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const u32x4 w = *(const u32x4 *)(s_keys[buffer] + R::slot(32 * h + n32, 2 * c + kq));
                // byte 0 for the unit's lower half, 2 for its upper one
                const uint32_t by = s_scales[buffer][2 * c + kq][n32 % 16] >> shift;
                if constexpr (R::kF32) {
                    const float f = scale_at(by, 2 * h);
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const bf16x8 k = as_bf16(eight(w[t], f));
#pragma unroll
                        for (int part = 2; part >= 0; part--)
                            s[h] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                                k, as_bf16(u32x4{q[part][c][4 * t], q[part][c][4 * t + 1], q[part][c][4 * t + 2], q[part][c][4 * t + 3]}),
                                s[h], 0, 0, 0);
                    }
                } else {
                    const i32x8 k = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
#pragma unroll
                    for (int part = 1; part >= 0; part--) {
                        i32x8 x;
#pragma unroll
                        for (int j = 0; j < 8; j++) x[j] = (int)q[0][c][8 * part + j];
                        // fp4 times e4m3
                        const auto product = [&](auto k_byte, auto q_byte) {
                            s[h] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, x, s[h], 4, 0, k_byte, by, q_byte, q_scale);
                        };
                        const std::integral_constant<int, 0> b0;
                        const std::integral_constant<int, 1> b1;
                        const std::integral_constant<int, 2> b2;
                        if (h == 0 && part == 0) product(b0, b0);
                        if (h == 0 && part == 1) product(b0, b1);
                        if (h == 1 && part == 0) product(b2, b0);
                        if (h == 1 && part == 1) product(b2, b1);
                    }
                }
            }
        }
    };
    const auto softmax = [&](int u, int id, auto whole) {
        const int kq = here(lane / 32), p0 = position_of(u);
        if (!whole && (id < 0 || p0 < w_all || p0 + kUnit - 1 > w_early)) {
            const int from_t = id < 0 ? 64 : lo - p0 - 4 * kq, to_t = hi - p0 - 4 * kq;
#pragma unroll
            for (int h = 0; h < kHalves; h++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int t = 32 * h + i / 4 * 8 + i % 4;
                    if (t < from_t || t > to_t) s[h][i] = kNone;
                }
        }
        float top = kNone;
#pragma unroll
        for (int h = 0; h < kHalves; h++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, s[h][i]);
        const float best = max_of_halves(top);
        top = best * a.scale_log2;
        float from = m;
        // the maximum is raised once scores pass it by 2^8: any number near it does
        if (__any(top > m + 8.0f || special(top, m))) {
            if (fabsf(top) >= kFar) top = best * far_scale(a.scale_log2);
            const float to = __any(top > m + 8.0f) ? fmaxf(m, top) : m, by = m == kNone ? 0.0f : __builtin_amdgcn_exp2f(m - to);
            m = from = to;
            sum *= by;
#pragma unroll
            for (int b = 0; b < kBlocks; b++) o[b] *= by;
            if (special(m, 0.0f)) {
                from = 0.0f;
#pragma unroll
                for (int h = 0; h < kHalves; h++)
#pragma unroll
                    for (int i = 0; i < 16; i++) s[h][i] = far_score(s[h][i], far_scale(a.scale_log2), m);
            }
        }
        float sums[2] = {sum, 0.0f};
#pragma unroll
        for (int h = 0; h < kHalves; h++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[h][2 * j], a.scale_log2, -from));
                const float y = __builtin_amdgcn_exp2f(fmaf(s[h][2 * j + 1], a.scale_log2, -from));
                sums[j % 2] += x;
                sums[j % 2] += y;
                if constexpr (R::kF32) {
                    uint32_t part[3];
                    three_parts(x, y, part);
#pragma unroll
                    for (int t = 0; t < 3; t++) p[t][h][j / 4][j % 4] = part[t];
                } else {
                    p[0][h][j / 4][j % 4] = kv4::bf16_pair(x, y);
                }
            }
        sum = sums[0] + sums[1];
    };
    // O^T: dimensions 32 b + 8 (i / 4) + 4 kq + i % 4 of row n32
    const auto products = [&](int u, auto whole) {
        const uint32_t l = here(lane);
        const int n32 = l % 32, kq = l / 32, p0 = position_of(u);
        // a block's values are read some products ahead: longer than LDS takes to answer
        constexpr int kAhead = 4, kSteps = kGroups * kBlocks;
        u32x4 v[kAhead];
        const auto read = [&](int i) {
            v[i % kAhead] = *(const u32x4 *)(s_values[u & 1] + ((i % kBlocks * kGroups + i / kBlocks) * 2 + kq) * 512 + n32 * 16);
        };
#pragma unroll
        for (int i = 0; i < kAhead - 1; i++) read(i);
#pragma unroll
        for (int i = 0; i < kSteps; i++) {
            if (i + kAhead - 1 < kSteps) read(i + kAhead - 1);
            if (NC < 3) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = R::kParts - 1; t >= 0; t--) {
                const uint32_t *x = p[t][i / kBlocks / 2][i / kBlocks % 2];
                o[i % kBlocks] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16(v[i % kAhead]), as_bf16(u32x4{x[0], x[1], x[2], x[3]}),
                                                                         o[i % kBlocks], 0, 0, 0);
            }
        }
        if (!whole && (p0 < all_lo || p0 + kUnit - 1 > early)) {
#pragma unroll
            for (int b = 0; b < kBlocks; b++) {
                const uint64_t nan = s_nan[u & 3][b];
                if (!__any(nan != 0)) continue;
                // the row's positions of this unit: bits from lo to hi
                const int from_bit = min(max(lo - p0, 0), 64), to_bit = min(max(hi + 1 - p0, 0), 64);
                const uint64_t below = to_bit == 64 ? ~0ull : (1ull << to_bit) - 1, above = from_bit == 64 ? 0ull : ~0ull << from_bit;
                const float poison = nan & below & above ? NAN : 0.0f;
#pragma unroll
                for (int i = 0; i < 16; i++) o[b][i] += poison;
            }
        }
    };

    const std::true_type whole;
    const std::false_type any;
    const bool later = wave >= 4;  // half a turn behind
    if (units > 0) {
        sm::lds_barrier();
        if (later) sm::lds_barrier();
    }
    // units that are whole, and so are those beside them, go without questions
    int u = 0, from = works ? min(whole_from + 1, units) : units, to = works ? whole_to - 1 : 0;
    while (u < units) {
        for (; u < from; u++) {
            if (threadIdx.x < kBlocks) s_nan[(u + 1) & 3][threadIdx.x] = 0;  // the next unit's
            stage(u, any);
            if (R::kScoresFirst && is_live(position_of(u))) scores(u);
            if (u > 0 && is_live(position_of(u - 1))) products(u - 1, any);
            if (!R::kScoresFirst && is_live(position_of(u))) scores(u);
            sm::lds_barrier();
            advance(u);
            if (is_live(position_of(u))) softmax(u, id_now, any);
            if (!later || u + 1 < units) sm::lds_barrier();
        }
        from = units;
        for (; u < to && !holes; u++) {
            if (R::kScoresFirst) scores(u);
            stage(u, whole);
            products(u - 1, whole);
            if (!R::kScoresFirst) scores(u);
            sm::lds_barrier();
            advance(u);
            softmax(u, 0, whole);
            sm::lds_barrier();
        }
    }
    if (units > 0 && is_live(position_of(units - 1))) products(units - 1, any);

    if (32 * wave + (int)(lane % 32) >= rows) return;
    const int kq = lane / 32;
    sum = sum_of_halves(sum);
    const int64_t part = (int64_t)(piece.at + tile * a.kv_heads + head) * R::kRows + 32 * wave + lane % 32;
    const int64_t out = ((int64_t)(span.row + token) * a.heads + hq) * a.dim;
    const T *g = G ? G + (int64_t)(span.row + token) * a.g_view.stride + hq * a.g_view.head + a.g_view.offset : nullptr;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int b = 0; b < kBlocks; b++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = 32 * b + 2 * i + 4 * kq;
            if (piece.count > 1) {
                if (units > 0) *(f32x4 *)(parts + part * kPitch + d) = f32x4{o[b][i], o[b][i + 1], o[b][i + 2], o[b][i + 3]};
            } else if (d < a.dim) {
                float y[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    y[j] = sum == 0.0f ? 0.0f : o[b][i + j] * inv;
                    if (g) y[j] = gated(y[j], kv4::value(g[d + j]));
                }
                if constexpr (R::kF32) *(f32x4 *)(Y + out + d) = f32x4{y[0], y[1], y[2], y[3]};
                else *(uint2 *)(Y + out + d) = make_uint2(kv4::bf16_pair(y[0], y[1]), kv4::bf16_pair(y[2], y[3]));
            }
        }
    if (piece.count > 1 && kq == 0) stats[part] = make_float2(m, sum);
}

// ------------------------------------------------------------ pieces joined
// The pieces of one row: its sequence's partial sums, each brought to the
// largest of their maxima. kWaves waves a row share out the pieces; with one,
// four rows a workgroup.
template <int NC, typename T, int kWaves>
__global__ void __launch_bounds__(kWaves == 1 ? 256 : 64 * kWaves) k_kv4_join(Kv4Attention a, const T *G, T *Y, const float *parts,
                                                                              const float2 *stats, const int2 *info, int tiles,
                                                                              int row_bits) {
    constexpr int kPitch = 64 * NC, kSome = 8;
    const int s = blockIdx.y, group = a.heads / a.kv_heads;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int number = kWaves == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
    const int token = number / a.heads, h = number % a.heads;
    const kv4::Span span = kv4::span(a.q, s);
    if (token >= span.n) return;
    const int2 pieces = info[s];  // the first, how many
    if (pieces.y <= 1) return;
    const int head = h / group, row = token * group + h % group, tile = row >> row_bits;
    // tiles from a piece to the next: as many for all sequences, or (0) the sequence's own, and the first piece's tile is named
    int apart = tiles, first = pieces.x * tiles;
    if (tiles == 0) apart = (span.n * group + (1 << row_bits) - 1) >> row_bits, first = pieces.x;
    const int64_t step = (int64_t)a.kv_heads * apart << row_bits;
    const int64_t base = ((int64_t)((first + tile) * a.kv_heads + head) << row_bits) + row - (tile << row_bits);
    float top = kNone, all = 0.0f, v[NC] = {};
    const int share = (pieces.y + kWaves - 1) / kWaves, from = kWaves == 1 ? 0 : wave * share, end = min(from + share, pieces.y);
    for (int c0 = from; c0 < end; c0 += kSome) {
        float2 st[kSome];
        float x[kSome][NC];
#pragma unroll
        for (int j = 0; j < kSome; j++) {
            const int64_t at = base + min(c0 + j, end - 1) * step;
            st[j] = stats[at];
#pragma unroll
            for (int n = 0; n < NC; n++) x[j][n] = parts[at * kPitch + NC * lane + n];
        }
        float to = top;
#pragma unroll
        for (int j = 0; j < kSome; j++) to = fmaxf(to, st[j].x);  // those past the end repeat the last one
        const float was = top == kNone ? 0.0f : __builtin_amdgcn_exp2f(top - to);
        all *= was;
#pragma unroll
        for (int n = 0; n < NC; n++) v[n] *= was;
#pragma unroll
        for (int j = 0; j < kSome; j++) {
            if (c0 + j >= end) break;
            // a sum that is not a number, of scores that are none, stays one; else such a piece has left no values
            if (st[j].x == kNone) {
                all += st[j].y == 0.0f ? 0.0f : NAN;
                continue;
            }
            const float by = __builtin_amdgcn_exp2f(st[j].x - to);
            all += st[j].y * by;
#pragma unroll
            for (int n = 0; n < NC; n++) v[n] += x[j][n] * by;
        }
        top = to;
    }
    if constexpr (kWaves > 1) {
        __shared__ float s_v[kWaves][kPitch], s_top[kWaves], s_all[kWaves];
#pragma unroll
        for (int n = 0; n < NC; n++) s_v[wave][NC * lane + n] = v[n];
        if (lane == 0) s_top[wave] = top, s_all[wave] = all;
        __syncthreads();
        if (wave > 0) return;
        top = s_top[0];
#pragma unroll
        for (int w = 1; w < kWaves; w++) top = fmaxf(top, s_top[w]);
        all = 0.0f;
#pragma unroll
        for (int n = 0; n < NC; n++) v[n] = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const float by = s_top[w] == kNone ? 0.0f : __builtin_amdgcn_exp2f(s_top[w] - top);
            all += s_top[w] == kNone ? s_all[w] : s_all[w] * by;
#pragma unroll
            for (int n = 0; n < NC; n++) v[n] += s_v[w][NC * lane + n] * by;
        }
    }
    const T *g = G ? G + (int64_t)(span.row + token) * a.g_view.stride + h * a.g_view.head + a.g_view.offset : nullptr;
    T *y = Y + ((int64_t)(span.row + token) * a.heads + h) * a.dim;
#pragma unroll
    for (int n = 0; n < NC; n++) {
        const int d = NC * lane + n;
        if (d >= a.dim) break;
        const float out = all == 0.0f ? 0.0f : v[n] / all;
        kv4::store1(y + d, g ? gated(out, kv4::value(g[d])) : out);
    }
}

template <int NC, typename T>
void launch(sm_ctx *ctx, Kv4Attention a, const Kv4Shape &s, const T *Q, const uint8_t *pool, const T *G, T *Y, void *workspace) {
    a.pieces = s.pieces, a.least = s.budget > 0 ? kKv4FarLeast : s.least, a.budget = s.budget, a.units = (int)s.units;
    float *parts = (float *)workspace;
    float2 *stats = (float2 *)((char *)workspace + s.part_bytes);
    const bool cut = s.pieces > 1 || s.budget > 0;
    a.info = cut ? (int2 *)((char *)workspace + s.part_bytes + s.stat_bytes) : nullptr;
    const dim3 grid = s.pieces > 1 ? dim3((uint32_t)(a.kv_heads * s.tiles), (uint32_t)s.slots)
                                   : dim3((uint32_t)(a.kv_heads * (s.units + s.budget)));
    const auto run = [&](auto by_rows) {
        if constexpr (Prompt<NC, T>::kThere)
            if (s.prompt)
                k_kv4_prompt<NC, T, by_rows><<<grid, Prompt<NC, T>::kThreads, 0, ctx->stream>>>(a, Q, pool, G, Y, parts, stats, s.tiles);
        if (!s.prompt) k_kv4_rows<NC, T, by_rows><<<grid, 256, 0, ctx->stream>>>(a, Q, pool, G, Y, parts, stats);
    };
    if (s.budget > 0) run(std::true_type());
    else run(std::false_type());
    if (!cut) return;
    const int tiles = s.budget > 0 ? 0 : s.tiles, row_bits = s.prompt ? 8 : 4;
    static_assert(kKv4PromptRows == 1 << 8, "a tile's rows");
    const uint32_t all = (uint32_t)a.q.longest * a.heads;
    if ((int64_t)all * a.q.count < kKv4JoinRows)
        k_kv4_join<NC, T, 16><<<dim3(all, a.q.count), 1024, 0, ctx->stream>>>(a, G, Y, parts, stats, a.info, tiles, row_bits);
    else
        k_kv4_join<NC, T, 1><<<dim3((all + 3) / 4, a.q.count), 256, 0, ctx->stream>>>(a, G, Y, parts, stats, a.info, tiles, row_bits);
}
template <typename T>
void launch(sm_ctx *ctx, const Kv4Attention &a, const T *Q, const uint8_t *pool, const T *G, T *Y, void *workspace) {
    const Kv4Shape s = kv4_shape(a.q, a.heads, a.kv_heads, a.dim, a.window, sizeof(T) == 2);
    switch (kv4_pitch(a.dim) / 64) {
        case 1: return launch<1, T>(ctx, a, s, Q, pool, G, Y, workspace);
        case 2: return launch<2, T>(ctx, a, s, Q, pool, G, Y, workspace);
        case 3: return launch<3, T>(ctx, a, s, Q, pool, G, Y, workspace);
        default: return launch<4, T>(ctx, a, s, Q, pool, G, Y, workspace);
    }
}

}  // namespace

namespace smi {

int kv4_attention_launch(sm_ctx *ctx, const Kv4Attention &a, const void *Q, const uint8_t *pool, const void *G, void *Y, bool bf16,
                         void *workspace) {
    if (bf16) launch(ctx, a, (const uint16_t *)Q, pool, (const uint16_t *)G, (uint16_t *)Y, workspace);
    else launch(ctx, a, (const float *)Q, pool, (const float *)G, (float *)Y, workspace);
    return launched(ctx);
}

}  // namespace smi
