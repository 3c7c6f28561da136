// How the 8-bit products (f8_project.hip) are shared out over the GPU: plain
// arithmetic on sizes, for the host.
#pragma once
#include <stdint.h>

namespace f8 {

enum Out { kF32, kBf16, kHidden, kCodes };  // kHidden, kCodes: silu(gate) * up in f32, in 8 bits

// A way to share out a product: a workgroup's tokens and rows (of each matrix),
// how many of them a CU holds, the blocks of 128 columns in a step of theirs,
// what a step takes where a CU has one of them and where it has all, and what a
// round over the GPU takes beside its steps, in us: fitted to whole calls on one
// MI355X, 1 to 1024 tokens, 640 to 20,480 rows, 1280 to 10,240 columns. Over
// those the choice is 1.5% slower than the best shape on average (to f32; to
// bf16 1.7%, a gated pair 0.4%), 25% at worst (512 tokens, 8192 x 8192, to bf16).
// The times are from before neighbouring workgroups of an XCD shared their rows,
// which some thousand tokens in 64 x 64 streams gain from (2048 tokens, 6144 to
// 2560, to f32 70 us; the table says 77).
// Both sides in us, to f32: 16 x 16 against 32 x 32 for 1 token, 2560 columns to
// 10,240 rows 5.9 and 7.0, 16 tokens, 8192 x 8192 15.0 and 13.1; 32 x 16 against
// 16 x 16 for 32 tokens, 6144 to 2560 6.5 and 7.9; 64 x 32 against 64 x 64 for 64
// tokens, 8192 x 8192 17.0 and 22.2, for 256 51.5 and 37.9; 32 x 64 against 64 x 64
// for 256 tokens, 2560 to 10,240 21.2 and 22.7; 64 x 64 of streams against tiles
// of 128 x 128 there 22.7 and 30.2. To bf16, 512 tokens: streams 26.7, tiles of
// 64 x 64 27.2, of 256 x 128 25.3; 1024 tokens, 4096 x 4096 tiles of 64 x 64 30.6,
// of 128 x 128 36.9.
struct Shape {
    int tokens, rows, resident, blocks;
    float one, all, round;
};
constexpr int kShapeCount = 10;
constexpr Shape kShapes[3][kShapeCount] = {  // by Out
    {{16, 16, 4, 8, 0.73f, 2.56f, 0.0f}, {32, 16, 3, 8, 0.89f, 2.27f, 0.5f}, {32, 32, 2, 8, 1.18f, 2.16f, 0.7f},
     {64, 32, 1, 8, 1.55f, 1.55f, 1.9f}, {32, 64, 3, 4, 0.78f, 2.10f, 3.7f}, {64, 64, 2, 4, 1.19f, 2.10f, 4.2f},
     {128, 128, 2, 1, 1.15f, 1.80f, 7.0f}, {256, 128, 1, 1, 1.50f, 1.50f, 11.0f}, {256, 256, 1, 1, 2.50f, 2.50f, 11.0f}},
    {{16, 16, 4, 8, 0.68f, 2.53f, 0.0f}, {32, 16, 3, 8, 0.88f, 2.26f, 0.0f}, {32, 32, 2, 8, 1.15f, 2.16f, 0.0f},
     {64, 32, 1, 8, 1.50f, 1.50f, 1.0f}, {32, 64, 3, 4, 0.69f, 1.93f, 3.1f}, {64, 64, 2, 4, 0.94f, 1.83f, 3.3f},
     {128, 128, 2, 1, 0.75f, 0.97f, 6.0f}, {256, 128, 1, 1, 0.96f, 0.96f, 4.5f}, {256, 256, 1, 1, 1.35f, 1.35f, 9.0f},
     {64, 64, 4, 1, 0.35f, 0.85f, 3.0f}},
    {{16, 16, 3, 8, 0.94f, 2.58f, 0.0f}, {32, 16, 2, 8, 1.14f, 2.02f, 0.4f}, {32, 32, 1, 8, 1.40f, 1.40f, 1.9f},
     {64, 32, 2, 4, 1.12f, 2.05f, 3.3f}}};

// The shape whose rounds over `cus` CUs take least, for kb blocks of 128
// columns: its index in kShapes, and that time in us.
inline int best_shape(int tokens, int rows, int kb, Out out, int cus, float *us) {
    int best = -1;
    for (int i = 0; i < kShapeCount; i++) {
        const Shape &s = kShapes[out][i];
        if (s.tokens == 0) continue;
        const int64_t n = (int64_t)((tokens + s.tokens - 1) / s.tokens) * ((rows + s.rows - 1) / s.rows);
        const int64_t slots = (int64_t)cus * s.resident, over = (n % slots + cus - 1) / cus;  // workgroups of a CU in the last round
        const int steps = (kb + s.blocks - 1) / s.blocks;
        const float last = s.resident == 1 ? s.one : s.one + (s.all - s.one) * (over - 1) / (s.resident - 1);
        const float time = n / slots * (s.all * steps + s.round) + (over ? last * steps + s.round : 0.0f);
        if (best < 0 || time < *us) *us = time, best = i;
    }
    return best;
}

// Workgroups that go through n persistent tiles, a multiple of the eight XCDs:
// as many as the GPU holds, or one a tile. With one block of columns, nothing
// is left of a tile's steps to bring the next in.
inline int tile_grid(int n, int kb, int cus, int resident) {
    const int all = (n + 7) / 8, held = (cus / 8 > 1 ? cus / 8 : 1) * resident;
    return (kb < 2 || all < held ? all : held) * 8;
}

// A gated pair: sums to f32 into the workspace and the conversion of rows, or
// one kernel whose tiles of 128 columns end in codes: 2.6 us a step and 16 us a
// round of tiles of 256 tokens, 1.55 and 9 of 128. Fitted as above, 96 to 8192
// tokens, 640 to 8192 columns out, 1280 to 6144 in: 0.2% slower than the best of
// the three on average, 7% at worst. In us, of 256 tokens, of 128, apart: 4096
// tokens, 2560 to 8192 268, 288 and 394; 1536 tokens, 2560 to 2560 63, 40 and 56;
// 256 tokens, 2560 to 8192 61, 38 and 32.
inline int gated_tile(int tokens, int ff, int kb, int cus) {
    auto rounds = [&](int n) { return ((int64_t)((tokens + n - 1) / n) * ((ff + 127) / 128) + cus - 1) / cus; };
    float apart = 0.0f;
    best_shape(tokens, ff, kb, kHidden, cus, &apart);
    apart += 3.0f + 5.0f * tokens * ff / 4e6f;  // and the conversion
    const float wide = rounds(256) * (2.6f * kb + 16.0f), narrow = rounds(128) * (1.55f * kb + 9.0f);
    return wide < apart && wide < narrow ? 256 : narrow < apart ? 128 : 0;
}

}  // namespace f8
