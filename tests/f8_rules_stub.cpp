// The host-side rules of the 8-bit products' kernels (csrc/internal.h,
// csrc/f8_shapes.h) as C functions, for tests without a GPU.
#include <hip/hip_runtime.h>

#include "../stratacuda_amd/csrc/f8_shapes.h"
#include "../stratacuda_amd/csrc/internal.h"

extern "C" {
void rule_piece(int first, int left, int rows, int most, int *to) {
    const smi::F8Piece p = smi::f8_piece(first, left, rows, most);
    to[0] = p.first, to[1] = p.count;
}
// {tokens, rows, resident, blocks} of the shape that a product of this output takes
int rule_shape(int out, int tokens, int rows, int kb, int cus, int *to) {
    float us = 0.0f;
    const int i = f8::best_shape(tokens, rows, kb, (f8::Out)out, cus, &us);
    const f8::Shape &s = f8::kShapes[out][i];
    to[0] = s.tokens, to[1] = s.rows, to[2] = s.resident, to[3] = s.blocks;
    return i;
}
// The same of the tables' i-th
void rule_listed(int out, int i, int *to) {
    const f8::Shape &s = f8::kShapes[out][i];
    to[0] = s.tokens, to[1] = s.rows, to[2] = s.resident, to[3] = s.blocks;
}
int rule_gated(int tokens, int ff, int kb, int cus) { return f8::gated_tile(tokens, ff, kb, cus); }
int rule_grid(int n, int kb, int cus, int resident) { return f8::tile_grid(n, kb, cus, resident); }
}
