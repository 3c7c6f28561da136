// The host-side rules of the 8-bit products' kernels (csrc/internal.h) as C
// functions, for tests without a GPU.
#include <hip/hip_runtime.h>

#include "../stratacuda_amd/csrc/internal.h"

extern "C" void rule_piece(int first, int left, int rows, int most, int *to) {
    const smi::F8Piece p = smi::f8_piece(first, left, rows, most);
    to[0] = p.first, to[1] = p.count;
}
