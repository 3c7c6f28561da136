// The host-side rules of the 8-bit products' kernels (csrc/internal.h) as C
// functions, for tests without a GPU.
#include <hip/hip_runtime.h>

#include "../stratacuda_amd/csrc/internal.h"

extern "C" void rule_piece(int left, int most, uint32_t pitch, int block, uint32_t *bytes, uint32_t *offset) {
    const smi::F8Piece p = smi::f8_piece(left, most, pitch, block);
    *bytes = p.bytes, *offset = p.offset;
}
