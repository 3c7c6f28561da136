// What csrc/kv4_shapes.h says of batches whose sequences' rows differ, as C
// functions, for tests without a GPU.
#include <hip/hip_runtime.h>

#include "../stratacuda_amd/csrc/kv4_shapes.h"

extern "C" {
// {many rows' kernel, tile rows, tiles, pieces, budget, units, workspace bytes, least of a piece by rows}
void rule_unlike(int count, int tokens, int longest, int table_pages, int heads, int kv_heads, int dim, int window, int bf16, long long *to) {
    const smi::Kv4Shape s = smi::kv4_shape({count, tokens, longest, table_pages, nullptr, nullptr, nullptr}, heads, kv_heads, dim, window, bf16);
    to[0] = s.prompt, to[1] = s.tile_rows, to[2] = s.tiles, to[3] = s.pieces, to[4] = s.budget, to[5] = s.units,
    to[6] = (long long)s.workspace, to[7] = smi::kKv4FarLeast;
}
unsigned long long rule_workspace(int count, int tokens, int longest, int table_pages, int heads, int kv_heads, int dim) {
    return smi::kv4_workspace({count, tokens, longest, table_pages, nullptr, nullptr, nullptr}, heads, kv_heads, dim);
}
}
