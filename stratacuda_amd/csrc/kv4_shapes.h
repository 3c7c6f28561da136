// Which kernel a call of attention over a 4-bit cache runs, and how it cuts the
// context: plain numbers, the same on every machine.
#pragma once
#include <algorithm>

#include "internal.h"

namespace smi {

// The least pages that are worth a piece: one a wave.
constexpr int kKv4Least = 4;
// From so many rows a wave joins a row's pieces: they fill the GPU.
constexpr int kKv4JoinRows = 512;
constexpr int kKv4PromptRows = 256;

// Sixteen rows a workgroup, or 256. The first takes W (17 + p) of its turns, W workgroups of p pages on average (17 pages
// are what a workgroup costs besides); the second half as many of theirs and 14 us more to begin and end with, but only
// where several workgroups read the same pages, so from 1024 rows of a key-value head. Measured, in us, sixteen rows
// against 256, 32 heads on 8 of dimension 128, bf16: 1024 tokens 32 and 45, 2048 tokens 81 and 66, 512 tokens over 4096
// positions 60 and 52, 8 prompts of 512 tokens 95 and 62, 8 times 64 tokens over 4096 positions 67 and 114. Dimensions
// up to 64 (16 heads, 4096 tokens 86 and 89, 512 over 32768 152 and 95) and f32 (512 over 8192 173 and 165, 8 of 512 tokens
// 164 and 104) gain later; f32 of more than 128 dimensions has no second kind.
constexpr int kKv4PromptLeast = 1024;
constexpr int64_t kKv4PromptTurns = 53 << 10, kKv4PromptTurnsF32 = 140 << 10, kKv4PromptTurns64 = 220 << 10;

struct Kv4Shape {
    bool prompt;
    int tile_rows, tiles, pieces, least;
    uint64_t slots, part_bytes, stat_bytes, bytes;
};
inline Kv4Shape kv4_shape(const Kv4Sequences &q, int heads, int kv_heads, int dim, int window, bool bf16) {
    Kv4Shape s;
    const int64_t rows = (int64_t)q.longest * (heads / kv_heads);
    const int pitch = kv4_pitch(dim);
    const int64_t pages = window > 0 ? std::min<int64_t>(q.table_pages, ((int64_t)window + q.longest) / 64 + 2) : q.table_pages;
    const int64_t reached = std::max<int64_t>(pages - q.longest / 128, 1);  // a row's on average, of the longest sequence's
    const int64_t turns = (int64_t)q.count * kv_heads * ((rows + 15) / 16) * (17 + reached);
    s.prompt = (bf16 || pitch <= 128) && rows >= kKv4PromptLeast &&
               turns >= (pitch == 64 ? kKv4PromptTurns64 : bf16 ? kKv4PromptTurns : kKv4PromptTurnsF32);
    s.tile_rows = s.prompt ? kKv4PromptRows : 16;
    s.tiles = (int)((rows + s.tile_rows - 1) / s.tile_rows);
    s.least = kKv4Least;
    const int64_t each = (int64_t)kv_heads * s.tiles;
    const int64_t most = q.table_pages <= s.least ? 1 : (int64_t)q.count * ((q.table_pages + s.least - 1) / s.least);
    // Sixteen rows: a workgroup for each CU, or three for two CUs where registers leave room for three on each (32 sequences
    // of dimension 128: 51 us with one for each, 42 with these). Prompts that leave CUs idle: what one round holds, two
    // where most of the context is the prompt itself, whose first rows reach little of it (4096 tokens, 12 heads on 4 of
    // dimension 192: 179 us whole, 128 in pieces).
    const int64_t whole = each * q.count;
    int64_t pieces = !s.prompt ? ((pitch > 128 || !bf16 ? 256 : 384) + each - 1) / each
                     : whole >= 256 ? 1 : (64 * (int64_t)q.table_pages <= 2 * (int64_t)q.longest ? 512 : 256) / whole;
    if (pieces > most) pieces = most;
    s.pieces = pieces < 1 ? 1 : (int)pieces;
    s.slots = (uint64_t)(s.pieces > 1 ? s.pieces + q.count : q.count);
    s.part_bytes = s.pieces > 1 ? s.slots * each * s.tile_rows * pitch * 4 : 0;
    s.stat_bytes = s.pieces > 1 ? s.slots * each * s.tile_rows * 8 : 0;
    s.bytes = s.part_bytes + s.stat_bytes + (s.pieces > 1 ? (uint64_t)q.count * 8 : 0);
    if (s.pieces == 1) s.least = q.table_pages + 1;  // one piece a sequence: as large as any
    return s;
}

// Enough for either type, with a window and without one: a window only decides which kernel it is.
inline uint64_t kv4_workspace(const Kv4Sequences &q, int heads, int kv_heads, int dim) {
    uint64_t most = 0;
    for (int bf16 = 0; bf16 < 2; bf16++)
        for (int window = 0; window < 2; window++) most = std::max(most, kv4_shape(q, heads, kv_heads, dim, window, bf16).bytes);
    return most;
}

}  // namespace smi
