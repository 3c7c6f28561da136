// Which kernel a call of attention over a 4-bit cache runs, and how it cuts the
// context: plain numbers, the same on every machine.
#pragma once
#include <algorithm>

#include "internal.h"

namespace smi {

// The least pages that are worth a piece: one a wave. 2048 positions of 24 heads on 2 of dimension 256, f32: 16.9 us, 16.7 with
// 2 and 19.5 with 8.
constexpr int kKv4Least = 4;
// Rows that reach up to so many pages are not cut: two or three turns of four pages take less than the launch that joins
// them. In pieces of 4 pages and whole, us: 500 positions, 32 heads on 8 of dimension 128 in bf16, 11.0 and 8.8 (32 sequences 11.9 and
// 10.0), 24 heads on 2 of 256 in f32 18.0 and 17.2; 700 positions 10.9 and 9.5 (32 sequences 14.3 and 11.1) but 17.5 and 19.9
// (bf16 14.6 and 15.6): f32 and more than 128 dimensions, whose turns are longer, from fewer pages.
constexpr int kKv4Whole = 12, kKv4WholeWide = 8;
// From so many rows a wave joins a row's pieces, else sixteen do. Sixteen against one, us: 24 rows of 128 pieces 26 and 47, 64
// rows of 32 14.8 and 16.8, 256 rows of 43 22.6 and 22.4, 512 rows of 25 38.8 and 37.3, 1024 rows 46.5 and 42.6.
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
    int64_t units;  // kv4_units
    uint64_t slots, part_bytes, stat_bytes, bytes;
};
// A window past every position of the tables is none (0). Any other is below 2^30 and a row's position above -2^24, so that
// the kernels' differences of the two stay within 32 bits.
inline int kv4_window(int window, int table_pages) { return window >= 64 * (int64_t)table_pages ? 0 : window; }
// The pages that a sequence's rows reach at most.
inline int64_t kv4_pages(const Kv4Sequences &q, int window) {
    return window > 0 ? std::min<int64_t>(q.table_pages, ((int64_t)window + q.longest) / 64 + 2) : q.table_pages;
}
// Tiles of all sequences at most.
inline int64_t kv4_units(const Kv4Sequences &q, int group, int tile_rows) {
    const int64_t rows = (int64_t)q.longest * group;
    return std::min(q.count * ((rows + tile_rows - 1) / tile_rows), (int64_t)q.tokens * group / tile_rows + q.count);
}
inline bool kv4_prompt(const Kv4Sequences &q, int heads, int kv_heads, int dim, int window, bool bf16) {
    const int64_t rows = (int64_t)q.longest * (heads / kv_heads);
    const int pitch = kv4_pitch(dim);
    const int64_t reached = std::max<int64_t>(kv4_pages(q, window) - q.longest / 128, 1);  // a row's on average, of the longest sequence's
    const int64_t turns = (int64_t)q.count * kv_heads * ((rows + 15) / 16) * (17 + reached);
    // a prompt among many single tokens, each of which would take 256 rows (255 tokens over 1000 positions each and 2048 new
    // ones: 152 us, where 256 rows a tile and as many tiles for each sequence took 1920)
    if (8 * kv4_units(q, heads / kv_heads, kKv4PromptRows) > kv4_units(q, heads / kv_heads, 16)) return false;
    return (bf16 || pitch <= 128) && rows >= kKv4PromptLeast &&
           turns >= (pitch == 64 ? kKv4PromptTurns64 : bf16 ? kKv4PromptTurns : kKv4PromptTurnsF32);
}
inline Kv4Shape kv4_cut(const Kv4Sequences &q, int heads, int kv_heads, int dim, int window, bool bf16, bool prompt) {
    Kv4Shape s;
    const int64_t rows = (int64_t)q.longest * (heads / kv_heads), pages = kv4_pages(q, window);
    const int pitch = kv4_pitch(dim);
    const bool wide = pitch > 128 || !bf16;
    s.prompt = prompt;
    s.tile_rows = s.prompt ? kKv4PromptRows : 16;
    s.tiles = (int)((rows + s.tile_rows - 1) / s.tile_rows);
    s.least = kKv4Least;
    s.units = kv4_units(q, heads / kv_heads, s.tile_rows);
    const int64_t each = (int64_t)kv_heads * s.tiles;
    const int64_t most = pages <= (wide ? kKv4WholeWide : kKv4Whole) ? 1 : (int64_t)q.count * ((q.table_pages + s.least - 1) / s.least);
    // Sixteen rows: a workgroup for each CU, or three for two CUs where registers leave room for three on each (32 sequences
    // of dimension 128: 51 us with one for each, 42 with these). Prompts that leave CUs idle: what one round holds, two
    // where most of the context is the prompt itself, whose first rows reach little of it (4096 tokens, 12 heads on 4 of
    // dimension 192: 179 us whole, 128 in pieces).
    const int64_t whole = each * q.count;
    int64_t pieces = !s.prompt ? ((wide ? 256 : 384) + each - 1) / each
                     : whole >= 256 ? 1 : (64 * (int64_t)q.table_pages <= 2 * (int64_t)q.longest ? 512 : 256) / whole;
    // pieces come for every tile of the longest sequence: not where nearly all of these would be empty
    if (pieces > most) pieces = most;
    if ((int64_t)s.tiles * q.count > 4 * s.units) pieces = 1;
    s.pieces = pieces < 1 ? 1 : (int)pieces;
    s.slots = (uint64_t)(s.pieces > 1 ? s.pieces + q.count : q.count);
    s.part_bytes = s.pieces > 1 ? s.slots * each * s.tile_rows * pitch * 4 : 0;
    s.stat_bytes = s.pieces > 1 ? s.slots * each * s.tile_rows * 8 : 0;
    s.bytes = s.part_bytes + s.stat_bytes + (s.pieces > 1 ? (uint64_t)q.count * 8 : 0);
    if (s.pieces == 1) s.least = q.table_pages + 1;  // one piece a sequence: as large as any
    return s;
}
inline Kv4Shape kv4_shape(const Kv4Sequences &q, int heads, int kv_heads, int dim, int window, bool bf16) {
    return kv4_cut(q, heads, kv_heads, dim, window, bf16, kv4_prompt(q, heads, kv_heads, dim, window, bf16));
}

// Enough for either type and every window: the narrowest and none tell which kernels it may be, and none has the most pieces.
inline uint64_t kv4_workspace(const Kv4Sequences &q, int heads, int kv_heads, int dim) {
    uint64_t most = 0;
    for (int bf16 = 0; bf16 < 2; bf16++)
        for (int window = 0; window < 2; window++)
            most = std::max(most, kv4_cut(q, heads, kv_heads, dim, 0, bf16, kv4_prompt(q, heads, kv_heads, dim, window, bf16)).bytes);
    return most;
}

}  // namespace smi
