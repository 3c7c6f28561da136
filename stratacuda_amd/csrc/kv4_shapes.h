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

// Sequences whose rows differ (a prompt or some tokens among single ones), so that they have two thirds or less of the tiles
// which as many of the longest one's would make, are cut by rows: equal pieces of all tiles' pages. In tables of so many
// pages, and where their tiles leave CUs idle; 256 rows a workgroup from the larger number on where the rule for equal
// sequences makes three pieces or more. Pieces of at least kKv4FarLeast pages. In us, by that rule and by rows, 24 heads on 2
// of dimension 256, bf16: 512 tokens and one over 32768 positions each 1376 and 393 (over 16384 703 and 220, over 8192 370
// and 134), 64 tokens and four single ones over 131072 positions 1221 and 77, 96 tokens and 8 over 9000 91 and 28, 8, 5, 3
// and 1 tokens over 32768 and fewer 71 and 54 (f32 64 and 54). Where the tiles are fewer by less: 2 tokens and 7 single ones
// over 1000 positions in a table for 8200 20.7 and 30.8. Least 8, 16 and 32: 96 tokens and 8 27, 28 and 33; 16 tokens and
// 3 over 8192, 32 heads on 8 of 128 in f32, 32, 32 and 27.
constexpr int kKv4Far = 512, kKv4FarRows = 128, kKv4FarLeast = 16;

struct Kv4Shape {
    bool prompt;
    int tile_rows, tiles;
    int64_t units;      // kv4_units
    // pieces of all sequences' pages, of at least so many, for each of the longest one's tiles; 1: none is cut
    int pieces, least;
    uint64_t slots, bytes;
    int budget;         // or, where none is: pieces of all tiles' pages, for each sequence's own tiles; 0: no
    uint64_t part_bytes, stat_bytes, workspace;
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
inline Kv4Shape kv4_cut(const Kv4Sequences &q, int heads, int kv_heads, int dim, int window, bool bf16, bool prompt,
                        bool by_rows = true) {
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
    if (pieces > most) pieces = most;
    // By rows: where one workgroup fills a CU, as many as one round holds, each tile's last pieces with them; else those besides.
    const bool alone = s.prompt || (!bf16 && pitch > 128);  // one workgroup a CU
    const int64_t fill = (!s.prompt && !wide ? 384 : 256) / kv_heads, budget = alone ? fill - s.units : fill;
    const bool far = pages >= (s.prompt && pieces > 2 ? kKv4Far : kKv4FarRows);
    s.budget = by_rows && far && 3 * s.units <= 2 * (int64_t)s.tiles * q.count && budget >= s.units ? (int)budget : 0;
    // pieces come for every tile of the longest sequence: not where nearly all of these would be empty
    if (s.budget || (int64_t)s.tiles * q.count > 4 * s.units) pieces = 1;
    s.pieces = pieces < 1 ? 1 : (int)pieces;
    s.slots = (uint64_t)(s.pieces > 1 ? s.pieces + q.count : q.count);
    const uint64_t held = s.budget ? (uint64_t)kv_heads * (s.units + s.budget) : s.pieces > 1 ? s.slots * each : 0;
    s.part_bytes = held * s.tile_rows * pitch * 4;
    s.stat_bytes = held * s.tile_rows * 8;
    s.workspace = held ? s.part_bytes + s.stat_bytes + (uint64_t)q.count * 8 : 0;
    s.bytes = s.pieces > 1 ? s.workspace : 0;
    if (s.pieces == 1) s.least = q.table_pages + 1;  // what is not cut is one piece, as large as any; no launch reads it
    return s;
}
inline Kv4Shape kv4_shape(const Kv4Sequences &q, int heads, int kv_heads, int dim, int window, bool bf16) {
    return kv4_cut(q, heads, kv_heads, dim, window, bf16, kv4_prompt(q, heads, kv_heads, dim, window, bf16));
}

// Enough for either type and every window: the narrowest and none tell which kernels it may be, and none has the most pieces,
// or those by rows in their place.
inline uint64_t kv4_workspace(const Kv4Sequences &q, int heads, int kv_heads, int dim) {
    uint64_t most = 0;
    for (int bf16 = 0; bf16 < 2; bf16++)
        for (int window = 0; window < 2; window++) {
            const bool prompt = kv4_prompt(q, heads, kv_heads, dim, window, bf16);
            for (const bool by_rows : {false, true}) most = std::max(most, kv4_cut(q, heads, kv_heads, dim, 0, bf16, prompt, by_rows).workspace);
        }
    return most;
}

}  // namespace smi
