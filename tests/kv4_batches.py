"""Batches that reach each kernel of attention over a 4-bit cache, by
csrc/kv4_shapes.h: (rows, length) of the sequences, heads, key-value heads and
the width of the page tables. No counterpart in the reference."""

# 256 rows a workgroup, the context whole and in pieces
WHOLE = dict(sequences=[(70, 200), (130, 300), (1, 129), (33, 33), (3, 3)] + [(0, 9)] * 19, heads=64, kv=1, width=8)
PIECES = dict(sequences=[(17, 1500), (130, 700), (5, 0), (1, 64), (96, 256), (2, 130)], heads=16, kv=2, width=400)
# more than 64 pages a workgroup
LONG = dict(sequences=[(130, 4300)] + [(0, 9)] * 3, heads=128, kv=8, width=70)
# 16 rows a workgroup, in pieces: of a row by sixteen waves joined, and by one
FEW = dict(sequences=[(1, 1500), (3, 700), (2, 0), (1, 64), (1, 1100)], heads=8, kv=2, width=40)
SOME = dict(sequences=[(20, 1500), (16, 700), (5, 0), (1, 64)], heads=8, kv=2, width=40)
# a prompt among single tokens
MIXED = dict(sequences=[(1, 100)] * 20 + [(200, 300)] + [(1, 1000 - 40 * i) for i in range(24)], heads=24, kv=2, width=16)
LONG_WINDOWS = (70, 300, 1000)
# more than 64 pages each; more than 128 pieces of a row
LONG_ROWS = dict(sequences=[(96, 96)] + [(2, 4700)] * 7, heads=8, kv=1, width=74)
FAR_ROWS = dict(sequences=[(1, 520 * 64 - 5)], heads=4, kv=1, width=520)

TYPES = [("bf16", 64), ("bf16", 40), ("bf16", 128), ("bf16", 72), ("bf16", 192), ("bf16", 256), ("bf16", 200), ("f32", 64), ("f32", 24),
         ("f32", 128), ("f32", 104)]  # those that have the many rows' kernel
WINDOWS = (1, 63, 64, 65, 100)

# sequences' rows differ, in tables of long contexts: each sequence's own tiles cut, of 16 rows and of 256
UNLIKE = dict(sequences=[(1, 1500), (60, 2900), (0, 9), (1, 64), (5, 0), (1, 6500), (7, 4)], heads=12, kv=2, width=200)
UNLIKE_PROMPT = dict(sequences=[(1, 5000), (130, 3000), (0, 9), (17, 2200), (20, 7)], heads=32, kv=2, width=600)
