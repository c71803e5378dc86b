// What both the launches of prefix attention (prefix_attention.cu) and the rule of which steps take it (host/fork.cpp, ops.prefix_attention_pays)
// go by: sizes of tiles, and into how many pieces tiles are cut.
#pragma once

namespace llmb_prefix {

constexpr int SMS = 148;
constexpr int FEW_ROWS = 16;         // rows of a sequence (new tokens times the query heads of a key head) above which a group's tiles walk own pages too
constexpr int TILE_ROWS = 128;       // of a group, up to which two blocks share an SM
constexpr int WIDE_ROWS = 256;       // of a tile of larger groups
constexpr int MAX_SPLITS = 64;       // pieces of a tile

// the least power of two that is no less than n: replayed steps of one bucket make the same launches
inline int bucket(int n) {
    int b = 1;
    while (b < n) b *= 2;
    return b;
}

// A few shared pages are read by every sequence itself: they come from L2, and a launch, its start and its parts are saved. One page always (three
// sequences of a small 32-bit model 14.5 us from the host for 22). Instead of the wide kernel up to 4,096 pages of a key head in all: heads of 128
// over 8, 64 sequences behind 2, 4 and 8 pages 12.3, 15.0, 20.3 us for 20.5, 22.5, 22.8; behind 16 pages 24 either way. Instead of the tile kernel up to
// 512, while no SM has two sequences: 8 behind 4, 8 and 16 pages 7.1, 7.7 and 12.7 for 9.3, 9.6 and 10.1; 32 behind 2 pages 12.7 for 11.2.
// walks: sequences times key heads; shared: pages, a bucket's; group_rows: of the largest group; whole: tiles walk own pages too.
inline bool reads_alone(long long walks, int shared, long long group_rows, bool tc, bool whole) {
    if (whole || shared <= 1) return !whole && shared == 1;
    return tc && group_rows > FEW_ROWS && (group_rows > TILE_ROWS ? walks * shared <= 4096 : walks * shared <= 512 && walks <= SMS);
}

// Pieces of each of `rest` tiles, the last round of blocks, whose walks have up to `walk` pages: four pages a piece at least.
inline int wide_pieces(long long rest, int walk, int head_dim) {
    long long best = 0;
    int pieces = 1;
    for (int n = 1; n <= MAX_SPLITS && (n == 1 || 4 * n <= walk) && rest > 0; ++n) {
        // In pages' time (0.85 us): rounds of blocks times what one takes, its pages and about twelve for its start and its end, and the parts
        // written and read again at some 5 TB/s.
        long long time = (rest * n + SMS - 1) / SMS * ((walk + n - 1) / n + 12) + (n > 1 ? rest * n * WIDE_ROWS * head_dim * 8 / 4300000 : 0);
        if (n == 1 || time < best) {
            best = time;
            pieces = n;
        }
    }
    return pieces;
}

}  // namespace llmb_prefix
