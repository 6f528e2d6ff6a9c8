// Which of their kernels the operators for several experts per token take: rules on sizes, types and alignment, host code without
// a device header, so that the tests can ask what a shape reaches.  The comments beside the kernels have what each was measured at.
#pragma once

#include <algorithm>

namespace infmoe {
namespace forms {

// ---------------------------------------------------------------- adapters (lora.hip)
// The adapters' first product: a wave per row and rank, a wave per row and four ranks, or tiles of rows on the matrix cores.
enum class Shrink { ONE_RANK, FOUR_RANKS, TILES };

constexpr int kFewShrink = 1024;  // rows up to which u takes waves of their own per row

inline Shrink shrink_form(int T, int padded_ranks) {
    if ((long long)T * padded_ranks <= 4096) return Shrink::ONE_RANK;
    return T <= kFewShrink ? Shrink::FOUR_RANKS : Shrink::TILES;
}

// The projection: W streamed past blocks of 16 * fm rows, 16 * fn of its rows a workgroup; tall tiles of 32 * fm rows, their K cut
// over `splits` workgroups; or tiles of 64 x 128.
struct Project {
    enum Kind { STREAM, TALL, TILES } kind;
    int fm, fn, splits;
};

constexpr int kStreamRows = 16;  // rows up to which W is streamed in any case
constexpr int kTallCutCols = 256, kTallCutBytes = 128;  // a tall tile's columns, its bytes of K per pair of steps

// Tiles of 32 * fm rows, their K cut over `splits` workgroups: the cut that takes least time by this model, in units of 0.2 us
// (what a pair of steps of one block of rows takes in 16 bits; a tile's weights count as one block more): a round of up to 256
// tiles costs its pairs of steps and 20 for its beginning and end, a join 20 and the FP32 sums at 4 TB/s there and back.  f32
// takes eight times as long a pair.  4096 x 10240: 64 rows are cut (2, 5) and take 37 us, where one workgroup a tile would need
// 60; 1024 rows (6, 1), 240 tiles, where 160 of full height or 320 of half of it need 115 to 121; 8192 rows (8, 1).
inline Project best_cut(int T, int d, int n, int size) {
    const int pairs = (int)(((long long)d * size + kTallCutBytes - 1) / kTallCutBytes), each = size == 4 ? 8 : 1;
    const long long cols = (n + kTallCutCols - 1) / kTallCutCols;
    Project best{Project::TALL, 8, 4, 1};
    double least = 0;
    for (int fm = 8; fm >= 2; --fm) {
        const long long tiles = (T + 32ll * fm - 1) / (32 * fm) * cols;
        for (int s = 1; s <= 8 && (s == 1 || (pairs >= 4 * s && tiles * s <= 512)); ++s) {
            const double rounds = (double)((tiles * s + 255) / 256);
            const double time = rounds * ((double)(fm + 1) * each * pairs / s + 20) + (s > 1 ? 20 + (double)s * T * n / 1e5 : 0);
            if (least == 0 || time < least) least = time, best.fm = fm, best.splits = s;
        }
    }
    return best;
}

// Up to 16 rows, and rows that are not whole 16-byte pieces: streams, W passing once per 16 to 64 rows.  The rows come through the
// caches, fm / fn of the weights' bytes, so as many weight rows per workgroup as leave at least 128 workgroups (64 rows by 10240
// x 4096: 16 weight rows 64 us, 64 of them 45).  With more rows, as long as tiles of 64 x 128 would leave compute units without
// work.
inline Project project_form(int T, int d, int n, int size, bool aligned) {
    if (aligned && T > kStreamRows) return best_cut(T, d, n, size);
    const long long row_tiles = (T + 63) / 64;
    auto stream = [](int fm, int fn) { return Project{Project::STREAM, fm, fn, 1}; };
    if (T <= 16) return stream(1, n >= 32 * 512 ? 2 : 1);
    if (T <= 32) return stream(2, n >= 32 * 128 ? 2 : 1);
    if (T <= 64 || row_tiles * ((n + 127) / 128) < 256)
        return stream(4, row_tiles * ((n + 63) / 64) >= 128 ? 4 : row_tiles * ((n + 31) / 32) >= 128 ? 2 : 1);
    return Project{Project::TILES, 4, 2, 1};
}

// ---------------------------------------------------------------- experts (experts_topk_run.h)
struct Experts {
    enum Kind { STREAM, TALL, TILES } kind;
    int blocks;     // STREAM: blocks of 16 rows a tile
    int tile_rows;
    bool mini;      // STREAM without a plan
    int max_tiles;  // row tiles there can be
};

constexpr int kMiniSlots = 64, kTallTileRows = 256, kSmallTileRows = 64;

// `aligned`: all rows are whole 16-byte pieces on 16-byte boundaries.  Tall tiles, if about as many as compute units can be
// expected (f32, whose small tiles are as fast while they last) or half; few rows per expert: tiles of 16 or 32 rows.
inline Experts experts_form(int slots, int E, int d, int h, int size, bool aligned) {
    const bool tall = aligned && (slots / kTallTileRows + std::min(E, slots) / 2) * (long long)((std::min(d, h) + kTallCutCols - 1) / kTallCutCols) >=
                                     (size == 4 ? 200 : 100);
    Experts f{};
    f.blocks = slots <= 4 * E ? 1 : slots <= (tall ? 8 : 16) * E ? 2 : 0;
    f.kind = f.blocks > 0 ? Experts::STREAM : tall ? Experts::TALL : Experts::TILES;
    f.mini = f.blocks > 0 && slots <= kMiniSlots;
    f.tile_rows = f.blocks > 0 ? 16 * f.blocks : tall ? kTallTileRows : kSmallTileRows;
    f.max_tiles = (f.mini ? 0 : slots / f.tile_rows) + std::min(E, slots);
    return f;
}

// Weight rows per workgroup of a streamed product, in blocks of 16: 64 (32 hidden columns of a gated product) where that leaves
// every compute unit two workgroups, down to 16 otherwise.
inline int stream_blocks(int max_tiles, int N, bool gated) {
    const long long blocks16 = (long long)max_tiles * ((N + 15) / 16) * (gated ? 2 : 1);
    return blocks16 >= 4 * 512 ? 4 : gated || blocks16 >= 2 * 512 ? 2 : 1;
}

}  // namespace forms
}  // namespace infmoe
