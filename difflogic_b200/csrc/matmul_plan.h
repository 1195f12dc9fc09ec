// How a matrix product is cut into tiles, and what it needs of memory: host code shared by the entry points.
#pragma once

#include "common.cuh"

namespace dl {

// What a caller wants of a plan (dl_matmul_choice), in the bits of a type above the lowest eight.  The plan depends on nothing but the
// arguments of a call, so that the one that asks for a workspace and the one that uses it make the same.
static inline int matmul_choice(int *type) {
    const int choice = *type >> 8;
    *type &= 0xff;
    return choice;
}

struct MatmulPlan {
    int columns;            // of a tile: 64 or 128, or 256 with two CTAs to a tile of 256 rows
    bool pair;
    int splits, steps_per_split;
    int64_t partial_bytes;  // of the sums of the splits; 0: one split
};

// Tiles of a matrix; symmetric: those that reach to or below the diagonal.
static inline int64_t tiles_of(int64_t m, int64_t n, int64_t rows, int64_t columns, bool symmetric) {
    const int64_t down = ceil_div(m, rows), across = ceil_div(n, columns);
    if (!symmetric) return down * across;
    int64_t tiles = 0;
    for (int64_t i = 0; i < down; ++i) {
        const int64_t c = ceil_div((i + 1) * rows, columns);
        tiles += c < across ? c : across;
    }
    return tiles;
}

// Clocks of one SM, fitted to measured times.  A step of 64 takes the longest of three: its products (128 x 16 by 64, 128 columns 32, 64
// clocks; a pair's 256 x 256 128); its copies, 60 bytes a clock; shared memory, which the products read and the copies write, 125 bytes a
// clock.  A tile ends with its epilogue, which the next tile's steps hide, the last one's do not; a join of splits costs a launch and
// moves the sums once more.  The cheapest of the tile widths and splits is taken.
static inline MatmulPlan plan_matmul(int64_t m, int64_t n, int64_t k, int64_t batch, int planes, bool symmetric, int sms, int choice) {
    MatmulPlan best = {};
    double best_clocks = 0;
    const int64_t steps = ceil_div(k, 64);
    const int products = planes == 1 ? 1 : planes == 2 ? 3 : 6;
    const int wanted = choice & 0x3ff, only_columns = wanted == 64 || wanted == 128 || wanted == 256 ? wanted : 0, only_splits = choice >> 10;
    for (int columns = 64; columns <= 256; columns *= 2) {
        const bool pair = columns == 256;
        if (only_columns > 0 ? columns != only_columns : columns > 64 && n <= columns / 2) continue;
        const int64_t per_matrix = tiles_of(m, n, pair ? 256 : 128, columns, symmetric);
        const int own = pair ? 128 : columns;   // columns' operands that a CTA copies and reads
        const double multiply = products * 2.0 * columns, copied = planes * (128 + own) * 128;
        const double copy = copied / 60, shared = (products * 4 * (128 + own) * 32 + copied) / 125;
        double step = multiply > copy ? multiply : copy;
        if (shared > step) step = shared;
        const double share = columns == 64 ? 32 : columns == 128 ? 64 : 128;   // columns of an epilogue warp
        const double end = 500 + share * (planes == 2 ? symmetric ? 110 : 80 : 70);
        for (int64_t splits = 1; splits <= 64 && (splits == 1 || steps / splits >= 4); splits += splits < 4 ? 1 : splits / 2) {
            const int64_t per = ceil_div(steps, splits), really = ceil_div(steps, per);
            if (really != splits || (only_splits > 0 && splits > only_splits)) continue;
            const int64_t tiles = per_matrix * batch * splits, waves = ceil_div(tiles, pair ? sms / 2 : sms);
            const int64_t partial = splits > 1 ? tiles * (pair ? 256 : 128) * columns * 4 : 0;
            if (partial > (int64_t)64 << 20) continue;
            const double tile = per * step, finish = splits > 1 ? 500 + share * 40 : end;
            double clocks = 6000 + tile + (waves - 1) * (tile > finish ? tile : finish) + finish;
            if (splits > 1) clocks += 8000 + partial / 1300.0;
            if (best.columns == 0 || clocks < best_clocks || (only_splits > 0 && splits > best.splits)) {
                best = {columns, pair, (int)splits, (int)per, partial};
                best_clocks = clocks;
            }
        }
    }
    return best;
}

}  // namespace dl
