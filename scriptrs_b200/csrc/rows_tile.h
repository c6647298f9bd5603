// Which tile a product of rows_kernel.cuh takes.  Host arithmetic only (plain C++, no CUDA types), so that it can be swept
// without a GPU.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace sb {

struct RowsTileShape {
    int bn;    // columns (128 rows per CTA)
    int ctas;  // 2: a pair of CTAs on 256 rows
};

// The tile with the least waves x cost of a step of K (64 columns, in 0.01 us; of gemm_tile.h).  The groups' sizes are on the
// device; the rows are taken as spread evenly over the groups, half a tile of each lost.  A result in 32 bits keeps its sums in
// registers: 128 columns, or a pair where no warps gather rows (`picked`).  The end of a pair's last tile, 128 columns a thread, is
// not hidden: a third of a wave more.  us, 128 columns / pairs, 32-bit results; rows (groups) x N x K:
//   2503 (8) x 1030 x 640    12.7 / 14.1     4000 (1) x 1024 x 1024   12.2 / 12.8     1504 (1) x 4096 x 1024    16.8 / 18.4
//   13160 (1) x 1024 x 1024  31.7 / 27.6     13160 (1) x 1024 x 4096   99 / 84        13160 (1) x 4096 x 1024   115 / 100
//   8064 (16) x 1024 x 1024  23.7 / 28.0     13160 (16) x 1024 x 1024  36.4 / 39.1    52360 (32) x 1024 x 4096  406 / 350
// Measured, us, at 32 / 64 / 128 / 256 columns / pairs, bf16 results with SiLU; rows (groups) x N x K:
//   128 (1) x 4096 x 1024    8.4 / 9.7 / 11.0 / 16.5 / 18.0     376 (1) x 4096 x 1024    17.0 / 15.0 / 12.1 / 17.3 / 18.3
//   1504 (1) x 4096 x 1024   48 / 31 / 22.5 / 26.4 / 26.2       13160 (1) x 4096 x 1024  354 / 162 / 109 / 101 / 91
//   8064 (16) x 4096 x 1024  179 / 102 / 75 / 69 / 69           8064 (16) x 1024 x 1024  47 / 30 / 22.3 / 21.0 / 25.3
//   2000 (32) x 4096 x 1024  113 / 65 / 53 / 53 / 61            64 (32) x 4096 x 1024    87 / 52 / 47 / 50 / 57
// e4m3, whose steps of K take half the time, by the same costs: 13160 (16) x 4096 x 1024 gathered 211 / 137 / 88 / 76 / 79, 13160 (1)
// 142 / 97 / 64 / 57 / 62: 5 to 8 % off the best.
inline RowsTileShape rows_tile(int64_t M, int N, int n_groups, bool f32, bool picked, int sm_count) {
    const int64_t groups = std::min<int64_t>(n_groups, M);
    RowsTileShape best{128, 1};
    int64_t least = INT64_MAX;
    auto offer = [&](int bn, int ctas, int cost, int end = 0) {
        const int64_t rows = 128 * ctas;
        const int64_t m_tiles = groups > 1 ? std::max(groups, (2 * M + groups * rows) / (2 * rows)) : (M + rows - 1) / rows;
        const int64_t slots = std::max(sm_count / ctas, 1);
        const int64_t waves = (m_tiles * ((N + bn - 1) / bn) + slots - 1) / slots;
        const int64_t all = waves * cost + end;
        if (all < least) { least = all; best = {bn, ctas}; }
    };
    if (!f32) {
        offer(256, 2, 34);
        offer(256, 1, 39);
    } else if (!picked) {
        offer(256, 2, 35, 10);
    }
    offer(128, 1, 22);
    offer(64, 1, 18);
    offer(32, 1, 15);
    return best;
}

}  // namespace sb
