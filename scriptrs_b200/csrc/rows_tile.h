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
// registers, 64 a thread at most, hence 128 columns; a pair of CTAs on 256 x 128 of it gained nothing (33 against 32 us at 13160 x
// 1024 x 1024, 99 against 99 at 1024 x 4096) and lost with ragged groups (27 against 24).
// Measured, us, at 32 / 64 / 128 / 256 columns / pairs, bf16 results; rows (groups) x N x K:
//   128 (1) x 4096 x 1024    5.7 / 6.3 / 6.9 / 9.9 / 11.0       376 (1) x 4096 x 1024    11.1 / 9.5 / 7.6 / 10.7 / 11.6
//   1504 (1) x 4096 x 1024   32 / 21 / 15.3 / 17.1 / 17.1       13160 (1) x 4096 x 1024  228 / 130 / 99 / 89 / 79
//   8064 (16) x 4096 x 1024  165 / 101 / 79 / 71 / 67           8064 (16) x 1024 x 1024  48 / 29 / 21.5 / 19.8 / 23.6
//   2000 (32) x 4096 x 1024  121 / 68 / 53 / 53 / 59            64 (32) x 4096 x 1024    118 / 64 / 48 / 50 / 53
inline RowsTileShape rows_tile(int64_t M, int N, int n_groups, bool f32, int sm_count) {
    const int64_t groups = std::min<int64_t>(n_groups, M);
    RowsTileShape best{128, 1};
    int64_t least = INT64_MAX;
    auto offer = [&](int bn, int ctas, int cost) {
        const int64_t rows = 128 * ctas;
        const int64_t m_tiles = groups > 1 ? std::max(groups, (2 * M + groups * rows) / (2 * rows)) : (M + rows - 1) / rows;
        const int64_t slots = std::max(sm_count / ctas, 1);
        const int64_t waves = (m_tiles * ((N + bn - 1) / bn) + slots - 1) / slots;
        if (waves * cost < least) { least = waves * cost; best = {bn, ctas}; }
    };
    if (!f32) {
        offer(256, 2, 34);
        offer(256, 1, 39);
    }
    offer(128, 1, 22);
    offer(64, 1, 18);
    offer(32, 1, 15);
    return best;
}

}  // namespace sb
