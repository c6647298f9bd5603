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

// The tile with the least waves x cost of a step of K (64 columns, 0.01 us; of gemm_tile.h).  The groups' sizes are on the
// device; the rows are taken as spread evenly over the groups, half a tile of each lost.
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
    if (!f32) offer(256, 2, 34);
    else offer(128, 2, 20);
    if (!f32) offer(256, 1, 39);
    offer(128, 1, 22);
    offer(64, 1, 18);
    offer(32, 1, 15);
    return best;
}

}  // namespace sb
