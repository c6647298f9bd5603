// Which tile a product of rows.cu takes.  Host arithmetic only (plain C++, no CUDA types), so that it can be swept without a GPU.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace sb {

// Columns of a tile (128 rows): the width with the least waves x cost of a step of K.  The groups' sizes are on the device;
// the rows are taken as spread evenly over the groups.
inline int rows_tile(int64_t M, int N, int n_groups, bool f32, int sm_count) {
    const int64_t groups = std::min<int64_t>(n_groups, M);
    const int64_t m_tiles = groups * ((M + groups * 128 - 1) / (groups * 128));
    const int widths[4] = {256, 128, 64, 32};
    const int cost[4] = {39, 22, 18, 15};  // of 64 columns of K, 0.01 us
    int best = 128;
    int64_t least = INT64_MAX;
    for (int i = f32 ? 1 : 0; i < 4; ++i) {
        const int64_t waves = (m_tiles * ((N + widths[i] - 1) / widths[i]) + sm_count - 1) / sm_count;
        if (waves * cost[i] < least) { least = waves * cost[i]; best = widths[i]; }
    }
    return best;
}

}  // namespace sb
