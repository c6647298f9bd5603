// The adapters among the rows of a tile, found by a warp.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace sb {

// ROWS / 32 neighbouring rows a lane; next() gives the adapters in the order of their first rows, -1 after the last one.  All lanes
// of the warp call together.  Ids outside [0, n_adapters) are no adapters.
template <int ROWS>
struct AdapterIds {
    static constexpr int kPer = ROWS / 32;
    int ids[kPer];
    __device__ __forceinline__ void load(const int32_t* row_adapter, int n_adapters, int row0, int row1, int lane) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int r = row0 + kPer * lane + j;
            ids[j] = r < row1 ? __ldg(row_adapter + r) : -1;
            if ((unsigned)ids[j] >= (unsigned)n_adapters) ids[j] = -1;
        }
    }
    __device__ __forceinline__ int next() {
        int first = -1;
#pragma unroll
        for (int j = kPer - 1; j >= 0; --j)
            if (ids[j] >= 0) first = ids[j];
        const uint32_t have = __ballot_sync(0xffffffffu, first >= 0);
        if (!have) return -1;
        const int cur = __shfl_sync(0xffffffffu, first, __ffs(have) - 1);
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (ids[j] == cur) ids[j] = -1;
        return cur;
    }
};

}  // namespace sb
