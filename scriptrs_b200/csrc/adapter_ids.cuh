// The adapters among the rows of a tile, found by a warp.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace sb {

// Row 32 q + lane of the tile in ids[q]; next() gives the adapters in the order of their first rows, -1 after the last one, and the
// rows of each: the first row left names the adapter, ballots find its other rows.  All lanes of the warp call together.  Ids
// outside [0, n_adapters) are no adapters.
template <int ROWS>
struct AdapterIds {
    static constexpr int kWords = ROWS / 32;
    int ids[kWords];
    uint32_t left[kWords];  // rows whose adapter has not been given yet
    __device__ __forceinline__ void load(const int32_t* row_adapter, int n_adapters, int row0, int row1, int lane) {
#pragma unroll
        for (int q = 0; q < kWords; ++q) {
            const int r = row0 + 32 * q + lane;
            ids[q] = r < row1 ? __ldg(row_adapter + r) : -1;
        }
#pragma unroll
        for (int q = 0; q < kWords; ++q) {
            if ((unsigned)ids[q] >= (unsigned)n_adapters) ids[q] = -1;
            left[q] = __ballot_sync(0xffffffffu, ids[q] >= 0);
        }
    }
    __device__ __forceinline__ int next(uint32_t (&rows)[kWords]) {
        int held = -1;
        uint32_t word = 0;
#pragma unroll
        for (int q = kWords - 1; q >= 0; --q)
            if (left[q]) { held = ids[q]; word = left[q]; }
        const int id = __shfl_sync(0xffffffffu, held, __ffs(word) - 1);  // (held is -1 everywhere where nothing is left)
#pragma unroll
        for (int q = 0; q < kWords; ++q) {
            rows[q] = __ballot_sync(0xffffffffu, ids[q] == id);
            left[q] &= ~rows[q];
        }
        return id;
    }
    __device__ __forceinline__ int next() {
        uint32_t rows[kWords];
        return next(rows);
    }
    __device__ __forceinline__ bool any() const {
        uint32_t all = 0;
#pragma unroll
        for (int q = 0; q < kWords; ++q) all |= left[q];
        return all != 0;
    }
};

}  // namespace sb
