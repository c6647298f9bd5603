// Products whose weights a row chooses, on tcgen05 tensor cores:
//   grouped:   out[i] = alpha act(s W_e x[rows[i]] + b_e)            for offsets[e] <= i < offsets[e + 1]
//   adapters:  out[i] = alpha act(W x[i] + U_a low[i] + b)           with the adapter a of row i, low = scale_a D_a x[i]
//
// One CTA per SM, warp-specialised like the shared product of gemm.cu: a TMA producer, an MMA issuer (128 rows x BN columns per
// CTA in tensor memory, two accumulators), eight epilogue warps (sixteen for pairs in e4m3).  What differs:
//   - The tiles are found on the device.  A tile belongs to one group: 128 consecutive rows of it per CTA (the last ones of a
//     group may be missing) times BN columns.  Every warp walks the offsets 128 groups at a time with a prefix sum over its
//     lanes, so no table of groups is kept and the host never learns the sizes.
//   - Rows picked by an index arrive by TMA gathers of four rows each, issued by four or eight warps from one elected
//     lane (from every lane by turns a gather takes ten times as long); a tile with few rows fetches only those.
//   - Rows leave through a swizzled slab per warp: 32 rows of one group by a TMA store (or reduce-add), which clips at column N;
//     the last rows of a group, behind which its neighbour's begin, results off the 16-byte boundaries, and the last columns where N
//     ends inside 16 bytes (the store clips at whole ones) by ordinary stores.
//   - The low-rank addition is K = rank more columns of the same product, accumulated in the same tensor memory, `low` against the
//     rows of U_a, as bf16 terms: two where the result is bf16 (an error of at most 2^-16 of |low| |U_a|, below the result's own rounding
//     even where the addition cancels in part; one term, 2^-8, takes 5 % less, 448 against 472 us for 52360 rows x 4096 x 1024 at rank
//     64 with two adapters a tile, but a row's numbers then depend on whether its call has more than 32 rows), three where it is stored in 32 bits (2^-24).
//     A tile may hold rows of several adapters: its MMAs run once for each, with the lanes of the other rows disabled, so that
//     nothing of one adapter (not even a NaN) reaches rows of another, and the shared weights are read once whatever the adapters.
//   - Up to 32 rows (live streams, as a rule each with an adapter of its own): an MMA per adapter would take longer than all of
//     K, so the addition is formed on CUDA cores by the four warps that stage `low` otherwise, in 32 bits, U_a on its way before
//     `low` is there, and the epilogue adds it (24 rows with as many adapters, rank 16, 1024 -> 4096: 14.8 -> 10.1 us,
//     and 7.1 us with A stages of 32 rows; 33 rows, by MMAs, 13.8 us).
//   - The tensor core adds into its accumulator by truncation, 1e-6 of the result at K = 1024 and 4.4e-6 at 4096 (measured).
//     Where the result is stored in 32 bits, it is collected in registers every 512 columns of K, rounded to nearest (4.7e-7 at
//     either K in bf16; every 256 columns: 2.5e-7, but 16384 x 1024 x 1024 then takes 48 us instead of 36, a handshake per segment.  e4m3:
//     13160 x 4096 x 1024 takes 95 us, 84 if collected every 1024 columns, where a product of a large value and small ones loses 2.7e-5
//     instead of 1.3e-5).
// Every wait on an mbarrier is bounded; when one runs out the kernel sets *error, drains, frees its tensor memory and returns.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "adapter_ids.cuh"
#include "gemm_tile.h"
#include "launch.cuh"
#include "rows.h"
#include "tc_ptx.cuh"

namespace sb {

namespace {

using namespace ptx;

constexpr int kBM = 128;
constexpr int kRowBytes = 128;  // of an operand row in a stage: one swizzle row
constexpr int kFewRows = 32, kFewPitch = kFewRows + 1;  // rows of the few-row forms; an odd pitch spreads both sides over the banks
constexpr int kSegmentCols = 512;  // columns of K between two collections of a 32-bit result

enum RowsMode : int { kGrouped = 0, kGathered = 1, kAdapters = 2, kFewAdapters = 3, kFewGathered = 4 };
constexpr bool rows_few(int mode) { return mode == kFewAdapters || mode == kFewGathered; }
constexpr bool rows_gathers(int mode) { return mode == kGathered || mode == kFewGathered; }

// Parts of a tile's columns, four epilogue warps (128 rows) each.  A pair's e4m3 tile is over in half the time, so its epilogue sets the
// pace: sixteen warps instead of eight (16384 x 4096 x 1024: 75 -> 71 us, gathered 84 -> 76, 16 groups 87 -> 84; their slabs take a
// stage, which costs 26000 x 1024 x 4096 1 %).  bf16 gains nothing by them.
constexpr int rows_parts(int bn, int ctas, bool fp8, bool f32) { return bn == 256 && ctas == 2 && fp8 && !f32 ? 4 : gemm_halves(bn); }

// CTAS = 2: a cluster of two CTAs on 256 rows x BN columns (tcgen05 cta_group::2); each stages its own 128 rows of A and its own
// half of the W rows.
template <int BN, int CTAS, bool FP8, int MODE, bool F32>
struct RCfg {
    static constexpr int kParts = rows_parts(BN, CTAS, FP8, F32), kEpiWarps = kParts == 4 ? 16 : 8;
    static constexpr int kPartCols = BN / kParts;
    static constexpr int kOutCols = F32 || kPartCols < 64 ? 32 : 64;  // that a warp sends off at a time
    static constexpr int kSlabBytes = 32 * 128;
    // Warps more where rows are picked (gathers) or have adapters (`low`): four, 32 rows each; two beside an epilogue that keeps 128
    // sums a thread in registers (168 registers for 12 warps, 144 for 14); eight for the gathers of bf16 results, which four warps only
    // just issue in a stage's time (16384 x 4096 x 1024: 111 -> 106 us, 8064 rows of 16 groups 73 -> 71), where registers allow.
    static constexpr int kAuxWarps = MODE == kGrouped ? 0 : (F32 && BN == 256 ? 2 : (MODE == kGathered && kEpiWarps == 8 && !F32 ? 8 : 4));
    static constexpr int kThreads = 32 * (2 + kEpiWarps + kAuxWarps);
    // The few-row forms stage 32 rows of A.  The MMA reads 128: the others are whatever lies behind, and so are their lanes of the
    // accumulator, which nobody reads.  What that saves goes into stages: narrow tiles are paced by the weights in flight
    // (24 rows with adapters, 1024 -> 4096: 10.1 -> 7.1 us, both kernels).
    static constexpr int kABytes = (rows_few(MODE) ? kFewRows : kBM) * kRowBytes;
    static constexpr int kBBytes = BN / CTAS * kRowBytes;
    static constexpr int kStageBytes = kABytes + kBBytes;
    // `low` of the tile's rows as an operand: blocks of 16 of its columns (32 bytes a row), four to an operand tile
    static constexpr int kTerms = F32 ? 3 : 2, kGroups = F32 ? 2 : 4;  // bf16 terms, blocks of columns that are held at once
    static constexpr int kLowBytes = MODE == kAdapters ? (kTerms * kGroups + 3) / 4 * kBM * kRowBytes
                                                       : (MODE == kFewAdapters ? (BN * kFewPitch * 4 + 1023) / 1024 * 1024 : 0);  // the addition, by column
    static constexpr int kColumnSets = kParts == 4 ? 1 : 2;  // by turns, where a stage does not go for it
    static constexpr int kColumnBytes = kColumnSets * (FP8 ? 2 : 1) * BN * 4;  // bias and column scales of a tile
    static constexpr int kIndexBytes = rows_gathers(MODE) ? kBM * 4 : 0;
    static constexpr int kBarBytes = 384;
    static constexpr int kFixedBytes = kLowBytes + kEpiWarps * kSlabBytes + kColumnBytes + kIndexBytes + kBarBytes;
    static constexpr int kStages = std::min((227 * 1024 - kFixedBytes) / kStageBytes, rows_few(MODE) ? 16 : 8);
    static constexpr int kSmemBytes = kStages * kStageBytes + kFixedBytes;
    static_assert(kLowBytes % 1024 == 0 && kStages >= 3 && 8 * (2 * kStages + 6) + 16 <= kBarBytes, "shared memory");
    static constexpr int kUps = kStageBytes / kBBytes;  // adapters' tiles of `up` in a stage
    static constexpr uint32_t kTmemCols = 2 * BN;
};

template <int BN, int CTAS, bool FP8>
__device__ __forceinline__ uint32_t rows_idesc() {
    const uint32_t fmt = FP8 ? 0u : 1u;  // e4m3 / bf16; fp32 accumulate, both operands K-major
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)((kBM * CTAS) >> 4) << 24);
}

// Four rows of the map (box one row high) to four consecutive 128-byte rows; CTAS = 2: `bar` is a shared::cluster address.
template <int CTAS>
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int r0, int r1, int r2, int r3) {
    if constexpr (CTAS == 2) {
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(r0), "r"(r1), "r"(r2), "r"(r3)
            : "memory");
    } else {
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(r0), "r"(r1), "r"(r2), "r"(r3)
            : "memory");
    }
}
template <int CTAS>
__device__ __forceinline__ void rows_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    if constexpr (CTAS == 2) tma_load_2d_pair(dst, map, bar, c0, c1);
    else tma_load_2d(dst, map, bar, c0, c1);
}
template <int CTAS, bool FP8>
__device__ __forceinline__ void rows_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CTAS == 2) tc_mma_pair<FP8>(d, a, b, idesc, accumulate);
    else tc_mma<FP8>(d, a, b, idesc, accumulate);
}
template <int CTAS>
__device__ __forceinline__ void rows_mma_lanes(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, const uint32_t (&off)[4 * CTAS]) {
    if constexpr (CTAS == 2) tc_mma_lanes_pair(d, a, b, idesc, off, 1u);
    else tc_mma_lanes(d, a, b, idesc, off, 1u);
}
template <int CTAS>
__device__ __forceinline__ void rows_commit(uint32_t bar) {
    if constexpr (CTAS == 2) tc_commit_both(bar);
    else tc_commit(bar);
}
// Bounded wait for a barrier on which the other CTA of the pair arrives after writing its shared memory.
template <int CTAS>
__device__ __forceinline__ bool rows_wait_pair(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    if constexpr (CTAS == 1) return mbar_wait(bar, parity, abort_flag);
    const long long t0 = clock64();
    while (true) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
        if (ok) return true;
        if (*abort_flag) return false;
        if (clock64() - t0 > kWaitCycles) {
            *abort_flag = 1;
            return false;
        }
    }
}

// The gathering warps go by a count of the stages that the producer has begun.  They do not wait on the barriers themselves: a
// warp without rows in a tile holds up nobody, could fall two turns of the ring behind, and would then wait for the parity of
// another turn.  (Arriving on every stage instead, across the pair, costs twice the product's time.)
__device__ __forceinline__ void rows_set_turn(uint32_t at, uint32_t n) {
    asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(at), "r"(n) : "memory");
}
__device__ __forceinline__ bool rows_wait_turn(uint32_t at, uint32_t n, volatile int* abort_flag) {
    const long long t0 = clock64();
    while (true) {
        uint32_t now;
        asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(now) : "r"(at) : "memory");
        if ((int32_t)(now - n) >= 0) return true;
        if (*abort_flag) return false;
        if (clock64() - t0 > kWaitCycles) {
            *abort_flag = 1;
            return false;
        }
    }
}

struct RowsParams {
    const int32_t* rows;
    const int32_t* offsets;
    const float* bias;
    const float* row_scale;
    const float* col_scale;
    void* out;
    int64_t a_rows, ldo;
    int M, N, K, n_groups, act, out_mode;
    float alpha;
    bool out_vec;    // output rows on 16-byte boundaries
    bool n_vec;      // and N columns end on one (a TMA store clips at column N in whole 16 bytes)
    // adapters
    const int32_t* row_adapter;
    const float* low;
    const void* up;
    int rank, n_adapters;
};

// A tile: rows [row0, row1) of the output, columns from col0, weights of group `group`.
struct RowsTile {
    int group, row0, row1, col0;
};

// Finds tile t.  All lanes of a warp call it together, with ascending t.  A lane holds kEach neighbouring groups.
template <int ROWS>
struct TileWalk {
    static constexpr int kEach = 4;
    const int32_t* offsets;
    int M, n_groups, n_tiles, lane;
    int first_group;      // of the groups that the lanes hold
    long long first_tile; // tiles of the groups before them
    int at[kEach + 1];    // this lane's groups: rows [at[j], at[j + 1]), ascending
    int own, upto;        // tiles of this lane's groups, of the lanes' up to and including this one
    int total;            // tiles of the groups that the lanes hold

    __device__ __forceinline__ TileWalk(const int32_t* off, int m, int groups, int nt, int ln)
        : offsets(off), M(m), n_groups(groups), n_tiles(nt), lane(ln), first_group(0), first_tile(0) {
        load();
    }
    __device__ __forceinline__ int tiles_of(int j) const { return (at[j + 1] - at[j] + ROWS - 1) / ROWS * n_tiles; }
    __device__ __forceinline__ void load() {
        const int g0 = first_group + kEach * lane;
        // whatever the offsets hold, rows stay inside [0, M), and a group behind the last one has none
#pragma unroll
        for (int j = 0; j <= kEach; ++j)
            at[j] = offsets ? min(max(__ldg(offsets + min(g0 + j, n_groups)), 0), M) : (g0 + j > 0 ? M : 0);
        own = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            at[j + 1] = max(at[j + 1], at[j]);
            own += tiles_of(j);
        }
        upto = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += v;
        }
        total = __shfl_sync(0xffffffffu, upto, 31);
    }
    __device__ __forceinline__ bool find(long long t, int bn, RowsTile& out) {
        while (t >= first_tile + total) {
            if (first_group + 32 * kEach >= n_groups) return false;
            first_tile += total;
            first_group += 32 * kEach;
            load();
        }
        const int r = (int)(t - first_tile);
        const int src = __ffs(__ballot_sync(0xffffffffu, upto > r)) - 1;
        int mine = r - (upto - own), j = 0, glo = at[0], ghi = at[1], skip = 0, before = 0;
#pragma unroll
        for (int i = 1; i < kEach; ++i) {
            before += tiles_of(i - 1);
            if (mine >= before) { j = i; glo = at[i]; ghi = at[i + 1]; skip = before; }
        }
        const int rest = __shfl_sync(0xffffffffu, mine - skip, src);
        glo = __shfl_sync(0xffffffffu, glo, src);
        ghi = __shfl_sync(0xffffffffu, ghi, src);
        out.group = first_group + kEach * src + __shfl_sync(0xffffffffu, j, src);
        const int mt = rest / n_tiles;
        out.row0 = glo + mt * ROWS;
        out.row1 = min(ghi, out.row0 + ROWS);
        out.col0 = (rest - mt * n_tiles) * bn;
        return true;
    }
};

// x sigmoid(x), its relative error a few 2^-22 on either side of 0 and 2^-23 |x| by the exponential's argument; 0 below -87, where the
// result is under 2^-118.  The exponential of -|x| does not overflow and the divisor lies in [1, 2].  (Through one tanh, x / 2 (1 + tanh),
// the sum cancels where x is negative: 1 % of the result at -4, 70 % at -8.  13160 rows x 4096 x 1024 took 80 us then and take 84, in
// e4m3 58 and 63.)
__device__ __forceinline__ float rows_silu(float x) {
    const float e = ex2_approx(-1.44269504f * fabsf(x));
    return (x < 0.0f ? x * e : x) * rcp_approx(1.0f + e);
}

// 32 accumulator columns -> scales, bias, activation.  bias, scale: of these columns, in shared memory.  (From global memory the
// same loads cost a trip to L2 every 32 columns even where they had been touched before: 28 us of 75 in a product of 16384 x 4096
// with K = 64; handed round by shuffles 7 us, but as many again for the scales.)
template <bool FP8, bool F32>
__device__ __forceinline__ void rows_finish(float (&x)[32], const RowsParams& p, const float4* bias, const float4* scale, float rs, bool known) {
    if (!known) {
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] = 0.0f;
    }
    if (FP8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float4 c = scale[j];
            x[4 * j] *= rs * c.x; x[4 * j + 1] *= rs * c.y; x[4 * j + 2] *= rs * c.z; x[4 * j + 3] *= rs * c.w;
        }
    }
    if (p.bias) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float4 b = bias[j];
            x[4 * j] += b.x; x[4 * j + 1] += b.y; x[4 * j + 2] += b.z; x[4 * j + 3] += b.w;
        }
    }
    if (p.act == kActSilu) {
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] = rows_silu(x[j]);
    } else if (p.act == kActRelu) {
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] = x[j] < 0.0f ? 0.0f : x[j];  // NaN stays
    }
}

// Stored, or added in memory as the TMA reduce does for whole boxes: no load to wait for (8064 rows of 16 groups x 1024 x 1024, 32-bit
// results added: 42 us with loads, 23 without).  An element is added to once.  Predicated: branches over the same two instructions cost
// 3 us of 11.5 at 2503 rows x 1030 x 640.
__device__ __forceinline__ void put(float* at, uint32_t v, int how) {  // 0: not at all, 1: stored, 2: added
    asm volatile(
        "{\n\t.reg .pred a, s;\n\tsetp.gt.s32 a, %2, 1;\n\tsetp.eq.s32 s, %2, 1;\n\t"
        "@a red.global.add.f32 [%0], %1;\n\t@s st.global.f32 [%0], %1;\n\t}" ::"l"(at),
        "f"(__uint_as_float(v)), "r"(how)
        : "memory");
}
__device__ __forceinline__ void put4(float* at, uint4 v, bool add) {
    asm volatile(
        "{\n\t.reg .pred a;\n\tsetp.ne.u32 a, %5, 0;\n\t"
        "@a red.global.add.v4.f32 [%0], {%1, %2, %3, %4};\n\t@!a st.global.v4.f32 [%0], {%1, %2, %3, %4};\n\t}" ::"l"(at),
        "f"(__uint_as_float(v.x)), "f"(__uint_as_float(v.y)), "f"(__uint_as_float(v.z)), "f"(__uint_as_float(v.w)), "r"((uint32_t)add)
        : "memory");
}

// The slab's 32 rows x COLS columns to memory, the rows below row1 and the columns below N.
template <typename T, int COLS>
__device__ __forceinline__ void rows_store(const unsigned char* slab, const RowsParams& p, int row0, int row1, int col0, int lane) {
    constexpr int kBytes = COLS * (int)sizeof(T), kChunks = kBytes / 16, kPer = 16 / (int)sizeof(T), kStep = 32 / kChunks;
    constexpr int kShift = kBytes == 64 ? 1 : 0, kMask = kChunks - 1;
    T* out = static_cast<T*>(p.out);
    const bool add = p.out_mode == kOutResidual;
    if (p.out_vec) {
        const int ch = lane % kChunks, col = col0 + ch * kPer;
#pragma unroll
        for (int i = 0; i < 32; i += kStep) {
            const int r = i + lane / kChunks;
            if (row0 + r >= row1 || col >= p.N) continue;
            const uint4 v = *reinterpret_cast<const uint4*>(slab + r * kBytes + ((ch ^ ((r >> kShift) & kMask)) << 4));
            T* dst = out + (int64_t)(row0 + r) * p.ldo + col;
            if (col + kPer <= p.N) {
                if constexpr (sizeof(T) == 4) put4(dst, v, add);
                else *reinterpret_cast<uint4*>(dst) = v;
            } else {
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    if (col + j >= p.N) break;
                    if constexpr (sizeof(T) == 4) put(dst + j, w[j], add ? 2 : 1);
                    else dst[j] = __ushort_as_bfloat16((unsigned short)(w[j / 2] >> (16 * (j & 1))));
                }
            }
        }
    } else {
        // eight rows' pieces out of the slab at once: a load that waits for the store before it costs 60 cycles a row
        const int rows = min(row1 - row0, 32);
        for (int r0 = 0; r0 < rows; r0 += 8) {
#pragma unroll
            for (int c = 0; c < COLS; c += 32) {
                const int cc = c + lane, byte = cc * (int)sizeof(T);
                T* dst = out + (int64_t)(row0 + r0) * p.ldo + col0 + cc;
                const bool in = col0 + cc < p.N;
                const int how = in ? (add ? 2 : 1) : 0;
                uint32_t v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = r0 + i;
                    const unsigned char* at = slab + r * kBytes + (((byte >> 4) ^ ((r >> kShift) & kMask)) << 4) + (byte & 15);
                    v[i] = sizeof(T) == 4 ? *reinterpret_cast<const uint32_t*>(at) : *reinterpret_cast<const unsigned short*>(at);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (sizeof(T) == 4) put(dst + i * p.ldo, v[i], r0 + i < rows ? how : 0);
                    else if (in && r0 + i < rows) dst[i * p.ldo] = __ushort_as_bfloat16((unsigned short)v[i]);
                }
            }
        }
    }
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}
// What rounding to bf16 leaves of v; nothing where that is not finite (inf - inf).
__device__ __forceinline__ float bf16_rest(float v) {
    const float d = v - __bfloat162float(__float2bfloat16_rn(v));
    return fabsf(d) < INFINITY ? d : 0.0f;
}

template <int BN, int CTAS, bool FP8, int MODE, bool F32>
__global__ void __launch_bounds__(RCfg<BN, CTAS, FP8, MODE, F32>::kThreads, 1)
rows_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_w,
            const __grid_constant__ CUtensorMap tma_up, const __grid_constant__ CUtensorMap tma_out, const RowsParams p,
            int* __restrict__ error) {
    using C = RCfg<BN, CTAS, FP8, MODE, F32>;
    constexpr int S = C::kStages;
    constexpr int kStepCols = FP8 ? 128 : 64, kSegment = kSegmentCols / kStepCols;
    constexpr int kTerms = C::kTerms, kGroups = C::kGroups, kPhaseCols = 16 * kGroups;
    constexpr int kEpiWarps = C::kEpiWarps, kAuxWarps = C::kAuxWarps;
    // rank of this CTA in its pair (the leader, rank 0, owns the barriers that the MMAs wait on)
    const uint32_t rank = CTAS == 2 ? __shfl_sync(0xffffffffu, cluster_ctarank(), 0) : 0u;
    extern __shared__ __align__(1024) unsigned char smem_dyn[];  // the operands' swizzle wants 1024-byte boundaries
    const uint32_t base = smem_u32(smem_dyn);
    unsigned char* base_ptr = smem_dyn;
    const uint32_t a_base = base, b_base = base + C::kABytes;  // of stage 0; a stage holds its A and its W side by side
    constexpr int kLowAt = S * C::kStageBytes, kSlabAt = kLowAt + C::kLowBytes, kColumnAt = kSlabAt + kEpiWarps * C::kSlabBytes;
    constexpr int kIndexAt = kColumnAt + C::kColumnBytes;
    constexpr int kBarAt = kIndexAt + C::kIndexBytes;
    const uint32_t bar_base = base + kBarAt;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (S + s); };
    auto tfull_bar = [&](int a) { return bar_base + 8u * (2 * S + a); };
    auto tempty_bar = [&](int a) { return bar_base + 8u * (2 * S + 2 + a); };
    const uint32_t low_bar = bar_base + 8u * (2 * S + 4);   // `low` of a tile is there
    const uint32_t lowfree_bar = bar_base + 8u * (2 * S + 5);  // and has been read
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base_ptr + kBarAt + 8 * (2 * S + 6));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const uint32_t turn_at = bar_base + 8u * (2 * S + 6) + 8;  // stages that the producer has begun, counted from the kernel's start
    // full barriers of the leader, as its own or as the pair's address
    auto lead = [&](uint32_t bar) { return CTAS == 2 ? mapa(bar, 0) : bar; };

    const int warp = warp_index(), lane = threadIdx.x & 31;
    const int n_tiles = (p.N + BN - 1) / BN;
    const int k_tiles = (p.K + kStepCols - 1) / kStepCols;
    const int phases = MODE == kAdapters ? (p.rank + kPhaseCols - 1) / kPhaseCols : 0;
    const long long tile0 = blockIdx.x / CTAS, tile_step = gridDim.x / CTAS;
    const int cta_row = (int)rank * kBM;

    if (base & 1023u) {  // dynamic shared memory begins on such a boundary where there is no static one
        if (threadIdx.x == 0) atomicExch(error, 1);
        return;
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), 4 * C::kParts * CTAS);
        }
        mbar_init(low_bar, std::max(kAuxWarps, 1) * CTAS);
        mbar_init(lowfree_bar, MODE == kFewAdapters ? C::kParts : 1);
        *abort_flag = 0;
        rows_set_turn(turn_at, 0);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (CTAS == 2) {
            tmem_alloc_pair(smem_u32(tmem_slot), C::kTmemCols);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CTAS == 2) cluster_sync();  // the peer's barriers exist before anything arrives on them
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_trigger();
    // The adapters' kernel ahead in the stream waits for everything before it and lets this one start after that: only what
    // it writes itself (low) has to be waited for here, by the warps that read it.
    constexpr bool kHasAdapters = MODE == kAdapters || MODE == kFewAdapters;
    if (!kHasAdapters) pdl_wait();
    constexpr int kTileRows = kBM * CTAS;

    TileWalk<kTileRows> walk(kHasAdapters ? nullptr : p.offsets, p.M, kHasAdapters ? 1 : p.n_groups, n_tiles, lane);
    RowsTile tile;

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        int stage = 0;
        uint32_t ph = 0, begun = 0;
        bool ok = true;
        for (long long t = tile0; ok && walk.find(t, BN, tile); t += tile_step) {
            const int w_col = tile.col0 + (int)rank * (BN / CTAS);
            const int w_row = tile.group * p.N + w_col;
            // bytes of A that the pair fetches: whole boxes, or the quads of rows that the gathers bring
            uint32_t a_bytes = CTAS * C::kABytes;
            if (rows_gathers(MODE)) {
                a_bytes = 0;
#pragma unroll
                for (int c = 0; c < CTAS; ++c) a_bytes += (uint32_t)((min(max(tile.row1 - tile.row0 - c * kBM, 0), kBM) + 3) >> 2) * (4 * kRowBytes);
            }
            AdapterIds<kTileRows> all;  // on their way while the shared columns of K are fetched
            if (MODE == kAdapters) all.load(p.row_adapter, p.n_adapters, tile.row0, tile.row1, lane);
            bool failed = false;
            if (elect_one()) {
                int s = stage;
                uint32_t sp = ph;
                for (int kt = 0; kt < k_tiles; ++kt) {
                    if (!mbar_wait(empty_bar(s), sp ^ 1, abort_flag)) { failed = true; break; }
                    if (rows_gathers(MODE)) rows_set_turn(turn_at, begun + (uint32_t)kt + 1);
                    if (rank == 0) mbar_expect_tx(full_bar(s), CTAS * C::kBBytes + a_bytes);
                    if (!rows_gathers(MODE))
                        rows_load<CTAS>(a_base + s * C::kStageBytes, &tma_a, lead(full_bar(s)), kt * kStepCols, tile.row0 + cta_row);
                    rows_load<CTAS>(b_base + s * C::kStageBytes, &tma_w, lead(full_bar(s)), kt * kStepCols, w_row);
                    if (++s == S) { s = 0; sp ^= 1; }
                }
            }
            ok = !__any_sync(0xffffffffu, failed);
            begun += k_tiles;
            stage += k_tiles;
            ph ^= (uint32_t)(stage / S) & 1u;
            stage %= S;
            if constexpr (MODE == kAdapters) {
                for (int c = 0; c < phases; ++c) {
                    AdapterIds<kTileRows> ids = all;
                    while (ok && ids.any()) {
                        int u_row[C::kUps], n = 0;
#pragma unroll
                        for (int u = 0; u < C::kUps; ++u) {
                            const int id = ids.next();
                            u_row[u] = id * p.N + w_col;
                            n += id >= 0;
                        }
                        ok = __all_sync(0xffffffffu, mbar_wait(empty_bar(stage), ph ^ 1, abort_flag));
                        if (!ok) break;
                        if (elect_one()) {
                            if (rank == 0) mbar_expect_tx(full_bar(stage), CTAS * C::kBBytes * n);
#pragma unroll
                            for (int u = 0; u < C::kUps; ++u)
                                if (u < n) rows_load<CTAS>(a_base + stage * C::kStageBytes + u * C::kBBytes, &tma_up, lead(full_bar(stage)), c * kPhaseCols, u_row[u]);
                        }
                        __syncwarp();
                        if (++stage == S) { stage = 0; ph ^= 1; }
                    }
                }
            }
        }
        if (!ok) {
            // copies already in flight land before the CTA exits
            const long long t0 = clock64();
            while (clock64() - t0 < 2000000) {}
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        const uint32_t idesc = rows_idesc<BN, CTAS, FP8>();
        int stage = 0;
        uint32_t ph = 0, seg = 0, low_ph = 0;
        bool ok = true;
        for (long long t = tile0; rank == 0 && ok && walk.find(t, BN, tile); t += tile_step) {
            AdapterIds<kTileRows> all;
            if (MODE == kAdapters) all.load(p.row_adapter, p.n_adapters, tile.row0, tile.row1, lane);
            int kt = 0;
            while (ok && kt < k_tiles) {
                const int acc = seg & 1;
                const uint32_t d_tmem = tmem_base + acc * BN;
                const int kt_end = F32 ? min(kt + kSegment, k_tiles) : k_tiles;
                const bool last = kt_end == k_tiles;
                bool failed = false;
                if (elect_one()) {
                    int s = stage;
                    uint32_t sp = ph;
                    if (!mbar_wait(tempty_bar(acc), ((seg >> 1) & 1) ^ 1, abort_flag)) failed = true;
                    tc_fence_after();
                    for (int k = kt; k < kt_end && !failed; ++k) {
                        if (!mbar_wait(full_bar(s), sp, abort_flag)) { failed = true; break; }
                        tc_fence_after();
                        const uint64_t adesc = make_smem_desc(a_base + s * C::kStageBytes), bdesc = make_smem_desc(b_base + s * C::kStageBytes);
#pragma unroll
                        for (int i = 0; i < 4; ++i) rows_mma<CTAS, FP8>(d_tmem, adesc + 2 * i, bdesc + 2 * i, idesc, (k > kt || i) ? 1u : 0u);
                        rows_commit<CTAS>(empty_bar(s));
                        if (++s == S) { s = 0; sp ^= 1; }
                    }
                    if (!failed && (MODE != kAdapters || !last)) rows_commit<CTAS>(tfull_bar(acc));
                }
                ok = !__any_sync(0xffffffffu, failed);
                stage += kt_end - kt;
                ph ^= (uint32_t)(stage / S) & 1u;
                stage %= S;
                if constexpr (MODE == kAdapters) {
                    if (ok && last) {
                        for (int c = 0; ok && c < phases; ++c) {
                            AdapterIds<kTileRows> ids = all;
                            if (!ids.any()) break;
                            ok = __all_sync(0xffffffffu, rows_wait_pair<CTAS>(low_bar, low_ph, abort_flag));
                            low_ph ^= 1;
                            const int groups = min(kGroups, (p.rank - c * kPhaseCols + 15) / 16);
                            while (ok && ids.any()) {
                                ok = __all_sync(0xffffffffu, mbar_wait(full_bar(stage), ph, abort_flag));
                                if (!ok) break;
                                tc_fence_after();
                                uint32_t off[C::kUps][4 * CTAS];  // lanes of other rows
                                int n = 0;
#pragma unroll
                                for (int u = 0; u < C::kUps; ++u) {
                                    n += ids.next(off[u]) >= 0;
#pragma unroll
                                    for (int q = 0; q < 4 * CTAS; ++q) off[u][q] = ~off[u][q];
                                }
                                if (elect_one()) {
                                    const uint64_t adesc = make_smem_desc(base + kLowAt), bdesc = make_smem_desc(a_base + stage * C::kStageBytes);
#pragma unroll
                                    for (int u = 0; u < C::kUps; ++u) {
                                        if (u >= n) break;
#pragma unroll
                                        for (int g = 0; g < kGroups; ++g) {
                                            if (g >= groups) break;
#pragma unroll
                                            for (int e = 0; e < kTerms; ++e) {
                                                constexpr int kTile = kBM * kRowBytes / 16;  // in the descriptor's 16-byte units
                                                const int at = g * kTerms + e;
                                                rows_mma_lanes<CTAS>(d_tmem, adesc + at / 4 * kTile + 2 * (at % 4), bdesc + u * (C::kBBytes / 16) + 2 * g, idesc,
                                                                     off[u]);
                                            }
                                        }
                                    }
                                    rows_commit<CTAS>(empty_bar(stage));
                                    if (!ids.any()) rows_commit<CTAS>(lowfree_bar);
                                }
                                __syncwarp();
                                if (++stage == S) { stage = 0; ph ^= 1; }
                            }
                        }
                        if (ok && elect_one()) rows_commit<CTAS>(tfull_bar(acc));
                        __syncwarp();
                    }
                }
                kt = kt_end;
                ++seg;
            }
        }
    } else if (warp < 2 + kEpiWarps) {
        // ------------------------------------------------------------ epilogue
        const int ew = warp - 2, quad = warp & 3, part = ew >> 2;
        unsigned char* slab = base_ptr + kSlabAt + ew * C::kSlabBytes;
        uint32_t seg = 0;
        bool ok = true;
        const int cbeg = part * C::kPartCols;
        float* columns = reinterpret_cast<float*>(base_ptr + kColumnAt) + cbeg;  // bias of this tile; the scales 2 BN further on
        // the four warps of a part bring in its columns' bias and scales, fetched a tile ahead
        float next_bias = 0.0f, next_scale = 1.0f;
        auto fetch_columns = [&](const RowsTile& at) {
            const int c = quad * 32 + lane, col = at.col0 + cbeg + c;
            const bool in = c < C::kPartCols && col < p.N;
            next_bias = p.bias && in ? __ldg(p.bias + (int64_t)at.group * p.N + col) : 0.0f;
            if (FP8) next_scale = p.col_scale && in ? __ldg(p.col_scale + (int64_t)at.group * p.N + col) : 1.0f;
        };
        static_assert(C::kPartCols <= 128, "a thread brings in one column");
        uint32_t tiles = 0;
        auto next_columns = [&]() { return reinterpret_cast<float*>(base_ptr + kColumnAt) + cbeg + (C::kColumnSets == 2 ? (tiles & 1) * BN : 0); };
        bool more = part < C::kParts && walk.find(tile0, BN, tile);
        RowsTile ahead;
        if (more) fetch_columns(tile);
        for (long long t = tile0; more; t += tile_step, tile = ahead, columns = next_columns()) {
            // Where a wait ran out in one of the four warps, all of them leave here.
            auto meet = [&]() {
                uint32_t all_ok;
                asm volatile(
                    "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %2, 0;\n\t"
                    "barrier.cta.red.and.pred p, %1, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                    : "=r"(all_ok)
                    : "r"(1 + part), "r"(ok ? 1u : 0u)
                    : "memory");
                ok = all_ok != 0;
            };
            if (C::kColumnSets == 1) meet();  // the tile before has been read (of two sets: the tile before the last, its readers met since)
            if (quad * 32 + lane < C::kPartCols) {
                columns[quad * 32 + lane] = next_bias;
                if (FP8) columns[C::kColumnSets * BN + quad * 32 + lane] = next_scale;
            }
            meet();
            if (!ok) break;
            more = walk.find(t + tile_step, BN, ahead);
            if (more) fetch_columns(ahead);
            const int row0 = tile.row0 + cta_row + quad * 32;  // of this warp
            const int row = row0 + lane;
            const bool live = row < tile.row1;
            int src = row;
            if (rows_gathers(MODE) && p.rows && live) src = __ldg(p.rows + row);
            const bool known = !rows_gathers(MODE) || (unsigned)src < (unsigned long long)p.a_rows;
            const float rs = FP8 && p.row_scale && live && known ? __ldg(p.row_scale + src) : 1.0f;
            const bool any = row0 < tile.row1;  // rows of this warp in the tile
            auto taddr = [&]() { return tmem_base + ((uint32_t)(quad * 32) << 16) + (seg & 1) * BN + cbeg; };
            auto release = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (CTAS == 2) mbar_arrive_cluster(mapa(tempty_bar(seg & 1), 0));
                    else mbar_arrive(tempty_bar(seg & 1));
                }
                ++seg;
            };
            const bool whole = p.out_vec && row0 + 32 <= tile.row1;  // 32 rows of this group: one TMA store
            const float* addition = reinterpret_cast<const float*>(base_ptr + kLowAt) + lane;  // of this row; columns kFewPitch apart
            if (MODE == kFewAdapters && any) {
                ok = __all_sync(0xffffffffu, mbar_wait(low_bar, tiles & 1, abort_flag));
                if (!ok) continue;
            }
            ++tiles;
            auto added = [&]() {
                __syncwarp();
                if (MODE == kFewAdapters && lane == 0) mbar_arrive(lowfree_bar);
            };
            auto ready = [&]() {  // the store before has read the slab
                if (elect_one()) bulk_wait_read0();
                __syncwarp();
            };
            auto leave = [&](int col0, int cols, auto&& store) {
                if (whole && (p.n_vec || col0 + cols <= p.N)) {
                    fence_proxy_async();
                    __syncwarp();
                    if (elect_one()) {
                        if (F32 && p.out_mode == kOutResidual) tma_reduce_add_2d(&tma_out, smem_u32(slab), col0, row0);
                        else tma_store_2d(&tma_out, smem_u32(slab), col0, row0);
                        bulk_commit();
                    }
                } else {
                    __syncwarp();
                    store();
                }
                __syncwarp();
            };
            if constexpr (F32) {
                constexpr int kCols = C::kPartCols;
                float sum[kCols];
#pragma unroll
                for (int j = 0; j < kCols; ++j) sum[j] = 0.0f;
                for (int kt = 0; kt < k_tiles; kt += kSegment) {
                    ok = __all_sync(0xffffffffu, mbar_wait(tfull_bar(seg & 1), (seg >> 1) & 1, abort_flag));
                    if (!ok) break;
                    tc_fence_after();
                    if (any) {
#pragma unroll
                        for (int c = 0; c < kCols; c += 32) {
                            uint32_t v[32];
                            tmem_ld32(taddr() + c, v);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; ++j) sum[c + j] += __uint_as_float(v[j]);
                        }
                    }
                    release();
                }
                if (!ok || !any) continue;
                if (MODE == kFewAdapters) {
#pragma unroll
                    for (int j = 0; j < kCols; ++j) sum[j] += addition[(cbeg + j) * kFewPitch];
                    added();
                }
#pragma unroll
                for (int c = 0; c < kCols; c += 32) {
                    const int col0 = tile.col0 + cbeg + c;
                    if (col0 >= p.N) break;
                    float x[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) x[j] = sum[c + j];
                    rows_finish<FP8, F32>(x, p, reinterpret_cast<const float4*>(columns + c), reinterpret_cast<const float4*>(columns + C::kColumnSets * BN + c), rs, known);
                    ready();
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        *reinterpret_cast<float4*>(slab + lane * 128 + ((q ^ (lane & 7)) << 4)) =
                            make_float4(p.alpha * x[4 * q], p.alpha * x[4 * q + 1], p.alpha * x[4 * q + 2], p.alpha * x[4 * q + 3]);
                    leave(col0, 32, [&]() { rows_store<float, 32>(slab, p, row0, tile.row1, col0, lane); });
                }
            } else {
                constexpr int kCols = C::kOutCols;
                constexpr int kShift = kCols == 32 ? 1 : 0, kMask = kCols / 8 - 1;
                ok = __all_sync(0xffffffffu, mbar_wait(tfull_bar(seg & 1), (seg >> 1) & 1, abort_flag));
                if (!ok) continue;
                tc_fence_after();
                bool held = true;
                if (any) {
#pragma unroll 1
                    for (int c = 0; c < C::kPartCols; c += kCols) {
                        const int col0 = tile.col0 + cbeg + c;
                        if (col0 >= p.N) break;
#pragma unroll
                        for (int sub = 0; sub < kCols / 32; ++sub) {
                            uint32_t v[32];
                            tmem_ld32(taddr() + c + 32 * sub, v);
                            tmem_wait_ld();
                            if (c + 32 * (sub + 1) >= C::kPartCols) {  // the accumulator is free for the tile after the next
                                release();
                                held = false;
                            }
                            float x[32];
#pragma unroll
                            for (int j = 0; j < 32; ++j) x[j] = __uint_as_float(v[j]);
                            if (MODE == kFewAdapters) {
#pragma unroll
                                for (int j = 0; j < 32; ++j) x[j] += addition[(cbeg + c + 32 * sub + j) * kFewPitch];
                            }
                            rows_finish<FP8, F32>(x, p, reinterpret_cast<const float4*>(columns + c + 32 * sub),
                                                  reinterpret_cast<const float4*>(columns + C::kColumnSets * BN + c + 32 * sub), rs, known);
                            if (sub == 0) ready();
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                *reinterpret_cast<uint4*>(slab + lane * (kCols * 2) + (((4 * sub + q) ^ ((lane >> kShift) & kMask)) << 4)) =
                                    make_uint4(pack_bf16(x[8 * q], x[8 * q + 1]), pack_bf16(x[8 * q + 2], x[8 * q + 3]),
                                               pack_bf16(x[8 * q + 4], x[8 * q + 5]), pack_bf16(x[8 * q + 6], x[8 * q + 7]));
                        }
                        leave(col0, kCols, [&]() { rows_store<__nv_bfloat16, kCols>(slab, p, row0, tile.row1, col0, lane); });
                    }
                }
                if (held) release();
                if (any) added();
            }
        }
        if (elect_one()) bulk_wait_all();
        __syncwarp();
    } else if constexpr (rows_gathers(MODE)) {
        // ------------------------------------------------------------ gathers, kGatherRows rows a warp
        constexpr int kGatherRows = kBM / kAuxWarps;
        const int gw = warp - 2 - kEpiWarps;
        int32_t* index = reinterpret_cast<int32_t*>(base_ptr + kIndexAt) + gw * kGatherRows;
        uint32_t begun = 0;
        bool ok = true;
        int next = 0;  // the index of this lane's row, fetched a tile ahead
        auto fetch_index = [&](const RowsTile& at) {
            const int i = min(at.row0 + cta_row + gw * kGatherRows + (lane % kGatherRows), at.row1 - 1);
            next = p.rows ? __ldg(p.rows + i) : i;
        };
        bool more = walk.find(tile0, BN, tile);
        RowsTile ahead;
        if (more) fetch_index(tile);
        for (long long t = tile0; ok && more; t += tile_step, tile = ahead, begun += k_tiles) {
            const int count = tile.row1 - (tile.row0 + cta_row + gw * kGatherRows), v = next;
            more = walk.find(t + tile_step, BN, ahead);
            if (more) fetch_index(ahead);
            if (count <= 0) continue;
            if (lane < kGatherRows) index[lane] = (unsigned)v < (unsigned long long)p.a_rows ? v : 0;
            __syncwarp();
            bool failed = false;
            if (elect_one()) {
                int4 r[kGatherRows / 4];
#pragma unroll
                for (int j = 0; j < kGatherRows / 4; ++j) r[j] = reinterpret_cast<const int4*>(index)[j];
                int s = (int)(begun % S);
                for (int kt = 0; kt < k_tiles; ++kt) {
                    if (!rows_wait_turn(turn_at, begun + (uint32_t)kt + 1, abort_flag)) { failed = true; break; }
                    const uint32_t dst = a_base + s * C::kStageBytes + gw * kGatherRows * kRowBytes, bar = lead(full_bar(s));
#pragma unroll
                    for (int j = 0; j < kGatherRows / 4; ++j)
                        if (4 * j < count) tma_gather4<CTAS>(dst + j * 4 * kRowBytes, &tma_a, bar, kt * kStepCols, r[j].x, r[j].y, r[j].z, r[j].w);
                    if (++s == S) s = 0;
                }
            }
            ok = !__any_sync(0xffffffffu, failed);
        }
        if (!ok) {
            const long long t0 = clock64();
            while (clock64() - t0 < 2000000) {}
        }
    } else if constexpr (MODE == kFewAdapters) {
        // ------------------------------------------------------------ the addition: a column a lane, every fourth row a warp
        const int w = warp - 2 - kEpiWarps;
        constexpr int kEach = kFewRows / kAuxWarps;
        float* addition = reinterpret_cast<float*>(base_ptr + kLowAt);
        const __nv_bfloat16* up = static_cast<const __nv_bfloat16*>(p.up);
        int ids[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int row = w + kAuxWarps * i;
            ids[i] = row < p.M ? __ldg(p.row_adapter + row) : -1;
        }
        uint32_t ph = 0;
        bool ok = true, waited = false;
        for (long long t = tile0; ok && walk.find(t, BN, tile); t += tile_step, ph ^= 1) {
            for (int c = 0; ok && c < BN; c += 32) {
                const int col = tile.col0 + c + lane;
                float acc[kEach];
#pragma unroll
                for (int i = 0; i < kEach; ++i) acc[i] = 0.0f;
                for (int r = 0; r < p.rank; r += 8) {
                    uint4 u[kEach];
#pragma unroll
                    for (int i = 0; i < kEach; ++i) {
                        u[i] = make_uint4(0, 0, 0, 0);
                        if ((unsigned)ids[i] < (unsigned)p.n_adapters && col < p.N)
                            u[i] = __ldg(reinterpret_cast<const uint4*>(up + ((int64_t)ids[i] * p.N + col) * p.rank + r));
                    }
                    if (!waited) { pdl_wait(); waited = true; }
                    // a row without an adapter has zeros in `low`, one beyond M borrows the last one's; no branches between the loads
                    float4 x[kEach], y[kEach];
#pragma unroll
                    for (int i = 0; i < kEach; ++i) {
                        const float4* low = reinterpret_cast<const float4*>(p.low + (int64_t)min(w + kAuxWarps * i, p.M - 1) * p.rank + r);
                        x[i] = low[0];
                        y[i] = low[1];
                    }
#pragma unroll
                    for (int i = 0; i < kEach; ++i) {
                        auto part = [](float a, float b, uint32_t v, float s) {
                            return fmaf(b, __uint_as_float(v & 0xffff0000u), fmaf(a, __uint_as_float(v << 16), s));
                        };
                        acc[i] = part(y[i].z, y[i].w, u[i].w, part(y[i].x, y[i].y, u[i].z, part(x[i].z, x[i].w, u[i].y, part(x[i].x, x[i].y, u[i].x, acc[i]))));
                    }
                }
                if (c == 0) ok = __all_sync(0xffffffffu, mbar_wait(lowfree_bar, ph ^ 1, abort_flag));
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < kEach; ++i) addition[(c + lane) * kFewPitch + w + kAuxWarps * i] = acc[i];
            }
            __syncwarp();
            if (ok && lane == 0) mbar_arrive(low_bar);
        }
    } else if constexpr (MODE == kAdapters) {
        // ------------------------------------------------------------ `low` of the tile's rows as an operand, a row per thread at a time
        const int r0 = (warp - 2 - kEpiWarps) * 32 + lane;
        uint32_t ph = 0;
        bool ok = true;
        pdl_wait();
        for (long long t = tile0; ok && walk.find(t, BN, tile); t += tile_step) {
            AdapterIds<kTileRows> ids;
            ids.load(p.row_adapter, p.n_adapters, tile.row0, tile.row1, lane);
            if (!ids.any()) continue;
            for (int c = 0; ok && c < phases; ++c) {
#pragma unroll 1
                for (int r = r0; r < kBM; r += 32 * kAuxWarps) {
                    const int row = tile.row0 + cta_row + r;
                    unsigned char* dst = base_ptr + kLowAt + r * kRowBytes;
                    float f[kPhaseCols];
#pragma unroll
                    for (int i = 0; i < kPhaseCols; i += 4) {
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (row < tile.row1 && c * kPhaseCols + i < p.rank)
                            v = *reinterpret_cast<const float4*>(p.low + (int64_t)row * p.rank + c * kPhaseCols + i);
                        f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
                    }
                    if (r == r0) ok = __all_sync(0xffffffffu, mbar_wait(lowfree_bar, ph ^ 1, abort_flag));
                    if (!ok) break;
#pragma unroll
                    for (int g = 0; g < kGroups; ++g)
#pragma unroll
                        for (int e = 0; e < kTerms; ++e) {
                            uint32_t w[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                float& x = f[16 * g + 2 * i];
                                float& y = f[16 * g + 2 * i + 1];
                                w[i] = pack_bf16(x, y);
                                x = bf16_rest(x);
                                y = bf16_rest(y);
                            }
                            const int at = g * kTerms + e, chunk = 2 * (at % 4);
                            unsigned char* d = dst + at / 4 * kBM * kRowBytes;
                            *reinterpret_cast<uint4*>(d + ((chunk ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                            *reinterpret_cast<uint4*>(d + (((chunk + 1) ^ (r & 7)) << 4)) = make_uint4(w[4], w[5], w[6], w[7]);
                        }
                }
                if (!ok) break;
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (CTAS == 2) mbar_arrive_cluster(mapa(low_bar, 0));
                    else mbar_arrive(low_bar);
                }
                ph ^= 1;
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if constexpr (CTAS == 2) cluster_sync();  // neither CTA leaves while the other may still touch its memory
    if (warp == 1) {
        tc_fence_after();
        if constexpr (CTAS == 2) tmem_dealloc_pair(tmem_base, C::kTmemCols);
        else tmem_dealloc(tmem_base, C::kTmemCols);
    }
    if (threadIdx.x == 0 && *abort_flag) atomicExch(error, 1);
}

template <int BN, int CTAS, bool FP8, int MODE, bool F32>
cudaError_t rows_launch_t(const RowsArgs& g, int sm_count, int* d_error, cudaStream_t stream) {
    alignas(64) CUtensorMap ma, mw, mu, mo;
    if (!rows_map(&ma, g.a, g.a_rows, g.K, g.lda, FP8, rows_gathers(MODE) ? 1 : RCfg<BN, CTAS, FP8, MODE, F32>::kABytes / kRowBytes) ||
        !rows_map(&mw, g.w, (int64_t)g.n_groups * g.N, g.K, g.K, FP8, BN / CTAS))
        return cudaErrorInvalidValue;
    mu = mw;
    if (MODE == kAdapters && !rows_map(&mu, g.up, (int64_t)g.n_adapters * g.N, g.rank, g.rank, false, BN / CTAS)) return cudaErrorInvalidValue;
    const int eb = F32 ? 4 : 2;
    RowsParams p{};
    p.rows = g.rows; p.offsets = g.offsets; p.bias = g.bias; p.row_scale = g.row_scale; p.col_scale = g.col_scale; p.out = g.out;
    p.a_rows = g.a_rows; p.ldo = g.ldo; p.M = g.M; p.N = g.N; p.K = g.K; p.n_groups = g.n_groups; p.act = g.act; p.out_mode = g.out_mode;
    p.alpha = g.alpha;
    p.out_vec = !(reinterpret_cast<uintptr_t>(g.out) & 15) && !((g.ldo * eb) & 15);
    p.n_vec = (int64_t)g.N * eb % 16 == 0;
    mo = mw;  // stores by TMA want 32 rows of a group
    if (p.out_vec && g.M >= 32 && !rows_out_map(&mo, g.out, g.M, g.N, g.ldo, F32, F32 || RCfg<BN, CTAS, FP8, MODE, F32>::kOutCols == 64 ? 128 : 64)) return cudaErrorInvalidValue;
    p.row_adapter = g.row_adapter; p.low = g.low; p.up = g.up; p.rank = g.rank; p.n_adapters = g.n_adapters;
    // at most this many tiles: a group's last one may be short
    const int64_t n_tiles = (g.N + BN - 1) / BN;
    const int64_t tiles = ((int64_t)(g.M + kBM * CTAS - 1) / (kBM * CTAS) + std::min(g.n_groups - 1, g.M)) * n_tiles;
    const int grid = CTAS * (int)std::min<int64_t>(tiles, sm_count / CTAS);
    return launch_pdl(rows_kernel<BN, CTAS, FP8, MODE, F32>, dim3(grid), RCfg<BN, CTAS, FP8, MODE, F32>::kThreads, RCfg<BN, CTAS, FP8, MODE, F32>::kSmemBytes, stream, CTAS, ma, mw, mu, mo, p,
                      d_error);
}

template <int BN, int CTAS, bool FP8, int MODE, bool F32>
cudaError_t rows_set() {
    return cudaFuncSetAttribute(rows_kernel<BN, CTAS, FP8, MODE, F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, RCfg<BN, CTAS, FP8, MODE, F32>::kSmemBytes);
}

// The tiles of one form of the product: columns per tile, CTAs per tile.  A 32-bit result keeps its sums in registers; 128 a thread
// leave no room for the gathering warps, so the widest tile of such rows has 128 columns.
template <bool FP8, int MODE>
cudaError_t rows_pick(const RowsArgs& g, RowsTileShape t, int sm_count, int* err, cudaStream_t st) {
    if constexpr (rows_few(MODE)) t.ctas = 1;
    if (g.out_mode != kOutBf16) {
        if constexpr (!rows_few(MODE) && !rows_gathers(MODE))
            if (t.ctas == 2) return rows_launch_t<256, 2, FP8, MODE, true>(g, sm_count, err, st);
        switch (t.bn) {
            case 32: return rows_launch_t<32, 1, FP8, MODE, true>(g, sm_count, err, st);
            case 64: return rows_launch_t<64, 1, FP8, MODE, true>(g, sm_count, err, st);
            default: return rows_launch_t<128, 1, FP8, MODE, true>(g, sm_count, err, st);
        }
    }
    if constexpr (!rows_few(MODE))
        if (t.ctas == 2) return rows_launch_t<256, 2, FP8, MODE, false>(g, sm_count, err, st);
    switch (t.bn) {
        case 32: return rows_launch_t<32, 1, FP8, MODE, false>(g, sm_count, err, st);
        case 64: return rows_launch_t<64, 1, FP8, MODE, false>(g, sm_count, err, st);
        case 128: return rows_launch_t<128, 1, FP8, MODE, false>(g, sm_count, err, st);
        default: return rows_launch_t<256, 1, FP8, MODE, false>(g, sm_count, err, st);
    }
}

template <bool FP8, int MODE>
cudaError_t rows_set_all() {
    const cudaError_t e[7] = {rows_set<32, 1, FP8, MODE, true>(),  rows_set<64, 1, FP8, MODE, true>(),   rows_set<128, 1, FP8, MODE, true>(),
                              rows_set<32, 1, FP8, MODE, false>(), rows_set<64, 1, FP8, MODE, false>(), rows_set<128, 1, FP8, MODE, false>(),
                              rows_set<256, 1, FP8, MODE, false>()};
    if constexpr (!rows_few(MODE)) {
        cudaError_t pair = rows_set<256, 2, FP8, MODE, false>();
        if constexpr (!rows_gathers(MODE))
            if (pair == cudaSuccess) pair = rows_set<256, 2, FP8, MODE, true>();
        if (pair != cudaSuccess) return pair;
    }
    for (cudaError_t x : e)
        if (x != cudaSuccess) return x;
    return cudaSuccess;
}

}  // namespace

}  // namespace sb
