// grouped.hpp -- shared by the grouped products: arguments and the tiles of
// ragged groups.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"
#include "device_utils.hpp"
#include "tinygnn_amd.h"

namespace tg {

constexpr int64_t kMaxGroups = 1024;

// Rows [offsets[g], offsets[g + 1]), whatever the offsets hold within [0, m].
__device__ __forceinline__ void group_rows(const int32_t* __restrict__ offsets, int g, int m,
                                           int* lo, int* hi) {
    const int a = offsets[g], b = offsets[g + 1];
    *lo = a < 0 ? 0 : a > m ? m : a;
    *hi = b < *lo ? *lo : b > m ? m : b;
}

// The tile of `unit` rows with number t over all groups, each cut from its own
// first row: its group and rows [*r0, *r1); false past the last.  Every
// wavefront finds it by itself, 64 groups at a time (offsets come from L2).
// offsets null: one group of all m rows.  `slot` (or null): the tile's number among
// those of groups of several.
__device__ __forceinline__ bool find_tile(const int32_t* __restrict__ offsets, int groups, int m,
                                          int unit, int t, int* g, int* r0, int* r1,
                                          int* slot = nullptr) {
    if (offsets == nullptr) {
        *g = 0;
        *r0 = t * unit;
        *r1 = m - *r0 > unit ? *r0 + unit : m;
        return *r0 < m;
    }
    const int lane = threadIdx.x & (kWave - 1);
    int slots = 0;
    for (int base = 0; base < groups; base += kWave) {
        int lo = 0, hi = 0;
        if (base + lane < groups) group_rows(offsets, base + lane, m, &lo, &hi);
        const int n = static_cast<int>((static_cast<int64_t>(hi) - lo + unit - 1) / unit);
        const int upto = wave_inclusive_scan(n);
        const int several = n > 1 ? n : 0;
        const int mine = slot ? wave_inclusive_scan(several) : 0;
        const uint64_t past = __ballot(upto > t);
        if (past) {
            const int w = __ffsll(static_cast<unsigned long long>(past)) - 1;
            const int first = __builtin_amdgcn_readlane(upto - n, w);
            const int a = __builtin_amdgcn_readlane(lo, w), b = __builtin_amdgcn_readlane(hi, w);
            *g = base + w;
            *r0 = a + (t - first) * unit;
            *r1 = b - *r0 > unit ? *r0 + unit : b;
            if (slot) *slot = slots + __builtin_amdgcn_readlane(mine - several, w) + t - first;
            return true;
        }
        if (slot) slots += __builtin_amdgcn_readlane(mine, kWave - 1);
        t -= __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    return false;
}

// Row tiles of `unit` rows of all groups.  (Their number decides which tiles an
// XCD takes: with the most that there can be instead, the last XCDs had only
// tiles that do not exist, and 256 tiles took two rounds of the 256 CUs.)  Falling
// offsets can name more rows than m, 512 times at most: the lanes' counts stop at
// 2^24, below which a launch's tiles are, and their sum is a whole number.
__device__ __forceinline__ int count_tiles(const int32_t* __restrict__ offsets, int groups, int m,
                                           int unit) {
    if (offsets == nullptr) return static_cast<int>((static_cast<int64_t>(m) + unit - 1) / unit);
    const int lane = threadIdx.x & (kWave - 1);
    int n = 0;
    for (int base = 0; base < groups; base += kWave) {
        int lo = 0, hi = 0;
        if (base + lane < groups) group_rows(offsets, base + lane, m, &lo, &hi);
        n += static_cast<int>((static_cast<int64_t>(hi) - lo + unit - 1) / unit);
    }
    return __builtin_amdgcn_readfirstlane(wave_sum(std::min(n, 1 << 24)));
}

// Most tiles of `unit` rows that m rows in `groups` groups can make.
inline int64_t most_tiles(int64_t m, int64_t groups, int64_t unit) {
    return m / unit + std::min(groups, m);
}

// exp(x) - 1 for x < 0 within a few units in the last place: its series near 0,
// where the difference loses digits (|x|^8 / 8! of 0.35 is below 2^-27 of x),
// else the difference (a size of 0.29 at least, and an exp off by 2^-24 of its
// own).  No branch and 14 instructions: the epilogues have 128 copies of it.
__device__ __forceinline__ float expm1_negative(float x) {
    float p = 1.0f / 40320.0f;
    p = __builtin_fmaf(p, x, 1.0f / 5040.0f);
    p = __builtin_fmaf(p, x, 1.0f / 720.0f);
    p = __builtin_fmaf(p, x, 1.0f / 120.0f);
    p = __builtin_fmaf(p, x, 1.0f / 24.0f);
    p = __builtin_fmaf(p, x, 1.0f / 6.0f);
    p = __builtin_fmaf(p, x, 0.5f);
    const float near = __builtin_fmaf(p * x, x, x);
    const float far = __expf(x) - 1.0f;
    return x > -0.35f ? near : far;
}

// x + bias, then TG_EPI_*.
template <int EPI>
__device__ __forceinline__ float grouped_epilogue(float x, float bias) {
    x += bias;
    if (EPI == TG_EPI_RELU) return 0.0f < x ? x : 0.0f;
    if (EPI == TG_EPI_ELU) return x < 0.0f ? expm1_negative(x) : x;
    return x;
}

// fn with the epilogue as a constant.
template <typename F>
__device__ __forceinline__ void with_epilogue(int epi, F&& fn) {
    if (epi == TG_EPI_RELU)
        fn(std::integral_constant<int, TG_EPI_RELU>{});
    else if (epi == TG_EPI_ELU)
        fn(std::integral_constant<int, TG_EPI_ELU>{});
    else
        fn(std::integral_constant<int, TG_EPI_NONE>{});
}

}  // namespace tg
