// linear.hpp -- arguments and plans of the dense layers' kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"
#include "types.hpp"

namespace tg {

struct LinearArgs {
    int m, n, k;  // results and contraction of this product
    const void* x;
    int64_t ldx;
    const void* w;
    int64_t ldw;
    const void* bias;
    int act;
    const void* residual;
    int64_t ldr;
    void* y;
    int64_t ldy;
    void* pre;
    int64_t ldp;
    uint32_t mt, nt;
    int unit;     // contraction of a part
    int parts;    // (join) whose sums stand at part
    bool more;    // (join) and others come: no results yet
    float* part;  // [kept parts][m][n], or null: one part, straight to y
};

struct ActArgs {
    int64_t m, n, rows;  // rows of a workgroup
    int log_wide;        // ... and 16-byte chunks of columns
    const void* dy;
    int64_t lddy;
    const void* pre;
    int64_t ldp;
    void* d;  // [m x ldd], or null
    int64_t ldd;
    float* part;  // [row parts][n], or null
};

struct LinearPlan {
    int64_t em, en;  // the tile
    int64_t mt, nt, unit, parts;
    int64_t kept;  // parts whose sums stand in the workspace at a time
    size_t bytes(int64_t m, int64_t n) const {
        return parts > 1 ? static_cast<size_t>(kept) * m * n * 4 : 0;
    }
};

// The launches of one element type: a product whose operands run across the
// contraction (ax, aw) or along it (p.em 0: of few rows, both along), d and its
// columns' sums by parts of rows, and the join of those.
template <typename T>
void linear_product(LinearArgs& a, const LinearPlan& p, bool ax, bool aw, bool direct,
                    hipStream_t s);
template <typename T>
void linear_act(const ActArgs& a, int act, hipStream_t s);
template <typename T>
void linear_columns(const float* part, int64_t n, int64_t parts, void* out, hipStream_t s);

}  // namespace tg
