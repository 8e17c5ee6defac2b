// norm.hip -- layer norm over rows, forward and backward.
//
// Forward: the row is held in registers, so x is read once: its sum, then the
// sum of squared deviations from the mean (no cancellation of large means),
// then the store.  Backward: dx needs two sums of a row (t and t * xh, t = dy *
// gamma); x and dy are read once, and the same values feed the columns' sums
// for dgamma and dbeta, which every workgroup keeps in registers over the rows
// that it walks and writes once, as one partial row; a second kernel adds the
// partials in order (no atomics: equal calls give equal bits).  Both are bound
// by HBM: 2 RC and 3 RC elements.
//
// A row is taken by as many threads as one 16-byte load of x each covers, 64
// (four rows a workgroup, no barrier) to 1,024, then by 1,024 with two or four
// loads each: forward up to 16,384 columns, backward up to 8,192.  Few registers, so
// many wavefronts a SIMD (16 values a thread kept the backward pass at two of
// them: 16,384 x 4,096 bf16 170 us against 105).  Wider rows are walked by 1,024
// threads, out of L2 after the first time.
#include "common.hpp"
#include "device_utils.hpp"
#include "types.hpp"

#include <string>

namespace tg {
namespace {

constexpr int kWideThreads = 1024;

struct NormArgs {
    int64_t rows, cols;
    const void* x;
    int64_t ldx;
    const void* gamma;
    const void* beta;
    int weight_f32;  // gamma, beta and their gradients are floats, else T
    float eps;
    void* y;
    int64_t ldy;
    float* mean;
    float* rstd;
    // backward
    const void* dy;
    int64_t lddy;
    void* dx;
    int64_t lddx;
    float* part;  // [gridDim.x][2][cols], or null
};

// N weights from column c on as floats; `none` for missing weights.
template <typename T, int N>
__device__ __forceinline__ void load_weights(const void* w, int f32, int64_t c, int64_t cols,
                                             float none, float (&v)[N]) {
    if (w == nullptr) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = none;
    } else if (f32) {
        load_floats<float, N>(static_cast<const float*>(w) + c, cols - c, v);
    } else {
        load_floats<T, N>(static_cast<const T*>(w) + c, cols - c, v);
    }
}

// Sum over the TPR threads of a row, to all of them; for TPR > 64 through `lds`,
// the row's own, and a barrier that the whole workgroup joins (one before the
// next use of lds is the caller's: two buffers alternate).
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*lds)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    if constexpr (TPR > kWave) {
        const int wave = threadIdx.x % TPR / kWave;
        if ((threadIdx.x & (kWave - 1)) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) lds[wave][i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < TPR / kWave; ++w) s += lds[w][i];
            v[i] = s;
        }
    }
}

template <typename T, int TPR, int ITEMS>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_kernel(NormArgs a) {
    constexpr int VEC = kVec<T>, RPB = TPR > 256 ? 1 : 256 / TPR;
    __shared__ float lds[2][RPB][TPR / kWave][1];
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * RPB + sub;
    const int64_t row = at < a.rows ? at : a.rows - 1;  // again, for the barriers
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    float v[ITEMS][VEC];
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int64_t c = static_cast<int64_t>(i * TPR + lane) * VEC;
        load_floats<T, VEC>(x + c, a.cols - c, v[i]);
#pragma unroll
        for (int u = 0; u < VEC; ++u) s[0] += v[i][u];
    }
    row_sums<TPR>(s, lds[0][sub]);
    const float n = static_cast<float>(a.cols);
    const float mean = s[0] / n;
    float q[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int64_t c = static_cast<int64_t>(i * TPR + lane) * VEC;
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
            const float d = v[i][u] - mean;
            v[i][u] = d;
            if (c + u < a.cols) q[0] = __builtin_fmaf(d, d, q[0]);
        }
    }
    row_sums<TPR>(q, lds[1][sub]);
    if (at >= a.rows) return;
    const float rstd = 1.0f / sqrtf(q[0] / n + a.eps);
    if (lane == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.ldy;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int64_t c = static_cast<int64_t>(i * TPR + lane) * VEC;
        if (c >= a.cols) break;
        float g[VEC], b[VEC];
        load_weights<T, VEC>(a.gamma, a.weight_f32, c, a.cols, 1.0f, g);
        load_weights<T, VEC>(a.beta, a.weight_f32, c, a.cols, 0.0f, b);
#pragma unroll
        for (int u = 0; u < VEC; ++u) v[i][u] = __builtin_fmaf(v[i][u] * rstd, g[u], b[u]);
        store_floats<T, VEC>(y + c, a.cols - c, v[i]);
    }
}

// Rows of any width: the workgroup walks the row three times.
template <typename T>
__global__ __launch_bounds__(kWideThreads) void norm_wide_kernel(NormArgs a) {
    constexpr int VEC = kVec<T>;
    __shared__ float lds[2][kWideThreads / kWave][1];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const float n = static_cast<float>(a.cols);
    float v[VEC];
    float s[1] = {0.0f}, q[1] = {0.0f};
    for (int64_t c = threadIdx.x * VEC; c < a.cols; c += kWideThreads * VEC) {
        load_floats<T, VEC>(x + c, a.cols - c, v);
#pragma unroll
        for (int u = 0; u < VEC; ++u) s[0] += v[u];
    }
    row_sums<kWideThreads>(s, lds[0]);
    const float mean = s[0] / n;
    for (int64_t c = threadIdx.x * VEC; c < a.cols; c += kWideThreads * VEC) {
        load_floats<T, VEC>(x + c, a.cols - c, v);
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
            const float d = v[u] - mean;
            if (c + u < a.cols) q[0] = __builtin_fmaf(d, d, q[0]);
        }
    }
    row_sums<kWideThreads>(q, lds[1]);
    const float rstd = 1.0f / sqrtf(q[0] / n + a.eps);
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.ldy;
    for (int64_t c = threadIdx.x * VEC; c < a.cols; c += kWideThreads * VEC) {
        float g[VEC], b[VEC];
        load_floats<T, VEC>(x + c, a.cols - c, v);
        load_weights<T, VEC>(a.gamma, a.weight_f32, c, a.cols, 1.0f, g);
        load_weights<T, VEC>(a.beta, a.weight_f32, c, a.cols, 0.0f, b);
#pragma unroll
        for (int u = 0; u < VEC; ++u) v[u] = __builtin_fmaf((v[u] - mean) * rstd, g[u], b[u]);
        store_floats<T, VEC>(y + c, a.cols - c, v);
    }
}

// The backward pass of rows b, b + B, ... for workgroup (or, TPR = 64, a
// quarter of one) b of B; the next row is loaded while this one is summed.
template <typename T, int TPR, int ITEMS>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_backward_kernel(NormArgs a) {
    constexpr int VEC = kVec<T>, RPB = TPR > 256 ? 1 : 256 / TPR;
    __shared__ float lds[2][RPB][TPR / kWave][2];
    __shared__ float sums[RPB > 1 ? RPB : 1][RPB > 1 ? TPR * ITEMS * VEC : 1];
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const int64_t step = static_cast<int64_t>(gridDim.x) * RPB;
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.dy);
    const float n = static_cast<float>(a.cols);
    float g[ITEMS][VEC], dg[ITEMS][VEC] = {}, db[ITEMS][VEC] = {};
    float xv[ITEMS][VEC], dv[ITEMS][VEC], mean = 0.0f, rstd = 0.0f;
    auto fetch = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int64_t c = static_cast<int64_t>(i * TPR + lane) * VEC;
            load_floats<T, VEC>(x + row * a.ldx + c, a.cols - c, xv[i]);
            load_floats<T, VEC>(dy + row * a.lddy + c, a.cols - c, dv[i]);
        }
        mean = a.mean[row];
        rstd = a.rstd[row];
    };
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int64_t c = static_cast<int64_t>(i * TPR + lane) * VEC;
        load_weights<T, VEC>(a.gamma, a.weight_f32, c, a.cols, 1.0f, g[i]);
    }
    int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + sub;
    int64_t first = row - sub;  // the workgroup's; rows past the last join its barriers
    if (row < a.rows) fetch(row);
    for (int buf = 0; first < a.rows; first += step, row += step, buf ^= 1) {
        const bool in = row < a.rows;
        float t[ITEMS][VEC], xh[ITEMS][VEC];
        float s[2] = {0.0f, 0.0f};
        const float r = rstd;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int64_t c = static_cast<int64_t>(i * TPR + lane) * VEC;
#pragma unroll
            for (int u = 0; u < VEC; ++u) {
                // past the row's end dy and g are 0, and so are the sums' terms
                const float d = in ? dv[i][u] : 0.0f;
                xh[i][u] = in && c + u < a.cols ? (xv[i][u] - mean) * r : 0.0f;
                t[i][u] = d * g[i][u];
                s[0] += t[i][u];
                s[1] = __builtin_fmaf(t[i][u], xh[i][u], s[1]);
                dg[i][u] = __builtin_fmaf(d, xh[i][u], dg[i][u]);
                db[i][u] += d;
            }
        }
        if (row + step < a.rows) fetch(row + step);
        row_sums<TPR>(s, lds[buf][sub]);
        if (a.dx == nullptr || !in) continue;
        const float m0 = s[0] / n, m1 = s[1] / n;
        T* dx = static_cast<T*>(a.dx) + row * a.lddx;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int64_t c = static_cast<int64_t>(i * TPR + lane) * VEC;
            if (c >= a.cols) break;
#pragma unroll
            for (int u = 0; u < VEC; ++u)
                t[i][u] = r * (t[i][u] - __builtin_fmaf(xh[i][u], m1, m0));
            store_floats<T, VEC>(dx + c, a.cols - c, t[i]);
        }
    }
    if (a.part == nullptr) return;
    float* out = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float(&v)[ITEMS][VEC] = which ? db : dg;
        if constexpr (RPB > 1) {  // the workgroup's rows, in order
            __syncthreads();
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                for (int u = 0; u < VEC; ++u) sums[sub][(i * TPR + lane) * VEC + u] = v[i][u];
            __syncthreads();
            for (int64_t c = threadIdx.x; c < a.cols; c += 256) {
                float z = 0.0f;
#pragma unroll
                for (int w = 0; w < RPB; ++w) z += sums[w][c];
                out[which * a.cols + c] = z;
            }
        } else {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int64_t c = static_cast<int64_t>(i * TPR + lane) * VEC;
                store_floats<float, VEC>(out + which * a.cols + c, a.cols - c, v[i]);
            }
        }
    }
}

// Rows of any width: twice over the row, the columns' sums in the workgroup's
// own partial row in memory (each element is one thread's).
template <typename T>
__global__ __launch_bounds__(kWideThreads) void norm_backward_wide_kernel(NormArgs a) {
    constexpr int VEC = kVec<T>;
    __shared__ float lds[2][kWideThreads / kWave][2];
    float* part = a.part ? a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.cols : nullptr;
    const float n = static_cast<float>(a.cols);
    int buf = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, buf ^= 1) {
        const T* x = static_cast<const T*>(a.x) + row * a.ldx;
        const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
        const float mean = a.mean[row], r = a.rstd[row];
        const bool first = row == blockIdx.x;
        float xv[VEC], dv[VEC], g[VEC];
        float s[2] = {0.0f, 0.0f};
        for (int64_t c = threadIdx.x * VEC; c < a.cols; c += kWideThreads * VEC) {
            load_floats<T, VEC>(x + c, a.cols - c, xv);
            load_floats<T, VEC>(dy + c, a.cols - c, dv);
            load_weights<T, VEC>(a.gamma, a.weight_f32, c, a.cols, 1.0f, g);
            float dg[VEC] = {}, db[VEC] = {};
            if (part && !first) {
                load_floats<float, VEC>(part + c, a.cols - c, dg);
                load_floats<float, VEC>(part + a.cols + c, a.cols - c, db);
            }
#pragma unroll
            for (int u = 0; u < VEC; ++u) {
                if (c + u >= a.cols) break;
                const float xh = (xv[u] - mean) * r, t = dv[u] * g[u];
                s[0] += t;
                s[1] = __builtin_fmaf(t, xh, s[1]);
                dg[u] = __builtin_fmaf(dv[u], xh, dg[u]);
                db[u] += dv[u];
            }
            if (part) {
                store_floats<float, VEC>(part + c, a.cols - c, dg);
                store_floats<float, VEC>(part + a.cols + c, a.cols - c, db);
            }
        }
        row_sums<kWideThreads>(s, lds[buf]);
        if (a.dx == nullptr) continue;
        const float m0 = s[0] / n, m1 = s[1] / n;
        T* dx = static_cast<T*>(a.dx) + row * a.lddx;
        for (int64_t c = threadIdx.x * VEC; c < a.cols; c += kWideThreads * VEC) {
            load_floats<T, VEC>(x + c, a.cols - c, xv);
            load_floats<T, VEC>(dy + c, a.cols - c, dv);
            load_weights<T, VEC>(a.gamma, a.weight_f32, c, a.cols, 1.0f, g);
#pragma unroll
            for (int u = 0; u < VEC; ++u)
                dv[u] = r * (dv[u] * g[u] - __builtin_fmaf((xv[u] - mean) * r, m1, m0));
            store_floats<T, VEC>(dx + c, a.cols - c, dv);
        }
    }
}

// dgamma and dbeta: the `parts` partial rows added in order by 16 threads a
// column (consecutive shares), their sums in order.
template <typename T>
__global__ __launch_bounds__(1024) void norm_reduce_kernel(const float* __restrict__ part,
                                                           int64_t parts, int64_t cols,
                                                           void* dgamma, void* dbeta, int f32) {
    __shared__ float lds[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = (static_cast<int64_t>(blockIdx.z) * gridDim.x + blockIdx.x) * 64 + lane;
    const int which = blockIdx.y;
    const int64_t share = (parts + 15) / 16;
    const int64_t lo = w * share, hi = lo + share < parts ? lo + share : parts;
    float s = 0.0f;
    if (c < cols) {
        const float* p = part + which * cols + c;
#pragma unroll 8
        for (int64_t i = lo; i < hi; ++i) s += p[i * 2 * cols];
    }
    lds[w][lane] = s;
    __syncthreads();
    void* out = which ? dbeta : dgamma;
    if (w == 0 && c < cols && out) {
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) z += lds[i][lane];
        if (f32)
            static_cast<float*>(out)[c] = z;
        else
            static_cast<T*>(out)[c] = static_cast<T>(z);
    }
}

// Threads of a row and 16-byte loads of each (0: rows that are walked).
struct RowShape {
    int threads, items;
};

RowShape row_shape(int64_t cols, int type) {
    const int64_t loads = ceil_div(cols, 16 / type_size(type));
    for (int t = 64; t < 1024; t *= 2)
        if (loads <= t) return {t, 1};
    const int items = loads <= 1024 ? 1 : loads <= 2048 ? 2 : 4;
    return {1024, cols > 16384 ? 0 : items};
}

// The backward pass holds a thread's values of x and dy, of the next row's, of
// gamma and of two sums: up to 8 of each in registers (16 spilled), wider rows are
// walked.
constexpr int kBackwardValues = 8;

bool in_registers(RowShape r, int type) {
    return r.items > 0 && r.items * 16 / type_size(type) <= kBackwardValues;
}

// fn(threads, items) as constants, for shapes that hold the row.
template <typename T, typename F>
void with_row_shape(RowShape r, F&& fn) {
    auto call = [&](auto threads, auto items) { fn(threads, items); };
    std::integral_constant<int, 1> one;
    if (r.threads == 64)
        call(std::integral_constant<int, 64>{}, one);
    else if (r.threads == 128)
        call(std::integral_constant<int, 128>{}, one);
    else if (r.threads == 256)
        call(std::integral_constant<int, 256>{}, one);
    else if (r.threads == 512)
        call(std::integral_constant<int, 512>{}, one);
    else if (r.items == 1)
        call(std::integral_constant<int, 1024>{}, one);
    else if (r.items == 2)
        call(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{});
    else if constexpr (sizeof(T) == 4)
        call(std::integral_constant<int, 1024>{}, std::integral_constant<int, 4>{});
}

// Workgroups of the backward pass: enough to fill the 256 CUs, few enough that
// the partial rows cost little beside the data.
int64_t backward_blocks(int64_t rows, int64_t cols, int type) {
    const RowShape r = row_shape(cols, type);
    const int64_t rpb = r.threads < 256 ? 256 / r.threads : 1;
    const int64_t most = 256 * std::max(1, std::min(4, 1024 / r.threads));  // that many fit
    return std::min(ceil_div(rows, rpb), most);
}

void check_norm(const char* what, int64_t rows, int64_t cols, int type, int weight_type,
                bool has_weights) {
    const std::string w = what;
    require(rows >= 0 && cols >= 0, w + ": negative dimension");
    require(rows < (int64_t(1) << 31) && cols < (int64_t(1) << 28),
            w + ": rows must be < 2^31 and cols < 2^28");
    require(rows == 0 || cols > 0, w + ": rows of 0 columns have no mean");
    require(type >= TG_TYPE_F32 && type <= TG_TYPE_F16, w + ": unknown element type " +
                                                            std::to_string(type));
    require(!has_weights || weight_type == TG_TYPE_F32 || weight_type == type,
            w + ": gamma and beta must have x's type or be floats");
}

}  // namespace
}  // namespace tg

using tg::guard;
using tg::require;

extern "C" {

int tg_layer_norm(int64_t rows, int64_t cols, int type, const void* x, int64_t ldx,
                  const void* gamma, const void* beta, int weight_type, float eps, void* y,
                  int64_t ldy, float* mean, float* rstd, tg_stream_t stream) {
    return guard([&] {
        tg::check_norm("layer_norm", rows, cols, type, weight_type, gamma || beta);
        if (rows == 0) return;
        require(x && y, "layer_norm: null pointer");
        require(ldx >= cols && ldy >= cols, "layer_norm: leading dimension below cols");
        tg::NormArgs a{};
        a.cols = cols;
        a.ldx = ldx;
        a.gamma = gamma;
        a.beta = beta;
        a.weight_f32 = weight_type == TG_TYPE_F32;
        a.eps = eps;
        a.ldy = ldy;
        hipStream_t s = static_cast<hipStream_t>(stream);
        const tg::RowShape shape = tg::row_shape(cols, type);
        const int64_t z = tg::type_size(type);
        tg::for_slices(rows, std::max(shape.threads, 64), [&](int64_t first, int64_t count) {
            a.rows = count;
            a.x = static_cast<const char*>(x) + first * ldx * z;
            a.y = static_cast<char*>(y) + first * ldy * z;
            a.mean = mean ? mean + first : nullptr;
            a.rstd = rstd ? rstd + first : nullptr;
            const unsigned n = static_cast<unsigned>(count);
            tg::with_type(type, "layer_norm", [&](auto t) {
                using T = decltype(t);
                if (shape.items == 0) {
                    tg::norm_wide_kernel<T><<<n, tg::kWideThreads, 0, s>>>(a);
                    return;
                }
                tg::with_row_shape<T>(shape, [&](auto threads, auto items) {
                    constexpr int TPR = decltype(threads)::value, RPB = TPR > 256 ? 1 : 256 / TPR;
                    tg::norm_kernel<T, TPR, decltype(items)::value>
                        <<<(n + RPB - 1) / RPB, TPR > 256 ? TPR : 256, 0, s>>>(a);
                });
            });
            TG_LAUNCH_CHECK();
        });
    });
}

size_t tg_layer_norm_backward_workspace_size(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    // of any type
    const int64_t blocks = std::max(tg::backward_blocks(rows, cols, TG_TYPE_F32),
                                    tg::backward_blocks(rows, cols, TG_TYPE_BF16));
    tg::Carver c(nullptr, 0);
    c.take<float>(static_cast<size_t>(blocks) * 2 * static_cast<size_t>(cols));
    return c.bytes();
}

int tg_layer_norm_backward(int64_t rows, int64_t cols, int type, const void* dy, int64_t lddy,
                           const void* x, int64_t ldx, const void* gamma, int weight_type,
                           const float* mean, const float* rstd, void* dx, int64_t lddx,
                           void* dgamma, void* dbeta, void* workspace, size_t workspace_bytes,
                           tg_stream_t stream) {
    return guard([&] {
        tg::check_norm("layer_norm_backward", rows, cols, type, weight_type,
                       gamma || dgamma || dbeta);
        if (cols == 0 || (!dx && !dgamma && !dbeta)) return;
        hipStream_t s = static_cast<hipStream_t>(stream);
        const bool sums = dgamma || dbeta;
        tg::NormArgs a{};
        tg::TempBuffer temp;
        const int64_t blocks = tg::backward_blocks(rows, cols, type);
        if (rows > 0) {
            require(dy && x && mean && rstd, "layer_norm_backward: null pointer");
            require(ldx >= cols && lddy >= cols && (!dx || lddx >= cols),
                    "layer_norm_backward: leading dimension below cols");
            a.rows = rows;
            a.cols = cols;
            a.x = x;
            a.ldx = ldx;
            a.gamma = gamma;
            a.weight_f32 = weight_type == TG_TYPE_F32;
            a.mean = const_cast<float*>(mean);
            a.rstd = const_cast<float*>(rstd);
            a.dy = dy;
            a.lddy = lddy;
            a.dx = dx;
            a.lddx = lddx;
            if (sums) {
                const size_t need = tg_layer_norm_backward_workspace_size(rows, cols);
                if (!workspace) {
                    temp.allocate(need, s);
                    workspace = temp.get();
                    workspace_bytes = need;
                }
                tg::Carver c(workspace, workspace_bytes);
                a.part = c.take<float>(static_cast<size_t>(blocks) * 2 *
                                       static_cast<size_t>(cols));
            }
        }
        tg::with_type(type, "layer_norm_backward", [&](auto t) {
            using T = decltype(t);
            const unsigned n = static_cast<unsigned>(blocks);
            if (rows > 0) {
                const tg::RowShape shape = tg::row_shape(cols, type);
                if (!tg::in_registers(shape, type))
                    tg::norm_backward_wide_kernel<T><<<n, tg::kWideThreads, 0, s>>>(a);
                else
                    tg::with_row_shape<T>(shape, [&](auto threads, auto items) {
                        constexpr int TPR = decltype(threads)::value, I = decltype(items)::value;
                        if constexpr (I * tg::kVec<T> <= tg::kBackwardValues)
                            tg::norm_backward_kernel<T, TPR, I>
                                <<<n, TPR > 256 ? TPR : 256, 0, s>>>(a);
                    });
                TG_LAUNCH_CHECK();
            }
            if (sums) {
                // (2^22 workgroups of 1,024 threads are more than a grid's x takes)
                const int64_t b = tg::ceil_div(cols, 64), z = tg::ceil_div(b, 1 << 21);
                const dim3 grid(static_cast<unsigned>(tg::ceil_div(b, z)), 2,
                                static_cast<unsigned>(z));
                tg::norm_reduce_kernel<T><<<grid, 1024, 0, s>>>(a.part, rows > 0 ? blocks : 0, cols,
                                                                dgamma, dbeta,
                                                                weight_type == TG_TYPE_F32);
                TG_LAUNCH_CHECK();
            }
        });
    });
}

}  // extern "C"
