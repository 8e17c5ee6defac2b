// grouped.hip -- products grouped by expert or node type, with ragged groups.
#include "grouped.hpp"

#include <string>

#include "types.hpp"

namespace tg {
namespace {

struct GroupedArgs {
    int m, k, n, groups;
    const void* x;
    int64_t x_rows, ldx;
    const int32_t* rows;
    const int32_t* offsets;
    const void* w;  // forward
    int64_t ldw, w_stride;
    int transposed;
    const void* bias;
    int epi;
    void* y;
    int64_t ldy;
    const void* dy;  // gradient of w
    int64_t lddy;
    void* dw;
    void* dbias;
};

constexpr int kT = 64, kTK = 16;  // tile edge and depth

// One 64 x 64 tile, 4 x 4 outputs a thread: a(i, c), b(c, j) give the operands
// (0 outside), out(i, j, v) takes the sums.
template <typename A, typename B, typename O>
__device__ void plain_tile(int depth, A&& a, B&& b, O&& out) {
    __shared__ float as[kTK][kT + 4], bs[kTK][kT + 4];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    for (int c0 = 0; c0 < depth; c0 += kTK) {
        for (int i = threadIdx.x; i < kT * kTK; i += 256) {
            as[i % kTK][i / kTK] = a(i / kTK, c0 + i % kTK);
            bs[i / kT][i % kT] = b(c0 + i / kT, i % kT);
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kTK; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = __builtin_fmaf(as[c][ty * 4 + i], bs[c][tx * 4 + j], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) out(ty * 4 + i, tx * 4 + j, acc[i][j]);
}

template <typename T>
__global__ __launch_bounds__(256) void grouped_kernel(GroupedArgs a) {
    int g, r0, r1;
    if (!find_tile(a.offsets, a.groups, a.m, kT, blockIdx.y, &g, &r0, &r1)) return;
    const int n0 = blockIdx.x * kT;
    const T* x = static_cast<const T*>(a.x);
    const T* w = static_cast<const T*>(a.w) + g * a.w_stride;
    plain_tile(
        a.k,
        [&](int i, int c) {
            if (r0 + i >= r1 || c >= a.k) return 0.0f;
            const int64_t r = a.rows ? a.rows[r0 + i] : r0 + i;
            return r < 0 || r >= a.x_rows ? 0.0f : static_cast<float>(x[r * a.ldx + c]);
        },
        [&](int c, int j) {
            if (c >= a.k || n0 + j >= a.n) return 0.0f;
            return static_cast<float>(a.transposed ? w[(n0 + j) * a.ldw + c]
                                                   : w[c * a.ldw + n0 + j]);
        },
        [&](int i, int j, float v) {
            if (r0 + i >= r1 || n0 + j >= a.n) return;
            const float b = a.bias ? static_cast<float>(static_cast<const T*>(
                                         a.bias)[static_cast<int64_t>(g) * a.n + n0 + j])
                                   : 0.0f;
            static_cast<T*>(a.y)[(r0 + i) * a.ldy + n0 + j] =
                static_cast<T>(grouped_epilogue(v, b, a.epi));
        });
}

template <typename T>
__global__ __launch_bounds__(256) void wgrad_kernel(GroupedArgs a) {
    const int g = blockIdx.z, k0 = blockIdx.y * kT, n0 = blockIdx.x * kT;
    int lo, hi;
    group_rows(a.offsets, g, a.m, &lo, &hi);
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.dy);
    auto grad = [&](int c, int j) {
        return lo + c >= hi || n0 + j >= a.n
                   ? 0.0f
                   : static_cast<float>(dy[(lo + c) * a.lddy + n0 + j]);
    };
    if (a.dw)
        plain_tile(
            hi - lo,
            [&](int i, int c) {
                if (lo + c >= hi || k0 + i >= a.k) return 0.0f;
                const int64_t r = a.rows ? a.rows[lo + c] : lo + c;
                return r < 0 || r >= a.x_rows ? 0.0f : static_cast<float>(x[r * a.ldx + k0 + i]);
            },
            grad,
            [&](int i, int j, float v) {
                if (k0 + i < a.k && n0 + j < a.n)
                    static_cast<T*>(
                        a.dw)[(static_cast<int64_t>(g) * a.k + k0 + i) * a.n + n0 + j] =
                        static_cast<T>(v);
            });
    if (a.dbias && blockIdx.y == 0 && threadIdx.x < kT && n0 + threadIdx.x < a.n) {
        float s = 0.0f;
        for (int c = 0; c < hi - lo; ++c) s += grad(c, threadIdx.x);
        static_cast<T*>(a.dbias)[static_cast<int64_t>(g) * a.n + n0 + threadIdx.x] =
            static_cast<T>(s);
    }
}

void check_grouped(const std::string& w, int64_t m, int64_t k, int64_t n, int64_t groups, int type,
                   int64_t x_rows) {
    require(m >= 0 && k >= 0 && n >= 0 && groups >= 0 && x_rows >= 0, w + ": negative dimension");
    require(m < (int64_t(1) << 31) - 4096 && k < (int64_t(1) << 31) - 4096 &&
                n < (int64_t(1) << 31) - 4096 && x_rows < (int64_t(1) << 31),
            w + ": m, k and n must be < 2^31 - 4096");
    require(groups <= kMaxGroups, w + ": at most 1024 groups, got " + std::to_string(groups));
    require(type >= TG_TYPE_F32 && type <= TG_TYPE_F16, w + ": unknown element type " +
                                                            std::to_string(type));
}

}  // namespace
}  // namespace tg

using tg::guard;
using tg::require;

extern "C" {

int tg_grouped_matmul(int64_t m, int64_t k, int64_t n, int64_t groups, int type, const void* x,
                      int64_t x_rows, int64_t ldx, const int32_t* rows, const int32_t* offsets,
                      const void* w, int64_t ldw, int64_t w_stride, int transposed,
                      const void* bias, int epilogue, void* y, int64_t ldy,
                      tg_stream_t stream) {
    return guard([&] {
        const std::string what = "grouped_matmul";
        tg::check_grouped(what, m, k, n, groups, type, x_rows);
        require(epilogue >= TG_EPI_NONE && epilogue <= TG_EPI_ELU,
                what + ": unknown epilogue " + std::to_string(epilogue));
        require(rows || x_rows >= m, what + ": x has fewer than m rows");
        if (m == 0 || n == 0 || groups == 0) return;
        require(offsets && y && (k == 0 || (w && (x || x_rows == 0))), what + ": null pointer");
        require(ldy >= n && ldx >= k && ldw >= (transposed ? k : n),
                what + ": leading dimension below the columns");
        tg::GroupedArgs a{};
        a.m = static_cast<int>(m);
        a.k = static_cast<int>(k);
        a.n = static_cast<int>(n);
        a.groups = static_cast<int>(groups);
        a.x = x;
        a.x_rows = x_rows;
        a.ldx = ldx;
        a.rows = rows;
        a.offsets = offsets;
        a.w = w;
        a.ldw = ldw;
        a.w_stride = w_stride;
        a.transposed = transposed != 0;
        a.bias = bias;
        a.epi = epilogue;
        a.y = y;
        a.ldy = ldy;
        hipStream_t s = static_cast<hipStream_t>(stream);
        const dim3 grid(static_cast<unsigned>(tg::ceil_div(n, tg::kT)),
                        static_cast<unsigned>(tg::most_tiles(m, groups, tg::kT)));
        tg::with_type(type, "grouped_matmul", [&](auto t) {
            tg::grouped_kernel<decltype(t)><<<grid, 256, 0, s>>>(a);
        });
        TG_LAUNCH_CHECK();
    });
}

size_t tg_grouped_matmul_wgrad_workspace_size(int64_t, int64_t, int64_t, int64_t, int) { return 0; }

int tg_grouped_matmul_wgrad(int64_t m, int64_t k, int64_t n, int64_t groups, int type,
                            const void* x, int64_t x_rows, int64_t ldx, const int32_t* rows,
                            const void* dy, int64_t lddy, const int32_t* offsets, void* dw,
                            void* dbias, void*, size_t, tg_stream_t stream) {
    return guard([&] {
        const std::string what = "grouped_matmul_wgrad";
        tg::check_grouped(what, m, k, n, groups, type, x_rows);
        require(rows || x_rows >= m, what + ": x has fewer than m rows");
        if (k == 0) dw = nullptr;
        if (n == 0 || groups == 0 || (!dw && !dbias)) return;
        require(offsets && (m == 0 || (dy && (!dw || x || x_rows == 0))), what + ": null pointer");
        require(lddy >= n && (!dw || ldx >= k), what + ": leading dimension below the columns");
        tg::GroupedArgs a{};
        a.m = static_cast<int>(m);
        a.k = static_cast<int>(k);
        a.n = static_cast<int>(n);
        a.groups = static_cast<int>(groups);
        a.x = x;
        a.x_rows = x_rows;
        a.ldx = ldx;
        a.rows = rows;
        a.offsets = offsets;
        a.dy = dy;
        a.lddy = lddy;
        a.dw = dw;
        a.dbias = dbias;
        hipStream_t s = static_cast<hipStream_t>(stream);
        const dim3 grid(static_cast<unsigned>(tg::ceil_div(n, tg::kT)),
                        static_cast<unsigned>(dw ? tg::ceil_div(k, tg::kT) : 1),
                        static_cast<unsigned>(groups));
        tg::with_type(type, "grouped_matmul_wgrad", [&](auto t) {
            tg::wgrad_kernel<decltype(t)><<<grid, 256, 0, s>>>(a);
        });
        TG_LAUNCH_CHECK();
    });
}

}  // extern "C"
