// fp8.hip -- products in e4m3 with a scale for each block of 128.
#include "grouped.hpp"

#include <string>

#include "types.hpp"

namespace tg {
namespace {

constexpr int kBlock = 128;
constexpr float kPerE4m3Max = 1.0f / 448.0f;  // of the largest e4m3 value
constexpr float kLeastScale = 1.17549435e-38f;  // 2^-126: x / scale stays finite

__device__ __forceinline__ float block_scale(float largest) {
    return fmaxf(largest * kPerE4m3Max, kLeastScale);
}

// Four quotients as e4m3, to nearest even; |q| <= 448 rounded to fp32.
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
    return static_cast<uint32_t>(v);
}

// One 128-column block of a row by eight lanes, 16 values each.
template <typename T>
__global__ __launch_bounds__(256) void quantize_kernel(int64_t rows, int64_t cols, int64_t blocks,
                                                       const T* __restrict__ x, int64_t ldx,
                                                       uint8_t* __restrict__ q,
                                                       float* __restrict__ scale) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x / 8;
    const int lane = threadIdx.x % 8;
    const int64_t at = i < rows * blocks ? i : rows * blocks - 1;  // every lane joins the maximum
    const int64_t r = at / blocks, b = at % blocks;
    const int64_t c = b * kBlock + lane * 16;
    float v[16], largest = 0.0f;
    load_floats<T, 16>(x + r * ldx + c, cols - c, v);
#pragma unroll
    for (int u = 0; u < 16; ++u) largest = fmaxf(largest, fabsf(v[u]));
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) largest = fmaxf(largest, __shfl_xor(largest, d, 8));
    const float s = block_scale(largest);
    uint4 out;
    uint32_t* o = &out.x;
#pragma unroll
    for (int u = 0; u < 4; ++u)
        o[u] = to_e4m3(v[4 * u] / s, v[4 * u + 1] / s, v[4 * u + 2] / s, v[4 * u + 3] / s);
    if (i >= rows * blocks) return;
    *reinterpret_cast<uint4*>(q + (r * blocks + b) * kBlock + lane * 16) = out;
    if (lane == 0) scale[b * rows + r] = s;
}

// One 128 x 128 block of a matrix, read along its rows, written along k.
template <typename T>
__global__ __launch_bounds__(256) void quantize_weight_kernel(int64_t k, int64_t n, const T* w,
                                                              int64_t ldw, int64_t w_stride,
                                                              int transposed,
                                                              uint8_t* __restrict__ q,
                                                              float* __restrict__ scale) {
    __shared__ float tile[kBlock][kBlock + 1];  // [n][k]
    __shared__ float top[4];
    const int64_t kb = gridDim.x, nb = gridDim.y, g = blockIdx.z;
    const int64_t k0 = static_cast<int64_t>(blockIdx.x) * kBlock;
    const int64_t n0 = static_cast<int64_t>(blockIdx.y) * kBlock;
    w += g * w_stride;
    float largest = 0.0f;
    for (int i = threadIdx.x; i < kBlock * kBlock; i += 256) {
        const int in = transposed ? i / kBlock : i % kBlock;
        const int ik = transposed ? i % kBlock : i / kBlock;
        float v = 0.0f;
        if (k0 + ik < k && n0 + in < n)
            v = static_cast<float>(transposed ? w[(n0 + in) * ldw + k0 + ik]
                                              : w[(k0 + ik) * ldw + n0 + in]);
        tile[in][ik] = v;
        largest = fmaxf(largest, fabsf(v));
    }
    largest = wave_max(largest);
    if (threadIdx.x % kWave == 0) top[threadIdx.x / kWave] = largest;
    __syncthreads();
    const float s = block_scale(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
    const int64_t kp = kb * kBlock;
    for (int i = threadIdx.x; i < kBlock * kBlock / 4; i += 256) {
        const int in = i / (kBlock / 4), ik = i % (kBlock / 4) * 4;
        if (n0 + in >= n) break;
        const float* t = &tile[in][ik];
        *reinterpret_cast<uint32_t*>(q + (g * n + n0 + in) * kp + k0 + ik) =
            to_e4m3(t[0] / s, t[1] / s, t[2] / s, t[3] / s);
    }
    if (threadIdx.x == 0) scale[(g * nb + blockIdx.y) * kb + blockIdx.x] = s;
}

struct Fp8Args {
    int m, n, kb, groups;  // kb: blocks of 128 along k
    const uint8_t* xq;
    const float* xscale;
    int64_t x_rows;
    const int32_t* rows;
    const int32_t* offsets;
    const uint8_t* wq;
    const float* wscale;
    const void* bias;
    int epi;
    void* y;
    int64_t ldy;
};

typedef float v4f __attribute__((ext_vector_type(4)));
typedef f16 v2h __attribute__((ext_vector_type(2)));
typedef f16 v8h __attribute__((ext_vector_type(8)));

// Eight e4m3 values as fp16, which holds each of them exactly.
__device__ __forceinline__ v8h to_f16(uint2 b) {
    const v2h x[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b.x, 1.0f, false),
                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b.x, 1.0f, true),
                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b.y, 1.0f, false),
                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b.y, 1.0f, true)};
    v8h v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = x[i].x;
        v[2 * i + 1] = x[i].y;
    }
    return v;
}

// One wavefront: 16 rows x 16 columns.  The e4m3 matrix instructions line the
// products up with the largest of them and drop what lies far below it: against
// 64 bits a block's sum is off by up to 2^-12.8 of the sum of its products'
// sizes for operands of random bits, 2^-16.3 (2^-18.9 in the mean) for normal
// ones.  That is below a 16-bit result's own rounding; for fp32 results the
// operands are widened to fp16, exactly, whose products are added in fp32.
template <typename T>
__global__ __launch_bounds__(64) void fp8_kernel(Fp8Args a) {
    int g, r0, r1;
    if (!find_tile(a.offsets, a.groups, a.m, 16, blockIdx.y, &g, &r0, &r1)) return;
    const int lane = threadIdx.x, r = lane % 16, q = lane / 16;
    const int n0 = blockIdx.x * 16;
    auto source = [&](int i) -> int64_t {
        const int p = r0 + i < r1 ? r0 + i : r1 - 1;
        const int64_t s = a.rows ? a.rows[p] : p;
        return s < 0 || s >= a.x_rows ? -1 : s;
    };
    const int64_t ra = source(r);
    const int col = n0 + r < a.n ? n0 + r : a.n - 1;
    const int64_t kp = static_cast<int64_t>(a.kb) * kBlock;
    const uint8_t* pa = a.xq + (ra < 0 ? 0 : ra) * kp;
    const uint8_t* pb = a.wq + (static_cast<int64_t>(g) * a.n + col) * kp;
    const float* ws = a.wscale + (static_cast<int64_t>(g) * ((a.n + 127) / 128) + col / 128) * a.kb;
    v4f acc = {};
    for (int b = 0; b < a.kb; ++b) {
        v4f part = {};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int64_t c = b * kBlock + s * 32 + q * 8;
            const uint2 av = *reinterpret_cast<const uint2*>(pa + c);
            const uint2 bv = *reinterpret_cast<const uint2*>(pb + c);
            if constexpr (sizeof(T) == 4)
                part = __builtin_amdgcn_mfma_f32_16x16x32_f16(to_f16(av), to_f16(bv), part, 0, 0,
                                                              0);
            else
                part = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(
                    __builtin_bit_cast(long, av), __builtin_bit_cast(long, bv), part, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t rr = source(4 * q + i);
            const float xs = rr < 0 ? 0.0f : a.xscale[static_cast<int64_t>(b) * a.x_rows + rr];
            acc[i] = rr < 0 ? 0.0f : __builtin_fmaf(xs * ws[b], part[i], acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int p = r0 + 4 * q + i;
        if (p >= r1 || n0 + r >= a.n) continue;
        const float bias = a.bias ? static_cast<float>(static_cast<const T*>(
                                        a.bias)[static_cast<int64_t>(g) * a.n + n0 + r])
                                  : 0.0f;
        static_cast<T*>(a.y)[p * a.ldy + n0 + r] =
            static_cast<T>(grouped_epilogue(acc[i], bias, a.epi));
    }
}

}  // namespace
}  // namespace tg

using tg::guard;
using tg::require;

extern "C" {

int tg_quantize(int64_t rows, int64_t cols, int type, const void* x, int64_t ldx, void* q,
                float* scale, tg_stream_t stream) {
    return guard([&] {
        require(rows >= 0 && cols >= 0, "quantize: negative dimension");
        require(rows < (int64_t(1) << 31) && cols < (int64_t(1) << 31) - 4096,
                "quantize: rows and cols must be < 2^31 - 4096");
        if (rows == 0 || cols == 0) return;
        require(x && q && scale, "quantize: null pointer");
        require(ldx >= cols, "quantize: leading dimension below cols");
        require(reinterpret_cast<uintptr_t>(q) % 16 == 0, "quantize: q must be 16-byte aligned");
        const int64_t blocks = tg::ceil_div(cols, tg::kBlock);
        const int64_t grid = tg::ceil_div(rows * blocks, 32);
        require(grid < (int64_t(1) << 31), "quantize: too many elements");
        tg::with_type(type, "quantize", [&](auto t) {
            using T = decltype(t);
            tg::quantize_kernel<T><<<static_cast<unsigned>(grid), 256, 0,
                                     static_cast<hipStream_t>(stream)>>>(
                rows, cols, blocks, static_cast<const T*>(x), ldx, static_cast<uint8_t*>(q), scale);
        });
        TG_LAUNCH_CHECK();
    });
}

int tg_quantize_weight(int64_t groups, int64_t k, int64_t n, int type, const void* w,
                       int64_t ldw, int64_t w_stride, int transposed, void* q, float* scale,
                       tg_stream_t stream) {
    return guard([&] {
        require(groups >= 0 && k >= 0 && n >= 0, "quantize_weight: negative dimension");
        require(groups <= tg::kMaxGroups && k < (int64_t(1) << 31) - 4096 &&
                    n < (int64_t(65535) * tg::kBlock),
                "quantize_weight: at most 1024 groups, k < 2^31 - 4096 and n <= 8388480");
        if (groups == 0 || k == 0 || n == 0) return;
        require(w && q && scale, "quantize_weight: null pointer");
        require(ldw >= (transposed ? k : n),
                "quantize_weight: leading dimension below the columns");
        require(reinterpret_cast<uintptr_t>(q) % 16 == 0,
                "quantize_weight: q must be 16-byte aligned");
        const dim3 grid(static_cast<unsigned>(tg::ceil_div(k, tg::kBlock)),
                        static_cast<unsigned>(tg::ceil_div(n, tg::kBlock)),
                        static_cast<unsigned>(groups));
        tg::with_type(type, "quantize_weight", [&](auto t) {
            using T = decltype(t);
            tg::quantize_weight_kernel<T><<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(
                k, n, static_cast<const T*>(w), ldw, w_stride, transposed,
                static_cast<uint8_t*>(q), scale);
        });
        TG_LAUNCH_CHECK();
    });
}

int tg_matmul_fp8(int64_t m, int64_t k, int64_t n, int64_t groups, const void* xq,
                  const float* xscale, int64_t x_rows, const int32_t* rows,
                  const int32_t* offsets, const void* wq, const float* wscale, int type,
                  const void* bias, int epilogue, void* y, int64_t ldy, tg_stream_t stream) {
    return guard([&] {
        require(m >= 0 && k >= 0 && n >= 0 && groups >= 0 && x_rows >= 0,
                "matmul_fp8: negative dimension");
        require(m < (int64_t(1) << 31) - 4096 && k < (int64_t(1) << 31) - 4096 &&
                    n < (int64_t(1) << 31) - 4096 && x_rows < (int64_t(1) << 31),
                "matmul_fp8: m, k and n must be < 2^31 - 4096");
        require(groups <= tg::kMaxGroups, "matmul_fp8: at most 1024 groups, got " +
                                              std::to_string(groups));
        require(offsets || groups == 1, "matmul_fp8: several groups need offsets");
        require(rows || x_rows >= m, "matmul_fp8: x has fewer than m rows");
        require(epilogue >= TG_EPI_NONE && epilogue <= TG_EPI_ELU,
                "matmul_fp8: unknown epilogue " + std::to_string(epilogue));
        require(type >= TG_TYPE_F32 && type <= TG_TYPE_F16,
                "matmul_fp8: unknown element type " + std::to_string(type));
        if (m == 0 || n == 0 || groups == 0) return;
        require(y && (k == 0 || (wq && wscale && (x_rows == 0 || (xq && xscale)))),
                "matmul_fp8: null pointer");
        require(ldy >= n, "matmul_fp8: leading dimension below the columns");
        require(reinterpret_cast<uintptr_t>(xq) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(wq) % 16 == 0,
                "matmul_fp8: xq and wq must be 16-byte aligned");
        tg::Fp8Args a{};
        a.m = static_cast<int>(m);
        a.n = static_cast<int>(n);
        a.kb = static_cast<int>(tg::ceil_div(k, tg::kBlock));
        a.groups = static_cast<int>(groups);
        a.xq = static_cast<const uint8_t*>(xq);
        a.xscale = xscale;
        a.x_rows = x_rows;
        a.rows = rows;
        a.offsets = offsets;
        a.wq = static_cast<const uint8_t*>(wq);
        a.wscale = wscale;
        a.bias = bias;
        a.epi = epilogue;
        a.y = y;
        a.ldy = ldy;
        if (x_rows == 0) a.kb = 0;  // every row is one of zeros
        const dim3 grid(static_cast<unsigned>(tg::ceil_div(n, 16)),
                        static_cast<unsigned>(tg::most_tiles(m, groups, 16)));
        tg::with_type(type, "matmul_fp8", [&](auto t) {
            tg::fp8_kernel<decltype(t)><<<grid, 64, 0, static_cast<hipStream_t>(stream)>>>(a);
        });
        TG_LAUNCH_CHECK();
    });
}

}  // extern "C"
