// fp8.hip -- products in e4m3 with a scale for each block of 128.
#include "grouped.hpp"

#include <string>

#include "tiles.hpp"
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
    uint32_t mt, nt;  // row tiles (most) and column tiles
};

typedef f16 v2h __attribute__((ext_vector_type(2)));
typedef int v8i __attribute__((ext_vector_type(8)));

// A wavefront's operand of one tile of 16 rows: the lane's chunks q and 4 + q
// of a block, 32 values in all.
struct Operand {
    Frag c[2];
};

// Eight e4m3 values as fp16, which holds each of them exactly.
__device__ __forceinline__ v8h to_f16(uint32_t lo, uint32_t hi) {
    const v2h x[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false),
                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true),
                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false),
                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true)};
    v8h v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = x[i].x;
        v[2 * i + 1] = x[i].y;
    }
    return v;
}

// The sum of a block's products, 16 x 16.  The e4m3 matrix instructions (of any
// shape) line the products up with the largest of them and drop what lies far
// below it: against 64 bits a block's sum is off by up to 2^-12.5 of the sum of its
// products' sizes for operands of random bits, 2^-16.1 (2^-19.6 in the mean) for
// normal ones.  A 16-bit result of many rows takes that for twice the rate: it is
// far below the operands' own rounding to e4m3 (2^-4 of each product), though where
// a sum cancels it can be far above the result's to 2^-9 or 2^-12.
// Where the rate does not count (few rows) and for fp32 results the operands
// are widened to fp16, exactly (WIDE).
template <bool WIDE>
__device__ __forceinline__ v4f block_products(const Operand& a, const Operand& b) {
    v4f p = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (WIDE) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const v4u& x = a.c[s / 2].u;
            const v4u& y = b.c[s / 2].u;
            p = __builtin_amdgcn_mfma_f32_16x16x32_f16(to_f16(x[s % 2 * 2], x[s % 2 * 2 + 1]),
                                                       to_f16(y[s % 2 * 2], y[s % 2 * 2 + 1]), p,
                                                       0, 0, 0);
        }
    } else {
        v8i x, y;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = static_cast<int>(a.c[e / 4].u[e % 4]);
            y[e] = static_cast<int>(b.c[e / 4].u[e % 4]);
        }
        p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, p, 0, 0, 0, 0, 0, 0);
    }
    return p;
}

// x's quantised row for row p of the product, or -1.
__device__ __forceinline__ int source_row(const Fp8Args& a, int p) {
    const int r = a.rows ? a.rows[p] : p;
    return r < 0 || r >= a.x_rows ? -1 : r;
}

// bias n .. n + 3 of group g.
template <typename T>
__device__ __forceinline__ v4f bias_of(const Fp8Args& a, int g, int n) {
    float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (a.bias)
        load_floats<T, 4>(static_cast<const T*>(a.bias) + static_cast<int64_t>(g) * a.n + n,
                          a.n - n, b);
    return v4f{b[0], b[1], b[2], b[3]};
}

// Columns n .. n + 3 of row p: bias, epilogue, store.
template <typename T, int EPI>
__device__ __forceinline__ void store_outputs(const Fp8Args& a, int p, int n, const v4f& acc,
                                              const v4f& bias) {
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = grouped_epilogue<EPI>(acc[e], bias[e]);
    store_floats<T, 4>(static_cast<T*>(a.y) + p * a.ldy + n, a.n - n, v);
}

// BM x BN outputs, a tile a block of 128: the products of a block go to fresh
// registers and from there, times x's scale of the row and w's of the columns,
// to the sums (16 multiply-adds beside each 32-cycle instruction).  As in the
// 16-bit products the outputs are computed transposed, so a lane's row of x is
// one; x's scales of the block come to LDS with its tile.
//
// FAR: x and its scales come through registers, for rows gathered from places
// past 2 GB, which the offsets of loads to LDS do not reach.
template <typename T, typename S, bool FAR>
__global__ __launch_bounds__(S::kThreads) void fp8_kernel(Fp8Args a) {
    constexpr int kScales = S::kM * kRowBytes;  // behind x's tile
    __shared__ __attribute__((aligned(16))) char a0[kScales + S::kThreads * 4];
    __shared__ __attribute__((aligned(16))) char b0[S::kN * kRowBytes];
    __shared__ __attribute__((aligned(16))) char a1[kScales + S::kThreads * 4];
    __shared__ __attribute__((aligned(16))) char b1[S::kN * kRowBytes];
    constexpr bool WIDE = sizeof(T) == 4;
    uint32_t mt, ntile;
    if (!tile_of(blockIdx.x, count_tiles(a.offsets, a.groups, a.m, S::kM), a.nt, &mt, &ntile))
        return;
    int g, r0, r1;
    if (!find_tile(a.offsets, a.groups, a.m, S::kM, static_cast<int>(mt), &g, &r0, &r1)) return;
    const int n0 = static_cast<int>(ntile) * S::kN;
    const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / S::kWC * S::kMI * 16, wn = wave % S::kWC * S::kNJ * 16;
    const int64_t kp = static_cast<int64_t>(a.kb) * kBlock;
    const uint8_t* w = a.wq + static_cast<int64_t>(g) * a.n * kp;
    static_assert(kBlock % (S::kNJ * 16) == 0, "one scale of w a wavefront");
    const int nb = (a.n + kBlock - 1) / kBlock;
    const int wblock = (n0 + wn) / kBlock < nb ? (n0 + wn) / kBlock : nb - 1;
    const float* ws = a.wscale + (static_cast<int64_t>(g) * nb + wblock) * a.kb;

    // a tile's rows of x from its first (gathered: from x's first), w's columns
    const uint8_t* xb = a.rows ? a.xq : a.xq + static_cast<int64_t>(r0) * kp;
    const uint8_t* wb = w + static_cast<int64_t>(n0) * kp;
    uint32_t ao[S::kCA], bo[S::kCB];
    const uint8_t* far[S::kCA];  // null: zeros
    v4u held[S::kCA];            // the next tile's
    float held_scale = 0.0f;
#pragma unroll
    for (int t = 0; t < S::kCA; ++t) {
        int row, c;
        chunk_place<uint8_t, S::kM, false>(t * S::kThreads + tid, &row, &c);
        const int src = r0 + row < r1 ? source_row(a, r0 + row) : -1;
        far[t] = FAR && src >= 0 ? a.xq + src * kp + c : nullptr;
        ao[t] = src < 0 ? kOutside
                        : static_cast<uint32_t>((a.rows ? src : row) * kp + c);
    }
#pragma unroll
    for (int t = 0; t < S::kCB; ++t) {
        int col, c;
        chunk_place<uint8_t, S::kN, false>(t * S::kThreads + tid, &col, &c);
        bo[t] = n0 + col < a.n ? static_cast<uint32_t>(col * kp + c) : kOutside;
    }
    // one row's scale for each thread; outside, and of threads past the rows: 0
    uint32_t so = kOutside;
    const float* far_scale = nullptr;
    if (tid < S::kM && r0 + tid < r1) {
        const int src = source_row(a, r0 + tid);
        if (src >= 0) so = static_cast<uint32_t>(src) * 4;
        if (FAR && src >= 0) far_scale = a.xscale + src;
    }
    // load p of tile kt (zeros past the last tile)
    constexpr int kLoads = 1 + S::kCA + S::kCB;
    auto load = [&](int kt, char* la, char* lb, int p) {
        const int64_t size = kt < a.kb ? kDirectBytes : 0;
        const int64_t at = static_cast<int64_t>(kt) * kBlock;
        if (FAR && p == 0) {
            held_scale = far_scale && kt < a.kb ? far_scale[kt * a.x_rows] : 0.0f;
        } else if (FAR && p <= S::kCA) {
            const v4u none = {0, 0, 0, 0};
            const uint8_t* x = far[p - 1];
            held[p - 1] = x && kt < a.kb ? *reinterpret_cast<const v4u*>(x + at) : none;
        } else if (p == 0) {
            const float* xs = a.xscale + static_cast<int64_t>(kt) * a.x_rows;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                buffer_of(xs, kt < a.kb ? 4 * a.x_rows : 0),
                (TG_LDS void*)(la + kScales + wave * 256), 4, static_cast<int>(so), 0, 0, 0);
        } else if (p <= S::kCA) {
            load_to_lds(buffer_of(xb + at, size), la + ((p - 1) * S::kThreads + wave * 64) * 16,
                        ao[p - 1]);
        } else {
            const int t = p - 1 - S::kCA;
            load_to_lds(buffer_of(wb + at, size), lb + (t * S::kThreads + wave * 64) * 16, bo[t]);
        }
    };
    // what FAR holds, to where load() puts it otherwise
    auto put = [&](char* la) {
        if (!FAR) return;
#pragma unroll
        for (int t = 0; t < S::kCA; ++t)
            *reinterpret_cast<v4u*>(la + (t * S::kThreads + tid) * 16) = held[t];
        *reinterpret_cast<float*>(la + kScales + tid * 4) = held_scale;
    };
    Acc<S> acc = {};
    const Reader<uint8_t, S::kM, false, S::kMI> ra(wm, lane);
    const Reader<uint8_t, S::kN, false, S::kNJ> rb(wn, lane);
    int kt = 0;
    // the products of the tile in la and lb, the next one's loads among them
    auto compute = [&](const char* la, const char* lb, char* na, char* nb) {
        const float scale = scalar_load(ws + kt++);
        const float* xs = reinterpret_cast<const float*>(la + kScales) + wm + r;
        // While row tile i's products run, x's operands of i + 1 are read, the
        // products of i - 1 scaled and added, and a share of the next tile's loads
        // asked for (asked for at once, they held the reads and the first products
        // back: 8,192 x 4,096 x 8,192 330 us against 301).  No more than that may
        // be live (registers).
        auto row_tile = [&](int i) {
            Operand x;
#pragma unroll
            for (int s = 0; s < 2; ++s) x.c[s] = ra.read(la, i, s);
            return x;
        };
        Operand b[S::kNJ], x[2];
#pragma unroll
        for (int j = 0; j < S::kNJ; ++j)
#pragma unroll
            for (int s = 0; s < 2; ++s) b[j].c[s] = rb.read(lb, j, s);
        x[0] = row_tile(0);
        v4f part[2][S::kNJ];
#pragma unroll
        for (int i = 0; i <= S::kMI; ++i) {
            if (i + 1 < S::kMI) x[(i + 1) & 1] = row_tile(i + 1);
            if (i < S::kMI) {
#pragma unroll
                for (int j = 0; j < S::kNJ; ++j)
                    part[i & 1][j] = block_products<WIDE>(b[j], x[i & 1]);
#pragma unroll
                for (int p = i * kLoads / S::kMI; p < (i + 1) * kLoads / S::kMI; ++p)
                    load(kt, na, nb, p);
            }
            if (i > 0) {
                const float f = xs[(i - 1) * 16] * scale;
#pragma unroll
                for (int j = 0; j < S::kNJ; ++j) {
                    v4f& sum = acc[i - 1][j];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sum[e] = __builtin_fmaf(part[(i - 1) & 1][j][e], f, sum[e]);
                    asm volatile("" : "+v"(sum));  // here, not at the tile's end
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        put(na);
    };
    if (a.kb > 0) {
#pragma unroll
        for (int p = 0; p < kLoads; ++p) load(0, a0, b0, p);
        put(a0);
    }
    while (kt + 1 < a.kb) {  // compute() counts
        loads_border();
        compute(a0, b0, a1, b1);
        loads_border();
        compute(a1, b1, a0, b0);
    }
    if (kt < a.kb) {
        loads_border();
        compute(a0, b0, a1, b1);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    v4f bias[S::kNJ];
#pragma unroll
    for (int j = 0; j < S::kNJ; ++j) bias[j] = bias_of<T>(a, g, n0 + wn + j * 16 + 4 * q);
    with_epilogue(a.epi, [&](auto epi) {
#pragma unroll
        for (int i = 0; i < S::kMI; ++i) {
            const int p = r0 + wm + i * 16 + r;
            if (p >= r1) continue;
#pragma unroll
            for (int j = 0; j < S::kNJ; ++j)
                store_outputs<T, decltype(epi)::value>(a, p, n0 + wn + j * 16 + 4 * q, acc[i][j],
                                                       bias[j]);
        }
    });
}

// Few rows: 16 rows x 16 columns, each of four wavefronts a quarter of the
// blocks straight from memory (w is read once, and that is what counts), four
// blocks in flight; their sums are joined in LDS, in order.  The products are exact
// (5 rows of 4,096 x 4,096 6.0 us, 64 x 2,048 x 4,096 10.6; with the e4m3
// instructions' dropped bits 6.6 and 10.6).
constexpr int kThinWaves = 4, kThinAhead = 4;

template <typename T>
__global__ __launch_bounds__(64 * kThinWaves) void fp8_thin_kernel(Fp8Args a) {
    __shared__ v4f join[kThinWaves - 1][64];
    uint32_t mt, ntile;
    if (!tile_of(blockIdx.x, count_tiles(a.offsets, a.groups, a.m, 16), a.nt, &mt, &ntile)) return;
    int g, r0, r1;
    if (!find_tile(a.offsets, a.groups, a.m, 16, static_cast<int>(mt), &g, &r0, &r1)) return;
    const int n0 = static_cast<int>(ntile) * 16;
    const int lane = threadIdx.x & 63, q = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t kp = static_cast<int64_t>(a.kb) * kBlock;
    const int src = r0 + r < r1 ? source_row(a, r0 + r) : -1;
    const int col = n0 + r < a.n ? n0 + r : a.n - 1;  // past the last: computed, not stored
    const int nb = (a.n + kBlock - 1) / kBlock;
    const uint8_t* px = a.xq + (src < 0 ? 0 : src) * kp + 16 * q;  // (any: not used)
    const uint8_t* pw = a.wq + (static_cast<int64_t>(g) * a.n + col) * kp + 16 * q;
    const float* xs = a.xscale + (src < 0 ? 0 : src);
    const float* ws = a.wscale + (static_cast<int64_t>(g) * nb + n0 / kBlock) * a.kb;
    const int share = (a.kb + kThinWaves - 1) / kThinWaves;
    const int b0 = wave * share, b1 = b0 + share < a.kb ? b0 + share : a.kb;
    const uint32_t keep = src < 0 ? 0 : ~0u;
    const v4u kept = {keep, keep, keep, keep};
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int base = b0; base < b1; base += kThinAhead) {
        Operand x[kThinAhead], w[kThinAhead];
        float sx[kThinAhead], sw[kThinAhead];
#pragma unroll
        for (int u = 0; u < kThinAhead; ++u) {
            const int b = base + u < b1 ? base + u : b1 - 1;  // again, for nothing
            const int64_t at = static_cast<int64_t>(b) * kBlock;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                w[u].c[h].u = *reinterpret_cast<const v4u*>(pw + at + 64 * h);
                x[u].c[h].u = *reinterpret_cast<const v4u*>(px + at + 64 * h);
            }
            sx[u] = xs[static_cast<int64_t>(b) * a.x_rows];
            sw[u] = ws[b];
        }
        if (a.rows) {  // an index outside x is a row of zeros
#pragma unroll
            for (int u = 0; u < kThinAhead; ++u) {
#pragma unroll
                for (int h = 0; h < 2; ++h) x[u].c[h].u &= kept;
                if (src < 0) sx[u] = 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < kThinAhead; ++u) {
            const v4f p = block_products<true>(w[u], x[u]);
            if (base + u >= b1) break;
            const float s = sx[u] * sw[u];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(p[e], s, acc[e]);
        }
    }
    if (wave > 0) join[wave - 1][lane] = acc;
    __syncthreads();
    if (wave > 0 || r0 + r >= r1) return;
#pragma unroll
    for (int u = 0; u < kThinWaves - 1; ++u) acc += join[u][lane];
    const v4f bias = bias_of<T>(a, g, n0 + 4 * q);
    with_epilogue(a.epi, [&](auto epi) {
        store_outputs<T, decltype(epi)::value>(a, r0 + r, n0 + 4 * q, acc, bias);
    });
}

using Large = Shape<256, 256, 2, 4>;
using Medium = Shape<128, 128, 2, 2>;
using Small = Shape<64, 64, 2, 2>;

unsigned set_grid(Fp8Args& a, int bm, int bn, int threads) {
    a.mt = static_cast<uint32_t>(most_tiles(a.m, a.groups, bm));
    a.nt = static_cast<uint32_t>(ceil_div(a.n, bn));
    const int64_t grid = static_cast<int64_t>(a.mt) * a.nt;
    return grid_of("matmul_fp8", grid, threads);
}

template <typename T>
void launch_fp8(Fp8Args& a, hipStream_t s) {
    const int64_t kp = static_cast<int64_t>(a.kb) * kBlock;
    // loads' offsets to LDS have 31 bits
    const bool near = (a.rows ? a.x_rows : 256) * kp < kDirectBytes && 4 * a.x_rows < kDirectBytes;
    auto tiled = [&](auto shape) {
        using S = decltype(shape);
        const unsigned grid = set_grid(a, S::kM, S::kN, S::kThreads);
        fp8_kernel<T, S, false><<<grid, S::kThreads, 0, s>>>(a);
    };
    auto tiles = [&](int64_t edge) {
        return most_tiles(a.m, a.groups, edge) * ceil_div(a.n, edge);
    };
    // Few rows: the thin form while its workgroups are few (5 rows of 4,096 x
    // 4,096 6.0 us, 12 in 64 x 64; 150 rows of 32 groups, 2,048 x 4,096, 62 us
    // against 41).  Large tiles where there are 160 of them of 1,024 values and the
    // groups fill them (2,500 x 2,048 x 4,096 46 us against 50; 40,000 x 512 x 512
    // 36 against 32; 16,384 rows of 32 groups, 2,048 x 4,096, 220 against 300, 4,096
    // rows of 16 groups 80 to 90 both), 128 x 128 where there are one for
    // each CU (10,000 x 512 x 512 the same as 64 x 64, 10,000 x 2,048 x 4,096 126
    // us against 177), else 64 x 64 (600 x 2,048 x 1,024 12 us against 18).  fp32
    // results stay below the large tile, whose widened operands do not fit the
    // registers beside its sums (18 spilled; 2,500 x 2,048 x 4,096 58 us against
    // 53 of 128 x 128, 40,000 x 1,024 x 1,024 106 against 95, 8,192 x 4,096 x 8,192
    // 477 against 499).
    if (256 * kp >= kDirectBytes || tiles(16) <= 1024) {
        const unsigned grid = set_grid(a, 16, 16, 64 * kThinWaves);
        fp8_thin_kernel<T><<<grid, 64 * kThinWaves, 0, s>>>(a);
    } else if (!near) {
        const unsigned grid = set_grid(a, Medium::kM, Medium::kN, Medium::kThreads);
        fp8_kernel<T, Medium, true><<<grid, Medium::kThreads, 0, s>>>(a);
    } else if (sizeof(T) == 2 && a.kb >= 8 && tiles(256) * a.kb >= 160 * 8 &&
               a.m >= 256 * a.groups) {
        if constexpr (sizeof(T) == 2) tiled(Large{});
    } else if (tiles(128) >= 300 && a.m >= 100 * a.groups) {
        tiled(Medium{});
    } else {
        tiled(Small{});
    }
    TG_LAUNCH_CHECK();
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
        const unsigned grid = tg::grid_of("quantize", tg::ceil_div(rows * blocks, 32), 256);
        tg::with_type(type, "quantize", [&](auto t) {
            using T = decltype(t);
            tg::quantize_kernel<T><<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(
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
        if (x_rows == 0) {  // every row is one of zeros: read, and not used
            a.xq = a.wq;
            a.xscale = a.wscale;
        }
        tg::with_type(type, "matmul_fp8", [&](auto t) {
            tg::launch_fp8<decltype(t)>(a, static_cast<hipStream_t>(stream));
        });
    });
}

}  // extern "C"
