// linear_kernels.hpp -- the kernels of the dense layers, compiled for one element
// type by each of linear_f32.hip, linear_bf16.hip and linear_f16.hip.
//
// All three products (x w; d w^T; x^T d) are one kernel, out [m x n] = the sum
// over the contraction of X's row and W's column, whose operands run along or
// across the contraction (tiles.hpp): x w has x along and w across (or along, if
// transposed), d w^T the other of the two for w, x^T d both across.  16-bit types go
// through v_mfma_f32_16x16x32, floats through v_mfma_f32_16x16x4f32; sums are
// fp32.  Where the tiles are too few for the CUs, or a chain of floats too long,
// the contraction is cut in parts whose fp32 sums a second kernel adds in order,
// with the epilogue.  The epilogue is in float, one rounding for each stored value:
//   pre = sum + bias,  y = residual + act(pre),  d = dy act'(pre), dbias = sum of d;
// d is rounded to the element type before d w^T and x^T d read it (the operands of the
// matrix instructions; dbias sums the values before that).
#pragma once

#include "grouped.hpp"
#include "linear.hpp"
#include "tiles.hpp"
#include "types.hpp"

namespace tg {
namespace {

constexpr float kGeluScale = 1.5957691216f;  // 2 sqrt(2 / pi)
constexpr float kGeluCube = 0.044715f;
constexpr float kLog2e = 1.4426950409f;

// 1 / (1 + 2^e), e = -s log2(e): the sigmoid of s, and GELU's (1 + tanh(s / 2)) / 2,
// whose constants take the logarithm.  (The reciprocal instruction is within one unit
// in the last place.)
__device__ __forceinline__ float sigmoid_of_log2(float e) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(e));
}
__device__ __forceinline__ float gelu_log2(float v) {
    return v * __builtin_fmaf(v * v, -kGeluScale * kGeluCube * kLog2e, -kGeluScale * kLog2e);
}

template <int ACT>
__device__ __forceinline__ float act_of(float v) {
    if constexpr (ACT == TG_EPI_RELU) return 0.0f < v ? v : 0.0f;
    if constexpr (ACT == TG_EPI_ELU) return v < 0.0f ? expm1_negative(v) : v;
    if constexpr (ACT == TG_EPI_GELU)
        return v * sigmoid_of_log2(gelu_log2(v));
    if constexpr (ACT == TG_EPI_SILU) return v * sigmoid_of_log2(-kLog2e * v);
    return v;
}

// act'(v).  Where p (1 - p) is 0, so is its term, however large v's powers are.
template <int ACT>
__device__ __forceinline__ float slope_of(float v) {
    if constexpr (ACT == TG_EPI_RELU) return 0.0f < v ? 1.0f : 0.0f;
    if constexpr (ACT == TG_EPI_ELU) return v < 0.0f ? __expf(v) : 1.0f;
    if constexpr (ACT == TG_EPI_GELU || ACT == TG_EPI_SILU) {
        const float ds =
            ACT == TG_EPI_GELU
                ? __builtin_fmaf(v * v, 3.0f * kGeluScale * kGeluCube, kGeluScale)
                : 1.0f;
        const float p = sigmoid_of_log2(ACT == TG_EPI_GELU ? gelu_log2(v) : -kLog2e * v);
        const float t = p * (1.0f - p);
        return t == 0.0f ? p : __builtin_fmaf(t * v, ds, p);
    }
    return 1.0f;
}

template <typename F>
__device__ __forceinline__ void with_act(int act, F&& fn) {
    switch (act) {
        case TG_EPI_RELU: return fn(std::integral_constant<int, TG_EPI_RELU>{});
        case TG_EPI_ELU: return fn(std::integral_constant<int, TG_EPI_ELU>{});
        case TG_EPI_GELU: return fn(std::integral_constant<int, TG_EPI_GELU>{});
        case TG_EPI_SILU: return fn(std::integral_constant<int, TG_EPI_SILU>{});
        default: return fn(std::integral_constant<int, TG_EPI_NONE>{});
    }
}

// The residual's W values of a row from column n on (zeros without one).
template <typename T, int W>
__device__ __forceinline__ void residual_of(const LinearArgs& a, int64_t row, int n, float (&r)[W]) {
    const bool in = a.residual && row < a.m;
    load_floats<T, W>(static_cast<const T*>(a.residual) + (in ? row * a.ldr + n : 0),
                      in ? a.n - n : 0, r);
}

// W consecutive results of a row: bias, the value before the activation, the
// activation, the residual.
template <typename T, int ACT, int W>
__device__ __forceinline__ void finish(const LinearArgs& a, int64_t row, int n,
                                       const float (&sum)[W], const float (&bias)[W],
                                       const float (&r)[W]) {
    float v[W];
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] = sum[e] + bias[e];
    if (a.pre) store_floats<T, W>(static_cast<T*>(a.pre) + row * a.ldp + n, a.n - n, v);
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] = act_of<ACT>(v[e]) + r[e];
    store_floats<T, W>(static_cast<T*>(a.y) + row * a.ldy + n, a.n - n, v);
}

// fn(row, column, W sums, W values) for a wavefront's sums from row m0, column n0
// on.  Lane (q, r) holds row r of a tile, columns 4 q .. 4 q + 3; 16 rows at a time
// go through `lds` (16 (16 NJ + 4) floats of the wavefront's own), so that memory is
// reached 16 bytes a lane and whole lines a row.  ahead(row, column, values) loads
// the values, 16 rows before they are used.
template <int W, int MI, int NJ, typename P, typename F>
__device__ __forceinline__ void each_sums(const LinearArgs& a, int m0, int n0, int lane,
                                          const v4f (&acc)[MI][NJ], float* lds, P&& ahead,
                                          F&& fn) {
    constexpr int kStride = NJ * 16 + 4, L = NJ * 16 / W, R = 64 / L, N = 16 / R;
    static_assert(L <= 64 && 16 % R == 0, "lanes of a row");
    const int q = lane >> 4, r = lane & 15, row = lane / L, col = lane % L * W;
    float next[N][W];
#pragma unroll
    for (int p = 0; p < N; ++p) ahead(m0 + p * R + row, n0 + col, next[p]);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
            *reinterpret_cast<v4f*>(lds + r * kStride + j * 16 + 4 * q) = acc[i][j];
        float now[N][W];
#pragma unroll
        for (int p = 0; p < N; ++p) {
#pragma unroll
            for (int e = 0; e < W; ++e) now[p][e] = next[p][e];
            if (i + 1 < MI) ahead(m0 + (i + 1) * 16 + p * R + row, n0 + col, next[p]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int p = 0; p < N; ++p) {
            float v[W];
#pragma unroll
            for (int c = 0; c < W; c += 4) {
                const v4f f = *reinterpret_cast<const v4f*>(lds + (p * R + row) * kStride + col + c);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[c + e] = f[e];
            }
            const int m = m0 + i * 16 + p * R + row;
            if (m < a.m) fn(m, n0 + col, v, now[p]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// PLAIN: a product without an epilogue.  Every wavefront is past its reads of the
// tiles, whose place lds is.
template <typename T, bool PLAIN, int MI, int NJ>
__device__ __forceinline__ void store_sums(const LinearArgs& a, int part, int m0, int n0, int lane,
                                           const v4f (&acc)[MI][NJ], float* lds) {
    constexpr int W = kVec<T>;
    if (a.part) {
        auto none = [](int, int, float(&)[4]) {};
        each_sums<4>(a, m0, n0, lane, acc, lds, none,
                     [&](int m, int n, const float (&v)[4], const float(&)[4]) {
            float* to = a.part + (static_cast<int64_t>(part) * a.m + m) * a.n;
            store_floats<float, 4>(to + n, a.n - n, v);
        });
        return;
    }
    if (PLAIN || (a.act == TG_EPI_NONE && !a.bias && !a.residual && !a.pre)) {
        auto none = [](int, int, float(&)[W]) {};
        each_sums<W>(a, m0, n0, lane, acc, lds, none,
                     [&](int m, int n, const float (&v)[W], const float(&)[W]) {
            store_floats<T, W>(static_cast<T*>(a.y) + m * a.ldy + n, a.n - n, v);
        });
        return;
    }
    if constexpr (PLAIN) return;
    float bias[W] = {};
    if (a.bias) {
        const int n = n0 + lane % (NJ * 16 / W) * W;
        load_floats<T, W>(static_cast<const T*>(a.bias) + n, a.n - n, bias);
    }
    auto residual = [&](int m, int n, float (&r)[W]) { residual_of<T, W>(a, m, n, r); };
    with_act(a.act, [&](auto act) {
        each_sums<W>(a, m0, n0, lane, acc, lds, residual,
                     [&](int m, int n, const float (&v)[W], const float (&r)[W]) {
            finish<T, decltype(act)::value>(a, m, n, v, bias, r);
        });
    });
}

// y = the epilogue of the parts' sums: Y threads take every Y-th part of four
// results, whose sums are added in order.  Where more parts come, the sum takes the
// place of the first part, which the thread that stores it has read.  Bound by
// reading the parts: 4,000 x 2,048 in two 19.4 us.
template <typename T, int Y>
__global__ __launch_bounds__(256) void join_kernel(LinearArgs a) {
    constexpr int X = 256 / Y;
    __shared__ float sums[Y > 1 ? Y - 1 : 1][X][4];
    const int x = threadIdx.x % X, y = threadIdx.x / X;
    const uint32_t chunks = (static_cast<uint32_t>(a.n) + 3) / 4;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * X + x;
    const int64_t row = t / chunks;
    const int n = static_cast<int>(t - row * chunks) * 4;
    const int64_t size = static_cast<int64_t>(a.m) * a.n;
    const float* p = a.part + row * a.n + n;
    float s[4] = {}, r[4] = {};
    if (row < a.m) {
        if (y == 0) residual_of<T, 4>(a, row, n, r);
#pragma unroll 8
        for (int i = y; i < a.parts; i += Y) {
            float v[4];
            load_floats<float, 4>(p + i * size, a.n - n, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += v[e];
        }
    }
    if constexpr (Y > 1) {
        if (y > 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[y - 1][x][e] = s[e];
        }
        __syncthreads();
        if (y > 0) return;
#pragma unroll
        for (int i = 0; i < Y - 1; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += sums[i][x][e];
    }
    if (row >= a.m) return;
    if (a.more) {
        store_floats<float, 4>(a.part + row * a.n + n, a.n - n, s);
        return;
    }
    float bias[4] = {};
    if (a.bias) load_floats<T, 4>(static_cast<const T*>(a.bias) + n, a.n - n, bias);
    with_act(a.act, [&](auto act) { finish<T, decltype(act)::value>(a, row, n, s, bias, r); });
}

// ---------------------------------------------------------------------------
// One operand's side of the tiles: R rows (of X) or columns (of W) from `first`
// on of `count`, the contraction from k0 to k1.
// ---------------------------------------------------------------------------
template <typename T, int R, bool ACROSS, int CHUNKS, int THREADS>
struct Side {
    static constexpr int Z = sizeof(T);
    const T* base;
    int64_t ld;
    int left;          // of count
    int k1;
    int k_held;        // (through registers) where the tile held begins
    int maj[CHUNKS], min[CHUNKS];
    uint32_t offset[CHUNKS];
    v4u held[CHUNKS];
    __device__ __forceinline__ Side(const void* p, int64_t ld_, int first, int count, int k1_)
        : ld(ld_), left(count - first), k1(k1_) {
        base = static_cast<const T*>(p) + (ACROSS ? first : first * ld);
#pragma unroll
        for (int t = 0; t < CHUNKS; ++t) {
            chunk_place<T, R, ACROSS>(t * THREADS + static_cast<int>(threadIdx.x), &maj[t],
                                      &min[t]);
            const bool in = (ACROSS ? min[t] : maj[t]) < left;
            offset[t] = in ? static_cast<uint32_t>(Z * (maj[t] * ld + min[t])) : kOutside;
        }
    }
    // The tile from contraction value k0 on, straight to LDS.  What lies past k1
    // is 0: across, past the buffer (which ends with its last row's columns) or
    // past k1; along, whole chunks past it, and the one that k1 ends in by registers.
    __device__ __forceinline__ void direct(int k0, char* lds, int wave) {
        const auto buf =
            ACROSS ? buffer_of(base + k0 * ld, Z * ((k1 - k0 - 1) * ld + left))
                   : buffer_of(base + k0, kDirectBytes);
        const bool part = k0 + kDepth<T> > k1;
        const bool split = !ACROSS && part && (k1 - k0) % kVec<T> != 0;
#pragma unroll
        for (int t = 0; t < CHUNKS; ++t) {
            const int k = k0 + (ACROSS ? maj[t] : min[t]);
            if (split) {
                const bool out = offset[t] == kOutside;
                const T* p = reinterpret_cast<const T*>(
                    reinterpret_cast<const char*>(base + k0) + (out ? 0 : offset[t]));
                *reinterpret_cast<v4u*>(lds + (t * THREADS + threadIdx.x) * 16) =
                    load_chunk(p, out ? 0 : k1 - k);
            } else {
                load_to_lds(buf, lds + (t * THREADS + wave * 64) * 16,
                            part && k >= k1 ? kOutside : offset[t]);
            }
        }
    }
    // The same through registers: chunk by chunk from rows that there are, one that the
    // row's values (along: k1) end in from the last kVec of them, so that no branch
    // stands between the loads; put() moves and clears what that left wrong.  (With
    // a branch for each chunk's length every load waited for the one before: bf16
    // 2,805 x 1,973 both across, contraction 28,511, 2,539 us -> 791.)  Rows and columns past
    // the last hold anything: their results are not stored.
    __device__ __forceinline__ void fetch(int k0) {
        constexpr int VEC = kVec<T>;
        const int n = ACROSS ? left : k1;
        k_held = k0;
        if (n < VEC) {
#pragma unroll
            for (int t = 0; t < CHUNKS; ++t) {
                const int k = k0 + (ACROSS ? maj[t] : min[t]);
                const int at = ACROSS ? min[t] : maj[t];
                const int64_t most = ACROSS ? (k < k1 ? left - at : 0) : (at < left ? k1 - k : 0);
                const int64_t from = most <= 0 ? 0 : ACROSS ? k * ld + at : at * ld + k;
                held[t] = load_chunk(base + from, most);
            }
            return;
        }
        typedef T Whole __attribute__((ext_vector_type(VEC)));
#pragma unroll
        for (int t = 0; t < CHUNKS; ++t) {
            const int row = ACROSS ? smaller(k0 + maj[t], k1 - 1) : smaller(maj[t], left - 1);
            const int at = smaller(ACROSS ? min[t] : k0 + min[t], n - VEC);
            held[t] = __builtin_bit_cast(
                v4u, static_cast<Whole>(
                         *reinterpret_cast<const typename Pack<T, VEC>::V*>(base + row * ld + at)));
        }
    }
    __device__ __forceinline__ void put(char* lds) {
        constexpr int VEC = kVec<T>;
        const int n = ACROSS ? left : k1;
        if (n >= VEC && (k_held + kDepth<T> > k1 || left < R)) {
#pragma unroll
            for (int t = 0; t < CHUNKS; ++t) {
                const int past = (ACROSS ? min[t] : k_held + min[t]) - (n - VEC);
                if (past > 0) held[t] = without_first(held[t], past);
                if (ACROSS && k_held + maj[t] >= k1) held[t] = v4u{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int t = 0; t < CHUNKS; ++t)
            *reinterpret_cast<v4u*>(lds + (t * THREADS + threadIdx.x) * 16) = held[t];
    }
    static __device__ __forceinline__ int smaller(int a, int b) { return a < b ? a : b; }
    // v without its first s values, zeros behind the others.
    static __device__ __forceinline__ v4u without_first(v4u v, int s) {
        typedef unsigned __int128 Bits;
        return __builtin_bit_cast(
            v4u, s >= kVec<T> ? Bits(0) : __builtin_bit_cast(Bits, v) >> (8 * Z * s));
    }
};

// Part, row tile and column tile of this workgroup; false past the last.
__device__ __forceinline__ bool place_of(const LinearArgs& a, int* part, uint32_t* mt,
                                         uint32_t* nt) {
    const uint32_t per = 8 * ((a.mt * a.nt + 7) / 8);
    *part = static_cast<int>(blockIdx.x / per);
    return tile_of(blockIdx.x % per, a.mt, a.nt, mt, nt);
}

// (Wavefronts a SIMD that floats' tiles of 64 x 128 are compiled for: one register
// more left two, 232,965 x 256 x 256 347 us against 332.)
template <typename T, typename S>
constexpr int kMinWaves = sizeof(T) == 4 && S::kM * S::kN == 8192 ? 3 : 1;

// A tile of S::kM x S::kN results in the registers of 256 threads, its operands by two
// tiles of LDS in turn.  Bound by the matrix instructions: floats, whose instruction
// has an eighth of the rate, and beside them by the results: 232,965 x 256 x 256 forward
// 380 us with residual, pre and y, 0.95 GB (80 TFLOP/s; 289 with bias alone, 106), its
// d w^T 322 (95), its x^T d 317 (96).  They are busy for 77% of the cycles, at the 2.1
// GHz that their power leaves.
template <typename T, typename S, bool AX, bool AW, bool DIRECT>
__global__ __launch_bounds__(S::kThreads, (kMinWaves<T, S>)) void linear_kernel(LinearArgs a) {
    __shared__ __attribute__((aligned(16))) char a0[S::kM * kRowBytes];
    __shared__ __attribute__((aligned(16))) char b0[S::kN * kRowBytes];
    __shared__ __attribute__((aligned(16))) char a1[S::kM * kRowBytes];
    __shared__ __attribute__((aligned(16))) char b1[S::kN * kRowBytes];
    int part;
    uint32_t mt, nt;
    if (!place_of(a, &part, &mt, &nt)) return;
    const int m0 = static_cast<int>(mt) * S::kM, n0 = static_cast<int>(nt) * S::kN;
    const int k0 = part * a.unit, k1 = a.k - k0 > a.unit ? k0 + a.unit : a.k;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / S::kWC * S::kMI * 16, wn = wave % S::kWC * S::kNJ * 16;
    const int tiles = (k1 - k0 + kDepth<T> - 1) / kDepth<T>;
    Side<T, S::kM, AX, S::kCA, S::kThreads> xs(a.x, a.ldx, m0, a.m, k1);
    Side<T, S::kN, AW, S::kCB, S::kThreads> ws(a.w, a.ldw, n0, a.n, k1);
    Sums<T, S::kMI, S::kNJ> acc;
    const Reader<T, S::kM, AX, S::kMI> ra(wm, lane);
    const Reader<T, S::kN, AW, S::kNJ> rb(wn, lane);
    auto compute = [&](const char* la, const char* lb) { multiply<T, S>(ra, rb, la, lb, acc.now); };
    auto join = [&] { acc.join(); };
    auto load = [&](int kt, char* la, char* lb) {
        const int k = k0 + kt * kDepth<T>;
        if constexpr (DIRECT) {
            xs.direct(k, la, wave);
            ws.direct(k, lb, wave);
        } else {
            xs.fetch(k);
            ws.fetch(k);
        }
    };
    auto store = [&](char* la, char* lb) {
        xs.put(la);
        ws.put(lb);
    };
    pipeline<DIRECT>(tiles, a0, b0, a1, b1, load, store, compute, join);
    __syncthreads();
    static_assert(S::kThreads == 256, "a place for each wavefront");
    char* const own = wave == 0 ? a0 : wave == 1 ? b0 : wave == 2 ? a1 : b1;
    // (both across: the weights' gradient)
    store_sums<T, AX>(a, part, m0 + wm, n0 + wn, lane, acc.result(),
                      reinterpret_cast<float*>(own));
}

// The large tile (tiles.hpp): 16-bit operands that can be loaded directly, in
// whole chunks (along the contraction, its length % 8 = 0; across it, the rows or
// columns % 8 = 0).  One workgroup a CU, so that nothing runs beside its first loads
// and its results: bf16 16,384 rows, 2,048 to 8,192, with GELU, pre and y 605 us (909
// TFLOP/s), its d w^T 466 (1,180), its x^T d 490 (1,122).
template <typename T, bool AX, bool AW>
__global__ __launch_bounds__(kRingThreads) void linear_ring_kernel(LinearArgs a) {
    TG_RING_LDS;
    int part;
    uint32_t mt, nt;
    if (!place_of(a, &part, &mt, &nt)) return;
    const int m0 = static_cast<int>(mt) * 256, n0 = static_cast<int>(nt) * 256;
    const int kb = part * a.unit, k1 = a.k - kb > a.unit ? kb + a.unit : a.k;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / 4 * 128, wn = wave % 4 * 64;
    const T* xb = static_cast<const T*>(a.x) + (AX ? m0 : m0 * a.ldx);
    const T* wb = static_cast<const T*>(a.w) + (AW ? n0 : n0 * a.ldw);
    uint32_t ao[2], bo[2];
    int ak[2], bk[2];  // the chunks' places along the contraction
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        int major, minor;
        part_place<AX>(t * kRingThreads + tid, &major, &minor);
        ak[t] = AX ? major : minor;
        ao[t] = m0 + (AX ? minor : major) < a.m ? static_cast<uint32_t>(2 * (major * a.ldx + minor))
                                                : kOutside;
        part_place<AW>(t * kRingThreads + tid, &major, &minor);
        bk[t] = AW ? major : minor;
        bo[t] = n0 + (AW ? minor : major) < a.n ? static_cast<uint32_t>(2 * (major * a.ldw + minor))
                                                : kOutside;
    }
    auto load = [&](int u, char* la, char* lb) {
        const int k0 = kb + u * kStep;
        // What lies behind k1 is 0: where both operands run across, past buffers
        // that end with it (no registers for the chunks' places; 11 were spilled).
        constexpr bool kEnds = AX && AW;
        const int64_t rows = k1 - k0, most = rows > 0 ? kDirectBytes : 0;
        const auto xbuf = buffer_of(AX ? xb + k0 * a.ldx : xb + k0,
                                    kEnds && rows > 0 ? 2 * ((rows - 1) * a.ldx + a.m - m0) : most);
        const auto wbuf = buffer_of(AW ? wb + k0 * a.ldw : wb + k0,
                                    kEnds && rows > 0 ? 2 * ((rows - 1) * a.ldw + a.n - n0) : most);
        const bool part = !kEnds && k0 + kStep > k1;
#pragma unroll
        for (int t = 0; t < 2; ++t)
            load_to_lds(xbuf, la + (t * kRingThreads + wave * 64) * 16,
                        part && k0 + ak[t] >= k1 ? kOutside : ao[t]);
#pragma unroll
        for (int t = 0; t < 2; ++t)
            load_to_lds(wbuf, lb + (t * kRingThreads + wave * 64) * 16,
                        part && k0 + bk[t] >= k1 ? kOutside : bo[t]);
    };
    v4f acc[8][4] = {};
    PartReader<AX, 8, true> ra(wm, lane);
    PartReader<AW, 4, AX> rb(wn, lane);
    ring<T>((k1 - kb + kStep - 1) / kStep, ra, rb, [](int) {}, load, a0, b0, a1, b1, a2, b2, a3, b3,
            acc);
    __syncthreads();
    char* const own = wave < 4 ? (wave == 0 ? a0 : wave == 1 ? b0 : wave == 2 ? a1 : b1)
                               : (wave == 4 ? a2 : wave == 5 ? b2 : wave == 6 ? a3 : b3);
    store_sums<T, AX>(a, part, m0 + wm, n0 + wn, lane, acc, reinterpret_cast<float*>(own));
}

using Medium = Shape<128, 128, 2, 2>;
using Small = Shape<64, 64, 2, 2>;
using Few = Shape<32, 128, 1, 4>;
using Wide = Shape<64, 128, 2, 2>;
using Tall = Shape<128, 64, 2, 2>;

// ---------------------------------------------------------------------------
// Up to 16 rows of x, w's rows along the contraction: 16 columns by the 16 wavefronts of
// a workgroup, which take turns of 128 bytes of the contraction, loaded straight to
// the matrix instructions' operands; their sums are added in order.  Bound by
// reading w once: 1 x 4,096 x 4,096 bf16 8.9 us (3.8 TB/s) where other work ran between;
// 7.2 after itself, when part of the 32 MB may still be in the last-level cache.
// ---------------------------------------------------------------------------
constexpr int kFewWaves = 16;

template <typename T>
__global__ __launch_bounds__(kFewWaves * 64) void few_kernel(LinearArgs a) {
    constexpr int VEC = kVec<T>, kTurn = 8 * VEC;
    __shared__ v4f sums[kFewWaves][64];
    const int lane = threadIdx.x & 63, q = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = static_cast<int>(blockIdx.x) * 16;
    // rows and columns past the last: the last one again, and not stored
    const T* w = static_cast<const T*>(a.w) + (n0 + r < a.n ? n0 + r : a.n - 1) * a.ldw + q * VEC;
    const T* x = static_cast<const T*>(a.x) + (r < a.m ? r : a.m - 1) * a.ldx + q * VEC;
    v4f acc = {};
    auto turns = [&](int k, auto count, auto whole) {
        constexpr int N = decltype(count)::value;
        Frag fw[N][2], fx[N][2];
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = k + u * kFewWaves * kTurn + h * 4 * VEC;
                const int64_t left = decltype(whole)::value ? VEC : a.k - at - q * VEC;
                fw[u][h].u = load_chunk(w + (left > 0 ? at : 0), left);
                fx[u][h].u = load_chunk(x + (left > 0 ? at : 0), left);
            }
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) acc = mfma<T>(fw[u][h], fx[u][h], acc);
    };
    constexpr int kMany = 4;
    using std::integral_constant;
    int k = wave * kTurn;
    for (; k + (kMany - 1) * kFewWaves * kTurn + kTurn <= a.k; k += kMany * kFewWaves * kTurn)
        turns(k, integral_constant<int, kMany>{}, std::true_type{});
    for (; k < a.k; k += kFewWaves * kTurn)
        turns(k, integral_constant<int, 1>{}, std::false_type{});
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
    v4f s = sums[0][lane];
#pragma unroll
    for (int v = 1; v < kFewWaves; ++v) s += sums[v][lane];
    const int n = n0 + 4 * q;
    if (r >= a.m) return;
    float bias[4] = {}, res[4];
    if (a.bias) load_floats<T, 4>(static_cast<const T*>(a.bias) + n, a.n - n, bias);
    residual_of<T, 4>(a, r, n, res);
    const float v[4] = {s[0], s[1], s[2], s[3]};
    with_act(a.act, [&](auto act) { finish<T, decltype(act)::value>(a, r, n, v, bias, res); });
}

template <typename T>
void launch_few(const LinearArgs& a, hipStream_t s) {
    const unsigned grid = grid_of("linear", ceil_div(a.n, 16), kFewWaves * 64);
    few_kernel<T><<<grid, kFewWaves * 64, 0, s>>>(a);
    TG_LAUNCH_CHECK();
}

template <typename T, bool AX, bool AW>
void launch_tiles(const LinearArgs& a, const LinearPlan& p, int64_t parts, bool direct,
                  hipStream_t s) {
    const int64_t per = 8 * ceil_div(p.mt * p.nt, 8);
    const unsigned grid = grid_of("linear", per * parts, kRingThreads);
    auto tiled = [&](auto shape) {
        using S = decltype(shape);
        linear_kernel<T, S, AX, AW, true><<<grid, S::kThreads, 0, s>>>(a);
    };
    auto by_registers = [&](auto shape) {
        using S = decltype(shape);
        linear_kernel<T, S, AX, AW, false><<<grid, S::kThreads, 0, s>>>(a);
    };
    constexpr bool kHalf = sizeof(T) == 2;
    if (!direct) {
        if (p.em == 64)
            by_registers(Small{});
        else if constexpr (kHalf)
            by_registers(Medium{});
    } else if (p.em == 32) {
        tiled(Few{});
    } else if (p.em == 64) {
        p.en == 64 ? tiled(Small{}) : tiled(Wide{});
    } else if (p.en == 64) {
        tiled(Tall{});
    } else if constexpr (kHalf) {
        if (p.em == 128)
            tiled(Medium{});
        else
            linear_ring_kernel<T, AX, AW><<<grid, kRingThreads, 0, s>>>(a);
    }
    TG_LAUNCH_CHECK();
}

// A product, p.kept parts at a time: the first of them is the sum of all before.  (fp32
// 8,192 x 8,192, contraction 1,000,000: 1 GB of sums where 62 parts are 16.6, 1.00 s.)
template <typename T, bool AX, bool AW>
void launch_product(LinearArgs& a, const LinearPlan& p, bool direct, hipStream_t s) {
    a.mt = static_cast<uint32_t>(p.mt);
    a.nt = static_cast<uint32_t>(p.nt);
    a.unit = static_cast<int>(p.unit);
    if (p.parts == 1) return launch_tiles<T, AX, AW>(a, p, 1, direct, s);
    const int64_t size = static_cast<int64_t>(a.m) * a.n;
    for (int64_t first = 0; first < p.parts;) {
        const int64_t before = first > 0 ? 1 : 0;
        const int64_t now = std::min(p.kept - before, p.parts - first), k0 = first * p.unit;
        LinearArgs b = a;
        b.x = static_cast<const T*>(a.x) + (AX ? k0 * a.ldx : k0);
        b.w = static_cast<const T*>(a.w) + (AW ? k0 * a.ldw : k0);
        b.k = static_cast<int>(std::min(a.k - k0, now * p.unit));
        b.part = a.part + before * size;
        launch_tiles<T, AX, AW>(b, p, now, direct, s);
        first += now;
        b.part = a.part;
        b.parts = static_cast<int>(before + now);
        b.more = first < p.parts;
        const int64_t threads = a.m * ceil_div(a.n, 4);
        auto join = [&](auto kernel, int64_t results) {
            kernel<<<grid_of("linear", ceil_div(threads, results), 256), 256, 0, s>>>(b);
        };
        b.parts > 48  ? join(join_kernel<T, 32>, 8)
        : b.parts > 8 ? join(join_kernel<T, 8>, 32)
                      : join(join_kernel<T, 1>, 256);
        TG_LAUNCH_CHECK();
    }
}

// ---------------------------------------------------------------------------
// d = dy act'(pre) and its columns' sums: a workgroup takes a.rows rows of up
// to 32 VEC columns, 8 rows or more at a time; the parts' sums are added in order by
// columns_kernel.  ACT NONE: the sums alone.  Bound by its two reads and one write:
// 232,965 x 256 fp32 135 us (5.3 TB/s), 16,384 x 8,192 bf16 with GELU 180 (4.5).
// ---------------------------------------------------------------------------
template <typename T, int ACT>
__global__ __launch_bounds__(256) void act_backward_kernel(ActArgs a) {
    constexpr int VEC = kVec<T>;
    __shared__ float join[256 * VEC];
    const int wide = 1 << a.log_wide, high = 256 >> a.log_wide;
    const int x = threadIdx.x & (wide - 1), y = threadIdx.x >> a.log_wide;
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * wide + x) * VEC;
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * a.rows;
    const int64_t r1 = a.m - r0 > a.rows ? r0 + a.rows : a.m;
    float s[VEC] = {};
    for (int64_t r = r0 + y; r < r1;) {  // chains of 64 rows
        const int64_t stop = r1 - r > 64 * high ? r + 64 * high : r1;
        float now[VEC] = {};
#pragma unroll 4
        for (; r < stop; r += high) {
            float v[VEC], p[VEC];
            load_floats<T, VEC>(static_cast<const T*>(a.dy) + r * a.lddy + c, a.n - c, v);
            if constexpr (ACT != TG_EPI_NONE) {
                load_floats<T, VEC>(static_cast<const T*>(a.pre) + r * a.ldp + c, a.n - c, p);
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[e] *= slope_of<ACT>(p[e]);
                if (a.d) store_floats<T, VEC>(static_cast<T*>(a.d) + r * a.ldd + c, a.n - c, v);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) now[e] += v[e];
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[e] += now[e];
    }
    if (!a.part) return;
#pragma unroll
    for (int e = 0; e < VEC; ++e) join[(y * wide + x) * VEC + e] = s[e];
    __syncthreads();
    for (int i = threadIdx.x; i < wide * VEC; i += 256) {
        const int64_t at = static_cast<int64_t>(blockIdx.x) * wide * VEC + i;
        float v = 0.0f;
        for (int w = 0; w < high; ++w) v += join[w * wide * VEC + i];
        if (at < a.n) a.part[static_cast<int64_t>(blockIdx.y) * a.n + at] = v;
    }
}

template <typename T>
__global__ __launch_bounds__(1024) void columns_kernel(const float* __restrict__ part, int64_t n,
                                                       int64_t parts, T* __restrict__ out) {
    __shared__ float join[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
    float s = 0.0f;
    if (c < n) {
#pragma unroll 8
        for (int64_t p = wave; p < parts; p += 16) s += part[p * n + c];
    }
    join[wave][lane] = s;
    __syncthreads();
    if (wave > 0 || c >= n) return;
#pragma unroll
    for (int w = 1; w < 16; ++w) s += join[w][lane];
    out[c] = static_cast<T>(s);
}

template <typename T>
void launch_act(const ActArgs& a, int act, hipStream_t s) {
    const int64_t cols = ceil_div(a.n, kVec<T> << a.log_wide), parts = ceil_div(a.m, a.rows);
    require(cols * 256 < (int64_t(1) << 32) && parts < 65536, "linear_backward: too many elements");
    const dim3 grid(static_cast<unsigned>(cols), static_cast<unsigned>(parts));
    if (act == TG_EPI_NONE) act_backward_kernel<T, TG_EPI_NONE><<<grid, 256, 0, s>>>(a);
    if (act == TG_EPI_RELU) act_backward_kernel<T, TG_EPI_RELU><<<grid, 256, 0, s>>>(a);
    if (act == TG_EPI_ELU) act_backward_kernel<T, TG_EPI_ELU><<<grid, 256, 0, s>>>(a);
    if (act == TG_EPI_GELU) act_backward_kernel<T, TG_EPI_GELU><<<grid, 256, 0, s>>>(a);
    if (act == TG_EPI_SILU) act_backward_kernel<T, TG_EPI_SILU><<<grid, 256, 0, s>>>(a);
    TG_LAUNCH_CHECK();
}

template <typename T>
void launch_columns(const float* part, int64_t n, int64_t parts, void* out, hipStream_t s) {
    columns_kernel<T><<<grid_of("linear_backward", ceil_div(n, 64), 1024), 1024, 0, s>>>(
        part, n, parts, static_cast<T*>(out));
    TG_LAUNCH_CHECK();
}

}  // namespace

// What one of the .hip files compiles.
#define TG_LINEAR_OF(T)                                                                          \
    template <>                                                                                  \
    void linear_product<T>(LinearArgs & a, const LinearPlan& p, bool ax, bool aw, bool direct,    \
                           hipStream_t s) {                                                      \
        if (p.em == 0)                                                                           \
            launch_few<T>(a, s);                                                                 \
        else if (ax)                                                                             \
            launch_product<T, true, true>(a, p, direct, s);                                      \
        else if (aw)                                                                             \
            launch_product<T, false, true>(a, p, direct, s);                                     \
        else                                                                                     \
            launch_product<T, false, false>(a, p, direct, s);                                    \
    }                                                                                            \
    template <>                                                                                  \
    void linear_act<T>(const ActArgs& a, int act, hipStream_t s) {                               \
        launch_act<T>(a, act, s);                                                                \
    }                                                                                            \
    template <>                                                                                  \
    void linear_columns<T>(const float* part, int64_t n, int64_t parts, void* out,               \
                           hipStream_t s) {                                                      \
        launch_columns<T>(part, n, parts, out, s);                                               \
    }

}  // namespace tg
