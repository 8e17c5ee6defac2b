// grouped.hip -- products grouped by expert or node type, with ragged groups.
//
// Every product is cut into row tiles of its own groups (find_tile), so no
// group's size is known to the host and nothing waits for it.  16-bit types go
// through v_mfma_f32_16x16x32, floats through v_mfma_f32_16x16x4f32 (tiles.hpp);
// sums are fp32 and rounded once.
#include "grouped.hpp"

#include <string>

#include "tiles.hpp"
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
    const void* bias;
    int epi;
    void* y;
    int64_t ldy;
    uint32_t mt, nt;  // row tiles (most) and column tiles
    const void* dy;   // gradient of w
    int64_t lddy;
    void* dw;
    void* dbias;
    int unit;    // rows of a part of a group, 0: whole groups
    int slots;   // most parts of groups of several
    float* part;  // [slots][k][n] sums of those parts, [slots][n] of dy's
    float* part_bias;
};

// x's row for row p of the product, or -1.
__device__ __forceinline__ int64_t source_row(const GroupedArgs& a, int p) {
    const int64_t r = a.rows ? a.rows[p] : p;
    return r < 0 || r >= a.x_rows ? -1 : r;
}

// A wavefront's outputs from row p0, column n0 of group g: bias, epilogue and
// stores.  Lane (q, r) holds row r of a tile, columns 4 q .. 4 q + 3.
template <typename T, int MI, int NJ>
__device__ __forceinline__ void store_outputs(const GroupedArgs& a, int g, int p0, int r1, int n0,
                                              int lane, const v4f (&acc)[MI][NJ]) {
    const int q = lane >> 4, r = lane & 15;
    float bias[NJ][4];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const int n = n0 + j * 16 + 4 * q;
        if (a.bias)
            load_floats<T, 4>(static_cast<const T*>(a.bias) + static_cast<int64_t>(g) * a.n + n,
                              a.n - n, bias[j]);
        else
            bias[j][0] = bias[j][1] = bias[j][2] = bias[j][3] = 0.0f;
    }
    with_epilogue(a.epi, [&](auto epi) {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int p = p0 + i * 16 + r;
            if (p >= r1) continue;
            T* y = static_cast<T*>(a.y) + p * a.ldy;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int n = n0 + j * 16 + 4 * q;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = grouped_epilogue<decltype(epi)::value>(acc[i][j][e], bias[j][e]);
                store_floats<T, 4>(y + n, a.n - n, v);
            }
        }
    });
}

// A wavefront's sums of dw from row k0, column n0 on: of group (or part) `part`.
template <typename T, int MI, int NJ>
__device__ __forceinline__ void store_gradient(const GroupedArgs& a, bool split, int part, int k0,
                                               int n0, int lane, const v4f (&acc)[MI][NJ]) {
    const int q = lane >> 4, r = lane & 15;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int k = k0 + i * 16 + r;
        if (k >= a.k) continue;
        const int64_t row = (static_cast<int64_t>(part) * a.k + k) * a.n;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int n = n0 + j * 16 + 4 * q;
            const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
            if (split)
                store_floats<float, 4>(a.part + row + n, a.n - n, v);
            else
                store_floats<T, 4>(static_cast<T*>(a.dw) + row + n, a.n - n, v);
        }
    }
}

template <typename T, int NJ>
__device__ __forceinline__ void store_bias_gradient(const GroupedArgs& a, bool split, int part,
                                                    int n0, int lane, const v4f (&sum)[NJ]) {
    const int q = lane >> 4, r = lane & 15;
    if (r != 0) return;
    const int64_t row = static_cast<int64_t>(part) * a.n;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const int n = n0 + j * 16 + 4 * q;
        const float v[4] = {sum[j][0], sum[j][1], sum[j][2], sum[j][3]};
        if (split)
            store_floats<float, 4>(a.part_bias + row + n, a.n - n, v);
        else
            store_floats<T, 4>(static_cast<T*>(a.dbias) + row + n, a.n - n, v);
    }
}

// ---------------------------------------------------------------------------
// BM x BN outputs by WR x WC wavefronts, two tiles of both operands in LDS: while
// the matrix instructions read one, the other is loaded.  The wavefront's outputs
// are computed transposed (columns of w as the rows of the instruction), so a
// lane holds four consecutive columns of y.
//
// DIRECT: the tiles come by loads that write to LDS; else through registers,
// for 16-bit operands of odd rows or places and those that reach past 2 GB.
// ---------------------------------------------------------------------------
// The products of one tile pair.
template <typename T, typename S, typename RA, typename RB>
__device__ __forceinline__ void multiply(const RA& ra, const RB& rb, const char* la, const char* lb,
                                         Acc<S>& acc) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        Frag b[S::kNJ];
#pragma unroll
        for (int j = 0; j < S::kNJ; ++j) b[j] = rb.read(lb, j, s);
#pragma unroll
        for (int i = 0; i < S::kMI; ++i) {
            const Frag a = ra.read(la, i, s);
#pragma unroll
            for (int j = 0; j < S::kNJ; ++j) acc[i][j] = mfma<T>(b[j], a, acc[i][j]);
        }
    }
}

// Sums of floats keep their digits: kSumTiles tiles (256 values) are one chain in
// `now`, and the chains' sums another in `all`.  (One chain of n values is off by up
// to n 2^-24 of the sum of sizes: a training step of 233K rows of 7 types, 602 x
// 256, was 8.9e-7 off with it and is 3.1e-7; 2.27 -> 2.31 ms.)  16-bit products
// are one chain, to which the instructions add eight at a time: n of one sign are
// off by n 2^-27 of their sum at most, n^(1/2) 2^-25 or so of random ones; the
// result's own rounding is 2^-9 or 2^-12.
template <typename T, int N, int M>
struct Sums {
    v4f now[N][M] = {}, all[sizeof(T) == 4 ? N : 1][sizeof(T) == 4 ? M : 1] = {};
    __device__ __forceinline__ void join() {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int j = 0; j < M; ++j) {
                    all[i][j] += now[i][j];
                    now[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
                }
        }
    }
    __device__ __forceinline__ auto& result() {
        join();
        if constexpr (sizeof(T) == 4)
            return all;
        else
            return now;
    }
};

template <typename T, typename S, bool ALONG_W, bool DIRECT>
__global__ __launch_bounds__(S::kThreads) void grouped_kernel(GroupedArgs a) {
    __shared__ __attribute__((aligned(16))) char a0[S::kM * kRowBytes];
    __shared__ __attribute__((aligned(16))) char b0[S::kN * kRowBytes];
    __shared__ __attribute__((aligned(16))) char a1[S::kM * kRowBytes];
    __shared__ __attribute__((aligned(16))) char b1[S::kN * kRowBytes];
    constexpr int Z = sizeof(T);
    uint32_t mt, ntile;
    if (!tile_of(blockIdx.x, count_tiles(a.offsets, a.groups, a.m, S::kM), a.nt, &mt, &ntile))
        return;
    int g, r0, r1;
    if (!find_tile(a.offsets, a.groups, a.m, S::kM, static_cast<int>(mt), &g, &r0, &r1)) return;
    const int n0 = static_cast<int>(ntile) * S::kN;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / S::kWC * S::kMI * 16, wn = wave % S::kWC * S::kNJ * 16;
    const T* x = static_cast<const T*>(a.x);
    const T* w = static_cast<const T*>(a.w) + g * a.w_stride;
    const int tiles = (a.k + kDepth<T> - 1) / kDepth<T>;

    // chunk t of this thread: its row and first value of x's tile, ...
    int ac[S::kCA], bmaj[S::kCB], bmin[S::kCB];
    int64_t ar[S::kCA];  // x's row, -1: zeros
#pragma unroll
    for (int t = 0; t < S::kCA; ++t) {
        int row;
        chunk_place<T, S::kM, false>(t * S::kThreads + tid, &row, &ac[t]);
        ar[t] = r0 + row < r1 ? source_row(a, r0 + row) : -1;
    }
#pragma unroll
    for (int t = 0; t < S::kCB; ++t)
        chunk_place<T, S::kN, !ALONG_W>(t * S::kThreads + tid, &bmaj[t], &bmin[t]);

    Sums<T, S::kMI, S::kNJ> acc;
    const Reader<T, S::kM, false, S::kMI> ra(wm, lane);
    const Reader<T, S::kN, !ALONG_W, S::kNJ> rb(wn, lane);
    auto compute = [&](const char* la, const char* lb) { multiply<T, S>(ra, rb, la, lb, acc.now); };
    auto join = [&] { acc.join(); };
    if constexpr (DIRECT) {
        // offsets from the tile's first row (gathered: x's) and w's tile
        const T* xb = a.rows ? x : x + static_cast<int64_t>(r0) * a.ldx;
        uint32_t ao[S::kCA], bo[S::kCB];
#pragma unroll
        for (int t = 0; t < S::kCA; ++t) {
            const int64_t row = a.rows ? ar[t] : ar[t] - r0;
            ao[t] = ar[t] < 0 ? kOutside : static_cast<uint32_t>(Z * (row * a.ldx + ac[t]));
        }
#pragma unroll
        for (int t = 0; t < S::kCB; ++t) {
            if (ALONG_W)
                bo[t] = n0 + bmaj[t] < a.n
                            ? static_cast<uint32_t>(Z * (bmaj[t] * a.ldw + bmin[t]))
                            : kOutside;
            else
                bo[t] = n0 + bmin[t] < a.n
                            ? static_cast<uint32_t>(Z * (bmaj[t] * a.ldw + bmin[t]))
                            : kOutside;
        }
        const T* wb = ALONG_W ? w + n0 * a.ldw : w + n0;
        // a chunk of an operand along memory that k ends in: by registers
        auto last_chunk = [&](const T* base, uint32_t offset, int64_t left, char* to) {
            const T* p = reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) +
                                                    (offset == kOutside ? 0 : offset));
            *reinterpret_cast<v4u*>(to) = load_chunk(p, offset == kOutside ? 0 : left);
        };
        auto load = [&](int kt, char* la, char* lb) {
            const int k0 = kt * kDepth<T>;
            const auto xbuf = buffer_of(xb + k0, kDirectBytes);
            // (w across memory ends with its last row's columns)
            const auto wbuf =
                ALONG_W ? buffer_of(wb + k0, kDirectBytes)
                        : buffer_of(wb + k0 * a.ldw, Z * ((a.k - k0 - 1) * a.ldw + a.n - n0));
            const bool part = k0 + kDepth<T> > a.k;  // the last tile: what lies behind k is 0
            const bool split = part && a.k % kVec<T> != 0;
#pragma unroll
            for (int t = 0; t < S::kCA; ++t) {
                if (split)
                    last_chunk(xb + k0, ao[t], a.k - k0 - ac[t],
                               la + (t * S::kThreads + tid) * 16);
                else
                    load_to_lds(xbuf, la + (t * S::kThreads + wave * 64) * 16,
                                part && k0 + ac[t] >= a.k ? kOutside : ao[t]);
            }
#pragma unroll
            for (int t = 0; t < S::kCB; ++t) {
                if (ALONG_W && split)
                    last_chunk(wb + k0, bo[t], a.k - k0 - bmin[t],
                               lb + (t * S::kThreads + tid) * 16);
                else
                    load_to_lds(wbuf, lb + (t * S::kThreads + wave * 64) * 16,
                                part && k0 + (ALONG_W ? bmin[t] : bmaj[t]) >= a.k ? kOutside
                                                                                 : bo[t]);
            }
        };
        pipeline<true>(tiles, a0, b0, a1, b1, load, [](char*, char*) {}, compute, join);
    } else {
        v4u av[S::kCA], bv[S::kCB];
        auto load = [&](int kt, char*, char*) {
            const int k0 = kt * kDepth<T>;
#pragma unroll
            for (int t = 0; t < S::kCA; ++t) {
                const int k = k0 + ac[t];
                av[t] = load_chunk(x + (ar[t] < 0 ? 0 : ar[t]) * a.ldx + k,
                                   ar[t] < 0 ? 0 : a.k - k);
            }
#pragma unroll
            for (int t = 0; t < S::kCB; ++t) {
                const int n = n0 + (ALONG_W ? bmaj[t] : bmin[t]);
                const int k = k0 + (ALONG_W ? bmin[t] : bmaj[t]);
                if (ALONG_W)
                    bv[t] = load_chunk(w + n * a.ldw + k, n < a.n ? a.k - k : 0);
                else
                    bv[t] = load_chunk(w + k * a.ldw + n, k < a.k ? a.n - n : 0);
            }
        };
        auto store = [&](char* la, char* lb) {
#pragma unroll
            for (int t = 0; t < S::kCA; ++t)
                *reinterpret_cast<v4u*>(la + (t * S::kThreads + tid) * 16) = av[t];
#pragma unroll
            for (int t = 0; t < S::kCB; ++t)
                *reinterpret_cast<v4u*>(lb + (t * S::kThreads + tid) * 16) = bv[t];
        };
        pipeline<false>(tiles, a0, b0, a1, b1, load, store, compute, join);
    }

    store_outputs<T>(a, g, r0 + wm, r1, n0 + wn, lane, acc.result());
}

// The large tile (tiles.hpp): 16-bit operands that can be loaded directly, in
// whole chunks (k % 8 = 0, across memory n % 8 = 0: a buffer that ends with w's
// last value cost the loop 600 -> 1270 us of 32 experts' 32,768 x 2048 x 4096).
template <typename T, bool ALONG_W, bool WHOLE>
__global__ __launch_bounds__(kRingThreads) void grouped_ring_kernel(GroupedArgs a) {
    TG_RING_LDS;
    uint32_t mt, ntile;
    if (!tile_of(blockIdx.x, count_tiles(a.offsets, a.groups, a.m, 256), a.nt, &mt, &ntile)) return;
    int g, r0, r1;
    if (!find_tile(a.offsets, a.groups, a.m, 256, static_cast<int>(mt), &g, &r0, &r1)) return;
    const int n0 = static_cast<int>(ntile) * 256;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / 4 * 128, wn = wave % 4 * 64;
    const T* w = static_cast<const T*>(a.w) + g * a.w_stride;
    const T* xb = static_cast<const T*>(a.x) + (a.rows ? 0 : static_cast<int64_t>(r0) * a.ldx);
    const T* wb = ALONG_W ? w + n0 * a.ldw : w + n0;
    uint32_t ao[2], bo[2];
    int ac[2], bk[2];  // the chunks' places along the contraction
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        int row, col, kk;
        part_place<false>(t * kRingThreads + tid, &row, &ac[t]);
        const int64_t src = r0 + row < r1 ? source_row(a, r0 + row) : -1;
        ao[t] = src < 0 ? kOutside
                        : static_cast<uint32_t>(2 * ((a.rows ? src : row) * a.ldx + ac[t]));
        if (ALONG_W)
            part_place<false>(t * kRingThreads + tid, &col, &kk);
        else
            part_place<true>(t * kRingThreads + tid, &kk, &col);
        bk[t] = kk;
        bo[t] = n0 + col < a.n
                    ? static_cast<uint32_t>(2 * (ALONG_W ? col * a.ldw + kk : kk * a.ldw + col))
                    : kOutside;
    }
    auto load = [&](int u, char* la, char* lb) {
        const int k0 = u * kStep;
        const int64_t size = k0 < a.k ? kDirectBytes : 0;
        const auto xbuf = buffer_of(xb + k0, size);
        const auto wbuf = buffer_of(ALONG_W ? wb + k0 : wb + k0 * a.ldw, size);
        const bool part = !WHOLE && k0 + kStep > a.k;  // what lies behind k is 0
#pragma unroll
        for (int t = 0; t < 2; ++t)
            load_to_lds(xbuf, la + (t * kRingThreads + wave * 64) * 16,
                        part && k0 + ac[t] >= a.k ? kOutside : ao[t]);
#pragma unroll
        for (int t = 0; t < 2; ++t)
            load_to_lds(wbuf, lb + (t * kRingThreads + wave * 64) * 16,
                        part && k0 + bk[t] >= a.k ? kOutside : bo[t]);
    };
    v4f acc[8][4] = {};
    PartReader<false, 8, true> ra(wm, lane);
    PartReader<!ALONG_W, 4, false> rb(wn, lane);
    ring<T>((a.k + kStep - 1) / kStep, ra, rb, [](int) {}, load, a0, b0, a1, b1, a2, b2, a3, b3, acc);
    store_outputs<T>(a, g, r0 + wm, r1, n0 + wn, lane, acc);
}

// dw_g = x_g^T dy_g and, from the workgroups of dw's first row tile, dbias: dy's
// columns times ones on the matrix units.  With a.unit a workgroup sums that
// many of a group's rows to fp32 parts, which parts_kernel adds in order: where
// the groups' own tiles are too few for the CUs (233K rows of 7 types, 602 x 256:
// 70 tiles), and the chains over 33K rows too long for fp32's digits.
template <typename T, typename S, bool DIRECT, bool BIAS>
__global__ __launch_bounds__(S::kThreads, DIRECT ? 2 : 1) void wgrad_kernel(GroupedArgs a) {
    __shared__ __attribute__((aligned(16))) char a0[S::kM * kRowBytes];
    __shared__ __attribute__((aligned(16))) char b0[S::kN * kRowBytes];
    __shared__ __attribute__((aligned(16))) char a1[S::kM * kRowBytes];
    __shared__ __attribute__((aligned(16))) char b1[S::kN * kRowBytes];
    constexpr int Z = sizeof(T);
    const uint32_t per = a.mt * a.nt;
    const int part = static_cast<int>(blockIdx.x / per);
    uint32_t mt, ntile;
    tile_of(blockIdx.x % per, a.mt, a.nt, &mt, &ntile);
    int g = part, lo, hi, slot = 0;
    if (a.unit == 0)
        group_rows(a.offsets, g, a.m, &lo, &hi);
    else if (!find_tile(a.offsets, a.groups, a.m, a.unit, part, &g, &lo, &hi, &slot))
        return;
    const int k0 = static_cast<int>(mt) * S::kM, n0 = static_cast<int>(ntile) * S::kN;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / S::kWC * S::kMI * 16, wn = wave % S::kWC * S::kNJ * 16;
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.dy);
    const int tiles = (hi - lo + kDepth<T> - 1) / kDepth<T>;

    int ap[S::kCA], ac[S::kCA], bp[S::kCB], bc[S::kCB];
#pragma unroll
    for (int t = 0; t < S::kCA; ++t)
        chunk_place<T, S::kM, true>(t * S::kThreads + tid, &ap[t], &ac[t]);
#pragma unroll
    for (int t = 0; t < S::kCB; ++t)
        chunk_place<T, S::kN, true>(t * S::kThreads + tid, &bp[t], &bc[t]);

    Sums<T, S::kMI, S::kNJ> acc;
    Sums<T, 1, BIAS ? S::kNJ : 1> sum;
    const bool sums = BIAS && mt == 0 && wm == 0;  // uniform
    const Frag one = ones<T>();
    const Reader<T, S::kM, true, S::kMI> ra(wm, lane);
    const Reader<T, S::kN, true, S::kNJ> rb(wn, lane);
    auto compute = [&](const char* la, const char* lb) {
        multiply<T, S>(ra, rb, la, lb, acc.now);
        if (BIAS && sums) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int j = 0; j < S::kNJ; ++j)
                    sum.now[0][j] = mfma<T>(rb.read(lb, j, s), one, sum.now[0][j]);
        }
    };
    auto join = [&] {
        acc.join();
        sum.join();
    };
    if constexpr (DIRECT) {
        uint32_t ao[S::kCA], bo[S::kCB];
        int idx[S::kCA];  // the next tile's gathered rows
#pragma unroll
        for (int t = 0; t < S::kCA; ++t)
            ao[t] = k0 + ac[t] < a.k ? static_cast<uint32_t>(Z * (ap[t] * a.ldx + k0 + ac[t]))
                                     : kOutside;
#pragma unroll
        for (int t = 0; t < S::kCB; ++t)
            bo[t] = n0 + bc[t] < a.n ? static_cast<uint32_t>(Z * (bp[t] * a.lddy + n0 + bc[t]))
                                     : kOutside;
        auto fetch = [&](int kt) {
#pragma unroll
            for (int t = 0; t < S::kCA; ++t) {
                const int p = lo + kt * kDepth<T> + ap[t];
                idx[t] = p < hi ? a.rows[p] : -1;
            }
        };
        if (a.rows) fetch(0);
        auto load = [&](int kt, char* la, char* lb) {
            const int p0 = lo + kt * kDepth<T>;
            const int64_t left = hi - p0;  // rows: the buffers end with them
            const auto dbuf = buffer_of(dy + p0 * a.lddy, Z * ((left - 1) * a.lddy + a.n));
            if (a.rows) {
                const auto xbuf = buffer_of(x, static_cast<int64_t>(sizeof(T)) *
                                             ((a.x_rows - 1) * a.ldx + a.k));
#pragma unroll
                for (int t = 0; t < S::kCA; ++t) {
                    const bool in = idx[t] >= 0 && idx[t] < a.x_rows && k0 + ac[t] < a.k;
                    load_to_lds(xbuf, la + (t * S::kThreads + wave * 64) * 16,
                                in ? static_cast<uint32_t>(
                                         Z * (idx[t] * a.ldx + k0 + ac[t]))
                                   : kOutside);
                }
                fetch(kt + 1);
            } else {
                const auto xbuf = buffer_of(x + p0 * a.ldx, Z * ((left - 1) * a.ldx + a.k));
#pragma unroll
                for (int t = 0; t < S::kCA; ++t)
                    load_to_lds(xbuf, la + (t * S::kThreads + wave * 64) * 16, ao[t]);
            }
#pragma unroll
            for (int t = 0; t < S::kCB; ++t)
                load_to_lds(dbuf, lb + (t * S::kThreads + wave * 64) * 16, bo[t]);
        };
        pipeline<true>(tiles, a0, b0, a1, b1, load, [](char*, char*) {}, compute, join);
    } else {
        v4u av[S::kCA], bv[S::kCB];
        auto load = [&](int kt, char*, char*) {
#pragma unroll
            for (int t = 0; t < S::kCA; ++t) {
                const int p = lo + kt * kDepth<T> + ap[t];
                const int64_t row = p < hi ? source_row(a, p) : -1;
                av[t] = load_chunk(x + (row < 0 ? 0 : row) * a.ldx + k0 + ac[t],
                                   row < 0 ? 0 : a.k - k0 - ac[t]);
            }
#pragma unroll
            for (int t = 0; t < S::kCB; ++t) {
                const int p = lo + kt * kDepth<T> + bp[t];
                bv[t] = load_chunk(dy + p * a.lddy + n0 + bc[t], p < hi ? a.n - n0 - bc[t] : 0);
            }
        };
        auto store = [&](char* la, char* lb) {
#pragma unroll
            for (int t = 0; t < S::kCA; ++t)
                *reinterpret_cast<v4u*>(la + (t * S::kThreads + tid) * 16) = av[t];
#pragma unroll
            for (int t = 0; t < S::kCB; ++t)
                *reinterpret_cast<v4u*>(lb + (t * S::kThreads + tid) * 16) = bv[t];
        };
        pipeline<false>(tiles, a0, b0, a1, b1, load, store, compute, join);
    }

    // (a group that is one part goes straight to dw)
    int first = lo, last = hi;
    if (a.unit) group_rows(a.offsets, g, a.m, &first, &last);
    const bool split = lo != first || hi != last;
    if (split && slot >= a.slots) return;  // falling offsets name more than there are
    const int to = split ? slot : g;
    if (a.dw) store_gradient<T>(a, split, to, k0 + wm, n0 + wn, lane, acc.result());
    if (BIAS && sums) store_bias_gradient<T>(a, split, to, n0 + wn, lane, sum.result()[0]);
}

constexpr int kRowParts = 64;

// dw on the large tile: both operands run across memory, the contraction over
// the group's rows.
template <typename T>
__global__ __launch_bounds__(kRingThreads) void wgrad_ring_kernel(GroupedArgs a) {
    TG_RING_LDS;
    __shared__ uint32_t row_starts[8 * kRowParts * 4];
    const uint32_t per = a.mt * a.nt;
    const int g = static_cast<int>(blockIdx.x / per);
    uint32_t mt, ntile;
    tile_of(blockIdx.x % per, a.mt, a.nt, &mt, &ntile);
    int lo, hi;
    group_rows(a.offsets, g, a.m, &lo, &hi);
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    const int k0 = static_cast<int>(mt) * 256, n0 = static_cast<int>(ntile) * 256;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / 4 * 128, wn = wave % 4 * 64;
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.dy);
    // a wavefront's load takes two rows, 32 chunks of each
    uint32_t ao[2], bo[2], ax[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        int p, c;
        part_place<true>(t * kRingThreads + tid, &p, &c);
        ax[t] = k0 + c < a.k ? static_cast<uint32_t>(2 * (k0 + c)) : kOutside;
        ao[t] = k0 + c < a.k ? static_cast<uint32_t>(2 * (p * a.ldx + k0 + c)) : kOutside;
        bo[t] = n0 + c < a.n ? static_cast<uint32_t>(2 * (p * a.lddy + n0 + c)) : kOutside;
    }
    // Gathered rows: a wavefront's rows' starts, in LDS for kRowParts parts at a
    // time.  (The indices loaded a step ahead to scalar registers held every step
    // back: 866 us against 609 without a gather, 32 groups of 32,768 x 2,048 x
    // 4,096.)
    uint32_t* own = row_starts + wave * kRowParts * 4;
    auto ahead = [&](int u) {
        if (a.rows == nullptr || u % kRowParts != 0) return;
#pragma unroll
        for (int c = 0; c < kRowParts / 16; ++c) {
            const int e = c * 64 + lane, t = (e >> 1) & 1, h = e & 1;
            const int p = lo + (u + (e >> 2)) * kStep + t * 16 + wave * 2 + h;
            const int r = p < hi ? a.rows[p] : -1;
            own[e] = r >= 0 && r < a.x_rows ? static_cast<uint32_t>(2 * r * a.ldx) : kOutside;
        }
    };
    auto load = [&](int u, char* la, char* lb) {
        const int p0 = lo + u * kStep;
        const int64_t left = hi - p0;  // rows: the buffers end with them
        const auto dbuf = buffer_of(dy + p0 * a.lddy, left > 0 ? 2 * ((left - 1) * a.lddy + a.n)
                                                               : 0);
        if (a.rows) {
            const auto xbuf = buffer_of(x, static_cast<int64_t>(sizeof(T)) *
                                             ((a.x_rows - 1) * a.ldx + a.k));
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint32_t row = own[u % kRowParts * 4 + t * 2 + (lane >> 5)];
                load_to_lds(xbuf, la + (t * kRingThreads + wave * 64) * 16,
                            (row | ax[t]) >= kOutside ? kOutside : row + ax[t]);
            }
        } else {
            const auto xbuf = buffer_of(x + p0 * a.ldx, left > 0 ? 2 * ((left - 1) * a.ldx + a.k)
                                                                 : 0);
#pragma unroll
            for (int t = 0; t < 2; ++t)
                load_to_lds(xbuf, la + (t * kRingThreads + wave * 64) * 16, ao[t]);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
            load_to_lds(dbuf, lb + (t * kRingThreads + wave * 64) * 16, bo[t]);
    };
    v4f acc[8][4] = {};
    PartReader<true, 8, true> ra(wm, lane);
    PartReader<true, 4, true> rb(wn, lane);
    ring<T>((hi - lo + kStep - 1) / kStep, ra, rb, ahead, load, a0, b0, a1, b1, a2, b2, a3, b3, acc);
    store_gradient<T>(a, false, g, k0 + wm, n0 + wn, lane, acc);
}

// dbias beside the large tiles, which have no registers left for it: the rows of
// a group over 16 wavefronts, 64 chunks of columns, their sums joined in order.
template <typename T>
__global__ __launch_bounds__(1024) void column_sums_kernel(GroupedArgs a) {
    constexpr int VEC = kVec<T>;
    __shared__ float join[16][64][VEC];
    const int g = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int lo, hi;
    group_rows(a.offsets, g, a.m, &lo, &hi);
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * 64 + lane) * VEC;
    const T* dy = static_cast<const T*>(a.dy) + c;
    float s[VEC] = {};
    for (int p = lo + wave; p < hi;) {  // chains of 64 rows (a row an add, unlike the products)
        const int stop = hi - p > 1024 ? p + 1024 : hi;
        float now[VEC] = {};
#pragma unroll 8
        for (; p < stop; p += 16) {
            float v[VEC];
            load_floats<T, VEC>(dy + p * a.lddy, a.n - c, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) now[e] += v[e];
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[e] += now[e];
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) join[wave][lane][e] = s[e];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < 16; ++w)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[e] += join[w][lane][e];
    store_floats<T, VEC>(static_cast<T*>(a.dbias) + static_cast<int64_t>(g) * a.n + c, a.n - c, s);
}

// out[g] = the sum of group g's parts, in order: `size` values each; zeros of no
// part.  A group of one part has none here: its sum is in out.
template <typename T>
__global__ __launch_bounds__(256) void parts_kernel(const int32_t* __restrict__ offsets, int m,
                                                    int unit, int slots,
                                                    const float* __restrict__ part, int64_t size,
                                                    T* __restrict__ out) {
    const int g = blockIdx.y, lane = threadIdx.x & (kWave - 1);
    int first = 0, lo, hi;
    for (int base = 0; base < g; base += kWave) {
        int n = 0;
        if (base + lane < g) {
            group_rows(offsets, base + lane, m, &lo, &hi);
            n = static_cast<int>((static_cast<int64_t>(hi) - lo + unit - 1) / unit);
        }
        first += wave_sum(n > 1 ? n : 0);
    }
    group_rows(offsets, g, m, &lo, &hi);
    // (falling offsets may name more parts than there are)
    int parts = static_cast<int>((static_cast<int64_t>(hi) - lo + unit - 1) / unit);
    if (parts == 1) return;
    parts = parts < slots - first ? parts : slots - first;
    const int64_t at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
    if (at >= size) return;
    const float* p = part + first * size + at;
    float s[4] = {};
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
        float v[4];
        load_floats<float, 4>(p + i * size, size - at, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += v[e];
    }
    store_floats<T, 4>(out + static_cast<int64_t>(g) * size + at, size - at, s);
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

// Whether an operand's tiles of up to `major` rows of `ld` elements can come by
// loads to LDS: from dword-aligned rows, within 2 GB of the tile's start; across
// memory, in whole dwords.
bool direct_operand(const void* p, int64_t ld, int64_t cols, int64_t stride, int64_t z,
                    int64_t major, bool across) {
    return reinterpret_cast<uintptr_t>(p) % 4 == 0 && ld * z % 4 == 0 && stride * z % 4 == 0 &&
           (!across || cols * z % 4 == 0) && (major * ld + cols) * z < kDirectBytes;
}

using Medium = Shape<128, 128, 2, 2>;
using Small = Shape<64, 64, 2, 2>;
using Wide = Shape<64, 128, 2, 2>;
using Few = Shape<32, 128, 1, 4>;

template <typename T, typename S>
void launch_grouped(GroupedArgs& a, bool along, bool direct, hipStream_t s) {
    a.mt = static_cast<uint32_t>(most_tiles(a.m, a.groups, S::kM));
    a.nt = static_cast<uint32_t>(ceil_div(a.n, S::kN));
    const unsigned grid = grid_of("grouped_matmul", static_cast<int64_t>(a.mt) * a.nt, S::kThreads);
    if (along)
        direct ? grouped_kernel<T, S, true, true><<<grid, S::kThreads, 0, s>>>(a)
               : grouped_kernel<T, S, true, false><<<grid, S::kThreads, 0, s>>>(a);
    else
        direct ? grouped_kernel<T, S, false, true><<<grid, S::kThreads, 0, s>>>(a)
               : grouped_kernel<T, S, false, false><<<grid, S::kThreads, 0, s>>>(a);
    TG_LAUNCH_CHECK();
}

template <typename T>
void launch_ring(GroupedArgs& a, bool along, hipStream_t s) {
    a.mt = static_cast<uint32_t>(most_tiles(a.m, a.groups, 256));
    a.nt = static_cast<uint32_t>(ceil_div(a.n, 256));
    const unsigned grid = grid_of("grouped_matmul", static_cast<int64_t>(a.mt) * a.nt, kRingThreads);
    if (a.k % kStep == 0)
        along ? grouped_ring_kernel<T, true, true><<<grid, kRingThreads, 0, s>>>(a)
              : grouped_ring_kernel<T, false, true><<<grid, kRingThreads, 0, s>>>(a);
    else
        along ? grouped_ring_kernel<T, true, false><<<grid, kRingThreads, 0, s>>>(a)
              : grouped_ring_kernel<T, false, false><<<grid, kRingThreads, 0, s>>>(a);
    TG_LAUNCH_CHECK();
}

// How a gradient of w is cut: tiles of `edge` x `edge` of whole groups where they
// are two for each of the 256 CUs, or the rows few; else of parts of `unit` rows
// for about four, 512 rows at least.  Edge 256 (16-bit types, direct loads) where
// that gives two or four tiles a CU of enough rows (32 groups of 40,000 x 1,024
// x 4,096 375 us against 459 of edge 128; 10,000 rows of 8 groups 122 against
// 113), 64 where the groups make few tiles (40,000 x 512 x 512 52 us against
// 69; in 8 groups 88 against 67).
// In fp32, whose digits the result keeps, no part has more than kLongChain rows
// (64 chains of kSumTiles tiles).
constexpr int64_t kLongChain = 16384;

struct WgradPlan {
    int64_t edge, mt, nt, unit, parts, slots;  // most parts, most of groups of several
    size_t bytes(int64_t k, int64_t n, float** part, float** part_bias, void* ws,
                 size_t size) const {
        Carver c(ws, size);
        if (unit == 0) return 0;
        float* p = c.take<float>(static_cast<size_t>(slots * k * n));
        float* b = c.take<float>(static_cast<size_t>(slots * n));
        if (part) *part = p;
        if (part_bias) *part_bias = b;
        return c.bytes();
    }
};

WgradPlan wgrad_plan(int64_t m, int64_t k, int64_t n, int64_t groups, int type, bool direct) {
    WgradPlan p{};
    const auto tiles_of = [&](int64_t edge) {
        return std::max<int64_t>(1, ceil_div(k, edge)) * ceil_div(n, edge);
    };
    const int64_t t256 = groups * tiles_of(256);
    p.edge = 128;
    if (type != TG_TYPE_F32 && direct &&
        ((t256 >= 1024 && m >= 192 * groups) || (t256 >= 512 && m >= 4096 * groups)))
        p.edge = 256;
    else if (groups * tiles_of(128) <= 64)
        p.edge = 64;
    p.mt = std::max<int64_t>(1, ceil_div(k, p.edge));
    p.nt = ceil_div(n, p.edge);
    p.parts = groups;
    const int64_t tiles = p.mt * p.nt;
    int64_t unit = std::max<int64_t>(512, ceil_div(ceil_div(m * tiles, 1024), 64) * 64);
    if (tiles * groups >= 512 || m < 1024) unit = m;
    if (type == TG_TYPE_F32) unit = std::min(unit, kLongChain);
    if (unit >= m) return p;
    p.unit = unit;
    p.parts = most_tiles(m, groups, unit);
    // a group of several has more than `unit` rows: m / unit such groups at most
    p.slots = m / unit + std::min(groups, m / unit);
    return p;
}

template <typename T>
void launch_wgrad(GroupedArgs& a, const WgradPlan& p, bool direct, hipStream_t s) {
    a.mt = static_cast<uint32_t>(p.mt);
    a.nt = static_cast<uint32_t>(p.nt);
    a.unit = static_cast<int>(p.unit);
    a.slots = static_cast<int>(p.slots);
    const unsigned grid = grid_of("grouped_matmul_wgrad", p.mt * p.nt * p.parts, kRingThreads);
    auto tiled = [&](auto shape) {
        using S = decltype(shape);
        if (a.dbias)
            direct ? wgrad_kernel<T, S, true, true><<<grid, S::kThreads, 0, s>>>(a)
                   : wgrad_kernel<T, S, false, true><<<grid, S::kThreads, 0, s>>>(a);
        else
            direct ? wgrad_kernel<T, S, true, false><<<grid, S::kThreads, 0, s>>>(a)
                   : wgrad_kernel<T, S, false, false><<<grid, S::kThreads, 0, s>>>(a);
    };
    if (p.edge == 64)
        tiled(Small{});
    else if (p.edge == 128)
        tiled(Medium{});
    if constexpr (sizeof(T) == 2) {
        if (p.edge == 256) {
            wgrad_ring_kernel<T><<<grid, kRingThreads, 0, s>>>(a);
            TG_LAUNCH_CHECK();
            if (a.dbias) {
                const dim3 blocks(static_cast<unsigned>(ceil_div(a.n, 64 * kVec<T>)),
                                  static_cast<unsigned>(a.groups));
                column_sums_kernel<T><<<blocks, 1024, 0, s>>>(a);
            }
        }
    }
    TG_LAUNCH_CHECK();
    if (!p.unit) return;
    auto add = [&](const float* part, int64_t size, void* out) {
        const dim3 blocks(grid_of("grouped_matmul_wgrad", ceil_div(size, 1024), 256),
                          static_cast<unsigned>(a.groups));
        parts_kernel<T><<<blocks, 256, 0, s>>>(a.offsets, a.m, a.unit,
                                               a.slots, part, size,
                                               static_cast<T*>(out));
        TG_LAUNCH_CHECK();
    };
    if (a.dw) add(a.part, static_cast<int64_t>(a.k) * a.n, a.dw);
    if (a.dbias) add(a.part_bias, a.n, a.dbias);
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
        a.bias = bias;
        a.epi = epilogue;
        a.y = y;
        a.ldy = ldy;
        const bool along = transposed != 0;
        const int64_t z = tg::type_size(type);
        const bool direct =
            tg::direct_operand(x, ldx, k, 0, z, rows ? x_rows : 256, false) &&
            tg::direct_operand(w, ldw, along ? k : n, groups > 1 ? w_stride : 0, z, 256, !along);
        hipStream_t s = static_cast<hipStream_t>(stream);
        tg::with_type(type, "grouped_matmul", [&](auto t) {
            using T = decltype(t);
            // Tiles of 32 rows for groups of about 20 (150 rows of 32 groups in
            // fp32 59 us against 79 of 64 x 64, in bf16 23 both); for 16-bit
            // types the large tile where there are 160 of them of 1,024 values
            // (2,500 x 1,024 x 4,096 38 us against 47; 40,000 x 512 x 512 45
            // against 42) and the groups fill them, 128 x 128 where there are
            // two for each CU (40,000 x 512 x 512 42 against 50), else 64 x 64.
            // For floats 64 x 128 where there are as many and no column more to
            // compute (7 groups of 232,965 x 602 x 256 704 us against 742, 40,000
            // x 2,048 x 1,024 1.30 ms against 1.34; 3,000 x 256 x 256 22 against
            // 18; 128 x 128 and 128 x 64 are between the two).
            const auto tiles = [&](int64_t edge) {
                return tg::most_tiles(m, groups, edge) * tg::ceil_div(n, edge);
            };
            if (m <= 24 * groups) {
                tg::launch_grouped<T, tg::Few>(a, along, direct, s);
            } else if constexpr (sizeof(T) == 2) {
                if (direct && k % 8 == 0 && (along || n % 8 == 0) && k >= 512 &&
                    tiles(256) * k >= 160 * 1024 && m >= 192 * groups)
                    tg::launch_ring<T>(a, along, s);
                else if (tiles(128) >= 600)
                    tg::launch_grouped<T, tg::Medium>(a, along, direct, s);
                else
                    tg::launch_grouped<T, tg::Small>(a, along, direct, s);
            } else if (tg::ceil_div(n, 64) % 2 == 0 &&
                       tg::most_tiles(m, groups, 64) * tg::ceil_div(n, 128) >= 600) {
                tg::launch_grouped<T, tg::Wide>(a, along, direct, s);
            } else {
                tg::launch_grouped<T, tg::Small>(a, along, direct, s);
            }
        });
    });
}

size_t tg_grouped_matmul_wgrad_workspace_size(int64_t m, int64_t k, int64_t n, int64_t groups,
                                              int type) {
    if (m <= 0 || k < 0 || n <= 0 || groups <= 0 || groups > tg::kMaxGroups) return 0;
    // either tile (which one depends on the operands' alignment)
    // and k is 0 where only dbias is wanted
    size_t most = 0;
    for (const bool direct : {false, true})
        for (const int64_t d : {k, int64_t(0)})
            most = std::max(most, tg::wgrad_plan(m, d, n, groups, type, direct)
                                      .bytes(d, n, nullptr, nullptr, nullptr, 0));
    return most;
}

int tg_grouped_matmul_wgrad(int64_t m, int64_t k, int64_t n, int64_t groups, int type,
                            const void* x, int64_t x_rows, int64_t ldx, const int32_t* rows,
                            const void* dy, int64_t lddy, const int32_t* offsets, void* dw,
                            void* dbias, void* workspace, size_t workspace_bytes,
                            tg_stream_t stream) {
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
        a.k = static_cast<int>(dw ? k : 0);
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
        const int64_t z = tg::type_size(type);
        const bool direct = tg::direct_operand(x, ldx, a.k, 0, z, rows ? x_rows : 64, true) &&
                            tg::direct_operand(dy, lddy, n, 0, z, 64, true);
        hipStream_t s = static_cast<hipStream_t>(stream);
        const tg::WgradPlan plan = tg::wgrad_plan(m, a.k, n, groups, type, direct);
        tg::TempBuffer temp;
        if (plan.unit) {
            const size_t need = plan.bytes(a.k, n, nullptr, nullptr, nullptr, 0);
            if (!workspace) {
                temp.allocate(need, s);
                workspace = temp.get();
                workspace_bytes = need;
            }
            plan.bytes(a.k, n, &a.part, &a.part_bias, workspace, workspace_bytes);
        }
        tg::with_type(type, "grouped_matmul_wgrad", [&](auto t) {
            tg::launch_wgrad<decltype(t)>(a, plan, direct, s);
        });
    });
}

}  // extern "C"
