// tiles.hpp -- operand tiles of the matrix products in LDS: how they lie
// there, how they come from memory and how the matrix instructions' operands
// are read.
//
// A tile holds 128 bytes of values along the contraction (64 of 16 bits, 32
// floats, 128 of 8 bits) for each of its R rows (of x) or columns (of w).  Two
// forms:
//   * along: the contraction runs along memory.  [R][128 bytes], a row's eight
//     16-byte chunks at positions c ^ (row & 7): sixteen lanes that read one
//     chunk each of sixteen rows meet every bank equally.
//   * across: the contraction runs across memory (w [k x n] in x * w; both
//     operands in x^T * dy).  [depth][R], in slots of 16 values that are
//     permuted within a row of the tile by its k, so that what the lanes of an
//     operand read (one slot in several rows) falls in different banks.  Floats
//     are read one by one; 16-bit values by the transposing LDS load, whose
//     sixteen lanes cover four rows of one slot: lane l reads 8 bytes of row
//     l / 4 and gets column l of the four rows.
// A thread moves the same 16-byte chunks in every tile, chunk (t threads + its
// number) to LDS address 16 x that: what the loads that write straight to LDS
// need (a wavefront's 64 chunks are consecutive there), so the permutations are
// applied to the addresses in memory.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "device_utils.hpp"
#include "types.hpp"

namespace tg {

constexpr int kRowBytes = 128;    // of a tile along the contraction
template <typename T>
constexpr int kDepth = kRowBytes / static_cast<int>(sizeof(T));

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef bf16 v8bf __attribute__((ext_vector_type(8)));
typedef f16 v8h __attribute__((ext_vector_type(8)));
#define TG_LDS __attribute__((address_space(3)))

// 16 bytes of consecutive contraction values of a row or column.
union Frag {
    v4u u;
    v4f f;
    v4s s[2];
    v8bf b;
    v8h h;
};

template <typename T>
__device__ __forceinline__ Frag ones() {
    Frag v;
    if constexpr (std::is_same_v<T, float>) {
        v.f = v4f{1.0f, 1.0f, 1.0f, 1.0f};
    } else {
        const uint32_t one = std::is_same_v<T, bf16> ? 0x3F80u : 0x3C00u;
        v.u = v4u{one * 0x10001u, one * 0x10001u, one * 0x10001u, one * 0x10001u};
    }
    return v;
}

// c + the products of 64 (16 floats) contraction values' fragments.
template <typename T>
__device__ __forceinline__ v4f mfma(const Frag& a, const Frag& b, v4f c) {
    if constexpr (std::is_same_v<T, bf16>) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.b, b.b, c, 0, 0, 0);
    } else if constexpr (std::is_same_v<T, f16>) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, b.h, c, 0, 0, 0);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.f[e], b.f[e], c, 0, 0, 0);
        return c;
    }
}

// The permutation of an across tile's slots in row k (of R / 16 slots).  16-bit
// operands: a read covers rows 8 q + 0 .. 3 of lanes' quarters q; floats: row
// 4 q of each.
template <typename T, int R>
__device__ __forceinline__ int slot_swizzle(int k) {
    const int s = sizeof(T) == 2 ? (k & 3) | ((k >> 3) & 1) << 2 : (k >> 2) & 3;
    return s & (R / 16 - 1);
}

// Where a thread's chunk number e lies in the tile: (row, first value), the
// permutation undone.  ACROSS: (k, first column).
template <typename T, int R, bool ACROSS>
__device__ __forceinline__ void chunk_place(int e, int* major, int* minor) {
    constexpr int EPC = kVec<T>;
    if constexpr (ACROSS) {
        constexpr int CPR = R / EPC, CPS = 16 / EPC;  // chunks of a row, of a slot
        const int k = e / CPR, p = e % CPR;
        *major = k;
        *minor = ((p / CPS) ^ slot_swizzle<T, R>(k)) * 16 + p % CPS * EPC;
    } else {
        *major = e >> 3;
        *minor = ((e & 7) ^ (*major & 7)) * EPC;
    }
}

// A wavefront's operands of N tiles of 16 rows (columns) from row `first` on.
template <typename T, int R, bool ACROSS, int N>
struct Reader {
    int at[ACROSS ? N : 2];
    __device__ __forceinline__ Reader(int first, int lane) {
        const int q = lane >> 4, r = lane & 15;
        if constexpr (ACROSS) {
            const int k = sizeof(T) == 2 ? 8 * q + (r >> 2) : 4 * q;
            const int in = sizeof(T) == 2 ? (r & 3) * 8 : r * 4;
#pragma unroll
            for (int i = 0; i < N; ++i)
                at[i] = (k * R + (((first >> 4) + i) ^ slot_swizzle<T, R>(k)) * 16) *
                            static_cast<int>(sizeof(T)) +
                        in;
        } else {
#pragma unroll
            for (int s = 0; s < 2; ++s)
                at[s] = (first + r) * kRowBytes + (((4 * s + q) ^ (r & 7)) << 4);
        }
    }
    // Tile i, chunk 4 s + q of the contraction (s = 0, 1).
    __device__ __forceinline__ Frag read(const char* lds, int i, int s) const {
        Frag f;
        if constexpr (!ACROSS) {
            f.u = *reinterpret_cast<const v4u*>(lds + at[s] + i * 16 * kRowBytes);
        } else if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                f.s[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (TG_LDS v4s*)(lds + at[i] + (32 * s + 4 * h) * R * 2));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                f.f[e] = *reinterpret_cast<const float*>(lds + at[i] + (16 * s + e) * R * 4);
        }
        return f;
    }
};

// The memory side.  `Direct`: buffer loads that write to LDS by themselves, 16
// bytes from a dword-aligned address, each dword zero that lies outside the
// buffer: offsets of 32 bits from a base that moves with the tile.
constexpr uint32_t kOutside = 0x80000000u;  // added to an offset: outside any buffer below
constexpr int64_t kDirectBytes = int64_t(1) << 31;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, int64_t bytes) {
    const int64_t n = bytes < 0 ? 0 : bytes > kDirectBytes ? kDirectBytes : bytes;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, static_cast<int>(n),
                                             0x00020000);
}

__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t b, char* lds, uint32_t offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (TG_LDS void*)lds, 16, static_cast<int>(offset), 0,
                                             0, 0);
}

// 16 bytes of T's values at any address of theirs, zeros from `left` values on.
template <typename T>
__device__ __forceinline__ v4u load_chunk(const T* p, int64_t left) {
    constexpr int EPC = kVec<T>;
    v4u v = {0, 0, 0, 0};
    if (left >= EPC) {
        typedef T Whole __attribute__((ext_vector_type(EPC)));
        v = __builtin_bit_cast(v4u, static_cast<Whole>(
                                        *reinterpret_cast<const typename Pack<T, EPC>::V*>(p)));
    } else if (left > 0) {
        if constexpr (sizeof(T) == 4) {
            const uint32_t* e = reinterpret_cast<const uint32_t*>(p);
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < left) v[i] = e[i];
        } else {
            const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (i < left) v[i / 2] |= static_cast<uint32_t>(e[i]) << (i % 2 * 16);
        }
    }
    return v;
}

// Tile b of mt x nt, taken `kBand` row tiles by all columns at a time on each
// of 8 XCDs (every eighth workgroup), whose runs of consecutive tiles share
// their rows and columns in its L2; false where there are fewer.
constexpr int kBand = 4;
__device__ __forceinline__ bool tile_of(uint32_t b, uint32_t mt, uint32_t nt, uint32_t* i,
                                        uint32_t* j) {
    const uint32_t all = mt * nt, per = all / 8, rest = all % 8, x = b % 8;
    if (b / 8 >= per + (x < rest ? 1 : 0)) return false;
    uint32_t t = x * per + (x < rest ? x : rest) + b / 8;
    const uint32_t band = t / (kBand * nt), first = band * kBand;
    const uint32_t high = mt - first < kBand ? mt - first : kBand;
    t -= band * kBand * nt;
    *i = first + t % high;
    *j = t / high;
    return true;
}

// BM x BN outputs by WR x WC wavefronts.
template <int BM, int BN, int WR, int WC>
struct Shape {
    static constexpr int kM = BM, kN = BN, kWR = WR, kWC = WC, kThreads = 64 * WR * WC;
    static constexpr int kMI = BM / WR / 16, kNJ = BN / WC / 16;
    static constexpr int kCA = BM * 8 / kThreads, kCB = BN * 8 / kThreads;  // chunks a thread
    static_assert(kCA * kThreads == BM * 8 && kCB * kThreads == BN * 8, "chunks");
};

template <typename S>
using Acc = v4f[S::kMI][S::kNJ];

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
// result's own rounding is 2^-8 or 2^-11 at most.  (The dense layers' chains stop at
// half of it.)
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

// The barrier of a loop over tiles that loads write straight to LDS: what this
// wavefront asked for is there, then the same of every wavefront.
// __syncthreads() alone orders reads and writes, not these loads: the compiler may
// wait for a loop's first entry alone, and did where registers were spilled.  (The
// wait is the builtin, which the compiler counts: written as inline assembly it cost
// fp32 233K x 602 x 256 700 us against 615.)
__device__ __forceinline__ void loads_border() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

// The loop over `tiles` tiles: load(kt, la, lb) brings tile kt.  With DIRECT
// the loads are in flight until the barrier; else load keeps them in registers
// and store(la, lb) writes them.  join() comes after every kSumTiles tiles: in a
// loop around theirs, for a branch among them was made into selects, which read
// the sums in every tile.
constexpr int kSumTiles = 8;
template <bool DIRECT, typename L, typename W, typename C, typename J>
__device__ __forceinline__ void pipeline(int tiles, char* a0, char* b0, char* a1, char* b1,
                                         L&& load, W&& store, C&& compute, J&& join) {
    if (tiles == 0) return;
    auto border = [] {
        if constexpr (DIRECT)
            loads_border();
        else
            __syncthreads();
    };
    load(0, a0, b0);
    if (!DIRECT) store(a0, b0);
    int kt = 0;
    while (kt + 1 < tiles) {
        const int stop = tiles - kt > kSumTiles ? kt + kSumTiles : tiles;
        for (; kt + 1 < stop; kt += 2) {
            border();
            load(kt + 1, a1, b1);
            compute(a0, b0);
            if (!DIRECT) store(a1, b1);
            border();
            if (kt + 2 < tiles) load(kt + 2, a0, b0);
            compute(a1, b1);
            if (!DIRECT && kt + 2 < tiles) store(a0, b0);
        }
        join();
    }
    if (kt < tiles) {
        border();
        compute(a0, b0);
    }
}

// ---------------------------------------------------------------------------
// The large tile: 256 x 256 outputs of a 16-bit type by eight wavefronts of 128
// x 64, two on each SIMD.  The operands lie in a ring of four parts of 32
// contraction values (64 bytes a row along, 32 rows across).  While a
// wavefront's 32 matrix instructions of one part run (512 cycles), it reads its
// operands of the next one from LDS to other registers and asks for the part
// that takes the place of this one, three steps before it is read; one barrier a
// step.
// ---------------------------------------------------------------------------
constexpr int kStep = 32;                // contraction values of a part
constexpr int kPartBytes = 256 * 64;     // of one operand
constexpr int kRingThreads = 512;

template <bool ACROSS>
__device__ __forceinline__ void part_place(int e, int* major, int* minor) {
    if constexpr (ACROSS) {
        chunk_place<bf16, 256, true>(e, major, minor);
    } else {
        *major = e >> 2;
        *minor = ((e & 3) ^ ((*major >> 1) & 3)) * 8;
    }
}

// Tile i's address across memory is the first one's with i in the slot's bits.
// KEEP: the N addresses stay in registers, else each step makes them: whichever
// leaves room for the sums and two parts' operands (8192^3, w [k x n]: 10
// registers spilled with them kept, 1129 TFLOP/s against 1393; the weights'
// gradient: 11 spilled without, 898 against 1283).
template <bool ACROSS, int N, bool KEEP>
struct PartReader {
    static constexpr int kKept = ACROSS && KEEP ? N : 1;
    int at[kKept];
    __device__ __forceinline__ PartReader(int first, int lane) {
        const int q = lane >> 4, r = lane & 15;
        if constexpr (ACROSS) {
            const Reader<bf16, 256, true, 1> one(first, lane);
#pragma unroll
            for (int i = 0; i < kKept; ++i) at[i] = one.at[0] ^ (i * 32);
        } else {
            at[0] = (first + r) * 64 + ((q ^ ((r >> 1) & 3)) << 4);
        }
    }
    // Before a step's reads.
    __device__ __forceinline__ void begin() {
        if constexpr (ACROSS && !KEEP) asm volatile("" : "+v"(at[0]));
    }
    __device__ __forceinline__ Frag read(const char* lds, int i) const {
        Frag f;
        if constexpr (ACROSS) {
            const int a = KEEP ? at[KEEP ? i : 0] : at[0] ^ (i * 32);
#pragma unroll
            for (int h = 0; h < 2; ++h)
                f.s[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (TG_LDS v4s*)(lds + a + 4 * h * 512));
        } else {
            f.u = *reinterpret_cast<const v4u*>(lds + at[0] + i * 1024);
        }
        return f;
    }
};

// A step's border: what this wavefront asked of LDS is there, and all but
// LOADS of its loads; then the same of every wavefront.
template <int LOADS>
__device__ __forceinline__ void step_border() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// acc += the products of `steps` parts; load(u, la, lb) asks for part u (four
// loads a thread; zeros from `steps` on), ahead(u) comes before the loads of u ..
// u + 3.
template <typename T, typename RA, typename RB, typename P, typename L>
__device__ __forceinline__ void ring(int steps, RA& ra, RB& rb, P&& ahead, L&& load, char* a0,
                                     char* b0, char* a1, char* b1, char* a2, char* b2, char* a3,
                                     char* b3, v4f (&acc)[8][4]) {
    constexpr int kLoads = 4;
    if (steps == 0) return;
    struct Operands {
        Frag x[8], w[4];
    };
    auto read = [&](Operands& o, const char* la, const char* lb) {
        ra.begin();
        rb.begin();
#pragma unroll
        for (int j = 0; j < 4; ++j) o.w[j] = rb.read(lb, j);
#pragma unroll
        for (int i = 0; i < 8; ++i) o.x[i] = ra.read(la, i);
    };
    // part u in `now`; part u + 1, in na and nb, to `next`; part u + 4 to u's place
    auto step = [&](int u, Operands& now, Operands& next, char* la, char* lb, const char* na,
                    const char* nb) {
        step_border<2 * kLoads>();
        load(u + 4, la, lb);
        read(next, na, nb);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = mfma<T>(now.w[j], now.x[i], acc[i][j]);
        // An LDS read beside each of the first matrix instructions, then a load
        // beside every fourth: the reads have the rest of the step to arrive
        // (left to itself, the compiler puts them last, where the border waits
        // for them), and the loads of eight wavefronts, 16 cycles each, do not
        // hold back the first products.
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
        }
    };
    ahead(0);
    load(0, a0, b0);
    load(1, a1, b1);
    load(2, a2, b2);
    load(3, a3, b3);
    step_border<3 * kLoads>();
    Operands even, odd;
    read(even, a0, b0);
    int u = 0;
    for (; u + 4 <= steps; u += 4) {
        ahead(u + 4);
        step(u, even, odd, a0, b0, a1, b1);
        step(u + 1, odd, even, a1, b1, a2, b2);
        step(u + 2, even, odd, a2, b2, a3, b3);
        step(u + 3, odd, even, a3, b3, a0, b0);
    }
    if (u < steps) {
        ahead(u + 4);
        step(u, even, odd, a0, b0, a1, b1);
        if (u + 1 < steps) {
            step(u + 1, odd, even, a1, b1, a2, b2);
            if (u + 2 < steps) step(u + 2, even, odd, a2, b2, a3, b3);
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
}

#define TG_RING_LDS                                                       \
    __shared__ __attribute__((aligned(16))) char a0[kPartBytes];          \
    __shared__ __attribute__((aligned(16))) char b0[kPartBytes];          \
    __shared__ __attribute__((aligned(16))) char a1[kPartBytes];          \
    __shared__ __attribute__((aligned(16))) char b1[kPartBytes];          \
    __shared__ __attribute__((aligned(16))) char a2[kPartBytes];          \
    __shared__ __attribute__((aligned(16))) char b2[kPartBytes];          \
    __shared__ __attribute__((aligned(16))) char a3[kPartBytes];          \
    __shared__ __attribute__((aligned(16))) char b3[kPartBytes]

}  // namespace tg
