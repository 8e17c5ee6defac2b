// losses_kernels.hpp -- the losses' kernels, compiled for one element type by each
// of losses_f32.hip, losses_bf16.hip and losses_f16.hip: log probabilities of given
// classes with the entropy and the likeliest classes, the divergence from a teacher's
// top logits, and their gradients.  With z = (x - max x) / T and s = sum of exp z,
//   log p = z - log s             entropy = log s - (sum of z exp z) / s
//   divergence = sum over the teacher's classes of q (log q - log p), q their softmax
// and the gradients, of the weights g of log p[y] and h of the entropy,
//   g ([c == y] - p) - h p (log p + entropy)   and   g (p - q),   each over T.
//
// All are bound by reading the logits (and writing the gradient), so a row is
// read once: kept in registers between its maximum, its sums and its gradient.
//   * few classes: a thread takes a row, 64 rows of a wavefront through LDS;
//   * up to 256 KB of a row in the registers of 16 to 1,024 threads;
//   * longer rows, and long rows where there are few, are cut in segments, whose
//     sums and top classes a second kernel joins, in order.
// Everything between the values read and the results rounded is float; sums are made
// in an order that the shape alone gives.
#pragma once

#include "device_utils.hpp"
#include "losses.hpp"

namespace tg {
namespace {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

enum { kLogProbs = 0, kDistill = 1, kSegment = 2 };

// ---------------------------------------------------------------------------
// A row's statistics: m its largest logit, s the sum of exp(z) over z =
// (x - m) / T, u the sum of exp(z) z / ln 2.  Exponentials are of two, of arguments
// made in two roundings: (x - m) * (log2(e) / T).
// ---------------------------------------------------------------------------
struct RowSums {
    float m, s, u;
};

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

struct RowStats {
    float m, log_s;  // log_s: natural
    __device__ __forceinline__ explicit RowStats(const RowSums& r)
        : m(r.m), log_s(r.s == 0.0f ? 0.0f : logf(r.s)) {}
    __device__ __forceinline__ RowStats(float m_, float log_s_) : m(m_), log_s(log_s_) {}
    __device__ __forceinline__ bool empty() const { return m == -INFINITY && log_s == 0.0f; }
    // Half of x - m, which may lie past the largest float where both are finite and
    // their log probability is.
    __device__ __forceinline__ float half_gap(float x) const {
        return __builtin_fmaf(0.5f, x, -0.5f * m);
    }
    __device__ __forceinline__ float logp(float x, float inv) const {
        return half_gap(x) * (2.0f * inv) - log_s;
    }
    // q (log_q - log p), q > 0: infinite only where that is.
    __device__ __forceinline__ float divergence(float q, float log_q, float x, float inv) const {
        if (empty()) return q * INFINITY;
        return __builtin_fmaf(q, log_q + log_s, -(q * half_gap(x)) * (2.0f * inv));
    }
    __device__ __forceinline__ float entropy(const RowSums& r) const {
        return r.s == 0.0f ? 0.0f : log_s - kLn2 * r.u / r.s;
    }
};

// What a row's gradient needs: e = exp2(z), z = (x - m) c, and
//   d = e (f + h z), f and h of the row, 1 / s among them.
// (With log2 s in the exponent its rounding, of numbers up to 17, was one of every p:
// rows of 130,051 equal logits 21 u off, 3 u and the logarithm's own 8 now.)
struct RowGradient {
    float m, f, h;
    __device__ __forceinline__ float operator()(float x, float c) const {
        return exp2_of((x - m) * c) * f;
    }
    // (h z: below -300, e is 0)
    __device__ __forceinline__ float with_entropy(float x, float c) const {
        const float z = (x - m) * c;
        return exp2_of(z) * __builtin_fmaf(h, __builtin_fmaxf(z, -300.0f), f);
    }
};

// That of g log p[y] + h entropy: -(g + h (log p + entropy)) p, log p = ln 2 z - log s.
template <bool ENTROPY>
__device__ __forceinline__ RowGradient log_probs_gradient(const LossArgs& a, int64_t row,
                                                          const RowStats& st, float g, float h) {
    const float per = expf(-st.log_s);
    if constexpr (ENTROPY)
        return {st.m, __builtin_fmaf(h, a.entropy[row] - st.log_s, -g) * per, h * kLn2 * per};
    return {st.m, -g * per, 0.0f};
}

// ---------------------------------------------------------------------------
// Reductions over a wavefront: within 16 lanes by DPP, across them by the swaps of
// rows of two registers.
// ---------------------------------------------------------------------------
template <int K>
__device__ __forceinline__ uint32_t lane_flip(uint32_t v) {
    if constexpr (K >= 16) {
        typedef uint32_t v2u __attribute__((ext_vector_type(2)));
        const v2u r = K == 32 ? __builtin_bit_cast(v2u, __builtin_amdgcn_permlane32_swap(v, v, false, false))
                              : __builtin_bit_cast(v2u, __builtin_amdgcn_permlane16_swap(v, v, false, false));
        // (one of the two is the lane's own)
        return (threadIdx.x & K) ? r[0] : r[1];
    } else {
        return static_cast<uint32_t>(
            __float_as_int(dpp_flip<K>(__int_as_float(static_cast<int>(v)))));
    }
}

template <int K>
__device__ __forceinline__ float lane_flip(float v) {
    return __uint_as_float(lane_flip<K>(__float_as_uint(v)));
}
template <int K>
__device__ __forceinline__ Key lane_flip(Key v) {
    return static_cast<Key>(lane_flip<K>(static_cast<uint32_t>(v >> 32))) << 32 |
           lane_flip<K>(static_cast<uint32_t>(v));
}

struct Add {
    template <typename V>
    __device__ __forceinline__ V operator()(V a, V b) const {
        return a + b;
    }
};
struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const {
        return __builtin_fmaxf(a, b);
    }
    __device__ __forceinline__ Key operator()(Key a, Key b) const { return a > b ? a : b; }
};

// (The partners of 8 and 4 are mirrored lanes: the other half's, in some order.)
template <typename V, typename O>
__device__ __forceinline__ V wave_all(V v, O op) {
    v = op(v, lane_flip<8>(v));
    v = op(v, lane_flip<4>(v));
    v = op(v, lane_flip<2>(v));
    v = op(v, lane_flip<1>(v));
    v = op(v, lane_flip<16>(v));
    return op(v, lane_flip<32>(v));
}

// What a row's threads wrote to LDS is there for all of them.
template <int NT>
__device__ __forceinline__ void group_sync() {
    if constexpr (NT > kWave) {
        __syncthreads();
    } else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
    }
}

// Over the NT threads of a row.  `lds`: NT / 64 values of its own for each call
// between two barriers.
template <int NT, typename V, typename O>
__device__ __forceinline__ V group_all(V v, O op, V* lds) {
    if constexpr (NT == 16) {
        v = op(v, lane_flip<8>(v));
        v = op(v, lane_flip<4>(v));
        v = op(v, lane_flip<2>(v));
        return op(v, lane_flip<1>(v));
    }
    v = wave_all(v, op);
    if constexpr (NT > kWave) {
        constexpr int NW = NT / kWave;
        if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
        __syncthreads();
        v = lds[threadIdx.x % NW];
        // NW values in each NW lanes
        if constexpr (NW >= 16) v = op(v, lane_flip<8>(v));
        if constexpr (NW >= 8) v = op(v, lane_flip<4>(v));
        if constexpr (NW >= 4) v = op(v, lane_flip<2>(v));
        v = op(v, lane_flip<1>(v));
    }
    return v;
}

// ---------------------------------------------------------------------------
// Top classes.  A class's key orders as the choice does: the value's bits in
// order, then the lower class; 0 for NaN and -inf, which are no choice.
// ---------------------------------------------------------------------------
__device__ __forceinline__ Key key_of(float x, uint32_t i) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t o = b >> 31 ? ~b : b | 0x80000000u;
    return x > -INFINITY ? static_cast<Key>(o) << 32 | static_cast<uint32_t>(~i) : 0;
}
__device__ __forceinline__ float key_value(Key k) {
    const uint32_t o = static_cast<uint32_t>(k >> 32);
    return __uint_as_float(o >> 31 ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ int key_class(Key k) {
    return static_cast<int>(~static_cast<uint32_t>(k));
}

// The value of lane ^ J, for every lane.
template <int J>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
    const int x = static_cast<int>(v);
    if constexpr (J == 4) {  // banks 0, 2 from four lanes up, 1, 3 from four down
        const int up = __builtin_amdgcn_update_dpp(x, x, 0x104, 0xF, 0x5, false);
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(up, x, 0x114, 0xF, 0xA, false));
    } else if constexpr (J == 8) {
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, x, 0x128, 0xF, 0xF, false));
    } else {
        return lane_flip<J>(v);
    }
}

// A step of a bitonic sort of the wavefront's keys.
template <int J>
__device__ __forceinline__ Key sort_step(Key v, bool high) {
    const Key o = static_cast<Key>(lane_xor<J>(static_cast<uint32_t>(v >> 32))) << 32 |
                  lane_xor<J>(static_cast<uint32_t>(v));
    return (v > o) == high ? v : o;
}

// The wavefront's 64 keys in falling order over its lanes.
__device__ __forceinline__ Key sort_falling(Key v) {
    const int lane = threadIdx.x & (kWave - 1);
    static_for<1, 7>([&](auto s) {
        constexpr int S = decltype(s)::value, SIZE = 1 << S;
        const bool falling = SIZE == kWave || !(lane & SIZE);
        static_for<0, S>([&](auto t) {
            constexpr int J = SIZE >> (decltype(t)::value + 1);
            v = sort_step<J>(v, falling == !(lane & J));
        });
    });
    return v;
}

// The 64 largest of two such lists, in falling order: `v` lane by lane, `o` given
// reversed.
__device__ __forceinline__ Key merge_falling(Key v, Key o) {
    const int lane = threadIdx.x & (kWave - 1);
    v = v > o ? v : o;
    static_for<0, 6>([&](auto t) {
        constexpr int J = 32 >> decltype(t)::value;
        v = sort_step<J>(v, !(lane & J));
    });
    return v;
}

// The key of the k-th largest of the threads' keys (1 <= k <= 64).  `lds`: NT keys.
template <int NT>
__device__ __forceinline__ Key kth_of(Key v, int k, Key* lds) {
    v = sort_falling(v);
    if constexpr (NT > kWave) {
        const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
        for (int half = NT / kWave / 2; half >= 1; half /= 2) {
            if (wave >= half && wave < 2 * half) lds[wave * kWave + lane] = v;
            __syncthreads();
            if (wave < half) v = merge_falling(v, lds[(wave + half) * kWave + 63 - lane]);
        }
        if (wave == 0) lds[lane] = v;
        __syncthreads();
        return lds[k - 1];
    }
    return static_cast<Key>(__shfl(v, k - 1, kWave));
}

// ---------------------------------------------------------------------------
// A row (or a segment of one) in the registers of NT threads: NV chunks of 16
// bytes a thread, chunk i of thread t the (i NT + t)-th of the row.
// ---------------------------------------------------------------------------
template <typename T>
constexpr uint32_t kMasked = sizeof(T) == 4                ? 0xFF800000u
                             : std::is_same_v<T, bf16> ? 0xFF80FF80u
                                                       : 0xFC00FC00u;  // -inf

template <typename T>
__device__ __forceinline__ v4u load_classes(const T* p, int left) {
    constexpr int VEC = kVec<T>;
    typedef T Whole __attribute__((ext_vector_type(VEC)));
    v4u v = {kMasked<T>, kMasked<T>, kMasked<T>, kMasked<T>};
    if (left >= VEC) {
        v = __builtin_bit_cast(v4u, static_cast<Whole>(
                                        *reinterpret_cast<const typename Pack<T, VEC>::V*>(p)));
    } else if (left > 0) {
        Whole w = __builtin_bit_cast(Whole, v);
#pragma unroll
        for (int e = 0; e < VEC - 1; ++e)
            if (e < left) w[e] = p[e];
        v = __builtin_bit_cast(v4u, w);
    }
    return v;
}

// v without its first s values, -inf behind the others.
template <typename T>
__device__ __forceinline__ v4u shifted(v4u v, int s) {
    const uint32_t fill = kMasked<T>;
    const int words = sizeof(T) == 4 ? s : s >> 1;
    const bool two = words & 2, one = words & 1;
    v4u a = {two ? v[2] : v[0], two ? v[3] : v[1], two ? fill : v[2], two ? fill : v[3]};
    v4u b = {one ? a[1] : a[0], one ? a[2] : a[1], one ? a[3] : a[2], one ? fill : a[3]};
    if constexpr (sizeof(T) == 2) {
        if (s & 1)
            b = v4u{__builtin_amdgcn_alignbit(b[1], b[0], 16), __builtin_amdgcn_alignbit(b[2], b[1], 16),
                    __builtin_amdgcn_alignbit(b[3], b[2], 16), __builtin_amdgcn_alignbit(fill, b[3], 16)};
    }
    return s >= kVec<T> ? v4u{fill, fill, fill, fill} : b;
}

// Chunks [at, at + VEC), at = at0 + i * step, of the n values at p, -inf behind them;
// `before`: as many values in front of p may be read.  A chunk that n ends in comes
// from the last VEC values, and all loads are asked for before the first is looked
// at (a branch for cut chunks among them had each wait for the one before).
template <typename T, int N>
__device__ __forceinline__ void load_chunks(const T* p, int at0, int step, int n, int64_t before,
                                            v4u (&x)[N]) {
    constexpr int VEC = kVec<T>;
    typedef T Whole __attribute__((ext_vector_type(VEC)));
    if (n + before < VEC) {  // (uniform, and fewer than one chunk)
        x[0] = load_classes<T>(p + at0, n - at0);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int at = at0 + i * step, from = at < n - VEC ? at : n - VEC;
        if (i == 0 || i * step < n)
            x[i] = __builtin_bit_cast(v4u, static_cast<Whole>(
                *reinterpret_cast<const typename Pack<T, VEC>::V*>(p + from)));
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int past = at0 + i * step - (n - VEC);
        if ((i == 0 || i * step < n) && past > 0) x[i] = shifted<T>(x[i], past);
    }
}

template <typename T>
__device__ __forceinline__ void floats_of(v4u v, float (&x)[kVec<T>]) {
    typedef T Whole __attribute__((ext_vector_type(kVec<T>)));
    const Whole w = __builtin_bit_cast(Whole, v);
#pragma unroll
    for (int e = 0; e < kVec<T>; ++e) x[e] = static_cast<float>(w[e]);
}

// Keys of LDS that a row's top classes need: its threads' and its candidates'.
__host__ __device__ constexpr int candidates(int top) { return 12 * top + 64; }
__host__ __device__ constexpr int top_keys(int nt, int top) {
    return top == 0 ? 0 : nt + candidates(top);
}

template <typename T, int NT, int NV>
struct Held {
    static constexpr int VEC = kVec<T>, NW = NT < kWave ? 1 : NT / kWave;
    v4u x[NV];
    int n, tid;
    __device__ __forceinline__ Held(const T* p, int n_, int64_t before)
        : n(n_), tid(threadIdx.x % NT) {
        load_chunks<T>(p, at(0), NT * VEC, n, before, x);
    }
    __device__ __forceinline__ int at(int i) const { return (i * NT + tid) * VEC; }
    // Whether any thread has a chunk i (n is the same in all).
    __device__ __forceinline__ bool used(int i) const { return i == 0 || i * NT * VEC < n; }
    // Chunk i's values.  (Each pass makes them again: kept from one to the next,
    // by the compiler, they took twice the registers that there are.)
    __device__ __forceinline__ void values(int i, float (&v)[VEC]) {
        asm volatile("" : "+v"(x[i]));
        floats_of<T>(x[i], v);
    }
    __device__ __forceinline__ float largest(int i) {
        float v[VEC];
        values(i, v);
        float m = v[0];
#pragma unroll
        for (int e = 1; e < VEC; ++e) m = __builtin_fmaxf(m, v[e]);
        return m;
    }
    // `lds`: 3 * NW floats.
    template <bool ENTROPY>
    __device__ __forceinline__ RowSums sums(float c, float* lds) {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (used(i)) m = __builtin_fmaxf(m, largest(i));
        m = group_all<NT>(m, Max{}, lds);
        // (a row of -inf alone: its z are -inf, not NaN; a NaN stays one)
        const float base = m == -INFINITY ? 0.0f : m;
        float s = 0.0f, u = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!used(i)) continue;
            float v[VEC], si = 0.0f, ui = 0.0f;
            values(i, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float z = (v[e] - base) * c;
                const float ex = exp2_of(z);
                si += ex;
                // (a masked one's z is kept finite: its exponential is 0)
                if (ENTROPY) ui = __builtin_fmaf(ex, __builtin_fmaxf(z, -1000.0f), ui);
            }
            s += si;
            if (ENTROPY) u += ui;
            asm volatile("" : "+v"(s), "+v"(u));  // (u's terms are not left for after s)
            __builtin_amdgcn_sched_barrier(0);
        }
        s = group_all<NT>(s, Add{}, lds + NW);
        if (ENTROPY) u = group_all<NT>(u, Add{}, lds + 2 * NW);
        return {m, s, u};
    }
    // The keys of the `top` largest classes: put(j, key) by some thread for each
    // place j that there is; classes count from `first`.  `lds`: top_keys keys;
    // `count`: one int of LDS.  The k-th largest of the threads' largest classes is no
    // more than the k-th largest class, so that few others are as large (44 in the
    // mean for 32 places of 64 threads, 270 for 64): those are counted against each
    // other.  A row that puts more of its largest classes on few threads takes a
    // round over all classes for each place.
    template <typename P>
    __device__ __forceinline__ void tops(int top, uint32_t first, Key* lds, int* count, P&& put) {
        float best = -INFINITY;
        int which = 0;
        v4u w = x[0];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!used(i)) continue;
            const float m = largest(i);
            const bool more = m > best;
            best = more ? m : best;
            which = more ? i : which;
            // (words of a copy: else the compiler indexes x, and keeps it in memory)
            v4u xi = x[i];
            asm volatile("" : "+v"(xi));
#pragma unroll
            for (int d = 0; d < 4; ++d) w[d] = more ? xi[d] : w[d];
        }
        float v[VEC];
        floats_of<T>(w, v);
        int e0 = 0;
#pragma unroll
        for (int e = VEC - 1; e >= 0; --e) e0 = v[e] == best ? e : e0;
        const Key mine = key_of(best, first + static_cast<uint32_t>(at(which) + e0));
        if (top == 1) {
            const Key k = group_all<NT>(mine, Max{}, lds);
            if (tid == 0) put(0, k);
            return;
        }
        if constexpr (NT >= kWave) many_tops(top, first, mine, lds, count, put);
    }
    template <typename P>
    __device__ __forceinline__ void many_tops(int top, uint32_t first, Key mine, Key* lds,
                                              int* count, P&& put) {
        float v[VEC];
        if (tid == 0) *count = 0;
        const Key limit = kth_of<NT>(mine, top, lds);
        if constexpr (NT == kWave) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        Key* cand = lds + NT;
        const float floor = limit ? key_value(limit) : -INFINITY;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (used(i)) {
                values(i, v);
                int these = 0;  // places of the chunk
#pragma unroll
                for (int e = 0; e < VEC; ++e) these |= v[e] >= floor ? 1 << e : 0;
                while (these) {
                    const int e = __builtin_ctz(these);
                    these &= these - 1;
                    float value = v[0];
#pragma unroll
                    for (int u = 1; u < VEC; ++u) value = e == u ? v[u] : value;
                    const Key k = key_of(value, first + static_cast<uint32_t>(at(i) + e));
                    if (k != 0 && k >= limit) {
                        const int to = atomicAdd(count, 1);
                        if (to < candidates(top)) cand[to] = k;
                    }
                }
            }
        }
        group_sync<NT>();
        const int many = *count;
        if (many > candidates(top)) {
            Key last = ~Key(0);
            for (int j = 0; j < top; ++j) {
                Key next = 0;
#pragma unroll 1
                for (int i = 0; i < NV; ++i) {
                    if (!used(i)) break;
#pragma unroll
                    for (int c = 0; c < NV; ++c)
                        if (c == i) values(c, v);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const Key k = key_of(v[e], first + static_cast<uint32_t>(at(i) + e));
                        next = k < last && k > next ? k : next;
                    }
                }
                last = group_all<NT>(next, Max{}, lds);
                if (tid == 0) put(j, last);
                group_sync<NT>();
            }
            return;
        }
        if (many > 2 * kWave && NT <= 256) {  // 64 at a time
            if (tid >= kWave) return;
            Key best = sort_falling(cand[tid]);
            for (int base = kWave; base < many; base += kWave) {
                const Key k = sort_falling(base + tid < many ? cand[base + tid] : Key(0));
                best = merge_falling(best, static_cast<Key>(__shfl(k, 63 - tid, kWave)));
            }
            if (tid < top) put(tid, best);
            return;
        }
        for (int i = tid; i < many; i += NT) {
            const Key k = cand[i];
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < many; ++j) rank += cand[j] > k ? 1 : 0;
            if (rank < top) put(rank, k);
        }
        for (int j = many + tid; j < top; j += NT) put(j, Key(0));
    }
};

// The chunk of 16 bytes' gradients to memory.
template <typename T>
__device__ __forceinline__ void store_classes(T* p, int left, const float (&d)[kVec<T>]) {
    store_floats<T, kVec<T>>(p, left, d);
}

__device__ __forceinline__ float teacher_at(const LossArgs& a, int64_t i) {
    if (a.teacher_type == TG_TYPE_F32) return static_cast<const float*>(a.teacher)[i];
    if (a.teacher_type == TG_TYPE_BF16)
        return static_cast<float>(static_cast<const bf16*>(a.teacher)[i]);
    return static_cast<float>(static_cast<const f16*>(a.teacher)[i]);
}

// Every 64th of the teacher's values from `first` on, where there are (`left`).
template <int N>
__device__ __forceinline__ void teachers_at(const LossArgs& a, int64_t first, int left,
                                            float (&t)[N]) {
    auto load = [&](auto type) {
        const auto* p = static_cast<const decltype(type)*>(a.teacher) + first;
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = static_cast<float>(p[i * kWave < left ? i * kWave : 0]);
    };
    if (a.teacher_type == TG_TYPE_F32)
        load(float{});
    else if (a.teacher_type == TG_TYPE_BF16)
        load(bf16{});
    else
        load(f16{});
}

// What a row of log probabilities gives out, by one thread.
template <typename T>
__device__ __forceinline__ void put_row(const LossArgs& a, int64_t row, const RowSums& r,
                                        const RowStats& st) {
    if (a.stats) {
        a.stats[2 * row] = st.m;
        a.stats[2 * row + 1] = st.log_s;
    }
    if (a.value) {
        const int y = a.labels[row];
        float v = 0.0f;
        if (y >= 0 && y < a.classes)
            v = st.empty() ? -INFINITY
                           : st.logp(static_cast<float>(
                                         static_cast<const T*>(a.logits)[row * a.ld + y]),
                                     a.inv);
        a.value[row] = v;
    }
    if (a.entropy) a.entropy[row] = st.entropy(r);
}

__device__ __forceinline__ void put_top(const LossArgs& a, int64_t row, int j, Key k,
                                        const RowStats& st) {
    a.top_values[row * a.top + j] = k ? st.logp(key_value(k), a.inv) : -INFINITY;
    a.top_ids[row * a.top + j] = k ? key_class(k) : -1;
}

// The teacher's places of a row, by the first wavefront of the row's threads:
// q of place j to q[j] (LDS or memory) and class to id[j] (-1: none); returns the
// loss and the sum of the exponentials (0: no places).
struct Teacher {
    float loss, total;
};

template <typename T, int N, typename Q, typename I>
__device__ __forceinline__ Teacher teach_of(const LossArgs& a, int64_t row, const RowStats& st,
                                         Q&& put_q, I&& put_id) {
    const int lane = threadIdx.x & (kWave - 1);
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    float t[N], xs[N];
    float tm = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int j = i * kWave + lane;
        t[i] = -INFINITY;
        xs[i] = 0.0f;
        if (j < a.k) {
            const int c = a.ids[row * a.k + j];
            const bool in = c >= 0 && c < a.classes;
            put_id(j, in ? c : -1);
            if (in) {
                t[i] = teacher_at(a, row * a.k + j);
                xs[i] = static_cast<float>(x[c]);
            }
        }
        tm = __builtin_fmaxf(tm, t[i]);
    }
    tm = wave_all(tm, Max{});
    float total = 0.0f;
    float e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        // (places of -inf alone: 0, not NaN)
        e[i] = t[i] == -INFINITY ? 0.0f : exp2_of((t[i] - tm) * a.c);
        total += e[i];
    }
    total = wave_all(total, Add{});
    const float log_total = logf(total);
    float loss = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int j = i * kWave + lane;
        const float q = total == 0.0f ? 0.0f : e[i] / total;
        if (j < a.k) put_q(j, q);
        if (j < a.k && q != 0.0f)
            loss += st.divergence(q, (t[i] - tm) * a.inv - log_total, xs[i], a.inv);
    }
    return {wave_all(loss, Add{}), total};
}

template <typename T, typename Q, typename I>
__device__ __forceinline__ Teacher teach(const LossArgs& a, int64_t row, const RowStats& st,
                                         Q&& put_q, I&& put_id) {
    return a.k <= kWave ? teach_of<T, 1>(a, row, st, put_q, put_id)
                        : teach_of<T, kMaxTeacher / kWave>(a, row, st, put_q, put_id);
}

// The factor of a row's distillation gradient; 0: the row's gradient is 0.  A NaN
// among the teacher's values is one in the whole row.
__device__ __forceinline__ float distill_factor(const LossArgs& a, int64_t row, float total,
                                                const RowStats& st) {
    const float g = a.dloss[row];
    return g == 0.0f || total == 0.0f || st.empty() ? 0.0f : g * a.inv * (total / total);
}

// d[at] -= v.
template <int VEC>
__device__ __forceinline__ void subtract(int at, float v, float (&d)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) d[e] -= at == e ? v : 0.0f;
}

// A teacher's places by the thread that holds their class: id and q of each (id -1:
// none, or its class in a place before, whose q has its own, added in order) and lists
// of a thread's places, whose order therefore changes nothing.
template <int NT>
struct Places {
    float q[kMaxTeacher];
    int id[kMaxTeacher];
    int before[kMaxTeacher];  // the place before in its list, -1: none
    int last[NT];
    // id and q are there, last is -1; of `k` places.  NT threads.
    template <int VEC>
    __device__ __forceinline__ void build(int tid, int k) {
        constexpr int N = kMaxTeacher / kWave;
        float sum[N];
        group_sync<NT>();
        if (tid < kWave) {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int j = u * kWave + tid;
                sum[u] = -1.0f;
                if (j >= k || id[j] < 0) continue;
                const int c = id[j];
                bool other = false;
                float s = 0.0f;
                for (int w = 0; w < k; ++w) {
                    const bool same = id[w] == c;
                    other |= same && w < j;
                    s += same ? q[w] : 0.0f;
                }
                sum[u] = other ? -1.0f : s;
            }
        }
        group_sync<NT>();
        if (tid < kWave) {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int j = u * kWave + tid;
                if (j >= k) continue;
                if (sum[u] == -1.0f) {
                    id[j] = -1;
                } else {
                    q[j] = sum[u];
                    before[j] = atomicExch(&last[id[j] / VEC % NT], j);
                }
            }
        }
        group_sync<NT>();
    }
};

// A thread's places: two in registers, the others looked up.
template <int NT, int VEC>
struct MyPlaces {
    int c0 = -1, c1 = -1, more = -1;
    float q0 = 0.0f, q1 = 0.0f;
    __device__ __forceinline__ MyPlaces(const Places<NT>& p, int tid) {
        const int j0 = p.last[tid];
        if (j0 < 0) return;
        c0 = p.id[j0];
        q0 = p.q[j0];
        const int j1 = p.before[j0];
        if (j1 < 0) return;
        c1 = p.id[j1];
        q1 = p.q[j1];
        more = p.before[j1];
    }
    // d -= g q of the places of the chunk at `at`.
    __device__ __forceinline__ void subtract_from(const Places<NT>& p, int at, float g,
                                                  float (&d)[VEC]) const {
        if (static_cast<uint32_t>(c0 - at) < VEC) subtract(c0 - at, q0 * g, d);
        if (static_cast<uint32_t>(c1 - at) < VEC) subtract(c1 - at, q1 * g, d);
        for (int j = more; j >= 0; j = p.before[j])
            if (static_cast<uint32_t>(p.id[j] - at) < VEC) subtract(p.id[j] - at, p.q[j] * g, d);
    }
};

// One row (kSegment: one segment) for each NT threads: one read of the logits, and
// for distillation one write of the gradient.  8,192 x 32,000 bf16: log probabilities
// 128 us (4.1 TB/s) behind the gradient of other rows, whose writes still leave the
// caches, 92 after each other; 4,096 x 65,536 bf16 with 32 places and gradient 224 (4.8).  Top
// classes cost beside it the largest of each thread, one sort of those and the few
// candidates: 64 x 32,000 bf16 with 64 of them 12.7 us.  (TOPS apart: their registers,
// 77 of 42, leave one workgroup of 1,024 a CU; 4,096 x 65,536 bf16 134 us -> 95.)
template <typename T, int NT, int NV, int MODE, bool ENTROPY, bool TOPS>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void row_kernel(LossArgs a) {
    constexpr int kBlock = NT < 256 ? 256 : NT, kRows = kBlock / NT, VEC = kVec<T>;
    extern __shared__ __attribute__((aligned(16))) Key top_lds[];
    __shared__ float reduce[kRows][3 * (NT < kWave ? 1 : NT / kWave)];
    __shared__ int count[kRows];
    const int sub = NT < kWave   ? threadIdx.x / NT
                    : kRows == 1 ? 0
                                 : __builtin_amdgcn_readfirstlane(threadIdx.x / NT);
    int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + sub;
    int seg = 0;
    if constexpr (MODE == kSegment) {
        const int64_t all = row;
        row = all / a.segments;
        seg = static_cast<int>(all - row * a.segments);
    }
    row += a.row0;
    if (row >= a.rows) return;  // (all of a row's lanes; no barriers where rows share a workgroup)
    const int64_t first = MODE == kSegment ? seg * a.segment : 0;
    const int n = static_cast<int>(MODE == kSegment && a.classes - first > a.segment
                                       ? a.segment
                                       : a.classes - first);
    const T* p = static_cast<const T*>(a.logits) + row * a.ld + first;
    Held<T, NT, NV> x(p, n, first);
    const RowSums r = x.template sums<ENTROPY>(a.c, reduce[sub]);
    Key* lds = top_lds + sub * top_keys(NT, a.top);
    if constexpr (MODE == kSegment) {
        const int64_t at = row * a.segments + seg;
        if (x.tid == 0) {
            a.part[4 * at] = r.m;
            a.part[4 * at + 1] = r.s;
            a.part[4 * at + 2] = r.u;
        }
        if constexpr (TOPS)
            x.tops(a.top, static_cast<uint32_t>(first), lds, &count[sub],
                   [&](int j, Key k) { a.part_keys[at * a.top + j] = k; });
    } else if constexpr (MODE == kLogProbs) {
        const RowStats st(r);
        if (x.tid == 0) put_row<T>(a, row, r, st);
        if constexpr (TOPS)
            x.tops(a.top, 0, lds, &count[sub], [&](int j, Key k) { put_top(a, row, j, k, st); });
    } else {
        __shared__ Places<NT> places[kRows];
        __shared__ float factor[kRows];
        const RowStats st(r);
        Places<NT>& pl = places[sub];
        pl.last[x.tid] = -1;
        if (NT == kWave || threadIdx.x < kWave) {
            const Teacher t = teach<T>(
                a, row, st, [&](int j, float v) { pl.q[j] = v; },
                [&](int j, int v) { pl.id[j] = v; });
            if (x.tid == 0) {
                a.loss[row] = t.loss;
                if (a.dlogits) factor[sub] = distill_factor(a, row, t.total, st);
            }
        }
        if (!a.dlogits) return;
        pl.template build<VEC>(x.tid, a.k);
        const MyPlaces<NT, VEC> mine(pl, x.tid);
        const float g = factor[sub];
        const RowGradient grad{st.m, g / r.s, 0.0f};
        T* out = static_cast<T*>(a.dlogits) + row * a.lddl;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!x.used(i)) continue;
            float v[VEC], d[VEC];
            x.values(i, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) d[e] = grad(v[e], a.c);
            mine.subtract_from(pl, x.at(i), g, d);
            if (g == 0.0f) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) d[e] = 0.0f;
            }
            store_classes<T>(out + x.at(i), n - x.at(i), d);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// ---------------------------------------------------------------------------
// The segments of a row joined: the sums by the first wavefront, the top classes by
// all NT / 64: each merges its share of the segments' lists (in falling order, 64
// at most), then pairs of wavefronts theirs.  Bound by its launch and latencies: 4 us.
// ---------------------------------------------------------------------------
template <typename T, int MODE, int NT>
__global__ __launch_bounds__(NT) void join_kernel(LossArgs a) {
    const int64_t row = a.row0 + blockIdx.x;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const float* part = a.part + 4 * row * a.segments;
    // (every wavefront needs the sums: the values of the top classes are by wave 0)
    float m = -INFINITY;
    for (int i = lane; i < a.segments; i += kWave) m = __builtin_fmaxf(m, part[4 * i]);
    m = wave_all(m, Max{});
    float s = 0.0f, u = 0.0f;
    for (int i = lane; i < a.segments; i += kWave) {
        const float si = part[4 * i + 1], mi = part[4 * i];
        if (si == 0.0f) continue;  // all masked
        const float z = (mi - m) * a.c;
        const float f = exp2_of(z);
        s += si * f;
        // (the sums of masked differences are kept finite)
        u += f * __builtin_fmaf(si, __builtin_fmaxf(z, -1000.0f), part[4 * i + 2]);
    }
    const RowSums r{m, wave_all(s, Add{}), wave_all(u, Add{})};
    const RowStats st(r);
    if constexpr (MODE == kLogProbs) {
        if (threadIdx.x == 0) put_row<T>(a, row, r, st);
        if constexpr (NT > kWave) {  // top classes
            __shared__ Key lists[NT];
            const Key* keys = a.part_keys + row * a.segments * a.top;
            auto list = [&](int i, int at) {
                return i < a.segments && at < a.top ? keys[static_cast<int64_t>(i) * a.top + at]
                                                    : Key(0);
            };
            constexpr int kStride = NT / kWave;
            Key v = list(wave, lane), next = list(wave + kStride, 63 - lane);
            for (int i = wave + kStride; i < a.segments; i += kStride) {
                const Key o = next;
                next = list(i + kStride, 63 - lane);
                v = merge_falling(v, o);
            }
#pragma unroll
            for (int half = NT / kWave / 2; half >= 1; half /= 2) {
                if (wave >= half && wave < 2 * half) lists[threadIdx.x] = v;
                __syncthreads();
                if (wave < half) v = merge_falling(v, lists[(wave + half) * kWave + 63 - lane]);
            }
            if (wave == 0 && lane < a.top) put_top(a, row, lane, v, st);
        }
    } else {
        const Teacher t = teach<T>(
            a, row, st, [&](int j, float v) { if (a.q) a.q[row * a.k + j] = v; }, [](int, int) {});
        if (lane == 0) {
            a.loss[row] = t.loss;
            if (a.dlogits) {
                float* o = a.row_part + 4 * row;
                const float g = distill_factor(a, row, t.total, st);
                o[0] = st.m;
                o[1] = g / r.s;
                o[2] = g;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// The gradient of rows whose statistics are known: a wavefront takes kSpan chunks
// a lane of one row, one read and one write; 8,192 x 32,000 bf16 174 us (6.0 TB/s,
// the end of what log_probs read still in the caches).
// ---------------------------------------------------------------------------
constexpr int kSpan = 4;

template <typename T, int MODE, bool ENTROPY>
__global__ __launch_bounds__(256) void gradient_kernel(LossArgs a, int64_t spans) {
    constexpr int VEC = kVec<T>;
    __shared__ Places<kWave> places[MODE == kDistill ? 4 : 1];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    // (from the last row on: what log_probs read last may still be in the caches,
    // 8,192 x 32,000 bf16 with the forward pass 315 us -> 305)
    const int64_t row = a.rows - 1 - w / spans;
    if (row < a.row0) return;
    const int64_t first = (w % spans) * kSpan * kWave * VEC;
    const int n = static_cast<int>(a.classes - first < kSpan * kWave * VEC ? a.classes - first
                                                                            : kSpan * kWave * VEC);
    const T* p = static_cast<const T*>(a.logits) + row * a.ld + first;
    T* out = static_cast<T*>(a.dlogits) + row * a.lddl + first;
    RowGradient grad;
    float g = 0.0f;
    int64_t y = -1;  // the label's place
    bool zero;
    Places<kWave>& pl = places[MODE == kDistill ? wave : 0];
    if constexpr (MODE == kLogProbs) {
        const RowStats st(a.stats[2 * row], a.stats[2 * row + 1]);
        if (a.labels) {
            const int label = a.labels[row];
            if (label >= 0 && label < a.classes) {
                g = a.dvalue[row] * a.inv;
                y = label - first;
            }
        }
        const float h = ENTROPY ? -a.dentropy[row] * a.inv : 0.0f;
        grad = log_probs_gradient<ENTROPY>(a, row, st, g, h);
        zero = (g == 0.0f && h == 0.0f) || st.empty();
    } else {
        const float* o = a.row_part + 4 * row;
        g = o[2];
        grad = {o[0], o[1], 0.0f};
        zero = g == 0.0f;
        pl.last[lane] = -1;
        for (int j = lane; j < a.k; j += kWave) {
            const int c = a.ids[row * a.k + j];
            const int64_t at = c - first;
            pl.id[j] = c >= 0 && c < a.classes && at >= 0 && at < n ? static_cast<int>(at) : -1;
            pl.q[j] = a.q[row * a.k + j];
        }
        pl.template build<VEC>(lane, a.k);
    }
    float d[VEC];
    if (zero) {  // whatever the logits hold
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[e] = 0.0f;
#pragma unroll
        for (int i = 0; i < kSpan; ++i) {
            const int at = (i * kWave + lane) * VEC;
            if (i * kWave * VEC < n) store_classes<T>(out + at, n - at, d);
        }
        return;
    }
    v4u x[kSpan];
    load_chunks<T>(p, lane * VEC, kWave * VEC, n, first, x);
    struct None {
        __device__ None(const Places<kWave>&, int) {}
    };
    const std::conditional_t<MODE == kDistill, MyPlaces<kWave, VEC>, None> mine(pl, lane);
#pragma unroll
    for (int i = 0; i < kSpan; ++i) {
        const int at = (i * kWave + lane) * VEC;
        if (i * kWave * VEC >= n) continue;
        float v[VEC];
        floats_of<T>(x[i], v);
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            d[e] = ENTROPY ? grad.with_entropy(v[e], a.c) : grad(v[e], a.c);
        if constexpr (MODE == kLogProbs) {
            if (static_cast<uint64_t>(y - at) < VEC) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) d[e] += y - at == e ? g : 0.0f;
            }
        } else {
            mine.subtract_from(pl, at, g, d);
        }
        store_classes<T>(out + at, n - at, d);
    }
}

// ---------------------------------------------------------------------------
// Few classes: a thread takes a row.  64 rows come through LDS (so that memory is
// read and written in whole lines), their rows an odd number of floats apart.  A
// workgroup is one wavefront, so that many stand at different points of load, sums and
// store; 232,965 x 41 fp32: log probabilities 14.1 us (2.8 TB/s), their gradient 23.5
// (3.4), distillation with its gradient 34.8.  What it waits for is the
// turns of the three in a wavefront; the next rows' loads ahead of the sums spilled.
// ---------------------------------------------------------------------------
// e / classes: magic = 2^32 / classes rounded up (0 for one class); exact below
// 2^32 / classes.
__device__ __forceinline__ int row_of(int e, uint32_t magic) {
    return magic == 0 ? e : static_cast<int>(__umulhi(static_cast<uint32_t>(e), magic));
}

// fn(i-th value, its place in LDS) for the VEC values from e on of rows that lie
// one behind the other.
template <int VEC, typename F>
__device__ __forceinline__ void each_value(int e, int left, int classes, uint32_t magic, F&& fn) {
    const int stride = classes | 1;
    int row = row_of(e, magic), c = e - row * classes, at = row * stride + c;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        if (i < left) fn(i, at);
        const bool next = ++c == classes;
        c = next ? 0 : c;
        at += next ? stride - classes + 1 : 1;
    }
}

template <typename T, int MODE, bool ENTROPY, bool GRADIENT>
__global__ __launch_bounds__(kWave) void tiny_kernel(LossArgs a, uint32_t magic, uint32_t magic_k) {
    constexpr int VEC = kVec<T>;
    // [64][classes | 1], and of the teacher [64][k | 1] values and classes
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int classes = static_cast<int>(a.classes), stride = classes | 1;
    const int64_t r0 = a.row0 + static_cast<int64_t>(blockIdx.x) * kWave, row = r0 + threadIdx.x;
    const int rows = static_cast<int>(a.rows - r0 < kWave ? a.rows - r0 : kWave);
    const T* p = static_cast<const T*>(a.logits) + r0 * a.ld;
    const int all = rows * classes;
    if (a.ld == classes) {
        constexpr int kBatch = 8;  // loads in flight
        for (int base = 0; base < all; base += kBatch * kWave * VEC) {
            v4u v[kBatch];
            if (base + kBatch * kWave * VEC <= all) {  // no branch among the loads
#pragma unroll
                for (int b = 0; b < kBatch; ++b)
                    v[b] = load_classes<T>(p + base + (b * kWave + threadIdx.x) * VEC, VEC);
            } else {
#pragma unroll
                for (int b = 0; b < kBatch; ++b) {
                    const int e = base + (b * kWave + threadIdx.x) * VEC;
                    v[b] = load_classes<T>(p + e, all - e);
                }
            }
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int e = base + (b * kWave + threadIdx.x) * VEC;
                if (e >= all) continue;
                float f[VEC];
                floats_of<T>(v[b], f);
                each_value<VEC>(e, all - e, classes, magic, [&](int i, int at) { lds[at] = f[i]; });
            }
        }
    } else {
        for (int e = threadIdx.x; e < all; e += kWave) {
            const int r = row_of(e, magic);
            lds[e + r * (stride - classes)] = static_cast<float>(p[r * a.ld + e - r * classes]);
        }
    }
    float* const taught = lds + kWave * stride;
    const int stride_k = a.k | 1;
    if constexpr (MODE == kDistill) {
        const int places = rows * a.k;
        constexpr int kBatch = 8;  // loads in flight
        for (int base = threadIdx.x; base < places; base += kBatch * kWave) {
            int c[kBatch];
            float t[kBatch];
            teachers_at(a, r0 * a.k + base, places - base, t);
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                c[b] = a.ids[r0 * a.k + base + (b * kWave < places - base ? b * kWave : 0)];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int e = base + b * kWave;
                if (e >= places) continue;
                const int to = e + row_of(e, magic_k) * (stride_k - a.k);
                const bool in = c[b] >= 0 && c[b] < classes;
                taught[to] = in ? t[b] : -INFINITY;
                taught[kWave * stride_k + to] = __int_as_float(in ? c[b] : 0);
            }
        }
    }
    __syncthreads();
    float* x = lds + threadIdx.x * stride;
    if (threadIdx.x < rows) {
        RowSums r{-INFINITY, 0.0f, 0.0f};
        const bool sums = MODE == kDistill || !GRADIENT;
        if (sums) {
#pragma unroll 8
            for (int i = 0; i < classes; ++i) r.m = __builtin_fmaxf(r.m, x[i]);
            const float base = r.m == -INFINITY ? 0.0f : r.m;
#pragma unroll 8
            for (int i = 0; i < classes; ++i) {
                const float z = (x[i] - base) * a.c, e = exp2_of(z);
                r.s += e;
                if (ENTROPY) r.u = __builtin_fmaf(e, __builtin_fmaxf(z, -1000.0f), r.u);
            }
        }
        if constexpr (MODE == kLogProbs && !GRADIENT) {
            const RowStats st(r);
            if (a.stats) {
                a.stats[2 * row] = st.m;
                a.stats[2 * row + 1] = st.log_s;
            }
            if (a.value) {
                const int y = a.labels[row];
                const bool in = y >= 0 && y < classes;
                a.value[row] = !in          ? 0.0f
                               : st.empty() ? -INFINITY
                                            : st.logp(x[in ? y : 0], a.inv);
            }
            if (a.entropy) a.entropy[row] = st.entropy(r);
            if (a.top) {
                // The largest of each of kBlocks runs of classes in registers; a round
                // takes the first largest and looks its run through again.  (All
                // classes in each round: 137,852 x 98 fp32 with 32 places 198 us.)
                constexpr int kBlocks = 12;
                const int size = (classes + kBlocks - 1) / kBlocks;
                float most[kBlocks];
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    most[b] = -INFINITY;
                    const int end = (b + 1) * size < classes ? (b + 1) * size : classes;
                    for (int i = b * size; i < end; ++i)
                        most[b] = __builtin_fmaxf(most[b], x[i]);
                }
                for (int j = 0; j < a.top; ++j) {
                    float best = -INFINITY;
                    int run = 0;
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b) {
                        const bool more = most[b] > best;
                        best = more ? most[b] : best;
                        run = more ? b : run;
                    }
                    int at = -1;
                    float rest = -INFINITY;
                    const int first = run * size;
                    for (int i = 0; i < size; ++i) {
                        const bool in = first + i < classes;
                        const float v = in ? x[in ? first + i : 0] : -INFINITY;
                        const bool it = at < 0 && v == best && v > -INFINITY;
                        at = it ? first + i : at;
                        rest = it ? rest : __builtin_fmaxf(rest, v);
                    }
                    a.top_values[row * a.top + j] = at < 0 ? -INFINITY : st.logp(best, a.inv);
                    a.top_ids[row * a.top + j] = at;
                    if (at >= 0) x[at] = -INFINITY;
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b) most[b] = b == run ? rest : most[b];
                }
            }
        } else if constexpr (MODE == kLogProbs) {
            const RowStats st(a.stats[2 * row], a.stats[2 * row + 1]);
            const int y = a.labels ? a.labels[row] : -1;
            const bool in = y >= 0 && y < classes;
            const float g = in ? a.dvalue[row] * a.inv : 0.0f;
            const float h = ENTROPY ? -a.dentropy[row] * a.inv : 0.0f;
            const RowGradient grad = log_probs_gradient<ENTROPY>(a, row, st, g, h);
            const bool zero = (g == 0.0f && h == 0.0f) || st.empty();
#pragma unroll 8
            for (int i = 0; i < classes; ++i) {
                const float d = ENTROPY ? grad.with_entropy(x[i], a.c) : grad(x[i], a.c);
                x[i] = zero ? 0.0f : d;
            }
            if (in && !zero) x[y] += g;
        } else {
            const RowStats st(r);
            float* t = taught + threadIdx.x * stride_k;
            const float* c = t + kWave * stride_k;
            auto each = [&](auto&& fn) {
#pragma unroll 4
                for (int j = 0; j < a.k; ++j) fn(t[j], __float_as_int(c[j]));
            };
            float tm = -INFINITY, total = 0.0f, loss = 0.0f;
            auto exp_of = [&](float tj) {
                return tj == -INFINITY ? 0.0f : exp2_of((tj - tm) * a.c);
            };
            each([&](float tj, int) { tm = __builtin_fmaxf(tm, tj); });
            each([&](float tj, int) { total += exp_of(tj); });
            // Place by place: log total taken from the sum of all lost what the two have in
            // common (41 classes, 8 places: 3.2e-7 off in the 2-norm, 2.2e-7 so).
            const float per = total == 0.0f ? 0.0f : 1.0f / total, log_total = logf(total);
            each([&](float& tj, int cj) {
                const float q = exp_of(tj) * per;
                if (q != 0.0f)
                    loss += st.divergence(q, (tj - tm) * a.inv - log_total, x[cj], a.inv);
                if (GRADIENT) tj = q;
            });
            a.loss[row] = loss;
            if (GRADIENT) {
                const float g = distill_factor(a, row, total, st);
                const RowGradient grad{st.m, g / r.s, 0.0f};
#pragma unroll 8
                for (int i = 0; i < classes; ++i) x[i] = g == 0.0f ? 0.0f : grad(x[i], a.c);
                if (g != 0.0f)
                    each([&](float q, int cj) {
                        if (q != 0.0f) x[cj] -= g * q;
                    });
            }
        }
    }
    if constexpr (GRADIENT) {
        __syncthreads();
        T* out = static_cast<T*>(a.dlogits) + r0 * a.lddl;
        if (a.lddl == classes) {
            for (int e = threadIdx.x * VEC; e < all; e += kWave * VEC) {
                float v[VEC] = {};
                each_value<VEC>(e, all - e, classes, magic, [&](int i, int at) { v[i] = lds[at]; });
                store_classes<T>(out + e, all - e, v);
            }
        } else {
            for (int e = threadIdx.x; e < all; e += kWave) {
                const int r = row_of(e, magic);
                out[r * a.lddl + e - r * classes] = static_cast<T>(lds[e + r * (stride - classes)]);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
// fn with NT threads and NV chunks a thread for rows (or segments) of n classes.
// Many rows: few threads a row, so that several rows' loads, sums and stores run
// beside each other on a CU; where rows are few, more threads for each.  LANES16:
// 16 lanes may take a row, without a step across 16 lanes (a wavefront a row against
// that: 227,701 x 470 bf16 with the gradient 326 us -> 171, the likeliest class of
// 200,000 x 300 bf16 95 -> 41).
template <bool LANES16, typename F>
void with_shape(int64_t rows, int64_t n, int vec, F&& fn) {
    const int64_t chunks = ceil_div(n, vec);
    const bool few = rows < 512;
    using std::integral_constant;
    auto shape = [&](auto nt, auto nv) {
        if (chunks > decltype(nt)::value * decltype(nv)::value) return false;
        fn(nt, nv);
        return true;
    };
    constexpr integral_constant<int, 64> t64{};
    constexpr integral_constant<int, 256> t256{};
    constexpr integral_constant<int, 1024> t1024{};
    constexpr integral_constant<int, 1> v1{};
    constexpr integral_constant<int, 4> v4{};
    constexpr integral_constant<int, 8> v8{};
    constexpr integral_constant<int, 16> v16{};
    if constexpr (LANES16) {
        constexpr integral_constant<int, 16> t16{};
        if (!few && (shape(t16, v4) || shape(t16, v8))) return;
    }
    if (few) {
        shape(t64, v1) || shape(t256, v4) || shape(t1024, v4) || shape(t1024, v8) ||
            shape(t1024, v16);
    } else {
        shape(t64, v1) || shape(t64, v4) || shape(t64, v16) || shape(t256, v16) ||
            shape(t1024, v8) || shape(t1024, v16);
    }
}

// fn(a, its rows) for the slices of rows that one launch of `threads` threads a
// row can take.
template <typename F>
void sliced(LossArgs a, int64_t threads, F&& fn) {
    const int64_t end = a.rows;
    for_slices(end, threads, [&](int64_t first, int64_t rows) {
        a.row0 = first;
        a.rows = first + rows;
        fn(a, rows);
    });
}

template <typename T, int MODE, bool ENTROPY, bool TOPS>
void launch_rows(const char* what, const LossArgs& all, hipStream_t s) {
    const int64_t each = MODE == kSegment ? all.segments : 1;
    const int64_t length = MODE == kSegment ? all.segment : all.classes;
    auto launch = [&](auto nt, auto nv) {
        constexpr int NT = decltype(nt)::value, NV = decltype(nv)::value;
        constexpr int kBlock = NT < 256 ? 256 : NT, kRows = kBlock / NT;
        // (rows that fill the registers, read alone: LDS for four workgroups a CU.  Six
        // have more loads in flight than the memory likes: 8,192 x 32,000 bf16, the
        // same rows again, 95 us -> 90, with its gradient 303 -> 296; 8,192 x 16,000 fp32 87 -> 85; but 20,000 x
        // 10,000 bf16, which leaves most registers empty, 71 -> 86)
        const bool four = NT == 256 && !TOPS && MODE != kDistill && length > 12 * NT * kVec<T>;
        const size_t lds = four ? 36 * 1024 : sizeof(Key) * kRows * top_keys(NT, all.top);
        auto kernel = row_kernel<T, NT, NV, MODE, ENTROPY, TOPS>;
        sliced(all, each * NT, [&](const LossArgs& a, int64_t rows) {
            const unsigned grid = grid_of(what, ceil_div(rows * each, kRows), kBlock);
            kernel<<<grid, kBlock, lds, s>>>(a);
            TG_LAUNCH_CHECK();
        });
    };
    if (MODE == kLogProbs && all.top <= 1)
        with_shape<MODE == kLogProbs>(all.rows * each, length, kVec<T>, launch);
    else
        with_shape<false>(all.rows * each, length, kVec<T>, launch);
}

template <typename T, int MODE, bool ENTROPY, bool GRADIENT>
void launch_tiny(const char* what, const LossArgs& a, hipStream_t s) {
    const unsigned grid = grid_of(what, ceil_div(a.rows, kWave), kWave);
    const uint32_t magic =
        static_cast<uint32_t>(((uint64_t(1) << 32) + a.classes - 1) / a.classes);
    const uint32_t magic_k =
        a.k ? static_cast<uint32_t>(((uint64_t(1) << 32) + a.k - 1) / a.k) : 0;
    const size_t lds = sizeof(float) * kWave * ((a.classes | 1) + (a.k ? 2 * (a.k | 1) : 0));
    auto kernel = tiny_kernel<T, MODE, ENTROPY, GRADIENT>;
    if (lds > 48 * 1024)
        TG_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                   hipFuncAttributeMaxDynamicSharedMemorySize,
                                   static_cast<int>(lds)));
    kernel<<<grid, kWave, lds, s>>>(a, magic, magic_k);
    TG_LAUNCH_CHECK();
}

template <typename T, int MODE, bool ENTROPY>
void launch_gradient(const char* what, const LossArgs& all, hipStream_t s) {
    const int64_t spans = ceil_div(all.classes, kSpan * kWave * kVec<T>);
    sliced(all, spans * kWave, [&](const LossArgs& a, int64_t rows) {
        const unsigned grid = grid_of(what, ceil_div(rows * spans, 4), 256);
        gradient_kernel<T, MODE, ENTROPY><<<grid, 256, 0, s>>>(a, spans);
        TG_LAUNCH_CHECK();
    });
}

// Joins the rows' segments.
template <typename T, int MODE>
void launch_join(const char* what, const LossArgs& all, hipStream_t s) {
    constexpr int kTop = 1024;
    const int threads = all.top ? kTop : kWave;
    sliced(all, threads, [&](const LossArgs& a, int64_t rows) {
        const unsigned grid = grid_of(what, rows, threads);
        if constexpr (MODE == kLogProbs)
            a.top ? join_kernel<T, MODE, kTop><<<grid, kTop, 0, s>>>(a)
                  : join_kernel<T, MODE, kWave><<<grid, kWave, 0, s>>>(a);
        else
            join_kernel<T, MODE, kWave><<<grid, kWave, 0, s>>>(a);
        TG_LAUNCH_CHECK();
    });
}

// Whether a thread takes a row: up to 64 classes, but where it would look for many
// top classes of few rows; up to 128 where many rows have top classes or a teacher
// (a wavefront's work on a row is the same for 65 as for 256).
bool tiny_rows(const LossArgs& a) {
    if (a.k > kTinyPlaces || a.classes > kTinyClasses) return false;
    if (a.rows < 8192) return a.classes <= 64 && a.top * a.classes <= 512;
    return a.classes <= 64 || a.top > 0 || a.k > 0;
}

template <typename F>
void with_bool(bool b, F&& fn) {
    b ? fn(std::true_type{}) : fn(std::false_type{});
}

template <typename T>
void launch_log_probs(const LossArgs& a, bool cut, hipStream_t s) {
    with_bool(a.entropy != nullptr, [&](auto ent) {
        constexpr bool E = decltype(ent)::value;
        if (tiny_rows(a)) {
            launch_tiny<T, kLogProbs, E, false>("log_probs", a, s);
            return;
        }
        with_bool(a.top > 0, [&](auto tops) {
            constexpr bool K = decltype(tops)::value;
            if (cut) {
                launch_rows<T, kSegment, E, K>("log_probs", a, s);
                launch_join<T, kLogProbs>("log_probs", a, s);
            } else {
                launch_rows<T, kLogProbs, E, K>("log_probs", a, s);
            }
        });
    });
}

template <typename T>
void launch_log_probs_backward(const LossArgs& a, hipStream_t s) {
    with_bool(a.dentropy != nullptr, [&](auto ent) {
        constexpr bool E = decltype(ent)::value;
        if (a.classes <= 64)
            launch_tiny<T, kLogProbs, E, true>("log_probs_backward", a, s);
        else
            launch_gradient<T, kLogProbs, E>("log_probs_backward", a, s);
    });
}

template <typename T>
void launch_distill(const LossArgs& a, bool cut, hipStream_t s) {
    if (tiny_rows(a)) {
        with_bool(a.dlogits != nullptr, [&](auto grad) {
            launch_tiny<T, kDistill, false, decltype(grad)::value>("distill", a, s);
        });
    } else if (cut) {
        launch_rows<T, kSegment, false, false>("distill", a, s);
        launch_join<T, kDistill>("distill", a, s);
        if (a.dlogits) launch_gradient<T, kDistill, false>("distill", a, s);
    } else {
        launch_rows<T, kDistill, false, false>("distill", a, s);
    }
}

}  // namespace

// What one of the .hip files compiles.
#define TG_LOSSES_OF(T)                                                              \
    template <>                                                                      \
    void losses_log_probs<T>(const LossArgs& a, bool cut, hipStream_t s) {           \
        launch_log_probs<T>(a, cut, s);                                              \
    }                                                                                \
    template <>                                                                      \
    void losses_log_probs_backward<T>(const LossArgs& a, hipStream_t s) {            \
        launch_log_probs_backward<T>(a, s);                                          \
    }                                                                                \
    template <>                                                                      \
    void losses_distill<T>(const LossArgs& a, bool cut, hipStream_t s) {             \
        launch_distill<T>(a, cut, s);                                                \
    }

}  // namespace tg
