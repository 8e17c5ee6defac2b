// route.hip -- routing rows to experts: softmax and the k largest, the rows'
// order by expert, the weighted join of the experts' results, and the backward
// passes of the first and the last.
//
// Top k.  16 lanes take a row of up to 256 experts (16 values a lane, so no
// step crosses a DPP row), a wavefront one of up to 1,024.  A value and its
// column make one key that orders as the choice does: the value's bits in order,
// then the lower column (32 bits for 16-bit logits, 64 for floats).  A lane sorts
// its keys once; each of the k rounds is one maximum over the lanes' heads, whose
// lane drops its own.  (A search by the lane that lost its largest value, in each
// round, took 46 us of 65,536 rows of 128 and 8 places; 31 now.)
//
// Order.  A stable counting sort of the slots by expert: workgroup b counts its
// share of the slots (in the top-k kernel, whose rows they are), then places
// them after the shares before it.  A wavefront ranks 64 slots at a time by the
// ballots of their ids' bits.  No atomics decide an order.
//
// The join is bound by reading y once, top k by its rounds (31 us where reading
// the logits takes 4; twice the wavefronts changed nothing), the order by the
// shares' counts (11 us; 17 with 512 shares), small sizes by their launches: up to
// kOneTokens rows or kOneSlots slots one workgroup does everything in one launch.
#include "common.hpp"
#include "device_utils.hpp"
#include "grouped.hpp"
#include "types.hpp"

#include <string>

namespace tg {
namespace {

constexpr int64_t kMaxTop = 32;
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int64_t kSortBlocks = 256;  // shares of the slots: each reads every share's counts
// Sizes that one workgroup routes and sorts by itself.
constexpr int64_t kOneSlots = 8192, kOneTokens = 256;

struct RouteArgs {
    int64_t tokens, k;
    int experts, renorm;
    const void* logits;
    int64_t ld;
    float* weights;
    int32_t* ids;
    int64_t share;    // tokens of a workgroup
    int32_t* counts;  // [workgroups][experts + 1] (last: none), or null
    // backward
    const float* dweights;
    void* dlogits;
    int64_t lddl;
};

struct PlanArgs {
    int64_t slots, k, share;  // share: slots of a workgroup
    int groups;
    const int32_t* ids;
    int32_t* offsets;
    int32_t* rows;
    int32_t* position;
    const int32_t* counts;  // [blocks][groups + 1], or null (one workgroup)
    int blocks;
};

// Reductions over the LPR lanes of a row.
template <int LPR, int K>
__device__ __forceinline__ uint32_t flip(uint32_t v) {
    if constexpr (LPR == 16)
        return static_cast<uint32_t>(
            __float_as_int(dpp_flip<K>(__int_as_float(static_cast<int>(v)))));
    else
        return static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), K, kWave));
}

template <int LPR, int K>
__device__ __forceinline__ uint64_t flip(uint64_t v) {
    return static_cast<uint64_t>(flip<LPR, K>(static_cast<uint32_t>(v >> 32))) << 32 |
           flip<LPR, K>(static_cast<uint32_t>(v));
}

template <int LPR, int K, typename V>
__device__ __forceinline__ V group_max(V v) {
    const V o = flip<LPR, K>(v);
    v = o > v ? o : v;
    if constexpr (K > 1) return group_max<LPR, K / 2>(v);
    return v;
}

template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
    if constexpr (LPR == 16) {
        v += dpp_flip<8>(v);
        v += dpp_flip<4>(v);
        v += dpp_flip<2>(v);
        return v + dpp_flip<1>(v);
    } else {
        return wave_sum(v);
    }
}

// The key of value x in column c: larger for a larger x, then for a smaller c;
// 0 for NaN and -inf, which are no choice.  -0 and 0 are equal.
template <typename T>
struct KeyOf {
    typedef uint32_t Key;
    typedef uint16_t Bits;
    static constexpr int kShift = 16;
};
template <>
struct KeyOf<float> {
    typedef uint64_t Key;
    typedef uint32_t Bits;
    static constexpr int kShift = 32;
};

template <typename T>
__device__ __forceinline__ typename KeyOf<T>::Key key_of(float x, int c) {
    using K = KeyOf<T>;
    typedef typename K::Bits Bits;
    constexpr Bits sign = Bits(1) << (K::kShift - 1);
    const Bits b = __builtin_bit_cast(Bits, static_cast<T>(x + 0.0f));
    const Bits o = b & sign ? static_cast<Bits>(~b) : static_cast<Bits>(b | sign);
    return x > -INFINITY ? static_cast<typename K::Key>(o) << K::kShift |
                               static_cast<Bits>(~static_cast<Bits>(c))
                         : 0;
}

template <typename T>
__device__ __forceinline__ float value_of(typename KeyOf<T>::Key key) {
    using K = KeyOf<T>;
    typedef typename K::Bits Bits;
    constexpr Bits sign = Bits(1) << (K::kShift - 1);
    const Bits o = static_cast<Bits>(key >> K::kShift);
    return static_cast<float>(__builtin_bit_cast(
        T, o & sign ? static_cast<Bits>(o & ~sign) : static_cast<Bits>(~o)));
}

template <typename T>
__device__ __forceinline__ int column_of(typename KeyOf<T>::Key key) {
    return static_cast<typename KeyOf<T>::Bits>(~key);
}

// v in falling order: Batcher's odd-even merge sort.
template <int N, typename V>
__device__ __forceinline__ void sort_falling(V (&v)[N]) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i) {
                    const int a = i + j, b = i + j + k;
                    if (b < N && a / (p * 2) == b / (p * 2)) {
                        const V x = v[a], y = v[b];
                        v[a] = x > y ? x : y;
                        v[b] = x > y ? y : x;
                    }
                }
}

// A lane's logits: VEC consecutive ones, every LPR * VEC; -inf past the row.
template <typename T, int LPR, int ITEMS>
struct RowOf {
    static constexpr int VEC = ITEMS < kVec<T> ? ITEMS : kVec<T>;
    __device__ static int column(int lane, int i) {
        return (i / VEC * LPR + lane) * VEC + i % VEC;
    }
    __device__ static void load(const T* __restrict__ p, int experts, int lane, float (&x)[ITEMS]) {
#pragma unroll
        for (int b = 0; b < ITEMS / VEC; ++b) {
            const int c = (b * LPR + lane) * VEC;
            float v[VEC];
            load_floats<T, VEC>(p + c, experts - c, v);
#pragma unroll
            for (int u = 0; u < VEC; ++u) x[b * VEC + u] = c + u < experts ? v[u] : -INFINITY;
        }
    }
    // The row's largest value, NaN left out, and the sum of x = exp(x - it).
    __device__ static float largest(const float (&x)[ITEMS]) {
        float top = x[0] > -INFINITY ? x[0] : -INFINITY;
#pragma unroll
        for (int i = 1; i < ITEMS; ++i) top = x[i] > top ? x[i] : top;
        return order_value(group_max<LPR, LPR / 2>(order_bits(top)));
    }
    __device__ static float exps(float top, float (&x)[ITEMS]) {
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            x[i] = x[i] == -INFINITY ? 0.0f : __expf(x[i] - top);
            total += x[i];
        }
        return group_sum<LPR>(total);
    }
    // floats as whole numbers of the same order (the group's maximum has one
    // form for both)
    __device__ static uint32_t order_bits(float x) {
        const uint32_t b = __float_as_uint(x);
        return b >> 31 ? ~b : b | 0x80000000u;
    }
    __device__ static float order_value(uint32_t o) {
        return __uint_as_float(o >> 31 ? o & 0x7FFFFFFFu : ~o);
    }
};

// The k largest of the row x: place j's expert and weight in lane j of the group.
template <typename T, int LPR, int ITEMS>
__device__ __forceinline__ void route_row(const RouteArgs& a, float (&x)[ITEMS], int lane,
                                          int* expert, float* weight) {
    using R = RowOf<T, LPR, ITEMS>;
    typedef typename KeyOf<T>::Key Key;
    Key key[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) key[i] = key_of<T>(x[i], R::column(lane, i));
    sort_falling(key);
    Key mine = 0, first = 0;
    const int k = static_cast<int>(a.k);
    for (int j = 0; j < k; ++j) {
        const Key best = group_max<LPR, LPR / 2>(key[0]);
        if (j == 0) first = best;
        if (lane == j) mine = best;
        const bool drop = key[0] == best;  // one lane's (or none is left: 0s)
#pragma unroll
        for (int i = 0; i + 1 < ITEMS; ++i) key[i] = drop ? key[i + 1] : key[i];
        if (drop) key[ITEMS - 1] = 0;
    }
    const float top = first ? value_of<T>(first) : -INFINITY;
    float total = R::exps(top, x);   // NaN where a logit is NaN or +inf
    const float e = mine ? __expf(value_of<T>(mine) - top) : 0.0f;
    const bool bad = total != total;
    if (a.renorm) {
        const float chosen = group_sum<LPR>(lane < k ? e : 0.0f);
        if (!bad) total = chosen;
    }
    *expert = mine ? column_of<T>(mine) : -1;
    *weight = mine || bad ? e / total : 0.0f;
}

// Places the slots [s0, s1) of one workgroup, `lds` holding kSortWaves *
// (groups + 1) + 2 * kSortThreads + 2 * kSortWaves ints.  id(s): the slot's
// group, `groups` for none.
template <typename F>
__device__ void place_slots(const PlanArgs& p, int64_t s0, int64_t s1, int* lds, F&& id) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int n = p.groups + 1;
    int* cursor = lds;                          // [wave][n]
    int* total = lds + kSortWaves * n;          // [<= kSortThreads + 1]: all workgroups' counts
    int* before = total + kSortThreads + kSortWaves;  // ... of those before this one
    int* mine = cursor + wave * n;

    // what each wavefront holds of each group
    for (int i = tid; i < kSortWaves * n; i += kSortThreads) cursor[i] = 0;
    __syncthreads();
    const int64_t seg = ((s1 - s0 + kSortWaves - 1) / kSortWaves + kWave - 1) / kWave * kWave;
    const int64_t lo = s0 + wave * seg, hi = lo + seg < s1 ? lo + seg : s1;
    for (int64_t s = lo + lane; s < hi; s += kWave) atomicAdd(&mine[id(s)], 1);
    __syncthreads();

    // all slots' counts and those before this workgroup
    if (p.counts == nullptr) {
        for (int e = tid; e < n; e += kSortThreads) {
            int t = 0;
            for (int w = 0; w < kSortWaves; ++w) t += cursor[w * n + e];
            total[e] = t;
            before[e] = 0;
        }
        __syncthreads();
    } else {
        for (int e = tid; e < n; e += kSortThreads) total[e] = before[e] = 0;
        __syncthreads();
        const int parts = n < kSortThreads ? kSortThreads / n : 1;
        for (int i = tid; i < parts * n; i += kSortThreads) {
            const int e = i % n, part = i / n;
            const int share = (p.blocks + parts - 1) / parts;
            const int b0 = part * share, b1 = b0 + share < p.blocks ? b0 + share : p.blocks;
            int t = 0, f = 0;
#pragma unroll 8
            for (int b = b0; b < b1; ++b) {
                const int c = p.counts[static_cast<int64_t>(b) * n + e];
                t += c;
                f += b < static_cast<int>(blockIdx.x) ? c : 0;
            }
            atomicAdd(&total[e], t);  // whole numbers: any order
            atomicAdd(&before[e], f);
        }
        __syncthreads();
    }

    // each group's first place, then each wavefront's
    __shared__ int scan[kSortWaves];
    int all;
    const int c = tid < p.groups ? total[tid] : 0;
    const int first = block_exclusive_scan<kSortThreads>(c, scan, &all);
    if (tid < p.groups) {
        if (blockIdx.x == 0) p.offsets[tid] = first;
        int at = first + before[tid];
        for (int w = 0; w < kSortWaves; ++w) {
            const int x = cursor[w * n + tid];
            cursor[w * n + tid] = at;
            at += x;
        }
    }
    if (tid == kSortThreads - 1) {
        if (blockIdx.x == 0) p.offsets[p.groups] = all;
        int at = all + before[p.groups];
        for (int w = 0; w < kSortWaves; ++w) {
            const int x = cursor[w * n + p.groups];
            cursor[w * n + p.groups] = at;
            at += x;
        }
    }
    __syncthreads();

    const int bits = 32 - __clz(p.groups);
    const uint32_t k = static_cast<uint32_t>(p.k);
    for (int64_t s = lo + lane; s - lane < hi; s += kWave) {
        const bool in = s < hi;
        const int g = in ? id(s) : 0;
        uint64_t peers = __ballot(in);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot((g >> b) & 1);
            peers &= (g >> b) & 1 ? set : ~set;
        }
        const int rank = __popcll(peers & ((uint64_t(1) << lane) - 1));
        const int start = in ? mine[g] : 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (in && rank == 0) mine[g] = start + __popcll(peers);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (in) {
            const int at = start + rank;
            const bool none = g == p.groups;
            p.position[s] = none ? -1 : at;
            p.rows[at] = none ? -1 : static_cast<int>(static_cast<uint32_t>(s) / k);
        }
    }
}

size_t place_lds_bytes(int64_t groups) {
    return 4 * static_cast<size_t>(kSortWaves * (groups + 1) + 2 * (kSortThreads + kSortWaves));
}

// The tokens of workgroup b's share.  ONE: the only workgroup, which goes on
// to the plan with the ids in LDS.
template <typename T, int LPR, int ITEMS, bool ONE>
__global__ __launch_bounds__(kSortThreads) void route_kernel(RouteArgs a, PlanArgs p) {
    extern __shared__ int lds[];
    __shared__ int ids[ONE ? kOneSlots : 1];
    constexpr int RPB = kSortThreads / LPR;
    const int lane = threadIdx.x % LPR;
    const int n = a.experts + 1;
    if (a.counts) {
        for (int e = threadIdx.x; e < n; e += kSortThreads) lds[e] = 0;
        __syncthreads();
    }
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.share;
    const int64_t t1 = t0 + a.share < a.tokens ? t0 + a.share : a.tokens;
    for (int64_t base = t0; base < t1; base += RPB) {
        const int64_t t = base + threadIdx.x / LPR;
        int id;
        float w, x[ITEMS];
        RowOf<T, LPR, ITEMS>::load(static_cast<const T*>(a.logits) + (t < t1 ? t : t1 - 1) * a.ld,
                                   a.experts, lane, x);  // past the last: again
        route_row<T, LPR, ITEMS>(a, x, lane, &id, &w);
        if (t < t1 && lane < a.k) {
            a.weights[t * a.k + lane] = w;
            a.ids[t * a.k + lane] = id;
            if (a.counts) atomicAdd(&lds[id < 0 ? a.experts : id], 1);
            if constexpr (ONE) ids[t * a.k + lane] = id < 0 ? a.experts : id;
        }
    }
    if constexpr (ONE) {
        __syncthreads();
        place_slots(p, 0, p.slots, lds, [&](int64_t s) { return ids[s]; });
    } else if (a.counts) {
        __syncthreads();
        for (int e = threadIdx.x; e < n; e += kSortThreads)
            a.counts[static_cast<int64_t>(blockIdx.x) * n + e] = lds[e];
    }
}

__device__ __forceinline__ int group_of(const PlanArgs& p, int64_t s) {
    const int g = p.ids[s];
    return static_cast<uint32_t>(g) < static_cast<uint32_t>(p.groups) ? g : p.groups;
}

__global__ __launch_bounds__(kSortThreads) void plan_count_kernel(PlanArgs p, int32_t* counts) {
    extern __shared__ int lds[];
    const int n = p.groups + 1;
    for (int e = threadIdx.x; e < n; e += kSortThreads) lds[e] = 0;
    __syncthreads();
    const int64_t s0 = static_cast<int64_t>(blockIdx.x) * p.share;
    const int64_t s1 = s0 + p.share < p.slots ? s0 + p.share : p.slots;
    for (int64_t s = s0 + threadIdx.x; s < s1; s += kSortThreads)
        atomicAdd(&lds[group_of(p, s)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e < n; e += kSortThreads)
        counts[static_cast<int64_t>(blockIdx.x) * n + e] = lds[e];
}

__global__ __launch_bounds__(kSortThreads) void plan_place_kernel(PlanArgs p) {
    extern __shared__ int lds[];
    const int64_t s0 = static_cast<int64_t>(blockIdx.x) * p.share;
    const int64_t s1 = s0 + p.share < p.slots ? s0 + p.share : p.slots;
    place_slots(p, s0, s1, lds, [&](int64_t s) { return group_of(p, s); });
}

// dlogits of one row by a group of LPR lanes.
template <typename T, int LPR, int ITEMS>
__global__ __launch_bounds__(256) void route_backward_kernel(RouteArgs a) {
    using R = RowOf<T, LPR, ITEMS>;
    const int lane = threadIdx.x % LPR;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / LPR) + threadIdx.x / LPR;
    const int64_t t = row < a.tokens ? row : a.tokens - 1;  // every lane joins the shuffles
    int id = -1;
    float w = 0.0f, dw = 0.0f;
    if (lane < a.k) {
        id = a.ids[t * a.k + lane];
        w = a.weights[t * a.k + lane];
        if (id >= 0) dw = a.dweights[t * a.k + lane];
    }
    // without an expert the place's weight is 0 (NaN in a row of NaN: kept)
    const float inner = group_sum<LPR>(id >= 0 ? dw * w : 0.0f);
    const float at_chosen = a.renorm ? w * (dw - inner) : dw;
    float g[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) g[i] = 0.0f;
    const int k = static_cast<int>(a.k);
    for (int j = 0; j < k; ++j) {
        const int c = __shfl(id, j, LPR);
        const float v = __shfl(at_chosen, j, LPR);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (R::column(lane, i) == c) g[i] = v;
    }
    if (!a.renorm) {
        float x[ITEMS];
        R::load(static_cast<const T*>(a.logits) + t * a.ld, a.experts, lane, x);
        const float total = R::exps(R::largest(x), x);
        const float r = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) g[i] = x[i] * r * (g[i] - inner);
    }
    if (row >= a.tokens) return;
    T* out = static_cast<T*>(a.dlogits) + t * a.lddl;
#pragma unroll
    for (int b = 0; b < ITEMS / R::VEC; ++b) {
        const int c = (b * LPR + lane) * R::VEC;
        float v[R::VEC];
#pragma unroll
        for (int u = 0; u < R::VEC; ++u) v[u] = g[b * R::VEC + u];
        store_floats<T, R::VEC>(out + c, a.experts - c, v);
    }
}

// The lanes and values a lane of a row: 16 lanes where its experts and places
// fit (65,536 rows of 128: fewer reduction steps and four rows a wavefront).
template <typename F>
void with_row_shape(int64_t experts, int64_t k, F&& fn) {
    if (k <= 16 && experts <= 64)
        fn(std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
    else if (k <= 16 && experts <= 128)
        fn(std::integral_constant<int, 16>{}, std::integral_constant<int, 8>{});
    else if (experts <= 256 && k <= 16)
        fn(std::integral_constant<int, 16>{}, std::integral_constant<int, 16>{});
    else if (experts <= 256)
        fn(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
    else
        fn(std::integral_constant<int, 64>{}, std::integral_constant<int, 16>{});
}

// ---------------------------------------------------------------------------
// The join: a wavefront takes 64 VEC columns of a row, its places and weights
// wave-uniform; four rows of y are in flight.
// ---------------------------------------------------------------------------
struct CombineArgs {
    int64_t tokens, k, cols, y_rows;
    const void* y;
    int64_t ldy;
    const int32_t* position;
    const float* weights;
    void* out;
    int64_t ldo;
    const void* dout;  // backward
    int64_t lddo;
    void* dy;
    int64_t lddy;
    float* dweights;
    int chunks;  // forward: column chunks of a row
};

template <typename T>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a) {
    constexpr int VEC = kVec<T>;
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 +
                      __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t t = w / a.chunks;
    if (t >= a.tokens) return;
    const int64_t c = ((w % a.chunks) * kWave + lane) * VEC;
    const T* y = static_cast<const T*>(a.y);
    float s[VEC] = {};
    for (int64_t j0 = 0; j0 < a.k; j0 += 4) {
        float v[4][VEC], f[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t i = t * a.k + j0 + u;
            const int64_t p = j0 + u < a.k ? a.position[i] : -1;
            const bool in = p >= 0 && p < a.y_rows;
            f[u] = !in ? 0.0f : a.weights ? a.weights[i] : 1.0f;
            load_floats<T, VEC>(y + (in ? p * a.ldy : 0) + c, in ? a.cols - c : 0, v[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < VEC; ++e) s[e] = __builtin_fmaf(f[u], v[u][e], s[e]);
    }
    store_floats<T, VEC>(static_cast<T*>(a.out) + t * a.ldo + c, a.cols - c, s);
}

// A wavefront takes a row: dout stays in registers for kDoutChunks chunks of
// columns while the row's places go by, eight at a time.
constexpr int kDoutChunks = 2, kPlaces = 8;

template <typename T>
__global__ __launch_bounds__(256) void combine_backward_kernel(CombineArgs a) {
    constexpr int VEC = kVec<T>;
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 +
                      __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (t >= a.tokens) return;
    const T* dout = static_cast<const T*>(a.dout) + t * a.lddo;
    for (int64_t j0 = 0; j0 < a.k; j0 += kPlaces) {
        float dot[kPlaces] = {};
        for (int64_t c0 = 0; c0 < a.cols; c0 += kDoutChunks * kWave * VEC) {
            float d[kDoutChunks][VEC];
#pragma unroll
            for (int b = 0; b < kDoutChunks; ++b) {
                const int64_t c = c0 + (b * kWave + lane) * VEC;
                load_floats<T, VEC>(dout + c, a.cols - c, d[b]);
            }
#pragma unroll
            for (int u = 0; u < kPlaces; ++u) {
                if (j0 + u >= a.k) break;
                const int64_t p = a.position[t * a.k + j0 + u];
                if (p < 0 || p >= a.y_rows) continue;
                const float f = a.weights ? a.weights[t * a.k + j0 + u] : 1.0f;
#pragma unroll
                for (int b = 0; b < kDoutChunks; ++b) {
                    const int64_t c = c0 + (b * kWave + lane) * VEC;
                    float v[VEC];
                    if (a.dweights) {
                        load_floats<T, VEC>(static_cast<const T*>(a.y) + p * a.ldy + c, a.cols - c,
                                            v);
#pragma unroll
                        for (int e = 0; e < VEC; ++e)
                            dot[u] = __builtin_fmaf(d[b][e], v[e], dot[u]);
                    }
                    if (a.dy) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) v[e] = f * d[b][e];
                        store_floats<T, VEC>(static_cast<T*>(a.dy) + p * a.lddy + c, a.cols - c, v);
                    }
                }
            }
        }
        if (a.dweights == nullptr) continue;
#pragma unroll
        for (int u = 0; u < kPlaces; ++u) {
            if (j0 + u >= a.k) break;
            const float s = wave_sum(dot[u]);
            if (lane == 0) a.dweights[t * a.k + j0 + u] = s;
        }
    }
}

void check_route(const char* what, int64_t tokens, int64_t experts, int64_t k, int64_t ld,
                 int type) {
    const std::string w = what;
    require(tokens >= 0 && experts >= 0 && k >= 0, w + ": negative dimension");
    require(experts >= 1 && experts <= kMaxGroups, w + ": between 1 and 1024 experts, got " +
                                                       std::to_string(experts));
    require(k >= 1 && k <= kMaxTop && k <= experts,
            w + ": k must be between 1 and min(32, experts), got " + std::to_string(k));
    require(tokens * k < (int64_t(1) << 31), w + ": tokens * k must be < 2^31");
    require(ld >= experts, w + ": leading dimension below experts");
    require(type >= TG_TYPE_F32 && type <= TG_TYPE_F16, w + ": unknown element type " +
                                                            std::to_string(type));
}

// Workgroups that n rows or slots go to, `least` each at least.
int64_t plan_blocks(int64_t n, int64_t least) { return std::min(kSortBlocks, ceil_div(n, least)); }

bool one_route(int64_t tokens, int64_t k) {
    return tokens <= kOneTokens && tokens * k <= kOneSlots;
}

size_t counts_bytes(int64_t blocks, int64_t groups) {
    Carver c(nullptr, 0);
    c.take<int32_t>(static_cast<size_t>(blocks * (groups + 1)));
    return c.bytes();
}

// Workgroups that route `tokens` rows: 64 rows each at least.
int64_t route_blocks(int64_t tokens) { return plan_blocks(tokens, 64); }

}  // namespace
}  // namespace tg

using tg::guard;
using tg::require;

extern "C" {

size_t tg_route_workspace_size(int64_t tokens, int64_t experts, int64_t k) {
    if (tokens <= 0 || experts <= 0 || k <= 0 || tg::one_route(tokens, k)) return 0;
    return tg::counts_bytes(tg::route_blocks(tokens), experts);
}

int tg_route(int64_t tokens, int64_t experts, int64_t k, int type, const void* logits,
             int64_t ld, int renormalize, float* weights, int32_t* expert_ids,
             int32_t* offsets, int32_t* rows, int32_t* position, void* workspace,
             size_t workspace_bytes, tg_stream_t stream) {
    return guard([&] {
        tg::check_route("route", tokens, experts, k, ld, type);
        const bool plan = offsets || rows || position;
        require(!plan || offsets, "route: offsets, rows and position go together");
        require(tokens == 0 || (logits && weights && expert_ids), "route: null pointer");
        require(!plan || tokens == 0 || (rows && position),
                "route: offsets, rows and position go together");
        hipStream_t s = static_cast<hipStream_t>(stream);
        if (tokens == 0) {
            if (plan) tg::fill_i32(offsets, experts + 1, 0, s);
            return;
        }
        tg::RouteArgs a{};
        a.tokens = tokens;
        a.k = k;
        a.experts = static_cast<int>(experts);
        a.renorm = renormalize != 0;
        a.logits = logits;
        a.ld = ld;
        a.weights = weights;
        a.ids = expert_ids;
        tg::PlanArgs p{};
        p.slots = tokens * k;
        p.k = k;
        p.groups = a.experts;
        p.ids = expert_ids;
        p.offsets = offsets;
        p.rows = rows;
        p.position = position;
        const bool one = plan && tg::one_route(tokens, k);
        int64_t blocks = one ? 1 : tg::route_blocks(tokens);
        a.share = tg::ceil_div(tokens, blocks);
        blocks = tg::ceil_div(tokens, a.share);
        tg::TempBuffer temp;
        if (plan && !one) {
            const size_t need = tg::counts_bytes(blocks, experts);
            if (!workspace) {
                temp.allocate(need, s);
                workspace = temp.get();
                workspace_bytes = need;
            }
            tg::Carver c(workspace, workspace_bytes);
            a.counts = c.take<int32_t>(static_cast<size_t>(blocks * (experts + 1)));
            p.counts = a.counts;
            p.blocks = static_cast<int>(blocks);
            p.share = a.share * k;
        }
        const unsigned n = static_cast<unsigned>(blocks);
        const size_t sort_lds = tg::place_lds_bytes(experts);
        tg::with_type(type, "route", [&](auto t) {
            using T = decltype(t);
            tg::with_row_shape(experts, k, [&](auto lpr, auto items) {
                constexpr int L = decltype(lpr)::value, I = decltype(items)::value;
                if (one)
                    tg::route_kernel<T, L, I, true><<<1, tg::kSortThreads, sort_lds, s>>>(a, p);
                else
                    tg::route_kernel<T, L, I, false>
                        <<<n, tg::kSortThreads, plan ? 4 * (experts + 1) : 0, s>>>(a, p);
            });
        });
        TG_LAUNCH_CHECK();
        if (plan && !one) {
            tg::plan_place_kernel<<<n, tg::kSortThreads, sort_lds, s>>>(p);
            TG_LAUNCH_CHECK();
        }
    });
}

size_t tg_route_plan_workspace_size(int64_t n, int64_t groups) {
    if (n <= tg::kOneSlots || groups <= 0) return 0;
    return tg::counts_bytes(tg::plan_blocks(n, 4096), groups);
}

int tg_route_plan(int64_t n, int64_t groups, int64_t k, const int32_t* ids, int32_t* offsets,
                  int32_t* rows, int32_t* position, void* workspace, size_t workspace_bytes,
                  tg_stream_t stream) {
    return guard([&] {
        require(n >= 0 && n < (int64_t(1) << 31), "route_plan: n must be within [0, 2^31)");
        require(groups >= 1 && groups <= tg::kMaxGroups,
                "route_plan: between 1 and 1024 groups, got " + std::to_string(groups));
        require(k >= 1 && k < (int64_t(1) << 31), "route_plan: k must be positive");
        require(offsets, "route_plan: null pointer");
        hipStream_t s = static_cast<hipStream_t>(stream);
        if (n == 0) {
            tg::fill_i32(offsets, groups + 1, 0, s);
            return;
        }
        require(ids && rows && position, "route_plan: null pointer");
        tg::PlanArgs p{};
        p.slots = p.share = n;
        p.k = k;
        p.groups = static_cast<int>(groups);
        p.ids = ids;
        p.offsets = offsets;
        p.rows = rows;
        p.position = position;
        p.blocks = 1;
        tg::TempBuffer temp;
        if (n > tg::kOneSlots) {
            p.share = tg::ceil_div(n, tg::plan_blocks(n, 4096));
            p.blocks = static_cast<int>(tg::ceil_div(n, p.share));
            const size_t need = tg::counts_bytes(p.blocks, groups);
            if (!workspace) {
                temp.allocate(need, s);
                workspace = temp.get();
                workspace_bytes = need;
            }
            tg::Carver c(workspace, workspace_bytes);
            int32_t* counts = c.take<int32_t>(static_cast<size_t>(p.blocks * (groups + 1)));
            p.counts = counts;
            tg::plan_count_kernel<<<p.blocks, tg::kSortThreads, 4 * (groups + 1), s>>>(p, counts);
            TG_LAUNCH_CHECK();
        }
        tg::plan_place_kernel<<<p.blocks, tg::kSortThreads, tg::place_lds_bytes(groups), s>>>(p);
        TG_LAUNCH_CHECK();
    });
}

int tg_route_backward(int64_t tokens, int64_t experts, int64_t k, int type, const void* logits,
                      int64_t ld, int renormalize, const float* weights,
                      const int32_t* expert_ids, const float* dweights, void* dlogits,
                      int64_t lddl, tg_stream_t stream) {
    return guard([&] {
        tg::check_route("route_backward", tokens, experts, k, ld, type);
        require(lddl >= experts, "route_backward: leading dimension below experts");
        if (tokens == 0) return;
        require(logits && weights && expert_ids && dweights && dlogits,
                "route_backward: null pointer");
        tg::RouteArgs a{};
        a.tokens = tokens;
        a.k = k;
        a.experts = static_cast<int>(experts);
        a.renorm = renormalize != 0;
        a.logits = logits;
        a.ld = ld;
        a.weights = const_cast<float*>(weights);
        a.ids = const_cast<int32_t*>(expert_ids);
        a.dweights = dweights;
        a.dlogits = dlogits;
        a.lddl = lddl;
        hipStream_t s = static_cast<hipStream_t>(stream);
        tg::with_type(type, "route_backward", [&](auto t) {
            using T = decltype(t);
            tg::with_row_shape(experts, k, [&](auto lpr, auto items) {
                constexpr int L = decltype(lpr)::value, I = decltype(items)::value;
                tg::for_slices(tokens, L, [&](int64_t first, int64_t count) {
                    tg::RouteArgs b = a;
                    b.tokens = count;
                    b.logits = static_cast<const T*>(logits) + first * ld;
                    b.weights += first * k;
                    b.ids += first * k;
                    b.dweights += first * k;
                    b.dlogits = static_cast<T*>(dlogits) + first * lddl;
                    const unsigned n = static_cast<unsigned>(tg::ceil_div(count, 256 / L));
                    tg::route_backward_kernel<T, L, I><<<n, 256, 0, s>>>(b);
                });
            });
        });
        TG_LAUNCH_CHECK();
    });
}

int tg_route_combine(int64_t tokens, int64_t k, int64_t cols, int type, const void* y,
                     int64_t y_rows, int64_t ldy, const int32_t* position,
                     const float* weights, void* out, int64_t ldo, tg_stream_t stream) {
    return guard([&] {
        require(tokens >= 0 && k >= 0 && cols >= 0 && y_rows >= 0,
                "route_combine: negative dimension");
        require(tokens < (int64_t(1) << 31) && cols < (int64_t(1) << 31) &&
                    (k == 0 || tokens * k < (int64_t(1) << 31)),
                "route_combine: tokens * k and cols must be < 2^31");
        require(ldo >= cols && ldy >= cols, "route_combine: leading dimension below cols");
        require(type >= TG_TYPE_F32 && type <= TG_TYPE_F16,
                "route_combine: unknown element type " + std::to_string(type));
        if (tokens == 0 || cols == 0) return;
        require(out && (k == 0 || position) && (y_rows == 0 || y), "route_combine: null pointer");
        tg::CombineArgs a{};
        a.tokens = tokens;
        a.k = k;
        a.cols = cols;
        a.y_rows = y_rows;
        a.y = y;
        a.ldy = ldy;
        a.position = position;
        a.weights = weights;
        a.out = out;
        a.ldo = ldo;
        hipStream_t s = static_cast<hipStream_t>(stream);
        tg::with_type(type, "route_combine", [&](auto t) {
            using T = decltype(t);
            const int64_t chunks = tg::ceil_div(cols, tg::kWave * tg::kVec<T>);
            a.chunks = static_cast<int>(chunks);
            tg::for_slices(tokens, chunks * tg::kWave, [&](int64_t first, int64_t count) {
                tg::CombineArgs b = a;
                b.tokens = count;
                b.position += first * k;
                if (weights) b.weights += first * k;
                b.out = static_cast<T*>(out) + first * ldo;
                const unsigned n = static_cast<unsigned>(tg::ceil_div(count * chunks, 4));
                tg::combine_kernel<T><<<n, 256, 0, s>>>(b);
            });
        });
        TG_LAUNCH_CHECK();
    });
}

int tg_route_combine_backward(int64_t tokens, int64_t k, int64_t cols, int type,
                              const void* dout, int64_t lddo, const void* y, int64_t y_rows,
                              int64_t ldy, const int32_t* position, const float* weights,
                              void* dy, int64_t lddy, float* dweights, tg_stream_t stream) {
    return guard([&] {
        require(tokens >= 0 && k >= 0 && cols >= 0 && y_rows >= 0,
                "route_combine_backward: negative dimension");
        require(tokens < (int64_t(1) << 31) && cols < (int64_t(1) << 31) &&
                    (k == 0 || tokens * k < (int64_t(1) << 31)),
                "route_combine_backward: tokens * k and cols must be < 2^31");
        require(lddo >= cols && (!dweights || ldy >= cols) && (!dy || lddy >= cols),
                "route_combine_backward: leading dimension below cols");
        require(type >= TG_TYPE_F32 && type <= TG_TYPE_F16,
                "route_combine_backward: unknown element type " + std::to_string(type));
        if (tokens == 0 || k == 0 || (!dy && !dweights)) return;
        require(position && (cols == 0 || (dout && (!dweights || y_rows == 0 || y))),
                "route_combine_backward: null pointer");
        tg::CombineArgs a{};
        a.tokens = tokens;
        a.k = k;
        a.cols = cols;
        a.y_rows = y_rows;
        a.y = y;
        a.ldy = ldy;
        a.position = position;
        a.weights = weights;
        a.dout = dout;
        a.lddo = lddo;
        a.dy = dy;
        a.lddy = lddy;
        a.dweights = dweights;
        hipStream_t s = static_cast<hipStream_t>(stream);
        tg::with_type(type, "route_combine_backward", [&](auto t) {
            using T = decltype(t);
            tg::for_slices(tokens, tg::kWave, [&](int64_t first, int64_t count) {
                tg::CombineArgs b = a;
                b.tokens = count;
                b.position += first * k;
                if (weights) b.weights += first * k;
                if (dweights) b.dweights += first * k;
                b.dout = static_cast<const T*>(dout) + first * lddo;
                const unsigned n = static_cast<unsigned>(tg::ceil_div(count, 4));
                tg::combine_backward_kernel<T><<<n, 256, 0, s>>>(b);
            });
        });
        TG_LAUNCH_CHECK();
    });
}

}  // extern "C"
