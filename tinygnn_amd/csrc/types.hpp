// types.hpp -- element types of the expert-layer operators: float, bf16, fp16
// in memory, float in the kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <string>

#include "tinygnn_amd.h"

namespace tg {

typedef __bf16 bf16;
typedef _Float16 f16;

// Runs fn with a value of the element type that `type` (TG_TYPE_*) names.
template <typename F>
void with_type(int type, const char* what, F&& fn) {
    if (type == TG_TYPE_F32)
        fn(float{});
    else if (type == TG_TYPE_BF16)
        fn(bf16{});
    else if (type == TG_TYPE_F16)
        fn(f16{});
    else
        throw std::invalid_argument(std::string(what) + ": unknown element type " +
                                    std::to_string(type));
}

inline int64_t type_size(int type) { return type == TG_TYPE_F32 ? 4 : 2; }

// N consecutive elements at any address their type allows: gfx950's global
// loads and stores of up to 128 bits need no alignment of their own.
template <typename T, int N>
struct Pack {
    typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

// Elements in 16 bytes.
template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));

// x[0, N) = p[0, N) as floats, zeros from `left` on (left may be <= 0 or > N).
template <typename T, int N>
__device__ __forceinline__ void load_floats(const T* __restrict__ p, int64_t left, float (&x)[N]) {
    if (left >= N) {
        const auto v = *reinterpret_cast<const typename Pack<T, N>::V*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = static_cast<float>(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = i < left ? static_cast<float>(p[i]) : 0.0f;
    }
}

// p[0, min(N, left)) = x, each rounded to T once.
template <typename T, int N>
__device__ __forceinline__ void store_floats(T* __restrict__ p, int64_t left, const float (&x)[N]) {
    if (left >= N) {
        typename Pack<T, N>::V v;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = static_cast<T>(x[i]);
        *reinterpret_cast<typename Pack<T, N>::V*>(p) = v;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) p[i] = static_cast<T>(x[i]);
    }
}

// Workgroups of one launch, which has fewer than 2^32 threads.
inline unsigned grid_of(const char* what, int64_t blocks, int64_t threads) {
    require(blocks * threads < (int64_t(1) << 32), std::string(what) + ": too many elements");
    return static_cast<unsigned>(blocks);
}

// fn(first, count) for the slices of `rows` that one launch of `threads` threads
// a row can take.
template <typename F>
void for_slices(int64_t rows, int64_t threads, F&& fn) {
    const int64_t most = ((int64_t(1) << 32) - 1024) / threads;
    for (int64_t first = 0; first < rows; first += most)
        fn(first, first + most < rows ? most : rows - first);
}

}  // namespace tg
