// losses.hpp -- arguments of the losses' kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"
#include "types.hpp"

namespace tg {

constexpr int64_t kMaxTop = 64, kMaxTeacher = 256;
constexpr int kTinyClasses = 128, kTinyPlaces = 64;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

typedef unsigned long long Key;

struct LossArgs {
    int64_t row0, rows, classes;  // rows [row0, rows)
    const void* logits;
    int64_t ld;
    float c;    // log2(e) / temperature
    float inv;  // 1 / temperature
    const int32_t* labels;
    int top;
    float* value;
    float* entropy;
    float* top_values;
    int32_t* top_ids;
    float* stats;
    // backward
    const float* dvalue;
    const float* dentropy;
    void* dlogits;
    int64_t lddl;
    // teacher
    int k, teacher_type;
    const void* teacher;
    const int32_t* ids;
    const float* dloss;
    float* loss;
    // segments
    int64_t segment;  // classes of one
    int segments;
    float* part;      // [rows][segments][4]: m, s, u
    Key* part_keys;   // [rows][segments][top]
    float* row_part;  // distillation: [rows][4]: m, factor / s, factor
    float* q;         // [rows][k]
};

// The most chunks of 16 bytes of a row or segment that a workgroup holds.
constexpr int64_t kMostChunks = 1024 * 16;

// The launches of one element type.
template <typename T>
void losses_log_probs(const LossArgs& a, bool cut, hipStream_t s);
template <typename T>
void losses_log_probs_backward(const LossArgs& a, hipStream_t s);
template <typename T>
void losses_distill(const LossArgs& a, bool cut, hipStream_t s);

}  // namespace tg
