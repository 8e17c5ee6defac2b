// losses.hip -- what a classifier answers and learns from: log probabilities of
// given classes with the entropy and the likeliest classes, the divergence from a
// teacher's top logits, and their gradients.
//
// One workgroup a row, which reads it from memory for the maximum, for the sums,
// once for each of the top places and for the gradient.
#include "common.hpp"
#include "device_utils.hpp"
#include "types.hpp"

#include <cmath>
#include <string>

namespace tg {
namespace {

constexpr int64_t kMaxTop = 64, kMaxTeacher = 256;
constexpr int kThreads = 256;

struct LossArgs {
    int64_t rows, classes;
    const void* logits;
    int64_t ld;
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
    int k;
    const void* teacher;
    const int32_t* ids;
    const float* dloss;
    float* loss;
};

// What a row's sums say: z = (x - m) / T, s = sum of exp(z), log s.
struct RowStats {
    float m, log_s;
    __device__ bool empty() const { return m == -INFINITY && log_s == 0.0f; }
    __device__ float logp(float x, float inv) const { return (x - m) * inv - log_s; }
    __device__ float p(float x, float inv) const { return __expf(logp(x, inv)); }
};

template <int OP>
__device__ float block_reduce(float v) {
    __shared__ float lds[kThreads / kWave];
    v = OP ? wave_max(v) : wave_sum(v);
    __syncthreads();
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    v = lds[0];
    for (int w = 1; w < kThreads / kWave; ++w) v = OP ? (lds[w] > v ? lds[w] : v) : v + lds[w];
    return v;
}

template <typename T>
__device__ RowStats row_stats(const T* x, int64_t n, float inv, float* s_out, float* u_out) {
    float m = -INFINITY;
    for (int64_t i = threadIdx.x; i < n; i += kThreads) {
        const float v = static_cast<float>(x[i]);
        m = v > m ? v : m;
    }
    m = block_reduce<1>(m);
    float s = 0.0f, u = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += kThreads) {
        const float v = static_cast<float>(x[i]);
        if (v == -INFINITY) continue;
        const float z = (v - m) * inv, e = __expf(z);
        s += e;
        u += e == 0.0f ? 0.0f : e * z;
    }
    *s_out = s = block_reduce<0>(s);
    *u_out = block_reduce<0>(u);
    return {m, s == 0.0f ? 0.0f : logf(s)};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void log_probs_kernel(LossArgs a) {
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    float s, u;
    const RowStats r = row_stats(x, a.classes, a.inv, &s, &u);
    if (threadIdx.x == 0) {
        if (a.stats) {
            a.stats[2 * row] = r.m;
            a.stats[2 * row + 1] = r.log_s;
        }
        if (a.value) {
            const int y = a.labels[row];
            const bool in = y >= 0 && y < a.classes;
            a.value[row] = !in ? 0.0f : r.empty() ? -INFINITY
                                                  : r.logp(static_cast<float>(x[y]), a.inv);
        }
        if (a.entropy) a.entropy[row] = s == 0.0f ? 0.0f : r.log_s - u / s;
    }
    // place j: the largest behind place j - 1
    float last = INFINITY;
    int at = -1;
    for (int j = 0; j < a.top; ++j) {
        __shared__ int best_at;
        float best = -INFINITY;
        int mine = 0x7fffffff;
        for (int64_t i = threadIdx.x; i < a.classes; i += kThreads) {
            const float v = static_cast<float>(x[i]);
            const bool behind = v < last || (v == last && i > at);
            if (behind && v > best) {
                best = v;
                mine = static_cast<int>(i);
            }
        }
        const float v = block_reduce<1>(best);
        if (threadIdx.x == 0) best_at = 0x7fffffff;
        __syncthreads();
        if (best == v && v > -INFINITY) atomicMin(&best_at, mine);
        __syncthreads();
        const bool none = v == -INFINITY;
        last = v;
        at = best_at;
        __syncthreads();
        if (threadIdx.x == 0) {
            a.top_values[row * a.top + j] = none ? -INFINITY : r.logp(v, a.inv);
            a.top_ids[row * a.top + j] = none ? -1 : at;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void log_probs_backward_kernel(LossArgs a) {
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    T* out = static_cast<T*>(a.dlogits) + row * a.lddl;
    const RowStats r = {a.stats[2 * row], a.stats[2 * row + 1]};
    const int y = a.labels ? a.labels[row] : -1;
    const float g = y >= 0 && y < a.classes && a.dvalue ? a.dvalue[row] * a.inv : 0.0f;
    const float h = a.dentropy ? a.dentropy[row] * a.inv : 0.0f;
    const float entropy = a.dentropy ? a.entropy[row] : 0.0f;
    const bool zero = (g == 0.0f && h == 0.0f) || r.empty();
    for (int64_t i = threadIdx.x; i < a.classes; i += kThreads) {
        const float v = static_cast<float>(x[i]);
        const float p = r.p(v, a.inv);
        float d = (i == y ? g : 0.0f) - g * p;
        if (h != 0.0f && p != 0.0f) d -= h * p * (r.logp(v, a.inv) + entropy);
        out[i] = static_cast<T>(zero ? 0.0f : d);
    }
}

template <typename T, typename U>
__global__ __launch_bounds__(kThreads) void distill_kernel(LossArgs a) {
    __shared__ float q[kMaxTeacher], xs[kMaxTeacher];
    __shared__ int id[kMaxTeacher];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    float s, u;
    const RowStats r = row_stats(x, a.classes, a.inv, &s, &u);
    float t = -INFINITY;
    const int j = threadIdx.x;
    if (j < a.k) {
        const int c = a.ids[row * a.k + j];
        const bool in = c >= 0 && c < a.classes;
        id[j] = in ? c : -1;
        xs[j] = in ? static_cast<float>(x[c]) : 0.0f;
        if (in) t = static_cast<float>(static_cast<const U*>(a.teacher)[row * a.k + j]);
    }
    const float tm = block_reduce<1>(t);
    const float z = (t - tm) * a.inv, e = t == -INFINITY ? 0.0f : __expf(z);
    const float total = block_reduce<0>(e);
    const float mine = total == 0.0f ? 0.0f : e / total;
    if (j < a.k) q[j] = mine;
    const float logp = j >= a.k || mine == 0.0f ? 0.0f
                       : r.empty()              ? -INFINITY
                                                : r.logp(xs[j], a.inv);
    const float loss =
        block_reduce<0>(mine == 0.0f ? 0.0f : mine * (z - logf(total) - logp));
    if (j == 0) a.loss[row] = loss;
    if (!a.dlogits) return;
    T* out = static_cast<T*>(a.dlogits) + row * a.lddl;
    const float g = a.dloss[row] * a.inv * (total / total);  // NaN in the teacher: in the row
    const bool zero = a.dloss[row] == 0.0f || total == 0.0f || r.empty();
    __syncthreads();
    for (int64_t i = threadIdx.x; i < a.classes; i += kThreads) {
        float d = r.p(static_cast<float>(x[i]), a.inv);
        for (int w = 0; w < a.k; ++w)
            if (id[w] == i) d -= q[w];
        out[i] = static_cast<T>(zero ? 0.0f : g * d);
    }
}

void check_losses(const std::string& w, int64_t rows, int64_t classes, int type,
                  float temperature) {
    require(rows >= 0 && classes >= 0, w + ": negative dimension");
    require(classes >= 1, w + ": no classes");
    require(rows < (int64_t(1) << 31) && classes < (int64_t(1) << 31) - 4096,
            w + ": rows and classes must be < 2^31 - 4096");
    require(type >= TG_TYPE_F32 && type <= TG_TYPE_F16, w + ": unknown element type " +
                                                            std::to_string(type));
    require(std::isfinite(temperature) && temperature >= 1e-4f && temperature <= 1e4f,
            w + ": temperature must be between 1e-4 and 1e4");
}

LossArgs loss_args(int64_t rows, int64_t classes, const void* logits, int64_t ld,
                   float temperature) {
    LossArgs a{};
    a.rows = rows;
    a.classes = classes;
    a.logits = logits;
    a.ld = ld;
    a.inv = static_cast<float>(1.0 / static_cast<double>(temperature));
    return a;
}

}  // namespace
}  // namespace tg

using tg::guard;
using tg::require;

extern "C" {

size_t tg_log_probs_workspace_size(int64_t rows, int64_t classes, int64_t top, int type) {
    (void)rows, (void)classes, (void)top, (void)type;
    return 0;
}

int tg_log_probs(int64_t rows, int64_t classes, int type, const void* logits, int64_t ld,
                 const int32_t* labels, float temperature, int64_t top, float* value,
                 float* entropy, float* top_values, int32_t* top_ids, float* stats,
                 void* workspace, size_t workspace_bytes, tg_stream_t stream) {
    return guard([&] {
        const std::string what = "log_probs";
        (void)workspace, (void)workspace_bytes;
        tg::check_losses(what, rows, classes, type, temperature);
        require(top >= 0 && top <= tg::kMaxTop && top <= classes,
                what + ": top must be between 0 and min(64, classes), got " + std::to_string(top));
        require(ld >= classes, what + ": leading dimension below classes");
        require((labels == nullptr) == (value == nullptr),
                what + ": labels and their values go together");
        if (rows == 0) return;
        require(logits && (top == 0 || (top_values && top_ids)), what + ": null pointer");
        tg::LossArgs a = tg::loss_args(rows, classes, logits, ld, temperature);
        a.labels = labels;
        a.top = static_cast<int>(top);
        a.value = value;
        a.entropy = entropy;
        a.top_values = top_values;
        a.top_ids = top_ids;
        a.stats = stats;
        hipStream_t s = static_cast<hipStream_t>(stream);
        tg::with_type(type, "log_probs", [&](auto t) {
            tg::log_probs_kernel<decltype(t)><<<rows, tg::kThreads, 0, s>>>(a);
        });
        TG_LAUNCH_CHECK();
    });
}

int tg_log_probs_backward(int64_t rows, int64_t classes, int type, const void* logits, int64_t ld,
                          const int32_t* labels, float temperature, const float* stats,
                          const float* entropy, const float* dvalue, const float* dentropy,
                          void* dlogits, int64_t lddl, tg_stream_t stream) {
    return guard([&] {
        const std::string what = "log_probs_backward";
        tg::check_losses(what, rows, classes, type, temperature);
        require(ld >= classes && lddl >= classes, what + ": leading dimension below classes");
        require((labels == nullptr) == (dvalue == nullptr),
                what + ": labels and dvalue go together");
        require(!dentropy || entropy || rows == 0, what + ": dentropy needs the entropy");
        if (rows == 0) return;
        require(logits && stats && dlogits, what + ": null pointer");
        tg::LossArgs a = tg::loss_args(rows, classes, logits, ld, temperature);
        a.labels = labels;
        a.stats = const_cast<float*>(stats);
        a.entropy = const_cast<float*>(entropy);
        a.dvalue = dvalue;
        a.dentropy = dentropy;
        a.dlogits = dlogits;
        a.lddl = lddl;
        hipStream_t s = static_cast<hipStream_t>(stream);
        tg::with_type(type, "log_probs_backward", [&](auto t) {
            tg::log_probs_backward_kernel<decltype(t)><<<rows, tg::kThreads, 0, s>>>(a);
        });
        TG_LAUNCH_CHECK();
    });
}

size_t tg_distill_workspace_size(int64_t rows, int64_t classes, int64_t k, int type) {
    (void)rows, (void)classes, (void)k, (void)type;
    return 0;
}

int tg_distill(int64_t rows, int64_t classes, int64_t k, int type, const void* logits, int64_t ld,
               int teacher_type, const void* teacher, const int32_t* ids, float temperature,
               float* loss, const float* dloss, void* dlogits, int64_t lddl, void* workspace,
               size_t workspace_bytes, tg_stream_t stream) {
    return guard([&] {
        const std::string what = "distill";
        (void)workspace, (void)workspace_bytes;
        tg::check_losses(what, rows, classes, type, temperature);
        require(teacher_type >= TG_TYPE_F32 && teacher_type <= TG_TYPE_F16,
                what + ": unknown element type " + std::to_string(teacher_type));
        require(k >= 1 && k <= tg::kMaxTeacher,
                what + ": k must be between 1 and 256, got " + std::to_string(k));
        require(ld >= classes && (!dlogits || lddl >= classes),
                what + ": leading dimension below classes");
        require((dloss == nullptr) == (dlogits == nullptr),
                what + ": dloss and dlogits go together");
        if (rows == 0) return;
        require(logits && teacher && ids && loss, what + ": null pointer");
        tg::LossArgs a = tg::loss_args(rows, classes, logits, ld, temperature);
        a.k = static_cast<int>(k);
        a.teacher = teacher;
        a.ids = ids;
        a.loss = loss;
        a.dloss = dloss;
        a.dlogits = dlogits;
        a.lddl = lddl;
        hipStream_t s = static_cast<hipStream_t>(stream);
        tg::with_type(type, "distill", [&](auto t) {
            tg::with_type(teacher_type, "distill", [&](auto u) {
                tg::distill_kernel<decltype(t), decltype(u)><<<rows, tg::kThreads, 0, s>>>(a);
            });
        });
        TG_LAUNCH_CHECK();
    });
}

}  // extern "C"
