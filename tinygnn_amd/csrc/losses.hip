// losses.hip -- what a classifier answers and learns from: how rows are cut, and the
// entry points (losses_kernels.hpp has the kernels).
#include "losses.hpp"

#include <cmath>
#include <string>

namespace tg {
namespace {

void check_losses(const std::string& w, int64_t rows, int64_t classes, int type,
                  float temperature) {
    require(rows >= 0 && classes >= 0, w + ": negative dimension");
    require(classes >= 1, w + ": no classes");
    require(rows < (int64_t(1) << 31) - 4096 && classes < (int64_t(1) << 31) - 4096,
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
    a.c = static_cast<float>(1.4426950408889634 / static_cast<double>(temperature));
    return a;
}

// How rows are cut: one segment, but few long rows: of more than 80,000 bytes where
// there are fewer than 128 (as many as give 256 workgroups), of 190,000, with top
// classes 300,000, where fewer than 1,024 (1,024 workgroups), each of 4,096 classes at
// least, 64 at most; and rows longer than a workgroup holds.  Over 1 to 1,500 rows of
// 20,000 to 250,000 fp32 and bf16 within 3% in the mean of the best of 1, 256, 512
// and 1,024 workgroups: 1 x 131,072 fp32 with 20 top classes 18.0 us in two, 10.5 in
// 32; 200 x 131,072 fp32 28.0 in 400, 21.3 in 1,200; but 1 x 20,000 fp32 4.3 in one, 5.2
// in five, 200 x 100,003 bf16 15.9 in 200, 20.6 in 400.  (A distillation with its
// gradient reads cut rows twice, the others once.)
struct Cut {
    int64_t segment, segments;
};

Cut cut_of(int64_t rows, int64_t classes, int type, bool tops) {
    const int64_t vec = 16 / type_size(type), most = kMostChunks * vec;
    const bool some = rows < 128;
    int64_t segments = 1;
    if (rows < 1024 && classes * type_size(type) > (some ? 80000 : tops ? 300000 : 190000))
        segments =
            std::min<int64_t>({ceil_div(some ? 256 : 1024, rows), ceil_div(classes, 4096), 64});
    segments = std::max(segments, ceil_div(classes, most));
    const int64_t segment = ceil_div(ceil_div(classes, segments), vec) * vec;
    return {segment, ceil_div(classes, segment)};
}

struct LossPlace {
    float* part;
    Key* keys;
    float* row_part;
    float* q;
    size_t bytes;
};

LossPlace loss_place(int64_t rows, int64_t classes, int64_t top, int64_t k, int type, void* ws,
                     size_t size) {
    LossPlace p{};
    const Cut cut = cut_of(rows, classes, type, top > 0);
    if (cut.segments == 1) return p;
    Carver c(ws, size);
    const size_t parts = static_cast<size_t>(rows) * cut.segments;
    p.part = c.take<float>(4 * parts);
    if (top) p.keys = c.take<Key>(parts * top);
    if (k) {
        p.row_part = c.take<float>(4 * static_cast<size_t>(rows));
        p.q = c.take<float>(static_cast<size_t>(rows) * k);
    }
    p.bytes = c.bytes();
    return p;
}

// The workspace's pieces into a; whether the rows are cut.
bool place_segments(LossArgs& a, int type, void* workspace, size_t bytes, TempBuffer* temp,
                    hipStream_t s) {
    const Cut cut = cut_of(a.rows, a.classes, type, a.top > 0);
    a.segment = cut.segment;
    a.segments = static_cast<int>(cut.segments);
    if (cut.segments == 1) return false;
    const size_t need = loss_place(a.rows, a.classes, a.top, a.k, type, nullptr, 0).bytes;
    if (!workspace) {
        temp->allocate(need, s);
        workspace = temp->get();
        bytes = need;
    }
    const LossPlace p = loss_place(a.rows, a.classes, a.top, a.k, type, workspace, bytes);
    a.part = p.part;
    a.part_keys = p.keys;
    a.row_part = p.row_part;
    a.q = p.q;
    return true;
}

size_t loss_bytes(int64_t rows, int64_t classes, int64_t top, int64_t k, int type) {
    if (rows <= 0 || classes <= 0 || type < TG_TYPE_F32 || type > TG_TYPE_F16) return 0;
    return loss_place(rows, classes, top, k, type, nullptr, 0).bytes;
}

}  // namespace
}  // namespace tg

using tg::guard;
using tg::require;

extern "C" {

size_t tg_log_probs_workspace_size(int64_t rows, int64_t classes, int64_t top, int type) {
    return tg::loss_bytes(rows, classes, top < 0 ? 0 : top, 0, type);
}

int tg_log_probs(int64_t rows, int64_t classes, int type, const void* logits, int64_t ld,
                 const int32_t* labels, float temperature, int64_t top, float* value,
                 float* entropy, float* top_values, int32_t* top_ids, float* stats,
                 void* workspace, size_t workspace_bytes, tg_stream_t stream) {
    return guard([&] {
        const std::string what = "log_probs";
        tg::check_losses(what, rows, classes, type, temperature);
        require(top >= 0 && top <= tg::kMaxTop && top <= classes,
                what + ": top must be between 0 and min(64, classes), got " + std::to_string(top));
        require(ld >= classes, what + ": leading dimension below classes");
        require((labels == nullptr) == (value == nullptr) || rows == 0,
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
        tg::TempBuffer temp;
        const bool cut = tg::place_segments(a, type, workspace, workspace_bytes, &temp, s);
        tg::with_type(type, "log_probs",
                      [&](auto t) { tg::losses_log_probs<decltype(t)>(a, cut, s); });
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
        require((labels == nullptr) == (dvalue == nullptr) || rows == 0,
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
        tg::with_type(type, "log_probs_backward",
                      [&](auto t) { tg::losses_log_probs_backward<decltype(t)>(a, s); });
    });
}

size_t tg_distill_workspace_size(int64_t rows, int64_t classes, int64_t k, int type) {
    return tg::loss_bytes(rows, classes, 0, k < 0 ? 0 : k, type);
}

int tg_distill(int64_t rows, int64_t classes, int64_t k, int type, const void* logits, int64_t ld,
               int teacher_type, const void* teacher, const int32_t* ids, float temperature,
               float* loss, const float* dloss, void* dlogits, int64_t lddl, void* workspace,
               size_t workspace_bytes, tg_stream_t stream) {
    return guard([&] {
        const std::string what = "distill";
        tg::check_losses(what, rows, classes, type, temperature);
        require(teacher_type >= TG_TYPE_F32 && teacher_type <= TG_TYPE_F16,
                what + ": unknown element type " + std::to_string(teacher_type));
        require(k >= 1 && k <= tg::kMaxTeacher,
                what + ": k must be between 1 and 256, got " + std::to_string(k));
        require(ld >= classes && (!dlogits || lddl >= classes),
                what + ": leading dimension below classes");
        require((dloss == nullptr) == (dlogits == nullptr) || rows == 0,
                what + ": dloss and dlogits go together");
        if (rows == 0) return;
        require(logits && teacher && ids && loss, what + ": null pointer");
        tg::LossArgs a = tg::loss_args(rows, classes, logits, ld, temperature);
        a.k = static_cast<int>(k);
        a.teacher_type = teacher_type;
        a.teacher = teacher;
        a.ids = ids;
        a.loss = loss;
        a.dloss = dloss;
        a.dlogits = dlogits;
        a.lddl = lddl;
        hipStream_t s = static_cast<hipStream_t>(stream);
        tg::TempBuffer temp;
        const bool cut = tg::place_segments(a, type, workspace, workspace_bytes, &temp, s);
        tg::with_type(type, "distill",
                      [&](auto t) { tg::losses_distill<decltype(t)>(a, cut, s); });
    });
}

}  // extern "C"
