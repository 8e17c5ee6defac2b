// linear.hip -- dense layers: y = residual + act(x w + bias), and the gradients:
// shapes, parts and entry points (linear_kernels.hpp has the kernels).
#include "linear.hpp"

#include <string>

#include "device_utils.hpp"
#include "tiles.hpp"

namespace tg {
namespace {

constexpr int64_t kLongChain = 16384;  // of floats: 64 chains of kSumTiles tiles

// How an out [m x n] with contraction k is cut.
LinearPlan linear_plan(int64_t m, int64_t n, int64_t k, int type, bool ring) {
    LinearPlan p{};
    const int64_t z = type_size(type), depth = kRowBytes / z;
    const auto tiles = [&](int64_t a, int64_t b) { return ceil_div(m, a) * ceil_div(n, b); };
    if (ring && tiles(256, 256) >= 160) {
        p.em = p.en = 256;
    } else if (m <= 32) {
        p.em = 32;
        p.en = 128;
    } else if (tiles(128, 128) >= 400) {
        p.em = p.en = 128;
    } else {
        p.em = p.en = 64;
    }
    p.mt = ceil_div(m, p.em);
    p.nt = ceil_div(n, p.en);
    const int64_t all = p.mt * p.nt;
    // parts of 4 tiles of the contraction at least, for about 512 workgroups
    int64_t parts = all >= 256 ? 1 : std::min(ceil_div(512, all), ceil_div(k, 4 * depth));
    if (type == TG_TYPE_F32) parts = std::max(parts, ceil_div(k, kLongChain));
    p.unit = std::max(depth, ceil_div(ceil_div(k, std::max<int64_t>(parts, 1)), depth) * depth);
    p.parts = std::max<int64_t>(1, ceil_div(k, p.unit));
    return p;
}

// Whether an operand's tiles of up to 256 of its rows or columns can come by
// loads to LDS: from dword-aligned rows, within 2 GB of the tile's start; across
// the contraction, in whole dwords.
bool direct_side(const void* p, int64_t ld, int64_t cols, int64_t z, bool across) {
    return reinterpret_cast<uintptr_t>(p) % 4 == 0 && ld * z % 4 == 0 &&
           (!across || cols * z % 4 == 0) && (256 * ld + cols) * z < kDirectBytes;
}

// One product with the operands' layouts; part: room for its parts.
void product(LinearArgs& a, int type, bool ax, bool aw, float* part, hipStream_t s) {
    const int64_t z = type_size(type);
    const bool direct = direct_side(a.x, a.ldx, ax ? a.m : a.k, z, ax) &&
                        direct_side(a.w, a.ldw, aw ? a.n : a.k, z, aw);
    const bool ring = direct && z == 2 && ((ax && aw) || a.k % 8 == 0) && (!ax || a.m % 8 == 0) &&
                      (!aw || a.n % 8 == 0);
    const LinearPlan p = linear_plan(a.m, a.n, a.k, type, ring);
    a.part = p.parts > 1 ? part : nullptr;
    with_type(type, "linear", [&](auto t) {
        linear_product<decltype(t)>(a, p, ax, aw, direct, s);
    });
}

// Bytes for the parts of a product, whichever tiles its operands allow.
size_t parts_bytes(int64_t m, int64_t n, int64_t k, int type) {
    if (m <= 0 || n <= 0) return 0;
    return std::max(linear_plan(m, n, k, type, false).bytes(m, n),
                    linear_plan(m, n, k, type, true).bytes(m, n));
}

constexpr int64_t kActRows = 256;

struct BackwardPlace {
    void* d;
    float* columns;
    float* part;
    size_t bytes;
};

BackwardPlace backward_place(int64_t m, int64_t k, int64_t n, int type, void* ws, size_t size) {
    Carver c(ws, size);
    BackwardPlace p{};
    p.d = c.take<char>(static_cast<size_t>(m) * n * type_size(type));
    p.columns = c.take<float>(static_cast<size_t>(ceil_div(m, kActRows)) * n);
    // dx's parts, then dw's, in the same place
    const size_t part = std::max(parts_bytes(m, k, n, type),
                                 std::max(parts_bytes(k, n, m, type), parts_bytes(n, k, m, type)));
    p.part = reinterpret_cast<float*>(c.take<char>(part));
    p.bytes = c.bytes();
    return p;
}

void check_linear(const std::string& w, int64_t m, int64_t k, int64_t n, int type, int act) {
    require(m >= 0 && k >= 0 && n >= 0, w + ": negative dimension");
    const int64_t most = (int64_t(1) << 31) - 4096;
    require(m < most && k < most && n < most, w + ": m, k and n must be < 2^31 - 4096");
    require(type >= TG_TYPE_F32 && type <= TG_TYPE_F16, w + ": unknown element type " +
                                                            std::to_string(type));
    require(act >= TG_EPI_NONE && act <= TG_EPI_SILU, w + ": unknown epilogue " +
                                                          std::to_string(act));
}

}  // namespace
}  // namespace tg

using tg::guard;
using tg::require;

extern "C" {

size_t tg_linear_workspace_size(int64_t m, int64_t k, int64_t n, int type) {
    if (m <= 0 || k < 0 || n <= 0 || type < TG_TYPE_F32 || type > TG_TYPE_F16) return 0;
    return tg::parts_bytes(m, n, k, type);
}

int tg_linear(int64_t m, int64_t k, int64_t n, int type, const void* x, int64_t ldx, const void* w,
              int64_t ldw, int transposed, const void* bias, int act, const void* residual,
              int64_t ldr, void* y, int64_t ldy, void* pre, int64_t ldp, void* workspace,
              size_t workspace_bytes, tg_stream_t stream) {
    return guard([&] {
        const std::string what = "linear";
        tg::check_linear(what, m, k, n, type, act);
        if (m == 0 || n == 0) return;
        require(y && (k == 0 || (x && w)), what + ": null pointer");
        require(ldx >= k && ldw >= (transposed ? k : n) && ldy >= n && (!residual || ldr >= n) &&
                    (!pre || ldp >= n),
                what + ": leading dimension below the columns");
        tg::LinearArgs a{};
        a.m = static_cast<int>(m);
        a.n = static_cast<int>(n);
        a.k = static_cast<int>(k);
        a.x = x;
        a.ldx = ldx;
        a.w = w;
        a.ldw = ldw;
        a.bias = bias;
        a.act = act;
        a.residual = residual;
        a.ldr = ldr;
        a.y = y;
        a.ldy = ldy;
        a.pre = pre;
        a.ldp = ldp;
        hipStream_t s = static_cast<hipStream_t>(stream);
        const size_t need = tg::parts_bytes(m, n, k, type);
        tg::TempBuffer temp;
        if (need && !workspace) {
            temp.allocate(need, s);
            workspace = temp.get();
            workspace_bytes = need;
        }
        tg::Carver c(workspace, workspace_bytes);
        float* part = reinterpret_cast<float*>(c.take<char>(need));
        tg::product(a, type, false, !transposed, part, s);
    });
}

size_t tg_linear_backward_workspace_size(int64_t m, int64_t k, int64_t n, int type) {
    if (m <= 0 || k < 0 || n <= 0 || type < TG_TYPE_F32 || type > TG_TYPE_F16) return 0;
    return tg::backward_place(m, k, n, type, nullptr, 0).bytes;
}

int tg_linear_backward(int64_t m, int64_t k, int64_t n, int type, const void* dy, int64_t lddy,
                       const void* x, int64_t ldx, const void* w, int64_t ldw, int transposed,
                       const void* pre, int64_t ldp, int act, void* dx, int64_t lddx, void* dw,
                       void* dbias, void* workspace, size_t workspace_bytes, tg_stream_t stream) {
    return guard([&] {
        const std::string what = "linear_backward";
        tg::check_linear(what, m, k, n, type, act);
        const bool slopes = act != TG_EPI_NONE;
        const bool given = m > 0 && n > 0;
        if (m == 0 || k == 0) dx = nullptr;
        if (n == 0 || k == 0) dw = nullptr;
        if (n == 0) dbias = nullptr;
        if (!dx && !dw && !dbias) return;
        require(!given || (dy && (!slopes || pre) && (!dw || x) && (!dx || w)),
                what + ": null pointer");
        require((!given || (lddy >= n && (!slopes || ldp >= n) && (!dw || ldx >= k) &&
                            (!dx || ldw >= (transposed ? k : n)))) &&
                    (!dx || lddx >= k),
                what + ": leading dimension below the columns");
        hipStream_t s = static_cast<hipStream_t>(stream);
        tg::BackwardPlace at{};
        tg::TempBuffer temp;
        if (given) {
            const size_t need = tg::backward_place(m, k, n, type, nullptr, 0).bytes;
            if (!workspace) {
                temp.allocate(need, s);
                workspace = temp.get();
                workspace_bytes = need;
            }
            at = tg::backward_place(m, k, n, type, workspace, workspace_bytes);
        }
        tg::with_type(type, "linear_backward", [&](auto t) {
            using T = decltype(t);
            tg::ActArgs a{};
            a.m = m;
            a.n = n;
            a.rows = tg::kActRows;
            a.dy = dy;
            a.lddy = lddy;
            a.pre = pre;
            a.ldp = ldp;
            a.d = dx || dw ? at.d : nullptr;
            a.ldd = n;
            a.part = dbias ? at.columns : nullptr;
            const int64_t parts = given ? tg::ceil_div(m, tg::kActRows) : 0;
            if (given && (slopes || dbias)) tg::linear_act<T>(a, act, s);
            if (dbias) tg::linear_columns<T>(at.columns, n, parts, dbias, s);
        });
        const void* d = slopes ? at.d : dy;
        const int64_t ldd = slopes ? n : lddy;
        tg::LinearArgs g{};
        if (dx) {
            g.m = static_cast<int>(m);
            g.n = static_cast<int>(k);
            g.k = static_cast<int>(n);
            g.x = d;
            g.ldx = ldd;
            g.w = w;
            g.ldw = ldw;
            g.y = dx;
            g.ldy = lddx;
            tg::product(g, type, false, transposed != 0, at.part, s);
        }
        if (dw) {
            g = tg::LinearArgs{};
            g.m = static_cast<int>(transposed ? n : k);
            g.n = static_cast<int>(transposed ? k : n);
            g.k = static_cast<int>(m);
            g.x = transposed ? d : x;
            g.ldx = transposed ? ldd : ldx;
            g.w = transposed ? x : d;
            g.ldw = transposed ? ldx : ldd;
            g.y = dw;
            g.ldy = g.n;
            tg::product(g, type, true, true, at.part, s);
        }
    });
}

}  // extern "C"
