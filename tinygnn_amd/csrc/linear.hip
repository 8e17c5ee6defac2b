// linear.hip -- dense layers: y = residual + act(x w + bias), and the gradients:
// shapes, parts and entry points (linear_kernels.hpp has the kernels).
#include "linear.hpp"

#include <string>

#include "device_utils.hpp"
#include "tiles.hpp"

namespace tg {
namespace {

// The longest contraction of one part.  Floats: 64 chains of kSumTiles tiles.  16-bit
// operands, whose sums are one chain that the instructions add eight products at a
// time to: n values of one sign are off by n 2^-27 of their sum at most, here
// half the result's own rounding (2^-11, 2^-8).  (In one chain, fp16 4,096 x 4,096 of
// constant columns, contraction 262,144, was 9.8e-4 off; one rounding is 4.9e-4.  In
// eight parts the product takes 7.51 ms, in one 7.50.)
int64_t long_chain(int type) {
    return type == TG_TYPE_F32 ? 16384 : type == TG_TYPE_F16 ? 32768 : 262144;
}

// Bytes of the parts' sums that a product keeps at a time, where it can: two of
// them, one of which is the sum of those before, at the least.
constexpr int64_t kKeptBytes = int64_t(1) << 30;

// The time of a product in us by tile, as measured: a tile of `m` x `n` results
// alone on a CU takes `alone` for each value of the contraction, one of many `busy`
// of the CU's time, and `fixed` beside that (lookup, first loads, results).
struct TileCost {
    int64_t m, n;
    double alone, busy, fixed;
};
constexpr TileCost kTiles16[] = {
    {32, 128, 0.0082, 0.0035, 0.6},  {64, 64, 0.0078, 0.0031, 0.6},
    {64, 128, 0.0105, 0.0051, 1.4},  {128, 64, 0.0105, 0.0051, 1.4},
    {128, 128, 0.0126, 0.0084, 2.5}, {256, 256, 0.0183, 0.0268, 8.0},
};
constexpr TileCost kTiles32[] = {
    {32, 128, 0.0290, 0.0170, 0.7},
    {64, 64, 0.0262, 0.0172, 0.7},
    {64, 128, 0.0420, 0.0325, 1.3},
    {128, 64, 0.0420, 0.0325, 1.3},
};

// How both operands come: through registers, straight to LDS, or to the ring of the
// large tile.
enum Loads { kRegisters, kDirect, kRing };

struct LinearPlans {
    LinearPlan of[3];  // by Loads
};

int64_t kept_parts(int64_t m, int64_t n, int64_t parts) {
    const int64_t fit = m > 0 && n > 0 ? kKeptBytes / 4 / m / n : parts;
    return std::min(parts, std::max<int64_t>(2, fit));
}

// How an out [m x n] with contraction k is cut: the tile and the parts of the
// contraction that the costs above and the parts' join (2.5 us, its bytes at 9 TB/s,
// past 200 MB at 5.3) make cheapest.  What it takes is within 10% of the best of 30
// measured tiles and parts for 19 of 22 products, and within 17% for the others:
// bf16 4,000 x 2,048, contraction 8,192: 256 x 256 in 2 parts 125 us (128 x 128 in
// one 134); 512 x 4,096 x 4,096: 64 x 128 in 2 parts 35 (128 x 128 in 4 32); 2,048^3:
// 64 x 128 29 (128 x 128 32, 256 x 256 51); fp32 232,965 x 256 x 256: 64 x 128 281
// (64 x 64 311, 128 x 128, which leaves one wavefront a SIMD, 362).
// Operands that come through registers (kRegisters) take 64 x 64 or, of 16 bits,
// 128 x 128.
LinearPlans linear_plans(int64_t m, int64_t n, int64_t k, int type) {
    const int64_t z = type_size(type), depth = kRowBytes / z;
    LinearPlans best{};
    double least[3] = {1e300, 1e300, 1e300};
    auto consider = [&](const TileCost& t) {
        const int64_t mt = ceil_div(m, t.m), nt = ceil_div(n, t.n), tiles = mt * nt;
        const bool square = t.m == t.n, large = t.m == 256;
        for (int64_t parts = 1; parts <= 256; parts *= 2) {
            if (parts > 1 && (k < 2 * depth * parts || tiles * parts > 2048)) break;
            int64_t unit = ceil_div(ceil_div(k, parts), depth) * depth;
            unit = std::max(std::min(unit, long_chain(type)), depth);
            const int64_t real = std::max<int64_t>(1, ceil_div(k, unit)), groups = tiles * real;
            const double load = groups < 256 ? static_cast<double>(groups) * (1.0 / 256)
                                             : static_cast<double>((groups + 255) / 256);
            const double u = static_cast<double>(unit);
            double us = std::max(t.alone * u + t.fixed, load * (t.busy * u + t.fixed));
            if (real > 1) {
                const double bytes = 8.0 * static_cast<double>(real) * static_cast<double>(m) *
                                     static_cast<double>(n);
                us += 2.5 + bytes * (bytes < 2e8 ? 1 / 9e6 : 1 / 5.3e6);
            }
            for (const Loads l : {kRegisters, kDirect, kRing}) {
                if ((l == kRegisters && !square) || (l != kRing && large) || us >= least[l])
                    continue;
                least[l] = us;
                best.of[l] = {t.m, t.n, mt, nt, unit, real, kept_parts(m, n, real)};
            }
        }
    };
    if (type == TG_TYPE_F32)
        for (const TileCost& t : kTiles32) consider(t);
    else
        for (const TileCost& t : kTiles16) consider(t);
    return best;
}

// Few rows of x with w's rows along the contraction (few_kernel): one launch, no
// parts.  Measured against the tiles with theirs, each after itself (bf16, 1 row: 4,096 x 4,096 7.2 us
// against 8.5, 512 x 8,192 4.2 against 6.0, 2,048 x 128 4.5 against 5.6; but 8,192 x
// 1,024 11.5 against 7.1, 4,096 x 64 6.6 against 5.3, 1,024 x 32,000 17.3 against 14.8;
// 32 rows of 4,096 x 4,096 14.6 against 13.2; fp32, 16 rows of 2,048 x 128 10.9 against
// 8.0).
bool few_rows(const LinearArgs& a, int64_t z, bool ax, bool aw) {
    return !ax && !aw && a.m <= 16 && a.k <= 4096 && a.n <= 16384 &&
           (a.n >= 1024 || (a.k <= 2048 && a.m * z <= 32));
}

// Whether an operand's tiles of up to 256 of its rows or columns can come by
// loads to LDS: from dword-aligned rows, within 2 GB of the tile's start; across
// the contraction, in whole dwords.
bool direct_side(const void* p, int64_t ld, int64_t cols, int64_t z, bool across) {
    return reinterpret_cast<uintptr_t>(p) % 4 == 0 && ld * z % 4 == 0 &&
           (!across || cols * z % 4 == 0) && (256 * ld + cols) * z < kDirectBytes;
}

// One product with the operands' layouts; `room` bytes at `part` for its parts.
void product(LinearArgs& a, int type, bool ax, bool aw, void* part, size_t room, hipStream_t s) {
    const int64_t z = type_size(type);
    const bool direct = direct_side(a.x, a.ldx, ax ? a.m : a.k, z, ax) &&
                        direct_side(a.w, a.ldw, aw ? a.n : a.k, z, aw);
    const bool ring = direct && z == 2 && ((ax && aw) || a.k % 8 == 0) && (!ax || a.m % 8 == 0) &&
                      (!aw || a.n % 8 == 0);
    LinearPlan p{};
    if (!few_rows(a, z, ax, aw)) {
        p = linear_plans(a.m, a.n, a.k, type).of[ring ? kRing : direct ? kDirect : kRegisters];
        if (p.parts > 1) {
            Carver c(part, room);
            a.part = reinterpret_cast<float*>(c.take<char>(p.bytes(a.m, a.n)));
        }
    }
    with_type(type, "linear", [&](auto t) {
        linear_product<decltype(t)>(a, p, ax, aw, direct, s);
    });
}

// Bytes for the parts of a product, whichever tiles its operands allow.
size_t parts_bytes(int64_t m, int64_t n, int64_t k, int type) {
    if (m <= 0 || n <= 0) return 0;
    const LinearPlans plans = linear_plans(m, n, k, type);
    size_t most = 0;
    for (const LinearPlan& p : plans.of) most = std::max(most, p.bytes(m, n));
    return most;
}

// Chunks of columns of a workgroup of act_backward_kernel, as a power of two, and
// its rows: for about 1,024 workgroups.
int act_log_wide(int64_t n, int type) {
    const int64_t chunks = ceil_div(n, 16 / type_size(type));
    int log = 0;
    while (log < 5 && (int64_t(1) << log) < chunks) ++log;
    return log;
}

int64_t act_rows(int64_t m, int64_t n, int type) {
    const int64_t chunks = std::max<int64_t>(1, ceil_div(n, 16 / type_size(type)));
    const int log = act_log_wide(n, type);
    const int64_t cols = ceil_div(chunks, int64_t(1) << log), high = 256 >> log;
    const int64_t parts = std::max<int64_t>(1, 1024 / cols);
    return std::max(high, ceil_div(ceil_div(m, parts), high) * high);
}

struct BackwardPlace {
    void* d;
    float* columns;
    void* part;  // dx's parts, then dw's: what is left of the workspace
    size_t room;
    size_t bytes;  // without the parts
};

BackwardPlace backward_place(int64_t m, int64_t n, int type, int act, bool dbias, void* ws,
                             size_t size) {
    Carver c(ws, size);
    BackwardPlace p{};
    if (act != TG_EPI_NONE) p.d = c.take<char>(static_cast<size_t>(m) * n * type_size(type));
    if (dbias) p.columns = c.take<float>(static_cast<size_t>(ceil_div(m, act_rows(m, n, type))) * n);
    p.bytes = c.bytes();
    p.part = ws ? static_cast<char*>(ws) + p.bytes : nullptr;
    p.room = size > p.bytes ? size - p.bytes : 0;
    return p;
}

size_t backward_bytes(int64_t m, int64_t k, int64_t n, int type, int act, bool dbias) {
    return backward_place(m, n, type, act, dbias, nullptr, 0).bytes +
           std::max(parts_bytes(m, k, n, type),
                    std::max(parts_bytes(k, n, m, type), parts_bytes(n, k, m, type)));
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
        tg::TempBuffer temp;
        if (!workspace) {
            workspace_bytes = tg::parts_bytes(m, n, k, type);
            if (workspace_bytes) {
                temp.allocate(workspace_bytes, s);
                workspace = temp.get();
            }
        }
        tg::product(a, type, false, !transposed, workspace, workspace_bytes, s);
    });
}

size_t tg_linear_backward_workspace_size(int64_t m, int64_t k, int64_t n, int type) {
    return tg_linear_backward_call_workspace_size(m, k, n, type, TG_EPI_SILU, 1);
}

size_t tg_linear_backward_call_workspace_size(int64_t m, int64_t k, int64_t n, int type, int act,
                                              int dbias) {
    if (m <= 0 || k < 0 || n <= 0 || type < TG_TYPE_F32 || type > TG_TYPE_F16) return 0;
    if (act < TG_EPI_NONE || act > TG_EPI_SILU) return 0;
    return tg::backward_bytes(m, k, n, type, act, dbias != 0);
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
            if (!workspace) {
                workspace_bytes = tg::backward_bytes(m, k, n, type, act, dbias != nullptr);
                if (workspace_bytes) {
                    temp.allocate(workspace_bytes, s);
                    workspace = temp.get();
                }
            }
            at = tg::backward_place(m, n, type, act, dbias != nullptr, workspace, workspace_bytes);
        }
        tg::with_type(type, "linear_backward", [&](auto t) {
            using T = decltype(t);
            tg::ActArgs a{};
            a.m = m;
            a.n = n;
            a.rows = tg::act_rows(m, n, type);
            a.log_wide = tg::act_log_wide(n, type);
            a.dy = dy;
            a.lddy = lddy;
            a.pre = pre;
            a.ldp = ldp;
            a.d = dx || dw ? at.d : nullptr;
            a.ldd = n;
            a.part = dbias ? at.columns : nullptr;
            const int64_t parts = given ? tg::ceil_div(m, a.rows) : 0;
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
            tg::product(g, type, false, transposed != 0, at.part, at.room, s);
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
            tg::product(g, type, true, true, at.part, at.room, s);
        }
    });
}

}  // extern "C"
