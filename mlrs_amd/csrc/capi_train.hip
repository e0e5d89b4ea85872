// C-ABI layer of the training operators: validation (before any launch),
// packing of operands that the kernels cannot read in place, and dispatch.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "../../include/mlrs_hip_knn.h"
#include "capi_shared.hpp"
#include "train_kernels.hpp"

using namespace mlrs;
using namespace mlrs::train;

namespace {

constexpr int64_t kMaxCount = 0x7FFFFFFF - 512;  // a tile past it must not overflow
constexpr int64_t kMaxRowBytes = (int64_t)1 << 22;  // 256 rows of a tile within a buffer descriptor's 2^31

constexpr int64_t kStatsBytes = (int64_t)256 << 20;  // of a loss's partial statistics

int32_t null_error(const char* operand) {
    return capi::error(MLRS_ERR_NULL_POINTER, operand, 0, 0, 0, "null pointer");
}

// Carves a call's scratch: first a pass that only adds up, then one that hands
// out addresses.
struct Scratch {
    char* base = nullptr;
    size_t used = 0;
    template <typename T>
    T* take(size_t n) {
        used = (used + 255) & ~(size_t)255;
        T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
        used += n * sizeof(T);
        return p;
    }
};

template <typename T>
int64_t padded(int64_t cols) {
    constexpr int64_t E = 16 / (int64_t)sizeof(T);
    return (cols + E - 1) / E * E;
}

template <typename T>
bool readable(const T* p, int64_t cols) {
    return (uintptr_t)p % 16 == 0 && padded<T>(cols) == cols;
}

// Where the rows of a packed matrix lie: a cache line apart or a multiple of it,
// from a few lines on.
template <typename T>
int64_t spaced(int64_t cols) {
    constexpr int64_t L = 128 / (int64_t)sizeof(T);
    return cols < 4 * L ? padded<T>(cols) : (cols + L - 1) / L * L;
}

// An operand as the kernels read it: in place (f32 of any rows, word by word), or
// packed.
template <typename T>
struct Op {
    const T* src;
    int64_t rows, cols;
    bool words;
    T* packed = nullptr;
    Op(const T* p, int64_t r, int64_t c, bool by_words) : src(p), rows(r), cols(c), words(by_words) {}
    bool in_place() const { return words || readable(src, cols); }
    void plan(Scratch& sc) {
        if (!in_place()) packed = sc.take<T>((size_t)(rows * spaced<T>(cols)));
    }
    PackJob job() const { return PackJob{src, packed, in_place() ? 0 : rows, cols, spaced<T>(cols)}; }
    Mat mat() const { return in_place() ? Mat{src, cols} : Mat{packed, spaced<T>(cols)}; }
};

// f32 operands whose rows are no multiple of 16 bytes: whether their products (`us`
// by words, `packed_us` else) copy them word by word, which makes a product about
// 6% slower (3001 x 10007 by 250 backwards: 372 us, 358 packed), or `elements` of
// them are packed: a launch, and their bytes twice (300 x 7001 by 501 forwards: 36
// us by words, 49 packed).
bool by_words(double us, double packed_us, double elements) {
    return 1.06 * us < packed_us + 4.5 + elements * 8.0 / 4.5e6;
}

// f32 products may run on the bf16 matrix cores, in three parts of each operand
// (train_split.hpp).  What packing `elements` of them costs, in microseconds: 10
// bytes each at 5.5 TB/s, its launch, and the launches of the
// f32 kernels that take over where an element is not finite.
double split_us(double elements) { return elements * 10.0 / 5.5e6 + 9.0; }

// A mark that no earlier call has left behind, and that what else lies in the
// workspace (indices, counts) does not look like; were it there all the same, the
// f32 kernels would compute the call.
uint32_t next_mark() {
    static uint32_t mark = 0;  // under the call lock
    mark += 0x9E3779B1u;
    return mark;
}

// The split kernels of a call and the f32 ones that stand in for them.
struct Sides {
    uint32_t* flag = nullptr;
    uint32_t mark = 0;
    Only split() const { return Only{flag, mark, false}; }
    Only plain() const { return Only{flag, mark, true}; }
};

constexpr Cut kPlainCut{0, 1, 0, 0.0};  // of the kernels that stand in
constexpr PairCut kPlainPair{kPlainCut, kPlainCut, true, 0.0};

// Sizes that both layers of operators share: a (n x d) and w (m x d).
template <typename T>
int32_t check_sizes(const char* a_name, int64_t a_len, int64_t n, int64_t d, int64_t w_len, int64_t m) {
    if (!capi::geometry(n, d, a_len)) return capi::shape_error(a_name, n, d, a_len);
    if (!capi::geometry(m, d, w_len)) return capi::shape_error("w", m, d, w_len);
    if (d < 1 || m < 1) return capi::shape_error("features", m, d, 0);
    if (d > kMaxRowBytes / (int64_t)sizeof(T) || m > kMaxCount)
        return capi::error(MLRS_ERR_UNSUPPORTED, "features", m, d, 0, "rows are limited to 2^22 bytes");
    if (n > kMaxCount) return capi::error(MLRS_ERR_UNSUPPORTED, "rows", n, d, 0, "row counts are limited to 2^31 - 513");
    return MLRS_OK;
}

// A product's grid must fit, in the largest tiles.
bool grid_fits(int64_t m, int64_t n) { return launchable(((m + 255) / 256) * ((n + 255) / 256), 512); }
int32_t grid_error(int64_t m, int64_t n) {
    return capi::error(MLRS_ERR_UNSUPPORTED, "rows", n, m, 0, "the product has more tiles than a launch");
}

// What a call writes may be no part of what it reads or else writes: workgroups
// read operands while others write results.
struct Span {
    const void* p;
    int64_t bytes;
    template <typename T>
    Span(const T* t, int64_t len) : p(t), bytes(t ? len * (int64_t)sizeof(T) : 0) {}
    bool meets(const Span& o) const {
        const uintptr_t a = (uintptr_t)p, b = (uintptr_t)o.p;
        return bytes > 0 && o.bytes > 0 && a < b + (uintptr_t)o.bytes && b < a + (uintptr_t)bytes;
    }
    bool meets(std::initializer_list<Span> others) const {
        for (const Span& o : others)
            if (meets(o)) return true;
        return false;
    }
};
int32_t overlap_error(const char* out) {
    return capi::error(MLRS_ERR_INVALID_PARAM, out, 0, 0, 0, "an output overlaps another operand");
}

#define MLRS_TRY(call)                                      \
    do {                                                    \
        const hipError_t e_ = (call);                       \
        if (e_ != hipSuccess) return capi::hip_error(e_, where); \
    } while (0)

// ---------------------------------------------------------------------------
template <typename T>
int32_t linear_impl(const T* x, int64_t x_len, int64_t n, int64_t k, const T* w, int64_t w_len, int64_t m,
                    const T* bias, int64_t bias_len, const T* residual, int64_t residual_len, int32_t act, T* y,
                    int64_t y_len, T* z, int64_t z_len, void* stream) {
    const char* where = "linear";
    return capi::call([&]() -> int32_t {
        int32_t rc = check_sizes<T>("x", x_len, n, k, w_len, m);
        if (rc) return rc;
        if (bias ? bias_len != m : bias_len != 0) return capi::shape_error("bias", 1, m, bias_len);
        if (residual ? !capi::geometry(n, m, residual_len) : residual_len != 0)
            return capi::shape_error("residual", n, m, residual_len);
        if (!capi::geometry(n, m, y_len)) return capi::shape_error("out", n, m, y_len);
        if (z ? !capi::geometry(n, m, z_len) : z_len != 0) return capi::shape_error("preact", n, m, z_len);
        if (act < MLRS_ACT_NONE || act > MLRS_ACT_SILU)
            return capi::error(MLRS_ERR_UNSUPPORTED, "activation", act, 0, 0, "unknown activation");
        if (n == 0) return MLRS_OK;
        if (!x || !w || !y) return null_error(!x ? "x" : !w ? "w" : "out");
        if (!grid_fits(m, n)) return grid_error(m, n);
        const Span sx(x, x_len), sw(w, w_len), sb(bias, bias_len), sr(residual, residual_len), sy(y, y_len);
        if (sy.meets({sx, sw, sb}) || (y != residual && sy.meets(sr))) return overlap_error("out");
        if (Span(z, z_len).meets({sx, sw, sb, sr, sy})) return overlap_error("preact");
        const hipStream_t s = (hipStream_t)stream;
        const LinearOut o{bias, residual, y, z, act};
        int cus = 0;
        rc = capi::cu_count(&cus);
        if (rc) return rc;
        Cut cut = choose_cut((int)sizeof(T), m, n, k, cus);
        if (few_rows((int)sizeof(T), n, m, k, cut)) {
            capi::Timed timed(s, "linear_few");
            MLRS_TRY(launch_linear_few<T>(x, w, n, m, k, o, s));
            return MLRS_OK;
        }
        bool split = false, words = false;
        if constexpr (std::is_same<T, float>::value) {
            const Cut other = choose_cut_split(m, n, k, cus);
            split = split_launchable(m, n) && other.us + split_us((double)(n + m) * (double)k) < cut.us;
            if (split) cut = other;
            const bool rx = readable(x, k), rw = readable(w, k);
            const Cut by = choose_cut((int)sizeof(T), m, n, k, cus, 64, true);
            words = !split && !(rx && rw) && by_words(by.us, cut.us, (double)((rx ? 0 : n) + (rw ? 0 : m)) * (double)k);
            if (words) cut = by;
        }
        Op<T> xo(x, n, k, words), wo(w, m, k, words);
        float* part = nullptr;
        char *xs = nullptr, *ws = nullptr;
        Sides sides;
        Scratch sc;
        for (int pass = 0; pass < 2; ++pass) {
            xo.plan(sc);
            wo.plan(sc);
            part = sc.take<float>(cut.part_bytes(m, n) / 4);
            if (split) {
                xs = sc.take<char>(split_bytes(n, k));
                ws = sc.take<char>(split_bytes(m, k));
                sides.flag = sc.take<uint32_t>(1);
            }
            if (sc.used == 0) break;
            if (pass == 0) {
                rc = capi::scratch(sc.used, s, &sc.base, &cus);
                if (rc) return rc;
                sc.used = 0;
            }
        }
        if constexpr (std::is_same<T, float>::value) {
            if (split) {
                sides.mark = next_mark();
                MLRS_TRY(launch_pack_split(split_job(x, k, n, k, xs, false), split_job(w, k, m, k, ws, false),
                                           sides.flag, sides.mark, s));
                capi::Timed timed(s, "linear");
                MLRS_TRY(launch_linear_split(split_mat(xs, k, false), split_mat(ws, k, false), n, m, k, o, cut, part,
                                             sides.split(), s));
                MLRS_TRY(launch_pack<T>(xo.job(), wo.job(), sides.plain(), s));
                MLRS_TRY(launch_linear<T>(xo.mat(), wo.mat(), n, m, k, o, kPlainCut, nullptr, sides.plain(), s));
                return MLRS_OK;
            }
        }
        MLRS_TRY(launch_pack<T>(xo.job(), wo.job(), Only{}, s));
        capi::Timed timed(s, "linear");
        MLRS_TRY(launch_linear<T>(xo.mat(), wo.mat(), n, m, k, o, cut, part, Only{}, s));
        return MLRS_OK;
    });
}

template <typename T>
int32_t linear_grad_impl(const T* dy, int64_t dy_len, const T* x, int64_t x_len, int64_t n, int64_t k, const T* w,
                         int64_t w_len, int64_t m, const T* z, int64_t z_len, int32_t act, T* dx, int64_t dx_len,
                         T* dw, int64_t dw_len, T* db, int64_t db_len, void* stream) {
    const char* where = "linear_grad";
    return capi::call([&]() -> int32_t {
        int32_t rc = check_sizes<T>("x", x_len, n, k, w_len, m);
        if (rc) return rc;
        if (m > kMaxRowBytes / (int64_t)sizeof(T))
            return capi::error(MLRS_ERR_UNSUPPORTED, "features", m, k, 0, "rows are limited to 2^22 bytes");
        if (!capi::geometry(n, m, dy_len)) return capi::shape_error("dy", n, m, dy_len);
        if (dx ? !capi::geometry(n, k, dx_len) : dx_len != 0) return capi::shape_error("dx", n, k, dx_len);
        if (dw ? !capi::geometry(m, k, dw_len) : dw_len != 0) return capi::shape_error("dw", m, k, dw_len);
        if (db ? db_len != m : db_len != 0) return capi::shape_error("dbias", 1, m, db_len);
        if (act < MLRS_ACT_NONE || act > MLRS_ACT_SILU)
            return capi::error(MLRS_ERR_UNSUPPORTED, "activation", act, 0, 0, "unknown activation");
        if (act == MLRS_ACT_NONE ? z_len != 0 : !capi::geometry(n, m, z_len))
            return capi::shape_error("preact", n, m, z_len);
        if (!dx && !dw && !db) return MLRS_OK;
        if (n > 0) {
            if (!dy) return null_error("dy");
            if (dw && !x) return null_error("x");
            if (act != MLRS_ACT_NONE && !z) return null_error("preact");
        }
        if (dx && !w) return null_error("w");
        if (!grid_fits(k, n) || !grid_fits(k, m)) return grid_error(k, std::max(m, n));
        const Span ody(dy, dy_len), ox(x, x_len), ow(w, w_len), oz(z, z_len), odx(dx, dx_len), odw(dw, dw_len);
        if (odx.meets({ody, ox, ow, oz})) return overlap_error("dx");
        if (odw.meets({ody, ox, ow, oz, odx})) return overlap_error("dw");
        if (Span(db, db_len).meets({ody, ox, ow, oz, odx, odw})) return overlap_error("dbias");
        const hipStream_t s = (hipStream_t)stream;
        int cus = 0;
        rc = capi::cu_count(&cus);
        if (rc) return rc;
        const bool products = (dx && n > 0) || dw;
        // dy itself serves as dz where there is no slope and its rows can be read
        const bool make_dz = products && n > 0 && (act != MLRS_ACT_NONE || !readable(dy, m));
        bool words = false;
        const bool want_x = dx && n > 0;
        PairCut cut = choose_pair((int)sizeof(T), k, n, m, k, m, n, cus);
        Cut sx{}, sw{};  // of those that run in parts
        bool split_x = false, split_w = false;
        if constexpr (std::is_same<T, float>::value) {
            const Cut cx = choose_cut((int)sizeof(T), k, n, m, cus), cw = choose_cut((int)sizeof(T), k, m, n, cus);
            sx = choose_cut_split(k, n, m, cus);
            sw = choose_cut_split(k, m, n, cus);
            split_x = want_x && split_launchable(k, n) && sx.us + split_us((double)(n + k) * (double)m) < cx.us;
            split_w = dw && n > 0 && split_launchable(k, m) && sw.us + split_us((double)(m + k) * (double)n) < cw.us;
            if (split_x || split_w) cut = PairCut{cx, cw, false, 0.0};
            const bool rw = !want_x || readable(w, k), rx = !dw || readable(x, k);
            const PairCut by = choose_pair((int)sizeof(T), k, n, m, k, m, n, cus, true);
            words = !split_x && !split_w && !(rx && rw) &&
                    by_words(by.us, cut.us, (double)((rx ? 0 : n) + (rw ? 0 : m)) * (double)k);
            if (words) cut = by;
        }
        if (!want_x || !dw)
            cut = PairCut{choose_cut((int)sizeof(T), k, n, m, cus, 64, words),
                          choose_cut((int)sizeof(T), k, m, n, cus, 64, words), false, 0.0};
        const int parts = column_parts(n, m, cus);
        char *w_r = nullptr, *dz_k = nullptr, *x_r = nullptr, *dz_r = nullptr;
        Sides sides;
        Op<T> xo(x, n, k, words), wo(w, m, k, words);
        T* dz = nullptr;
        float *part = nullptr, *sums = nullptr;
        Scratch sc;
        for (int pass = 0; pass < 2; ++pass) {
            if (dw) xo.plan(sc);
            if (dx) wo.plan(sc);
            if (make_dz) dz = sc.take<T>((size_t)(n * spaced<T>(m)));
            if (db) sums = sc.take<float>((size_t)parts * (size_t)m);
            part = sc.take<float>(std::max(cut.part_bytes(k, n, k, m),
                                           std::max(split_x ? sx.part_bytes(k, n) : 0, split_w ? sw.part_bytes(k, m) : 0)) / 4);
            if (split_x) {
                w_r = sc.take<char>(split_bytes(m, k));
                dz_k = sc.take<char>(split_bytes(n, m));
            }
            if (split_w) {
                x_r = sc.take<char>(split_bytes(n, k));
                dz_r = sc.take<char>(split_bytes(n, m));
            }
            if (split_x || split_w) sides.flag = sc.take<uint32_t>(1);
            if (sc.used == 0) break;
            if (pass == 0) {
                rc = capi::scratch(sc.used, s, &sc.base, &cus);
                if (rc) return rc;
                sc.used = 0;
            }
        }
        ColumnSums<T> col{db, sums, parts, nullptr};
        if (make_dz || db)
            MLRS_TRY(launch_act_grad<T>(dy, act == MLRS_ACT_NONE ? nullptr : z, act, n, m, dz, spaced<T>(m), col, s));
        if (parts == 1) col.out = nullptr;  // done
        const Mat dzm = make_dz ? Mat{dz, spaced<T>(m)} : Mat{dy, m};
        PackJob xj = xo.job(), wj = wo.job();
        if (!dw || split_w) xj.rows = 0;
        if (!dx || split_x) wj.rows = 0;
        MLRS_TRY(launch_pack<T>(xj, wj, Only{}, s));
        capi::Timed timed(s, "linear_grad");
        const StoreTo to_x{dx, k, nullptr, nullptr, 0, nullptr}, to_w{dw, k, nullptr, nullptr, 0, nullptr};
        Product px{wo.mat(), dzm, k, n, m, to_x}, pw{xo.mat(), dzm, k, m, n, to_w};
        if constexpr (std::is_same<T, float>::value) {
            if (split_x || split_w) {
                sides.mark = next_mark();
                const float* z32 = (const float*)dzm.p;
                if (split_x) {
                    MLRS_TRY(launch_pack_split(split_job(w, k, m, k, w_r, true),
                                               split_job(z32, dzm.ld, n, m, dz_k, false), sides.flag, sides.mark, s));
                    MLRS_TRY(launch_product_split(split_mat(w_r, k, true), split_mat(dz_k, m, false), true, k, n, m,
                                                  to_x, sx, part, sides.split(), s));
                }
                if (split_w) {
                    MLRS_TRY(launch_pack_split(split_job(x, k, n, k, x_r, true),
                                               split_job(z32, dzm.ld, n, m, dz_r, true), sides.flag, sides.mark, s));
                    MLRS_TRY(launch_product_split(split_mat(x_r, k, true), split_mat(dz_r, m, true), false, k, m, n,
                                                  to_w, sw, part, sides.split(), s));
                }
                // what dw's packing marked is marked for dx as well, whose
                // product the f32 kernel then computes again, to the same values
                PackJob xp = xo.job(), wp = wo.job();
                if (!split_w) xp.rows = 0;
                if (!split_x) wp.rows = 0;
                MLRS_TRY(launch_pack<T>(xp, wp, sides.plain(), s));
                MLRS_TRY(launch_products<T>(split_x ? px : Product{}, split_w ? pw : Product{}, kPlainPair, nullptr,
                                            ColumnSums<T>{}, 0, sides.plain(), s));
            }
        }
        if (!want_x || split_x) px.m = 0;
        if (!dw || split_w) pw.m = 0;
        if (px.m || pw.m)
            MLRS_TRY(launch_products<T>(px, pw, cut, part, col, m, Only{}, s));
        else
            MLRS_TRY(launch_sum_parts<T>(col, m, s));
        return MLRS_OK;
    });
}

// ---------------------------------------------------------------------------
template <typename T>
int32_t check_xent(int64_t h_len, int64_t n, int64_t d, int64_t w_len, int64_t v, const T* bias, int64_t bias_len,
                   int64_t target_len, int64_t out_len) {
    const int32_t rc = check_sizes<T>("h", h_len, n, d, w_len, v);
    if (rc) return rc;
    if (bias ? bias_len != v : bias_len != 0) return capi::shape_error("bias", 1, v, bias_len);
    if (target_len != n) return capi::shape_error("target", n, 1, target_len);
    if (out_len != n) return capi::shape_error("out", n, 1, out_len);
    return MLRS_OK;
}

template <typename T>
int32_t xent_impl(const T* h, int64_t h_len, int64_t n, int64_t d, const T* w, int64_t w_len, int64_t v,
                  const T* bias, int64_t bias_len, const int64_t* target, int64_t target_len, int64_t ignore,
                  float* loss, float* lse, int64_t out_len, void* stream) {
    const char* where = "softmax_xent";
    return capi::call([&]() -> int32_t {
        int32_t rc = check_xent<T>(h_len, n, d, w_len, v, bias, bias_len, target_len, out_len);
        if (rc) return rc;
        if (n == 0) return MLRS_OK;
        if (!h || !w || !target || !loss || !lse)
            return null_error(!h ? "h" : !w ? "w" : !target ? "target" : "out");
        const Span sh(h, h_len), sw(w, w_len), sb(bias, bias_len), st(target, target_len), sl(loss, out_len);
        if (sl.meets({sh, sw, sb, st}) || Span(lse, out_len).meets({sh, sw, sb, st, sl})) return overlap_error("out");
        const hipStream_t s = (hipStream_t)stream;
        int cus = 0;
        rc = capi::cu_count(&cus);
        if (rc) return rc;
        const Cut cut = choose_cut((int)sizeof(T), v, n, d, cus, 1);
        int tile = cut.tile;
        int64_t parts = stats_parts(tile, v), parts_s = 0;
        bool split = false, words = false;
        if constexpr (std::is_same<T, float>::value) {
            // (256 rows, or as many as leave a few tiles)
            split = split_launchable(v, std::min<int64_t>(n, 256)) &&
                    choose_cut_split(v, n, d, cus, 1).us + split_us((double)(n + v) * (double)d) < cut.us;
            if (split) {
                tile = kPlainCut.tile;
                parts = stats_parts(tile, v);
                parts_s = stats_parts_split(v);
            }
            const bool rh = readable(h, d), rw = readable(w, d);
            const Cut by = choose_cut((int)sizeof(T), v, n, d, cus, 1, true);
            words = !split && !(rh && rw) && by_words(by.us, cut.us, (double)((rh ? 0 : n) + (rw ? 0 : v)) * (double)d);
            if (words) {
                tile = by.tile;
                parts = stats_parts(tile, v);
            }
        }
        // few tiles and long rows: the logits in parts
        const Cut zc = choose_cut((int)sizeof(T), v, n, d, cus, 64, words);
        const bool in_parts = !split && zc.splits > 1;
        // the statistics of as many rows at a time as their parts have room for
        const int64_t room = std::max(parts, parts_s);
        const int64_t rows = std::min(n, std::max<int64_t>(256, kStatsBytes / (8 * room) / 256 * 256));
        Op<T> ho(h, n, d, words), wo(w, v, d, words);
        float *top = nullptr, *total = nullptr, *hit = nullptr, *z = nullptr;
        char *hs = nullptr, *ws = nullptr;
        Sides sides;
        Scratch sc;
        for (int pass = 0; pass < 2; ++pass) {
            ho.plan(sc);
            wo.plan(sc);
            if (in_parts) {
                z = sc.take<float>(zc.part_bytes(v, n) / 4);
            } else {
                top = sc.take<float>((size_t)(room * rows));
                total = sc.take<float>((size_t)(room * rows));
                hit = sc.take<float>((size_t)rows);
            }
            if (split) {
                hs = sc.take<char>(split_bytes(n, d));
                ws = sc.take<char>(split_bytes(v, d));
                sides.flag = sc.take<uint32_t>(1);
            }
            if (pass == 0) {
                rc = capi::scratch(sc.used, s, &sc.base, &cus);
                if (rc) return rc;
                sc.used = 0;
            }
        }
        if constexpr (std::is_same<T, float>::value) {
            if (split) {
                sides.mark = next_mark();
                MLRS_TRY(launch_pack_split(split_job(h, d, n, d, hs, false), split_job(w, d, v, d, ws, false),
                                           sides.flag, sides.mark, s));
            }
        }
        const Only plain = split ? sides.plain() : Only{};
        MLRS_TRY(launch_pack<T>(ho.job(), wo.job(), plain, s));
        const Mat hm = ho.mat();
        capi::Timed timed(s, "softmax_xent");
        if (in_parts) {
            MLRS_TRY(launch_logit_parts<T>(hm, wo.mat(), n, v, d, zc, z, s));
            MLRS_TRY(launch_xent_rows<T>(z, zc, bias, target, n, v, ignore, loss, lse, s));
            return MLRS_OK;
        }
        for (int64_t r0 = 0; r0 < n; r0 += rows) {
            const int64_t r = std::min(rows, n - r0);
            if constexpr (std::is_same<T, float>::value) {
                if (split) {
                    MLRS_TRY(launch_xent_stats_split(split_mat(hs + split_bytes(r0, d), d, false),
                                                     split_mat(ws, d, false), bias, target + r0, r, v, d, top, total,
                                                     hit, sides.split(), s));
                    MLRS_TRY(launch_xent_join(top, total, parts_s, hit, target + r0, r, v, ignore, loss + r0, lse + r0,
                                              sides.split(), s));
                }
            }
            MLRS_TRY(launch_xent_stats<T>(Mat{(const T*)hm.p + r0 * hm.ld, hm.ld}, wo.mat(), bias, target + r0, r, v,
                                          d, tile, top, total, hit, plain, s));
            MLRS_TRY(launch_xent_join(top, total, parts, hit, target + r0, r, v, ignore, loss + r0, lse + r0, plain,
                                      s));
        }
        return MLRS_OK;
    });
}

template <typename T>
int32_t xent_grad_impl(const T* h, int64_t h_len, int64_t n, int64_t d, const T* w, int64_t w_len, int64_t v,
                       const T* bias, int64_t bias_len, const int64_t* target, int64_t target_len, int64_t ignore,
                       const float* lse, const float* grad, int64_t out_len, T* dh, int64_t dh_len, T* dw,
                       int64_t dw_len, T* db, int64_t db_len, void* stream) {
    const char* where = "softmax_xent_grad";
    return capi::call([&]() -> int32_t {
        int32_t rc = check_xent<T>(h_len, n, d, w_len, v, bias, bias_len, target_len, out_len);
        if (rc) return rc;
        if (dh ? !capi::geometry(n, d, dh_len) : dh_len != 0) return capi::shape_error("dh", n, d, dh_len);
        if (dw ? !capi::geometry(v, d, dw_len) : dw_len != 0) return capi::shape_error("dw", v, d, dw_len);
        if (db ? db_len != v : db_len != 0) return capi::shape_error("dbias", 1, v, db_len);
        if (!dh && !dw && !db) return MLRS_OK;
        if (!w) return null_error("w");
        if (n > 0 && (!h || !target || !lse || !grad))
            return null_error(!h ? "h" : !target ? "target" : !lse ? "lse" : "grad");
        const Span oh(h, h_len), ow(w, w_len), ob(bias, bias_len), ot(target, target_len), ol(lse, out_len),
            og(grad, out_len), odh(dh, dh_len), odw(dw, dw_len);
        if (odh.meets({oh, ow, ob, ot, ol, og})) return overlap_error("dh");
        if (odw.meets({oh, ow, ob, ot, ol, og, odh})) return overlap_error("dw");
        if (Span(db, db_len).meets({oh, ow, ob, ot, ol, og, odh, odw})) return overlap_error("dbias");
        const hipStream_t s = (hipStream_t)stream;
        int cus = 0;
        rc = capi::cu_count(&cus);
        if (rc) return rc;
        if (n == 0) {
            // no rows: the products over them are empty sums
            if (dw) {
                const StoreTo o{dw, d, nullptr, nullptr, 0, nullptr};
                const Product p{Mat{w, padded<T>(d)}, Mat{w, padded<T>(v)}, d, v, 0, o};
                const Cut c{0, 1, 0, 0.0};
                MLRS_TRY(launch_products<T>(Product{}, p, PairCut{c, c, false, 0.0}, nullptr, ColumnSums<T>{}, 0, Only{}, s));
            }
            constexpr int64_t kMost = (int64_t)1 << 27;  // columns of a launch
            for (int64_t c = 0; db && c < v; c += kMost)
                MLRS_TRY(launch_sum_parts<T>(ColumnSums<T>{db + c, nullptr, 0, nullptr}, std::min(kMost, v - c), s));
            return MLRS_OK;
        }
        // classes of a piece: a multiple of 256, at least one tile, and a row of
        // them within the kernels' limit
        const int64_t fit = std::min<int64_t>(MLRS_XENT_PIECE_BYTES / ((int64_t)sizeof(T) * n),
                                              kMaxRowBytes / (int64_t)sizeof(T)) / 256 * 256;
        const int64_t pieces = (v + std::max<int64_t>(fit, 256) - 1) / std::max<int64_t>(fit, 256);
        const int64_t piece = pieces == 1 ? v : ((v + pieces - 1) / pieces + 255) / 256 * 256;
        const int64_t ld = spaced<T>(std::min(piece, v)), dh_ld = (d + 3) / 4 * 4;
        const bool scaled = sizeof(T) == 2 && std::is_same<T, _Float16>::value;
        const int64_t most = std::min(piece, v);  // classes of the largest piece
        PairCut cut = choose_pair((int)sizeof(T), d, n, most, d, most, n, cus);
        // f32: which of a piece's three products run in parts; the gradient of the
        // logits is packed for each of the two that take it
        Cut sh{}, sw{};
        bool split_z = false, split_h = false, split_w = false;
        if constexpr (std::is_same<T, float>::value) {
            const double nv = (double)n * (double)most, nd = (double)n * (double)d, vd = (double)most * (double)d;
            const Cut ch = choose_cut((int)sizeof(T), d, n, most, cus), cw = choose_cut((int)sizeof(T), d, most, n, cus);
            sh = choose_cut_split(d, n, most, cus);
            sw = choose_cut_split(d, most, n, cus);
            split_z = split_launchable(most, n) && choose_cut_split(most, n, d, cus, 1).us + split_us(nd + vd) <
                      choose_cut((int)sizeof(T), most, n, d, cus, 1).us;
            split_h = dh && split_launchable(d, n) && sh.us + split_us(nv + vd) < ch.us;
            split_w = dw && split_launchable(d, most) && sw.us + split_us(nv + nd) < cw.us;
            if (split_h || split_w) cut = PairCut{ch, cw, false, 0.0};
        }
        const bool split = split_z || split_h || split_w;
        bool words = false;
        if constexpr (std::is_same<T, float>::value) {
            const bool rh = readable(h, d), rw = readable(w, d);
            const PairCut by = choose_pair((int)sizeof(T), d, n, most, d, most, n, cus, true);
            const double z = choose_cut((int)sizeof(T), most, n, d, cus, 1).us * (double)pieces;
            words = !split && !(rh && rw) &&
                    by_words(by.us * (double)pieces + z, cut.us * (double)pieces + z,
                             (double)((rh ? 0 : n) + (rw ? 0 : v)) * (double)d);
            if (words) cut = by;
        }
        if (!dh || !dw)
            cut = PairCut{choose_cut((int)sizeof(T), d, n, most, cus, 64, words),
                          choose_cut((int)sizeof(T), d, most, n, cus, 64, words), false, 0.0};
        // one tile for every piece: its column sums are of as many parts
        const int z_tile = split_z ? kPlainCut.tile : choose_cut((int)sizeof(T), most, n, d, cus, 1, words).tile;
        const Cut zc = choose_cut((int)sizeof(T), most, n, d, cus, 64, words);
        const bool in_parts = !split && pieces == 1 && zc.splits > 1;  // as the loss
        const int parts = in_parts ? column_parts(n, most, cus) : (int)logit_grad_parts(z_tile, n);
        Op<T> ho(h, n, d, words), wo(w, v, d, words);
        T* dz = nullptr;
        float *acc = nullptr, *part = nullptr, *sums = nullptr, *up = nullptr, *z = nullptr;
        char *h_k = nullptr, *w_k = nullptr, *h_r = nullptr, *w_r = nullptr, *dz_k = nullptr, *dz_r = nullptr;
        Sides sides;
        Scratch sc;
        for (int pass = 0; pass < 2; ++pass) {
            ho.plan(sc);
            wo.plan(sc);
            dz = sc.take<T>((size_t)(n * ld));
            if (dh && pieces > 1) acc = sc.take<float>((size_t)(n * dh_ld));
            if (db) sums = sc.take<float>((size_t)parts * (size_t)most);
            if (in_parts) z = sc.take<float>(zc.part_bytes(most, n) / 4);
            if (scaled) up = sc.take<float>(2);
            size_t bytes = cut.part_bytes(d, n, d, most);
            if (split_h) bytes = std::max(bytes, sh.part_bytes(d, n));
            if (split_w) bytes = std::max(bytes, sw.part_bytes(d, most));
            part = sc.take<float>(bytes / 4);
            if (split_z) {
                h_k = sc.take<char>(split_bytes(n, d));
                w_k = sc.take<char>(split_bytes(most, d));
            }
            if (split_w) {
                h_r = sc.take<char>(split_bytes(n, d));
                dz_r = sc.take<char>(split_bytes(n, most));
            }
            if (split_h) {
                w_r = sc.take<char>(split_bytes(most, d));
                dz_k = sc.take<char>(split_bytes(n, most));
            }
            if (split) sides.flag = sc.take<uint32_t>(1);
            if (pass == 0) {
                rc = capi::scratch(sc.used, s, &sc.base, &cus);
                if (rc) return rc;
                sc.used = 0;
            }
        }
        if (split) sides.mark = next_mark();
        // f32 operands that every product has in parts are needed only where the
        // plain kernels stand in
        const Only plain = split ? sides.plain() : Only{};
        const bool all_split = split_z && (!dh || split_h) && (!dw || split_w);
        if (scaled) MLRS_TRY(launch_grad_scale(grad, target, n, ignore, up, s));
        const bool first_row = std::is_same<T, __bf16>::value;
        const float* down = scaled ? up + 1 : first_row ? grad : nullptr;
        const float* lift = scaled ? up : down;
        const Mat hm = ho.mat(), wm = wo.mat();
        capi::Timed timed(s, "softmax_xent_grad");
        if constexpr (std::is_same<T, float>::value) {
            SplitJob hk = split_job(h, d, n, d, h_k, false), hr = split_job(h, d, n, d, h_r, true);
            if (!split_z) hk.rows = 0;
            if (!split_w) hr.rows = 0;
            if (split) MLRS_TRY(launch_pack_split(hk, hr, sides.flag, sides.mark, s));
        }
        if (!all_split) MLRS_TRY(launch_pack<T>(ho.job(), wo.job(), Only{}, s));
        for (int64_t v0 = 0; v0 < v; v0 += piece) {
            const int64_t vp = std::min(piece, v - v0);
            const bool last = v0 + vp == v;
            const Mat dzm{dz, ld};
            const ColumnSums<T> col{db ? db + v0 : nullptr, sums, parts, down};
            if constexpr (std::is_same<T, float>::value) {
                const float* wp = w + v0 * d;
                SplitJob wk = split_job(wp, d, vp, d, w_k, false), wr = split_job(wp, d, vp, d, w_r, true);
                if (!split_z) wk.rows = 0;
                if (!split_h) wr.rows = 0;
                if (split) MLRS_TRY(launch_pack_split(wk, wr, sides.flag, sides.mark, s));
                if (all_split) MLRS_TRY(launch_pack<T>(ho.job(), wo.job(), plain, s));
                if (split_z)
                    MLRS_TRY(launch_logit_grad_split(split_mat(h_k, d, false), split_mat(w_k, d, false), bias, target,
                                                     lse, grad, n, v0, vp, v, d, ignore, dz, ld, sums, sides.split(), s));
            }
            if (in_parts) {
                MLRS_TRY(launch_logit_parts<T>(hm, wm, n, v, d, zc, z, s));
                MLRS_TRY(launch_logit_grad_rows<T>(z, zc, bias, target, lse, grad, lift, n, v, ignore, dz, ld, sums,
                                                   parts, s));
            } else {
                MLRS_TRY(launch_logit_grad<T>(hm, wm, bias, target, lse, grad, lift, n, v0, vp, v, d, ignore, dz, ld, sums,
                                              z_tile, split_z ? plain : Only{}, s));
            }
            const StoreTo to_w{dw ? dw + v0 * d : nullptr, d, nullptr, nullptr, 0, down};
            StoreTo to_h{};
            to_h.ld = d;
            to_h.acc = acc;
            to_h.acc_ld = dh_ld;
            to_h.add = v0 > 0 ? acc : nullptr;
            if (last) {
                to_h.out = dh;
                to_h.alpha = down;
            }
            if constexpr (std::is_same<T, float>::value) {
                SplitJob zk = split_job(dz, ld, n, vp, dz_k, false), zr = split_job(dz, ld, n, vp, dz_r, true);
                if (!split_h) zk.rows = 0;
                if (!split_w) zr.rows = 0;
                if (split_h || split_w) MLRS_TRY(launch_pack_split(zk, zr, sides.flag, sides.mark, s));
                if (all_split) MLRS_TRY(launch_pack<T>(ho.job(), wo.job(), plain, s));
                if (split_w)
                    MLRS_TRY(launch_product_split(split_mat(h_r, d, true), split_mat(dz_r, vp, true), false, d, vp, n,
                                                  to_w, sw, part, sides.split(), s));
                // a last piece's parts of the contraction may be empty ones
                Cut c = sh;
                if (vp < most) c = Cut{0, 1, 0, 0.0};
                if (split_h)
                    MLRS_TRY(launch_product_split(split_mat(w_r, d, true), split_mat(dz_k, vp, false), true, d, n, vp,
                                                  to_h, c, part, sides.split(), s));
            }
            Product ph{Mat{(const T*)wm.p + v0 * wm.ld, wm.ld}, dzm, d, n, vp, to_h}, pw{hm, dzm, d, vp, n, to_w};
            if (split_h || split_w)
                MLRS_TRY(launch_products<T>(split_h ? ph : Product{}, split_w ? pw : Product{}, kPlainPair, nullptr,
                                            ColumnSums<T>{}, 0, plain, s));
            if (!dh || split_h) ph.m = 0;
            if (!dw || split_w) pw.m = 0;
            PairCut c = cut;  // a last piece's contraction may have fewer parts
            if (c.x.splits > 1) c.x.splits = (int)((vp + c.x.k_split - 1) / c.x.k_split);
            if (ph.m || pw.m)
                MLRS_TRY(launch_products<T>(ph, pw, c, part, col, vp, Only{}, s));
            else
                MLRS_TRY(launch_sum_parts<T>(col, vp, s));
        }
        return MLRS_OK;
    });
}

bool dtype_ok(int32_t t) { return t >= MLRS_DTYPE_F32 && t <= MLRS_DTYPE_BF16; }

}  // namespace

extern "C" {

#define MLRS_TRAIN_ENTRY(SUFFIX, ABI, T)                                                                             \
    int32_t mlrs_linear_##SUFFIX(const ABI* x, int64_t x_len, int64_t n, int64_t d_in, const ABI* w, int64_t w_len,  \
                                 int64_t d_out, const ABI* bias, int64_t bias_len, const ABI* residual,              \
                                 int64_t residual_len, int32_t activation, ABI* y, int64_t y_len, ABI* preact,       \
                                 int64_t preact_len, void* stream) {                                                 \
        return linear_impl<T>((const T*)x, x_len, n, d_in, (const T*)w, w_len, d_out, (const T*)bias, bias_len,      \
                              (const T*)residual, residual_len, activation, (T*)y, y_len, (T*)preact, preact_len,    \
                              stream);                                                                               \
    }                                                                                                                \
    int32_t mlrs_linear_grad_##SUFFIX(                                                                               \
        const ABI* dy, int64_t dy_len, const ABI* x, int64_t x_len, int64_t n, int64_t d_in, const ABI* w,           \
        int64_t w_len, int64_t d_out, const ABI* preact, int64_t preact_len, int32_t activation, ABI* dx,            \
        int64_t dx_len, ABI* dw, int64_t dw_len, ABI* dbias, int64_t dbias_len, void* stream) {                      \
        return linear_grad_impl<T>((const T*)dy, dy_len, (const T*)x, x_len, n, d_in, (const T*)w, w_len, d_out,     \
                                   (const T*)preact, preact_len, activation, (T*)dx, dx_len, (T*)dw, dw_len,         \
                                   (T*)dbias, dbias_len, stream);                                                    \
    }                                                                                                                \
    int32_t mlrs_softmax_xent_##SUFFIX(const ABI* h, int64_t h_len, int64_t n, int64_t d, const ABI* w,              \
                                       int64_t w_len, int64_t classes, const ABI* bias, int64_t bias_len,            \
                                       const int64_t* target, int64_t target_len, int64_t ignore_index, float* loss, \
                                       float* lse, int64_t out_len, void* stream) {                                  \
        return xent_impl<T>((const T*)h, h_len, n, d, (const T*)w, w_len, classes, (const T*)bias, bias_len, target, \
                            target_len, ignore_index, loss, lse, out_len, stream);                                   \
    }                                                                                                                \
    int32_t mlrs_softmax_xent_grad_##SUFFIX(                                                                         \
        const ABI* h, int64_t h_len, int64_t n, int64_t d, const ABI* w, int64_t w_len, int64_t classes,             \
        const ABI* bias, int64_t bias_len, const int64_t* target, int64_t target_len, int64_t ignore_index,          \
        const float* lse, const float* grad, int64_t out_len, ABI* dh, int64_t dh_len, ABI* dw, int64_t dw_len,      \
        ABI* dbias, int64_t dbias_len, void* stream) {                                                               \
        return xent_grad_impl<T>((const T*)h, h_len, n, d, (const T*)w, w_len, classes, (const T*)bias, bias_len,    \
                                 target, target_len, ignore_index, lse, grad, out_len, (T*)dh, dh_len, (T*)dw,       \
                                 dw_len, (T*)dbias, dbias_len, stream);                                              \
    }
MLRS_TRAIN_ENTRY(f32, float, float)
MLRS_TRAIN_ENTRY(f16, uint16_t, _Float16)
MLRS_TRAIN_ENTRY(bf16, uint16_t, __bf16)

int32_t mlrs_grad_clip_scale(const mlrs_grad_tensor* tensors, int64_t count, double max_norm, float* norm,
                             float* scale, void* stream) {
    const char* where = "grad_clip_scale";
    return capi::call([&]() -> int32_t {
        if (count < 0) return capi::shape_error("tensors", count, 1, 0);
        if (count > 0 && !tensors) return null_error("tensors");
        for (int64_t i = 0; i < count; ++i) {
            if (tensors[i].len < 0) return capi::shape_error("tensors", i, 1, tensors[i].len);
            if (!dtype_ok(tensors[i].dtype))
                return capi::error(MLRS_ERR_UNSUPPORTED, "dtype", tensors[i].dtype, i, 0, "unknown element type");
            if (tensors[i].len > 0 && !tensors[i].grad) return null_error("grad");
        }
        if (!(max_norm > 0.0))
            return capi::error(MLRS_ERR_INVALID_PARAM, "max_norm", 0, 0, 0, "max_norm is invalid (must be > 0)");
        if (!norm || !scale) return null_error("out");
        const hipStream_t s = (hipStream_t)stream;
        const int64_t parts = norm_parts(tensors, count);
        char* ws = nullptr;
        int cus = 0;
        const int32_t rc = capi::scratch((size_t)parts * sizeof(double), s, &ws, &cus);
        if (rc) return rc;
        capi::Timed timed(s, "grad_clip_scale");
        MLRS_TRY(launch_clip_scale(tensors, count, max_norm, (double*)ws, norm, scale, s));
        return MLRS_OK;
    });
}

int32_t mlrs_adamw_step(const mlrs_adamw_tensor* tensors, int64_t count, int32_t state_bits, double lr, double beta1,
                        double beta2, double eps, int64_t step, const float* scale, uint32_t seed, void* stream) {
    const char* where = "adamw_step";
    return capi::call([&]() -> int32_t {
        if (count < 0) return capi::shape_error("tensors", count, 1, 0);
        if (count > 0 && !tensors) return null_error("tensors");
        if (state_bits != 32 && state_bits != 8)
            return capi::error(MLRS_ERR_UNSUPPORTED, "state_bits", state_bits, 0, 0, "states have 32 or 8 bits");
        auto invalid = [](const char* name, const char* message) {
            return capi::error(MLRS_ERR_INVALID_PARAM, name, 0, 0, 0, message);
        };
        if (!(lr >= 0.0) || std::isinf(lr)) return invalid("lr", "lr is invalid (must be finite and >= 0)");
        if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0))
            return invalid("betas", "betas are invalid (must be in [0, 1))");
        if (!(eps >= 0.0) || std::isinf(eps)) return invalid("eps", "eps is invalid (must be finite and >= 0)");
        if (step < 1) return invalid("step", "step is invalid (counts from 1)");
        for (int64_t i = 0; i < count; ++i) {
            const mlrs_adamw_tensor& t = tensors[i];
            if (t.len < 0) return capi::shape_error("tensors", i, 1, t.len);
            if (!dtype_ok(t.param_dtype) || !dtype_ok(t.grad_dtype))
                return capi::error(MLRS_ERR_UNSUPPORTED, "dtype", t.param_dtype, t.grad_dtype, 0,
                                   "unknown element type");
            if (!(t.weight_decay >= 0.0) || std::isinf(t.weight_decay))
                return invalid("weight_decay", "weight_decay is invalid (must be finite and >= 0)");
            if (!adamw_launchable(t.len))
                return capi::error(MLRS_ERR_UNSUPPORTED, "tensors", i, 1, t.len, "a tensor has at most 2^36 - 4096 elements");
            if (t.len == 0) continue;
            if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return null_error("tensors");
            if (t.param_dtype != MLRS_DTYPE_F32 && !t.master) return null_error("master");
            if (state_bits == 8 && (!t.avg_scale || !t.avg_sq_scale)) return null_error("scales");
        }
        const double c1 = 1.0 - std::pow(beta1, (double)step), c2 = 1.0 - std::pow(beta2, (double)step);
        AdamwHyper hy;
        hy.b1 = (float)beta1;
        hy.c1 = (float)(1.0 - beta1);
        hy.b2 = (float)beta2;
        hy.c2 = (float)(1.0 - beta2);
        hy.step = (float)(lr / c1);
        hy.root = (float)(1.0 / std::sqrt(c2));
        hy.eps = (float)eps;
        hy.lr = lr;
        hy.seed = seed;
        const hipStream_t s = (hipStream_t)stream;
        capi::Timed timed(s, "adamw_step");
        MLRS_TRY(launch_adamw(tensors, count, state_bits, hy, scale, s));
        return MLRS_OK;
    });
}

int32_t mlrs_adamw_state_values(const uint8_t* codes, int64_t len, const float* scales, int64_t scales_len,
                                int32_t which, float* out, int64_t out_len, void* stream) {
    const char* where = "adamw_state_values";
    return capi::call([&]() -> int32_t {
        if (len < 0) return capi::shape_error("codes", len, 1, len);
        if (scales_len != (len + MLRS_STATE_BLOCK - 1) / MLRS_STATE_BLOCK)
            return capi::shape_error("scales", (len + MLRS_STATE_BLOCK - 1) / MLRS_STATE_BLOCK, 1, scales_len);
        if (out_len != len) return capi::shape_error("out", len, 1, out_len);
        if (which != 0 && which != 1)
            return capi::error(MLRS_ERR_UNSUPPORTED, "which", which, 0, 0, "which is 0 (exp_avg) or 1 (exp_avg_sq)");
        if (len == 0) return MLRS_OK;
        if (!codes || !scales || !out) return null_error(!codes ? "codes" : !scales ? "scales" : "out");
        MLRS_TRY(launch_state_values(codes, scales, len, which, out, (hipStream_t)stream));
        return MLRS_OK;
    });
}

}  // extern "C"
