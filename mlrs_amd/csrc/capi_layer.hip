// C-ABI layer of the operators of an encoder's layer beside its product:
// validation (before any launch) and dispatch.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/mlrs_hip_knn.h"
#include "capi_train.hpp"
#include "train_kernels.hpp"

using namespace mlrs;
using namespace mlrs::train;

namespace {

int32_t invalid(const char* name, const char* message) {
    return capi::error(MLRS_ERR_INVALID_PARAM, name, 0, 0, 0, message);
}

bool activation_ok(int32_t act) { return act >= MLRS_ACT_NONE && act <= MLRS_ACT_SILU; }
int32_t activation_error(int32_t act) {
    return capi::error(MLRS_ERR_UNSUPPORTED, "activation", act, 0, 0, "unknown activation");
}

bool probability_ok(double p) { return p >= 0.0 && p < 1.0; }
int32_t probability_error() { return invalid("p", "p is invalid (must be in [0, 1))"); }

Drop drop_of(double p, uint64_t seed, uint64_t offset, const int64_t* step) {
    Drop d;
    d.threshold = (uint32_t)std::min(65535.0, std::floor(p * 65536.0 + 0.5));
    d.factor = (float)(65536.0 / (65536.0 - (double)d.threshold));
    d.k0 = (uint32_t)seed;
    d.k1 = (uint32_t)(seed >> 32);
    d.offset = offset;
    d.step = step;
    return d;
}

template <typename T>
int32_t dropout_impl(const T* x, int64_t x_len, double p, uint64_t seed, uint64_t offset, const int64_t* step,
                     const T* residual, int64_t residual_len, T* y, int64_t y_len, void* stream) {
    const char* where = "dropout";
    return capi::call([&]() -> int32_t {
        if (x_len < 0) return capi::shape_error("x", x_len, 1, x_len);
        if (residual ? residual_len != x_len : residual_len != 0)
            return capi::shape_error("residual", x_len, 1, residual_len);
        if (y_len != x_len) return capi::shape_error("out", x_len, 1, y_len);
        if (!probability_ok(p)) return probability_error();
        if (x_len == 0) return MLRS_OK;
        if (!x || !y) return null_error(!x ? "x" : "out");
        const Span sx(x, x_len), sr(residual, residual_len), sy(y, y_len);
        if ((y != x && sy.meets(sx)) || (y != residual && sy.meets(sr)) || sy.meets(Span(step, 1)))
            return overlap_error("out");
        int cus = 0;
        const int32_t rc = capi::cu_count(&cus);
        if (rc) return rc;
        const hipStream_t s = (hipStream_t)stream;
        capi::Timed timed(s, "dropout");
        MLRS_TRY(launch_dropout<T>(x, residual, y, x_len, drop_of(p, seed, offset, step), cus, s));
        return MLRS_OK;
    });
}

// Whether n x s x c is `len`, without overflow.
bool volume(int64_t n, int64_t s, int64_t c, int64_t len) {
    int64_t rows;
    return n >= 0 && s >= 0 && !__builtin_mul_overflow(n, s, &rows) && capi::geometry(rows, c, len);
}

int32_t check_norm(int64_t x_len, int64_t n, int64_t s, int64_t c, int64_t g, const void* w, int64_t w_len,
                   const void* b, int64_t b_len) {
    if (!volume(n, s, c, x_len)) return capi::shape_error("x", n, c, x_len);
    if (s < 1 || c < 1) return capi::shape_error("features", s, c, 0);
    if (g < 1 || c % g != 0) return capi::shape_error("groups", g, c, 0);
    if (c / g > kNormGroup)
        return capi::error(MLRS_ERR_UNSUPPORTED, "groups", g, c, 0, "a group is limited to 8192 channels");
    if (c > (int64_t)1 << 22 || s > (int64_t)1 << 31 || n > (int64_t)1 << 40)
        return capi::error(MLRS_ERR_UNSUPPORTED, "features", s, c, 0,
                           "channels are limited to 2^22, positions to 2^31, samples to 2^40");
    if (w ? w_len != c : w_len != 0) return capi::shape_error("weight", 1, c, w_len);
    if (b ? b_len != c : b_len != 0) return capi::shape_error("bias", 1, c, b_len);
    return MLRS_OK;
}

template <typename T>
int32_t norm_impl(const T* x, int64_t x_len, int64_t n, int64_t s, int64_t c, int64_t g, const T* w, int64_t w_len,
                  const T* b, int64_t b_len, double eps, int32_t act, double p, uint64_t seed, uint64_t offset,
                  const int64_t* step, T* y, int64_t y_len, float* mean, float* rstd, int64_t stats_len,
                  void* stream) {
    const char* where = "group_norm";
    return capi::call([&]() -> int32_t {
        int32_t rc = check_norm(x_len, n, s, c, g, w, w_len, b, b_len);
        if (rc) return rc;
        if (!volume(n, s, c, y_len)) return capi::shape_error("out", n, c, y_len);
        if (mean || rstd ? !capi::geometry(n, g, stats_len) : stats_len != 0)
            return capi::shape_error("stats", n, g, stats_len);
        if (!activation_ok(act)) return activation_error(act);
        if (!(eps >= 0.0) || std::isinf(eps)) return invalid("eps", "eps is invalid (must be finite and >= 0)");
        if (!probability_ok(p)) return probability_error();
        if (n == 0) return MLRS_OK;
        if (!x || !y) return null_error(!x ? "x" : "out");
        if (!mean != !rstd) return null_error("stats");
        const Span sx(x, x_len), sw(w, w_len), sb(b, b_len), sy(y, y_len), sm(mean, stats_len), so(step, 1);
        if (sy.meets({sx, sw, sb, so})) return overlap_error("out");
        if (sm.meets({sx, sw, sb, so, sy}) || Span(rstd, stats_len).meets({sx, sw, sb, so, sy, sm}))
            return overlap_error("stats");
        int cus = 0;
        rc = capi::cu_count(&cus);
        if (rc) return rc;
        NormCall k{x, w, b, nullptr, y, mean, rstd, nullptr, nullptr, n, s, c, g, (float)eps, act,
                   drop_of(p, seed, offset, step)};
        const hipStream_t st = (hipStream_t)stream;
        char* room = nullptr;
        if (const size_t bytes = norm_scratch((int)sizeof(T), k, cus)) {
            rc = eager_scratch(bytes, st, &room, &cus);
            if (rc) return rc;
        }
        capi::Timed timed(st, "group_norm");
        MLRS_TRY(launch_norm<T>(k, (float*)room, cus, st));
        return MLRS_OK;
    });
}

template <typename T>
int32_t norm_grad_impl(const T* dy, int64_t dy_len, const T* x, int64_t x_len, int64_t n, int64_t s, int64_t c,
                       int64_t g, const T* w, int64_t w_len, const T* b, int64_t b_len, const float* mean,
                       const float* rstd, int64_t stats_len, int32_t act, double p, uint64_t seed, uint64_t offset,
                       const int64_t* step, T* dx, int64_t dx_len, T* dw, int64_t dw_len, T* db, int64_t db_len,
                       void* stream) {
    const char* where = "group_norm_grad";
    return capi::call([&]() -> int32_t {
        int32_t rc = check_norm(x_len, n, s, c, g, w, w_len, b, b_len);
        if (rc) return rc;
        if (!volume(n, s, c, dy_len)) return capi::shape_error("dy", n, c, dy_len);
        if (!capi::geometry(n, g, stats_len)) return capi::shape_error("stats", n, g, stats_len);
        if (dx ? !volume(n, s, c, dx_len) : dx_len != 0) return capi::shape_error("dx", n, c, dx_len);
        if (dw ? dw_len != c : dw_len != 0) return capi::shape_error("dweight", 1, c, dw_len);
        if (db ? db_len != c : db_len != 0) return capi::shape_error("dbias", 1, c, db_len);
        if (!activation_ok(act)) return activation_error(act);
        if (!probability_ok(p)) return probability_error();
        if (!dx && !dw && !db) return MLRS_OK;
        if (n > 0 && (!dy || !x || !mean || !rstd)) return null_error(!dy ? "dy" : !x ? "x" : "stats");
        const Span sd(dy, dy_len), sx(x, x_len), sw(w, w_len), sb(b, b_len), sm(mean, stats_len), sr(rstd, stats_len),
            so(step, 1), sdx(dx, dx_len), sdw(dw, dw_len);
        if (sdx.meets({sd, sx, sw, sb, sm, sr, so})) return overlap_error("dx");
        if (sdw.meets({sd, sx, sw, sb, sm, sr, so, sdx})) return overlap_error("dweight");
        if (Span(db, db_len).meets({sd, sx, sw, sb, sm, sr, so, sdx, sdw})) return overlap_error("dbias");
        int cus = 0;
        rc = capi::cu_count(&cus);
        if (rc) return rc;
        NormCall k{x, w, b, dy, dx, const_cast<float*>(mean), const_cast<float*>(rstd), dw, db, n, s, c, g, 0.0f, act,
                   drop_of(p, seed, offset, step)};
        const hipStream_t st = (hipStream_t)stream;
        char* room = nullptr;
        if (const size_t bytes = norm_grad_scratch((int)sizeof(T), k, cus)) {
            rc = eager_scratch(bytes, st, &room, &cus);
            if (rc) return rc;
        }
        capi::Timed timed(st, "group_norm_grad");
        MLRS_TRY(launch_norm_grad<T>(k, (float*)room, cus, st));
        return MLRS_OK;
    });
}

// ---------------------------------------------------------------------------
// 8-bit floating point
// ---------------------------------------------------------------------------
constexpr int64_t kMaxCount = 0x7FFFFFFF - 512;    // a tile past it must not overflow
constexpr int64_t kMaxColumns = (int64_t)1 << 22;  // 256 rows of codes within a buffer descriptor's 2^31

int64_t tiles128(int64_t n) { return (n + 127) / 128; }

// Sizes of a layer: n rows (x) by k, and m x k weights.
int32_t check_layer(int64_t x_len, int64_t n, int64_t k, int64_t m) {
    if (!capi::geometry(n, k, x_len)) return capi::shape_error("x", n, k, x_len);
    if (k < 1 || m < 1) return capi::shape_error("features", m, k, 0);
    if (k > kMaxColumns || m > kMaxColumns)
        return capi::error(MLRS_ERR_UNSUPPORTED, "features", m, k, 0, "features are limited to 2^22");
    if (n > kMaxCount) return capi::error(MLRS_ERR_UNSUPPORTED, "rows", n, k, 0, "row counts are limited to 2^31 - 513");
    return MLRS_OK;
}
int32_t check_codes(const char* codes_name, const char* scales_name, const uint8_t* codes, int64_t codes_len,
                    const uint8_t* scales, int64_t scales_len, int64_t rows, int64_t k) {
    if (codes_len != rows * fp8_columns(k)) return capi::shape_error(codes_name, rows, fp8_columns(k), codes_len);
    if (scales_len != tiles128(rows) * fp8_scale_row(k))
        return capi::shape_error(scales_name, tiles128(rows), fp8_scale_row(k), scales_len);
    if ((uintptr_t)codes % 16 != 0) return invalid(codes_name, "codes must be aligned to 16 bytes");
    if ((uintptr_t)scales % 4 != 0) return invalid(scales_name, "scales must be aligned to 4 bytes");
    return MLRS_OK;
}
// A product's grid must fit, in the largest tiles.
bool grid_fits(int64_t m, int64_t n) { return launchable(((m + 255) / 256) * ((n + 255) / 256), 512); }
bool codes_fit(int64_t n, int64_t k) { return launchable(tiles128(n) * tiles128(k), 512); }
int32_t grid_error(int64_t m, int64_t n) {
    return capi::error(MLRS_ERR_UNSUPPORTED, "rows", n, m, 0, "the product has more tiles than a launch");
}

template <typename T>
int32_t fp8_weight_impl(const T* w, int64_t w_len, int64_t m, int64_t k, uint8_t* codes, int64_t codes_len,
                        uint8_t* scales, int64_t scales_len, uint8_t* codes_t, int64_t codes_t_len, uint8_t* scales_t,
                        int64_t scales_t_len, void* stream) {
    const char* where = "fp8_weight";
    return capi::call([&]() -> int32_t {
        if (!capi::geometry(m, k, w_len)) return capi::shape_error("w", m, k, w_len);
        int32_t rc = check_layer(0, 0, k, m);
        if (rc) return rc;
        rc = check_codes("codes", "scales", codes, codes_len, scales, scales_len, m, k);
        if (rc) return rc;
        if (codes_t || scales_t || codes_t_len || scales_t_len) {
            rc = check_codes("codes_t", "scales_t", codes_t, codes_t_len, scales_t, scales_t_len, k, m);
            if (rc) return rc;
            if (!codes_t || !scales_t) return null_error(!codes_t ? "codes_t" : "scales_t");
        }
        if (!w || !codes || !scales) return null_error(!w ? "w" : !codes ? "codes" : "scales");
        if (!codes_fit(m, k)) return grid_error(k, m);
        const Span sw(w, w_len), sc(codes, codes_len), ss(scales, scales_len), st(codes_t, codes_t_len);
        if (sc.meets(sw)) return overlap_error("codes");
        if (ss.meets({sw, sc})) return overlap_error("scales");
        if (st.meets({sw, sc, ss})) return overlap_error("codes_t");
        if (Span(scales_t, scales_t_len).meets({sw, sc, ss, st})) return overlap_error("scales_t");
        const hipStream_t s = (hipStream_t)stream;
        capi::Timed timed(s, "fp8_weight");
        MLRS_TRY(launch_fp8_weight<T>(w, m, k, Fp8Mat{codes, scales, true}, Fp8Mat{codes_t, scales_t, true}, s));
        return MLRS_OK;
    });
}

template <typename T>
int32_t linear_fp8_impl(const T* x, int64_t x_len, int64_t n, int64_t k, const uint8_t* codes, int64_t codes_len,
                        const uint8_t* scales, int64_t scales_len, int64_t m, const T* bias, int64_t bias_len,
                        const T* residual, int64_t residual_len, int32_t act, T* y, int64_t y_len, T* z,
                        int64_t z_len, void* stream) {
    const char* where = "linear_fp8";
    return capi::call([&]() -> int32_t {
        int32_t rc = check_layer(x_len, n, k, m);
        if (rc) return rc;
        rc = check_codes("codes", "scales", codes, codes_len, scales, scales_len, m, k);
        if (rc) return rc;
        if (bias ? bias_len != m : bias_len != 0) return capi::shape_error("bias", 1, m, bias_len);
        if (residual ? !capi::geometry(n, m, residual_len) : residual_len != 0)
            return capi::shape_error("residual", n, m, residual_len);
        if (!capi::geometry(n, m, y_len)) return capi::shape_error("out", n, m, y_len);
        if (z ? !capi::geometry(n, m, z_len) : z_len != 0) return capi::shape_error("preact", n, m, z_len);
        if (!activation_ok(act)) return activation_error(act);
        if (n == 0) return MLRS_OK;
        if (!x || !codes || !scales || !y) return null_error(!x ? "x" : !codes ? "codes" : !scales ? "scales" : "out");
        if (!grid_fits(m, n) || !codes_fit(n, k)) return grid_error(m, n);
        const Span sx(x, x_len), sc(codes, codes_len), ss(scales, scales_len), sb(bias, bias_len),
            sr(residual, residual_len), sy(y, y_len);
        if (sy.meets({sx, sc, ss, sb}) || (y != residual && sy.meets(sr))) return overlap_error("out");
        if (Span(z, z_len).meets({sx, sc, ss, sb, sr, sy})) return overlap_error("preact");
        const hipStream_t s = (hipStream_t)stream;
        const LinearOut o{bias, residual, y, z, act};
        const Fp8Mat w{codes, scales, true};
        int cus = 0;
        rc = capi::cu_count(&cus);
        if (rc) return rc;
        if (fp8_few_rows(n, m, k)) {
            capi::Timed timed(s, "linear_fp8_few");
            MLRS_TRY(launch_fp8_few<T>(x, w, n, m, k, o, s));
            return MLRS_OK;
        }
        constexpr bool kValues = sizeof(T) == 4;
        const Cut cut = choose_cut_fp8((int)sizeof(T), m, n, k, cus);
        uint8_t *xc = nullptr, *xs = nullptr, *wv = nullptr;
        float* part = nullptr;
        Scratch sc8;
        for (int pass = 0; pass < 2; ++pass) {
            xc = sc8.take<uint8_t>((size_t)(n * fp8_columns(k)) * (kValues ? 2 : 1));
            if (kValues)
                wv = sc8.take<uint8_t>((size_t)(m * fp8_columns(k)) * 2);
            else
                xs = sc8.take<uint8_t>((size_t)(n * fp8_scale_row(k)));
            part = sc8.take<float>(cut.part_bytes(m, n) / 4);
            if (pass == 0) {
                rc = eager_scratch(sc8.used, s, &sc8.base, &cus);
                if (rc) return rc;
                sc8.used = 0;
            }
        }
        const Fp8Mat xm{xc, xs, false};
        MLRS_TRY(launch_fp8_rows<T>(x, n, k, xm, s));
        if (kValues) MLRS_TRY(launch_fp8_values(w, m, k, wv, s));
        capi::Timed timed(s, "linear_fp8");
        MLRS_TRY(launch_fp8_linear<T>(xm, kValues ? Fp8Mat{wv, nullptr, false} : w, n, m, k, o, cut, part, s));
        return MLRS_OK;
    });
}

template <typename T>
int32_t linear_fp8_grad_impl(const T* dy, int64_t dy_len, const T* x, int64_t x_len, int64_t n, int64_t k,
                             const uint8_t* codes_t, int64_t codes_t_len, const uint8_t* scales_t,
                             int64_t scales_t_len, int64_t m, const T* z, int64_t z_len, int32_t act, T* dx,
                             int64_t dx_len, T* dw, int64_t dw_len, T* db, int64_t db_len, void* stream) {
    const char* where = "linear_fp8_grad";
    return capi::call([&]() -> int32_t {
        int32_t rc = check_layer(x_len, n, k, m);
        if (rc) return rc;
        if (codes_t || scales_t || codes_t_len || scales_t_len) {
            rc = check_codes("codes_t", "scales_t", codes_t, codes_t_len, scales_t, scales_t_len, k, m);
            if (rc) return rc;
        }
        if (!capi::geometry(n, m, dy_len)) return capi::shape_error("dy", n, m, dy_len);
        if (dx ? !capi::geometry(n, k, dx_len) : dx_len != 0) return capi::shape_error("dx", n, k, dx_len);
        if (dw ? !capi::geometry(m, k, dw_len) : dw_len != 0) return capi::shape_error("dw", m, k, dw_len);
        if (db ? db_len != m : db_len != 0) return capi::shape_error("dbias", 1, m, db_len);
        if (!activation_ok(act)) return activation_error(act);
        if (act == MLRS_ACT_NONE ? z_len != 0 : !capi::geometry(n, m, z_len))
            return capi::shape_error("preact", n, m, z_len);
        if (n > kMaxColumns)
            return capi::error(MLRS_ERR_UNSUPPORTED, "rows", n, k, 0, "rows of a gradient are limited to 2^22");
        if (!dx && !dw && !db) return MLRS_OK;
        if (n > 0) {
            if (!dy) return null_error("dy");
            if (dw && !x) return null_error("x");
            if (act != MLRS_ACT_NONE && !z) return null_error("preact");
        }
        if (dx && (!codes_t || !scales_t)) return null_error(!codes_t ? "codes_t" : "scales_t");
        if (!grid_fits(k, n) || !grid_fits(k, m) || !launchable(tiles128(n) * (tiles128(m) + tiles128(k)), 512))
            return grid_error(k, std::max(m, n));
        const Span ody(dy, dy_len), ox(x, x_len), oc(codes_t, codes_t_len), os(scales_t, scales_t_len), oz(z, z_len),
            odx(dx, dx_len), odw(dw, dw_len);
        if (odx.meets({ody, ox, oc, os, oz})) return overlap_error("dx");
        if (odw.meets({ody, ox, oc, os, oz, odx})) return overlap_error("dw");
        if (Span(db, db_len).meets({ody, ox, oc, os, oz, odx, odw})) return overlap_error("dbias");
        const hipStream_t s = (hipStream_t)stream;
        int cus = 0;
        rc = capi::cu_count(&cus);
        if (rc) return rc;
        if (n == 0) {  // sums of nothing
            constexpr int64_t kMost = (int64_t)1 << 27;  // columns of a launch
            const ColumnSums<T> none[2] = {{dw, nullptr, 0, nullptr}, {db, nullptr, 0, nullptr}};
            const int64_t len[2] = {dw_len, db_len};
            for (int i = 0; i < 2; ++i)
                for (int64_t c = 0; none[i].out && c < len[i]; c += kMost)
                    MLRS_TRY(launch_sum_parts<T>(ColumnSums<T>{none[i].out + c, nullptr, 0, nullptr},
                                                 std::min(kMost, len[i] - c), s));
            return MLRS_OK;
        }
        Cut cx{}, cw{};
        if (dx && dw)
            choose_pair_fp8((int)sizeof(T), k, n, m, k, m, n, cus, &cx, &cw);
        else if (dx)
            cx = choose_cut_fp8((int)sizeof(T), k, n, m, cus);
        else if (dw)
            cw = choose_cut_fp8((int)sizeof(T), k, m, n, cus);
        const int64_t runs = tiles128(n);
        constexpr bool kValues = sizeof(T) == 4;
        constexpr size_t kCode = kValues ? 2 : 1;  // bytes
        uint8_t *zc = nullptr, *zs = nullptr, *zct = nullptr, *zst = nullptr, *xct = nullptr, *xst = nullptr;
        uint8_t* wv = nullptr;
        float *sums = nullptr, *part = nullptr;
        Scratch sc;
        for (int pass = 0; pass < 2; ++pass) {
            if (dx) {
                zc = sc.take<uint8_t>((size_t)(n * fp8_columns(m)) * kCode);
                zs = sc.take<uint8_t>((size_t)(n * fp8_scale_row(m)));
                if (kValues) wv = sc.take<uint8_t>((size_t)(k * fp8_columns(m)) * kCode);
            }
            if (dw) {
                zct = sc.take<uint8_t>((size_t)(m * fp8_columns(n)) * kCode);
                zst = sc.take<uint8_t>((size_t)(m * fp8_scale_row(n)));
                xct = sc.take<uint8_t>((size_t)(k * fp8_columns(n)) * kCode);
                xst = sc.take<uint8_t>((size_t)(k * fp8_scale_row(n)));
            }
            if (db) sums = sc.take<float>((size_t)(runs * m));
            part = sc.take<float>(((dx ? cx.part_bytes(k, n) : 0) + (dw ? cw.part_bytes(k, m) : 0)) / 4);
            if (pass == 0) {
                rc = eager_scratch(sc.used, s, &sc.base, &cus);
                if (rc) return rc;
                sc.used = 0;
            }
        }
        const Fp8Mat dz{zc, zs, false}, dz_t{zct, zst, false}, x_t{xct, xst, false};
        MLRS_TRY(launch_fp8_grad_codes<T>(dy, act == MLRS_ACT_NONE ? nullptr : z, act, n, m, dz, dz_t, sums,
                                          dw ? x : nullptr, k, x_t, s));
        const Fp8Mat wt{codes_t, scales_t, true};
        if (kValues && dx) MLRS_TRY(launch_fp8_values(wt, k, m, wv, s));
        capi::Timed timed(s, "linear_fp8_grad");
        Fp8Product px{kValues ? Fp8Mat{wv, nullptr, false} : wt, dz, k, n, m, StoreTo{dx, k, nullptr, nullptr, 0, nullptr}};
        Fp8Product pw{x_t, dz_t, k, m, n, StoreTo{dw, k, nullptr, nullptr, 0, nullptr}};
        if (!dx) px.m = 0;
        if (!dw) pw.m = 0;
        MLRS_TRY(launch_fp8_products<T>(px, pw, cx, cw, part, ColumnSums<T>{db, sums, (int)runs, nullptr}, m, s));
        return MLRS_OK;
    });
}

}  // namespace

extern "C" {

#define MLRS_LAYER_ENTRY(SUFFIX, ABI, T)                                                                               \
    int32_t mlrs_dropout_##SUFFIX(const ABI* x, int64_t x_len, double p, uint64_t seed, uint64_t offset,              \
                                  const int64_t* step, const ABI* residual, int64_t residual_len, ABI* y,             \
                                  int64_t y_len, void* stream) {                                                      \
        return dropout_impl<T>((const T*)x, x_len, p, seed, offset, step, (const T*)residual, residual_len, (T*)y,    \
                               y_len, stream);                                                                        \
    }                                                                                                                 \
    int32_t mlrs_group_norm_##SUFFIX(const ABI* x, int64_t x_len, int64_t n, int64_t positions, int64_t channels,     \
                                     int64_t groups, const ABI* weight, int64_t weight_len, const ABI* bias,          \
                                     int64_t bias_len, double eps, int32_t activation, double p, uint64_t seed,       \
                                     uint64_t offset, const int64_t* step, ABI* y, int64_t y_len, float* mean,        \
                                     float* rstd, int64_t stats_len, void* stream) {                                  \
        return norm_impl<T>((const T*)x, x_len, n, positions, channels, groups, (const T*)weight, weight_len,         \
                            (const T*)bias, bias_len, eps, activation, p, seed, offset, step, (T*)y, y_len, mean,     \
                            rstd, stats_len, stream);                                                                 \
    }                                                                                                                 \
    int32_t mlrs_group_norm_grad_##SUFFIX(                                                                            \
        const ABI* dy, int64_t dy_len, const ABI* x, int64_t x_len, int64_t n, int64_t positions, int64_t channels,   \
        int64_t groups, const ABI* weight, int64_t weight_len, const ABI* bias, int64_t bias_len, const float* mean,  \
        const float* rstd, int64_t stats_len, int32_t activation, double p, uint64_t seed, uint64_t offset,           \
        const int64_t* step, ABI* dx, int64_t dx_len, ABI* dweight, int64_t dweight_len, ABI* dbias,                  \
        int64_t dbias_len, void* stream) {                                                                            \
        return norm_grad_impl<T>((const T*)dy, dy_len, (const T*)x, x_len, n, positions, channels, groups,            \
                                 (const T*)weight, weight_len, (const T*)bias, bias_len, mean, rstd, stats_len,       \
                                 activation, p, seed, offset, step, (T*)dx, dx_len, (T*)dweight, dweight_len,         \
                                 (T*)dbias, dbias_len, stream);                                                       \
    }
#define MLRS_FP8_ENTRY(SUFFIX, ABI, T)                                                                                \
    int32_t mlrs_fp8_weight_##SUFFIX(const ABI* w, int64_t w_len, int64_t d_out, int64_t d_in, uint8_t* codes,        \
                                     int64_t codes_len, uint8_t* scales, int64_t scales_len, uint8_t* codes_t,        \
                                     int64_t codes_t_len, uint8_t* scales_t, int64_t scales_t_len, void* stream) {    \
        return fp8_weight_impl<T>((const T*)w, w_len, d_out, d_in, codes, codes_len, scales, scales_len, codes_t,     \
                                  codes_t_len, scales_t, scales_t_len, stream);                                       \
    }                                                                                                                 \
    int32_t mlrs_linear_fp8_##SUFFIX(const ABI* x, int64_t x_len, int64_t n, int64_t d_in, const uint8_t* codes,      \
                                     int64_t codes_len, const uint8_t* scales, int64_t scales_len, int64_t d_out,     \
                                     const ABI* bias, int64_t bias_len, const ABI* residual, int64_t residual_len,    \
                                     int32_t activation, ABI* y, int64_t y_len, ABI* preact, int64_t preact_len,      \
                                     void* stream) {                                                                  \
        return linear_fp8_impl<T>((const T*)x, x_len, n, d_in, codes, codes_len, scales, scales_len, d_out,           \
                                  (const T*)bias, bias_len, (const T*)residual, residual_len, activation, (T*)y,      \
                                  y_len, (T*)preact, preact_len, stream);                                             \
    }                                                                                                                 \
    int32_t mlrs_linear_fp8_grad_##SUFFIX(                                                                            \
        const ABI* dy, int64_t dy_len, const ABI* x, int64_t x_len, int64_t n, int64_t d_in, const uint8_t* codes_t,  \
        int64_t codes_t_len, const uint8_t* scales_t, int64_t scales_t_len, int64_t d_out, const ABI* preact,         \
        int64_t preact_len, int32_t activation, ABI* dx, int64_t dx_len, ABI* dw, int64_t dw_len, ABI* dbias,         \
        int64_t dbias_len, void* stream) {                                                                            \
        return linear_fp8_grad_impl<T>((const T*)dy, dy_len, (const T*)x, x_len, n, d_in, codes_t, codes_t_len,       \
                                       scales_t, scales_t_len, d_out, (const T*)preact, preact_len, activation,       \
                                       (T*)dx, dx_len, (T*)dw, dw_len, (T*)dbias, dbias_len, stream);                 \
    }
MLRS_FP8_ENTRY(f32, float, float)
MLRS_FP8_ENTRY(f16, uint16_t, _Float16)
MLRS_FP8_ENTRY(bf16, uint16_t, __bf16)
MLRS_LAYER_ENTRY(f32, float, float)
MLRS_LAYER_ENTRY(f16, uint16_t, _Float16)
MLRS_LAYER_ENTRY(bf16, uint16_t, __bf16)

}  // extern "C"
