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
MLRS_LAYER_ENTRY(f32, float, float)
MLRS_LAYER_ENTRY(f16, uint16_t, _Float16)
MLRS_LAYER_ENTRY(bf16, uint16_t, __bf16)

}  // extern "C"
