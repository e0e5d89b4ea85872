// Softmax cross entropy of h w^T + bias over many classes, without the logits
// in memory.  Forwards, a tile of logits is reduced in registers to the
// largest and the sum of exponentials of each row; backwards, the gradient of
// a piece of the vocabulary is made from recomputed logits and goes into the
// two products of the gradient before the next piece.
#include "train_launch.hpp"

namespace mlrs {
namespace train {

static const int kWaveRows[4] = {128, 64, 32, 32};  // classes of a wave, by tile

int64_t stats_parts(int tile, int64_t classes) {
    const int rows = kTileRows[tile];
    return (classes + rows - 1) / rows * (rows / kWaveRows[tile]);
}

template <typename T>
hipError_t launch_xent_stats(Mat h, Mat w, const T* bias, const int64_t* target, int64_t n, int64_t classes, int64_t k,
                             int tile, float* top, float* total, float* hit, const Only& only, hipStream_t s) {
    const StatsEpi<T> e{bias, target, top, total, hit};
    return launch_gemm<T>(tile, w, h, classes, n, k, 1, 0, only, e, s);
}

// A workgroup joins the parts of 16 rows: sixteen threads take every sixteenth
// part of a row, four at a time, with a running largest and sum; then one of
// them joins the sixteen.  Fixed order, so a row's loss does not depend on the
// others.
__global__ __launch_bounds__(256) void xent_join_kernel(const float* __restrict__ top, const float* __restrict__ total,
                                                        int64_t parts, const float* __restrict__ hit,
                                                        const int64_t* __restrict__ target, int64_t n,
                                                        int64_t classes, int64_t ignore, float* __restrict__ loss,
                                                        float* __restrict__ lse, Only only) {
    if (skipped(only.flag, only.mark, only.wanted)) return;
    constexpr int kRows = 16, kSlices = 16, kAtOnce = 4;
    __shared__ float tops[kSlices][kRows], sums[kSlices][kRows];
    const int c = threadIdx.x % kRows, p0 = threadIdx.x / kRows;
    const int64_t i = (int64_t)blockIdx.x * kRows + c;
    const float none = -__builtin_huge_valf();
    float mx = none, sum = 0.0f;
    if (i < n) {
        for (int64_t p = p0; p < parts; p += kSlices * kAtOnce) {
            float t[kAtOnce], s[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int64_t at = p + u * kSlices;
                t[u] = at < parts ? top[at * n + i] : none;
                s[u] = at < parts ? total[at * n + i] : 0.0f;
            }
            float most = mx;
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) most = fmaxf(most, t[u]);
            const float base = most == none ? 0.0f : most;
            sum *= exp_fast(mx - base);
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) sum += s[u] * exp_fast(t[u] - base);
            mx = most;
        }
    }
    tops[p0][c] = mx;
    sums[p0][c] = sum;
    __syncthreads();
    if (p0 != 0 || i >= n) return;
#pragma unroll
    for (int p = 1; p < kSlices; ++p) mx = fmaxf(mx, tops[p][c]);
    const float base = mx == none ? 0.0f : mx;
    sum = 0.0f;
#pragma unroll
    for (int p = 0; p < kSlices; ++p) sum += sums[p][c] * exp_fast(tops[p][c] - base);
    const float l = base + logf(sum);
    lse[i] = l;
    const int64_t t = target[i];
    float v = 0.0f;
    if (t != ignore) v = t >= 0 && t < classes ? l - hit[i] : __builtin_nanf("");
    loss[i] = v;
}

hipError_t launch_xent_join(const float* top, const float* total, int64_t parts, const float* hit,
                            const int64_t* target, int64_t n, int64_t classes, int64_t ignore, float* loss, float* lse,
                            const Only& only, hipStream_t s) {
    if (!launchable((n + 15) / 16, 256)) return hipErrorInvalidConfiguration;  // the caller's chunks are shorter
    xent_join_kernel<<<dim3((unsigned)((n + 15) / 16)), 256, 0, s>>>(top, total, parts, hit, target, n, classes,
                                                                    ignore, loss, lse, only);
    return hipGetLastError();
}

// up_down[0]: the factor that brings the largest |gradient| of a kept row to 2^13,
// so that the products of it with probabilities down to 2^-27 are normal numbers of
// half precision; up_down[1]: its inverse.
__global__ __launch_bounds__(1024) void grad_scale_kernel(const float* __restrict__ grad,
                                                          const int64_t* __restrict__ target, int64_t n,
                                                          int64_t ignore, float* __restrict__ up_down) {
    __shared__ float most[16];
    float mx = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += 1024)
        if (target[i] != ignore) mx = fmaxf(mx, fabsf(grad[i]));
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
    if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = mx;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, most[i]);
    int e = (int)((__float_as_uint(mx) >> 23) & 255u) - 127;  // mx in 2^e .. 2^(e+1)
    // nothing to scale, or nothing finite; and both factors stay normal
    const bool as_is = mx == 0.0f || e == 128;
    const float f = as_is ? 1.0f : fraction_of(mx);
    e = as_is ? 0 : 13 - e;
    e = e < -120 ? -120 : e > 120 ? 120 : e;
    up_down[0] = __uint_as_float((uint32_t)(127 + e) << 23) / f;
    up_down[1] = __uint_as_float((uint32_t)(127 - e) << 23) * f;
}

hipError_t launch_grad_scale(const float* grad, const int64_t* target, int64_t n, int64_t ignore, float* up_down,
                             hipStream_t s) {
    grad_scale_kernel<<<1, 1024, 0, s>>>(grad, target, n, ignore, up_down);
    return hipGetLastError();
}

int64_t logit_grad_parts(int tile, int64_t n) { return tile < 2 ? (n + 63) / 64 : (n + 31) / 32; }

template <typename T>
hipError_t launch_logit_grad(Mat h, Mat w, const T* bias, const int64_t* target, const float* lse, const float* grad,
                             const float* up, int64_t n, int64_t first, int64_t piece, int64_t classes, int64_t k,
                             int64_t ignore, T* out, int64_t ld, float* sums, int tile, const Only& only,
                             hipStream_t s) {
    const LogitGradEpi<T> e{bias ? bias + first : nullptr, target, lse, grad, up, out, sums, ld, ignore, (int32_t)first,
                            (int32_t)classes};
    const Mat wp{(const T*)w.p + first * w.ld, w.ld};
    return launch_gemm<T>(tile, wp, h, piece, n, k, 1, 0, only, e, s);
}

// ---------------------------------------------------------------------------
// few classes and few rows, long rows
// ---------------------------------------------------------------------------
// A dozen tiles would leave most CUs idle, and statistics need whole sums: the
// logits' contraction is split, and a second kernel joins its parts on the way to
// the loss or the gradient, as small a matrix as they are then.  76 x 344 by 3473
// in f32: 92 us in twelve tiles, 21 so; 64 x 1000 by 2048 48 and 18.
template <typename T>
struct LogitParts {
    const float* part;
    int splits;
    int64_t stride, ld;
    const T* bias;
    __device__ __forceinline__ f32x4 at(int64_t row, int64_t c, int64_t classes) const {
        const float* from = part + row * ld + c;
        f32x4 z = *reinterpret_cast<const f32x4*>(from);
        for (int s = 1; s < splits; ++s) z += *reinterpret_cast<const f32x4*>(from + s * stride);
        if (bias) z += load4(bias, c, classes);
        return z;
    }
};
template <typename T>
static LogitParts<T> logit_parts(const float* part, const Cut& cut, const T* bias, int64_t n, int64_t classes) {
    const int64_t ld = (classes + 3) & ~(int64_t)3;
    return LogitParts<T>{part, cut.splits, n * ld, ld, bias};
}

// A workgroup computes a row's loss, in two walks over its logits.
template <typename T>
__global__ __launch_bounds__(256) void xent_rows_kernel(LogitParts<T> z, const int64_t* __restrict__ target,
                                                        int64_t classes, int64_t ignore, float* __restrict__ loss,
                                                        float* __restrict__ lse) {
    __shared__ float join[4];
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float none = -__builtin_huge_valf();
    float mx = none;
    for (int64_t c = threadIdx.x * 4; c < classes; c += 1024) {
        const f32x4 v = z.at(row, c, classes);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < classes) mx = fmaxf(mx, v[e]);
    }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor(mx, s));
    if (lane == 0) join[wave] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(join[0], join[1]), fmaxf(join[2], join[3]));
    __syncthreads();
    // as in the tiles' statistics: a NaN logit reaches the sum
    const float base = mx == none ? 0.0f : mx;
    float sum = 0.0f;
    for (int64_t c = threadIdx.x * 4; c < classes; c += 1024) {
        const f32x4 v = z.at(row, c, classes);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < classes) sum += exp_fast(v[e] - base);
    }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) sum += __shfl_xor(sum, s);
    if (lane == 0) join[wave] = sum;
    __syncthreads();
    if (threadIdx.x != 0) return;
    const float l = base + logf((join[0] + join[1]) + (join[2] + join[3]));
    lse[row] = l;
    const int64_t t = target[row];
    float v = 0.0f;
    if (t != ignore) v = __builtin_nanf("");
    if (t != ignore && t >= 0 && t < classes) {
        const f32x4 q = z.at(row, t & ~(int64_t)3, classes);
        const int e = (int)(t & 3);
        v = l - (e == 0 ? q[0] : e == 1 ? q[1] : e == 2 ? q[2] : q[3]);
    }
    loss[row] = v;
}

// The gradient of the logits, as LogitGradEpi's; 256 columns and a run of rows to
// a workgroup, whose column sums are left as its part.
template <typename T>
__global__ __launch_bounds__(256) void logit_grad_rows_kernel(LogitParts<T> z, const int64_t* __restrict__ target,
                                                              const float* __restrict__ lse,
                                                              const float* __restrict__ grad,
                                                              const float* __restrict__ up, int64_t n, int64_t classes,
                                                              int64_t ignore, T* __restrict__ out, int64_t ld,
                                                              float* __restrict__ sums, int64_t rows_per) {
    __shared__ f32x4 join[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = ((int64_t)blockIdx.x * 64 + lane) * 4;
    const int64_t r0 = (int64_t)blockIdx.y * rows_per;
    const int64_t r1 = r0 + rows_per < n ? r0 + rows_per : n;
    const float scale = up ? up_factor<T>(up) : 1.0f;
    f32x4 sum = {};
    if (c < ld) {
        for (int64_t r = r0 + wave; r < r1; r += 4) {
            const int64_t t = target[r];
            const bool valid = t >= 0 && t < classes;
            const float l = lse[r], by = valid ? grad[r] * scale : __builtin_nanf("");
            typename Elem<T>::Vec4 v = {};
            if (t != ignore && c < classes) {
                const f32x4 q = z.at(r, c, classes);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = sizeof(T) == 2 ? __builtin_amdgcn_exp2f(__builtin_fmaf(q[e], kLog2E, -l * kLog2E))
                                                   : exp_fast(q[e] - l);
                    if (c + e < classes) v[e] = (T)((p - (t == c + e ? 1.0f : 0.0f)) * by);
                }
            }
            *reinterpret_cast<typename Elem<T>::Vec4*>(out + r * ld + c) = v;
            sum += widen(v);
        }
    }
    if (!sums) return;
    join[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && c < classes) {
#pragma unroll
        for (int i = 1; i < 4; ++i) sum += join[i][lane];
        store4(sums + (int64_t)blockIdx.y * classes, c, classes, sum);
    }
}

template <typename T>
hipError_t launch_xent_rows(const float* part, const Cut& cut, const T* bias, const int64_t* target, int64_t n,
                            int64_t classes, int64_t ignore, float* loss, float* lse, hipStream_t s) {
    if (!launchable(n, 256)) return hipErrorInvalidConfiguration;  // so many rows are no few tiles
    xent_rows_kernel<T><<<dim3((unsigned)n), 256, 0, s>>>(logit_parts(part, cut, bias, n, classes), target, classes,
                                                          ignore, loss, lse);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_logit_grad_rows(const float* part, const Cut& cut, const T* bias, const int64_t* target,
                                  const float* lse, const float* grad, const float* up, int64_t n, int64_t classes,
                                  int64_t ignore, T* out, int64_t ld, float* sums, int parts, hipStream_t s) {
    const int64_t rows_per = (n + parts - 1) / parts;
    logit_grad_rows_kernel<T><<<dim3((unsigned)((ld + 255) / 256), (unsigned)parts), 256, 0, s>>>(
        logit_parts(part, cut, bias, n, classes), target, lse, grad, up, n, classes, ignore, out, ld, sums, rows_per);
    return hipGetLastError();
}

#define MLRS_INST(T)                                                                                              \
    template hipError_t launch_xent_stats<T>(Mat, Mat, const T*, const int64_t*, int64_t, int64_t, int64_t, int,  \
                                             float*, float*, float*, const Only&, hipStream_t);                   \
    template hipError_t launch_logit_grad<T>(Mat, Mat, const T*, const int64_t*, const float*, const float*,      \
                                             const float*, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,  \
                                             T*, int64_t, float*, int, const Only&, hipStream_t);                 \
    template hipError_t launch_xent_rows<T>(const float*, const Cut&, const T*, const int64_t*, int64_t, int64_t, \
                                            int64_t, float*, float*, hipStream_t);                                \
    template hipError_t launch_logit_grad_rows<T>(const float*, const Cut&, const T*, const int64_t*,             \
                                                  const float*, const float*, const float*, int64_t, int64_t,     \
                                                  int64_t, T*, int64_t, float*, int, hipStream_t);
MLRS_INST(float)
MLRS_INST(_Float16)
MLRS_INST(__bf16)

}  // namespace train
}  // namespace mlrs
