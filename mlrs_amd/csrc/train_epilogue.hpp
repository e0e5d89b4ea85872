// What is done with a product's tile while it is in registers: the layer's
// bias, activation and residual; plain, scaled or accumulated stores; the
// softmax statistics of a tile of logits; the gradient of the logits.
#pragma once
#include "train_gemm.hpp"

namespace mlrs {
namespace train {

enum Activation { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4, kActCount = 5 };

constexpr float kLog2E = 1.44269504088896340736f;
constexpr float kGeluC = 0.79788456080286535588f;  // sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;

// e^x through the hardware's 2^x: x * log2(e) is rounded once, which costs
// |x| 2^-24 relative -- under 2^-20 wherever the result is not lost in a sum.
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * kLog2E); }

// the hardware's reciprocal is within one unit in the last place
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_fast(-x)); }

__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
    case kActRelu: return z > 0.0f ? z : (z != z ? z : 0.0f);
    case kActGelu: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752440f));
    // (1 + tanh u) / 2 = sigmoid(2 u); a product with a zero sigmoid is zero
    // only for finite z, as in the formula
    case kActGeluTanh: return z * sigmoid(2.0f * kGeluC * (z + kGeluB * z * z * z));
    case kActSilu: return z * sigmoid(z);
    default: return z;
    }
}

// d activate / dz
__device__ __forceinline__ float activate_slope(float z, int act) {
    switch (act) {
    case kActRelu: return z > 0.0f ? 1.0f : 0.0f;
    case kActGelu:
        return 0.5f * (1.0f + erff(z * 0.70710678118654752440f)) + z * (0.5f * kGeluC) * exp_fast(-0.5f * z * z);
    case kActGeluTanh: {
        const float s = sigmoid(2.0f * kGeluC * (z + kGeluB * z * z * z));
        return s + z * s * (1.0f - s) * 2.0f * kGeluC * (1.0f + 3.0f * kGeluB * z * z);
    }
    case kActSilu: {
        const float s = sigmoid(z);
        return s + z * s * (1.0f - s);
    }
    default: return 1.0f;
    }
}

// Four consecutive elements of a row from m on, those at or past `end` left
// out.  `wide`: the row's start and m are aligned for one access.
template <typename T>
__device__ __forceinline__ f32x4 load4(const T* row, int64_t m, int64_t end, bool wide) {
    f32x4 v;
    if (wide && m + 4 <= end) {
        const typename Elem<T>::Vec4 t = *reinterpret_cast<const typename Elem<T>::Vec4*>(row + m);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)t[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = m + e < end ? (float)row[m + e] : 0.0f;
    }
    return v;
}

template <typename T>
__device__ __forceinline__ void store4(T* row, int64_t m, int64_t end, bool wide, f32x4 v) {
    if (wide && m + 4 <= end) {
        typename Elem<T>::Vec4 t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = (T)v[e];
        *reinterpret_cast<typename Elem<T>::Vec4*>(row + m) = t;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (m + e < end) row[m + e] = (T)v[e];
    }
}

// Hands every element of the wave's part with m < m_end to f(n, m, v): four consecutive m of
// one n, the lanes along the row, so that a row leaves in whole lines.  The
// accumulators (a lane holds four m of one n, lanes run along n) are turned
// through the wave's own part of LDS, 32 rows at a time; a row's 16-byte
// chunks are kept at c ^ (n & 7).
template <int MB, int NB, typename F>
__device__ __forceinline__ void for_rows(const f32x16 (&acc)[MB][NB], const Place& p, char* lds, int32_t m_end,
                                         F f) {
    constexpr int kRow = MB * 128;                // bytes
    constexpr int kLanes = MB * 8;                // of a row
    constexpr int kStep = 64 / kLanes;            // rows per access
    char* mine = lds + p.wave * 32 * kRow;
    const int h = p.lane >> 5, r = p.lane & 31;
    __syncthreads();  // the tiles in LDS are no longer read
#pragma unroll
    for (int j = 0; j < NB; ++j) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e];
                *reinterpret_cast<f32x4*>(mine + r * kRow + (((8 * i + 2 * q + h) ^ (r & 7)) << 4)) = v;
            }
        // the wave's LDS accesses are in order; nothing else touches `mine`
        __builtin_amdgcn_wave_barrier();
        const int c = p.lane % kLanes;
#pragma unroll 1
        for (int t = 0; t < 32; t += kStep) {
            const int row = t + p.lane / kLanes;
            const f32x4 v = *reinterpret_cast<const f32x4*>(mine + row * kRow + ((c ^ (row & 7)) << 4));
            const int32_t n = p.n0 + j * 32 + row, m = p.m0 + 4 * c;
            if (n < p.n && m < m_end) f(n, m, v);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// y = act(P + bias) + residual, and z = P + bias where it is kept.
template <typename T>
struct LinearEpi {
    const T* bias;
    const T* residual;
    T* y;
    T* z;
    int64_t ld;  // of residual, y and z
    int32_t act;
    bool wide;

    __device__ __forceinline__ void point(int64_t n, int64_t m, int64_t end, f32x4 v) const {
        if (bias) v += load4(bias, m, end, false);
        if (z) store4(z + n * ld, m, end, wide, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = activate(v[e], act);
        if (residual) v += load4(residual + n * ld, m, end, wide);
        store4(y + n * ld, m, end, wide, v);
    }
    template <int WM, int WN, int MB, int NB>
    __device__ __forceinline__ void run(f32x16 (&acc)[MB][NB], const Place& p, char* lds) const {
        for_rows(acc, p, lds, p.m, [&](int32_t n, int32_t m, f32x4 v) { point(n, m, p.m, v); });
    }
};

// out = alpha * (P + add), rounded to out's type; or the parts of a split
// contraction, or a running sum, in f32.
template <typename T>
struct StoreEpi {
    T* out;              // null: `part` is written instead
    float* part;         // + split * part_stride
    const float* add;    // may be null
    const float* alpha;  // device scalar; may be null
    int64_t ld, part_ld, part_stride;
    bool wide;

    __device__ __forceinline__ void finish(int64_t n, int64_t m, int64_t end, f32x4 v) const {
        if (add) v += load4(add + n * part_ld, m, end, true);
        if (alpha) v *= *alpha;
        store4(out + n * ld, m, end, wide, v);
    }
    template <int WM, int WN, int MB, int NB>
    __device__ __forceinline__ void run(f32x16 (&acc)[MB][NB], const Place& p, char* lds) const {
        if (out) {
            for_rows(acc, p, lds, p.m, [&](int32_t n, int32_t m, f32x4 v) { finish(n, m, p.m, v); });
        } else {
            float* to = part + p.split * part_stride;
            for_rows(acc, p, lds, p.m, [&](int32_t n, int32_t m, f32x4 v) {
                if (add) v += load4(add + n * part_ld, m, p.m, true);
                store4(to + n * part_ld, m, p.m, true, v);  // part_ld is a multiple of 4
            });
        }
    }
};

// The statistics of a tile of logits z = P + bias (rows: classes, columns:
// rows of the batch): the largest and the sum of e^(z - largest) over the
// wave's classes, and the target's logit from the wave that has it.  Classes
// whose logit is -inf add nothing, also where that is all of them.
template <typename T>
struct StatsEpi {
    const T* bias;
    const int64_t* target;
    float* top;      // parts x n
    float* total;    // parts x n
    float* hit;      // n

    template <int WM, int WN, int MB, int NB>
    __device__ __forceinline__ void run(f32x16 (&acc)[MB][NB], const Place& p, char*) const {
        const int h = p.lane >> 5, r = p.lane & 31;
        const int64_t at = ((int64_t)p.tile_m * WM + p.wm) * p.n;
        if (bias) {
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 bv = load4(bias, p.m0 + i * 32 + 8 * q + 4 * h, p.m, false);
#pragma unroll
                    for (int j = 0; j < NB; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] += bv[e];
                }
        }
        const float none = -__builtin_huge_valf();
        if (p.m0 + MB * 32 > p.m) {  // classes past the end
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int q = 0; q < 16; ++q)
                    if (p.m0 + i * 32 + 8 * (q >> 2) + 4 * h + (q & 3) >= p.m)
#pragma unroll
                        for (int j = 0; j < NB; ++j) acc[i][j][q] = none;
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int32_t n = p.n0 + j * 32 + r;
            float mx = none;
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int q = 0; q < 16; ++q) mx = fmaxf(mx, acc[i][j][q]);
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            // the sum is relative to a finite value where there is one to be
            // had: a NaN logit reaches it, and +inf - +inf is NaN
            const float base = mx == none ? 0.0f : mx;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int q = 0; q < 16; ++q) sum += exp_fast(acc[i][j][q] - base);
            sum += __shfl_xor(sum, 32);
            if (n < p.n) {
                if (h == 0) {
                    top[at + n] = mx;
                    total[at + n] = sum;
                }
                const int64_t t = target[n] - p.m0;
                if (t >= 0 && t < MB * 32 && t < p.m - p.m0) {
                    float v = 0.0f;
                    bool found = false;
#pragma unroll
                    for (int i = 0; i < MB; ++i)
#pragma unroll
                        for (int q = 0; q < 16; ++q)
                            if (t == i * 32 + 8 * (q >> 2) + 4 * h + (q & 3)) {
                                v = acc[i][j][q];
                                found = true;
                            }
                    if (found) hit[n] = v;
                }
            }
        }
    }
};

// The gradient of the logits: (e^(z - lse) - [class is the target]) * grad,
// zero in ignored rows, NaN in rows whose target is no class.  Rounded to the
// operands' type, as it goes into two matrix products with them: the products
// still add in f32, and a 16-bit gradient's own rounding is of the same size.
// `up` scales it by a power of two first (f16: the gradients of a mean over a
// batch times the probabilities of a large vocabulary lie below f16's range).
template <typename T>
struct LogitGradEpi {
    const T* bias;
    const int64_t* target;
    const float* lse;
    const float* grad;
    const float* up;  // device scalar; may be null
    T* out;
    int64_t ld;
    int64_t ignore;
    int32_t first;    // the piece's first class
    int32_t classes;  // of the whole vocabulary

    template <int WM, int WN, int MB, int NB>
    __device__ __forceinline__ void run(f32x16 (&acc)[MB][NB], const Place& p, char* lds) const {
        const float scale = up ? *up : 1.0f;
        for_rows(acc, p, lds, (int32_t)ld, [&](int32_t n, int32_t m, f32x4 v) {
            const int64_t t = target[n];
            const bool kept = t != ignore;
            float g = grad[n] * scale;
            if (t < 0 || t >= classes) g = __builtin_nanf("");
            const float l = lse[n];
            if (bias) v += load4(bias, m, p.m, false);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = exp_fast(v[e] - l);
                if (t == first + m + e) x -= 1.0f;
                v[e] = kept ? x * g : 0.0f;
            }
            // the columns up to ld, a multiple of 16 bytes, are read by the
            // products and must be zero
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (m + e >= p.m) v[e] = 0.0f;
            store4(out + (int64_t)n * ld, m, ld, true, v);
        });
    }
};

}  // namespace train
}  // namespace mlrs
