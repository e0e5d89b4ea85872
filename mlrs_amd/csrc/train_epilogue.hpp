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

// The normal distribution function, and e^(-z^2/2) in `bell`.  For u = |z|,
// Phi(-u) = erfc(u / sqrt 2) / 2 = e^(-u^2/2) q(1 / (1 + 0.36 u)) / 2 with a
// polynomial q of degree 9 without constant term, fitted to the scaled
// complementary error function for u in 0 .. 40 by iteratively reweighted
// least squares: its largest relative error there is 9.0e-8.
__device__ __forceinline__ float normal_cdf(float z, float& bell) {
    const float u = fabsf(z);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.36f, u, 1.0f));
    float q = -0.06048248215007038f;
    q = __builtin_fmaf(q, t, 0.27904132186964825f);
    q = __builtin_fmaf(q, t, -0.44724105480219f);
    q = __builtin_fmaf(q, t, 0.21477676823808028f);
    q = __builtin_fmaf(q, t, -0.0007932018218880397f);
    q = __builtin_fmaf(q, t, 0.19208110241674273f);
    q = __builtin_fmaf(q, t, 0.2480183825361184f);
    q = __builtin_fmaf(q, t, 0.28736386334573727f);
    q = __builtin_fmaf(q, t, 0.2872353260570751f);
    bell = exp_fast(-0.5f * z * z);
    const float below = 0.5f * (q * t) * bell;
    return z < 0.0f ? below : 1.0f - below;
}

__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
    case kActRelu: return z > 0.0f ? z : (z != z ? z : 0.0f);
    case kActGelu: {
        float bell;
        return z * normal_cdf(z, bell);
    }
    // (1 + tanh u) / 2 = sigmoid(2 u); a product with a zero sigmoid is zero
    // only for finite z, as in the formula
    case kActGeluTanh: return z * sigmoid(2.0f * kGeluC * (z + kGeluB * z * z * z));
    case kActSilu: return z * sigmoid(z);
    default: return z;
    }
}

// The same over a group: one switch for all of it.
template <int N>
__device__ __forceinline__ void activate_all(f32x4 (&v)[N], int act) {
    auto each = [&](auto f) {
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[u][e] = f(v[u][e]);
    };
    switch (act) {
    case kActRelu: each([](float z) { return activate(z, kActRelu); }); break;
    case kActGelu: each([](float z) { return activate(z, kActGelu); }); break;
    case kActGeluTanh: each([](float z) { return activate(z, kActGeluTanh); }); break;
    case kActSilu: each([](float z) { return activate(z, kActSilu); }); break;
    default: break;
    }
}

// d activate / dz
__device__ __forceinline__ float activate_slope(float z, int act) {
    switch (act) {
    case kActRelu: return z > 0.0f ? 1.0f : 0.0f;
    case kActGelu: {
        float bell;
        const float cdf = normal_cdf(z, bell);
        return cdf + z * (0.5f * kGeluC) * bell;
    }
    case kActGeluTanh: {
        // from |z| = 16 on s is 0 or 1, and z^2 may leave f32's range
        const float s = sigmoid(2.0f * kGeluC * (z + kGeluB * z * z * z));
        return s + z * s * (1.0f - s) * 2.0f * kGeluC * (1.0f + 3.0f * kGeluB * fminf(z * z, 256.0f));
    }
    case kActSilu: {
        const float s = sigmoid(z);
        return s + z * s * (1.0f - s);
    }
    default: return 1.0f;
    }
}

// A 16-bit gradient of the logits is rounded before its products.  The rows of a
// mean share one gradient, 1 / n, and where the other classes' shares are small the
// target's element is nearly that in every row: its rounding error, up to 2^-8 of
// bf16's, would be common to all and show in the results as it is.  So the
// gradients are divided by the fraction of one of them (1 <= f < 2), which puts such
// elements just below a power of two, where a rounding error is 2^-9 at most and
// goes by each row's probability; the products and the sums are multiplied by it.
// bf16 takes the first row's gradient's; f16 a factor from memory that also lifts
// the gradients into the type's range.
__device__ __forceinline__ float fraction_of(float x) {
    return __uint_as_float((__float_as_uint(x) & 0x7FFFFFu) | 0x3F800000u);  // in [1, 2), whatever x is
}
template <typename T>
__device__ __forceinline__ float up_factor(const float* p) {
    return __is_same(T, __bf16) ? 1.0f / fraction_of(*p) : *p;
}
template <typename T>
__device__ __forceinline__ float down_factor(const float* p) {
    return __is_same(T, __bf16) ? fraction_of(*p) : *p;
}

// Four consecutive elements of a row from m on, those at or past `end` left
// out.  Global accesses need no more than their elements' alignment, so rows of
// any length are read and written four elements at a time.
template <typename T>
__device__ __forceinline__ typename Elem<T>::Vec4 load_raw4(const T* row, int64_t m, int64_t end) {
    typename Elem<T>::Vec4 v;
    if (m + 4 <= end) {
        __builtin_memcpy(&v, row + m, sizeof v);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = m + e < end ? row[m + e] : (T)0.0f;
    }
    return v;
}

template <typename V>
__device__ __forceinline__ f32x4 widen(V v) {
    return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}

template <typename T>
__device__ __forceinline__ f32x4 load4(const T* row, int64_t m, int64_t end) {
    return widen(load_raw4(row, m, end));
}

template <typename T>
__device__ __forceinline__ void store4(T* row, int64_t m, int64_t end, f32x4 v) {
    if (m + 4 <= end) {
        typename Elem<T>::Vec4 t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = (T)v[e];
        __builtin_memcpy(row + m, &t, sizeof t);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (m + e < end) row[m + e] = (T)v[e];
    }
}

// Hands the wave's part with m < m_end to f(n, m, v, with) in groups: v[u] holds
// four consecutive m of row n + u * step (which may be past the last row), the
// lanes along the row, so that a row leaves in whole lines; a lane's m is the
// same in every call.  `with` is what load(n, m, with) read for the same rows, a
// group ahead: a group's loads are under way at once and while the group before
// is worked on (a residual of 16384 x 4096 bf16 beside a product costs 75 us when
// a group loads its own, 26 so).  The accumulators (a lane holds four m of one n,
// sixteen lanes run along n) are turned through the wave's own part of LDS, 32
// rows at a time.
template <int MB>
constexpr int row_step() {
    return 64 / (MB * 4);  // rows that the lanes cover together
}
template <int MB>
constexpr int row_group() {
    return MB == 2 ? 4 : 8;
}
// Rows of BYTES bytes in LDS: piece c (16 bytes) of row r lies at c ^ this, and
// sixteen rows read or written at one c touch all banks.
template <int BYTES>
__device__ __forceinline__ int turn_swizzle(int r) {
    return BYTES >= 256 ? r & 15 : BYTES == 128 ? (r >> 1) & 7 : (r >> 2) & 3;
}
template <typename With, int MB, int NB, typename L, typename F>
__device__ __forceinline__ void for_rows(const f32x4 (&acc)[MB][NB], const Place& p, char* lds, int32_t m_end, L load,
                                         F f) {
    constexpr int kRow = MB * 64;       // bytes
    constexpr int kLanes = MB * 4;      // of a row
    constexpr int kStep = row_step<MB>(), kGroup = row_group<MB>(), kRows = kStep * kGroup;
    char* mine = lds + p.wave * 32 * kRow;
    const int g = p.lane >> 4, r = p.lane & 15;
    const int c = p.lane % kLanes;
    const int32_t m = p.m0 + 4 * c, n_first = p.n0 + p.lane / kLanes;
    With with[kGroup], next[kGroup];
    if (n_first < p.n && m < m_end) load(n_first, m, with);
    __syncthreads();  // the panels in LDS are no longer read
#pragma unroll
    for (int j = 0; j < NB; j += 2) {
#pragma unroll
        for (int jj = 0; jj < 2; ++jj)
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const int row = 16 * jj + r;
                *reinterpret_cast<f32x4*>(mine + row * kRow + (((4 * i + g) ^ turn_swizzle<kRow>(row)) << 4)) =
                    acc[i][j + jj];
            }
        // the wave's LDS accesses are in order; nothing else touches `mine`
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int t = 0; t < 32; t += kRows) {
            const int32_t n = n_first + j * 16 + t;
            if (j * 16 + t + kRows < NB * 16 && n + kRows < p.n && m < m_end) load(n + kRows, m, next);
            f32x4 v[kGroup];
#pragma unroll
            for (int u = 0; u < kGroup; ++u) {
                const int row = t + u * kStep + p.lane / kLanes;
                v[u] = *reinterpret_cast<const f32x4*>(mine + row * kRow + ((c ^ turn_swizzle<kRow>(row)) << 4));
            }
            if (n < p.n && m < m_end) f(n, m, v, with);
#pragma unroll
            for (int u = 0; u < kGroup; ++u) with[u] = next[u];
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

    typedef typename Elem<T>::Vec4 Vec4;
    // rows n, n + step, ... of them those before n_end
    template <int N>
    __device__ __forceinline__ void load(int64_t n, int64_t step, int64_t n_end, int64_t m, int64_t end,
                                         Vec4 (&res)[N]) const {
        if (!residual) return;
#pragma unroll
        for (int u = 0; u < N; ++u)
            if (n + u * step < n_end) res[u] = load_raw4(residual + (n + u * step) * ld, m, end);
    }
    template <int N>
    __device__ __forceinline__ void rows(int64_t n, int64_t step, int64_t n_end, int64_t m, int64_t end, f32x4 bv,
                                         f32x4 (&v)[N], const Vec4 (&res)[N]) const {
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] += bv;
        if (z) {
#pragma unroll
            for (int u = 0; u < N; ++u)
                if (n + u * step < n_end) store4(z + (n + u * step) * ld, m, end, v[u]);
        }
        activate_all(v, act);
        if (residual) {
#pragma unroll
            for (int u = 0; u < N; ++u) v[u] += widen(res[u]);
        }
#pragma unroll
        for (int u = 0; u < N; ++u)
            if (n + u * step < n_end) store4(y + (n + u * step) * ld, m, end, v[u]);
    }
    // one group of four elements
    __device__ __forceinline__ void point(int64_t n, int64_t m, int64_t end, f32x4 v) const {
        f32x4 one[1] = {v};
        Vec4 res[1] = {};
        load(n, 0, n + 1, m, end, res);
        rows(n, 0, n + 1, m, end, bias_at(m, end), one, res);
    }
    __device__ __forceinline__ f32x4 bias_at(int64_t m, int64_t end) const {
        f32x4 bv = {};
        if (bias && m < end) bv = load4(bias, m, end);
        return bv;
    }
    template <int WM, int WN, int MB, int NB>
    __device__ __forceinline__ void run(f32x4 (&acc)[MB][NB], const Place& p, char* lds) const {
        const f32x4 bv = bias_at(p.m0 + 4 * (p.lane % (MB * 4)), p.m);
        constexpr int kGroup = row_group<MB>(), kStep = row_step<MB>();
        for_rows<Vec4>(
            acc, p, lds, p.m,
            [&](int32_t n, int32_t m, Vec4 (&res)[kGroup]) { load(n, kStep, p.n, m, p.m, res); },
            [&](int32_t n, int32_t m, f32x4 (&v)[kGroup], const Vec4 (&res)[kGroup]) {
                rows(n, kStep, p.n, m, p.m, bv, v, res);
            });
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

    template <int N>
    __device__ __forceinline__ void load(int64_t n, int64_t step, int64_t n_end, int64_t m, int64_t end,
                                         f32x4 (&old)[N]) const {
        if (!add) return;
#pragma unroll
        for (int u = 0; u < N; ++u)
            if (n + u * step < n_end) old[u] = load4(add + (n + u * step) * part_ld, m, end);
    }
    template <int N>
    __device__ __forceinline__ void rows(int64_t n, int64_t step, int64_t n_end, int64_t m, int64_t end, int split,
                                         f32x4 (&v)[N], const f32x4 (&old)[N]) const {
        if (add) {
#pragma unroll
            for (int u = 0; u < N; ++u) v[u] += old[u];
        }
        if (out) {
            const float by = alpha ? down_factor<T>(alpha) : 1.0f;
#pragma unroll
            for (int u = 0; u < N; ++u)
                if (n + u * step < n_end) store4(out + (n + u * step) * ld, m, end, v[u] * by);
        } else {
            float* to = part + split * part_stride;  // part_ld is a multiple of 4
#pragma unroll
            for (int u = 0; u < N; ++u)
                if (n + u * step < n_end) store4(to + (n + u * step) * part_ld, m, end, v[u]);
        }
    }
    __device__ __forceinline__ void point(int64_t n, int64_t m, int64_t end, f32x4 v) const {
        f32x4 one[1] = {v}, old[1] = {};
        load(n, 0, n + 1, m, end, old);
        rows(n, 0, n + 1, m, end, 0, one, old);
    }
    template <int WM, int WN, int MB, int NB>
    __device__ __forceinline__ void run(f32x4 (&acc)[MB][NB], const Place& p, char* lds) const {
        constexpr int kGroup = row_group<MB>(), kStep = row_step<MB>();
        for_rows<f32x4>(
            acc, p, lds, p.m,
            [&](int32_t n, int32_t m, f32x4 (&old)[kGroup]) { load(n, kStep, p.n, m, p.m, old); },
            [&](int32_t n, int32_t m, f32x4 (&v)[kGroup], const f32x4 (&old)[kGroup]) {
                rows(n, kStep, p.n, m, p.m, p.split, v, old);
            });
    }
};

// acc += bias, along m.
template <typename T, int MB, int NB>
__device__ __forceinline__ void add_bias(f32x4 (&acc)[MB][NB], const T* bias, const Place& p) {
    if (!bias) return;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const int32_t m = p.m0 + i * 16 + 4 * (p.lane >> 4);
        const f32x4 bv = m < p.m ? load4(bias, m, p.m) : f32x4{};
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] += bv;
    }
}

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
    __device__ __forceinline__ void run(f32x4 (&acc)[MB][NB], const Place& p, char*) const {
        const int g = p.lane >> 4, r = p.lane & 15;
        const int64_t at = ((int64_t)p.tile_m * WM + p.wm) * p.n;
        add_bias(acc, bias, p);
        const float none = -__builtin_huge_valf();
        if (p.m0 + MB * 16 > p.m) {  // classes past the end
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (p.m0 + i * 16 + 4 * g + e >= p.m)
#pragma unroll
                        for (int j = 0; j < NB; ++j) acc[i][j][e] = none;
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int32_t n = p.n0 + j * 16 + r;
            float mx = none;
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, acc[i][j][e]);
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            // the sum is relative to a finite value where there is one to be
            // had: a NaN logit reaches it, and +inf - +inf is NaN
            const float base = mx == none ? 0.0f : mx;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += exp_fast(acc[i][j][e] - base);
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (n < p.n) {
                if (g == 0) {
                    top[at + n] = mx;
                    total[at + n] = sum;
                }
                const int64_t t = target[n] - p.m0;
                if (t >= 0 && t < MB * 16 && t < p.m - p.m0) {
                    const int32_t place = (int32_t)t;
                    if (((place >> 2) & 3) == g) {  // this lane has it
                        float v = 0.0f;
#pragma unroll
                        for (int i = 0; i < MB; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) v = place == i * 16 + 4 * g + e ? acc[i][j][e] : v;
                        hit[n] = v;
                    }
                }
            }
        }
    }
};

// The gradient of the logits: (e^(z - lse) - [class is the target]) * grad,
// zero in ignored rows, NaN in rows whose target is no class.  Rounded to the
// operands' type, as it goes into two matrix products with them: the products
// still add in f32, and a 16-bit gradient's own rounding is of the same size.
// The column sums add up the rounded elements, as they leave LDS in lines (within
// 2.7e-4 of the sums of unrounded ones in f16, as the products are).
// `up` scales it first (f16: the gradients of a mean over a batch times the
// probabilities of a large vocabulary lie below f16's range).
template <typename T>
struct LogitGradEpi {
    const T* bias;
    const int64_t* target;
    const float* lse;
    const float* grad;
    const float* up;  // device scalar; may be null
    T* out;
    float* sums;  // null, or the column sums of every wave's rows, piece by piece of NB * 16 rows
    int64_t ld;
    int64_t ignore;
    int32_t first;    // the piece's first class
    int32_t classes;  // of the whole vocabulary

    // A lane's accumulators belong to one row of the batch for each block of
    // columns, so the row's target, lse and gradient are three registers; the
    // result is turned through LDS in its own type, and leaves in 16-byte pieces.
    template <int WM, int WN, int MB, int NB>
    __device__ __forceinline__ void run(f32x4 (&acc)[MB][NB], const Place& p, char* lds) const {
        constexpr int kEach = 16 / (int)sizeof(T);      // elements of a piece
        constexpr int kRow = MB * 16 * (int)sizeof(T);  // bytes of a row
        constexpr int kPieces = kRow / 16;
        constexpr int kStep = 64 / kPieces;             // rows that the lanes cover together
        const int g = p.lane >> 4, r = p.lane & 15;
        const float scale = up ? up_factor<T>(up) : 1.0f;
        float l[NB], by[NB];
        int32_t hot[NB];    // the target's place among the wave's classes
        uint32_t keep[NB];  // all ones, or none in an ignored row
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int32_t n = p.n0 + j * 16 + r;
            const int32_t at = n < p.n ? n : p.n - 1;
            const int64_t t = target[at];
            const bool valid = t >= 0 && t < classes;
            l[j] = sizeof(T) == 2 ? lse[at] * kLog2E : lse[at];
            keep[j] = t != ignore ? 0xFFFFFFFFu : 0u;
            by[j] = valid ? grad[at] * scale : __builtin_nanf("");
            hot[j] = valid ? (int32_t)t - first - p.m0 : -1;
        }
        add_bias(acc, bias, p);
        // Three vector operations and an exponential for an element where no
        // lane holds its row's target and the wave's classes are whole (the
        // rest of a piece): vector work is what this epilogue costs.  16-bit
        // types fold the subtraction into the multiplication by log2(e), which
        // costs |lse| 2^-24 of a probability that is then rounded to 2^-8 or 2^-11.
        auto element = [&](int i, int j, int e) {
            const float z = acc[i][j][e];
            return sizeof(T) == 2 ? __builtin_amdgcn_exp2f(__builtin_fmaf(z, kLog2E, -l[j])) : exp_fast(z - l[j]);
        };
        auto mask = [&](typename Elem<T>::Vec4 v, uint32_t by_row) {
            typedef uint32_t Words __attribute__((ext_vector_type(sizeof(T))));
            Words w = __builtin_bit_cast(Words, v);
            w &= by_row;
            return __builtin_bit_cast(typename Elem<T>::Vec4, w);
        };
        char* mine = lds + p.wave * 32 * kRow;
        float col[kEach] = {};
        __syncthreads();  // the panels in LDS are no longer read
#pragma unroll
        for (int j0 = 0; j0 < NB; j0 += 2) {
            auto place = [&](int i, int jj) {
                const int row = 16 * jj + r, at = (i * 16 + 4 * g) * (int)sizeof(T);
                return reinterpret_cast<typename Elem<T>::Vec4*>(
                    mine + row * kRow + (((at >> 4) ^ turn_swizzle<kRow>(row)) << 4) + (at & 15));
            };
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) {
                const int j = j0 + jj;
                const bool odd = p.m0 + MB * 16 > p.m || __any(hot[j] >= 0 && hot[j] < MB * 16);
                if (!odd) {
#pragma unroll
                    for (int i = 0; i < MB; ++i) {
                        typename Elem<T>::Vec4 v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = (T)(element(i, j, e) * by[j]);
                        *place(i, jj) = mask(v, keep[j]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < MB; ++i) {
                        const int32_t m = i * 16 + 4 * g;  // of the wave's classes
                        typename Elem<T>::Vec4 v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = element(i, j, e) - (hot[j] == m + e ? 1.0f : 0.0f);
                            // the columns up to ld, a multiple of 16 bytes, are
                            // read by the products and must be zero
                            v[e] = (T)(p.m0 + m + e < p.m ? x * by[j] : 0.0f);
                        }
                        *place(i, jj) = mask(v, keep[j]);
                    }
                }
            }
            // the wave's LDS accesses are in order; nothing else touches `mine`
            __builtin_amdgcn_wave_barrier();
            const int c = p.lane % kPieces;
#pragma unroll
            for (int t = 0; t < 32; t += kStep) {
                const int row = t + p.lane / kPieces;
                const typename Elem<T>::Frag v = *reinterpret_cast<const typename Elem<T>::Frag*>(
                    mine + row * kRow + ((c ^ turn_swizzle<kRow>(row)) << 4));
                const int32_t n = p.n0 + j0 * 16 + row, m = p.m0 + kEach * c;
                if (n < p.n && m < ld) {
                    *reinterpret_cast<typename Elem<T>::Frag*>(out + (int64_t)n * ld + m) = v;
                    if (sums) {
#pragma unroll
                        for (int e = 0; e < kEach; ++e) col[e] += (float)v[e];
                    }
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
        if (!sums || p.n0 >= p.n) return;
#pragma unroll
        for (int s = kPieces; s < 64; s <<= 1)
#pragma unroll
            for (int e = 0; e < kEach; ++e) col[e] += __shfl_xor(col[e], s);
        if (p.lane >= kPieces) return;
#pragma unroll
        for (int e = 0; e < kEach; e += 4)
            store4(sums + (int64_t)(p.n0 / (NB * 16)) * p.m, p.m0 + kEach * p.lane + e, p.m,
                   f32x4{col[e], col[e + 1], col[e + 2], col[e + 3]});
    }
};

}  // namespace train
}  // namespace mlrs
