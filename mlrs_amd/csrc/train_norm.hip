// Group norm with an activation and dropout, channels last, and its gradient.
//
// x is n samples of s positions of c channels, in g groups of d = c / g adjacent
// channels.  With mean and variance over the s d elements of a sample's group,
// rstd = 1 / sqrt(var + eps), xh = (x - mean) rstd and z = xh w + b:
//   y = drop(act(z)).
// Backwards, with dz = drop(dy) act'(z) and t = dz w: db = sum dz and dw = sum dz xh
// over samples and positions, dx = rstd (t - (sum t + xh sum t xh) / (s d)), the
// sums over the sample's group.
//
// Few operations for each byte: the elements are read once and kept in registers
// between the sums and what needs them, but where a group is too large for that.
// What bounds it is memory only without an activation; with one it is the vector
// instructions, 26 an element forwards with silu and 48 backwards.  Three ways:
//   rows      s = 1: a group is d adjacent elements, which some lanes of a wave, or
//             a workgroup, hold.  16384 x 2048 bf16 in 16 groups, gelu, dropout: 45 us
//             (3.0 TB/s), backwards 63 (3.2).
//   resident  a workgroup holds a slab, some whole groups of a sample: a thread has
//             eight adjacent channels at every so-manieth position.  16 x 1024 x 640
//             bf16 in 32 groups, silu: 17 us (2.4 TB/s), backwards 32 (2.0).
//   split     groups past that: partial sums of runs of positions, then a second
//             pass over the elements; it reads the sums first, so that it is the
//             second launch of two.  16 x 4096 x 320 f16 in 32 groups, silu: 15 and
//             21 us, bf16 as long, f32 53 together, backwards 55 and 88; the second
//             pass finds its elements in the last cache.
// The parameters' gradients are added up per thread while its channels stay the
// same over samples and positions; a last launch adds those in order.
#include <algorithm>
#include <cmath>

#include "train_epilogue.hpp"
#include "train_random.hpp"

namespace mlrs {
namespace train {

namespace {

template <typename T>
struct NormOperands {
    const T *x, *w, *b;  // w and b may be null
    const T* dy;         // backwards
    T* y;                // or dx
    float *mean, *rstd;  // n x g; forwards may be null
    float *pw, *pb;      // the parameters' partial sums (rows x c); may be null
    int64_t n, s, c, g, d;
    float eps;
    int act;
    bool aligned;  // every thread's eight channels are whole and one block of random bits
    Drop drop;
};

// ---------------------------------------------------------------------------
// what is done with an element
// ---------------------------------------------------------------------------
// gelu is z Phi(z) = max(z, 0) - |z| Phi(-|z|), and Phi(-u) = e^(-u^2/2) q(t) with t =
// 1 / (1 + 0.36 u), as train_epilogue.hpp's: a polynomial of degree 9 fitted to the
// scaled complementary error function for u in 0 .. 40, relative error 3.8e-7 as it is
// computed: a layer's gelu is as exact with a norm as without, in every type.  (Degree 6,
// relative error 1.1e-5, saves 3 us of 106 of 16384 x 2048 bf16 there and back, but
// rounds 65 of 38400 f16 slopes to the wrong side.)
__device__ __forceinline__ float normal_tail(float u, float& bell) {
    bell = __builtin_amdgcn_exp2f(u * u * (-0.5f * kLog2E));
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.36f, u, 1.0f));
    float q = -0.030237516661021768f;
    q = __builtin_fmaf(q, t, 0.13950534889597813f);
    q = __builtin_fmaf(q, t, -0.22359445728159374f);
    q = __builtin_fmaf(q, t, 0.10736457851476656f);
    q = __builtin_fmaf(q, t, -0.00038397830051628453f);
    q = __builtin_fmaf(q, t, 0.09603661840218482f);
    q = __builtin_fmaf(q, t, 0.1240098852248856f);
    q = __builtin_fmaf(q, t, 0.14368186910198438f);
    q = __builtin_fmaf(q, t, 0.14361766520603944f);
    return q * t * bell;
}

template <int ACT>
__device__ __forceinline__ float value_of(float z) {
    if constexpr (ACT == kActGelu) {
        float bell;
        const float u = __builtin_elementwise_minimum(fabsf(z), 1e18f);  // these two keep a NaN
        const float tail = normal_tail(u, bell);
        return __builtin_fmaf(-u, tail, __builtin_elementwise_maximum(z, 0.0f));
    } else {
        return activate(z, ACT);
    }
}
template <int ACT>
__device__ __forceinline__ float slope_of(float z) {
    if constexpr (ACT == kActGelu) {
        float bell;
        const float tail = normal_tail(__builtin_elementwise_minimum(fabsf(z), 1e18f), bell);
        const float cdf = 0.5f + __builtin_copysignf(0.5f - tail, z);
        return __builtin_fmaf(z * (0.5f * kGeluC), bell, cdf);
    } else {
        return activate_slope(z, ACT);
    }
}

// One switch for eight elements: v = value(z), or v *= slope(z).
__device__ __forceinline__ void values_of(int act, float (&v)[8]) {
    auto each = [&](auto f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = f(v[e]);
    };
    switch (act) {
    case kActRelu: each([](float z) { return value_of<kActRelu>(z); }); break;
    case kActGelu: each([](float z) { return value_of<kActGelu>(z); }); break;
    case kActGeluTanh: each([](float z) { return value_of<kActGeluTanh>(z); }); break;
    case kActSilu: each([](float z) { return value_of<kActSilu>(z); }); break;
    default: break;
    }
}
__device__ __forceinline__ void times_slopes(int act, const float (&xh)[8], const float (&w)[8], const float (&b)[8],
                                             float (&v)[8]) {
    auto each = [&](auto f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= f(__builtin_fmaf(xh[e], w[e], b[e]));
    };
    switch (act) {
    case kActRelu: each([](float z) { return slope_of<kActRelu>(z); }); break;
    case kActGelu: each([](float z) { return slope_of<kActGelu>(z); }); break;
    case kActGeluTanh: each([](float z) { return slope_of<kActGeluTanh>(z); }); break;
    case kActSilu: each([](float z) { return slope_of<kActSilu>(z); }); break;
    default: break;
    }
}

// y of eight elements from their xh.
template <typename T>
__device__ __forceinline__ void forward_oct(const NormOperands<T>& a, uint64_t offset, int64_t i, const float (&w)[8],
                                            const float (&b)[8], float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(v[e], w[e], b[e]);
    values_of(a.act, v);
    if (a.drop.threshold) drop_oct(a.drop, offset, i, a.aligned, v);
}

// dz of eight elements: dy becomes it.
template <typename T>
__device__ __forceinline__ void backward_oct(const NormOperands<T>& a, uint64_t offset, int64_t i,
                                             const float (&w)[8], const float (&b)[8], const float (&xh)[8],
                                             float (&dy)[8]) {
    if (a.drop.threshold) drop_oct(a.drop, offset, i, a.aligned, dy);
    times_slopes(a.act, xh, w, b, dy);
}

// 1 / sqrt(v): the hardware's, to one unit, and a step of Newton's.
__device__ __forceinline__ float inverse_root(float v) {
    const float y = __builtin_amdgcn_rsqf(v);
    const float better = y * __builtin_fmaf(-0.5f * v * y, y, 1.5f);
    return y < 1e18f && y > 1e-18f ? better : y;  // v y is out of range beyond, or v 0 or infinite
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_huge_valf(); }
// Squares about a place, less what that place is off their mean: not negative, whatever
// is rounded; infinite where they are past f32's range, and NaN where they are.
__device__ __forceinline__ float squares_less(float squares, float less) {
    return __builtin_elementwise_maximum(squares - (finite(less) ? less : 0.0f), 0.0f);
}
// sum / count, by its reciprocal and a step: the quotient rounded, so that the mean of
// equal elements is theirs where their sum is exact.
__device__ __forceinline__ float mean_of(float sum, float count, float inv) {
    const float m = sum * inv;
    const float rest = __builtin_fmaf(-m, count, sum);
    return rest - rest == 0.0f ? __builtin_fmaf(rest, inv, m) : m;
}

// ---------------------------------------------------------------------------
// sums
// ---------------------------------------------------------------------------
__device__ __forceinline__ float other_rows(float v, bool halves) {
#if defined(__HIP_DEVICE_COMPILE__)
    const unsigned u = __float_as_uint(v);
    if (halves) {
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        const unsigned lo = r[0], hi = r[1];
        return __uint_as_float(lo) + __uint_as_float(hi);
    }
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned even = r[0], odd = r[1];
    return __uint_as_float(even) + __uint_as_float(odd);
#else
    (void)halves;
    return v;
#endif
}

// Sums over the lanes of a unit (a power of two of them, up to a wave), in every one
// of them, by moves within the vector unit: neighbours, pairs, mirrored halves of
// eight and of sixteen, rows of sixteen, halves of the wave.
template <int N>
__device__ __forceinline__ void lane_sums(float (&v)[N], int lanes) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (lanes > 1) v[i] += from_lane<kNeighbour>(v[i]);
        if (lanes > 2) v[i] += from_lane<kPair>(v[i]);
        if (lanes > 4) v[i] += from_lane<kMirror8>(v[i]);
        if (lanes > 8) v[i] += from_lane<kMirror16>(v[i]);
        if (lanes > 16) v[i] = other_rows(v[i], false);
        if (lanes > 32) v[i] = other_rows(v[i], true);
    }
}

// The same over a workgroup of THREADS; `lds` holds N * THREADS / 64 floats that
// the call before last was done with before the last one's barrier.
template <int N, int THREADS>
__device__ __forceinline__ void block_sums(float (&v)[N], float* lds) {
    lane_sums(v, 64);
    constexpr int kWaves = THREADS / 64;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) lds[i * kWaves + wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) v[i] += lds[i * kWaves + k];
    }
}

// w and b of eight channels, 1 and 0 where there are none.
template <typename T>
__device__ __forceinline__ void load_affine(const NormOperands<T>& a, int64_t at, int64_t end, float (&w)[8],
                                            float (&b)[8]) {
    const Oct<T> vw = a.w ? load_oct(a.w, at, end) : Oct<T>{}, vb = a.b ? load_oct(a.b, at, end) : Oct<T>{};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        w[e] = a.w ? (float)vw[e] : 1.0f;
        b[e] = (float)vb[e];
    }
}

// ---------------------------------------------------------------------------
// rows
// ---------------------------------------------------------------------------
// THREADS 0: `lanes` lanes of a wave to a unit (a row's group), a workgroup of
// four waves; else THREADS of them.  A unit's place decides its group, so its
// lanes' channels stay the same: place p takes the samples p / g, + passes, ...
struct RowPlan {
    int lanes;       // of a unit
    int64_t places;  // a multiple of g
    int64_t passes;  // samples side by side: places / g
};

struct RowPlace {
    int li;      // the lane in its unit
    int step;    // channels from one of a lane's octs to the next
    int64_t row0, gi;
    bool live;
};
template <int THREADS, typename T>
__device__ __forceinline__ RowPlace row_place(const NormOperands<T>& a, const RowPlan& plan) {
    constexpr bool kWide = THREADS > 0;
    RowPlace q;
    const int lane = threadIdx.x & 63;
    q.li = kWide ? threadIdx.x : lane & (plan.lanes - 1);
    q.step = 8 * (kWide ? THREADS : plan.lanes);
    const int per = 64 / (kWide ? 64 : plan.lanes);
    const int64_t place = kWide ? (int64_t)blockIdx.x
                                : ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * per + lane / plan.lanes;
    q.row0 = place / a.g;
    q.gi = place - q.row0 * a.g;
    q.live = place < plan.places;
    return q;
}

template <typename T, int CPL, int THREADS>
__global__ __launch_bounds__(THREADS ? THREADS : 256) void norm_rows_kernel(NormOperands<T> a, RowPlan plan) {
    constexpr bool kWide = THREADS > 0;
    __shared__ float lds[2][2][kWide ? THREADS / 64 : 1];
    const RowPlace q = row_place<THREADS>(a, plan);
    const uint64_t offset = drop_offset(a.drop);
    const float count = (float)a.d, inv = 1.0f / count;
    const int32_t d = (int32_t)a.d;
    float w[CPL][8], b[CPL][8];
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
        const int32_t c = 8 * q.li + j * q.step;
        load_affine(a, q.gi * a.d + c, q.live && c < d ? (q.gi + 1) * a.d : 0, w[j], b[j]);
    }
    int turn = 0;
    Oct<T> raw[CPL] = {};
    auto load = [&](int64_t row) {
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const int32_t c = 8 * q.li + j * q.step;
            if (q.live && row < a.n && c < d) raw[j] = load_oct(a.x + (row * a.g + q.gi) * a.d, c, d);
        }
    };
    load(q.row0);
    for (int64_t r0 = 0; r0 < a.n; r0 += plan.passes, turn ^= 1) {
        const int64_t row = r0 + q.row0;
        const bool ok = q.live && row < a.n;
        if (kWide && !ok) break;  // the whole workgroup
        const int64_t unit = row * a.g + q.gi, base = unit * a.d;
        float v[CPL][8];
        float sum[1] = {0.0f};
#pragma unroll
        for (int j = 0; j < CPL; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[j][e] = (float)raw[j][e];
                sum[0] += v[j][e];
            }
        load(row + plan.passes);  // under way while this one is worked on
        if constexpr (kWide)
            block_sums<1, THREADS>(sum, lds[turn][0]);
        else
            lane_sums(sum, plan.lanes);
        const float mean = mean_of(sum[0], count, inv);
        sum[0] = 0.0f;
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const int32_t c = 8 * q.li + j * q.step;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] -= mean;
            if (c + 8 <= d) {
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[0] = __builtin_fmaf(v[j][e], v[j][e], sum[0]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < d) sum[0] = __builtin_fmaf(v[j][e], v[j][e], sum[0]);
            }
        }
        if constexpr (kWide)
            block_sums<1, THREADS>(sum, lds[turn][1]);
        else
            lane_sums(sum, plan.lanes);
        const float rstd = inverse_root(__builtin_fmaf(sum[0], inv, a.eps));
        if (ok && q.li == 0 && a.mean) {
            a.mean[unit] = mean;
            a.rstd[unit] = rstd;
        }
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const int32_t c = 8 * q.li + j * q.step;
            if (!ok || c >= d) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] *= rstd;
            forward_oct(a, offset, base + c, w[j], b[j], v[j]);
            store_oct(a.y + base, c, d, v[j]);
        }
    }
}

template <typename T, int CPL, int THREADS>
__global__ __launch_bounds__(THREADS ? THREADS : 256) void norm_rows_grad_kernel(NormOperands<T> a, RowPlan plan) {
    constexpr bool kWide = THREADS > 0;
    __shared__ float lds[2][2 * (kWide ? THREADS / 64 : 1)];
    const RowPlace q = row_place<THREADS>(a, plan);
    const uint64_t offset = drop_offset(a.drop);
    const float inv = 1.0f / (float)a.d;
    const int32_t d = (int32_t)a.d;
    float w[CPL][8], b[CPL][8], dw[CPL][8] = {}, db[CPL][8] = {};
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
        const int32_t c = 8 * q.li + j * q.step;
        load_affine(a, q.gi * a.d + c, q.live && c < d ? (q.gi + 1) * a.d : 0, w[j], b[j]);
    }
    int turn = 0;
    Oct<T> rx[CPL] = {}, rd[CPL] = {};
    float next_mean = 0.0f, next_rstd = 0.0f;
    auto load = [&](int64_t row) {
        if (!q.live || row >= a.n) return;
        const int64_t unit = row * a.g + q.gi;
        next_mean = a.mean[unit];
        next_rstd = a.rstd[unit];
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const int32_t c = 8 * q.li + j * q.step;
            if (c < d) {
                rx[j] = load_oct(a.x + unit * a.d, c, d);
                rd[j] = load_oct(a.dy + unit * a.d, c, d);
            }
        }
    };
    load(q.row0);
    for (int64_t r0 = 0; r0 < a.n; r0 += plan.passes, turn ^= 1) {
        const int64_t row = r0 + q.row0;
        const bool ok = q.live && row < a.n;
        if (kWide && !ok) break;  // the whole workgroup
        const int64_t base = (row * a.g + q.gi) * a.d;
        float xh[CPL][8], t[CPL][8];
        const float mean = next_mean, rstd = next_rstd;
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                xh[j][e] = ((float)rx[j][e] - mean) * rstd;
                t[j][e] = (float)rd[j][e];
            }
        }
        load(row + plan.passes);  // under way while this one is worked on
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const int32_t c = 8 * q.li + j * q.step;
            if (c + 8 > d)  // past the group's end dy is zero, and so is what comes of it
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e >= d) xh[j][e] = 0.0f;
            if (!ok || c >= d) continue;
            backward_oct(a, offset, base + c, w[j], b[j], xh[j], t[j]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                db[j][e] += t[j][e];
                dw[j][e] = __builtin_fmaf(t[j][e], xh[j][e], dw[j][e]);
                t[j][e] *= w[j][e];
                sum[0] += t[j][e];
                sum[1] = __builtin_fmaf(t[j][e], xh[j][e], sum[1]);
            }
        }
        if constexpr (kWide)
            block_sums<2, THREADS>(sum, lds[turn]);
        else
            lane_sums(sum, plan.lanes);
        const float m1 = sum[0] * inv, m2 = sum[1] * inv;
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const int32_t c = 8 * q.li + j * q.step;
            if (!a.y || !ok || c >= d) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) t[j][e] = rstd * (t[j][e] - __builtin_fmaf(xh[j][e], m2, m1));
            store_oct(a.y + base, c, d, t[j]);
        }
    }
    if (!q.live) return;
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
        const int32_t c = 8 * q.li + j * q.step;
        if (c >= d) continue;
        if (a.pw) store_oct(a.pw + q.row0 * a.c + q.gi * a.d, c, d, dw[j]);
        if (a.pb) store_oct(a.pb + q.row0 * a.c + q.gi * a.d, c, d, db[j]);
    }
}

// ---------------------------------------------------------------------------
// slabs of whole groups
// ---------------------------------------------------------------------------
struct SlabPlan {
    int32_t groups;   // of a slab
    int32_t octs;     // of a slab's row: ceil(groups * d / 8)
    int32_t rows;     // positions side by side
    int32_t slabs;    // of a row of channels
    int64_t across;   // resident: samples side by side; split: runs of positions
    int64_t run;      // split: positions of a run
};

constexpr int kSlabGroups = 256;  // of a slab, at most

// A thread's place in a slab: eight channels of every so-manieth position; and, where
// the threads' sums are added up, a channel (or several) of a slice of those.
struct SlabPlace {
    int32_t oct, row;       // row: -1 where the thread has nothing to do
    int32_t width;          // channels of the slab
    int32_t groups, d;
    int32_t slices;         // 1 where there are more channels than threads
    int32_t slice, column;  // column: the first of the thread's, then + THREADS
    int64_t c0, g0;         // the slab's first channel and group
};
template <int THREADS, typename T>
__device__ __forceinline__ SlabPlace slab_place(const NormOperands<T>& a, const SlabPlan& p, int32_t slab) {
    SlabPlace q;
    const int t = threadIdx.x;
    q.row = t / p.octs;
    q.oct = t - q.row * p.octs;
    q.d = (int32_t)a.d;
    q.g0 = (int64_t)slab * p.groups;
    q.c0 = q.g0 * a.d;
    const int64_t left = a.g - q.g0;
    q.groups = (int32_t)(left < p.groups ? left : p.groups);
    q.width = q.groups * q.d;
    if (q.row >= p.rows || q.oct * 8 >= q.width) q.row = -1;
    q.slices = THREADS / q.width;
    if (q.slices > p.rows) q.slices = p.rows;
    if (q.slices < 1) q.slices = 1;
    q.slice = q.slices > 1 ? t / q.width : 0;
    q.column = t - q.slice * q.width;
    return q;
}

// The groups of a thread's eight channels, of the slab (0 past its end).
template <typename F>
__device__ __forceinline__ void each_group(const SlabPlace& q, F f) {
    const int32_t c0 = 8 * q.oct;
    int32_t g = q.row >= 0 ? c0 / q.d : 0, in = c0 - g * q.d;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        f(e, q.row >= 0 && c0 + e < q.width ? g : 0);
        if (++in == q.d) {
            in = 0;
            ++g;
        }
    }
}

// Adds up N values of each of the threads' channels over the rows: first over every
// `slices`th row, a channel's and slice's handed to seen(place in a row of lds, sums);
// then over slices and a group's channels, times what weight(channel) says, and
// done(group, sums) once for each.  `lds`: N * rows *
// octs * 8 floats; what channels past the slab's end hold is not read.
template <int N, int THREADS, typename Seen, typename Weight, typename Done>
__device__ __forceinline__ void group_sums(const float (&v)[N][8], const SlabPlan& p, const SlabPlace& q, float* lds,
                                           bool groups, Seen seen, Weight weight, Done done) {
    const int32_t line = p.octs * 8, size = p.rows * line;
    const int t = threadIdx.x;
    __syncthreads();  // what was there has been read
    if (t < p.rows * p.octs) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < 8; e += 4)
                *reinterpret_cast<f32x4*>(lds + i * size + t * 8 + e) =
                    f32x4{v[i][e], v[i][e + 1], v[i][e + 2], v[i][e + 3]};
    }
    __syncthreads();
    if (q.slice < q.slices) {
        constexpr int U = 4;  // rows under way
#pragma unroll 1
        for (int c = q.column; c < q.width; c += THREADS) {
            float sum[N] = {};
#pragma unroll 1
            for (int r = q.slice; r < p.rows; r += U * q.slices) {
                float u[U][N] = {};
#pragma unroll
                for (int j = 0; j < U; ++j)
                    if (r + j * q.slices < p.rows)
#pragma unroll
                        for (int i = 0; i < N; ++i) u[j][i] = lds[i * size + (r + j * q.slices) * line + c];
#pragma unroll
                for (int j = 0; j < U; ++j)
#pragma unroll
                    for (int i = 0; i < N; ++i) sum[i] += u[j][i];
            }
            // row `slice` of the column is this thread's own
#pragma unroll
            for (int i = 0; i < N; ++i) lds[i * size + q.slice * line + c] = sum[i];
            seen(q.slice * line + c, sum);
        }
    }
    if (!groups) return;
    __syncthreads();
    if (q.slices * q.d <= 32) {  // a thread to a group; a wave alone may have more groups than threads
        for (int g = t; g < q.groups; g += THREADS) {
            float sum[N] = {};
#pragma unroll 1
            for (int c = g * q.d; c < (g + 1) * q.d; ++c) {
                const float by = weight(c);
                for (int r = 0; r < q.slices; ++r)
#pragma unroll
                    for (int i = 0; i < N; ++i) sum[i] = __builtin_fmaf(lds[i * size + r * line + c], by, sum[i]);
            }
            done(g, sum);
        }
    } else {  // a wave to a group
        const int lane = t & 63, wave = t >> 6;
        // as many slices side by side as the lanes have room for
        const int wide = q.d < 64 ? q.d : 64, side = 64 / wide, first = lane / wide;
        for (int g = wave; g < q.groups; g += THREADS / 64) {
            float sum[N] = {};
            for (int r = first < side ? first : q.slices; r < q.slices; r += side)
                for (int c = lane - first * wide; c < q.d; c += 64)
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        sum[i] = __builtin_fmaf(lds[i * size + r * line + g * q.d + c], weight(g * q.d + c), sum[i]);
            lane_sums(sum, 64);
            if (lane == 0) done(g, sum);
        }
    }
    __syncthreads();
}

__device__ __forceinline__ float weight_one(int) { return 1.0f; }
struct Nothing {
    template <int N>
    __device__ __forceinline__ void operator()(int, const float (&)[N]) const {}
};

// What was made of these elements is made again from here on: 16-bit ones would be
// kept as f32 besides, in twice the registers.
template <typename T, int M>
__device__ __forceinline__ void forget(Oct<T> (&v)[M]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < M; ++i) {
            u32x4 w = __builtin_bit_cast(u32x4, v[i]);
            asm volatile("" : "+v"(w));
            v[i] = __builtin_bit_cast(Oct<T>, w);
        }
    }
}

// The workgroup's slab and sample: adjacent slabs, which have lines of memory in
// common, in one chiplet (workgroups go to the eight in turn).
__device__ __forceinline__ void slab_of(int32_t& slab, int64_t& sample) {
    const uint32_t id = blockIdx.y * gridDim.x + blockIdx.x, each = gridDim.x * gridDim.y / 8;
    const uint32_t to = id < each * 8 ? (id & 7) * each + (id >> 3) : id;
    sample = to / gridDim.x;
    slab = (int32_t)(to - (uint32_t)sample * gridDim.x);
}

template <typename T, int M, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_resident_kernel(NormOperands<T> a, SlabPlan p) {
    __shared__ __attribute__((aligned(16))) float lds[THREADS * 8];
    __shared__ float means[kSlabGroups], rstds[kSlabGroups];
    const uint64_t offset = drop_offset(a.drop);
    const float count = (float)a.s * (float)a.d, inv = 1.0f / count;
    int32_t slab;
    int64_t place;
    slab_of(slab, place);
    const SlabPlace q = slab_place<THREADS>(a, p, slab);
    const int32_t c0 = 8 * q.oct;  // within the slab
    int32_t gi[8];
    each_group(q, [&](int e, int32_t g) { gi[e] = g; });
    float w[8], b[8];
    load_affine(a, q.c0 + c0, q.row >= 0 ? q.c0 + q.width : 0, w, b);
    for (int64_t n = place; n < a.n; n += gridDim.y) {
        const int64_t base = n * a.s * a.c + q.c0;
        Oct<T> raw[M] = {};
        if (q.row >= 0) {
#pragma unroll
            for (int i = 0; i < M; ++i) {
                const int64_t pos = q.row + (int64_t)i * p.rows;
                if (pos < a.s) raw[i] = load_oct(a.x + base + pos * a.c, c0, q.width);
            }
        }
        float v[1][8] = {};
#pragma unroll
        for (int i = 0; i < M; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[0][e] += (float)raw[i][e];
        group_sums<1, THREADS>(v, p, q, lds, true, Nothing{}, weight_one,
                               [&](int g, const float (&sum)[1]) { means[g] = mean_of(sum[0], count, inv); });
        forget<T>(raw);
        float mean[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            mean[e] = means[gi[e]];
            v[0][e] = 0.0f;
        }
        if (q.row >= 0) {
#pragma unroll
            for (int i = 0; i < M; ++i) {
                if (q.row + (int64_t)i * p.rows >= a.s) continue;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float u = (float)raw[i][e] - mean[e];
                    v[0][e] = __builtin_fmaf(u, u, v[0][e]);
                }
            }
        }
        group_sums<1, THREADS>(v, p, q, lds, true, Nothing{}, weight_one, [&](int g, const float (&sum)[1]) {
            const float rstd = inverse_root(__builtin_fmaf(sum[0], inv, a.eps));
            rstds[g] = rstd;
            if (a.mean) {
                a.mean[n * a.g + q.g0 + g] = means[g];
                a.rstd[n * a.g + q.g0 + g] = rstd;
            }
        });
        if (q.row < 0) continue;
        forget<T>(raw);
        float rstd[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) rstd[e] = rstds[gi[e]];
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const int64_t pos = q.row + (int64_t)i * p.rows;
            if (pos >= a.s) continue;
            float u[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = ((float)raw[i][e] - mean[e]) * rstd[e];
            forward_oct(a, offset, base + pos * a.c + c0, w, b, u);
            store_oct(a.y + base + pos * a.c, c0, q.width, u);
        }
    }
}

// The weights of a slab's channels, for what is added up of each of them.
template <int THREADS, typename T>
__device__ __forceinline__ void slab_weights(const NormOperands<T>& a, const SlabPlace& q, float* lds) {
    for (int c = threadIdx.x; c < q.width; c += THREADS) lds[c] = a.w ? (float)a.w[q.c0 + c] : 1.0f;
}

// Workgroup (slab, place): samples place, place + across, ...  dz is kept for the second
// use of the elements where there are registers for it.
template <typename T, int M, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_resident_grad_kernel(NormOperands<T> a, SlabPlan p) {
    __shared__ __attribute__((aligned(16))) float lds[2 * THREADS * 8];
    __shared__ float totals[2 * THREADS * 8];  // of the channels' slices, each its thread's own
    __shared__ float weights[THREADS * 8], m1s[kSlabGroups], m2s[kSlabGroups];
    constexpr int kSize = THREADS * 8;
    constexpr bool kKeep = M <= 4;
    int32_t slab;
    int64_t place;
    slab_of(slab, place);
    const uint64_t offset = drop_offset(a.drop);
    const float inv = 1.0f / ((float)a.s * (float)a.d);
    const SlabPlace q = slab_place<THREADS>(a, p, slab);
    const int32_t c0 = 8 * q.oct;
    slab_weights<THREADS>(a, q, weights);
    for (int i = threadIdx.x; i < 2 * kSize; i += THREADS) totals[i] = 0.0f;
    float w[8], b[8];
    int32_t gi[8];
    load_affine(a, q.c0 + c0, q.row >= 0 ? q.c0 + q.width : 0, w, b);
    each_group(q, [&](int e, int32_t g) { gi[e] = g; });
    for (int64_t n = place; n < a.n; n += p.across) {
        const int64_t base = n * a.s * a.c + q.c0;
        Oct<T> rx[M] = {}, rd[M] = {};
        float mean[8], rstd[8], dz[kKeep ? M : 1][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int64_t at = n * a.g + q.g0 + gi[e];
            mean[e] = a.mean[at];
            rstd[e] = a.rstd[at];
        }
        float v[2][8] = {};
        if (q.row >= 0) {
#pragma unroll
            for (int i = 0; i < M; ++i) {
                const int64_t pos = q.row + (int64_t)i * p.rows;
                if (pos < a.s) {
                    rx[i] = load_oct(a.x + base + pos * a.c, c0, q.width);
                    rd[i] = load_oct(a.dy + base + pos * a.c, c0, q.width);
                }
            }
#pragma unroll
            for (int i = 0; i < M; ++i) {
                const int64_t pos = q.row + (int64_t)i * p.rows;
                if (pos >= a.s) continue;
                float xh[8], t[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    xh[e] = ((float)rx[i][e] - mean[e]) * rstd[e];
                    t[e] = (float)rd[i][e];
                }
                backward_oct(a, offset, base + pos * a.c + c0, w, b, xh, t);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[0][e] += t[e];
                    v[1][e] = __builtin_fmaf(t[e], xh[e], v[1][e]);
                    if constexpr (kKeep) dz[i][e] = t[e];
                }
            }
        }
        group_sums<2, THREADS>(
            v, p, q, lds, a.y != nullptr,
            [&](int at, const float (&sum)[2]) {
                totals[at] += sum[0];
                totals[kSize + at] += sum[1];
            },
            [&](int c) { return weights[c]; },
            [&](int g, const float (&sum)[2]) {
                m1s[g] = sum[0] * inv;
                m2s[g] = sum[1] * inv;
            });
        if (!a.y || q.row < 0) continue;
        forget<T>(rx);
        if constexpr (!kKeep) forget<T>(rd);
        float m1[8], m2[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            m1[e] = m1s[gi[e]];
            m2[e] = m2s[gi[e]];
        }
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const int64_t pos = q.row + (int64_t)i * p.rows;
            if (pos >= a.s) continue;
            float xh[8], t[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                xh[e] = ((float)rx[i][e] - mean[e]) * rstd[e];
                t[e] = kKeep ? dz[kKeep ? i : 0][e] : (float)rd[i][e];
            }
            if constexpr (!kKeep) backward_oct(a, offset, base + pos * a.c + c0, w, b, xh, t);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                t[e] = rstd[e] * (t[e] * w[e] - __builtin_fmaf(xh[e], m2[e], m1[e]));
            store_oct(a.y + base + pos * a.c, c0, q.width, t);
        }
    }
    if (!a.pw && !a.pb) return;
    __syncthreads();
    for (int c = threadIdx.x; c < q.width; c += THREADS) {
        float sum[2] = {0.0f, 0.0f};
        for (int r = 0; r < q.slices; ++r) {
            sum[0] += totals[r * p.octs * 8 + c];
            sum[1] += totals[kSize + r * p.octs * 8 + c];
        }
        if (a.pb) a.pb[place * a.c + q.c0 + c] = sum[0];
        if (a.pw) a.pw[place * a.c + q.c0 + c] = sum[1];
    }
}

// ---------------------------------------------------------------------------
// split
// ---------------------------------------------------------------------------
// A run's statistics of every group: its mean, and the sum of squares about it; the
// counts follow from the run.  Each thread sums differences from its first row, a
// channel of its own, so that a large mean costs nothing.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_split_stats_kernel(NormOperands<T> a, SlabPlan p, float* part) {
    __shared__ __attribute__((aligned(16))) float lds[THREADS * 8];
    __shared__ float means[kSlabGroups];
    const int64_t run = blockIdx.y;
    const SlabPlace q = slab_place<THREADS>(a, p, (int32_t)blockIdx.x);
    const int32_t c0 = 8 * q.oct;
    const int64_t s0 = run * p.run, s1 = s0 + p.run < a.s ? s0 + p.run : a.s;
    const float size = (float)(s1 - s0) * (float)a.d, inv = 1.0f / size;
    const int64_t step = (int64_t)p.rows * a.c;
    for (int64_t n = blockIdx.z; n < a.n; n += gridDim.z) {
        float first[8] = {}, sum[8] = {}, square[8] = {};
        int32_t rows = 0;
        if (q.row >= 0 && s0 + q.row < s1) {
            const T* from = a.x + (n * a.s + s0 + q.row) * a.c + q.c0;
            rows = (int32_t)((s1 - s0 - q.row + p.rows - 1) / p.rows);
            constexpr int U = sizeof(T) == 2 ? 8 : 4;
            const Oct<T> raw = load_oct(from, c0, q.width);
#pragma unroll
            for (int e = 0; e < 8; ++e) {  // differences from what is no number would be none
                sum[e] = (float)raw[e];
                first[e] = finite(sum[e]) ? sum[e] : 0.0f;
                sum[e] -= first[e];
                square[e] = fabsf(sum[e]);
            }
            from += step;
            for (int32_t r = 1; r < rows; r += U, from += U * step) {
                Oct<T> v[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (r + u < rows) v[u] = load_oct(from + u * step, c0, q.width);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (r + u >= rows) continue;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float t = (float)v[u][e] - first[e];
                        sum[e] += t;
                        square[e] = __builtin_fmaf(t, t, square[e]);
                    }
                }
            }
        }
        // to each channel's own mean, then to the group's
        float v[1][8];
        const float by = rows ? 1.0f / (float)rows : 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float m = sum[e] * by;
            square[e] = squares_less(square[e], sum[e] * m);
            first[e] += m;  // the channel's mean
            v[0][e] = first[e] * (float)rows;
        }
        const int64_t at = (n * p.across + run) * a.g + q.g0;
        group_sums<1, THREADS>(v, p, q, lds, true, Nothing{}, weight_one, [&](int g, const float (&total)[1]) {
            means[g] = mean_of(total[0], size, inv);
            part[2 * (at + g)] = means[g];
        });
        each_group(q, [&](int e, int32_t g) {
            const float far = first[e] - means[g];
            v[0][e] = rows ? __builtin_fmaf(far * far, (float)rows, square[e]) : 0.0f;
        });
        group_sums<1, THREADS>(v, p, q, lds, true, Nothing{}, weight_one,
                               [&](int g, const float (&total)[1]) { part[2 * (at + g) + 1] = total[0]; });
    }
}

// Rows under way: the first of DEPTH is worked on while the others are loaded.  Rows
// are moved up rather than the loop unrolled, as the code of every activation times
// the depth takes the registers of as many waves.
template <typename T, int DEPTH>
struct RowQueue {
    Oct<T> v[DEPTH];
    __device__ __forceinline__ void fill(const T* from, int64_t step, int32_t c, int32_t width, int32_t rows) {
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            v[i] = Oct<T>{};
            if (i < rows) v[i] = load_oct(from + i * step, c, width);
        }
    }
    // the row in front is done; `left` rows from it on
    __device__ __forceinline__ void next(const T* from, int64_t step, int32_t c, int32_t width, int32_t left) {
#pragma unroll
        for (int i = 0; i + 1 < DEPTH; ++i) v[i] = v[i + 1];
        if (left > DEPTH) v[DEPTH - 1] = load_oct(from + DEPTH * step, c, width);
    }
};

template <typename T>
constexpr int kRowsAhead = sizeof(T) == 2 ? 4 : 3;

// A run's positions.
__device__ __forceinline__ float run_count(const SlabPlan& p, int64_t s, int64_t r) {
    return (float)(r + 1 < p.across ? p.run : s - r * p.run);
}

// The lanes that add up a group's runs: so many that the workgroup has all groups at
// once, a power of two.
template <int THREADS>
__device__ __forceinline__ int join_lanes(const SlabPlan& p) {
    int lanes = 64;
    while (lanes > 1 && lanes * p.groups > THREADS) lanes >>= 1;
    return lanes;
}
template <typename F>
__device__ __forceinline__ void each_join(const SlabPlace& q, int lanes, F f) {
    const int g = threadIdx.x / lanes;
    if (g < q.groups) f(g, threadIdx.x & (lanes - 1));
}

// Joins the runs of a sample's groups: the mean, and the squares about it; then y.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_split_kernel(NormOperands<T> a, SlabPlan p, const float* part) {
    __shared__ float means[kSlabGroups], rstds[kSlabGroups];
    const int lanes = join_lanes<THREADS>(p);
    const float inv = 1.0f / ((float)a.s * (float)a.d);
    const uint64_t offset = drop_offset(a.drop);
    const int64_t run = blockIdx.y;
    const SlabPlace q = slab_place<THREADS>(a, p, (int32_t)blockIdx.x);
    const int32_t c0 = 8 * q.oct;
    const int64_t s0 = run * p.run, s1 = s0 + p.run < a.s ? s0 + p.run : a.s;
    const int64_t step = (int64_t)p.rows * a.c;
    float w[8], b[8];
    load_affine(a, q.c0 + c0, q.row >= 0 ? q.c0 + q.width : 0, w, b);
    for (int64_t n = blockIdx.z; n < a.n; n += gridDim.z) {
        __syncthreads();
        // as a sum over the first run's mean: sum of n (m - m0), and of the squares
        // about m0, from which what the mean is off m0 is taken; infinities and NaN go
        // where the definition has them
        each_join(q, lanes, [&](int g, int li) {
            const float* f = part + 2 * (n * p.across * a.g + q.g0 + g);
            const int64_t next = 2 * a.g;
            const float first = finite(f[0]) ? f[0] : 0.0f;
            float sum[2] = {0.0f, 0.0f};
#pragma unroll 4
            for (int64_t r = li; r < p.across; r += lanes) {
                const float far = f[r * next] - first, count = run_count(p, a.s, r) * (float)a.d;
                sum[0] = __builtin_fmaf(far, count, sum[0]);
                sum[1] += __builtin_fmaf(far * far, count, f[r * next + 1]);
            }
            lane_sums(sum, lanes);
            if (li) return;
            const float beyond = sum[0] * inv, mean = first + beyond;
            const float rstd = inverse_root(squares_less(sum[1] * inv, beyond * beyond) + a.eps);
            means[g] = mean;
            rstds[g] = rstd;
            if (a.mean && run == 0) {
                a.mean[n * a.g + q.g0 + g] = mean;
                a.rstd[n * a.g + q.g0 + g] = rstd;
            }
        });
        __syncthreads();
        if (q.row < 0 || s0 + q.row >= s1) continue;
        float mean[8], rstd[8];
        each_group(q, [&](int e, int32_t g) {
            mean[e] = means[g];
            rstd[e] = rstds[g];
        });
        int64_t at = (n * a.s + s0 + q.row) * a.c + q.c0;
        const int32_t rows = (int32_t)((s1 - s0 - q.row + p.rows - 1) / p.rows);
        RowQueue<T, kRowsAhead<T>> rows_x;
        rows_x.fill(a.x + at, step, c0, q.width, rows);
#pragma unroll 1
        for (int32_t r = 0; r < rows; ++r, at += step) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = ((float)rows_x.v[0][e] - mean[e]) * rstd[e];
            rows_x.next(a.x + at, step, c0, q.width, rows - r);
            forward_oct(a, offset, at + c0, w, b, f);
            store_oct(a.y + at, c0, q.width, f);
        }
    }
}

// Backwards: of every run the groups' two sums (part), and the channels' (pw, pb).
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_split_sums_kernel(NormOperands<T> a, SlabPlan p, float* part) {
    __shared__ __attribute__((aligned(16))) float lds[2 * THREADS * 8];
    __shared__ float weights[THREADS * 8];
    const uint64_t offset = drop_offset(a.drop);
    const int64_t run = blockIdx.y;
    const SlabPlace q = slab_place<THREADS>(a, p, (int32_t)blockIdx.x);
    const int32_t c0 = 8 * q.oct;
    const int64_t s0 = run * p.run, s1 = s0 + p.run < a.s ? s0 + p.run : a.s;
    const int64_t step = (int64_t)p.rows * a.c;
    slab_weights<THREADS>(a, q, weights);
    float w[8], b[8];
    load_affine(a, q.c0 + c0, q.row >= 0 ? q.c0 + q.width : 0, w, b);
    for (int64_t n = blockIdx.z; n < a.n; n += gridDim.z) {
        float mean[8], rstd[8], v[2][8] = {};
        each_group(q, [&](int e, int32_t g) {
            mean[e] = a.mean[n * a.g + q.g0 + g];
            rstd[e] = a.rstd[n * a.g + q.g0 + g];
        });
        if (q.row >= 0 && s0 + q.row < s1) {
            int64_t at = (n * a.s + s0 + q.row) * a.c + q.c0;
            const int32_t rows = (int32_t)((s1 - s0 - q.row + p.rows - 1) / p.rows);
            RowQueue<T, 3> rows_x, rows_d;
            rows_x.fill(a.x + at, step, c0, q.width, rows);
            rows_d.fill(a.dy + at, step, c0, q.width, rows);
#pragma unroll 1
            for (int32_t r = 0; r < rows; ++r, at += step) {
                float xh[8], t[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    xh[e] = ((float)rows_x.v[0][e] - mean[e]) * rstd[e];
                    t[e] = (float)rows_d.v[0][e];
                }
                rows_x.next(a.x + at, step, c0, q.width, rows - r);
                rows_d.next(a.dy + at, step, c0, q.width, rows - r);
                backward_oct(a, offset, at + c0, w, b, xh, t);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[0][e] += t[e];
                    v[1][e] = __builtin_fmaf(t[e], xh[e], v[1][e]);
                }
            }
        }
        const int64_t line = n * p.across + run;
        group_sums<2, THREADS>(
            v, p, q, lds, true, Nothing{}, [&](int c) { return weights[c]; },
            [&](int g, const float (&sum)[2]) {
                float* const to = part + 2 * (line * a.g + q.g0 + g);
                to[0] = sum[0];
                to[1] = sum[1];
            });
        if (!a.pw && !a.pb) continue;
        const int32_t row = p.octs * 8, size = p.rows * row;  // where the slices' sums are
        for (int c = threadIdx.x; c < q.width; c += THREADS) {
            float sum[2] = {0.0f, 0.0f};
            for (int r = 0; r < q.slices; ++r) {
                sum[0] += lds[r * row + c];
                sum[1] += lds[size + r * row + c];
            }
            if (a.pb) a.pb[line * a.c + q.c0 + c] = sum[0];
            if (a.pw) a.pw[line * a.c + q.c0 + c] = sum[1];
        }
    }
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_split_grad_kernel(NormOperands<T> a, SlabPlan p, const float* part) {
    __shared__ float m1s[kSlabGroups], m2s[kSlabGroups];
    const int lanes = join_lanes<THREADS>(p);
    const uint64_t offset = drop_offset(a.drop);
    const float inv = 1.0f / ((float)a.s * (float)a.d);
    const int64_t run = blockIdx.y;
    const SlabPlace q = slab_place<THREADS>(a, p, (int32_t)blockIdx.x);
    const int32_t c0 = 8 * q.oct;
    const int64_t s0 = run * p.run, s1 = s0 + p.run < a.s ? s0 + p.run : a.s;
    const int64_t step = (int64_t)p.rows * a.c;
    float w[8], b[8];
    load_affine(a, q.c0 + c0, q.row >= 0 ? q.c0 + q.width : 0, w, b);
    for (int64_t n = blockIdx.z; n < a.n; n += gridDim.z) {
        __syncthreads();
        each_join(q, lanes, [&](int g, int li) {
            const float* f = part + 2 * (n * p.across * a.g + q.g0 + g);
            float sum[2] = {0.0f, 0.0f};
#pragma unroll 4
            for (int64_t r = li; r < p.across; r += lanes) {
                sum[0] += f[2 * r * a.g];
                sum[1] += f[2 * r * a.g + 1];
            }
            lane_sums(sum, lanes);
            if (li) return;
            m1s[g] = sum[0] * inv;
            m2s[g] = sum[1] * inv;
        });
        __syncthreads();
        if (q.row < 0 || s0 + q.row >= s1) continue;
        float mean[8], rstd[8], m1[8], m2[8];
        each_group(q, [&](int e, int32_t g) {
            mean[e] = a.mean[n * a.g + q.g0 + g];
            rstd[e] = a.rstd[n * a.g + q.g0 + g];
            m1[e] = m1s[g];
            m2[e] = m2s[g];
        });
        int64_t at = (n * a.s + s0 + q.row) * a.c + q.c0;
        const int32_t rows = (int32_t)((s1 - s0 - q.row + p.rows - 1) / p.rows);
        RowQueue<T, 3> rows_x, rows_d;
        rows_x.fill(a.x + at, step, c0, q.width, rows);
        rows_d.fill(a.dy + at, step, c0, q.width, rows);
#pragma unroll 1
        for (int32_t r = 0; r < rows; ++r, at += step) {
            float xh[8], t[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                xh[e] = ((float)rows_x.v[0][e] - mean[e]) * rstd[e];
                t[e] = (float)rows_d.v[0][e];
            }
            rows_x.next(a.x + at, step, c0, q.width, rows - r);
            rows_d.next(a.dy + at, step, c0, q.width, rows - r);
            backward_oct(a, offset, at + c0, w, b, xh, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = rstd[e] * (t[e] * w[e] - __builtin_fmaf(xh[e], m2[e], m1[e]));
            store_oct(a.y + at, c0, q.width, t);
        }
    }
}

// ---------------------------------------------------------------------------
// the parameters' gradients: `rows` partial sums of every channel, in order
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(1024) void norm_join_kernel(const float* pw, const float* pb, int64_t rows, int64_t c,
                                                         T* dw, T* db) {
    __shared__ float join[32][33];
    const float* from = blockIdx.y ? pb : pw;
    T* to = blockIdx.y ? db : dw;
    if (!to) return;
    const int col = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t at = (int64_t)blockIdx.x * 32 + col;
    float sum = 0.0f;
    if (at < c) {
        int64_t r = slice;
        for (; r + 3 * 32 < rows; r += 4 * 32) {
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = from[(r + 32 * u) * c + at];
#pragma unroll
            for (int u = 0; u < 4; ++u) sum += v[u];
        }
        for (; r < rows; r += 32) sum += from[r * c + at];
    }
    join[slice][col] = sum;
    __syncthreads();
    if (slice) return;
#pragma unroll
    for (int i = 1; i < 32; ++i) sum += join[i][col];
    if (at < c) to[at] = (T)sum;
}

// ---------------------------------------------------------------------------
// which way, and its sizes
// ---------------------------------------------------------------------------
struct Way {
    enum { kRows, kResident, kSplit } kind;
    int cpl, threads;  // rows: octs of a lane, and 0 or the unit's threads; else the workgroup's threads
    int m;             // resident: positions of a thread
    RowPlan row;
    SlabPlan slab;
    int64_t blocks;  // rows
    int64_t side;    // slabs: samples side by side
    int64_t parts;  // rows of the parameters' partial sums
};

// Positions of a thread of 512: backwards as many as spill no registers (11 take 254 of
// 256, six of f32 250); forwards one more than that (12 take 179, of f32 212).
constexpr int most_positions(int elem_bytes, bool grad) { return !grad ? 12 : elem_bytes == 4 ? 6 : 11; }

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

Way choose(int elem_bytes, int64_t n, int64_t s, int64_t c, int64_t g, bool grad, int cus) {
    Way o{};
    const int64_t d = c / g, octs = ceil_div(d, 8);
    if (s == 1) {
        o.kind = Way::kRows;
        int64_t units;  // of a workgroup
        if (octs <= 64) {
            o.cpl = 1;
            o.row.lanes = 1;
            while (o.row.lanes < octs) o.row.lanes *= 2;
            units = 4 * (64 / o.row.lanes);
        } else if (octs <= 128) {
            o.cpl = 2;
            o.row.lanes = 64;
            units = 4;
        } else {
            o.cpl = octs <= 256 ? 1 : 2;
            o.threads = octs <= 512 ? 256 : 512;
            units = 1;
        }
        const int64_t most = std::max(ceil_div((int64_t)cus * (grad ? 4 : 8), 1), ceil_div(g, units));
        int64_t blocks = std::min(most, ceil_div(n * g, units));
        int64_t side = std::max<int64_t>(1, blocks * units / g);  // samples side by side
        // Backwards a unit's sample takes 1 us, after which 2.7 ns go into adding up each
        // unit's sums: 20 sqrt(n) make both together least.  100,000 rows of 64 bf16
        // channels in 4 groups take 44 us with 4096 side by side, 84 with all, 113 with 1024.
        if (grad) side = std::min(side, (int64_t)(20.0 * std::sqrt((double)n)));
        o.row.passes = ceil_div(n, ceil_div(n, side));
        o.row.places = o.row.passes * g;
        o.blocks = ceil_div(o.row.places, units);
        o.parts = o.row.passes;
        return o;
    }
    // samples side by side, each in `blocks` workgroups: a launch has fewer than 2^32 threads
    auto beside = [&](int64_t blocks, int threads) {
        return std::max<int64_t>(1, std::min<int64_t>({n, 65535, ((int64_t)1 << 31) / (blocks * threads)}));
    };
    // the slab: whole groups, as few as make a line of memory, or half of one
    auto slab = [&](int threads, int64_t groups) {
        SlabPlan p{};
        p.groups = (int32_t)groups;
        p.octs = (int32_t)ceil_div(groups * d, 8);
        p.rows = threads / p.octs;
        p.slabs = (int32_t)ceil_div(g, groups);
        return p;
    };
    auto bytes = [&](int64_t line) {
        return std::min<int64_t>({g, kSlabGroups, std::max<int64_t>(1, ceil_div(line / elem_bytes, d))});
    };
    const int most = most_positions(elem_bytes, grad), middle = elem_bytes == 4 && grad ? 4 : 8;
    // Slabs of half a line, and as many positions as there are registers for, leave a CU
    // one workgroup at a time, whose loads, sums and stores follow one another: they are
    // taken where no CU gets a second one, whole octs first.  16 samples of 1024 positions
    // of 640 bf16 channels in 32 groups take 17.6 us so and 28.9 backwards, split 27.8
    // and 46.6 (whole calls: 17 and 36; of 17 samples, split, 29 and 41); 64 samples 62 and
    // 111, split 53 and 86; 16 of 600 positions of 320, slabs of 70 channels, 21.8 and 38.5,
    // split 18.2 and 24.
    // A wave alone takes a row of channels that it can hold.  Where few positions would
    // leave most of 256 threads without work, a slab has more groups, as long as every
    // CU has four: 2499 samples of 5 positions of 2025 f16 channels in 27 groups take 266
    // us, there and back, in slabs of a line 1015; 3302 of 4 of 18, a wave each, 34, 72.
    auto wide = [&](int64_t groups) {
        const int64_t line = groups;
        for (int64_t more = 2 * groups;; more *= 2) {
            more = std::min<int64_t>({more, g, kSlabGroups});
            const SlabPlan p = slab(256, more);
            if (more == groups || p.octs > 256 || ceil_div(s, p.rows) > 4 || n * p.slabs < 4 * (int64_t)cus) break;
            groups = more;
        }
        return groups == line ? line : ceil_div(g, ceil_div(g, groups));  // all slabs alike
    };
    struct { int threads, line, most; } tries[] = {
        {64, 0, 2}, {256, 128, middle}, {512, 128, middle}, {512, 64, most}, {512, 128, most}, {512, 64, middle}};
    for (int i = 0; i < 6; ++i) {
        const auto& t = tries[i];
        const int threads = t.threads;
        const SlabPlan p = slab(threads, i == 0 ? std::min<int64_t>(g, kSlabGroups) : i == 1 ? wide(bytes(128)) : bytes(t.line));
        if (p.octs > threads || ceil_div(s, p.rows) > t.most) continue;
        if (i == 0 && p.slabs > 1) continue;
        if (i >= 3 && n * p.slabs > cus) continue;
        if ((i == 3 || i == 4) && p.groups * d % 8) continue;
        o.kind = Way::kResident;
        o.threads = threads;
        const int64_t m = ceil_div(s, p.rows);
        o.m = m <= 2 ? 2 : m <= 4 ? 4 : m <= middle ? middle : most;
        o.slab = p;
        const int64_t side = std::max<int64_t>(1, (int64_t)cus * (threads == 64 ? 8 : threads == 256 ? 4 : 2) / p.slabs);
        o.slab.across = grad ? ceil_div(n, ceil_div(n, std::min<int64_t>({n, side, 65535}))) : n;
        o.side = grad ? o.slab.across : beside(p.slabs, threads);
        o.parts = o.slab.across;
        return o;
    }
    // As many workgroups as run at once in the 16-bit types, four to a CU (114 to 126
    // registers a thread), backwards three (148 to 166), and six positions to a thread at
    // least: a run's first and last steps cost as much as its rows.  16 x 4096 x 320 f16 in
    // 32 groups backwards: 54 us, of four to a CU 58, of eight 78; forwards 36, 36 and 51.
    // 4 x 4096 x 320: 22 us, with four positions 27.  f32's statistics run four to a CU as
    // well, but its second pass three (139 registers) and its gradient's two (176, 191):
    // their grids end in a part of a round; other counts were not measured there.
    // Groups of more than 2048 channels take 1024 threads of 128 registers, which spill
    // but for 16-bit forwards (f32 10 of them, backwards 41 and 53; 16 bits backwards 14
    // to 29): 2 x 300 x 20000 in 4 groups, silu, 51 us in f16 and 85 backwards, f32 59, 142.
    o.kind = Way::kSplit;
    o.threads = octs <= 256 ? 256 : 1024;
    // as many whole groups as the threads have room for
    const int64_t groups = std::max<int64_t>(1, std::min<int64_t>({g, kSlabGroups, (int64_t)o.threads * 8 / d}));
    o.slab = slab(o.threads, groups);
    const int64_t want = ceil_div((int64_t)cus * (grad ? 3 : 4), n * o.slab.slabs);
    const int64_t rows = std::max<int64_t>(ceil_div(s, std::max<int64_t>(1, want)), 6 * (int64_t)o.slab.rows);
    o.slab.run = std::min(rows, s);
    o.slab.across = ceil_div(s, o.slab.run);
    o.side = beside(o.slab.slabs * o.slab.across, o.threads);
    o.parts = n * o.slab.across;
    return o;
}

template <typename T, bool GRAD>
hipError_t launch_rows(const NormOperands<T>& a, const Way& o, hipStream_t s) {
    const dim3 grid((unsigned)o.blocks);
    auto go = [&](auto kernel, int threads) {
        kernel<<<grid, threads, 0, s>>>(a, o.row);
        return hipGetLastError();
    };
#define MLRS_ROWS(CPL, THREADS)                                                    \
    if (o.cpl == CPL && o.threads == THREADS) {                                    \
        if constexpr (GRAD)                                                        \
            return go(norm_rows_grad_kernel<T, CPL, THREADS>, THREADS ? THREADS : 256); \
        else                                                                       \
            return go(norm_rows_kernel<T, CPL, THREADS>, THREADS ? THREADS : 256); \
    }
    MLRS_ROWS(1, 0)
    MLRS_ROWS(2, 0)
    MLRS_ROWS(1, 256)
    MLRS_ROWS(2, 256)
    MLRS_ROWS(2, 512)
#undef MLRS_ROWS
    return hipErrorInvalidValue;
}

template <typename T, bool GRAD>
hipError_t launch_resident(const NormOperands<T>& a, const Way& o, hipStream_t s) {
    const dim3 grid((unsigned)o.slab.slabs, (unsigned)o.side);
    auto go = [&](auto kernel) {
        kernel<<<grid, o.threads, 0, s>>>(a, o.slab);
        return hipGetLastError();
    };
#define MLRS_SLAB(M, THREADS)                                            \
    if (o.m == M && o.threads == THREADS) {                              \
        if constexpr (GRAD)                                              \
            return go(norm_resident_grad_kernel<T, M, THREADS>);         \
        else                                                             \
            return go(norm_resident_kernel<T, M, THREADS>);              \
    }
    MLRS_SLAB(2, 64)
    MLRS_SLAB(2, 256)
    MLRS_SLAB(4, 256)
    MLRS_SLAB(2, 512)
    MLRS_SLAB(4, 512)
    if constexpr (!GRAD || sizeof(T) == 2) {
        MLRS_SLAB(8, 256)
        MLRS_SLAB(8, 512)
    }
    MLRS_SLAB(most_positions((int)sizeof(T), GRAD), 512)
#undef MLRS_SLAB
    return hipErrorInvalidValue;
}

template <typename T>
NormOperands<T> operands(const NormCall& k, const Way& o) {
    NormOperands<T> a{};
    a.x = (const T*)k.x;
    a.w = (const T*)k.w;
    a.b = (const T*)k.b;
    a.dy = (const T*)k.dy;
    a.y = (T*)k.y;
    a.mean = k.mean;
    a.rstd = k.rstd;
    a.n = k.n;
    a.s = k.s;
    a.c = k.c;
    a.g = k.g;
    a.d = k.c / k.g;
    a.eps = k.eps;
    a.act = k.act;
    a.drop = k.drop;
    a.aligned = k.c % 8 == 0 && (o.kind == Way::kRows ? a.d : o.slab.groups * a.d) % 8 == 0;
    return a;
}

}  // namespace

size_t norm_scratch(int elem_bytes, const NormCall& k, int cus) {
    const Way o = choose(elem_bytes, k.n, k.s, k.c, k.g, false, cus);
    return o.kind == Way::kSplit ? (size_t)(k.n * o.slab.across * k.g * 2) * 4 : 0;
}

template <typename T>
hipError_t launch_norm(const NormCall& k, float* scratch, int cus, hipStream_t s) {
    const Way o = choose((int)sizeof(T), k.n, k.s, k.c, k.g, false, cus);
    const NormOperands<T> a = operands<T>(k, o);
    if (o.kind == Way::kRows) return launch_rows<T, false>(a, o, s);
    if (o.kind == Way::kResident) return launch_resident<T, false>(a, o, s);
    const dim3 grid((unsigned)o.slab.slabs, (unsigned)o.slab.across, (unsigned)o.side);
    if (o.threads == 256)
        norm_split_stats_kernel<T, 256><<<grid, 256, 0, s>>>(a, o.slab, scratch);
    else
        norm_split_stats_kernel<T, 1024><<<grid, 1024, 0, s>>>(a, o.slab, scratch);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (o.threads == 256)
        norm_split_kernel<T, 256><<<grid, 256, 0, s>>>(a, o.slab, scratch);
    else
        norm_split_kernel<T, 1024><<<grid, 1024, 0, s>>>(a, o.slab, scratch);
    return hipGetLastError();
}

size_t norm_grad_scratch(int elem_bytes, const NormCall& k, int cus) {
    if (k.n == 0) return 0;
    const Way o = choose(elem_bytes, k.n, k.s, k.c, k.g, true, cus);
    size_t floats = 0;
    if (k.dw) floats += (size_t)(o.parts * k.c);
    if (k.db) floats += (size_t)(o.parts * k.c);
    if (o.kind == Way::kSplit) floats += (size_t)(k.n * o.slab.across * k.g * 2);
    return floats * 4;
}

template <typename T>
hipError_t launch_norm_grad(const NormCall& k, float* scratch, int cus, hipStream_t s) {
    Way o{};  // of no samples, the parameters' sums have no parts
    if (k.n) o = choose((int)sizeof(T), k.n, k.s, k.c, k.g, true, cus);
    NormOperands<T> a = operands<T>(k, o);
    float* at = scratch;
    if (k.dw) {
        a.pw = at;
        at += o.parts * k.c;
    }
    if (k.db) {
        a.pb = at;
        at += o.parts * k.c;
    }
    hipError_t e = hipSuccess;
    if (k.n == 0) {
    } else if (o.kind == Way::kRows) {
        e = launch_rows<T, true>(a, o, s);
    } else if (o.kind == Way::kResident) {
        e = launch_resident<T, true>(a, o, s);
    } else {
        const dim3 grid((unsigned)o.slab.slabs, (unsigned)o.slab.across, (unsigned)o.side);
        if (o.threads == 256)
            norm_split_sums_kernel<T, 256><<<grid, 256, 0, s>>>(a, o.slab, at);
        else
            norm_split_sums_kernel<T, 1024><<<grid, 1024, 0, s>>>(a, o.slab, at);
        e = hipGetLastError();
        if (e == hipSuccess && k.y) {
            if (o.threads == 256)
                norm_split_grad_kernel<T, 256><<<grid, 256, 0, s>>>(a, o.slab, at);
            else
                norm_split_grad_kernel<T, 1024><<<grid, 1024, 0, s>>>(a, o.slab, at);
            e = hipGetLastError();
        }
    }
    if (e != hipSuccess || (!k.dw && !k.db)) return e;
    norm_join_kernel<T><<<dim3((unsigned)((k.c + 31) / 32), 2), 1024, 0, s>>>(a.pw, a.pb, o.parts, k.c, (T*)k.dw,
                                                                             (T*)k.db);
    return hipGetLastError();
}

#define MLRS_INST(T)                                                                \
    template hipError_t launch_norm<T>(const NormCall&, float*, int, hipStream_t);  \
    template hipError_t launch_norm_grad<T>(const NormCall&, float*, int, hipStream_t);
MLRS_INST(float)
MLRS_INST(_Float16)
MLRS_INST(__bf16)

}  // namespace train
}  // namespace mlrs
