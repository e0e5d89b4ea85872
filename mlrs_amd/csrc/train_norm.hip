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
// All of it is bound by memory: the elements are read once and kept in registers
// between the sums and what needs them, but where a group is too large for that.
// Three ways:
//   rows      s = 1: a group is d adjacent elements, which some lanes of a wave, or
//             a workgroup, hold.
//   resident  a workgroup holds a slab, some whole groups of a sample: a thread has
//             eight adjacent channels at every so-manieth position.
//   split     groups past that: partial sums of runs of positions, then a second
//             pass over the elements; it reads the sums first, so that it is the
//             second launch of two.
// The parameters' gradients are added up per thread while its channels stay the
// same over samples and positions; a last launch adds those in order.
#include <algorithm>

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
    Drop drop;
};

template <int A>
struct Act {
    static constexpr int id = A;
};
template <typename F>
__device__ __forceinline__ void with_activation(int act, F f) {
    switch (act) {
    case kActRelu: f(Act<kActRelu>{}); break;
    case kActGelu: f(Act<kActGelu>{}); break;
    case kActGeluTanh: f(Act<kActGeluTanh>{}); break;
    case kActSilu: f(Act<kActSilu>{}); break;
    default: f(Act<kActNone>{}); break;
    }
}

// Sums over the lanes of a unit (a power of two of them, up to a wave).
template <int N>
__device__ __forceinline__ void lane_sums(float (&v)[N], int lanes) {
    for (int o = lanes >> 1; o; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o);
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

// y of eight elements from their xh.
template <typename T>
__device__ __forceinline__ void forward_oct(const NormOperands<T>& a, uint64_t offset, int64_t i, const float (&w)[8],
                                            const float (&b)[8], float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(v[e], w[e], b[e]);
    with_activation(a.act, [&](auto act) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = activate(v[e], decltype(act)::id);
    });
    if (a.drop.threshold) drop_oct(a.drop, offset, i, v);
    __builtin_amdgcn_sched_barrier(0);  // one after another: interleaved, they take twice the registers
}

// dz of eight elements: dy becomes it.
template <typename T>
__device__ __forceinline__ void backward_oct(const NormOperands<T>& a, uint64_t offset, int64_t i,
                                             const float (&w)[8], const float (&b)[8], const float (&xh)[8],
                                             float (&dy)[8]) {
    if (a.drop.threshold) drop_oct(a.drop, offset, i, dy);
    if (a.act != kActNone)
        with_activation(a.act, [&](auto act) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                dy[e] *= activate_slope(__builtin_fmaf(xh[e], w[e], b[e]), decltype(act)::id);
        });
    __builtin_amdgcn_sched_barrier(0);
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

template <typename T, int CPL, int THREADS>
__global__ __launch_bounds__(THREADS ? THREADS : 256) void norm_rows_kernel(NormOperands<T> a, RowPlan plan) {
    constexpr bool kWide = THREADS > 0;
    constexpr int kWaves = kWide ? THREADS / 64 : 1;
    __shared__ float lds[2][2][kWaves];
    int turn = 0;
    const int lane = threadIdx.x & 63;
    const int li = kWide ? threadIdx.x : lane & (plan.lanes - 1);
    const int per = 64 / (kWide ? 64 : plan.lanes);
    const int64_t place = kWide ? (int64_t)blockIdx.x
                                : ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * per + lane / plan.lanes;
    const int64_t row0 = place / a.g, gi = place - row0 * a.g;
    const bool live = place < plan.places;
    const uint64_t offset = drop_offset(a.drop);
    const float inv = 1.0f / (float)a.d;
    const int step = 8 * (kWide ? THREADS : plan.lanes);
    for (int64_t r0 = 0; r0 < a.n; r0 += plan.passes, turn ^= 1) {
        const int64_t row = r0 + row0;
        const bool ok = live && row < a.n;
        if (kWide && !ok) break;  // the whole workgroup
        const int64_t base = (row * a.g + gi) * a.d;
        float v[CPL][8];
        float sum[1] = {0.0f};
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const int64_t c = 8 * li + j * step;
            Oct<T> raw = {};
            if (ok && c < a.d) raw = load_oct(a.x + base, c, a.d);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[j][e] = (float)raw[e];
                sum[0] += v[j][e];
            }
        }
        if constexpr (kWide)
            block_sums<1, THREADS>(sum, lds[turn][0]);
        else
            lane_sums(sum, plan.lanes);
        const float mean = sum[0] / (float)a.d;  // exact where all are equal and few
        sum[0] = 0.0f;
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const int64_t c = 8 * li + j * step;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] -= mean;
            if (c + 8 <= a.d) {
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[0] = __builtin_fmaf(v[j][e], v[j][e], sum[0]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < a.d) sum[0] = __builtin_fmaf(v[j][e], v[j][e], sum[0]);
            }
        }
        if constexpr (kWide)
            block_sums<1, THREADS>(sum, lds[turn][1]);
        else
            lane_sums(sum, plan.lanes);
        const float rstd = 1.0f / sqrtf(__builtin_fmaf(sum[0], inv, a.eps));
        if (ok && li == 0 && a.mean) {
            a.mean[row * a.g + gi] = mean;
            a.rstd[row * a.g + gi] = rstd;
        }
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const int64_t c = 8 * li + j * step;
            if (!ok || c >= a.d) continue;
            float w[8], b[8];
            load_affine(a, gi * a.d + c, (gi + 1) * a.d, w, b);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] *= rstd;
            forward_oct(a, offset, base + c, w, b, v[j]);
            store_oct(a.y + base, c, a.d, v[j]);
        }
    }
}

template <typename T, int CPL, int THREADS>
__global__ __launch_bounds__(THREADS ? THREADS : 256) void norm_rows_grad_kernel(NormOperands<T> a, RowPlan plan) {
    constexpr bool kWide = THREADS > 0;
    constexpr int kWaves = kWide ? THREADS / 64 : 1;
    __shared__ float lds[2][2 * kWaves];
    const int lane = threadIdx.x & 63;
    const int li = kWide ? threadIdx.x : lane & (plan.lanes - 1);
    const int per = 64 / (kWide ? 64 : plan.lanes);
    const int64_t place = kWide ? (int64_t)blockIdx.x
                                : ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * per + lane / plan.lanes;
    const int64_t row0 = place / a.g, gi = place - row0 * a.g;
    const bool live = place < plan.places;
    const uint64_t offset = drop_offset(a.drop);
    const float inv = 1.0f / (float)a.d;
    const int step = 8 * (kWide ? THREADS : plan.lanes);
    float w[CPL][8], b[CPL][8], dw[CPL][8] = {}, db[CPL][8] = {};
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
        const int64_t c = 8 * li + j * step;
        load_affine(a, gi * a.d + c, live && c < a.d ? (gi + 1) * a.d : 0, w[j], b[j]);
    }
    int turn = 0;
    for (int64_t r0 = 0; r0 < a.n; r0 += plan.passes, turn ^= 1) {
        const int64_t row = r0 + row0;
        const bool ok = live && row < a.n;
        if (kWide && !ok) break;  // the whole workgroup
        const int64_t unit = row * a.g + gi, base = unit * a.d;
        float xh[CPL][8], t[CPL][8];
        const float mean = ok ? a.mean[unit] : 0.0f, rstd = ok ? a.rstd[unit] : 0.0f;
        Oct<T> rx[CPL] = {}, rd[CPL] = {};
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const int64_t c = 8 * li + j * step;
            if (ok && c < a.d) {
                rx[j] = load_oct(a.x + base, c, a.d);
                rd[j] = load_oct(a.dy + base, c, a.d);
            }
        }
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const int64_t c = 8 * li + j * step;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                xh[j][e] = ((float)rx[j][e] - mean) * rstd;
                t[j][e] = (float)rd[j][e];
                // past the group's end dy is zero, and so is what comes of it
                if (c + 8 > a.d && c + e >= a.d) xh[j][e] = 0.0f;
            }
            if (!ok || c >= a.d) continue;
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
            const int64_t c = 8 * li + j * step;
            if (!a.y || !ok || c >= a.d) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) t[j][e] = rstd * (t[j][e] - __builtin_fmaf(xh[j][e], m2, m1));
            store_oct(a.y + base, c, a.d, t[j]);
        }
    }
    if (!live) return;
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
        const int64_t c = 8 * li + j * step;
        if (c >= a.d) continue;
        if (a.pw) store_oct(a.pw + row0 * a.c + gi * a.d, c, a.d, dw[j]);
        if (a.pb) store_oct(a.pb + row0 * a.c + gi * a.d, c, a.d, db[j]);
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

// A thread's place in a slab.
struct SlabPlace {
    int32_t oct, row;   // row: -1 where the thread has nothing to do
    int32_t c0, width;  // the slab's first channel, and its channels
    int32_t groups;
};
template <typename T>
__device__ __forceinline__ SlabPlace slab_place(const NormOperands<T>& a, const SlabPlan& p, int32_t slab) {
    SlabPlace q;
    const int t = threadIdx.x;
    q.row = t / p.octs;
    q.oct = t - q.row * p.octs;
    const int64_t left = a.g - (int64_t)slab * p.groups;
    q.groups = (int32_t)(left < p.groups ? left : p.groups);
    q.c0 = (int32_t)(slab * p.groups * a.d);
    q.width = (int32_t)(q.groups * a.d);
    if (q.row >= p.rows || q.oct * 8 >= q.width) q.row = -1;
    return q;
}

// Where sums of the slab's groups are: few groups are added up by several waves each.
struct GroupSums {
    float* at;      // N x parts x groups
    int32_t parts, groups;
    __device__ __forceinline__ float get(int i, int32_t g) const {
        float v = at[i * parts * groups + g];
        for (int k = 1; k < parts; ++k) v += at[(i * parts + k) * groups + g];
        return v;
    }
};

// The sums over every group of N values of each of a thread's channels, in LDS.
// `lds`: N * rows * octs * 8 floats.  What channels past the slab's end hold is not
// read.
template <int N, int THREADS>
__device__ __forceinline__ GroupSums group_sums(const float (&v)[N][8], const SlabPlan& p, const SlabPlace& q,
                                                int32_t d, float* lds, float* out) {
    constexpr int kWaves = THREADS / 64;
    const int32_t line = p.octs * 8, size = p.rows * line;
    __syncthreads();  // what was there has been read
    if ((int)threadIdx.x < p.rows * p.octs) {
        const int t = threadIdx.x;  // row * octs + oct
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < 8; e += 4)
                *reinterpret_cast<f32x4*>(lds + i * size + t * 8 + e) =
                    f32x4{v[i][e], v[i][e + 1], v[i][e + 2], v[i][e + 3]};
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int parts = 1;
    while (parts * 2 * p.groups <= kWaves) parts *= 2;
    // the lanes of a wave side by side over the group's channels, and over rows
    int span = 1, shift = 0;
    while (span < 64 && span < d) {
        span *= 2;
        ++shift;
    }
    const int side = (64 >> shift) * parts, lc = lane & (span - 1);
    constexpr int U = 4;  // rows under way
    for (int w = wave; w < q.groups * parts; w += kWaves) {
        const int g = w / parts, part = w - g * parts;
        const int lr = (lane >> shift) * parts + part;
        float sum[N] = {};
        for (int c = lc; c < d; c += span) {
            const float* from = lds + g * d + c;
            for (int r = lr; r < p.rows; r += U * side) {
                float u[U][N] = {};
#pragma unroll
                for (int k = 0; k < U; ++k)
                    if (r + k * side < p.rows)
#pragma unroll
                        for (int i = 0; i < N; ++i) u[k][i] = from[i * size + (r + k * side) * line];
#pragma unroll
                for (int k = 0; k < U; ++k)
#pragma unroll
                    for (int i = 0; i < N; ++i) sum[i] += u[k][i];
            }
        }
        lane_sums(sum, 64);
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) out[(i * parts + part) * p.groups + g] = sum[i];
    }
    __syncthreads();
    return GroupSums{out, parts, p.groups};
}

// The groups of a thread's eight channels, of the slab (0 past its end).
template <typename F>
__device__ __forceinline__ void each_group(const SlabPlace& q, int32_t d, F f) {
    const int32_t c0 = 8 * q.oct;
    int32_t g = q.row >= 0 ? c0 / d : 0, in = c0 - g * d;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        f(e, q.row >= 0 && c0 + e < q.width ? g : 0);
        if (++in == d) {
            in = 0;
            ++g;
        }
    }
}

// The same sums over the rows alone, to memory.
template <int N>
__device__ __forceinline__ void channel_sums(const float (&v)[N][8], const SlabPlan& p, const SlabPlace& q,
                                             int threads, float* lds, float* const (&to)[N]) {
    const int32_t line = p.octs * 8, size = p.rows * line;
    __syncthreads();
    if ((int)threadIdx.x < p.rows * p.octs) {
        const int t = threadIdx.x;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < 8; e += 4)
                *reinterpret_cast<f32x4*>(lds + i * size + t * 8 + e) =
                    f32x4{v[i][e], v[i][e + 1], v[i][e + 2], v[i][e + 3]};
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (!to[i]) continue;
        for (int c = threadIdx.x; c < q.width; c += threads) {
            float sum = 0.0f;
            for (int r = 0; r < p.rows; ++r) sum += lds[i * size + r * line + c];
            to[i][q.c0 + c] = sum;
        }
    }
}

constexpr int kSlabGroups = 256;  // of a slab, at most

template <typename T, int M, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_resident_kernel(NormOperands<T> a, SlabPlan p) {
    __shared__ __attribute__((aligned(16))) float lds[THREADS * 8];
    __shared__ float sums[kSlabGroups];
    const uint64_t offset = drop_offset(a.drop);
    const float count = (float)a.s * (float)a.d, inv = 1.0f / count;
    const int32_t slab = (int32_t)blockIdx.x;
    const SlabPlace q = slab_place(a, p, slab);
    const int32_t d = (int32_t)a.d;
    int32_t gi[8];
    each_group(q, d, [&](int e, int32_t g) { gi[e] = g; });
    for (int64_t n = blockIdx.y; n < a.n; n += gridDim.y) {
        const int64_t c0 = 8 * (int64_t)q.oct;  // within the slab
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
        GroupSums total = group_sums<1, THREADS>(v, p, q, d, lds, sums);
        float mean[8], rstd[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            mean[e] = total.get(0, gi[e]) / count;
            v[0][e] = 0.0f;
        }
        if (q.row >= 0) {
#pragma unroll
            for (int i = 0; i < M; ++i) {
                if (q.row + (int64_t)i * p.rows >= a.s) continue;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float u = (float)raw[i][e] - mean[e];
                    if (c0 + e < q.width) v[0][e] = __builtin_fmaf(u, u, v[0][e]);
                }
            }
        }
        total = group_sums<1, THREADS>(v, p, q, d, lds, sums);
#pragma unroll
        for (int e = 0; e < 8; ++e) rstd[e] = 1.0f / sqrtf(__builtin_fmaf(total.get(0, gi[e]), inv, a.eps));
        if (q.row < 0) continue;
        if (a.mean && q.row == 0) {
            const int64_t at = n * a.g + (int64_t)slab * p.groups;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c0 + e < q.width && (int32_t)c0 + e == gi[e] * d) {
                    a.mean[at + gi[e]] = mean[e];
                    a.rstd[at + gi[e]] = rstd[e];
                }
        }
        float w[8], b[8];
        load_affine(a, q.c0 + c0, q.c0 + q.width, w, b);
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

// Workgroup (slab, place): samples place, place + across, ...
template <typename T, int M, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_resident_grad_kernel(NormOperands<T> a, SlabPlan p) {
    __shared__ __attribute__((aligned(16))) float lds[2 * THREADS * 8];
    __shared__ float sums[2 * kSlabGroups];
    const int32_t slab = (int32_t)blockIdx.x;
    const int64_t place = blockIdx.y;
    const uint64_t offset = drop_offset(a.drop);
    const float inv = 1.0f / ((float)a.s * (float)a.d);
    const SlabPlace q = slab_place(a, p, slab);
    const int32_t d = (int32_t)a.d;
    const int64_t c0 = 8 * (int64_t)q.oct;
    float w[8], b[8], total[2][8] = {};
    int32_t gi[8];
    load_affine(a, q.c0 + c0, q.row >= 0 ? q.c0 + q.width : 0, w, b);
    each_group(q, d, [&](int e, int32_t g) { gi[e] = g; });
    for (int64_t n = place; n < a.n; n += p.across) {
        const int64_t base = n * a.s * a.c + q.c0;
        Oct<T> rx[M] = {}, rd[M] = {};
        float mean[8], rstd[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int64_t at = n * a.g + (int64_t)slab * p.groups + gi[e];
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
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                total[k][e] += v[k][e];
                v[k][e] *= w[e];
            }
        if (!a.y) continue;
        const GroupSums group = group_sums<2, THREADS>(v, p, q, d, lds, sums);
        if (q.row < 0) continue;
        float m1[8], m2[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            m1[e] = group.get(0, gi[e]) * inv;
            m2[e] = group.get(1, gi[e]) * inv;
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
            for (int e = 0; e < 8; ++e)
                t[e] = rstd[e] * (t[e] * w[e] - __builtin_fmaf(xh[e], m2[e], m1[e]));
            store_oct(a.y + base + pos * a.c, c0, q.width, t);
        }
    }
    if (!a.pw && !a.pb) return;
    float* const to[2] = {a.pb ? a.pb + place * a.c : nullptr, a.pw ? a.pw + place * a.c : nullptr};
    channel_sums(total, p, q, THREADS, lds, to);
}

// ---------------------------------------------------------------------------
// split
// ---------------------------------------------------------------------------
// A run's statistics of every group: three floats, its mean, the sum of squares
// about it, and nothing else is needed: the counts follow from the run.  Each
// thread sums differences from its first row, a channel of its own, so that a
// large mean costs nothing.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS, 4) void norm_split_stats_kernel(NormOperands<T> a, SlabPlan p, float* part) {
    __shared__ __attribute__((aligned(16))) float lds[THREADS * 8];
    __shared__ float sums[kSlabGroups];
    const int32_t slab = (int32_t)blockIdx.x;
    const int64_t run = blockIdx.y;
    const SlabPlace q = slab_place(a, p, slab);
    const int32_t d = (int32_t)a.d;
    const int64_t c0 = 8 * (int64_t)q.oct;
    for (int64_t n = blockIdx.z; n < a.n; n += gridDim.z) {
        const int64_t s0 = run * p.run, s1 = s0 + p.run < a.s ? s0 + p.run : a.s;
        const T* from = a.x + n * a.s * a.c + q.c0;
        float first[8] = {}, sum[8] = {}, square[8] = {};
        int32_t count = 0;
        if (q.row >= 0 && s0 + q.row < s1) {
            const Oct<T> raw = load_oct(from + (s0 + q.row) * a.c, c0, q.width);
#pragma unroll
            for (int e = 0; e < 8; ++e) first[e] = (float)raw[e];
            count = 1;
            constexpr int U = 4;
            for (int64_t pos = s0 + q.row + p.rows; pos < s1; pos += U * p.rows) {
                Oct<T> v[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (pos + u * p.rows < s1) v[u] = load_oct(from + (pos + u * p.rows) * a.c, c0, q.width);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (pos + u * p.rows >= s1) continue;
                    ++count;
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
        float v[1][8], about[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float m = count ? sum[e] / (float)count : 0.0f;
            about[e] = square[e] - sum[e] * m;
            first[e] += m;  // the channel's mean
            v[0][e] = first[e] * (float)count;
        }
        GroupSums total = group_sums<1, THREADS>(v, p, q, d, lds, sums);
        const float size = (float)(s1 - s0) * (float)d;
        each_group(q, d, [&](int e, int32_t g) {
            const float far = first[e] - total.get(0, g) / size;
            v[0][e] = count ? __builtin_fmaf(far * far, (float)count, about[e]) : 0.0f;
        });
        const int64_t at = (n * p.across + run) * a.g + (int64_t)slab * p.groups;
        for (int g = threadIdx.x; g < q.groups; g += THREADS) part[2 * (at + g)] = total.get(0, g) / size;
        total = group_sums<1, THREADS>(v, p, q, d, lds, sums);
        for (int g = threadIdx.x; g < q.groups; g += THREADS) part[2 * (at + g) + 1] = total.get(0, g);
    }
}

// A run's share of the positions.
__device__ __forceinline__ float run_share(const SlabPlan& p, int64_t s, int64_t r) {
    return (float)(r + 1 < p.across ? p.run : s - r * p.run) / (float)s;
}

// Joins the runs of a sample's groups: the mean, and the squares about it.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS, 4) void norm_split_kernel(NormOperands<T> a, SlabPlan p, const float* part) {
    __shared__ float means[kSlabGroups], rstds[kSlabGroups];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t offset = drop_offset(a.drop);
    const int32_t slab = (int32_t)blockIdx.x;
    const int64_t run = blockIdx.y;
    const SlabPlace q = slab_place(a, p, slab);
    const int32_t d = (int32_t)a.d;
    const int64_t c0 = 8 * (int64_t)q.oct;
    for (int64_t n = blockIdx.z; n < a.n; n += gridDim.z) {
        __syncthreads();
        // a wave to a group, its lanes over the runs
        for (int g = wave; g < q.groups; g += THREADS / 64) {
            const float* f = part + 2 * (n * p.across * a.g + (int64_t)slab * p.groups + g);
            const int64_t step = 2 * a.g;
            const float first = f[0];
            float sum[1] = {0.0f};  // what the mean is beyond the first run's
            for (int64_t r = lane; r < p.across; r += 64)
                sum[0] = __builtin_fmaf(f[r * step] - first, run_share(p, a.s, r), sum[0]);
            lane_sums(sum, 64);
            const float mean = first + sum[0];
            sum[0] = 0.0f;
            for (int64_t r = lane; r < p.across; r += 64) {
                const float far = f[r * step] - mean;
                sum[0] += __builtin_fmaf(far * far, run_share(p, a.s, r) * (float)a.s * (float)d, f[r * step + 1]);
            }
            lane_sums(sum, 64);
            const float rstd = 1.0f / sqrtf(sum[0] / ((float)a.s * (float)d) + a.eps);
            if (lane) continue;
            means[g] = mean;
            rstds[g] = rstd;
            if (a.mean && run == 0) {
                a.mean[n * a.g + (int64_t)slab * p.groups + g] = mean;
                a.rstd[n * a.g + (int64_t)slab * p.groups + g] = rstd;
            }
        }
        __syncthreads();
        if (q.row < 0) continue;
        float w[8], b[8], mean[8], rstd[8];
        load_affine(a, q.c0 + c0, q.c0 + q.width, w, b);
        each_group(q, d, [&](int e, int32_t g) {
            mean[e] = means[g];
            rstd[e] = rstds[g];
        });
        const int64_t s0 = run * p.run, s1 = s0 + p.run < a.s ? s0 + p.run : a.s;
        const int64_t base = n * a.s * a.c + q.c0;
        constexpr int U = 4;
        for (int64_t pos = s0 + q.row; pos < s1; pos += U * p.rows) {
            Oct<T> v[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (pos + u * p.rows < s1) v[u] = load_oct(a.x + base + (pos + u * p.rows) * a.c, c0, q.width);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t at = pos + u * p.rows;
                if (at >= s1) continue;
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = ((float)v[u][e] - mean[e]) * rstd[e];
                forward_oct(a, offset, base + at * a.c + c0, w, b, f);
                store_oct(a.y + base + at * a.c, c0, q.width, f);
            }
        }
    }
}

// Backwards: of every run the groups' two sums (part), and the channels' (pw, pb).
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS, 4) void norm_split_sums_kernel(NormOperands<T> a, SlabPlan p, float* part) {
    __shared__ __attribute__((aligned(16))) float lds[2 * THREADS * 8];
    __shared__ float sums[2 * kSlabGroups];
    const uint64_t offset = drop_offset(a.drop);
    const int32_t slab = (int32_t)blockIdx.x;
    const int64_t run = blockIdx.y;
    const SlabPlace q = slab_place(a, p, slab);
    const int32_t d = (int32_t)a.d;
    const int64_t c0 = 8 * (int64_t)q.oct;
    for (int64_t n = blockIdx.z; n < a.n; n += gridDim.z) {
        const int64_t s0 = run * p.run, s1 = s0 + p.run < a.s ? s0 + p.run : a.s;
        const int64_t base = n * a.s * a.c + q.c0;
        float w[8], b[8], mean[8], rstd[8], v[2][8] = {};
        load_affine(a, q.c0 + c0, q.row >= 0 ? q.c0 + q.width : 0, w, b);
        each_group(q, d, [&](int e, int32_t g) {
            mean[e] = a.mean[n * a.g + (int64_t)slab * p.groups + g];
            rstd[e] = a.rstd[n * a.g + (int64_t)slab * p.groups + g];
        });
        if (q.row >= 0) {
            constexpr int U = 2;
            for (int64_t pos = s0 + q.row; pos < s1; pos += U * p.rows) {
                Oct<T> rx[U], rd[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (pos + u * p.rows < s1) {
                        rx[u] = load_oct(a.x + base + (pos + u * p.rows) * a.c, c0, q.width);
                        rd[u] = load_oct(a.dy + base + (pos + u * p.rows) * a.c, c0, q.width);
                    }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t at = pos + u * p.rows;
                    if (at >= s1) continue;
                    float xh[8], t[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        xh[e] = ((float)rx[u][e] - mean[e]) * rstd[e];
                        t[e] = (float)rd[u][e];
                    }
                    backward_oct(a, offset, base + at * a.c + c0, w, b, xh, t);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        v[0][e] += t[e];
                        v[1][e] = __builtin_fmaf(t[e], xh[e], v[1][e]);
                    }
                }
            }
        }
        const int64_t at = n * p.across + run;
        float* const to[2] = {a.pb ? a.pb + at * a.c : nullptr, a.pw ? a.pw + at * a.c : nullptr};
        channel_sums(v, p, q, THREADS, lds, to);
        if (!a.y) continue;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] *= w[e];
        const GroupSums group = group_sums<2, THREADS>(v, p, q, d, lds, sums);
        for (int g = threadIdx.x; g < q.groups; g += THREADS) {
            float* const to2 = part + 2 * (at * a.g + (int64_t)slab * p.groups + g);
            to2[0] = group.get(0, g);
            to2[1] = group.get(1, g);
        }
    }
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS, 4) void norm_split_grad_kernel(NormOperands<T> a, SlabPlan p, const float* part) {
    __shared__ float m1s[kSlabGroups], m2s[kSlabGroups];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t offset = drop_offset(a.drop);
    const float inv = 1.0f / ((float)a.s * (float)a.d);
    const int32_t slab = (int32_t)blockIdx.x;
    const int64_t run = blockIdx.y;
    const SlabPlace q = slab_place(a, p, slab);
    const int32_t d = (int32_t)a.d;
    const int64_t c0 = 8 * (int64_t)q.oct;
    for (int64_t n = blockIdx.z; n < a.n; n += gridDim.z) {
        __syncthreads();
        for (int g = wave; g < q.groups; g += THREADS / 64) {  // a wave to a group, its lanes over the runs
            const float* f = part + 2 * (n * p.across * a.g + (int64_t)slab * p.groups + g);
            float sum[2] = {0.0f, 0.0f};
            for (int64_t r = lane; r < p.across; r += 64) {
                sum[0] += f[2 * r * a.g];
                sum[1] += f[2 * r * a.g + 1];
            }
            lane_sums(sum, 64);
            if (lane) continue;
            m1s[g] = sum[0] * inv;
            m2s[g] = sum[1] * inv;
        }
        __syncthreads();
        if (q.row < 0) continue;
        float w[8], b[8], mean[8], rstd[8], m1[8], m2[8];
        load_affine(a, q.c0 + c0, q.c0 + q.width, w, b);
        each_group(q, d, [&](int e, int32_t g) {
            mean[e] = a.mean[n * a.g + (int64_t)slab * p.groups + g];
            rstd[e] = a.rstd[n * a.g + (int64_t)slab * p.groups + g];
            m1[e] = m1s[g];
            m2[e] = m2s[g];
        });
        const int64_t s0 = run * p.run, s1 = s0 + p.run < a.s ? s0 + p.run : a.s;
        const int64_t base = n * a.s * a.c + q.c0;
        constexpr int U = 2;
        for (int64_t pos = s0 + q.row; pos < s1; pos += U * p.rows) {
            Oct<T> rx[U], rd[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (pos + u * p.rows < s1) {
                    rx[u] = load_oct(a.x + base + (pos + u * p.rows) * a.c, c0, q.width);
                    rd[u] = load_oct(a.dy + base + (pos + u * p.rows) * a.c, c0, q.width);
                }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t at = pos + u * p.rows;
                if (at >= s1) continue;
                float xh[8], t[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    xh[e] = ((float)rx[u][e] - mean[e]) * rstd[e];
                    t[e] = (float)rd[u][e];
                }
                backward_oct(a, offset, base + at * a.c + c0, w, b, xh, t);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    t[e] = rstd[e] * (t[e] * w[e] - __builtin_fmaf(xh[e], m2[e], m1[e]));
                store_oct(a.y + base + at * a.c, c0, q.width, t);
            }
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
        const int64_t side = std::max<int64_t>(1, blocks * units / g);  // samples side by side
        o.row.passes = ceil_div(n, ceil_div(n, side));
        o.row.places = o.row.passes * g;
        o.blocks = ceil_div(o.row.places, units);
        o.parts = o.row.passes;
        return o;
    }
    // the slab: whole groups, as few as make a line of memory
    auto slab = [&](int threads, int64_t groups) {
        SlabPlan p{};
        p.groups = (int32_t)groups;
        p.octs = (int32_t)ceil_div(groups * d, 8);
        p.rows = threads / p.octs;
        p.slabs = (int32_t)ceil_div(g, groups);
        return p;
    };
    const int64_t line = std::min<int64_t>(g, std::max<int64_t>(1, ceil_div(128 / elem_bytes, d)));
    const int most = elem_bytes == 4 && grad ? 4 : 8;
    for (int threads : {256, 512}) {
        const SlabPlan p = slab(threads, std::min<int64_t>(line, kSlabGroups));
        if (p.octs > threads || ceil_div(s, p.rows) > most) continue;
        o.kind = Way::kResident;
        o.threads = threads;
        const int64_t m = ceil_div(s, p.rows);
        o.m = m <= 2 ? 2 : m <= 4 ? 4 : 8;
        o.slab = p;
        const int64_t side = std::max<int64_t>(1, (int64_t)cus * (threads == 256 ? 4 : 2) / p.slabs);
        o.slab.across = grad ? ceil_div(n, ceil_div(n, std::min<int64_t>({n, side, 65535}))) : n;
        o.side = std::min<int64_t>(grad ? o.slab.across : n, 65535);
        o.parts = o.slab.across;
        return o;
    }
    o.kind = Way::kSplit;
    o.threads = octs <= 512 ? 512 : 1024;
    // as many whole groups as the threads have room for
    const int64_t groups = std::max<int64_t>(1, std::min<int64_t>({g, kSlabGroups, (int64_t)o.threads * 8 / d}));
    o.slab = slab(o.threads, groups);
    const int64_t want = ceil_div((int64_t)cus * 4, n * o.slab.slabs);
    const int64_t rows = std::max<int64_t>(ceil_div(s, std::max<int64_t>(1, want)), 4 * (int64_t)o.slab.rows);
    o.slab.run = std::min(rows, s);
    o.slab.across = ceil_div(s, o.slab.run);
    o.side = std::min<int64_t>(n, 65535);
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
    MLRS_SLAB(2, 256)
    MLRS_SLAB(4, 256)
    MLRS_SLAB(2, 512)
    MLRS_SLAB(4, 512)
    if constexpr (!GRAD || sizeof(T) == 2) {
        MLRS_SLAB(8, 256)
        MLRS_SLAB(8, 512)
    }
#undef MLRS_SLAB
    return hipErrorInvalidValue;
}

template <typename T>
NormOperands<T> operands(const NormCall& k) {
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
    const NormOperands<T> a = operands<T>(k);
    if (o.kind == Way::kRows) return launch_rows<T, false>(a, o, s);
    if (o.kind == Way::kResident) return launch_resident<T, false>(a, o, s);
    const dim3 grid((unsigned)o.slab.slabs, (unsigned)o.slab.across, (unsigned)o.side);
    if (o.threads == 512)
        norm_split_stats_kernel<T, 512><<<grid, 512, 0, s>>>(a, o.slab, scratch);
    else
        norm_split_stats_kernel<T, 1024><<<grid, 1024, 0, s>>>(a, o.slab, scratch);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (o.threads == 512)
        norm_split_kernel<T, 512><<<grid, 512, 0, s>>>(a, o.slab, scratch);
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
    NormOperands<T> a = operands<T>(k);
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
        if (o.threads == 512)
            norm_split_sums_kernel<T, 512><<<grid, 512, 0, s>>>(a, o.slab, at);
        else
            norm_split_sums_kernel<T, 1024><<<grid, 1024, 0, s>>>(a, o.slab, at);
        e = hipGetLastError();
        if (e == hipSuccess && k.y) {
            if (o.threads == 512)
                norm_split_grad_kernel<T, 512><<<grid, 512, 0, s>>>(a, o.slab, at);
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
