// A layer forwards and backwards: y = act(x w^T + bias) + residual, and the
// products dz w and dz^T x of its gradient.
#include <cmath>

#include "train_launch.hpp"

namespace mlrs {
namespace train {

// ---------------------------------------------------------------------------
// how a product is cut
// ---------------------------------------------------------------------------
// The time of each choice, in microseconds, from measurements on this chip:
// a staged width (128 bytes of k) of the one, two, ... tiles that a CU holds at
// a time, and what a round of tiles costs besides (its first copies, its
// epilogue).  16-bit tiles are bound by LDS and copies, so a CU that holds one
// of the smaller tiles is far from twice as fast as one that holds two; f32
// tiles are bound by the matrix cores, and only the count matters.  Measured at
// 2048 x 1024 x 4096 in bf16: 32.1 us in 256 x 256 tiles, 24.8 in 128 x 128,
// 33.8 in 64 x 64; at 16384 x 4096 x 4096: 433, 513, -.
static const double kStage16[3][3] = {{1.6}, {0.62, 0.98}, {0.27, 0.5, 0.75}};
static const double kStage32[3][3] = {{7.4}, {2.0, 4.0}, {0.68, 1.05, 1.55}};
static const double kRoundUs[3] = {6.0, 4.5, 4.0};
static const int kResident[3] = {1, 2, 3};

// Joining parts: a launch, and their bytes twice.
static double join_us(int64_t elements) { return elements ? 10.0 + (double)elements * 8.0 / 4.5e6 : 0.0; }

Cut choose_cut(int elem_bytes, int64_t m, int64_t n, int64_t k, int cus, int max_splits, bool words) {
    const int64_t per = kStageBytes / elem_bytes;
    const int64_t stages = std::max<int64_t>(1, (k + per - 1) / per);
    Cut best{0, 1, 0, 1e300};
    for (int t = words ? 2 : 0; t < 3; ++t) {
        const double* stage = elem_bytes == 2 ? kStage16[t] : kStage32[t];
        const int rows = kTileRows[t];
        const int64_t tiles = ((m + rows - 1) / rows) * ((n + rows - 1) / rows);
        for (int64_t sp = 1; sp <= max_splits && sp <= stages; sp = sp < 4 ? sp + 1 : sp * 2) {
            const int64_t each = (stages + sp - 1) / sp;
            if (sp > 1 && (each < 3 || (sp - 1) * each >= stages)) continue;
            if ((t > 0 || sp > 1) && !launchable(tiles * sp, kTileThreads[t])) continue;
            const int64_t on_cu = (tiles * sp + cus - 1) / cus;  // tiles that the busiest CU computes
            const int64_t rounds = on_cu / kResident[t], rest = on_cu % kResident[t];
            double cost = (double)rounds * ((double)each * stage[kResident[t] - 1] + kRoundUs[t]);
            if (rest) cost += (double)each * stage[rest - 1] + kRoundUs[t];
            if (sp > 1) cost += join_us(sp * m * n);
            if (cost < best.us) best = Cut{words ? 3 : t, (int)sp, (int32_t)(each * per), cost};
        }
    }
    return best;
}

// When the last of two kinds of workgroups is done, `first` of which go to `slots`
// places before `then` of the other: places that fall free together are taken
// together.
static double last_done(int64_t first, double first_us, int64_t then, double then_us, int64_t slots) {
    struct Group {
        double at;
        int64_t size;
    } g[3] = {{(double)(first / slots) * first_us, slots - first % slots},
              {(double)(first / slots + 1) * first_us, first % slots},
              {0.0, 0}};
    const int64_t rounds = std::max<int64_t>(0, then / slots - 8);  // of many, all but a few at once
    then -= rounds * slots;
    for (Group& o : g) o.at += (double)rounds * then_us;
    while (then > 0) {
        Group& o = g[1].size && g[1].at < g[0].at ? g[1] : g[0];
        const int64_t n = std::min(then, o.size);
        if (n < o.size) g[2] = Group{o.at + then_us, n};
        else o.at += then_us;
        then -= n;
    }
    double end = 0.0;
    for (const Group& o : g)
        if (o.size) end = std::max(end, o.at);
    return end;
}

// Two products in one grid: what the places of a full CU need for both, and of
// what its last workgroups need beyond that a part, as a CU that is left to few of
// them is faster for each; no less than the longest workgroup alone.  Over thirty
// layers in bf16 and f32 of 64 to 30,000 rows and 96 to 10,000 columns the choice
// was 2% slower than the best of some sixty cuts each, 13% at most, and in bf16 a
// fifth to a third faster than the best two launches below 100 us: 4099 x 2056 by
// 1000 takes 55 us, 66 in two; 2048^3 36 and 53; 16020 x 960 by 2816 174 and 202.
PairCut choose_pair(int elem_bytes, int64_t xm, int64_t xn, int64_t xk, int64_t wm, int64_t wn, int64_t wk, int cus,
                    bool words) {
    PairCut best{choose_cut(elem_bytes, xm, xn, xk, cus, 64, words), choose_cut(elem_bytes, wm, wn, wk, cus, 64, words),
                 false, 0.0};
    best.us = best.x.us + best.w.us + 3.0;  // another launch
    const int64_t per = kStageBytes / elem_bytes;
    const int64_t xs = std::max<int64_t>(1, (xk + per - 1) / per), ws = std::max<int64_t>(1, (wk + per - 1) / per);
    auto next = [](int64_t sp) { return sp < 4 ? sp + 1 : sp * 2; };
    for (int t = words ? 2 : 0; t < 3; ++t) {
        const double* stage = elem_bytes == 2 ? kStage16[t] : kStage32[t];
        const int rows = kTileRows[t];
        const int64_t xt = ((xm + rows - 1) / rows) * ((xn + rows - 1) / rows);
        const int64_t wt = ((wm + rows - 1) / rows) * ((wn + rows - 1) / rows);
        for (int64_t sx = 1; sx <= 64; sx = next(sx)) {
            const int64_t ex = (xs + sx - 1) / sx;
            if (sx > 1 && (ex < 3 || (sx - 1) * ex >= xs || xt * sx > 8 * cus)) continue;
            for (int64_t sw = 1; sw <= 64; sw = next(sw)) {
                const int64_t ew = (ws + sw - 1) / sw;
                if (sw > 1 && (ew < 3 || (sw - 1) * ew >= ws || wt * sw > 8 * cus)) continue;
                const int64_t count = xt * sx + wt * sw;
                if (!launchable(count, kTileThreads[t])) continue;
                const int64_t full = std::min<int64_t>(kResident[t], (count + cus - 1) / cus), slots = full * cus;
                const double ux = (double)ex * stage[full - 1] + kRoundUs[t], uw = (double)ew * stage[full - 1] + kRoundUs[t];
                const double all = ((double)(xt * sx) * ux + (double)(wt * sw) * uw) / (double)slots;
                const double end = ex >= ew ? last_done(xt * sx, ux, wt * sw, uw, slots)
                                            : last_done(wt * sw, uw, xt * sx, ux, slots);
                double cost = std::max(all + 0.6 * (end - all) * stage[0] / stage[full - 1],
                                       (double)std::max(ex, ew) * stage[0] + kRoundUs[t]);
                cost += join_us((sx > 1 ? sx * xm * xn : 0) + (sw > 1 ? sw * wm * wn : 0));
                if (cost < best.us) {
                    const int tile = words ? 3 : t;
                    best = PairCut{Cut{tile, (int)sx, (int32_t)(ex * per), cost},
                                   Cut{tile, (int)sw, (int32_t)(ew * per), cost}, true, cost};
                }
            }
        }
    }
    return best;
}

// ---------------------------------------------------------------------------
// packing
// ---------------------------------------------------------------------------
// Two matrices in a launch: both operands of a product are usually packed.
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(PackJob a, PackJob b, Only only) {
    if (skipped(only.flag, only.mark, only.wanted)) return;
    constexpr int E = 16 / (int)sizeof(T);
    const int64_t total_a = a.rows * (a.ld / E), total = total_a + b.rows * (b.ld / E);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const PackJob& j = i < total_a ? a : b;
        const int64_t at = i < total_a ? i : i - total_a;
        const int64_t chunks = j.ld / E, r = at / chunks, c = (at - r * chunks) * E;
        const T* from = (const T*)j.src + r * j.cols;
        typename Elem<T>::Frag v;
        if (c + E <= j.cols) {
            __builtin_memcpy(&v, from + c, sizeof v);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = c + e < j.cols ? from[c + e] : (T)0.0f;
        }
        *reinterpret_cast<typename Elem<T>::Frag*>((T*)j.dst + r * j.ld + c) = v;
    }
}

template <typename T>
hipError_t launch_pack(const PackJob& a, const PackJob& b, const Only& only, hipStream_t s) {
    const int64_t total = (a.rows * a.ld + b.rows * b.ld) / (16 / (int64_t)sizeof(T));
    if (total == 0) return hipSuccess;
    const int64_t blocks = std::min<int64_t>((total + 255) / 256, 16384);
    pack_kernel<T><<<dim3((unsigned)blocks), 256, 0, s>>>(a, b, only);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// forwards
// ---------------------------------------------------------------------------
template <typename T>
hipError_t launch_linear(Mat x, Mat w, int64_t n, int64_t m, int64_t k, const LinearOut& o, const Cut& cut,
                         float* part, const Only& only, hipStream_t s) {
    const LinearEpi<T> e = linear_epi<T>(o, m);
    if (cut.splits == 1) return launch_gemm<T>(cut.tile, w, x, m, n, k, 1, 0, only, e, s);
    const hipError_t r = launch_gemm<T>(cut.tile, w, x, m, n, k, cut.splits, cut.k_split, only,
                                                    parts_epi<T>(part, m, n), s);
    if (r != hipSuccess) return r;
    return launch_join(part, cut.splits, m, n, LinearPoint<T>{e}, only, s);
}

template <typename T>
hipError_t launch_logit_parts(Mat h, Mat w, int64_t n, int64_t classes, int64_t k, const Cut& cut, float* part,
                              hipStream_t s) {
    return launch_gemm<T>(cut.tile, w, h, classes, n, k, cut.splits, cut.k_split, Only{},
                          parts_epi<T>(part, classes, n), s);
}

// A few rows: the weights are read once, straight into registers as the
// fragments of the matrix instructions.  A workgroup computes
// sixteen outputs of every row; its waves take the contraction axis in turn
// and their sums are joined in LDS, in the order of the waves.
template <typename T>
__device__ __forceinline__ typename Elem<T>::Frag chunk_at(const T* row, int64_t c, int64_t k) {
    constexpr int E = 16 / (int)sizeof(T);
    typename Elem<T>::Frag f;
    if (c + E <= k) {
        __builtin_memcpy(&f, row + c, sizeof f);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = c + e < k ? row[c + e] : (T)0.0f;
    }
    return f;
}

template <typename T, int NB, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void linear_few_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                                int32_t n, int32_t m, int64_t k, int32_t first,
                                                                LinearEpi<T> epi) {
    constexpr int E = 16 / (int)sizeof(T);
    constexpr int STEP = 4 * E;  // of k per wave and step
    __shared__ f32x4 sums[WAVES][NB][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int32_t m0 = first + (int32_t)blockIdx.x * 16;
    const T* wr = w + (int64_t)(m0 + r < m ? m0 + r : m - 1) * k;
    const T* xr[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) xr[b] = x + (int64_t)(b * 16 + r < n ? b * 16 + r : n - 1) * k;
    f32x4 acc[NB] = {};
    constexpr int U = 4;  // steps in flight
    for (int64_t k0 = (int64_t)wave * (U * STEP); k0 < k; k0 += (int64_t)WAVES * (U * STEP)) {
        typename Elem<T>::Frag a[U], bx[NB][U];
#pragma unroll
        for (int u = 0; u < U; ++u) a[u] = chunk_at<T>(wr, k0 + u * STEP + q * E, k);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int u = 0; u < U; ++u) bx[b][u] = chunk_at<T>(xr[b], k0 + u * STEP + q * E, k);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int u = 0; u < U; ++u) acc[b] = mfma_step<T>(a[u], bx[b][u], acc[b]);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) sums[wave][b][lane] = acc[b];
    __syncthreads();
    // wave b joins the sums of rows 16 b .. 16 b + 15
    for (int b = wave; b < NB; b += WAVES) {
        f32x4 v = sums[0][b][lane];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) v += sums[i][b][lane];
        const int32_t row = b * 16 + r, c = m0 + 4 * q;
        if (row < n && c < m) epi.point(row, c, m, v);
    }
}

template <typename T, int NB>
static hipError_t launch_few_nb(const T* x, const T* w, int64_t n, int64_t m, int64_t k, const LinearEpi<T>& e,
                                hipStream_t s) {
    constexpr int64_t kMost = (int64_t)1 << 26;  // outputs of a launch: half of what its threads could be
    for (int64_t first = 0; first < m; first += kMost) {
        const int64_t here = std::min(kMost, m - first);
        linear_few_kernel<T, NB, 8><<<dim3((unsigned)((here + 15) / 16)), 512, 0, s>>>(x, w, (int32_t)n, (int32_t)m, k,
                                                                                      (int32_t)first, e);
        const hipError_t r = hipGetLastError();
        if (r != hipSuccess) return r;
    }
    return hipSuccess;
}

template <typename T>
hipError_t launch_linear_few(const T* x, const T* w, int64_t n, int64_t m, int64_t k, const LinearOut& o,
                             hipStream_t s) {
    const LinearEpi<T> e = linear_epi<T>(o, m);
    return n <= 16 ? launch_few_nb<T, 1>(x, w, n, m, k, e, s) : launch_few_nb<T, 2>(x, w, n, m, k, e, s);
}

// Sixteen rows are bound by reading the weights (8192 x 8192 bf16: 29 us at one
// row, 35 at sixteen, of a floor of 28; in 64 x 64 tiles 35 from the first row
// on); thirty-two read twice as many fragments of x from the caches for them (47
// us), and the tiles are as fast or faster where there are weights enough.
bool few_rows(int elem_bytes, int64_t n, int64_t m, int64_t k, const Cut& cut) {
    if (n <= 16) return true;
    if (n > 32) return false;
    return 4.0 + 1.6 * (double)elem_bytes * (double)m * (double)k / 4.75e6 < cut.us;
}

// ---------------------------------------------------------------------------
// backwards
// ---------------------------------------------------------------------------
// A workgroup takes 256 columns (four per lane) and a run of rows, at least eight
// where there are more; its four waves take rows in turn and their sums are joined
// in order.  A single run is the column sum itself: it goes out at once; the grid
// of the products joins several, so that they cost no launch.
int column_parts(int64_t n, int64_t m, int cus) {
    const int64_t across = std::max<int64_t>(1, (m + 255) / 256);
    const int64_t want = std::max<int64_t>(1, (int64_t)cus * 8 / across);
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, 256), (n + 7) / 8));
}

// dz leaves in the operands' type, as the matrix instructions of the two products
// take it; the column sums add it up in f32, unrounded.  With a 16-bit dz the
// products' error against 64 bits is 2.3e-3 in bf16 (8192 x 2048 by 8192) and
// 2.9e-4 in f16, where rounding the results alone makes 1.7e-3 and 2.1e-4; a dz in
// two parts would double the products.
template <typename T>
__global__ __launch_bounds__(256) void act_grad_kernel(const T* __restrict__ dy, const T* __restrict__ z, int act,
                                                       int64_t n, int64_t m, T* __restrict__ dz, int64_t ld,
                                                       ColumnSums<T> sums, int64_t rows_per) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = ((int64_t)blockIdx.x * 64 + lane) * 4;
    const int64_t r0 = (int64_t)blockIdx.y * rows_per;
    const int64_t r1 = r0 + rows_per < n ? r0 + rows_per : n;
    f32x4 sum = {};
    if (c < (dz ? ld : m)) {
        constexpr int kRows = 2;  // of a wave, under way at once
        for (int64_t r = r0 + wave; r < r1; r += 4 * kRows) {
            f32x4 v[kRows] = {}, zz[kRows] = {};
#pragma unroll
            for (int u = 0; u < kRows; ++u)
                if (r + 4 * u < r1) v[u] = load4(dy + (r + 4 * u) * m, c, m);
            if (z) {
#pragma unroll
                for (int u = 0; u < kRows; ++u)
                    if (r + 4 * u < r1) zz[u] = load4(z + (r + 4 * u) * m, c, m);
            }
#pragma unroll
            for (int u = 0; u < kRows; ++u) {
                if (z) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[u][e] *= activate_slope(zz[u][e], act);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e >= m || r + 4 * u >= r1) v[u][e] = 0.0f;
                sum += v[u];
                if (dz && r + 4 * u < r1) store4(dz + (r + 4 * u) * ld, c, ld, v[u]);
            }
        }
    }
    if (!sums.out) return;
    __shared__ f32x4 join[4][64];
    join[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && c < m) {
        f32x4 v = join[0][lane];
#pragma unroll
        for (int i = 1; i < 4; ++i) v += join[i][lane];
        if (gridDim.y == 1)
            store4(sums.out, c, m, v);
        else
            store4(sums.sums + (int64_t)blockIdx.y * m, c, m, v);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void sum_parts_kernel(ColumnSums<T> to, int64_t m) {
    __shared__ float join[256];
    sum_parts<T, 256>(to, m, blockIdx.x, join);
}

template <typename T>
hipError_t launch_act_grad(const T* dy, const T* z, int act, int64_t n, int64_t m, T* dz, int64_t ld,
                           const ColumnSums<T>& sums, hipStream_t s) {
    const int64_t across = ((dz ? ld : m) + 255) / 256;
    if (across == 0 || (n == 0 && !sums.out)) return hipSuccess;
    const int64_t rows_per = (n + sums.parts - 1) / sums.parts;
    act_grad_kernel<T><<<dim3((unsigned)across, (unsigned)sums.parts), 256, 0, s>>>(dy, z, act, n, m, dz, ld, sums,
                                                                                   rows_per);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_sum_parts(const ColumnSums<T>& to, int64_t m, hipStream_t s) {
    if (!to.out) return hipSuccess;
    if (!launchable((m + 15) / 16, 256)) return hipErrorInvalidConfiguration;  // the caller has checked
    sum_parts_kernel<T><<<dim3((unsigned)((m + 15) / 16)), 256, 0, s>>>(to, m);
    return hipGetLastError();
}

// Both products of a gradient in one grid, and the column sums' join: none needs
// another's results, and the workgroups of one fill the CUs that the last ones
// of the other leave.
template <typename T>
struct PairArgs {
    GemmArgs x, w;
    StoreEpi<T> to_x, to_w;
    int32_t x_wgs, w_wgs;
    bool x_first;  // the one with the longer workgroups
    ColumnSums<T> sums;
    int64_t columns;
};
template <typename T, int WM, int WN, int MB, int NB, int BYTES = 16>
__global__ __launch_bounds__(WM* WN * 64, 2) void pair_kernel(PairArgs<T> q) {
    __shared__ __attribute__((aligned(1024))) char buf[gemm_lds<WM, MB, NB>()];
    if (skipped(q.x)) return;  // both have the same flag
    int32_t wg = blockIdx.x;
    const int32_t lead = q.x_first ? q.x_wgs : q.w_wgs;
    if (wg >= q.x_wgs + q.w_wgs) {
        sum_parts<T, WM * WN * 64>(q.sums, q.columns, wg - q.x_wgs - q.w_wgs, reinterpret_cast<float*>(buf));
        return;
    }
    const bool second = wg >= lead;
    if (second) wg -= lead;
    if (second != q.x_first)
        gemm_workgroup<T, false, true, WM, WN, MB, NB, StoreEpi<T>, BYTES>(q.x, q.to_x, wg, buf);
    else
        gemm_workgroup<T, false, false, WM, WN, MB, NB, StoreEpi<T>, BYTES>(q.w, q.to_w, wg, buf);
}

template <typename T>
static hipError_t launch_pair(const Product& x, const Product& w, const Cut& cx, const Cut& cw, float* part,
                              const ColumnSums<T>& sums, int64_t columns, const Only& only, hipStream_t s) {
    PairArgs<T> q;
    const int tile = x.m ? cx.tile : cw.tile;
    int64_t wgs[2];
    float* parts[2] = {part, part + (x.m ? cx.part_bytes(x.m, x.n) / 4 : 0)};
    const StoreEpi<T> to[2] = {store_epi<T>(x.to), store_epi<T>(w.to)};
    wgs[0] = gemm_args(q.x, tile, x.a, x.b, x.m, x.n, x.k, cx.splits, cx.k_split, only);
    wgs[1] = gemm_args(q.w, tile, w.a, w.b, w.m, w.n, w.k, cw.splits, cw.k_split, only);
    q.to_x = cx.splits > 1 ? parts_epi<T>(parts[0], x.m, x.n) : to[0];
    q.to_w = cw.splits > 1 ? parts_epi<T>(parts[1], w.m, w.n) : to[1];
    q.x_wgs = (int32_t)wgs[0];
    q.w_wgs = (int32_t)wgs[1];
    q.x_first = q.x.k_split >= q.w.k_split;
    q.sums = sums;
    q.columns = columns;
    int64_t blocks = wgs[0] + wgs[1] + (sums.out ? (columns + 15) / 16 : 0);
    if (blocks == 0) return hipSuccess;
    if (sums.out && !launchable(blocks, kTileThreads[tile])) {
        const hipError_t e = launch_sum_parts(sums, columns, s);
        if (e != hipSuccess) return e;
        blocks = wgs[0] + wgs[1];
    }
    if (!launchable(blocks, kTileThreads[tile])) return hipErrorInvalidConfiguration;  // the caller has checked
    const dim3 grid((unsigned)blocks);
    if (tile == 0)
        pair_kernel<T, 2, 4, 8, 4><<<grid, 512, 0, s>>>(q);
    else if (tile == 1)
        pair_kernel<T, 2, 2, 4, 4><<<grid, 256, 0, s>>>(q);
    else if (tile == 2)
        pair_kernel<T, 2, 2, 2, 2><<<grid, 256, 0, s>>>(q);
    else if constexpr (sizeof(T) == 4)
        pair_kernel<T, 2, 2, 2, 2, 4><<<grid, 256, 0, s>>>(q);
    else
        return hipErrorInvalidValue;
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    typedef JoinJob<StorePoint<T>> Job;
    return launch_join(Job{parts[0], x.m && cx.splits > 1 ? cx.splits : 0, x.m, x.n, StorePoint<T>{to[0]}},
                       Job{parts[1], w.m && cw.splits > 1 ? cw.splits : 0, w.m, w.n, StorePoint<T>{to[1]}}, only, s);
}

template <typename T>
hipError_t launch_products(const Product& x, const Product& w, const PairCut& cut, float* part,
                           const ColumnSums<T>& sums, int64_t columns, const Only& only, hipStream_t s) {
    if (cut.together || !x.m || !w.m) return launch_pair<T>(x, w, cut.x, cut.w, part, sums, columns, only, s);
    const hipError_t e = launch_pair<T>(Product{}, w, Cut{}, cut.w, part, sums, columns, only, s);
    if (e != hipSuccess) return e;
    return launch_pair<T>(x, Product{}, cut.x, Cut{}, part, ColumnSums<T>{}, 0, only, s);
}

#define MLRS_INST(T)                                                                                               \
    template hipError_t launch_pack<T>(const PackJob&, const PackJob&, const Only&, hipStream_t);                  \
    template hipError_t launch_linear<T>(Mat, Mat, int64_t, int64_t, int64_t, const LinearOut&, const Cut&, float*, \
                                         const Only&, hipStream_t);                                                \
    template hipError_t launch_logit_parts<T>(Mat, Mat, int64_t, int64_t, int64_t, const Cut&, float*,             \
                                              hipStream_t);                                                        \
    template hipError_t launch_linear_few<T>(const T*, const T*, int64_t, int64_t, int64_t, const LinearOut&,      \
                                             hipStream_t);                                                         \
    template hipError_t launch_act_grad<T>(const T*, const T*, int, int64_t, int64_t, T*, int64_t,                 \
                                           const ColumnSums<T>&, hipStream_t);                                     \
    template hipError_t launch_sum_parts<T>(const ColumnSums<T>&, int64_t, hipStream_t);                           \
    template hipError_t launch_products<T>(const Product&, const Product&, const PairCut&, float*,                 \
                                           const ColumnSums<T>&, int64_t, const Only&, hipStream_t);
MLRS_INST(float)
MLRS_INST(_Float16)
MLRS_INST(__bf16)

}  // namespace train
}  // namespace mlrs
