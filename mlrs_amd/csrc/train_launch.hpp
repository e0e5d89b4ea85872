// Launching the matrix-core products of the training operators.
#pragma once
#include <algorithm>

#include "train_epilogue.hpp"
#include "train_kernels.hpp"

namespace mlrs {
namespace train {

constexpr int kTileRows[4] = {256, 128, 64, 64};
constexpr int kTileThreads[4] = {512, 256, 256, 256};

// Tiles of m walked together along n.  The workgroups that run at once on an
// XCD (32 CUs) then share about as many panels of either operand.
inline int32_t band_of(int tile, int32_t tiles_m) { return std::min<int32_t>(tiles_m, tile == 0 ? 4 : 8); }

// The arguments of a product in tiles of `rows` on a side, and its workgroups.
inline int64_t gemm_args(GemmArgs& g, int tile, Mat a, Mat b, int64_t m, int64_t n, int64_t k, int splits,
                         int32_t k_split, const Only& only) {
    const int rows = kTileRows[tile];
    g.a = Operand{a.p, a.ld};
    g.b = Operand{b.p, b.ld};
    g.m = (int32_t)m;
    g.n = (int32_t)n;
    g.k = (int32_t)k;
    g.tiles_m = (int32_t)((m + rows - 1) / rows);
    g.tiles_n = (int32_t)((n + rows - 1) / rows);
    g.splits = splits;
    g.k_split = splits > 1 ? k_split : (int32_t)std::max<int64_t>(k, 1);
    g.band = band_of(tile, g.tiles_m);
    g.flag = only.flag;
    g.mark = only.mark;
    g.wanted = only.wanted;
    return (int64_t)g.tiles_m * g.tiles_n * splits;
}

template <typename T, typename Epi>
hipError_t launch_gemm(int tile, Mat a, Mat b, int64_t m, int64_t n, int64_t k, int splits, int32_t k_split,
                       const Only& only, const Epi& epi, hipStream_t s) {
    GemmArgs g;
    const int64_t blocks = gemm_args(g, tile, a, b, m, n, k, splits, k_split, only);
    if (!launchable(blocks, kTileThreads[tile])) return hipErrorInvalidConfiguration;  // the caller has checked
    const dim3 grid((unsigned)blocks);
    if (tile == 0)
        gemm_kernel<T, 2, 4, 8, 4, Epi><<<grid, 512, 0, s>>>(g, epi);
    else if (tile == 1)
        gemm_kernel<T, 2, 2, 4, 4, Epi><<<grid, 256, 0, s>>>(g, epi);
    else if (tile == 2)
        gemm_kernel<T, 2, 2, 2, 2, Epi><<<grid, 256, 0, s>>>(g, epi);
    else if constexpr (sizeof(T) == 4)
        gemm_kernel<T, 2, 2, 2, 2, Epi, 4><<<grid, 256, 0, s>>>(g, epi);
    else
        return hipErrorInvalidValue;
    return hipGetLastError();
}

// The parts of split contractions, joined in order: of one product or of two.
template <typename Point>
struct JoinJob {
    const float* part;
    int32_t splits;  // none: nothing to do
    int64_t m, n;
    Point point;
    __host__ __device__ int64_t quads() const { return (m + 3) / 4; }  // of a row
    __host__ __device__ int64_t total() const { return splits ? quads() * n : 0; }
};

template <typename Point>
__global__ __launch_bounds__(256) void join_kernel(JoinJob<Point> x, JoinJob<Point> w, Only only) {
    if (skipped(only.flag, only.mark, only.wanted)) return;
    const int64_t first = x.total(), total = first + w.total();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const JoinJob<Point>& j = i < first ? x : w;
        const int64_t at = i < first ? i : i - first, quads = j.quads();
        const int64_t r = at / quads, c = (at - r * quads) * 4;
        const float* from = j.part + at * 4;
        f32x4 v = *reinterpret_cast<const f32x4*>(from);
        for (int s = 1; s < j.splits; ++s) v += *reinterpret_cast<const f32x4*>(from + s * quads * 4 * j.n);
        j.point(r, c, j.m, v);
    }
}

template <typename Point>
hipError_t launch_join(const JoinJob<Point>& x, const JoinJob<Point>& w, const Only& only, hipStream_t s) {
    const int64_t total = x.total() + w.total();
    if (total == 0) return hipSuccess;
    const int64_t blocks = std::min<int64_t>((total + 255) / 256, 16384);
    join_kernel<Point><<<dim3((unsigned)blocks), 256, 0, s>>>(x, w, only);
    return hipGetLastError();
}
template <typename Point>
hipError_t launch_join(const float* part, int splits, int64_t m, int64_t n, const Point& point, const Only& only,
                       hipStream_t s) {
    return launch_join(JoinJob<Point>{part, splits, m, n, point}, JoinJob<Point>{nullptr, 0, 0, 0, point}, only, s);
}

template <typename T>
struct LinearPoint {
    LinearEpi<T> e;
    __device__ __forceinline__ void operator()(int64_t n, int64_t c, int64_t m, f32x4 v) const { e.point(n, c, m, v); }
};
template <typename T>
struct StorePoint {
    StoreEpi<T> e;
    __device__ __forceinline__ void operator()(int64_t n, int64_t c, int64_t m, f32x4 v) const { e.point(n, c, m, v); }
};

template <typename T>
inline StoreEpi<T> parts_epi(float* part, int64_t m, int64_t n) {
    StoreEpi<T> e{};
    e.part = part;
    e.part_ld = (m + 3) & ~(int64_t)3;
    e.part_stride = n * e.part_ld;
    return e;
}

template <typename T>
inline LinearEpi<T> linear_epi(const LinearOut& o, int64_t m) {
    LinearEpi<T> e;
    e.bias = (const T*)o.bias;
    e.residual = (const T*)o.residual;
    e.y = (T*)o.y;
    e.z = (T*)o.z;
    e.ld = m;
    e.act = o.act;
    return e;
}

template <typename T>
inline StoreEpi<T> store_epi(const StoreTo& o) {
    StoreEpi<T> e{};
    e.out = (T*)o.out;
    e.part = o.acc;
    e.add = o.add;
    e.alpha = o.alpha;
    e.ld = o.ld;
    e.part_ld = o.acc_ld;
    e.part_stride = 0;
    return e;
}

}  // namespace train
}  // namespace mlrs
