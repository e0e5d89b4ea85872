// Launching the matrix-core products of the training operators.
#pragma once
#include <algorithm>

#include "train_epilogue.hpp"
#include "train_kernels.hpp"

namespace mlrs {
namespace train {

constexpr int kTileRows[3] = {256, 128, 64};

// Tiles of m walked together along n.  The workgroups that run at once on an
// XCD (32 CUs) then share about as many panels of either operand.
inline int32_t band_of(int tile, int32_t tiles_m) { return std::min<int32_t>(tiles_m, tile == 0 ? 4 : 8); }

template <typename T, bool AKC, bool BKC, typename Epi>
hipError_t launch_gemm(int tile, Mat a, Mat b, int64_t m, int64_t n, int64_t k, int splits, int32_t k_split,
                       const Epi& epi, hipStream_t s) {
    const int rows = kTileRows[tile];
    GemmArgs g;
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
    const int64_t blocks = (int64_t)g.tiles_m * g.tiles_n * splits;
    if (blocks > INT32_MAX) return hipErrorInvalidValue;  // the caller has checked
    const dim3 grid((unsigned)blocks);
    if (tile == 0)
        gemm_kernel<T, AKC, BKC, 2, 4, 8, 4, Epi><<<grid, 512, 0, s>>>(g, epi);
    else if (tile == 1)
        gemm_kernel<T, AKC, BKC, 2, 2, 4, 4, Epi><<<grid, 256, 0, s>>>(g, epi);
    else
        gemm_kernel<T, AKC, BKC, 2, 2, 2, 2, Epi><<<grid, 256, 0, s>>>(g, epi);
    return hipGetLastError();
}

// How many elements of rows `ld` elements apart from p on an access may hold.
template <typename T>
inline int row_width(const void* p, int64_t ld) {
    if ((uintptr_t)p % (4 * sizeof(T)) == 0 && ld % 4 == 0) return 4;
    return (uintptr_t)p % (2 * sizeof(T)) == 0 && ld % 2 == 0 ? 2 : 1;
}

}  // namespace train
}  // namespace mlrs
