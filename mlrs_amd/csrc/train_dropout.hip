// Dropout with a residual: y = drop(x) + residual.
#include <algorithm>

#include "train_random.hpp"

namespace mlrs {
namespace train {

// A lane takes eight elements, one block of random bits, at a time; two of them
// under way at once.  Bound by memory: 16384 x 4096 bf16 with a residual, 402 MB, take
// 80 us, 5.0 TB/s, where a large copy reaches 5.1.
template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, const T* residual, T* y, int64_t len, Drop drop) {
    const uint64_t offset = drop_offset(drop);
    const int64_t octs = (len + 7) / 8, stride = (int64_t)gridDim.x * 256;
    constexpr int U = 2;
    for (int64_t o = (int64_t)blockIdx.x * 256 + threadIdx.x; o < octs; o += U * stride) {
        Oct<T> v[U], r[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (o + u * stride < octs) v[u] = load_oct(x, (o + u * stride) * 8, len);
        if (residual) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (o + u * stride < octs) r[u] = load_oct(residual, (o + u * stride) * 8, len);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = o + u * stride;
            if (at >= octs) continue;
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = (float)v[u][e];
            if (drop.threshold) drop_oct(drop, offset, at * 8, true, f);
            if (residual) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] += (float)r[u][e];
            }
            store_oct(y, at * 8, len, f);
        }
    }
}

template <typename T>
hipError_t launch_dropout(const T* x, const T* residual, T* y, int64_t len, const Drop& drop, int cus, hipStream_t s) {
    const int64_t blocks = std::min<int64_t>((len + 2047) / 2048, (int64_t)cus * 16);
    dropout_kernel<T><<<dim3((unsigned)blocks), 256, 0, s>>>(x, residual, y, len, drop);
    return hipGetLastError();
}

#define MLRS_INST(T) \
    template hipError_t launch_dropout<T>(const T*, const T*, T*, int64_t, const Drop&, int, hipStream_t);
MLRS_INST(float)
MLRS_INST(_Float16)
MLRS_INST(__bf16)

}  // namespace train
}  // namespace mlrs
