// Random bits from a counter, for dropout: the mask of an element is computed
// where it is needed, forwards and backwards, and never stored.
//
// Philox 4x32 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011) with seven rounds, the fewest that the paper found to pass
// all of its tests: two 32 x 32 -> 64 bit products a round, for which the vector
// unit takes four times as long as for other instructions.  A block of 128 bits
// serves eight elements, 16 bits each: of 16384 x 4096 bf16 the generator's share
// is then below what reading and writing take.
#pragma once
#include "train_gemm.hpp"
#include "train_kernels.hpp"

namespace mlrs {
namespace train {

// Eight consecutive elements, as they are loaded and stored.
template <typename T>
struct OctOf;
template <>
struct OctOf<float> {
    typedef float V __attribute__((ext_vector_type(8)));
};
template <>
struct OctOf<_Float16> {
    typedef f16x8 V;
};
template <>
struct OctOf<__bf16> {
    typedef bf16x8 V;
};
template <typename T>
using Oct = typename OctOf<T>::V;

// Elements c .. c + 7 of a row of `end`, those past it as zeros or left out;
// global accesses need no more than their elements' alignment.
template <typename T>
__device__ __forceinline__ Oct<T> load_oct(const T* row, int64_t c, int64_t end) {
    Oct<T> v = {};
    if (c + 8 <= end) {
        __builtin_memcpy(&v, row + c, sizeof v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < end) v[e] = row[c + e];
    }
    return v;
}
template <typename T>
__device__ __forceinline__ void store_oct(T* row, int64_t c, int64_t end, const float (&f)[8]) {
    Oct<T> v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (T)f[e];
    if (c + 8 <= end) {
        __builtin_memcpy(row + c, &v, sizeof v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < end) row[c + e] = v[e];
    }
}

// Another lane's value, by a move within the vector unit: the neighbour's, that of the
// other pair of four, that of the mirror image in eight or sixteen lanes.
enum { kNeighbour = 0xB1, kPair = 0x4E, kMirror8 = 0x141, kMirror16 = 0x140 };
template <int CTRL>
__device__ __forceinline__ float from_lane(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_bit_cast(float,
                              __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
#else
    return v;
#endif
}
// The largest of sixteen adjacent lanes' values, in each of them.
__device__ __forceinline__ float max16(float v) {
    v = fmaxf(v, from_lane<kNeighbour>(v));
    v = fmaxf(v, from_lane<kPair>(v));
    v = fmaxf(v, from_lane<kMirror8>(v));
    return fmaxf(v, from_lane<kMirror16>(v));
}

typedef uint32_t RandomWords[4];

__device__ __forceinline__ void random_block(uint64_t block, uint64_t offset, uint32_t k0, uint32_t k1,
                                             RandomWords& out) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    out[0] = c0;
    out[1] = c1;
    out[2] = c2;
    out[3] = c3;
}

// The offset of a call, with what the device adds to it.
__device__ __forceinline__ uint64_t drop_offset(const Drop& d) {
    return d.offset + (d.step ? (uint64_t)*d.step : 0);
}

// Multiplies elements i .. i + 7 by their factor, 0 (whatever they hold) or
// d.factor.  aligned: i is a multiple of 8, in every lane; else the eight may lie
// in two blocks.
__device__ __forceinline__ void drop_oct(const Drop& d, uint64_t offset, int64_t i, bool aligned, float (&v)[8]) {
    RandomWords w;
    random_block((uint64_t)i >> 3, offset, d.k0, d.k1, w);
    const int r = (int)(i & 7);
    if (!aligned) {
        asm volatile("");  // not to be computed where it is not needed
        RandomWords next;
        random_block(((uint64_t)i >> 3) + 1, offset, d.k0, d.k1, next);
        uint32_t all[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            all[e] = w[e];
            all[e + 4] = next[e];
        }
        // down by r halves: four words, two, one, and half a word
#pragma unroll
        for (int e = 0; e < 6; ++e)
            if (r & 4) all[e] = all[e + 2];
#pragma unroll
        for (int e = 0; e < 5; ++e)
            if (r & 2) all[e] = all[e + 1];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = r & 1 ? (all[e] >> 16) | (all[e + 1] << 16) : all[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t u = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu;
        v[e] = u >= d.threshold ? v[e] * d.factor : 0.0f;
    }
}

}  // namespace train
}  // namespace mlrs
