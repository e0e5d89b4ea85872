// A layer in 8-bit floating point: making the codes, and its three products.
#include <cmath>
#include <type_traits>

#include "train_fp8.hpp"
#include "train_random.hpp"

namespace mlrs {
namespace train {

namespace {

// The exponent of a block's scale: the least e with top <= 448 * 2^e (448 is 1.75 *
// 2^8), 0 for a block of zeros.
__device__ __forceinline__ int scale_exponent(float top) {
    const uint32_t bits = __float_as_uint(top);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return top > 0.0f ? (e < -127 ? -127 : e) : 0;
}
// 2^-e
__device__ __forceinline__ float scale_inverse(int e) { return __uint_as_float((uint32_t)(127 - e) << 23); }

// Four values that 448 bounds as codes, to nearest even; a NaN has code NaN.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
#if defined(__HIP_DEVICE_COMPILE__)
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
#else
    (void)a;
    (void)b;
    (void)c;
    (void)d;
    return 0;
#endif
}

// The values of eight codes as bf16, which holds them: exact but for magnitudes
// outside its range.
__device__ __forceinline__ bf16x8 values8(uint32_t lo, uint32_t hi, float up) {
    bf16x8 v = {};
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int w = (int)(h ? hi : lo);
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        v[4 * h] = (__bf16)(a[0] * up);
        v[4 * h + 1] = (__bf16)(a[1] * up);
        v[4 * h + 2] = (__bf16)(b[0] * up);
        v[4 * h + 3] = (__bf16)(b[1] * up);
    }
#else
    (void)lo;
    (void)hi;
    (void)up;
#endif
    return v;
}

// 2^e, from -127 on
__device__ __forceinline__ float scale_of(int e) { return __uint_as_float(e > -127 ? (uint32_t)(e + 127) << 23 : 1u << 22); }

__device__ __forceinline__ bool unbounded(float x) { return fabsf(x) == __builtin_huge_valf(); }

// ---------------------------------------------------------------------------
// making codes
// ---------------------------------------------------------------------------
// A workgroup takes 128 x 128 elements, a thread four by eight of them: rows 4 (t /
// 16) on and columns 8 (t % 16) on, so that it has eight adjacent codes of a row and
// four of a column (eight by eight take 210 registers and the same time).  Bound by
// memory: the codes of 8192 x 8192 with act'(z) and of x of 8192 x 4096, 535 MB in bf16,
// take 127 to 152 us, 3.5 to 4.2 TB/s.  The elements are read once, whatever is made of
// them: codes with a scale for each row, codes of the transpose with a scale for each
// column (turned through LDS), or both with one scale for the tile; and column sums.
// Infinities and NaN have code NaN and no part in the scale.
// VALUES: bf16 values and no scales in the codes' place.
template <typename T>
struct CodeJob {
    const T *src, *z;  // z: null, or src is multiplied by act'(z)
    int act;
    int64_t rows, cols;
    uint8_t *codes, *scales, *codes_t, *scales_t;  // null where not wanted
    float* sums;                                   // null, or the column sums of every 128 rows
    bool tile;                                     // one scale for all of it
    __host__ __device__ int64_t tiles_c() const { return (cols + 127) / 128; }
    __host__ __device__ int64_t tiles() const { return (rows + 127) / 128 * tiles_c(); }
};

constexpr int kCodeThreads = 512;

template <typename T, bool VALUES>
__global__ __launch_bounds__(kCodeThreads, 4) void codes_kernel(CodeJob<T> first, CodeJob<T> second) {
    constexpr int R = 4, WAVES = kCodeThreads / 64;
    __shared__ __attribute__((aligned(16))) char turn[128 * 128 * (VALUES ? 2 : 1)];
    __shared__ float tops[WAVES][128], sums[WAVES][128];
    const bool one = (int64_t)blockIdx.x < first.tiles();
    const CodeJob<T>& j = one ? first : second;
    const int64_t t = one ? blockIdx.x : blockIdx.x - first.tiles();
    const int64_t tr = t / j.tiles_c(), tc = t - tr * j.tiles_c();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int o = threadIdx.x & 15, p = threadIdx.x >> 4;
    const int64_t r0 = tr * 128 + R * p, c0 = tc * 128 + 8 * o;
    float v[R][8];
    {
        Oct<T> raw[R] = {}, z[R] = {};
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (r0 + i < j.rows && c0 < j.cols) raw[i] = load_oct(j.src + (r0 + i) * j.cols, c0, j.cols);
        if (j.z) {
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (r0 + i < j.rows && c0 < j.cols) z[i] = load_oct(j.z + (r0 + i) * j.cols, c0, j.cols);
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = (float)raw[i][e];
        if (j.z) {
            auto slope = [&](auto f) {
#pragma unroll
                for (int i = 0; i < R; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[i][e] *= f((float)z[i][e]);
            };
            switch (j.act) {
            case kActRelu: slope([](float x) { return activate_slope(x, kActRelu); }); break;
            case kActGelu: slope([](float x) { return activate_slope(x, kActGelu); }); break;
            case kActGeluTanh: slope([](float x) { return activate_slope(x, kActGeluTanh); }); break;
            case kActSilu: slope([](float x) { return activate_slope(x, kActSilu); }); break;
            default: break;
            }
        }
    }
    // the largest magnitudes; maxima leave out NaN by themselves
    float row_top[R], col_top[8], col_sum[8] = {};
    auto maxima = [&](auto magnitude) {
#pragma unroll
        for (int e = 0; e < 8; ++e) col_top[e] = 0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            row_top[i] = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float a = magnitude(v[i][e]);
                row_top[i] = fmaxf(row_top[i], a);
                col_top[e] = fmaxf(col_top[e], a);
            }
        }
    };
    if (j.sums) {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) col_sum[e] += v[i][e];
    }
    maxima([](float x) { return fabsf(x); });
    bool odd = false;
#pragma unroll
    for (int i = 0; i < R; ++i) odd |= unbounded(row_top[i]);
    if (odd) {
        maxima([](float x) { return unbounded(x) ? 0.0f : fabsf(x); });
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (unbounded(v[i][e])) v[i][e] = __builtin_nanf("");
    }
    if (j.codes_t || j.tile) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            col_top[e] = fmaxf(col_top[e], __shfl_xor(col_top[e], 16));
            col_top[e] = fmaxf(col_top[e], __shfl_xor(col_top[e], 32));
        }
        if (lane < 16)
#pragma unroll
            for (int e = 0; e < 8; ++e) tops[wave][8 * o + e] = col_top[e];
    }
    if (j.sums) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            col_sum[e] += __shfl_xor(col_sum[e], 16);
            col_sum[e] += __shfl_xor(col_sum[e], 32);
        }
        if (lane < 16)
#pragma unroll
            for (int e = 0; e < 8; ++e) sums[wave][8 * o + e] = col_sum[e];
    }
    float whole = 0.0f;
    if (j.codes_t || j.tile || j.sums) {
        __syncthreads();
        if (j.sums && threadIdx.x < 128) {
            const int c = threadIdx.x;
            float sum = sums[0][c];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) sum += sums[w][c];
            if (tc * 128 + c < j.cols) j.sums[tr * j.cols + tc * 128 + c] = sum;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            col_top[e] = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) col_top[e] = fmaxf(col_top[e], tops[w][8 * o + e]);
            whole = fmaxf(whole, col_top[e]);
        }
    }
    if (j.tile) {
        whole = max16(whole);
#pragma unroll
        for (int e = 0; e < 8; ++e) col_top[e] = whole;
#pragma unroll
        for (int i = 0; i < R; ++i) row_top[i] = whole;
    } else if (j.codes) {
#pragma unroll
        for (int i = 0; i < R; ++i) row_top[i] = max16(row_top[i]);
    }
    // weights' rows of scales are whole words: the last tile writes what is behind it
    auto put_scale = [](uint8_t* row, int64_t at, int64_t blocks, int e) {
        row[at] = (uint8_t)(e + 127);
        if (at + 1 == blocks)
            for (int64_t b = blocks; b & 3; ++b) row[b] = 127;
    };
    const int64_t blocks = j.tiles_c(), blocks_t = (j.rows + 127) / 128;
    const int64_t ld = (blocks + 3) / 4 * 4, ld_t = (blocks_t + 3) / 4 * 4;
    if (j.codes) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int e = scale_exponent(row_top[i]);
            const float by = scale_inverse(e);
            if (r0 + i >= j.rows) continue;
            const uint32_t lo = codes4(v[i][0] * by, v[i][1] * by, v[i][2] * by, v[i][3] * by);
            const uint32_t hi = codes4(v[i][4] * by, v[i][5] * by, v[i][6] * by, v[i][7] * by);
            const int64_t at = (r0 + i) * blocks * 128 + c0;
            if constexpr (VALUES) {
                *reinterpret_cast<bf16x8*>(j.codes + 2 * at) = values8(lo, hi, scale_of(e));
                continue;
            }
            *reinterpret_cast<uint64_t*>(j.codes + at) = lo | (uint64_t)hi << 32;
            if (!j.tile && o == 0) j.scales[((tc >> 2) * j.rows + r0 + i) * 4 + (tc & 3)] = (uint8_t)(e + 127);
        }
        if (!VALUES && j.tile && threadIdx.x == 0) put_scale(j.scales + tr * ld, tc, blocks, scale_exponent(whole));
    }
    if (!j.codes_t) return;
    // column c's line in LDS: its pieces of sixteen bytes at piece ^ (c / 8), so that the
    // lanes that write one row's eighths of the columns are in different banks
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int x = scale_exponent(col_top[e]);
        const float by = scale_inverse(x);
        const uint32_t w = codes4(v[0][e] * by, v[1][e] * by, v[2][e] * by, v[3][e] * by);
        if constexpr (VALUES) {
            const bf16x8 u = values8(w, 0, scale_of(x));
            *reinterpret_cast<bf16x4*>(turn + (8 * o + e) * 256 + (((p >> 1) ^ o) << 4) + (p & 1) * 8) =
                __builtin_shufflevector(u, u, 0, 1, 2, 3);
            continue;
        }
        *reinterpret_cast<uint32_t*>(turn + (8 * o + e) * 128 + (((p >> 2) ^ (o & 7)) << 4) + (p & 3) * 4) = w;
        if (!j.tile && p == 0 && c0 + e < j.cols)
            j.scales_t[((tr >> 2) * j.cols + c0 + e) * 4 + (tr & 3)] = (uint8_t)(x + 127);
    }
    if (!VALUES && j.tile && threadIdx.x == 0) put_scale(j.scales_t + tc * ld_t, tr, blocks_t, scale_exponent(whole));
    __syncthreads();
    constexpr int kPieces = VALUES ? 16 : 8;  // of a line
#pragma unroll
    for (int i = 0; i < 128 * kPieces / kCodeThreads; ++i) {
        const int at = threadIdx.x + kCodeThreads * i, c = at / kPieces, piece = at % kPieces;
        const u32x4 w = *reinterpret_cast<const u32x4*>(turn + c * 16 * kPieces + ((piece ^ ((c >> 3) & (kPieces - 1))) << 4));
        if (tc * 128 + c < j.cols)
            *reinterpret_cast<u32x4*>(j.codes_t + ((tc * 128 + c) * blocks_t * 128 + tr * 128) * (VALUES ? 2 : 1) + 16 * piece) = w;
    }
}

template <bool VALUES, typename T>
hipError_t launch_codes(const CodeJob<T>& a, const CodeJob<T>& b, hipStream_t s) {
    const int64_t tiles = a.tiles() + b.tiles();
    if (tiles == 0) return hipSuccess;
    if (!launchable(tiles, kCodeThreads)) return hipErrorInvalidConfiguration;  // the caller has checked
    codes_kernel<T, VALUES><<<dim3((unsigned)tiles), kCodeThreads, 0, s>>>(a, b);
    return hipGetLastError();
}

// Weights' values as bf16, from their codes.
__global__ __launch_bounds__(256) void values_kernel(const uint8_t* __restrict__ codes,
                                                     const uint8_t* __restrict__ scales, int64_t rows, int64_t blocks,
                                                     char* __restrict__ out) {
    const int64_t ld = (blocks + 3) / 4 * 4, total = rows * blocks * 8;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / (blocks * 8), b = (i - r * blocks * 8) >> 3;
        const u32x4 c = *reinterpret_cast<const u32x4*>(codes + 16 * i);
        const float up = scale_of((int)scales[(r >> 7) * ld + b] - 127);
        *reinterpret_cast<bf16x8*>(out + 32 * i) = values8(c[0], c[1], up);
        *reinterpret_cast<bf16x8*>(out + 32 * i + 16) = values8(c[2], c[3], up);
    }
}

// ---------------------------------------------------------------------------
// a few rows
// ---------------------------------------------------------------------------
// Bound by reading the codes of the weights, once, straight into registers as the
// fragments of the matrix instructions.  A workgroup computes sixteen outputs of
// every row.  In passes of 1024 U columns its threads first make the codes of the rows
// in LDS, sixteen lanes to a block, while the pass's weights are on their way; then
// each wave multiplies its U blocks.  The waves' sums are joined in LDS, in order.  No
// launch and no workspace besides.  (Each wave making the codes of its own blocks, as
// it needs them, took 12.1 us of one row by 8192 x 4096: the codes of a row are then
// made sixteen times over.)
constexpr int kFewWaves = 8;
template <int U>
__host__ __device__ constexpr int few_row_bytes() {  // of a row in LDS: codes and scales
    return kFewWaves * U * (128 + 4);
}

template <typename T, int NB, int U>
__global__ __launch_bounds__(kFewWaves * 64) void fp8_few_kernel(const T* __restrict__ x,
                                                                 const uint8_t* __restrict__ codes,
                                                                 const uint8_t* __restrict__ scales, int32_t n,
                                                                 int32_t m, int64_t k, LinearEpi<T> epi) {
    extern __shared__ __attribute__((aligned(16))) char rows[];  // n rows of few_row_bytes
    __shared__ f32x4 sums[kFewWaves][NB][64];
    constexpr int kBlocks = kFewWaves * U, kOcts = kBlocks * 16;  // of a pass
    char* const row_scales = rows + n * kBlocks * 128;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int32_t m0 = (int32_t)blockIdx.x * 16;
    const int64_t blocks = (k + 127) / 128;
    const uint8_t* wr = codes + (int64_t)(m0 + r < m ? m0 + r : m - 1) * blocks * 128 + 16 * g;
    const uint8_t* ws = scales + (m0 >> 7) * ((blocks + 3) / 4 * 4);
    f32x4 acc[NB] = {};
    for (int64_t pass = 0; pass < blocks; pass += kBlocks) {
        const int64_t b0 = pass + wave * U;
        u32x4 lo[U] = {}, hi[U] = {};
        int sw[U] = {};
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (b0 + u < blocks) {
                lo[u] = *reinterpret_cast<const u32x4*>(wr + (b0 + u) * 128);
                hi[u] = *reinterpret_cast<const u32x4*>(wr + (b0 + u) * 128 + 64);
                sw[u] = ws[b0 + u];
            }
        if (pass) __syncthreads();  // the last pass's codes have been read
        for (int at = threadIdx.x; at < n * kOcts; at += kFewWaves * 64) {
            const int row = at / kOcts, oct = at % kOcts;
            const int64_t c = pass * 128 + 8 * oct;
            Oct<T> raw = {};
            if (c < k) raw = load_oct(x + row * k, c, k);
            float v[8], top = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = (float)raw[e];
                top = fmaxf(top, fabsf(v[e]));
            }
            if (unbounded(top)) {
                top = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (unbounded(v[e])) v[e] = __builtin_nanf("");
                    top = fmaxf(top, fabsf(v[e]));
                }
            }
            const int e = scale_exponent(max16(top));
            const float by = scale_inverse(e);
            const uint64_t w = codes4(v[0] * by, v[1] * by, v[2] * by, v[3] * by) |
                               (uint64_t)codes4(v[4] * by, v[5] * by, v[6] * by, v[7] * by) << 32;
            *reinterpret_cast<uint64_t*>(rows + (row * kBlocks + oct / 16) * 128 +
                                         ((((oct >> 1) & 7) ^ k_swizzle(row)) << 4) + (oct & 1) * 8) = w;
            if ((oct & 15) == 0) *reinterpret_cast<int*>(row_scales + (row * kBlocks + oct / 16) * 4) = e + 127;
        }
        __syncthreads();
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int row = b * 16 + r < n ? b * 16 + r : n - 1;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (b0 + u >= blocks) continue;
                const char* from = rows + (row * kBlocks + wave * U + u) * 128;
                const u32x4 x0 = *reinterpret_cast<const u32x4*>(from + ((g ^ k_swizzle(row)) << 4));
                const u32x4 x1 = *reinterpret_cast<const u32x4*>(from + (((4 + g) ^ k_swizzle(row)) << 4));
                const int sx = *reinterpret_cast<const int*>(row_scales + (row * kBlocks + wave * U + u) * 4);
                if constexpr (sizeof(T) == 2) {
                    acc[b] = mfma_fp8(join_halves(lo[u], hi[u]), join_halves(x0, x1), acc[b], sw[u], sx);
                } else {  // in f32 the codes go through the bf16 instructions, the scales to their sums
                    f32x4 block = {};
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const u32x4 &w = h < 2 ? lo[u] : hi[u], &y = h < 2 ? x0 : x1;
                        block = mfma_step<__bf16>(values8(w[2 * (h & 1)], w[2 * (h & 1) + 1], 1.0f),
                                                  values8(y[2 * (h & 1)], y[2 * (h & 1) + 1], 1.0f), block);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[b][e] += ldexpf(block[e], sw[u] + sx - 254);
                }
            }
        }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) sums[wave][b][lane] = acc[b];
    __syncthreads();
    for (int b = wave; b < NB; b += kFewWaves) {  // wave b joins the sums of rows 16 b .. 16 b + 15
        f32x4 v = sums[0][b][lane];
#pragma unroll
        for (int i = 1; i < kFewWaves; ++i) v += sums[i][b][lane];
        const int32_t row = b * 16 + r, c = m0 + 4 * g;
        if (row < n && c < m) epi.point(row, c, m, v);
    }
}

// ---------------------------------------------------------------------------
// the products
// ---------------------------------------------------------------------------
int64_t product_args(GemmArgs& g, int tile, const Fp8Mat& a, const Fp8Mat& b, int64_t m, int64_t n, int64_t k,
                     int splits, int32_t k_split) {
    const int64_t kp = fp8_columns(k);
    return gemm_args(g, tile, Mat{a.codes, kp}, Mat{b.codes, kp}, m, n, kp, splits, k_split, Only{});
}
int64_t product_args(Fp8Args& q, int tile, const Fp8Mat& a, const Fp8Mat& b, int64_t m, int64_t n, int64_t k,
                     int splits, int32_t k_split) {
    const int64_t blocks = product_args(q.g, tile, a, b, m, n, k, splits, k_split);
    auto where = [&](const Fp8Mat& x, int64_t rows) {
        return x.tile ? ScaleRows{x.scales, fp8_scale_row(k), 4, (rows + 127) / 128, 7}
                      : ScaleRows{x.scales, 4, 4 * rows, rows, 0};
    };
    q.sa = where(a, m);
    q.sb = where(b, n);
    return blocks;
}

// The product of two operands in either form: 16-bit results from codes, f32 ones
// from values.
template <typename T, typename Epi>
hipError_t launch_fp8(int tile, const Fp8Mat& a, const Fp8Mat& b, int64_t m, int64_t n, int64_t k, int splits,
                      int32_t k_split, const Epi& epi, hipStream_t s) {
    if constexpr (sizeof(T) == 4) {
        const int64_t kp = fp8_columns(k);
        return launch_gemm<__bf16>(tile, Mat{a.codes, kp}, Mat{b.codes, kp}, m, n, kp, splits, k_split, Only{}, epi, s);
    } else {
        Fp8Args q;
        const int64_t blocks = product_args(q, tile, a, b, m, n, k, splits, k_split);
        if (!launchable(blocks, kTileThreads[tile])) return hipErrorInvalidConfiguration;  // the caller has checked
        const dim3 grid((unsigned)blocks);
        if (tile == 0)
            fp8_kernel<2, 4, 8, 4, Epi><<<grid, 512, 0, s>>>(q, epi);
        else if (tile == 1)
            fp8_kernel<2, 2, 4, 4, Epi><<<grid, 256, 0, s>>>(q, epi);
        else
            fp8_kernel<2, 2, 2, 2, Epi><<<grid, 256, 0, s>>>(q, epi);
        return hipGetLastError();
    }
}

// The two products of a gradient in one grid, as train_linear.hip's, with the column
// sums' last step: of codes, or in f32 of values.  Of 3001 x 2050 by 1000 in f32 they
// take 37 us, in a launch each and one for the sums 62.
template <typename T>
struct Fp8Pair {
    std::conditional_t<sizeof(T) == 4, GemmArgs, Fp8Args> x, w;
    StoreEpi<T> to_x, to_w;
    int32_t x_wgs, w_wgs;
    bool x_first;  // the one with the longer workgroups
    ColumnSums<T> sums;
    int64_t columns;
};
template <typename T, int WM, int WN, int MB, int NB>
__global__ __launch_bounds__(WM* WN * 64, 2) void fp8_pair_kernel(Fp8Pair<T> q) {
    constexpr int kLds = sizeof(T) == 4 ? gemm_lds<WM, MB, NB>() : fp8_lds<WM, WN, MB, NB>();
    __shared__ __attribute__((aligned(1024))) char buf[kLds];
    int32_t wg = blockIdx.x;
    const int32_t lead = q.x_first ? q.x_wgs : q.w_wgs;
    if (wg >= q.x_wgs + q.w_wgs) {
        sum_parts<T, WM * WN * 64>(q.sums, q.columns, wg - q.x_wgs - q.w_wgs, reinterpret_cast<float*>(buf));
        return;
    }
    const bool second = wg >= lead;
    if (second) wg -= lead;
    const bool is_x = second != q.x_first;
    if constexpr (sizeof(T) == 4)
        gemm_workgroup<__bf16, true, true, WM, WN, MB, NB, StoreEpi<T>>(is_x ? q.x : q.w, is_x ? q.to_x : q.to_w, wg, buf);
    else
        fp8_workgroup<WM, WN, MB, NB>(is_x ? q.x : q.w, is_x ? q.to_x : q.to_w, wg, buf);
}

// The time of each choice, in microseconds, as of the 16-bit products: a staged width
// (128 of k) of the one, two, ... tiles that a CU holds, a round's other costs, and the
// join of split sums.  Measured over every tile and count of splits of 17 products from
// 64 x 4096 x 8192 to 4096^3: the choice is the fastest or within 6 % of it, for a
// gradient's two within 16 %, where others take up to 8 times as long.
constexpr double kStage8[3][3] = {{1.31}, {0.67, 0.96}, {0.265, 0.43, 0.6}};
constexpr double kRound8[3] = {6.0, 4.0, 3.4};
constexpr int kResident8[3] = {1, 2, 3};
double join_us(int64_t elements) { return elements ? 4.5 + (double)elements * 8.0 / 4.5e6 : 0.0; }

}  // namespace

// Parts of the contraction are whole words of scales.
Cut choose_cut_fp8(int elem_bytes, int64_t m, int64_t n, int64_t k, int cus, int tile) {
    if (elem_bytes == 4) return choose_cut(2, m, n, fp8_columns(k), cus);
    const int64_t quads = std::max<int64_t>(1, (k + 511) / 512);
    Cut best{std::max(tile, 0), 1, 0, 1e300};
    for (int t = 0; t < 3; ++t) {
        if (tile >= 0 && t != tile) continue;
        const int rows = kTileRows[t];
        const int64_t tiles = ((m + rows - 1) / rows) * ((n + rows - 1) / rows);
        for (int64_t sp = 1; sp <= 64 && sp <= quads; sp = sp < 4 ? sp + 1 : sp * 2) {
            const int64_t each = (quads + sp - 1) / sp;
            if (sp > 1 && (sp - 1) * each >= quads) continue;
            if ((t > 0 || sp > 1) && !launchable(tiles * sp, kTileThreads[t])) continue;
            const double widths = sp > 1 ? 4.0 * (double)each : (double)((k + 127) / 128);
            const int64_t on_cu = (tiles * sp + cus - 1) / cus;
            const int64_t rounds = on_cu / kResident8[t], rest = on_cu % kResident8[t];
            double cost = (double)rounds * (widths * kStage8[t][kResident8[t] - 1] + kRound8[t]);
            if (rest) cost += widths * kStage8[t][rest - 1] + kRound8[t];
            if (sp > 1) cost += join_us(sp * m * n);
            if (cost < best.us) best = Cut{t, (int)sp, (int32_t)(each * 512), cost};
        }
    }
    return best;
}

// Both products of a gradient: in tiles of one size, so that one grid holds them.
void choose_pair_fp8(int elem_bytes, int64_t xm, int64_t xn, int64_t xk, int64_t wm, int64_t wn, int64_t wk, int cus, Cut* x, Cut* w) {
    if (elem_bytes == 4) {
        const PairCut p = choose_pair(2, xm, xn, fp8_columns(xk), wm, wn, fp8_columns(wk), cus, false);
        *x = p.x;
        *w = p.w;
        return;
    }
    double best = 1e300;
    for (int t = 0; t < 3; ++t) {
        const Cut cx = choose_cut_fp8(elem_bytes, xm, xn, xk, cus, t), cw = choose_cut_fp8(elem_bytes, wm, wn, wk, cus, t);
        if (cx.us + cw.us < best) {
            best = cx.us + cw.us;
            *x = cx;
            *w = cw;
        }
    }
}

template <typename T>
hipError_t launch_fp8_weight(const T* w, int64_t rows, int64_t cols, const Fp8Mat& to, const Fp8Mat& to_t, hipStream_t s) {
    CodeJob<T> j{w, nullptr, 0, rows, cols, (uint8_t*)to.codes, (uint8_t*)to.scales, (uint8_t*)to_t.codes,
                 (uint8_t*)to_t.scales, nullptr, true};
    return launch_codes<false>(j, CodeJob<T>{}, s);
}

template <typename T>
hipError_t launch_fp8_rows(const T* x, int64_t n, int64_t k, const Fp8Mat& to, hipStream_t s) {
    CodeJob<T> j{x, nullptr, 0, n, k, (uint8_t*)to.codes, (uint8_t*)to.scales, nullptr, nullptr, nullptr, false};
    return launch_codes<sizeof(T) == 4>(j, CodeJob<T>{}, s);
}

hipError_t launch_fp8_values(const Fp8Mat& w, int64_t rows, int64_t k, void* out, hipStream_t s) {
    const int64_t blocks = (k + 127) / 128, total = rows * blocks * 8;
    const dim3 grid((unsigned)std::min<int64_t>((total + 255) / 256, 16384));
    values_kernel<<<grid, 256, 0, s>>>((const uint8_t*)w.codes, w.scales, rows, blocks, (char*)out);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_fp8_grad_codes(const T* dy, const T* z, int act, int64_t n, int64_t m, const Fp8Mat& dz,
                                 const Fp8Mat& dz_t, float* sums, const T* x, int64_t k, const Fp8Mat& x_t,
                                 hipStream_t s) {
    CodeJob<T> a{dy, z, act, n, m, (uint8_t*)dz.codes, (uint8_t*)dz.scales, (uint8_t*)dz_t.codes,
                 (uint8_t*)dz_t.scales, sums, false};
    CodeJob<T> b{};
    if (x) b = CodeJob<T>{x, nullptr, 0, n, k, nullptr, nullptr, (uint8_t*)x_t.codes, (uint8_t*)x_t.scales, nullptr, false};
    return launch_codes<sizeof(T) == 4>(a, b, s);
}

template <typename T>
hipError_t launch_fp8_linear(const Fp8Mat& x, const Fp8Mat& w, int64_t n, int64_t m, int64_t k, const LinearOut& o,
                             const Cut& cut, float* part, hipStream_t s) {
    const LinearEpi<T> e = linear_epi<T>(o, m);
    if (cut.splits == 1) return launch_fp8<T>(cut.tile, w, x, m, n, k, 1, 0, e, s);
    const hipError_t r = launch_fp8<T>(cut.tile, w, x, m, n, k, cut.splits, cut.k_split, parts_epi<T>(part, m, n), s);
    if (r != hipSuccess) return r;
    return launch_join(part, cut.splits, m, n, LinearPoint<T>{e}, Only{}, s);
}

template <typename T>
hipError_t launch_fp8_few(const T* x, const Fp8Mat& w, int64_t n, int64_t m, int64_t k, const LinearOut& o,
                          hipStream_t s) {
    const LinearEpi<T> e = linear_epi<T>(o, m);
    const dim3 grid((unsigned)((m + 15) / 16));
    const uint8_t* c = (const uint8_t*)w.codes;
    // as many columns at a time as leave several workgroups a CU
    if (n <= 8)
        fp8_few_kernel<T, 1, 4><<<grid, kFewWaves * 64, n * few_row_bytes<4>(), s>>>(x, c, w.scales, (int32_t)n, (int32_t)m, k, e);
    else if (n <= 16)
        fp8_few_kernel<T, 1, 2><<<grid, kFewWaves * 64, n * few_row_bytes<2>(), s>>>(x, c, w.scales, (int32_t)n, (int32_t)m, k, e);
    else
        fp8_few_kernel<T, 2, 1><<<grid, kFewWaves * 64, n * few_row_bytes<1>(), s>>>(x, c, w.scales, (int32_t)n, (int32_t)m, k, e);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_fp8_products(const Fp8Product& x, const Fp8Product& w, const Cut& cx, const Cut& cw, float* part,
                               const ColumnSums<T>& sums, int64_t columns, hipStream_t s) {
    const Fp8Product* ps[2] = {&x, &w};
    const Cut* cs[2] = {&cx, &cw};
    float* parts[2] = {part, part + (x.m ? cx.part_bytes(x.m, x.n) / 4 : 0)};
    if (x.m && w.m && cx.tile == cw.tile) {
        Fp8Pair<T> q;
        decltype(q.x)* args[2] = {&q.x, &q.w};
        StoreEpi<T>* to[2] = {&q.to_x, &q.to_w};
        int32_t* wgs[2] = {&q.x_wgs, &q.w_wgs};
        for (int i = 0; i < 2; ++i) {
            const Fp8Product& p = *ps[i];
            *wgs[i] = (int32_t)product_args(*args[i], cs[i]->tile, p.a, p.b, p.m, p.n, p.k, cs[i]->splits, cs[i]->k_split);
            *to[i] = cs[i]->splits > 1 ? parts_epi<T>(parts[i], p.m, p.n) : store_epi<T>(p.to);
        }
        auto each = [](const auto& a) {
            if constexpr (sizeof(T) == 4)
                return a.k_split;
            else
                return a.g.k_split;
        };
        q.x_first = each(q.x) >= each(q.w);
        int64_t blocks = (int64_t)q.x_wgs + q.w_wgs + (sums.out ? (columns + 15) / 16 : 0);
        q.sums = sums;
        q.columns = columns;
        if (sums.out && !launchable(blocks, kTileThreads[cx.tile])) {
            const hipError_t e = launch_sum_parts(sums, columns, s);
            if (e != hipSuccess) return e;
            blocks = (int64_t)q.x_wgs + q.w_wgs;
        }
        if (!launchable(blocks, kTileThreads[cx.tile])) return hipErrorInvalidConfiguration;  // the caller has checked
        const dim3 grid((unsigned)blocks);
        if (cx.tile == 0)
            fp8_pair_kernel<T, 2, 4, 8, 4><<<grid, 512, 0, s>>>(q);
        else if (cx.tile == 1)
            fp8_pair_kernel<T, 2, 2, 4, 4><<<grid, 256, 0, s>>>(q);
        else
            fp8_pair_kernel<T, 2, 2, 2, 2><<<grid, 256, 0, s>>>(q);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    } else {
        const hipError_t r = launch_sum_parts(sums, columns, s);
        if (r != hipSuccess) return r;
        for (int i = 0; i < 2; ++i) {
            const Fp8Product& p = *ps[i];
            if (!p.m) continue;
            const hipError_t e = launch_fp8<T>(cs[i]->tile, p.a, p.b, p.m, p.n, p.k, cs[i]->splits, cs[i]->k_split,
                                            cs[i]->splits > 1 ? parts_epi<T>(parts[i], p.m, p.n) : store_epi<T>(p.to), s);
            if (e != hipSuccess) return e;
        }
    }
    typedef JoinJob<StorePoint<T>> Job;
    return launch_join(
        Job{parts[0], x.m && cx.splits > 1 ? cx.splits : 0, x.m, x.n, StorePoint<T>{store_epi<T>(x.to)}},
        Job{parts[1], w.m && cw.splits > 1 ? cw.splits : 0, w.m, w.n, StorePoint<T>{store_epi<T>(w.to)}}, Only{}, s);
}

#define MLRS_INST(T)                                                                                                \
    template hipError_t launch_fp8_weight<T>(const T*, int64_t, int64_t, const Fp8Mat&, const Fp8Mat&, hipStream_t); \
    template hipError_t launch_fp8_rows<T>(const T*, int64_t, int64_t, const Fp8Mat&, hipStream_t);                 \
    template hipError_t launch_fp8_grad_codes<T>(const T*, const T*, int, int64_t, int64_t, const Fp8Mat&,          \
                                                 const Fp8Mat&, float*, const T*, int64_t, const Fp8Mat&,           \
                                                 hipStream_t);                                                      \
    template hipError_t launch_fp8_linear<T>(const Fp8Mat&, const Fp8Mat&, int64_t, int64_t, int64_t,               \
                                             const LinearOut&, const Cut&, float*, hipStream_t);                    \
    template hipError_t launch_fp8_few<T>(const T*, const Fp8Mat&, int64_t, int64_t, int64_t, const LinearOut&,     \
                                          hipStream_t);                                                             \
    template hipError_t launch_fp8_products<T>(const Fp8Product&, const Fp8Product&, const Cut&, const Cut&, float*, \
                                               const ColumnSums<T>&, int64_t, hipStream_t);
MLRS_INST(float)
MLRS_INST(_Float16)
MLRS_INST(__bf16)

}  // namespace train
}  // namespace mlrs
