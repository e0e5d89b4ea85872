// The optimizer step over many tensors: the norm of all gradients with the
// factor that clips it, and AdamW with its two moments in 32 or in 8 bits.
//
// A launch takes as many tensors as its arguments have room for with their
// addresses and sizes (45 of a step, 135 of a norm; no table in memory, nothing
// kept between calls), and cuts them into runs of kRun elements, one per
// workgroup; a workgroup finds its tensor by bisection of the running counts.
#include <algorithm>
#include <cmath>

#include "train_epilogue.hpp"
#include "train_kernels.hpp"

namespace mlrs {
namespace train {

constexpr int kTableBytes = 3800;  // of the 4 KB of a launch's arguments
constexpr int kRun = 4096;         // elements of a workgroup: 16 per thread
constexpr int kBlock = 256;        // elements that share a scale of an 8-bit state
constexpr int64_t kMostRuns = ((int64_t)1 << 24) - 1;  // of a launch: 2^32 threads are one too many

enum { kF32 = 0, kF16 = 1, kBF16 = 2 };

template <typename Item>
struct Batch {
    static constexpr int kTensors = kTableBytes / (int)(sizeof(Item) + 4);
    Item item[kTensors];
    int32_t first[kTensors + 1];  // running counts of runs
    int32_t count;
};

template <typename Item>
__device__ __forceinline__ int find_item(const Batch<Item>& b, int32_t run) {
    int lo = 0, hi = b.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (b.first[mid] <= run)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

// Four elements from i on as floats; those at or past `end` are 0.
__device__ __forceinline__ f32x4 load_any(const void* p, int dtype, int64_t i, int64_t end) {
    switch (dtype) {
    case kF32: return load4((const float*)p, i, end);
    case kF16: return load4((const _Float16*)p, i, end);
    default: return load4((const __bf16*)p, i, end);
    }
}
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, int64_t end, f32x4 v) {
    switch (dtype) {
    case kF32: store4((float*)p, i, end, v); break;
    case kF16: store4((_Float16*)p, i, end, v); break;
    default: store4((__bf16*)p, i, end, v); break;
    }
}


// ---------------------------------------------------------------------------
// the norm of all gradients
// ---------------------------------------------------------------------------
struct NormItem {
    const void* g;
    int64_t len;
    int32_t dtype;
};

// A workgroup's sum of squares, in f64 from the squares on, as f32 and bf16
// elements past 2^64 or below 2^-75 have squares that f32 cannot hold.  Added in a
// fixed order: a thread's sixteen, the threads', the workgroups'.  202M bf16
// gradients: 112 us with the join, 110 with the squares in f32.
__global__ __launch_bounds__(256) void norm_kernel(Batch<NormItem> b, double* __restrict__ parts) {
    const int t = find_item(b, (int32_t)blockIdx.x);
    const NormItem& it = b.item[t];
    const int64_t at = (int64_t)((int32_t)blockIdx.x - b.first[t]) * kRun;
    double d = 0.0;
#pragma unroll
    for (int u = 0; u < kRun / 1024; ++u) {
        const int64_t i = at + u * 1024 + threadIdx.x * 4;
        if (i >= it.len) continue;
        const f32x4 v = load_any(it.g, it.dtype, i, it.len);
#pragma unroll
        for (int e = 0; e < 4; ++e) d = __builtin_fma((double)v[e], (double)v[e], d);
    }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) d += __shfl_xor(d, s);
    __shared__ double join[4];
    if ((threadIdx.x & 63) == 0) join[threadIdx.x >> 6] = d;
    __syncthreads();
    if (threadIdx.x == 0) parts[blockIdx.x] = (join[0] + join[1]) + (join[2] + join[3]);
}

// norm, and scale = min(1, max_norm / norm); NaN where the norm is not finite.
__global__ __launch_bounds__(1024) void norm_join_kernel(const double* __restrict__ parts, int64_t n, double max_norm,
                                                         float* __restrict__ norm, float* __restrict__ scale) {
    double d = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) d += parts[i];
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) d += __shfl_xor(d, s);
    __shared__ double join[16];
    if ((threadIdx.x & 63) == 0) join[threadIdx.x >> 6] = d;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int i = 1; i < 16; ++i) d += join[i];
    const double root = sqrt(d);
    *norm = (float)root;
    const bool finite = (float)root < __builtin_huge_valf();  // false for NaN too
    *scale = !finite ? __builtin_nanf("") : root > max_norm ? (float)(max_norm / root) : 1.0f;
}

static int64_t runs_of(int64_t len) { return (len + kRun - 1) / kRun; }

int64_t norm_parts(const mlrs_grad_tensor* t, int64_t count) {
    int64_t n = 0;
    for (int64_t i = 0; i < count; ++i) n += runs_of(t[i].len);
    return n;
}

// Fills batches of tensors and launches each: add(item, index, from, len) describes
// `len` elements of a tensor, all of them but where a launch cannot hold as many;
// go(batch, runs) launches.
template <typename Item, typename Len, typename Add, typename Go>
static hipError_t in_batches(int64_t count, Len len, Add add, Go go) {
    Batch<Item> b;
    int n = 0;
    int64_t runs = 0;
    for (int64_t i = 0; i < count; ++i) {
        const int64_t whole = len(i);
        for (int64_t from = 0; from < whole; from += kMostRuns * kRun) {
            const int64_t part = std::min(whole - from, kMostRuns * kRun), r = runs_of(part);
            if (n == Batch<Item>::kTensors || (n > 0 && runs + r > kMostRuns)) {
                b.first[n] = (int32_t)runs;
                b.count = n;
                const hipError_t e = go(b, runs);
                if (e != hipSuccess) return e;
                n = 0;
                runs = 0;
            }
            b.first[n] = (int32_t)runs;
            add(b.item[n], i, from, part);
            ++n;
            runs += r;
        }
    }
    if (n == 0) return hipSuccess;
    b.first[n] = (int32_t)runs;
    b.count = n;
    return go(b, runs);
}

hipError_t launch_clip_scale(const mlrs_grad_tensor* t, int64_t count, double max_norm, double* parts, float* norm,
                             float* scale, hipStream_t s) {
    int64_t at = 0;
    hipError_t e = in_batches<NormItem>(
        count, [&](int64_t i) { return t[i].len; },
        [&](NormItem& it, int64_t i, int64_t from, int64_t len) {
            it.g = (const char*)t[i].grad + from * (t[i].dtype == kF32 ? 4 : 2);
            it.len = len;
            it.dtype = t[i].dtype;
        },
        [&](const Batch<NormItem>& b, int64_t runs) {
            norm_kernel<<<dim3((unsigned)runs), 256, 0, s>>>(b, parts + at);
            at += runs;
            return hipGetLastError();
        });
    if (e != hipSuccess) return e;
    norm_join_kernel<<<1, 1024, 0, s>>>(parts, at, max_norm, norm, scale);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// AdamW
// ---------------------------------------------------------------------------
struct AdamwItem {
    void* param;
    const void* grad;
    void* avg;     // f32, or codes
    void* sq;      // f32, or codes of the root
    float* master;
    float* avg_scale;
    float* sq_scale;
    int64_t len;
    float decay;   // 1 - lr * weight_decay
    uint32_t key;  // of the roundings
    uint8_t param_dtype, grad_dtype;
};

// 8-bit states.  The first moment is a sign and seven bits, four of exponent
// and three of fraction; the second is kept as its root, whose range is half
// as many powers of two, in four bits each.  A block's scale is its largest
// magnitude over the format's largest value, so exponent 15 stands for 2^0 and
// the smallest step is 2^-17 or 2^-18 of about the largest.  A decaying average
// moves by less than half a step from one call to the next, and rounding to
// nearest would hold it where it is: a value is rounded up with the probability
// of its remainder, by bits of a hash of the element and the call's seed.
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x6A09E667u;  // odd 32-bit fractions of sqrt(2) and sqrt(3)
    x = (x ^ (x >> 15)) * 0xBB67AE85u;
    return x ^ (x >> 16);
}

template <int MANT>
__device__ __forceinline__ float code_value(uint32_t code) {
    const uint32_t e = code >> MANT, f = code & ((1u << MANT) - 1u);
    const float small = (float)f * __uint_as_float((uint32_t)(127 - 14 - MANT) << 23);
    return e ? __uint_as_float((code + (112u << MANT)) << (23 - MANT)) : small;
}

// y >= 0, at most about the format's largest value; r16: sixteen random bits.
template <int MANT>
__device__ __forceinline__ uint32_t value_code(float y, uint32_t r16) {
    const uint32_t big = ((__float_as_uint(y) + (r16 << (7 - MANT))) >> (23 - MANT)) - (112u << MANT);
    const uint32_t small = (uint32_t)floorf(y * (float)(1u << (14 + MANT)) + (float)r16 * 1.52587890625e-05f);
    const uint32_t c = y < 6.103515625e-05f ? small : big;  // 2^-14
    constexpr uint32_t most = (16u << MANT) - 1u;
    return c < most ? c : most;
}

__device__ __forceinline__ float avg_value(uint32_t code) {
    const float v = code_value<3>(code & 127u);
    return code > 127u ? -v : v;
}

// The largest of a wave's non-negative floats, by their bits: a NaN is larger
// than infinity and so marks its block.
__device__ __forceinline__ float wave_most(float v) {
    uint32_t b = __float_as_uint(v);
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)b, s);
        b = o > b ? o : b;
    }
    return __uint_as_float(b);
}

__device__ __forceinline__ float most4(f32x4 v) {
    uint32_t b = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t o = __float_as_uint(v[e]) & 0x7FFFFFFFu;
        b = o > b ? o : b;
    }
    return __uint_as_float(b);
}

// Every operation is rounded by itself, in the order written (the build
// contracts nothing), so that an 8-bit state follows from its inputs alone.
// A wave holds 256 consecutive elements, the block of an 8-bit scale.  Bound by
// memory: 28 bytes an element with 32-bit states (202M bf16 parameters with
// masters in 1.06 to 1.22 ms by the card with their norm, 4.65 TB/s on the one where
// a copy reaches 4.75), 16 with 8-bit states and f32 parameters (164M in 0.89 ms
// with reading the values back, 4.4 TB/s).
template <int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(Batch<AdamwItem> b, AdamwHyper hy,
                                                    const float* __restrict__ scale_p) {
    const int t = find_item(b, (int32_t)blockIdx.x);
    const AdamwItem& it = b.item[t];
    const int64_t at = (int64_t)((int32_t)blockIdx.x - b.first[t]) * kRun;
    const float scale = scale_p ? *scale_p : 1.0f;
    if (!(fabsf(scale) < __builtin_huge_valf())) return;  // gradients that are not finite: no step
#pragma unroll
    for (int u = 0; u < kRun / 1024; ++u) {
        const int64_t i = at + u * 1024 + threadIdx.x * 4;
        if (i - (int64_t)(threadIdx.x & 63) * 4 >= it.len) return;  // the wave is past the end
        const int64_t end = it.len;
        f32x4 p = {}, g = {}, m = {}, r = {}, v = {};
        float* master = it.master;
        if (i < end) {
            p = master ? load4(master, i, end) : load_any(it.param, it.param_dtype, i, end);
            g = load_any(it.grad, it.grad_dtype, i, end);
            if (scale_p) g *= scale;
            if constexpr (BITS == 32) {
                m = load4((const float*)it.avg, i, end);
                v = load4((const float*)it.sq, i, end);
            } else {
                const float ms = it.avg_scale[i / kBlock], rs = it.sq_scale[i / kBlock];
                uint32_t mc = 0, rc = 0;
                if (i + 4 <= end) {
                    __builtin_memcpy(&mc, (const uint8_t*)it.avg + i, 4);
                    __builtin_memcpy(&rc, (const uint8_t*)it.sq + i, 4);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (i + e < end) {
                            mc |= (uint32_t)((const uint8_t*)it.avg)[i + e] << (8 * e);
                            rc |= (uint32_t)((const uint8_t*)it.sq)[i + e] << (8 * e);
                        }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    m[e] = avg_value((mc >> (8 * e)) & 255u) * ms;
                    const float root = code_value<4>((rc >> (8 * e)) & 255u) * rs;
                    v[e] = root * root;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            m[e] = m[e] * hy.b1 + g[e] * hy.c1;
            v[e] = v[e] * hy.b2 + (g[e] * hy.c2) * g[e];
            r[e] = sqrtf(v[e]);
            p[e] = p[e] * it.decay - (m[e] / (r[e] * hy.root + hy.eps)) * hy.step;
            if constexpr (BITS == 8)
                if (i + e >= end) m[e] = r[e] = 0.0f;  // no part of the block
        }
        if (i < end) {
            if (master) store4(master, i, end, p);
            store_any(it.param, it.param_dtype, i, end, p);
        }
        if constexpr (BITS == 32) {
            if (i < end) {
                store4((float*)it.avg, i, end, m);
                store4((float*)it.sq, i, end, v);
            }
        } else {
            const float ms = wave_most(most4(m)) / 1.875f, rs = wave_most(most4(r)) / 1.9375f;
            uint32_t mc = 0, rc = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint64_t idx = (uint64_t)(i + e);
                const uint32_t h = mix32(((uint32_t)idx ^ it.key) + (uint32_t)(idx >> 32) * 0x9E3779B1u);
                uint32_t c = value_code<3>(ms > 0.0f ? fabsf(m[e]) / ms : 0.0f, h & 0xFFFFu);
                if (m[e] < 0.0f) c |= 128u;
                mc |= c << (8 * e);
                c = value_code<4>(rs > 0.0f ? r[e] / rs : 0.0f, h >> 16);
                // a root that is not zero stays so: it divides
                if (r[e] > 0.0f && c == 0) c = 1;
                rc |= c << (8 * e);
            }
            if (i < end) {
                if (i + 4 <= end) {
                    __builtin_memcpy((uint8_t*)it.avg + i, &mc, 4);
                    __builtin_memcpy((uint8_t*)it.sq + i, &rc, 4);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (i + e < end) {
                            ((uint8_t*)it.avg)[i + e] = (uint8_t)(mc >> (8 * e));
                            ((uint8_t*)it.sq)[i + e] = (uint8_t)(rc >> (8 * e));
                        }
                }
            }
            if ((threadIdx.x & 63) == 0) {  // i < end: the wave is not past the end
                it.avg_scale[i / kBlock] = ms;
                it.sq_scale[i / kBlock] = rs;
            }
        }
    }
}

bool adamw_launchable(int64_t len) { return runs_of(len) <= kMostRuns; }

hipError_t launch_adamw(const mlrs_adamw_tensor* t, int64_t count, int bits, const AdamwHyper& hy, const float* scale,
                        hipStream_t s) {
    return in_batches<AdamwItem>(
        count, [&](int64_t i) { return t[i].len; },
        [&](AdamwItem& it, int64_t i, int64_t, int64_t) {  // whole: mlrs_adamw_step has checked
            const mlrs_adamw_tensor& x = t[i];
            it.param = x.param;
            it.grad = x.grad;
            it.avg = x.exp_avg;
            it.sq = x.exp_avg_sq;
            it.master = x.master;
            it.avg_scale = x.avg_scale;
            it.sq_scale = x.avg_sq_scale;
            it.len = x.len;
            it.decay = (float)(1.0 - hy.lr * x.weight_decay);
            it.key = mix32(hy.seed + (uint32_t)i * 0x9E3779B1u);
            it.param_dtype = (uint8_t)x.param_dtype;
            it.grad_dtype = (uint8_t)x.grad_dtype;
        },
        [&](const Batch<AdamwItem>& b, int64_t runs) {
            if (bits == 32)
                adamw_kernel<32><<<dim3((unsigned)runs), 256, 0, s>>>(b, hy, scale);
            else
                adamw_kernel<8><<<dim3((unsigned)runs), 256, 0, s>>>(b, hy, scale);
            return hipGetLastError();
        });
}

// The values that 8-bit codes stand for.
template <bool ROOT>
__global__ __launch_bounds__(256) void state_values_kernel(const uint8_t* __restrict__ codes,
                                                           const float* __restrict__ scales, int64_t len,
                                                           float* __restrict__ out) {
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < len; i += (int64_t)gridDim.x * 1024) {
        uint32_t c = 0;
        if (i + 4 <= len) {
            __builtin_memcpy(&c, codes + i, 4);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < len) c |= (uint32_t)codes[i + e] << (8 * e);
        }
        const float sc = scales[i / kBlock];
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t x = (c >> (8 * e)) & 255u;
            v[e] = (ROOT ? code_value<4>(x) : avg_value(x)) * sc;
        }
        store4(out, i, len, v);
    }
}

hipError_t launch_state_values(const uint8_t* codes, const float* scales, int64_t len, int which, float* out,
                               hipStream_t s) {
    const int64_t blocks = std::min<int64_t>((len + 1023) / 1024, 65536);
    if (which == 0)
        state_values_kernel<false><<<dim3((unsigned)blocks), 256, 0, s>>>(codes, scales, len, out);
    else
        state_values_kernel<true><<<dim3((unsigned)blocks), 256, 0, s>>>(codes, scales, len, out);
    return hipGetLastError();
}

}  // namespace train
}  // namespace mlrs
