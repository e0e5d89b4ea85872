// f32 products on the bf16 matrix cores.  A float is the sum of three bf16
// numbers (8 bits of its significand each, rounded to nearest, so the remainders
// are signed), and a b = a0 b0 + a0 b1 + a1 b0 + a1 b1 + a0 b2 + a2 b0 up to
// 2^-25 of |a b|: six instructions that run at sixteen times the f32 rate.  The
// exponent range is f32's, so nothing is scaled.  An infinity or a NaN has no
// such parts: packing marks the call, and the f32 kernels take it over
// (GemmArgs::flag).
//
// Layouts, made by pack_split_kernel.  K layout: eight k of a row are 48 bytes,
// the first parts of all eight, the second, the third.  R layout: the row of a
// k is three rows, one of each part.
#pragma once
#include "train_gemm.hpp"

namespace mlrs {
namespace train {

constexpr int kSplitBK = 32;                  // k of a staged width
constexpr int kSplitRowBytes = 6 * kSplitBK;  // of a row in it (K layout)

// An operand's copy into LDS: 96 of its rows of one k and part (R layout), or
// 192 bytes of each row (K layout).
template <bool KC, int ROWS, int WAVES>
struct SplitStager {
    static constexpr int kInstr = ROWS * kSplitRowBytes / 1024 / WAVES;
    static constexpr int kChunks = ROWS * 2 / 16;
    static_assert(kInstr * WAVES * 1024 == ROWS * kSplitRowBytes, "whole copies");
    const char* base;
    int64_t bytes, step;
    int32_t chunk[kInstr];
    uint32_t off[kInstr];

    // o.ld: bytes of a row (K layout) or elements of one of the three (R layout)
    __device__ __forceinline__ void init(const Operand& o, int32_t row0, int32_t rows, int32_t k, int wave, int lane) {
        const int64_t ldb = KC ? o.ld : o.ld * 2;
        const int64_t at = KC ? (int64_t)row0 * ldb : (int64_t)row0 * 2;
        base = reinterpret_cast<const char*>(o.p) + at;
        bytes = (KC ? (int64_t)rows * ldb : (int64_t)k * 3 * ldb) - at;
        step = KC ? 6 : 3 * ldb;
#pragma unroll
        for (int i = 0; i < kInstr; ++i) {
            const int q = (wave * kInstr + i) * 64 + lane;
            chunk[i] = 0;
            if constexpr (KC) {
                const int r = q / 12, c = (q % 12) ^ ((r >> 2) & 3);
                chunk[i] = 16 * c;
                off[i] = (uint32_t)r * (uint32_t)ldb + 16u * (uint32_t)c;
            } else {
                const int row = q / kChunks;
                const int c = (q % kChunks) ^ r_swizzle<__bf16, ROWS>(row / 3);
                off[i] = (uint32_t)row * (uint32_t)ldb + 16u * (uint32_t)c;
            }
        }
    }

    // k: the end of the contraction, of K layout padded to eight
    __device__ __forceinline__ void load(char* lds, int32_t k0, int32_t k, int wave) const {
#if defined(__HIP_DEVICE_COMPILE__)
        const int64_t skip = (int64_t)k0 * step;
        const int64_t left = bytes - skip;
        const uint64_t at = (uint64_t)(base + skip);
        u32x4 rsrc;
        rsrc[0] = (uint32_t)at;
        rsrc[1] = (uint32_t)(at >> 32) & 0xFFFFu;
        rsrc[2] = left < 0x7FFFFFFF ? (left > 0 ? (uint32_t)left : 0u) : 0x7FFFFFFFu;
        rsrc[3] = 0x00027000u;
        const int32_t row_left = (k - k0) * 6;  // bytes of a row
#pragma unroll
        for (int i = 0; i < kInstr; ++i)
            copy_to_lds(rsrc, lds + (wave * kInstr + i) * 1024, KC && chunk[i] >= row_left ? 0x80000000u : off[i]);
#else
        (void)lds;
        (void)k0;
        (void)k;
        (void)wave;
#endif
    }
};

template <bool KC, int ROWS, int BLOCKS>
struct SplitReader {
    int at[KC ? 3 : BLOCKS];

    __device__ __forceinline__ void init(int first, int lane) {
        const int g = lane >> 4, r = lane & 15;
        if constexpr (KC) {
            // (row >> 2) & 3 is the same in every block
#pragma unroll
            for (int p = 0; p < 3; ++p) at[p] = (first + r) * kSplitRowBytes + (((3 * g + p) ^ ((r >> 2) & 3)) << 4);
        } else {
            const int q = r >> 2, p = lane & 3;
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
                const int c = ((first >> 4) + b) * 2 + (p >> 1);
                at[b] = (8 * g + q) * 3 * (ROWS * 2) + ((c ^ r_swizzle<__bf16, ROWS>(8 * g + q)) << 4) + (p & 1) * 8;
            }
        }
    }
    __device__ __forceinline__ bf16x8 get(const char* lds, int part, int b) const {
#if defined(__HIP_DEVICE_COMPILE__)
        if constexpr (KC) {
            return *reinterpret_cast<const bf16x8*>(lds + at[part] + b * 16 * kSplitRowBytes);
        } else {
            const char* q = lds + at[b] + part * (ROWS * 2);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MLRS_LDS s16x4*)q);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MLRS_LDS s16x4*)(q + 4 * 3 * (ROWS * 2)));
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
#else
        (void)lds;
        (void)part;
        (void)b;
        return bf16x8{};
#endif
    }
};

// 256 x 128 tiles, eight waves of 64 x 64.  A staged width of both operands is 72
// KB, two of them are in LDS.  Its six products go from the small ones to the
// large; fragments of the next width are read over those that are done with,
// the parts a1, b1, a2, b2 in this width, a0 and b0 during the next one's first
// product, so one set of registers serves: the barrier stands after the second
// product, where every fragment of this width is in registers.  4096^3: 600 us,
// 229 TFLOP/s of f32 work or 1370 of bf16, and 55 for packing.
template <bool AKC, bool BKC, typename Epi>
__global__ __launch_bounds__(512, 2) void gemm_split_kernel(GemmArgs g, Epi epi) {
    constexpr int WM = 4, WN = 2, MB = 4, NB = 4, WAVES = 8;
    constexpr int BM = WM * MB * 16, BN = WN * NB * 16;
    constexpr int kA = BM * kSplitRowBytes, kB = BN * kSplitRowBytes, kStage = kA + kB;
    constexpr int BK = kSplitBK;
    __shared__ __attribute__((aligned(1024))) char buf[2 * kStage];
    if (skipped(g)) return;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const TilePlace t = tile_place(g, blockIdx.x);
    const int32_t m0 = t.tm * BM, n0 = t.tn * BN;
    const int32_t k_lo = t.split * g.k_split;
    const int32_t k_hi = g.k - k_lo < g.k_split ? g.k : k_lo + g.k_split;
    // of K layout: the zeros behind a row belong to it
    const int32_t k_end = k_hi == g.k ? (k_hi + 7) & ~7 : k_hi;

    SplitStager<AKC, BM, WAVES> sa;
    SplitStager<BKC, BN, WAVES> sb;
    sa.init(g.a, m0, g.m, k_hi, wave, lane);
    sb.init(g.b, n0, g.n, k_hi, wave, lane);
    SplitReader<AKC, BM, MB> ra;
    SplitReader<BKC, BN, NB> rb;
    ra.init(wm * MB * 16, lane);
    rb.init(wn * NB * 16, lane);

    f32x4 acc[MB][NB] = {};
    bf16x8 a0[MB], a1[MB], a2[MB], b0[NB], b1[NB], b2[NB];
    auto fetch_a = [&](bf16x8(&f)[MB], const char* from, int part) {
#pragma unroll
        for (int i = 0; i < MB; ++i) f[i] = ra.get(from, part, i);
    };
    auto fetch_b = [&](bf16x8(&f)[NB], const char* from, int part) {
#pragma unroll
        for (int j = 0; j < NB; ++j) f[j] = rb.get(from + kA, part, j);
    };
    auto multiply = [&](const bf16x8(&a)[MB], const bf16x8(&b)[NB]) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int i = 0; i < MB; ++i) acc[i][j] = mfma_step<__bf16>(a[i], b[j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
    };
    constexpr int IA = decltype(sa)::kInstr, IB = decltype(sb)::kInstr;

    sa.load(buf, k_lo, k_end, wave);
    sb.load(buf + kA, k_lo, k_end, wave);
    sa.load(buf + kStage, k_lo + BK, k_end, wave);
    sb.load(buf + kStage + kA, k_lo + BK, k_end, wave);
    wait_copies<IA + IB>();
    __builtin_amdgcn_s_barrier();
    fetch_a(a1, buf, 1);
    fetch_b(b1, buf, 1);
    fetch_a(a2, buf, 2);
    fetch_b(b2, buf, 2);
    int cur = 0;
    for (int32_t k0 = k_lo; k0 < k_hi; k0 += BK) {
        const char *here = buf + cur, *next = buf + (kStage - cur);
        __builtin_amdgcn_sched_barrier(0);
        fetch_b(b0, here, 0);
        fetch_a(a0, here, 0);
        multiply(a1, b1);
        multiply(a2, b0);
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        wait_copies<0>();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        sa.load(buf + cur, k0 + 2 * BK, k_end, wave);
        fetch_a(a2, next, 2);
        multiply(a0, b2);
        sb.load(buf + cur + kA, k0 + 2 * BK, k_end, wave);
        fetch_b(b2, next, 2);
        multiply(a1, b0);
        fetch_a(a1, next, 1);
        multiply(a0, b1);
        fetch_b(b1, next, 1);
        multiply(a0, b0);
        cur = kStage - cur;
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);
    wait_copies<0>();  // of widths past the end

    Place p;
    p.m0 = m0 + wm * MB * 16;
    p.n0 = n0 + wn * NB * 16;
    p.m = g.m;
    p.n = g.n;
    p.split = t.split;
    p.tile_m = t.tm;
    p.lane = lane;
    p.wave = wave;
    p.wm = wm;
    p.wn = wn;
    epi.template run<WM, WN, MB, NB>(acc, p, buf);
}

}  // namespace train
}  // namespace mlrs
