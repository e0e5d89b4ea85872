// The f32 products on the bf16 matrix cores: packing into parts, and the
// launches with the training operators' epilogues.
#include <cmath>

#include "train_launch.hpp"
#include "train_split.hpp"

namespace mlrs {
namespace train {

// Measured on this chip, in microseconds: a staged width (32 of k) of a tile,
// and what a round of tiles costs besides.
Cut choose_cut_split(int64_t m, int64_t n, int64_t k, int cus, int max_splits) {
    constexpr double kWidth = 2.4, kRound = 7.0;
    const int64_t widths = std::max<int64_t>(1, (k + kSplitBK - 1) / kSplitBK);
    const int64_t tiles = ((m + 255) / 256) * ((n + 127) / 128);
    Cut best{0, 1, 0, 1e300};
    for (int64_t sp = 1; sp <= max_splits && sp <= widths; sp = sp < 4 ? sp + 1 : sp * 2) {
        const int64_t each = (widths + sp - 1) / sp;
        if (sp > 1 && (each < 3 || (sp - 1) * each >= widths)) continue;
        const double rounds = (double)((tiles * sp + cus - 1) / cus);
        double cost = rounds * ((double)each * kWidth + kRound);
        if (sp > 1) cost += 7.0 + (double)sp * (double)m * (double)n * 8.0 / 4.5e6;
        if (cost < best.us) best = Cut{0, (int)sp, (int32_t)(each * kSplitBK), cost};
    }
    return best;
}

// Two matrices in a launch.  Eight floats of a row become three chunks of bf16;
// one that is not finite (or rounds to an infinity) marks the call.
__global__ __launch_bounds__(256) void pack_split_kernel(SplitJob a, SplitJob b, uint32_t* flag, uint32_t mark) {
    const int64_t total_a = a.rows * ((a.cols + 7) / 8), total = total_a + b.rows * ((b.cols + 7) / 8);
    bool odd = false;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const SplitJob& j = i < total_a ? a : b;
        const int64_t at = i < total_a ? i : i - total_a;
        const int64_t groups = (j.cols + 7) / 8, r = at / groups, c = at - r * groups;
        const float* from = j.src + r * j.src_ld;
        const f32x4 lo = load4(from, 8 * c, j.cols), hi = load4(from, 8 * c + 4, j.cols);
        bf16x8 p0, p1, p2;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = e < 4 ? lo[e] : hi[e - 4];
            p0[e] = (__bf16)x;
            const float x1 = x - (float)p0[e];
            p1[e] = (__bf16)x1;
            p2[e] = (__bf16)(x1 - (float)p1[e]);
            odd |= !(fabsf((float)p0[e]) < __builtin_huge_valf());
        }
        char* to = (char*)j.dst;
        int64_t step;
        if (j.r_layout) {
            to += (r * 3 * groups + c) * 16;
            step = groups * 16;
        } else {
            to += (r * groups + c) * 48;
            step = 16;
        }
        *reinterpret_cast<bf16x8*>(to) = p0;
        *reinterpret_cast<bf16x8*>(to + step) = p1;
        *reinterpret_cast<bf16x8*>(to + 2 * step) = p2;
    }
    if (odd) *flag = mark;
}

SplitJob split_job(const float* src, int64_t src_ld, int64_t rows, int64_t cols, void* dst, bool r_layout) {
    return SplitJob{src, src_ld, dst, rows, cols, r_layout};
}

hipError_t launch_pack_split(const SplitJob& a, const SplitJob& b, uint32_t* flag, uint32_t mark, hipStream_t s) {
    const int64_t total = a.rows * ((a.cols + 7) / 8) + b.rows * ((b.cols + 7) / 8);
    if (total == 0) return hipSuccess;
    const int64_t blocks = std::min<int64_t>((total + 255) / 256, 16384);
    pack_split_kernel<<<dim3((unsigned)blocks), 256, 0, s>>>(a, b, flag, mark);
    return hipGetLastError();
}

template <bool AKC, bool BKC, typename Epi>
static hipError_t launch_split(Mat a, Mat b, int64_t m, int64_t n, int64_t k, const Cut& cut, const Only& only,
                               const Epi& epi, hipStream_t s) {
    GemmArgs g;
    g.a = Operand{a.p, a.ld};
    g.b = Operand{b.p, b.ld};
    g.m = (int32_t)m;
    g.n = (int32_t)n;
    g.k = (int32_t)k;
    g.tiles_m = (int32_t)((m + 255) / 256);
    g.tiles_n = (int32_t)((n + 127) / 128);
    g.splits = cut.splits;
    g.k_split = cut.splits > 1 ? cut.k_split : (int32_t)std::max<int64_t>(k, 1);
    g.band = std::min<int32_t>(g.tiles_m, 4);
    g.flag = only.flag;
    g.mark = only.mark;
    g.wanted = only.wanted;
    const int64_t blocks = (int64_t)g.tiles_m * g.tiles_n * cut.splits;
    if (!launchable(blocks, 512)) return hipErrorInvalidConfiguration;  // the caller has checked
    gemm_split_kernel<AKC, BKC, Epi><<<dim3((unsigned)blocks), 512, 0, s>>>(g, epi);
    return hipGetLastError();
}

hipError_t launch_linear_split(Mat x, Mat w, int64_t n, int64_t m, int64_t k, const LinearOut& o, const Cut& cut,
                               float* part, const Only& only, hipStream_t s) {
    const LinearEpi<float> e = linear_epi<float>(o, m);
    if (cut.splits == 1) return launch_split<true, true>(w, x, m, n, k, cut, only, e, s);
    const hipError_t r = launch_split<true, true>(w, x, m, n, k, cut, only, parts_epi<float>(part, m, n), s);
    if (r != hipSuccess) return r;
    return launch_join(part, cut.splits, m, n, LinearPoint<float>{e}, only, s);
}

hipError_t launch_product_split(Mat a, Mat b, bool b_k, int64_t m, int64_t n, int64_t k, const StoreTo& o,
                                const Cut& cut, float* part, const Only& only, hipStream_t s) {
    const StoreEpi<float> e = store_epi<float>(o);
    if (cut.splits == 1)
        return b_k ? launch_split<false, true>(a, b, m, n, k, cut, only, e, s)
                   : launch_split<false, false>(a, b, m, n, k, cut, only, e, s);
    const StoreEpi<float> pe = parts_epi<float>(part, m, n);
    const hipError_t r = b_k ? launch_split<false, true>(a, b, m, n, k, cut, only, pe, s)
                             : launch_split<false, false>(a, b, m, n, k, cut, only, pe, s);
    if (r != hipSuccess) return r;
    return launch_join(part, cut.splits, m, n, StorePoint<float>{e}, only, s);
}

int64_t stats_parts_split(int64_t classes) { return (classes + 255) / 256 * 4; }

hipError_t launch_xent_stats_split(Mat h, Mat w, const float* bias, const int64_t* target, int64_t n, int64_t classes,
                                   int64_t k, float* top, float* total, float* hit, const Only& only, hipStream_t s) {
    const StatsEpi<float> e{bias, target, top, total, hit};
    return launch_split<true, true>(w, h, classes, n, k, Cut{0, 1, 0, 0.0}, only, e, s);
}

hipError_t launch_logit_grad_split(Mat h, Mat w, const float* bias, const int64_t* target, const float* lse,
                                   const float* grad, int64_t n, int64_t first, int64_t piece, int64_t classes,
                                   int64_t k, int64_t ignore, float* out, int64_t ld, float* sums,
                                   const Only& only, hipStream_t s) {
    const LogitGradEpi<float> e{bias ? bias + first : nullptr, target, lse, grad, nullptr, out, sums, ld, ignore,
                                (int32_t)first, (int32_t)classes};
    return launch_split<true, true>(w, h, piece, n, k, Cut{0, 1, 0, 0.0}, only, e, s);
}

}  // namespace train
}  // namespace mlrs
