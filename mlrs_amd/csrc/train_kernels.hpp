// Host side of the training operators' kernels: what capi_train.hip calls.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/mlrs_hip_knn.h"

namespace mlrs {
namespace train {

// Whether a launch may have so many workgroups: a grid holds fewer than 2^32
// threads along an axis, and a larger one is cut short without an error.
inline bool launchable(int64_t workgroups, int threads) { return workgroups * threads < (int64_t)1 << 32; }

// A row-major matrix the matrix-core kernels can read: 16-byte aligned, rows
// a multiple of 16 bytes apart (of f32 in tiles copied by words, any).
struct Mat {
    const void* p;
    int64_t ld;
};

// How a product is cut: the tile, and the parts of its contraction axis.
struct Cut {
    int tile;         // 0: 256 x 256, 1: 128 x 128, 2: 64 x 64, 3: the same, f32 copied by words
    int splits;
    int32_t k_split;
    double us;        // the estimate it was chosen by
    size_t part_bytes(int64_t m, int64_t n) const {
        return splits > 1 ? (size_t)splits * (size_t)n * (size_t)((m + 3) & ~(int64_t)3) * 4 : 0;
    }
};
// Of choices whose grid is launchable, and the largest tiles in any case.
Cut choose_cut(int elem_bytes, int64_t m, int64_t n, int64_t k, int cus, int max_splits = 64, bool words = false);

// A launch that runs only where (*flag == mark) == wanted (flag null: always).
struct Only {
    const uint32_t* flag = nullptr;
    uint32_t mark = 0;
    bool wanted = true;
};

// dst (rows x ld, ld >= cols) := src (rows x cols), zeros behind each row; no
// rows: nothing to do.
struct PackJob {
    const void* src;
    void* dst;
    int64_t rows, cols, ld;
};
template <typename T>
hipError_t launch_pack(const PackJob& a, const PackJob& b, const Only& only, hipStream_t s);

// y (n x m) = act(x w^T + bias) + residual; z, where not null, x w^T + bias.
struct LinearOut {
    const void* bias;
    const void* residual;
    void* y;
    void* z;
    int act;
};
template <typename T>
hipError_t launch_linear(Mat x, Mat w, int64_t n, int64_t m, int64_t k, const LinearOut& o, const Cut& cut,
                         float* part, const Only& only, hipStream_t s);
// The same for at most 32 rows, straight from the caller's unpacked operands, and
// whether that is the faster way.
bool few_rows(int elem_bytes, int64_t n, int64_t m, int64_t k, const Cut& cut);
template <typename T>
hipError_t launch_linear_few(const T* x, const T* w, int64_t n, int64_t m, int64_t k, const LinearOut& o,
                             hipStream_t s);

// Column sums that are still to be joined: out (null: none) := alpha * the sum of
// `parts` runs of rows, parts x columns floats.
template <typename T>
struct ColumnSums {
    T* out;
    float* sums;
    int parts;
    const float* alpha;  // device scalar; may be null
};
int column_parts(int64_t n, int64_t m, int cus);
// dz (n x ld) := dy * act'(z), zeros behind each row (dz may be null), and where
// sums.out its column sums: done with one part, else for launch_products or
// launch_sum_parts.
template <typename T>
hipError_t launch_act_grad(const T* dy, const T* z, int act, int64_t n, int64_t m, T* dz, int64_t ld,
                           const ColumnSums<T>& sums, hipStream_t s);
template <typename T>
hipError_t launch_sum_parts(const ColumnSums<T>& to, int64_t m, hipStream_t s);

// Stores of a product P (m x n, element (i, j) at out[j * ld + i]): a (rows m)
// with its row index contiguous, b (rows n) with k contiguous (b_k) or not.
struct StoreTo {
    void* out;           // of type T, or null: the running sum `acc` is written
    int64_t ld;
    const float* add;    // added first; may be null
    float* acc;          // n x acc_ld
    int64_t acc_ld;      // a multiple of 4
    const float* alpha;  // device scalar; may be null
};
// The two products of a gradient: x (dz w: b with k contiguous) and w (dz^T x: b
// with its row index contiguous); one of m = 0 is not wanted.
struct Product {
    Mat a, b;
    int64_t m, n, k;
    StoreTo to;
};
struct PairCut {
    Cut x, w;
    bool together;  // in one grid
    double us;      // the estimate, of both
    size_t part_bytes(int64_t xm, int64_t xn, int64_t wm, int64_t wn) const {
        return x.part_bytes(xm, xn) + w.part_bytes(wm, wn);
    }
};
PairCut choose_pair(int elem_bytes, int64_t xm, int64_t xn, int64_t xk, int64_t wm, int64_t wn, int64_t wk, int cus,
                    bool words = false);
// sums: of `columns` columns.
template <typename T>
hipError_t launch_products(const Product& x, const Product& w, const PairCut& cut, float* part,
                           const ColumnSums<T>& sums, int64_t columns, const Only& only, hipStream_t s);

// Softmax cross entropy: the statistics of every wave's classes, joined into
// lse and loss; the scale of a half-precision gradient; a piece's gradient.
int64_t stats_parts(int tile, int64_t classes);
template <typename T>
hipError_t launch_xent_stats(Mat h, Mat w, const T* bias, const int64_t* target, int64_t n, int64_t classes, int64_t k,
                             int tile, float* top, float* total, float* hit, const Only& only, hipStream_t s);
hipError_t launch_xent_join(const float* top, const float* total, int64_t parts, const float* hit,
                            const int64_t* target, int64_t n, int64_t classes, int64_t ignore, float* loss, float* lse,
                            const Only& only, hipStream_t s);
hipError_t launch_grad_scale(const float* grad, const int64_t* target, int64_t n, int64_t ignore, float* up_down,
                             hipStream_t s);
// sums: null, or logit_grad_parts(tile, n) runs of rows' column sums (f32's split
// kernels: as of tile 0).
int64_t logit_grad_parts(int tile, int64_t n);
template <typename T>
hipError_t launch_logit_grad(Mat h, Mat w, const T* bias, const int64_t* target, const float* lse, const float* grad,
                             const float* up, int64_t n, int64_t first, int64_t piece, int64_t classes, int64_t k,
                             int64_t ignore, T* out, int64_t ld, float* sums, int tile, const Only& only,
                             hipStream_t s);

// The logits in parts of their contraction (cut.splits > 1, cut.part_bytes(classes,
// n)), and what joins them: every row's loss, or the gradient with `parts` runs of
// rows' column sums (sums may be null).
template <typename T>
hipError_t launch_logit_parts(Mat h, Mat w, int64_t n, int64_t classes, int64_t k, const Cut& cut, float* part,
                              hipStream_t s);
template <typename T>
hipError_t launch_xent_rows(const float* part, const Cut& cut, const T* bias, const int64_t* target, int64_t n,
                            int64_t classes, int64_t ignore, float* loss, float* lse, hipStream_t s);
template <typename T>
hipError_t launch_logit_grad_rows(const float* part, const Cut& cut, const T* bias, const int64_t* target,
                                  const float* lse, const float* grad, const float* up, int64_t n, int64_t classes,
                                  int64_t ignore, T* out, int64_t ld, float* sums, int parts, hipStream_t s);

// f32 products on the bf16 matrix cores (train_split.hpp).  K layout: ld is
// bytes, split_row_bytes of the columns; R layout: ld is elements, a multiple of
// 8, of the three rows of one k.
struct SplitJob {
    const float* src;
    int64_t src_ld;
    void* dst;
    int64_t rows, cols;
    bool r_layout;
};
SplitJob split_job(const float* src, int64_t src_ld, int64_t rows, int64_t cols, void* dst, bool r_layout);
inline int64_t split_row_bytes(int64_t cols) { return (cols + 7) / 8 * 48; }
inline size_t split_bytes(int64_t rows, int64_t cols) { return (size_t)rows * (size_t)split_row_bytes(cols); }
inline Mat split_mat(const void* p, int64_t cols, bool r_layout) {
    return Mat{p, r_layout ? (cols + 7) / 8 * 8 : split_row_bytes(cols)};
}
inline bool split_launchable(int64_t m, int64_t n) { return launchable(((m + 255) / 256) * ((n + 127) / 128), 512); }
Cut choose_cut_split(int64_t m, int64_t n, int64_t k, int cus, int max_splits = 64);
// *flag := mark where an element is not finite.
hipError_t launch_pack_split(const SplitJob& a, const SplitJob& b, uint32_t* flag, uint32_t mark, hipStream_t s);
hipError_t launch_linear_split(Mat x, Mat w, int64_t n, int64_t m, int64_t k, const LinearOut& o, const Cut& cut,
                               float* part, const Only& only, hipStream_t s);
hipError_t launch_product_split(Mat a, Mat b, bool b_k, int64_t m, int64_t n, int64_t k, const StoreTo& o,
                                const Cut& cut, float* part, const Only& only, hipStream_t s);
int64_t stats_parts_split(int64_t classes);
hipError_t launch_xent_stats_split(Mat h, Mat w, const float* bias, const int64_t* target, int64_t n, int64_t classes,
                                   int64_t k, float* top, float* total, float* hit, const Only& only, hipStream_t s);
// w: the piece's classes; bias: the whole vocabulary's.
hipError_t launch_logit_grad_split(Mat h, Mat w, const float* bias, const int64_t* target, const float* lse,
                                   const float* grad, int64_t n, int64_t first, int64_t piece, int64_t classes,
                                   int64_t k, int64_t ignore, float* out, int64_t ld, float* sums,
                                   const Only& only, hipStream_t s);

// Optimizer.
int64_t norm_parts(const mlrs_grad_tensor* t, int64_t count);
hipError_t launch_clip_scale(const mlrs_grad_tensor* t, int64_t count, double max_norm, double* parts, float* norm,
                             float* scale, hipStream_t s);
struct AdamwHyper {
    float b1, c1, b2, c2, step, root, eps;  // c1 = 1 - b1, c2 = 1 - b2
    double lr;
    uint32_t seed;
};
bool adamw_launchable(int64_t len);  // elements of a tensor
hipError_t launch_adamw(const mlrs_adamw_tensor* t, int64_t count, int bits, const AdamwHyper& hy, const float* scale,
                        hipStream_t s);
hipError_t launch_state_values(const uint8_t* codes, const float* scales, int64_t len, int which, float* out,
                               hipStream_t s);

}  // namespace train
}  // namespace mlrs
