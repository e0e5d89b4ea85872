/*
 * mlrs_hip_knn.h -- C ABI of the MI355X (gfx950) brute-force kNN engine.
 *
 * Drop-in replacement for the kernel launches behind mlrs-backend's
 * brute-force kNN / k-means-assignment / pairwise-distance prims.  Every entry
 * point:
 *   - takes DEVICE pointers (HIP, owned by the caller) plus each buffer's
 *     element count, so the geometry checks of the Rust prims can run here;
 *   - validates everything BEFORE any launch and returns 0 or a negative
 *     MLRS_ERR_* code; mlrs_last_error() then describes the failure with the
 *     same fields as mlrs_core::PrimError (crates/mlrs-core/src/error.rs:62);
 *   - enqueues its work on `stream` (a hipStream_t; NULL = the null stream)
 *     and returns without synchronizing, except when it must grow one of its
 *     cached device buffers: growth synchronizes the WHOLE device (every
 *     stream, other libraries' work included) before freeing the old buffer;
 *   - is callable from any thread, one call at a time per process (the
 *     Rust side serializes through its global pool mutex,
 *     crates/mlrs-py/src/lib.rs:104-186); calls are serialized internally;
 *   - runs after the previous call on the same device even when the two
 *     calls name different streams: the cached buffers are shared, so a call
 *     on another stream than the last call's first makes its stream wait for
 *     the last call's work (an event recorded at the end of every call), as
 *     the reference's single stream orders them
 *     (crates/mlrs-backend/src/stream_cap.rs:69).  The caller still orders
 *     its own reads of the outputs after the call's stream.
 * Results equal mlrs's cpu-backend arithmetic bit for bit: the same arm
 * (direct / metric / host) the cpu dispatch would pick for the shape
 * (crates/mlrs-algos/src/neighbors/nearest.rs:891-953) is evaluated in the same
 * operation order, and selection uses the (value, index) order with the lowest
 * index winning ties.
 */
#ifndef MLRS_HIP_KNN_H
#define MLRS_HIP_KNN_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ---- */
#define MLRS_OK 0
#define MLRS_ERR_SHAPE_MISMATCH (-1) /* PrimError::ShapeMismatch{operand, rows, cols, len} */
#define MLRS_ERR_DIM_MISMATCH (-2)   /* PrimError::DimMismatch{dim(operand), lhs(rows), rhs(cols)} */
#define MLRS_ERR_UNSUPPORTED (-3)    /* metric or shape this build does not serve */
#define MLRS_ERR_NULL_POINTER (-4)   /* a required pointer was NULL */
#define MLRS_ERR_HIP (-5)            /* a HIP runtime call failed (hip_error holds it) */
#define MLRS_ERR_ALLOC (-6)          /* device workspace allocation failed */
#define MLRS_ERR_INVALID_PARAM (-7)  /* AlgoError::InvalidEps-style rejection of a scalar (operand names it) */

/* ---- metrics: the variants of the Metric enum of crates/mlrs-backend/src/prims/knn_graph.rs:61-75
 *      (numbered here, not in the enum's declaration order) ---- */
#define MLRS_METRIC_EUCLIDEAN 0
#define MLRS_METRIC_COSINE 1
#define MLRS_METRIC_MANHATTAN 2
#define MLRS_METRIC_CHEBYSHEV 3
#define MLRS_METRIC_MINKOWSKI 4 /* exponent in the `p` argument, p >= 1 */

typedef struct mlrs_error_info {
    int32_t code;        /* the MLRS_ERR_* value returned */
    char operand[32];    /* PrimError operand / dim name, e.g. "x", "y", "k", "out" */
    int64_t rows;        /* ShapeMismatch rows   | DimMismatch lhs */
    int64_t cols;        /* ShapeMismatch cols   | DimMismatch rhs */
    int64_t len;         /* ShapeMismatch len */
    int32_t hip_error;   /* hipError_t for MLRS_ERR_HIP / MLRS_ERR_ALLOC */
    char message[160];   /* human-readable, PrimError's Display text */
} mlrs_error_info;

/* Details of the calling thread's last failed call. Returns its code. */
int32_t mlrs_last_error(mlrs_error_info *out);
/* Static description of a status code. */
const char *mlrs_status_string(int32_t code);
/* ABI version of this header (bumped on any signature change). */
int32_t mlrs_abi_version(void);
#define MLRS_ABI_VERSION 5

/*
 * Brute-force k nearest training rows of every query row.
 *
 * Replaces: the arm chosen by metric_topk (nearest.rs:891-953) --
 *   cpu_rows_topk (crates/mlrs-backend/src/prims/knn.rs:491-671),
 *   cpu_metric_rows_topk (prims/knn.rs:732-898),
 *   knn_host_topk (crates/mlrs-backend/src/prims/knn_host.rs:210-304),
 *   fused_distance_topk (prims/knn.rs:1070-1323) and
 *   tiled_distance_topk / tiled_metric_distance_topk (nearest.rs:1058-1512).
 * Layout: xq is n_query x n_features, x_train n_train x n_features, both
 *   row-major; out_dist / out_idx are n_query x k row-major, each row ascending
 *   by (distance, index).  Distances are TRUE distances (Euclidean: the root of
 *   the selected squared values; cosine: 1 - cos, clamped to [0, 2];
 *   Manhattan: sum |x-y|; Chebyshev: max |x-y| by select, NaN never replacing;
 *   Minkowski: (sum |x-y|^p)^(1/p), |x-y|^p by a multiply chain for an integer
 *   p in 3..8 (minkowski_powi, prims/knn.rs:680-687), pow otherwise, and the
 *   root pow(v, (F)(1/p)) on the selected values).  A slot no admissible
 *   (non-NaN) candidate filled holds (+inf, 0).
 * Errors (checked in this order, before any launch, mirroring
 *   cpu_metric_rows_topk / knn_host_topk):
 *   ShapeMismatch "x"        n_query*n_features != xq_len
 *   ShapeMismatch "y"        n_train*n_features != xt_len
 *   ShapeMismatch "k"        k < 1 or k > n_train           (rows=1, cols=k, len=n_train)
 *   ShapeMismatch "features" n_features < 1
 *   ShapeMismatch "rows"     n_query or n_train > UINT32_MAX
 *   ShapeMismatch "out"      out_len != n_query*k
 *   MLRS_ERR_UNSUPPORTED     metric not served, or a Minkowski p below 1 (or NaN)
 * Every 1 <= k <= n_train is served (knn_host_possible,
 *   crates/mlrs-backend/src/prims/knn_host.rs:182-184; top_k,
 *   crates/mlrs-backend/src/prims/topk.rs:208-212).
 * `p` is the Minkowski exponent, ignored by the other metrics.
 */
int32_t mlrs_knn_topk_f32(const float *xq, int64_t xq_len, int64_t n_query, int64_t n_features,
                          const float *x_train, int64_t xt_len, int64_t n_train, int32_t k,
                          int32_t metric, double p, float *out_dist, uint32_t *out_idx,
                          int64_t out_len, void *stream);
int32_t mlrs_knn_topk_f64(const double *xq, int64_t xq_len, int64_t n_query, int64_t n_features,
                          const double *x_train, int64_t xt_len, int64_t n_train, int32_t k,
                          int32_t metric, double p, double *out_dist, uint32_t *out_idx,
                          int64_t out_len, void *stream);
/* Largest k served for (dtype_bytes, n_features, metric): INT32_MAX, i.e.
 * every k up to n_train (the arguments are kept for ABI stability). */
int32_t mlrs_knn_max_k(int32_t dtype_bytes, int64_t n_features, int32_t metric);

/*
 * mlrs_knn_topk_f32 for callers that cannot allocate device memory (code
 * under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  No counterpart in the reference.  Same arguments, validation,
 * kernels and bits as mlrs_knn_topk_f32; the only difference is where the
 * kernels' scratch (the copied operands, norms, group minima, lists, exact
 * tiles) lives: in a static device array of MLRS_NOALLOC_SCRATCH_BYTES per
 * GPU, held until the process ends, instead of the library's cached
 * workspace.  The call makes no hipMalloc / hipFree / allocating library
 * call; its first call on a device looks the array's device address
 * (hipGetSymbolAddress) and the CU count up once: make that first call, which
 * may have n_query = 0, outside a graph capture.  After it, calls can be
 * captured into a HIP graph (every step is a kernel launch: no memset, no
 * copy, no event) and replayed with new data in the same buffers.  The
 * searches for d <= 256 and k <= 128 cut the index and the queries to fit the
 * array; what cannot be cut (the low-d kernel's lists, a row of the exact
 * tiles for every query) and exceeds it, and searches of more than 2^32
 * n_query * n_train * n_features whose d or k is past the low-d kernel's range
 * and for which 12 bytes per row, a list per query and index segment and
 * their queues would exceed it (about 100,000 queries at n_train = 1M, d =
 * 128, k = 32), return MLRS_ERR_UNSUPPORTED, operand "scratch" {rows = bytes
 * needed, len = MLRS_NOALLOC_SCRATCH_BYTES}, before any launch.  Every call on
 * a GPU shares that GPU's
 * array: calls that overlap on one GPU (two streams, no ordering between
 * them) RACE -- order them yourself.  Not ordered against the other entry
 * points' calls (they use other memory), and no timing events are recorded.
 */
#define MLRS_NOALLOC_SCRATCH_BYTES 134217728 /* 128 MiB */
int32_t mlrs_knn_topk_f32_noalloc(const float *xq, int64_t xq_len, int64_t n_query, int64_t n_features,
                                  const float *x_train, int64_t xt_len, int64_t n_train, int32_t k,
                                  int32_t metric, double p, float *out_dist, uint32_t *out_idx,
                                  int64_t out_len, void *stream);

/*
 * Nearest-centre assignment (the k-means assignment step, k = 1 search).
 *
 * Replaces: assign_min (crates/mlrs-backend/src/prims/kmeans.rs:635-750) --
 *   dist_direct_2d_c4 + argmin_dist_rows (crates/mlrs-kernels/src/kmeans.rs:
 *   206-310) -- without its n x n_centers staging matrix.
 * Writes labels[i] = argmin_c ||x_i - c||^2 (lowest index on a tie; a NaN
 *   distance to centre 0 wins with label 0, as argmin_dist_rows seeds from
 *   centre 0) and sqdist[i] = that SQUARED distance.
 * Errors (validate_geometry, prims/kmeans.rs:1416-1454, then assign_min):
 *   ShapeMismatch "x"        n*n_features != x_len
 *   ShapeMismatch "k"        n_centers < 1 or n_centers > n
 *   ShapeMismatch "n"/"d"/"k" a dimension > UINT32_MAX
 *   ShapeMismatch "centers"  n_centers*n_features != centers_len
 *   ShapeMismatch "labels"   labels_len != n or dist_len != n
 * The reference's extra guard n*n_centers <= UINT32_MAX existed only for its
 * staging matrix, which this kernel does not have; it is not enforced.
 */
int32_t mlrs_kmeans_assign_f32(const float *x, int64_t x_len, int64_t n, int64_t n_features,
                               const float *centers, int64_t centers_len, int64_t n_centers,
                               uint32_t *labels, int64_t labels_len, float *sqdist, int64_t dist_len,
                               void *stream);
int32_t mlrs_kmeans_assign_f64(const double *x, int64_t x_len, int64_t n, int64_t n_features,
                               const double *centers, int64_t centers_len, int64_t n_centers,
                               uint32_t *labels, int64_t labels_len, double *sqdist, int64_t dist_len,
                               void *stream);

/*
 * Full pairwise distance matrix out[i*rows_y + j].
 *
 * Replaces: distance_direct (crates/mlrs-backend/src/prims/distance.rs:428-551,
 *   kernel euclidean_sq_dist, crates/mlrs-kernels/src/distance.rs:411-440) for
 *   MLRS_METRIC_EUCLIDEAN -- SQUARED distance, with the boundary root of
 *   sqrt_elem (crates/mlrs-kernels/src/elementwise.rs:131-136) when
 *   do_sqrt != 0 -- and metric_distance's cosine_dist
 *   (crates/mlrs-kernels/src/distance.rs:257-310) for MLRS_METRIC_COSINE.
 *   MLRS_METRIC_MANHATTAN / _CHEBYSHEV / _MINKOWSKI are manhattan_dist,
 *   chebyshev_dist and minkowski_dist (distance.rs:67-227; Minkowski with pow
 *   per feature and the root pow(acc, 1/p) with 1/p formed in F); do_sqrt is
 *   ignored for them, p is read for Minkowski only.
 * Errors (validate_geometry, prims/distance.rs:260-302):
 *   ShapeMismatch "x" / "y", DimMismatch "cols", ShapeMismatch "out".
 */
int32_t mlrs_pairwise_distance_f32(const float *x, int64_t x_len, int64_t rows_x, int64_t cols,
                                   const float *y, int64_t y_len, int64_t rows_y, int64_t cols_y,
                                   int32_t metric, int32_t do_sqrt, double p, float *out, int64_t out_len,
                                   void *stream);
int32_t mlrs_pairwise_distance_f64(const double *x, int64_t x_len, int64_t rows_x, int64_t cols,
                                   const double *y, int64_t y_len, int64_t rows_y, int64_t cols_y,
                                   int32_t metric, int32_t do_sqrt, double p, double *out, int64_t out_len,
                                   void *stream);

/*
 * Per-row squared L2 norms, out[r] = sum_c x[r,c]^2 accumulated in column
 * order with separate multiply and add.
 *
 * Replaces: row_sqnorms (crates/mlrs-backend/src/prims/kmeans.rs:805-832,
 *   kernel row_sqnorm, crates/mlrs-kernels/src/kmeans.rs:610) and the
 *   row_sumsq norm feeder (crates/mlrs-kernels/src/knn.rs:2130-2149).
 * Errors: ShapeMismatch "x" (n*n_features != x_len), ShapeMismatch "out".
 */
int32_t mlrs_row_sqnorms_f32(const float *x, int64_t x_len, int64_t n, int64_t n_features, float *out,
                             int64_t out_len, void *stream);
int32_t mlrs_row_sqnorms_f64(const double *x, int64_t x_len, int64_t n, int64_t n_features,
                             double *out, int64_t out_len, void *stream);

/*
 * kNN regressor prediction from a neighbour set (device-resident predict).
 *
 * Replaces: knn_regress_mean_gather (crates/mlrs-backend/src/prims/knn.rs:59-
 *   150, kernel knn_regress_mean, crates/mlrs-kernels/src/knn.rs:95-147) for
 *   weighted == 0 and n_outputs == 1, and knn_regress_gather_weighted
 *   (prims/knn.rs:151-323, kernel knn_regress_gather, knn.rs:197-316)
 *   otherwise.
 * Layout: y_train is n_train x n_outputs row-major; idx / dist are the
 *   n_query x k neighbour indices and TRUE distances of a search (dist is read
 *   only when weighted != 0 and may be NULL otherwise); out is n_query x
 *   n_outputs.  out = sum_j w_j y[idx_j] / sum_j w_j with w = 1 (uniform) or
 *   1/d (weighted; a row with a zero distance weighs its zero-distance
 *   neighbours 1 and the rest 0), both sums Neumaier-compensated.
 * Errors, before any launch: ShapeMismatch "k" (k < 1, n_query < 1,
 *   n_outputs < 1 or n_train < 1), "idx", "dist", "y_train", "n_query" /
 *   "n_train" / "n_outputs" (> UINT32_MAX), "out".  After the gather (the call
 *   synchronizes on `stream` to check): ShapeMismatch "knn.train_idx"
 *   {rows = first query row holding an index >= n_train, cols = k,
 *   len = n_train}; such an index contributes nothing.
 */
int32_t mlrs_knn_regress_f32(const float *y_train, int64_t y_len, int64_t n_train, int64_t n_outputs,
                             const uint32_t *idx, int64_t idx_len, const float *dist, int64_t dist_len,
                             int64_t n_query, int32_t k, int32_t weighted, float *out, int64_t out_len,
                             void *stream);
int32_t mlrs_knn_regress_f64(const double *y_train, int64_t y_len, int64_t n_train, int64_t n_outputs,
                             const uint32_t *idx, int64_t idx_len, const double *dist, int64_t dist_len,
                             int64_t n_query, int32_t k, int32_t weighted, double *out, int64_t out_len,
                             void *stream);

/*
 * kNN classifier vote from a neighbour set (device-resident predict).
 *
 * Replaces: KNeighborsClassifier::predict_proba_host / predict_labels_host
 *   (crates/mlrs-algos/src/neighbors/classifier.rs:782-930), the host f64
 *   vote after the search.
 * y_class holds each training row's DENSE class index (0..n_classes-1).
 *   proba (n_query x n_classes) = per-class sums of the f64 weights (1, or 1/d
 *   with the zero-distance indicator rule), divided by the row total (an
 *   all-zero row is left at zero), cast to F; labels (n_query) = the argmax
 *   over the F probabilities, lowest class index on a tie.
 * Errors, before any launch: ShapeMismatch "k", "idx", "dist", "n_classes",
 *   "proba", "labels".  After the vote (synchronizes on `stream`): the first
 *   bad neighbour in row-major order gives ShapeMismatch "knn.train_idx"
 *   {rows = the index, cols = 1, len = n_train} or "knn.class_id" {rows =
 *   max(class, 0), cols = 1, len = n_classes}.
 */
int32_t mlrs_knn_classify_f32(const int32_t *y_class, int64_t n_train, int32_t n_classes, const uint32_t *idx,
                              int64_t idx_len, const float *dist, int64_t dist_len, int64_t n_query, int32_t k,
                              int32_t weighted, float *proba, int64_t proba_len, int32_t *labels,
                              int64_t labels_len, void *stream);
int32_t mlrs_knn_classify_f64(const int32_t *y_class, int64_t n_train, int32_t n_classes, const uint32_t *idx,
                              int64_t idx_len, const double *dist, int64_t dist_len, int64_t n_query, int32_t k,
                              int32_t weighted, double *proba, int64_t proba_len, int32_t *labels,
                              int64_t labels_len, void *stream);

/*
 * Every training row within `radius` of each query row.
 *
 * Replaces: radius_neighbor_indices_metric (crates/mlrs-algos/src/neighbors/
 *   nearest.rs:609-749) with its default arm, radius_host_scan
 *   (crates/mlrs-backend/src/prims/radius_host.rs:140-234); the result is the
 *   RadiusNeighbors layout (nearest.rs:564-582): counts[q] (n_query, device)
 *   is row q's match count, and out_dist / out_idx (device) hold the matches
 *   of row 0, then row 1, ..., each row's in ascending training index -- a CSR
 *   matrix without its indptr.  Values are the host scan's: the knn_host lane
 *   arithmetic compared as `v <= th` against th = (F)(radius^2 | radius^p |
 *   radius) formed in f64 (NaN never matches), then sqrt (Euclidean),
 *   pow(v, (F)(1/p)) (Minkowski) or identity on the matches; indices are the
 *   training row numbers as int32.
 * Sizes: *total (host) receives the number of matches.  With out_dist and
 *   out_idx both NULL the call only counts (counts and *total filled).  With
 *   buffers of `capacity` entries and *total > capacity nothing is written to
 *   them and the call returns ShapeMismatch "out" {rows = total, cols = 1,
 *   len = capacity}.  The usual sequence is a counting call, then a call with
 *   buffers of the returned size and otherwise the same arguments, which
 *   starts from the first call's counts (the second call re-checks them and
 *   counts again if the data changed in between).  A call that brings
 *   buffers without a counting call before it (a caller that knows a bound
 *   on the total, e.g. from an earlier search) is served by one pass when
 *   the f32 matrix-core path keeps every strip's matches (at most 1,024 per
 *   strip and row): they are counted, kept and copied into place in the
 *   same call.  Buffers too small: as above, and the counts are kept for
 *   the next call.
 * Errors, before any launch: InvalidParam "radius" (radius not >= 0, NaN
 *   included; the text of AlgoError::InvalidEps), ShapeMismatch "xq" (n_query
 *   or n_features zero, or a length mismatch), DimMismatch "n_features",
 *   ShapeMismatch "y" / "rows" (n_train above u32::MAX) / "counts",
 *   Unsupported "metric" / "p" (Minkowski p < 1).
 * Synchronous: returns after `stream` has finished the call's work.
 */
int32_t mlrs_radius_neighbors_f32(const float *xq, int64_t xq_len, int64_t n_query, int64_t n_features,
                                  const float *x_train, int64_t x_train_len, int64_t n_train,
                                  int64_t train_features, int32_t metric, double p, double radius, uint32_t *counts,
                                  int64_t counts_len, float *out_dist, int32_t *out_idx, int64_t capacity,
                                  int64_t *total, void *stream);
int32_t mlrs_radius_neighbors_f64(const double *xq, int64_t xq_len, int64_t n_query, int64_t n_features,
                                  const double *x_train, int64_t x_train_len, int64_t n_train,
                                  int64_t train_features, int32_t metric, double p, double radius, uint32_t *counts,
                                  int64_t counts_len, double *out_dist, int32_t *out_idx, int64_t capacity,
                                  int64_t *total, void *stream);

/*
 * Directed k-nearest-neighbour graph of a row set against itself.
 *
 * Replaces: knn_graph (crates/mlrs-backend/src/prims/knn_graph.rs:180-311) as
 *   the cpu backend serves its callers, through host_knn (crates/mlrs-algos/src/
 *   manifold/umap_host_knn.rs:212-515, UMAP, include_self = 0) and the
 *   self-inclusive graph HDBSCAN reads (include_self = 1).  The arithmetic is
 *   that host scan's, in f64 (f32 rows are widened first): Euclidean
 *   sqrt(sum diff*diff), cosine 0.5*|x^ - y^|^2 over L2-normalised rows,
 *   Manhattan, Chebyshev (NaN never replaces the running max), Minkowski
 *   pow(sum pow(|diff|, p), 1/p).  out_idx / out_dist (n x k, device): per row
 *   ascending (distance, index); include_self = 0 leaves out the row's own
 *   index (by identity, not by distance: a duplicate point stays); an entry
 *   the scan cannot fill is (0, 0.0).  As in the host scan's KNearest
 *   (umap_host_knn.rs:171-198, pushing the final distance at :494), the lists
 *   are ranked by the final distance, not by the aggregate before the root:
 *   two aggregates that root to the same double are ordered by index.
 * Errors (knn_graph.rs:475-539): ShapeMismatch "x" {n, d, len} (or a
 *   dimension above u32::MAX), "k" {1, k, max_k} with max_k = n - 1 (n with
 *   include_self), "p" {1, 0, 1} (Minkowski p < 1), "out"; Unsupported
 *   "metric".  Every k up to max_k is served.
 */
int32_t mlrs_knn_graph_f32(const float *x, int64_t x_len, int64_t n, int64_t n_features, int64_t k, int32_t metric,
                           double p, int32_t include_self, uint32_t *out_idx, double *out_dist, int64_t out_len,
                           void *stream);
int32_t mlrs_knn_graph_f64(const double *x, int64_t x_len, int64_t n, int64_t n_features, int64_t k,
                           int32_t metric, double p, int32_t include_self, uint32_t *out_idx, double *out_dist,
                           int64_t out_len, void *stream);

/*
 * HDBSCAN core distances: out[i] (n, device, f64) = the (k-1)-th smallest
 *   distance from row i to every row, itself included, k = clamp(min_samples,
 *   1, n); +inf when fewer than k distances are finite.
 * Replaces: the core-distance step of feature_metric_single_linkage
 *   (crates/mlrs-algos/src/cluster/hdbscan.rs:1495-1566), served on the cpu
 *   backend by core_distances_host (cluster/hdbscan/host_core.rs:253-540); same
 *   f64 arithmetic as mlrs_knn_graph_*.  Cosine is not served (the reference
 *   takes cosine core distances from a dense matrix): Unsupported "metric".
 */
int32_t mlrs_hdbscan_core_distances_f32(const float *x, int64_t x_len, int64_t n, int64_t n_features,
                                        int32_t metric, double p, int64_t min_samples, double *out, int64_t out_len,
                                        void *stream);
int32_t mlrs_hdbscan_core_distances_f64(const double *x, int64_t x_len, int64_t n, int64_t n_features,
                                        int32_t metric, double p, int64_t min_samples, double *out, int64_t out_len,
                                        void *stream);

/*
 * k-means fit: restarts, initialisation and the Lloyd loop around the fused
 * nearest-centre assignment.
 *
 * Replaces: KMeans::fit (crates/mlrs-algos/src/cluster/kmeans.rs:1353-1580)
 *   with single_run (:929-1155) and the prims it drives (crates/mlrs-backend/
 *   src/prims/kmeans.rs): feature_mean_var (tol scaled by the mean feature
 *   variance), kmeanspp_sample / random_sample on SplitMix64 seeded
 *   seed + restart, assign_min, centroid_sums_dev (F sums over the reference's
 *   row blocks, block partials summed in order, widened to f64),
 *   relocate_empty_clusters, the f64 mean update, the strict label-equality
 *   break then the tol break, inertia_rows + sum_device, and the restart rule
 *   (strictly lower inertia on a partition that is not a relabelling).
 * algorithm: MLRS_KMEANS_LLOYD runs the fused k = 1 assignment over every row
 *   each iteration (assign_min); MLRS_KMEANS_ELKAN the bound-pruned one
 *   (elkan_init_bounds / elkan_assign_device / elkan_relax_bounds,
 *   prims/kmeans.rs:1523-1717), without the reference's n x k lower bounds:
 *   per row an upper bound on its centre distance, the sorted k x k half
 *   centre distances, and the fused search for the rows those cannot settle.
 *   Both return the same fit, bit for bit (labels, centres, inertia, n_iter),
 *   as the reference pins for its two arms; 'elkan' serves k <= 4096 with
 *   finite rows and runs Lloyd otherwise.
 * init_kind: 0 explicit centres (init, device, k x n_features; one run), 1
 *   k-means++, 2 random.  out_centers (k x n_features, device, F),
 *   out_labels (n, device), *out_inertia and *out_n_iter (host) of the
 *   winning restart.  Synchronous.
 * Errors: InvalidParam "k" (AlgoError::InvalidK text), "n_init", "max_iter",
 *   "tol", "algorithm"; ShapeMismatch "x", "init", "centers", "labels", and "labels"
 *   {n, k, empty clusters} when an empty cluster finds no donor row;
 *   Unsupported "init".
 */
#define MLRS_KMEANS_LLOYD 0
#define MLRS_KMEANS_ELKAN 1
int32_t mlrs_kmeans_fit_f32(const float *x, int64_t x_len, int64_t n, int64_t n_features, int64_t n_clusters,
                            int32_t init_kind, const float *init, int64_t init_len, uint64_t seed, int64_t n_init,
                            int64_t max_iter, double tol, int32_t algorithm, float *out_centers, int64_t centers_len,
                            uint32_t *out_labels, int64_t labels_len, double *out_inertia, int64_t *out_n_iter,
                            void *stream);
int32_t mlrs_kmeans_fit_f64(const double *x, int64_t x_len, int64_t n, int64_t n_features, int64_t n_clusters,
                            int32_t init_kind, const double *init, int64_t init_len, uint64_t seed, int64_t n_init,
                            int64_t max_iter, double tol, int32_t algorithm, double *out_centers,
                            int64_t centers_len,
                            uint32_t *out_labels, int64_t labels_len, double *out_inertia, int64_t *out_n_iter,
                            void *stream);

/*
 * Fit-time ownership copy: dst[0..len) = src[0..len) on `stream` (device
 * pointers, any alignment; 16-byte vectors when both are 16-byte aligned).
 * Replaces: device_copy (crates/mlrs-backend/src/prims/knn.rs:358-386) with
 *   its copy_elem / copy_elem_cpu_chunked kernels (crates/mlrs-kernels/src/
 *   elementwise.rs:71-125), which NearestNeighbors' Rust Fit::fit runs to own
 *   the training matrix.  The reference's u32 element ceiling (a CubeCL launch
 *   limit) does not apply.
 * Errors: ShapeMismatch "src" (len < 0), "dst" {len, 1, dst_len} when
 *   dst_len != len; NullPointer when len > 0 and a pointer is NULL.
 */
int32_t mlrs_device_copy_f32(const float *src, int64_t len, float *dst, int64_t dst_len, void *stream);
int32_t mlrs_device_copy_f64(const double *src, int64_t len, double *dst, int64_t dst_len, void *stream);

/*
 * Buffer counters of the current device: PoolStats (crates/mlrs-backend/src/
 * pool.rs:27-56) over the library's cached device buffers (the main and
 * auxiliary workspaces and the radius plan memory).  allocations: buffers
 * grown with hipMalloc; reuses: requests the held buffer already covered;
 * live_bytes: capacity currently held; peak_bytes: its high-water mark;
 * read_backs: device-to-host copies the library made (radius totals and
 * flags, the consumers' error checks, the k-means fit's per-iteration state)
 * -- the search, assignment, pairwise, norm and graph paths make none, so a
 * memory gate can assert read_backs does not move across them.
 * mlrs_pool_stats_reset zeroes allocations, reuses and read_backs and sets
 * peak_bytes to live_bytes.  The allocation-free entry point's static
 * scratch is not a cached buffer and is not counted.
 */
typedef struct mlrs_pool_stats {
    uint64_t allocations;
    uint64_t reuses;
    uint64_t peak_bytes;
    uint64_t live_bytes;
    uint64_t read_backs;
} mlrs_pool_stats;
int32_t mlrs_pool_stats_get(mlrs_pool_stats *out);
int32_t mlrs_pool_stats_reset(void);

/*
 * ---- training an embedding ----
 * What a table of embeddings is trained with before it is searched: a layer
 * forwards and backwards, the softmax cross entropy of many classes with its
 * gradient, and the optimizer step.  No counterpart in the reference.
 *
 * Element types: _f32 (float), _f16 (IEEE half) and _bf16 (bfloat16; 16-bit
 * elements are passed as uint16_t).  Products, sums and softmax statistics are
 * held in f32 whatever the type, norms in f64; a result is rounded to its type
 * once, to nearest even.  Matrices are contiguous and row-major, aligned to
 * their element size; other alignments than 16 bytes (or rows that are no
 * multiple of 16 bytes) cost a copy of the operand into the workspace.
 * Results do not depend on the stream or on other calls, and the same call
 * gives the same bits.  Row, column and class counts are limited to 2^31 - 513
 * and a row to 2^22 bytes (MLRS_ERR_UNSUPPORTED "features").  What a call
 * writes overlaps neither its operands nor its other outputs (InvalidParam with
 * the output's name, after the other checks), but where it says so.
 */
#define MLRS_ACT_NONE 0
#define MLRS_ACT_RELU 1
#define MLRS_ACT_GELU 2      /* z (1 + erf(z / sqrt 2)) / 2 */
#define MLRS_ACT_GELU_TANH 3 /* z (1 + tanh(sqrt(2/pi) (z + 0.044715 z^3))) / 2 */
#define MLRS_ACT_SILU 4      /* z / (1 + e^-z) */

/*
 * z = x w^T + bias; y = act(z) + residual.  x is n x d_in, w d_out x d_in,
 * bias d_out (may be NULL), residual n x d_out (may be NULL), y n x d_out;
 * preact (n x d_out, may be NULL) receives z.  y may be the residual's buffer.
 * Errors, in this order:
 *   ShapeMismatch "x" / "w"       n*d_in != x_len, d_out*d_in != w_len
 *   ShapeMismatch "features"      d_in < 1 or d_out < 1
 *   MLRS_ERR_UNSUPPORTED "features" / "rows"  sizes past the limits above
 *   ShapeMismatch "bias" / "residual" / "out" / "preact"
 *   MLRS_ERR_UNSUPPORTED "activation"
 */
int32_t mlrs_linear_f32(const float *x, int64_t x_len, int64_t n, int64_t d_in, const float *w, int64_t w_len,
                        int64_t d_out, const float *bias, int64_t bias_len, const float *residual,
                        int64_t residual_len, int32_t activation, float *y, int64_t y_len, float *preact,
                        int64_t preact_len, void *stream);
int32_t mlrs_linear_f16(const uint16_t *x, int64_t x_len, int64_t n, int64_t d_in, const uint16_t *w, int64_t w_len,
                        int64_t d_out, const uint16_t *bias, int64_t bias_len, const uint16_t *residual,
                        int64_t residual_len, int32_t activation, uint16_t *y, int64_t y_len, uint16_t *preact,
                        int64_t preact_len, void *stream);
int32_t mlrs_linear_bf16(const uint16_t *x, int64_t x_len, int64_t n, int64_t d_in, const uint16_t *w, int64_t w_len,
                         int64_t d_out, const uint16_t *bias, int64_t bias_len, const uint16_t *residual,
                         int64_t residual_len, int32_t activation, uint16_t *y, int64_t y_len, uint16_t *preact,
                         int64_t preact_len, void *stream);

/*
 * The gradient of mlrs_linear: dz = dy * act'(preact); dx = dz w (n x d_in),
 * dw = dz^T x (d_out x d_in), dbias = the column sums of dz (d_out); the
 * residual's gradient is dy.  Any of dx, dw and dbias may be NULL (length 0).
 * preact is what mlrs_linear kept, NULL (length 0) with MLRS_ACT_NONE.  16-bit
 * types: dz is rounded to the type before the two products (dbias sums it
 * unrounded).  n = 0 gives dw = 0 and dbias = 0.
 * Errors, in this order: as mlrs_linear ("x", "w", "features", "rows"), then
 *   ShapeMismatch "dy" / "dx" / "dw" / "dbias", MLRS_ERR_UNSUPPORTED
 *   "activation", ShapeMismatch "preact".
 */
int32_t mlrs_linear_grad_f32(const float *dy, int64_t dy_len, const float *x, int64_t x_len, int64_t n, int64_t d_in,
                             const float *w, int64_t w_len, int64_t d_out, const float *preact, int64_t preact_len,
                             int32_t activation, float *dx, int64_t dx_len, float *dw, int64_t dw_len, float *dbias,
                             int64_t dbias_len, void *stream);
int32_t mlrs_linear_grad_f16(const uint16_t *dy, int64_t dy_len, const uint16_t *x, int64_t x_len, int64_t n,
                             int64_t d_in, const uint16_t *w, int64_t w_len, int64_t d_out, const uint16_t *preact,
                             int64_t preact_len, int32_t activation, uint16_t *dx, int64_t dx_len, uint16_t *dw,
                             int64_t dw_len, uint16_t *dbias, int64_t dbias_len, void *stream);
int32_t mlrs_linear_grad_bf16(const uint16_t *dy, int64_t dy_len, const uint16_t *x, int64_t x_len, int64_t n,
                              int64_t d_in, const uint16_t *w, int64_t w_len, int64_t d_out, const uint16_t *preact,
                              int64_t preact_len, int32_t activation, uint16_t *dx, int64_t dx_len, uint16_t *dw,
                              int64_t dw_len, uint16_t *dbias, int64_t dbias_len, void *stream);

/*
 * Softmax cross entropy of z = h w^T + bias: lse_i = log sum_v e^(z_iv) and
 * loss_i = lse_i - z_i,target(i), without z in memory (but for a few tiles of
 * long rows, whose z is computed in parts in the workspace).  h is n x d, w
 * classes x d, bias `classes` long (may be NULL; -inf leaves a class out);
 * target, loss and lse hold n elements.  A row whose target is `ignore_index`
 * has loss 0 (its lse is still written); a target that is no class, loss NaN.
 * A row all of whose logits are -inf has lse -inf, and loss NaN; one with a
 * logit of +inf or NaN has NaN for both (a loss of 0 where it is ignored).
 * Errors, in this order: ShapeMismatch "h" / "w", "features" (d or classes
 *   < 1), MLRS_ERR_UNSUPPORTED "features" / "rows", ShapeMismatch "bias" /
 *   "target" / "out".
 */
int32_t mlrs_softmax_xent_f32(const float *h, int64_t h_len, int64_t n, int64_t d, const float *w, int64_t w_len,
                              int64_t classes, const float *bias, int64_t bias_len, const int64_t *target,
                              int64_t target_len, int64_t ignore_index, float *loss, float *lse, int64_t out_len,
                              void *stream);
int32_t mlrs_softmax_xent_f16(const uint16_t *h, int64_t h_len, int64_t n, int64_t d, const uint16_t *w,
                              int64_t w_len, int64_t classes, const uint16_t *bias, int64_t bias_len,
                              const int64_t *target, int64_t target_len, int64_t ignore_index, float *loss, float *lse,
                              int64_t out_len, void *stream);
int32_t mlrs_softmax_xent_bf16(const uint16_t *h, int64_t h_len, int64_t n, int64_t d, const uint16_t *w,
                               int64_t w_len, int64_t classes, const uint16_t *bias, int64_t bias_len,
                               const int64_t *target, int64_t target_len, int64_t ignore_index, float *loss,
                               float *lse, int64_t out_len, void *stream);

/*
 * The gradient of sum_i grad_i loss_i: with dz_iv = grad_i (e^(z_iv - lse_i) -
 * [v = target(i)]), zero in ignored rows, dh = dz w (n x d), dw = dz^T h
 * (classes x d) and dbias = the column sums of dz.  lse is mlrs_softmax_xent's
 * of the same operands; z is computed again, in pieces of the vocabulary (256
 * classes at least) whose dz takes at most MLRS_XENT_PIECE_BYTES of workspace;
 * of several pieces, dh is added up in f32.  f32's large products take dz in six
 * bytes an element more each, up to four times MLRS_XENT_PIECE_BYTES with it.  Any
 * of dh, dw and dbias may be NULL (length 0).
 * 16-bit types: dz is rounded to the type before the products, and dbias adds up
 * what is rounded.  It is scaled for that, and the results back: divided by the
 * fraction (1 to 2) of grad_0 in bf16, of the largest |grad_i| of a row that is not
 * ignored in f16, where a power of two also lifts that to 2^13.  So how an
 * element of one row is rounded depends on another row's grad.
 * n = 0 gives dw = 0 and dbias = 0.
 * Errors, in this order: as mlrs_softmax_xent ("out" being lse's and grad's
 *   length), then ShapeMismatch "dh" / "dw" / "dbias".
 */
#define MLRS_XENT_PIECE_BYTES 1073741824 /* 1 GiB */
int32_t mlrs_softmax_xent_grad_f32(const float *h, int64_t h_len, int64_t n, int64_t d, const float *w, int64_t w_len,
                                   int64_t classes, const float *bias, int64_t bias_len, const int64_t *target,
                                   int64_t target_len, int64_t ignore_index, const float *lse, const float *grad,
                                   int64_t out_len, float *dh, int64_t dh_len, float *dw, int64_t dw_len,
                                   float *dbias, int64_t dbias_len, void *stream);
int32_t mlrs_softmax_xent_grad_f16(const uint16_t *h, int64_t h_len, int64_t n, int64_t d, const uint16_t *w,
                                   int64_t w_len, int64_t classes, const uint16_t *bias, int64_t bias_len,
                                   const int64_t *target, int64_t target_len, int64_t ignore_index, const float *lse,
                                   const float *grad, int64_t out_len, uint16_t *dh, int64_t dh_len, uint16_t *dw,
                                   int64_t dw_len, uint16_t *dbias, int64_t dbias_len, void *stream);
int32_t mlrs_softmax_xent_grad_bf16(const uint16_t *h, int64_t h_len, int64_t n, int64_t d, const uint16_t *w,
                                    int64_t w_len, int64_t classes, const uint16_t *bias, int64_t bias_len,
                                    const int64_t *target, int64_t target_len, int64_t ignore_index, const float *lse,
                                    const float *grad, int64_t out_len, uint16_t *dh, int64_t dh_len, uint16_t *dw,
                                    int64_t dw_len, uint16_t *dbias, int64_t dbias_len, void *stream);

/*
 * ---- the rest of an encoder's layer ----
 * Dropout, group norm with an activation and dropout, and the layer in 8-bit
 * floating point.  Element types, overlaps and errors as above.  No call here
 * synchronizes or reads back.  A call that takes no workspace can be captured into
 * a graph and replayed; one that does is refused there (MLRS_ERR_UNSUPPORTED
 * "stream").
 *
 * Random bits come from a counter: element i of the tensor takes 16 bits of
 * Philox 4x32 with seven rounds (Salmon et al., SC 2011), key `seed`, counter
 * (i / 8, offset): the low half of word (i % 8) / 2 where i is even, else the
 * high one.  It is kept where they are at least t = round(65536 p) (65535 at
 * most), and then multiplied by 65536 / (65536 - t); else it is 0, whatever it
 * held.  So the mask is not stored: the backward pass takes the same seed and
 * offset.  `step` may be NULL, or an int64_t on the device that is added to
 * `offset` when the call runs (a replayed graph then draws other bits each time).
 */

/*
 * y = drop(x) + residual; all hold x_len elements, residual may be NULL.  y may
 * be x's or the residual's buffer.  The gradient of x is drop(dy), of the
 * residual dy.
 * Errors, in this order: ShapeMismatch "x" / "residual" / "out", InvalidParam
 *   "p" (not in [0, 1)).
 */
int32_t mlrs_dropout_f32(const float *x, int64_t x_len, double p, uint64_t seed, uint64_t offset, const int64_t *step,
                         const float *residual, int64_t residual_len, float *y, int64_t y_len, void *stream);
int32_t mlrs_dropout_f16(const uint16_t *x, int64_t x_len, double p, uint64_t seed, uint64_t offset,
                         const int64_t *step, const uint16_t *residual, int64_t residual_len, uint16_t *y,
                         int64_t y_len, void *stream);
int32_t mlrs_dropout_bf16(const uint16_t *x, int64_t x_len, double p, uint64_t seed, uint64_t offset,
                          const int64_t *step, const uint16_t *residual, int64_t residual_len, uint16_t *y,
                          int64_t y_len, void *stream);

/*
 * Group norm, channels last: x is n x positions x channels, in `groups` groups of
 * adjacent channels (8192 at most).  With mean and variance (over all of them, not
 * one less) of a sample's group over its positions, and rstd = 1 / sqrt(var + eps):
 *   z = (x - mean) rstd weight + bias,  y = drop(act(z)).
 * Sums are f32: a group with an infinity or a NaN has rstd NaN and so all of its y;
 * squares past f32's range give rstd 0.
 * weight and bias hold `channels` elements and may be NULL (1 and 0).  mean and
 * rstd (n x groups, f32) may both be NULL; the gradient takes them.
 * Errors, in this order: ShapeMismatch "x" / "features" (positions or channels
 *   < 1) / "groups" (< 1, or channels no multiple), MLRS_ERR_UNSUPPORTED "groups"
 *   / "features" (channels > 2^22, positions > 2^31, n > 2^40), ShapeMismatch
 *   "weight" / "bias" / "out" / "stats", MLRS_ERR_UNSUPPORTED "activation",
 *   InvalidParam "eps" / "p".
 */
int32_t mlrs_group_norm_f32(const float *x, int64_t x_len, int64_t n, int64_t positions, int64_t channels,
                            int64_t groups, const float *weight, int64_t weight_len, const float *bias,
                            int64_t bias_len, double eps, int32_t activation, double p, uint64_t seed,
                            uint64_t offset, const int64_t *step, float *y, int64_t y_len, float *mean, float *rstd,
                            int64_t stats_len, void *stream);
int32_t mlrs_group_norm_f16(const uint16_t *x, int64_t x_len, int64_t n, int64_t positions, int64_t channels,
                            int64_t groups, const uint16_t *weight, int64_t weight_len, const uint16_t *bias,
                            int64_t bias_len, double eps, int32_t activation, double p, uint64_t seed,
                            uint64_t offset, const int64_t *step, uint16_t *y, int64_t y_len, float *mean,
                            float *rstd, int64_t stats_len, void *stream);
int32_t mlrs_group_norm_bf16(const uint16_t *x, int64_t x_len, int64_t n, int64_t positions, int64_t channels,
                             int64_t groups, const uint16_t *weight, int64_t weight_len, const uint16_t *bias,
                             int64_t bias_len, double eps, int32_t activation, double p, uint64_t seed,
                             uint64_t offset, const int64_t *step, uint16_t *y, int64_t y_len, float *mean,
                             float *rstd, int64_t stats_len, void *stream);

/*
 * Its gradient: with dz = drop(dy) act'(z) and t = dz weight, dbias = the sums of
 * dz over samples and positions, dweight those of dz (x - mean) rstd, and dx =
 * rstd (t - (mean of t) - (x - mean) rstd (mean of t (x - mean) rstd)), the means
 * over the sample's group.  z is computed again.  Any of dx, dweight and dbias may
 * be NULL (length 0); n = 0 gives dweight = 0 and dbias = 0.
 * Errors, in this order: as mlrs_group_norm to "bias", ShapeMismatch "dy" /
 *   "stats" / "dx" / "dweight" / "dbias", MLRS_ERR_UNSUPPORTED "activation",
 *   InvalidParam "p".
 */
int32_t mlrs_group_norm_grad_f32(const float *dy, int64_t dy_len, const float *x, int64_t x_len, int64_t n,
                                 int64_t positions, int64_t channels, int64_t groups, const float *weight,
                                 int64_t weight_len, const float *bias, int64_t bias_len, const float *mean,
                                 const float *rstd, int64_t stats_len, int32_t activation, double p, uint64_t seed,
                                 uint64_t offset, const int64_t *step, float *dx, int64_t dx_len, float *dweight,
                                 int64_t dweight_len, float *dbias, int64_t dbias_len, void *stream);
int32_t mlrs_group_norm_grad_f16(const uint16_t *dy, int64_t dy_len, const uint16_t *x, int64_t x_len, int64_t n,
                                 int64_t positions, int64_t channels, int64_t groups, const uint16_t *weight,
                                 int64_t weight_len, const uint16_t *bias, int64_t bias_len, const float *mean,
                                 const float *rstd, int64_t stats_len, int32_t activation, double p, uint64_t seed,
                                 uint64_t offset, const int64_t *step, uint16_t *dx, int64_t dx_len,
                                 uint16_t *dweight, int64_t dweight_len, uint16_t *dbias, int64_t dbias_len,
                                 void *stream);
int32_t mlrs_group_norm_grad_bf16(const uint16_t *dy, int64_t dy_len, const uint16_t *x, int64_t x_len, int64_t n,
                                  int64_t positions, int64_t channels, int64_t groups, const uint16_t *weight,
                                  int64_t weight_len, const uint16_t *bias, int64_t bias_len, const float *mean,
                                  const float *rstd, int64_t stats_len, int32_t activation, double p, uint64_t seed,
                                  uint64_t offset, const int64_t *step, uint16_t *dx, int64_t dx_len,
                                  uint16_t *dweight, int64_t dweight_len, uint16_t *dbias, int64_t dbias_len,
                                  void *stream);

/*
 * ---- a layer in 8-bit floating point ----
 * Values are held as e4m3 codes (OCP: largest 448, no infinities, a NaN) with a
 * power of two for every block of 128 elements of a contraction axis, the least
 * with which no finite magnitude of the block passes 448 (1 for a block of zeros);
 * a code is the value over its scale, rounded to nearest even, so that a value is
 * rounded once.  Infinities and NaN have code NaN and no part in the scale.
 * Weights: one scale for each 128 x 128.  codes: d_out x C bytes, C = d_in rounded
 * up to 128, zeros behind a row; scales: a byte (the exponent + 127) for each tile,
 * ceil(d_out / 128) rows of S bytes, S = ceil(d_in / 128) rounded up to 4, 127
 * behind a row.  codes_t / scales_t: the same of the transpose (d_in rows), which
 * the gradient takes.  Codes are aligned to 16 bytes, scales to 4.
 */

/*
 * The codes of weights w (d_out x d_in); codes_t and scales_t may both be NULL
 * (lengths 0).
 * Errors, in this order: ShapeMismatch "w" / "features", MLRS_ERR_UNSUPPORTED
 *   "features" (> 2^22), ShapeMismatch and then InvalidParam (alignment) "codes" /
 *   "scales", "codes_t" / "scales_t".
 */
int32_t mlrs_fp8_weight_f32(const float *w, int64_t w_len, int64_t d_out, int64_t d_in, uint8_t *codes,
                            int64_t codes_len, uint8_t *scales, int64_t scales_len, uint8_t *codes_t,
                            int64_t codes_t_len, uint8_t *scales_t, int64_t scales_t_len, void *stream);
int32_t mlrs_fp8_weight_f16(const uint16_t *w, int64_t w_len, int64_t d_out, int64_t d_in, uint8_t *codes,
                            int64_t codes_len, uint8_t *scales, int64_t scales_len, uint8_t *codes_t,
                            int64_t codes_t_len, uint8_t *scales_t, int64_t scales_t_len, void *stream);
int32_t mlrs_fp8_weight_bf16(const uint16_t *w, int64_t w_len, int64_t d_out, int64_t d_in, uint8_t *codes,
                             int64_t codes_len, uint8_t *scales, int64_t scales_len, uint8_t *codes_t,
                             int64_t codes_t_len, uint8_t *scales_t, int64_t scales_t_len, void *stream);

/*
 * mlrs_linear with such weights: z = x' w'^T + bias, y = act(z) + residual, where x'
 * is what 8 bits hold of x, a scale for each 128 of a row, and w' what the codes
 * stand for.  Products are exact.  f16, bf16: the matrix instruction adds eight
 * adjacent products after cutting off what lies below 2^-13 of the largest one's
 * power of two, all else in f32.  f32: added up in f32, the values of more than 16
 * rows in bf16's range.  Up to 16 rows take no workspace.
 * Errors, in this order: ShapeMismatch "x" / "features", MLRS_ERR_UNSUPPORTED
 *   "features" / "rows", "codes" and "scales" as above, then as mlrs_linear from
 *   "bias" on.
 */
int32_t mlrs_linear_fp8_f32(const float *x, int64_t x_len, int64_t n, int64_t d_in, const uint8_t *codes,
                            int64_t codes_len, const uint8_t *scales, int64_t scales_len, int64_t d_out,
                            const float *bias, int64_t bias_len, const float *residual, int64_t residual_len,
                            int32_t activation, float *y, int64_t y_len, float *preact, int64_t preact_len,
                            void *stream);
int32_t mlrs_linear_fp8_f16(const uint16_t *x, int64_t x_len, int64_t n, int64_t d_in, const uint8_t *codes,
                            int64_t codes_len, const uint8_t *scales, int64_t scales_len, int64_t d_out,
                            const uint16_t *bias, int64_t bias_len, const uint16_t *residual, int64_t residual_len,
                            int32_t activation, uint16_t *y, int64_t y_len, uint16_t *preact, int64_t preact_len,
                            void *stream);
int32_t mlrs_linear_fp8_bf16(const uint16_t *x, int64_t x_len, int64_t n, int64_t d_in, const uint8_t *codes,
                             int64_t codes_len, const uint8_t *scales, int64_t scales_len, int64_t d_out,
                             const uint16_t *bias, int64_t bias_len, const uint16_t *residual, int64_t residual_len,
                             int32_t activation, uint16_t *y, int64_t y_len, uint16_t *preact, int64_t preact_len,
                             void *stream);

/*
 * Its gradient, of the values in 8 bits as if they were x and w: dz = dy
 * act'(preact), dx = dz' w' with a scale for each 128 of a row of dz, dw = dz''^T
 * x'' with one for each 128 rows of a column of dz and of x; dbias = the column sums
 * of dz itself.  Any of dx, dw and dbias may be NULL (length 0); codes_t and scales_t
 * may be where dx is.  n is limited to 2^22; n = 0 gives dw = 0 and dbias = 0.
 * Errors, in this order: as mlrs_linear_fp8 to "scales" ("codes_t" / "scales_t"
 *   where they are given), ShapeMismatch "dy" / "dx" / "dw" / "dbias",
 *   MLRS_ERR_UNSUPPORTED "activation", ShapeMismatch "preact", MLRS_ERR_UNSUPPORTED
 *   "rows".
 */
int32_t mlrs_linear_fp8_grad_f32(const float *dy, int64_t dy_len, const float *x, int64_t x_len, int64_t n,
                                 int64_t d_in, const uint8_t *codes_t, int64_t codes_t_len, const uint8_t *scales_t,
                                 int64_t scales_t_len, int64_t d_out, const float *preact, int64_t preact_len,
                                 int32_t activation, float *dx, int64_t dx_len, float *dw, int64_t dw_len,
                                 float *dbias, int64_t dbias_len, void *stream);
int32_t mlrs_linear_fp8_grad_f16(const uint16_t *dy, int64_t dy_len, const uint16_t *x, int64_t x_len, int64_t n,
                                 int64_t d_in, const uint8_t *codes_t, int64_t codes_t_len, const uint8_t *scales_t,
                                 int64_t scales_t_len, int64_t d_out, const uint16_t *preact, int64_t preact_len,
                                 int32_t activation, uint16_t *dx, int64_t dx_len, uint16_t *dw, int64_t dw_len,
                                 uint16_t *dbias, int64_t dbias_len, void *stream);
int32_t mlrs_linear_fp8_grad_bf16(const uint16_t *dy, int64_t dy_len, const uint16_t *x, int64_t x_len, int64_t n,
                                  int64_t d_in, const uint8_t *codes_t, int64_t codes_t_len, const uint8_t *scales_t,
                                  int64_t scales_t_len, int64_t d_out, const uint16_t *preact, int64_t preact_len,
                                  int32_t activation, uint16_t *dx, int64_t dx_len, uint16_t *dw, int64_t dw_len,
                                  uint16_t *dbias, int64_t dbias_len, void *stream);

#define MLRS_DTYPE_F32 0
#define MLRS_DTYPE_F16 1
#define MLRS_DTYPE_BF16 2

typedef struct mlrs_grad_tensor {
    const void *grad;
    int64_t len;
    int32_t dtype; /* MLRS_DTYPE_* */
} mlrs_grad_tensor;

/*
 * norm = the root of the sum of squares of every element of `count` gradients;
 * scale = min(1, max_norm / norm), the factor that clips them, NaN where the
 * norm is not finite.  Both are single floats on the device, so the step that
 * takes the factor needs no read-back.  `tensors` is host memory, read before
 * the call returns.
 * Errors: MLRS_ERR_NULL_POINTER, ShapeMismatch "tensors" (count < 0 or a
 *   negative length), MLRS_ERR_UNSUPPORTED "dtype", InvalidParam "max_norm"
 *   (not > 0).
 */
int32_t mlrs_grad_clip_scale(const mlrs_grad_tensor *tensors, int64_t count, double max_norm, float *norm,
                             float *scale, void *stream);

typedef struct mlrs_adamw_tensor {
    void *param;          /* f32, or f16 / bf16 with a master */
    const void *grad;     /* f32, f16 or bf16 */
    void *exp_avg;        /* 32 bits: f32; 8 bits: codes */
    void *exp_avg_sq;     /* 32 bits: f32; 8 bits: codes of the root */
    float *master;        /* f32 value of the parameter; NULL for f32 parameters */
    float *avg_scale;     /* 8 bits: a scale per MLRS_STATE_BLOCK elements; else NULL */
    float *avg_sq_scale;  /* likewise */
    int64_t len;
    double weight_decay;
    int32_t param_dtype, grad_dtype; /* MLRS_DTYPE_* */
} mlrs_adamw_tensor;
#define MLRS_STATE_BLOCK 256

/*
 * One AdamW step of `count` tensors in place, `step` counting from 1:
 *   g = grad * scale;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;
 *   p = p (1 - lr weight_decay) - lr / (1 - b1^step) * m / (sqrt(v / (1 - b2^step)) + eps)
 * `scale` is a float on the device (mlrs_grad_clip_scale's, the inverse of a
 * loss scale; NULL = 1); where it is not finite nothing is changed.
 * state_bits 32: m and v are f32.  state_bits 8: a block of MLRS_STATE_BLOCK
 * elements of a tensor has one scale each for m and for sqrt(v), which are kept
 * as a sign, four bits of exponent and three of fraction (m) and four and four
 * (the root), rounded up or down at random by `seed`, the tensor's place and
 * the element's index: give every step another seed.  All codes and scales 0 is
 * the state before the first step.  `tensors` is host memory, read before the
 * call returns; no tensor may appear twice.
 * Errors: MLRS_ERR_NULL_POINTER ("master" for a 16-bit parameter without one),
 *   ShapeMismatch "tensors", MLRS_ERR_UNSUPPORTED "dtype" / "state_bits" /
 *   "tensors" (one of more than 2^36 - 4096 elements), InvalidParam "lr" /
 *   "betas" / "eps" / "weight_decay" / "step".
 */
int32_t mlrs_adamw_step(const mlrs_adamw_tensor *tensors, int64_t count, int32_t state_bits, double lr, double beta1,
                        double beta2, double eps, int64_t step, const float *scale, uint32_t seed, void *stream);

/*
 * The values that an 8-bit state stands for: `which` 0 = exp_avg, 1 = the root
 * of exp_avg_sq.  scales_len = the blocks of `len` elements.
 * Errors: ShapeMismatch "codes" / "scales" / "out", MLRS_ERR_UNSUPPORTED
 *   "which", MLRS_ERR_NULL_POINTER.
 */
int32_t mlrs_adamw_state_values(const uint8_t *codes, int64_t len, const float *scales, int64_t scales_len,
                                int32_t which, float *out, int64_t out_len, void *stream);

/* Release the cached device workspace of the current device. */
int32_t mlrs_release_workspace(void);

/*
 * Measurement hook (no counterpart in the reference; for benchmarks).
 * While enabled, every call records a pair of HIP events on its own stream
 * around the launch of its dominant kernel (the group-minimum scan or tiles,
 * the resident or Gram kernel, the low-d ALU kernel, or the generic path's
 * distance tile; k-means fit also times
 * its centroid-sum pass).  mlrs_timing_read waits for the recorded events,
 * picks the name with the largest summed time, and returns that sum, the
 * number of launches timed under the name and the name; enabling again
 * clears the records.
 */
int32_t mlrs_timing_enable(int32_t on);
int32_t mlrs_timing_read(double *total_ms, int64_t *launches, char *kernel_name, int32_t name_len);

/*
 * Peak probe (no counterpart in the reference; the basis of the roofline
 * fractions the benchmark reports).  Runs register-only chains on every CU
 * with `waves_per_simd` waves on each SIMD (1..8) and returns the achieved
 * TFLOP/s (an FMA counts two flops) of the second of two launches, timed with
 * HIP events on `stream`:
 *   kind 0: v_fma_f32 (eight independent chains per lane, no packed math)
 *   kind 1: v_fma_f64 (likewise)
 *   kind 2: v_mfma_f32_32x32x2f32 (two independent accumulator chains)
 *   kind 3: v_mfma_f64_16x16x4f64 (four independent accumulator chains)
 * Synchronous.  Errors: Unsupported "kind" / "waves_per_simd".
 */
int32_t mlrs_probe_peak(int32_t kind, int32_t waves_per_simd, double *tflops, void *stream);

/*
 * Kernel-family override (no counterpart in the reference; for tests and
 * benchmarks).  Every family returns the same bits, so this only changes
 * speed: 0 = automatic choice (default); 1 = the matrix-core kernels wherever
 * they serve the shape (Euclidean and cosine searches with d <= 256 and k <=
 * 128: the group-minimum search, the resident one for k = 1; k-means: d <= 256);
 * 2 = the low-d ALU kernel wherever it serves the shape (f32 and f64, Euclidean
 * and cosine, d <= 16, k <= 32); 3 = the generic exact-tile path.  A family that
 * does not serve
 * a shape falls back to the automatic choice.  radius_neighbors: 1 = the
 * matrix-core screen wherever it serves (f32 Euclidean / cosine, d <= 128),
 * 3 = the host-scan kernel.  Process-wide.
 */
#define MLRS_PATH_AUTO 0
#define MLRS_PATH_FUSED 1
#define MLRS_PATH_LOWD 2
#define MLRS_PATH_GENERIC 3
int32_t mlrs_force_path(int32_t path);

#ifdef __cplusplus
}
#endif

#endif /* MLRS_HIP_KNN_H */
