/*
 * mlxvs C ABI for the MI355X (gfx950) exact k-nearest-neighbour engine.
 *
 * The first three functions and both enums are the drop-in surface of the
 * reference's C API (include/mlxvs/mlxvs_c.h:24-45, 243-256 and
 * src/c_api.cpp:190-196 in mikepapadim/mlxvs 0.16.1): same names, argument
 * order, enum values, status codes and per-thread error string, so a caller
 * that binds the reference (Java FFM, ctypes, cgo) binds this library
 * unchanged.  Everything after the marked line is an extension with no
 * counterpart in the reference's C API; each says which reference function
 * it exposes.
 *
 * Conventions (as the reference):
 *  - every function returns MLXVS_OK (0) or an mlxvs_status error code, and
 *    mlxvs_last_error() then describes the failure for the calling thread
 *    ("" after a success);
 *  - host arrays are row-major and owned by the caller: inputs are copied in,
 *    outputs are written into the caller's buffers;
 *  - ids are int32 [nq, k], -1 where fewer than k rows exist; distances are
 *    float32 [nq, k], nearest first: squared L2 ascending (+inf when
 *    missing), inner product / cosine similarity descending (-inf when
 *    missing), Hamming distance ascending (+inf when missing).
 *
 * Device-pointer variants (suffix _device) take pointers to device memory
 * (hipMalloc'ed on the current HIP device) and a hipStream_t passed as
 * void* (NULL = the null stream).  They enqueue all work on that stream and
 * return without waiting for it: every step, including the exhaustive
 * search of the queries a merge flags, is decided on the device.  Calls on
 * one device plan their work one at a time (a per-device lock, held only
 * while a call enqueues), and a call's work is ordered after the previous
 * call's on that device, whatever the streams.
 */
#ifndef MLXVS_C_H
#define MLXVS_C_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MLXVS_C_API __attribute__((visibility("default")))

/** C API version, major * 10000 + minor (reference mlxvs_c.h:25). */
#define MLXVS_C_API_VERSION 100

/** Status codes (reference include/mlxvs/mlxvs_c.h:27-35). */
typedef enum {
  MLXVS_OK = 0,
  /** An argument was out of range (mlxvs_last_error says which). */
  MLXVS_ERROR_INVALID_ARGUMENT = 1,
  /** A file could not be read or written (unused by the k-NN functions). */
  MLXVS_ERROR_IO = 2,
  /** Anything else: no GPU, out of device memory, a HIP runtime error. */
  MLXVS_ERROR_INTERNAL = 3,
} mlxvs_status;

/** How two rows compare (reference include/mlxvs/mlxvs_c.h:37-45). */
typedef enum {
  /** Dot product, larger is closer. */
  MLXVS_INNER_PRODUCT = 0,
  /** Squared Euclidean distance, smaller is closer. */
  MLXVS_L2 = 1,
  /** Cosine similarity, larger is closer; rows are normalised on the fly. */
  MLXVS_COSINE = 2,
} mlxvs_metric;

/**
 * The calling thread's message for its last failed call, "" after a
 * success.  Replaces reference src/c_api.cpp:190-192.
 */
MLXVS_C_API const char* mlxvs_last_error(void);

/** Library version string, "0.16.1" (the reference version this library
 * replaces).  Replaces src/c_api.cpp:194-196. */
MLXVS_C_API const char* mlxvs_version(void);

/**
 * Exact k-nearest neighbours of nq queries among n base rows (float32,
 * row-major, d columns).  1 <= k <= 256 (checked only when n >= 1, as the
 * reference).  distances may be NULL.  Replaces reference
 * include/mlxvs/mlxvs_c.h:243-256 / src/c_api.cpp:468-489.
 */
MLXVS_C_API int mlxvs_brute_force_knn(
    const float* base,
    int64_t n,
    const float* queries,
    int64_t nq,
    int32_t d,
    int32_t k,
    mlxvs_metric metric,
    int32_t* ids,
    float* distances);

/* ---- extensions: no counterpart in the reference's C API ---------------- */

/**
 * Exact Hamming k-NN of bit-packed rows (uint8 [n, bytes], as
 * numpy.packbits) for bit-packed queries (uint8 [nq, bytes]); 1 <= k <= 256.
 * Distances are popcounts of the XOR, as float32, ascending, lowest id first
 * among equal distances.  Exposes reference mlxvs::hamming_knn
 * (include/mlxvs/mlxvs.h:775-784, src/ivf.cpp:1343-1403), which the
 * reference binds to Python only (python/bindings.cpp:681-709).
 */
MLXVS_C_API int mlxvs_hamming_knn(
    const uint8_t* rows,
    int64_t n,
    const uint8_t* queries,
    int64_t nq,
    int32_t bytes,
    int32_t k,
    int32_t* ids,
    float* distances);

/**
 * As mlxvs_brute_force_knn, for float16 rows (IEEE binary16 bit patterns,
 * uint16 [n, d]) multiplied on the fp16 MFMA units with float32
 * accumulation.  The reference upcasts float16 input to float32
 * (src/utils.h:28) and computes in float32; products of binary16 values are
 * exact in float32, so the two differ only in summation order.
 */
MLXVS_C_API int mlxvs_brute_force_knn_f16(
    const uint16_t* base,
    int64_t n,
    const uint16_t* queries,
    int64_t nq,
    int32_t d,
    int32_t k,
    mlxvs_metric metric,
    int32_t* ids,
    float* distances);

/**
 * The k-NN graph of rows against themselves with each row's own id dropped:
 * ids int32 [n, k] and distances float32 [n, k].  rows are float32
 * (f16 == 0) or binary16 bit patterns (f16 != 0).  1 <= k <= 255, n >= 2.
 * Exposes the single-cluster brute-force route of reference
 * mlxvs::all_neighbors (src/all_neighbors.cpp:250-263, 56-95, 265-272).
 */
MLXVS_C_API int mlxvs_knn_self_graph(
    const void* rows,
    int64_t n,
    int32_t d,
    int32_t f16,
    int32_t k,
    mlxvs_metric metric,
    int32_t* ids,
    float* distances);

/**
 * The m nearest centroids of every row: labels int32 [n, m], nearest first
 * (squared L2, lowest index among equal distances).  x [n, d] and
 * centroids [c, d] are float32 (f16 == 0) or binary16 (f16 != 0) host
 * arrays; 1 <= m <= min(c, 256).  Extension: exposes mlxvs::kmeans_predict
 * (reference include/mlxvs/mlxvs.h:89-99, src/kmeans.cpp:136-169), which the
 * reference binds to C++ and Python only.
 */
MLXVS_C_API int mlxvs_kmeans_predict(
    const void* x,
    int64_t n,
    const void* centroids,
    int64_t c,
    int32_t d,
    int32_t f16,
    int32_t m,
    int32_t* labels);

/**
 * IVF-Flat search (extension; exposes mlxvs::ivf_flat_search, reference
 * include/mlxvs/mlxvs.h:561-571 / src/ivf.cpp:327-416, which the reference
 * binds to C++ and Python only).  The index: centers [lists, d] float32,
 * data [n, d] float32 grouped by list (unit rows for MLXVS_COSINE), indices
 * [n] int32 (the id of each row), offsets [lists + 1] int32.  queries
 * [nq, d]; n_probes lists scanned per query (clamped to [1, lists]);
 * 1 <= k <= 256.  ids / distances [nq, k] as mlxvs_brute_force_knn, -1 /
 * +-inf where the scanned lists hold fewer than k rows.  Host arrays.
 */
MLXVS_C_API int mlxvs_ivf_flat_search(
    const float* centers,
    int64_t lists,
    const float* data,
    int64_t n,
    const int32_t* indices,
    const int32_t* offsets,
    int32_t d,
    mlxvs_metric metric,
    const float* queries,
    int64_t nq,
    int32_t k,
    int32_t n_probes,
    int32_t* ids,
    float* distances);

/** mlxvs_ivf_flat_search with every array in device memory, enqueued on
 * stream (a hipStream_t); returns without waiting.  The work is planned on
 * the device from the probes and the offsets, which are not read on the
 * host and so not checked: they must run from 0 to n without decreasing. */
MLXVS_C_API int mlxvs_ivf_flat_search_device(
    const float* centers,
    int64_t lists,
    const float* data,
    int64_t n,
    const int32_t* indices,
    const int32_t* offsets,
    int32_t d,
    mlxvs_metric metric,
    const float* queries,
    int64_t nq,
    int32_t k,
    int32_t n_probes,
    int32_t* ids,
    float* distances,
    void* stream);

/**
 * mlxvs_brute_force_knn on device memory: base [n, d] and queries [nq, d]
 * float32 (f16 == 0) or binary16 (f16 != 0), outputs ids / distances
 * [nq, k] in device memory (distances may be NULL).  Enqueued on stream;
 * returns without waiting.
 */
MLXVS_C_API int mlxvs_brute_force_knn_device(
    const void* base,
    int64_t n,
    const void* queries,
    int64_t nq,
    int32_t d,
    int32_t f16,
    int32_t k,
    mlxvs_metric metric,
    int32_t* ids,
    float* distances,
    void* stream);

/**
 * mlxvs_brute_force_knn_device without allocating: no counterpart in the
 * reference; for callers that cannot call hipMalloc (code under HIP graph
 * capture, serving loops, harnesses that forbid allocation).  Its
 * workspace (norms, per-lane lists, bounds, merge levels) is a fixed device
 * array of 64 MiB on each GPU the library runs on, held until the process
 * ends; the call itself allocates nothing.  Limits: a workspace of at most
 * 64 MiB (about 10,000 queries against 1,000,000 rows of 128 dims at
 * k = 10) and shapes the fused kernels take; anything else returns
 * MLXVS_ERROR_INVALID_ARGUMENT before any work is enqueued.  Enqueued on
 * stream, returns without waiting.  Calls that overlap on one GPU share the
 * array and race: order them (one stream, or events).
 */
MLXVS_C_API int mlxvs_brute_force_knn_device_noalloc(
    const void* base,
    int64_t n,
    const void* queries,
    int64_t nq,
    int32_t d,
    int32_t f16,
    int32_t k,
    mlxvs_metric metric,
    int32_t* ids,
    float* distances,
    void* stream);

/** mlxvs_hamming_knn on device memory (see mlxvs_brute_force_knn_device). */
MLXVS_C_API int mlxvs_hamming_knn_device(
    const uint8_t* rows,
    int64_t n,
    const uint8_t* queries,
    int64_t nq,
    int32_t bytes,
    int32_t k,
    int32_t* ids,
    float* distances,
    void* stream);

/** mlxvs_knn_self_graph on device memory (see mlxvs_brute_force_knn_device). */
MLXVS_C_API int mlxvs_knn_self_graph_device(
    const void* rows,
    int64_t n,
    int32_t d,
    int32_t f16,
    int32_t k,
    mlxvs_metric metric,
    int32_t* ids,
    float* distances,
    void* stream);

/**
 * One merge step of the exact k-NN: the best k of each row of scores
 * (float32 [nq, t], row-major; column c has id id_offset + c) together with
 * the running lists ids (int32 [nq, k]) and best (float32 [nq, k]) unless
 * first != 0 (then ids and best are not read and may be NULL).  Writes
 * out_ids / out_scores [nq, k] (out_scores may be NULL), best first: score
 * descending with -0 equal to +0, then id ascending; among entries of equal
 * key the lowest (unsigned) ids are kept; -1 / -inf past min(k, t + (first ?
 * 0 : k)) entries.  1 <= k <= 256.  Extension: exposes mlxvs::topk_merge
 * (reference include/mlxvs/mlxvs.h:892-905, src/knn.cpp:37-69), which the
 * reference binds to C++ only.  Host arrays.
 */
MLXVS_C_API int mlxvs_topk_merge(
    const float* scores,
    int64_t nq,
    int64_t t,
    const int32_t* ids,
    const float* best,
    int32_t id_offset,
    int32_t first,
    int32_t k,
    int32_t* out_ids,
    float* out_scores);

/**
 * mlxvs_topk_merge on device memory, enqueued on stream (a hipStream_t);
 * returns without waiting.  out_ids / out_scores may be ids / best
 * themselves (each row's running entries are read before it is written).
 * Uses no workspace.
 */
MLXVS_C_API int mlxvs_topk_merge_device(
    const float* scores,
    int64_t nq,
    int64_t t,
    const int32_t* ids,
    const float* best,
    int32_t id_offset,
    int32_t first,
    int32_t k,
    int32_t* out_ids,
    float* out_scores,
    void* stream);

/*
 * Host-array entries on a caller's stream.  The same as the entries without
 * the suffix, except that the copies in, the kernels and the copies out are
 * enqueued on stream (a hipStream_t; NULL: the null stream) and the call
 * waits for that stream, not the device, before it returns with the results
 * in the caller's buffers.  Extension: the reference's Python binding takes
 * a stream for brute_force_knn and kmeans_predict (python/bindings.cpp:55,
 * 125) and runs on it (src/utils.h:31-38 gpu_stream); hamming_knn takes one
 * in the C++ entry (include/mlxvs/mlxvs.h:775-784).  f16 != 0: binary16
 * rows, as mlxvs_brute_force_knn_f16.
 */
MLXVS_C_API int mlxvs_brute_force_knn_on_stream(
    const void* base,
    int64_t n,
    const void* queries,
    int64_t nq,
    int32_t d,
    int32_t f16,
    int32_t k,
    mlxvs_metric metric,
    int32_t* ids,
    float* distances,
    void* stream);

MLXVS_C_API int mlxvs_hamming_knn_on_stream(
    const uint8_t* rows,
    int64_t n,
    const uint8_t* queries,
    int64_t nq,
    int32_t bytes,
    int32_t k,
    int32_t* ids,
    float* distances,
    void* stream);

MLXVS_C_API int mlxvs_kmeans_predict_on_stream(
    const void* x,
    int64_t n,
    const void* centroids,
    int64_t c,
    int32_t d,
    int32_t f16,
    int32_t m,
    int32_t* labels,
    void* stream);

MLXVS_C_API int mlxvs_topk_merge_on_stream(
    const float* scores,
    int64_t nq,
    int64_t t,
    const int32_t* ids,
    const float* best,
    int32_t id_offset,
    int32_t first,
    int32_t k,
    int32_t* out_ids,
    float* out_scores,
    void* stream);

/** Prefilter kinds (cuVS's filters; reference
 * python/mlxvs/cuvs/neighbors/filters.py:39-50). */
enum {
  /** every row (the filter words are not read) */
  MLXVS_FILTER_NONE = 0,
  /** one bit per base row: bit i % 32 of word i / 32 set when row i may be
   * returned; ceil(n / 32) words */
  MLXVS_FILTER_BITSET = 1,
  /** one bit per (query, row), row-major over nq * n bits and not padded
   * per query: bit q n + i set when row i may be returned for query q;
   * ceil(nq n / 32) words */
  MLXVS_FILTER_BITMAP = 2
};

/**
 * Extension: exact k-NN over the rows a prefilter allows.  As
 * mlxvs_brute_force_knn_on_stream (host arrays, enqueued on stream, waits
 * for that stream), with filter_kind one of MLXVS_FILTER_* and filter its
 * host words: each query's k nearest allowed rows, ids numbering all rows,
 * -1 / +inf (L2) or -inf (similarities) past the allowed rows there are.
 * Rows the filter leaves out never enter the fused select's lists.  No C
 * counterpart in the reference, whose prefiltered search is the
 * Python-level cuvs.neighbors.brute_force.search (python/mlxvs/cuvs/
 * neighbors/brute_force.py:97-136: scores of excluded rows set to the
 * worst value before the selection, such picks returned as -1).
 */
MLXVS_C_API int mlxvs_brute_force_knn_filtered(
    const void* base,
    int64_t n,
    const void* queries,
    int64_t nq,
    int32_t d,
    int32_t f16,
    int32_t k,
    mlxvs_metric metric,
    const uint32_t* filter,
    int32_t filter_kind,
    int32_t* ids,
    float* distances,
    void* stream);

/**
 * mlxvs_brute_force_knn_filtered on device memory (inputs, filter words
 * and outputs); returns once the work is enqueued on stream.
 */
MLXVS_C_API int mlxvs_brute_force_knn_filtered_device(
    const void* base,
    int64_t n,
    const void* queries,
    int64_t nq,
    int32_t d,
    int32_t f16,
    int32_t k,
    mlxvs_metric metric,
    const uint32_t* filter,
    int32_t filter_kind,
    int32_t* ids,
    float* distances,
    void* stream);

/**
 * Extension: exact k-NN under one of cuVS's distances that the fused
 * kernels do not serve, for cuVS's brute_force.search: distance_type is
 * cuVS's DistanceType value -- 3 L1 (cityblock), 7 Linf (chebyshev), 8
 * Canberra, 9 Lp (minkowski, exponent metric_arg), 10 correlation, 12
 * Hellinger, 14 Bray-Curtis, 15 Jensen-Shannon, 16 Hamming (the share of
 * differing columns), 17 KL divergence, 18 Russell-Rao -- with the
 * reference's definitions (python/mlxvs/cuvs/distance.py:85-151, which
 * brute_force.search applies at python/mlxvs/cuvs/neighbors/brute_force.py:
 * 118-136).  float32 host rows; 1 <= k <= 256 (any n: -1 / +inf past the
 * rows a query may return); each query's k smallest distances, nearest
 * first, lower id first among equal ones; filter / filter_kind as
 * mlxvs_brute_force_knn_filtered.  No C counterpart in the reference, whose
 * search computes these distance matrices in Python.  Waits for its stream.
 */
MLXVS_C_API int mlxvs_pairwise_knn(
    const float* base,
    int64_t n,
    const float* queries,
    int64_t nq,
    int32_t d,
    int32_t k,
    int32_t distance_type,
    float metric_arg,
    const uint32_t* filter,
    int32_t filter_kind,
    int32_t* ids,
    float* distances,
    void* stream);

/* ---- the paged key-value cache (extensions) -------------------------------
 *
 * A cache of attention keys and values in pages of page_size tokens, and
 * retrieval over it: a step's block tables and slots from the requests'
 * lengths (mlxvs_kv_plan_device), the write of its tokens
 * (mlxvs_kv_append_device), the blocks that a cheap score selects for each of
 * them (mlxvs_kv_select_device) and their attention, over every block or the
 * selected ones (mlxvs_kv_attend_device).  Queries and keys get their positions
 * from mlxvs_kv_rotate_device; a budget is kept by the attention that each key got
 * (mlxvs_kv_weigh_device), the tokens that have most of it
 * (mlxvs_kv_keep_device), and a cut to those (mlxvs_kv_compact_device).  All
 * arrays are device memory; the calls enqueue their work on `stream`, allocate nothing, keep nothing and can
 * be captured into graphs.  Calls that depend on one another go to one stream
 * or are ordered by the caller; a workspace serves one call at a time.
 */

/** Element type of keys, values, queries and outputs. */
typedef enum {
  MLXVS_KV_F16 = 0,  /* IEEE binary16 */
  MLXVS_KV_BF16 = 1, /* bfloat16 */
} mlxvs_kv_type;

/**
 * A cache.  page_size: a power of two from 16 to 256; dim: a multiple of 8, at
 * most 256.  keys [pages][heads][page_size][dim]; values
 * [pages][heads][dim][page_size], transposed within a page; both 16-byte
 * aligned.  summaries int8 [pages][heads][dim] with scales float32
 * [pages][heads] describe complete pages for mlxvs_kv_select_device: code x
 * scale is the mean of a page's keys (null, both: the cache keeps none).
 */
typedef struct {
  void* keys;
  void* values;
  int8_t* summaries;
  float* scales;
  int64_t pages;
  int32_t heads;
  int32_t page_size;
  int32_t dim;
  mlxvs_kv_type type;
} mlxvs_kv_cache;

/**
 * Queries of `tokens` tokens and where they stand: q [tokens][q_heads][dim] of
 * the cache's type, strides in values (multiples of 8; the values of a head
 * are contiguous; 16-byte aligned), q_heads a multiple of the cache's heads
 * (query head i reads kv head i / (q_heads / heads)).  table int32
 * [requests][columns], rows table_stride apart: the page of each block of a
 * request.  token_request[t] and positions[t] int32: token t belongs to that
 * request and sees its keys 0 .. position, itself among them; a token with
 * position -1 (or a request out of range) sees nothing.  A page id outside
 * [0, pages) stands for a block that is absent.
 */
typedef struct {
  const void* q;
  int64_t token_stride;
  int64_t head_stride;
  int64_t tokens;
  int32_t q_heads;
  int32_t columns;
  const int32_t* table;
  int64_t table_stride;
  int64_t requests;
  const int32_t* token_request;
  const int32_t* positions;
} mlxvs_kv_queries;

/**
 * A step's block tables and slot maps.  Request r holds past[r] tokens and gets
 * fresh[r] more (0: none).  Its table row has the pages of the tokens it holds;
 * the pages that the new ones need are taken from free_pages (page ids, used
 * from entry cursor[0] on) in the requests' order and written into the row.  A
 * request whose blocks exceed `columns` or whose pages the free list does not
 * reach is not admitted, nor is any later one that needs pages in the second
 * case: it takes none.  Written, all int32 but slots:
 *   slots int64 [tokens], token_request [tokens], positions [tokens]: the new
 *     tokens in the requests' order: page x page_size + offset, the request,
 *     the position; slot and position -1 for a request that was not admitted,
 *     all three -1 past the last token (tokens: the batch's size; tokens past
 *     it get no entry);
 *   starts [requests + 1]: each request's first token in the batch;
 *   lengths [requests]: tokens held after the step;
 *   first [requests]: a request's first entry of free_pages, -1 if it was not
 *     admitted (0 if it needs none);
 *   cursor_out[0]: the first unused entry after the step.
 * What is written may not overlap what is read, the table apart.
 * columns x page_size must be below 2^31.
 */
MLXVS_C_API int mlxvs_kv_plan_device(
    const int32_t* past,
    const int32_t* fresh,
    int64_t requests,
    int32_t* table,
    int64_t table_stride,
    int32_t columns,
    const int32_t* free_pages,
    int64_t free_count,
    const int32_t* cursor,
    int32_t page_size,
    int64_t tokens,
    int64_t* slots,
    int32_t* token_request,
    int32_t* positions,
    int32_t* starts,
    int32_t* lengths,
    int32_t* first,
    int32_t* cursor_out,
    void* stream);

/**
 * Writes keys and values of tokens into their slots (page x page_size +
 * offset; outside the cache: skipped), k and v [tokens][heads][dim] with
 * token and head strides in values (multiples of 8, 16-byte aligned), and then
 * the summaries of the pages whose last slot is among them (over all their
 * slots), if the cache keeps summaries.
 */
MLXVS_C_API int mlxvs_kv_append_device(
    const mlxvs_kv_cache* cache,
    const void* k,
    int64_t k_token_stride,
    int64_t k_head_stride,
    const void* v,
    int64_t v_token_stride,
    int64_t v_head_stride,
    const int64_t* slots,
    int64_t tokens,
    void* stream);

/**
 * The n best blocks of each token and kv head: blocks int32
 * [tokens][heads][n], ascending, -1 after the last.  Candidates are the blocks
 * up to the token's own; its own and the last - 1 before it (last >= 1) and the
 * first `first` of the request are always taken (first + last <= n <= 256),
 * the others by score, the lowest block among equal ones.  A score is the int8
 * dot product of a block's summary with the codes of the query (the sum over
 * the group's heads), times the summary's scale: the same list from every
 * implementation.  workspace: mlxvs_kv_select_workspace bytes (may be 0).
 */
MLXVS_C_API int mlxvs_kv_select_device(
    const mlxvs_kv_cache* cache,
    const mlxvs_kv_queries* queries,
    int32_t n,
    int32_t first,
    int32_t last,
    int32_t* blocks,
    void* workspace,
    int64_t workspace_bytes,
    void* stream);

/** Bytes of workspace of a call with these arguments, -1 if they are invalid
 * (mlxvs_last_error says why). */
MLXVS_C_API int64_t mlxvs_kv_select_workspace(const mlxvs_kv_cache* cache,
                                              const mlxvs_kv_queries* queries, int32_t n);

/**
 * Attention of the tokens over the cache: out [tokens][q_heads][dim] (the
 * cache's type, contiguous) and, unless null, lse float32 [tokens][q_heads],
 * the logarithm of the sum of exponentials.  blocks null: over all of a
 * request's blocks; else int32 [tokens][heads][n] (n <= 256): over the listed
 * ones, an entry outside the table or past the token's own block showing
 * nothing (one listed twice counts twice).  Keys past the token's position
 * never count, whatever their places hold.  A token that sees nothing: zeros,
 * lse -inf.  scale > 0 multiplies the scores.  longest: tokens that the longest
 * request holds, as far as the caller knows (0: all that the table can hold);
 * it guides how work is split and never what is computed.  workspace:
 * mlxvs_kv_attend_workspace bytes (may be 0).
 */
MLXVS_C_API int mlxvs_kv_attend_device(
    const mlxvs_kv_cache* cache,
    const mlxvs_kv_queries* queries,
    const int32_t* blocks,
    int32_t n,
    float scale,
    int64_t longest,
    void* out,
    float* lse,
    void* workspace,
    int64_t workspace_bytes,
    void* stream);

/** Bytes of workspace of a call with these arguments (n 0: over all blocks), -1
 * if they are invalid. */
MLXVS_C_API int64_t mlxvs_kv_attend_workspace(const mlxvs_kv_cache* cache,
                                              const mlxvs_kv_queries* queries, int32_t n,
                                              int64_t longest);

/** Which values of a head are turned together: the first half of the rotated
 * ones with the second, or neighbours. */
typedef enum {
  MLXVS_KV_HALVES = 0, /* (x[i], x[i + rotated / 2]) */
  MLXVS_KV_PAIRS = 1,  /* (x[2 i], x[2 i + 1]) */
} mlxvs_kv_rotary_layout;

/** How the frequencies of positions are scaled for texts `factor` times as long as
 * those (of `context` tokens) that a model learnt on. */
typedef enum {
  MLXVS_KV_SCALING_NONE = 0,   /* f_i = base^(-2 i / rotated) */
  MLXVS_KV_SCALING_LINEAR = 1, /* f_i / factor */
  MLXVS_KV_SCALING_BASE = 2,   /* base x factor^(rotated / (rotated - 2)) for base */
  /* f_i where it makes 32 turns or more over the context, f_i / factor where it
   * makes one or less, between them a straight line in the turns; rotated values by
   * 0.1 ln(factor) + 1 (Peng et al. 2023, YaRN) */
  MLXVS_KV_SCALING_RAMP = 3,
} mlxvs_kv_rotary_scaling;

/**
 * Radians a position of each pair of rotated values, frequencies [rotated / 2], and
 * the factor of the rotated values, magnitude[0].  On the host, no GPU needed.
 */
MLXVS_C_API int mlxvs_kv_rotary_frequencies(int32_t rotated, double base,
                                            mlxvs_kv_rotary_scaling scaling, double factor,
                                            double context, double* frequencies,
                                            float* magnitude);

/** n radians a position as turns a position in 2^-64 of a turn (whole turns
 * left out), for mlxvs_kv_rotary.  On the host, no GPU needed. */
MLXVS_C_API int mlxvs_kv_rotary_turns(const double* frequencies, int32_t n, uint64_t* turns);

/**
 * Positions as rotations of heads of `dim` values (a multiple of 8, at most 256):
 * their first `rotated` ones (even, at most dim) are turned, the others pass.
 * turns [rotated / 2] in device memory, from mlxvs_kv_rotary_turns.
 */
typedef struct {
  const uint64_t* turns;
  int32_t dim;
  int32_t rotated;
  mlxvs_kv_rotary_layout layout;
  float magnitude;
  mlxvs_kv_type type; /* of the heads */
} mlxvs_kv_rotary;

/** Type of a norm's weights. */
typedef enum {
  MLXVS_KV_NORM_OWN = 0, /* the heads' own */
  MLXVS_KV_NORM_F32 = 1,
} mlxvs_kv_norm;

/**
 * Heads of tokens: x [tokens][heads][dim] and the place of their results, strides
 * in values (multiples of 8; 16-byte aligned).  `out` may be x, with its strides;
 * else the results may overlap nothing that the call reads.  norm [dim]: weights of
 * a norm before the rotation, x rsqrt(mean(x^2) + eps) norm over the whole head,
 * 16-byte aligned; null: none.  heads 0: nothing.
 */
typedef struct {
  const void* x;
  int64_t token_stride;
  int64_t head_stride;
  int32_t heads;
  const void* norm;
  mlxvs_kv_norm norm_type;
  void* out;
  int64_t out_token_stride;
  int64_t out_head_stride;
} mlxvs_kv_heads;

/**
 * Queries and keys (either may be null) normed and rotated by positions int32
 * [tokens].  With evicted int32 [requests], a token's position in its text is
 * positions[t] + evicted[token_request[t]]: what its request's cache has lost
 * (mlxvs_kv_compact_device) still counts (a request out of range: nothing).  A
 * token with a negative position is turned by nothing, as at position 0 (its norm and
 * the magnitude of its rotated values are as for any other).  Computed in float32 and
 * rounded once.  A position times the given turns is exact modulo a turn, at every
 * position; the angle is then rounded to 2^-26 of a turn.  (What a frequency was rounded
 * by as a double grows with the position: for one just below a radian it is 2^-25.6 of a
 * turn at position 2^31.)  out may be x with its strides; otherwise what is written may
 * overlap neither what is read nor the other results.
 */
MLXVS_C_API int mlxvs_kv_rotate_device(const mlxvs_kv_rotary* rotary, const mlxvs_kv_heads* q,
                                       const mlxvs_kv_heads* k, int64_t tokens,
                                       const int32_t* positions, const int32_t* token_request,
                                       const int32_t* evicted, int64_t requests, float eps,
                                       void* stream);

/**
 * The attention that each key gets from the step's tokens, added to what it got
 * before: mass float32 [requests][heads][slots], slots >= columns x page_size.  The
 * tokens of request r (a row of queries->table) are starts[r] .. starts[r + 1] - 1
 * (int32 [requests + 1]), their positions one after another, as
 * mlxvs_kv_plan_device makes them (a request's first one is read, no other);
 * queries->token_request is not read and may be null.  lse float32
 * [tokens][q_heads]: what mlxvs_kv_attend_device over every block returned for
 * the same queries and scale.  For the positions p up to the last token's
 *   mass[p] = (p < first ? decay x mass[p] : 0) + the sum over the tokens that see p
 *             and the head's query heads of exp(scale x q.k_p - lse),
 * first being the first token's position: the step's own keys start from zero.  The
 * others, and requests without tokens (or with position -1), stay as they are: the
 * keys of a step that is left out have what their places held before.  A key of an
 * absent page gets nothing, and one with values that are not finite may get NaN.
 * decay in [0, 1]; with 0 masses are not read.  A page that several rows share has a
 * mass in each.  longest guides how work is split, as in mlxvs_kv_attend_device.  The
 * same bits every time.  workspace: mlxvs_kv_weigh_workspace bytes (may be 0).
 */
MLXVS_C_API int mlxvs_kv_weigh_device(const mlxvs_kv_cache* cache,
                                      const mlxvs_kv_queries* queries, const int32_t* starts,
                                      const float* lse, float scale, float decay,
                                      int64_t longest, float* mass, int64_t slots,
                                      void* workspace, int64_t workspace_bytes, void* stream);

/** Bytes of workspace of a call with these arguments, -1 if they are invalid. */
MLXVS_C_API int64_t mlxvs_kv_weigh_workspace(const mlxvs_kv_cache* cache,
                                             const mlxvs_kv_queries* queries, int64_t longest);

/**
 * The tokens that a budget of n leaves: kept int32 [requests][heads][n], ascending.
 * Request r holds lengths[r] tokens (at most slots count).  Of more than `above`
 * (>= n) its first `first` and last `recent` (first + recent <= n) are kept, and of
 * the others those of the largest mass, the lowest among equal ones; NaN counts
 * as less than any other.  A request of at most `above` keeps all: its list is -1
 * throughout.  workspace: mlxvs_kv_keep_workspace bytes (may be 0).
 */
MLXVS_C_API int mlxvs_kv_keep_device(const float* mass, int64_t requests, int32_t heads,
                                     int64_t slots, const int32_t* lengths, int32_t n,
                                     int32_t first, int32_t recent, int32_t above, int32_t* kept,
                                     void* workspace, int64_t workspace_bytes, void* stream);

/** Bytes of workspace of a call with these sizes, -1 if they are invalid. */
MLXVS_C_API int64_t mlxvs_kv_keep_workspace(int64_t requests, int32_t heads, int64_t slots);

/**
 * Cuts requests to the tokens of their lists, kept int32 [requests][heads][n]
 * (mlxvs_kv_keep_device's, or others: n ascending positions below the request's
 * length for each head, the same requests in all heads).  Key, value and mass (mass
 * float32 [requests][heads][slots], or null) of position kept[j] move to position
 * j, in place; what lies past position n stays in its places.  Complete pages of
 * which a token changed get new summaries, if the cache keeps any.  The table stays
 * as it is: the request's pages past the new end, columns ceil(n / page_size) ..
 * ceil(length / page_size) - 1, are written into free_pages before entry cursor[0],
 * in the requests' order from there down, so that entries from cursor_out[0] on are
 * free (a column of an absent block gives its entry, whatever it is).  Not cut, and given back nothing: a request whose list starts with -1, one
 * of at most n tokens or of more than the table holds, and, from the first one on
 * whose pages find no room in free_pages, each that would give pages back.
 * lengths_out [requests], cursor_out [1]: the lengths and the cursor after it.  The
 * pages of a request that is cut have to be its own: in place of shared ones the
 * requests' tokens would be mixed up.  workspace: mlxvs_kv_compact_workspace bytes.
 */
MLXVS_C_API int mlxvs_kv_compact_device(const mlxvs_kv_cache* cache, const int32_t* table,
                                        int64_t table_stride, int32_t columns, int64_t requests,
                                        const int32_t* lengths, const int32_t* kept, int32_t n,
                                        int32_t* free_pages, int64_t free_count,
                                        const int32_t* cursor, float* mass, int64_t slots,
                                        int32_t* lengths_out, int32_t* cursor_out,
                                        void* workspace, int64_t workspace_bytes, void* stream);

/** Bytes of workspace of a call with these sizes, -1 if they are invalid. */
MLXVS_C_API int64_t mlxvs_kv_compact_workspace(const mlxvs_kv_cache* cache, int32_t columns,
                                               int64_t requests, int32_t n);

/**
 * Releases the workspace the library keeps on the current device between
 * calls (it is grown on demand and reused).  Safe to call at any time when
 * no other call is running on that device.
 */
MLXVS_C_API int mlxvs_release_workspace(void);

/**
 * Per-stage kernel timing: with enable != 0 every kernel launch of later
 * calls is bracketed by HIP events on its stream (stages: prep, fused_f32,
 * fused_f16, hamming, merge, scores, select, pack, fill, self_drop, kv_plan,
 * kv_append, kv_select, kv_attend, kv_rotate, kv_weigh, kv_keep, kv_compact).
 * Enabling or disabling clears the totals.
 */
MLXVS_C_API int mlxvs_profile(int enable);

/**
 * Writes "stage launches total_ms" lines for the launches since the last
 * report into buf (NUL-terminated, truncated to len), waiting for their
 * events, and clears the totals.
 */
MLXVS_C_API int mlxvs_profile_report(char* buf, int64_t len);

#ifdef __cplusplus
}
#endif

#endif /* MLXVS_C_H */
