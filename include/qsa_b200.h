/*
 * qsa_b200.h -- C ABI of the B200 (sm_100a) sparse paged GQA FP8 decode
 * attention library (libqsa_b200.so).
 *
 * The operation, for each Top-K row r, query head h and KV head g = h / G:
 *
 *   out[r,h,:] = softmax_t( q[r,h] . K[slot_t, g] * k_scale * softmax_scale )
 *                . V[slot_t, g] * v_scale  (*)  sigmoid(gate[r,h,:])
 *
 *   slot_t = btable[t2r[r], t / P] * P + t % P   for each selected token t
 *
 * with bf16 q / gate / out [rows, Hq, 128], FP8 E4M3FN K/V caches
 * [num_pages, P, Hkv, 128], int32 block table, Top-K indices and request map.
 *
 * All pointers are device pointers owned by the caller. Calls are
 * asynchronous on the given stream and never synchronise, trap or allocate.
 * Entry points return 0 or a negative QSA_B200_ERR_* status.
 *
 * Reference interfaces this library replaces (Ammar-Alnagar/QSA-FP8-SM89):
 *   - the C-ABI launcher  launch_qsa_cuda        sm89_cuda.cu:232-253
 *   - the Python entry    run(q, k, v, k_scale, v_scale, btable, t2r,
 *                          indices, gate)        sm89_cutedsl.py:311-351
 *   - the eager oracle    torch_eager(...)       sm89_torch.py:27-54
 *   - the Triton launch   launch(q, k, v, indices, btable, t2r, gate, out,
 *                          k_scale, v_scale)     sm89_triton.py:118-142
 *   - the cache producer  (randn * 0.1).to(float8_e4m3fn) into the paged
 *                          [num_pages, P, Hkv, 128] layout, with the scales
 *                          returned beside it    sm89_cutedsl.py:48-62, :79
 *                          (qsa_b200_cache_write: the same layout, written
 *                          at given token slots, saturating at +-448)
 */
#ifndef QSA_B200_H_
#define QSA_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define QSA_B200_API __attribute__((visibility("default")))
#else
#define QSA_B200_API
#endif

/* A CUDA stream handle (cudaStream_t / CUstream); NULL is the legacy stream. */
typedef struct CUstream_st* qsa_b200_stream_t;

#define QSA_B200_ABI_VERSION 1

enum {
  QSA_B200_OK = 0,
  QSA_B200_ERR_NULL_POINTER = -1, /* a required pointer is NULL */
  QSA_B200_ERR_BAD_SHAPE = -2,    /* a size is negative / inconsistent */
  QSA_B200_ERR_UNSUPPORTED = -3,  /* head_dim != 128, group > 32, or past a tensor-core kernel limit */
  QSA_B200_ERR_MISALIGNED = -4,   /* a tensor is not 16-byte aligned */
  QSA_B200_ERR_WORKSPACE = -5,    /* workspace missing or too small */
  QSA_B200_ERR_DEVICE = -6,       /* current device is not sm_100 */
  QSA_B200_ERR_LAUNCH = -7,       /* the CUDA launch itself failed */
  QSA_B200_ERR_KERNEL = -8,       /* a kernel reported a device-side failure */
  QSA_B200_ERR_TOO_LARGE = -9,    /* workspace above the fixed scratch of qsa_b200_decode_noalloc */
  QSA_B200_ERR_BAD_VALUE = -10    /* a scale is not a positive finite number */
};

/* Kernel selection. AUTO picks the tensor-core kernel for every group size
 * (Hq / Hkv) from 1 to 32; above 16 each KV head's query heads go in two
 * halves, each half reading the KV rows. The CUDA-core kernel (SIMT) takes
 * the same sizes. The tensor-core kernel (explicit or through AUTO)
 * returns QSA_B200_ERR_UNSUPPORTED for a cache of more than 2^31 - 1 rows of
 * 128 bytes (num_pages * page_size * num_kv_heads; 256 GiB per cache) and
 * for more than 2^30 - 1 work items (rows * num_kv_heads * ceil(topk / 512)). */
enum { QSA_B200_KERNEL_AUTO = 0, QSA_B200_KERNEL_TC = 1, QSA_B200_KERNEL_SIMT = 2 };

typedef struct qsa_b200_decode_args {
  const void* q;          /* bf16 [rows, num_q_heads, head_dim], contiguous */
  const void* k_cache;    /* fp8 e4m3fn [num_pages, page_size, num_kv_heads, head_dim] */
  const void* v_cache;    /* same layout as k_cache */
  const int32_t* indices; /* [rows, indices_stride]; first `topk` columns = logical tokens, <0 = masked */
  const int32_t* counts;  /* optional [rows]: only the first counts[r] columns may be valid */
  const int32_t* btable;  /* [num_reqs, btable_stride]; first pages_per_req columns = physical pages */
  const int32_t* t2r;     /* optional [rows]: Top-K row -> block-table row (NULL = identity) */
  const void* gate;       /* bf16 [rows, num_q_heads, head_dim], contiguous */
  void* out;              /* bf16 [rows, num_q_heads, head_dim], contiguous */
  float softmax_scale;    /* natural-log domain score scale, e.g. 1/sqrt(head_dim) */
  float k_scale;          /* K dequantisation scale (folded into the score scale) */
  float v_scale;          /* V dequantisation scale */
  int32_t rows;
  int32_t num_q_heads;
  int32_t num_kv_heads;
  int32_t head_dim;       /* must be 128 */
  int32_t page_size;
  int32_t pages_per_req;
  int32_t num_reqs;
  int64_t num_pages;
  int32_t topk;
  int64_t indices_stride; /* >= topk (+1 with count_column) */
  int32_t count_column;   /* nonzero: counts[r] = indices[r * indices_stride + topk] */
  int64_t btable_stride;  /* >= pages_per_req */
  int32_t kernel;         /* QSA_B200_KERNEL_* */
} qsa_b200_decode_args;

/* Bytes of device workspace qsa_b200_decode needs, each part 256-byte
 * aligned: the tensor-core kernel's row map (one int32 token slot per Top-K
 * entry: rows x chunks x 512 entries), its tile flags (16 bytes per row and
 * chunk) and its item claim counter (256 bytes), then, when a Top-K row spans
 * more than one chunk, the split partial outputs and log-sum-exps.
 * 0 only for the CUDA-core kernel without a split. Negative on invalid
 * arguments. */
QSA_B200_API int64_t qsa_b200_workspace_bytes(const qsa_b200_decode_args* args);

/* The decode. `workspace` (256-byte aligned) must hold
 * qsa_b200_workspace_bytes(args) bytes; it may be NULL when that is 0. The
 * workspace needs no clearing and may be reused by the next call on the same
 * stream.
 * Replaces launch_qsa_cuda (sm89_cuda.cu:232-301) / run (sm89_cutedsl.py:311). */
QSA_B200_API int qsa_b200_decode(const qsa_b200_decode_args* args, void* workspace, size_t workspace_bytes,
                    qsa_b200_stream_t stream);

/* The index decode alone: slots[r * topk + c] = physical token slot
 * (phys_page * page_size + t % page_size) of Top-K entry (r, c), or -1 when it
 * is masked -- the bit-exact part of the path (sm89_torch.py:30-39;
 * sm89_cuda.cu:110-115, :147-164). Only the index/table fields of `args` are
 * read; q, caches, gate and out may be NULL. */
QSA_B200_API int qsa_b200_slots(const qsa_b200_decode_args* args, int64_t* slots, qsa_b200_stream_t stream);

/* Drop-in for the reference's C-ABI launcher, same signature and argument
 * meaning (sm89_cuda.cu:232-253): indices are [nreqs, topk + 1] with the valid
 * count in the last column, softmax_scale is in the log2 domain
 * (k_scale * log2(e) / sqrt(head_dim)), rows == nreqs and t2r is required.
 * Returns void like the reference; the status of the call is available from
 * qsa_b200_last_status(). Rows with an out-of-range t2r entry or no valid
 * token are written as zeros (the reference leaves them unwritten). This
 * signature takes no workspace: the call runs as qsa_b200_decode_noalloc, on
 * the library's fixed per-device scratch (QSA_B200_ERR_TOO_LARGE beyond it),
 * so calls that overlap in time on one device race. */
QSA_B200_API void launch_qsa_cuda(const void* q, const void* k, const void* v, const void* indices, const void* btable,
                     const int32_t* t2r, const void* gate, void* out, float softmax_scale, float v_scale,
                     int32_t nblocks, int32_t nreqs, int32_t num_q_heads, int32_t num_kv_heads, int32_t topk,
                     int32_t page_sz, int32_t max_pages, int32_t head_dim, int32_t group_sz,
                     qsa_b200_stream_t stream);

/* Status of the calling thread's last launch_qsa_cuda. */
QSA_B200_API int qsa_b200_last_status(void);

/* Reads the device-side error word of the current device (nonzero when a
 * kernel gave up on a bounded wait); clears it when `clear` is nonzero.
 * Synchronous; returns a negative status if the read itself fails. */
QSA_B200_API int qsa_b200_device_error(int clear);

/* Human-readable text of a status code. */
QSA_B200_API const char* qsa_b200_status_string(int status);

/* QSA_B200_ABI_VERSION of the loaded library. */
QSA_B200_API int qsa_b200_abi_version(void);

/* Fixed workspace of qsa_b200_decode_noalloc, per device: 32 MiB, room for
 * the row map and split partials of, for example, 128 rows x 64 query heads x
 * 4 chunks of 512 Top-K entries (18 MiB). */
#define QSA_B200_NOALLOC_SCRATCH_BYTES (32u * 1024u * 1024u)

/* Allocation-free qsa_b200_decode. This entry point has NO counterpart in
 * the reference. It serves callers that cannot allocate device memory at
 * call time: a runtime with a fixed device budget, a latency-critical loop,
 * an FFI caller without an allocator.
 *   - The workspace (row map and split partials) is a file-scope device
 *     array of QSA_B200_NOALLOC_SCRATCH_BYTES per device; the call makes no
 *     cudaMalloc, cudaFree or other allocating call.
 *   - Returns QSA_B200_ERR_TOO_LARGE, before touching the device, when
 *     qsa_b200_workspace_bytes(args) exceeds that maximum; otherwise the
 *     statuses and results of qsa_b200_decode.
 *   - The first call on each device looks up the array's address
 *     (cudaGetSymbolAddress) with that device current: make that first call
 *     before any stream capture.
 *   - Calls that overlap in time on one device (other streams or threads)
 *     share the scratch and race; the caller serialises them. */
QSA_B200_API int qsa_b200_decode_noalloc(const qsa_b200_decode_args* args, qsa_b200_stream_t stream);

/* Element types of the new keys and values of qsa_b200_cache_write. */
enum { QSA_B200_DTYPE_BF16 = 0, QSA_B200_DTYPE_F16 = 1, QSA_B200_DTYPE_F32 = 2 };

typedef struct qsa_b200_cache_write_args {
  const void* k;         /* new keys [tokens, num_kv_heads, head_dim] of input_dtype */
  const void* v;         /* new values, same shape, type and strides as k */
  const int64_t* slots;  /* [tokens]: physical token slot phys_page * page_size + offset of each token;
                            a negative slot or one past the cache is skipped */
  void* k_cache;         /* fp8 e4m3fn [num_pages, page_size, num_kv_heads, head_dim] */
  void* v_cache;         /* same layout as k_cache */
  float k_scale;         /* dequantisation scales (cache value * scale = stored value) */
  float v_scale;
  int32_t tokens;
  int32_t num_kv_heads;
  int32_t head_dim;      /* must be 128 */
  int32_t page_size;
  int64_t num_pages;
  int64_t token_stride;  /* elements from one token of k / v to the next, >= num_kv_heads * head_dim */
  int32_t input_dtype;   /* QSA_B200_DTYPE_* */
} qsa_b200_cache_write_args;

/* Quantises new keys and values into the paged FP8 caches:
 *   cache[slot, g, d] = e4m3fn(x[t, g, d] * inv)   for slot = slots[t]
 * with inv = 1 / scale rounded to fp32 once, an fp32 product, and the
 * conversion rounding to the nearest E4M3FN value (ties to even), saturating
 * at +-448: a finite value
 * beyond the range and an infinity become +-448, NaN stays NaN (torch's cast
 * turns |x| >= 464 into NaN instead). Rows of skipped tokens are left as they
 * were. Two tokens with the same slot race (the caller gives each slot once).
 * Needs k, v 16-byte aligned with token_stride * element size a multiple of
 * 16, and 16-byte aligned caches. Asynchronous on `stream`. */
QSA_B200_API int qsa_b200_cache_write(const qsa_b200_cache_write_args* args, qsa_b200_stream_t stream);

typedef struct qsa_b200_topk_args {
  const float* scores;    /* [rows, ctx] fp32 per-position scores, row stride score_stride */
  const int32_t* lengths; /* optional [rows]: valid positions of each row (clamped to [0, ctx]); NULL = ctx */
  int32_t* out;           /* [rows, k] int32 Top-K indices, row stride out_stride */
  int32_t rows;
  int32_t ctx;            /* positions per row, 1 .. QSA_B200_TOPK_MAX_CTX */
  int32_t k;              /* selections per row, >= 1 */
  int64_t score_stride;   /* >= ctx */
  int64_t out_stride;     /* >= k */
} qsa_b200_topk_args;

#define QSA_B200_TOPK_MAX_CTX (1 << 20)

/* The Top-K index producer, the step before the decode: for each row, the
 * positions of the k highest scores, in ascending position order, as the
 * decode's [rows, k] int32 indices. A position t is a candidate when t is
 * below the row's length and its score is neither NaN nor -inf; at the k-th
 * score lower positions win; a row with fewer than k candidates is padded
 * with -1. No reference counterpart: the reference consumes Top-K indices but
 * does not produce them (sm89_cutedsl.py:72-76 builds sequential ones).
 * Needs 4-byte aligned scores, lengths and out. Asynchronous on `stream`. */
QSA_B200_API int qsa_b200_topk_select(const qsa_b200_topk_args* args, qsa_b200_stream_t stream);

/* ---- The block-scaled cache ----------------------------------------------
 * Paged E4M3FN caches [num_pages, P, Hkv, 128] with one fp32 scale for each
 * block of `block_size` consecutive tokens of a page and each KV head:
 *   stored value = code * scales[page, (t % P) / block_size, g],
 * scales fp32 [num_pages, P / block_size, Hkv] for K and for V. block_size
 * divides P; block_size 1 is a scale for every token, P one for every page. Up to
 * (2^31 - 1) / 128 heads of a kind.
 * Three entry points serve one attention layer over it: qsa_b200_qk_rope (the
 * queries), qsa_b200_block_append (new keys and values) and
 * qsa_b200_block_decode. None has a counterpart in the reference, whose
 * caches have one scale each (sm89_cutedsl.py:48-62, :79). */

/* Position rotation of a 128-element head. The first rotary_dim elements form
 * rotary_dim / 2 pairs: pair j is elements (j, j + rotary_dim / 2), or with
 * `interleaved` (2j, 2j + 1). Pair (a, b) becomes (a c - b s, b c + a s) with
 * c = table[p * rotary_dim + j], s = table[p * rotary_dim + rotary_dim / 2 + j].
 * p is the token's position on pair j's axis: the first sections[0] pairs go by
 * axis 0, the next sections[1] by axis 1, and so on. */
#define QSA_B200_ROPE_MAX_AXES 4
typedef struct qsa_b200_rotation {
  const float* table;       /* fp32 [table_len, rotary_dim]: cosines, then sines; NULL = no rotation */
  const int32_t* positions; /* [num_axes, tokens], rows axis_stride apart */
  int64_t axis_stride;      /* elements from one axis to the next, >= tokens with several axes */
  int32_t table_len;        /* a token with a position outside [0, table_len) gets a row of zeros */
  int32_t rotary_dim;       /* a multiple of 16 up to 128 */
  int32_t interleaved;
  int32_t num_axes;         /* 1 .. QSA_B200_ROPE_MAX_AXES */
  int32_t sections[QSA_B200_ROPE_MAX_AXES]; /* pairs of each axis, sum rotary_dim / 2 (not read with one axis) */
} qsa_b200_rotation;

typedef struct qsa_b200_qk_rope_args {
  const void* q;        /* [tokens, num_q_heads, head_dim] of dtype, heads contiguous */
  const void* k;        /* optional [tokens, num_kv_heads, head_dim] */
  void* q_out;          /* shaped like q; may be q itself */
  void* k_out;          /* shaped like k; may be k itself */
  const void* q_weight; /* optional [head_dim] of weight_dtype: RMS norm of each query head */
  const void* k_weight; /* optional [head_dim]: the same for each key head */
  float eps;            /* >= 0, added to the mean square */
  int32_t tokens;
  int32_t num_q_heads;
  int32_t num_kv_heads; /* 0 without k */
  int32_t head_dim;     /* must be 128 */
  int64_t q_stride;     /* elements from one token to the next */
  int64_t k_stride;
  int64_t q_out_stride;
  int64_t k_out_stride;
  int32_t dtype;        /* QSA_B200_DTYPE_* of q, k and the outputs */
  int32_t weight_dtype; /* QSA_B200_DTYPE_* of the weights */
  qsa_b200_rotation rope;
} qsa_b200_qk_rope_args;

/* RMS norm of every query and key head and the position rotation, in one pass:
 *   y = x * rsqrt(mean(x^2) + eps) * weight (where a weight is given), rotated,
 * in fp32 and rounded once to dtype. The outputs may be the inputs (same
 * pointer and stride); they must not overlap otherwise. Needs 16-byte aligned
 * tensors with token strides a multiple of 16 bytes, and a 16-byte aligned
 * table. Asynchronous on `stream`. */
QSA_B200_API int qsa_b200_qk_rope(const qsa_b200_qk_rope_args* args, qsa_b200_stream_t stream);

typedef struct qsa_b200_block_append_args {
  const void* k;            /* new keys [tokens, num_kv_heads, head_dim] of input_dtype, heads contiguous */
  const void* v;            /* new values, same shape, type and strides as k */
  void* k_cache;            /* fp8 e4m3fn [num_pages, page_size, num_kv_heads, head_dim] */
  void* v_cache;
  float* k_scales;          /* fp32 [num_pages, page_size / block_size, num_kv_heads] */
  float* v_scales;
  const int32_t* btable;    /* [num_reqs, btable_stride]; first pages_per_req columns = physical pages */
  const int32_t* reqs;      /* optional [entries]: block-table row of each entry (NULL = identity) */
  const int32_t* starts;    /* [entries]: logical position of the entry's first new token */
  const int32_t* cu_tokens; /* optional [entries + 1]: entry e has the tokens cu_tokens[e] .. cu_tokens[e + 1] - 1;
                               NULL: one token each (tokens == entries) */
  const void* k_weight;     /* optional [head_dim] of weight_dtype: RMS norm of each key head */
  float eps;
  int32_t entries;
  int32_t tokens;
  int32_t num_kv_heads;
  int32_t head_dim;         /* must be 128 */
  int32_t page_size;
  int32_t block_size;       /* divides page_size */
  int32_t pages_per_req;
  int32_t num_reqs;
  int64_t num_pages;
  int64_t btable_stride;
  int64_t token_stride;     /* elements from one token of k / v to the next */
  int32_t input_dtype;      /* QSA_B200_DTYPE_* */
  int32_t weight_dtype;
  qsa_b200_rotation rope;   /* of the keys; positions NULL = the tokens' logical positions (one axis) */
} qsa_b200_block_append_args;

/* Appends new keys (normed and rotated on the way, in fp32) and values to the
 * block-scaled caches. Entry e's tokens go to the logical positions starts[e],
 * starts[e] + 1, ... of its request. For each block and head that gets a token:
 *   s = max(s_old, max |x| / 448, 2^-126) over the block's new rows x, with
 *       s_old the block's scale where it keeps tokens before starts[e], else 0;
 *   each new row is stored as e4m3fn(x / s), each kept row as
 *   e4m3fn(code * (s_old / s)); ties to even, saturating at +-448.
 * Rows at and after the last new token stay as they were. Infinities count
 * for no maximum and are stored as +-448; NaN stays NaN. Tokens whose page
 * lies outside the table or the cache are skipped, as are entries with a
 * negative start or a reqs entry out of range. Two entries that write to one
 * block race: a page that gets tokens belongs to one request, and a request
 * comes once in a call. Needs 16-byte aligned k, v, caches and table, token
 * strides a multiple of 16 bytes. Asynchronous on `stream`. */
QSA_B200_API int qsa_b200_block_append(const qsa_b200_block_append_args* args, qsa_b200_stream_t stream);

typedef struct qsa_b200_block_decode_args {
  const void* q;          /* bf16 [rows, num_q_heads, head_dim], contiguous */
  const void* k_cache;    /* fp8 e4m3fn [num_pages, page_size, num_kv_heads, head_dim] */
  const void* v_cache;
  const float* k_scales;  /* fp32 [num_pages, page_size / block_size, num_kv_heads] */
  const float* v_scales;
  const int32_t* indices; /* [rows, indices_stride], first `topk` columns = logical tokens, <0 = masked;
                             NULL = every token in order (topk is then pages_per_req * page_size) */
  const int32_t* counts;  /* optional [rows]: only the first counts[r] columns may be valid */
  const int32_t* btable;  /* [num_reqs, btable_stride] */
  const int32_t* t2r;     /* optional [rows]: row -> block-table row (NULL = identity) */
  const void* gate;       /* optional bf16 [rows, num_q_heads, head_dim]: out is multiplied by sigmoid(gate) */
  void* out;              /* bf16 [rows, num_q_heads, head_dim] */
  float softmax_scale;
  int32_t rows;
  int32_t num_q_heads;
  int32_t num_kv_heads;
  int32_t head_dim;       /* must be 128 */
  int32_t page_size;
  int32_t block_size;     /* divides page_size */
  int32_t pages_per_req;
  int32_t num_reqs;
  int64_t num_pages;      /* num_pages * page_size <= 2^31 - 1 */
  int32_t topk;           /* not read without indices; a row's columns (topk, or pages_per_req * page_size) are
                             up to 2^31 - 2049, and times num_kv_heads below 2^36 */
  int64_t indices_stride;
  int64_t btable_stride;
} qsa_b200_block_decode_args;

/* Bytes of device workspace qsa_b200_block_decode needs (256-byte aligned;
 * split partial results), negative on invalid arguments. */
QSA_B200_API int64_t qsa_b200_block_decode_workspace_bytes(const qsa_b200_block_decode_args* args);

/* Attention over the block-scaled caches, for row r and query head h of KV
 * head g = h / (num_q_heads / num_kv_heads), groups of 1 to 32:
 *   out[r,h] = softmax_t(q[r,h] . K[t,g] ks[t,g] softmax_scale) . V[t,g] vs[t,g]
 *              (*) sigmoid(gate[r,h])
 * with the masks of qsa_b200_decode: entries that are negative, past the
 * count, past the block table or on a page outside the cache do not count,
 * and what lies in the cache there (NaN too) is not read. A row without a
 * valid entry gives zeros. The workspace needs no clearing and may be reused
 * by the next call on the same stream. Asynchronous on `stream`. */
QSA_B200_API int qsa_b200_block_decode(const qsa_b200_block_decode_args* args, void* workspace, size_t workspace_bytes,
                                       qsa_b200_stream_t stream);

/* ---- The latent cache ------------------------------------------------------
 * Keys and values of all heads come from one vector a token: `rank` latent
 * values, which are key and value, and 64 rotated values, which are key only.
 * A paged cache keeps E4M3FN codes of the latent, the rotated part in bf16 and
 * one fp32 scale a token:
 *   key = scale * (codes, rope)      value = scale * codes.
 * qsa_b200_latent_append writes scales that are powers of two from 2^-60 to
 * 2^60; readers take any scale clamped to that range, and NaN as NaN. Four
 * entry points serve one attention layer over it: qsa_b200_latent_append,
 * qsa_b200_latent_read, qsa_b200_latent_decode (the absorbed form) and
 * qsa_b200_latent_prefill (the expanded form, which needs no cache). None has a
 * counterpart in the reference, whose caches hold a key and a value for each KV
 * head (sm89_cutedsl.py:48-62). */
typedef struct qsa_b200_latent_cache {
  void* codes;           /* fp8 e4m3fn [num_pages, page_size, rank] */
  void* rope;            /* bf16 [num_pages, page_size, rope_dim] */
  float* scales;         /* fp32 [num_pages, page_size] */
  const int32_t* btable; /* [num_reqs, btable_stride]; first pages_per_req columns = physical pages */
  int32_t rank;          /* 128, 256, 384 or 512 */
  int32_t rope_dim;      /* must be 64 */
  int32_t page_size;
  int32_t pages_per_req; /* pages_per_req * page_size and num_pages * page_size up to 2^31 - 1024 */
  int32_t num_reqs;
  int64_t num_pages;
  int64_t btable_stride;
} qsa_b200_latent_cache;

typedef struct qsa_b200_latent_append_args {
  qsa_b200_latent_cache cache;
  const void* c;            /* new latents [tokens, rank] of input_dtype, rows c_stride elements apart */
  const void* r;            /* their rotated part, before the rotation [tokens, rope_dim], rows r_stride apart */
  const int32_t* starts;    /* [entries]: logical position of the entry's first new token */
  const int32_t* reqs;      /* optional [entries]: block-table row of each entry (NULL = identity) */
  const int32_t* cu_tokens; /* optional [entries + 1]: entry e has the tokens cu_tokens[e] .. cu_tokens[e + 1] - 1;
                               NULL: one token each (tokens == entries) */
  const void* c_weight;     /* optional [rank] of weight_dtype: RMS norm of the latent */
  float eps;
  int32_t entries;
  int32_t tokens;
  int32_t input_dtype;      /* QSA_B200_DTYPE_* */
  int32_t weight_dtype;
  int64_t c_stride;
  int64_t r_stride;
  qsa_b200_rotation rotation; /* of r: one axis, rotary_dim up to 64; positions NULL = the tokens' logical positions */
} qsa_b200_latent_append_args;

/* Appends new tokens to the latent cache, in fp32 up to the stored roundings.
 * Entry e's tokens go to the logical positions starts[e], starts[e] + 1, ... of
 * its request:
 *   y     = c * rsqrt(mean(c^2) + eps) * c_weight   (c itself without a weight)
 *   scale = 2^e, e the least with max|y| <= 448 * 2^e, from -60 to 60
 *   codes = e4m3fn(y / scale), ties to even, saturating at +-448
 *   rope  = bf16(rotated r / scale)
 * Infinities of y count for no maximum and are stored as +-448. A token with a
 * NaN in y gets the scale NaN and zero codes. A position outside the rotation
 * table gives a zero rotated part. Tokens outside the block table or the cache
 * are skipped, as are entries with a negative start or a reqs entry out of
 * range. A cache place is named once in a call. Needs 16-byte aligned c, r,
 * codes, rope, c_weight and table, strides a multiple of 16 bytes.
 * Asynchronous on `stream`. */
QSA_B200_API int qsa_b200_latent_append(const qsa_b200_latent_append_args* args, qsa_b200_stream_t stream);

typedef struct qsa_b200_latent_read_args {
  qsa_b200_latent_cache cache;
  void* c;                  /* [tokens, rank] of output_dtype, contiguous */
  void* r;                  /* [tokens, rope_dim] of output_dtype, contiguous */
  const int32_t* starts;    /* [entries] */
  const int32_t* reqs;      /* optional [entries] */
  const int32_t* cu_tokens; /* optional [entries + 1]; NULL: one token each (tokens == entries) */
  int32_t entries;
  int32_t tokens;
  int32_t output_dtype;     /* QSA_B200_DTYPE_* */
} qsa_b200_latent_read_args;

/* Reads tokens back: scale * codes and scale * rope, rounded once. Entry e's
 * rows are the logical positions starts[e], starts[e] + 1, ... of its request,
 * laid out as in qsa_b200_latent_append. Positions outside the block table or
 * the cache give zeros; rows that no entry names are left as they are. Needs
 * 16-byte aligned tensors. Asynchronous on `stream`. */
QSA_B200_API int qsa_b200_latent_read(const qsa_b200_latent_read_args* args, qsa_b200_stream_t stream);

#define QSA_B200_LATENT_MAX_NODES 256
typedef struct qsa_b200_latent_decode_args {
  qsa_b200_latent_cache cache;
  const void* q;          /* bf16 [rows, nodes, heads, rank + rope_dim], contiguous, in the latent's space */
  void* out;              /* bf16 [rows, nodes, heads, rank], contiguous */
  const int32_t* indices; /* [rows, indices_stride], first `topk` columns = logical tokens, <0 = masked;
                             NULL = every token in order */
  const int32_t* counts;  /* optional [rows]: only the first counts[r] columns (without indices: tokens) may be valid */
  const int32_t* t2r;     /* optional [rows]: row -> block-table row (NULL = identity) */
  const int32_t* tree;    /* optional [rows, nodes, tree_words], contiguous: what each node sees of the row's nodes */
  float softmax_scale;
  int32_t rows;
  int32_t nodes;          /* query tokens of a row, 1 .. QSA_B200_LATENT_MAX_NODES; 1 with indices */
  int32_t heads;          /* 1 .. 128 */
  int32_t topk;           /* not read without indices; up to 2^31 - 1024 */
  int32_t tree_words;     /* >= (nodes + 31) / 32 */
  int64_t indices_stride;
} qsa_b200_latent_decode_args;

/* Bytes of device workspace qsa_b200_latent_decode needs (256-byte aligned),
 * negative on invalid arguments. */
QSA_B200_API int64_t qsa_b200_latent_decode_workspace_bytes(const qsa_b200_latent_decode_args* args);

/* Attention in the latent's space (the absorbed form), for row r, node i, head h:
 *   out[r,i,h] = softmax_t(q[r,i,h] . key_t * softmax_scale) . value_t
 * over the tokens that the node sees. With one node: the first counts[r]
 * columns (all without counts). With several, the row's nodes are the last
 * `nodes` of its counts[r] tokens; each node sees the tokens before them and,
 * of the nodes, those j whose bit j % 32 is set in word j / 32 of its tree
 * words, or without a tree nodes 0 to i. Masked entries (those, and as in
 * qsa_b200_decode negative ones and ones on a page outside the table or the
 * cache) do not count, and what the cache holds there is not read, apart from
 * tokens that another node of the row sees. A node without a visible token
 * gives zeros; a head whose query has an infinity or NaN gives NaN where it sees
 * a token. The workspace needs no clearing and may be reused by the next
 * call on the same stream. Needs 16-byte aligned tensors. Asynchronous on
 * `stream`. */
QSA_B200_API int qsa_b200_latent_decode(const qsa_b200_latent_decode_args* args, void* workspace, size_t workspace_bytes,
                                        qsa_b200_stream_t stream);

typedef struct qsa_b200_latent_prefill_args {
  const void* q;       /* [q_tokens, heads, 192]: 128 values, then the 64 rotated ones */
  const void* k;       /* [k_tokens, heads, 128] */
  const void* k_rope;  /* [k_tokens, 64], for all heads */
  const void* v;       /* [k_tokens, heads, 128] */
  void* out;           /* [q_tokens, heads, 128], contiguous */
  const int32_t* cu_q; /* [entries + 1]: entry e has the query tokens cu_q[e] .. cu_q[e + 1] - 1 */
  const int32_t* cu_k; /* [entries + 1]: and the key tokens cu_k[e] .. cu_k[e + 1] - 1 */
  float softmax_scale;
  int32_t entries;
  int32_t q_tokens;
  int32_t k_tokens;
  int32_t heads;
  int32_t causal;      /* query i of n sees the keys up to i + (m - n) of m */
  int32_t dtype;       /* QSA_B200_DTYPE_BF16 or _F16, of all tensors */
  int64_t q_stride, q_head_stride; /* elements from one token, and one head, to the next */
  int64_t k_stride, k_head_stride;
  int64_t v_stride, v_head_stride;
  int64_t k_rope_stride;
} qsa_b200_latent_prefill_args;

/* Attention of prompts in the expanded form, for query token i of an entry and
 * head h over the entry's visible keys j:
 *   out[i,h] = softmax_j((q[i,h,:128] . k[j,h] + q[i,h,128:] . k_rope[j]) * softmax_scale) . v[j,h]
 * A query without a visible key gives zeros; query tokens that no entry names
 * are left as they are. Needs 16-byte aligned tensors and strides (at least the
 * rows they separate) a multiple of 16 bytes. Asynchronous on `stream`. */
QSA_B200_API int qsa_b200_latent_prefill(const qsa_b200_latent_prefill_args* args, qsa_b200_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* QSA_B200_H_ */
