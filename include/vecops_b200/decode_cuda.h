/*
 * One decode step of an attention block on the GPU: products of block-scaled 8-bit floating point, and attention over a
 * paged key/value cache whose sequences share a prefix.
 *
 * These stand next to the quantised matmul rows and the attention caller of matmul_cuda.h and follow its rules: all
 * pointers are DEVICE pointers on `device_index`, strides count elements, nothing allocates device memory, errors come
 * back as VecopsStatusCode with a message, calls are synchronous unless VECOPS_B200_MATMUL_FLAG_ASYNC is set, and there
 * is no CPU fallback.  The first call on a device sets it up; make it before any stream capture begins.  Calls whose outputs
 * and scratch are apart may run at once, on any streams.  The reference has no counterpart of these operators.
 *
 *     vecops_b200_quantize_blocks     x -> e4m3 values and an fp32 scale per 1 x 128 or 128 x 128 block
 *     vecops_b200_matmul_f8_run       C = sum over 128-blocks of K of a_scale * b_scale * (A_block . B_block^T)
 *     vecops_b200_cache_append        rotate queries and keys by position, write keys and values into cache pages
 *     vecops_b200_prefix_sdpa_run     attention over a shared prefix plus each sequence's own suffix, both in pages
 */
#ifndef VECOPS_B200_DECODE_CUDA_H
#define VECOPS_B200_DECODE_CUDA_H

#include "vecops_b200/matmul_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------------------------------------------------------
 * Block quantiser.  For every block of `block_rows` x 128 elements (the last ones may be smaller)
 *
 *     amax  = largest |x| of the block, taken to lie in [2^-110, largest finite f32]
 *     scale = amax / 448
 *     q     = x * (448 / amax) rounded to the nearest e4m3 value, ties to even, saturating at +-448
 *
 * NaN elements become NaN and do not count towards amax; infinities become +-448 of a block whose scale is that of the
 * largest finite f32.  q * scale stands for x. */
typedef struct VecopsB200QuantizeBlocks {
  uint32_t struct_size;
  uint32_t block_rows;        /* 1 (activations) or 128 (weights) */
  int64_t rows, cols;
  const void* src;            /* [rows, cols] */
  int64_t src_stride_row, src_stride_col;
  uint32_t src_dtype;         /* F32 | BF16 | F16 */
  uint32_t flags;             /* VECOPS_B200_MATMUL_FLAG_ASYNC */
  void* dst;                  /* [rows, cols] e4m3, one byte each, contiguous along cols */
  int64_t dst_stride_row;     /* >= cols; a multiple of 16 (and a 16-byte aligned dst) lets the product read it by TMA */
  float* scale;               /* [ceil(rows / block_rows), ceil(cols / 128)] */
  int64_t scale_stride_row, scale_stride_col;
  void* stream;
  int32_t device_index;
  uint32_t reserved;
} VecopsB200QuantizeBlocks;

VECOPS_B200_EXPORT int32_t vecops_b200_quantize_blocks(const VecopsB200QuantizeBlocks* quantize, VecopsError* error);

/* ---------------------------------------------------------------------------------------------------------------
 * Product of block-scaled e4m3 operands, B as everywhere [N,K]:
 *
 *     C[m,n] = sum_b a_scale[m,b] * b_scale[n / 128, b] * sum_{k in block b} A[m,k] * B[n,k]        (blocks of 128 along K)
 *
 * Each block's sum is accumulated in fp32 and enters the total in fp32 with its scale; one rounding to C's type.  The two scales
 * are multiplied with each other first: where that product leaves fp32's normal range, 2^-126 to 2^128, a block's share loses digits or
 * becomes inf, or NaN beside a sum of 0.  K == 0 stores zeros. */
typedef enum VecopsB200MatmulF8Kernel {
  VECOPS_B200_F8_AUTO = 0,
  VECOPS_B200_F8_GENERIC = 1, /* CUDA cores; any strides */
  VECOPS_B200_F8_STREAM = 2,  /* up to 128 rows of A: weights streamed once through tcgen05 as its 128-row operand */
  VECOPS_B200_F8_TILED = 3,   /* tcgen05 kind::f8f6f4 on 256 x 256 tiles of CTA pairs */
  VECOPS_B200_F8_COUNT_ = 4
} VecopsB200MatmulF8Kernel;

typedef struct VecopsB200MatmulF8 {
  uint32_t struct_size;
  uint32_t kernel;            /* VecopsB200MatmulF8Kernel; AUTO = pick by rules */
  int64_t m, n, k;
  const void* a;              /* [M,K] e4m3 */
  int64_t a_stride_m, a_stride_k;
  const float* a_scale;       /* [M, ceil(K/128)] */
  int64_t a_scale_stride_m, a_scale_stride_k;
  const void* b;              /* [N,K] e4m3 */
  int64_t b_stride_n, b_stride_k;
  const float* b_scale;       /* [ceil(N/128), ceil(K/128)] */
  int64_t b_scale_stride_n, b_scale_stride_k;
  void* c;                    /* [M,N] */
  int64_t c_stride_m, c_stride_n;
  uint32_t c_dtype;           /* BF16 | F16 | F32 */
  uint32_t flags;             /* VECOPS_B200_MATMUL_FLAG_ASYNC */
  void* stream;
  int32_t device_index;       /* -1: the calling thread's current device */
  uint32_t reserved;
} VecopsB200MatmulF8;

/* Pure host logic: which kernel the rules choose.  INVALID_ARGUMENT for a record that no kernel serves, NOT_APPLICABLE
 * when `kernel` was forced to one that cannot serve it. */
VECOPS_B200_EXPORT int32_t vecops_b200_matmul_f8_select(const VecopsB200MatmulF8* problem, uint32_t* kernel, VecopsError* error);
VECOPS_B200_EXPORT int32_t vecops_b200_matmul_f8_run(const VecopsB200MatmulF8* problem, VecopsError* error);

/* ---------------------------------------------------------------------------------------------------------------
 * Appending to a paged key/value cache, with the rotation by position on the way.  For token t
 *
 *     (c, s) = row positions[t] of cos_sin, c its first half and s its second
 *     pair (x1, x2) -> (x1 * c - x2 * s, x2 * c + x1 * s)          on the first `rotary` dims of every query and key head;
 *     pairs are (i, i + rotary/2), or (2i, 2i + 1) with `interleaved`; the other dims are copied
 *
 * in fp32 with one rounding.  The rotated query goes to q_out[t], the rotated key and the value to cache row slots[t] =
 * page * page_size + offset.  A token whose slot is outside the cache (-1 for padding) or whose position is outside the
 * table writes nothing into the cache and zeros into q_out[t]; no other cache row is touched.  Slots of one call that are
 * inside the cache must differ from one another.  q and q_out may be NULL together (keys and values only); q_out may be
 * q itself. */
typedef struct VecopsB200CacheAppend {
  uint32_t struct_size;
  uint32_t dtype;             /* BF16 | F16: q, k, v, q_out and the cache */
  int64_t tokens, q_heads, kv_heads, head_dim;
  const void* q;              /* [tokens, q_heads, head_dim], contiguous along head_dim like every operand here */
  int64_t q_stride_token, q_stride_head;
  const void* k;              /* [tokens, kv_heads, head_dim] */
  int64_t k_stride_token, k_stride_head;
  const void* v;
  int64_t v_stride_token, v_stride_head;
  void* q_out;                /* [tokens, q_heads, head_dim] */
  int64_t q_out_stride_token, q_out_stride_head;
  void* k_cache;              /* [pages, page_size, kv_heads, head_dim] */
  int64_t k_stride_page, k_stride_slot, k_cache_stride_head;
  void* v_cache;
  int64_t v_stride_page, v_stride_slot, v_cache_stride_head;
  int64_t pages, page_size;
  const int64_t* slots;       /* [tokens] */
  const int64_t* positions;   /* [tokens] */
  const float* cos_sin;       /* [max_positions, rotary], contiguous rows */
  int64_t cos_sin_stride;     /* from row to row */
  int64_t max_positions, rotary; /* rotary even, 0..head_dim; 0 = no rotation (cos_sin and positions are not read) */
  uint32_t interleaved;
  uint32_t flags;             /* VECOPS_B200_MATMUL_FLAG_ASYNC */
  void* stream;
  int32_t device_index;
  uint32_t reserved;
} VecopsB200CacheAppend;

VECOPS_B200_EXPORT int32_t vecops_b200_cache_append(const VecopsB200CacheAppend* append, VecopsError* error);

/* ---------------------------------------------------------------------------------------------------------------
 * Attention of a batch whose sequences share one prefix, over paged caches.  Sequence b owns the query tokens
 * [query_starts[b], query_starts[b+1]) - one each, token b, when query_starts is NULL - which are its newest: the last one
 * sees the whole prefix and all lengths[b] suffix keys (its own among them), the one before it one suffix key less, and
 * so on.  Query head h reads key/value head h / (q_heads / kv_heads).
 *
 *     out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q.k_j - max)      over prefix keys [0, prefix_len) and the seen suffix keys
 *
 * Scores, maxima, both sums and the result before its one rounding are fp32; in the first sum the kernels on the tensor cores round p_j to q's
 * type, which a 16-bit product takes (the second keeps all of it): an error of half a step a key, under the rounding of the result
 * where many keys have weight.
 *
 * Prefix key j lies in page prefix_pages[j / page_size], suffix key j of sequence b in page page_table[b][j / page_size].
 * Keys of a page number outside [0, pages) count as absent, as do suffix keys past the table's width.  A query that sees
 * no key, a token of no sequence and the tokens of a sequence with a negative length (padding of a captured batch) get
 * zeros.  A NaN in a query or in a key that it sees gives NaN, and so do scores that are +inf or all -inf (0 / 0 by the formula).
 * What lies in the cache behind the last key is never used, NaN included.  lengths, query_starts and both tables
 * are read on the device, so a captured call follows their later contents; prefix_len is fixed at the call. */
typedef struct VecopsB200PrefixAttention {
  uint32_t struct_size;
  uint32_t dtype;             /* BF16 | F16: q, the caches and out */
  int64_t tokens, batch, q_heads, kv_heads, head_dim; /* head_dim 1..256 */
  const void* q;              /* [tokens, q_heads, head_dim], contiguous along head_dim like every operand here */
  int64_t q_stride_token, q_stride_head;
  void* out;                  /* [tokens, q_heads, head_dim] */
  int64_t out_stride_token, out_stride_head;
  const void* k_cache;        /* [pages, page_size, kv_heads, head_dim] */
  int64_t k_stride_page, k_stride_slot, k_stride_head;
  const void* v_cache;
  int64_t v_stride_page, v_stride_slot, v_stride_head;
  int64_t pages, page_size;
  const int32_t* prefix_pages; /* [ceil(prefix_len / page_size)] */
  int64_t prefix_len;
  const int32_t* page_table;  /* [batch, table_width], contiguous rows */
  int64_t table_stride, table_width;
  const int32_t* lengths;     /* [batch] */
  const int32_t* query_starts; /* [batch + 1], not decreasing, or NULL; what passes [0, tokens] counts as 0 or tokens */
  float scale;
  uint32_t flags;             /* VECOPS_B200_MATMUL_FLAG_ASYNC */
  void* workspace;            /* 256-byte aligned device scratch of vecops_b200_prefix_sdpa_workspace bytes */
  uint64_t workspace_size;
  void* stream;
  int32_t device_index;
  uint32_t reserved;
} VecopsB200PrefixAttention;

/* Scratch of a call: by the record's extents, whether it has query_starts, and the device's SM count - whatever the pointers, strides and
 * contents are, so one size serves every call of a shape.  A call whose rows lie off 16-byte boundaries does without. */
VECOPS_B200_EXPORT int32_t vecops_b200_prefix_sdpa_workspace(const VecopsB200PrefixAttention* attention, uint64_t* bytes, VecopsError* error);
VECOPS_B200_EXPORT int32_t vecops_b200_prefix_sdpa_run(const VecopsB200PrefixAttention* attention, VecopsError* error);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* VECOPS_B200_DECODE_CUDA_H */
