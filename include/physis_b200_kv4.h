/*
 * physis_b200_kv4.h -- C ABI of the paged 4-bit K/V cache on B200 (sm_100a):
 * appending (RMSNorm + RoPE + quantisation in one launch), reading rows back,
 * and attention over the cache.
 *
 * The ring of physis_b200.h holds a stream's rotated K and V in the activation
 * type: 4*C bytes a token in bf16.  At full state (a ring per stream, denoising
 * step and block) that is what limits the streams a GPU serves, and attention
 * with few query rows is bound by reading it.  This cache holds the same rows in
 * 4.5 bits an element (1.125*C bytes a token) in pages of one pool, so that
 * cells of unlike window length share the memory.
 *
 * Format.  The pool is uint8 [num_pages, kv_heads, 2, page_rows * 72]: for each
 * head K (index 0) and V (index 1), page_rows rows of 64 code bytes, then
 * page_rows rows of 8 scale bytes.  A row is one token's 128 elements of one
 * head.  Code byte j holds elements 2j (low four bits) and 2j+1 (high four bits)
 * as e2m1; scale byte i is the (non-negative) e4m3 scale of elements 16i..16i+15.
 * An element is code * scale * tensor scale (k_scale or v_scale of the call).
 * Logical row r of the cache lies in page table[r / page_rows] at row
 * r % page_rows; a member's rows start at member * table_pages * page_rows.
 *
 * Quantisation of a block of 16 elements x (rounded to the activation type, as
 * the bf16 or fp32 ring would hold them): scale = e4m3(max|x| / (6 * tensor
 * scale)), codes = e2m1(x / (scale * tensor scale)), both to nearest, ties to
 * even, saturating.  The format has no infinities and no NaN: an infinite
 * element saturates, a NaN is stored as zero, and each such block is counted.
 *
 * A table entry outside [0, num_pages) is never followed: an append skips the
 * row, a read returns zeros, an attention leaves the page's keys out, and each
 * counts it in its own measure.  ps_kv4_counters reads both counts.
 *
 * Status codes, PS_API, ps_seq and the table modes come from physis_b200.h.
 * Every entry point validates on the host first, allocates nothing and is
 * asynchronous on the given stream.
 */
#ifndef PHYSIS_B200_KV4_H
#define PHYSIS_B200_KV4_H

#include "physis_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define PS_KV4_HEAD_DIM 128 /* elements of a row */
#define PS_KV4_ROW_BYTES 72 /* 64 of codes, 8 of scales */

/* The cache a call works on. */
typedef struct ps_kv4_cache {
  void* pages;           /* uint8 [num_pages, kv_heads, 2, page_rows * 72], 16-byte aligned */
  const int32_t* table;  /* device [members, table_pages], row-contiguous */
  int64_t num_pages;
  int64_t members;
  int64_t table_pages;   /* table entries per member */
  int32_t kv_heads;      /* >= 1 */
  int32_t page_rows;     /* 16, 32, 64 or 128 */
  float k_scale;         /* tensor scales, > 0 */
  float v_scale;
} ps_kv4_cache;

/* Arguments of ps_qk_norm_rope_kv4.  As ps_qk_prep_args, with the K and V rows
 * going to the cache: ring_row, ring_frames and ring_slot0 of a sequence name
 * logical rows of the cache (a member's rows start at member * table_pages *
 * page_rows).  No two tokens of a launch may go to the same row of the same page,
 * by equal ring rows or by a page that stands in the table twice: which of them
 * the row then holds is not defined. */
typedef struct ps_kv4_prep_args {
  int32_t dtype;      /* ps_dtype of q, k, v, q_out, k_pre and k_sink */
  int32_t heads;      /* query heads */
  int32_t head_dim;   /* 128 */
  int32_t table_mode; /* ps_table_mode */
  int32_t t_dim, h_dim, w_dim; /* axis split of head_dim (even parts); PS_TABLE_AXES only */
  int32_t n_seqs;     /* 1..PS_MAX_SEQS */
  float eps;          /* RMSNorm epsilon */
  int32_t weight_f32; /* 0: weights are of dtype; 1: fp32 */
  int32_t launch;     /* ps_launch; PS_LAUNCH_PDL_EARLY_INPUTS reads the page table before
                       * the wait too: no kernel still running may write it */
  int32_t reserved;   /* 0 */

  int64_t in_rows;                    /* rows of q, k, v, q_out, k_pre */
  const void* q;  int64_t q_stride;   /* [in_rows, heads*128]; NULL: no Q role */
  const void* k;  int64_t k_stride;   /* [in_rows, kv_heads*128]; NULL: no K role */
  const void* v;  int64_t v_stride;   /* [in_rows, kv_heads*128]; NULL: no V role */
  const void* q_weight;               /* [heads*128]; both weights NULL: no RMSNorm */
  const void* k_weight;               /* [kv_heads*128] */
  const float* cos;                   /* [table_rows, 128] fp32 */
  const float* sin;
  int64_t table_rows;
  void* q_out;  int64_t q_out_stride; /* rotated Q rows */
  void* k_pre;  int64_t k_pre_stride; /* optional: normalised K before RoPE */
  const void* k_sink; int64_t k_sink_stride; /* pre-RoPE K rows of PS_SEQ_SINK sequences */
  int64_t k_sink_rows;
  ps_kv4_cache cache;
  const ps_seq* seqs;                 /* host array of n_seqs descriptors */
} ps_kv4_prep_args;

/* Arguments of ps_kv4_read: rows [row0, row0 + rows) of every member, as
 * [members, rows, kv_heads*128] with a row and a member stride (elements). */
typedef struct ps_kv4_read_args {
  int32_t dtype;      /* ps_dtype of k_out and v_out */
  int32_t reserved;   /* 0 */
  int64_t row0, rows; /* logical rows of each member */
  void* k_out; int64_t k_member_stride; int64_t k_row_stride; /* NULL: K is not read */
  void* v_out; int64_t v_member_stride; int64_t v_row_stride; /* NULL: V is not read */
  ps_kv4_cache cache;
} ps_kv4_read_args;

/* Which kernel ps_attention_kv4 runs. */
typedef enum ps_kv4_kernel {
  PS_KV4_AUTO = 0,
  PS_KV4_ROWS = 1, /* 8 query rows of a K/V head at a time, bound by reading the cache */
  PS_KV4_TILES = 2 /* 256 query rows of a K/V head at a time on the tcgen05 tensor cores */
} ps_kv4_kernel;

/* Arguments of ps_attention_kv4.  Query row t of member b, head h starts at
 * q + b*q_member_stride + t*q_row_stride + h*128 (elements); head h reads K/V
 * head h / (heads / kv_heads).  Member b sees the rows [0, n_b) of its cache:
 * n_b = kv_lens[b] clamped to [0, kv_tokens], or kv_tokens without kv_lens.
 * With causal_block c > 0, query row t sees the rows
 *   [0, min(n_b, n_b - q_tokens + (t / c + 1) * c)):
 * c = 1 is the causal mask of the last q_tokens rows, c = tokens of a frame lets
 * a frame see itself and the frames before it.  A row that sees nothing gets
 * zeros. */
typedef struct ps_kv4_attn_args {
  int32_t heads;        /* query heads, a multiple of cache.kv_heads */
  int32_t q_tokens;     /* query rows per member (>= 0) */
  int32_t kv_tokens;    /* most window rows of a member, 0 .. table_pages * page_rows */
  int32_t causal_block; /* 0: no mask */
  float scale;          /* softmax scale; <= 0 selects 1/sqrt(128) */
  int32_t kernel;       /* ps_kv4_kernel */
  int32_t key_chunks;   /* rows kernel: key chunks per block of rows, 1..64; 0 = automatic */
  int32_t reserved;     /* 0 */
  const void* q;  int64_t q_member_stride;   int64_t q_row_stride;   /* bf16 */
  void* out;      int64_t out_member_stride; int64_t out_row_stride; /* bf16 */
  const int32_t* kv_lens; /* device [members], or NULL */
  void* workspace;        /* device scratch of ps_kv4_attention_workspace() bytes, 16-byte aligned;
                           * calls that may run at once need one each */
  int64_t workspace_bytes;
  ps_kv4_cache cache;
} ps_kv4_attn_args;

/* RMSNorm(Q), RMSNorm(K), RoPE of Q and K, and the quantised write of rotated K
 * and of V: ps_qk_norm_rope_kv with the cache in the place of the ring.  Same
 * roundings; K's sum of squares is accumulated in 64 bits, so that the rows that
 * are quantised do not depend on the order of that sum (but for one in some 2^28
 * of those rows whose squares do not sum exactly in 64 bits). */
PS_API int32_t ps_qk_norm_rope_kv4(const ps_kv4_prep_args* args, void* stream);
PS_API int32_t ps_kv4_prep_validate(const ps_kv4_prep_args* args);

/* Cache rows as numbers: code * scale * tensor scale, rounded once to dtype. */
PS_API int32_t ps_kv4_read(const ps_kv4_read_args* args, void* stream);
PS_API int32_t ps_kv4_read_validate(const ps_kv4_read_args* args);

/* Softmax attention of every query row over the window rows it sees.  Q and the
 * dequantised K and V enter the products in fp16: code * scale has six
 * significant bits, so K and V are exact, and a query row is scaled by the power
 * of two that brings its largest element to [1, 2) ([2, 4) from 2^127 on), so
 * that nothing of it that matters at 24 bits is lost (the tensor scales and that
 * power are applied to the scores in fp32).  Scores, softmax statistics and sums
 * are fp32; probabilities are rounded to fp16 for P V, with an absolute error of
 * 2^-32 of the row's largest at most where that is more than 2^-11 of their own;
 * the output is rounded once to bf16. */
PS_API int32_t ps_attention_kv4(const ps_kv4_attn_args* args, void* stream);
PS_API int32_t ps_kv4_attention_validate(const ps_kv4_attn_args* args);
/* Bytes of scratch that ps_attention_kv4 needs for these arguments on the current device (of the pointers
 * only kv_lens matters: whether it is NULL). */
PS_API int32_t ps_kv4_attention_workspace(const ps_kv4_attn_args* args, int64_t* bytes);

/* What ps_kv4_counters clears after reading (any other value clears every count). */
typedef enum ps_kv4_reset {
  PS_KV4_KEEP = 0,
  PS_KV4_RESET = 1,          /* every count */
  PS_KV4_RESET_TIMEOUTS = 2  /* counts[2] alone */
} ps_kv4_reset;

/* Counts on the current device since each was last cleared: counts[0] pages outside
 * the pool that calls came upon (an append counts each token of such a page, a read
 * each 16 elements of a row and head, an attention each thread block that takes
 * its keys), counts[1] blocks that held an infinity or a NaN, counts[2]
 * bounded waits that ran out (the outputs of that call are undefined).
 * Synchronises the device first. */
PS_API int32_t ps_kv4_counters(uint32_t counts[3], int32_t reset);

#ifdef __cplusplus
}
#endif

#endif /* PHYSIS_B200_KV4_H */
