/* Rotary positions, appends to a cache in pages, and attention of sequences that share prefixes over
 * such a cache (C ABI of liblogkv_hip.so, gfx950).
 *
 * Conventions are logkv_hip.h's: device pointers, strides in elements, a hipStream_t as void*;
 * an entry point validates, enqueues on the caller's stream, never allocates and never
 * synchronizes; LOGKV_EINVAL leaves every buffer as it was and logkv_last_error() says why.
 *
 * A paged cache is k_pages [n_pages, n_groups, page, dk] and v_pages [n_pages, n_groups, page, dv];
 * row i of sequence b is slot i % page of page table[b, i / page], page a power of two from 16 on.
 *
 * No counterpart in the reference, which rotates in torch (litgpt/model.py:918-925) and keeps dense
 * caches. */
#ifndef LOGKV_PAGED_H
#define LOGKV_PAGED_H

#include <stdint.h>

#include "logkv_rows.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { LOGKV_F32 = 2 };

/* x [n_batch, heads, tokens, dim] for x = q (n_heads) and k (n_groups), either of them NULL for none:
 * features are turned in pairs i < rotated / 2 by the angle t = sign pos frequencies[i],
 *
 *   (a, b) -> amplitude (a cos t - b sin t, b cos t + a sin t),
 *
 * (a, b) = (x[i], x[i + rotated / 2]), or (x[2 i], x[2 i + 1]) where interleaved; features from
 * `rotated` on pass through. Angles are formed in 64 bits and reduced to a turn before their sine,
 * products are float32, rounded once to the output's type. dtype: LOGKV_BF16, LOGKV_F16 or LOGKV_F32
 * for q, k, v and q_out. rotated: even, 0 (no frequencies needed) to dim; dim up to 512. Features are
 * contiguous; any other strides. frequencies: double, or float with freq_float.
 *
 * pos of token t of batch row b: positions[b pos_sb + t pos_st] (int64, int32 with pos_int), or
 * without positions first + (first_dev ? first_dev[b] : 0) + t; an append adds the row n_b.
 *
 * The other fields are those of logkv_paged_append: n_b = lengths[b] (NULL: 0) + len_add rows in use,
 * token t < counts[b] (NULL: all) is stored at row n_b + t of its sequence, its turned key rounded to
 * the cache's type (cache_dtype: LOGKV_BF16 or LOGKV_F16), its value v as it is. A row at or past
 * table_len pages, below row 0 or on a page outside [0, n_pages) is not stored. k_out (optional there)
 * takes every key in the cache's type. Rows of one call must not share slots. */
typedef struct logkv_rotary_args {
  const void* q;
  int64_t q_sb, q_sh, q_st;
  void* q_out;
  int64_t qo_sb, qo_sh, qo_st;
  const void* k;
  int64_t k_sb, k_sh, k_st;
  void* k_out;
  int64_t ko_sb, ko_sh, ko_st;
  const void* v;
  int64_t v_sb, v_sh, v_st;
  uint16_t* k_pages;
  int64_t kp_sp, kp_sg, kp_st;
  uint16_t* v_pages;
  int64_t vp_sp, vp_sg, vp_st;
  const int32_t* table;
  int64_t table_sb;
  const int32_t* lengths;
  const int32_t* counts;
  const void* frequencies;
  const void* positions;
  int64_t pos_sb, pos_st;
  const int64_t* first_dev;
  int64_t first;
  int32_t n_batch, n_heads, n_groups, tokens, dim, dim_v, rotated, dtype, cache_dtype, interleaved;
  int32_t freq_float, pos_int, len_add, page, table_len, n_pages;
  float amplitude, sign;
} logkv_rotary_args;

int logkv_rotary(const logkv_rotary_args* args, void* stream);

int logkv_paged_append(const logkv_rotary_args* args, void* stream);

/* tq queries per head q [n_batch, n_heads, tq, dk] over, in this order, a prefix that n_batch /
 * n_prefixes consecutive sequences share, the sequence's own rows in its pages and the call's rows
 * k / v [n_batch, n_groups, tq, dk / dv]:
 *
 *   s = scale q . k (+ bias_scale bias, prefix rows);  out = softmax(s) v  (zeros where nothing is seen)
 *
 * Own rows: the first n_b = lengths[b len_stride] + len_add, held to [0, table_len page]. The call's rows:
 * those up to the query's own, or the ones that visible (uint8, as in logkv_rows_args) shows it; with
 * counts (no visible) only the first counts[b] queries and rows exist, the others' outputs are zeros.
 * Prefix (n_prefixes 0: none): rows of pages by prefix_table [n_prefixes, prefix_len pages], or, where
 * prefix_table is NULL, of prefix_k / prefix_v [n_prefixes, n_groups, prefix_len rows, dk / dv] with an
 * optional bias as in logkv_rows_args; the first prefix_lengths[i prefix_stride] + prefix_lengths2[0] +
 * prefix_add rows of each.
 * A table's entry outside [0, n_pages) stands for a page of zeros. Sizes, types, alignment, arithmetic
 * and what infinities and NaNs reach are logkv_rows_args'. */
typedef struct logkv_paged_args {
  const uint16_t* q;
  int64_t q_sb, q_sh, q_st;
  const uint16_t* k;
  int64_t k_sb, k_sg, k_st;
  const uint16_t* v;
  int64_t v_sb, v_sg, v_st;
  uint16_t* k_pages;
  int64_t kp_sp, kp_sg, kp_st;
  uint16_t* v_pages;
  int64_t vp_sp, vp_sg, vp_st;
  const int32_t* table;
  int64_t table_sb;
  const int32_t* lengths;
  const int32_t* counts;
  const uint8_t* visible;
  int64_t vis_sb, vis_st;
  const int32_t* prefix_table;
  int64_t prefix_sb;
  uint16_t* prefix_k;
  int64_t pk_sb, pk_sg, pk_st;
  uint16_t* prefix_v;
  int64_t pv_sb, pv_sg, pv_st;
  const void* bias;
  int64_t b_sb, b_sg, b_st;
  const int32_t* prefix_lengths;
  const int32_t* prefix_lengths2;
  uint16_t* out;
  int64_t o_sb, o_sh, o_st;
  int32_t n_batch, n_heads, n_groups, tq, dk, dv, dtype, page, table_len, n_pages, n_prefixes, prefix_len;
  int32_t len_stride, len_add, prefix_stride, prefix_add, bias_half;
  float scale, bias_scale;
} logkv_paged_args;

/* Scratch of one call. */
int64_t logkv_paged_workspace_bytes(const logkv_paged_args* args);

/* How a call of these sizes is run (no buffer is needed or read), four numbers for the pass over the
 * sequences' own rows, then four for the prefixes' (zeros without one): waves of 32 queries in a block
 * of the tiled kernel, or 0; columns of 16 queries in a block of the streamed kernel, or 0; shares that
 * a lane's rows are dealt in; the most that one may take where tensors of lengths deal them anew. */
int logkv_paged_plan(const logkv_paged_args* args, int32_t plan[8]);

int logkv_paged_attention(const logkv_paged_args* args, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LOGKV_PAGED_H */
