/*
 * pa_mi355x_ext.h — entries of the same library for models beyond the reference operator's
 * attributes: rotary positions of several axes, masks by document and prefix with a bias by
 * distance, and prefixes that several sequences hold in the same pages.  They have no counterpart
 * in the reference; conventions and layouts are pa_mi355x.h's, which declares the entries beside the
 * others.  Here are their descriptors and contracts.
 *
 * The attention entries read every key and value, the new tokens' rows included, from the
 * block-table pages (pa_multi_axis_rotary_append, pa_rotary_append or pa_reshape_and_cache wrote
 * them earlier on the same stream); batch->slot_mapping must be NULL there.  A workspace carries
 * nothing from one call to the next; calls in flight on different streams, and captured graphs
 * whose replays may overlap, need a workspace each.
 */
#ifndef PA_MI355X_EXT_H
#define PA_MI355X_EXT_H

#include "pa_mi355x.h"

/* Rotary positions of several axes (time, height and width of images and video).  Frequency i of
 * [0, rotary_half) turns by the cos / sin row of positions[axis(i)][t].  axes_interleaved 0: the
 * axes' sections follow each other (the first sections[0] frequencies on axis 0, the next
 * sections[1] on axis 1, ...); 1: they take turns, axis(i) = i % axes while i < axes *
 * sections[i % axes], axis 0 beyond.  A pair whose position lies outside [0, rotary_positions) is
 * left unturned.  (One row of positions for every axis: axes 1 and one section.) */
#define PA_MAX_AXES 4
typedef struct pa_axis_rotary {
  const int64_t* positions; /* [axes, num_tokens] */
  int64_t position_stride;  /* elements from one axis' row to the next; 0 = num_tokens */
  int32_t axes;             /* 1 .. PA_MAX_AXES */
  int32_t sections[PA_MAX_AXES]; /* frequencies of each axis; their sum is rotary_half */
  int32_t axes_interleaved;
  const void* cos_cache; /* [rotary_positions, rotary_half] in table_dtype */
  const void* sin_cache;
  pa_dtype table_dtype; /* the activation dtype or PA_DTYPE_FLOAT32 */
  int64_t rotary_positions;
  int32_t rotary_half;        /* rotary_offset + 2 * rotary_half <= head_dim */
  int32_t rotary_offset;      /* first rotated element of a head row */
  int32_t rotary_interleaved; /* 0: pairs (i, rotary_half + i); 1: pairs (2 i, 2 i + 1) */
} pa_axis_rotary;

/* pa_multi_axis_rotary_append: RMSNorm (optional) and multi-axis rotary positions on the query and key rows, queries into
 * q_out, keys and values into their pages.
 *   query/key/value  [num_tokens, heads * head_dim] in act_dtype, consecutive tokens q_stride /
 *                    k_stride / v_stride elements apart (0 = dense; views of packed QKV rows)
 *   q_out            [num_tokens, num_heads * head_dim], dense; the query buffer itself (dense
 *                    rows) or one apart from every input.  query and q_out NULL: keys and values
 *                    alone.
 *   q_norm/k_norm    [head_dim] act_dtype, both or neither
 * A row is normalised, scaled by the weights and turned in fp32 and rounded to act_dtype once;
 * fp8 and integer caches encode that rounded row.  Slots, -1 entries of batch->slot_mapping and
 * tokens that share a slot are treated as by pa_rotary_append. */

/* Masks and a bias by distance, each optional (NULL).  Token t = row r of sequence b stands at
 * position i = past[b] + r and sees key j of its sequence iff
 *   max(document_starts[t], i - local_window_size + 1) <= j < max(i + 1, prefix_lens[b])
 * (is_causal 0: up to the sequence's last key; local_window_size -1: no window, else at least 1),
 * and its score there is
 *   softcap(scale * q.k) - distance_slopes[h] * |i - j|.
 * A row that sees no key is zero. */
typedef struct pa_mask {
  const float* distance_slopes;   /* [num_heads] fp32 */
  const int32_t* prefix_lens;     /* [batch]: leading keys that every row of the sequence sees */
  const int32_t* document_starts; /* [num_tokens]: first key of the token's document */
} pa_mask;

/* pa_masked_attention: attention over the pages under such a mask (mask NULL: plain paged
 * attention).  Layouts of q and out and the attributes as pa_attention; the SEPARATE cache layout; out
 * apart from q.  Workspace: at least the size that pa_masked_attention_workspace_bytes gives.
 * fp16 / bf16 activations and pages at heads 64, 96, 128 and 256, from caches that begin at 16 bytes,
 * run on matrix cores and want q, out and the workspace at 16 bytes too (refused otherwise).
 * Everything else runs without them, many times as long on prompts: other types and heads, byte-coded
 * pages, and calls whose blocks of 128 rows times their tables' tiles of 64 keys pass 2^30 (a prompt of
 * 400,000 tokens at 64 heads). */

/* Groups of consecutive sequences whose first keys are the same, in the same pages: group i holds
 * sequences [group_cum[i], group_cum[i + 1]) and their first prefix_lens[i] keys.  The caller
 * guarantees that the block tables of a group's sequences name the same pages for those keys; the
 * library may read them through any one of the tables.  Sequences outside every group share
 * nothing. */
typedef struct pa_shared_prefix {
  const int32_t* group_cum;   /* [groups + 1], non-decreasing, within [0, batch] */
  const int32_t* prefix_lens; /* [groups] */
  int32_t groups;             /* >= 1 */
  int32_t max_prefix_len;     /* host-known bound on prefix_lens, for the plan and its workspace;
                               * 0 = the context's own bound */
} pa_shared_prefix;

/* pa_shared_prefix_attention: pa_masked_attention for such groups, with the same results up to
 * rounding.  On matrix cores the keys and values of a prefix are read once for all the rows of its
 * group (once per 128 of them), otherwise for every row. */

#endif /* PA_MI355X_EXT_H */
