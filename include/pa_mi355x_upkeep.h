/*
 * pa_mi355x_upkeep.h — entries of the same library that keep a paged cache at work: attention of
 * drafted trees and what is accepted of them, attention that keeps account of what its keys weigh,
 * and the eviction that goes by that account.  They have no counterpart in the reference;
 * conventions and layouts are pa_mi355x.h's, which declares the entries beside the others.  Here
 * are their descriptors and contracts.
 *
 * A block-table entry that names no page is read as the nearest one and never written through.
 *
 * The attention entries read every key and value, the new tokens' rows included, from the
 * block-table pages; batch->slot_mapping must be NULL.  A workspace carries nothing from one call to
 * the next; calls in flight on different streams, and captured graphs whose replays may overlap,
 * need a workspace each.
 */
#ifndef PA_MI355X_UPKEEP_H
#define PA_MI355X_UPKEEP_H

#include "pa_mi355x.h"

/* ---- Drafted trees ---------------------------------------------------------------------------
 * The new tokens of a sequence may be the nodes of a tree of drafted tokens: parents[t] is the row
 * (within the sequence's new tokens) of the node's parent, which comes before it; -1, and whatever
 * names no earlier row, makes it a root.  A node of depth d (0: a root) stands at position past + d
 * of its text; its key and value are in slot past + row, like any new token's
 * (pa_multi_axis_rotary_append with one axis appends rows turned to positions of their own).  At
 * most PA_MAX_TREE_NODES nodes to a sequence. */
#define PA_MAX_TREE_NODES 4096

/* pa_tree_attention: attention in which a node sees the keys [0, past) and, of the new rows, its
 * ancestors and itself; under a window the keys and ancestors less than local_window_size positions
 * before it.  parents [num_tokens] int32.  Layouts, attributes (is_causal must be 1) and types as
 * pa_masked_attention's; out apart from q.  max_query_len bounds the nodes of a
 * sequence (0: num_tokens, at most PA_MAX_TREE_NODES); nodes beyond the bound see the keys before
 * the tree at most, and what they yield is unspecified.  Workspace: at least the size that
 * pa_tree_attention_workspace_bytes gives; 16-byte aligned. */

/* pa_accept_drafts: the accepted path of every sequence, and its rows moved to where the cached
 * sequence goes on: row path[i] of the new tokens to slot past + i, keys and values of every head.
 * The path begins with row 0 and goes on, while there is one, to the first child of its last node
 * whose token is that node's target (parents, tokens, targets given; path, path_lens and next_tokens
 * are then written), or it is given (parents NULL: rising rows in path, path_lens of them).  A step
 * without new tokens has empty paths (parents, tokens, targets not NULL; nothing is read there).  Other
 * rows of the new tokens keep what they held or lose it to the path's.  fp8 rows that move to a page
 * of another scale are encoded anew (x / scale as the append does); other rows keep their bytes.
 * The pages of the new tokens must belong to their sequence alone. */
typedef struct pa_drafts {
  const int32_t* parents;  /* [num_tokens], or NULL */
  const int64_t* tokens;   /* [num_tokens]: the drafted tokens */
  const int64_t* targets;  /* [num_tokens]: the model's choice after each of them */
  int32_t* path;           /* [batch, max_path] rows; those behind the path are set to -1 */
  int32_t* path_lens;      /* [batch] */
  int64_t* next_tokens;    /* [batch]: the target of the path's last node (-1: no new tokens); or NULL */
  int32_t max_path;        /* >= 1; longer paths end there */
  float* key_weights;      /* the cache's accounts (see below), which the path's rows begin anew at
                            * zero; or NULL */
} pa_drafts;

/* ---- Accounts and eviction -------------------------------------------------------------------
 * An account holds what every cached key weighed, per kv-head, beside the pages and in their order:
 * key_weights [num_blocks, kv_heads, block_size] fp32.
 *
 * pa_accumulating_attention: attention over the pages (the new tokens' rows among them) that adds to
 * every key's account the probabilities, sinks in their denominator, that the rows which count gave
 * it, over the heads of its kv-head: the last `observed_rows` new tokens of each sequence (0: all of
 * them).  Keys of the new tokens begin at zero, whatever their slots held.  The same call on the
 * same inputs gives the same bits.  Windows, softcaps, sinks, types and layouts as
 * pa_masked_attention's; out apart from q, key_weights 4-byte aligned and apart from
 * everything else.  Where several sequences of the call hold a page, each of them writes its entries,
 * which are then unspecified (the outputs are not).  Workspace: at least the size that
 * pa_accumulating_attention_workspace_bytes gives (up to 32 rows of one kv-head per sequence: 4
 * bytes for every row and key of the context bound); 16-byte aligned.  A sequence whose context
 * exceeds max_context_len leaves its account unspecified. */

/* pa_evict_keys: the keys of every (sequence, kv-head) that stay.  A sequence that holds
 * n = batch->past_seqlens[b] <= budget keys keeps them all; of more stay the first `sinks`, the last
 * `recent` and of those between them the budget - sinks - recent that weigh most, the lower position
 * of equals first (-0 like +0; NaN weighs more than all).  They keep their order: kept names their
 * positions (-1 behind them), row i of the pages becomes row kept[i], key, value and account.  The
 * rows go to the sequence's own pages (block_table_out NULL; rows behind the new length keep what
 * they held or lose it) or to other ones, no page of which any sequence of the batch holds.  Pages
 * that are written belong to one sequence alone.  Heads keep different keys; keys carry their rotary
 * positions with them, so that attention without a window goes on as before over fewer keys.  fp8
 * rows as in pa_accept_drafts.  Of batch, only past_seqlens, block_table, batch, max_blocks and
 * max_context_len (0: the tables' capacity; keys beyond it are not looked at) are read. */
typedef struct pa_eviction {
  float* key_weights;
  int32_t budget, sinks, recent; /* budget >= 1; sinks, recent >= 0, sinks + recent <= budget */
  const int32_t* block_table_out; /* [batch, max_blocks_out], or NULL */
  int32_t max_blocks_out;         /* pages for min(budget, the context bound) rows at least */
  int32_t* kept;                  /* [batch, kv_heads, budget] */
  int32_t* lens_out;              /* [batch]: min(n, budget); past_seqlens itself is refused */
} pa_eviction;

#endif /* PA_MI355X_UPKEEP_H */
