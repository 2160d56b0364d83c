/* C ABI of the serving-step operators of libexactattn_cuda.so: what a decoding loop over draft
 * trees runs next to the certified attention of exactattn_cuda.h.
 *
 *   ea_plan_step_cuda       page allocation, slot map, positions and lengths of a step
 *   ea_rope_cuda            rotary positions (1 to 4 axes), optionally written into the paged cache
 *   ea_tree_attention_cuda  attention of drafted tokens (tree, chain, single token) over a paged cache
 *   ea_process_logits_cuda  penalties for repeated tokens, biases and grammar masks
 *
 * These are ordinary floating-point operators: they serve the draft side of speculative decoding,
 * whose results the certified attention verifies. Arithmetic is 32-bit and outputs are rounded once,
 * except that the attention's weights enter the product with the values as 16-bit numbers (below).
 * Every pointer is a device pointer, every call is asynchronous on `stream` (a cudaStream_t, NULL =
 * default), allocates nothing, never waits for the host, and may be captured in a CUDA graph.
 * Calls share no state: they may run on several streams at once.
 *
 * Return codes as exactattn_cuda.h: 0 OK, -1 bad dimensions, -4 CUDA error, -9 unsupported layout.
 * ea_serving_last_error() has the message of this thread's last failure. */
#ifndef EXACTATTN_SERVING_H
#define EXACTATTN_SERVING_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
enum { EA_BF16 = 0, EA_FP16 = 1, EA_FP32 = 2 };

/* One step's paging. Sequence b holds context_lens[b] cached keys and receives new_lens[b] tokens
 * (a prompt chunk, a draft tree, one token, none). Negative lengths count as 0. It owns
 * ceil(context / page_size) pages; the pages it lacks are taken from free_pages[free_head ..] in
 * sequence order and written into its row of page_table (-1 once the list has run out). Token t of
 * the step is the i-th of sequence b = token_seq[t], i = t - q_start[b]:
 *   slot_map[t]  page * page_size + offset of cache position context + i (-1: no page)
 *   positions[t] context + depths[t] (depths NULL: context + i)
 * Slots t past the step's tokens are padding: slot -1, position 0, token_seq -1.
 * status (one int, overwritten): 0, or bits EA_PLAN_NO_PAGES (the free list ran out),
 * EA_PLAN_TABLE_FULL (a sequence needs more than max_pages pages), EA_PLAN_TOO_MANY (the step has
 * more than max_tokens tokens; the first max_tokens are planned). */
enum { EA_PLAN_NO_PAGES = 1, EA_PLAN_TABLE_FULL = 2, EA_PLAN_TOO_MANY = 4 };
#define EA_PLAN_MAX_SEQS 16384
typedef struct ea_plan_step {
  const int32_t* context_lens; /* (batch,) */
  const int32_t* new_lens;     /* (batch,) */
  int32_t* page_table;         /* (batch, max_pages), rows table_stride apart, updated in place */
  const int32_t* free_pages;   /* (num_free,) */
  const int32_t* free_head;    /* (1,) first unused entry of free_pages; NULL: 0 */
  const int32_t* depths;       /* (max_tokens,) or NULL */
  int64_t* slot_map;           /* (max_tokens,) out */
  int32_t* positions;          /* (max_tokens,) out */
  int32_t* token_seq;          /* (max_tokens,) out */
  int32_t* q_start;            /* (batch + 1,) out: prefix sums of new_lens */
  int32_t* seq_lens;           /* (batch,) out: context + new */
  int32_t* next_free_head;     /* (1,) out, may not alias free_head */
  int32_t* status;             /* (1,) out */
  int64_t table_stride;
  int batch, max_pages, page_size, num_free, max_tokens;
} ea_plan_step_t;
int ea_plan_step_cuda(const ea_plan_step_t* args, void* stream);

/* Rotary positions. Pair i < rot / 2 of every q and k head of token t is turned by the angle
 * positions[axes[i]][t] * inv_freq[i] (axes NULL: axis 0; positions axis_stride apart), or by its
 * negative (inverse: the gradient of the forward call). adjacent == 0: pair i is (x[i], x[i + rot / 2]);
 * adjacent != 0: (x[2 i], x[2 i + 1]). Channels from rot on are copied. q_out (tokens, q_heads, d)
 * and k_out (tokens, kv_heads, d) are contiguous; with slot_map, k is instead written to row
 * slot_map[t] of k_cache and v copied to that row of v_cache (nothing is written at -1): slot s is
 * row s % page_size of page s / page_size, strides in elements. v and the caches are NULL without
 * slot_map. q (or k and v) may be NULL with its head count 0. Outputs may not overlap inputs.
 * d at most 1024. Angles keep 32-bit accuracy at positions of any size and frequencies up to 2^40. */
typedef struct ea_rope {
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;                /* between tokens, in elements */
  int64_t q_head_stride, k_head_stride, v_head_stride; /* between heads; channels are contiguous */
  const int32_t* positions;                            /* (num_axes, tokens) */
  int64_t axis_stride;
  const float* inv_freq; /* (rot / 2,) */
  const int32_t* axes;   /* (rot / 2,) each 0 .. num_axes - 1, or NULL */
  void *q_out, *k_out;
  const int64_t* slot_map; /* (tokens,) or NULL */
  void *k_cache, *v_cache;
  int64_t k_page_stride, k_cache_head_stride, k_row_stride;
  int64_t v_page_stride, v_cache_head_stride, v_row_stride;
  int64_t tokens, num_slots; /* num_slots: rows of the caches; slots outside 0 .. num_slots - 1 are skipped */
  int q_heads, kv_heads, d, rot, num_axes, page_size;
  int dtype, adjacent, inverse;
} ea_rope_t;
int ea_rope_cuda(const ea_rope_t* args, void* stream);

/* Attention of a step's tokens over the paged cache, which already holds their keys and values.
 * Sequence b has seq_lens[b] keys, the last q_start[b + 1] - q_start[b] of them its step's tokens.
 * Token t = q_start[b] + i sees every earlier key and, of the step's tokens, the j-th where bit j
 * of its row of tree_mask (mask_words 32-bit words, bit j % 32 of word j / 32) is set; tree_mask
 * NULL: j <= i. Key j of sequence b is row j % page_size of page page_table[b][j / page_size].
 * With w_j = 2^(alpha q . k_j) over the visible keys: out = sum w v / sum w, lse = log2 sum w (NULL: not
 * written); a row that sees no key gives 0 and -inf. Head h reads kv head h / (q_heads / kv_heads).
 * What a row does not see cannot reach its output, NaN and infinities included; an infinite value that it
 * sees with a weight that rounds to zero may give NaN. For up to 16 query rows a kv head (max_new * q_heads /
 * kv_heads) w enters sum w v as a pair of 16-bit numbers, 2^-17 off or less; for more it is rounded once to
 * the caches' type (in fp16 to within 2^-35 of the row's largest weight). sum w is 32-bit.
 * bf16 or fp16 (q, caches and out alike), d a multiple of 8 up to 128, rows on 16-byte boundaries (-9
 * otherwise).
 * max_new: the most tokens any sequence has in this step (a hint: it sizes tiles, not results). tokens *
 * q_heads, max_pages * page_size and the tiles that these allow stay below 2^31 (-1 otherwise).
 * workspace: ea_tree_attention_workspace(args) bytes, 16-byte aligned, any contents; calls that
 * may overlap need workspaces of their own. Page ids outside 0 .. num_pages - 1 and keys past the table's
 * columns are read as keys no row sees; tokens past `tokens` have no row, but still count among the step's.
 * Deterministic for equal inputs on one GPU model (no atomics).
 * Waits inside the kernels are bounded (2 s): rows whose block gave one up are NaN in out and lse, so that an error
 * shows in the results; it has never been seen outside of the test hook (ea_set_test_hooks). */
#define EA_TREE_MAX_SEQS 8192
typedef struct ea_tree_attention {
  const void* q; /* (tokens, q_heads, d) */
  int64_t q_stride, q_head_stride;
  const void *k_cache, *v_cache;
  int64_t k_page_stride, k_head_stride, k_row_stride;
  int64_t v_page_stride, v_head_stride, v_row_stride;
  const int32_t* page_table; /* (batch, max_pages), rows table_stride apart */
  int64_t table_stride;
  const int32_t* seq_lens;  /* (batch,) */
  const int32_t* q_start;   /* (batch + 1,) */
  const int32_t* tree_mask; /* (tokens, mask_words) or NULL */
  void* out;                /* (tokens, q_heads, d) contiguous */
  float* lse;               /* (tokens, q_heads) or NULL */
  void* workspace;
  int64_t tokens, num_pages;
  float alpha;
  int batch, q_heads, kv_heads, d, page_size, max_pages, mask_words, max_new, dtype;
} ea_tree_attention_t;
int64_t ea_tree_attention_workspace(const ea_tree_attention_t* args);
int ea_tree_attention_cuda(const ea_tree_attention_t* args, void* stream);

/* Logits of row r, sequence b = row_seq[r] (NULL: r), token v, in 32 bits, in this order:
 *   c = how often v occurs in history[b][prompt_lens[b] .. history_lens[b]) and among the drafted
 *       tokens on the row's path: draft_tokens[q_start[b] + j] for the set bits j of tree_mask[r]
 *       (tree_mask NULL: j <= r - q_start[b])
 *   x > 0 ? x / repetition[b] : x * repetition[b]  if c > 0 or v is in history[b][0 .. prompt_lens[b])
 *   x - frequency[b] * c;  x - presence[b] if c > 0
 *   x + bias_values[b][e] for the entries e with bias_ids[b][e] == v, in their order
 *   -inf if bit v of allowed_bits[mask_rows[r]] is clear (mask_rows NULL: r; a mask row outside
 *       0 .. num_masks - 1 allows every token)
 * rounded once to the type of logits. NULL history / repetition / frequency / presence / biases /
 * allowed_bits / draft_tokens leave their step out. Token ids outside 0 .. vocab - 1 are ignored;
 * rows with row_seq outside 0 .. batch - 1 are copied, unmasked too. out may be logits itself. At most
 * EA_LOGITS_MAX_SEQS sequences, EA_LOGITS_MAX_HISTORY history entries, EA_LOGITS_MAX_PATH drafted
 * tokens (later ones are not counted) and EA_LOGITS_MAX_BIASES biases a sequence. */
#define EA_LOGITS_MAX_HISTORY 1000000
#define EA_LOGITS_MAX_PATH 32768
#define EA_LOGITS_MAX_BIASES 2000
#define EA_LOGITS_MAX_SEQS (1 << 30)
typedef struct ea_process_logits {
  const void* logits; /* (rows, vocab), rows logits_stride elements apart */
  void* out;          /* (rows, vocab), rows out_stride apart */
  int64_t logits_stride, out_stride;
  const int32_t* row_seq;
  const int32_t* history; /* (batch, ..), rows history_stride apart */
  int64_t history_stride;
  const int32_t *history_lens, *prompt_lens; /* (batch,); prompt_lens NULL: 0 */
  const float *repetition, *frequency, *presence; /* (batch,) */
  const int32_t* bias_ids; /* (batch, num_biases), negative: unused */
  const float* bias_values;
  const int32_t* allowed_bits; /* (mask states, mask_stride words) */
  int64_t mask_stride;
  const int32_t* mask_rows;    /* (rows,) */
  const int32_t* draft_tokens; /* (rows,) */
  const int32_t* q_start;      /* (batch + 1,) */
  const int32_t* tree_mask;    /* (rows, tree_words) */
  int64_t rows;
  int vocab, batch, max_history, num_biases, num_masks, tree_words, dtype;
} ea_process_logits_t;
int ea_process_logits_cuda(const ea_process_logits_t* args, void* stream);

/* Message of the calling thread's last failed call of this header. */
const char* ea_serving_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* EXACTATTN_SERVING_H */
