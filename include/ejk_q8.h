/*
 * C ABI of the serving step around a paged KV cache held in 8 bits (sm_100a): page tables and slot maps from request
 * lengths, the cache's write and read, and ragged attention over it.  Same library, conventions, return codes, status
 * word and call attributes as ejk_rpa.h; these operators have no counterpart in the reference.
 *
 * The cache
 *   kv_pages   [num_pages, num_kv_heads, 2, page_size, head_dim]            codes, one byte each (e4m3 or int8); 2 = K, V
 *   kv_scales  [num_pages, num_kv_heads, 2, page_size / scale_block]         float32, positive and finite
 * A value is its code times the scale of its block of `scale_block` tokens.  A write makes no NaN codes; e4m3 codes that are NaN
 * (a cache that was filled otherwise) make NaN of the rows that see them, and where they are V's also of rows that the mask keeps
 * from them but not from the other keys of the same tile.  Behind a sequence's end and before the window of all its rows any bytes
 * may lie, scales included.  The page of one head is contiguous (the
 * pool of ejk_rpa_launch interleaves the heads of a token): the attention kernel fetches runs of page_size * head_dim
 * bytes, where one token of one head is 64 to 256 bytes of an 8-bit cache -- shorter than what DRAM serves well.
 *
 * Every call only enqueues work on `stream`, allocates nothing and does not synchronise.
 */
#ifndef EJK_Q8_H_
#define EJK_Q8_H_

#include "ejk_rpa.h"

#ifdef __cplusplus
extern "C" {
#endif

/* code types (ejk_q8_shape.code_dtype); EJK_RPA_E4M3 = 2 is the other */
#define EJK_Q8_I8 3

/* status bits beside EJK_RPA_ST_* */
#define EJK_Q8_ST_POOL 64u       /* the free list ran out of pages, or of room for returned ones */
#define EJK_Q8_ST_NONFINITE 128u /* a NaN or an infinity was written to the cache (as 0, or the largest code) */

typedef struct ejk_q8_shape {
  int32_t total_tokens;  /* rows of queries / keys / slots */
  int32_t max_num_seqs;  /* block_tables.shape[0] */
  int32_t pages_per_seq; /* block_tables.shape[1] */
  int32_t num_pages;
  int32_t page_size;     /* tokens; num_pages * page_size < 2^31 */
  int32_t num_q_heads;
  int32_t num_kv_heads;
  int32_t head_dim;      /* 64, 128 or 256 */
  int32_t dtype;         /* EJK_RPA_BF16 | EJK_RPA_F16: queries, out, keys, values */
  int32_t code_dtype;    /* EJK_RPA_E4M3 | EJK_Q8_I8 */
  int32_t scale_block;   /* tokens that share a scale: a power of two that divides page_size */
} ejk_q8_shape;

/* A status word for `status` of the calls below that lives as long as the library, one on each device (that of the current
 * device is given): zero at first, the caller clears it.  It can be had while a stream is being captured. */
EJK_RPA_API int ejk_q8_status_word(int32_t** word);

/* The first bytes of an attention workspace: counters that have to be zero when a workspace is used for the first time.  Every
 * call leaves them zero, one whose waits ran out (EJK_RPA_ST_TIMEOUT) included; the rest needs no initialisation. */
#define EJK_Q8_TICKET_BYTES 16384

/* Scratch that ejk_q8_attention_launch needs for this static shape on the current device (0: invalid shape), in calls with
 * these attributes (of which num_queries_per_block counts; null: without it).  One workspace serves any number of calls that are
 * ordered on the device, of any shapes that fit. */
EJK_RPA_API size_t ejk_q8_attention_workspace_bytes(const ejk_q8_shape* shape, const ejk_rpa_attrs* attrs);
/* The same without attributes. */
EJK_RPA_API size_t ejk_q8_workspace_bytes(const ejk_q8_shape* shape);

/* Ragged attention over the 8-bit cache.  Operands, masks, sinks and zero rows as ejk_rpa_launch; `attrs.q_scale` and
 * `attrs.out_scale` must be 0.  With x = softmax_scale * k_scale[j] * sum_d q[d] * k_code[j, d], soft cap and masks on
 * x, the output is sum_j softmax(x)[j] * v_scale[j] * v_code[j].
 * Accuracy, per row, with p the softmax weights and the sums over the keys that the row sees: within 2^-10 sum p |v| (2^-9 where
 * scales are no powers of two) + 2^-24 max |v| + the output's rounding, for logits of a few units.
 * Sequences with many query rows are served by tensor tiles (head_dim 64 and 128): those of num_queries_per_block tokens and more
 * where the caller gives it, otherwise those of 32 rows and more in batches with more tokens than block_tables has rows.  In a
 * table with idle rows only the hint tells a chunk of a prompt from decode rows.  Every row of `out` is written: rows of no sequence, and of
 * sequences whose offsets are refused (EJK_RPA_ST_QLEN: they decrease, or lie outside [0, total_tokens]), are zero.  Where
 * offsets decrease, sequences can claim the same rows: whose such a row is, or whether it is zero, is open. */
EJK_RPA_API int ejk_q8_attention_launch(const void* queries, const void* kv_pages, const float* kv_scales,
                                        const int32_t* context_lens, const int32_t* block_tables,
                                        const int32_t* query_start_loc, const int32_t* num_seqs, const float* softmax_aux,
                                        void* out, void* workspace, size_t workspace_bytes, int32_t* status,
                                        const ejk_q8_shape* shape, const ejk_rpa_attrs* attrs, void* stream);

/* Writes rows keys / values [total_tokens, num_kv_heads, head_dim] (rows `key_stride` / `value_stride` elements apart, a
 * multiple of 8) to the cache, in place.  slots[t] = page * page_size + offset, or negative: the row is skipped.
 * Rows of one scale block have to be neighbours in the batch, with ascending slots -- what ejk_page_tables_launch
 * gives -- and no slot may occur twice.  Per (scale block, head, K or V), with A the largest finite |x| of the new rows and
 * qmax = 448 (e4m3) or 127 (int8):
 *   s_new = the smallest power of two, not below 2^-126, with A <= qmax * s_new
 *   o     = the offset of the first new row inside the block: the rows [0, o) are kept
 *   o == 0: scale = s_new;  o > 0: scale = max(old scale, s_new), kept rows get code' = round(code * old / scale)
 *   code  = round(clamp(x / scale, -qmax, qmax)), to the nearest, ties to even; NaN is written as 0
 * With powers of two every quotient is exact, so that a code is the correctly rounded one and the result does not depend
 * on the order of execution.  Of the shape, the sequence and query-head fields are not read. */
EJK_RPA_API int ejk_q8_write_launch(const void* keys, const void* values, int64_t key_stride, int64_t value_stride,
                                    void* kv_pages, float* kv_scales, const int32_t* slots, int32_t* status,
                                    const ejk_q8_shape* shape, void* stream);

/* The rows at `slots` as 16-bit keys / values [total_tokens, num_kv_heads, head_dim]: code * scale, rounded, saturated at
 * the largest finite value; a code that is a NaN gives a NaN.  A negative slot gives zeros. */
EJK_RPA_API int ejk_q8_read_launch(const void* kv_pages, const float* kv_scales, const int32_t* slots, void* keys,
                                   void* values, int32_t* status, const ejk_q8_shape* shape, void* stream);

/* Page tables and slot maps of one step from the requests' lengths, without the host.
 *   in:     query_lens, context_lens (tokens cached before this step) [max_num_seqs]; num_seqs [1] (later rows are idle);
 *           finished [max_num_seqs] bytes or null; num_free [1]
 *   in/out: block_tables [max_num_seqs, pages_per_seq]; free_pages [capacity], a stack whose first num_free entries are free
 *   out:    new_context_lens [max_num_seqs], query_start_loc [max_num_seqs + 1], slots [total_tokens], new_num_free [1]
 * First the pages of finished rows go on top of the stack, in row and page order (such a row takes no tokens in this
 * call).  Then every row that lacks pages for its context_len + query_len tokens takes them from the top, rows in
 * order.  A row that cannot be served -- the stack is empty, the row's table too short, the batch longer than
 * total_tokens -- takes no page, keeps its context length, gets slots of -1 and sets a status bit.  Its tokens still count in
 * query_start_loc: a write skips them, and attention takes them as the LAST tokens of the old context length and returns numbers for
 * them.  Whoever lets a step go on without reading the status has to drop such rows' results (their new length is the old one).
 * slots[t] = page * page_size + offset of token t; -1 behind the last sequence.  max_num_seqs is 16384 at most.
 * No output may overlap an input other than as named above. */
EJK_RPA_API int ejk_page_tables_launch(const int32_t* query_lens, const int32_t* context_lens, int32_t* block_tables,
                                       int32_t* free_pages, const int32_t* num_free, const int32_t* num_seqs,
                                       const uint8_t* finished, int32_t* new_context_lens, int32_t* query_start_loc,
                                       int32_t* slots, int32_t* new_num_free, int32_t* status, int32_t max_num_seqs,
                                       int32_t pages_per_seq, int32_t page_size, int32_t capacity, int32_t total_tokens,
                                       void* stream);

#ifdef __cplusplus
}
#endif
#endif /* EJK_Q8_H_ */
