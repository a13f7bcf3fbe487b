/* C ABI of the attention half of a served block, next to the experts' half of tetris_mx4.h: the residual's addition with a
 * root-mean-square norm, rotary positions, a cache of keys and values in MX4, attention over that cache.  Part of
 * libtetris_spconv2d.so; conventions, types and leading dimensions as in tetris_mx4.h.
 */
#ifndef TETRIS_ATTENTION_H_
#define TETRIS_ATTENTION_H_

#include "tetris_mx4.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------------------------------
 * s = x + residual and y = s / sqrt(mean(s^2) + eps) * weight, row by row.  d_residual NULL: s = x.  d_weight: cols floats, or
 * NULL for ones.  d_sum, NULL or rows of `type` for s rounded; d_sum may be d_residual (with ld_sum = ld_residual), nothing else overlaps.
 * The norm is of s in 32 bits, before it is rounded, also where its squares are beyond them or vanish in them.  Columns up to 2^20.
 * ---------------------------------------------------------------------------------------------- */
int tetris_rms_norm(const void* d_x, int type, int64_t rows, int cols, int64_t ldx, const void* d_residual, int64_t ld_residual,
                    const float* d_weight, float eps, void* d_sum, int64_t ld_sum, void* d_y, int64_t ldy, void* stream);

/* ------------------------------------------------------------------------------------------------
 * Rotary positions.  A head's first `dims` elements are dims / 2 pairs (u, v), which become (u cos a - v sin a, u sin a + v cos a);
 * the other head - dims are copied.  Pair i is elements i and i + dims / 2 (TETRIS_PAIR_HALVES) or 2 i and 2 i + 1
 * (TETRIS_PAIR_NEIGHBOURS).  Its angle is position * base^(-2 i / dims), the position that of the axis whose section holds i: the
 * first sections[0] pairs turn with axis 0 (time), the next sections[1] with axis 1 (height), and so on; `axes` sections add up to
 * dims / 2.  TETRIS_RATE_AXIS: every axis has all rates, pair i of a section of n the rate base^(-i' / n), i' its place in the section.
 * Angles are formed in 64 bits and are those of positions up to 2^31.
 * d_position: a row of `tokens` int32 for each axis, ld_position elements apart.  A token's heads lie one after another.
 * backward: by -a, which carries the gradient of y to x.  d_y may be d_x, with ldy = ldx.
 * Limits: head <= 1024, even dims <= head, axes 1 to 4, base positive and finite.
 * ---------------------------------------------------------------------------------------------- */
enum { TETRIS_PAIR_HALVES = 0, TETRIS_PAIR_NEIGHBOURS = 1 };
enum { TETRIS_RATE_HEAD = 0, TETRIS_RATE_AXIS = 1 };
typedef struct {
  int32_t head, dims, axes, sections[4], pairing, rate;
  double base;
} tetris_rotary;
int tetris_rotate(const tetris_rotary* r, const void* d_x, int type, int tokens, int heads, int64_t ldx, const int32_t* d_position,
                  int64_t ld_position, int backward, void* d_y, int64_t ldy, void* stream);

/* ------------------------------------------------------------------------------------------------
 * A cache of keys and values: `pages` pages of `page` tokens of kv_heads heads of `head` elements, each head's key and value an MX4
 * row (tetris_mx4.h).  d_pages is the caller's memory, pages * tetris_cache_page_bytes(kv_heads, head, page) bytes on 16, and
 * stays its own; how a page is laid out is the kernels' matter, and what has not been appended is not defined.  A slot is
 * page number * page + place in the page.  Limits: head a multiple of 32 up to 256, page a multiple of 16 up to 4096, kv_heads
 * up to 1024, fewer than 2^31 slots.  The handle belongs to the HIP device that is current when it is made.
 *
 * tetris_cache_append rounds `tokens` keys and values (rows of kv_heads * head elements) into the slots d_slot, as
 * tetris_mx4_quantize does.  The slots of one call are distinct (one named twice holds a mix of both tokens).
 * tetris_cache_read: the values that slots hold, rounded once to `type` (exact in TETRIS_BF16 and TETRIS_F32).
 * A negative slot, or one past the last page, is passed over: nothing is written for it, and it reads as zeros.
 * ---------------------------------------------------------------------------------------------- */
typedef struct tetris_cache tetris_cache;
size_t tetris_cache_page_bytes(int kv_heads, int head, int page);
int tetris_cache_create(int kv_heads, int head, int page, int64_t pages, void* d_pages, tetris_cache** out);
void tetris_cache_destroy(tetris_cache* c); /* no launch that uses it may be under way */
int tetris_cache_append(tetris_cache* c, const void* d_k, int64_t ldk, const void* d_v, int64_t ldv, int type, int tokens,
                        const int64_t* d_slot, void* stream);
int tetris_cache_read(tetris_cache* c, const int64_t* d_slot, int tokens, void* d_k, int64_t ldk, void* d_v, int64_t ldv, int type,
                      void* stream);

/* ------------------------------------------------------------------------------------------------
 * Attention over the cache.  `rows` queries (rows of heads * head elements, head h's keys and values those of kv head
 * h / (heads / kv_heads)) of `sequences` sequences: sequence s has rows d_first[s] .. d_first[s + 1] - 1, the newest tokens of
 * the d_length[s] that are cached of it, or without d_first row s alone.  Token j of a sequence lies in page d_table[s][j / page]
 * at place j % page.  Row i of n of a sequence of length L is at position p = L - n + i, sees tokens j with j <= p and, with a window,
 * j > p - window, and becomes  y = sum_j softmax_j(scale * q.k_j) v_j; a row that sees nothing becomes zeros (a score of
 * minus infinity counts as not seen).  Keys and values that a row does not see do not touch it, whatever they are.
 * most_length (up to 2^28) and most_rows: no sequence is longer, nor has more rows; what is longer counts as most_length, rows beyond most_rows are left as they
 * are, as are those of no sequence.  d_table: a row of ceil(most_length / page) page numbers for each sequence, ld_table
 * apart; a number outside of the pool stands for a page that no row sees.  The lengths, tables and offsets are read on the device: a captured
 * launch serves whatever they hold when it is replayed.
 * Products are of the cache's exact values and of q in 1, 2 or 3 bf16 parts (bf16, f16, f32: no bit is lost), summed in 32 bits, as are
 * the softmax and its sums.  Its weights enter the second product with 16 bits, for f32 with 24; where a call has many rows in bf16, with 11 (2^-11 of a weight),
 * an eighth of what the output is rounded by.  Results do not depend on the order in which anything runs.
 * Workspace is the cache's, one per stream as in tetris_mx4.h; tetris_cache_prepare makes it ahead of a graph capture, for calls of
 * these sizes or smaller sequences, most_rows and most_length with as many or fewer rows.
 * Sizes that are more than a launch has (2^24 workgroups, or for all sequences' kv heads and rows together some 2^31 times 128 tokens) are refused with
 * TETRIS_EUNSUPPORTED.
 * ---------------------------------------------------------------------------------------------- */
typedef struct {
  int32_t heads, sequences, rows, most_rows, most_length, window; /* window 0: none */
  float scale;
} tetris_attention;
int tetris_cache_prepare(tetris_cache* c, const tetris_attention* a, int type, void* stream);
int tetris_cache_attend(tetris_cache* c, const tetris_attention* a, const void* d_q, int64_t ldq, int type, const int32_t* d_first,
                        const int32_t* d_length, const int32_t* d_table, int64_t ld_table, void* d_y, int64_t ldy, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* TETRIS_ATTENTION_H_ */
