/* C ABI of the operators on compressed weights: 4-bit floating point with shared scales (MX4), products with MX4
 * weights, routing of tokens to experts, and the experts' products.  Part of libtetris_spconv2d.so; conventions as in
 * tetris_spconv2d.h: d_* is memory of the current HIP device, `stream` a hipStream_t passed as void*, every function
 * returns 0 or a TETRIS_E* code with a message in tetris_last_error(), launches are asynchronous on `stream`.
 *
 * `type` names the elements of activations, logits and outputs: TETRIS_F32, TETRIS_F16 or TETRIS_BF16.  A leading
 * dimension (`ld`) is the distance of two rows in elements.  Rows and bases need no alignment beyond their element's;
 * rows that start on 16 bytes and widths that are multiples of eight are read without a copy.
 * Outputs may not overlap inputs.  A call with no rows does nothing and succeeds.  Launches of one handle on one stream come from one
 * thread at a time (they share that stream's workspace; hipStreamPerThread is a stream of each thread).  A graph keeps the workspace of the stream
 * that its launches were captured on: on whatever stream it is replayed, it may not overlap other launches of the handle on that stream, nor
 * other graphs that were captured there with the handle.
 */
#ifndef TETRIS_MX4_H_
#define TETRIS_MX4_H_

#include "tetris_spconv2d.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { TETRIS_F32 = 0, TETRIS_F16 = 1, TETRIS_BF16 = 2 };

/* ------------------------------------------------------------------------------------------------
 * MX4 rows.  A row of `cols` values is ceil(cols / 32) blocks; a block is 16 bytes of codes (element 2i in the low half
 * of byte i) and one scale byte.  Value = code * 2^(scale - 127); codes 0..7 are 0, 0.5, 1, 1.5, 2, 3, 4, 6, 8..15 the
 * same negated; scale 255 makes the block NaN; what
 * lies beyond 32 bits' range (scales 253 and 254 have such codes; no quantised number has them) counts as infinite, and a sum with
 * one may be NaN in place of an infinity (rows are multiplied in parts, some of them zero).  Elements past `cols` in the last block are zero codes.
 *
 * tetris_mx4_quantize: the scale of a block is 2^(floor(log2 a) - 2), a its largest magnitude, and at least 2^-127; an
 * element goes to the nearest value, to the even code where two are as near, and to 6 beyond 6; a block that holds an
 * infinity or a NaN becomes NaN.  d_codes: rows x tetris_mx4_code_bytes(cols), 16-byte aligned; d_scales: rows x
 * tetris_mx4_scale_bytes(cols).
 * tetris_mx4_dequantize: the values, rounded once to `type` (exact in TETRIS_BF16 and TETRIS_F32).
 * ---------------------------------------------------------------------------------------------- */
size_t tetris_mx4_code_bytes(int cols);
size_t tetris_mx4_scale_bytes(int cols);
int tetris_mx4_quantize(const void* d_x, int type, int64_t rows, int cols, int64_t ld, uint8_t* d_codes,
                        uint8_t* d_scales, void* stream);
int tetris_mx4_dequantize(const uint8_t* d_codes, const uint8_t* d_scales, int64_t rows, int cols, void* d_y, int type,
                          int64_t ld, void* stream);

/* ------------------------------------------------------------------------------------------------
 * Weights in MX4, laid out once for the kernels: `experts` matrices of n rows and k columns.
 * tetris_mx4_create takes MX4 rows (experts * n of them, as tetris_mx4_quantize writes them), tetris_mx4_create_values
 * numbers of any type, which it quantises.  gated: the first n / 2 rows of a matrix are a gate's and the others the rows
 * it gates (tetris_experts); n is then even.  At most 1024 matrices, sides up to 2^21.  Both wait for `stream`: the arrays may be freed afterwards, and the handle
 * used on any stream.
 * ---------------------------------------------------------------------------------------------- */
typedef struct tetris_mx4 tetris_mx4;
int tetris_mx4_create(const uint8_t* d_codes, const uint8_t* d_scales, int experts, int n, int k, int gated, void* stream,
                      tetris_mx4** out);
int tetris_mx4_create_values(const void* d_w, int type, int experts, int n, int k, int64_t ld, int gated, void* stream,
                             tetris_mx4** out);
void tetris_mx4_destroy(tetris_mx4* w); /* no launch that uses it may be under way */

/* ------------------------------------------------------------------------------------------------
 * y[i] = x[i] W^T + bias for m rows x[i] of k and y[i] of n elements of `type`; d_bias: n floats or NULL.  W is one
 * matrix, not gated.  Products are exact and summed in 32 bits.  mx4_input: the rows of x are rounded to MX4 (as
 * tetris_mx4_quantize does) before the product, on the fly; large m then runs on the matrix cores' 4-bit products.
 * Workspace is the handle's, one per stream it is launched on; tetris_mx4_prepare makes it ahead, for up to m rows (of a graph capture,
 * under which a launch that would have to allocate is refused with TETRIS_EINVAL).
 * ---------------------------------------------------------------------------------------------- */
int tetris_mx4_prepare(tetris_mx4* w, int m, int type, int mx4_input, void* stream);
int tetris_mx4_linear(tetris_mx4* w, const void* d_x, int type, int m, int64_t ldx, void* d_y, int64_t ldy,
                      const float* d_bias, int mx4_input, void* stream);

/* ------------------------------------------------------------------------------------------------
 * Routing: for each of `tokens` rows of `experts` logits the `top` experts (d_index, best first) and their weights
 * (d_weight), both [tokens][top].
 *   scores  s = softmax(logits) over the row, or 1 / (1 + exp(-logit)), in 32 bits
 *   rank    s + d_bias[expert], or without a bias the logit itself, whose order is that of the scores
 *   groups  experts / groups neighbouring experts form a group; only the top_groups groups of largest rank stay, a group
 *           ranking by its best expert (TETRIS_GROUP_MAX) or by the sum of its two best s + bias (TETRIS_GROUP_TWO)
 *   choice  the `top` of largest rank; ties, of groups too, go to the lowest index
 *   weight  scale * s, with renorm scale * s / (sum of the chosen s); zero where that sum is zero
 * The bias decides the choice and enters no weight.  A logit of -inf scores zero (a row of them: all weights are zero and the
 * first experts of the groups that stay are named); a NaN ranks as -inf and its row's softmax weights are NaN.  +inf logits share a softmax's weight.
 * Limits: experts <= 1024, top <= 32 and <= experts in the groups that stay, groups <= 64 dividing experts.
 *
 * tetris_route_backward: the gradient of the weights (d_dweight, [tokens][top]) carried to the logits for the choice
 * d_index (distinct experts), which itself has no gradient, nor has the bias.  Zero for a row whose weights are zero for
 * want of scores.  Entries of d_index outside the experts are passed over.
 * ---------------------------------------------------------------------------------------------- */
enum { TETRIS_SCORE_SOFTMAX = 0, TETRIS_SCORE_SIGMOID = 1 };
enum { TETRIS_GROUP_MAX = 0, TETRIS_GROUP_TWO = 1 };
typedef struct {
  int32_t experts, top, score, groups, top_groups, group_by, renorm;
  float scale;
} tetris_router;
int tetris_route(const tetris_router* r, const void* d_logits, int type, int tokens, int64_t ld, const float* d_bias,
                 int32_t* d_index, float* d_weight, void* stream);
int tetris_route_backward(const tetris_router* r, const void* d_logits, int type, int tokens, int64_t ld,
                          const int32_t* d_index, const float* d_dweight, void* d_dlogits, int64_t ld_out, void* stream);

/* ------------------------------------------------------------------------------------------------
 * The experts' products: y[t] = sum over j of d_weight[t][j] * down_e(silu(gate_e x[t]) * up_e x[t]), e = d_index[t][j].
 * `up` is gated, experts x 2 hidden x width; `down` experts x width x hidden.  Entries of d_index outside the experts
 * add nothing (a token of nothing but such entries gets zeros).  Sums are of 32 bits and in the order of j; between the
 * products numbers are held in `type`'s precision or better, with the range of 32 bits.  Workspace: up's, as for tetris_mx4_linear;
 * tetris_experts_prepare makes it ahead.
 * ---------------------------------------------------------------------------------------------- */
int tetris_experts_prepare(tetris_mx4* up, tetris_mx4* down, int tokens, int top, int type, void* stream);
int tetris_experts(tetris_mx4* up, tetris_mx4* down, const void* d_x, int type, int tokens, int64_t ldx, int top,
                   const int32_t* d_index, const float* d_weight, void* d_y, int64_t ldy, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* TETRIS_MX4_H_ */
