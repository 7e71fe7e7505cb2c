/*
 * phyai_layer.h - C ABI of the kernels that surround attention in a decoder layer on MI355X (gfx950): the fp8 linear whose
 * weights have one scale per block of 128 x 128, the norms of query and key heads with the position rotation and the write
 * into a paged cache, and attention of new tokens over the cache's pages.  Same library, same rules as phyai_fp8.h: device
 * pointers, sizes and a HIP stream (`void*`); work is enqueued on that stream of the current device; nothing is allocated
 * and nothing synchronises, so every call can be recorded into a HIP graph.  Return value 0, or a negative PHYAI_FP8_E*
 * code (phyai_fp8.h) with the message in phyai_layer_last_error() of the calling thread.
 */
#ifndef PHYAI_LAYER_H
#define PHYAI_LAYER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PHYAI_LAYER_ABI_VERSION 1

int phyai_layer_abi_version(void);
const char *phyai_layer_last_error(void);

/*
 * Activations with one scale per 128 elements of a row: for block g of row m
 *     scale = max(amax |x|, 1e-12) / 448   (fp32),     codes = e4m3fn(x / scale)   (round to nearest even),
 * the last block of a row may be shorter.  x: [M, K] bf16, row stride ldx (elements, a multiple of 8), 16-byte aligned;
 * xq: [M, K] bytes, dense; the scale of block g of row m goes to x_scale[m * xs_row + g * xs_block].  K % 8 == 0.
 */
int phyai_layer_block_quant(const void *x, int64_t ldx, int64_t M, int64_t K, void *xq, float *x_scale, int64_t xs_row,
                            int64_t xs_block, void *stream);

/*
 * out[m, n] = bf16(sum_g x_scale[m, g] * w_scale[n / 128, g] * (sum over block g of xq[m, k] * w[n, k]) + bias[n]).
 * w: [N, K] e4m3fn bytes, dense, 16-byte aligned; w_scale: [ceil(N / 128), ceil(K / 128)] fp32, dense; x_scale as above
 * (xs_block = 0: one scale per row); bias: [N] bf16 or NULL; out: [M, N] bf16, row stride ldo (a multiple of 4), 8-byte
 * aligned.  N % 16 == 0 and K % 16 == 0.  Products of one block are summed by the matrix units (of eight neighbouring
 * k, what lies more than 13 bits below the largest product is cut off by the hardware), blocks in fp32.  out must not
 * overlap xq.
 */
int phyai_layer_block_gemm(const void *xq, const float *x_scale, int64_t xs_row, int64_t xs_block, const void *w,
                           const float *w_scale, const void *bias, void *out, int64_t ldo, int64_t M, int64_t N, int64_t K,
                           void *stream);

/*
 * Both as one call.  Few token rows: one kernel, no workspace (phyai_layer_block_linear_workspace_bytes() says 0).
 * out must not overlap x there, since some rows are read while others are written.
 * Otherwise codes and scales go through the workspace, behind its first PHYAI_FP8_WORKSPACE_HEADER_BYTES (which this
 * call leaves alone); 256-byte aligned, not shared by calls that may overlap.
 */
size_t phyai_layer_block_linear_workspace_bytes(int64_t M, int64_t N, int64_t K);
int phyai_layer_block_linear(const void *x, int64_t ldx, const void *w, const float *w_scale, const void *bias, void *out,
                             int64_t ldo, int64_t M, int64_t N, int64_t K, void *workspace, size_t workspace_bytes, void *stream);

/* Types of query, key and value elements. */
enum { PHYAI_LAYER_BF16 = 0, PHYAI_LAYER_F16 = 1 };

/*
 * Query and key heads of a fused projection normed and rotated, keys and values written into a paged cache, in one pass.
 * qkv: [T, (heads + 2 kv_heads) * head_dim] = q | k | v, row stride ld.  For a query or key head x of the token t:
 *     n = x * rsqrt(mean(x^2) + eps) * w   (w + 1 with gemma != 0; weights NULL: n = x),
 * then its first rot elements are turned by the angles of row positions[t] of cos_sin ([table_rows, rot] fp32: rot / 2
 * cosines, then rot / 2 sines), pair i being elements (i, i + rot / 2), or (2 i, 2 i + 1) with interleaved != 0; fp32
 * throughout, one rounding.  A position outside the table turns those elements of its token's query and key into NaNs.
 * q_out: [T, heads, head_dim].  With k_out ([T, kv_heads, head_dim]) keys go there and values nowhere; with k_out NULL keys
 * and values go to k_pages / v_pages (strides in elements: page, token, head): token t to token slots[t] % page_size of
 * page slots[t] / page_size.  A slot outside [0, n_pages * page_size) is not written (padding); slots must differ, and
 * so must the places that the strides give them.
 * Limits: rot and head_dim multiples of 8, rot <= head_dim <= 512; strides multiples of 8; pointers 16-byte aligned.
 */
int phyai_layer_head_rope(const void *qkv, int64_t ld, const void *q_weight, const void *k_weight, const float *cos_sin,
                          int64_t table_rows, const int64_t *positions, void *q_out, void *k_out, void *k_pages, void *v_pages,
                          const int64_t *k_strides, const int64_t *v_strides, const int64_t *slots, int64_t n_pages,
                          int64_t page_size, int64_t T, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rot, float eps,
                          int gemma, int interleaved, int type, void *stream);

/*
 * Attention of new tokens over a paged cache.  Sequence b has the tokens q_offsets[b] .. q_offsets[b + 1] - 1 of q ([T,
 * heads, head_dim], strides in elements) and kv_lens[b] keys, its new tokens' among them: new token i stands at position
 * p = kv_lens[b] - (q_offsets[b + 1] - q_offsets[b]) + i and sees the keys j < kv_lens[b] with j <= p (causal) and j > p -
 * window (window > 0).  out[t, h] = sum_j softmax_j(scale * q.k_j) v_j with key head h / (heads / kv_heads), zero if it
 * sees nothing and NaN if it sees only scores of -inf; out: [T, heads, head_dim] dense.  Key j lies in token j % page_size of
 * page page_table[b, j / page_size] (table_stride between its rows; 0: one row for all).  Rows outside every sequence are left
 * as they are; keys beyond the table's width do not exist (where the tokens stand goes by kv_lens all the same); a page number
 * outside [0, n_pages) makes the rows that see its keys NaN.  K and V have the same strides (elements: page, token, head).
 * out may be q, token for token and head for head; it must not overlap it otherwise.
 * Sums, maxima and products' sums are fp32; probabilities are rounded to the element type for the second product.
 * Limits: head_dim a multiple of 8 up to 256; strides multiples of 8; pointers 16-byte aligned; scale and scale * log2(e)
 * positive and finite; T * heads and page_table's width * page_size below 2^30.
 * Workspace as for phyai_layer_block_linear; max_kv: table width * page_size.
 */
size_t phyai_layer_paged_attention_workspace_bytes(int64_t T, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                   int64_t max_kv);
int phyai_layer_paged_attention(const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *k_pages, const void *v_pages,
                                const int64_t *kv_strides, int64_t n_pages, int64_t page_size, const int32_t *page_table,
                                int64_t table_stride, int64_t table_width, const int32_t *q_offsets, const int32_t *kv_lens, void *out,
                                int64_t T, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, float scale, int causal,
                                int64_t window, int type, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* PHYAI_LAYER_H */
