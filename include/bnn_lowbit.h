/* bnn_lowbit.h - 4-bit linear layers and the block-scaled key/value cache
 * with the attention that reads it: the low-bit operators of language-model
 * decoding beside the binary layers of bnn_b200.h. No reference counterpart
 * (Sboyle132/BNNs_to_C runs one convolutional network).
 *
 * The manner is that of bnn_bconv_layer_*: an opaque handle is created once
 * on a device and owns its device memory; the calls on it take device
 * pointers and a stream (cudaStream_t as void*, NULL = the legacy default
 * stream), enqueue, and return without synchronising; status codes and
 * bnn_last_error as in bnn_b200.h. The handle's device is made current for
 * the call and the caller's device restored. No call but the create and
 * destroy ones allocates, so all others can be captured into a graph (whose
 * last replay a handle has to outlive). A
 * handle may be used from several host threads and streams; calls that
 * overlap must not write what another one reads (positions of a cache,
 * outputs, the workspace of an attention).
 *
 * device = -1 makes a handle without device memory, for a machine without
 * a GPU: it answers sizes and checks arguments, and every call that would
 * compute returns BNN_ERR_CUDA after its checks.
 *
 * Real values are 16-bit: `type` is BNN_BF16 or BNN_FP16, chosen when a
 * handle is created. Sums, softmax statistics and scales of sums are 32-bit
 * floats.
 */
#ifndef BNN_LOWBIT_H
#define BNN_LOWBIT_H
#include <stddef.h>
#include <stdint.h>
#include "bnn_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { BNN_BF16 = 0, BNN_FP16 = 1 };

/* ---------------- 4-bit linear layer ----------------
 * y[m][o] = bias[o] + sum_i x[m][i] * (q[o][i] - z[o][i / group]) * s[o][i / group]
 * q: codes 0..15, two a byte, the even i in the low half: [n_out][ceil(n_in / 2)].
 * s: scales in the layer's type, [n_out][ceil(n_in / group)]; the last group
 *    may be cut short. z: zero points 0..15, uint8 of the same shape; NULL = 8.
 * bias: float32 [n_out]; NULL = none. group: a multiple of 32.
 * The arrays are host or device memory (of `device`); they are laid out anew
 * for the kernels and not needed afterwards. Arrays that another stream is
 * still writing must be complete before the call. */
typedef struct bnn_q4_layer bnn_q4_layer;
int bnn_q4_layer_create(int device, int n_in, int n_out, int group, int type,
                        const uint8_t *codes, const void *scales,
                        const uint8_t *zeros, const float *bias,
                        bnn_q4_layer **out);

/* rows (0 .. 2^19) vectors: x [rows] at a distance of x_stride elements
 * (>= n_in) -> y [rows] at y_stride (>= n_out), both in the layer's type, any
 * alignment of the type. x and y must not overlap. Up to 8 rows, and up to 16
 * in a layer of fewer than 2^23 weights (n_out rounded up to a multiple of 16
 * times n_in to one of 64), the codes are multiplied exactly and a group's
 * scale is applied to its 32-bit sum (finite for |x| below 2^112); else each
 * weight (q - z) * s is rounded to the type first (tensor memory operands),
 * which adds half a step of the type to each product. So a row's result
 * depends, within that, on how many rows share the call. A layer with a weight
 * that would round to an infinity of the type is multiplied in the first way
 * with any number of rows. */
int bnn_q4_layer_run(const bnn_q4_layer *L, const void *d_x, int64_t x_stride,
                     int rows, void *d_y, int64_t y_stride, void *stream);
void bnn_q4_layer_destroy(bnn_q4_layer *L);

/* Number of CTAs of that kernel whose bounded wait (mbarriers of its TMA /
 * tcgen05 pipeline) gave up on `device` since the library was loaded: the
 * counterpart of bnn_device_error. Expected to stay 0; another number means
 * that some output of a layer is not to be trusted. */
int bnn_q4_device_error(int device, unsigned int *wait_timeouts);

/* ---------------- block-scaled key/value cache ----------------
 * `pages` pages of page_tokens (16, 32, 64, 128 or 256) tokens. A token has
 * kv_heads keys and as many values of head_dim numbers (a multiple of 8, at
 * most 256), kept in `bits` = 8 or 4 bits with one scale for each `group`
 * neighbouring numbers (32, 64, 128, or head_dim for one scale per head;
 * 0 = head_dim; the last group may be cut short):
 *   scale = bf16(max |x| / top), top = 127 (8 bits) or 7 (4 bits)
 *   code  = x / scale rounded to the nearest (even on a tie), held to
 *           [-top, top]; 0 where the scale is 0
 *   value = code * scale
 * bf16() rounds to the nearest, even on a tie. A group that holds an
 * infinity or a NaN reads back as NaN throughout. A new cache reads back
 * zeros. */
typedef struct bnn_kv_cache bnn_kv_cache;
int bnn_kv_cache_create(int device, int pages, int page_tokens, int kv_heads,
                        int head_dim, int bits, int group, int type,
                        bnn_kv_cache **out);
void bnn_kv_cache_destroy(bnn_kv_cache *c);
size_t bnn_kv_cache_bytes(const bnn_kv_cache *c); /* device memory it holds */

/* Which tokens a write or a read is about. Sequence b's position p lies in
 * page d_table[b * table_pages + p / page_tokens] at p % page_tokens.
 * Row t of the given n_tokens belongs to the sequence b with
 * d_offsets[b] <= t < d_offsets[b + 1] (n_seqs + 1 ascending numbers) and
 * stands at position d_start[b] + t - d_offsets[b]; with d_offsets = NULL
 * row t is one token of sequence t (n_tokens = n_seqs). All arrays are int32
 * device memory. Rows before d_offsets[0] or from d_offsets[n_seqs] on are
 * left alone: not stored, not written by a read. So are positions that have
 * no page: p < 0, p / page_tokens >= table_pages, or an entry of the table
 * outside 0 .. pages - 1 (-1 marks a page that is not there). One write must
 * not name a position of a page twice (two sequences writing into a page
 * they share): which of the two is kept, code by code, is not defined. */

/* Quantise keys and values as they are stored: k and v in the cache's type,
 * row t and head h at k + t * k_token + h * k_head (elements, below 2^31; the
 * head_dim numbers of a head are contiguous). n_tokens: at most 2^30. */
int bnn_kv_cache_write(bnn_kv_cache *c, const void *d_k, int64_t k_token,
                       int64_t k_head, const void *d_v, int64_t v_token,
                       int64_t v_head, int n_tokens, int n_seqs,
                       const int32_t *d_table, int table_pages,
                       const int32_t *d_start, const int32_t *d_offsets,
                       void *stream);

/* The values that such tokens have in the cache, rounded to its type. Strides
 * that put two heads of an output over one another are refused. */
int bnn_kv_cache_read(const bnn_kv_cache *c, void *d_k, int64_t k_token,
                      int64_t k_head, void *d_v, int64_t v_token,
                      int64_t v_head, int n_tokens, int n_seqs,
                      const int32_t *d_table, int table_pages,
                      const int32_t *d_start, const int32_t *d_offsets,
                      void *stream);

/* Attention of one query token per sequence over the cache:
 *   out[b][i] = sum_t softmax_t(scale * q[b][i] . key_t) * value_t
 * for query heads i of kv head i / (q_heads / kv_heads), over the positions
 * 0 .. d_lengths[b] - 1 of sequence b, behind the positions
 * 0 .. prefix_tokens - 1 of a prefix that all sequences share, whose pages
 * are d_prefix[0 ..] (prefix_tokens = 0: none). The prefix is read once for
 * the whole batch, not once per sequence. Positions without a page are not
 * there (see above), a negative length counts as 0. A row that sees no
 * position gets zeros, and a log-sum of -infinity. A NaN in a key, value or
 * query (in a query an infinity, too) makes NaN of what depends on it, and of
 * nothing else.
 * Scores, their maximum and sum, and the sums of values are 32-bit. A weight
 * times the scale of a value is rounded to 11 bits: a term of the sum is off by
 * 2^-11 of itself, or, where it is less than 2^-22 of the largest such product
 * of the row in the scale group, by 2^-33 of that product for each step of its
 * code. Keys of 2^100 and more make scores that are not finite.
 * q and out: the cache's type, sequence b and head i at
 * q + b * q_seq + i * q_head; they must not overlap (strides of out that put
 * two heads over one another are refused). d_lse, unless NULL:
 * float32 [n_seqs][q_heads], the natural logarithm of
 * sum_t exp(scale * q . key_t).
 * d_work: bnn_kv_attend_work(...) bytes of device memory, 16-byte aligned,
 * with any content, for this call alone until it has run: two calls (or two
 * captured graphs) that may overlap need one each. q_heads is a multiple of
 * kv_heads; n_seqs <= 16384. */
size_t bnn_kv_attend_work(const bnn_kv_cache *c, int n_seqs, int q_heads,
                          int prefix_tokens);
int bnn_kv_attend(const bnn_kv_cache *c, const void *d_q, int64_t q_seq,
                  int64_t q_head, int n_seqs, int q_heads,
                  const int32_t *d_lengths, const int32_t *d_table,
                  int table_pages, const int32_t *d_prefix, int prefix_pages,
                  int prefix_tokens, float scale, void *d_out, int64_t o_seq,
                  int64_t o_head, float *d_lse, void *d_work,
                  size_t work_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif
