/*
 * operatorlib C ABI, language-model operators: a paged key-value cache with
 * the rotation applied on the way in, the attention of one new token per
 * sequence over it, and the attention of a prompt's tokens to each other.
 * Exported by liboperatorlib_lm.so, which links liboperatorlib.so (status
 * texts: operatorlib_status_string; scratch: the arena described at the top
 * of operatorlib/operatorlib_c.h).
 *
 * The conventions are operatorlib_c.h's: device pointers that the caller
 * owns, plain sizes, an opaque stream, an int hipError_t; arguments are
 * checked before any HIP call, work is enqueued on `stream` and nothing
 * synchronizes or allocates. Every pointer is to memory of the GPU that is
 * current when the function is called. Outputs must not overlap inputs.
 *
 * Index tensors (positions, slots, page tables, lengths, documents,
 * prefixes) are int32 in device memory. They are read by the kernels, so a
 * bad value cannot be reported; each function says what it does with one,
 * and none reads or writes outside the tensors it was given.
 *
 * A paged cache is two tensors, keys and values, each
 * [pages, kv_heads, page_size, head_dim], contiguous. Slot s of the cache is
 * token s % page_size of page s / page_size.
 *
 * Tensors are accessed 16 bytes at a time: those named "16-byte rows" below
 * need a 16-byte aligned base, strides that are multiples of 16 bytes, and a
 * head_dim that is a multiple of 8 (fp16) or 4 (fp32).
 *
 * The reference has none of these operators.
 */
#ifndef OPERATORLIB_LM_C_H_
#define OPERATORLIB_LM_C_H_

#include <stddef.h>
#include <stdint.h>

#include "operatorlib/operatorlib_c.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Version of this header's ABI; bumped on any incompatible change. */
#define OPERATORLIB_LM_ABI_VERSION 1
int operatorlib_lm_abi_version(void);

/*
 * Rotates the queries and keys of `tokens` tokens by their positions and
 * stores the rotated keys and the values in a paged cache.
 *
 * q [tokens, q_heads, head_dim], k and v [tokens, kv_heads, head_dim]; the
 * rows of a token are contiguous, tokens are *_token_stride elements apart
 * (the parts of one fused projection can be passed in place).
 *
 * Rotation: the first rotary_dim dims of each head are rotary_dim / 2 pairs;
 * pair i is dims (i, i + rotary_dim / 2), or (2 i, 2 i + 1) with
 * interleaved != 0, and (a, b) becomes
 *   (a cos t - b sin t, b cos t + a sin t),  t = position * frequencies[i].
 * Dims from rotary_dim on are copied. rotary_dim = 0 rotates nothing (and
 * frequencies and positions may be NULL). The angle is reduced in 64 bits:
 * exact to 1e-6 radians for any int32 position times |frequency| up to 1.
 * positions is [position_rows, tokens]; pair i uses row axes[i] (axes NULL:
 * row 0 for every pair). A pair whose axis is outside [0, position_rows) is
 * not rotated.
 *
 * q_out [tokens, q_heads, head_dim] gets the rotated queries, k_out (NULL: not
 * wanted) [tokens, kv_heads, head_dim] the rotated keys, both contiguous and
 * for every token. Token t's rotated keys and values go to slot slots[t] of
 * the cache of `pages` pages; a token whose slot is outside
 * [0, pages * page_size) is not stored (use -1 for padding), and no other
 * slot is written. Slots must differ: of two tokens with the same slot, each
 * element keeps one or the other's.
 *
 * Errors: a NULL pointer other than axes, k_out, and, with rotary_dim 0,
 * positions and frequencies; key_cache and value_cache overlapping; a size <= 0
 * (rotary_dim: < 0); rotary_dim odd or over head_dim; a stride below
 * heads * head_dim; pages * page_size over INT32_MAX; a token of more than
 * 2^31 - 2^20 - 1 elements (q, k and v); tokens over 2^24 - 8.
 * Any head_dim and alignment is accepted; 16-byte rows and a rotary_dim / 2
 * (interleaved: rotary_dim) that is a multiple of 8 (fp16) or 4 (fp32) are
 * the fast form.
 */
int operatorlib_rope_append_f16(
    const operatorlib_half_t* q, int64_t q_token_stride, const operatorlib_half_t* k,
    int64_t k_token_stride, const operatorlib_half_t* v, int64_t v_token_stride,
    const int32_t* positions, int position_rows, const int32_t* axes, const float* frequencies,
    const int32_t* slots, operatorlib_half_t* q_out, operatorlib_half_t* k_out,
    operatorlib_half_t* key_cache, operatorlib_half_t* value_cache, int tokens, int q_heads,
    int kv_heads, int head_dim, int rotary_dim, int interleaved, int pages, int page_size,
    void* stream);
int operatorlib_rope_append_f32(
    const float* q, int64_t q_token_stride, const float* k, int64_t k_token_stride, const float* v,
    int64_t v_token_stride, const int32_t* positions, int position_rows, const int32_t* axes,
    const float* frequencies, const int32_t* slots, float* q_out, float* k_out, float* key_cache,
    float* value_cache, int tokens, int q_heads, int kv_heads, int head_dim, int rotary_dim,
    int interleaved, int pages, int page_size, void* stream);

/*
 * Attention of one new token per sequence over a paged cache.
 *
 * q [batch, q_heads, head_dim] (sequences q_stride elements apart), cache as
 * above, page_table [batch, max_pages] (rows table_stride elements apart):
 * token j of sequence b is token j % page_size of page
 * page_table[b][j / page_size]. The sequence has n = lengths[b] tokens, the
 * new one included (it is the last). Query head h reads key head
 * h / (q_heads / kv_heads).
 *   s_j = scale * (q . k_j);  softcap > 0: s_j = softcap * tanh(s_j / softcap);
 *   slopes [q_heads], or NULL: s_j -= slopes[h] * (n - 1 - j);
 *   output = sum_j softmax(s)_j v_j over j in [max(0, n - window), n)
 *   (window 0: all j < n); output [batch, q_heads, head_dim] contiguous, fp32
 *   arithmetic, one rounding to the output's type; the fp16 form rounds the
 *   probabilities to fp16 for the product with v.
 * n below 0 counts as 0, n over max_pages * page_size as that; a sequence
 * with no token gives zeros. Tokens on a page outside [0, pages) are left out
 * as if masked. What cache rows outside a sequence's window hold (infinities
 * and NaN too) has no effect, and page_table entries past its last token are
 * not read.
 *
 * Scratch (the arena, or the *_ws forms' workspace): partial results where
 * the grid splits a sequence; the query depends on the sizes only.
 *
 * Errors: a NULL pointer other than slopes; a size <= 0; q_heads not a
 * multiple of kv_heads; head_dim over 128; window < 0; scale outside
 * [2^-100, 2^100]; softcap not 0 and softcap or scale / softcap outside of that;
 * q, cache and output not 16-byte rows; q_stride below q_heads * head_dim,
 * table_stride below max_pages; pages * kv_heads * page_size over 2^32 - 1;
 * max_pages * page_size over INT32_MAX - 1024; batch * q_heads over INT32_MAX,
 * or over 2^31 blocks of 64 keys in batch * kv_heads * max_pages * page_size;
 * *_ws: a workspace smaller than the query's answer, NULL, or not 256-byte
 * aligned. The queries return 0 for invalid sizes.
 */
size_t operatorlib_paged_attention_f16_workspace_size(int batch, int q_heads, int kv_heads,
                                                      int head_dim, int page_size, int max_pages);
int operatorlib_paged_attention_f16_ws(
    const operatorlib_half_t* q, int64_t q_stride, const operatorlib_half_t* key_cache,
    const operatorlib_half_t* value_cache, const int32_t* page_table, int64_t table_stride,
    const int32_t* lengths, const float* slopes, operatorlib_half_t* output, int batch, int q_heads,
    int kv_heads, int head_dim, int pages, int page_size, int max_pages, float scale, int window,
    float softcap, void* workspace, size_t workspace_bytes, void* stream);
int operatorlib_paged_attention_f16(
    const operatorlib_half_t* q, int64_t q_stride, const operatorlib_half_t* key_cache,
    const operatorlib_half_t* value_cache, const int32_t* page_table, int64_t table_stride,
    const int32_t* lengths, const float* slopes, operatorlib_half_t* output, int batch, int q_heads,
    int kv_heads, int head_dim, int pages, int page_size, int max_pages, float scale, int window,
    float softcap, void* stream);
size_t operatorlib_paged_attention_f32_workspace_size(int batch, int q_heads, int kv_heads,
                                                      int head_dim, int page_size, int max_pages);
int operatorlib_paged_attention_f32_ws(
    const float* q, int64_t q_stride, const float* key_cache, const float* value_cache,
    const int32_t* page_table, int64_t table_stride, const int32_t* lengths, const float* slopes,
    float* output, int batch, int q_heads, int kv_heads, int head_dim, int pages, int page_size,
    int max_pages, float scale, int window, float softcap, void* workspace, size_t workspace_bytes,
    void* stream);
int operatorlib_paged_attention_f32(
    const float* q, int64_t q_stride, const float* key_cache, const float* value_cache,
    const int32_t* page_table, int64_t table_stride, const int32_t* lengths, const float* slopes,
    float* output, int batch, int q_heads, int kv_heads, int head_dim, int pages, int page_size,
    int max_pages, float scale, int window, float softcap, void* stream);

/* Element strides of a [batch, heads, sequence, head_dim] tensor whose
 * head_dim is contiguous. */
typedef struct {
  int64_t batch;
  int64_t head;
  int64_t token;
} operatorlib_strides_t;

/*
 * Attention of a prompt's tokens to each other, with the masks and score
 * rules of language models.
 *
 * q and output [batch, q_heads, sequence, head_dim], k and v [batch, kv_heads,
 * sequence, head_dim], strided ("16-byte rows"). Query head h reads key head
 * h / (q_heads / kv_heads).
 *   s_ij = scale * (q_i . k_j);  softcap > 0: softcap * tanh(s_ij / softcap);
 *   slopes [q_heads], or NULL: s_ij -= slopes[h] * |i - j|;
 *   output_i = sum_j softmax(s_i)_j v_j over the visible j.
 * Key j is visible to query i of batch row b if
 *   documents [batch, sequence] is NULL, or documents[b][i] is >= 0 and equal
 *   to documents[b][j]; and
 *   j < prefixes[b] (prefixes [batch] not NULL), or
 *   (causal == 0 or j <= i) and (window == 0 or |i - j| < window).
 * A query that sees no key gives zeros. What masked keys and values hold
 * (infinities and NaN too) has no effect on the queries that do not see them.
 * fp32 arithmetic, one rounding to the output's type; the fp16 form rounds
 * the probabilities to fp16 for the product with v.
 *
 * Errors: a NULL pointer other than slopes, documents, prefixes; a size <= 0;
 * q_heads not a multiple of kv_heads; head_dim over 128; window < 0; scale
 * outside [2^-100, 2^100]; softcap not 0 and softcap or scale / softcap outside of
 * that; tensors not 16-byte rows; a token stride below head_dim, or a negative
 * stride; 64 tokens or a whole head of a tensor spanning 2^31 bytes or more;
 * sequence over 2^20; batch * q_heads * blocks of 32 queries over 2^24 - 8.
 * (q, k and v may repeat rows, with batch and head strides of 0; the rows of
 * output must be apart, which is not checked.)
 */
int operatorlib_masked_attention_f16(
    const operatorlib_half_t* q, operatorlib_strides_t q_strides, const operatorlib_half_t* k,
    operatorlib_strides_t k_strides, const operatorlib_half_t* v, operatorlib_strides_t v_strides,
    const float* slopes, const int32_t* documents, const int32_t* prefixes,
    operatorlib_half_t* output, operatorlib_strides_t output_strides, int batch, int q_heads,
    int kv_heads, int sequence, int head_dim, float scale, int causal, int window, float softcap,
    void* stream);
int operatorlib_masked_attention_f32(
    const float* q, operatorlib_strides_t q_strides, const float* k,
    operatorlib_strides_t k_strides, const float* v, operatorlib_strides_t v_strides,
    const float* slopes, const int32_t* documents, const int32_t* prefixes, float* output,
    operatorlib_strides_t output_strides, int batch, int q_heads, int kv_heads, int sequence,
    int head_dim, float scale, int causal, int window, float softcap, void* stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* OPERATORLIB_LM_C_H_ */
