/*
 * hipvoc_ops.h -- operators of ONE TOKEN STEP of the token models next to the vocoder, in libhipvoc.
 *
 * The codes that hipvoc.h turns into sound are written by two autoregressive models (the talker and the code predictor,
 * src/worker/candle_qwen3.rs, src/worker/talker.rs, src/worker/code_predictor_candle.rs of the reference).  Their weights
 * and caches are read once per token, so a step is bound by memory and by launches.  These are the operators such a step
 * needs besides its rotation: a paged key/value cache that can be held in 8 bits, the attention that reads it, the norm
 * with the residual's addition (and 8-bit rows), and products with 4-bit weights.
 *
 * Conventions are hipvoc.h's: opaque handle, int 0 / negative HIPVOC_E_* codes, text in hipvoc_last_error(h), no
 * exception or abort across the boundary, released with hipvoc_free().  Different from hipvoc.h: calls on one handle may
 * come from several threads at once (a handle keeps no workspace; the text is that of its last failure, whichever
 * thread's), and every call names the stream it is enqueued on (`stream`: a hipStream_t of the handle's device, NULL = the
 * null stream), since these operators are parts of the caller's own step.  All tensors are DEVICE memory of the handle's
 * device; they are read and written when the stream gets there.  No call allocates, synchronises (but for hipvoc_ops_sync /
 * hipvoc_sync) or changes the calling thread's current device, so all of them can be captured into a HIP graph (which must
 * not outlive the handle: the kernels report into it); every kernel writes all it reads back, so two graphs share nothing
 * that they are not given both.  A call whose threads do not count in 32 bits is refused, and so are more than 2^28 rows of a
 * cache call, 65535 sequences, 1024 key heads, 16384 query heads, 2^24 rows of weights or 2^20 columns.
 *
 * Deferred errors: what only the device sees (a page number, a length or an offset out of range) is never followed out of
 * bounds.  The kernel records it in the handle, leaves such a row of the cache unwritten, fills such a row of an output
 * with NaN, and the next hipvoc_ops_sync / hipvoc_sync returns HIPVOC_E_CODE and clears the record.  The record is the handle's: a
 * sync reports what any stream's calls raised until then, once.  A caller that has to tell streams or threads apart opens a handle
 * for each (they hold 256 bytes of device memory).
 *
 * Types: "act" is the type of the step's own vectors, one of F32, F16, BF16.  Pointers to vectors are 16-byte aligned and
 * strides are counted in elements of their tensor.  Every sum, maximum, softmax statistic and scale is kept in 32 bits.
 */
#ifndef HIPVOC_OPS_H
#define HIPVOC_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "hipvoc.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HIPVOC_T_F32 0
#define HIPVOC_T_F16 1
#define HIPVOC_T_BF16 2
#define HIPVOC_T_INT8 3     /* code * scale, codes -127 .. 127, scale = max|x| * (1/127), the reciprocal a 32-bit number */
#define HIPVOC_T_E4M3 4     /* code * scale, 8-bit floats (4 exponent, 3 mantissa bits, largest 448, no infinities), scale = max|x| * (1/448) */

/* A handle for the operators below on one device; NULL on failure (text in hipvoc_last_error(NULL)).  The vocoder and
 * encoder entry points refuse it. */
void *hipvoc_ops_open(int device_id);

/* Waits for `stream` (hipvoc_sync(h): for the whole device) and returns the handle's deferred error, if any, clearing it.  Callers
 * that wait for different streams do not wait for each other. */
int hipvoc_ops_sync(void *h, void *stream);

/*
 * A paged key/value cache: `n_pages` pages of `page` tokens (a power of two, 8 .. 1024), each holding for every key head
 * (kv_heads of them) the rows of its tokens, head_dim (64 or 128) values long:
 *   k, v               [n_pages][kv_heads][page][head_dim], page p at p * page_stride elements (>= kv_heads*page*head_dim,
 *                      a multiple of 16 bytes), so K and V may be halves of one allocation
 *   k_scale, v_scale   [n_pages][kv_heads][page] f32, for INT8 / E4M3 only (NULL otherwise)
 * dtype: the act type (kept as it is), INT8 or E4M3.  Values may lie past 2^31 elements.
 */
typedef struct {
    void *k, *v;
    float *k_scale, *v_scale;
    int64_t page_stride;
    int32_t n_pages, kv_heads, page, head_dim, dtype;
} hipvoc_kv_cache;

/* The tokens of a call in the cache: a batch of n_seqs sequences, sequence b's rows being rows cu[b] .. cu[b+1]-1 of the
 * call's tensors and standing at its positions first[b], first[b]+1, ...; position p lives in page table[b*table_stride +
 * p/page], place p%page.  cu [n_seqs+1] is ascending and starts at 0 (rows at or behind cu[n_seqs] are padding: nothing is
 * written for them, and nothing that they hold is used; the call's tensors have n_rows rows, those among them).  table_width:
 * pages listed per sequence.  All int32, device memory. */
typedef struct {
    const int32_t *table, *cu, *first;
    int64_t table_stride;
    int32_t table_width, n_seqs;
} hipvoc_kv_rows;

/* Writes n_rows new tokens' keys and values (act type `dtype`; row i of k at k + i*k_stride, [kv_heads][head_dim]) into the
 * cache.  8-bit types: one scale per token and head, code = x / scale rounded to nearest, ties to even (the quotient itself
 * rounded to 32 bits first); a row of zeros has scale 0; a row that holds an infinity or NaN reads back as NaN.
 * A page that is written belongs to ONE sequence (shared prefix pages are for reading). */
int hipvoc_kv_write(void *h, const hipvoc_kv_cache *cache, const void *k, const void *v, int64_t k_stride, int64_t v_stride,
                    int dtype, const hipvoc_kv_rows *rows, int n_rows, void *stream);

/* Reads n_rows tokens back: code * scale in 32 bits, rounded once to act type `dtype`.  A cache of an act type is read in
 * that type. */
int hipvoc_kv_read(void *h, const hipvoc_kv_cache *cache, void *k, void *v, int64_t k_stride, int64_t v_stride, int dtype,
                   const hipvoc_kv_rows *rows, int n_rows, void *stream);

/*
 * Attention of one new token per sequence over its cached tokens: with n = lens[b] tokens in the cache (the new one among
 * them) and query head i reading key head i / (n_heads / kv_heads),
 *   out[b][i] = sum_t p_t v_t,   p = softmax_t(scale * q[b][i] . k_t),   lse[b][i] = log sum_t exp(scale * q . k_t)
 * over the positions max(0, n - window) <= t < n (window 0: all).  n = 0: out is 0 and lse -infinity.
 * q, out: act type, row b at b*q_stride / b*out_stride, [n_heads][head_dim]; lse [n_seqs][n_heads] f32 or NULL.  out may be q
 * itself (same stride); else it overlaps no input.
 * max_len: no lens[b] is larger (a larger one is a deferred error); the host cuts the length into parts by it, so a
 * tight bound costs least.  At most table_width * page.
 * Where act has 16 bits the weights p enter the product with V as the sum of two f16 (an f16 cache) or two bf16 (any other), so an
 * infinity among the values that are seen gives NaN (in an F32 cache it stays one); scores, sums and the product itself are in
 * 32 bits.
 * How a sequence is cut, and with it the order of its sums, depends on all lengths of the call; the same call gives the same bits.
 * workspace: hipvoc_attention_workspace() bytes (it may be 0), 16-byte aligned, not used by another call in flight.
 */
size_t hipvoc_attention_workspace(const hipvoc_kv_cache *cache, int n_heads, int n_seqs, int max_len, int window);
int hipvoc_attention(void *h, const hipvoc_kv_cache *cache, const void *q, int64_t q_stride, void *out, int64_t out_stride,
                     float *lse, int dtype, int n_heads, const int32_t *table, int64_t table_stride, int table_width,
                     const int32_t *lens, int n_seqs, int max_len, int window, float scale, void *workspace,
                     size_t workspace_bytes, void *stream);

/*
 * s = x + residual (in 32 bits; residual NULL: s = x), y = s / sqrt(mean(s^2) + eps) * weight, per row of `cols` values.
 * eps may be 0: a row of zeros (or whose mean square is 0 in 32 bits) then has no norm, and its zeros give NaN (8 bits: scale NaN).
 * sum (act type; NULL: not wanted, and without a residual it has to be NULL) gets s rounded; y is made from s before that
 * rounding.  sum may be x or residual themselves (same stride); y overlaps no input and not sum.
 * out_dtype = dtype: y [rows][cols] in the act type.  INT8 / E4M3: y holds codes (bytes) and scales [rows][cols/group] f32,
 * one per `group` columns (32, 64, 128, or 0 for one per row; group divides cols), code and scale as in the cache.
 * Fewer than 2^22 rows; any cols from 1 to 2^20, any alignment.
 */
int hipvoc_add_rmsnorm(void *h, const void *x, int64_t x_stride, const void *residual, int64_t residual_stride,
                       const void *weight, void *sum, int64_t sum_stride, void *y, int64_t y_stride, float *scales,
                       int dtype, int out_dtype, int group, float eps, int rows, int cols, void *stream);

/*
 * y[m][n] = sum_k x[m][k] * w[n][k] for a few rows m, w in 4 bits:
 *   codes  [n_out][n_in/2] bytes, code k in the low half of byte k/2 for even k, the high half for odd k; row-major, dense
 *   scales [n_out][n_in/group] f16; mins the same or NULL; group 32, 64 or 128, a divisor of n_in
 *   w = scale * (code - 8), or with mins: w = scale * code + min
 * x: row m at m*x_stride, act type, or INT8 with x_scale [n_rows][x_groups] f32 (x_groups = n_in/group, or 1 for one
 * scale per row).  y: act type y_dtype at m*y_stride; for x of an act type y_dtype is that type.
 * Every product is exact; sums of a group, and of groups, are kept in 32 bits (8-bit rows: a group's sum is an integer).
 * Codes enter with 16 added that is taken off the sum, so a row of x that holds an infinity or NaN gives NaN, and one whose
 * sum of |x| * scale is within a factor of 31 of the largest 32-bit number may.
 * Bits of a 32-bit x under 2^-133 count as 0 (values under 2^-109 lose accuracy).  y overlaps no input.
 * Up to 65535 rows: the weights are read once for every 16.  x_stride is a multiple of 16 bytes.
 */
int hipvoc_q4_matvec(void *h, const uint8_t *codes, const void *scales, const void *mins, int n_out, int n_in, int group,
                     const void *x, int64_t x_stride, int x_dtype, const float *x_scale, int x_groups, void *y,
                     int64_t y_stride, int y_dtype, int n_rows, void *stream);

#ifdef __cplusplus
}
#endif
#endif
