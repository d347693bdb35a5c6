/* Paged 8-bit key/value cache and the attention over it (MI355X, gfx950).
 *
 * The cache holds keys and values as int8 codes with one fp32 scale for each
 * page (page_size consecutive tokens of one sequence) and head, keys and
 * values apart; a value is code * scale, scales at least 0. Its layout is the one the attention
 * kernels' matrix operands are read in:
 *
 *   k_codes  [pages, heads, head_size / 16, page_size, 16]
 *   v_codes  [pages, heads, head_size, page_size]
 *   k_scales, v_scales  [pages, heads]
 *
 * A sequence's pages are named by its row of a block table (int32
 * [requests, table_width], -1 for none); token t of sequence b is at slot
 * tables[b][t / page_size] * page_size + t % page_size.
 *
 * No counterpart in the reference, which holds weights only: this is the
 * step between the q/k/v projections and the output projection of a decoder
 * layer around its gemv() (python/decode_kernel/__init__.py:32-83).
 *
 * Every entry point is asynchronous on the given stream, allocates nothing
 * and copies nothing to the host. Status codes and dk_last_error() are those
 * of dk_gemv.h; the dispatch stamp is not touched.
 */
#ifndef DECODE_KERNEL_DK_KV_H_
#define DECODE_KERNEL_DK_KV_H_

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime.h>

#include "decode_kernel/dk_gemv.h" /* status codes */

#ifdef __cplusplus
extern "C" {
#endif

/* Requests dk_kv_plan takes at most (their prefix sums are held in LDS). */
#define DK_KV_MAX_REQUESTS 4096

/* Element types of activations. */
#define DK_KV_F16 0
#define DK_KV_BF16 1
#define DK_KV_F32 2

/* head_size 64 or 128; page_size 16, 32, 64 or 128; code pointers 16-byte
 * aligned. */
typedef struct dk_kv_cache {
  int8_t* k_codes;
  int8_t* v_codes;
  float* k_scales;
  float* v_scales;
  int pages;
  int heads;
  int head_size;
  int page_size;
} dk_kv_cache;

/* Pages and slots of a step's new tokens. Request b holds held[b] tokens and
 * gets added[b] more (both taken as 0 if negative), in the order of the
 * requests, num_tokens in all at most. Writes
 *   query_offsets [requests + 1]  where each request's tokens start in the step,
 *   seq_lens [requests]           tokens held after the step (at most
 *                                 table_width * page_size),
 *   slots, positions [num_tokens] of each token (-1 past the last one),
 *   tables                        the entries of newly opened pages,
 *   *free_count_out               *free_count less the pages opened.
 * Pages come off the end of free_pages[0 .. *free_count), in the order of
 * the requests. Where none is left the entry is -1, the slots of its tokens
 * are -1 and *free_count_out is negative by what was missing; slots past the
 * table's end are -1 too. A token without a slot stays without: an entry of -1
 * is not filled in later. After a shortage take the missing tokens off held
 * (down to the end of the last page that is there), or drop their requests, and
 * set the count to 0 before pages are put back from there; a negative one is
 * subtracted from what comes after it. Every result is a function of the inputs
 * alone, so the same call again gives the same. free_count_out must not be
 * free_count. */
int dk_kv_plan(int32_t* tables, int table_width, const int32_t* held, const int32_t* added,
               int requests, const int32_t* free_pages, int free_capacity,
               const int32_t* free_count, int page_size, int num_tokens, int64_t* slots,
               int32_t* positions, int32_t* query_offsets, int32_t* seq_lens,
               int32_t* free_count_out, hipStream_t stream);

/* Writes k and v [num_tokens, heads, head_size] (DK_KV_F16 or DK_KV_BF16; strides in
 * elements of tokens and heads, multiples of 8; 16-byte aligned) at slots.
 * Tokens of one page must stand together and in order, as dk_kv_plan gives
 * them (token t + i at slot s + i); slots outside the cache (-1) are skipped,
 * also among them. For each page and head that the step writes, with amax over
 * its new tokens:
 *   scale = max(old scale, amax * (1 / 127))  (old scale 0 if token 0 of the
 *                                              page is among the new ones)
 *   inv = 1 / scale                           (0 for a scale under 2^-126,
 *                                              which so stores zeros)
 *   code = clamp(rint(x * inv), -127, 127)
 * and where the scale grows the page's earlier codes become
 * clamp(rint(code * (old scale * inv)), -127, 127); each operation is rounded
 * to fp32. A NaN or infinity makes the scale NaN, and with it every value of
 * the page for that head. */
int dk_kv_append(const dk_kv_cache* cache, const void* k, const void* v, int dtype,
                 long long k_token_stride, long long k_head_stride, long long v_token_stride,
                 long long v_head_stride, const int64_t* slots, int num_tokens,
                 hipStream_t stream);

/* k and v [num_tokens, heads, head_size] = code * scale at slots, in fp32 and
 * from there rounded to dtype (F16, BF16 or F32); zeros for a slot outside the
 * cache. */
int dk_kv_read(const dk_kv_cache* cache, const int64_t* slots, int num_tokens, int dtype, void* k,
               void* v, hipStream_t stream);

/* Bytes of workspace dk_kv_attend takes for these sizes (partial results of
 * sequences that several workgroups share). max_query_len: as in the call. */
size_t dk_kv_attend_workspace_bytes(int num_tokens, int requests, int q_heads, int heads,
                                    int head_size, int table_width, int page_size,
                                    int max_query_len);

/* out[t, hq] = sum_j softmax_j(scale * q[t, hq] . k[j]) v[j] over the keys j
 * of t's sequence, heads hq / (q_heads / heads). Sequence b has seq_lens[b]
 * keys (at most table_width * page_size) and the queries
 * query_offsets[b] .. query_offsets[b + 1] - 1 (NULL: query b alone, and
 * num_tokens == requests; where offsets decrease, all of out is 0). With causal,
 * query i of n sees the keys up to seq_lens[b] - n + i: the queries are the
 * sequence's last tokens, and their keys are in the cache already. Keys on a page outside the cache (-1) are
 * not seen. A query that sees no key gives 0, and so does one that belongs to no
 * sequence (before the first offset or from the last one on), which is not read.
 *
 * q and out: DK_KV_F16 or DK_KV_BF16, out contiguous, q with strides (in
 * elements, multiples of 8) of tokens and heads, both 16-byte aligned.
 * max_query_len: the most queries that a sequence has. It only picks
 * kernels; sequences with more are right too. Work is counted in 31 bits: heads
 * times tiles of 256 rows (queries times the group; of 16 or 32 where all
 * sequences have up to 128) times tiles of 64 keys (of the tables' width) over
 * 2^30 is DK_ERR_UNSUPPORTED, and so are keys or num_tokens times the group over
 * 2^30. */
int dk_kv_attend(const void* q, int dtype, long long q_token_stride, long long q_head_stride,
                 const dk_kv_cache* cache, const int32_t* tables, int table_width,
                 const int32_t* seq_lens, const int32_t* query_offsets, int num_tokens,
                 int requests, int q_heads, int max_query_len, float scale, int causal, void* out,
                 void* workspace, size_t workspace_bytes, hipStream_t stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* DECODE_KERNEL_DK_KV_H_ */
