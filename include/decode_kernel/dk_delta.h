/* Gated delta rule and the short convolution before it (MI355X, gfx950): the
 * token mixing of a decoder's layers that keep a state of fixed size for each
 * request instead of a cache that grows.
 *
 * A step's tokens stand request after request, as dk_kv_plan (dk_kv.h) orders
 * them: request b has the rows offsets[b] .. offsets[b + 1] - 1 of num_tokens
 * (offsets NULL: row b alone, and num_tokens == requests). held[b] is what it
 * had before the step (dk_kv_plan's held): a request that held nothing starts
 * from zeros, whatever its state or window contains (held NULL: all go on from
 * theirs). A request without new tokens keeps its state and window as they
 * are, and the results of rows that belong to no request (before the first
 * offset or from the last one on) are 0. Where offsets decrease, or leave
 * 0 .. num_tokens, all results are 0 and nothing is updated.
 *
 * No counterpart in the reference, which holds weights only: these stand
 * between the projections that its gemv() computes
 * (python/decode_kernel/__init__.py:32-83), where a layer with a cache has
 * dk_kv_append and dk_kv_attend.
 *
 * Every entry point is asynchronous on the given stream, allocates nothing
 * and copies nothing to the host. Status codes and dk_last_error() are those
 * of dk_gemv.h; the dispatch stamp is not touched.
 */
#ifndef DECODE_KERNEL_DK_DELTA_H_
#define DECODE_KERNEL_DK_DELTA_H_

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime.h>

#include "decode_kernel/dk_gemv.h" /* status codes */
#include "decode_kernel/dk_kv.h"   /* element types */

#ifdef __cplusplus
extern "C" {
#endif

/* What dk_delta_rule works on. q and k: [num_tokens, qk_heads, key_size], v:
 * [num_tokens, v_heads, value_size], of type dtype (DK_KV_F16 or DK_KV_BF16),
 * strides in elements of tokens (0 .. 2^24) and heads, multiples of 8, 16-byte
 * aligned; log_decay and beta: fp32 [num_tokens, v_heads]; states: fp32
 * [requests, v_heads, key_size, value_size], 16-byte aligned. v_heads is a
 * multiple of qk_heads (head h has the keys of head h / (v_heads / qk_heads)),
 * key_size and value_size are 64 or 128. */
typedef struct dk_delta_args {
  const void* q;
  const void* k;
  const void* v;
  long long q_token_stride, q_head_stride;
  long long k_token_stride, k_head_stride;
  long long v_token_stride, v_head_stride;
  const float* log_decay;
  const float* beta;
  float* states;
  const int32_t* held;
  const int32_t* offsets;
  int dtype;
  int num_tokens;
  int requests;
  int qk_heads;
  int v_heads;
  int key_size;
  int value_size;
  int max_query_len; /* the most tokens that a request gets. It only picks
                        kernels, the better the closer it is; requests with
                        more are right too */
  int normalize;     /* nonzero: q and k as x / sqrt(|x|^2 + 1e-6) */
  float scale;
} dk_delta_args;

/* Bytes of workspace dk_delta_rule takes for these sizes: 0 where every
 * request gets few tokens (max_query_len), else what the chunks of 64 tokens
 * of its prompts need. Returns 0 for invalid arguments. */
size_t dk_delta_workspace_bytes(int num_tokens, int requests, int qk_heads, int v_heads,
                                int key_size, int max_query_len);

/* Token by token of each request, for each head, from its state S:
 *   S <- exp(log_decay) S
 *   S <- S + k (beta (v - S^T k))^T
 *   out = scale S^T q
 * with S as it is after the last token written back. out: dtype, contiguous
 * [num_tokens, v_heads, value_size], 16-byte aligned; it and states are
 * apart from all inputs. log_decay is at most 0 (over a chunk of 64 tokens its sum
 * has to stay in fp32's exponents); -infinity empties the state. With
 * beta |k|^2 over 2 (over 2 of normalised keys' beta) the rule itself
 * amplifies what the state holds; long prompts then leave fp32's range sooner
 * than tokens one by one would. Sums and states are fp32, and a result is off by
 * their roundings at the token's own time, whatever came before or comes later:
 * in a prompt's products the state has 22 bits, counted from the largest value of
 * its column, and values, decays and corrections have 24 of their own. With beta
 * |k|^2 near 2 and keys that hardly differ nothing fades, and the corrections of a
 * prompt's 64 tokens cancel: they can lose up to 2e-3 of values and state (150
 * tokens one by one up to 1e-4). A NaN or infinity
 * stays in its request, and one in v in its column of the state; in a prompt it
 * may reach the results of up to 63 tokens before its own, too (a chunk's
 * products multiply what comes later by 0). The
 * workspace is 256-byte aligned, needs no clearing and holds nothing between
 * calls; calls that overlap in time need workspaces of their own. From 2^24
 * chunks of 64 tokens (one more a request) times heads on it is DK_ERR_UNSUPPORTED. */
int dk_delta_rule(const dk_delta_args* args, void* out, void* workspace, size_t workspace_bytes,
                  hipStream_t stream);

/* The causal convolution of width taps (2, 3 or 4) over each request's own
 * tokens, channel by channel:
 *   y[t, c] = act(bias[c] + sum_j weight[c, j] x[t - (width - 1) + j, c])
 * where inputs before the step come from windows [requests, width - 1,
 * channels] (the oldest first), which then hold the last width - 1 inputs. act
 * is z / (1 + exp(-z)) with silu nonzero, else nothing. x, weight [channels,
 * width], bias (or NULL), windows and y have type dtype (F16 or BF16); sums
 * are fp32. x has a stride of tokens, y is contiguous; max_query_len as in dk_delta_args; both, weight and
 * windows aligned as their elements are (16-byte rows of x, y and windows,
 * and 16-byte weights, take the wide loads). y and windows are apart from all
 * inputs. A call takes fewer than 2^24 tiles of 4 or 8 tokens (one more a request;
 * of one token without offsets), else it is DK_ERR_UNSUPPORTED. */
int dk_short_conv(const void* x, long long x_token_stride, const void* weight, const void* bias,
                  void* windows, const int32_t* held, const int32_t* offsets, int dtype,
                  int num_tokens, int requests, int channels, int width, int max_query_len,
                  int silu, void* y, hipStream_t stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* DECODE_KERNEL_DK_DELTA_H_ */
