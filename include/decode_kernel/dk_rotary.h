/* Rotary positions of one or several axes (MI355X, gfx950): what queries and
 * keys go through between their projection and dk_kv_append / dk_kv_attend
 * (dk_kv.h).
 *
 * No counterpart in the reference, which holds weights only (the step behind
 * its gemv(), python/decode_kernel/__init__.py:32-83). Asynchronous on the
 * given stream, allocates nothing and copies nothing to the host. Status
 * codes and dk_last_error() are those of dk_gemv.h; the dispatch stamp is not
 * touched.
 */
#ifndef DECODE_KERNEL_DK_ROTARY_H_
#define DECODE_KERNEL_DK_ROTARY_H_

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime.h>

#include "decode_kernel/dk_gemv.h" /* status codes */
#include "decode_kernel/dk_kv.h"   /* element types */

#ifdef __cplusplus
extern "C" {
#endif

/* The most frequencies (half of the elements that rotate) and elements of a
 * head that dk_rotate_qk takes. */
#define DK_ROTARY_MAX_FREQUENCIES 256
#define DK_ROTARY_MAX_HEAD_SIZE 1024

/* q [num_tokens, q_heads, head_size] and k [num_tokens, k_heads, head_size] of
 * type dtype (DK_KV_F16 or DK_KV_BF16), strides in elements of tokens and
 * heads, the last dimension contiguous, into contiguous q_out and k_out of the
 * same shapes. With angle(t, i) = positions[axis[i]][t] * frequencies[i] for
 * i < num_frequencies, the pair (a, b) of elements (i, num_frequencies + i) of
 * a head, or (2 i, 2 i + 1) with adjacent nonzero, becomes
 *   (a cos - b sin, a sin + b cos)
 * and with inverse nonzero the rotation by -angle (the transposed one: the
 * gradient of q and k from that of the results). Elements from 2
 * num_frequencies on are copied as they are. positions: int32 or, with
 * positions64 nonzero, int64, [num_axes, num_tokens]; axis: int32
 * [num_frequencies], values outside 0 .. num_axes - 1 taken as the nearest of
 * them, NULL for all 0. The angle is formed in 64 bits and reduced to one turn
 * there, so far positions cost no accuracy; cos, sin and the products are fp32.
 * q or k may have 0 heads. Outputs are apart from all inputs. From 2^26 - 3 tokens
 * on it is DK_ERR_UNSUPPORTED. */
int dk_rotate_qk(const void* q, long long q_token_stride, long long q_head_stride, int q_heads,
                 const void* k, long long k_token_stride, long long k_head_stride, int k_heads,
                 int dtype, int head_size, int num_tokens, const void* positions, int positions64,
                 int num_axes, const float* frequencies, const int32_t* axis, int num_frequencies,
                 int adjacent, int inverse, void* q_out, void* k_out, hipStream_t stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* DECODE_KERNEL_DK_ROTARY_H_ */
