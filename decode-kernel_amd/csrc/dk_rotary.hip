// Rotary positions of queries and keys. Contract in
// include/decode_kernel/dk_rotary.h.
//
// A workgroup serves a few tokens of a range of heads. It forms the cosines
// and sines of their angles once, into LDS, where all heads read them: a
// frequency's angle is a 64-bit product reduced to a part of one turn there,
// so that only that part is rounded to fp32 (a position of 10^6 has 20 bits
// before the point, which a 32-bit angle would lose behind it). Each element
// is read and written once, 32 bytes a lane: bound by HBM for prompts (8192
// tokens of 72 heads of 128, 302 MB, 53 us with the result's memory used again and
// 64 into new memory, where a copy takes 59) and by latency for a decode step (64
// tokens 3.3 us).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "dk_host.hpp"
#include "dk_kv.hpp"
#include "decode_kernel/dk_rotary.h"

namespace dk {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryTokens = 4;  // tokens a workgroup serves at most

struct RotaryArgs {
  const uint16_t* in[2];  // q, k
  uint16_t* out[2];
  long long token_stride[2], head_stride[2];
  int heads[2];
  int head_size, tokens, axes, freqs;
  const void* positions;
  const float* frequencies;
  const int32_t* axis;
  int positions64, inverse;
  int tokens_each, heads_each;  // what a workgroup serves
};

template <bool kBf16>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  constexpr int kType = kBf16 ? DK_KV_BF16 : DK_KV_F16;
  return (uint32_t)to_half_bits<kType>(lo) | (uint32_t)to_half_bits<kType>(hi) << 16;
}

// kWide: an item is 16 elements of a head, as two loads of 8: the halves' i ..
// i + 7 (or 16 in a row, for adjacent pairs and for what is only copied). Else
// one pair, or one copied element.
template <bool kBf16, bool kAdjacent, bool kWide>
__global__ __launch_bounds__(kRotaryThreads) void rotate_kernel(RotaryArgs a) {
  __shared__ float2 turn[kRotaryTokens * DK_ROTARY_MAX_FREQUENCIES];  // cos, sin
  constexpr int kType = kBf16 ? DK_KV_BF16 : DK_KV_F16;
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * a.tokens_each, nt = min(a.tokens_each, a.tokens - t0);
  const int h0 = blockIdx.y * a.heads_each, nh = min(a.heads_each, a.heads[0] + a.heads[1] - h0);
  const int rotated = 2 * a.freqs;
  const unsigned units = kWide ? a.head_size / 16 : a.freqs + (a.head_size - rotated);
  const unsigned turning = kWide ? a.freqs / 8 : a.freqs;  // units that rotate
  const unsigned items = units * (unsigned)nh * (unsigned)nt;

  struct Item {
    long long from, to;
    int which, t, first, second, freq;
    bool turns;
  };
  auto item_of = [&](unsigned it) {
    Item x;
    const unsigned row = it / units, u = it - row * units;
    const unsigned t = row / (unsigned)nh;
    const int h = h0 + (int)(row - t * nh);
    x.which = h >= a.heads[0];
    const int hh = h - (x.which ? a.heads[0] : 0);
    x.t = (int)t;
    x.turns = u < turning;
    if constexpr (kWide) {
      x.freq = 8 * u;
      if (kAdjacent || !x.turns) {
        x.first = 16 * u;
        x.second = 16 * u + 8;
      } else {
        x.first = 8 * u;
        x.second = a.freqs + 8 * u;
      }
    } else {
      x.freq = u;
      if (!x.turns) x.first = x.second = a.freqs + u;  // freqs past the last pair's number
      else if (kAdjacent) x.first = 2 * u, x.second = 2 * u + 1;
      else x.first = u, x.second = a.freqs + u;
    }
    x.from = (long long)(t0 + x.t) * a.token_stride[x.which] + (long long)hh * a.head_stride[x.which];
    x.to = ((long long)(t0 + x.t) * a.heads[x.which] + hh) * a.head_size;
    return x;
  };
  using Part = typename std::conditional<kWide, uint4, uint16_t>::type;
  auto load = [&](const Item& x, Part& p, Part& q) {
    const uint16_t* src = a.in[x.which] + x.from;
    p = *reinterpret_cast<const Part*>(src + x.first);
    q = *reinterpret_cast<const Part*>(src + x.second);
  };

  // The first item's loads are under way while the angles are formed.
  unsigned it = tid;
  Item now;
  Part p{}, q{};
  if (it < items) {
    now = item_of(it);
    load(now, p, q);
  }
  for (int i = tid; i < nt * a.freqs; i += kRotaryThreads) {
    const int t = i / a.freqs, f = i - t * a.freqs;
    const int ax = a.axis ? min(max(a.axis[f], 0), a.axes - 1) : 0;
    const long long at = (long long)ax * a.tokens + t0 + t;
    const double pos = a.positions64 ? (double)static_cast<const int64_t*>(a.positions)[at]
                                     : (double)static_cast<const int32_t*>(a.positions)[at];
    const double turns = pos * (double)a.frequencies[f] * 0.15915494309189533577;  // 1 / (2 pi)
    const float part = (float)(turns - rint(turns));
    float s, c;
    sincospif(2.0f * part, &s, &c);
    turn[i] = make_float2(c, a.inverse ? -s : s);
  }
  __syncthreads();

  while (it < items) {
    const unsigned next = it + kRotaryThreads;
    Item after;
    Part pn{}, qn{};
    if (next < items) {
      after = item_of(next);
      load(after, pn, qn);
    }
    uint16_t* dst = a.out[now.which] + now.to;
    if (now.turns) {
      const float2* cs = turn + now.t * a.freqs + now.freq;
      if constexpr (kWide) {
        uint32_t x[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
        if constexpr (kAdjacent) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float u = pair_lo<kBf16>(x[j]), v = pair_hi<kBf16>(x[j]);
            x[j] = pack_pair<kBf16>(u * cs[j].x - v * cs[j].y, u * cs[j].y + v * cs[j].x);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 c0 = cs[2 * j], c1 = cs[2 * j + 1];
            const float u0 = pair_lo<kBf16>(x[j]), u1 = pair_hi<kBf16>(x[j]);
            const float v0 = pair_lo<kBf16>(x[4 + j]), v1 = pair_hi<kBf16>(x[4 + j]);
            x[j] = pack_pair<kBf16>(u0 * c0.x - v0 * c0.y, u1 * c1.x - v1 * c1.y);
            x[4 + j] = pack_pair<kBf16>(u0 * c0.y + v0 * c0.x, u1 * c1.y + v1 * c1.x);
          }
        }
        p = make_uint4(x[0], x[1], x[2], x[3]);
        q = make_uint4(x[4], x[5], x[6], x[7]);
      } else {
        const float u = pair_lo<kBf16>(p), v = pair_lo<kBf16>(q);
        p = to_half_bits<kType>(u * cs->x - v * cs->y);
        q = to_half_bits<kType>(u * cs->y + v * cs->x);
      }
    }
    *reinterpret_cast<Part*>(dst + now.first) = p;
    if (kWide || now.turns) *reinterpret_cast<Part*>(dst + now.second) = q;
    it = next;
    now = after;
    p = pn;
    q = qn;
  }
}

}  // namespace dk

extern "C" int dk_rotate_qk(const void* q, long long q_token_stride, long long q_head_stride,
                            int q_heads, const void* k, long long k_token_stride,
                            long long k_head_stride, int k_heads, int dtype, int head_size,
                            int num_tokens, const void* positions, int positions64, int num_axes,
                            const float* frequencies, const int32_t* axis, int num_frequencies,
                            int adjacent, int inverse, void* q_out, void* k_out,
                            hipStream_t stream) {
  auto aligned = [](const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  if (dtype != DK_KV_F16 && dtype != DK_KV_BF16)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "q and k must be fp16 or bf16");
  if (num_tokens < 0 || q_heads < 0 || k_heads < 0 || q_heads > 65535 || k_heads > 65535)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "num_tokens must be >= 0 and heads in [0, 65535]");
  if (head_size < 1 || head_size > DK_ROTARY_MAX_HEAD_SIZE)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "head_size=%d must be in [1, %d]", head_size,
                         DK_ROTARY_MAX_HEAD_SIZE);
  if (num_frequencies < 0 || num_frequencies > DK_ROTARY_MAX_FREQUENCIES ||
      2 * num_frequencies > head_size)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT,
                         "num_frequencies=%d must be in [0, %d] and at most half of head_size",
                         num_frequencies, DK_ROTARY_MAX_FREQUENCIES);
  if (num_axes < 1) return dk::set_error(DK_ERR_INVALID_ARGUMENT, "num_axes must be >= 1");
  if (num_tokens == 0 || q_heads + k_heads == 0) return DK_OK;
  if ((q_heads > 0 && (!q || !q_out)) || (k_heads > 0 && (!k || !k_out)) || !positions ||
      (num_frequencies > 0 && !frequencies))
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "rotate's arrays must not be NULL");
  if (!aligned(q, 2) || !aligned(k, 2) || !aligned(q_out, 2) || !aligned(k_out, 2) ||
      !aligned(frequencies, 4) || !aligned(axis, 4) || !aligned(positions, positions64 ? 8 : 4))
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "rotate's arrays must be aligned as their elements");

  const int heads = q_heads + k_heads;
  // Wide loads where each of them is 16 bytes from an address that 16 divides.
  const bool wide = head_size % 16 == 0 && num_frequencies % 8 == 0 && aligned(q_out, 16) && aligned(k_out, 16) &&
                    (q_heads == 0 || (aligned(q, 16) && q_token_stride % 8 == 0 && q_head_stride % 8 == 0)) &&
                    (k_heads == 0 || (aligned(k, 16) && k_token_stride % 8 == 0 && k_head_stride % 8 == 0));
  const int units = wide ? head_size / 16 : num_frequencies + head_size - 2 * num_frequencies;
  // A workgroup takes as many heads as its threads serve in one go, and all of
  // a few tokens' where that still leaves several workgroups a CU.
  int heads_each = units >= dk::kRotaryThreads ? 1 : dk::kRotaryThreads / units;
  int tokens_each = 1;
  if (heads_each >= heads) {
    heads_each = heads;
    while (tokens_each < dk::kRotaryTokens && units * heads * tokens_each < dk::kRotaryThreads) tokens_each *= 2;
  }
  const long long work = (long long)num_tokens * heads * units;
  if (work > 2048LL * 4 * dk::kRotaryThreads) {
    heads_each = std::min(heads, std::max(1, 4096 / units));
    tokens_each = dk::kRotaryTokens;
  }
  const long long groups = ((long long)num_tokens + tokens_each - 1) / tokens_each;
  const unsigned splits = (unsigned)((heads + heads_each - 1) / heads_each);
  if (!dk::fits_launch(groups, dk::kRotaryThreads))
    return dk::set_error(DK_ERR_UNSUPPORTED, "too many tokens for one call");
  if (splits > 65535)
    return dk::set_error(DK_ERR_UNSUPPORTED, "too many heads for this head size");
  const dk::RotaryArgs a{{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k)},
                         {static_cast<uint16_t*>(q_out), static_cast<uint16_t*>(k_out)},
                         {q_token_stride, k_token_stride},
                         {q_head_stride, k_head_stride},
                         {q_heads, k_heads},
                         head_size,
                         num_tokens,
                         num_axes,
                         num_frequencies,
                         positions,
                         frequencies,
                         axis,
                         positions64,
                         inverse,
                         tokens_each,
                         heads_each};
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups, splits), dim3(dk::kRotaryThreads), 0, stream, a);
  };
  auto pick = [&](auto bf16, auto adj) {
    constexpr bool b = decltype(bf16)::value, j = decltype(adj)::value;
    wide ? launch(dk::rotate_kernel<b, j, true>) : launch(dk::rotate_kernel<b, j, false>);
  };
  using yes = std::true_type;
  using no = std::false_type;
  if (dtype == DK_KV_BF16) adjacent ? pick(yes{}, yes{}) : pick(yes{}, no{});
  else adjacent ? pick(no{}, yes{}) : pick(no{}, no{});
  return dk::check_launch("rotate launch");
}
