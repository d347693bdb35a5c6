// The gated delta rule token by token, the short convolution before it, and
// the entry points of both. Contracts in include/decode_kernel/dk_delta.h, the
// chunked form of long prompts in dk_delta_chunk.hip.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "dk_delta.hpp"
#include "dk_host.hpp"

namespace dk {

// ---------------------------------------------------------------------------
// Token by token: a wave holds all rows of 32 columns of one head's state in
// registers, from the first of a request's tokens to its last. Columns do not
// meet: both products over the rows, S^T k and S^T q, are taken of the old
// state in one pass, since with u = beta (v - e^g S^T k)
//   S_new^T q = e^g S^T q + u (k . q).
// A lane has 4 columns (16 bytes of a row) of dk / 8 rows that follow one
// another; 8 lanes read a line of 128 bytes, and sums over the rows go over
// the other three lane bits. One new token a request is bound by reading and
// writing its state once: 61 requests of 32 heads of 128 x 128, 250 MB, take 49.8
// us, 5.0 TB/s, where a copy reaches 5.1. More tokens are bound by the chain from
// token to token.
// ---------------------------------------------------------------------------
constexpr int kStepColumns = 32;

__device__ __forceinline__ float sum_rows(float v) {
  v += dpp<0x128>(v);  // row_ror:8: the lane 8 away in its row of 16
  // Through LDS, 22 of them on their way at once: swaps of register halves
  // (v_permlane*_swap) take one wait each, 13.0 against 11.8 us for 4 tokens of
  // 96 requests.
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  return v;
}

template <int kDk, bool kBf16>
__global__ __launch_bounds__(64) void delta_step_kernel(DeltaArgs a, int value_size) {
  constexpr int kRows = kDk / 8;
  constexpr int kType = kBf16 ? DK_KV_BF16 : DK_KV_F16;
  const int lane = threadIdx.x;
  const int slices = value_size / kStepColumns;
  const int h = blockIdx.x / slices, b = blockIdx.y;
  const int col = (blockIdx.x % slices) * kStepColumns + (lane & 7) * 4;
  const int row = (lane >> 3) * kRows;
  uint16_t* out = a.out + (long long)h * value_size + col;
  const long long out_token = (long long)a.v_heads * value_size;
  auto clear = [&](int from, int to) {
    for (int t = from + (lane >> 3); t < to; t += 8)
      *reinterpret_cast<uint2*>(out + t * out_token) = make_uint2(0u, 0u);
  };

  int first = b, last = b + 1;
  bool ok = a.requests > 0;
  if (!ok) {
    clear(0, a.tokens);
  } else if (a.offsets) {
    first = a.offsets[b];
    last = a.offsets[b + 1];
    ok = wave_offsets_ok(a.offsets, a.requests, a.tokens);
    if (ok) {
      if (b == 0) clear(0, first);
      if (b == a.requests - 1) clear(last, a.tokens);
    } else if (b == 0) {
      clear(0, a.tokens);
    }
  }
  if (!ok || last == first || last - first > a.limit) return;

  float* state = a.states + (((long long)b * a.v_heads + h) * kDk + row) * value_size + col;
  f4_t s[kRows];
  if (a.held && a.held[b] <= 0) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) s[r] = f4_t{0.f, 0.f, 0.f, 0.f};
  } else {
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      s[r] = *reinterpret_cast<const f4_t*>(state + (long long)r * value_size);
  }

  const uint16_t* kp = a.k + (long long)(h / a.group) * a.k_head + row;
  const uint16_t* qp = a.q + (long long)(h / a.group) * a.q_head + row;
  const uint16_t* vp = a.v + (long long)h * a.v_head + col;
  struct Token {
    uint4 k[kRows / 8], q[kRows / 8];
    uint2 v;
    float g, beta;
  };
  auto load = [&](int t) {
    Token x;
#pragma unroll
    for (int i = 0; i < kRows / 8; ++i) {
      x.k[i] = *reinterpret_cast<const uint4*>(kp + t * a.k_token + 8 * i);
      x.q[i] = *reinterpret_cast<const uint4*>(qp + t * a.q_token + 8 * i);
    }
    x.v = *reinterpret_cast<const uint2*>(vp + t * a.v_token);
    x.g = a.log_decay[(long long)t * a.v_heads + h];
    x.beta = a.beta[(long long)t * a.v_heads + h];
    return x;
  };
  Token next = load(first);
  for (int t = first; t < last; ++t) {
    const Token now = next;
    if (t + 1 < last) next = load(t + 1);
    float k[kRows], q[kRows];
#pragma unroll
    for (int i = 0; i < kRows / 8; ++i) {
      const uint32_t kw[4] = {now.k[i].x, now.k[i].y, now.k[i].z, now.k[i].w};
      const uint32_t qw[4] = {now.q[i].x, now.q[i].y, now.q[i].z, now.q[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        k[8 * i + 2 * j] = pair_lo<kBf16>(kw[j]);
        k[8 * i + 2 * j + 1] = pair_hi<kBf16>(kw[j]);
        q[8 * i + 2 * j] = pair_lo<kBf16>(qw[j]);
        q[8 * i + 2 * j + 1] = pair_hi<kBf16>(qw[j]);
      }
    }
    float kk = 0.f, qq = 0.f, kq = 0.f;
    f4_t sk{0.f, 0.f, 0.f, 0.f}, sq{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      kk = fmaf(k[r], k[r], kk);
      qq = fmaf(q[r], q[r], qq);
      kq = fmaf(k[r], q[r], kq);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        sk[c] = fmaf(s[r][c], k[r], sk[c]);
        sq[c] = fmaf(s[r][c], q[r], sq[c]);
      }
    }
    kq = sum_rows(kq);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      sk[c] = sum_rows(sk[c]);
      sq[c] = sum_rows(sq[c]);
    }
    float kr = 1.f, qr = a.scale;
    if (a.normalize) {
      // The hardware's reciprocal root, 1 ulp: a root and a division are 25
      // instructions of a token's 400.
      kr = __builtin_amdgcn_rsqf(sum_rows(kk) + kUnitEps);
      qr *= __builtin_amdgcn_rsqf(sum_rows(qq) + kUnitEps);
    }
    const float keep = expf(now.g);
    const float v[4] = {pair_lo<kBf16>(now.v.x), pair_hi<kBf16>(now.v.x), pair_lo<kBf16>(now.v.y),
                        pair_hi<kBf16>(now.v.y)};
    float u[4], o[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      u[c] = kr * now.beta * (v[c] - keep * kr * sk[c]);
      o[c] = qr * fmaf(keep, sq[c], u[c] * kq);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[r][c] = fmaf(k[r], u[c], keep * s[r][c]);
    if (lane < 8)
      *reinterpret_cast<uint2*>(out + t * out_token) =
          make_uint2((uint32_t)to_half_bits<kType>(o[0]) | (uint32_t)to_half_bits<kType>(o[1]) << 16,
                     (uint32_t)to_half_bits<kType>(o[2]) | (uint32_t)to_half_bits<kType>(o[3]) << 16);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) *reinterpret_cast<f4_t*>(state + (long long)r * value_size) = s[r];
}

// ---------------------------------------------------------------------------
// The short convolution: a workgroup takes a tile of one request's tokens and
// a block of channels, a thread 8 channels (or one, where rows are not made of
// aligned 16-byte pieces) down the tile with the last inputs in registers, so
// that each input is read once but for the width - 1 before a tile. The tile
// that holds a request's first tokens is the only reader of its window, so
// the same threads write it. Bound by HBM for prompts (8192 tokens of 8192
// channels, 268 MB, 54 us, 5.0 TB/s) and by latency for single tokens (64 tokens
// 3.6 us): every load is asked for before the first is waited for.
// ---------------------------------------------------------------------------
struct ConvArgs {
  const uint16_t* x;
  long long x_token;
  const uint16_t* weight;
  const uint16_t* bias;
  uint16_t* windows;
  const int32_t* held;
  const int32_t* offsets;
  uint16_t* y;
  int tokens, requests, channels, silu;
};

// z / (1 + e^-z) on the hardware's exponential and reciprocal, 1 ulp each: with
// a division and expf() the arithmetic of 67 million elements takes as long as
// their bytes (62 of 80 us).
__device__ __forceinline__ float silu_of(float z) {
  return z * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f));
}

template <int kWidth, int kTile, bool kBf16, bool kWide>
__global__ __launch_bounds__(256) void short_conv_kernel(ConvArgs a) {
  constexpr int kEach = kWide ? 8 : 1, kPast = kWidth - 1;
  constexpr int kType = kBf16 ? DK_KV_BF16 : DK_KV_F16;
  using Part = typename std::conditional<kWide, uint4, uint16_t>::type;
  const int c = (blockIdx.y * 256 + threadIdx.x) * kEach;
  const bool mine = c < a.channels;
  auto clear = [&](long long from, long long to) {
    if (mine)
      for (long long t = from; t < to; ++t) *reinterpret_cast<Part*>(a.y + t * a.channels + c) = Part{};
  };
  Tile tile{(int)blockIdx.x, (int)blockIdx.x, 1, 0, 1, 0, 0};
  if (a.offsets) {
    const long long part = (long long)blockIdx.x * kTile;
    if (a.requests == 0 || !find_tile(a.offsets, a.requests, a.tokens, kTile, blockIdx.x, &tile)) {
      clear(min(part, (long long)a.tokens), min(part + kTile, (long long)a.tokens));
      return;
    }
    clear(min(part, (long long)tile.head), min(part + kTile, (long long)tile.head));
    clear(min(tile.end + part, (long long)a.tokens), min(tile.end + part + kTile, (long long)a.tokens));
    if (tile.request < 0) return;
  }
  if (!mine) return;

  auto get = [&](const Part& p, float (&f)[kEach]) {
    if constexpr (kWide) {
      const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[2 * j] = pair_lo<kBf16>(w[j]);
        f[2 * j + 1] = pair_hi<kBf16>(w[j]);
      }
    } else {
      f[0] = pair_lo<kBf16>(p);
    }
  };
  // Rows before the request's first come from the window, those behind the
  // tile's last are that one again.
  const uint16_t* x = a.x + (long long)tile.row * a.x_token + c;
  uint16_t* window = a.windows + (long long)tile.request * kPast * a.channels + c;
  const bool first = tile.index == 0;
  const int n = tile.total;
  Part in[kPast + kTile];
#pragma unroll
  for (int i = 0; i < kPast; ++i)
    in[i] = *reinterpret_cast<const Part*>(first ? window + (long long)i * a.channels
                                                 : x + (long long)(i - kPast) * a.x_token);
#pragma unroll
  for (int i = 0; i < kTile; ++i)
    in[kPast + i] = *reinterpret_cast<const Part*>(x + (long long)min(i, tile.count - 1) * a.x_token);
  Part w_raw[kWidth];
#pragma unroll
  for (int i = 0; i < kWidth; ++i)  // 8 channels' weights are kWidth pieces of 16 bytes in a row
    w_raw[i] = *reinterpret_cast<const Part*>(a.weight + (long long)c * kWidth + kEach * i);
  if (first) {
    if (a.held && a.held[tile.request] <= 0)
#pragma unroll
      for (int i = 0; i < kPast; ++i) in[i] = Part{};
    // The window's row i is then the request's new row n - kPast + i, or, where
    // that is below 0, its own row n + i.
    Part keep[kPast];
#pragma unroll
    for (int i = 0; i < kPast; ++i)
      keep[i] = *reinterpret_cast<const Part*>(x + (long long)max(n - kPast + i, 0) * a.x_token);
#pragma unroll
    for (int i = 0; i < kPast; ++i) {
#pragma unroll
      for (int j = 0; j < kPast; ++j)
        if (n + i == j) keep[i] = in[j];
      *reinterpret_cast<Part*>(window + (long long)i * a.channels) = keep[i];
    }
  }

  float w[kEach][kWidth], bias[kEach];
  if constexpr (kWide) {
    uint16_t flat[8 * kWidth];
#pragma unroll
    for (int i = 0; i < kWidth; ++i) {
      const uint32_t pw[4] = {w_raw[i].x, w_raw[i].y, w_raw[i].z, w_raw[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        flat[8 * i + 2 * j] = (uint16_t)pw[j];
        flat[8 * i + 2 * j + 1] = (uint16_t)(pw[j] >> 16);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int j = 0; j < kWidth; ++j) w[e][j] = pair_lo<kBf16>(flat[e * kWidth + j]);
  } else {
#pragma unroll
    for (int j = 0; j < kWidth; ++j) w[0][j] = pair_lo<kBf16>(w_raw[j]);
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) bias[e] = a.bias ? pair_lo<kBf16>(a.bias[c + e]) : 0.f;

  float past[kWidth][kEach];
#pragma unroll
  for (int i = 0; i < kPast; ++i) get(in[i], past[i]);
  uint16_t* y = a.y + (long long)tile.row * a.channels + c;
#pragma unroll
  for (int i = 0; i < kTile; ++i) {
    get(in[kPast + i], past[kPast]);
    uint16_t o[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      float z = bias[e];
#pragma unroll
      for (int j = 0; j < kWidth; ++j) z = fmaf(past[j][e], w[e][j], z);
      o[e] = to_half_bits<kType>(a.silu ? silu_of(z) : z);
    }
    if (i < tile.count) {
      if constexpr (kWide) {
        uint32_t p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = (uint32_t)o[2 * j] | (uint32_t)o[2 * j + 1] << 16;
        *reinterpret_cast<uint4*>(y + (long long)i * a.channels) = make_uint4(p[0], p[1], p[2], p[3]);
      } else {
        y[(long long)i * a.channels] = o[0];
      }
    }
#pragma unroll
    for (int j = 0; j < kPast; ++j)
#pragma unroll
      for (int e = 0; e < kEach; ++e) past[j][e] = past[j + 1][e];
  }
}

// Requests of up to so many tokens go token by token, 1.1 us each; a chunk costs
// its 64 tokens' work also where few are there. 17 tokens, token by token and as
// a chunk, us: 1 request of 32 heads 22 and 17, 8 of them 27 and 43, 64 of 4 heads
// 25 and 48, 200 of 8 heads 110 and 197; 32 tokens 37 and 18, 44 and 42, 43 and 48,
// 165 and 209. One line for all: where it is wrong, for a single request or for
// many with 17 to about 40 tokens each, a call takes up to twice as long.
constexpr int kStepTokens = 16;

}  // namespace dk

namespace {

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

bool delta_size(int n) { return n == 64 || n == 128; }

}  // namespace

extern "C" size_t dk_delta_workspace_bytes(int num_tokens, int requests, int qk_heads, int v_heads,
                                           int key_size, int max_query_len) {
  if (num_tokens <= 0 || requests <= 0 || qk_heads <= 0 || v_heads <= 0 || v_heads % qk_heads ||
      !delta_size(key_size) || max_query_len <= dk::kStepTokens)
    return 0;
  return dk::delta_chunk_bytes(num_tokens, requests, dk::kStepTokens, qk_heads, v_heads, key_size);
}

extern "C" int dk_delta_rule(const dk_delta_args* p, void* out, void* workspace,
                             size_t workspace_bytes, hipStream_t stream) {
  if (!p) return dk::set_error(DK_ERR_INVALID_ARGUMENT, "args must not be NULL");
  if (p->dtype != DK_KV_F16 && p->dtype != DK_KV_BF16)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "q, k and v must be fp16 or bf16");
  if (p->num_tokens < 0 || p->requests < 0)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "num_tokens and requests must be >= 0");
  if (p->requests > 65535)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "requests must be at most 65535");
  if (p->qk_heads < 1 || p->v_heads < 1 || p->v_heads > 65535 || p->v_heads % p->qk_heads)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT,
                         "v_heads (1..65535) must be a multiple of qk_heads");
  if (!delta_size(p->key_size) || !delta_size(p->value_size))
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "key_size and value_size must be 64 or 128");
  if (p->max_query_len < 1)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "max_query_len must be >= 1");
  if (!p->offsets && p->num_tokens != p->requests)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT,
                         "without offsets each request has one token: num_tokens must be requests");
  if (p->num_tokens == 0) return DK_OK;
  if (!p->q || !p->k || !p->v || !p->log_decay || !p->beta || !out ||
      (p->requests > 0 && !p->states))
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "delta_rule's arrays must not be NULL");
  if (!aligned(p->q, 16) || !aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(out, 16) ||
      !aligned(p->states, 16))
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "q, k, v, states and out must be 16-byte aligned");
  if (!aligned(p->log_decay, 4) || !aligned(p->beta, 4) || !aligned(p->held, 4) ||
      !aligned(p->offsets, 4))
    return dk::set_error(DK_ERR_INVALID_ARGUMENT,
                         "log_decay, beta, held and offsets must be 4-byte aligned");
  if (p->q_token_stride % 8 || p->q_head_stride % 8 || p->k_token_stride % 8 ||
      p->k_head_stride % 8 || p->v_token_stride % 8 || p->v_head_stride % 8)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "the strides of q, k and v must be multiples of 8");
  for (const long long stride : {p->q_token_stride, p->k_token_stride, p->v_token_stride})
    if (stride < 0 || stride > 1 << 24)  // 64 of them are counted in 32 bits
      return dk::set_error(DK_ERR_INVALID_ARGUMENT, "the token strides of q, k and v must be in [0, 2^24]");
  // Without offsets a request has one token whatever max_query_len says.
  const bool chunks = p->offsets && p->max_query_len > dk::kStepTokens && p->requests > 0;
  const size_t need = chunks ? dk_delta_workspace_bytes(p->num_tokens, p->requests, p->qk_heads, p->v_heads,
                                                        p->key_size, p->max_query_len) : 0;
  if (chunks) {
    if (!dk::fits_launch(dk::chunk_slots(p->num_tokens, p->requests, dk::kStepTokens) * p->v_heads, dk::kPrepareThreads))
      return dk::set_error(DK_ERR_UNSUPPORTED, "too large: chunks times heads must be under 2^24");
    if (!workspace || !aligned(workspace, 256) || workspace_bytes < need)
      return dk::set_error(DK_ERR_INVALID_ARGUMENT,
                           "workspace must be 256-byte aligned and of %zu bytes", need);
  }
  const dk::DeltaArgs a{static_cast<const uint16_t*>(p->q),
                        static_cast<const uint16_t*>(p->k),
                        static_cast<const uint16_t*>(p->v),
                        p->q_token_stride,
                        p->q_head_stride,
                        p->k_token_stride,
                        p->k_head_stride,
                        p->v_token_stride,
                        p->v_head_stride,
                        p->log_decay,
                        p->beta,
                        p->states,
                        p->held,
                        p->offsets,
                        static_cast<uint16_t*>(out),
                        p->num_tokens,
                        p->requests,
                        p->qk_heads,
                        p->v_heads,
                        p->v_heads / p->qk_heads,
                        chunks ? dk::kStepTokens : INT32_MAX,
                        p->max_query_len,
                        p->normalize,
                        p->scale};
  const bool bf16 = p->dtype == DK_KV_BF16;
  const dim3 grid((unsigned)(p->v_heads * (p->value_size / dk::kStepColumns)),
                  (unsigned)(p->requests > 0 ? p->requests : 1));
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(64), 0, stream, a, p->value_size);
  };
  if (p->key_size == 64)
    bf16 ? launch(dk::delta_step_kernel<64, true>) : launch(dk::delta_step_kernel<64, false>);
  else
    bf16 ? launch(dk::delta_step_kernel<128, true>) : launch(dk::delta_step_kernel<128, false>);
  if (const int rc = dk::check_launch("delta_rule launch")) return rc;
  if (!chunks) return DK_OK;
  return dk::delta_chunk_launch(a, p->key_size, p->value_size, bf16, workspace, stream);
}

extern "C" int dk_short_conv(const void* x, long long x_token_stride, const void* weight,
                             const void* bias, void* windows, const int32_t* held,
                             const int32_t* offsets, int dtype, int num_tokens, int requests,
                             int channels, int width, int max_query_len, int silu, void* y,
                             hipStream_t stream) {
  if (dtype != DK_KV_F16 && dtype != DK_KV_BF16)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "x must be fp16 or bf16");
  if (num_tokens < 0 || requests < 0 || channels < 0)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "num_tokens, requests and channels must be >= 0");
  if (width < 2 || width > 4)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "width=%d must be 2, 3 or 4", width);
  if (max_query_len < 1)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "max_query_len must be >= 1");
  if (!offsets && num_tokens != requests)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT,
                         "without offsets each request has one token: num_tokens must be requests");
  if (num_tokens == 0 || channels == 0) return DK_OK;
  if (!x || !weight || !y || (requests > 0 && !windows))
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "short_conv's arrays must not be NULL");
  if (!aligned(x, 2) || !aligned(weight, 2) || !aligned(bias, 2) || !aligned(windows, 2) ||
      !aligned(y, 2) || !aligned(held, 4) || !aligned(offsets, 4))
    return dk::set_error(DK_ERR_INVALID_ARGUMENT,
                         "short_conv's arrays must be aligned as their elements");
  const bool wide = channels % 8 == 0 && x_token_stride % 8 == 0 && aligned(x, 16) &&
                    aligned(weight, 16) && aligned(windows, 16) && aligned(y, 16);
  const long long blocks = ((long long)channels - 1) / (wide ? 2048 : 256) + 1;
  // Tokens of a request that a workgroup takes. Where there are many, 8: each
  // input is read 11 times in 8, not 7 in 4 (8192 tokens of 8192 channels 50.6
  // against 55.8 us; with 16 fewer loads are on their way at once, 60.2). Where 8
  // would leave the chip few workgroups, or requests have few tokens, 4 (4100
  // tokens of 1544 channels 10.1 against 11.5 us).
  const int tile = !offsets ? 1 : max_query_len <= 4 || (long long)num_tokens / 8 * blocks < 1024 ? 4 : 8;
  const long long tiles = offsets ? (long long)num_tokens / tile + requests + 1 : requests;
  if (!dk::fits_launch(tiles, 256) || blocks > 65535)
    return dk::set_error(DK_ERR_UNSUPPORTED, "too many tokens or channels for one call");
  const dk::ConvArgs a{static_cast<const uint16_t*>(x), x_token_stride,
                       static_cast<const uint16_t*>(weight), static_cast<const uint16_t*>(bias),
                       static_cast<uint16_t*>(windows), held, offsets, static_cast<uint16_t*>(y),
                       num_tokens, requests, channels, silu};
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, (unsigned)blocks), dim3(256), 0, stream, a);
  };
  auto pick = [&](auto bf16, auto w) {
    constexpr bool b = decltype(bf16)::value;
    constexpr int n = decltype(w)::value;
    if (tile == 1) wide ? launch(dk::short_conv_kernel<n, 1, b, true>) : launch(dk::short_conv_kernel<n, 1, b, false>);
    else if (tile == 4) wide ? launch(dk::short_conv_kernel<n, 4, b, true>) : launch(dk::short_conv_kernel<n, 4, b, false>);
    else wide ? launch(dk::short_conv_kernel<n, 8, b, true>) : launch(dk::short_conv_kernel<n, 8, b, false>);
  };
  auto by_width = [&](auto bf16) {
    if (width == 2) pick(bf16, std::integral_constant<int, 2>{});
    else if (width == 3) pick(bf16, std::integral_constant<int, 3>{});
    else pick(bf16, std::integral_constant<int, 4>{});
  };
  dtype == DK_KV_BF16 ? by_width(std::true_type{}) : by_width(std::false_type{});
  return dk::check_launch("short_conv launch");
}
