// The gated delta rule over long prompts, 64 tokens at a time.
//
// Inside a chunk with the state S before it, G_i = the sum of the logarithms
// of the decays up to token i, and the rule's corrections u_i = beta_i (v_i -
// (what the state before token i gives for k_i)):
//   (1 + A) u = beta v - beta e^G (K S),   A_ij = beta_i e^(G_i - G_j) k_i.k_j  (j < i)
//   out_i     = e^(G_i) q_i S + sum_(j <= i) e^(G_i - G_j) (q_i.k_j) u_j
//   S_after   = e^(G_last) S + sum_j e^(G_last - G_j) k_j u_j
// so a chunk is a few products of matrices. What does not depend on the state
// (T = (1 + A)^-1, P = the decayed q.k, and the operands in the order that the
// matrix instructions read them) is computed for all chunks at once by
// delta_prepare_kernel; delta_scan_kernel then goes through a request's
// chunks one after another, with the state in registers.
//
// Precision: the state is fp32 and keeps what 32-bit products would give. The
// matrix cores take fp16, so an fp32 operand goes in as two fp16 parts, 22
// bits together, after its column (one element of v's axis) was scaled by a
// power of two to just below fp16's top: a part's own range then reaches 2^-39
// of the column's largest. Keys and queries are exact in one part: a row is
// scaled by a power of two (k = 2^e k'), which takes bf16's range away and
// leaves its 8 bits. The power and the length that a row is divided by go into
// the rows' factors: with c_i = 2^e / |k_i| and w_i = c_i u_i,
//   A'_ij = beta_i c_i^2 e^(G_i - G_j) k'_i.k'_j,
//   w = T' (beta c v - beta c^2 e^G (K' S)),  S_after = e^G_last S + sum_j k'_j (e^(..) w_j).
#include <hip/hip_runtime.h>

#include "dk_delta.hpp"
#include "dk_host.hpp"

namespace dk {

namespace {

// What T and P are multiplied by before they become two fp16 parts, so that the
// second part of a small entry is not lost below fp16's smallest: elements of
// k' and q' are under 2, so P stays under 4 * 128 * 64 = 2^15, and T under 2 *
// 22.7 * 512 = 2^14.5 where beta |k|^2 is at most 2 (an entry is at most beta
// |k_i| |k_j| in the rule's own keys, and k' of 1 to 22.7 in length).
constexpr float kInverseScale = 512.f, kScoreScale = 64.f;
constexpr int kFragments = 6;  // 16 x 32 pieces of a lower triangle of 64: (0,0) (1,0) (2,0) (2,1) (3,0) (3,1)

// The prepared operands of a chunk, as matrix operands A: for a piece of 16
// rows and 32 columns lane l holds row l % 16 and the columns 4 q .. 4 q + 3
// and 16 + 4 q .. 16 + 4 q + 3 of q = l / 16, which are the rows that the
// lane's 4 values of two stacked result tiles stand in: a product's result is
// the next one's operand B as it stands.
struct ChunkSpace {
  h8_t* k;    // [qk head][slot][4][dk / 32][64]   K', rows = tokens
  h8_t* q;    // [qk head][slot][4][dk / 32][64]   Q'
  h8_t* kt;   // [qk head][slot][dk / 16][2][64]   K' transposed, rows = elements
  h8_t* t;    // [v head][slot][6][2][64]          T' * 512: first and second part
  h8_t* p;    // [v head][slot][6][2][64]          P * 64, of q' and k'
  float* s;   // [v head][slot][kFactors * 64]     the rows' factors
  long long slots;
};
constexpr int kFactors = 6;  // beta c, beta c^2 e^G, e^G, d, e^(G_last - G), e^G_last (all alike)

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

long long slots_of(int tokens, int requests) { return (long long)tokens / kChunk + requests; }

ChunkSpace chunk_space(void* workspace, int tokens, int requests, int qk_heads, int v_heads, int dk,
                       size_t* bytes) {
  const size_t slots = (size_t)slots_of(tokens, requests);
  char* at = static_cast<char*>(workspace);
  auto take = [&](size_t n) {
    char* p = at;
    at += up256(n);
    return p;
  };
  ChunkSpace c;
  const size_t rows = slots * qk_heads * kChunk * dk * 2, lower = slots * v_heads * kFragments * 2 * 1024;
  c.k = reinterpret_cast<h8_t*>(take(rows));
  c.q = reinterpret_cast<h8_t*>(take(rows));
  c.kt = reinterpret_cast<h8_t*>(take(rows));
  c.t = reinterpret_cast<h8_t*>(take(lower));
  c.p = reinterpret_cast<h8_t*>(take(lower));
  c.s = reinterpret_cast<float*>(take(slots * v_heads * kFactors * kChunk * 4));
  c.slots = (long long)slots;
  *bytes = (size_t)(at - static_cast<char*>(workspace));
  return c;
}

__device__ __forceinline__ f4_t mfma(h8_t a, h8_t b, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f4_t mfma32(float a, float b, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ int exponent_of(float m) {
  return (int)(__builtin_bit_cast(uint32_t, m) >> 23 & 0xFF) - 127;
}

__device__ __forceinline__ float power2(int e) {  // -126 <= e <= 127
  return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}

// The largest over the lanes l, l + 16, l + 32 and l + 48.
__device__ __forceinline__ float max_rows(float m) {
  const uint32_t x = __builtin_bit_cast(uint32_t, m);
  const auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  const float y = fmaxf(__builtin_bit_cast(float, (uint32_t)p[0]), __builtin_bit_cast(float, (uint32_t)p[1]));
  const uint32_t z = __builtin_bit_cast(uint32_t, y);
  const auto q = __builtin_amdgcn_permlane32_swap(z, z, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)q[0]), __builtin_bit_cast(float, (uint32_t)q[1]));
}

// The power of two that brings a column's largest (over this lane's values and
// those of the lanes 16, 32 and 48 away) to 2^14 .. 2^15, as an exponent.
__device__ __forceinline__ int column_shift(float m) { return min(14 - exponent_of(max_rows(m)), 126); }

__device__ __forceinline__ float max4(float m, f4_t x) {
  m = fmaxf(fmaxf(m, fabsf(x[0])), fabsf(x[1]));
  return fmaxf(fmaxf(m, fabsf(x[2])), fabsf(x[3]));
}

// Two stacked result tiles times a power of two as an operand B of 32 rows, in
// two fp16 parts of one rounding each.
__device__ __forceinline__ void split_tiles(f4_t x, f4_t y, float scale, h8_t* hi, h8_t* lo) {
  const float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    // As one instruction of mixed width, not a product and a conversion.
    const _Float16 h = (_Float16)fmaf(v[j], scale, 0.f);
    (*hi)[j] = h;
    (*lo)[j] = (_Float16)fmaf(v[j], scale, -(float)h);
  }
}

// ---------------------------------------------------------------------------
// One workgroup a chunk and head; wave w has its rows 16 w .. 16 w + 15.
// ---------------------------------------------------------------------------
constexpr int kPad = 68;  // floats a row of 64 takes in LDS

template <int kDk, bool kBf16>
__global__ __launch_bounds__(256) void delta_prepare_kernel(DeltaArgs a, ChunkSpace ws) {
  constexpr int kS = kDk / 32;
  __shared__ h8_t keys[4][kS][64];
  __shared__ float m[kChunk][kPad];
  __shared__ float c_of[kChunk], d_of[kChunk], hi_of[kChunk], lo_of[kChunk], b2_of[kChunk];
  __shared__ int found[2];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, i = lane & 15, q4 = lane >> 4;
  const long long slot = blockIdx.x / a.v_heads;
  const int h = blockIdx.x % a.v_heads, hq = h / a.group;
  Tile tile;
  if (!find_tile(a.offsets, a.requests, a.tokens, kChunk, (int)slot, found, &tile)) return;
  if (tile.request < 0) return;
  if (a.offsets[tile.request + 1] - a.offsets[tile.request] <= a.limit) return;
  const bool first_of_group = h % a.group == 0;

  // Rows of keys and queries, scaled to fp16.
  const int r = 16 * wave + i;
  const bool real = r < tile.count;
  h8_t kf[kS], qf[kS];
  auto rows = [&](const uint16_t* x, h8_t(&f)[kS], float* length2) {
    uint2 raw[kS][2];
#pragma unroll
    for (int s = 0; s < kS; ++s)
#pragma unroll
      for (int p = 0; p < 2; ++p)
        raw[s][p] = real ? *reinterpret_cast<const uint2*>(x + 32 * s + 16 * p + 4 * q4) : make_uint2(0u, 0u);
    float top = 0.f, sum = 0.f;
#pragma unroll
    for (int s = 0; s < kS; ++s)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const float e[4] = {pair_lo<kBf16>(raw[s][p].x), pair_hi<kBf16>(raw[s][p].x),
                            pair_lo<kBf16>(raw[s][p].y), pair_hi<kBf16>(raw[s][p].y)};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          top = fmaxf(top, fabsf(e[j]));
          sum = fmaf(e[j], e[j], sum);
        }
      }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    const int e2 = exponent_of(top);
#pragma unroll
    for (int s = 0; s < kS; ++s)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        f[s][4 * p] = (_Float16)ldexpf(pair_lo<kBf16>(raw[s][p].x), -e2);
        f[s][4 * p + 1] = (_Float16)ldexpf(pair_hi<kBf16>(raw[s][p].x), -e2);
        f[s][4 * p + 2] = (_Float16)ldexpf(pair_lo<kBf16>(raw[s][p].y), -e2);
        f[s][4 * p + 3] = (_Float16)ldexpf(pair_hi<kBf16>(raw[s][p].y), -e2);
      }
    *length2 = sum;
    return top == 0.f ? INT32_MIN : e2;  // NaN has an exponent too
  };
  const long long row = tile.row + (real ? r : 0);
  float kk, qq;
  const int ke = rows(a.k + row * a.k_token + (long long)hq * a.k_head, kf, &kk);
  const int qe = rows(a.q + row * a.q_token + (long long)hq * a.q_head, qf, &qq);
  float c = 0.f, d = 0.f;  // a row of zeros has no part in anything
  if (ke != INT32_MIN) c = ldexpf(a.normalize ? 1.f / sqrtf(kk + kUnitEps) : 1.f, ke);
  if (qe != INT32_MIN) d = ldexpf(a.normalize ? a.scale / sqrtf(qq + kUnitEps) : a.scale, qe);
  const size_t qk_at = (hq * ws.slots + slot) * (4 * kS * 64);
#pragma unroll
  for (int s = 0; s < kS; ++s) {
    keys[wave][s][lane] = kf[s];
    if (first_of_group) {
      ws.k[qk_at + (wave * kS + s) * 64 + lane] = kf[s];
      ws.q[qk_at + (wave * kS + s) * 64 + lane] = qf[s];
    }
  }
  if (q4 == 0) {
    c_of[r] = c;
    d_of[r] = d;
  }
  __syncthreads();

  // Sums of the decays' logarithms, in 64 bits: a sum's difference to another
  // has to be exact where both are large. Kept as two fp32, to the base 2.
  if (wave == 0) {
    const bool live = lane < tile.count;
    const long long at = (long long)(tile.row + (live ? lane : 0)) * a.v_heads + h;
    const float beta = live ? a.beta[at] : 0.f;
    double g = live ? (double)cut_log(a.log_decay[at]) : 0.0;
#pragma unroll
    for (int dd = 1; dd < 64; dd *= 2) {
      const double o = __shfl_up(g, dd);
      if (lane >= dd) g += o;
    }
    g *= 1.4426950408889634074;  // log2(e)
    const double rest = __shfl(g, 63) - g;
    const float hi = (float)g, lo = (float)(g - (double)hi);
    const float cc = c_of[lane], since = exp2f(hi) * fmaf(lo, 0.69314718f, 1.f);
    const float until = exp2f((float)rest);
    hi_of[lane] = hi;
    lo_of[lane] = lo;
    b2_of[lane] = beta * cc * cc;
    float* f = ws.s + (h * ws.slots + slot) * (kFactors * kChunk) + lane;
    f[0] = beta * cc;
    f[64] = beta * cc * cc * since;
    f[128] = since;
    f[192] = d_of[lane];
    f[256] = until;
    f[320] = __shfl(since, 63);
  }
  // The transposed keys, element by element out of the operands' order.
  if (first_of_group) {
    const uint16_t* flat = reinterpret_cast<const uint16_t*>(&keys[0][0][0]);
    for (int f = wave; f < kDk / 16 * 2; f += 4) {
      const int e = 16 * (f >> 1) + i;  // the element
      union {
        uint16_t u[8];
        h8_t v;
      } x;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int t = 32 * (f & 1) + 16 * (j >> 2) + 4 * q4 + (j & 3);
        x.u[j] = flat[(((t >> 4) * kS + (e >> 5)) * 64 + (t & 15) + 16 * ((e & 15) >> 2)) * 8 +
                      ((e >> 4) & 1) * 4 + (e & 3)];
      }
      ws.kt[qk_at + f * 64 + lane] = x.v;
    }
  }
  f4_t kkt[4], qkt[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    kkt[j] = qkt[j] = f4_t{0.f, 0.f, 0.f, 0.f};
    if (j <= wave) {
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        const h8_t b = keys[j][s][lane];
        kkt[j] = mfma(kf[s], b, kkt[j]);
        qkt[j] = mfma(qf[s], b, qkt[j]);
      }
    }
  }
  __syncthreads();

  // Decayed products: P to LDS and out; A stays here.
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int col = 16 * j + i;
    const float hc = hi_of[col], lc = lo_of[col];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int rr = 16 * wave + 4 * q4 + e;
      const float decay = exp2f((hi_of[rr] - hc) + (lo_of[rr] - lc));
      m[rr][col] = rr >= col ? decay * qkt[j][e] : 0.f;
      kkt[j][e] = rr > col ? b2_of[rr] * decay * kkt[j][e] : 0.f;
    }
  }
  const size_t v_at = (h * ws.slots + slot) * (kFragments * 2 * 64);
  const int piece0 = wave == 0 ? 0 : wave == 1 ? 1 : wave == 2 ? 2 : 4;
  auto pieces_out = [&](h8_t* to, float scale) {
    for (int s = 0; s <= wave / 2; ++s) {
      h8_t hi, lo;
      const f4_t x = *reinterpret_cast<const f4_t*>(&m[16 * wave + i][32 * s + 4 * q4]);
      const f4_t y = *reinterpret_cast<const f4_t*>(&m[16 * wave + i][32 * s + 16 + 4 * q4]);
      split_tiles(x, y, scale, &hi, &lo);
      to[v_at + (2 * (piece0 + s)) * 64 + lane] = hi;
      to[v_at + (2 * (piece0 + s) + 1) * 64 + lane] = lo;
    }
  };
  __syncthreads();
  pieces_out(ws.p, kScoreScale);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) m[16 * wave + 4 * q4 + e][16 * j + i] = kkt[j][e];
  __syncthreads();

  // T = (1 + A)^-1: the blocks of 16 on the diagonal by substitution, a lane a
  // column, then the blocks below from them, a wave a column of blocks, with
  // 32-bit matrix products:  T_ij = -T_ii sum_(j <= k < i) A_ik T_kj.
  {
    float t[16];
    const int base = 16 * wave;
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      float sum = x == i ? 1.f : 0.f;
#pragma unroll
      for (int k = 0; k < x; ++k) sum = fmaf(-m[base + x][base + k], t[k], sum);
      t[x] = sum;
    }
    __builtin_amdgcn_wave_barrier();
    if (q4 == 0)
#pragma unroll
      for (int x = 0; x < 16; ++x) m[base + x][base + i] = t[x];
  }
  __syncthreads();
  f4_t below[4];
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    if (wave != j) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) below[j][e] = m[16 * j + 4 * q4 + e][16 * j + i];
#pragma unroll
    for (int x = j + 1; x < 4; ++x) {
      f4_t sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = j; k < x; ++k) {
        const f4_t ak = *reinterpret_cast<const f4_t*>(&m[16 * x + i][16 * k + 4 * q4]);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = mfma32(ak[e], below[k][e], sum);
      }
      const f4_t tx = *reinterpret_cast<const f4_t*>(&m[16 * x + i][16 * x + 4 * q4]);
      f4_t got{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e) got = mfma32(tx[e], sum[e], got);
      below[x] = -got;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    if (wave != j) continue;
#pragma unroll
    for (int x = j + 1; x < 4; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) m[16 * x + 4 * q4 + e][16 * j + i] = below[x][e];
  }
  __syncthreads();
  pieces_out(ws.t, kInverseScale);
}

// ---------------------------------------------------------------------------
// A request's chunks one after another, 32 columns of one head's state a
// workgroup. Waves 0 and 1 hold 16 columns each and go from state to state;
// columns do not meet, and a result tile is the next product's operand B, so
// nothing but the prepared operands comes from outside a wave. Waves 2 and 3
// compute the same columns' outputs one chunk behind, from the parts of the
// state and of the corrections that waves 0 and 1 leave in LDS, and bring the
// next chunk's operands there: what only the outputs need is off the chain
// that bounds a long prompt.
// ---------------------------------------------------------------------------
constexpr int kScanTiles = 2;  // tiles of 16 columns a workgroup holds

using lds_ptr = __attribute__((address_space(3))) void*;

// Buffers: a chunk's rows behind the request's last are out of their range, so
// that they load zeros and store nothing.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}

__device__ __forceinline__ h8_t load_piece(__amdgpu_buffer_rsrc_t r, uint32_t offset) {
  return __builtin_bit_cast(h8_t, __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 0));
}

template <int kDk, bool kBf16>
__global__ __launch_bounds__(256, 1) void delta_scan_kernel(DeltaArgs a, ChunkSpace ws, int value_size) {
  constexpr int kS = kDk / 32, kTiles = kDk / 16;
  constexpr int kType = kBf16 ? DK_KV_BF16 : DK_KV_F16;
  constexpr int kKeys = 4 * kS, kInverse = 2 * kFragments, kTurned = 2 * kTiles;  // pieces of 1 KB
  constexpr f4_t kZero{0.f, 0.f, 0.f, 0.f};
  __shared__ h8_t stage[2][kKeys + kInverse + kTurned][64];
  __shared__ h8_t left_s[2][kScanTiles][2 * kS][64];  // the state's parts
  __shared__ h8_t left_w[2][kScanTiles][4][64];       // the corrections'
  __shared__ float left_scale[2][kScanTiles][2][16];  // what both are divided by
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, i = lane & 15, q4 = lane >> 4;
  const int tile = wave & 1;
  const int h = blockIdx.x % a.v_heads, hq = h / a.group, b = blockIdx.y;
  const int col = ((blockIdx.x / a.v_heads) * kScanTiles + tile) * 16 + i;
  if (!wave_offsets_ok(a.offsets, a.requests, a.tokens)) return;
  const int from = a.offsets[b], n = a.offsets[b + 1] - from;
  if (n <= a.limit) return;
  const long long slot0 = from / kChunk + b;
  const int chunks = (n + kChunk - 1) / kChunk;
  // A chunk's operands and factors, whole pieces of 1 KB, 16 bytes a lane.
  constexpr uint32_t kQkBytes = kKeys * 1024, kVBytes = kInverse * 1024, kFactorBytes = kFactors * kChunk * 4;
  auto of_qk = [&](const h8_t* base, int c) {
    return buffer_of(reinterpret_cast<const char*>(base) + (hq * ws.slots + slot0 + c) * kQkBytes, kQkBytes);
  };
  auto of_v = [&](const h8_t* base, int c) {
    return buffer_of(reinterpret_cast<const char*>(base) + (h * ws.slots + slot0 + c) * kVBytes, kVBytes);
  };
  auto of_factors = [&](int c) {
    return buffer_of(reinterpret_cast<const char*>(ws.s) + (h * ws.slots + slot0 + c) * kFactorBytes, kFactorBytes);
  };
  const uint32_t piece_at = lane * 16;
  auto rows4 = [&](__amdgpu_buffer_rsrc_t r, int which, int y) {
    return __builtin_bit_cast(
        f4_t, __builtin_amdgcn_raw_buffer_load_b128(r, 16 * q4 + (which * kChunk + 16 * y) * 4, 0, 0));
  };

  // Both output waves bring half of chunk c's operands.
  auto bring = [&](int c) {
    h8_t* to = &stage[c & 1][0][0];
    const auto keys = of_qk(ws.k, c), inverse = of_v(ws.t, c), turned = of_qk(ws.kt, c);
    auto one = [&](__amdgpu_buffer_rsrc_t r, int from, int piece) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(to + piece * 64), 16, piece_at + from * 1024, 0, 0, 0);
    };
#pragma unroll
    for (int p = 0; p < kKeys; p += 2) one(keys, p + tile, p + tile);
#pragma unroll
    for (int p = 0; p < kInverse; p += 2) one(inverse, p + tile, kKeys + p + tile);
#pragma unroll
    for (int p = 0; p < kTurned; p += 2) one(turned, p + tile, kKeys + kInverse + p + tile);
  };

  if (wave < 2) {
    float* state = a.states + ((long long)b * a.v_heads + h) * kDk * value_size + col;
    f4_t s[kTiles];
    const bool fresh = a.held && a.held[b] <= 0;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][e] = fresh ? 0.f : state[(long long)(16 * t + 4 * q4 + e) * value_size];
    // A chunk's rows are loaded as soon as those of the chunk before are used.
    const uint16_t* values = a.v + (long long)from * a.v_token + (long long)h * a.v_head;
    uint32_t v_at[16];
#pragma unroll
    for (int z = 0; z < 16; ++z) v_at[z] = ((16 * (z >> 2) + (z & 3) + 4 * q4) * (uint32_t)a.v_token + col) * 2;
    uint16_t v[16];
    f4_t b1[4], b2[4], until[4];
    auto load_values = [&](int c) {
      const uint32_t count = min(n - c * kChunk, kChunk);
      const auto rows = buffer_of(values + (long long)c * kChunk * a.v_token, ((count - 1) * (uint32_t)a.v_token + value_size) * 2);
      const auto f = of_factors(c);
#pragma unroll
      for (int z = 0; z < 16; ++z) v[z] = __builtin_amdgcn_raw_buffer_load_b16(rows, v_at[z], 0, 0);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        b1[y] = rows4(f, 0, y);
        b2[y] = rows4(f, 1, y);
      }
    };
    float whole;
    auto load_until = [&](int c) {
      const auto f = of_factors(c);
#pragma unroll
      for (int y = 0; y < 4; ++y) until[y] = rows4(f, 4, y);
      whole = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(f, 5 * kChunk * 4, 0, 0));
    };
    load_values(0);
    load_until(0);
    float top = 0.f;  // the largest of the state's values here
#pragma unroll
    for (int t = 0; t < kTiles; ++t) top = max4(top, s[t]);
    for (int c = 0; c <= chunks; ++c) {
      __syncthreads();  // chunk c's operands are there, and chunk c - 2's parts read
      if (c == chunks) break;
      const int after = min(c + 1, chunks - 1);
      const h8_t(*keys)[64] = &stage[c & 1][0];
      const h8_t(*inverse)[64] = &stage[c & 1][kKeys];
      const h8_t(*turned)[64] = &stage[c & 1][kKeys + kInverse];

      // Operands are read from LDS a product ahead: left to itself the compiler
      // reads two, waits for them and goes on, 22 times a chunk.
      h8_t kf[kKeys], tf[kInverse], uf[kTurned];
#pragma unroll
      for (int z = 0; z < kKeys; ++z) kf[z] = keys[z][lane];
      __builtin_amdgcn_sched_barrier(0);
      // K' S.
      int shift = column_shift(top);
      float up = power2(shift), down = power2(-shift);
      if (q4 == 0) left_scale[c & 1][tile][0][i] = down;
      f4_t x[4] = {kZero, kZero, kZero, kZero};
#pragma unroll
      for (int t = 0; t < kS; ++t) {
        h8_t hi, lo;
        split_tiles(s[2 * t], s[2 * t + 1], up, &hi, &lo);
        left_s[c & 1][tile][2 * t][lane] = hi;
        left_s[c & 1][tile][2 * t + 1][lane] = lo;
#pragma unroll
        for (int y = 0; y < 4; ++y) x[y] = mfma(kf[y * kS + t], hi, x[y]);
#pragma unroll
        for (int y = 0; y < 4; ++y) x[y] = mfma(kf[y * kS + t], lo, x[y]);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int z = 0; z < kInverse; ++z) tf[z] = inverse[z][lane];
      __builtin_amdgcn_sched_barrier(0);
      // What each token finds wrong in the state before the chunk.
      float m = 0.f;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[y][e] = b1[y][e] * pair_lo<kBf16>(v[4 * y + e]) - b2[y][e] * (down * x[y][e]);
        m = max4(m, x[y]);
      }
      load_values(after);
      // The corrections w = T x.
      shift = column_shift(m);
      up = power2(shift);
      down = power2(-shift) / kInverseScale;
      h8_t hi[2], lo[2];
      split_tiles(x[0], x[1], up, &hi[0], &lo[0]);
      split_tiles(x[2], x[3], up, &hi[1], &lo[1]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int z = 0; z < kTurned; ++z) uf[z] = turned[z][lane];
      __builtin_amdgcn_sched_barrier(0);
      f4_t w[4] = {kZero, kZero, kZero, kZero};
#pragma unroll
      for (int part = 0; part < 3; ++part)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int y = 2 * t; y < 4; ++y) {
            const int piece = (y == 0 ? 0 : y == 1 ? 1 : y == 2 ? 2 : 4) + t;
            w[y] = mfma(tf[2 * piece + (part == 2)], part == 1 ? lo[t] : hi[t], w[y]);
          }
      float m2 = 0.f;
      f4_t w2[4];
      m = 0.f;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        w[y] *= down;
        w2[y] = w[y] * until[y];
        m = max4(m, w[y]);
        m2 = max4(m2, w2[y]);
      }
      // The state after the chunk.
      shift = column_shift(m2);
      up = power2(shift);
      down = power2(-shift);
      split_tiles(w2[0], w2[1], up, &hi[0], &lo[0]);
      split_tiles(w2[2], w2[3], up, &hi[1], &lo[1]);
      top = 0.f;
#pragma unroll
      for (int t = 0; t < kTiles; t += 4) {
        f4_t add[4] = {kZero, kZero, kZero, kZero};
#pragma unroll
        for (int y = 0; y < 2; ++y) {
#pragma unroll
          for (int z = 0; z < 4; ++z) add[z] = mfma(uf[2 * (t + z) + y], hi[y], add[z]);
#pragma unroll
          for (int z = 0; z < 4; ++z) add[z] = mfma(uf[2 * (t + z) + y], lo[y], add[z]);
        }
#pragma unroll
        for (int z = 0; z < 4; ++z) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t + z][e] = fmaf(add[z][e], down, whole * s[t + z][e]);
          top = max4(top, s[t + z]);
        }
      }
      load_until(after);
      // The corrections for the outputs.
      shift = column_shift(m);
      up = power2(shift);
      if (q4 == 0) left_scale[c & 1][tile][1][i] = power2(-shift) / kScoreScale;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        split_tiles(w[2 * t], w[2 * t + 1], up, &hi[t], &lo[t]);
        left_w[c & 1][tile][2 * t][lane] = hi[t];
        left_w[c & 1][tile][2 * t + 1][lane] = lo[t];
      }
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) state[(long long)(16 * t + 4 * q4 + e) * value_size] = s[t][e];
  } else {
    uint16_t* out = a.out + ((long long)from * a.v_heads + h) * value_size;
    const uint32_t out_token = a.v_heads * value_size;
    uint32_t out_at[16];
#pragma unroll
    for (int z = 0; z < 16; ++z) out_at[z] = ((16 * (z >> 2) + (z & 3) + 4 * q4) * out_token + col) * 2;
    struct Operands {
      h8_t q[kKeys], p[kInverse];
    };
    // Outputs of chunk c - 1, whose operands are in `now`; chunk c's go to `next`,
    // so that all loads have a chunk's time to arrive.
    auto outputs = [&](int c, const Operands& now, Operands& next) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // bring()'s pieces are in LDS
      __syncthreads();
      if (c + 1 < chunks) bring(c + 1);
      if (c < chunks) {
        const auto qs = of_qk(ws.q, c), ps = of_v(ws.p, c);
#pragma unroll
        for (int z = 0; z < kKeys; ++z) next.q[z] = load_piece(qs, piece_at + z * 1024);
#pragma unroll
        for (int z = 0; z < kInverse; ++z) next.p[z] = load_piece(ps, piece_at + z * 1024);
      }
      if (c == 0) return;
      const int at = c - 1;
      f4_t x[4] = {kZero, kZero, kZero, kZero}, y2[4] = {kZero, kZero, kZero, kZero}, since[4], d[4];
      const auto f = of_factors(at);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        since[y] = rows4(f, 2, y);
        d[y] = rows4(f, 3, y);
      }
      const float down_s = left_scale[at & 1][tile][0][i], down_w = left_scale[at & 1][tile][1][i];
      h8_t sp[2 * kS], wp[4];
#pragma unroll
      for (int t = 0; t < 2 * kS; ++t) sp[t] = left_s[at & 1][tile][t][lane];
#pragma unroll
      for (int t = 0; t < 4; ++t) wp[t] = left_w[at & 1][tile][t][lane];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < 2 * kS; ++t)
#pragma unroll
        for (int y = 0; y < 4; ++y) x[y] = mfma(now.q[y * kS + t / 2], sp[t], x[y]);
#pragma unroll
      for (int part = 0; part < 3; ++part)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int y = 2 * t; y < 4; ++y) {
            const int piece = (y == 0 ? 0 : y == 1 ? 1 : y == 2 ? 2 : 4) + t;
            y2[y] = mfma(now.p[2 * piece + (part == 2)], wp[2 * t + (part == 1)], y2[y]);
          }
      const uint32_t count = min(n - at * kChunk, kChunk);
      const auto rows = buffer_of(out + (long long)at * kChunk * out_token, ((count - 1) * out_token + value_size) * 2);
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float o = d[y][e] * fmaf(y2[y][e], down_w, since[y][e] * down_s * x[y][e]);
          __builtin_amdgcn_raw_buffer_store_b16(to_half_bits<kType>(o), rows, out_at[4 * y + e], 0, 0);
        }
    };
    bring(0);
    Operands even, odd;  // of chunks c - 1 and c, in turn
    for (int c = 0; c <= chunks; c += 2) {
      outputs(c, odd, even);
      if (c + 1 <= chunks) outputs(c + 1, even, odd);
    }
  }
}

}  // namespace

size_t delta_chunk_bytes(int num_tokens, int requests, int qk_heads, int v_heads, int key_size) {
  size_t bytes;
  chunk_space(nullptr, num_tokens, requests, qk_heads, v_heads, key_size, &bytes);
  return bytes;
}

int delta_chunk_launch(const DeltaArgs& a, int key_size, int value_size, bool bf16, void* workspace,
                       hipStream_t stream) {
  size_t bytes;
  const ChunkSpace ws = chunk_space(workspace, a.tokens, a.requests, a.qk_heads, a.v_heads, key_size, &bytes);
  const dim3 chunks((unsigned)(slots_of(a.tokens, a.requests) * a.v_heads));
  const dim3 columns((unsigned)(a.v_heads * (value_size / (16 * kScanTiles))), (unsigned)a.requests);
  auto launch = [&](auto prepare, auto scan) {
    hipLaunchKernelGGL(prepare, chunks, dim3(256), 0, stream, a, ws);
    hipLaunchKernelGGL(scan, columns, dim3(256), 0, stream, a, ws, value_size);
  };
  if (key_size == 64)
    bf16 ? launch(delta_prepare_kernel<64, true>, delta_scan_kernel<64, true>)
         : launch(delta_prepare_kernel<64, false>, delta_scan_kernel<64, false>);
  else
    bf16 ? launch(delta_prepare_kernel<128, true>, delta_scan_kernel<128, true>)
         : launch(delta_prepare_kernel<128, false>, delta_scan_kernel<128, false>);
  return check_launch("delta_rule launch");
}

}  // namespace dk
