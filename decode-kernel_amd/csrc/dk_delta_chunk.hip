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
  h8_t* k;    // [slot][qk head][4][dk / 32][64]   K', rows = tokens
  h8_t* q;    // [slot][qk head][4][dk / 32][64]   Q'
  h8_t* kt;   // [slot][qk head][dk / 16][2][64]   K' transposed, rows = elements
  h8_t* t;    // [slot][v head][6][2][64]          T' * 512: first and second part
  h8_t* p;    // [slot][v head][6][2][64]          P * 64, of q' and k'
  float* s;   // [slot][v head][kFactors * 64]     the rows' factors
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

// x as two fp16 parts.
__device__ __forceinline__ void split2(float x, _Float16* hi, _Float16* lo) {
  *hi = (_Float16)x;
  *lo = (_Float16)(x - (float)*hi);
}

// The power of two that brings a column's largest (over this lane's values and
// those of the lanes 16, 32 and 48 away) to 2^14 .. 2^15, as an exponent.
__device__ __forceinline__ int column_shift(float m) {
  m = fmaxf(m, __shfl_xor(m, 16));
  m = fmaxf(m, __shfl_xor(m, 32));
  return min(14 - exponent_of(m), 126);
}

__device__ __forceinline__ float max4(float m, f4_t x) {
  return fmaxf(fmaxf(m, fmaxf(fabsf(x[0]), fabsf(x[1]))), fmaxf(fabsf(x[2]), fabsf(x[3])));
}

// Two stacked result tiles as an operand B of 32 rows, in two parts.
__device__ __forceinline__ void split_tiles(f4_t x, f4_t y, float scale, h8_t* hi, h8_t* lo) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    _Float16 h, l;
    split2(x[j] * scale, &h, &l);
    (*hi)[j] = h;
    (*lo)[j] = l;
    split2(y[j] * scale, &h, &l);
    (*hi)[4 + j] = h;
    (*lo)[4 + j] = l;
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
  const size_t qk_at = (slot * a.qk_heads + hq) * (4 * kS * 64);
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
    float* f = ws.s + (slot * a.v_heads + h) * (kFactors * kChunk) + lane;
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
  const size_t v_at = (slot * a.v_heads + h) * (kFragments * 2 * 64);
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
// One wave 16 columns of one head's state, through a request's chunks.
// ---------------------------------------------------------------------------
template <int kDk, bool kBf16>
__global__ __launch_bounds__(64, 1) void delta_scan_kernel(DeltaArgs a, ChunkSpace ws, int value_size) {
  constexpr int kS = kDk / 32, kTiles = kDk / 16;
  constexpr int kType = kBf16 ? DK_KV_BF16 : DK_KV_F16;
  constexpr f4_t kZero{0.f, 0.f, 0.f, 0.f};
  const int lane = threadIdx.x, i = lane & 15, q4 = lane >> 4;
  const int h = blockIdx.x % a.v_heads, hq = h / a.group, b = blockIdx.y;
  const int col = (blockIdx.x / a.v_heads) * 16 + i;
  if (!wave_offsets_ok(a.offsets, a.requests, a.tokens)) return;
  const int from = a.offsets[b], n = a.offsets[b + 1] - from;
  if (n <= a.limit) return;
  const long long slot0 = from / kChunk + b;

  float* state = a.states + ((long long)b * a.v_heads + h) * kDk * value_size + col;
  f4_t s[kTiles];
  const bool fresh = a.held && a.held[b] <= 0;
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[t][e] = fresh ? 0.f : state[(long long)(16 * t + 4 * q4 + e) * value_size];

  const int chunks = (n + kChunk - 1) / kChunk;
  for (int c = 0; c < chunks; ++c) {
    const long long slot = slot0 + c;
    const int row0 = from + c * kChunk, count = min(kChunk, n - c * kChunk);
    const size_t qk_at = (slot * a.qk_heads + hq) * (4 * kS * 64) + lane;
    const size_t v_at = (slot * a.v_heads + h) * (kFragments * 2 * 64) + lane;
    const float* f = ws.s + (slot * a.v_heads + h) * (kFactors * kChunk);

    // K' S and Q' S.
    float m = 0.f;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) m = max4(m, s[t]);
    int shift = column_shift(m);
    float up = power2(shift), down = power2(-shift);
    f4_t x[4] = {kZero, kZero, kZero, kZero}, o[4] = {kZero, kZero, kZero, kZero};
#pragma unroll
    for (int t = 0; t < kS; ++t) {
      h8_t hi, lo;
      split_tiles(s[2 * t], s[2 * t + 1], up, &hi, &lo);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const h8_t kf = ws.k[qk_at + (y * kS + t) * 64], qf = ws.q[qk_at + (y * kS + t) * 64];
        x[y] = mfma(kf, hi, x[y]);
        x[y] = mfma(kf, lo, x[y]);
        o[y] = mfma(qf, hi, o[y]);
        o[y] = mfma(qf, lo, o[y]);
      }
    }
    // What each token finds wrong in the state before the chunk.
    m = 0.f;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const f4_t b1 = *reinterpret_cast<const f4_t*>(f + 16 * y + 4 * q4);
      const f4_t b2 = *reinterpret_cast<const f4_t*>(f + 64 + 16 * y + 4 * q4);
      const f4_t since = *reinterpret_cast<const f4_t*>(f + 128 + 16 * y + 4 * q4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 16 * y + 4 * q4 + e;
        float v = 0.f;
        if (r < count) v = pair_lo<kBf16>(a.v[(long long)(row0 + r) * a.v_token + (long long)h * a.v_head + col]);
        x[y][e] = b1[e] * v - b2[e] * (down * x[y][e]);
        o[y][e] *= since[e] * down;
      }
      m = max4(m, x[y]);
    }
    // The corrections w.
    shift = column_shift(m);
    up = power2(shift);
    h8_t hi[2], lo[2];
    split_tiles(x[0], x[1], up, &hi[0], &lo[0]);
    split_tiles(x[2], x[3], up, &hi[1], &lo[1]);
    down = power2(-shift) / kInverseScale;
    f4_t w[4] = {kZero, kZero, kZero, kZero};
    m = 0.f;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
#pragma unroll
      for (int t = 0; t <= y / 2; ++t) {
        const int piece = (y == 0 ? 0 : y == 1 ? 1 : y == 2 ? 2 : 4) + t;
        const h8_t th = ws.t[v_at + (2 * piece) * 64], tl = ws.t[v_at + (2 * piece + 1) * 64];
        w[y] = mfma(th, hi[t], w[y]);
        w[y] = mfma(th, lo[t], w[y]);
        w[y] = mfma(tl, hi[t], w[y]);
      }
      w[y] *= down;
      m = max4(m, w[y]);
    }
    // Out.
    shift = column_shift(m);
    up = power2(shift);
    down = power2(-shift) / kScoreScale;
    split_tiles(w[0], w[1], up, &hi[0], &lo[0]);
    split_tiles(w[2], w[3], up, &hi[1], &lo[1]);
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const f4_t d = *reinterpret_cast<const f4_t*>(f + 192 + 16 * y + 4 * q4);
      f4_t p = kZero;
#pragma unroll
      for (int t = 0; t <= y / 2; ++t) {
        const int piece = (y == 0 ? 0 : y == 1 ? 1 : y == 2 ? 2 : 4) + t;
        const h8_t ph = ws.p[v_at + (2 * piece) * 64], pl = ws.p[v_at + (2 * piece + 1) * 64];
        p = mfma(ph, hi[t], p);
        p = mfma(ph, lo[t], p);
        p = mfma(pl, hi[t], p);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 16 * y + 4 * q4 + e;
        if (r < count)
          a.out[((long long)(row0 + r) * a.v_heads + h) * value_size + col] =
              to_half_bits<kType>(d[e] * fmaf(p[e], down, o[y][e]));
      }
    }
    // The state after the chunk.
    m = 0.f;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const f4_t until = *reinterpret_cast<const f4_t*>(f + 256 + 16 * y + 4 * q4);
      w[y] *= until;
      m = max4(m, w[y]);
    }
    shift = column_shift(m);
    up = power2(shift);
    down = power2(-shift);
    split_tiles(w[0], w[1], up, &hi[0], &lo[0]);
    split_tiles(w[2], w[3], up, &hi[1], &lo[1]);
    const float whole = f[320];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      f4_t add = kZero;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const h8_t kt = ws.kt[qk_at + (2 * t + y) * 64];
        add = mfma(kt, hi[y], add);
        add = mfma(kt, lo[y], add);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][e] = fmaf(add[e], down, whole * s[t][e]);
    }
  }
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) state[(long long)(16 * t + 4 * q4 + e) * value_size] = s[t][e];
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
  const dim3 columns((unsigned)(a.v_heads * (value_size / 16)), (unsigned)a.requests);
  auto launch = [&](auto prepare, auto scan) {
    hipLaunchKernelGGL(prepare, chunks, dim3(256), 0, stream, a, ws);
    hipLaunchKernelGGL(scan, columns, dim3(64), 0, stream, a, ws, value_size);
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
