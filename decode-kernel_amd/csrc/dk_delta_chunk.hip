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
// matrix cores take 16 bits, and what stands behind a sum decides how an fp32
// operand goes in.
//  - Where all terms of a sum belong to one moment (the state in K S and Q S, the
//    corrections that are added to it, decayed to the chunk's end), what counts is
//    the largest of a column (one element of v's axis): two fp16 parts, 22 bits
//    together, after the column was scaled by a power of two to just below fp16's
//    top; their range reaches 2^-39 of the column's largest.
//  - Where a sum goes over tokens (T and what it multiplies, P and the
//    corrections), a decay of 2^-40 may meet a value 2^40 times its neighbours', and
//    neither has a scale that fits the others: three bf16 parts, which
//    are the fp32 number in all its bits and all its range. Of the nine products of
//    parts the six largest are taken, which leaves 2^-24 of a term.
//  - Keys and queries are one fp16 part: a row is scaled by a power of two (k = 2^e
//    k') that brings its largest to 1 .. 2, and elements keep all of their bits
//    down to 2^-14 (fp16's 11) or 2^-17 (bf16's 8) of that, below it 2^-25 of it.
// The power and the length that a row is divided by go into the rows' factors: with
// c_i = 2^e / |k_i| and w_i = c_i u_i,
//   A'_ij = beta_i c_i^2 e^(G_i - G_j) k'_i.k'_j,
//   w = T' (beta c v - beta c^2 e^G (K' S)),  S_after = e^G_last S + sum_j k'_j (e^(..) w_j).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "dk_delta.hpp"
#include "dk_host.hpp"

namespace dk {

namespace {

typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));

// A lower triangle of 64 as pieces of 16 rows (tile y) and 32 columns (from 32 t): in
// 1 .. 4 (1,0) (2,0) (3,0) (3,1), and in 0 what there is of (0,0) and (2,1), the 16
// columns up to the diagonal: a lane's first 8 bytes are of the one and its last of the
// other. Without the empty halves the operands of 8192 tokens of 32 heads are 200 MB,
// not 225, and a chunk's factors one piece, not two: 255 us instead of 287.
constexpr int kTriangle = 5;
constexpr int kParts = 3;  // bf16 parts of an entry of T and P

// The prepared operands of a chunk, as matrix operands A: for a piece of 16
// rows and 32 columns lane l holds row l % 16 and the columns 4 q .. 4 q + 3
// and 16 + 4 q .. 16 + 4 q + 3 of q = l / 16, which are the rows that the
// lane's 4 values of two stacked result tiles stand in: a product's result is
// the next one's operand B as it stands.
struct ChunkSpace {
  h8_t* k;    // [qk head][slot][4][dk / 32][64]   K', rows = tokens
  h8_t* q;    // [qk head][slot][4][dk / 32][64]   Q'
  b8_t* t;    // [v head][slot][kTriangle][kParts][64]  T'
  b8_t* p;    // [v head][slot][kTriangle][kParts][64]  P, of q' and k'
  float* s;   // [v head][slot][kFactors * 64]     the rows' factors
  long long slots;
};
constexpr int kCus = 256;
constexpr int kFactors = 5;  // beta c^2 e^G, e^G (the last one is the chunk's), d, e^(G_last - G): a piece of 1 KB; beta c

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

ChunkSpace chunk_space(void* workspace, size_t slots, int qk_heads, int v_heads, int dk, size_t* bytes) {
  char* at = static_cast<char*>(workspace);
  auto take = [&](size_t n) {
    char* p = at;
    at += up256(n);
    return p;
  };
  ChunkSpace c;
  const size_t rows = slots * qk_heads * kChunk * dk * 2, lower = slots * v_heads * kTriangle * kParts * 1024;
  c.k = reinterpret_cast<h8_t*>(take(rows));
  c.q = reinterpret_cast<h8_t*>(take(rows));
  c.t = reinterpret_cast<b8_t*>(take(lower));
  c.p = reinterpret_cast<b8_t*>(take(lower));
  c.s = reinterpret_cast<float*>(take(slots * v_heads * kFactors * kChunk * 4));
  c.slots = (long long)slots;
  *bytes = (size_t)(at - static_cast<char*>(workspace));
  return c;
}

__device__ __forceinline__ f4_t mfma(h8_t a, h8_t b, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f4_t mfma(b8_t a, b8_t b, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The same of 16 columns, a lane's 4 q .. 4 q + 3: the first half of a piece.
__device__ __forceinline__ f4_t mfma(short4_t a, b8_t b, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(
      a, __builtin_bit_cast(short4_t, __builtin_shufflevector(b, b, 0, 1, 2, 3)), c, 0, 0, 0);
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

__device__ __forceinline__ float max4(f4_t x) {
  return fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
}

// Two stacked result tiles times a power of two as an operand B of 32 rows, in
// two fp16 parts of one rounding each: an instruction of mixed width a part.
__device__ __forceinline__ void split_tiles(f4_t x, f4_t y, float scale, h8_t* hi, h8_t* lo) {
  const float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const h2_t pair = {(_Float16)fmaf(v[j], scale, 0.f), (_Float16)fmaf(v[j + 1], scale, 0.f)};
    uint32_t bits = __builtin_bit_cast(uint32_t, pair);
    asm("" : "+v"(bits));  // or each first part is computed twice, for itself and for the second
    const h2_t h = as_h2(bits);
    (*hi)[j] = h[0];
    (*hi)[j + 1] = h[1];
    (*lo)[j] = (_Float16)fmaf(v[j], scale, -(float)h[0]);
    (*lo)[j + 1] = (_Float16)fmaf(v[j + 1], scale, -(float)h[1]);
  }
}

// Two stacked result tiles as an operand of 32 rows in three bf16 parts: one of the
// number, one of what that leaves, and the rest, which has no more than 8 bits.
// kNearest: the nearest ones, each at most 2^-9 of the one before and of either sign;
// for T and P, where nothing waits. Else the upper 16 bits, at most 2^-7 of the one
// before, an instruction less (1.68 and 1.74 us a chunk). What the products left
// out then are is as small and of either sign. (An infinity's second part is NaN.)
struct Split {
  b8_t part[kParts];
};
template <bool kNearest>
__device__ __forceinline__ Split split_exact(f4_t x, f4_t y) {
  float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  uint32_t bits[kParts][4];
#pragma unroll
  for (int p = 0; p < kParts; ++p)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t a = __builtin_bit_cast(uint32_t, v[2 * j]), b = __builtin_bit_cast(uint32_t, v[2 * j + 1]);
      if constexpr (kNearest) {
        a = (uint32_t)f2bf(v[2 * j]) << 16;
        b = (uint32_t)f2bf(v[2 * j + 1]) << 16;
      }
      bits[p][j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      v[2 * j] -= __builtin_bit_cast(float, a & 0xFFFF0000u);
      v[2 * j + 1] -= __builtin_bit_cast(float, b & 0xFFFF0000u);
    }
  Split s;
#pragma unroll
  for (int p = 0; p < kParts; ++p)
    s.part[p] = __builtin_bit_cast(b8_t, make_uint4(bits[p][0], bits[p][1], bits[p][2], bits[p][3]));
  return s;
}

__device__ __forceinline__ uint2 first_half(b8_t x) {
  const uint4 w = __builtin_bit_cast(uint4, x);
  return make_uint2(w.x, w.y);
}

// The products of parts that are taken: of the first with all, and of the second with two.
constexpr int kProducts = 6;
__device__ constexpr int kLeft[kProducts] = {0, 0, 1, 1, 0, 2}, kRight[kProducts] = {0, 1, 0, 1, 2, 0};

// 2^(a - b) of two sums of logarithms in two fp32 parts each, a below b: the
// difference of the first parts is not exact, and what it leaves counts, since a
// difference of 40 has steps of 2^-18.
__device__ __forceinline__ float decay_of(float a, float a_rest, float b, float b_rest) {
  const float d = a - b;
  return exp2f(d) * fmaf((a - d) - b + (a_rest - b_rest), 0.69314718f, 1.f);
}

// ---------------------------------------------------------------------------
// One workgroup a chunk and head; wave w has its rows 16 w .. 16 w + 15. 8192
// tokens of 32 heads of 128 (16 of keys), 4096 workgroups, take 70 us: 76 MB read
// from memory and 199 written, 3.9 TB/s, which bounds it; a workgroup alone would
// take 8 us, and next to others' stores its first loads take 4 of 13.
// ---------------------------------------------------------------------------
constexpr int kPad = 68;  // floats a row of 64 takes in LDS

template <int kDk, bool kBf16>
__global__ __launch_bounds__(kPrepareThreads, 4) void delta_prepare_kernel(DeltaArgs a, ChunkSpace ws) {
  constexpr int kS = kDk / 32;
  __shared__ h8_t keys[4][kS][64];
  __shared__ float m[kChunk][kPad];
  __shared__ float c_of[kChunk], d_of[kChunk], beta_of[kChunk], hi_of[kChunk], lo_of[kChunk];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, i = lane & 15, q4 = lane >> 4;
  const long long slot = blockIdx.x / a.v_heads;
  const int h = blockIdx.x % a.v_heads, hq = h / a.group;
  Tile tile;
  if (!find_tile<true>(a.offsets, a.requests, a.tokens, kChunk, (int)slot, &tile, a.limit)) return;
  if (tile.request < 0) return;
  const bool first_of_group = h % a.group == 0;

  // Every load first; rows behind the last are row 0 again, and zeros below.
  const int r = 16 * wave + i;
  const bool real = r < tile.count;
  const long long row = tile.row + (real ? r : 0);
  const uint16_t* kp = a.k + row * a.k_token + (long long)hq * a.k_head + 4 * q4;
  const uint16_t* qp = a.q + row * a.q_token + (long long)hq * a.q_head + 4 * q4;
  uint2 k_raw[2 * kS], q_raw[2 * kS];
#pragma unroll
  for (int s = 0; s < 2 * kS; ++s) k_raw[s] = *reinterpret_cast<const uint2*>(kp + 16 * s);
#pragma unroll
  for (int s = 0; s < 2 * kS; ++s) q_raw[s] = *reinterpret_cast<const uint2*>(qp + 16 * s);
  const bool live = lane < tile.count;
  double g = 0.0;
  float beta = 0.f;
  if (wave == 0) {
    const long long at = (long long)(tile.row + (live ? lane : 0)) * a.v_heads + h;
    g = (double)cut_log(a.log_decay[at]);
    beta = a.beta[at];
  }

  // Rows of keys and queries, scaled to fp16.
  h8_t kf[kS], qf[kS];
  auto rows = [&](const uint2(&raw)[2 * kS], h8_t(&f)[kS], float* length2) {
    float top = 0.f, sum = 0.f;
    float e[kS][8];
#pragma unroll
    for (int s = 0; s < 2 * kS; ++s) {
      const uint32_t x = real ? raw[s].x : 0u, y = real ? raw[s].y : 0u;
      float* to = e[s >> 1] + 4 * (s & 1);
      to[0] = pair_lo<kBf16>(x);
      to[1] = pair_hi<kBf16>(x);
      to[2] = pair_lo<kBf16>(y);
      to[3] = pair_hi<kBf16>(y);
      top = fmaxf(fmaxf(top, fmaxf(fabsf(to[0]), fabsf(to[1]))), fmaxf(fabsf(to[2]), fabsf(to[3])));
      sum += fmaf(to[0], to[0], to[1] * to[1]) + fmaf(to[2], to[2], to[3] * to[3]);
    }
    top = max_rows(top);
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    const int e2 = exponent_of(top);
#pragma unroll
    for (int s = 0; s < kS; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) f[s][j] = (_Float16)ldexpf(e[s][j], -e2);
    *length2 = sum;
    return top == 0.f ? INT32_MIN : e2;  // NaN has an exponent too
  };
  float kk, qq;
  const int ke = rows(k_raw, kf, &kk);
  const size_t qk_at = (hq * ws.slots + slot) * (4 * kS * 64);
#pragma unroll
  for (int s = 0; s < kS; ++s) {
    keys[wave][s][lane] = kf[s];
    if (first_of_group) ws.k[qk_at + (wave * kS + s) * 64 + lane] = kf[s];
  }
  const int qe = rows(q_raw, qf, &qq);
  if (first_of_group)
#pragma unroll
    for (int s = 0; s < kS; ++s) ws.q[qk_at + (wave * kS + s) * 64 + lane] = qf[s];
  float c = 0.f, d = 0.f;  // a row of zeros has no part in anything
  if (ke != INT32_MIN) c = ldexpf(a.normalize ? 1.f / sqrtf(kk + kUnitEps) : 1.f, ke);
  if (qe != INT32_MIN) d = ldexpf(a.normalize ? a.scale / sqrtf(qq + kUnitEps) : a.scale, qe);
  if (q4 == 0) {
    c_of[r] = c;
    d_of[r] = d;
  }
  // Sums of the decays' logarithms, in 64 bits: a sum's difference to another
  // has to be exact where both are large. Kept as two fp32, to the base 2.
  float hi = 0.f, lo = 0.f, until = 0.f;
  if (wave == 0) {
    if (!live) g = 0.0, beta = 0.f;
#pragma unroll
    for (int dd = 1; dd < 64; dd *= 2) {
      const double o = __shfl_up(g, dd);
      if (lane >= dd) g += o;
    }
    g *= 1.4426950408889634074;  // log2(e)
    hi = (float)g;
    lo = (float)(g - (double)hi);
    until = decay_of(__shfl(hi, 63), __shfl(lo, 63), hi, lo);
    hi_of[lane] = hi;
    lo_of[lane] = lo;
    beta_of[lane] = beta;
  }
  __syncthreads();

  if (wave == 0) {
    const float cc = c_of[lane], since = decay_of(hi, lo, 0.f, 0.f);
    float* f = ws.s + (h * ws.slots + slot) * (kFactors * kChunk) + lane;
    f[0] = beta * cc * cc * since;
    f[64] = since;
    f[128] = d_of[lane];
    f[192] = until;
    f[256] = beta * cc;
  }
  // Decayed products of the wave's rows with those before them.
  const size_t v_at = (h * ws.slots + slot) * (kTriangle * kParts * 64);
  auto pieces_out = [&](b8_t* to) {
    for (int s = 0; s <= wave / 2; ++s) {
      const bool alone = (wave & 1) == 0 && s == wave / 2;
      const f4_t x = *reinterpret_cast<const f4_t*>(&m[16 * wave + i][32 * s + 4 * q4]);
      f4_t y{0.f, 0.f, 0.f, 0.f};
      if (!alone) y = *reinterpret_cast<const f4_t*>(&m[16 * wave + i][32 * s + 16 + 4 * q4]);
      const Split e = split_exact<true>(x, y);
      b8_t* at = to + v_at + (alone ? 0 : wave + s) * (kParts * 64) + lane;
#pragma unroll
      for (int p = 0; p < kParts; ++p)
        if (alone) reinterpret_cast<uint2*>(at + p * 64)[s] = first_half(e.part[p]);
        else at[p * 64] = e.part[p];
    }
  };
  const int rr0 = 16 * wave + 4 * q4;
  float hr[4], lr[4], b2[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    hr[e] = hi_of[rr0 + e];
    lr[e] = lo_of[rr0 + e];
    b2[e] = beta_of[rr0 + e] * c_of[rr0 + e] * c_of[rr0 + e];
  }
  f4_t kkt[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f4_t qkt{0.f, 0.f, 0.f, 0.f};
    kkt[j] = f4_t{0.f, 0.f, 0.f, 0.f};
    const int col = 16 * j + i;
    if (j <= wave) {
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        const h8_t b = keys[j][s][lane];
        kkt[j] = mfma(kf[s], b, kkt[j]);
        qkt = mfma(qf[s], b, qkt);
      }
      const float hc = hi_of[col], lc = lo_of[col];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float decay = decay_of(hr[e], lr[e], hc, lc);
        qkt[e] = rr0 + e >= col ? decay * qkt[e] : 0.f;
        kkt[j][e] = rr0 + e > col ? b2[e] * decay * kkt[j][e] : 0.f;
      }
    }
    if (j <= wave)
#pragma unroll
      for (int e = 0; e < 4; ++e) m[rr0 + e][col] = qkt[e];
  }
  // A wave's rows of m are its own until the barrier: P goes out from there, then
  // A comes in.
  pieces_out(ws.p);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j <= wave)
#pragma unroll
      for (int e = 0; e < 4; ++e) m[rr0 + e][16 * j + i] = kkt[j][e];

  // T = (1 + A)^-1: the blocks of 16 on the diagonal by substitution, a lane a
  // column, then the blocks below from them, a wave a column of blocks, with
  // 32-bit matrix products:  T_ij = -T_ii sum_(j <= k < i) A_ik T_kj.
  {
    float t[16];
    const int base = 16 * wave;
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      float even = x == i ? 1.f : 0.f, odd = 0.f;
#pragma unroll
      for (int k = 0; k < x; ++k) {
        float& sum = k & 1 ? odd : even;
        sum = fmaf(-m[base + x][base + k], t[k], sum);
      }
      t[x] = even + odd;
    }
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
  pieces_out(ws.t);
}

// ---------------------------------------------------------------------------
// A request's chunks one after another, kCols tiles of 16 columns of one head's
// state a workgroup, four waves a tile. Two waves hold half of the tile's rows
// each and go from state to state: their shares of K' S are added through LDS,
// the corrections both compute, and each brings its rows of the state forward.
// Columns do not meet, and a result tile is the next product's operand B as it
// stands. The other two waves compute half of the tokens' outputs each, one
// chunk behind, from the parts of the state and the corrections that the first
// two leave in LDS, and bring the next chunk's operands there: what only the
// outputs need is off the chain that bounds a long prompt. That chain is K' S and
// what the corrections add, each with its largest value, a scale and two parts
// before it, and between them the corrections, with three: 1.65 us a chunk where the
// chip has room, 1.95 to 2 on all of its CUs (1.5 and 1.8 with two fp16 parts
// there, too). One prompt of 8192 tokens of 32 heads takes 255 us on 256
// workgroups, of 4 heads 211 on 32, and 7 prompts of 3001 tokens of 16 heads 45.
// ---------------------------------------------------------------------------
using lds_ptr = __attribute__((address_space(3))) void*;
typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
using lds_short4_ptr = __attribute__((address_space(3))) short4_t*;
using lds_float_ptr = __attribute__((address_space(3))) float*;

// Buffers: a chunk's rows behind the request's last are out of their range, so
// that they load zeros and store nothing.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}

template <typename Piece>
__device__ __forceinline__ Piece load_piece(__amdgpu_buffer_rsrc_t r, uint32_t offset) {
  return __builtin_bit_cast(Piece, __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 0));
}

// A barrier for what was read from and written to LDS: __syncthreads() waits for
// loads to LDS too, which the output waves have under way across it.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int kDk, int kCols, bool kBf16>
__global__ __launch_bounds__(256 * kCols, 1) void delta_scan_kernel(DeltaArgs a, ChunkSpace ws, int value_size) {
  constexpr int kS = kDk / 32, kHalfS = kS / 2, kHalfTiles = kDk / 32;
  constexpr int kType = kBf16 ? DK_KV_BF16 : DK_KV_F16;
  constexpr int kKeys = 4 * kS, kInverse = kParts * kTriangle;  // pieces of 1 KB
  constexpr int kPieces = kKeys + kInverse + 1;
  constexpr f4_t kZero{0.f, 0.f, 0.f, 0.f};
  __shared__ h8_t stage[2][kPieces][64];         // a chunk's operands and its rows' factors
  __shared__ f4_t rows_v[2][kCols][4][64];       // beta c v of a chunk's rows
  __shared__ f4_t share[kCols][2][4][64];        // a half's share of K' S
  __shared__ h8_t left_s[kCols][2 * kS][64];     // the state's parts
  __shared__ f4_t left_w[kCols][4][64];          // the corrections
  __shared__ float left_scale[kCols][2][16];     // by which both halves of the state are to be multiplied
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool outputs = wave >= 2 * kCols;
  const int tile = (wave >> 1) & (kCols - 1), half = wave & 1;
  const int h = blockIdx.x % a.v_heads, hq = h / a.group;
  if (!wave_offsets_ok(a.offsets, a.requests, a.tokens)) return;
  // The grid has room for so many long requests; where there are more, a workgroup
  // takes several, one after another.
  for (int rank = blockIdx.y;; rank += gridDim.y) {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // or all addresses of both kinds of waves are kept across requests
  const int i = lane & 15, q4 = lane >> 4, col = ((blockIdx.x / a.v_heads) * kCols + tile) * 16 + i;
  const int b = __builtin_amdgcn_readfirstlane(find_long(a.offsets, a.requests, a.limit, rank));
  if (b < 0) return;
  const int from = __builtin_amdgcn_readfirstlane(a.offsets[b]);
  const int n = __builtin_amdgcn_readfirstlane(a.offsets[b + 1]) - from;
  const long long slot0 = from / kChunk + rank;
  const int chunks = (n + kChunk - 1) / kChunk;

  // A chunk takes two barriers. State waves: the first, K' S from the state, the
  // second, the corrections and the state after. Output waves: the first, P w
  // and the outputs of the chunk before, the second, Q' S and the next chunk's
  // loads. Each hands on what the other needs before a barrier and takes it
  // behind it, so that one buffer of each is enough.
  if (!outputs) {
    float* state = a.states + (((long long)b * a.v_heads + h) * kDk + half * (kDk / 2)) * value_size + col;
    f4_t s[kHalfTiles];
    const bool fresh = a.held && a.held[b] <= 0;
#pragma unroll
    for (int t = 0; t < kHalfTiles; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][e] = fresh ? 0.f : state[(long long)(16 * t + 4 * q4 + e) * value_size];
    for (int c = 0; c <= chunks; ++c) {
      lds_barrier();
      if (c == chunks) break;
      const h8_t(*keys)[64] = &stage[c & 1][0];
      const h8_t(*inverse)[64] = &stage[c & 1][kKeys];
      const float* factors = reinterpret_cast<const float*>(&stage[c & 1][kKeys + kInverse][0]);
      auto rows4 = [&](int which, int y) {
        return *reinterpret_cast<const f4_t*>(factors + which * kChunk + 16 * y + 4 * q4);
      };

      // Operands are read from LDS well ahead of their products: left to itself
      // the compiler reads two, waits for them and goes on.
      h8_t kf[4 * kHalfS], uf[2 * kHalfTiles];
      short4_t t_first[2][kParts];  // of (0,0) and (2,1)
      b8_t t_whole[4][kParts];      // (1,0) (2,0) (3,0) (3,1)
#pragma unroll
      for (int t = 0; t < kHalfS; ++t)
#pragma unroll
        for (int y = 0; y < 4; ++y) kf[y * kHalfS + t] = keys[y * kS + half * kHalfS + t][lane];
      __builtin_amdgcn_sched_barrier(0);
      // K' S, this half's share.
      float m = max4(s[0]);
#pragma unroll
      for (int t = 1; t < kHalfTiles; ++t) m = fmaxf(m, max4(s[t]));
      int shift = column_shift(m);
      float up = power2(shift), down = power2(-shift);
      f4_t x[4] = {kZero, kZero, kZero, kZero};
#pragma unroll
      for (int t = 0; t < kHalfS; ++t) {
        h8_t hi, lo;
        split_tiles(s[2 * t], s[2 * t + 1], up, &hi, &lo);
        left_s[tile][2 * (half * kHalfS + t)][lane] = hi;
        left_s[tile][2 * (half * kHalfS + t) + 1][lane] = lo;
#pragma unroll
        for (int y = 0; y < 4; ++y) x[y] = mfma(kf[y * kHalfS + t], hi, x[y]);
#pragma unroll
        for (int y = 0; y < 4; ++y) x[y] = mfma(kf[y * kHalfS + t], lo, x[y]);
      }
      __builtin_amdgcn_sched_barrier(0);
      // The keys once more, transposed: rows are elements 16 z .. of this half, and
      // the columns tokens in the order of an operand. Of each 16 lanes lane 4 r +
      // c reads the elements 4 c .. 4 c + 3 of token r, and lane l receives
      // element l of tokens 0 .. 3.
#pragma unroll
      for (int z = 0; z < kHalfTiles; ++z)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int e = half * kHalfTiles + z;
          const h8_t* from = &keys[y * kS + (e >> 1)][4 * q4 + (i >> 2) + 16 * (i & 3)];
          const h4_t part = __builtin_bit_cast(
              h4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_ptr)(reinterpret_cast<const uint16_t*>(from) + 4 * (e & 1))));
#pragma unroll
          for (int j = 0; j < 4; ++j) uf[2 * z + (y >> 1)][4 * (y & 1) + j] = part[j];
        }
      __builtin_amdgcn_sched_barrier(0);
      if (q4 == 0) left_scale[tile][half][i] = down;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        x[y] *= down;
        share[tile][half][y][lane] = x[y];
      }
      f4_t bv[4], b2[4], until[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) bv[y] = rows_v[c & 1][tile][y][lane];
      lds_barrier();
      f4_t other[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        other[y] = share[tile][1 - half][y][lane];
        b2[y] = rows4(0, y);
      }
#pragma unroll
      for (int n = 0; n < kParts; ++n) {
        t_first[0][n] = *reinterpret_cast<const short4_t*>(&inverse[n][lane]);
#pragma unroll
        for (int z = 0; z < 3; ++z) t_whole[z][n] = __builtin_bit_cast(b8_t, inverse[(z + 1) * kParts + n][lane]);
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) until[y] = rows4(3, y);
      const float whole = factors[2 * kChunk - 1];
      __builtin_amdgcn_sched_barrier(0);
      // What each token finds wrong in the state before the chunk.
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[y][e] = fmaf(-b2[y][e], x[y][e] + other[y][e], bv[y][e]);
      // The corrections w = T x.
      f4_t w[4] = {kZero, kZero, kZero, kZero};
      const Split x01 = split_exact<false>(x[0], x[1]);
#pragma unroll
      for (int n = 0; n < kParts; ++n) {
        t_first[1][n] = *(reinterpret_cast<const short4_t*>(&inverse[n][lane]) + 1);
        t_whole[3][n] = __builtin_bit_cast(b8_t, inverse[4 * kParts + n][lane]);
      }
#pragma unroll
      for (int n = 0; n < kProducts; ++n) {
        w[0] = mfma(t_first[0][kLeft[n]], x01.part[kRight[n]], w[0]);
#pragma unroll
        for (int y = 1; y < 4; ++y) w[y] = mfma(t_whole[y - 1][kLeft[n]], x01.part[kRight[n]], w[y]);
      }
      const Split x23 = split_exact<false>(x[2], x[3]);
#pragma unroll
      for (int n = 0; n < kProducts; ++n) {
        w[2] = mfma(t_first[1][kLeft[n]], x23.part[kRight[n]], w[2]);
        w[3] = mfma(t_whole[3][kLeft[n]], x23.part[kRight[n]], w[3]);
      }
      // The state after the chunk.
      f4_t w2[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) w2[y] = w[y] * until[y];
      shift = column_shift(fmaxf(fmaxf(max4(w2[0]), max4(w2[1])), fmaxf(max4(w2[2]), max4(w2[3]))));
      up = power2(shift);
      down = power2(-shift);
      h8_t hi[2], lo[2];
      f4_t add[kHalfTiles];
#pragma unroll
      for (int z = 0; z < kHalfTiles; ++z) add[z] = kZero;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        split_tiles(w2[2 * y], w2[2 * y + 1], up, &hi[y], &lo[y]);
#pragma unroll
        for (int z = 0; z < kHalfTiles; ++z) add[z] = mfma(uf[2 * z + y], hi[y], add[z]);
#pragma unroll
        for (int z = 0; z < kHalfTiles; ++z) add[z] = mfma(uf[2 * z + y], lo[y], add[z]);
      }
      if (half == 0) {  // one half of the tokens' corrections each
        left_w[tile][0][lane] = w[0];
        left_w[tile][1][lane] = w[1];
      } else {
        left_w[tile][2][lane] = w[2];
        left_w[tile][3][lane] = w[3];
      }
#pragma unroll
      for (int z = 0; z < kHalfTiles; ++z)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[z][e] = fmaf(add[z][e], down, whole * s[z][e]);
    }
#pragma unroll
    for (int t = 0; t < kHalfTiles; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) state[(long long)(16 * t + 4 * q4 + e) * value_size] = s[t][e];
  } else {
    // A chunk's operands and factors, whole pieces of 1 KB, 16 bytes a lane.
    constexpr uint32_t kQkBytes = kKeys * 1024, kVBytes = kInverse * 1024, kFactorBytes = kFactors * kChunk * 4;
    auto of_qk = [&](const h8_t* base, int c) {
      return buffer_of(reinterpret_cast<const char*>(base) + (hq * ws.slots + slot0 + c) * kQkBytes, kQkBytes);
    };
    auto of_v = [&](const b8_t* base, int c) {
      return buffer_of(reinterpret_cast<const char*>(base) + (h * ws.slots + slot0 + c) * kVBytes, kVBytes);
    };
    auto of_factors = [&](int c) {
      return buffer_of(reinterpret_cast<const char*>(ws.s) + (h * ws.slots + slot0 + c) * kFactorBytes, kFactorBytes);
    };
    const uint32_t piece_at = lane * 16;
    const uint16_t* values = a.v + (long long)from * a.v_token + (long long)h * a.v_head;
    uint16_t* out = a.out + ((long long)from * a.v_heads + h) * value_size;
    const uint32_t out_token = a.v_heads * value_size;
    // Of a chunk's outputs the rows 32 half .. 32 half + 31 are this wave's, and of
    // its values, a row a lane, the columns 8 half .. 8 half + 7.
    uint32_t out_at[8];
#pragma unroll
    for (int z = 0; z < 8; ++z) out_at[z] = ((32 * half + 16 * (z >> 2) + (z & 3) + 4 * q4) * out_token + col) * 2;
    const uint32_t v_at = (lane * (uint32_t)a.v_token + col - i + 8 * half) * 2;
    // All output waves bring a chunk's operands, each its share of the pieces. Past
    // the last chunk it is that one again, into a buffer that nobody reads: the
    // compiler counts what is on its way only where every turn asks for as much.
    auto bring = [&](int chunk, int which) {
      h8_t* to = &stage[chunk & 1][0][0];
      const int c = min(chunk, chunks - 1);
      auto some = [&](__amdgpu_buffer_rsrc_t r, int first, int count, int turn) {
#pragma unroll
        for (int p = 0; p < count; p += 2 * kCols)
          if (count % (2 * kCols) == 0 || p + turn < count)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(to + (first + p + turn) * 64), 16,
                                                     piece_at + (p + turn) * 1024, 0, 0, 0);
      };
      const int turn = wave - 2 * kCols;
      if (which == 0) {
        some(of_qk(ws.k, c), 0, kKeys, turn);
      } else {  // as many for each wave: the last has one of T less and the factors
        some(of_v(ws.t, c), kKeys, kInverse, turn);
        some(of_factors(c), kKeys + kInverse, 1, 2 * kCols - 1 - turn);
      }
    };
    auto in_order = [] {
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    // Until no more than so many of this wave's loads and stores are under way: they
    // come back in the order in which they were asked for.
    auto wait_but = [&](auto count) {
      constexpr int k = decltype(count)::value;
      static_assert(k < 64, "what vmcnt holds");
      in_order();
      __builtin_amdgcn_s_waitcnt((k & 15) | (k >> 4 << 14) | 0xF70);
      in_order();
    };
    constexpr int kLateLoads = 2 * kS + kKeys / (2 * kCols);  // queries, and a share of keys
    uint4 v;
    float b1;
    h8_t q[2 * kS];
    short4_t p_first[kParts];  // of (0,0) or (2,1)
    b8_t p[3 * kParts];        // (1,0), or (2,0) (3,0) (3,1)
    auto load_values = [&](int chunk) {
      const int c = min(chunk, chunks - 1);
      const uint32_t count = min(n - c * kChunk, kChunk);
      const auto r =
          buffer_of(values + (long long)c * kChunk * a.v_token, ((count - 1) * (uint32_t)a.v_token + value_size) * 2);
      v = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, v_at, 0, 0));
      b1 = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(of_factors(c), (4 * kChunk + lane) * 4, 0, 0));
    };
    auto give_values = [&](int c) {  // to where a result tile has row `lane`
      float* to = reinterpret_cast<float*>(&rows_v[c & 1][tile][lane >> 4][8 * half + 16 * ((lane & 15) >> 2)]) + (lane & 3);
      const uint32_t pairs[4] = {v.x, v.y, v.z, v.w};
      const uint32_t at = (uint32_t)(uintptr_t)(lds_float_ptr)to;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // Before a store to LDS the compiler waits for all loads to LDS, also where
        // they go elsewhere.
        asm volatile("ds_write_b32 %0, %1 offset:%2" ::"v"(at), "v"(b1 * pair_lo<kBf16>(pairs[j])), "n"(32 * j) : "memory");
        asm volatile("ds_write_b32 %0, %1 offset:%2" ::"v"(at), "v"(b1 * pair_hi<kBf16>(pairs[j])), "n"(32 * j + 16)
                     : "memory");
      }
    };
    auto load_queries = [&](int chunk) {
      const int c = min(chunk, chunks - 1);
      const auto qs = of_qk(ws.q, c);
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int t = 0; t < kS; ++t) q[y * kS + t] = load_piece<h8_t>(qs, piece_at + ((2 * half + y) * kS + t) * 1024);
    };
    load_values(0);
    give_values(0);
    load_values(1);
    bring(0, 0);
    bring(0, 1);
    load_queries(0);
    bring(1, 0);
    f4_t x[2], d[2], y2[2];  // of the last chunk: e^G Q' S, and the queries' factors
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0);  // chunk 0's operands are in LDS
    asm volatile("" ::: "memory");
    for (int c = 0; c <= chunks; ++c) {
      lds_barrier();
      if (c > 0) {
        const int at = c - 1;
        f4_t wv[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) wv[t] = left_w[tile][t][lane];
        y2[0] = y2[1] = kZero;
        const Split w01 = split_exact<false>(wv[0], wv[1]);
        if (half) {
#pragma unroll
          for (int n = 0; n < kProducts; ++n)
#pragma unroll
            for (int y = 0; y < 2; ++y) y2[y] = mfma(p[kParts * y + kLeft[n]], w01.part[kRight[n]], y2[y]);
          const Split w23 = split_exact<false>(wv[2], wv[3]);
#pragma unroll
          for (int n = 0; n < kProducts; ++n) {
            y2[0] = mfma(p_first[kLeft[n]], w23.part[kRight[n]], y2[0]);
            y2[1] = mfma(p[kParts * 2 + kLeft[n]], w23.part[kRight[n]], y2[1]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < kProducts; ++n) {
            y2[0] = mfma(p_first[kLeft[n]], w01.part[kRight[n]], y2[0]);
            y2[1] = mfma(p[kLeft[n]], w01.part[kRight[n]], y2[1]);
          }
        }
        give_values(c + 1);
        __builtin_amdgcn_sched_barrier(0);
        const uint32_t count = min(n - at * kChunk, kChunk);
        const auto r = buffer_of(out + (long long)at * kChunk * out_token, ((count - 1) * out_token + value_size) * 2);
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float o = d[y][e] * (y2[y][e] + x[y][e]);
            __builtin_amdgcn_raw_buffer_store_b16(to_half_bits<kType>(o), r, out_at[4 * y + e], 0, 0);
          }
      }
      if (c == chunks) break;
      // What the state waves read behind the barrier is there; the next chunk's
      // keys and queries, asked for last, and the 8 stores above may be under way.
      if (c > 0) wait_but(std::integral_constant<int, 8 + kLateLoads>{});
      else give_values(1);
      lds_barrier();
      h8_t sp[2 * kS];
#pragma unroll
      for (int t = 0; t < 2 * kS; ++t) sp[t] = left_s[tile][t][lane];
      const float ds0 = left_scale[tile][0][i], ds1 = left_scale[tile][1][i];
      const float* factors = reinterpret_cast<const float*>(&stage[c & 1][kKeys + kInverse][0]);
      f4_t since[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        since[y] = *reinterpret_cast<const f4_t*>(factors + kChunk + 32 * half + 16 * y + 4 * q4);
        d[y] = *reinterpret_cast<const f4_t*>(factors + 2 * kChunk + 32 * half + 16 * y + 4 * q4);
      }
      __builtin_amdgcn_sched_barrier(0);
      f4_t x0[2] = {kZero, kZero}, x1[2] = {kZero, kZero};  // of the state's halves
#pragma unroll
      for (int t = 0; t < kHalfS; ++t)
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            x0[y] = mfma(q[y * kS + t], sp[2 * t + part], x0[y]);
            x1[y] = mfma(q[y * kS + kHalfS + t], sp[2 * (kHalfS + t) + part], x1[y]);
          }
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[y][e] = since[y][e] * fmaf(ds0, x0[y][e], ds1 * x1[y][e]);
      __builtin_amdgcn_sched_barrier(0);
      // In the order in which it is waited for. The state waves are through with
      // this chunk's keys and with all of the last one's operands.
      const auto ps = of_v(ws.p, c);
      if (half)
#pragma unroll
        for (int z = kParts; z < 3 * kParts; ++z) p[z] = load_piece<b8_t>(ps, piece_at + (2 * kParts + z) * 1024);
#pragma unroll
      for (int z = 0; z < kParts; ++z) {
        p_first[z] = __builtin_bit_cast(short4_t, __builtin_amdgcn_raw_buffer_load_b64(ps, piece_at + z * 1024 + 8 * half, 0, 0));
        p[z] = load_piece<b8_t>(ps, piece_at + (kParts * (1 + half) + z) * 1024);
      }
      load_values(c + 2);
      bring(c + 1, 1);
      in_order();  // kLateLoads counts what comes behind this
      load_queries(c + 1);
      in_order();
      bring(c + 2, 0);
      in_order();
      // Chunk c + 1's keys, asked for before the last turn's stores, are there:
      // at least so many more were asked for since.
      static_assert((kInverse + 1) % (2 * kCols) == 0, "every wave brings as much");
      constexpr int kSince = 8 + 2 * kParts + 2 + (kInverse + 1) / (2 * kCols) + kLateLoads;
      wait_but(std::integral_constant<int, kSince>{});
    }
    __builtin_amdgcn_s_waitcnt(0);  // nothing is on its way to LDS behind the end
  }
  lds_barrier();  // the next request's first stores to LDS are behind this one's last reads
  }
}

}  // namespace

size_t delta_chunk_bytes(int num_tokens, int requests, int limit, int qk_heads, int v_heads, int key_size) {
  size_t bytes;
  chunk_space(nullptr, chunk_slots(num_tokens, requests, limit), qk_heads, v_heads, key_size, &bytes);
  return bytes;
}

int delta_chunk_launch(const DeltaArgs& a, int key_size, int value_size, bool bf16, void* workspace,
                       hipStream_t stream) {
  size_t bytes;
  const long long slots = chunk_slots(a.tokens, a.requests, a.limit);
  const ChunkSpace ws = chunk_space(workspace, slots, a.qk_heads, a.v_heads, key_size, &bytes);
  const dim3 chunks((unsigned)(slots * a.v_heads));
  // Tiles of 16 columns: two a workgroup where one each would not be at work at
  // once (its LDS leaves one workgroup a CU). One and two, us: 256 tiles (61 single
  // tokens and a prompt of 2048 of 32 heads) 124 and 144, 512 (4 prompts of 2048 of
  // 16 heads) 162 and 131, 1920 (60 prompts of 100 of 4 heads) 78 and 60. How many
  // requests are at work at once goes by the longest, or, where max_query_len says
  // no more than the number of tokens does, by their average (and is one where that
  // is under a chunk: single tokens and a prompt).
  const long long average = a.tokens / a.requests;
  const long long each = a.longest < a.tokens ? a.longest : average >= kChunk ? average : a.tokens;
  const long long at_once = std::min((long long)a.requests, std::max(1LL, a.tokens / each));
  const int cols = at_once * a.v_heads * (value_size / 16) > kCus ? 2 : 1;
  // Room for three times the requests that fill the chip, whatever max_query_len is:
  // workgroups take several where there are more, and one without any costs its
  // turn on a CU. Once, three times and room for all, us: 7 ragged prompts of 16
  // heads 77, 66 and 66; 8192 tokens and 100 prompts of 80 of 4 heads 316, 267 and
  // 242; the 62 requests above 126, 124 and 187; 64 prompts of 128 of 32 heads 411,
  // 411 and 471.
  const int workgroups = a.v_heads * (value_size / (16 * cols));
  const long long longs = std::min((long long)a.requests, (long long)a.tokens / (a.limit + 1));
  const unsigned room = (unsigned)std::max(1LL, std::min(longs, 3LL * ((kCus + workgroups - 1) / workgroups)));
  const dim3 columns((unsigned)workgroups, room);
  auto launch = [&](auto prepare, auto one, auto two) {
    hipLaunchKernelGGL(prepare, chunks, dim3(kPrepareThreads), 0, stream, a, ws);
    if (cols == 1) hipLaunchKernelGGL(one, columns, dim3(256), 0, stream, a, ws, value_size);
    else hipLaunchKernelGGL(two, columns, dim3(512), 0, stream, a, ws, value_size);
  };
  auto pick = [&](auto dk, auto type) {
    constexpr int d = decltype(dk)::value;
    constexpr bool t = decltype(type)::value;
    launch(delta_prepare_kernel<d, t>, delta_scan_kernel<d, 1, t>, delta_scan_kernel<d, 2, t>);
  };
  using std::integral_constant;
  if (key_size == 64)
    bf16 ? pick(integral_constant<int, 64>{}, std::true_type{}) : pick(integral_constant<int, 64>{}, std::false_type{});
  else
    bf16 ? pick(integral_constant<int, 128>{}, std::true_type{}) : pick(integral_constant<int, 128>{}, std::false_type{});
  return check_launch("delta_rule launch");
}

}  // namespace dk
