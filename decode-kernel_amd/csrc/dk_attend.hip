// Attention over the paged 8-bit key/value cache.
// Layouts in dk_kv.hpp, contract in include/decode_kernel/dk_kv.h.
//
// For a row (a query head of one token) with keys j:
//   s_j = scale q.k_j,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),
// in one pass with a running m (fp32, base 2). The rows of one key/value head
// and sequence (the group's query heads times the sequence's queries) are
// the columns of matrix products over a tile of 64 keys:
//   S^T [64 keys, 16 rows] = K Q^T,   O^T [elements, 16 rows] += V^T P^T,
// v_mfma_f32_16x16x32_f16 throughout. Codes are whole numbers up to 127,
// exact in fp16; a page's scale multiplies S after, P before, the product.
// Which key a product's row is, is free, so lane group g (16 lanes) takes the
// keys 16 g .. 16 g + 15 of the tile in both products: S comes out in the
// registers that P goes in, and a page's scales are one value a lane.
#include <hip/hip_runtime.h>

#include "dk_host.hpp"
#include "dk_kv.hpp"

namespace dk {

int kv_view(const dk_kv_cache* c, KvView* view);

constexpr int kTile = 64;          // keys of a tile
constexpr int kAttendWaves = 4;
constexpr float kNegInf = -__builtin_huge_valf();
// A row's maximum is moved only when a tile passes it by this much (base 2):
// P stays below 2^8, far inside fp16, and the usual tile rescales nothing.
constexpr float kLazy = 8.0f;

struct AttendArgs {
  KvView c;
  const uint16_t* q;
  long long qt, qh;  // strides of tokens and heads, elements
  uint16_t* out;
  const int32_t* tables;
  const int32_t* lens;
  const int32_t* offsets;
  float* partials;
  int4* starts;
  float scale_log2;
  int width, tokens, requests, group, bf16, causal;
};

// One sequence's share of the work.
struct Seq {
  int q0, n, len, row_tiles, tiles;
};

template <int NT>
__device__ __forceinline__ Seq sequence(const AttendArgs& a, int b) {
  Seq s;
  s.q0 = b, s.n = 1;
  if (a.offsets) {
    s.q0 = min(max(a.offsets[b], 0), a.tokens);
    s.n = max(min(a.offsets[b + 1], a.tokens) - s.q0, 0);
  }
  s.len = min((long long)max(a.lens[b], 0), (long long)a.width << a.c.page_shift);
  s.row_tiles = (int)(((long long)s.n * a.group + 16 * NT - 1) / (16 * NT));
  s.tiles = max((s.len + kTile - 1) / kTile, 1);  // an empty sequence's rows are written too
  return s;
}

__device__ __forceinline__ h8_t codes_to_f16(uint32_t lo, uint32_t hi) {
  // A byte u = code + 128 under 0x64 is the fp16 value 1024 + u.
  const uint32_t a = lo ^ 0x80808080u, b = hi ^ 0x80808080u;
  const h2_t bias = {(_Float16)-1152.0f, (_Float16)-1152.0f};
  const h2_t p0 = as_h2(__builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) + bias;
  const h2_t p1 = as_h2(__builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) + bias;
  const h2_t p2 = as_h2(__builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) + bias;
  const h2_t p3 = as_h2(__builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) + bias;
  h8_t r;
  r[0] = p0[0]; r[1] = p0[1]; r[2] = p1[0]; r[3] = p1[1];
  r[4] = p2[0]; r[5] = p2[1]; r[6] = p3[0]; r[7] = p3[1];
  return r;
}

// Eight elements of a query as fp32.
__device__ __forceinline__ void load_q8(const uint16_t* p, int bf16, float (&x)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16 ? pair_lo<true>(ws[i]) : pair_lo<false>(ws[i]);
    x[2 * i + 1] = bf16 ? pair_hi<true>(ws[i]) : pair_hi<false>(ws[i]);
  }
}

// A power of two that brings a row's largest element to [2^14, 2^15), and so
// makes a bf16 row exact in fp16 but for elements 2^-29 below its largest.
__device__ __forceinline__ int row_exponent(float amax) {
  const int e = (int)(__builtin_bit_cast(uint32_t, amax) >> 23) - 127;  // amax >= 0
  return amax == 0.0f ? 0 : min(14 - e, 126);
}
__device__ __forceinline__ float pow2i(int e) {
  return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}

__device__ __forceinline__ float max_groups(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float sum_groups(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

__device__ __forceinline__ void store_half4(const AttendArgs& a, uint16_t* at, const float (&x)[4]) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = a.bf16 ? f2bf(x[2 * i]) | (uint32_t)f2bf(x[2 * i + 1]) << 16
                  : f2h(x[2 * i]) | (uint32_t)f2h(x[2 * i + 1]) << 16;
  *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
}

// Where row r of a sequence and key/value head goes in the output.
template <int D>
__device__ __forceinline__ uint16_t* out_row(const AttendArgs& a, const Seq& s, int h, int r) {
  const int i = r / a.group;
  const long long head = (long long)h * a.group + (r - i * a.group);
  return a.out + ((long long)(s.q0 + i) * ((long long)a.c.heads * a.group) + head) * D;
}

template <int D, int NT>
struct AttendLds {
  static constexpr int kRows = 16 * NT;
  static constexpr int kStride = D + 4;
  float o[kAttendWaves][kRows][kStride];
  float m[kAttendWaves][kRows];
  float l[kAttendWaves][kRows];
  long long sums[kAttendWaves];
  int found;
  long long found_base;
};

// The keys tile0 .. tile1 of one (sequence, key/value head, row tile): the
// waves take tiles in turn and leave their O, m and l in LDS.
template <int D, int NT>
__device__ void attend_tiles(const AttendArgs& a, AttendLds<D, NT>& lds, const Seq& s, int b, int h,
                             int rt, int tile0, int tile1, int lane, int wave) {
  constexpr int kJ = D / 64;  // 16-byte pieces of a key a lane holds
  constexpr int kD = D / 16;
  const int n16 = lane & 15, g = lane >> 4;
  const int shift = a.c.page_shift, P = 1 << shift;
  const int rows = s.n * a.group;

  // This lane's columns: the row, the keys it sees, its query as fp16.
  h8_t qf[NT][kJ][2];
  float qs[NT], m[NT], l[NT];
  int limit[NT], most = 0, least = INT32_MAX;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = (rt * NT + t) * 16 + n16;
    const bool real = r < rows;
    const int i = real ? r / a.group : 0;
    limit[t] = !real ? 0 : a.causal ? s.len - s.n + i + 1 : s.len;
    const uint16_t* q = a.q + (long long)(s.q0 + i) * a.qt +
                        ((long long)h * a.group + (real ? r - i * a.group : 0)) * a.qh;
    float x[kJ][2][8];
    float amax = 0;
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        load_q8(q + 16 * (4 * j + g) + 8 * e, a.bf16, x[j][e]);
#pragma unroll
        for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(x[j][e][k]));
      }
    const int ex = row_exponent(max_groups(amax));
    const float f = pow2i(ex);
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 0; k < 8; ++k) qf[t][j][e][k] = (_Float16)(x[j][e][k] * f);
    qs[t] = a.scale_log2 * pow2i(-ex);
    m[t] = kNegInf;
    l[t] = 0;
    most = max(most, limit[t]);
    least = min(least, real ? limit[t] : INT32_MAX);
  }
#pragma unroll
  for (int d = 1; d < 16; d *= 2) {
    most = max(most, __shfl_xor(most, d));
    least = min(least, __shfl_xor(least, d));
  }
  most = __builtin_amdgcn_readfirstlane(most);
  least = __builtin_amdgcn_readfirstlane(least);

  f4_t o[NT][kD] = {};
  const int32_t* table = a.tables + (long long)b * a.width;
  const long long page_bytes = (long long)a.c.heads * D * P;
  const long long head_bytes = (long long)h * D * P;

  for (int tile = tile0 + wave; tile < tile1; tile += kAttendWaves) {
    const int key0 = tile * kTile;
    if (key0 >= most) break;
    // The page of this lane's key pieces (A rows 4 i + v of group n16 / 4)
    // and of its value pieces and scales (group g).
    const int kt = key0 + 16 * (n16 >> 2), vt = key0 + 16 * g;
    const int kcol = kt >> shift, vcol = vt >> shift;
    int kp = kcol < a.width && kt < s.len ? table[kcol] : -1;
    int vp = vcol < a.width && vt < s.len ? table[vcol] : -1;
    const bool have = vp >= 0 && vp < a.c.pages;
    kp = kp >= 0 && kp < a.c.pages ? kp : 0;
    vp = have ? vp : 0;
    const int8_t* kb = a.c.k + kp * page_bytes + head_bytes + ((kt & (P - 1)) + (n16 & 3)) * 16;
    const int8_t* vb = a.c.v + vp * page_bytes + head_bytes + n16 * P + (vt & (P - 1));
    uint4 kw[4][kJ], vw[kD];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < kJ; ++j)
        kw[i][j] = *reinterpret_cast<const uint4*>(kb + ((4 * j + g) * P + 4 * i) * 16);
#pragma unroll
    for (int d = 0; d < kD; ++d) vw[d] = *reinterpret_cast<const uint4*>(vb + 16 * d * P);
    const float sk = a.c.ks[(long long)vp * a.c.heads + h];
    const float sv = have ? a.c.vs[(long long)vp * a.c.heads + h] : 0.0f;

    f4_t st[NT][4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        const h8_t k0 = codes_to_f16(kw[i][j].x, kw[i][j].y);
        const h8_t k1 = codes_to_f16(kw[i][j].z, kw[i][j].w);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          st[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qf[t][j][0], st[t][i], 0, 0, 0);
          st[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qf[t][j][1], st[t][i], 0, 0, 0);
        }
      }

    // Value scales relative to the tile's largest, so that P in fp16 keeps
    // its bits whatever the values' size is; exactly 1 on a page alone.
    float top = max_groups(sv < __builtin_huge_valf() ? sv : 0.0f);
    top = top > 0 ? top : 1.0f;
    const float rel = sv / top;

    const bool whole = key0 + kTile <= least && __all(have);
    h8_t pf[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float c = sk * qs[t];
      float x[4][4], tm = kNegInf;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[i][v] = st[t][i][v] * c;
          if (!whole && !(have && vt + 4 * i + v < limit[t])) x[i][v] = kNegInf;
          tm = fmaxf(tm, x[i][v]);
        }
      if (__any(tm > m[t] + kLazy)) {
        const float mn = fmaxf(m[t], max_groups(tm));
        const float alpha = mn == kNegInf ? 1.0f : exp2f(m[t] - mn);
        l[t] *= alpha;
#pragma unroll
        for (int d = 0; d < kD; ++d) o[t][d] *= alpha;
        m[t] = mn;
      }
      const float base = m[t] == kNegInf ? 0.0f : m[t];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float p = exp2f(x[i][v] - base);
          l[t] += p;
          // A key that is not seen has p = 0 on a page of any scale.
          const float w = x[i][v] == kNegInf ? 0.0f : p * rel;
          pf[t][i >> 1][4 * (i & 1) + v] = (_Float16)w;
        }
    }
#pragma unroll
    for (int d = 0; d < kD; ++d) {
      const h8_t v0 = codes_to_f16(vw[d].x, vw[d].y);
      const h8_t v1 = codes_to_f16(vw[d].z, vw[d].w);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f4_t y = {};
        y = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[t][0], y, 0, 0, 0);
        y = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[t][1], y, 0, 0, 0);
#pragma unroll
        for (int v = 0; v < 4; ++v) o[t][d][v] = fmaf(top, y[v], o[t][d][v]);
      }
    }
  }

#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = 16 * t + n16;
    const float sum = sum_groups(l[t]);
    if (g == 0) {
      lds.m[wave][r] = m[t];
      lds.l[wave][r] = sum;
    }
#pragma unroll
    for (int d = 0; d < kD; ++d)
      *reinterpret_cast<f4_t*>(&lds.o[wave][r][16 * d + 4 * g]) = o[t][d];
  }
}

// The work is (sequence, key/value head, row tile, tile of keys), in that
// order; a workgroup takes an equal share of it, whatever the lengths are.
// What a share holds of an item that others share goes to the workspace, and
// attend_join adds it up.
template <int D, int NT>
__global__ __launch_bounds__(kAttendWaves * 64) void attend_kernel(AttendArgs a) {
  using Lds = AttendLds<D, NT>;
  constexpr int kRows = Lds::kRows;
  __shared__ Lds lds;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wg = blockIdx.x;

  // Every workgroup adds up all sequences' work to find its own.
  const int each = (a.requests + 255) / 256;
  const int b0 = min(tid * each, a.requests), b1 = min(b0 + each, a.requests);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    const Seq s = sequence<NT>(a, b);
    mine += (long long)a.c.heads * s.row_tiles * s.tiles;
  }
  long long inc = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const long long o = __shfl_up(inc, d);
    if (lane >= d) inc += o;
  }
  if (lane == 63) lds.sums[wave] = inc;
  __syncthreads();
  long long total = 0, before = inc - mine;
#pragma unroll
  for (int w = 0; w < kAttendWaves; ++w) {
    if (w < wave) before += lds.sums[w];
    total += lds.sums[w];
  }
  const long long share = max((total + gridDim.x - 1) / gridDim.x, (long long)kAttendWaves);
  const long long begin = wg * share, end = min(begin + share, total);
  if (tid == 0) a.starts[wg] = make_int4(-1, 0, 0, 0);
  if (begin >= end) return;
  if (begin >= before && begin < before + mine) {
    long long base = before;
    for (int b = b0; b < b1; ++b) {
      const Seq s = sequence<NT>(a, b);
      const long long w = (long long)a.c.heads * s.row_tiles * s.tiles;
      if (begin < base + w) {
        lds.found = b;
        lds.found_base = base;
        break;
      }
      base += w;
    }
  }
  __syncthreads();
  int b = lds.found;
  long long base = lds.found_base;

  for (long long cur = begin; cur < end;) {
    const Seq s = sequence<NT>(a, b);
    const long long w = (long long)a.c.heads * s.row_tiles * s.tiles;
    if (cur >= base + w) {
      base += w;
      ++b;
      continue;
    }
    const long long local = cur - base;
    const int item = (int)(local / s.tiles), tile0 = (int)(local % s.tiles);
    const int tile1 = (int)min((long long)s.tiles, tile0 + (end - cur));
    const int h = item / s.row_tiles, rt = item % s.row_tiles;
    attend_tiles<D, NT>(a, lds, s, b, h, rt, tile0, tile1, lane, wave);
    __syncthreads();

    const bool shared = tile0 > 0 || tile1 < s.tiles;
    const int slot = 2 * wg + (cur == begin ? 0 : 1);
    float* part = a.partials + (long long)slot * kRows * (D + 2);
    const int rows = min(kRows, s.n * a.group - rt * kRows);
    for (int u = tid; u < rows * (D / 4); u += 256) {
      const int r = u / (D / 4), d = u % (D / 4) * 4;
      float mx = kNegInf;
#pragma unroll
      for (int k = 0; k < kAttendWaves; ++k) mx = fmaxf(mx, lds.m[k][r]);
      float sum = 0, x[4] = {};
#pragma unroll
      for (int k = 0; k < kAttendWaves; ++k) {
        const float f = lds.m[k][r] == kNegInf ? 0.0f : exp2f(lds.m[k][r] - mx);
        sum += f * lds.l[k][r];
        if (f == 0.0f) continue;  // a wave without keys
        const f4_t y = *reinterpret_cast<const f4_t*>(&lds.o[k][r][d]);
#pragma unroll
        for (int v = 0; v < 4; ++v) x[v] = fmaf(f, y[v], x[v]);
      }
      if (shared) {
        *reinterpret_cast<f4_t*>(part + r * D + d) = f4_t{x[0], x[1], x[2], x[3]};
        if (d == 0) {
          part[kRows * D + r] = mx;
          part[kRows * D + kRows + r] = sum;
        }
      } else {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int v = 0; v < 4; ++v) x[v] *= inv;
        store_half4(a, out_row<D>(a, s, h, rt * kRows + r) + d, x);
      }
    }
    if (shared && tile0 == 0 && tid == 0) {
      // The pieces that follow are the first ones of the next workgroups.
      const int more = (int)((s.tiles - tile1 + share - 1) / share);
      a.starts[wg] = make_int4(b, item, slot, more);
    }
    __syncthreads();
    cur += tile1 - tile0;
  }
}

// Adds up the pieces of the item that starts in workgroup blockIdx.x and
// goes on in the next ones, in their order. A workgroup does four rows.
template <int D, int NT>
__global__ __launch_bounds__(4 * (D / 4)) void attend_join(AttendArgs a) {
  constexpr int kRows = 16 * NT;
  const int4 start = a.starts[blockIdx.x];
  if (start.x < 0) return;
  const Seq s = sequence<NT>(a, start.x);
  const int h = start.y / s.row_tiles, rt = start.y % s.row_tiles;
  const int r = blockIdx.y * 4 + threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
  if (r >= min(kRows, s.n * a.group - rt * kRows)) return;
  const long long size = (long long)kRows * (D + 2);
  float mx = kNegInf, sum = 0, x[4] = {};
  for (int k = 0; k <= start.w; ++k) {
    const float* part = a.partials + (k == 0 ? (long long)start.z : 2LL * (blockIdx.x + k)) * size;
    const float pm = part[kRows * D + r], pl = part[kRows * D + kRows + r];
    const f4_t y = *reinterpret_cast<const f4_t*>(part + r * D + d);
    const float mn = fmaxf(mx, pm);
    const float fo = mx == kNegInf ? 0.0f : exp2f(mx - mn);
    const float fn = pm == kNegInf ? 0.0f : exp2f(pm - mn);
    sum = sum * fo + pl * fn;
#pragma unroll
    for (int v = 0; v < 4; ++v) x[v] = x[v] * fo + (fn == 0.0f ? 0.0f : y[v] * fn);
    mx = mn;
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int v = 0; v < 4; ++v) x[v] *= inv;
  store_half4(a, out_row<D>(a, s, h, rt * kRows + r) + d, x);
}

}  // namespace dk

namespace {

constexpr int kWorkgroups = 512;  // two a CU

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Column tiles of a wave: 16 rows where no sequence has more.
int column_tiles(int max_query_len, int group) {
  return (long long)max_query_len * group <= 16 ? 1 : 2;
}

size_t workspace(int nt, int head_size) {
  return (size_t)kWorkgroups * sizeof(int4) +
         (size_t)kWorkgroups * 2 * 16 * nt * (head_size + 2) * sizeof(float);
}

}  // namespace

extern "C" size_t dk_kv_attend_workspace_bytes(int num_tokens, int requests, int q_heads, int heads,
                                               int head_size, int table_width, int page_size,
                                               int max_query_len) {
  (void)table_width;
  (void)page_size;
  if (num_tokens <= 0 || requests <= 0 || heads <= 0 || q_heads <= 0) return 0;
  return workspace(column_tiles(max_query_len, q_heads / heads), head_size);
}

extern "C" int dk_kv_attend(const void* q, int dtype, long long q_token_stride,
                            long long q_head_stride, const dk_kv_cache* cache,
                            const int32_t* tables, int table_width, const int32_t* seq_lens,
                            const int32_t* query_offsets, int num_tokens, int requests,
                            int q_heads, int max_query_len, float scale, int causal, void* out,
                            void* workspace_ptr, size_t workspace_bytes, hipStream_t stream) {
  dk::KvView view;
  if (const int rc = dk::kv_view(cache, &view)) return rc;
  if (dtype != DK_KV_F16 && dtype != DK_KV_BF16)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "q must be fp16 or bf16");
  if (num_tokens < 0 || requests < 0 || table_width < 0)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT,
                         "num_tokens, requests and table_width must be >= 0");
  if (q_heads < 1 || q_heads % view.heads != 0)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "q_heads=%d must be a multiple of the cache's heads (%d)",
                         q_heads, view.heads);
  if ((long long)num_tokens * (q_heads / view.heads) > INT32_MAX - 64)
    return dk::set_error(DK_ERR_UNSUPPORTED, "num_tokens * q_heads / heads too large");
  if (((long long)table_width << view.page_shift) > INT32_MAX - dk::kTile)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "table_width * page_size must fit in int32");
  if (!query_offsets && num_tokens != requests)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT,
                         "without query_offsets each of the %d requests has one query, got %d",
                         requests, num_tokens);
  if (max_query_len < 1)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "max_query_len must be >= 1");
  if (num_tokens == 0 || requests == 0) return DK_OK;
  if (!q || !out || !seq_lens || (!tables && table_width > 0) || !workspace_ptr)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT,
                         "q, out, tables, seq_lens and the workspace must not be NULL");
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(workspace_ptr, 16))
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "q, out and the workspace must be 16-byte aligned");
  if (q_token_stride % 8 || q_head_stride % 8)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "the strides of q must be multiples of 8");
  const int group = q_heads / view.heads;
  const int nt = column_tiles(max_query_len, group);
  if (workspace_bytes < workspace(nt, cache->head_size))
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "the workspace has %zu of %zu bytes",
                         workspace_bytes, workspace(nt, cache->head_size));
  dk::AttendArgs a{};
  a.c = view;
  a.q = static_cast<const uint16_t*>(q);
  a.qt = q_token_stride;
  a.qh = q_head_stride;
  a.out = static_cast<uint16_t*>(out);
  a.tables = tables;
  a.lens = seq_lens;
  a.offsets = query_offsets;
  a.starts = static_cast<int4*>(workspace_ptr);
  a.partials = reinterpret_cast<float*>(a.starts + kWorkgroups);
  a.scale_log2 = scale * 1.44269504088896340736f;
  a.width = cache->pages > 0 ? table_width : 0;  // no pages, no keys
  a.tokens = num_tokens;
  a.requests = requests;
  a.group = group;
  a.bf16 = dtype == DK_KV_BF16;
  a.causal = causal != 0;
  auto launch = [&](auto main, auto join) {
    hipLaunchKernelGGL(main, dim3(kWorkgroups), dim3(dk::kAttendWaves * 64), 0, stream, a);
    hipLaunchKernelGGL(join, dim3(kWorkgroups, 4 * nt), dim3(cache->head_size), 0, stream, a);
  };
  if (cache->head_size == 64) {
    if (nt == 1) launch(dk::attend_kernel<64, 1>, dk::attend_join<64, 1>);
    else launch(dk::attend_kernel<64, 2>, dk::attend_join<64, 2>);
  } else {
    if (nt == 1) launch(dk::attend_kernel<128, 1>, dk::attend_join<128, 1>);
    else launch(dk::attend_kernel<128, 2>, dk::attend_join<128, 2>);
  }
  return dk::check_launch("attend launch");
}
