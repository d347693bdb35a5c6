// Attention over the paged 8-bit key/value cache.
// Layouts in dk_kv.hpp, contract in include/decode_kernel/dk_kv.h.
//
// For a row (a query head of one token) with keys j:
//   s_j = scale q.k_j,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),
// in one pass with a running m (fp32, base 2). The rows of one key/value head
// and sequence (the group's query heads times the sequence's queries) are
// the columns of two matrix products over a tile of 64 keys,
//   S^T [64 keys, rows] = K Q^T,   O^T [elements, rows] += V^T P^T,
// on fp16 MFMAs with fp32 sums. Codes are whole numbers up to 127, exact in
// fp16; a page's scale multiplies S after, P before, the product. Which key a
// row of the first product is, is free: it is chosen so that S comes out in
// the registers that P goes into the second product from. Scales are taken to
// be at least 0 (or NaN), as append leaves them.
//
// attend_few reads the cache once and is bound by that; attend_many keeps the
// matrix units busy for long query rows. Which one takes a sequence: dispatch.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "dk_host.hpp"
#include "dk_kv.hpp"

namespace dk {

int kv_view(const dk_kv_cache* c, KvView* view);

constexpr int kTile = 64;          // keys of a tile
constexpr int kWorkgroups = 256;   // one a CU
constexpr float kNegInf = -__builtin_huge_valf();
// A row's maximum is moved only when a tile passes it by this much (base 2), so
// that the usual tile rescales nothing: P stays below 2^kLazy. Times 2^kLift it
// fills fp16 upwards, whose second part ends at 2^-25: a weight is kept down to
// 2^-36 of the row's largest, where 131072 of them add 2^-19.
constexpr float kLazy = 4.0f, kLift = 11.0f, kLower = 0x1p-11f;  // kLower: what undoes the lift

struct AttendArgs {
  KvView c;
  const uint16_t* q;
  long long qt, qh;  // strides of tokens and heads, elements
  uint16_t* out;
  const int32_t* tables;
  const int32_t* lens;
  const int32_t* offsets;
  float* partials;
  unsigned long long* flags;  // two a workgroup, as its pieces
  unsigned long long gen;
  float scale_log2;
  int width, tokens, requests, group, bf16, causal;
  int few_rows;  // sequences of more rows are attend_many's
  int clear;     // this kernel writes the rows of no sequence
};

// One sequence: its queries (below 0 of them: offsets that decrease), its keys,
// its row tiles and tiles of keys.
struct Seq {
  int q0, n, len, row_tiles, tiles;
};

__device__ __forceinline__ Seq sequence(const AttendArgs& a, int b, int rows_a_tile, bool many) {
  Seq s;
  s.q0 = b, s.n = 1;
  if (a.offsets) {
    s.q0 = min(max(a.offsets[b], 0), a.tokens);
    s.n = min(max(a.offsets[b + 1], 0), a.tokens) - s.q0;
  }
  s.len = min((long long)max(a.lens[b], 0), (long long)a.width << a.c.page_shift);
  const int rows = max(s.n, 0) * a.group;
  s.row_tiles = (rows > a.few_rows) == many ? (rows + rows_a_tile - 1) / rows_a_tile : 0;
  s.tiles = max((s.len + kTile - 1) / kTile, 1);  // an empty sequence's rows are written too
  return s;
}

// The tokens that belong to a sequence: first <= t < last.
struct Owned {
  int first, last;
};
__device__ __forceinline__ Owned owned_tokens(const AttendArgs& a) {
  Owned w{0, a.tokens};
  if (a.offsets) {
    w.first = min(max(a.offsets[0], 0), a.tokens);
    w.last = min(max(a.offsets[a.requests], w.first), a.tokens);
  }
  return w;
}

// The others' rows are zeros, each workgroup's part of them.
template <int D>
__device__ __forceinline__ void clear_rows(const AttendArgs& a, const Owned& w, int tid, int threads) {
  const long long row = (long long)a.c.heads * a.group * (D / 8);  // 16 bytes each
  const long long before = w.first * row, all = before + (a.tokens - w.last) * row;
  uint4* out = reinterpret_cast<uint4*>(a.out);
  for (long long u = (long long)blockIdx.x * threads + tid; u < all; u += (long long)kWorkgroups * threads)
    out[u < before ? u : u - before + w.last * row] = zero4();
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

// Two weights as their first fp16 parts. The second part is what these very
// bits leave: without the asm the compiler rounds a product to fp16 twice, from
// fp32 for the first part and exactly where that is taken off again, which
// differ on ties: one weight in some ten thousand was half a step of fp16 off.
__device__ __forceinline__ h2_t first_parts(float x, float y) {
  uint32_t w = __builtin_bit_cast(uint32_t, h2_t{(_Float16)x, (_Float16)y});
  asm("" : "+v"(w));
  return as_h2(w);
}

// Eight elements of a query as fp32.
__device__ __forceinline__ void q_floats(const uint4& w, int bf16, float (&x)[8]) {
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

// Of a value >= 0; 0 below the normal range.
__device__ __forceinline__ float floor_pow2(float v) {
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & 0x7F800000u);
}

// The four lane groups' values against each other: exchanges of half rows of
// registers, no LDS on the way.
__device__ __forceinline__ float max_groups(float v) {
  const auto h = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v),
                                                  __builtin_bit_cast(uint32_t, v), false, false);
  v = fmaxf(__builtin_bit_cast(float, (uint32_t)h[0]), __builtin_bit_cast(float, (uint32_t)h[1]));
  const auto q = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v),
                                                  __builtin_bit_cast(uint32_t, v), false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)q[0]), __builtin_bit_cast(float, (uint32_t)q[1]));
}
__device__ __forceinline__ float sum_groups(float v) {
  const auto h = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v),
                                                  __builtin_bit_cast(uint32_t, v), false, false);
  v = __builtin_bit_cast(float, (uint32_t)h[0]) + __builtin_bit_cast(float, (uint32_t)h[1]);
  const auto q = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v),
                                                  __builtin_bit_cast(uint32_t, v), false, false);
  return __builtin_bit_cast(float, (uint32_t)q[0]) + __builtin_bit_cast(float, (uint32_t)q[1]);
}

// The wave's halves against each other.
__device__ __forceinline__ float max_halves(float v) {
  const auto h = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v),
                                                  __builtin_bit_cast(uint32_t, v), false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)h[0]), __builtin_bit_cast(float, (uint32_t)h[1]));
}
__device__ __forceinline__ float sum_halves(float v) {
  const auto h = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v),
                                                  __builtin_bit_cast(uint32_t, v), false, false);
  return __builtin_bit_cast(float, (uint32_t)h[0]) + __builtin_bit_cast(float, (uint32_t)h[1]);
}

// The 16 lanes of a row against each other.
__device__ __forceinline__ float max_row(float v) {
  v = fmaxf(v, dpp<0xB1>(v));   // quad_perm [1,0,3,2]
  v = fmaxf(v, dpp<0x4E>(v));   // quad_perm [2,3,0,1]
  v = fmaxf(v, dpp<0x141>(v));  // row_half_mirror
  return fmaxf(v, dpp<0x140>(v));  // row_mirror
}
__device__ __forceinline__ float sum_row(float v) {
  v += dpp<0xB1>(v);
  v += dpp<0x4E>(v);
  v += dpp<0x141>(v);
  return v + dpp<0x140>(v);
}
__device__ __forceinline__ int max_row(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false));
  return max(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false));
}
// Of lanes 0..31, in lane 0.
__device__ __forceinline__ int max_half_wave(int v) {
  v = max_row(v);
  return max(v, __builtin_amdgcn_readlane(v, 16));
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

// ---------------------------------------------------------------------------
// Few rows: bound by the cache's bytes.
//
// The work is (sequence, key/value head, row tile, tile of keys), in that
// order. Every wave of the card's 256 workgroups takes an equal share of it,
// whatever the sequences' lengths are; an item (one row tile with all its
// keys) costs kItemCost tiles on top, for the latency of its start. Where
// items are few and short, a workgroup's share is one item (kAloneTiles). A
// wave writes what it has of a whole item, and leaves the piece of an item it
// shares, at its start or its end, in LDS; the workgroup joins the pieces of
// an item, and an item that several workgroups share goes through the
// workspace, where the last one to arrive adds the pieces up in their order.
//
// v_mfma_f32_16x16x32_f16, 16 rows to a product: lane group g (16 lanes) takes
// the keys 16 g .. 16 g + 15 of the tile in both products, and a page's scales
// are one value a lane. P goes in as two fp16 parts, which costs nothing here.
//
// 131071 keys of 8 heads of 128 for one token (8 rows a head): 268 MB in 60 us,
// 4.5 TB/s (a large read has 6.1). The tiles themselves run at 6.9 TB/s; 5 us
// go by before them (lengths, page numbers, first codes: three trips to
// memory) and 10 after (joining in LDS, flags, joining 32 workgroups' pieces).
// 64 ragged sequences in pages of 16: 185 MB in 46 us. 700 keys of 32 heads:
// 13 us, all of it such trips. With 32 rows and heads of 128 (NT 2) the state
// takes 256 registers and 112 accumulation registers, one wave a SIMD, and part
// of it moves between them in the loop; what is uniform and little used lies in
// vector lanes here and in attend_many (30 to 56 scalar registers). Equal shares
// a workgroup instead of a wave, its four waves on one item, took 50 us and more
// where short sequences stand together, and a second launch to join 5 us more.
// ---------------------------------------------------------------------------
constexpr int kItemCost = 1;

// With no more items than workgroups, each goes to one of its own where that
// makes a wave's share longer by no more than this many tiles (of a workgroup
// of eight waves; twice as many of four): a tile costs 2.5 us where a wave has
// few, meeting through the workspace 4 to 7. us, shared / alone, fp16, heads of
// 128, pages of 64, at 200, 500, 700, 1500 and 3000 keys:
//    1 sequence, 32 heads                15.1/9.0  14.7/10.9  14.4/13.3  15/19  14/24
//   16 sequences, 8 x 8 heads            15.7/9.2  15.6/11.2  15.5/14.0  21/20  23/26
//   32 sequences, 8 x 8 heads            15.7/9.3  20.1/12.0  19.6/15.7  28/23  36/36
//    8 sequences, 8 x 8, four queries    23.7/16   25.0/19    19.6/20    29/29  26/42
constexpr int kAloneTiles = 1;

template <int D, int NT>
struct Few {
  static constexpr int kRows = 16 * NT;
  static constexpr int kWaves = D * NT > 128 ? 4 : 8;  // as many as LDS holds two pieces of
  static constexpr int kThreads = kWaves * 64;
  static constexpr int kPiece = kRows * (D + 2);  // floats of a piece in the workspace
  struct Piece {
    int b, item, tile0, tile1;
    int start;  // of the item in the work
  };
  struct Shared {  // an item that several workgroups have pieces of
    int b, item, wg0, pieces;
    Seq s;
  };
  struct Lds {
    float o[kWaves][2][kRows][D + 4];
    float m[kWaves][2][kRows];
    float l[kWaves][2][kRows];
    Piece piece[kWaves][2];
    Seq of_piece[kWaves][2];
    float w[kRows][16];  // weights of the pieces being joined
    float sum[kRows];
    Shared shared[2];
    int last[2];
  };
  // In the place of o: maxima, then weights, and sums of an item's pieces.
  static constexpr int kMostPieces = kWorkgroups;
  static_assert(2 * kMostPieces * kRows + kThreads * 4 <= kWaves * 2 * kRows * (D + 4), "");
};

// What a wave holds of a row tile: lane (g, n) the sums of column n over
// elements 16 d + 4 g + v, its maximum, and l over its own keys alone.
template <int D, int NT>
struct Sums {
  f4_t o[NT][D / 16];
  float m[NT], l[NT];
};

// The queries of a row tile as the product's right operand, in fp16 times a
// power of two, and what multiplies a column's scores.
template <int D, int NT>
struct Queries {
  h8_t f[NT][D / 64][2];
  float scale[NT];
  int limit[NT];    // keys that a column's row sees
  int most, least;  // of all columns with a row
};

// A column's eight elements each as they lie in memory, on their way.
template <int D, int NT>
struct RawQueries {
  uint4 w[NT][D / 64][2];
};

template <int D, int NT>
__device__ __forceinline__ void load_queries(const AttendArgs& a, const Seq& s, int h, int rt, int lane,
                                             RawQueries<D, NT>& raw, Queries<D, NT>& y) {
  const int n16 = lane & 15, g = lane >> 4;
  const int rows = s.n * a.group;
  int most = 0, least = INT32_MAX;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = (rt * NT + t) * 16 + n16;
    const bool real = r < rows;
    const int i = real ? r / a.group : 0;
    y.limit[t] = !real ? 0 : a.causal ? s.len - s.n + i + 1 : s.len;
    const uint16_t* q = a.q + (long long)(s.q0 + i) * a.qt +
                        ((long long)h * a.group + (real ? r - i * a.group : 0)) * a.qh + 16 * g;
#pragma unroll
    for (int j = 0; j < D / 64; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) raw.w[t][j][e] = *reinterpret_cast<const uint4*>(q + 64 * j + 8 * e);
    most = max(most, y.limit[t]);
    least = min(least, real ? y.limit[t] : INT32_MAX);
  }
  y.most = __builtin_amdgcn_readfirstlane(max_row(most));
  y.least = -__builtin_amdgcn_readfirstlane(max_row(-least));
}

template <int D, int NT>
__device__ __forceinline__ void convert_queries(const AttendArgs& a, const RawQueries<D, NT>& raw,
                                                Queries<D, NT>& y) {
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float amax = 0;
#pragma unroll
    for (int j = 0; j < D / 64; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x[8];
        q_floats(raw.w[t][j][e], a.bf16, x);
#pragma unroll
        for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(x[k]));
      }
    const int ex = row_exponent(max_groups(amax));
    const float f = pow2i(ex);
#pragma unroll
    for (int j = 0; j < D / 64; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x[8];
        q_floats(raw.w[t][j][e], a.bf16, x);
#pragma unroll
        for (int k = 0; k < 8; ++k) y.f[t][j][e][k] = (_Float16)(x[k] * f);
      }
    y.scale[t] = a.scale_log2 * pow2i(-ex);
  }
}

// The pages of a tile that this lane's key pieces and value pieces lie on, -1
// where there is none.
struct Pages {
  int k, v;
};
__device__ __forceinline__ Pages tile_pages(const AttendArgs& a, const int32_t* table, int len,
                                            int key0, int lane) {
  const int kt = key0 + 16 * ((lane & 15) >> 2), vt = key0 + 16 * (lane >> 4);
  Pages p;
  p.k = kt < len ? table[kt >> a.c.page_shift] : -1;
  p.v = vt < len ? table[vt >> a.c.page_shift] : -1;
  return p;
}

// Keys tile0 .. tile1 of one item. The loads run a step ahead of the products:
// the next tile's keys go out when this one's scores are done, its values when
// this one's sums are, and page numbers a tile before them, so that a wave
// always has 8 KiB or more in flight.
template <int D, int NT>
__device__ __forceinline__ void attend_piece(const AttendArgs& a, const Seq& s, int b, int h, int rt,
                                             int tile0, int tile1, int lane, Sums<D, NT>& y) {
  constexpr int kJ = D / 64;  // 16-byte pieces of a key a lane holds
  constexpr int kD = D / 16;
  const int n16 = lane & 15, g = lane >> 4;
  const int shift = a.c.page_shift, P = 1 << shift;
  Queries<D, NT> q;
  const int32_t* table = a.tables + (long long)b * a.width;
  Pages next = tile_pages(a, table, s.len, tile0 * kTile, lane);
  RawQueries<D, NT> raw;
  load_queries<D, NT>(a, s, h, rt, lane, raw, q);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    y.m[t] = kNegInf;
    y.l[t] = 0;
#pragma unroll
    for (int d = 0; d < kD; ++d) y.o[t][d] = f4_t{0, 0, 0, 0};
  }
  tile1 = min(tile1, (q.most + kTile - 1) / kTile);
  if (tile0 >= tile1) return;

  const long long page_bytes = (long long)a.c.heads * D * P;
  const int8_t* kh = a.c.k + (long long)h * D * P + (g * P + (n16 & 3)) * 16;
  const int8_t* vh = a.c.v + (long long)h * D * P + n16 * P;
  const float* ksh = a.c.ks + h;
  const float* vsh = a.c.vs + h;
  uint4 kw[4][kJ], vw[kD];
  float sk, sv;
  bool have;
  int vpage;
  // Where the next tile's pieces are; a page that is not there is read as
  // page 0 and masked.
  const int8_t* kb;
  const int8_t* vb;
  auto locate = [&](int key0) {
    const int kt = key0 + 16 * (n16 >> 2), vt = key0 + 16 * g;
    const int kp = next.k >= 0 && next.k < a.c.pages ? next.k : 0;
    have = next.v >= 0 && next.v < a.c.pages;
    vpage = have ? next.v : 0;
    kb = kh + kp * page_bytes + (kt & (P - 1)) * 16;
    vb = vh + vpage * page_bytes + (vt & (P - 1));
  };
  auto load_keys = [&] {
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        kw[i][j] = *reinterpret_cast<const uint4*>(kb + (4 * j * P + 4 * i) * 16);
    sk = ksh[(long long)vpage * a.c.heads];
    sv = vsh[(long long)vpage * a.c.heads];
  };
  auto load_values = [&] {
#pragma unroll
    for (int d = 0; d < kD; ++d) vw[d] = *reinterpret_cast<const uint4*>(vb + 16 * d * P);
  };
  locate(tile0 * kTile);
  load_keys();
  load_values();
  next = tile_pages(a, table, s.len, (tile0 + 1) * kTile, lane);
  convert_queries<D, NT>(a, raw, q);

  for (int tile = tile0; tile < tile1; ++tile) {
    const int key0 = tile * kTile;
    const bool more = tile + 1 < tile1;
    f4_t st[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) st[t][i] = f4_t{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const h8_t k0 = codes_to_f16(kw[i][j].x, kw[i][j].y);
        const h8_t k1 = codes_to_f16(kw[i][j].z, kw[i][j].w);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          st[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q.f[t][j][0], st[t][i], 0, 0, 0);
          st[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q.f[t][j][1], st[t][i], 0, 0, 0);
        }
      }
    const float ck = sk;
    const bool here = have;
    const float cv = here ? sv : 0.0f;
    if (more) {
      locate(key0 + kTile);
      load_keys();
      next = tile_pages(a, table, s.len, key0 + 2 * kTile, lane);
    }

    // Value scales relative to the tile's largest, so that P in fp16 keeps
    // its bits whatever the values' size is; exactly 1 on a page alone.
    float top = max_groups(cv < __builtin_huge_valf() ? cv : 0.0f);
    top = top > 0 ? top : 1.0f;
    const float rel = cv / top;
    const float lowered = top * kLower;  // 12 bits at the least scale that has codes, 2^-126

    const bool whole = key0 + kTile <= q.least && __all(here);
    h8_t pf[NT][2], pl[NT][2];  // P in fp16 and what that leaves of it
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float c = ck * q.scale[t];
      float x[16], tm = kNegInf;
#pragma unroll
      for (int k = 0; k < 16; ++k) x[k] = st[t][k >> 2][k & 3] * c;
      const int left = here ? q.limit[t] - key0 - 16 * g : 0;  // keys seen of this lane's 16
      if (!whole) {
#pragma unroll
        for (int k = 0; k < 16; ++k) x[k] = k < left ? x[k] : kNegInf;
      }
#pragma unroll
      for (int k = 0; k < 16; ++k) tm = fmaxf(tm, x[k]);
      if (__any(tm > y.m[t] + kLazy)) {
        const float mn = fmaxf(y.m[t], max_groups(tm));
        const float alpha = mn == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(y.m[t] - mn);
        y.l[t] *= alpha;
#pragma unroll
        for (int d = 0; d < kD; ++d) y.o[t][d] *= alpha;
        y.m[t] = mn;
      }
      const float base = y.m[t] == kNegInf ? 0.0f : y.m[t] - kLift;
      float sum = 0;  // the tile's by itself: small weights are not lost one by one beside large ones
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        x[k] = __builtin_amdgcn_exp2f(x[k] - base);
        sum += x[k];
        x[k] *= rel;
      }
      y.l[t] += sum;
      if (!whole) {  // a key that is not seen has weight 0 on a page of any scale
#pragma unroll
        for (int k = 0; k < 16; ++k) x[k] = k < left ? x[k] : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < 16; k += 2) {
        const h2_t f = first_parts(x[k], x[k + 1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          pf[t][k >> 3][(k & 7) + i] = f[i];
          pl[t][k >> 3][(k & 7) + i] = (_Float16)(x[k + i] - (float)f[i]);
        }
      }
    }
#pragma unroll
    for (int d = 0; d < kD; ++d) {
      const h8_t v0 = codes_to_f16(vw[d].x, vw[d].y);
      const h8_t v1 = codes_to_f16(vw[d].z, vw[d].w);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f4_t z = {0, 0, 0, 0};
        z = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[t][0], z, 0, 0, 0);
        z = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[t][1], z, 0, 0, 0);
        z = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[t][0], z, 0, 0, 0);
        z = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[t][1], z, 0, 0, 0);
#pragma unroll
        for (int v = 0; v < 4; ++v) y.o[t][d][v] = fmaf(lowered, z[v], y.o[t][d][v]);
      }
    }
    if (more) load_values();
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) y.l[t] = sum_groups(y.l[t]) * kLower;
}

// Whether all pieces of an item are in the workspace. A workgroup sets its own
// piece's flag to the call's number when its stores are acknowledged, waits
// for that too, and looks at all flags of the item: the one whose flag is set
// last sees them all. Two that set theirs at once may both, and then write the
// same rows with the same bits. Nothing but the call's number counts as set,
// so the workspace needs no clearing; who sees them all clears them, and a
// replay of the same captured call starts clean. Relaxed accesses at agent
// scope go past the XCDs' L2s (see take_ticket in dk_kernels.hpp). One atomic
// counter an item instead took 32 workgroups that arrive together 12 us more.
__device__ __forceinline__ void set_flag(unsigned long long* f, unsigned long long v) {
  __hip_atomic_store(f, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ bool flags_set(const unsigned long long* flags, unsigned long long gen, int wg0,
                                          int pieces, int lane) {
  bool all = true;
  for (int k = lane; k < pieces; k += 64)
    all &= __hip_atomic_load(flags + 2 * (wg0 + k) + (k == 0), __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT) == gen;
  return __all(all);
}

// Two floats at once.
__device__ __forceinline__ void store_agent2(float* p, float x, float y) {
  const unsigned long long w = __builtin_bit_cast(uint32_t, x) | (unsigned long long)__builtin_bit_cast(uint32_t, y) << 32;
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_agent2(const float* p) {
  const unsigned long long w = __hip_atomic_load(reinterpret_cast<const unsigned long long*>(p),
                                                 __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__builtin_bit_cast(float, (uint32_t)w), __builtin_bit_cast(float, (uint32_t)(w >> 32)));
}

__device__ __forceinline__ float inverse_sum(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

// The last workgroup to arrive adds an item's pieces up, in their order, and
// writes its rows. The place of o in LDS is free by then.
template <int D, int NT>
__device__ __forceinline__ void join_pieces(const AttendArgs& a, typename Few<D, NT>::Lds& lds,
                                            const typename Few<D, NT>::Shared& x0, int tid) {
  using F = Few<D, NT>;
  constexpr int kRows = F::kRows, kUnits = D / 4;
  const Seq s = x0.s;
  const int wg0 = x0.wg0, pieces = x0.pieces;
  const int h = x0.item / s.row_tiles, rt = x0.item % s.row_tiles;
  const int rows = min(kRows, s.n * a.group - rt * kRows);
  const int lane = tid & 63, wave = tid >> 6;
  float* ms = &lds.o[0][0][0][0];           // [row][piece]
  float* ls = ms + F::kMostPieces * kRows;  // the same
  float* xs = ls + F::kMostPieces * kRows;  // [thread][4]
  auto piece = [&](int k) { return a.partials + (2LL * (wg0 + k) + (k == 0)) * F::kPiece; };
  if (pieces <= 16) {  // no need of LDS: each thread takes all pieces, eight at once
    for (int u = tid; u < rows * kUnits; u += F::kThreads) {
      const int r = u / kUnits, d = u % kUnits * 4;
      float mx = kNegInf, sum = 0, x[4] = {};
      for (int k0 = 0; k0 < pieces; k0 += 8) {
        float2 ml[8], o[8][2];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          ml[k] = make_float2(kNegInf, 0.0f);
          o[k][0] = o[k][1] = make_float2(0.0f, 0.0f);
          if (k0 + k < pieces) {
            const float* p = piece(k0 + k);
            ml[k] = load_agent2(p + kRows * D + 2 * r);
            o[k][0] = load_agent2(p + r * D + d);
            o[k][1] = load_agent2(p + r * D + d + 2);
          }
        }
        const float old = mx;
#pragma unroll
        for (int k = 0; k < 8; ++k) mx = fmaxf(mx, ml[k].x);
        const float f = old == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(old - mx);
        sum *= f;  // a NaN stays
#pragma unroll
        for (int v = 0; v < 4; ++v) x[v] *= f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float w = ml[k].x == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(ml[k].x - mx);
          sum += w * ml[k].y;
          x[0] = fmaf(w, o[k][0].x, x[0]);
          x[1] = fmaf(w, o[k][0].y, x[1]);
          x[2] = fmaf(w, o[k][1].x, x[2]);
          x[3] = fmaf(w, o[k][1].y, x[3]);
        }
      }
      sum = inverse_sum(sum);
#pragma unroll
      for (int v = 0; v < 4; ++v) x[v] *= sum;
      store_half4(a, out_row<D>(a, s, h, rt * kRows + r) + d, x);
    }
    return;
  }
  __syncthreads();
  for (int u = tid; u < pieces * kRows; u += F::kThreads) {
    const int k = u / kRows, r = u % kRows;
    if (r >= rows) continue;
    const float2 ml = load_agent2(piece(k) + kRows * D + 2 * r);
    ms[r * F::kMostPieces + k] = ml.x;
    ls[r * F::kMostPieces + k] = ml.y;
  }
  __syncthreads();
  for (int r = wave; r < rows; r += F::kWaves) {
    float* m = ms + r * F::kMostPieces;
    float mx = kNegInf, sum = 0;
    for (int k = lane; k < pieces; k += 64) mx = fmaxf(mx, m[k]);
    for (int d = 32; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
    for (int k = lane; k < pieces; k += 64) {
      const float w = m[k] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m[k] - mx);
      m[k] = w;
      sum += w * ls[r * F::kMostPieces + k];  // a NaN stays
    }
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) lds.sum[r] = inverse_sum(sum);
  }
  __syncthreads();
  // Where rows leave threads over, they take the pieces in `parts` turns.
  const int units = rows * kUnits;
  const int parts = max(F::kThreads / units, 1);
  const int part = units < F::kThreads ? tid / units : 0;
  for (int u0 = 0; u0 < units; u0 += F::kThreads) {
    const int u = units < F::kThreads ? tid % units : u0 + tid;
    const int r = u / kUnits, d = u % kUnits * 4;
    const bool on = part < parts && u < units;
    float x[4] = {};
    if (on) {
      for (int k0 = part; k0 < pieces; k0 += 8 * parts) {
        float2 o[8][2];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float* p = piece(min(k0 + e * parts, pieces - 1)) + r * D + d;
          o[e][0] = load_agent2(p);
          o[e][1] = load_agent2(p + 2);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (k0 + e * parts >= pieces) break;
          const float w = ms[r * F::kMostPieces + k0 + e * parts];
          x[0] = fmaf(w, o[e][0].x, x[0]);
          x[1] = fmaf(w, o[e][0].y, x[1]);
          x[2] = fmaf(w, o[e][1].x, x[2]);
          x[3] = fmaf(w, o[e][1].y, x[3]);
        }
      }
    }
    if (parts > 1) {
      if (on) *reinterpret_cast<f4_t*>(xs + 4 * tid) = f4_t{x[0], x[1], x[2], x[3]};
      __syncthreads();
      if (on && part == 0)
        for (int k = 1; k < parts; ++k) {
          const f4_t y = *reinterpret_cast<const f4_t*>(xs + 4 * (tid + k * units));
#pragma unroll
          for (int v = 0; v < 4; ++v) x[v] += y[v];
        }
    }
    if (on && part == 0) {
#pragma unroll
      for (int v = 0; v < 4; ++v) x[v] *= lds.sum[r];
      store_half4(a, out_row<D>(a, s, h, rt * kRows + r) + d, x);
    }
  }
}

// Of whole numbers >= 0, in lane 63.
__device__ __forceinline__ int wave_max(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));
  return v;
}

// Inclusive sums over the wave.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

__device__ __forceinline__ Seq lane_seq(const Seq& s, int lane) {
  Seq u;
  u.q0 = __builtin_amdgcn_readlane(s.q0, lane);
  u.n = __builtin_amdgcn_readlane(s.n, lane);
  u.len = __builtin_amdgcn_readlane(s.len, lane);
  u.row_tiles = __builtin_amdgcn_readlane(s.row_tiles, lane);
  u.tiles = __builtin_amdgcn_readlane(s.tiles, lane);
  return u;
}

__device__ __forceinline__ Seq uniform_seq(const Seq& s) {
  Seq u;
  u.q0 = __builtin_amdgcn_readfirstlane(s.q0);
  u.n = __builtin_amdgcn_readfirstlane(s.n);
  u.len = __builtin_amdgcn_readfirstlane(s.len);
  u.row_tiles = __builtin_amdgcn_readfirstlane(s.row_tiles);
  u.tiles = __builtin_amdgcn_readfirstlane(s.tiles);
  return u;
}

template <int D, int NT>
__global__ __launch_bounds__((Few<D, NT>::kThreads)) void attend_few(AttendArgs a) {
  using F = Few<D, NT>;
  constexpr int kRows = F::kRows, kWaves = F::kWaves, kSlots = 2 * F::kWaves;
  __shared__ typename F::Lds lds;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wg = blockIdx.x;

  if (lane < 2) lds.piece[wave][lane].b = -1;
  if (tid < 2) lds.shared[tid].pieces = 0;

  // Every wave adds up all sequences' work to find its own, by itself: the
  // lanes take `each` sequences in a row, then those of the block that the
  // share starts in one by one. The host has seen to it that the sum fits.
  int each_units = 0;  // of every item, if they are one workgroup's each
  auto units_of = [&](const Seq& s) { return each_units ? each_units : s.tiles + kItemCost; };
  auto cost = [&](const Seq& s) { return a.c.heads * s.row_tiles * units_of(s); };
  const Owned owned = owned_tokens(a);  // asked for along with the lengths
  const int each = (a.requests + 63) / 64;
  int b = lane * each;
  Seq s{};
  int work = 0, items = 0, longest = 0;
  bool ordered = true;
  for (int k = 0; k < each && b + k < a.requests; ++k) {
    s = sequence(a, b + k, kRows, false);
    ordered &= s.n >= 0;
    work += cost(s);
    items += a.c.heads * s.row_tiles;
    longest = max(longest, s.row_tiles ? s.tiles : 0);
  }
  int upto = wave_scan(work);
  int total = __builtin_amdgcn_readlane(upto, 63);
  // A wave's share, and below the workgroup's.
  int share = max((int)(((unsigned)total + kWorkgroups * kWaves - 1) / (kWorkgroups * kWaves)), 1);
  const int items_upto = wave_scan(items), most_items = __builtin_amdgcn_readlane(items_upto, 63);
  longest = __builtin_amdgcn_readlane(wave_max(longest), 63);
  const int alone = (longest + kItemCost + kWaves - 1) / kWaves;  // a wave's share of the longest item
  if (most_items <= kWorkgroups && alone <= share + kAloneTiles * 8 / kWaves) {
    share = alone;
    each_units = share * kWaves;
    work = items * each_units;
    upto = items_upto * each_units;
    total = most_items * each_units;
  }
  ordered = __all(ordered);
  if (a.clear) clear_rows<D>(a, ordered ? owned : Owned{0, 0}, tid, F::kThreads);
  if (!ordered) return;  // rows of two sequences: more work than is counted in 31 bits
  const int group_share = share * kWaves;
  if (wg >= (total + group_share - 1) / group_share) return;
  const int begin = wg * group_share + wave * share, end = min(begin + share, total);
  int base = 0;
  if (begin < end) {
    int at = __builtin_ctzll(__ballot(begin < upto));
    base = __builtin_amdgcn_readlane(upto - work, at);
    b = at * each;
    if (each > 1) {
      int first = b;
      for (;; first += 64) {
        const bool real = first + lane < min(b + each, a.requests);
        s = sequence(a, real ? first + lane : 0, kRows, false);
        work = real ? cost(s) : 0;
        upto = wave_scan(work);
        if (begin < base + __builtin_amdgcn_readlane(upto, 63)) break;
        base += __builtin_amdgcn_readlane(upto, 63);
      }
      at = __builtin_ctzll(__ballot(begin < base + upto));
      base += __builtin_amdgcn_readlane(upto - work, at);
      b = first + at;
    }
    s = lane_seq(s, at);
    for (int cur = begin; cur < end;) {
      const int c = cost(s);
      if (cur >= base + c) {
        base += c;
        s = sequence(a, ++b, kRows, false);
        continue;
      }
      const int units = units_of(s);
      const int item = (unsigned)(cur - base) / (unsigned)units, at = cur - base - item * units;
      const int stop = min(units, at + (end - cur));
      cur += stop - at;
      const int tile0 = max(at - kItemCost, 0), tile1 = min(stop - kItemCost, s.tiles);
      if (tile0 >= tile1) continue;  // the item's start alone, or past its end
      const int h = (unsigned)item / (unsigned)s.row_tiles, rt = item - h * s.row_tiles;
      Sums<D, NT> y;
      attend_piece<D, NT>(a, s, b, h, rt, tile0, tile1, lane, y);
      const int n16 = lane & 15, g = lane >> 4;
      if (tile0 == 0 && tile1 == s.tiles) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int r = (rt * NT + t) * 16 + n16;
          if (r >= s.n * a.group) continue;
          const float inv = inverse_sum(y.l[t]);
          uint16_t* out = out_row<D>(a, s, h, r) + 4 * g;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            const float x[4] = {y.o[t][d][0] * inv, y.o[t][d][1] * inv, y.o[t][d][2] * inv,
                                y.o[t][d][3] * inv};
            store_half4(a, out + 16 * d, x);
          }
        }
      } else {
        const int slot = tile0 == 0 ? 1 : 0;  // at the share's end, or its start
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int r = 16 * t + n16;
          if (g == 0) {
            lds.m[wave][slot][r] = y.m[t];
            lds.l[wave][slot][r] = y.l[t];
          }
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
            *reinterpret_cast<f4_t*>(&lds.o[wave][slot][r][16 * d + 4 * g]) = y.o[t][d];
        }
        if (lane == 0) {
          lds.piece[wave][slot] = typename F::Piece{b, item, tile0, tile1, base + item * units};
          lds.of_piece[wave][slot] = s;
        }
      }
    }
  }
  __syncthreads();

  // Pieces of one item stand in a row: a wave's end and the next one's start.
  // Lane i looks at piece i.
  typename F::Piece piece{-1, 0, 0, 0, 0};
  if (lane < kSlots) piece = lds.piece[lane / 2][lane % 2];
  const uint32_t filled = (uint32_t)__ballot(piece.b >= 0);
  const uint32_t below = filled & ((1u << (lane & 31)) - 1);
  const int prev = below ? 31 - __builtin_clz(below) : 0;
  const int prev_b = __shfl(piece.b, prev), prev_item = __shfl(piece.item, prev);  // by every lane
  const bool same = below && prev_b == piece.b && prev_item == piece.item;
  const uint32_t starts = (uint32_t)__ballot(piece.b >= 0 && !same);
  for (uint32_t todo = starts; todo; todo &= todo - 1) {
    const int i = __builtin_ctz(todo);
    const uint32_t after = todo & (todo - 1);
    const uint32_t group = filled & ~((1u << i) - 1) & (after ? (after & -after) - 1 : ~0u);
    const int last_piece = 31 - __builtin_clz(group);
    const int b = __builtin_amdgcn_readlane(piece.b, i);
    const int item = __builtin_amdgcn_readlane(piece.item, i);
    const int tile0 = __builtin_amdgcn_readlane(piece.tile0, i);
    const int tile1 = __builtin_amdgcn_readlane(piece.tile1, last_piece);
    const int start = __builtin_amdgcn_readlane(piece.start, i);
    const Seq s = uniform_seq(lds.of_piece[i / 2][i % 2]);
    const int h = (unsigned)item / (unsigned)s.row_tiles, rt = item - h * s.row_tiles;
    const int rows = min(kRows, s.n * a.group - rt * kRows);
    const bool whole = tile0 == 0 && tile1 == s.tiles;
    float* part = a.partials + (2LL * wg + (tile0 == 0)) * F::kPiece;
    // Weights: 16 lanes a row, a lane a piece.
    for (int u = tid; u < kRows * 16; u += F::kThreads) {
      const int r = u >> 4, p = u & 15;
      const bool on = group >> p & 1;
      const float m = on ? lds.m[p / 2][p % 2][r] : kNegInf;
      const float l = on ? lds.l[p / 2][p % 2][r] : 0.0f;
      const float mx = max_row(m);
      const float w = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - mx);
      const float sum = sum_row(w * l);  // a NaN stays
      lds.w[r][p] = w;
      if (p == 0) {
        lds.sum[r] = inverse_sum(sum);
        if (!whole && r < rows) store_agent2(part + kRows * D + 2 * r, mx, sum);
      }
    }
    __syncthreads();
    for (int u = tid; u < rows * (D / 4); u += F::kThreads) {
      const int r = u / (D / 4), d = u % (D / 4) * 4;
      float x[4] = {};
      for (uint32_t k = group; k;) {  // four pieces' loads at once
        f4_t o[4];
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int p = k ? __builtin_ctz(k) : last_piece;
          o[e] = *reinterpret_cast<const f4_t*>(&lds.o[p / 2][p % 2][r][d]);
          w[e] = k ? lds.w[r][p] : 0.0f;
          k &= k - 1;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int v = 0; v < 4; ++v) x[v] = fmaf(w[e], o[e][v], x[v]);
      }
      if (whole) {
#pragma unroll
        for (int v = 0; v < 4; ++v) x[v] *= lds.sum[r];
        store_half4(a, out_row<D>(a, s, h, rt * kRows + r) + d, x);
      } else {
        store_agent2(part + r * D + d, x[0], x[1]);
        store_agent2(part + r * D + d + 2, x[2], x[3]);
      }
    }
    if (!whole && tid == 0) {
      // The item's pieces are the end of the workgroup that its first tile
      // falls to and the starts of those after it.
      const int wg0 = tile0 == 0 ? wg : (start + kItemCost) / group_share;
      const int last = (start + s.tiles + kItemCost - 1) / group_share;
      lds.shared[tile0 == 0] = typename F::Shared{b, item, wg0, last - wg0 + 1, s};
    }
    __syncthreads();  // w and sum are free again
  }

  // At most two items of a workgroup are shared, at its start and at its end.
  __builtin_amdgcn_s_waitcnt(0);  // this wave's stores to the workspace
  __syncthreads();
  if (wave < 2) {
    const typename F::Shared x = lds.shared[wave];
    bool all = false;
    if (x.pieces > 0) {
      if (lane == 0) set_flag(a.flags + 2 * wg + wave, a.gen);
      __builtin_amdgcn_s_waitcnt(0);
      all = flags_set(a.flags, a.gen, x.wg0, x.pieces, lane);
    }
    if (lane == 0) lds.last[wave] = all;
  }
  __syncthreads();
  for (int k = 0; k < 2; ++k) {
    if (!lds.last[k]) continue;
    const typename F::Shared x = lds.shared[k];
    join_pieces<D, NT>(a, lds, x, tid);
    for (int p = tid; p < x.pieces; p += F::kThreads)
      set_flag(a.flags + 2 * (x.wg0 + p) + (p == 0), 0);
  }
}

// ---------------------------------------------------------------------------
// Many rows (prompts): bound by the matrix products.
//
// A workgroup of eight waves takes 256 rows of one sequence and key/value head
// over the tiles of keys, 32 rows a wave, v_mfma_f32_32x32x16_f16. It turns a
// tile's codes into fp16 in LDS once for all its rows (a thread 16 bytes of
// keys and of values), a tile ahead of the products. Rows of a product's right
// operand are a wave's lanes, so a row's maximum and sum need one exchange of
// the wave's halves. Values lie in LDS in the order in which lanes hold P's
// tokens.
//
// A page's value scale goes into P relative to a power of two, `unit`, which is
// what the sums are counted in. A tile's largest scale is kScaleLow to kScaleHigh
// units, so that P, 2^kLazy high, fills fp16 upwards and a weight is kept down to
// 2^-30 of the row's largest (2^-33 where the first tile's scale is the usual one).
// The unit moves no further than a tile asks for: scales within 2^5 of each other
// settle on one, and the sums are rescaled only when it moves. A row whose sums
// are 2^126 under a later tile's scale loses them, where that tile weighs nothing.
//
// The work is (sequence, head, row tile, tile of keys), with the tiles past a
// row tile's last visible key left out; the workgroups take equal shares, and
// pieces of an item that two or more share meet as those of attend_few do.
//
// A prompt of 4096 tokens, 64 query and 8 key/value heads, fp16: 275 GFLOP in
// 417 us, 660 TFLOP/s, with the products for P's second part on top (half as
// many again: 990 of the 1200 that a large library product has); 501 tokens on
// each of three long contexts, bf16: 281 GFLOP in 405 us. Per tile the vector
// instructions of two waves (scores to weights about 200, codes 50 each) take
// about as long as their products, with the matrix units busy 52% and 59% of the
// time at a clock that falls to 1.8 and 1.7 GHz. With P in one part, operand
// loads next to their products, in the compiler's order, cost a quarter, and the
// second took 383 us instead of 328 without the halves' shift.
// ---------------------------------------------------------------------------
constexpr int kManyRows = 256;
constexpr int kManyThreads = 512;
constexpr float kScaleLow = 0x1p5f, kScaleFirst = 0x1p8f, kScaleHigh = 0x1p11f;
constexpr int kManyItemCost = 6;  // an item's start and end against a tile, measured

typedef float f16_t __attribute__((ext_vector_type(16)));

template <int D>
struct Many {
  static constexpr int kPiece = kManyRows * (D + 2);      // floats in the workspace
  static constexpr int kBlock = D * 16 + 16;              // bytes of eight tokens' values, spread over the banks
  struct Lds {
    // Three tiles in turn: one is multiplied by P while the next is multiplied
    // by Q and the one after is written, with the workgroup's halves apart.
    alignas(16) char k[3][D / 8][kTile][16];  // eight elements of a key
    alignas(16) char v[3][8 * kBlock];        // [(16 tokens, half)][element][8 tokens]
    // Scales of a tile's 16-token groups, keys and values; -1: no page. Lanes
    // that bring none write to the second one.
    float scales[2][3][4], none[24];
    int last;
  };
};

// Whether a sequence's row tiles see different numbers of keys.
__device__ __forceinline__ bool slanted(const AttendArgs& a, const Seq& s) {
  return a.causal && s.n <= s.len && s.row_tiles > 1;
}

// Tiles of keys that row tile rt sees, j = rt + 1: its last row's token sees
// len - n + ceil(256 j / group) keys, or all, which is a number of tiles of
//   ceil(((len - n) group + 256 j) / (64 group)) = ceil((c + 4 j) / group),
// c = ceil((len - n) group / 64).
__device__ __forceinline__ unsigned keys_before(const AttendArgs& a, const Seq& s) {
  return ((unsigned)(s.len - s.n) * (unsigned)a.group + kTile - 1) / kTile;
}
__device__ __forceinline__ int tiles_seen(const AttendArgs& a, const Seq& s, int rt) {
  if (!slanted(a, s) || rt >= s.row_tiles - 1) return s.tiles;
  const unsigned G = a.group;
  return (keys_before(a, s) + (kManyRows / kTile) * (rt + 1) + G - 1) / G;
}

// The work of one head of a sequence: the sum of its row tiles'. Every `period`
// row tiles a row tile sees `rise` tiles of keys more, so those that stand
// `period` apart are an arithmetic series.
__device__ __forceinline__ int head_cost(const AttendArgs& a, const Seq& s) {
  if (!slanted(a, s)) return s.row_tiles * (s.tiles + kManyItemCost);
  static_assert(kManyRows / kTile == 4, "period and rise");
  const unsigned G = a.group, common = G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1;
  const unsigned period = G / common, rise = 4 / common, last = s.row_tiles - 1;
  const unsigned c = keys_before(a, s);
  unsigned sum = s.row_tiles * kManyItemCost + s.tiles;
  for (unsigned j = 1; j <= min(period, last); ++j) {
    const unsigned terms = (last - j) / period + 1;
    sum += terms * ((c + 4 * j + G - 1) / G) + rise * (terms * (terms - 1) / 2);
  }
  return (int)sum;
}

// A workgroup barrier for what is in LDS alone: __syncthreads() also waits for
// every load from memory under way, the next tiles' codes among them.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

constexpr int kAhead = 4;

// Uniform loads through it are scalar loads, stores elsewhere or not: what is
// read so (tables, scales) no kernel here writes while it is read.
template <typename T>
__device__ __forceinline__ const __attribute__((address_space(4))) T* as_constant(const T* p) {
  return (const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

// P goes in as two fp16 parts here too, which doubles the second product. With
// one, results were up to 4.4 (bf16) and 1.6 (fp16) times their own rounding
// away from 64 bits where few keys carry a row; with two they are not. The
// 501-token pieces took 303 us with one, 391 with two.
template <int D>
__global__ __launch_bounds__(kManyThreads) void attend_many(AttendArgs a) {
  using M = Many<D>;
  constexpr int kK = D / 16, kDt = D / 32;
  __shared__ typename M::Lds lds;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, hh = lane >> 5;
  const int wg = blockIdx.x;
  const int shift = a.c.page_shift, P = 1 << shift;

  // This workgroup's share, found by every wave for itself as in attend_few.
  const Owned owned = owned_tokens(a);
  const int each = (a.requests + 63) / 64;
  int b = lane * each;
  Seq s{};
  int work = 0;
  bool ordered = true;
  for (int k = 0; k < each && b + k < a.requests; ++k) {
    s = sequence(a, b + k, kManyRows, true);
    ordered &= s.n >= 0;
    work += a.c.heads * head_cost(a, s);
  }
  int upto = wave_scan(work);
  const int total = __builtin_amdgcn_readlane(upto, 63);
  const int share = max((int)(((unsigned)total + kWorkgroups - 1) / kWorkgroups), 1);
  const int begin = wg * share, end = min(begin + share, total);
  ordered = __all(ordered);
  if (a.clear) clear_rows<D>(a, ordered ? owned : Owned{0, 0}, tid, kManyThreads);
  if (!ordered || begin >= end) return;
  int at = __builtin_ctzll(__ballot(begin < upto));
  int base = __builtin_amdgcn_readlane(upto - work, at);
  b = at * each;
  if (each > 1) {
    int first = b;
    for (;; first += 64) {
      const bool real = first + lane < min(b + each, a.requests);
      s = sequence(a, real ? first + lane : 0, kManyRows, true);
      work = real ? a.c.heads * head_cost(a, s) : 0;
      upto = wave_scan(work);
      if (begin < base + __builtin_amdgcn_readlane(upto, 63)) break;
      base += __builtin_amdgcn_readlane(upto, 63);
    }
    at = __builtin_ctzll(__ballot(begin < base + upto));
    base += __builtin_amdgcn_readlane(upto - work, at);
    b = first + at;
  }
  s = lane_seq(s, at);

  // The item that the share starts in, and where: head, row tile.
  int per_head = __builtin_amdgcn_readfirstlane(head_cost(a, s));
  int h = (begin - base) / per_head, rt = 0;
  base += h * per_head;
  for (;; rt += 64) {
    const int u = rt + lane < s.row_tiles ? tiles_seen(a, s, rt + lane) + kManyItemCost : 0;
    const int scan = wave_scan(u);
    const int all = __builtin_amdgcn_readlane(scan, 63);
    if (begin < base + all) {
      const int i = __builtin_ctzll(__ballot(begin < base + scan));
      base += __builtin_amdgcn_readlane(scan - u, i);
      rt += i;
      break;
    }
    base += all;
  }

  for (int cur = begin; cur < end;) {
    const int tiles = tiles_seen(a, s, rt);
    const int units = tiles + kManyItemCost;
    const int from = cur - base, stop = min(units, from + (end - cur));
    const int tile0 = max(from - kManyItemCost, 0), tile1 = stop - kManyItemCost;
    const int start = base;
    cur += stop - from;
    if (tile0 < tile1) {
      const int row0 = rt * kManyRows + wave * 32;
      const int rows = s.n * a.group;
      const int32_t* table = a.tables + (long long)b * a.width;

      // A wave loads 16 tokens of a tile, group `wave % 4`: half of their keys'
      // pieces and of their values' elements, or with 64 elements all of the
      // one or the other. Its page is uniform, so addresses cost no vector
      // instruction. Loads run for every tile, past the last one too (of the
      // last key's page): under a condition they would be waited for where the
      // ways meet again.
      const bool loads_k = D == 128 || wave < 4;
      const int own = wave & 3, half = wave >> 2;
      const int kc = (D == 128 ? 4 * half : 0) + (lane >> 4), vd = (D == 128 ? 64 * half : 0) + lane;
      const uint32_t page_bytes = (uint32_t)a.c.heads * D * P;  // under 2^31
      const uint32_t head_bytes = (uint32_t)h * D * P;
      const uint32_t kat = (kc * P + (lane & 15)) * 16, vat = vd * P;
      uint4 kraw, vraw;  // with 64 elements kraw alone, of keys or values
      float ksraw, vsraw;
      int page, page_of_raw;
      const int last = s.len - 1;
      auto load_page = [&](int tile) {
        page = as_constant(table)[min(tile * kTile + 16 * own, last) >> shift];
      };
      auto load_scales = [&] {  // of `page`
        page_of_raw = page;
        const uint32_t at = page >= 0 && page < a.c.pages ? page : 0;
        ksraw = as_constant(a.c.ks)[(unsigned long long)at * (uint32_t)a.c.heads + h];
        vsraw = as_constant(a.c.vs)[(unsigned long long)at * (uint32_t)a.c.heads + h];
      };
      auto load_codes = [&](int tile, int step) {
        const uint32_t in = (tile * kTile + 16 * own) & (P - 1);
        const unsigned long long at =
            (unsigned long long)(uint32_t)(page >= 0 && page < a.c.pages ? page : 0) * page_bytes + head_bytes;
        if (step == 0) {
          if constexpr (D == 128)
            kraw = *reinterpret_cast<const uint4*>(a.c.k + (at + in * 16) + kat);
          else
            kraw = *reinterpret_cast<const uint4*>((loads_k ? a.c.k + (at + in * 16) : a.c.v + (at + in)) +
                                                   (loads_k ? kat : vat));
        } else if (D == 128) {
          vraw = *reinterpret_cast<const uint4*>(a.c.v + (at + in) + vat);
        }
      };
      char* const kto = lds.k[0][2 * kc][16 * own + (lane & 15)];
      char* const vto = lds.v[0] + 2 * own * M::kBlock + vd * 16;
      float* const sto = wave < 4 && lane == 0 ? &lds.scales[0][0][own] : lds.none;
      auto store_codes = [&](int buf, int step) {
        const uint4 v = D == 128 ? vraw : kraw;
        char* k = kto + buf * (int)sizeof(lds.k[0]);
        char* w = vto + buf * (int)sizeof(lds.v[0]);
        if (step == 0 && loads_k)
          *reinterpret_cast<h8_t*>(k) = codes_to_f16(kraw.x, kraw.y);
        else if (step == 1 && loads_k)
          *reinterpret_cast<h8_t*>(k + kTile * 16) = codes_to_f16(kraw.z, kraw.w);
        else if (step == 2 && (D == 128 || !loads_k))
          *reinterpret_cast<h8_t*>(w) = codes_to_f16(v.x, v.z);
        else if (step == 3 && (D == 128 || !loads_k))
          *reinterpret_cast<h8_t*>(w + M::kBlock) = codes_to_f16(v.y, v.w);
        else if (step == 4) {
          const bool there = page_of_raw >= 0 && page_of_raw < a.c.pages;
          sto[buf * 4] = there ? ksraw : -1.0f;
          sto[buf * 4 + 12] = there ? vsraw : -1.0f;
        }
      };
      // Steps to go between products: tile's successor out of the registers into
      // `buf`, the one after it into them.
      auto move_codes = [&](int tile, int buf, int step) {
        if (step < 5) store_codes(buf, step);
        else if (step < 7) load_codes(tile + 2, step - 5);
      };

      const bool keys = s.len > 0;  // a sequence without keys has no page to read
      if (keys) load_page(tile0);
      // The queries of this wave's rows.
      h8_t qf[kK];
      float qs;
      int limit, least;
      {
        const int r = row0 + n32;
        const bool real = r < rows;
        const int i = real ? r / a.group : 0;
        limit = !real ? 0 : a.causal ? s.len - s.n + i + 1 : s.len;
        const uint16_t* q = a.q + (long long)(s.q0 + i) * a.qt +
                            ((long long)h * a.group + (real ? r - i * a.group : 0)) * a.qh + 8 * hh;
        uint4 raw[kK];
#pragma unroll
        for (int k = 0; k < kK; ++k) raw[k] = *reinterpret_cast<const uint4*>(q + 16 * k);
        if (keys) {
          load_codes(tile0, 0);
          load_codes(tile0, 1);
          load_scales();
          load_page(tile0 + 1);
        }
        float amax = 0;
#pragma unroll
        for (int k = 0; k < kK; ++k) {
          float x[8];
          q_floats(raw[k], a.bf16, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[e]));
        }
        const int ex = row_exponent(max_halves(amax));
        const float f = a.scale_log2 < 0 ? -pow2i(ex) : pow2i(ex);
#pragma unroll
        for (int k = 0; k < kK; ++k) {
          float x[8];
          q_floats(raw[k], a.bf16, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) qf[k][e] = (_Float16)(x[e] * f);
        }
        qs = fabsf(a.scale_log2) * pow2i(-ex);
        least = -__builtin_amdgcn_readfirstlane(max_half_wave(real ? -limit : -INT32_MAX));
      }

      // Sums, and what the fast way through a tile compares with: `bound` the
      // score that moves a row's maximum, `sub` what is taken off a score.
      f16_t o[kDt], st[2];
      h8_t pf[4], pl[4];  // pl: what rounding to pf leaves
      float m = kNegInf, bound = kNegInf, sub = 0, l = 0;
      float unit = 0, per_unit = 0;
#pragma unroll
      for (int d = 0; d < kDt; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] = 0;

      // Products of the values of `vbuf` with P, then of the keys of `kbuf`
      // with Q: operands come from LDS kAhead products ahead of their own.
      auto products = [&](auto with_values, auto with_keys, int vbuf, int kbuf, auto between) {
        constexpr int kV = decltype(with_values)::value ? 4 * kDt : 0;
        constexpr int kN = kV + (decltype(with_keys)::value ? 2 * kK : 0);
        const char* v = lds.v[vbuf] + hh * M::kBlock + n32 * 16;
        const char* k = &lds.k[kbuf][hh][n32][0];
        h8_t ring[kAhead];
        auto load = [&](int i) {
          const char* from = i < kV ? v + 2 * (i / kDt) * M::kBlock + 32 * (i % kDt) * 16
                                    : k + (2 * ((i - kV) / 2) * kTile + 32 * ((i - kV) % 2)) * 16;
          ring[i % kAhead] = *reinterpret_cast<const h8_t*>(from);
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i) load(i);
        if constexpr (decltype(with_keys)::value) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) st[t][e] = 0;
        }
        auto step = [&](int i) {  // the operand after the ring's in the place of product i's
          if (i + kAhead < kN) load(i + kAhead);
          between(i - kV);
          // The compiler puts loads right before their products.
          __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (int q = 0; q < kV / kDt; ++q) {
#pragma unroll
          for (int d = 0; d < kDt; ++d) {
            const h8_t x = ring[(q * kDt + d) % kAhead];
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, pf[q], o[d], 0, 0, 0);
          }
#pragma unroll
          for (int d = 0; d < kDt; ++d) {  // after the others, whose sums they wait for
            const h8_t x = ring[(q * kDt + d) % kAhead];
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, pl[q], o[d], 0, 0, 0);
            step(q * kDt + d);
          }
        }
#pragma unroll
        for (int i = kV; i < kN; ++i) {
          const int k = i - kV;
          st[k % 2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[i % kAhead], qf[k / 2], st[k % 2], 0, 0, 0);
          step(i);
        }
      };

      // P of a tile from its scores.
      auto weights = [&](int tile, int buf, auto meanwhile) {
        const int key0 = tile * kTile;
        const f4_t cs = *reinterpret_cast<const f4_t*>(lds.scales[0][buf]);
        const f4_t vs = *reinterpret_cast<const f4_t*>(lds.scales[1][buf]);
        meanwhile();
        float ck[4], rel[4];
        const float top = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
        const float bottom = fminf(fminf(cs[0], cs[1]), fminf(cs[2], cs[3]));  // -1: a page is missing
#pragma unroll
        for (int q = 0; q < 4; ++q) ck[q] = cs[q] * qs;
        bool fix = false;
        // Places of this lane's tokens in the tile: 16 q + 8 (e / 4) + 4 hh + e % 4.
        int left = limit - key0 - 4 * hh;
        auto seen = [&](int q, int e) { return cs[q] != -1.0f && 16 * q + 8 * (e >> 2) + (e & 3) < left; };
        if (__builtin_expect(key0 + kTile > least || bottom < 0, 0)) {
          asm volatile("" : "+v"(left));  // keeps the comparisons in here
#pragma unroll
          for (int q = 0; q < 4; ++q) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float x = st[q >> 1][8 * (q & 1) + e];
              st[q >> 1][8 * (q & 1) + e] = seen(q, e) ? x * ck[q] : kNegInf;
            }
            ck[q] = 1.0f;
          }
          fix = !(fabsf(vs[0]) + fabsf(vs[1]) + fabsf(vs[2]) + fabsf(vs[3]) < __builtin_huge_valf());
        }
        float tm = kNegInf;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float g = st[q >> 1][8 * (q & 1)];
#pragma unroll
          for (int e = 1; e < 8; ++e) g = fmaxf(g, st[q >> 1][8 * (q & 1) + e]);
          tm = fmaxf(tm, g * ck[q]);
        }
        float alpha = 1.0f;  // what the sums so far are multiplied by
        bool move = false;
        if (__builtin_expect(__any(tm > bound), 0)) {
          const float mn = fmaxf(m, max_halves(tm));
          alpha = mn == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
          l *= alpha;
          m = mn;
          bound = mn + kLazy;
          sub = mn == kNegInf ? 0.0f : -mn;
          move = true;
        }
        auto fits = [&](float scale) { return scale >= unit * kScaleLow && scale <= unit * kScaleHigh; };
        if (__builtin_expect(!fits(top), 0)) {  // the unit moves, or there is none
          float t = 0;
#pragma unroll
          for (int q = 0; q < 4; ++q) t = fmaxf(t, vs[q] < __builtin_huge_valf() ? vs[q] : 0.0f);
          if (t > 0 && !fits(t)) {
            const float was = unit;
            const float units = was == 0 ? kScaleFirst : t > was * kScaleHigh ? kScaleHigh / 2 : kScaleLow;
            unit = fmaxf(floor_pow2(t) / units, 0x1p-126f);
            float most = 1.0f;
            if (unit < was) {  // not so far that the sums overflow: what such a tile adds is nothing to them
              most = 0;
#pragma unroll
              for (int d = 0; d < kDt; ++d)
#pragma unroll
                for (int v = 0; v < 16; ++v) most = fmaxf(most, fabsf(o[d][v]));
              most = max_halves(most) * alpha;
              const float least = most > 0 ? fmaxf(floor_pow2(was * (most * 0x1p-99f)), was * 0x1p-126f) : 0.0f;
              unit = fminf(fmaxf(unit, least), was);
            }
            if (most > 0) alpha *= was / unit;  // else there is nothing to multiply
            move |= unit != was;
            per_unit = 1.0f / unit;
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) rel[q] = vs[q] * per_unit;
        if (__builtin_expect(move, 0)) {
#pragma unroll
          for (int d = 0; d < kDt; ++d) o[d] *= alpha;
        }
        float sum = 0;  // the tile's by itself, as in attend_few
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            float w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float p = __builtin_amdgcn_exp2f(fmaf(st[q >> 1][8 * (q & 1) + e + i], ck[q], sub));
              sum += p;
              w[i] = p * rel[q];
            }
            const h2_t f = first_parts(w[0], w[1]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              pf[q][e + i] = f[i];
              pl[q][e + i] = (_Float16)fmaf((float)f[i], -1.0f, w[i]);
            }
          }
        l += sum;
        if (__builtin_expect(fix, 0)) {  // a key that is not seen has weight 0 on a page of any scale
          asm volatile("" : "+v"(left));
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              pf[q][e] = seen(q, e) ? pf[q][e] : (_Float16)0.0f;
              pl[q][e] = seen(q, e) ? pl[q][e] : (_Float16)0.0f;
            }
        }
      };

      if (keys) {
        constexpr std::true_type kYes;
        constexpr std::false_type kNo;
        // Tile tile0 + i is in buffer i % 3: the one before this one, this one
        // and the next.
        int prev = 2, buf = 0, next = 1;
        lds_barrier();  // the buffers may be in use by the item before
#pragma unroll
        for (int i = 0; i < 7; ++i) move_codes(tile0 - 1, 0, i);
        load_scales();
        load_page(tile0 + 2);
        lds_barrier();
        // The workgroup's two halves, a wave of each on every SIMD, run half a
        // tile apart: while one multiplies, the other works out its weights.
        // Both pass the same barriers. Who multiplies issues first: its few
        // vector instructions would hold its products up (340 against 322 us, P in
        // one part).
        if (wave >= 4) lds_barrier();
        auto nothing = [](int) {};
        for (int tile = tile0; tile < tile1; ++tile) {
          __builtin_amdgcn_s_setprio(1);
          if (tile > tile0) products(kYes, kNo, prev, buf, nothing);
          products(kNo, kYes, prev, buf, [&](int i) { move_codes(tile, next, i); });
          __builtin_amdgcn_s_setprio(0);
          lds_barrier();
          weights(tile, buf, [&] {
            load_scales();  // of the tile that is in the registers next
            load_page(tile + 3);
          });
          lds_barrier();
          const int free = prev;
          prev = buf, buf = next, next = free;
        }
        products(kYes, kNo, prev, buf, nothing);
        if (wave < 4) lds_barrier();
      }

      l = sum_halves(l);
#pragma unroll
      for (int d = 0; d < kDt; ++d) o[d] *= unit;  // 0 where no page had a scale above 0
      const int r = row0 + n32;
      bool write = true;
      if (tile0 > 0 || tile1 < tiles) {
        // A piece, as the registers lie: [wave][pair of registers][lane].
        auto place = [&](int k, int pair) {
          return a.partials + (2LL * k) * M::kPiece + ((wave * (8 * kDt) + pair) * 64 + lane) * 2;
        };
        auto stats = [&](int k) {
          return a.partials + (2LL * k) * M::kPiece + kManyRows * D + (wave * 32 + n32) * 2;
        };
        const int own = tile0 == 0 ? 1 : 0;
        float* slot = place(wg, 0) + own * M::kPiece;
#pragma unroll
        for (int d = 0; d < kDt; ++d)
#pragma unroll
          for (int v = 0; v < 8; ++v) store_agent2(slot + (8 * d + v) * 128, o[d][2 * v], o[d][2 * v + 1]);
        if (hh == 0) store_agent2(stats(wg) + own * M::kPiece, m, l);
        const int wg0 = tile0 == 0 ? wg : (start + kManyItemCost) / share;
        const int pieces = (start + units - 1) / share - wg0 + 1;
        __builtin_amdgcn_s_waitcnt(0);  // this wave's stores to the workspace
        __syncthreads();
        if (wave == 0) {
          if (lane == 0) set_flag(a.flags + 2 * wg + own, a.gen);
          __builtin_amdgcn_s_waitcnt(0);
          const bool all = flags_set(a.flags, a.gen, wg0, pieces, lane);
          if (lane == 0) lds.last = all;
        }
        __syncthreads();
        write = lds.last;
        if (write) {
          m = kNegInf, l = 0;
#pragma unroll
          for (int d = 0; d < kDt; ++d)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[d][v] = 0;
          for (int k = 0; k < pieces; ++k) {
            const long long off = k == 0 ? M::kPiece : 0;
            const float2 ml = load_agent2(stats(wg0 + k) + off);
            const float* p = place(wg0 + k, 0) + off;
            float2 x[kDt][8];
#pragma unroll
            for (int d = 0; d < kDt; ++d)
#pragma unroll
              for (int v = 0; v < 8; ++v) x[d][v] = load_agent2(p + (8 * d + v) * 128);
            const float mn = fmaxf(m, ml.x);
            const float fo = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
            const float fn = ml.x == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mn);
            l = l * fo + ml.y * fn;  // a NaN stays
            m = mn;
#pragma unroll
            for (int d = 0; d < kDt; ++d)
#pragma unroll
              for (int v = 0; v < 8; ++v) {
                o[d][2 * v] = fmaf(o[d][2 * v], fo, x[d][v].x * fn);
                o[d][2 * v + 1] = fmaf(o[d][2 * v + 1], fo, x[d][v].y * fn);
              }
          }
          for (int k = tid; k < pieces; k += kManyThreads)
            set_flag(a.flags + 2 * (wg0 + k) + (k == 0), 0);
        }
      }
      if (write && r < rows) {
        const float inv = inverse_sum(l);
        uint16_t* out = out_row<D>(a, s, h, r) + 4 * hh;
#pragma unroll
        for (int d = 0; d < kDt; ++d)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const float x[4] = {o[d][4 * v] * inv, o[d][4 * v + 1] * inv, o[d][4 * v + 2] * inv,
                                o[d][4 * v + 3] * inv};
            store_half4(a, out + 32 * d + 8 * v, x);
          }
      }
    }
    // On to the next item.
    base += units;
    if (++rt == s.row_tiles && cur < end) {
      rt = 0;
      if (++h == a.c.heads) {
        h = 0;
        do {
          s = sequence(a, ++b, kManyRows, true);
        } while (s.row_tiles == 0);
      }
    }
  }
}

}  // namespace dk

namespace {

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Which kernels a call runs and what they need. Sequences of at most 128 rows
// (queries times the group) are attend_few's, larger ones attend_many's. fp16,
// head size 128, 8 heads, us of the two kernels at 64, 128 and 256 rows:
//   64 sequences of 4000 keys   181 / 348   356 / 364   709 / 394
//    8 sequences of 4000 keys    38 / 64     55 / 68     98 / 74
//    1 sequence of 30000 keys    48 / 114    82 / 116   156 / 121
//   64 sequences of 500 keys     34 / 57     62 / 66    117 / 77
// bf16 differs by 4% at most.
// A call that by its sizes can have one kind alone runs one kernel, which then
// takes every size. attend_few takes 32 rows at a time where sequences have
// more than 16 and there are 32 sequences and heads to share the card (64 x 8,
// 4000 keys, 64 rows: 181 us against 199 for 16 at a time); with fewer, pieces
// of 16 rows are joined sooner (1 x 8, 30000 keys, 32 rows: 34 against 66).
constexpr int kFewRows = 128;

struct Dispatch {
  bool few, many;
  int nt;
};
Dispatch dispatch(int num_tokens, int requests, int heads, int group, int max_query_len) {
  Dispatch d;
  const long long rows = (long long)std::min(max_query_len, num_tokens) * group;
  d.many = rows > kFewRows;
  d.few = !d.many || requests > 1;
  d.nt = rows <= 16 || (long long)heads * requests < 32 ? 1 : 2;
  return d;
}

// The most that a kernel of the call may have to count, in 31 bits: heads, row
// tiles and tiles of keys with an item's own cost, all sequences as long as the
// tables are wide. Each kernel's sequences are those of its number of rows.
double most_work(const Dispatch& d, int num_tokens, int requests, int heads, int group, long long keys) {
  const double rows = (double)num_tokens * group;
  const int rows_a_tile = 16 * d.nt;
  double tiles = 0;
  if (d.few) tiles = rows / rows_a_tile + requests;
  if (d.few && d.many) tiles = std::min(tiles, (double)requests * (kFewRows / rows_a_tile));
  if (d.many) tiles = std::max(tiles, rows / dk::kManyRows + std::min((double)requests, rows / (d.few ? kFewRows : 1) + 1));
  return heads * tiles * ((double)keys / dk::kTile + 8);
}

// The number of a call, which never comes again in a process: what its pieces'
// flags hold when they are set.
unsigned long long next_call() {
  static std::atomic<unsigned long long> calls{0x9D8E6B1F37A95C41ull};  // no count that memory may hold
  return calls.fetch_add(1, std::memory_order_relaxed);
}

size_t flags_bytes() { return (size_t)dk::kWorkgroups * 2 * sizeof(unsigned long long); }

// Flags and pieces of each kernel that runs.
size_t workspace_bytes_of(const Dispatch& d, int head_size) {
  size_t rows = 0;
  if (d.few) rows += 16 * d.nt;
  if (d.many) rows += dk::kManyRows;
  return flags_bytes() * (d.few + d.many) +
         (size_t)dk::kWorkgroups * 2 * rows * (head_size + 2) * sizeof(float);
}

}  // namespace

extern "C" size_t dk_kv_attend_workspace_bytes(int num_tokens, int requests, int q_heads, int heads,
                                               int head_size, int table_width, int page_size,
                                               int max_query_len) {
  (void)table_width;
  (void)page_size;
  if (num_tokens <= 0 || requests <= 0 || heads <= 0 || q_heads <= 0 || head_size <= 0) return 0;
  return workspace_bytes_of(dispatch(num_tokens, requests, heads, q_heads / heads, max_query_len),
                            head_size);
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
  if (num_tokens == 0) return DK_OK;
  const int group = q_heads / view.heads;
  const Dispatch d = dispatch(num_tokens, requests, view.heads, group, max_query_len);
  const size_t need = requests > 0 ? workspace_bytes_of(d, cache->head_size) : 0;
  if (!q || !out || (requests > 0 && (!seq_lens || (!tables && table_width > 0))) || (!workspace_ptr && need > 0))
    return dk::set_error(DK_ERR_INVALID_ARGUMENT,
                         "q, out, tables, seq_lens and the workspace must not be NULL");
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(workspace_ptr, 16))
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "q, out and the workspace must be 16-byte aligned");
  if (q_token_stride % 8 || q_head_stride % 8)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "the strides of q must be multiples of 8");
  if (most_work(d, num_tokens, requests, view.heads, group, (long long)table_width << view.page_shift) > 1 << 30)
    return dk::set_error(DK_ERR_UNSUPPORTED, "heads * queries * keys too large");
  if (((double)table_width * cache->page_size + num_tokens + dk::kTile) * group > 1 << 30)
    return dk::set_error(DK_ERR_UNSUPPORTED, "keys * q_heads / heads too large");
  if (workspace_bytes < need)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "the workspace has %zu of %zu bytes", workspace_bytes, need);
  dk::AttendArgs a{};
  a.c = view;
  a.q = static_cast<const uint16_t*>(q);
  a.qt = q_token_stride;
  a.qh = q_head_stride;
  a.out = static_cast<uint16_t*>(out);
  a.tables = tables;
  a.lens = seq_lens;
  a.offsets = query_offsets;
  a.gen = next_call();
  a.scale_log2 = scale * 1.44269504088896340736f;
  a.width = cache->pages > 0 ? table_width : 0;  // no pages, no keys
  a.tokens = num_tokens;
  a.requests = requests;
  a.group = group;
  a.bf16 = dtype == DK_KV_BF16;
  a.causal = causal != 0;
  char* ws = static_cast<char*>(workspace_ptr);
  auto launch = [&](auto kernel, int threads, int rows) {
    a.flags = reinterpret_cast<unsigned long long*>(ws);
    a.partials = reinterpret_cast<float*>(ws + flags_bytes());
    hipLaunchKernelGGL(kernel, dim3(dk::kWorkgroups), dim3(threads), 0, stream, a);
    ws += flags_bytes() + (size_t)dk::kWorkgroups * 2 * rows * (cache->head_size + 2) * sizeof(float);
  };
  if (d.many) {
    a.few_rows = d.few ? kFewRows : 0;
    a.clear = !d.few;
    if (cache->head_size == 64) launch(dk::attend_many<64>, dk::kManyThreads, dk::kManyRows);
    else launch(dk::attend_many<128>, dk::kManyThreads, dk::kManyRows);
  }
  if (d.few) {
    a.few_rows = d.many ? kFewRows : INT32_MAX;
    a.clear = 1;
    if (cache->head_size == 64) {
      if (d.nt == 1) launch(dk::attend_few<64, 1>, dk::Few<64, 1>::kThreads, 16);
      else launch(dk::attend_few<64, 2>, dk::Few<64, 2>::kThreads, 32);
    } else {
      if (d.nt == 1) launch(dk::attend_few<128, 1>, dk::Few<128, 1>::kThreads, 16);
      else launch(dk::attend_few<128, 2>, dk::Few<128, 2>::kThreads, 32);
    }
  }
  return dk::check_launch("attend launch");
}
