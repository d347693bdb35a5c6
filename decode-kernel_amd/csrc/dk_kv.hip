// The paged 8-bit key/value cache: planning a step, appending and reading.
// Layouts in dk_kv.hpp, contracts in include/decode_kernel/dk_kv.h.
#include <hip/hip_runtime.h>

#include "dk_host.hpp"
#include "dk_kv.hpp"

namespace dk {

// ---------------------------------------------------------------------------
// Plan: from request lengths to offsets, pages and slots, in one launch.
//
// Every workgroup scans all requests into LDS (tokens, then pages, since the
// pages follow from the tokens that fit) and then serves its own tokens, one
// a thread: the request by bisection, the page from the table or, for a page
// that the step opens, from the free list at the rank that the scan gives. A
// token at a page's first place writes the table's entry, so no token waits
// for another. A few kilobytes, so latency alone: 3.9 us for 256 requests with
// a token each, 4.6 for 37 with 30011.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 256;

// Exclusive scan of one value a thread; the total in *total.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* wave_sums, T* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T inc = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const T o = __shfl_up(inc, d);
    if (lane >= d) inc += o;
  }
  __syncthreads();  // wave_sums may be in use from the scan before
  if (lane == 63) wave_sums[wave] = inc;
  __syncthreads();
  T before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) before += wave_sums[w];
    sum += wave_sums[w];
  }
  *total = sum;
  return before + inc - v;
}

struct PlanArgs {
  int32_t* tables;
  const int32_t* held;
  const int32_t* added;
  const int32_t* free_pages;
  const int32_t* free_count;
  int64_t* slots;
  int32_t* positions;
  int32_t* query_offsets;
  int32_t* seq_lens;
  int32_t* free_count_out;
  int width, requests, capacity, page_shift, tokens;
};

__device__ __forceinline__ int pages_of(long long tokens, int shift) {
  return (int)((tokens + (1 << shift) - 1) >> shift);
}

__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a) {
  __shared__ int offs[DK_KV_MAX_REQUESTS + 1];   // where request b's tokens start
  __shared__ int ranks[DK_KV_MAX_REQUESTS];      // pages opened before request b
  __shared__ long long token_sums[kPlanThreads / 64];
  __shared__ int page_sums[kPlanThreads / 64];
  const int tid = threadIdx.x;
  const int each = (a.requests + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * each, a.requests), b1 = min(b0 + each, a.requests);
  const long long room = (long long)a.width << a.page_shift;

  long long mine = 0, all;
  for (int b = b0; b < b1; ++b) mine += max(a.added[b], 0);
  long long at = block_scan(mine, token_sums, &all);
  for (int b = b0; b < b1; ++b) {
    offs[b] = (int)min(at, (long long)a.tokens);
    at += max(a.added[b], 0);
  }
  if (tid == 0) offs[a.requests] = (int)min(all, (long long)a.tokens);
  __syncthreads();

  int pages = 0, opened;
  for (int b = b0; b < b1; ++b) {
    const long long had = max(a.held[b], 0);
    const long long len = min(had + offs[b + 1] - offs[b], room);
    ranks[b] = pages;
    pages += max(pages_of(len, a.page_shift) - pages_of(had, a.page_shift), 0);
    if (blockIdx.x == 0) {
      a.seq_lens[b] = (int)len;
      a.query_offsets[b] = offs[b];
    }
  }
  const int first = block_scan(pages, page_sums, &opened);
  for (int b = b0; b < b1; ++b) ranks[b] += first;
  if (blockIdx.x == 0 && tid == 0) {
    a.query_offsets[a.requests] = offs[a.requests];
    *a.free_count_out = *a.free_count - opened;
  }
  __syncthreads();

  const int t = blockIdx.x * kPlanThreads + tid;
  if (t >= a.tokens) return;
  if (t >= offs[a.requests]) {
    a.slots[t] = -1;
    a.positions[t] = -1;
    return;
  }
  int lo = 0, hi = a.requests - 1;  // the first request that ends after t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (offs[mid + 1] > t) hi = mid;
    else lo = mid + 1;
  }
  const long long had = max(a.held[lo], 0);
  const long long pos = had + t - offs[lo];
  const long long col = pos >> a.page_shift;
  const int in_page = (int)(pos & ((1 << a.page_shift) - 1));
  long long slot = -1;
  if (col < a.width) {
    int32_t* entry = a.tables + (long long)lo * a.width + col;
    const int fresh = (int)col - pages_of(had, a.page_shift);
    int page;
    if (fresh >= 0) {
      const int i = min(*a.free_count, a.capacity) - 1 - (ranks[lo] + fresh);
      page = i >= 0 ? a.free_pages[i] : -1;
      if (in_page == 0) *entry = page;
    } else {
      page = *entry;
    }
    if (page >= 0) slot = ((long long)page << a.page_shift) + in_page;
  }
  a.slots[t] = slot;
  a.positions[t] = (int)min(pos, (long long)INT32_MAX);
}

// ---------------------------------------------------------------------------
// Append: bound by bytes for prompts, by latency for decode.
//
// A run is the step's tokens of one page; for one head, keys or values. Its
// tokens fall into groups of 16 places of the page. A group's elements stay in
// a wave's registers from the largest one's search to the codes' store, so
// they are read once, and everything that a run needs is asked for at once
// (elements, old scale, codes beside the new ones). Before that stand four loads
// of slots, each waiting for the one before: a workgroup's own, those before
// them, a run's first, those after it. A workgroup looks for runs that start
// among its `scan` tokens; runs of few tokens or within one group go to its waves
// in turn, longer ones to all of them. 8003 prompt tokens, 8 heads of 128, pages
// of 64: 49.5 MB in 22 us (2.2 TB/s); 10 us would be the rate of a large copy, but
// values are stored 8 or 16 bytes at a time, page_size apart, a page's rows in
// pieces by several waves. One wave a run, with the elements read twice, took 53.
// ---------------------------------------------------------------------------
struct AppendArgs {
  KvView c;
  const uint16_t* k;
  const uint16_t* v;
  long long kt, kh, vt, vh;  // strides of tokens and heads, elements
  const int64_t* slots;
  int tokens;
};

constexpr int kAppendWaves = 4;

// The new tokens of one page: token t0 + i goes to place off + i, for i < n
// with bit i of hi:lo (the others have no slot).
struct Run {
  unsigned long long lo, hi;
  int t0, n, page, off;
  __device__ __forceinline__ bool has(int i) const {
    return i >= 0 && i < n && (((i < 64 ? lo : hi) >> (i & 63)) & 1);
  }
};

// Largest of non-negative floats as bits: NaN above infinity above the rest.
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
  return v;
}

__device__ __forceinline__ uint32_t abs_bits(float f) {
  return __builtin_bit_cast(uint32_t, f) & 0x7FFFFFFFu;
}

__device__ __forceinline__ uint32_t quantise(float x, float inv) {
  // fminf/fmaxf drop a NaN, so a code is in range whatever comes in.
  return (uint32_t)(int)fminf(fmaxf(rintf(x * inv), -kCodeMax), kCodeMax) & 0xFFu;
}

__device__ __forceinline__ uint32_t requantise_word(uint32_t w, float ratio) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) r |= quantise((float)code_of(w, i), ratio) << (8 * i);
  return r;
}

// The scale a page gets, from the old one and the new tokens' largest bits.
struct PageScale {
  float scale, inv, ratio;
  bool grew;
};
__device__ __forceinline__ PageScale page_scale(float old, uint32_t amax) {
  PageScale s;
  // An infinity counts as a NaN: the page's values for this head are NaN then.
  const float top = amax >= 0x7F800000u ? __builtin_nanf("")
                                        : __builtin_bit_cast(float, amax) * (1.0f / kCodeMax);
  const uint32_t ob = abs_bits(old), tb = abs_bits(top);
  s.grew = tb > ob;
  s.scale = __builtin_bit_cast(float, max(ob, tb));
  s.inv = s.scale >= 0x1p-126f ? 1.0f / s.scale : 0.0f;
  s.ratio = old * s.inv;
  return s;
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pair_max_bits(uint32_t w) {
  return max(abs_bits(pair_lo<kBf16>(w)), abs_bits(pair_hi<kBf16>(w)));
}
template <bool kBf16>
__device__ __forceinline__ uint32_t quantise_pair(uint32_t w, float inv) {
  return quantise(pair_lo<kBf16>(w), inv) | quantise(pair_hi<kBf16>(w), inv) << 8;
}

// A group's keys: a lane has 16 elements of a token, kUnits times.
template <int D, bool kBf16>
struct KeyGroup {
  static constexpr int kC = D / 16, kUnits = kC / 4;
  uint4 w[kUnits][2];

  static __device__ __forceinline__ int place(int g, int u, int lane) { return 16 * g + (64 * u + lane) / kC; }

  __device__ __forceinline__ void load(const AppendArgs& a, const Run& run, int head, int g, int lane) {
    const uint16_t* x = a.k + (long long)run.t0 * a.kt + (long long)head * a.kh + lane % kC * 16;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int t = place(g, u, lane) - run.off;
      const bool on = run.has(t);
      const uint4* p = reinterpret_cast<const uint4*>(x + (long long)(on ? t : 0) * a.kt);
      w[u][0] = on ? p[0] : zero4();
      w[u][1] = on ? p[1] : zero4();
    }
  }
  __device__ __forceinline__ uint32_t max_bits() const {
    uint32_t m = 0;
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        m = max(max(m, max(pair_max_bits<kBf16>(w[u][h].x), pair_max_bits<kBf16>(w[u][h].y))),
                max(pair_max_bits<kBf16>(w[u][h].z), pair_max_bits<kBf16>(w[u][h].w)));
    return m;
  }
  __device__ __forceinline__ void store(const AppendArgs& a, const Run& run, long long ph, int g, int lane,
                                        const PageScale& s) const {
    const int P = 1 << a.c.page_shift;
    uint4* codes = reinterpret_cast<uint4*>(a.c.k + ph * D * P) + lane % kC * P;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int at = place(g, u, lane);
      if (!run.has(at - run.off)) continue;
      uint32_t q[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        q[2 * h] = quantise_pair<kBf16>(w[u][h].x, s.inv) | quantise_pair<kBf16>(w[u][h].y, s.inv) << 16;
        q[2 * h + 1] = quantise_pair<kBf16>(w[u][h].z, s.inv) | quantise_pair<kBf16>(w[u][h].w, s.inv) << 16;
      }
      codes[at] = make_uint4(q[0], q[1], q[2], q[3]);
    }
  }
  // The page's earlier tokens of a group, where the scale grew.
  static __device__ __forceinline__ void requantise(const AppendArgs& a, const Run& run, long long ph, int g,
                                                    int lane, const PageScale& s) {
    const int P = 1 << a.c.page_shift;
    uint4* codes = reinterpret_cast<uint4*>(a.c.k + ph * D * P) + lane % kC * P;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int at = place(g, u, lane);
      if (at >= run.off) continue;
      const uint4 c = codes[at];
      codes[at] = make_uint4(requantise_word(c.x, s.ratio), requantise_word(c.y, s.ratio),
                             requantise_word(c.z, s.ratio), requantise_word(c.w, s.ratio));
    }
  }
};

// A group's values: a lane has two elements of kTok consecutive places, which
// are two runs of bytes in the cache, so the transposition costs no shuffle.
// `old` is what lies there, asked for where not every place is written.
template <int D, bool kBf16>
struct ValueGroup {
  static constexpr int kTok = D / 8, kWords = kTok / 4;
  typedef uint32_t words_t __attribute__((ext_vector_type(kWords)));
  uint32_t w[kTok];
  words_t old[2];

  static __device__ __forceinline__ int place(int g, int lane) { return 16 * g + lane / (D / 2) * kTok; }
  static __device__ __forceinline__ words_t* row(const AppendArgs& a, long long ph, int g, int lane, int r) {
    const int P = 1 << a.c.page_shift;
    return reinterpret_cast<words_t*>(a.c.v + ph * D * P + (long long)(lane % (D / 2) * 2 + r) * P + place(g, lane));
  }
  __device__ __forceinline__ void load(const AppendArgs& a, const Run& run, int head, int g, int lane) {
    const uint16_t* x = a.v + (long long)run.t0 * a.vt + (long long)head * a.vh + lane % (D / 2) * 2;
    bool all = true;
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      const int t = place(g, lane) + i - run.off;
      const bool on = run.has(t);
      all &= on;
      w[i] = on ? *reinterpret_cast<const uint32_t*>(x + (long long)t * a.vt) : 0u;
    }
    if (!all) {
      const long long ph = (long long)run.page * a.c.heads + head;
      old[0] = *row(a, ph, g, lane, 0);
      old[1] = *row(a, ph, g, lane, 1);
    }
  }
  __device__ __forceinline__ uint32_t max_bits() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kTok; ++i) m = max(m, pair_max_bits<kBf16>(w[i]));
    return m;
  }
  __device__ __forceinline__ void store(const AppendArgs& a, const Run& run, long long ph, int g, int lane,
                                        const PageScale& s) {
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      const int first = place(g, lane) + 4 * k - run.off;
      if (!s.grew && (first + 4 <= 0 || first >= run.n)) continue;  // as it lies
      uint32_t c[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = first + i;
        const bool on = run.has(t);
        const uint32_t q = quantise_pair<kBf16>(w[4 * k + i], s.inv);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t y = q >> (8 * r) & 0xFFu;
          if (!on) {
            y = old[r][k] >> (8 * i) & 0xFFu;
            if (t < 0 && s.grew) y = quantise((float)code_of(old[r][k], i), s.ratio);
          }
          c[r] |= y << (8 * i);
        }
      }
      old[0][k] = c[0];
      old[1][k] = c[1];
    }
    *row(a, ph, g, lane, 0) = old[0];
    *row(a, ph, g, lane, 1) = old[1];
  }
  // A group of earlier tokens alone, where the scale grew.
  static __device__ __forceinline__ void requantise(const AppendArgs& a, const Run& run, long long ph, int g,
                                                    int lane, const PageScale& s) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      words_t* at = row(a, ph, g, lane, r);
      words_t c = *at;
#pragma unroll
      for (int k = 0; k < kWords; ++k) c[k] = requantise_word(c[k], s.ratio);
      *at = c;
    }
  }
};

// One run by `waves` waves, the workgroup's all or this one alone. With pages
// of at most 128 places a wave of four has at most two groups of a run, and a
// wave alone runs within one.
template <typename Group, bool kKeys>
__device__ __forceinline__ void append_run(const AppendArgs& a, const Run& run, int head, int wave, int waves,
                                           int lane, uint32_t* shared_max) {
  const long long ph = (long long)run.page * a.c.heads + head;
  float* scales = kKeys ? a.c.ks : a.c.vs;
  const int g0 = (run.off >> 4) + wave, g1 = (run.off + run.n + 15) >> 4;
  const float old = run.off == 0 ? 0.0f : scales[ph];
  Group x[2];
  uint32_t amax = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (g0 + j * waves < g1) x[j].load(a, run, head, g0 + j * waves, lane);
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (g0 + j * waves < g1) amax = max(amax, x[j].max_bits());
  amax = wave_max_bits(amax);
  if (waves > 1) {
    __syncthreads();  // the run before may still be read
    if (lane == 0) shared_max[wave] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendWaves; ++w) amax = max(amax, shared_max[w]);
  }
  const PageScale s = page_scale(old, amax);
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (g0 + j * waves < g1) x[j].store(a, run, ph, g0 + j * waves, lane, s);
  if (s.grew) {
    // Earlier tokens: all their groups, but for values the one that they share
    // with new tokens, which is written whole above.
    const int stop = kKeys ? (run.off + 15) >> 4 : run.off >> 4;
    for (int g = wave; g < stop; g += waves) Group::requantise(a, run, ph, g, lane, s);
  }
  if (wave == 0 && lane == 0 && (s.grew || run.off == 0)) scales[ph] = s.scale;
}

// A run of few tokens by this wave alone, token by token, two elements a lane:
// little code, since its time is latency and a workgroup fetches its
// instructions cold (200 runs of one token and 8 heads: 7 us, on append_run 10).
constexpr int kFewTokens = 8;
template <int D, bool kBf16, bool kKeys>
__device__ __forceinline__ void append_few(const AppendArgs& a, const Run& run, int head, int lane) {
  constexpr int kSide = 128 / D;  // tokens at once
  const int P = 1 << a.c.page_shift;
  const int d = lane % (D / 2) * 2, side = lane / (D / 2);
  const long long ph = (long long)run.page * a.c.heads + head;
  float* scales = kKeys ? a.c.ks : a.c.vs;
  int8_t* codes = (kKeys ? a.c.k : a.c.v) + ph * D * P;
  const long long stride = kKeys ? a.kt : a.vt;
  const uint16_t* x = (kKeys ? a.k + (long long)head * a.kh : a.v + (long long)head * a.vh) +
                      (long long)run.t0 * stride + d;
  const float old = run.off == 0 ? 0.0f : scales[ph];
  auto load = [&](int t) {
    return run.has(t) ? *reinterpret_cast<const uint32_t*>(x + (long long)t * stride) : 0u;
  };
  const uint32_t first = load(side);
  uint32_t amax = pair_max_bits<kBf16>(first);
#pragma unroll 4
  for (int t = side + kSide; t < run.n; t += kSide) amax = max(amax, pair_max_bits<kBf16>(load(t)));
  const PageScale s = page_scale(old, wave_max_bits(amax));
  for (int t = side; t < run.n; t += kSide) {
    if (!run.has(t)) continue;
    const uint32_t q = quantise_pair<kBf16>(t == side ? first : load(t), s.inv);
    const int at = run.off + t;
    if (kKeys) {
      *reinterpret_cast<uint16_t*>(codes + (d / 16 * P + at) * 16 + d % 16) = (uint16_t)q;
    } else {
      codes[d * P + at] = (int8_t)q;
      codes[(d + 1) * P + at] = (int8_t)(q >> 8);
    }
  }
  if (s.grew) {  // the page's earlier tokens, of which a word with new ones is done by bytes
    const int words = kKeys ? run.off * (D / 4) : (run.off + 3) / 4 * D;
    for (int u = lane; u < words; u += 64) {
      const int tok = kKeys ? u / (D / 4) : u / D * 4;
      uint32_t* w = reinterpret_cast<uint32_t*>(
          kKeys ? codes + (u % (D / 4) / 4 * P + tok) * 16 + u % 4 * 4 : codes + u % D * P + tok);
      if (kKeys || tok + 4 <= run.off) {
        *w = requantise_word(*w, s.ratio);
      } else {
        int8_t* c = reinterpret_cast<int8_t*>(w);
        for (int i = 0; tok + i < run.off; ++i) c[i] = (int8_t)quantise((float)c[i], s.ratio);
      }
    }
  }
  if (lane == 0 && (s.grew || run.off == 0)) scales[ph] = s.scale;
}

__device__ __forceinline__ bool in_cache(const AppendArgs& a, long long slot) {
  return slot >= 0 && slot >> a.c.page_shift < a.c.pages;
}

// Whether token t, which has a slot, is its page's first one in this step.
__device__ __forceinline__ bool starts_run(const AppendArgs& a, int t, long long slot) {
  const int off = (int)(slot & ((1 << a.c.page_shift) - 1));
  for (int k = 1; k <= min(t, off); ++k) {  // back over tokens without a slot
    const long long s = a.slots[t - k];
    if (s == slot - k) return false;
    if (in_cache(a, s)) return true;
  }
  return true;
}

template <int D, bool kBf16>
__global__ __launch_bounds__(kAppendWaves * 64) void append_kernel(AppendArgs a, int scan) {
  __shared__ uint32_t shared_max[kAppendWaves];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.y;
  const int base = blockIdx.x * scan;  // scan <= 64
  const int P = 1 << a.c.page_shift;
  bool starts = false;
  if (lane < scan && lane < a.tokens - base) {
    const long long slot = a.slots[base + lane];
    starts = in_cache(a, slot) && starts_run(a, base + lane, slot);
  }
  int i = 0;
  for (unsigned long long mask = __ballot(starts); mask; ++i, mask &= mask - 1) {
    Run run;
    run.t0 = base + __builtin_ctzll(mask);
    const long long slot = a.slots[run.t0];
    run.page = (int)(slot >> a.c.page_shift);
    run.off = (int)(slot & (P - 1));
    // The tokens that follow on in the page, over those without a slot.
    run.n = 0;
    const int most = min(P - run.off, a.tokens - run.t0);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int j = 64 * w + lane;
      const long long s = j < most ? a.slots[run.t0 + j] : 0;
      const bool mine = j < most && s == slot + j;
      const bool on = mine || (j < most && !in_cache(a, s));
      const unsigned long long follow = run.n == 64 * w ? __ballot(on) : 0;
      const int c = follow == ~0ull ? 64 : __builtin_ctzll(~follow);
      run.n += c;
      (w ? run.hi : run.lo) = __ballot(mine) & (c == 64 ? ~0ull : (1ull << c) - 1);
    }
    const bool all = run.n > kFewTokens && (run.off & 15) + run.n > 16;  // more than a group
    if (!all && i % kAppendWaves != wave) continue;
    const int w = all ? wave : 0, waves = all ? kAppendWaves : 1;
    if (run.n <= kFewTokens) {
      if (blockIdx.z == 0) append_few<D, kBf16, true>(a, run, head, lane);
      else append_few<D, kBf16, false>(a, run, head, lane);
    } else if (blockIdx.z == 0) {
      append_run<KeyGroup<D, kBf16>, true>(a, run, head, w, waves, lane, shared_max);
    } else {
      append_run<ValueGroup<D, kBf16>, false>(a, run, head, w, waves, lane, shared_max);
    }
  }
}

// ---------------------------------------------------------------------------
// Read: bound by bytes, two thirds of them written. A lane has 8 elements of
// four tokens, so that a wave writes rows of 128 and 256 bytes. Keys: 8 bytes
// of each token. Values lie the other way round: four tokens' bytes of each
// element in one word where the tokens follow each other in a page, turned
// round in registers; else byte by byte. 65000 tokens of 8 heads of 128, 400 MB
// in 93 us (4.3 TB/s; a large copy has 5.0), 5000 of 32 heads, 123 MB in 25.5
// (4.8); single bytes of the values took 178 and 50.
// ---------------------------------------------------------------------------
struct ReadArgs {
  KvView c;
  const int64_t* slots;
  void* k;
  void* v;
  int tokens;
};

typedef float read_f4 __attribute__((ext_vector_type(4)));
typedef uint32_t read_u4 __attribute__((ext_vector_type(4)));

// Eight codes, two words, times a scale.
template <int kDtype>
__device__ __forceinline__ void store_codes(void* out, long long at, uint32_t lo, uint32_t hi, float s) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = (float)code_of(i < 4 ? lo : hi, i & 3) * s;
    asm("" : "+v"(x[i]));  // in fp32, also where the product could go into fp16 in one instruction
  }
  if constexpr (kDtype == DK_KV_F32) {
    read_f4* o = reinterpret_cast<read_f4*>(static_cast<float*>(out) + at);
    __builtin_nontemporal_store(read_f4{x[0], x[1], x[2], x[3]}, o);
    __builtin_nontemporal_store(read_f4{x[4], x[5], x[6], x[7]}, o + 1);
  } else {
    read_u4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = to_half_bits<kDtype>(x[2 * i]) | (uint32_t)to_half_bits<kDtype>(x[2 * i + 1]) << 16;
    __builtin_nontemporal_store(w, reinterpret_cast<read_u4*>(static_cast<uint16_t*>(out) + at));
  }
}

template <int D, int kDtype>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
  constexpr int kLanes = D / 8;
  const int P = 1 << a.c.page_shift;
  const int head = blockIdx.y;
  const int t0 = (blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes) * 4;
  const int d = threadIdx.x % kLanes * 8;
  if (t0 >= a.tokens) return;
  const int n = min(4, a.tokens - t0);
  long long slot[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) slot[i] = a.slots[t0 + min(i, n - 1)];
  bool ok[4];
  long long ph[4];
  float scale[4];
  const float* scales = blockIdx.z == 0 ? a.c.ks : a.c.vs;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long page = slot[i] >> a.c.page_shift;
    ok[i] = slot[i] >= 0 && page < a.c.pages;
    ph[i] = ok[i] ? page * a.c.heads + head : 0;
    scale[i] = ok[i] ? scales[ph[i]] : 0.0f;
  }
  uint32_t lo[4] = {}, hi[4] = {};
  if (blockIdx.z == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (ok[i]) {
        const int off = (int)(slot[i] & (P - 1));
        const uint2 w = *reinterpret_cast<const uint2*>(a.c.k + ph[i] * D * P + ((d / 16) * P + off) * 16 + d % 16);
        lo[i] = w.x, hi[i] = w.y;
      }
  } else {
    const int off = (int)(slot[0] & (P - 1));
    const bool follow = n == 4 && ok[0] && off + 3 < P && slot[1] == slot[0] + 1 &&
                        slot[2] == slot[0] + 2 && slot[3] == slot[0] + 3;
    if (follow) {
      const int8_t* c = a.c.v + ph[0] * D * P + (long long)d * P + (off & ~3);
      const int by = off & 3;
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = *reinterpret_cast<const uint32_t*>(c + e * P);
      if (by)  // the four tokens lie in two words
#pragma unroll
        for (int e = 0; e < 8; ++e)
          w[e] = __builtin_amdgcn_alignbyte(*reinterpret_cast<const uint32_t*>(c + e * P + 4), w[e], by);
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // four elements of four tokens, turned round
        const uint32_t ab = __builtin_amdgcn_perm(w[4 * h + 1], w[4 * h], 0x05010400u);
        const uint32_t cd = __builtin_amdgcn_perm(w[4 * h + 3], w[4 * h + 2], 0x05010400u);
        const uint32_t ef = __builtin_amdgcn_perm(w[4 * h + 1], w[4 * h], 0x07030602u);
        const uint32_t gh = __builtin_amdgcn_perm(w[4 * h + 3], w[4 * h + 2], 0x07030602u);
        uint32_t* to = h ? hi : lo;
        to[0] = __builtin_amdgcn_perm(cd, ab, 0x05040100u);
        to[1] = __builtin_amdgcn_perm(cd, ab, 0x07060302u);
        to[2] = __builtin_amdgcn_perm(gh, ef, 0x05040100u);
        to[3] = __builtin_amdgcn_perm(gh, ef, 0x07060302u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (ok[i]) {
          const uint8_t* c = reinterpret_cast<const uint8_t*>(a.c.v) + ph[i] * D * P + (long long)d * P +
                             (slot[i] & (P - 1));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            lo[i] |= (uint32_t)c[e * P] << (8 * e);
            hi[i] |= (uint32_t)c[(e + 4) * P] << (8 * e);
          }
        }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n)
      store_codes<kDtype>(blockIdx.z == 0 ? a.k : a.v, ((long long)(t0 + i) * a.c.heads + head) * D + d,
                          lo[i], hi[i], scale[i]);
}

}  // namespace dk

namespace {

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int page_shift(int page_size) {
  switch (page_size) {
    case 16: return 4;
    case 32: return 5;
    case 64: return 6;
    case 128: return 7;
    default: return -1;
  }
}

}  // namespace

namespace dk {

int kv_view(const dk_kv_cache* c, KvView* view) {
  if (!c) return set_error(DK_ERR_INVALID_ARGUMENT, "cache must not be NULL");
  const int shift = page_shift(c->page_size);
  if (shift < 0)
    return set_error(DK_ERR_INVALID_ARGUMENT, "page_size=%d must be 16, 32, 64 or 128", c->page_size);
  if (c->head_size != 64 && c->head_size != 128)
    return set_error(DK_ERR_INVALID_ARGUMENT, "head_size=%d must be 64 or 128", c->head_size);
  if (c->pages < 0 || c->heads < 1 || c->heads > 65535)
    return set_error(DK_ERR_INVALID_ARGUMENT, "the cache needs pages >= 0 and 1..65535 heads");
  if (c->pages > 0) {
    if (!c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales)
      return set_error(DK_ERR_INVALID_ARGUMENT, "the cache's codes and scales must not be NULL");
    if (!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16) || !aligned(c->k_scales, 4) ||
        !aligned(c->v_scales, 4))
      return set_error(DK_ERR_INVALID_ARGUMENT,
                       "the cache's codes must be 16-byte and its scales 4-byte aligned");
  }
  *view = KvView{c->k_codes, c->v_codes, c->k_scales, c->v_scales, c->pages, c->heads, shift};
  return DK_OK;
}

}  // namespace dk

extern "C" int dk_kv_plan(int32_t* tables, int table_width, const int32_t* held,
                          const int32_t* added, int requests, const int32_t* free_pages,
                          int free_capacity, const int32_t* free_count, int page_size,
                          int num_tokens, int64_t* slots, int32_t* positions,
                          int32_t* query_offsets, int32_t* seq_lens, int32_t* free_count_out,
                          hipStream_t stream) {
  const int shift = page_shift(page_size);
  if (shift < 0)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "page_size=%d must be 16, 32, 64 or 128", page_size);
  if (requests < 0 || requests > DK_KV_MAX_REQUESTS)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "requests must be in [0, %d]", DK_KV_MAX_REQUESTS);
  if (table_width < 0 || num_tokens < 0 || free_capacity < 0)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT,
                         "table_width, num_tokens and free_capacity must be >= 0");
  if (((long long)table_width << shift) > INT32_MAX)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "table_width * page_size must fit in int32");
  if (!query_offsets || !free_count || !free_count_out ||
      (requests > 0 && (!held || !added || !seq_lens)) ||
      (requests > 0 && table_width > 0 && !tables) || (num_tokens > 0 && (!slots || !positions)) ||
      (free_capacity > 0 && !free_pages))
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "plan's arrays must not be NULL");
  if (free_count == free_count_out)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "free_count_out must not be free_count");
  const dk::PlanArgs a{tables, held, added, free_pages, free_count, slots, positions,
                       query_offsets, seq_lens, free_count_out, table_width, requests,
                       free_capacity, shift, num_tokens};
  const unsigned blocks = num_tokens == 0 ? 1u : (unsigned)((num_tokens - 1) / dk::kPlanThreads + 1);
  hipLaunchKernelGGL(dk::plan_kernel, dim3(blocks), dim3(dk::kPlanThreads), 0, stream, a);
  return dk::check_launch("plan launch");
}

extern "C" int dk_kv_append(const dk_kv_cache* cache, const void* k, const void* v, int dtype,
                            long long k_token_stride, long long k_head_stride,
                            long long v_token_stride, long long v_head_stride,
                            const int64_t* slots, int num_tokens, hipStream_t stream) {
  dk::KvView view;
  if (const int rc = dk::kv_view(cache, &view)) return rc;
  if (dtype != DK_KV_F16 && dtype != DK_KV_BF16)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "k and v must be fp16 or bf16");
  if (num_tokens < 0) return dk::set_error(DK_ERR_INVALID_ARGUMENT, "num_tokens must be >= 0");
  if (num_tokens == 0 || cache->pages == 0) return DK_OK;
  if (!k || !v || !slots) return dk::set_error(DK_ERR_INVALID_ARGUMENT, "k, v and slots must not be NULL");
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(slots, 8))
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "k and v must be 16-byte, slots 8-byte aligned");
  if (k_token_stride % 8 || k_head_stride % 8 || v_token_stride % 8 || v_head_stride % 8)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "the strides of k and v must be multiples of 8");
  const dk::AppendArgs a{view, static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
                         k_token_stride, k_head_stride, v_token_stride, v_head_stride, slots,
                         num_tokens};
  // Tokens that a workgroup looks for runs among: about 12 workgroups a CU. Runs
  // of one token go round its four waves, and one of four waves finds few of
  // them; of whole pages one workgroup in many finds the start, and the others
  // cost their launch. 8 heads of 128, us by 4 / 16 / 32 tokens:
  //   2 prompts, 2000 tokens   19 / 10 / 12    300 sequences, a token each   11 / 16 / 23
  //   4 prompts, 4000 tokens   44 / 17 / 15    600 sequences, a token each   17 / 19 / 28
  //   2 prompts, 60000 tokens  - / 229 / 125; 64 tokens take 115, but 30 instead
  //   of 22 for 2000 tokens of 32 heads, where each has a run or two: only far on
  const long long rows = (long long)num_tokens * view.heads;
  int scan = 4;
  while (scan < 32 && rows > 1536LL * scan) scan *= 2;
  if (rows > 1 << 18) scan = 64;
  const dim3 grid((unsigned)((num_tokens - 1) / scan + 1), (unsigned)view.heads, 2);
  const dim3 block(dk::kAppendWaves * 64);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, a, scan); };
  if (cache->head_size == 64)
    dtype == DK_KV_BF16 ? launch(dk::append_kernel<64, true>) : launch(dk::append_kernel<64, false>);
  else
    dtype == DK_KV_BF16 ? launch(dk::append_kernel<128, true>) : launch(dk::append_kernel<128, false>);
  return dk::check_launch("append launch");
}

extern "C" int dk_kv_read(const dk_kv_cache* cache, const int64_t* slots, int num_tokens, int dtype,
                          void* k, void* v, hipStream_t stream) {
  dk::KvView view;
  if (const int rc = dk::kv_view(cache, &view)) return rc;
  if (dtype != DK_KV_F16 && dtype != DK_KV_BF16 && dtype != DK_KV_F32)
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "dtype must be fp16, bf16 or fp32");
  if (num_tokens < 0) return dk::set_error(DK_ERR_INVALID_ARGUMENT, "num_tokens must be >= 0");
  if (num_tokens == 0) return DK_OK;
  if (!k || !v || !slots) return dk::set_error(DK_ERR_INVALID_ARGUMENT, "k, v and slots must not be NULL");
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(slots, 8))
    return dk::set_error(DK_ERR_INVALID_ARGUMENT, "k and v must be 16-byte, slots 8-byte aligned");
  const dk::ReadArgs a{view, slots, k, v, num_tokens};
  auto launch = [&](auto kernel, int lanes) {
    const int each = 256 / lanes * 4;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((num_tokens - 1) / each + 1), (unsigned)view.heads, 2),
                       dim3(256), 0, stream, a);
  };
  if (cache->head_size == 64) {
    if (dtype == DK_KV_F16) launch(dk::read_kernel<64, DK_KV_F16>, 8);
    else if (dtype == DK_KV_BF16) launch(dk::read_kernel<64, DK_KV_BF16>, 8);
    else launch(dk::read_kernel<64, DK_KV_F32>, 8);
  } else {
    if (dtype == DK_KV_F16) launch(dk::read_kernel<128, DK_KV_F16>, 16);
    else if (dtype == DK_KV_BF16) launch(dk::read_kernel<128, DK_KV_BF16>, 16);
    else launch(dk::read_kernel<128, DK_KV_F32>, 16);
  }
  return dk::check_launch("read launch");
}
