// Shared by the kernels of the gated delta rule and the short convolution.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "decode_kernel/dk_delta.h"
#include "dk_kv.hpp"

namespace dk {

constexpr int kChunk = 64;           // tokens that the chunked form takes at once
constexpr int kPrepareThreads = 256; // of the workgroup that prepares a chunk and head
constexpr float kUnitEps = 1e-6f;    // added to a squared length
// Below this a decay's exponential is 0 in fp32 (e^-128 < 2^-149): logarithms
// are cut there, so that sums over a chunk stay finite and differences exact.
constexpr float kLowestLog = -128.0f;

// The decay's logarithm as it is summed: cut at kLowestLog, NaN kept.
__device__ __forceinline__ float cut_log(float g) { return g < kLowestLog ? kLowestLog : g; }

struct DeltaArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  long long q_token, q_head, k_token, k_head, v_token, v_head;
  const float* log_decay;
  const float* beta;
  float* states;
  const int32_t* held;
  const int32_t* offsets;
  uint16_t* out;
  int tokens, requests, qk_heads, v_heads, group;
  int limit;  // requests of up to so many tokens go one by one, longer ones in chunks
  int longest;  // max_query_len
  int normalize;
  float scale;
};

// Whether offsets grow from at least 0 to at most `tokens`; by one wave.
__device__ __forceinline__ bool wave_offsets_ok(const int32_t* offsets, int requests, int tokens) {
  bool bad = false;
  for (int i = threadIdx.x & 63; i < requests; i += 64) bad |= offsets[i + 1] < offsets[i];
  if ((threadIdx.x & 63) == 0) bad |= offsets[0] < 0 || offsets[requests] > tokens;
  return __ballot(bad) == 0;
}

// The request that is number `rank` (from 0) of those with more than `limit`
// tokens, or -1; by one wave. Offsets have to be good.
__device__ __forceinline__ int find_long(const int32_t* offsets, int requests, int limit, int rank) {
  for (int first = 0; first < requests; first += 64) {
    const int i = first + (threadIdx.x & 63);
    unsigned long long is = __ballot(i < requests && offsets[min(i, requests - 1) + 1] - offsets[min(i, requests - 1)] > limit);
    const int count = __popcll(is);
    if (rank < count) {
      for (; rank > 0; --rank) is &= is - 1;
      return first + __ffsll(is) - 1;
    }
    rank -= count;
  }
  return -1;
}

// A tile of a request's new tokens. Tiles of `tile` tokens have numbers that
// need no sum over the requests: request b's begin at offsets[b] / tile + b,
// and since floor(x + n) - floor(x) + 1 >= ceil(n), they end before the next
// request's do begin. tokens / tile + requests numbers are enough. Where only
// requests of more than `limit` tokens have tiles, b is the request's number
// among those.
struct Tile {
  int request;    // -1: the number is nobody's
  int row;        // its first row
  int count;      // its rows
  int index;      // which tile of its request
  int total;      // its request's rows
  int head, end;  // the first row of all requests, and one past the last
};

// Numbers that the chunks of requests of more than `limit` tokens take.
inline long long chunk_slots(int tokens, int requests, int limit) {
  const int longs = tokens / (limit + 1);
  return (long long)(tokens / kChunk) + (requests < longs ? requests : longs);
}

// The tile with number `number` (kLong: of requests of more than `limit` tokens), and whether offsets are good; by each wave for
// itself, with the same answer in all. Offsets are loaded once, 64 requests at
// a time, and what is needed of them is taken from other lanes: a load that
// waits for another costs 1 to 2 us next to stores of a full chip.
template <bool kLong = false>
__device__ __forceinline__ bool find_tile(const int32_t* offsets, int requests, int tokens, int tile,
                                          int number, Tile* out, int limit = 0) {
  const int lane = threadIdx.x & 63;
  int b = -1, rank_b = 0, from_b = 0, to_b = 0, head = 0, end = 0, longs = 0;
  bool bad = false;
  for (int first = 0; first < requests; first += 64) {
    const int i = min(first + lane, requests - 1);
    const int from = offsets[i], to = offsets[i + 1];
    bad |= to < from;
    bool has = first + lane < requests;
    int rank = i;
    if constexpr (kLong) {
      has = has && to - from > limit;
      const unsigned long long is = __ballot(has);
      rank = longs + __builtin_amdgcn_mbcnt_hi((uint32_t)(is >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)is, 0));
      longs += __popcll(is);
    }
    const unsigned long long before = __ballot(has && from / tile + rank <= number);
    if (before) {  // requests' tiles begin one after another: the last that does before the number
      const int at = 63 - __clzll(before);
      b = first + at;
      rank_b = kLong ? __builtin_amdgcn_readlane(rank, at) : b;
      from_b = __builtin_amdgcn_readlane(from, at);
      to_b = __builtin_amdgcn_readlane(to, at);
    }
    if (first == 0) head = __builtin_amdgcn_readlane(from, 0);
    end = __builtin_amdgcn_readlane(to, 63);  // of the last request: i ends there
  }
  *out = Tile{-1, 0, 0, 0, 0, head, end};
  if (__ballot(bad) || head < 0 || end > tokens) return false;
  if (b < 0) return true;
  const int n = to_b - from_b, index = number - (from_b / tile + rank_b);
  if ((long long)index * tile >= n) return true;
  out->request = b;
  out->row = from_b + index * tile;
  out->count = min(tile, n - index * tile);
  out->index = index;
  out->total = n;
  return true;
}

size_t delta_chunk_bytes(int num_tokens, int requests, int limit, int qk_heads, int v_heads, int key_size);
int delta_chunk_launch(const DeltaArgs& a, int key_size, int value_size, bool bf16, void* workspace,
                       hipStream_t stream);

}  // namespace dk
