// Device side of the requests of one batch: which tokens a tile holds and which
// adapter they take.
//
// Requests are ranges of tokens of any length, known on the device only.  A
// kernel that works in tiles of M tokens is launched with T / M + R + 2 slots;
// segment i (the tokens in front of the first request, each request, the tokens
// behind the last) starts at slot a_i / M + i, where its first token is a_i:
// floor(b / M) + i + 1 - (floor(a / M) + i) is never less than the ceil((b - a) / M)
// tiles it needs, so no tile is shared by two requests, nothing is counted
// beforehand, and a block finds its segment by one or two 64-way searches.
// What the arrays hold is clamped before it is used as an index.
#pragma once

#include "ra_common.h"
#include "req_kernels.h"

namespace harp_req {

__device__ __forceinline__ int64_t load_int(const void* p, int is64, int64_t i) {
  return is64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}
// first token of request i (0 .. count), within 0 .. tokens
__device__ __forceinline__ int token_of(const Requests& q, int i) {
  const int64_t v = q.offsets ? load_int(q.offsets, q.offsets64, i) : (int64_t)i * q.len;
  return (int)min(max(v, (int64_t)0), (int64_t)q.tokens);
}
// adapter of request i, -1: none
__device__ __forceinline__ int adapter_of(const Requests& q, int i) {
  const int64_t v = load_int(q.index, q.index64, i);
  return v >= 0 && v < q.n ? (int)v : -1;
}
// first token of segment i: 0 in front of the requests, request i - 1, behind them
__device__ __forceinline__ int segment_start(const Requests& q, int i) {
  if (i <= 0) return 0;
  return i > q.count + 1 ? q.tokens : token_of(q, i - 1);
}

// The largest segment i (0 .. count + 1) with at(i), which holds for 0 and, in order, for no others than a first run
template <class F>
__device__ __forceinline__ int last_segment(const Requests& q, F at) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = q.count + 2;  // at(lo) holds; hi is behind the last segment or at(hi) does not hold
  while (hi - lo > 1) {          // (uniform, and hi - lo shrinks 64-fold)
    const int step = (hi - lo + 63) / 64;
    const int i = lo + lane * step;
    const uint64_t b = __ballot(i < hi && at(i)) | 1;
    const int k = b == ~0ull ? 63 : __ffsll((unsigned long long)~b) - 2;  // the last lane of the leading run
    hi = min(hi, lo + (k + 1) * step);
    lo = lo + k * step;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// A tile: rows first .. first + rows - 1 (rows <= M, or not positive) with one adapter (-1: none)
struct Tile {
  int first, rows, adapter;
};
template <int M>
__device__ __forceinline__ Tile tile_at(const Requests& q, int slot) {
  const int i = last_segment(q, [&](int s) { return segment_start(q, s) / M + s <= slot; });
  const int a = segment_start(q, i), b = segment_start(q, i + 1);
  Tile t;
  t.first = a + (slot - (a / M + i)) * M;
  t.rows = min(M, b - t.first);
  t.adapter = i >= 1 && i <= q.count ? adapter_of(q, i - 1) : -1;
  t.first = __builtin_amdgcn_readfirstlane(t.first);
  t.rows = __builtin_amdgcn_readfirstlane(t.rows);
  t.adapter = __builtin_amdgcn_readfirstlane(t.adapter);
  return t;
}
inline int64_t slots_of(const Requests& q, int M) { return (int64_t)q.tokens / M + q.count + 2; }

}  // namespace harp_req
