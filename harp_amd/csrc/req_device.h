// Device side of the requests of one batch: which tokens a tile holds and which
// adapter they take.
//
// Requests are ranges of tokens of any length, known on the device only.  A
// kernel that works in tiles of M tokens is launched with T / M + R + 2 slots;
// segment i (the tokens in front of the first request, each request, the tokens
// behind the last) starts at slot a_i / M + i, where its first token is a_i:
// floor(b / M) + i + 1 - (floor(a / M) + i) is never less than the ceil((b - a) / M)
// tiles it needs, so no tile is shared by two requests, nothing is counted
// beforehand, and a block finds its segment by a 64-way search.
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

// at(i) holds for segment 0 and, in order, for no others than a first run of the segments 0 .. count + 1.
// at(lo) holds, hi is behind the last segment or at(hi) does not: narrows both to at most `most` apart.
template <class F>
__device__ __forceinline__ void narrow(int& lo, int& hi, int most, F at) {
  const int lane = threadIdx.x & 63;
  while (hi - lo > most) {  // (uniform, and hi - lo shrinks 64-fold)
    const int step = (hi - lo + 63) / 64;
    const int i = lo + lane * step;
    const uint64_t b = __ballot(i < hi && at(i)) | 1;
    const int k = b == ~0ull ? 63 : __ffsll((unsigned long long)~b) - 2;  // the last lane of the leading run
    hi = min(hi, lo + (k + 1) * step);
    lo = lo + k * step;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);
}
// The largest segment i with at(i)
template <class F>
__device__ __forceinline__ int last_segment(const Requests& q, F at) {
  int lo = 0, hi = q.count + 2;
  narrow(lo, hi, 1, at);
  return lo;
}

// A tile: rows first .. first + rows - 1 (rows <= M, or not positive) with one adapter (-1: none)
struct Tile {
  int first, rows, adapter;
};
// (the last 62 candidates' starts and adapters come with one load each, one in every lane: each load that
// waits for another costs a short call most of a microsecond)
template <int M>
__device__ __forceinline__ Tile tile_at(const Requests& q, int slot) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = q.count + 2;
  narrow(lo, hi, 63, [&](int s) { return segment_start(q, s) / M + s <= slot; });
  const int i = lo + lane, start = segment_start(q, i);
  const int adapter = i >= 1 && i <= q.count ? adapter_of(q, i - 1) : -1;
  const uint64_t in = __ballot(i < hi && start / M + i <= slot) | 1;
  const int k = __ffsll((unsigned long long)~in) - 2;  // (0 .. 62: the segment is lo + k)
  Tile t;
  const int a = __builtin_amdgcn_readlane(start, k), b = __builtin_amdgcn_readlane(start, k + 1);
  t.first = a + (slot - (a / M + lo + k)) * M;
  t.rows = min(M, b - t.first);
  t.adapter = __builtin_amdgcn_readlane(adapter, k);
  return t;
}
inline int64_t slots_of(const Requests& q, int M) { return (int64_t)q.tokens / M + q.count + 2; }

}  // namespace harp_req
