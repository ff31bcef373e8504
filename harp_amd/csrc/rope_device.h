// Device side of the rotary embedding: the angle of a pair, formed in 64 bits as a
// share of a turn, and its cosine and sine.  For the kernels that rotate and for those
// that write the table.
#pragma once

#include "ra_common.h"
#include "req_kernels.h"

namespace harp_req {

// turns per unit of position of pair p, and its axis.  (The exponent is formed from the pair's place
// in its axis: from its place in the head, with the axes in front taken off again, it loses bits to
// them, 2^-18 of a turn at positions of 2^31 where the axes in front are 60 pairs and theta is 1e6;
// so formed the angle there is within 2^-22.9 of a turn: an ulp of exp2, the roundings of 1 / (2 pi),
// of the two products and of the exponent, which is small where the rate is not.)
__device__ __forceinline__ double rate_of(const RopeAxes& ax, int p, int& axis) {
  double c = ax.c[0];
  int first = 0;
  axis = 0;
#pragma unroll
  for (int a = 1; a < kMaxAxes; ++a)
    if (a < ax.n && p >= ax.end[a - 1]) {
      axis = a;
      first = ax.end[a - 1];
      c = ax.c[a];
    }
  return exp2(c * (double)(p - first)) * 0.15915494309189535;
}
// the elements at base + off[k]
template <int N>
__device__ __forceinline__ void load_pos(const RopePos& q, int64_t base, const int64_t (&off)[N], double (&v)[N]) {
  if (q.dtype == kI32) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = (double)((const int32_t*)q.p + base)[off[k]];
  } else if (q.dtype == kI64) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = (double)((const int64_t*)q.p + base)[off[k]];
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = (double)((const float*)q.p + base)[off[k]];
  }
}
// cos and sin of `turns` turns
__device__ __forceinline__ void cos_sin(double turns, float& c, float& s) {
  turns -= __builtin_rint(turns);                // within half a turn, exact
  const double q = __builtin_rint(4.0 * turns);  // quarters: -2 .. 2
  const float x = (float)__builtin_fma(4.0, turns, -q) * 1.57079632679489662f;  // within pi / 4
  const int n = (int)q;
  const float x2 = x * x;
  // x - x^3/3! + x^5/5! - x^7/7! + x^9/9!, and 1 - x^2/2! + x^4/4! - x^6/6! + x^8/8!
  const float sp = __builtin_fmaf(
      x * x2, __builtin_fmaf(x2, __builtin_fmaf(x2, __builtin_fmaf(x2, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f),
      x);
  const float cp = __builtin_fmaf(
      x2, __builtin_fmaf(x2, __builtin_fmaf(x2, __builtin_fmaf(x2, 1.f / 40320.f, -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
  const bool odd = n & 1;
  s = odd ? cp : sp;
  c = odd ? sp : cp;
  if (n == 2 || n == -2 || n == -1) s = -s;
  if (n == 2 || n == -2 || n == 1) c = -c;
}

// A block's share of the table, of `blocks`: a thread keeps one pair and walks the tokens
__device__ __forceinline__ void table_share(const RopeTable& t, int block, int blocks, int threads) {
  const int per = threads / t.pairs;  // tokens of a block's step
  const int p = threadIdx.x % t.pairs, at = threadIdx.x / t.pairs;
  if (at >= per) return;
  int axis;
  const double rate = rate_of(t.axes, p, axis);
#pragma unroll 4
  for (int64_t tok = (int64_t)block * per + at; tok < t.tokens; tok += (int64_t)blocks * per) {
    const int64_t b = tok / t.S, s = tok - b * t.S;
    const int64_t off[1] = {axis * t.pos.sa};
    double v[1];
    load_pos(t.pos, b * t.pos.sb + s * t.pos.ss, off, v);
    float2 cs;
    cos_sin(v[0] * rate, cs.x, cs.y);
    t.out[tok * t.pairs + p] = cs;
  }
}

}  // namespace harp_req
