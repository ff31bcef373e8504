// gfx950 kernels of the QK RMSNorm with a rotary embedding of several axes
// (time, height, width of a token), forward and backward, and of its table.
//
//   rho = 1 / sqrt(mean(x^2) + eps),  n = x rho w            (or n = x without a norm)
//   phi_p = position[axis of p] * theta^(-2 j / width)       (j: the pair's place in its axis)
//   (y0, y1) = (n0 cos - n1 sin, n0 sin + n1 cos)            pairs (2p, 2p + 1) or (p, p + D / 2)
//   d = dy turned back by phi,  g = d w,  dx = rho (g - x rho mean(g x rho)),  dw = sum_rows d x rho
//
// All arithmetic is fp32 over the stored inputs, every output rounded once, to
// nearest.  The angle is formed in 64 bits as a share of a turn (position *
// rate, less its whole turns and then its whole quarters), so that a far
// position loses nothing; what is left, within an eighth of a turn, takes the
// Taylor series of sine and cosine in 32 bits (remainders (pi/4)^11 / 11! =
// 1.8e-9 and (pi/4)^10 / 10! = 2.5e-8).
//
// Layout: LPR lanes (8, 16 or 32 for D <= 64, 128, 256) hold a row, 8 values
// (four pairs) each.  The angles of the few tokens that a block's rows are of are
// formed by all its threads while the rows' loads are on their way, and shared
// through LDS (each lane its own four, their rates' powers in 64 bits among them, the
// arithmetic took longer than the memory: 62 us for 8192 tokens x 60 heads).  No
// table is read.
//
// Bound by memory: at 8192 tokens x 60 heads of 128 in bf16 the forward moves 252 MB in
// 52 us (4.8 TB/s) and the backward, which reads x and dy, 377 MB in 85 us (4.4 TB/s),
// where a large copy moves 5.1 TB/s.  A call of few tokens is bound by its launch.
#include <algorithm>
#include <type_traits>

#include "ra_common.h"
#include "req_kernels.h"
#include "rope_device.h"

namespace harp_req {

namespace {

using harp_ra::bf16;
using harp_ra::f32x4;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// sum over the LPR lanes of a row's group, the same value in all of them
template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (LPR == 32)
    v += __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401f));  // lane ^ 16
  if constexpr (LPR >= 16) {
    v += dpp<0x128>(v);  // row_ror:8
    v += dpp<0x124>(v);  // row_ror:4
  } else {
    v += dpp<0x1b>(dpp<0x141>(v));  // row_half_mirror, then quad_perm:[3,2,1,0]: lane ^ 4
  }
  v += dpp<0x4e>(v);  // quad_perm:[2,3,0,1]
  v += dpp<0xb1>(v);  // quad_perm:[1,0,3,2]
  return v;
}

// A lane's 8 values as they are in memory: two runs of four, next to each
// other (pairs 2p, 2p + 1) or D / 2 apart (HALF).
template <bool F32>
struct Raw {
  typedef u32x2 Run;
  Run v[2];
};
template <>
struct Raw<true> {
  typedef f32x4 Run;
  Run v[2];
};

template <bool F32, bool HALF>
__device__ __forceinline__ Raw<F32> load_raw(const char* row, int sub, int D) {
  Raw<F32> r;
  constexpr int es = F32 ? 4 : 2;
  if constexpr (!HALF && !F32) {
    const u32x4 u = *(const u32x4*)(row + sub * 16);
    r.v[0] = u32x2{u[0], u[1]};
    r.v[1] = u32x2{u[2], u[3]};
  } else {
    const char* p = row + (HALF ? 4 * sub : 8 * sub) * es;
    r.v[0] = *(const typename Raw<F32>::Run*)p;
    r.v[1] = *(const typename Raw<F32>::Run*)(p + (HALF ? D / 2 : 4) * es);
  }
  return r;
}
// to fp32, in the order of the pairs: (v[0], v[1]) is pair 4 sub, and so on
template <bool F32, bool HALF>
__device__ __forceinline__ void unpack(const Raw<F32>& r, float (&v)[8]) {
  float t[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (F32) {
#pragma unroll
      for (int k = 0; k < 4; ++k) t[4 * i + k] = r.v[i][k];
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        t[4 * i + 2 * k] = __uint_as_float(r.v[i][k] << 16);
        t[4 * i + 2 * k + 1] = __uint_as_float(r.v[i][k] & 0xffff0000u);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[2 * k] = HALF ? t[k] : t[2 * k];
    v[2 * k + 1] = HALF ? t[4 + k] : t[2 * k + 1];
  }
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 v = {(bf16)lo, (bf16)hi};
  return __builtin_bit_cast(uint32_t, v);
}
template <bool F32, bool HALF>
__device__ __forceinline__ void store_row(char* row, int sub, int D, const float (&v)[8]) {
  float t[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    t[HALF ? k : 2 * k] = v[2 * k];
    t[HALF ? 4 + k : 2 * k + 1] = v[2 * k + 1];
  }
  constexpr int es = F32 ? 4 : 2;
  char* p = row + (HALF ? 4 * sub : 8 * sub) * es;
  char* q = p + (HALF ? D / 2 : 4) * es;
  if constexpr (F32) {
    *(f32x4*)p = f32x4{t[0], t[1], t[2], t[3]};
    *(f32x4*)q = f32x4{t[4], t[5], t[6], t[7]};
  } else {
    const u32x4 u = {pack_bf16(t[0], t[1]), pack_bf16(t[2], t[3]), pack_bf16(t[4], t[5]), pack_bf16(t[6], t[7])};
    if constexpr (HALF) {
      *(u32x2*)p = u32x2{u[0], u[1]};
      *(u32x2*)q = u32x2{u[2], u[3]};
    } else {
      *(u32x4*)p = u;
    }
  }
}
// a lane's weights, in the order of the pairs (any alignment of the vector)
template <bool HALF>
__device__ __forceinline__ void load_weight(const void* w, int w_f32, int sub, int D, float (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = 1.f;
  if (!w) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int e0 = HALF ? 4 * sub + k : 8 * sub + 2 * k, e1 = HALF ? e0 + D / 2 : e0 + 1;
    v[2 * k] = w_f32 ? ((const float*)w)[e0] : __uint_as_float((uint32_t)((const uint16_t*)w)[e0] << 16);
    v[2 * k + 1] = w_f32 ? ((const float*)w)[e1] : __uint_as_float((uint32_t)((const uint16_t*)w)[e1] << 16);
  }
}

// Workgroups are dealt to the 8 XCDs round-robin: each XCD takes one contiguous
// range of the work, so that what its L2 holds is one window of memory.
__device__ __forceinline__ uint32_t xcd_block(uint32_t bid, uint32_t blocks) {
  const uint32_t q = blocks / 8, r = blocks % 8, x = bid % 8, local = bid / 8;
  return x < r ? x * (q + 1) + local : r * (q + 1) + (x - r) * q + local;
}

// A launch's blocks: those of q, then those of k.  The heads of a token are dealt
// to J groups of lanes, R to each.
struct Blocks {
  int q, k;
  uint32_t q_steps, k_steps;  // of a block (the last one's may be fewer)
};
struct Unit {
  uint32_t b, s;
  int j;
};
__device__ __forceinline__ Unit unit_at(uint32_t S, uint32_t J, uint32_t unit) {
  const uint32_t tok = unit / J, b = tok / S;
  return Unit{b, tok - b * S, (int)(unit - tok * J)};
}
// n units on, in 32 bits (n is a block's groups)
__device__ __forceinline__ Unit unit_after(uint32_t S, uint32_t J, const Unit& u, uint32_t n) {
  const uint32_t v = u.j + n, dt = v / J, s = u.s + dt, db = s / S;
  return Unit{u.b + db, s - db * S, (int)(v - dt * J)};
}
__device__ __forceinline__ int64_t offset_of(const RopeStrides& st, const Unit& u, int h) {
  return u.b * st.b + (int64_t)h * st.h + (int64_t)u.s * st.s;
}

// The angles of a block's step: its kGroups units, one after the other, are of a
// few tokens (kGroups at most).  A thread keeps one pair, whose rate it forms
// once, and forms the angles of every 256 / kPairs-th token for all of them.
template <int LPR>
struct Angles {
  static constexpr int kPairs = 4 * LPR, kGroups = kThreads / LPR;
  typedef float2 Buf[kGroups][kPairs];
  double rate;
  int64_t axis;  // offset of the pair's axis in a token's position
  int pair, at;
  __device__ __forceinline__ explicit Angles(const RopeParams& p) {
    pair = threadIdx.x % kPairs;
    at = threadIdx.x / kPairs;
    int a;
    rate = rate_of(p.axes, min(pair, p.D / 2 - 1), a);
    axis = a * p.pos.sa;
  }
  // of the tokens from `first` (of unit u) on
  __device__ __forceinline__ void form(const RopeParams& p, const Unit& u, int tokens, float sign, Buf& buf) const {
    if (2 * pair >= p.D) return;
    for (int k = at; k < tokens; k += kThreads / kPairs) {
      const uint32_t s = u.s + k, db = s / (uint32_t)p.S;
      const int64_t off[1] = {axis};
      double v[1];
      load_pos(p.pos, (int64_t)(u.b + db) * p.pos.sb + (int64_t)(s - db * (uint32_t)p.S) * p.pos.ss, off, v);
      float2 cs;
      cos_sin(v[0] * rate, cs.x, cs.y);
      cs.y *= sign;
      buf[k][pair] = cs;
    }
  }
  static __device__ __forceinline__ void read(const Buf& buf, int token, int sub, float (&c)[4], float (&s)[4]) {
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
      const f32x4 v = *(const f32x4*)&buf[token][4 * sub + k];
      c[k] = v[0];
      s[k] = v[1];
      c[k + 1] = v[2];
      s[k + 1] = v[3];
    }
  }
};

__device__ __forceinline__ void rotate(float (&v)[8], const float (&c)[4], const float (&s)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float a = v[2 * k], b = v[2 * k + 1];
    v[2 * k] = __builtin_fmaf(-b, s[k], a * c[k]);
    v[2 * k + 1] = __builtin_fmaf(b, c[k], a * s[k]);
  }
}
__device__ __forceinline__ float dot8(const float (&a)[8], const float (&b)[8]) {
  float d = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) d = __builtin_fmaf(a[k], b[k], d);
  return d;
}
__device__ __forceinline__ float inv_rms(float ss, int D, float eps) {
  return __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(ss, (float)D) + eps));
}

}  // namespace

// ---------------------------------------------------------------------------
// Forward, and (sign -1, no norm) the rotation's own backward
// ---------------------------------------------------------------------------
namespace {

// A block's share bid of `blocks` of a tensor's steps, kGroups units each (a unit: R
// heads of one token): where each group of lanes is in them.
template <int LPR, int R>
struct Walk {
  static constexpr int kGroups = kThreads / LPR;
  uint32_t units, step, end, S;  // (at most 2^31 units: 64-bit divisions took a microsecond of a short call)
  int J, grp, groups, token;  // groups: that have a unit in this step; token: this one's among the step's
  Unit u0, u;                 // the step's first unit, this group's
  __device__ __forceinline__ Walk(const RopeParams& p, const RopeHeads& t, uint32_t bid, int blocks, uint32_t each) {
    J = (t.H + R - 1) / R;
    S = (uint32_t)p.S;
    grp = threadIdx.x / LPR;
    units = (uint32_t)p.B * S * (uint32_t)J;
    step = xcd_block(bid, blocks) * each;
    end = min(step + each, (units + kGroups - 1) / kGroups);
    if (step < end) {
      u0 = unit_at(p.S, J, step * kGroups);
      place();
    }
  }
  // a group behind the last unit repeats it (and counts for nothing)
  __device__ __forceinline__ void place() {
    groups = (int)min((uint32_t)kGroups, units - step * kGroups);
    const int at = min(grp, groups - 1);
    token = (u0.j + at) / J;
    u = unit_after(S, J, u0, at);
  }
  __device__ __forceinline__ int tokens() const { return (u0.j + groups - 1) / J + 1; }
  __device__ __forceinline__ bool next() {
    if (++step >= end) return false;
    u0 = unit_after(S, J, u0, kGroups);
    place();
    return true;
  }
};

// Forward: the blocks of long calls (four heads a group) walk their steps, a short one's have a
// step each (with the walk's second buffer and copies, 1024 tokens x 30 heads of 72 in fp32 took
// 12.2 us instead of 11.3 and one token's heads 7.2 instead of 4.5)
template <int R>
constexpr bool kWalk = R == 4;

template <bool F32, bool HALF, int LPR, int R>
__device__ __forceinline__ void forward_share(const RopeParams& p, const RopeHeads& t, const Angles<LPR>& ang,
                                              uint32_t bid, int blocks, uint32_t each,
                                              typename Angles<LPR>::Buf (&angles)[kWalk<R> ? 2 : 1]) {
  constexpr int es = F32 ? 4 : 2;
  const int sub = threadIdx.x % LPR;
  const bool lane_in = 8 * sub < p.D;
  const int lane = lane_in ? sub : 0;  // lanes behind D repeat the first values and store nothing
  Walk<LPR, R> at(p, t, bid, blocks, each);
  if (at.step >= at.end) return;
  float w[8];
  load_weight<HALF>(t.w, t.w_f32, lane, p.D, w);
  Raw<F32> raw[R];
  auto load = [&]() {
#pragma unroll
    for (int i = 0; i < R; ++i)
      raw[i] = load_raw<F32, HALF>((const char*)t.x + offset_of(t.sx, at.u, min(at.u.j + at.J * i, t.H - 1)) * es, lane, p.D);
  };
  load();
  bool more = true;
  for (int odd = 0; more; odd ^= 1) {
    ang.form(p, at.u0, at.tokens(), p.sign, angles[odd]);
    __syncthreads();  // (the other buffer's readers are past the barrier of the step before)
    float c[4], s[4];
    Angles<LPR>::read(angles[odd], at.token, lane, c, s);
    const Unit u = at.u;
    const bool in = lane_in && at.grp < at.groups;
    Raw<F32> cur[R];
#pragma unroll
    for (int i = 0; i < R; ++i) cur[i] = raw[i];
    more = kWalk<R> && at.next();
    if (more) load();
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int h = u.j + at.J * i;
      float v[8];
      unpack<F32, HALF>(cur[i], v);
      if (t.norm) {
        const float inv = inv_rms(group_sum<LPR>(lane_in ? dot8(v, v) : 0.f), p.D, t.eps);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = v[k] * inv * w[k];
      }
      rotate(v, c, s);
      if (in && h < t.H) store_row<F32, HALF>((char*)t.y + offset_of(t.sy, u, h) * es, lane, p.D, v);
    }
  }
}

}  // namespace

template <bool F32, bool HALF, int LPR, int R>
__global__ __launch_bounds__(kThreads) void rope_forward_kernel(RopeParams p, Blocks n) {
  __shared__ __attribute__((aligned(16))) typename Angles<LPR>::Buf angles[kWalk<R> ? 2 : 1];
  const Angles<LPR> ang(p);
  harp_ra::sched_fence();
  const bool is_k = (int)blockIdx.x >= n.q;
  if constexpr (kWalk<R>) {
    // (two copies of the walk: both tensors' strides side by side do not fit the scalar registers)
    if (!is_k) forward_share<F32, HALF, LPR, R>(p, p.t[0], ang, blockIdx.x, n.q, n.q_steps, angles);
    else forward_share<F32, HALF, LPR, R>(p, p.t[1], ang, blockIdx.x - n.q, n.k, n.k_steps, angles);
  } else {
    const RopeHeads t = is_k ? p.t[1] : p.t[0];
    forward_share<F32, HALF, LPR, R>(p, t, ang, blockIdx.x - (is_k ? n.q : 0), is_k ? n.k : n.q, 1, angles);
  }
}

// ---------------------------------------------------------------------------
// Backward: a block walks its share of the units with the sums of both weights'
// gradients in registers and writes one partial row of each; a second kernel
// adds those in a fixed order.
// ---------------------------------------------------------------------------
namespace {
// The block's share of one tensor, t: the next step's loads are on their way while one is worked on
template <bool F32, bool HALF, int LPR, int R>
__device__ __forceinline__ void backward_share(const RopeParams& p, const RopeHeads& t, const Angles<LPR>& ang,
                                               uint32_t bid, int blocks, uint32_t each,
                                               typename Angles<LPR>::Buf (&angles)[2],
                                               float (&wg)[8]) {
  constexpr int es = F32 ? 4 : 2;
  const int sub = threadIdx.x % LPR;
  const bool lane_in = 8 * sub < p.D;
  const int lane = lane_in ? sub : 0;
  Walk<LPR, R> at(p, t, bid, blocks, each);
  if (at.step >= at.end) return;
  float w[8];
  load_weight<HALF>(t.w, t.w_f32, lane, p.D, w);
  Raw<F32> rx[R], rd[R];
  auto load = [&]() {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int h = min(at.u.j + at.J * i, t.H - 1);
      rd[i] = load_raw<F32, HALF>((const char*)t.dy + offset_of(t.sdy, at.u, h) * es, lane, p.D);
      rx[i] = load_raw<F32, HALF>((const char*)t.x + offset_of(t.sx, at.u, h) * es, lane, p.D);
    }
  };
  load();
  bool more = true;
  for (int odd = 0; more; odd ^= 1) {
    ang.form(p, at.u0, at.tokens(), -1.f, angles[odd]);
    __syncthreads();  // (the other buffer's readers are past the barrier of the step before)
    float c[4], s[4];
    Angles<LPR>::read(angles[odd], at.token, lane, c, s);
    const Unit u = at.u;
    const bool in = lane_in && at.grp < at.groups;
    Raw<F32> cx[R], cd[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      cx[i] = rx[i];
      cd[i] = rd[i];
    }
    more = at.next();
    if (more) load();
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int h = u.j + at.J * i;
      const bool mine = in && h < t.H;
      float x[8], g[8];
      unpack<F32, HALF>(cd[i], g);
      unpack<F32, HALF>(cx[i], x);
      rotate(g, c, s);
      const float inv = inv_rms(group_sum<LPR>(lane_in ? dot8(x, x) : 0.f), p.D, t.eps);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[k] = lane_in ? x[k] * inv : 0.f;
        wg[k] = __builtin_fmaf(mine ? g[k] : 0.f, x[k], wg[k]);
        g[k] *= w[k];
      }
      const float mean = __fdiv_rn(group_sum<LPR>(dot8(g, x)), (float)p.D);
#pragma unroll
      for (int k = 0; k < 8; ++k) g[k] = inv * __builtin_fmaf(-x[k], mean, g[k]);
      if (mine) store_row<F32, HALF>((char*)t.y + offset_of(t.sy, u, h) * es, lane, p.D, g);
    }
  }
}
}  // namespace

template <bool F32, bool HALF, int LPR, int R>
__global__ __launch_bounds__(kThreads) void rope_backward_kernel(RopeParams p, Blocks n) {
  constexpr int kGroups = kThreads / LPR;
  __shared__ __attribute__((aligned(16))) typename Angles<LPR>::Buf angles[2];
  __shared__ float part[kGroups][LPR * 8 + 4];
  float wg[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) wg[k] = 0.f;
  const Angles<LPR> ang(p);
  harp_ra::sched_fence();
  if ((int)blockIdx.x < n.q) backward_share<F32, HALF, LPR, R>(p, p.t[0], ang, blockIdx.x, n.q, n.q_steps, angles, wg);
  else backward_share<F32, HALF, LPR, R>(p, p.t[1], ang, blockIdx.x - n.q, n.k, n.k_steps, angles, wg);
  if (!p.wpart) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) part[threadIdx.x / LPR][8 * (threadIdx.x % LPR) + k] = wg[k];
  __syncthreads();
  // value 2 k + e of the partial row is element e of pair k
  if ((int)threadIdx.x < p.D) {
    const int at = threadIdx.x, pair = at / 2;
    float sum = 0.f;
#pragma unroll
    for (int gi = 0; gi < kGroups; ++gi) sum += part[gi][at];
    p.wpart[(int64_t)blockIdx.x * p.D + (HALF ? pair + (at & 1) * (p.D / 2) : at)] = sum;
  }
}

// gw[e] = sum of wpart[block][e] over a tensor's blocks: 8 columns a block, 128
// lanes of rows, added in a fixed order
constexpr int kWgCols = 8, kWgLanes = 128;
__global__ __launch_bounds__(kWgCols* kWgLanes) void rope_wgrad_kernel(const float* src, int q_blocks, int k_blocks,
                                                                       int D, void* gq, int gq_f32, void* gk,
                                                                       int gk_f32) {
  __shared__ float part[kWgLanes][kWgCols + 1];
  const int tx = threadIdx.x % kWgCols, ty = threadIdx.x / kWgCols;
  const int t = blockIdx.y, e = blockIdx.x * kWgCols + tx;  // D is a multiple of 8
  void* const dst = t ? gk : gq;
  const int f32 = t ? gk_f32 : gq_f32;
  if (!dst) return;
  const int blocks = t ? k_blocks : q_blocks;
  if (t) src += (int64_t)q_blocks * D;
  float acc = 0.f;
#pragma unroll 4
  for (int i = ty; i < blocks; i += kWgLanes) acc += src[(int64_t)i * D + e];
  part[ty][tx] = acc;
  __syncthreads();
  if (ty < 8) {
    acc = 0.f;
#pragma unroll
    for (int k = 0; k < kWgLanes / 8; ++k) acc += part[ty * (kWgLanes / 8) + k][tx];
  }
  __syncthreads();
  if (ty < 8) part[ty][tx] = acc;
  __syncthreads();
  if (ty != 0) return;
  acc = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) acc += part[k][tx];
  if (f32) ((float*)dst)[e] = acc;
  else ((bf16*)dst)[e] = (bf16)acc;
}

// ---------------------------------------------------------------------------
// The table (table_share)
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kThreads) void rope_table_kernel(RopeTable t) {
  table_share(t, (int)blockIdx.x, (int)gridDim.x, kThreads);
}

// ---------------------------------------------------------------------------
// Launchers
// ---------------------------------------------------------------------------
namespace {

int lanes_per_row(int D) { return D > 128 ? 32 : D > 64 ? 16 : 8; }

constexpr int kFillBlocks = 1024;  // four blocks for each of 256 CUs
// A long call's blocks walk their steps, four of them at a time on a CU, all in one round.  8192 tokens x 60
// heads of 128: forward 52 us (58 with 1536 blocks), backward 85 (95 with 1280).
constexpr int kMaxBlocks = 1024;
constexpr int kOneStep = 1 << 30;  // no limit: a step to a block

int64_t blocks_of(const RopeParams& p, const RopeHeads& t, int R) {
  const int per = kThreads / lanes_per_row(p.D);
  return ((int64_t)p.B * p.S * ((t.H + R - 1) / R) + per - 1) / per;
}
int64_t blocks_of(const RopeParams& p, int R) { return blocks_of(p, p.t[0], R) + blocks_of(p, p.t[1], R); }
// heads of a token for one group of lanes: as many as leave kFillBlocks blocks
int heads_per_group(const RopeParams& p, int most) {
  for (int R = most; R > 1; R /= 2)
    if (blocks_of(p, R) >= kFillBlocks) return R;
  return 1;
}
template <template <bool, bool, int, int> class K>
hipError_t dispatch(const RopeParams& p, int R, const Blocks& r, hipStream_t st) {
  auto heads = [&](auto f32, auto half, auto l) {
    constexpr bool F = decltype(f32)::value, H = decltype(half)::value;
    constexpr int L = decltype(l)::value;
    if (R == 4) K<F, H, L, 4>::launch(p, r, st);
    else if (R == 2) K<F, H, L, 2>::launch(p, r, st);
    else K<F, H, L, 1>::launch(p, r, st);
  };
  auto lanes = [&](auto f32, auto half) {
    const int l = lanes_per_row(p.D);
    if (l == 32) heads(f32, half, std::integral_constant<int, 32>{});
    else if (l == 16) heads(f32, half, std::integral_constant<int, 16>{});
    else heads(f32, half, std::integral_constant<int, 8>{});
  };
  auto layout = [&](auto f32) { p.half ? lanes(f32, std::true_type{}) : lanes(f32, std::false_type{}); };
  p.f32 ? layout(std::true_type{}) : layout(std::false_type{});
  return hipGetLastError();
}
template <bool F, bool H, int L, int R>
struct Forward {
  static void launch(const RopeParams& p, const Blocks& r, hipStream_t st) {
    hipLaunchKernelGGL((rope_forward_kernel<F, H, L, R>), dim3((unsigned)(r.q + r.k)), dim3(kThreads), 0, st, p, r);
  }
};
constexpr int kBwdHeads = 2;  // rows of x and dy of four heads would leave a CU half the waves
template <bool F, bool H, int L, int R>
struct Backward {
  static void launch(const RopeParams& p, const Blocks& r, hipStream_t st) {
    constexpr int B = R > kBwdHeads ? kBwdHeads : R;
    hipLaunchKernelGGL((rope_backward_kernel<F, H, L, B>), dim3((unsigned)(r.q + r.k)), dim3(kThreads), 0, st, p, r);
  }
};

// each tensor's share of at most `most` blocks, as few as leave the busiest one no more steps
Blocks shares(const RopeParams& p, int R, int most) {
  auto share = [&](const RopeHeads& t, int& blocks, uint32_t& each) {
    const int64_t steps = blocks_of(p, t, R);
    if (!steps) return;
    const int64_t mine = std::max<int64_t>(1, (int64_t)most * t.H / (p.t[0].H + p.t[1].H));
    each = (uint32_t)((steps + mine - 1) / mine);
    blocks = (int)((steps + each - 1) / each);
  };
  Blocks n{};
  share(p.t[0], n.q, n.q_steps);
  share(p.t[1], n.k, n.k_steps);
  return n;
}

}  // namespace

hipError_t launch_rope_forward(const RopeParams& p, hipStream_t stream) {
  const int R = heads_per_group(p, 4);
  return dispatch<Forward>(p, R, shares(p, R, R == 4 ? kMaxBlocks : kOneStep), stream);
}

void rope_bwd_blocks(const RopeParams& p, int blocks[2]) {
  const Blocks n = shares(p, heads_per_group(p, kBwdHeads), kMaxBlocks);
  blocks[0] = n.q;
  blocks[1] = n.k;
}
hipError_t launch_rope_backward(const RopeParams& p, hipStream_t stream) {
  const int R = heads_per_group(p, kBwdHeads);
  return dispatch<Backward>(p, R, shares(p, R, kMaxBlocks), stream);
}

hipError_t launch_rope_wgrad(const float* wpart, const int blocks[2], int D, void* const gw[2], const int gw_f32[2],
                             hipStream_t stream) {
  hipLaunchKernelGGL(rope_wgrad_kernel, dim3((unsigned)(D / kWgCols), 2), dim3(kWgCols * kWgLanes), 0, stream, wpart,
                     blocks[0], blocks[1], D, gw[0], gw_f32[0], gw[1], gw_f32[1]);
  return hipGetLastError();
}

hipError_t launch_rope_table(const RopeTable& t, hipStream_t stream) {
  const int per = kThreads / t.pairs;
  const int64_t need = (t.tokens + per - 1) / per;
  hipLaunchKernelGGL(rope_table_kernel, dim3((unsigned)std::min<int64_t>(need, 2048)), dim3(kThreads), 0, stream, t);
  return hipGetLastError();
}

}  // namespace harp_req
