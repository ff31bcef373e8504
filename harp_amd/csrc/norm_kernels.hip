// gfx950 kernels of the residual addition with its RMSNorm, forward and
// backward, and of 8-bit rows (quantise, norm + quantise, dequantise).
//
//   h = x + r                          (rounded once, to r's type)
//   rho = 1 / sqrt(mean(h^2) + eps),   y = h * rho * w
//   g = dy * w,  c = mean(g * h * rho)
//   d = rho * (g - h * rho * c) + dh,  dx = d, dr = d,  dw = sum_rows dy * h * rho
//   8-bit rows: a = max |v|, s = a / 127, q = v * 127 / a to nearest (ties to even)
//
// All arithmetic and sums are fp32 over the stored inputs; every output is
// rounded once, to nearest.  y of the 8-bit rows is never rounded to bf16:
// with v = h * w the common factor rho cancels from q = 127 v / max |v|, and
// only the scale, rho * max |v| / 127, holds it, so the row's two reductions
// (sum of squares, maximum) need one exchange.
//
// The kernels are bound by memory: each row is read once into registers (8
// values per thread and vector) and finished there.  Rows need no alignment
// beyond their element's: a 16-byte global access at any address is one
// instruction on gfx950, and the vector at a row's end is taken apart.
//
// Measured, 8192 rows of 3840 (a copy of 1 GiB reaches 5.23 TB/s here): norm
// of a bf16 x with its fp32 residual 67 us (378 MB, 5.6 TB/s), backward 103 us
// (503 MB, 4.9 TB/s) and 5 us for the weight's gradient; norm to 8 bits of
// bf16 rows and residual 37 us (220 MB, 5.9 TB/s, part of it out of the last
// caches), dequantise 17.4 us (94 MB, 5.4 TB/s).  256 rows: 4.5, 6.2 + 2 .. 3
// us, which is a launch, a trip to HBM and an exchange; one row to 8 bits 3 us.
#include "blk_kernels.h"
#include "ra_common.h"

namespace harp_blk {

using harp_ra::bf16;

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef u32x4 u32x4u __attribute__((aligned(2)));

constexpr int kVec = 8;  // values per vector

template <int DT>
struct Elem;
template <>
struct Elem<kBf16> {
  typedef uint16_t type;
};
template <>
struct Elem<kF32> {
  typedef float type;
};
template <>
struct Elem<kNone> {
  typedef float type;
};

__device__ __forceinline__ float from_bits(uint32_t b) { return __uint_as_float(b); }
__device__ __forceinline__ uint16_t bf16_rne(float f) { return __builtin_bit_cast(uint16_t, (bf16)f); }

// n (1 .. 8) values at p; the rest are zero
template <int DT>
__device__ __forceinline__ f32x8 load8(const typename Elem<DT>::type* p, int n) {
  f32x8 v;
  if (n == kVec) {
    if constexpr (DT == kBf16) {
      const u32x4 u = *(const u32x4u*)p;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = from_bits(u[i] << 16);
        v[2 * i + 1] = from_bits(u[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const harp_ra::f32x4 u = *(const harp_ra::f32x4u*)(p + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * i + e] = u[e];
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      v[e] = 0.f;
      if (e < n) {
        if constexpr (DT == kBf16)
          v[e] = from_bits((uint32_t)p[e] << 16);
        else
          v[e] = p[e];
      }
    }
  }
  return v;
}

// A vector as it is in memory; zeros where it lies behind the row.  load_raw
// only loads: a vector that would reach past the row's end is read at the row's
// last 8 values instead, and unpack moves the n that count to the front, zeros
// behind them.  So a kernel's loads are all on their way before the first is
// waited for; converted where they are loaded, they went one by one (norm to 8
// bits of 8192 rows of 3840: 45 us, this way 37).  Rows of 8 values or more.
template <int DT>
struct Raw {
  u32x4 u;
};
template <>
struct Raw<kF32> {
  harp_ra::f32x4 lo, hi;
};
template <>
struct Raw<kNone> {};

template <int DT>
__device__ __forceinline__ Raw<DT> load_raw(const typename Elem<DT>::type* row, int c, int cols) {
  Raw<DT> r{};
  const auto* p = row + min(c, cols - kVec);
  if constexpr (DT == kBf16) {
    if (c < cols) r.u = *(const u32x4u*)p;
  } else if constexpr (DT == kF32) {
    if (c < cols) {
      r.lo = *(const harp_ra::f32x4u*)p;
      r.hi = *(const harp_ra::f32x4u*)(p + 4);
    }
  }
  return r;
}

template <int DT>
__device__ __forceinline__ f32x8 unpack(const Raw<DT>& r, int n) {
  f32x8 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == kBf16) {
      v[2 * i] = from_bits(r.u[i] << 16);
      v[2 * i + 1] = from_bits(r.u[i] & 0xffff0000u);
    } else {
      v[i] = r.lo[i];
      v[4 + i] = r.hi[i];
    }
  }
  if (n > 0 && n < kVec) {
    const int by = kVec - n;
#pragma unroll
    for (int step = 1; step < kVec; step *= 2)
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float next = e + step < kVec ? v[e + step] : 0.f;
        if (by & step) v[e] = next;
      }
  }
  return v;
}

template <int DT>
__device__ __forceinline__ void store8(typename Elem<DT>::type* p, const f32x8& v, int n) {
  if constexpr (DT == kBf16) {
    uint16_t h[kVec];
#pragma unroll
    for (int e = 0; e < kVec; ++e) h[e] = bf16_rne(v[e]);
    if (n == kVec) {
      u32x4 u;
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = (uint32_t)h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
      *(u32x4u*)p = u;
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (e < n) p[e] = h[e];
    }
  } else {
    if (n == kVec) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        harp_ra::f32x4 u;
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = v[4 * i + e];
        *(harp_ra::f32x4u*)(p + 4 * i) = u;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (e < n) p[e] = v[e];
    }
  }
}

// weight vector: a run-time type (its branch is the same in every thread)
__device__ __forceinline__ f32x8 load_w(const void* w, int dtype, int c, int n) {
  if (!w) {
    f32x8 v;
#pragma unroll
    for (int e = 0; e < kVec; ++e) v[e] = 1.f;
    return v;
  }
  return dtype == kF32 ? load8<kF32>((const float*)w + c, n) : load8<kBf16>((const uint16_t*)w + c, n);
}

// the same in two steps, for rows of 8 values or more
struct RawW {
  u32x4 lo, hi;  // bf16: lo alone
};
__device__ __forceinline__ void load_raw_w(RawW& r, const void* w, int dtype, int c, int cols) {
  if (dtype == kF32) {
    const Raw<kF32> f = load_raw<kF32>((const float*)w, c, cols);
    r.lo = __builtin_bit_cast(u32x4, f.lo);
    r.hi = __builtin_bit_cast(u32x4, f.hi);
  } else {
    r.lo = load_raw<kBf16>((const uint16_t*)w, c, cols).u;
  }
}
__device__ __forceinline__ f32x8 unpack_w(const RawW& r, const void* w, int dtype, int n) {
  if (!w) {
    f32x8 v;
#pragma unroll
    for (int e = 0; e < kVec; ++e) v[e] = 1.f;
    return v;
  }
  if (dtype == kF32)
    return unpack<kF32>({__builtin_bit_cast(harp_ra::f32x4, r.lo), __builtin_bit_cast(harp_ra::f32x4, r.hi)}, n);
  return unpack<kBf16>({r.lo}, n);
}

// x + r as it is kept: in r's type
template <int RD>
__device__ __forceinline__ float round_to(float v) {
  if constexpr (RD == kBf16) return (float)(bf16)v;
  return v;
}

// Sum, and maximum of unsigned words, over the TPR threads of a row; every
// thread gets the results.  Rows of one wave exchange within it; a row of
// several waves goes through LDS (one row per block then).
template <int TPR, bool SUM, bool MAX>
__device__ __forceinline__ void row_reduce(float& s, uint32_t& m, float* lds_s, uint32_t* lds_m) {
#pragma unroll
  for (int d = (TPR < 64 ? TPR : 64) / 2; d > 0; d >>= 1) {
    if (SUM) s += __shfl_xor(s, d);
    if (MAX) m = max(m, (uint32_t)__shfl_xor((int)m, d));
  }
  if constexpr (TPR > 64) {
    constexpr int kW = TPR / 64;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      if (SUM) lds_s[wave] = s;
      if (MAX) lds_m[wave] = m;
    }
    __syncthreads();
    if (SUM) {
      s = 0.f;
#pragma unroll
      for (int i = 0; i < kW; ++i) s += lds_s[i];
    }
    if (MAX) {
      m = 0;
#pragma unroll
      for (int i = 0; i < kW; ++i) m = max(m, lds_m[i]);
    }
  }
}

// The scale of a row and what turns its values into steps.  The maximum comes
// as the bits of |v|, which order as the values do with infinity and NaN on
// top: a row that holds one has the scale NaN (and steps of zero), so that
// whatever reads it is NaN too; so has a row whose normed values are not finite
// (factor infinite: eps 0 and squares that sum to 0).  A row of zeros has scale
// and steps zero.
// Maxima below 2^-100 are raised by 2^100 first, or 127 / a would overflow;
// those above 2^100 are lowered by it, or 127 v would.  (Values that become
// denormal or zero by that are far below a step.)
struct Steps {
  float pre, a, inv, scale;
};
__device__ __forceinline__ Steps row_steps(uint32_t max_bits, float factor) {
  Steps t;
  const float a = from_bits(max_bits);
  t.pre = a < 0x1p-100f ? 0x1p100f : a > 0x1p100f ? 0x1p-100f : 1.f;
  t.a = a * t.pre;
  t.inv = __fdiv_rn(127.f, t.a);
  t.scale = __fdiv_rn(a * factor, 127.f);
  if (max_bits == 0) t.inv = 0.f;
  if (!(t.scale < __builtin_inff())) {
    t.inv = 0.f;
    t.scale = __uint_as_float(0x7fc00000u);
  }
  return t;
}

// v * 127 / a to the nearest integer, ties to even, of one vector, packed.
// f = v * inv is off by 2^-23 of its size (two roundings; 127 steps: 1.52e-5),
// so only values that close to a border between two steps can round to the wrong
// one: where a vector has one, the sign of 254 v - m a decides, with m / 2 the
// border on f's side of q.  It is exact: m a is its rounding p and the rounding's
// error; 254 v - p is less than 2^-13 a beside a border and, v being at least
// a / 254, a multiple of 2^-31 a, so one fma forms it without a rounding.  (Taken
// from 127 v - q a in one fp32, 51 of 12000 values within one fp32 step of a
// border came out a step off; in 64 bits 8192 bf16 rows of 3840, many of whose
// values lie on a border, take 22.5 us instead of 20.5.)
__device__ __forceinline__ uint2 pack_steps(const f32x8& v, const Steps& t) {
  f32x8 q;
  float far = 0.f;
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    const float f = v[e] * t.pre * t.inv;
    q[e] = __builtin_rintf(f);
    far = __builtin_fmaxf(far, __builtin_fabsf(f - q[e]));
  }
  if (__builtin_expect(far > 0.49998f, 0)) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const float x = v[e] * t.pre, one = __builtin_copysignf(1.f, x * t.inv - q[e]), m = 2.f * q[e] + one;
      const float p = m * t.a, err = __builtin_fmaf(m, t.a, -p);
      const float over = one * (__builtin_fmaf(254.f, x, -p) - err);
      const bool odd = ((int)q[e] & 1) != 0;
      if (over > 0.f || (over == 0.f && odd)) q[e] += one;
    }
  }
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < kVec; ++e) w[e >> 2] |= ((uint32_t)(int)q[e] & 0xffu) << (8 * (e & 3));
  return make_uint2(w[0], w[1]);
}

}  // namespace

enum { kModeNorm = 0, kModeNorm8 = 1, kModeQuant = 2 };

// TPR threads per row, NV vectors of 8 per thread; blocks of max(TPR, 256)
// threads hold 256 / TPR rows, or one.  TPR is a quarter of a wave up to 128
// columns (20000 rows of 64 take 5 us, with a wave for each 9 to 12), a wave up
// to 1024 (no LDS, no barrier), then 256, and 512 where 256 would need more than
// 4 vectors each: the row's registers (16 of fp32 at 3840 columns) leave 7 or 8
// blocks on a CU, whose loads hide each other's exchanges.
template <int MODE, int XD, int RD, int TPR, int NV>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_kernel(NormParams p) {
  constexpr int kRows = TPR > 256 ? 1 : 256 / TPR;
  constexpr bool kEarlyW = MODE != kModeQuant && NV <= 2;  // the weight is loaded with the row (more have no room)
  typedef typename Elem<XD>::type TX;
  typedef typename Elem<RD>::type TR;
  __shared__ float lds_s[16];
  __shared__ uint32_t lds_m[16];
  const int64_t row = (int64_t)blockIdx.x * kRows + (kRows > 1 ? threadIdx.x / TPR : 0);
  if (row >= p.rows) return;  // whole rows: rows of several waves are alone in their block
  const int t = threadIdx.x % TPR;
  const TX* x = (const TX*)p.x + row * p.ldx;
  const TR* r = (const TR*)p.res + row * p.ldr;

  f32x8 v[NV];
  RawW wr[NV];
  float ss = 0.f;
  uint32_t mx = 0;
  if (TPR > 64 || NV > 1 || p.cols >= kVec) {
    Raw<XD> xr[NV];
    Raw<RD> rr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * kVec;
      xr[i] = load_raw<XD>(x, c, p.cols);
      if constexpr (RD != kNone) rr[i] = load_raw<RD>(r, c, p.cols);
    }
    if (kEarlyW && p.w) {
#pragma unroll
      for (int i = 0; i < NV; ++i) load_raw_w(wr[i], p.w, p.w_dtype, (i * TPR + t) * kVec, p.cols);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int n = p.cols - (i * TPR + t) * kVec;
      v[i] = unpack<XD>(xr[i], n);
      if constexpr (RD != kNone) {
        const f32x8 a = unpack<RD>(rr[i], n);
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[i][e] = round_to<RD>(v[i][e] + a[e]);
      }
    }
  } else {  // a row of fewer values than a vector (NV is 1)
    const int n = p.cols - t * kVec;
#pragma unroll
    for (int e = 0; e < kVec; ++e) v[0][e] = 0.f;
    if (n > 0) {
      v[0] = load8<XD>(x, n);
      if constexpr (RD != kNone) {
        const f32x8 a = load8<RD>(r, n);
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[0][e] = round_to<RD>(v[0][e] + a[e]);
      }
    }
  }
  auto weight = [&](int i, int c, int n) {
    return kEarlyW && (TPR > 64 || NV > 1 || p.cols >= kVec) ? unpack_w(wr[i], p.w, p.w_dtype, n)
                                                             : load_w(p.w, p.w_dtype, c, n);
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * kVec, n = min(kVec, p.cols - c);
    if constexpr (RD != kNone)
      if (p.h && n > 0) store8<RD>((TR*)p.h + row * p.ldh + c, v[i], n);
    if constexpr (MODE != kModeQuant)
#pragma unroll
      for (int e = 0; e < kVec; ++e) ss = __builtin_fmaf(v[i][e], v[i][e], ss);
    if constexpr (MODE == kModeNorm8)
      if (n > 0) {
        const f32x8 w = weight(i, c, n);
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[i][e] *= w[e];
      }
    if constexpr (MODE != kModeNorm)
#pragma unroll
      for (int e = 0; e < kVec; ++e) mx = max(mx, __float_as_uint(v[i][e]) & 0x7fffffffu);
  }
  row_reduce<TPR, MODE != kModeQuant, MODE != kModeNorm>(ss, mx, lds_s, lds_m);
  float rho = 1.f;
  if constexpr (MODE != kModeQuant) {
    rho = __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(ss, (float)p.cols) + p.eps));
    if (p.rstd && t == 0) p.rstd[row] = rho;
  }
  if constexpr (MODE == kModeNorm) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * kVec, n = min(kVec, p.cols - c);
      if (n > 0) {
        const f32x8 w = weight(i, c, n);
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[i][e] = v[i][e] * rho * w[e];
        store8<XD>((TX*)p.y + row * p.ldy + c, v[i], n);
      }
    }
  } else {
    const Steps st = row_steps(mx, rho);
    const bool bad = !(st.scale < __builtin_inff());
    if (t == 0) p.scale[row] = st.scale;
    int8_t* q = p.q + row * p.ldq;
    const int end = (p.cols + 15) & ~15;  // the last 16 bytes whole, zeros behind the row's values
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * kVec;
      if (c < end) *(uint2*)(q + c) = bad ? make_uint2(0, 0) : pack_steps(v[i], st);
    }
  }
}

// ---------------------------------------------------------------------------
// Backward.  A block of GROUPS groups of TPR threads walks its share of the
// rows, one row per group at a time, and keeps the weight gradient's sums of
// its columns in registers; the groups' sums are added in LDS at the end and
// written as one partial row, so the order of every sum is fixed by the
// launch alone.  At most 512 blocks, two to a CU: more would only lengthen the
// partial rows that wgrad_kernel reads (512 x 3840 fp32 are 8 MB, which stay in
// the caches: 5 us).  KEEP: dy and h stay in registers between the row's two
// passes; the longest rows have no room and read them again (out of L2).
template <int XD, int HD, int TPR, int NV, int GROUPS, bool KEEP>
__global__ __launch_bounds__(TPR* GROUPS) void norm_bwd_kernel(NormBwdParams p) {
  typedef typename Elem<XD>::type TX;
  typedef typename Elem<HD>::type TH;
  constexpr int kW = TPR / 64;
  __shared__ float lds_s[2][GROUPS][kW > 0 ? kW : 1];
  const int grp = threadIdx.x / TPR;
  int t = threadIdx.x % TPR;
  f32x8 gw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < kVec; ++e) gw[i][e] = 0.f;
  constexpr bool kEarlyDh = KEEP && NV <= 2;  // a row's dh is loaded with its dy and h (more have no room)
  const bool raw = KEEP && (TPR > 64 || NV > 1 || p.cols >= kVec);  // rows of a vector or more
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  const int64_t n_iter = (p.rows + step - 1) / step;
  for (int64_t it = 0; it < n_iter; ++it) {  // the same count in every group: the barrier below is in step
    const int64_t row = it * step + (int64_t)blockIdx.x * GROUPS + grp;
    const bool live = row < p.rows;
    // (opaque, or every vector's bounds tests would be kept in SGPRs over the loop: 34 spilled)
    asm volatile("" : "+v"(t));
    constexpr int kKeep = KEEP ? NV : 1;
    f32x8 gs[kKeep], hs[kKeep];
    Raw<HD> dhr[kEarlyDh ? NV : 1];
    float c1 = 0.f;
    const float rho = live ? p.rstd[row] : 0.f;
    const TX* dy = (const TX*)p.dy + row * p.ldy;
    const TH* hp = (const TH*)p.h + row * p.ldh;
    const TH* dhp = (const TH*)p.dh + row * p.lddh;
    auto load = [&](int i, f32x8& g, f32x8& h) {
      const int c = (i * TPR + t) * kVec, n = live ? min(kVec, p.cols - c) : 0;
      if (n > 0) {
        g = load8<XD>(dy + c, n);
        h = load8<HD>(hp + c, n);
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) g[e] = h[e] = 0.f;
      }
    };
    // g: dy -> dy w, h -> h rho
    auto scale = [&](int i, f32x8& g, f32x8& h, bool sums) {
      const int c = (i * TPR + t) * kVec, n = min(kVec, p.cols - c);
      if (n > 0) {
        const f32x8 w = load_w(p.w, p.w_dtype, c, n);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          h[e] *= rho;
          if (sums) gw[i][e] = __builtin_fmaf(g[e], h[e], gw[i][e]);
          g[e] *= w[e];
          if (sums) c1 = __builtin_fmaf(g[e], h[e], c1);
        }
      }
    };
    if constexpr (KEEP) {
      if (raw) {
        if (live) {
          Raw<XD> gr[NV];
          Raw<HD> hr[NV];
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * kVec;
            gr[i] = load_raw<XD>(dy, c, p.cols);
            hr[i] = load_raw<HD>(hp, c, p.cols);
          }
          if (kEarlyDh && p.dh) {
#pragma unroll
            for (int i = 0; i < NV; ++i) dhr[i] = load_raw<HD>(dhp, (i * TPR + t) * kVec, p.cols);
          }
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const int n = p.cols - (i * TPR + t) * kVec;
            gs[i] = unpack<XD>(gr[i], n);
            hs[i] = unpack<HD>(hr[i], n);
          }
        } else {
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < kVec; ++e) gs[i][e] = hs[i][e] = 0.f;
        }
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) load(i, gs[i], hs[i]);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) scale(i, gs[i], hs[i], true);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        load(i, gs[0], hs[0]);
        scale(i, gs[0], hs[0], true);
      }
    }
#pragma unroll
    for (int d = (TPR < 64 ? TPR : 64) / 2; d > 0; d >>= 1) c1 += __shfl_xor(c1, d);
    if constexpr (TPR > 64) {
      // two buffers in turn: the next row's writes meet no reader of this one
      float* s = lds_s[it & 1][grp];
      if ((t & 63) == 0) s[t >> 6] = c1;
      __syncthreads();
      c1 = 0.f;
#pragma unroll
      for (int i = 0; i < kW; ++i) c1 += s[i];
    }
    c1 = __fdiv_rn(c1, (float)p.cols);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * kVec, n = live ? min(kVec, p.cols - c) : 0;
      f32x8 &g = gs[KEEP ? i : 0], &h = hs[KEEP ? i : 0];
      if constexpr (!KEEP) {
        load(i, g, h);
        scale(i, g, h, false);
      }
      if (n > 0) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) g[e] = rho * __builtin_fmaf(-h[e], c1, g[e]);
        if (p.dh) {
          const f32x8 a = kEarlyDh && raw ? unpack<HD>(dhr[kEarlyDh ? i : 0], n) : load8<HD>(dhp + c, n);
#pragma unroll
          for (int e = 0; e < kVec; ++e) g[e] += a[e];
        }
        store8<XD>((TX*)p.dx + row * p.lddx + c, g, n);
        if (p.dres) store8<HD>((TH*)p.dres + row * p.lddr + c, g, n);
      }
    }
  }
  if (!p.wpart) return;
  // the groups' sums, in group order, one vector column at a time
  if constexpr (GROUPS > 1) {
    __shared__ float part[GROUPS][TPR * kVec];
    constexpr int kAtOnce = GROUPS > 8 ? 2 : GROUPS;  // (32 groups at once would take 229 registers)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kVec; ++e) part[grp][e * TPR + t] = gw[i][e];
      __syncthreads();
      if (grp == 0) {
#pragma unroll kAtOnce
        for (int k = 1; k < GROUPS; ++k)
#pragma unroll
          for (int e = 0; e < kVec; ++e) gw[i][e] += part[k][e * TPR + t];
      }
    }
    if (grp != 0) return;
  }
  float* out = p.wpart + (int64_t)blockIdx.x * p.cols;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * kVec, n = min(kVec, p.cols - c);
    if (n > 0) store8<kF32>(out + c, gw[i], n);
  }
}

// grad_weight[c] = sum over the blocks' partial rows, in a fixed order: 32
// columns per block, 8 row groups, then the groups in order.
constexpr int kWgCols = 32, kWgGroups = 8;
__global__ __launch_bounds__(kWgCols* kWgGroups) void wgrad_kernel(const float* part, int blocks, int cols, void* gw,
                                                                   int gw_f32) {
  __shared__ float sums[kWgGroups][kWgCols];
  const int j = threadIdx.x % kWgCols, g = threadIdx.x / kWgCols;
  const int c = blockIdx.x * kWgCols + j;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int b = g; b < blocks; b += kWgGroups) s += part[(int64_t)b * cols + c];
  }
  sums[g][j] = s;
  __syncthreads();
  if (g == 0 && c < cols) {
#pragma unroll
    for (int k = 1; k < kWgGroups; ++k) s += sums[k][j];
    if (gw_f32)
      ((float*)gw)[c] = s;
    else
      ((uint16_t*)gw)[c] = bf16_rne(s);
  }
}

// out = q * scale, 16 values per thread
template <int OD>
__global__ __launch_bounds__(256) void dequant_kernel(const int8_t* q, int64_t ldq, const float* scale,
                                                      typename Elem<OD>::type* out, int64_t ldo, int rows, int cols) {
  const int per_row = (cols + 15) / 16;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = id / per_row;
  if (row >= rows) return;
  const int c = (int)(id - row * per_row) * 16;
  const u32x4 u = *(const u32x4*)(q + row * ldq + c);
  const float s = scale[row];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int n = min(kVec, cols - c - half * kVec);
    f32x8 v;
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      v[e] = (float)((int)(u[half * 2 + (e >> 2)] << (24 - 8 * (e & 3))) >> 24) * s;
    if (n > 0) store8<OD>(out + row * ldo + c + half * kVec, v, n);
  }
}

// ---------------------------------------------------------------------------
namespace {

constexpr int kMaxBlocks = 1 << 22;  // of one launch: a grid holds fewer than 2^32 threads

// p without its first `rows` rows
template <int XD, int RD>
NormParams rows_from(NormParams p, int rows) {
  typedef typename Elem<XD>::type TX;
  typedef typename Elem<RD>::type TR;
  p.rows -= rows;
  p.x = (const TX*)p.x + rows * p.ldx;
  if (p.res) p.res = (const TR*)p.res + rows * p.ldr;
  if (p.h) p.h = (TR*)p.h + rows * p.ldh;
  if (p.y) p.y = (TX*)p.y + rows * p.ldy;
  if (p.rstd) p.rstd += rows;
  if (p.q) p.q += rows * p.ldq;
  if (p.scale) p.scale += rows;
  return p;
}

template <int MODE, int XD, int RD, int TPR, int NV>
hipError_t launch_fwd_rows(NormParams p, hipStream_t stream) {
  constexpr int kRows = TPR > 256 ? 1 : 256 / TPR;
  for (;;) {
    const int left = p.rows - kMaxBlocks * kRows;
    if (left > 0) p.rows = kMaxBlocks * kRows;
    hipLaunchKernelGGL((norm_kernel<MODE, XD, RD, TPR, NV>), dim3((unsigned)((p.rows + kRows - 1) / kRows)),
                       dim3(TPR > 256 ? TPR : 256), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || left <= 0) return e;
    p = rows_from<XD, RD>(p, p.rows);
    p.rows = left;
  }
}

template <int MODE, int XD, int RD>
hipError_t launch_fwd_t(const NormParams& p, hipStream_t stream) {
  const int vecs = (p.cols + kVec - 1) / kVec;
#define HARP_NORM_LAUNCH(TPR, NV) return launch_fwd_rows<MODE, XD, RD, TPR, NV>(p, stream);
  if (vecs <= 16) HARP_NORM_LAUNCH(16, 1)
  if (vecs <= 64) HARP_NORM_LAUNCH(64, 1)
  if (vecs <= 128) HARP_NORM_LAUNCH(64, 2)
  if (vecs <= 256) HARP_NORM_LAUNCH(256, 1)
  if (vecs <= 512) HARP_NORM_LAUNCH(256, 2)
  if (vecs <= 1024) HARP_NORM_LAUNCH(256, 4)
  if (vecs <= 2048) HARP_NORM_LAUNCH(512, 4)
  HARP_NORM_LAUNCH(512, 8)
#undef HARP_NORM_LAUNCH
}

template <int MODE>
hipError_t launch_fwd(const NormParams& p, hipStream_t stream) {
  if (MODE == kModeQuant || !p.res) {
    if (p.x_dtype == kBf16) return launch_fwd_t<MODE, kBf16, kNone>(p, stream);
    return launch_fwd_t<MODE, kF32, kNone>(p, stream);
  }
  if constexpr (MODE != kModeQuant) {
    if (p.x_dtype == kBf16)
      return p.r_dtype == kBf16 ? launch_fwd_t<MODE, kBf16, kBf16>(p, stream)
                                : launch_fwd_t<MODE, kBf16, kF32>(p, stream);
    return p.r_dtype == kBf16 ? launch_fwd_t<MODE, kF32, kBf16>(p, stream)
                              : launch_fwd_t<MODE, kF32, kF32>(p, stream);
  }
  return hipErrorInvalidValue;
}

// The backward's block by the row's vectors: TPR threads with NV vectors each for
// one row, GROUPS rows at a time.  The grid, the partial rows of the workspace and
// the kernel's instance all come from here.
template <int TPR_, int NV_, int GROUPS_>
struct BwdShape {
  static constexpr int TPR = TPR_, NV = NV_, GROUPS = GROUPS_;
};
template <class F>
auto with_bwd_shape(int cols, F f) {
  const int vecs = (cols + kVec - 1) / kVec;
  if (vecs <= 16) return f(BwdShape<16, 1, 32>());
  if (vecs <= 64) return f(BwdShape<64, 1, 8>());
  if (vecs <= 128) return f(BwdShape<64, 2, 8>());
  if (vecs <= 256) return f(BwdShape<256, 1, 2>());
  if (vecs <= 512) return f(BwdShape<256, 2, 2>());
  if (vecs <= 1024) return f(BwdShape<256, 4, 2>());
  if (vecs <= 2048) return f(BwdShape<512, 4, 1>());
  return f(BwdShape<1024, 4, 1>());
}

template <int XD, int HD>
hipError_t launch_bwd_t(const NormBwdParams& p, hipStream_t stream) {
  const unsigned blocks = (unsigned)bwd_blocks(p.rows, p.cols);
  return with_bwd_shape(p.cols, [&](auto s) {
    typedef decltype(s) S;
    hipLaunchKernelGGL((norm_bwd_kernel<XD, HD, S::TPR, S::NV, S::GROUPS, (S::NV * S::TPR <= 2048)>), dim3(blocks),
                       dim3(S::TPR * S::GROUPS), 0, stream, p);
    return hipGetLastError();
  });
}

}  // namespace

int bwd_blocks(int rows, int cols) {
  const int g = with_bwd_shape(cols, [](auto s) { return decltype(s)::GROUPS; });
  const int64_t need = ((int64_t)rows + g - 1) / g;
  return (int)(need < 512 ? need : 512);
}

hipError_t launch_norm(const NormParams& p, hipStream_t stream) { return launch_fwd<kModeNorm>(p, stream); }
hipError_t launch_norm_rows8(const NormParams& p, hipStream_t stream) { return launch_fwd<kModeNorm8>(p, stream); }
hipError_t launch_quantize(const NormParams& p, hipStream_t stream) { return launch_fwd<kModeQuant>(p, stream); }

hipError_t launch_norm_backward(const NormBwdParams& p, hipStream_t stream) {
  if (p.x_dtype == kBf16)
    return p.h_dtype == kBf16 ? launch_bwd_t<kBf16, kBf16>(p, stream) : launch_bwd_t<kBf16, kF32>(p, stream);
  return p.h_dtype == kBf16 ? launch_bwd_t<kF32, kBf16>(p, stream) : launch_bwd_t<kF32, kF32>(p, stream);
}

hipError_t launch_wgrad(const float* wpart, int blocks, int cols, void* gw, int gw_f32, hipStream_t stream) {
  hipLaunchKernelGGL(wgrad_kernel, dim3((unsigned)((cols + kWgCols - 1) / kWgCols)), dim3(kWgCols * kWgGroups), 0,
                     stream, wpart, blocks, cols, gw, gw_f32);
  return hipGetLastError();
}

hipError_t launch_dequantize(const int8_t* q, int64_t ldq, const float* scale, void* out, int64_t ldo, int o_dtype,
                             int rows, int cols, hipStream_t stream) {
  const int64_t per_row = (cols + 15) / 16;
  const int64_t most = (int64_t)kMaxBlocks * 256 / per_row;  // rows of one launch (cols < 2^31: at least 7)
  for (int64_t r0 = 0; r0 < rows; r0 += most) {
    const int n = (int)(rows - r0 < most ? rows - r0 : most);
    const dim3 grid((unsigned)((n * per_row + 255) / 256));
    if (o_dtype == kF32)
      hipLaunchKernelGGL((dequant_kernel<kF32>), grid, dim3(256), 0, stream, q + r0 * ldq, ldq, scale + r0,
                         (float*)out + r0 * ldo, ldo, n, cols);
    else
      hipLaunchKernelGGL((dequant_kernel<kBf16>), grid, dim3(256), 0, stream, q + r0 * ldq, ldq, scale + r0,
                         (uint16_t*)out + r0 * ldo, ldo, n, cols);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace harp_blk
