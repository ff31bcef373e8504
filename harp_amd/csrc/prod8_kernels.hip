// gfx950 kernels for the products of 8-bit rows: Linear layers whose weights
// and activations are 8-bit integers with one scale for each token (a) and
// one for each output feature (t):
//   y[m][n] = (sum_k x[m][k] w[n][k]) * a[m] * t[n] + b[n]
// and the q/k/v producer on them, which finishes each head of 128 features
// (QK RMSNorm, then RoPE) before its only store.
//
// The sums are exact: products of two 8-bit values add up in 32-bit integers,
// and K <= 2^16 terms of at most 2^14 stay below 2^31.  So the order of the
// contraction is free, nothing depends on how it is split, and the first
// rounding is the conversion of a sum to fp32.  The scales, the bias, the
// norm and the rotation are fp32; the result is rounded once, to nearest.
#include "blk_kernels.h"
#include "ra_common.h"

namespace harp_blk {

using harp_ra::bf16;
using harp_ra::f32x4;
using harp_ra::f32x4u;
using harp_ra::lds_dma_b128;
using harp_ra::lds_void;
using harp_ra::make_rsrc;
using harp_ra::rsrc_t;
using harp_ra::sched_fence;
using harp_ra::wait_lds_loads;
using harp_ra::wait_lds_loads_but;

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4u __attribute__((aligned(2)));

constexpr int kTokenGroups = 4;       // waves per feature group of a block, along the tokens
constexpr int kFeat = 128;            // features of one wave (one head)
constexpr int kRowBytes = kKTile8;    // 128: one row of a tile
constexpr int kGroupOrder = 4;        // feature tiles per group of the block order
constexpr int kLds8Bytes = 144 * 1024;

template <int I>
struct Int {
  static constexpr int value = I;
  constexpr operator int() const { return I; }
};

// 32 x 32 x 32: lane L holds row L % 32 of A and of B with the same 16 values
// of k, picked by L / 32; C as every 32 x 32 product (ra_common.h)
__device__ __forceinline__ i32x16 mfma32x32x32(i32x4 a, i32x4 b, i32x16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
}

// Tile layout: rows of 128 bytes = 8 chunks of 16; chunk c of row r sits at
// position c ^ ((r >> 1) & 7), so that the 16 lanes of a fragment read that
// are served together (rows r0 .. r0 + 15 at one chunk) touch every 16-byte
// bank group of the 256-byte bank line once.
__device__ __forceinline__ int tile_pos(int r, int c) { return c ^ ((r >> 1) & 7); }

// Source byte offset (within the tile's rows) of 16-byte LDS slot `slot`.
__device__ __forceinline__ uint32_t slot_src(int slot, int64_t ld) {
  const int r = slot >> 3;
  return (uint32_t)(r * ld + tile_pos(r, slot & 7) * 16);
}

__device__ __forceinline__ float bits_f32(uint32_t b) { return __uint_as_float(b); }
__device__ __forceinline__ uint32_t bf16_rne(float f) { return __builtin_bit_cast(uint16_t, (bf16)f); }
__device__ __forceinline__ float vec_at(const void* v, int f32, int64_t i) {
  return f32 ? ((const float*)v)[i] : bits_f32((uint32_t)((const uint16_t*)v)[i] << 16);
}

// byte mask of dword i of a 16-byte chunk whose first n (0 .. 16) bytes count
__device__ __forceinline__ uint32_t dword_mask(int n, int i) {
  const int b = n - 4 * i;
  return b >= 4 ? 0xffffffffu : (b <= 0 ? 0u : (1u << (8 * b)) - 1u);
}

template <int NJ>
struct Frags {
  i32x4 a[4];   // w rows: 32 features each
  i32x4 b[NJ];  // x rows: 32 tokens each
};

}  // namespace

// Tile kernel.  C^T = W x^T, so a lane holds one token and 16 features per
// accumulator.  A block is 4 x GROUPS waves and covers GROUPS x 128 features
// by 4 x TPW tokens; a wave 128 features by TPW tokens (4 x TPW / 32
// accumulators of 32 x 32).  K-tiles of 128 bytes a row are copied global ->
// LDS by buffer_load ... lds, STAGES of them in flight, one barrier per tile
// in its last k-step; fragment reads run on across tile boundaries.
// Rows past the last token or feature and bytes past the descriptors' ends
// load zeros; the last tile's bytes past K are cleared in the w tile, which
// makes whatever x holds there count for nothing.
template <int TPW, int GROUPS, int STAGES, bool NORM>
__global__ __launch_bounds__(64 * kTokenGroups * GROUPS, 1) void prod8_kernel(Prod8Params p) {
  constexpr int kWaves = kTokenGroups * GROUPS;
  constexpr int kThreads = 64 * kWaves;
  constexpr int kFeatures = GROUPS * kFeat;
  constexpr int kWBytes = kFeatures * kRowBytes;
  constexpr int kWPerWave = kWBytes / 1024 / kWaves;
  constexpr int NJ = TPW / 32;
  constexpr int kTok = kTokenGroups * TPW;
  constexpr int kXBytes = kTok * kRowBytes;
  constexpr int kXPerWave = kXBytes / 1024 / kWaves;
  constexpr int kDmaPerWave = kXPerWave + kWPerWave;
  constexpr int kMfma = 4 * NJ;
  constexpr int kRing = STAGES * (kXBytes + kWBytes);
  static_assert(kXBytes % (1024 * kWaves) == 0 && kWBytes % (1024 * kWaves) == 0, "copies split evenly");
  static_assert(kRing <= kLds8Bytes, "LDS budget");
  static_assert(kWaves * 32 * kFeat * 4 <= kRing, "a wave's staging of 32 fp32 rows fits the stages");
  __shared__ __attribute__((aligned(16))) char lds[kRing];
  __shared__ float wsc[kFeatures], wbias[kFeatures];  // feature scales; bias, or the norm's weight
  auto Xs = [&](int s) { return lds + s * kXBytes; };
  auto Ws = [&](int s) { return lds + STAGES * kXBytes + s * kWBytes; };

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, g = lane >> 5;
  const int hh = wave % GROUPS, tg = wave / GROUPS;

  // block -> (token tile, feature tile): each XCD (workgroups are dealt to
  // them round-robin) gets a contiguous range of an order that walks groups
  // of 4 feature tiles, within a group the token tiles, within a token tile
  // the group's feature tiles
  const int n_ft = (p.N + kFeatures - 1) / kFeatures, n_mt = (p.M + kTok - 1) / kTok;
  const int total = n_ft * n_mt, bid = (int)blockIdx.x;
  const int lin = (bid % 8) * (total / 8) + min(bid % 8, total % 8) + bid / 8;
  const int grp = lin / (n_mt * kGroupOrder), gs = min(kGroupOrder, n_ft - grp * kGroupOrder);
  const int rem = lin - grp * n_mt * kGroupOrder;
  const int mt = rem / gs, ft = grp * kGroupOrder + rem % gs;
  // (constant indices: a kernel-argument array indexed at run time would be
  // copied to scratch memory)
  const Prod8Out o = blockIdx.y == 0 ? p.out[0] : (blockIdx.y == 1 ? p.out[1] : p.out[2]);
  const int m0 = mt * kTok, n0 = ft * kFeatures;
  const int rows_x = min(kTok, p.M - m0), rows_w = min(kFeatures, p.N - n0);
  const int8_t* xb = p.x + (int64_t)m0 * p.ldx;
  const int8_t* wb = o.w + (int64_t)n0 * o.ldw;
  const int k16 = (p.K + 15) & ~15;
  const uint32_t x_bytes = (uint32_t)((rows_x - 1) * p.ldx + k16);
  const uint32_t w_bytes = (uint32_t)((rows_w - 1) * o.ldw + k16);

  uint32_t xsrc[kXPerWave], wsrc[kWPerWave];
#pragma unroll
  for (int k = 0; k < kXPerWave; ++k) xsrc[k] = slot_src((wave + kWaves * k) * 64 + lane, p.ldx);
#pragma unroll
  for (int k = 0; k < kWPerWave; ++k) wsrc[k] = slot_src((wave + kWaves * k) * 64 + lane, o.ldw);
  const int nt = (p.K + kKTile8 - 1) / kKTile8;
  const int k_last = p.K - (nt - 1) * kKTile8;  // bytes of the last tile, 1 .. 128
  // descriptors of tile t's rows; past the last tile they are empty (the
  // copies then write zeros and read nothing)
  auto x_rsrc = [&](int t) {
    const int k0 = t * kKTile8;
    return make_rsrc(xb + (t < nt ? k0 : 0), t < nt ? x_bytes - (uint32_t)k0 : 0u);
  };
  auto w_rsrc = [&](int t) {
    const int k0 = t * kKTile8;
    return make_rsrc(wb + (t < nt ? k0 : 0), t < nt ? w_bytes - (uint32_t)k0 : 0u);
  };
  const uint32_t lds_wave = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void*)(lds + wave * 1024));
  auto dma = [&](uint32_t base, const rsrc_t& xr, const rsrc_t& wr, int s, int j) {
    if (j < kXPerWave)
      lds_dma_b128(xr, base + s * kXBytes + kWaves * j * 1024, xsrc[j]);
    else
      lds_dma_b128(wr, base + STAGES * kXBytes + s * kWBytes + kWaves * (j - kXPerWave) * 1024,
                   wsrc[j - kXPerWave]);
  };
  // clear the bytes past K of the last w tile, in stage s (two threads a row)
  auto clear_tail = [&](int s) {
    static_assert(kThreads == 2 * kFeatures, "two threads per row of the w tile");
    const int r = tid >> 1;
#pragma unroll
    for (int c4 = 0; c4 < 4; ++c4) {
      const int c = 4 * (tid & 1) + c4, n = k_last - 16 * c;
      if (n < 16) {
        u32x4* q = (u32x4*)(Ws(s) + r * kRowBytes + (tile_pos(r, c) << 4));
        u32x4 v = *q;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] &= dword_mask(n, i);
        *q = v;
      }
    }
  };

  int foff[4];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) foff[ks] = l32 * kRowBytes + (tile_pos(l32, 2 * ks + g) << 4);
  auto load = [&](int s, int ks) {
    Frags<NJ> f;
    const char* xs = Xs(s) + tg * TPW * kRowBytes + foff[ks];
    const char* ws = Ws(s) + hh * kFeat * kRowBytes + foff[ks];
#pragma unroll
    for (int j = 0; j < NJ; ++j) f.b[j] = *(const i32x4*)(xs + 32 * j * kRowBytes);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.a[i] = *(const i32x4*)(ws + 32 * i * kRowBytes);
    return f;
  };

  i32x16 acc[4][NJ];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
  auto mma = [&](const Frags<NJ>& f, bool copy, const rsrc_t& xr, const rsrc_t& wr, int s) {
    // (opaque, or every stage's addresses would be kept in SGPRs over the loop)
    uint32_t base = lds_wave;
    asm volatile("" : "+s"(base));
#pragma unroll
    for (int u = 0; u < kMfma; ++u) {
      acc[u / NJ][u % NJ] = mfma32x32x32(f.a[u / NJ], f.b[u % NJ], acc[u / NJ][u % NJ]);
      if (copy) {
#pragma unroll
        for (int j = u * kDmaPerWave / kMfma; j < (u + 1) * kDmaPerWave / kMfma; ++j) dma(base, xr, wr, s, j);
      }
    }
  };

  // the features' scales and bias (or norm weight), loaded now and moved to
  // LDS after the main loop (older than every copy: the copy waits cover them)
  float r_sc = 0.f, r_b = 0.f;
  if (tid < kFeatures && n0 + tid < p.N) {
    r_sc = o.w_scale[n0 + tid];
    if (NORM) {
      if (o.norm_w) r_b = vec_at(o.norm_w, o.norm_w_f32, tid % kFeat);
    } else if (o.bias) {
      r_b = vec_at(o.bias, o.bias_f32, n0 + tid);
    }
  }

#pragma unroll
  for (int t = 0; t < STAGES; ++t) {
    const rsrc_t xr = x_rsrc(t), wr = w_rsrc(t);
#pragma unroll
    for (int j = 0; j < kDmaPerWave; ++j) dma(lds_wave, xr, wr, t, j);
  }
  wait_lds_loads_but<(STAGES - 1) * kDmaPerWave>();
  __syncthreads();
  if (nt == 1 && k_last < kKTile8) {
    clear_tail(0);
    __syncthreads();
  }
  Frags<NJ> f0 = load(0, 0), f1;

  // After the last tile the fragment reads of "tile t + 1" read a stale
  // stage and the copies of "tile t + STAGES" are empty: both stay in bounds
  // and their results are never used.
  auto tile = [&](auto SC, int t) {
    constexpr int S = decltype(SC)::value, S1 = (S + 1) % STAGES;
    f1 = load(S, 1);
    sched_fence();
    mma(f0, false, {}, {}, S);
    sched_fence();
    f0 = load(S, 2);
    sched_fence();
    mma(f1, false, {}, {}, S);
    sched_fence();
    f1 = load(S, 3);
    sched_fence();
    mma(f0, false, {}, {}, S);
    sched_fence();
    // every wave has its last fragments of tile t, and tile t + 1 is
    // complete: only the copies of tiles t + 2 .. t + STAGES - 1 are younger
    wait_lds_loads_but<(STAGES - 2) * kDmaPerWave>();
    __syncthreads();
    if (t + 2 == nt && k_last < kKTile8) {
      clear_tail(S1);
      __syncthreads();
    }
    const rsrc_t xr = x_rsrc(t + STAGES), wr = w_rsrc(t + STAGES);
    f0 = load(S1, 0);
    sched_fence();
    mma(f1, true, xr, wr, S);
    sched_fence();
  };
#pragma unroll 1
  for (int t = 0; t < nt; t += STAGES) {
    tile(Int<0>{}, t);
    if (t + 1 < nt) tile(Int<1>{}, t + 1);
    if constexpr (STAGES > 2) {
      if (t + 2 < nt) tile(Int<2>{}, t + 2);
    }
    if constexpr (STAGES > 3) {
      if (t + 3 < nt) tile(Int<3>{}, t + 3);
    }
  }
  // no copy may still write the LDS when the stages become staging rows
  wait_lds_loads();
  if (tid < kFeatures) {
    wsc[tid] = r_sc;
    wbias[tid] = r_b;
  }
  __syncthreads();

  // ---- epilogue: this lane holds tokens m0 + TPW tg + 32 j + l32 and
  // features 32 i + 8 q + 4 g + e of its wave's 128, e < 4
  const int fw = n0 + hh * kFeat;  // the wave's first feature
  if (fw >= p.N) return;
  const int lane_e = harp_ra::lane_id_fresh(), l32e = lane_e & 31, ge = lane_e >> 5;
  char* const stg = lds + wave * (32 * kFeat * 4);  // 32 rows of 256 or 512 bytes, one token block at a time
  const bool norm = NORM && o.norm_w != nullptr;
  const bool rope = norm && p.freqs != nullptr;

#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int mj = m0 + TPW * tg + 32 * j;  // the token block's first token
    const int m = min(mj + l32e, p.M - 1);
    const float sx = p.x_scale[m];
    f32x4 v[4][4];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int d0 = 32 * i + 8 * q + 4 * ge;
        const f32x4 ws = *(const f32x4*)(wsc + hh * kFeat + d0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[i][q][e] = (float)acc[i][j][4 * q + e] * sx * ws[e];
          if (NORM) ss = __builtin_fmaf(v[i][q][e], v[i][q][e], ss);
        }
        if (!NORM) {
          const f32x4 b = *(const f32x4*)(wbias + hh * kFeat + d0);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[i][q][e] += b[e];
        }
      }
    if (NORM && norm) {
      ss = harp_ra::wave_half_sum(ss);  // this lane's 64 features and its partner lane's
      const float rho = __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(ss, (float)kFeat) + o.eps));
      const float* fr = rope ? p.freqs + (int64_t)(m / p.S) * p.f_stride_b + (int64_t)(m % p.S) * p.f_stride_s : nullptr;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int d0 = 32 * i + 8 * q + 4 * ge;
          const f32x4 w = *(const f32x4*)(wbias + hh * kFeat + d0);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[i][q][e] = v[i][q][e] * rho * w[e];
          if (rope) {
            const f32x4 f = *(const f32x4*)(fr + d0);
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const float a = v[i][q][e], b = v[i][q][e + 1];
              v[i][q][e] = __builtin_fmaf(-b, f[e + 1], a * f[e]);
              v[i][q][e + 1] = __builtin_fmaf(a, f[e + 1], b * f[e]);
            }
          }
        }
    }
    // out through LDS: the wave's own rows (16-byte chunk c of row r at
    // position c ^ (r & 15)), then 16 bytes per lane along the rows; LDS
    // operations of one wave stay in order, so there is no barrier
    if (NORM || !o.y_f32) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *(uint2*)(stg + l32e * 256 + (((4 * i + q) ^ (l32e & 15)) << 4) + ge * 8) =
              make_uint2(bf16_rne(v[i][q][0]) | (bf16_rne(v[i][q][1]) << 16),
                         bf16_rne(v[i][q][2]) | (bf16_rne(v[i][q][3]) << 16));
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int r = 4 * k + (lane_e >> 4), c = lane_e & 15, n = fw + c * 8;
        const u32x4 u = *(const u32x4*)(stg + r * 256 + ((c ^ (r & 15)) << 4));
        uint16_t* dst = (uint16_t*)o.y + (int64_t)(mj + r) * o.ldy + n;
        if (mj + r < p.M) {
          if (n + 8 <= p.N) {
            *(u32x4u*)dst = u;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (n + e < p.N) dst[e] = (uint16_t)(u[e >> 1] >> (16 * (e & 1)));
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = 8 * i + 2 * q + ge;
          *(f32x4*)(stg + l32e * 512 + ((c ^ (l32e & 15)) << 4)) = v[i][q];
        }
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int r = 2 * k + (lane_e >> 5), c = lane_e & 31, n = fw + c * 4;
        const f32x4 u = *(const f32x4*)(stg + r * 512 + ((c ^ (r & 15)) << 4));
        float* dst = (float*)o.y + (int64_t)(mj + r) * o.ldy + n;
        if (mj + r < p.M) {
          if (n + 4 <= p.N) {
            *(f32x4u*)dst = u;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n + e < p.N) dst[e] = u[e];
          }
        }
      }
    }
  }
}

namespace {

template <int TPW, int GROUPS, int STAGES>
hipError_t launch_tiles(const Prod8Params& p, bool norm, hipStream_t stream) {
  constexpr int kTok = kTokenGroups * TPW, kFeatures = GROUPS * kFeat;
  const int64_t blocks = (int64_t)((p.M + kTok - 1) / kTok) * ((p.N + kFeatures - 1) / kFeatures);
  if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)blocks, (unsigned)p.n_outs), block(64 * kTokenGroups * GROUPS);
  if (norm)
    hipLaunchKernelGGL((prod8_kernel<TPW, GROUPS, STAGES, true>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((prod8_kernel<TPW, GROUPS, STAGES, false>), grid, block, 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_prod8(const Prod8Params& p, hipStream_t stream) {
  bool norm = false;
  for (int i = 0; i < p.n_outs; ++i) norm |= p.out[i].norm_w != nullptr;
  return launch_tiles<64, 2, 2>(p, norm, stream);
}

}  // namespace harp_blk
