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
using harp_ra::kOOB;
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
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2u __attribute__((aligned(2)));

constexpr int kFeat = 128;       // features of one head
constexpr int kGroupOrder = 4;   // feature tiles per group of the block order
constexpr int kLds8Bytes = 144 * 1024;

// 32 x 32 x 32: lane L holds row L % 32 of A and of B with the same 16 values
// of k, picked by L / 32; C as every 32 x 32 product (ra_common.h)
__device__ __forceinline__ i32x16 mfma32x32x32(i32x4 a, i32x4 b, i32x16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
}

// Tile layout: rows of KT bytes in chunks of 16; chunk c of row r sits at a
// position that differs from c by a few of r's bits, so that the 16 lanes of a
// fragment read that are served together (rows r0 .. r0 + 15 at one chunk)
// touch every 16-byte bank group of the 256-byte bank line once.
template <int KT>
__device__ __forceinline__ int tile_pos(int r, int c) {
  static_assert(KT == 256 || KT == 128 || KT == 64, "row bytes");
  return KT == 256 ? c ^ (r & 15) : KT == 128 ? c ^ ((r >> 1) & 7) : c ^ ((r >> 2) & 3);
}

// Source byte offset (within the tile's rows) of 16-byte LDS slot `slot`.
template <int KT>
__device__ __forceinline__ uint32_t slot_src(int slot, int64_t ld) {
  const int r = slot / (KT / 16);
  return (uint32_t)(r * ld + tile_pos<KT>(r, slot % (KT / 16)) * 16);
}

__device__ __forceinline__ float bits_f32(uint32_t b) { return __uint_as_float(b); }
__device__ __forceinline__ uint32_t bf16_rne(float f) { return __builtin_bit_cast(uint16_t, (bf16)f); }
__device__ __forceinline__ float vec_at(const void* v, int f32, int64_t i) {
  return f32 ? ((const float*)v)[i] : bits_f32((uint32_t)((const uint16_t*)v)[i] << 16);
}

// 16 bytes at byte offset off of a buffer (zeros past its end)
__device__ __forceinline__ i32x4 buffer_load16(rsrc_t r, uint32_t off) {
  const uint64_t a = (uint64_t)r.x | ((uint64_t)r.y << 32);
  const auto b = __builtin_amdgcn_make_buffer_rsrc((void*)a, 0, r.z, r.w);
  return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, 0));
}

// byte mask of dword i of a 16-byte chunk whose first n (0 .. 16) bytes count
__device__ __forceinline__ uint32_t dword_mask(int n, int i) {
  const int b = n - 4 * i;
  return b >= 4 ? 0xffffffffu : (b <= 0 ? 0u : (1u << (8 * b)) - 1u);
}

template <int FB, int NJ>
struct Frags {
  i32x4 a[FB];  // w rows: 32 features each
  i32x4 b[NJ];  // x rows: 32 tokens each
};

// v_permlane32_swap on two dwords: afterwards x holds (x of lanes 0 .. 31, y
// of lanes 0 .. 31) and y (x of lanes 32 .. 63, y of lanes 32 .. 63)
__device__ __forceinline__ void swap_halves(uint32_t& x, uint32_t& y) {
  const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  x = r[0];
  y = r[1];
}

// Chunks q and q + 1 (features 8 q .. 8 q + 15) of a lane's token: each half
// of the wave holds 4 of a chunk's 8 features; they exchange, and lane half 0
// has chunk q, half 1 chunk q + 1, as bf16.
__device__ __forceinline__ u32x4 pack_chunks(const f32x4& a, const f32x4& b) {
  uint32_t u[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    u[h] = bf16_rne(a[2 * h]) | (bf16_rne(a[2 * h + 1]) << 16);
    u[2 + h] = bf16_rne(b[2 * h]) | (bf16_rne(b[2 * h + 1]) << 16);
  }
  swap_halves(u[0], u[2]);
  swap_halves(u[1], u[3]);
  return u32x4{u[0], u[1], u[2], u[3]};
}

// The end of a token block: sums of OF feature blocks for this lane's token mj
// (features fw + 32 i + 8 q + 4 ge + e, e < 4) become results and are stored.
// wsc, wb: the scales, and bias or norm weight, from feature fw on; a norm's
// results are bf16.
template <int OF, bool NORM, class Combine>
__device__ __forceinline__ void finish_tokens(const Prod8Params& p, const Prod8Out& o, const i32x16 (&own)[OF],
                                              float sx, const float* wsc, const float* wb, int d_own, int fw, int mj,
                                              int ge, Combine combine) {
  const bool norm = NORM && o.norm_w != nullptr, rope = norm && p.freqs != nullptr;
  f32x4 v[OF][4];
  float sq[OF];  // sums of the squares of each feature block
#pragma unroll
  for (int i = 0; i < OF; ++i) {
    sched_fence();  // (one feature block's scales at a time: all would not fit beside the sums)
    sq[i] = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 ws = *(const f32x4*)(wsc + 32 * i + 8 * q + 4 * ge);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[i][q][e] = (float)own[i][4 * q + e] * sx * ws[e];
        if (NORM) sq[i] = __builtin_fmaf(v[i][q][e], v[i][q][e], sq[i]);
      }
      if (!NORM) {
        const f32x4 b = *(const f32x4*)(wb + 32 * i + 8 * q + 4 * ge);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][q][e] += b[e];
      }
      // (opaque, or the arithmetic would sink to the stores, behind their bounds tests, and its operands stay)
      if (!NORM) asm volatile("" : "+v"(v[i][q]));
    }
  }
  sched_fence();
  if (NORM && norm) {
    // the head's sum, of its four feature blocks' sums (this lane's features and its partner lane's) taken in pairs:
    // the same order in every kind, so that a token's result does not depend on the kind its call runs in
#pragma unroll
    for (int i = 0; i < OF; ++i) sq[i] = harp_ra::wave_half_sum(sq[i]);
    static_assert(OF == 1 || OF == 2 || OF == 4, "pairs of feature blocks");
    float ss = sq[0];
    if constexpr (OF > 1) ss += sq[1];
    if constexpr (OF > 2) ss += sq[2] + sq[3];
    ss = combine(ss);
    const float rho = __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(ss, (float)kFeat) + o.eps));
    const int mt = min(mj, p.M - 1) + p.m_base;  // the token among the call's
    const float* fr = p.freqs + (int64_t)(mt / p.S) * p.f_stride_b + (int64_t)(mt % p.S) * p.f_stride_s + d_own + 4 * ge;
    constexpr int kPart = OF > 1 ? 2 : 1;  // feature blocks whose row of the table is loaded at once
#pragma unroll
    for (int i0 = 0; i0 < OF; i0 += kPart) {
      f32x4 fq[kPart][4];
      if (rope) {
#pragma unroll
        for (int i = 0; i < kPart; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) fq[i][q] = *(const f32x4*)(fr + 32 * (i0 + i) + 8 * q);
      }
#pragma unroll
      for (int i = i0; i < i0 + kPart; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 w = *(const f32x4*)(wb + 32 * i + 8 * q + 4 * ge);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[i][q][e] = v[i][q][e] * rho * w[e];
        }
      if (rope) {
#pragma unroll
        for (int i = 0; i < kPart; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const f32x4 f = fq[i][q];
              const float a = v[i0 + i][q][e], b = v[i0 + i][q][e + 1];
              v[i0 + i][q][e] = __builtin_fmaf(-b, f[e + 1], a * f[e]);
              v[i0 + i][q][e + 1] = __builtin_fmaf(a, f[e + 1], b * f[e]);
            }
      }
    }
  }
  // stores: 16 bytes per lane, 32 in a row of y.  (The lane's half is opaque
  // at each guarded store, or every store's bounds tests would be formed ahead
  // and kept in SGPRs.)
  int gs = ge;
  if (NORM || !o.y_f32) {
#pragma unroll
    for (int i = 0; i < OF; ++i)
#pragma unroll
      for (int q = 0; q < 4; q += 2) {
        const u32x4 w = pack_chunks(v[i][q], v[i][q + 1]);
        asm volatile("" : "+v"(gs));
        const int n = fw + 32 * i + 8 * (q + gs);
        uint16_t* dst = (uint16_t*)o.y + (int64_t)mj * o.ldy + n;
        if (mj < p.M) {
          if (n + 8 <= p.N) {
            *(u32x4u*)dst = w;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (n + e < p.N) dst[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
          }
        }
      }
  } else {
#pragma unroll
    for (int i = 0; i < OF; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        asm volatile("" : "+v"(gs));
        const int n = fw + 32 * i + 8 * q + 4 * gs;
        float* dst = (float*)o.y + (int64_t)mj * o.ldy + n;
        if (mj < p.M) {
          if (n + 4 <= p.N) {
            *(f32x4u*)dst = v[i][q];
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n + e < p.N) dst[e] = v[i][q][e];
          }
        }
      }
  }
}

}  // namespace

// Tile kernel.  C^T = W x^T, so a lane holds one token and 16 features per
// accumulator.  A wave covers FB x NJ blocks of 32 features by 32 tokens; a
// block is GROUPS x FB x 32 features by TG x NJ x 32 tokens, each part covered
// by KG waves that share the k-steps of a tile and add their sums at the end.
// K-tiles of KT bytes a row are copied global -> LDS by buffer_load ... lds,
// STAGES of them in flight, one barrier per tile in its last k-step; fragment
// reads run on across tile boundaries.
// Rows past the last token or feature and bytes past the descriptors' ends
// load zeros; the last tile's bytes past K are cleared in the w tile, which
// makes whatever x holds there count for nothing.
template <int FB, int NJ, int TG, int GROUPS, int KG, int KT, int STAGES, bool NORM>
__global__ __launch_bounds__(64 * TG * GROUPS * KG, 1) void prod8_kernel(Prod8Params p) {
  constexpr int kWaves = TG * GROUPS * KG;
  constexpr int kThreads = 64 * kWaves;
  constexpr int kWaveFeat = 32 * FB, TPW = 32 * NJ;
  constexpr int kFeatures = GROUPS * kWaveFeat;
  constexpr int kWBytes = kFeatures * KT;
  constexpr int kWPerWave = kWBytes / 1024 / kWaves;
  constexpr int kTok = TG * TPW;
  constexpr int kXBytes = kTok * KT;
  constexpr int kXPerWave = kXBytes / 1024 / kWaves;
  constexpr int kDmaPerWave = kXPerWave + kWPerWave;
  constexpr int kMfma = FB * NJ;
  constexpr int kOwn = KT / 32 / KG;  // k-steps of a wave in a tile
  constexpr int kRing = STAGES * (kXBytes + kWBytes);
  static_assert(kXBytes % (1024 * kWaves) == 0 && kWBytes % (1024 * kWaves) == 0, "copies split evenly");
  static_assert(kRing <= kLds8Bytes, "LDS budget");
  static_assert(kOwn * KG * 32 == KT && (kOwn % 2 == 0 || STAGES % 2 == 0), "whole k-steps; fragments in turn");
  // what a wave finishes of the sums it shares: whole token blocks where there
  // is one for each (a head stays in one wave), else feature blocks of one
  // (with fewer blocks than waves, the last waves have none)
  constexpr int kOwnJ = NJ % KG == 0 ? NJ / KG : 1, kOwnF = FB * NJ >= KG ? FB * NJ / KG / kOwnJ : 1;
  static_assert((kOwnJ * kOwnF * KG == FB * NJ || FB * NJ < KG) && FB % kOwnF == 0, "equal shares");
  constexpr int kParts = kFeat / 32 / kOwnF;  // waves that finish a head's token block between them (norm)
  static_assert(!NORM || kFeatures % kFeat == 0, "whole heads");
  static_assert(KG == 1 || kWaves * FB * NJ * 4096 <= kRing, "the sums fit the stages");
  __shared__ __attribute__((aligned(16))) char lds[kRing];
  __shared__ float wsc[kFeatures], wbias[kFeatures];  // feature scales; bias, or the norm's weight
  __shared__ float part_ss[NORM ? kParts : 1][NORM ? kFeatures / kFeat : 1][NORM ? kTok : 1];
  auto Xs = [&](int s) { return lds + s * kXBytes; };
  auto Ws = [&](int s) { return lds + STAGES * kXBytes + s * kWBytes; };

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, g = lane >> 5;
  const int kg = wave % KG, hh = wave / KG % GROUPS, tg = wave / KG / GROUPS;

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
  for (int k = 0; k < kXPerWave; ++k) xsrc[k] = slot_src<KT>((wave + kWaves * k) * 64 + lane, p.ldx);
#pragma unroll
  for (int k = 0; k < kWPerWave; ++k) wsrc[k] = slot_src<KT>((wave + kWaves * k) * 64 + lane, o.ldw);
  const int nt = (p.K + KT - 1) / KT;
  const int k_last = p.K - (nt - 1) * KT;  // bytes of the last tile, 1 .. KT
  // descriptors of tile t's rows; past the last tile they are empty (the
  // copies then write zeros and read nothing)
  auto x_rsrc = [&](int t) {
    const int k0 = t * KT;
    return make_rsrc(xb + (t < nt ? k0 : 0), t < nt ? x_bytes - (uint32_t)k0 : 0u);
  };
  auto w_rsrc = [&](int t) {
    const int k0 = t * KT;
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
  // clear the bytes past K of the last w tile, in stage s
  auto clear_tail = [&](int s) {
    constexpr int kChunks = KT / 16;
#pragma unroll 1
    for (int id = tid; id < kFeatures * kChunks; id += kThreads) {
      const int r = id / kChunks, c = id % kChunks, n = k_last - 16 * c;
      if (n < 16) {
        u32x4* q = (u32x4*)(Ws(s) + r * KT + (tile_pos<KT>(r, c) << 4));
        u32x4 v = *q;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] &= dword_mask(n, i);
        *q = v;
      }
    }
  };

  // lane part of the fragments' LDS offsets: the wave's k-steps kg kOwn ..
  int foff[kOwn];
#pragma unroll
  for (int ks = 0; ks < kOwn; ++ks) foff[ks] = l32 * KT + (tile_pos<KT>(l32, 2 * (kg * kOwn + ks) + g) << 4);
  auto load = [&](int s, int ks) {
    Frags<FB, NJ> f;
    const char* xs = Xs(s) + tg * TPW * KT + foff[ks];
    const char* ws = Ws(s) + hh * kWaveFeat * KT + foff[ks];
#pragma unroll
    for (int j = 0; j < NJ; ++j) f.b[j] = *(const i32x4*)(xs + 32 * j * KT);
#pragma unroll
    for (int i = 0; i < FB; ++i) f.a[i] = *(const i32x4*)(ws + 32 * i * KT);
    return f;
  };

  i32x16 acc[FB][NJ];
#pragma unroll
  for (int i = 0; i < FB; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
  auto mma = [&](const Frags<FB, NJ>& f, bool copy, const rsrc_t& xr, const rsrc_t& wr, int s) {
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
  static_assert(kThreads >= kFeatures, "a thread per feature");
  // what the wave finishes (see the epilogue), and its tokens' scales
  const int i_own = kOwnF == FB ? 0 : kg / NJ * kOwnF, j_own = kOwnF == FB ? kg * kOwnJ : kg % NJ;
  const int f_own = hh * kWaveFeat + 32 * i_own, m_own = m0 + TPW * tg + 32 * j_own;
  float sx[kOwnJ];
#pragma unroll
  for (int j = 0; j < kOwnJ; ++j) sx[j] = p.x_scale[min(m_own + 32 * j + l32, p.M - 1)];

#pragma unroll
  for (int t = 0; t < STAGES; ++t) {
    const rsrc_t xr = x_rsrc(t), wr = w_rsrc(t);
#pragma unroll
    for (int j = 0; j < kDmaPerWave; ++j) dma(lds_wave, xr, wr, t, j);
  }
  wait_lds_loads_but<(STAGES - 1) * kDmaPerWave>();
  __syncthreads();
  if (nt == 1 && k_last < KT) {
    clear_tail(0);
    __syncthreads();
  }
  Frags<FB, NJ> f[2];
  f[0] = load(0, 0);

  // After the last tile the fragment reads of "tile t + 1" read a stale
  // stage and the copies of "tile t + STAGES" are empty: both stay in bounds
  // and their results are never used.
  auto tile = [&](int S, int t) {  // stage S, a constant of the unrolled loop below
    const int S1 = (S + 1) % STAGES;
    const int P = kOwn % 2 ? S & 1 : 0;  // the fragments of the tile's first k-step
#pragma unroll
    for (int ks = 0; ks + 1 < kOwn; ++ks) {
      f[(P + ks + 1) & 1] = load(S, ks + 1);
      sched_fence();
      mma(f[(P + ks) & 1], false, {}, {}, S);
      sched_fence();
    }
    // every wave has its last fragments of tile t, and tile t + 1 is
    // complete: only the copies of tiles t + 2 .. t + STAGES - 1 are younger
    wait_lds_loads_but<(STAGES - 2) * kDmaPerWave>();
    __syncthreads();
    if (t + 2 == nt && k_last < KT) {
      clear_tail(S1);
      __syncthreads();
    }
    const rsrc_t xr = x_rsrc(t + STAGES), wr = w_rsrc(t + STAGES);
    f[(P + kOwn) & 1] = load(S1, 0);
    sched_fence();
    mma(f[(P + kOwn - 1) & 1], true, xr, wr, S);
    sched_fence();
  };
#pragma unroll 1
  for (int t = 0; t < nt; t += STAGES) {
#pragma unroll
    for (int S = 0; S < STAGES; ++S)
      if (t + S < nt) tile(S, t + S);
  }
  // no copy may still write the LDS when the stages become staging rows
  wait_lds_loads();
  if (tid < kFeatures) {
    wsc[tid] = r_sc;
    wbias[tid] = r_b;
  }
  __syncthreads();

  // the KG waves of a sum put theirs into LDS, and each adds up its share
  i32x16 own[kOwnF][kOwnJ];
  if constexpr (KG > 1) {
    i32x4* const sums = (i32x4*)lds + lane;  // [wave][FB][NJ][4] x 64 lanes
#pragma unroll
    for (int i = 0; i < FB; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          sums[((((wave * FB) + i) * NJ + j) * 4 + q) * 64] =
              i32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kOwnF; ++i)
#pragma unroll
      for (int j = 0; j < kOwnJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const i32x4* s0 = sums + (((((wave - kg) * FB) + i_own + i) * NJ + j_own + j) * 4 + q) * 64;
          i32x4 v = s0[0];
#pragma unroll
          for (int k = 1; k < KG; ++k) v += s0[k * FB * NJ * 4 * 64];
#pragma unroll
          for (int e = 0; e < 4; ++e) own[i][j][4 * q + e] = v[e];
        }
  } else {
#pragma unroll
    for (int i = 0; i < kOwnF; ++i)
#pragma unroll
      for (int j = 0; j < kOwnJ; ++j) own[i][j] = acc[i][j];
  }

  // ---- epilogue: this lane holds tokens m_own + 32 j + l32 and features
  // f_own + 32 i + 8 q + 4 g + e of the block's, e < 4
  const int fw = n0 + f_own;
  // (with a norm every wave stays for the exchange; those past the last head store nothing)
  if ((!NORM && fw >= p.N) || (FB * NJ < KG && kg >= FB * NJ)) return;
  const int lane_e = harp_ra::lane_id_fresh(), l32e = lane_e & 31, ge = lane_e >> 5;
#pragma unroll
  for (int j = 0; j < kOwnJ; ++j) {
    i32x16 col[kOwnF];
#pragma unroll
    for (int i = 0; i < kOwnF; ++i) col[i] = own[i][j];
    finish_tokens<kOwnF, NORM>(p, o, col, sx[j], wsc + f_own, wbias + f_own, f_own % kFeat, fw, m_own + 32 * j + l32e,
                               ge, [&](float ss) {
                                 if constexpr (NORM && kParts > 1) {
                                   const int t = m_own - m0 + 32 * j + l32e, h = f_own / kFeat;
                                   part_ss[f_own % kFeat / (32 * kOwnF)][h][t] = ss;
                                   __syncthreads();
                                   static_assert(kParts == 2 || kParts == 4, "pairs of parts");
                                   ss = part_ss[0][h][t] + part_ss[1][h][t];
                                   if constexpr (kParts > 2) ss += part_ss[2][h][t] + part_ss[3][h][t];
                                 }
                                 return ss;
                               });
  }
}

// Few-token kernel, up to 16 tokens.  A block is 16 features and splits the
// contraction over 4 waves, which read their operands from global memory
// straight into the fragments of v_mfma_i32_16x16x64_i8 (each byte of w is
// used once, so LDS would only add a stop), 4 chunks of 128 bytes a row in
// flight.  The waves' sums are added in LDS.  Bound by the first bytes' way and
// then by HBM: one token x 3840 features of 3840 bytes takes 5.6 us, 10240
// features (39 MB) 10.8 us with the weights out of HBM, 4.9 and 9.7 with them in
// the caches.  The same with 32 tokens (two x fragments to each of w) takes
// 20.1 us at 32 x 3840 x 10240, where the 32 x 32 blocks take 18.0.
constexpr int kFewWaves = 4, kFewChunks = 4;
__global__ __launch_bounds__(64 * kFewWaves) void few8_kernel(Prod8Params p) {
  __shared__ i32x4 red[kFewWaves][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const Prod8Out o = blockIdx.y == 0 ? p.out[0] : (blockIdx.y == 1 ? p.out[1] : p.out[2]);
  const int n0 = (int)blockIdx.x * 16;
  const int rows_w = min(16, p.N - n0);
  const int k16 = (p.K + 15) & ~15;
  // rows past the last feature or token, and chunks past K, read as zeros
  const rsrc_t wr = make_rsrc(o.w + (int64_t)n0 * o.ldw, (uint32_t)((rows_w - 1) * o.ldw + k16));
  const rsrc_t xr = make_rsrc(p.x, (uint32_t)((p.M - 1) * p.ldx + k16));
  const uint32_t woff = l16 < rows_w ? (uint32_t)(l16 * o.ldw) : kOOB;
  const uint32_t xoff = l16 < p.M ? (uint32_t)(l16 * p.ldx) : kOOB;

  // the scales and bias of the result that this thread may finish come in
  // with the first operands: token l16, features n0 + 4 g + e
  float ws[4], bs[4], sx = 0.f;
  if (wave == 0) {
    sx = p.x_scale[min(l16, p.M - 1)];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = min(n0 + 4 * g + e, p.N - 1);
      ws[e] = o.w_scale[n];
      bs[e] = o.bias ? vec_at(o.bias, o.bias_f32, n) : 0.f;
    }
  }

  i32x4 acc = {0, 0, 0, 0};
  const int chunks = (p.K + 127) / 128, part = p.K & 15;
#pragma unroll 1
  for (int c0 = wave; c0 < chunks; c0 += kFewWaves * kFewChunks) {
    i32x4 a[kFewChunks][2], b[kFewChunks][2];
#pragma unroll
    for (int u = 0; u < kFewChunks; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int kk = (c0 + kFewWaves * u) * 128 + 64 * h + 16 * g;
        a[u][h] = buffer_load16(wr, kk < p.K ? woff + kk : kOOB);
        b[u][h] = buffer_load16(xr, kk < p.K ? xoff + kk : kOOB);
      }
#pragma unroll
    for (int u = 0; u < kFewChunks; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (part) {  // the chunk that ends inside 16 bytes: w's bytes past K count for nothing
          const int left = p.K - ((c0 + kFewWaves * u) * 128 + 64 * h + 16 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) a[u][h][i] &= dword_mask(left, i);
        }
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u][h], b[u][h], acc, 0, 0, 0);
      }
  }
  red[wave][lane] = acc;
  __syncthreads();
  if (wave != 0 || l16 >= p.M) return;
#pragma unroll
  for (int w = 1; w < kFewWaves; ++w) acc += red[w][lane];
  const int n = n0 + 4 * g;
  f32x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (float)acc[e] * sx * ws[e] + bs[e];
  if (o.y_f32) {
    float* dst = (float*)o.y + (int64_t)l16 * o.ldy + n;
    if (n + 4 <= p.N) {
      *(f32x4u*)dst = y;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.N) dst[e] = y[e];
    }
  } else {
    uint16_t* dst = (uint16_t*)o.y + (int64_t)l16 * o.ldy + n;
    if (n + 4 <= p.N) {
      *(u32x2u*)dst = u32x2{bf16_rne(y[0]) | (bf16_rne(y[1]) << 16), bf16_rne(y[2]) | (bf16_rne(y[3]) << 16)};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.N) dst[e] = (uint16_t)bf16_rne(y[e]);
    }
  }
}

namespace {

// Compute units of the current device (cached per device).
int device_cus() {
  static int cached[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (!cached[dev]) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess) cached[dev] = n;
  }
  return cached[dev] > 0 ? cached[dev] : 256;
}

template <int FB, int NJ, int TG, int GROUPS, int KG, int KT, int STAGES>
hipError_t launch_tiles(const Prod8Params& p, bool norm, hipStream_t stream) {
  constexpr int kTok = TG * NJ * 32, kFeatures = GROUPS * FB * 32;
  const int64_t blocks = (int64_t)((p.M + kTok - 1) / kTok) * ((p.N + kFeatures - 1) / kFeatures);
  const dim3 grid((unsigned)blocks, (unsigned)p.n_outs), block(64 * TG * GROUPS * KG);
  if constexpr (kFeatures % kFeat == 0)
    if (norm) {
      hipLaunchKernelGGL((prod8_kernel<FB, NJ, TG, GROUPS, KG, KT, STAGES, true>), grid, block, 0, stream, p);
      return hipGetLastError();
    }
  if (norm) return hipErrorInvalidValue;  // blocks without whole heads
  hipLaunchKernelGGL((prod8_kernel<FB, NJ, TG, GROUPS, KG, KT, STAGES, false>), grid, block, 0, stream, p);
  return hipGetLastError();
}

// p without its first `rows` tokens
Prod8Params rows_from(Prod8Params p, int rows) {
  p.M -= rows;
  p.m_base += rows;
  p.x += (int64_t)rows * p.ldx;
  p.x_scale += rows;
  for (int i = 0; i < p.n_outs; ++i)
    p.out[i].y = (char*)p.out[i].y + (int64_t)rows * p.out[i].ldy * (p.out[i].y_f32 ? 4 : 2);
  return p;
}

hipError_t launch_few(const Prod8Params& p, bool, hipStream_t stream) {
  hipLaunchKernelGGL(few8_kernel, dim3((unsigned)((p.N + 15) / 16), (unsigned)p.n_outs), dim3(64 * kFewWaves), 0,
                     stream, p);
  return hipGetLastError();
}

// The kinds of blocks and what they were measured to take (weights out of
// HBM): one round of the CUs takes base + per_tile microseconds for each 128
// bytes of K, a further round `more` and the tiles again.  At K = 3840: 32
// tokens x 32 features 8 us, 64 x 64 13, 128 x 128 22, 256 x 256 50 a round;
// 8192 tokens x 10240 features (5 rounds of the largest) take 290 us, in 128 x
// 128 blocks 384 and in 64 x 64 519.  What bounds them: the small ones the
// latency of a block's start, first bytes and end (their `base`), then 64
// bytes per clock and CU into the LDS; the large ones the board's power (the
// 256 x 256 blocks keep the matrix pipes 57% busy at 1.85 of 2.4 GHz; the
// copies into LDS cost a fifth of the rate, LDS reads 6%, the stores of the
// results, whether or not anything runs beside them, a tenth).
struct Kind {
  int tokens, features;
  bool heads;        // takes a norm: whole heads
  int max_tokens;    // of the call
  double base, per_tile, more;
  int per_cu;
  hipError_t (*launch)(const Prod8Params&, bool, hipStream_t);
};
constexpr int kAny = 0x7fffffff;
constexpr int64_t kMaxBlocks = 1 << 22;  // of one launch: a grid holds fewer than 2^32 threads
const Kind kKinds[] = {
    {16, 16, false, 16, 3.4, 0.11, 0.0, 2, launch_few},
    {32, 32, false, kAny, 3.6, 0.15, 0.0, 2, launch_tiles<1, 1, 1, 1, 4, 256, 4>},
    {32, 64, false, kAny, 4.0, 0.21, 0.0, 1, launch_tiles<2, 1, 1, 1, 2, 256, 4>},
    {64, 64, false, kAny, 4.0, 0.30, 0.0, 2, launch_tiles<2, 2, 1, 1, 4, 128, 4>},
    {32, 128, true, kAny, 5.0, 0.34, 0.0, 1, launch_tiles<4, 1, 1, 1, 4, 256, 3>},
    {64, 128, true, kAny, 5.5, 0.40, 1.0, 1, launch_tiles<4, 2, 1, 1, 4, 256, 3>},
    {128, 128, true, kAny, 6.0, 0.54, 4.0, 1, launch_tiles<2, 2, 2, 2, 2, 128, 4>},
    {128, 256, true, kAny, 7.5, 0.80, 8.0, 1, launch_tiles<2, 2, 2, 4, 1, 128, 3>},
    {256, 256, true, kAny, 11.0, 1.33, 15.0, 1, launch_tiles<2, 4, 2, 4, 1, 128, 2>},
};
constexpr int kNumKinds = sizeof(kKinds) / sizeof(kKinds[0]);

double kind_us(const Kind& k, const Prod8Params& p, int64_t rows, int cus) {
  const int64_t blocks = (int64_t)p.n_outs * ((p.N + k.features - 1) / k.features) * ((rows + k.tokens - 1) / k.tokens);
  const double tiles = (double)((p.K + kKTile8 - 1) / kKTile8);
  // blocks that share a CU run out one by one, larger ones round by round
  const double rounds = k.per_cu > 1 ? (blocks > cus ? (double)blocks / cus + 0.25 : 1.0) : (double)((blocks + cus - 1) / cus);
  return k.base + rounds * k.per_tile * tiles + (rounds - 1) * k.more;
}

bool takes(const Kind& k, const Prod8Params& p, bool norm, int64_t rows) {
  const int64_t tiles = (int64_t)((p.N + k.features - 1) / k.features) * ((rows + k.tokens - 1) / k.tokens);
  return (!norm || k.heads) && rows <= k.max_tokens && tiles <= kMaxBlocks;
}

// index of the kind with the smallest time, or -1
int best_kind(const Prod8Params& p, bool norm, int64_t rows, int cus, double* us) {
  int best = -1;
  for (int i = 0; i < kNumKinds; ++i) {
    if (!takes(kKinds[i], p, norm, rows)) continue;
    const double t = kind_us(kKinds[i], p, rows, cus);
    if (best < 0 || t < *us) {
      best = i;
      *us = t;
    }
  }
  return best;
}

// The launches of a call: kind of the first rows, and of the rest (-1: none).
struct Plan {
  int first = -1, rest = -1, rows = 0;
};

// The kind with the smallest time for the call; where a kind's last round
// would be part full, its whole rounds may run as one launch and the rows left
// as another of a smaller kind (2 us between the two): 2048 tokens x 10240 of
// 3840 take 91 us instead of 97, 5000 x 3840 79 instead of 94.  Blocks of the
// same kind start as others end, so a second launch of them only adds a stop
// (q, k, v of 8192 tokens: 372 us instead of 363).  Over 133 shapes from 1 to
// 8192 tokens the kind chosen for a whole call takes 0.4% more than the best.
Plan plan_of(const Prod8Params& p, bool norm, int cus) {
  double us = 0;
  Plan plan;
  plan.first = best_kind(p, norm, p.M, cus, &us);
  plan.rows = p.M;
  for (int i = 0; i < kNumKinds; ++i) {
    const Kind& k = kKinds[i];
    if (!takes(k, p, norm, 1) || k.per_cu > 1) continue;
    const int64_t per_row_tile = (int64_t)p.n_outs * ((p.N + k.features - 1) / k.features);
    const int64_t blocks = per_row_tile * ((p.M + k.tokens - 1) / k.tokens);
    const int64_t rows = blocks / cus * cus / per_row_tile * k.tokens;
    if (rows < 1 || rows >= p.M || !takes(k, p, norm, rows)) continue;
    double t2 = 0;
    const int r = best_kind(p, norm, p.M - rows, cus, &t2);
    if (r < 0 || r == i) continue;  // the same kind: no gain
    const double t = kind_us(k, p, rows, cus) + 2.0 + t2;
    if (plan.first < 0 || t < us) {
      us = t;
      plan = {i, r, (int)rows};
    }
  }
  return plan;
}

bool has_norm(const Prod8Params& p) {
  bool norm = false;
  for (int i = 0; i < p.n_outs; ++i) norm |= p.out[i].norm_w != nullptr;
  return norm;
}

}  // namespace

hipError_t launch_prod8(const Prod8Params& p, hipStream_t stream) {
  const bool norm = has_norm(p);
  const Plan plan = plan_of(p, norm, device_cus());
  if (plan.first < 0) return hipErrorInvalidConfiguration;
  Prod8Params a = p;
  a.M = plan.rows;
  const hipError_t e = kKinds[plan.first].launch(a, norm, stream);
  if (e != hipSuccess || plan.rest < 0) return e;
  return kKinds[plan.rest].launch(rows_from(p, plan.rows), norm, stream);
}

}  // namespace harp_blk

// Used by the tests, which have to reach every kind: what a product of M x N x
// K (n_outs of them) runs as.  out: tokens and features of the first launch's
// blocks, its rows, tokens and features of the second's (0: none); kinds: the
// table's (tokens, features, whole heads), `room` entries at most.  cus 0: the
// current device's.  Returns the number of kinds, or -1 for a call that none takes.
extern "C" __attribute__((visibility("default"))) int harp_prod8_plan(int M, int N, int K, int n_outs, int norm,
                                                                      int cus, int* out, int* kinds, int room) {
  using namespace harp_blk;
  Prod8Params p{};
  p.M = M;
  p.N = N;
  p.K = K;
  p.n_outs = n_outs;
  const Plan plan = plan_of(p, norm != 0, cus > 0 ? cus : device_cus());
  if (plan.first < 0) return -1;
  const Kind &a = kKinds[plan.first], *b = plan.rest < 0 ? nullptr : &kKinds[plan.rest];
  const int v[5] = {a.tokens, a.features, plan.rows, b ? b->tokens : 0, b ? b->features : 0};
  for (int i = 0; i < 5; ++i) out[i] = v[i];
  for (int i = 0; i < kNumKinds && i < room; ++i) {
    kinds[3 * i] = kKinds[i].tokens;
    kinds[3 * i + 1] = kKinds[i].features;
    kinds[3 * i + 2] = kKinds[i].heads;
  }
  return kNumKinds;
}
