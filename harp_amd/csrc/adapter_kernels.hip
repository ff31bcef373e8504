// gfx950 kernels of low-rank adapters beside a projection, for many requests
// at once: token m of request i takes adapter a = index[i],
//
//   t[m] = s_a x[m] A_a^T            (shrink: r sums over K)
//   y[m] = base[m] + t[m] B_a^T      (expand: N sums over r)
//   u[m] = s_a dy[m] B_a             (shrink of dy with B transposed)
//   dx[m] = u[m] A_a                 (expand of u with A transposed)
//   dA_a = sum_m u[m]^T x[m],  dB_a = sum_m dy[m]^T t[m]
//
// All sums are fp32.  t and u stay fp32 between the kernels; where expand
// multiplies them by bf16 on the matrix cores they are taken apart into two
// bf16 (three for an fp32 result) whose products are added in fp32: 2^-17 (2^-25)
// of a value is left out, far below the result's own rounding, and the
// second product costs nothing beside the memory these kernels wait for.
//
// Requests are ranges of tokens of any length, known on the device only.  A
// kernel that works in tiles of M tokens is launched with T / M + R + 2 slots;
// segment i (the tokens in front of the first request, each request, the tokens
// behind the last) starts at slot a_i / M + i, where its first token is a_i:
// floor(b / M) + i + 1 - (floor(a / M) + i) is never less than the ceil((b - a) / M)
// tiles it needs, so no tile is shared by two requests, nothing is counted
// beforehand, and a block finds its segment by one or two 64-way searches.
// What the arrays hold is clamped before it is used as an index.
#include <algorithm>

#include "ra_common.h"
#include "req_kernels.h"

namespace harp_req {

namespace {

using harp_ra::bf16;
using harp_ra::bf16x8;
using harp_ra::f32x16;
using harp_ra::f32x4;
using harp_ra::f32x4u;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4u __attribute__((aligned(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2u __attribute__((aligned(2)));

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------
// Which tokens, which adapter
// ---------------------------------------------------------------------------
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

// The largest i <= count + 1 whose segment starts at or before `slot`, M tokens a slot
template <int M>
__device__ __forceinline__ int segment_at(const Requests& q, int slot) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = q.count + 2;  // lo's start is <= slot; hi's is above, or hi is behind the last
  while (hi - lo > 1) {          // (uniform: hi - lo shrinks 64-fold)
    const int step = (hi - lo + 63) / 64;
    const int i = lo + lane * step;
    const bool at = i < hi && segment_start(q, i) / M + i <= slot;
    // the last lane of the leading run; lane 0 (lo itself) is in it
    const uint64_t b = __ballot(at) | 1;
    const int last = __ffsll((unsigned long long)~b) - 2;
    const int k = b == ~0ull ? 63 : last;
    hi = min(hi, lo + (k + 1) * step);
    lo = lo + k * step;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// A tile: rows first .. first + rows - 1 (rows <= M) with one adapter (-1: none)
struct Tile {
  int first, rows, adapter;
};
template <int M>
__device__ __forceinline__ Tile tile_at(const Requests& q, int slot) {
  const int i = segment_at<M>(q, slot);
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
int64_t slots_of(const Requests& q, int M) { return (int64_t)q.tokens / M + q.count + 2; }

// ---------------------------------------------------------------------------
// Fragments
// ---------------------------------------------------------------------------
// n (<= 8) bf16 at p, zeros behind them
__device__ __forceinline__ bf16x8 load_some(const bf16* p, int n) {
  bf16x8 v = harp_ra::zero8();
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) v[i] = p[i];
  return v;
}
__device__ __forceinline__ bf16x8 load_full(const bf16* p) { return __builtin_bit_cast(bf16x8, *(const u32x4u*)p); }

__device__ __forceinline__ float high_part(float f) { return (float)(bf16)f; }

}  // namespace

// ---------------------------------------------------------------------------
// Shrink.  A block takes a tile of 16 TB tokens and 16 RB ranks of one adapter;
// its WAVES waves take every WAVES-th 64 columns of K and their sums are added
// in LDS in the order of the waves.  v_mfma_f32_16x16x32_bf16 with A's rows as
// the first operand: a lane ends with four neighbouring ranks of one token.
// Fragments come straight from memory: a 64-column step reads whole 128-byte
// lines of x and of A, and nothing of x is used twice by a block.
// ---------------------------------------------------------------------------
template <int TB, int RB, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void shrink_kernel(ShrinkParams p) {
  constexpr int M = 16 * TB;
  __shared__ f32x4 sums[WAVES][TB * RB][64];
  const Tile tile = tile_at<M>(p.req, (int)blockIdx.x);
  if (tile.rows <= 0 || tile.adapter < 0) return;
  const int which = blockIdx.z, r0 = (int)blockIdx.y * 16 * RB;
  const ShrinkSet set = which == 0 ? p.set[0] : which == 1 ? p.set[1] : p.set[2];
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const bf16* xr[TB];
  const bf16* ar[RB];
  // rows behind the tile and ranks behind r repeat the last one; their sums are dropped
#pragma unroll
  for (int i = 0; i < TB; ++i)
    xr[i] = (const bf16*)p.x + (int64_t)(tile.first + min(16 * i + l16, tile.rows - 1)) * p.ldx + 8 * g;
#pragma unroll
  for (int j = 0; j < RB; ++j)
    ar[j] = (const bf16*)set.a + ((int64_t)tile.adapter * p.r + min(r0 + 16 * j + l16, p.r - 1)) * p.K + 8 * g;
  f32x4 acc[RB][TB];
#pragma unroll
  for (int j = 0; j < RB; ++j)
#pragma unroll
    for (int i = 0; i < TB; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int full = p.K / 64;
#pragma unroll 2
  for (int c = wave; c < full; c += WAVES) {
    bf16x8 xf[2][TB], af[2][RB];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < TB; ++i) xf[h][i] = load_full(xr[i] + c * 64 + 32 * h);
#pragma unroll
      for (int j = 0; j < RB; ++j) af[h][j] = load_full(ar[j] + c * 64 + 32 * h);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < RB; ++j)
#pragma unroll
        for (int i = 0; i < TB; ++i) acc[j][i] = harp_ra::mfma16x16x32(af[h][j], xf[h][i], acc[j][i]);
  }
  if (p.K % 64 && wave == full % WAVES) {  // the columns behind the last whole step
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = full * 64 + 32 * h, n = p.K - k - 8 * g;
      if (k < p.K) {
#pragma unroll
        for (int j = 0; j < RB; ++j) {
          const bf16x8 af = load_some(ar[j] + k, n);
#pragma unroll
          for (int i = 0; i < TB; ++i) acc[j][i] = harp_ra::mfma16x16x32(af, load_some(xr[i] + k, n), acc[j][i]);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < RB; ++j)
#pragma unroll
    for (int i = 0; i < TB; ++i) sums[wave][j * TB + i][lane] = acc[j][i];
  __syncthreads();
  const float scale = set.scale ? set.scale[tile.adapter] : 1.f;
  for (int e = threadIdx.x; e < TB * RB * 64; e += 64 * WAVES) {
    const int at = e >> 6, l = e & 63, j = at / TB, i = at % TB;
    f32x4 s = sums[0][at][l];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += sums[w][at][l];
    const int row = 16 * i + (l & 15), rank = r0 + 16 * j + 4 * (l >> 4);
    if (row >= tile.rows || rank >= p.rp) continue;
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] = rank + k < p.r ? s[k] * scale : 0.f;
    const int64_t m = tile.first + row;
    if (!p.pairs) {
      *(f32x4*)((float*)set.t + m * p.ldt + rank) = s;
    } else {
      bf16 hi[4], lo[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        hi[k] = (bf16)s[k];
        lo[k] = (bf16)(s[k] - (float)hi[k]);
      }
      bf16* t = (bf16*)set.t + m * p.ldt + rank;
      *(u32x2*)t = *(const u32x2*)hi;
      *(u32x2*)(t + p.rp) = *(const u32x2*)lo;
    }
  }
}

// ---------------------------------------------------------------------------
// Expand.  A wave takes 32 tokens and walks 64 features at a time:
// v_mfma_f32_32x32x16_bf16 with B's rows as the first operand, its row q of a
// 32-feature block reading feature 32 g + 16 block + r of the 64, so that a lane
// (token l % 32, half g) ends with 2 x 16 neighbouring features and the
// wave's base and out accesses are whole 128-byte lines of a row.  t's fragments
// stay in registers over the walk.
// ---------------------------------------------------------------------------
namespace {

// 16 (bf16: 32 bytes, fp32: 64 bytes) values of a row from column f on, columns below N
template <bool F32>
__device__ __forceinline__ void load16(const void* row, int f, int N, float (&v)[16]) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int c = f + 8 * q;
    if (c + 8 <= N) {
      if constexpr (F32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 u = *(const f32x4u*)((const float*)row + c + 4 * h);
#pragma unroll
          for (int k = 0; k < 4; ++k) v[8 * q + 4 * h + k] = u[k];
        }
      } else {
        const u32x4 u = *(const u32x4u*)((const bf16*)row + c);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[8 * q + 2 * k] = __uint_as_float(u[k] << 16);
          v[8 * q + 2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[8 * q + k] = 0.f;
        if (c + k < N) v[8 * q + k] = F32 ? ((const float*)row)[c + k] : (float)((const bf16*)row)[c + k];
      }
    }
  }
}
template <bool F32>
__device__ __forceinline__ void store16(void* row, int f, int N, const float (&v)[16]) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int c = f + 8 * q;
    if (c + 8 <= N) {
      if constexpr (F32) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *(f32x4u*)((float*)row + c + 4 * h) =
              f32x4{v[8 * q + 4 * h], v[8 * q + 4 * h + 1], v[8 * q + 4 * h + 2], v[8 * q + 4 * h + 3]};
      } else {
        bf16x8 o;
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = (bf16)v[8 * q + k];
        *(u32x4u*)((bf16*)row + c) = __builtin_bit_cast(u32x4, o);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c + k < N) {
          if constexpr (F32) ((float*)row)[c + k] = v[8 * q + k];
          else ((bf16*)row)[c + k] = (bf16)v[8 * q + k];
        }
    }
  }
}

}  // namespace

// RS: 16-rank steps (rp / 16); WT: waves of a block along the tokens (the other
// 4 / WT along the features); a block walks `span` features
template <bool F32, int RS, int WT>
__global__ __launch_bounds__(kThreads) void expand_kernel(ExpandParams p, int span) {
  constexpr int M = 32 * WT, WF = 4 / WT, PARTS = F32 ? 3 : 2;
  const Tile tile = tile_at<M>(p.req, (int)blockIdx.x);
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int row = 32 * (wave % WT) + l32;
  if (tile.rows <= 32 * (wave % WT)) return;
  const bool mine = row < tile.rows;
  const int64_t m = tile.first + (mine ? row : 0);
  const int f_end = min(p.N, ((int)blockIdx.y + 1) * span);
  constexpr int es = F32 ? 4 : 2;
  const char* const base = p.base ? (const char*)p.base + m * p.ld_base * es : nullptr;
  char* const out = (char*)p.out + m * p.ld_out * es;

  bf16x8 tf[RS][PARTS];
  if (tile.adapter >= 0) {
#pragma unroll
    for (int s = 0; s < RS; ++s) {
      const float* t = p.t + m * p.ldt + 16 * s + 8 * g;
      float v[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 u = *(const f32x4*)(t + 4 * h);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[4 * h + k] = u[k];
      }
#pragma unroll
      for (int part = 0; part < PARTS; ++part)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const bf16 b = (bf16)v[k];
          tf[s][part][k] = b;
          v[k] -= (float)b;
        }
    }
  }
  // the B row of operand row l32 in block q: feature 32 g' + 16 q + 4 a + b for l32 = 8 a + 4 g' + b
  const int feat = 32 * ((l32 >> 2) & 1) + 4 * (l32 >> 3) + (l32 & 3);
  const bool whole = p.r % 8 == 0;
  for (int f0 = (int)blockIdx.y * span + 64 * (wave / WT); f0 < f_end; f0 += 64 * WF) {
    float v[2][16];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (base) {
        load16<F32>(base, f0 + 32 * g + 16 * q, p.N, v[q]);
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) v[q][k] = 0.f;
      }
    }
    if (tile.adapter >= 0) {
      f32x16 acc[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const bf16* b = (const bf16*)p.b + ((int64_t)tile.adapter * p.N + min(f0 + feat + 16 * q, p.N - 1)) * p.r + 8 * g;
        acc[q] = harp_ra::zero16();
#pragma unroll
        for (int s = 0; s < RS; ++s) {
          const int n = p.r - 16 * s - 8 * g;  // ranks this lane has left: 8 or more but in the last step
          const bf16x8 bf = s < RS - 1 || n >= 8 ? load_full(b + 16 * s)
                            : whole              ? harp_ra::zero8()
                                                 : load_some(b + 16 * s, n);
#pragma unroll
          for (int part = 0; part < PARTS; ++part) acc[q] = harp_ra::mfma32x32x16(bf, tf[s][part], acc[q]);
        }
      }
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int k = 0; k < 16; ++k) v[q][k] += acc[q][k];
    }
    if (mine) {
#pragma unroll
      for (int q = 0; q < 2; ++q) store16<F32>(out, f0 + 32 * g + 16 * q, p.N, v[q]);
    }
  }
}

// ---------------------------------------------------------------------------
// Gradients of A and B: for each adapter the sum over its tokens of
// v[m]^T x[m], 16 RB ranks x 128 columns a block.  The WAVES waves take every
// WAVES-th four tokens; v_mfma_f32_16x16x4_f32 takes them as they lie in
// memory (a lane holds rank l % 16, or 8 columns 8 (l % 16) .., of token l / 16),
// so nothing is transposed and v keeps its 32 bits.  The waves' sums are
// added in LDS in order.  Where the blocks of all adapters would not fill the
// chip, each request's tokens are taken in `splits` parts whose sums a second
// kernel adds, in order too.
// ---------------------------------------------------------------------------
constexpr int kGradWaves = 8, kGradCols = 128;

template <int RB>
__global__ __launch_bounds__(64 * kGradWaves) void grad_kernel(GradParams p) {
  __shared__ f32x4 sums[kGradWaves][RB * 2][64];
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int c0_blocks = p.part[0].out ? (p.part[0].C + kGradCols - 1) / kGradCols : 0;
  const bool second = (int)blockIdx.x >= c0_blocks;
  const GradPart part = second ? p.part[1] : p.part[0];
  const int c0 = ((int)blockIdx.x - (second ? c0_blocks : 0)) * kGradCols;
  const int rgroups = (p.r + 16 * RB - 1) / (16 * RB);
  const int adapter = (int)blockIdx.y / rgroups, r0 = (int)blockIdx.y % rgroups * 16 * RB;
  const int split = blockIdx.z;
  const int col = c0 + 8 * l16;
  const int ncol = min(8, part.C - col);  // <= 0: no column of this lane

  f32x4 acc[RB][8];
#pragma unroll
  for (int j = 0; j < RB; ++j)
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[j][k] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int i0 = 0; i0 < p.req.count; i0 += 64) {
    const bool hit = i0 + lane < p.req.count && adapter_of(p.req, min(i0 + lane, p.req.count - 1)) == adapter;
    for (uint64_t todo = __ballot(hit); todo; todo &= todo - 1) {
      const int i = i0 + __ffsll((unsigned long long)todo) - 1;
      const int a = token_of(p.req, i), n = max(token_of(p.req, i + 1) - a, 0);
      const int begin = a + (int)((int64_t)n * split / p.splits), end = a + (int)((int64_t)n * (split + 1) / p.splits);
      for (int m0 = begin + 4 * wave; m0 < end; m0 += 4 * kGradWaves) {
        const int m = m0 + g;
        const bool in = m < end;
        bf16x8 xv = harp_ra::zero8();
        float vv[RB];
        if (in) {
          const bf16* x = (const bf16*)part.x + (int64_t)m * part.ldx + col;
          if (ncol == 8) xv = load_full(x);
          else if (ncol > 0) xv = load_some(x, ncol);
        }
#pragma unroll
        for (int j = 0; j < RB; ++j)
          vv[j] = in && r0 + 16 * j < p.rp ? part.v[(int64_t)m * part.ldv + r0 + 16 * j + l16] : 0.f;
#pragma unroll
        for (int j = 0; j < RB; ++j)
#pragma unroll
          for (int k = 0; k < 8; ++k)
            acc[j][k] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[j], (float)xv[k], acc[j][k], 0, 0, 0);
      }
    }
  }

  // columns 8 l16 + 2 h, + 1 of all waves at a time; a lane holds ranks 4 g .. + 3
#pragma unroll
  for (int h = 0; h < 4; ++h) {
#pragma unroll
    for (int j = 0; j < RB; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) sums[wave][2 * j + k][lane] = acc[j][2 * h + k];
    __syncthreads();
    for (int e = threadIdx.x; e < RB * 2 * 64; e += 64 * kGradWaves) {
      const int at = e >> 6, l = e & 63;
      f32x4 s = sums[0][at][l];
#pragma unroll
      for (int w = 1; w < kGradWaves; ++w) s += sums[w][at][l];
      const int c = c0 + 8 * (l & 15) + 2 * h + (at & 1), rank = r0 + 16 * (at >> 1) + 4 * (l >> 4);
      if (c >= part.C) continue;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (rank + k >= p.r) break;
        const int64_t o = part.cols_first ? ((int64_t)adapter * part.C + c) * p.r + rank + k
                                          : ((int64_t)adapter * p.r + rank + k) * part.C + c;
        if (p.splits == 1) ((bf16*)part.out)[o] = (bf16)s[k];
        else {
          const int64_t all = (int64_t)p.req.n * p.r * ((p.part[0].out ? p.part[0].C : 0) + (p.part[1].out ? p.part[1].C : 0));
          p.work[split * all + (second && p.part[0].out ? (int64_t)p.req.n * p.r * p.part[0].C : 0) + o] = s[k];
        }
      }
    }
    __syncthreads();
  }
}

__global__ __launch_bounds__(kThreads) void grad_sum_kernel(const float* work, int splits, int64_t n0, int64_t n1,
                                                            bf16* out0, bf16* out1) {
  const int64_t all = n0 + n1;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < all; i += (int64_t)gridDim.x * kThreads) {
    float s = work[i];
    for (int k = 1; k < splits; ++k) s += work[k * all + i];
    (i < n0 ? out0[i] : out1[i - n0]) = (bf16)s;
  }
}

// ---------------------------------------------------------------------------
// n matrices transposed, 64 x 64 values a block
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kThreads) void transpose_kernel(TransposeParams p, int tiles0) {
  __shared__ uint16_t t[64][65];
  const bool second = (int)blockIdx.x >= tiles0;
  const TransposePart part = second ? p.part[1] : p.part[0];
  const int across = (part.cols + 63) / 64;
  const int tile = (int)blockIdx.x - (second ? tiles0 : 0);
  const int r0 = tile / across * 64, c0 = tile % across * 64;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  for (int i = blockIdx.y; i < p.n; i += gridDim.y) {
    const uint16_t* src = (const uint16_t*)part.src + (int64_t)i * part.rows * part.cols;
    uint16_t* dst = (uint16_t*)part.dst + (int64_t)i * part.rows * part.cols;
    for (int y = ty; y < 64; y += 4)
      if (r0 + y < part.rows && c0 + tx < part.cols) t[y][tx] = src[(int64_t)(r0 + y) * part.cols + c0 + tx];
    __syncthreads();
    for (int y = ty; y < 64; y += 4)
      if (c0 + y < part.cols && r0 + tx < part.rows) dst[(int64_t)(c0 + y) * part.rows + r0 + tx] = t[tx][y];
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Launchers
// ---------------------------------------------------------------------------
namespace {
template <int TB, int RB, int WAVES>
hipError_t shrink_t(const ShrinkParams& p, hipStream_t st) {
  const dim3 grid((unsigned)slots_of(p.req, 16 * TB), (unsigned)((p.rp + 16 * RB - 1) / (16 * RB)), (unsigned)p.sets);
  hipLaunchKernelGGL((shrink_kernel<TB, RB, WAVES>), grid, dim3(64 * WAVES), 0, st, p);
  return hipGetLastError();
}
}  // namespace

hipError_t launch_shrink(const ShrinkParams& p, hipStream_t st) {
  // few tokens: 16 waves share a tile's K
  if (slots_of(p.req, 32) * p.sets < 512) return shrink_t<1, 1, 16>(p, st);
  return p.rp <= 16 ? shrink_t<2, 1, 4>(p, st) : p.rp <= 32 ? shrink_t<2, 2, 4>(p, st) : shrink_t<4, 4, 4>(p, st);
}

namespace {
template <bool F32, int RS, int WT>
hipError_t expand_t(const ExpandParams& p, hipStream_t st) {
  const int64_t slots = slots_of(p.req, 32 * WT);
  // enough blocks for the chip, in multiples of a block's 64-feature steps
  constexpr int step = 64 * (4 / WT);
  const int steps = (p.N + step - 1) / step;
  const int64_t want = std::max<int64_t>(1, 2048 / slots);
  const int each = (int)std::max<int64_t>(1, steps / std::min<int64_t>(want, steps));
  hipLaunchKernelGGL((expand_kernel<F32, RS, WT>), dim3((unsigned)slots, (unsigned)((steps + each - 1) / each)),
                     dim3(kThreads), 0, st, p, each * step);
  return hipGetLastError();
}
template <bool F32, int RS>
hipError_t expand_w(const ExpandParams& p, hipStream_t st) {
  // requests of 64 tokens and more on the average fill a block's waves along the tokens
  return p.req.tokens / std::max(p.req.count, 1) >= 64 ? expand_t<F32, RS, 4>(p, st) : expand_t<F32, RS, 1>(p, st);
}
template <bool F32>
hipError_t expand_r(const ExpandParams& p, hipStream_t st) {
  switch (p.rp / 16) {
    case 1: return expand_w<F32, 1>(p, st);
    case 2: return expand_w<F32, 2>(p, st);
    case 3: return expand_w<F32, 3>(p, st);
    case 4: return expand_w<F32, 4>(p, st);
    case 5: return expand_w<F32, 5>(p, st);
    case 6: return expand_w<F32, 6>(p, st);
    case 7: return expand_w<F32, 7>(p, st);
    default: return expand_w<F32, 8>(p, st);
  }
}
}  // namespace
hipError_t launch_expand(const ExpandParams& p, hipStream_t st) { return p.f32 ? expand_r<true>(p, st) : expand_r<false>(p, st); }

namespace {
int grad_ranks(const GradParams& p) { return p.rp <= 16 ? 1 : p.rp <= 32 ? 2 : 4; }  // RB
int grad_cols(const GradParams& p) {
  int n = 0;
  for (const GradPart& q : p.part) n += q.out ? (q.C + kGradCols - 1) / kGradCols : 0;
  return n;
}
template <int RB>
hipError_t grad_t(const GradParams& p, hipStream_t st) {
  const dim3 grid((unsigned)grad_cols(p), (unsigned)(p.req.n * ((p.r + 16 * RB - 1) / (16 * RB))), (unsigned)p.splits);
  hipLaunchKernelGGL((grad_kernel<RB>), grid, dim3(64 * kGradWaves), 0, st, p);
  return hipGetLastError();
}
}  // namespace
int grad_splits(const GradParams& p) {
  const int RB = grad_ranks(p);
  const int64_t blocks = (int64_t)grad_cols(p) * std::min(p.req.n, p.req.count) * ((p.r + 16 * RB - 1) / (16 * RB));
  if (!blocks) return 1;
  const int64_t want = (512 + blocks - 1) / blocks;                               // two blocks a CU
  const int64_t most = std::max<int64_t>(1, p.req.tokens / p.req.count / 128);    // of 128 tokens at least
  return (int)std::min(want, most);
}
hipError_t launch_adapter_grad(const GradParams& p, hipStream_t st) {
  const int RB = grad_ranks(p);
  const hipError_t e = RB == 1 ? grad_t<1>(p, st) : RB == 2 ? grad_t<2>(p, st) : grad_t<4>(p, st);
  if (e != hipSuccess || p.splits == 1) return e;
  const int64_t per = (int64_t)p.req.n * p.r;
  const int64_t n0 = p.part[0].out ? per * p.part[0].C : 0, n1 = p.part[1].out ? per * p.part[1].C : 0;
  const int64_t blocks = std::min<int64_t>((n0 + n1 + kThreads - 1) / kThreads, 4096);
  hipLaunchKernelGGL(grad_sum_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, st, (const float*)p.work, p.splits, n0,
                     n1, (bf16*)p.part[0].out, (bf16*)p.part[1].out);
  return hipGetLastError();
}

hipError_t launch_transpose(const TransposeParams& p, hipStream_t st) {
  auto tiles = [](const TransposePart& q) {
    return q.src ? (int64_t)((q.rows + 63) / 64) * ((q.cols + 63) / 64) : 0;
  };
  const int64_t t0 = tiles(p.part[0]), t1 = tiles(p.part[1]);
  hipLaunchKernelGGL(transpose_kernel, dim3((unsigned)(t0 + t1), (unsigned)std::min(p.n, 65535)), dim3(kThreads), 0, st,
                     p, (int)t0);
  return hipGetLastError();
}

}  // namespace harp_req
