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
// Which tokens a block works on: req_device.h.
#include <algorithm>
#include <type_traits>

#include "ra_common.h"
#include "req_device.h"
#include "req_kernels.h"
#include "rope_device.h"

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
constexpr int kCUs = 256;

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
// what the rounding b left of v; nothing behind an infinity, whose difference would be NaN
__device__ __forceinline__ float rest(float v, bf16 b) {
  constexpr float kMost = 0x1.fep127f;  // of bf16
  return __builtin_amdgcn_fmed3f(v, -kMost, kMost) - __builtin_amdgcn_fmed3f((float)b, -kMost, kMost);
}
__device__ __forceinline__ bf16x8 load_full(const bf16* p) { return __builtin_bit_cast(bf16x8, *(const u32x4u*)p); }

}  // namespace

namespace {
// t of a block's tile from its waves' sums: sum_of(wave, rank block * TB + token block, lane)
template <int TB, int RB, int WAVES, class F>
__device__ __forceinline__ void shrink_store(const ShrinkParams& p, const Tile& tile, int e0, int e_end, F sum_of) {
  const int per = p.rp / 16;
  for (int e = threadIdx.x; e < TB * RB * 64; e += 64 * WAVES) {
    const int at = e >> 6, l = e & 63, j = at / TB, i = at % TB;
    f32x4 s = sum_of(0, at, l);
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += sum_of(w, at, l);
    const int row = 16 * i + (l & 15);
    if (row >= tile.rows || e0 + j >= e_end) continue;
    const int which = (e0 + j) / per, rank = 16 * (e0 + j - which * per) + 4 * (l >> 4);
    const ShrinkSet set = which == 0 ? p.set[0] : which == 1 ? p.set[1] : p.set[2];
    const float scale = set.scale ? set.scale[tile.adapter] : 1.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] = rank + k < p.r ? s[k] * scale : 0.f;
    const int64_t m = tile.first + row;
    if (set.t) *(f32x4*)(set.t + m * p.ldt + rank) = s;
    if (set.pairs) {
      bf16 hi[4], lo[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        hi[k] = (bf16)s[k];
        lo[k] = (bf16)rest(s[k], hi[k]);
      }
      bf16* t = (bf16*)set.pairs + m * 2 * p.rp + rank;
      *(u32x2*)t = *(const u32x2*)hi;
      *(u32x2*)(t + p.rp) = *(const u32x2*)lo;
    }
  }
}
}  // namespace

// ---------------------------------------------------------------------------
// Shrink.  A block takes a tile of 16 TB tokens and RB blocks of 16 ranks (of the
// sets one after the other) of one adapter; its WAVES waves take every WAVES-th
// 64 columns of K and their sums are added in LDS in the order of the waves.
// v_mfma_f32_16x16x32_bf16 with A's rows as the first operand: a lane ends with
// four neighbouring ranks of one token.  Fragments come straight from memory: a
// 64-column step reads whole 128-byte lines of x and of A, and nothing of x is
// used twice by a block.  Bound by its start and the latency of its loads: 8 us for
// 1333 tokens x 2570 columns, rank 12, whose rows are 4-byte aligned.
// ---------------------------------------------------------------------------
template <int TB, int RB, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void shrink_kernel(ShrinkParams p) {
  constexpr int M = 16 * TB;
  __shared__ f32x4 sums[WAVES][TB * RB][64];
  const Tile tile = tile_at<M>(p.req, (int)blockIdx.x);
  if (tile.rows <= 0 || tile.adapter < 0) return;
  // this block's entries e0 .. e0 + RB - 1 (before e_end) of the sets' rank blocks; those of sets with an x of
  // their own are not shared
  const int per = p.rp / 16, groups = (per + RB - 1) / RB, own = (int)blockIdx.y / groups;
  const int e0 = p.apart ? own * per + ((int)blockIdx.y - own * groups) * RB : (int)blockIdx.y * RB;
  const int e_end = p.apart ? (own + 1) * per : per * p.sets;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  // (constant indices: a kernel-argument array indexed at run time would be copied to scratch memory)
  auto set_of = [&](int e) { return min(e, e_end - 1) / per; };
  auto a_of = [&](int i) { return (const bf16*)(i == 0 ? p.set[0].a : i == 1 ? p.set[1].a : p.set[2].a); };
  const int s0 = set_of(e0);
  const bf16* const x = (const bf16*)(s0 == 0 ? p.set[0].x : s0 == 1 ? p.set[1].x : p.set[2].x);
  const int64_t ldx = s0 == 0 ? p.set[0].ldx : s0 == 1 ? p.set[1].ldx : p.set[2].ldx;
  const bf16* xr[TB];
  const bf16* ar[RB];
  // rows behind the tile and ranks behind r repeat the last one; their sums are dropped
#pragma unroll
  for (int i = 0; i < TB; ++i) xr[i] = x + (int64_t)(tile.first + min(16 * i + l16, tile.rows - 1)) * ldx + 8 * g;
#pragma unroll
  for (int j = 0; j < RB; ++j) {
    const int set = set_of(e0 + j), rank = 16 * (min(e0 + j, e_end - 1) - set * per) + l16;
    ar[j] = a_of(set) + ((int64_t)tile.adapter * p.r + min(rank, p.r - 1)) * p.K + 8 * g;
  }
  f32x4 acc[RB][TB];
#pragma unroll
  for (int j = 0; j < RB; ++j)
#pragma unroll
    for (int i = 0; i < TB; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int full = p.K / 64;
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
  shrink_store<TB, RB, WAVES>(p, tile, e0, e_end, [&](int w, int at, int l) { return sums[w][at][l]; });
}

// The same where x's and A's rows are 16-byte aligned.  Fragments read straight
// from memory touch 16 rows with every 16 lanes, and the caches serve those one
// after the other; here each wave copies its 64 columns of the tile's rows to LDS
// (buffer_load ... lds, eight whole 128-byte lines an instruction) and reads the
// fragments from there.  A wave has STAGES such steps of its own, so the loop has
// no barrier: it waits for its oldest copies, reads, multiplies and sends the next
// copies into the same place.
// Bound by the read of x: 8192 tokens x 3840 columns, rank 32, 18 us (3.5 TB/s;
// 4.7 TB/s from one K to the next, and 6 us to start and end), 23.5 behind a kernel whose
// 168 MB of results are still on their way to memory.  Other waves, stages and LDS
// sizes of 96 KB and more came within 1 us of it.
// TABLE: the blocks behind the slots write the rotary table that the next launch reads.
template <bool TABLE>
struct TableArg {};
template <>
struct TableArg<true> {
  RopeTable v;
  int first;  // block
};
template <int TB, int RB, int WAVES, int STAGES, bool TABLE>
__global__ __launch_bounds__(64 * WAVES) void shrink_lds_kernel(ShrinkParams p, TableArg<TABLE> table) {
  if constexpr (TABLE) {
    if ((int)blockIdx.x >= table.first) {
      if (blockIdx.y == 0) table_share(table.v, (int)blockIdx.x - table.first, (int)gridDim.x - table.first, 64 * WAVES);
      return;
    }
  }
  constexpr int M = 16 * TB;
  constexpr int kCopies = 2 * (TB + RB);  // of 8 rows each, x's rows and then A's
  constexpr int kStage = 1024 * kCopies;  // bytes
  constexpr int kTiles = WAVES * STAGES * kStage, kSums = WAVES * TB * RB * 64 * 16;
  __shared__ __attribute__((aligned(16))) char lds[kTiles > kSums ? kTiles : kSums];
  const Tile tile = tile_at<M>(p.req, (int)blockIdx.x);
  if (tile.rows <= 0 || tile.adapter < 0) return;
  // this block's entries e0 .. e0 + RB - 1 (before e_end) of the sets' rank blocks; those of sets with an x of
  // their own are not shared
  const int per = p.rp / 16, groups = (per + RB - 1) / RB, own = (int)blockIdx.y / groups;
  const int e0 = p.apart ? own * per + ((int)blockIdx.y - own * groups) * RB : (int)blockIdx.y * RB;
  const int e_end = p.apart ? (own + 1) * per : per * p.sets;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int s0 = __builtin_amdgcn_readfirstlane(min(e0, e_end - 1) / per);
  const bf16* const x = (const bf16*)(s0 == 0 ? p.set[0].x : s0 == 1 ? p.set[1].x : p.set[2].x);
  const int64_t ldx = s0 == 0 ? p.set[0].ldx : s0 == 1 ? p.set[1].ldx : p.set[2].ldx;
  // copy j takes rows 8 j + lane / 8, the 16-byte chunk that sits at position lane % 8 of its row: chunk c of
  // row r at c ^ ((r >> 1) & 7), so that 16 rows' reads of one chunk hit every bank once
  const int row8 = lane >> 3, chunk = (lane & 7) ^ ((row8 >> 1) & 7);
  const harp_ra::rsrc_t xr =
      harp_ra::make_rsrc(x + (int64_t)tile.first * ldx, (uint32_t)(((int64_t)(tile.rows - 1) * ldx + p.K) * 2));
  uint32_t xsrc[2 * TB], asrc[2 * RB];
#pragma unroll
  for (int j = 0; j < 2 * TB; ++j) {
    const int r = 8 * j + row8;
    xsrc[j] = r < tile.rows ? (uint32_t)(r * ldx * 2 + (chunk ^ (4 * (j & 1))) * 16) : harp_ra::kOOB;
  }
  const bf16* ab[RB];
#pragma unroll
  for (int j = 0; j < RB; ++j) {
    const int e = min(e0 + j, e_end - 1), set = e / per;
    const void* a = set == 0 ? p.set[0].a : set == 1 ? p.set[1].a : p.set[2].a;
    ab[j] = (const bf16*)a + ((int64_t)tile.adapter * p.r + 16 * (e - set * per)) * p.K;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 8 * h + row8;
      asrc[2 * j + h] = 16 * (e - set * per) + r < p.r ? (uint32_t)(r * p.K * 2 + (chunk ^ (4 * h)) * 16) : harp_ra::kOOB;
    }
  }
  const uint32_t base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(harp_ra::lds_void*)lds) +
                        (uint32_t)(wave * STAGES * kStage);
  const char* const mine = lds + wave * STAGES * kStage;
  // the copies of columns 64 c .. 64 c + 63 into stage s; columns behind K are zeros (`live` false: all of them)
  auto copy = [&](int s, int c, bool live) {
    const int left = live ? p.K - 64 * c : 0;  // columns
#pragma unroll
    for (int j = 0; j < 2 * TB; ++j) {
      const bool in = 8 * (chunk ^ (4 * (j & 1))) < left;
      harp_ra::lds_dma_b128(xr, base + s * kStage + 1024 * j, in ? xsrc[j] + 128 * c : harp_ra::kOOB);
    }
#pragma unroll
    for (int j = 0; j < RB; ++j) {
      const harp_ra::rsrc_t arr = harp_ra::make_rsrc(ab[j], 16u * (uint32_t)p.K * 2u);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool in = 8 * (chunk ^ (4 * h)) < left;
        harp_ra::lds_dma_b128_fresh(arr, base + s * kStage + 1024 * (2 * TB + 2 * j + h),
                                    in ? asrc[2 * j + h] + 128 * c : harp_ra::kOOB);
      }
    }
  };
  f32x4 acc[RB][TB];
#pragma unroll
  for (int j = 0; j < RB; ++j)
#pragma unroll
    for (int i = 0; i < TB; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int steps = (p.K + 63) / 64;
#pragma unroll
  for (int s = 0; s < STAGES; ++s) copy(s, wave + WAVES * s, wave + WAVES * s < steps);
  auto step = [&](auto SC, int c) {
    constexpr int S = decltype(SC)::value;
    harp_ra::wait_lds_loads_but<(STAGES - 1) * kCopies>();
    bf16x8 xf[2][TB], af[2][RB];
    const char* const t = mine + S * kStage;
    auto frag = [&](int r, int h) {  // row r (16 of them in a block), columns 32 h + 8 g ..
      return *(const bf16x8*)(t + r * 128 + (((4 * h + g) ^ ((r >> 1) & 7)) << 4));
    };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < TB; ++i) xf[h][i] = frag(16 * i + l16, h);
#pragma unroll
      for (int j = 0; j < RB; ++j) af[h][j] = frag(16 * (TB + j) + l16, h);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < RB; ++j)
#pragma unroll
        for (int i = 0; i < TB; ++i) acc[j][i] = harp_ra::mfma16x16x32(af[h][j], xf[h][i], acc[j][i]);
    // the fragments are in registers: the stage is free
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    copy(S, c + STAGES * WAVES, c + STAGES * WAVES < steps);
  };
  for (int c = wave; c < steps; c += STAGES * WAVES) {
    step(std::integral_constant<int, 0>{}, c);
    if constexpr (STAGES > 1)
      if (c + WAVES < steps) step(std::integral_constant<int, 1>{}, c + WAVES);
    if constexpr (STAGES > 2)
      if (c + 2 * WAVES < steps) step(std::integral_constant<int, 2>{}, c + 2 * WAVES);
  }
  harp_ra::wait_lds_loads();  // (the empty copies too: the sums go over the stages)
  __syncthreads();
  f32x4* const sums = (f32x4*)lds;
#pragma unroll
  for (int j = 0; j < RB; ++j)
#pragma unroll
    for (int i = 0; i < TB; ++i) sums[(wave * TB * RB + j * TB + i) * 64 + lane] = acc[j][i];
  __syncthreads();
  shrink_store<TB, RB, WAVES>(p, tile, e0, e_end, [&](int w, int at, int l) { return sums[(w * TB * RB + at) * 64 + l]; });
}

// ---------------------------------------------------------------------------
// Expand.  A wave takes 32 tokens and walks 64 features at a time:
// v_mfma_f32_32x32x16_bf16 with B's rows as the first operand, so that a lane
// ends with runs of four features of one token.  Those go through the wave's
// 8 KB of LDS (16-byte chunk c of row r at c ^ (r % 16): no bank conflict either
// way), so that base is read and out written in whole 128-byte lines, 16 bytes a
// lane: straight from the accumulators' layout each access touched 64 rows'
// pieces and the kernel ran at half the rate.  t's fragments stay in registers
// over the walk.  Bound by base and out: 8192 tokens x 10240 features, rank 32, 336 MB in
// 70.5 us (4.8 TB/s); 3840 features, rank 64, 126 MB in 42 us, without a base 63 MB in 22.
// ---------------------------------------------------------------------------
namespace {

constexpr int kNoBase = 0, kBaseBf16 = 1, kBaseF32 = 2;

template <int E>
struct Run {
  float v[E];
};
// E values of a row from column c on as they are in memory, those below N
template <bool F32, int E>
struct RawRun {
  u32x4 u[E * (F32 ? 4 : 2) / 16];
};
template <bool F32, int E>
__device__ __forceinline__ RawRun<F32, E> load_run(const char* row, int c, int N) {
  constexpr int es = F32 ? 4 : 2, kWords = E * es / 16;
  RawRun<F32, E> r;
  if (c + E <= N) {
#pragma unroll
    for (int h = 0; h < kWords; ++h) r.u[h] = *(const u32x4u*)(row + (int64_t)c * es + 16 * h);
  } else {
    uint32_t w[4 * kWords] = {};
#pragma unroll
    for (int k = 0; k < E; ++k)
      if (c + k < N) {
        if constexpr (F32) w[k] = ((const uint32_t*)row)[c + k];
        else w[k / 2] |= (uint32_t)((const uint16_t*)row)[c + k] << (16 * (k & 1));
      }
#pragma unroll
    for (int h = 0; h < kWords; ++h) r.u[h] = u32x4{w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]};
  }
  return r;
}
template <bool F32, int E>
__device__ __forceinline__ Run<E> values(const RawRun<F32, E>& r) {
  Run<E> v;
#pragma unroll
  for (int k = 0; k < E; ++k) {
    if constexpr (F32) v.v[k] = __uint_as_float(r.u[k / 4][k % 4]);
    else v.v[k] = __uint_as_float((k & 1) ? r.u[k / 8][k / 2 % 4] & 0xffff0000u : r.u[k / 8][k / 2 % 4] << 16);
  }
  return v;
}
template <bool F32, int E>
__device__ __forceinline__ void store_run(char* row, int c, int N, const Run<E>& r) {
  if (c + E <= N) {
    if constexpr (F32) {
#pragma unroll
      for (int h = 0; h < E / 4; ++h)
        *(f32x4u*)((float*)row + c + 4 * h) = f32x4{r.v[4 * h], r.v[4 * h + 1], r.v[4 * h + 2], r.v[4 * h + 3]};
    } else {
      static_assert(E == 8);
      bf16x8 o;
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] = (bf16)r.v[k];
      *(u32x4u*)((bf16*)row + c) = __builtin_bit_cast(u32x4, o);
    }
  } else {
#pragma unroll
    for (int k = 0; k < E; ++k)
      if (c + k < N) {
        if constexpr (F32) ((float*)row)[c + k] = r.v[k];
        else ((bf16*)row)[c + k] = (bf16)r.v[k];
      }
  }
}

}  // namespace

namespace {

// What both kernels below share: a wave's 32 rows of a tile, its 8 KB of LDS
template <int BASE, bool F32, int RS>
struct Expand {
  static constexpr int PARTS = F32 ? 3 : 2;
  static constexpr int E = F32 ? 4 : 8;                   // features of a lane's access: 16 bytes of out
  static constexpr int kLanes = 64 / E, kPass = 32 / E;   // lanes of a row, passes over the 32 rows
  static constexpr int es = F32 ? 4 : 2, bs = BASE == kBaseF32 ? 4 : 2;
  typedef RawRun<BASE == kBaseF32, E> Raw;
  typedef Raw Raws[kPass];
  typedef bf16x8 Frags[RS][PARTS];
  const ExpandParams& p;
  f32x4* lds;
  int64_t m0;
  int rows, adapter;
  int l32, g, r_in, c_in;  // r_in, c_in: this lane's row and columns of a pass

  __device__ __forceinline__ Expand(const ExpandParams& p_, f32x4* lds_, const Tile& tile, int row0)
      : p(p_), lds(lds_), m0(tile.first + row0), rows(min(32, tile.rows - row0)), adapter(tile.adapter) {
    const int lane = threadIdx.x & 63;
    l32 = lane & 31;
    g = lane >> 5;
    r_in = lane / kLanes;
    c_in = E * (lane % kLanes);
  }
  // t as parts of bf16, from this lane's token's row of it
  __device__ __forceinline__ void load_t(Frags& tf) const {
    if (adapter >= 0) load_t(tf, p.t + (m0 + min(l32, rows - 1)) * p.ldt);
  }
  __device__ __forceinline__ void load_t(Frags& tf, const float* t) const {
    t += 8 * g;
#pragma unroll
    for (int s = 0; s < RS; ++s) {
      float v[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 u = *(const f32x4*)(t + 16 * s + 4 * h);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[4 * h + k] = u[k];
      }
#pragma unroll
      for (int part = 0; part < PARTS; ++part)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const bf16 b = (bf16)v[k];
          tf[s][part][k] = b;
          v[k] = rest(v[k], b);
        }
    }
  }
  __device__ __forceinline__ void load_base(Raws& raw, int f0) const {
    if constexpr (BASE != kNoBase) {
#pragma unroll
      for (int i = 0; i < kPass; ++i) {
        const int row = i * E + r_in;
        if (row < rows)
          raw[i] = load_run<BASE == kBaseF32, E>((const char*)p.base + (m0 + row) * p.ld_base * bs, f0 + c_in, p.N);
      }
    }
  }
  // features 32 q .. + 31 of the 64: registers 4 a .. + 3 are features 8 a + 4 g .. + 3 of token l32
  __device__ __forceinline__ void put(int q, const f32x16& acc) const {
#pragma unroll
    for (int a = 0; a < 4; ++a)
      lds[l32 * 16 + ((8 * q + 2 * a + g) ^ (l32 & 15))] =
          f32x4{acc[4 * a], acc[4 * a + 1], acc[4 * a + 2], acc[4 * a + 3]};
  }
  // base + what put() left (the wave's own LDS, whose operations stay in order)
  __device__ __forceinline__ void store(const Raws& raw, int f0) const {
#pragma unroll
    for (int i = 0; i < kPass; ++i) {
      const int row = i * E + r_in;
      Run<E> v{};
      if constexpr (BASE != kNoBase) v = values<BASE == kBaseF32, E>(raw[i]);
      if (adapter >= 0) {
#pragma unroll
        for (int h = 0; h < E / 4; ++h) {
          const f32x4 d = lds[row * 16 + ((c_in / 4 + h) ^ (row & 15))];
#pragma unroll
          for (int k = 0; k < 4; ++k) v.v[4 * h + k] += d[k];
        }
      }
      if (row < rows) store_run<F32, E>((char*)p.out + (m0 + row) * p.ld_out * es, f0 + c_in, p.N, v);
    }
  }
};

}  // namespace

// Long requests: a block's four waves take 128 tokens and walk `span` features
// together.  64 rows of B at a time are copied to LDS, whole lines, for all four
// (fragments read straight from memory touch a row's line with every lane: rank 64
// took 33 us for 63 MB of results), XOR-swizzled as the row length asks.  A step's
// copies and base loads go out one step ahead, before the stores of the step
// before: behind them they would wait for the stores to be done.
template <int BASE, bool F32, int RS>
__global__ __launch_bounds__(kThreads) void expand_kernel(ExpandParams p, int span) {
  typedef Expand<BASE, F32, RS> X;
  constexpr int kChunks = RS == 1 ? 2 : RS == 2 ? 4 : RS <= 4 ? 8 : 16;  // 16-byte chunks of a row of B in LDS
  constexpr int kRows = 16 / kChunks;                                  // rows of B in 256 bytes
  __shared__ f32x4 tiles[4][32 * 16];
  __shared__ __attribute__((aligned(16))) char bs[2][64 * kChunks * 16];
  const Tile tile = tile_at<128>(p.req, (int)blockIdx.x);
  if (tile.rows <= 0) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const X x(p, tiles[wave], tile, 32 * wave);  // (rows <= 0: the wave only helps to copy)
  const int f_begin = (int)blockIdx.y * span, f_end = min(p.N, f_begin + span);
  auto pos = [](int r, int c) { return c ^ (r / kRows & (kChunks - 1)); };  // of chunk c in row r
  const harp_ra::rsrc_t br = harp_ra::make_rsrc((const bf16*)p.b + (int64_t)max(tile.adapter, 0) * p.N * p.r,
                                                (uint32_t)p.N * (uint32_t)p.r * 2u);
  const uint32_t b_lds = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(harp_ra::lds_void*)bs);
  auto copy_b = [&](int f0, int stage) {
#pragma unroll
    for (int j = wave; j < kChunks; j += 4) {  // 64 chunks each
      const int slot = 64 * j + lane, r = slot / kChunks, c = pos(r, slot % kChunks);
      const bool in = f0 + r < p.N && 8 * c < p.r;
      harp_ra::lds_dma_b128(br, b_lds + stage * (64 * kChunks * 16) + 1024 * j,
                            in ? (uint32_t)((f0 + r) * p.r * 2 + 16 * c) : harp_ra::kOOB);
    }
  };
  typename X::Frags tf;
  typename X::Raws raw, cur;
  // (loads come back in order: once `tick` is there, the copies before it are too)
  uint32_t tick = 0;
  auto load_step = [&](int f0, int stage) {
    if (tile.adapter >= 0) {
      copy_b(f0, stage);
      tick = ((const uint16_t*)p.b)[((int64_t)tile.adapter * p.N + f0) * p.r + (lane & 7)];  // (r is 8 or more)
    }
    if (x.rows > 0) x.load_base(raw, f0);
  };
  if (x.rows > 0) x.load_t(tf);
  load_step(f_begin, 0);
  int stage = 0;
  for (int f0 = f_begin; f0 < f_end; f0 += 64, stage ^= 1) {
    asm volatile("" : "+v"(tick)::"memory");
    if (tile.adapter >= 0) {
      __syncthreads();
      if (x.rows > 0) {
        const char* const t = bs[stage];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          f32x16 acc = harp_ra::zero16();
#pragma unroll
          for (int s = 0; s < RS; ++s) {
            const int r = 32 * q + x.l32;
            const bf16x8 bf = *(const bf16x8*)(t + (r * kChunks + pos(r, 2 * s + x.g)) * 16);
#pragma unroll
            for (int part = 0; part < X::PARTS; ++part) acc = harp_ra::mfma32x32x16(bf, tf[s][part], acc);
          }
          x.put(q, acc);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < X::kPass; ++i) cur[i] = raw[i];
    if (f0 + 64 < f_end) load_step(f0 + 64, stage ^ 1);
    if (x.rows > 0) x.store(cur, f0);
  }
  harp_ra::wait_lds_loads();
}

// Short requests, and ranks whose rows of B are not 16-byte aligned: a tile of 32
// tokens, each wave 64 features of its own, B's fragments straight from memory.
// 1333 tokens x 1001 features in fp32, rank 12: 9.6 us, a third of it the start.
template <int BASE, bool F32, int RS>
__global__ __launch_bounds__(kThreads) void expand_short_kernel(ExpandParams p, int span) {
  typedef Expand<BASE, F32, RS> X;
  __shared__ f32x4 tiles[4][32 * 16];
  const Tile tile = tile_at<32>(p.req, (int)blockIdx.x);
  if (tile.rows <= 0) return;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const X x(p, tiles[wave], tile, 0);
  const int f_end = min(p.N, ((int)blockIdx.y + 1) * span);
  const bool whole = p.r % 8 == 0;
  typename X::Frags tf;
  typename X::Raws raw, cur;
  bf16x8 bf[2][RS];
  auto load_step = [&](int f0) {
    if (tile.adapter >= 0) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const bf16* b =
            (const bf16*)p.b + ((int64_t)tile.adapter * p.N + min(f0 + 32 * q + x.l32, p.N - 1)) * p.r + 8 * x.g;
#pragma unroll
        for (int s = 0; s < RS; ++s) {
          const int n = p.r - 16 * s - 8 * x.g;  // ranks this lane has left: 8 or more but in the last step
          bf[q][s] = s < RS - 1 || n >= 8 ? load_full(b + 16 * s) : whole ? harp_ra::zero8() : load_some(b + 16 * s, n);
        }
      }
    }
    x.load_base(raw, f0);
  };
  int f0 = (int)blockIdx.y * span + 64 * wave;
  if (f0 >= f_end) return;
  load_step(f0);
  x.load_t(tf);
  for (; f0 < f_end; f0 += 256) {
    if (tile.adapter >= 0) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        f32x16 acc = harp_ra::zero16();
#pragma unroll
        for (int s = 0; s < RS; ++s)
#pragma unroll
          for (int part = 0; part < X::PARTS; ++part) acc = harp_ra::mfma32x32x16(bf[q][s], tf[s][part], acc);
        x.put(q, acc);
      }
    }
#pragma unroll
    for (int i = 0; i < X::kPass; ++i) cur[i] = raw[i];
    if (f0 + 256 < f_end) load_step(f0 + 256);
    x.store(cur, f0);
  }
}

// One to four tokens to a request: both products in one launch, in fp32 on the
// vector units.  What counts is how long a block waits, not what it computes: every
// block forms t of its tokens anew (a wave sums 2 RS ranks with its lanes along K, so
// that each load is one run of 1 KB; fragments of the matrix instructions would touch
// 16 rows with every 16 lanes, and A's 123 KB of rank 16 over 3840 columns then took a
// CU 3.6 us), and its threads take a feature each, whose row of B and base were on their
// way meanwhile.  One token from 3840 to 10240 features, rank 16: 4.8 us, of which an
// empty launch is half; 32 tokens with an adapter each from 256 to 15360 features, 16 MB of
// B: 9 us.
constexpr int kFewFeatures = 512;  // of a block: a thread each

__device__ __forceinline__ float wave_sum(float v) {
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x128, 0xf, 0xf, true));  // row_ror:8
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x124, 0xf, 0xf, true));  // row_ror:4
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4e, 0xf, 0xf, true));   // quad_perm:[2,3,0,1]
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xb1, 0xf, 0xf, true));   // quad_perm:[1,0,3,2]
  v += __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401f));              // lane ^ 16
  return harp_ra::wave_half_sum(v);
}

template <bool F32, int RS, int M>
__global__ __launch_bounds__(kFewFeatures) void few_kernel(ExpandParams p, FewParams q) {
  constexpr int kWaves = kFewFeatures / 64, RJ = 16 * RS / kWaves;  // ranks of a wave
  __shared__ __attribute__((aligned(16))) float ts[M][16 * RS];
  const Tile tile = tile_at<M>(p.req, (int)blockIdx.x);
  if (tile.rows <= 0) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int f = (int)blockIdx.y * kFewFeatures + (int)threadIdx.x, fc = min(f, p.N - 1);
  float base[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const int64_t o = (int64_t)(tile.first + min(m, tile.rows - 1)) * p.ld_base + fc;
    base[m] = F32 ? ((const float*)p.base)[o] : (float)((const bf16*)p.base)[o];
  }
  if (tile.adapter >= 0) {  // (the same in every thread)
    const bool whole = p.r % 8 == 0;
    const bf16* const b = (const bf16*)p.b + ((int64_t)tile.adapter * p.N + fc) * p.r;
    bf16x8 bv[2 * RS];
#pragma unroll
    for (int s = 0; s < 2 * RS; ++s) {
      const int n = p.r - 8 * s;
      bv[s] = n >= 8 ? load_full(b + 8 * s) : whole ? harp_ra::zero8() : load_some(b + 8 * s, n);
    }
    const bf16* xr[M];
    const bf16* ar[RJ];
    float acc[RJ][M];
#pragma unroll
    for (int m = 0; m < M; ++m) xr[m] = (const bf16*)q.x + (int64_t)(tile.first + min(m, tile.rows - 1)) * q.ldx;
#pragma unroll
    for (int j = 0; j < RJ; ++j) {
      ar[j] = (const bf16*)q.a + ((int64_t)tile.adapter * p.r + min(RJ * wave + j, p.r - 1)) * q.K;
#pragma unroll
      for (int m = 0; m < M; ++m) acc[j][m] = 0.f;
    }
    auto add = [&](const bf16x8(&xv)[M], const bf16x8(&av)[RJ]) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int j = 0; j < RJ; ++j)
#pragma unroll
          for (int m = 0; m < M; ++m) acc[j][m] = __builtin_fmaf((float)av[j][k], (float)xv[m][k], acc[j][m]);
    };
    int k = 8 * lane;
    constexpr int U = RS * M <= 4 ? 4 : RS * M <= 8 ? 2 : 1;  // loads on their way, as the registers allow
#pragma unroll U
    for (; k + 8 <= q.K; k += 512) {
      bf16x8 xv[M], av[RJ];
#pragma unroll
      for (int m = 0; m < M; ++m) xv[m] = load_full(xr[m] + k);
#pragma unroll
      for (int j = 0; j < RJ; ++j) av[j] = load_full(ar[j] + k);
      add(xv, av);
    }
    if (k < q.K) {
      bf16x8 xv[M], av[RJ];
#pragma unroll
      for (int m = 0; m < M; ++m) xv[m] = load_some(xr[m] + k, q.K - k);
#pragma unroll
      for (int j = 0; j < RJ; ++j) av[j] = load_some(ar[j] + k, q.K - k);
      add(xv, av);
    }
    const float scale = q.scale ? q.scale[tile.adapter] : 1.f;
#pragma unroll
    for (int j = 0; j < RJ; ++j)
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const float v = wave_sum(acc[j][m]);
        if (lane == 0) ts[m][RJ * wave + j] = RJ * wave + j < p.r ? v * scale : 0.f;
      }
    __syncthreads();
    if (q.t && blockIdx.y == 0)
      for (int e = threadIdx.x; e < 16 * RS * min(M, tile.rows); e += kFewFeatures)
        q.t[(int64_t)(tile.first + e / (16 * RS)) * p.ldt + e % (16 * RS)] = ts[e / (16 * RS)][e % (16 * RS)];
    float y[M];
#pragma unroll
    for (int m = 0; m < M; ++m) y[m] = 0.f;
#pragma unroll
    for (int s = 0; s < 2 * RS; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < M; ++m) {
          const f32x4 t = *(const f32x4*)&ts[m][8 * s + 4 * h];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[m] = __builtin_fmaf(t[e], (float)bv[s][4 * h + e], y[m]);
        }
#pragma unroll
    for (int m = 0; m < M; ++m) base[m] += y[m];
  }
#pragma unroll
  for (int m = 0; m < M; ++m)
    if (f < p.N && m < tile.rows) {
      const int64_t o = (int64_t)(tile.first + m) * p.ld_out + f;
      if constexpr (F32) ((float*)p.out)[o] = base[m];
      else ((bf16*)p.out)[o] = (bf16)base[m];
    }
}

// ---------------------------------------------------------------------------
// Gradients of A and B: for each adapter the sum over its tokens of v[m]^T x[m].
// A block takes 128 columns and 32 RK ranks of one adapter.  Its G groups of four
// waves (32 columns each) walk the adapter's tokens, 64 in a group's step: the step's x
// (bf16) and v (taken apart into two bf16) lie in LDS as they come, and
// ds_read_b64_tr_b16 reads both transposed, tokens along the contraction of
// v_mfma_f32_32x32x16_bf16.  The next step's loads are on their way meanwhile, and the
// groups' sums are added in LDS in their order.
// (v_mfma_f32_16x16x4_f32 takes the values without a transpose, and runs at a
// sixteenth of the rate: rank 64 over 8192 tokens took 119 us.)  Where the
// blocks of all adapters would not fill the chip, each request's tokens are taken
// in `splits` parts whose sums a second kernel adds in order.
// Four adapters of rank 64 over 8192 tokens, 3840 columns of x and of dy: 42 us for
// 126 MB of them and as much of v again, out of the caches (7.9 TB/s into the CUs).  With
// one group a block and three splits, 12 waves of three blocks a CU, the same took 48 us,
// and 8 more for the sum of the splits.
// ---------------------------------------------------------------------------
namespace {
constexpr int kGradCols = 128, kGradStep = 64, kGradGroups = 4;

// Rows of W (128, 64 or 32) bf16: 16-byte chunk c of row r.  Row writes and the transposed reads below
// (64 bytes of each of four rows at a time) are free of bank conflicts.
template <int W>
__device__ __forceinline__ int grad_slot(int r, int c) {
  const int x = W == 128 ? harp_ra::swz(r) : W == 64 ? (r & 2) << 1 : 0;
  return r * W + ((c ^ x) << 3);
}

// T[r0 + {4 g .. + 3, 8 + 4 g .. + 3}][32 db + l32]: of two lanes with one g each
// register holds one token, the same for both operands.  In each group of 16
// lanes, lane i's value s is element i % 4 of the 8 bytes that lane 4 s + i / 4 addresses.
template <int W>
__device__ __forceinline__ bf16x8 tr_frag(const bf16* t, int r0, int db) {
  const int lane = threadIdx.x & 63, g = lane >> 5, s = (lane >> 2) & 3, m = lane & 3;
  const int c = 4 * db + 2 * ((lane >> 4) & 1) + (m >> 1);
  const int ra = r0 + 4 * g + s, rb = ra + 8;
  const auto lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((harp_ra::lds_bf16x4*)(t + grad_slot<W>(ra, c) + 4 * (m & 1)));
  const auto hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((harp_ra::lds_bf16x4*)(t + grad_slot<W>(rb, c) + 4 * (m & 1)));
  bf16x8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = lo[i];
    r[i + 4] = hi[i];
  }
  return r;
}

// The steps of an adapter's tokens: those of its requests one after the other
struct Steps {
  int i0;         // requests i0 .. i0 + 63 are in `todo`
  uint64_t todo;  // those of the adapter that are left
  int m, end;     // the next step's first token, the end of the request's part
};

}  // namespace

template <int RK, int G>
__global__ __launch_bounds__(kThreads* G) void grad_kernel(GradParams p, int64_t all) {
  constexpr int kRanks = 32 * RK, kPitch = kGradCols + 4;  // of the sums (a lane writes 4 columns of its rank)
  constexpr int kX = kGradStep * kGradCols, kV = kGradStep * kRanks, kGroup = 2 * (kX + 2 * kV), kSums = kRanks * kPitch * 4;
  __shared__ __attribute__((aligned(16))) char lds[G * (kGroup > kSums ? kGroup : kSums)];
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5, tid = threadIdx.x % kThreads;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kThreads);
  bf16* const xs = (bf16*)(lds + group * kGroup);
  bf16* const vs = xs + kX;  // the parts one after the other
  // this block's part and columns (constant indices: see the shrink kernel)
  GradPart part = p.part[0];
  int cb = blockIdx.x, which = 0;
#pragma unroll
  for (int i = 1; i < kMaxGradParts; ++i) {
    const int blocks = (part.C + kGradCols - 1) / kGradCols;
    if (i < p.parts && cb >= blocks) {
      cb -= blocks;
      part = p.part[i];
      which = i;
    } else {
      break;
    }
  }
  const int c0 = cb * kGradCols;
  const int rgroups = (p.rp + kRanks - 1) / kRanks;
  const int adapter = (int)blockIdx.y / rgroups, r0 = (int)blockIdx.y % rgroups * kRanks;
  const int split = blockIdx.z;
  harp_ra::sched_fence();  // (the parts' arguments and the walk's beside each other do not fit the scalar registers)

  f32x16 acc[RK];
#pragma unroll
  for (int j = 0; j < RK; ++j) acc[j] = harp_ra::zero16();

  Steps st{-64, 0, 0, 0};
  auto next = [&]() {  // whether there is another step; its tokens are st.m .. min(st.m + 64, st.end) - 1
    while (st.m >= st.end) {
      while (!st.todo) {
        st.i0 += 64;
        if (st.i0 >= p.req.count) return false;
        const int i = st.i0 + lane;
        st.todo = __ballot(i < p.req.count && adapter_of(p.req, min(i, p.req.count - 1)) == adapter);
      }
      const int i = st.i0 + __ffsll((unsigned long long)st.todo) - 1;
      st.todo &= st.todo - 1;
      const int a = token_of(p.req, i), n = max(token_of(p.req, i + 1) - a, 0);
      st.m = a + (int)((int64_t)n * split / p.splits);
      st.end = a + (int)((int64_t)n * (split + 1) / p.splits);
    }
    return true;
  };
  // the next step of every group, and whether there was one for the first; this group's is n tokens (or 0) from m on
  int m = 0, n = 0;
  auto deal = [&]() {
    bool any = false;
    n = 0;
#pragma unroll 1
    for (int q = 0; q < G && next(); ++q) {
      any = true;
      const int rows = min(kGradStep, st.end - st.m);
      if (q == group) {
        m = st.m;
        n = rows;
      }
      st.m += rows;
    }
    return any;
  };

  // a thread's share of a step: x row tid / 16 + 16 k, 8 columns; v row tid / (4 RK)
  // + 64 / RK k, 8 ranks
  constexpr int kVLanes = 4 * RK, kVRows = kThreads / kVLanes, kVPass = kGradStep / kVRows;
  bf16x8 xv[4];
  f32x4 vv[kVPass][2];
  const int xr = tid >> 4, xc = tid & 15, vr = tid / kVLanes, vc = tid % kVLanes;
  auto load = [&]() {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = xr + 16 * k, left = part.C - c0 - 8 * xc;
      xv[k] = harp_ra::zero8();
      if (row < n && left > 0) {
        const bf16* x = (const bf16*)part.x + (int64_t)(m + row) * part.ldx + c0 + 8 * xc;
        xv[k] = left >= 8 ? load_full(x) : load_some(x, left);
      }
    }
#pragma unroll
    for (int k = 0; k < kVPass; ++k) {
      const int row = vr + kVRows * k;
      vv[k][0] = vv[k][1] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (row < n && r0 + 8 * vc < p.rp) {
        const float* v = part.v + (int64_t)(m + row) * part.ldv + r0 + 8 * vc;
        vv[k][0] = *(const f32x4*)v;
        vv[k][1] = *(const f32x4*)(v + 4);
      }
    }
  };
  bool more = deal();
  load();
  while (more) {
    const int ksteps = (n + 15) / 16;
#pragma unroll
    for (int k = 0; k < 4; ++k) *(bf16x8*)(xs + grad_slot<kGradCols>(xr + 16 * k, xc)) = xv[k];
#pragma unroll
    for (int k = 0; k < kVPass; ++k) {
      bf16x8 hi, lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = vv[k][e / 4][e % 4];
        hi[e] = (bf16)f;
        lo[e] = (bf16)(f - (float)hi[e]);  // (an infinite t or u has no gradient to give: NaN)
      }
      *(bf16x8*)(vs + grad_slot<kRanks>(vr + kVRows * k, vc)) = hi;
      *(bf16x8*)(vs + kV + grad_slot<kRanks>(vr + kVRows * k, vc)) = lo;
    }
    __syncthreads();
    more = deal();
    load();
    for (int k = 0; k < ksteps; ++k) {
      const bf16x8 xf = tr_frag<kGradCols>(xs, 16 * k, wave);
#pragma unroll
      for (int j = 0; j < RK; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          acc[j] = harp_ra::mfma32x32x16(xf, tr_frag<kRanks>(vs + h * kV, 16 * k, j), acc[j]);
    }
    __syncthreads();
  }

  // a lane holds rank 32 j + l32 and columns 8 a + 4 g .. + 3 of the wave's 32
  float* const sums = (float*)lds;
#pragma unroll
  for (int j = 0; j < RK; ++j)
#pragma unroll
    for (int e = 0; e < 16; e += 4)
      *(f32x4*)(sums + (group * kRanks + 32 * j + l32) * kPitch + 32 * wave + harp_ra::c_row(e, g)) =
          f32x4{acc[j][e], acc[j][e + 1], acc[j][e + 2], acc[j][e + 3]};
  __syncthreads();
  // where the part's values go (found now: kept over the walk, it does not fit the scalar registers either)
  asm volatile("" : "+s"(which));
  const int64_t per = (int64_t)p.req.n * p.r;
  int64_t at = 0;  // of the part's values among all
  void* out = p.part[0].out;
  int cols_first = p.part[0].cols_first;
#pragma unroll
  for (int i = 1; i < kMaxGradParts; ++i)
    if (i <= which) {
      at += per * p.part[i - 1].C;
      out = p.part[i].out;
      cols_first = p.part[i].cols_first;
    }
  float* const work = p.work + split * all + at;
  // out as it lies in memory, one value a thread
  const int ranks = min(kRanks, p.r - r0), cols = min(kGradCols, part.C - c0);
  for (int i = threadIdx.x; i < kRanks * kGradCols; i += kThreads * G) {
    const int rank = cols_first ? i % kRanks : i / kGradCols, c = cols_first ? i / kRanks : i % kGradCols;
    if (rank >= ranks || c >= cols) continue;
    float sum = sums[rank * kPitch + c];
#pragma unroll
    for (int q = 1; q < G; ++q) sum += sums[(q * kRanks + rank) * kPitch + c];
    const int64_t o = cols_first ? ((int64_t)adapter * part.C + c0 + c) * p.r + r0 + rank
                                      : ((int64_t)adapter * p.r + r0 + rank) * part.C + c0 + c;
    if (p.splits == 1) ((bf16*)out)[o] = (bf16)sum;
    else work[o] = sum;
  }
}

// the sum of the splits, in order
__global__ __launch_bounds__(kThreads) void grad_sum_kernel(GradParams p, int64_t all) {
  const int64_t per = (int64_t)p.req.n * p.r;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < all; i += (int64_t)gridDim.x * kThreads) {
    float s = p.work[i];
    for (int k = 1; k < p.splits; ++k) s += p.work[k * all + i];
    int64_t o = i;
    void* out = p.part[0].out;
    int64_t n = per * p.part[0].C;
#pragma unroll
    for (int k = 1; k < kMaxGradParts; ++k)
      if (k < p.parts && o >= n) {
        o -= n;
        out = p.part[k].out;
        n = per * p.part[k].C;
      }
    ((bf16*)out)[o] = (bf16)s;
  }
}

// ---------------------------------------------------------------------------
// n matrices transposed, 64 x 64 values a block, all of a thread's loads on their way at
// once (8 matrices of 64 x 3840: 5 us; one after the other 9.4)
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kThreads) void transpose_kernel(TransposeParams p) {
  __shared__ uint16_t t[64][65];
  TransposePart part = p.part[0];
  int tile = blockIdx.x;
#pragma unroll
  for (int i = 1; i < 2 * kMaxSets; ++i) {
    const int tiles = (max(part.rows, part.fill) + 63) / 64 * ((part.cols + 63) / 64);
    if (i < p.parts && tile >= tiles) {
      tile -= tiles;
      part = p.part[i];
    } else {
      break;
    }
  }
  const int across = (part.cols + 63) / 64, fill = max(part.rows, part.fill);
  const int r0 = tile / across * 64, c0 = tile % across * 64;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  for (int i = blockIdx.y; i < p.n; i += gridDim.y) {
    const uint16_t* src = (const uint16_t*)part.src + (int64_t)i * part.rows * part.cols;
    uint16_t* dst = (uint16_t*)part.dst + (int64_t)i * part.cols * part.ld;
    uint16_t v[16];  // (all of them on their way at once)
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int r = r0 + ty + 4 * k, c = c0 + tx;
      v[k] = src[(int64_t)min(r, part.rows - 1) * part.cols + min(c, part.cols - 1)];
      if (r >= part.rows || c >= part.cols) v[k] = 0;
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) t[ty + 4 * k][tx] = v[k];
    __syncthreads();
#pragma unroll
    for (int y = ty; y < 64; y += 4)
      if (c0 + y < part.cols && r0 + tx < fill) dst[(int64_t)(c0 + y) * part.ld + r0 + tx] = t[tx][y];
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Launchers
// ---------------------------------------------------------------------------
namespace {
template <int RB>
unsigned shrink_groups(const ShrinkParams& p) {
  const int per = p.rp / 16;
  return (unsigned)(p.apart ? p.sets * ((per + RB - 1) / RB) : (per * p.sets + RB - 1) / RB);
}
template <int TB, int RB, int WAVES>
hipError_t shrink_t(const ShrinkParams& p, hipStream_t st) {
  hipLaunchKernelGGL((shrink_kernel<TB, RB, WAVES>), dim3((unsigned)slots_of(p.req, 16 * TB), shrink_groups<RB>(p)),
                     dim3(64 * WAVES), 0, st, p);
  return hipGetLastError();
}
template <int TB, int RB, int WAVES, int STAGES>
hipError_t shrink_lds_t(const ShrinkParams& p, hipStream_t st) {
  hipLaunchKernelGGL((shrink_lds_kernel<TB, RB, WAVES, STAGES, false>),
                     dim3((unsigned)slots_of(p.req, 16 * TB), shrink_groups<RB>(p)), dim3(64 * WAVES), 0, st, p,
                     TableArg<false>{});
  return hipGetLastError();
}
}  // namespace

hipError_t launch_shrink(const ShrinkParams& p, const RopeTable* table, hipStream_t st) {
  bool aligned = p.K % 8 == 0;
  for (int i = 0; i < p.sets; ++i) {
    const ShrinkSet& s = p.set[i];
    aligned &= s.ldx % 8 == 0 && s.ldx < (1 << 24) && (uintptr_t)s.x % 16 == 0 && (uintptr_t)s.a % 16 == 0;
  }
  // Few tokens: a block for every 16 ranks.  K = 3840, such blocks and the others (with t B^T): rank 64, 256 tokens 12.3
  // and 15.5 us, 1024 tokens 15.1 and 18.7, 2048 tokens 21.4 and 19.1; rank 16, 4096 tokens 14.4 and 14.6.
  const bool few = slots_of(p.req, 16) * (p.rp / 16) * p.sets <= 512;
  const int total = p.rp / 16 * (p.apart ? 1 : p.sets);
  if (table) {
    // The table beside few tokens' blocks, two pairs a thread, where both leave each other their CUs: 768 tokens, ranks of
    // 16 of three projections, 9.8 us against 9.0 and 5.2; at 8192 tokens 33 against 24 and 6.
    const int64_t slots = slots_of(p.req, 16);
    const int64_t more = (table->tokens * table->pairs + 2 * 512 - 1) / (2 * 512);
    if (aligned && few && slots * shrink_groups<1>(p) + more <= kCUs) {
      hipLaunchKernelGGL((shrink_lds_kernel<1, 1, 8, 3, true>), dim3((unsigned)(slots + more), shrink_groups<1>(p)),
                         dim3(512), 0, st, p, TableArg<true>{*table, (int)slots});
      return hipGetLastError();
    }
    const hipError_t e = launch_rope_table(*table, st);
    if (e != hipSuccess) return e;
  }
  if (aligned) {
    if (few) return shrink_lds_t<1, 1, 8, 3>(p, st);
    // Tiles of 64 tokens read A half as often and leave half as many blocks, one to a CU: they win where 32 tokens a
    // tile take more than one round.  K = 3840, rank 64: 16384 tokens 42 -> 36 us, 12000 tokens 38 -> 31, but 8192
    // tokens 22.5 -> 28; rank 32: 35 -> 29.5, 31 -> 28, 18 -> 22.
    if (p.req.tokens > 32 * kCUs && p.req.tokens / std::max(p.req.count, 1) >= 64)
      return total == 1   ? shrink_lds_t<4, 1, 4, 3>(p, st)
             : total == 2 ? shrink_lds_t<4, 2, 4, 3>(p, st)
                          : shrink_lds_t<4, 4, 4, 2>(p, st);
    // (96 KB and more of LDS each: blocks that leave room for a second one land on one CU in twos: 16 us, with half 22)
    return total == 1   ? shrink_lds_t<2, 1, 8, 2>(p, st)
           : total == 2 ? shrink_lds_t<2, 2, 4, 3>(p, st)
                        : shrink_lds_t<2, 4, 4, 3>(p, st);
  }
  // The waves of a block share K.  16 of them and 4: rank 64, 4096 tokens, K = 2052 25.1 and 30.8 us (with t B^T),
  // K = 324 17.2 and 18.3, K = 130 15.3 and 15.0; rank 128, 8192 tokens, K = 66 32.2 and 27.1.
  if (p.K < 256) return few ? shrink_t<1, 1, 4>(p, st) : shrink_t<2, 4, 4>(p, st);
  return few || total == 1 ? shrink_t<1, 1, 16>(p, st) : shrink_t<2, 4, 16>(p, st);
}

namespace {
template <int BASE, bool F32, int RS>
hipError_t expand_w(const ExpandParams& p, hipStream_t st) {
  // Requests of 128 tokens and more on the average fill a block's waves along the tokens.  To 3840 features, tall
  // and short: 32 requests of 256 tokens with rank 64 45 and 62 us, of 128 tokens 36 and 36, of 32 tokens 21.7 and
  // 22.3, with rank 16 13.4 and 13.7; of 16 tokens with rank 16 11.1 and 9.5.
  const bool tall = p.req.tokens / std::max(p.req.count, 1) >= 128 && p.r % 8 == 0 && (uintptr_t)p.b % 16 == 0;
  const int64_t slots = slots_of(p.req, tall ? 128 : 32);
  // blocks in multiples of their steps: of the long requests' three fit a CU at a time, and no more than that
  // keeps what a block does before its first step small (rank 64, 8192 x 3840: 22 us, with 2048 blocks 27)
  const int step = tall ? 64 : 256, steps = (p.N + step - 1) / step;
  const int64_t want = std::max<int64_t>(1, (tall ? 768 : 2048) / slots);
  const int each = (int)std::max<int64_t>(1, steps / std::min<int64_t>(want, steps));
  const dim3 grid((unsigned)slots, (unsigned)((steps + each - 1) / each));
  if (tall) hipLaunchKernelGGL((expand_kernel<BASE, F32, RS>), grid, dim3(kThreads), 0, st, p, each * step);
  else hipLaunchKernelGGL((expand_short_kernel<BASE, F32, RS>), grid, dim3(kThreads), 0, st, p, each * step);
  return hipGetLastError();
}
template <int BASE, bool F32>
hipError_t expand_r(const ExpandParams& p, hipStream_t st) {
  switch (p.rp / 16) {
    case 1: return expand_w<BASE, F32, 1>(p, st);
    case 2: return expand_w<BASE, F32, 2>(p, st);
    case 3: return expand_w<BASE, F32, 3>(p, st);
    case 4: return expand_w<BASE, F32, 4>(p, st);
    case 5: return expand_w<BASE, F32, 5>(p, st);
    case 6: return expand_w<BASE, F32, 6>(p, st);
    case 7: return expand_w<BASE, F32, 7>(p, st);
    default: return expand_w<BASE, F32, 8>(p, st);
  }
}
}  // namespace
hipError_t launch_expand(const ExpandParams& p, hipStream_t st) {
  if (p.out_f32) return expand_r<kBaseF32, true>(p, st);
  if (!p.base) return expand_r<kNoBase, false>(p, st);
  return p.base_f32 ? expand_r<kBaseF32, false>(p, st) : expand_r<kBaseBf16, false>(p, st);
}

namespace {
// One launch and two, K = 3840.  Of a token a request, rank 16: one request to 10240 features 4.7 and 8.6 us; to 3840
// features 16 requests (15.7 MB of A read by all blocks) 7.1 and 9.0, 24 requests (23.6 MB) 7.6 and 9.3, 64 requests
// 17.5 and 13.1; 32 requests from 256 to 15360 features 8.9 and 14.5.  Rank 64 (491 KB of A a block): 12.3 and 9.7.
// Of four tokens a request, rank 16: 4 requests (3.9 MB) 7.5 and 8.7, 8 (7.9 MB) 8.9 and 8.8, 16 (15.7 MB) 10.8
// and 9.1; rank 48 15.1 and 9.0.
constexpr int64_t kFewBytes = 24 << 20, kFewBytes4 = 8 << 20;  // of A that all blocks together read
constexpr int64_t kFewBlockBytes = 256 << 10;                  // and one of them
constexpr int kFewSteps4 = 3;  // 16-rank steps of four tokens' sums that fit the registers

int64_t few_blocks(const ExpandParams& p) { return (p.N + kFewFeatures - 1) / kFewFeatures; }

template <bool F32, int RS>
hipError_t few_t(const ExpandParams& p, const FewParams& q, hipStream_t st) {
  if (p.req.tokens <= p.req.count)
    hipLaunchKernelGGL((few_kernel<F32, RS, 1>), dim3((unsigned)slots_of(p.req, 1), (unsigned)few_blocks(p)),
                       dim3(kFewFeatures), 0, st, p, q);
  else if constexpr (RS <= kFewSteps4)
    hipLaunchKernelGGL((few_kernel<F32, RS, 4>), dim3((unsigned)slots_of(p.req, 4), (unsigned)few_blocks(p)),
                       dim3(kFewFeatures), 0, st, p, q);
  return hipGetLastError();
}
template <bool F32>
hipError_t few_r(const ExpandParams& p, const FewParams& q, hipStream_t st) {
  switch (p.rp / 16) {
    case 1: return few_t<F32, 1>(p, q, st);
    case 2: return few_t<F32, 2>(p, q, st);
    case 3: return few_t<F32, 3>(p, q, st);
    default: return few_t<F32, 4>(p, q, st);
  }
}
}  // namespace
bool few_tokens(const ExpandParams& p, int K) {
  const int64_t tiles = std::min<int64_t>(p.req.tokens, p.req.tokens / 4 + p.req.count);  // that have tokens
  const bool one = p.req.tokens <= p.req.count;
  const int64_t bytes = (int64_t)p.r * K * 2;
  return p.rp <= 16 * (one ? 4 : kFewSteps4) && p.base && p.base_f32 == p.out_f32 &&
         p.req.tokens <= 4 * (int64_t)p.req.count && bytes <= kFewBlockBytes &&
         tiles * few_blocks(p) * bytes <= (one ? kFewBytes : kFewBytes4);
}
hipError_t launch_few(const ExpandParams& p, const FewParams& q, hipStream_t st) {
  return p.out_f32 ? few_r<true>(p, q, st) : few_r<false>(p, q, st);
}

namespace {
int grad_blocks(const GradParams& p) {
  int n = 0;
  for (int i = 0; i < p.parts; ++i) n += (p.part[i].C + kGradCols - 1) / kGradCols;
  return n;
}
int grad_groups(const GradParams& p) { return (p.rp + 63) / 64; }  // 64 ranks a block (32 where that is all)
// that have tokens (of each split)
int64_t busy_blocks(const GradParams& p) {
  return (int64_t)grad_blocks(p) * std::min(p.req.n, p.req.count) * grad_groups(p);
}
template <int RK, int G>
hipError_t grad_t(const GradParams& p, hipStream_t st) {
  const dim3 grid((unsigned)grad_blocks(p), (unsigned)(p.req.n * ((p.rp + 32 * RK - 1) / (32 * RK))), (unsigned)p.splits);
  hipLaunchKernelGGL((grad_kernel<RK, G>), grid, dim3(kThreads * G), 0, st, p,
                     grad_values(p));
  return hipGetLastError();
}
// Four groups of waves where a block has a CU to itself, fewer where more blocks share it.  3840 columns of x and of
// dy, four, two groups and one: 4 adapters of rank 64 over 8192 tokens (240 blocks) 39, 41 and 54 us; 8 of them (480
// blocks) 44, 36 and 39; 16 over 2048 tokens (960) 33, 21 and 19; 32 of rank 16 over 4096 tokens (1920) 43, 24 and 20.
template <int RK>
hipError_t grad_g(const GradParams& p, hipStream_t st) {
  const int64_t blocks = busy_blocks(p) * p.splits;
  return blocks <= kCUs ? grad_t<RK, 4>(p, st) : blocks <= 2 * kCUs ? grad_t<RK, 2>(p, st) : grad_t<RK, 1>(p, st);
}
}  // namespace
int grad_splits(const GradParams& p) {
  const int64_t blocks = busy_blocks(p);
  if (!blocks) return 1;
  const int64_t want = kCUs / blocks;  // a CU to a block
  const int64_t most = p.req.tokens / p.req.count / (kGradStep * kGradGroups);  // a step for every group at least
  return (int)std::max<int64_t>(1, std::min(want, most));
}
hipError_t launch_adapter_grad(const GradParams& p, hipStream_t st) {
  const hipError_t e = p.rp <= 32 ? grad_g<1>(p, st) : grad_g<2>(p, st);
  if (e != hipSuccess || p.splits == 1) return e;
  const int64_t all = grad_values(p);
  const int64_t blocks = std::min<int64_t>((all + kThreads - 1) / kThreads, 4096);
  hipLaunchKernelGGL(grad_sum_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, st, p, all);
  return hipGetLastError();
}

hipError_t launch_transpose(const TransposeParams& p, hipStream_t st) {
  int64_t tiles = 0;
  for (int i = 0; i < p.parts; ++i)
    tiles += (int64_t)((std::max(p.part[i].rows, p.part[i].fill) + 63) / 64) * ((p.part[i].cols + 63) / 64);
  hipLaunchKernelGGL(transpose_kernel, dim3((unsigned)tiles, (unsigned)std::min(p.n, 65535)), dim3(kThreads), 0, st, p);
  return hipGetLastError();
}

}  // namespace harp_req
