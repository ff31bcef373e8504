// Parameter blocks and launchers of the kernels that give every request of a
// batch its own positions and its own adapter: the QK RMSNorm with a rotary
// embedding of several axes, and low-rank adapters beside a projection
// (internal to libharp_ra.so; the C ABI is in include/harp_request_ops.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace harp_req {

constexpr int kF32 = 0, kBf16 = 1, kI32 = 2, kI64 = 3;  // element types

// ---------------------------------------------------------------------------
// Rotary positions with several axes
// ---------------------------------------------------------------------------
constexpr int kMaxAxes = 4;
constexpr int kMaxRopeDim = 256;

// Pair p of a head (p < end[a], not before the axis), the axis' pair j, turns by
// 2^(c[a] * j) / (2 pi) turns per unit of its position along axis a.
struct RopeAxes {
  int n;
  int end[kMaxAxes];  // first pair behind the axis; the last one is D / 2
  double c[kMaxAxes];
};

// positions [B, S, n axes] (element strides, any of them 0)
struct RopePos {
  const void* p;
  int dtype;  // kI32, kI64 or kF32
  int64_t sb, ss, sa;
};

// q or k: [B, H, S, D] views with unit D stride
struct RopeStrides {
  int64_t b;
  int h, s;
};
struct RopeHeads {
  const void* x;
  const void* dy;  // backward: gradient of y
  void* y;         // forward: the result; backward: the gradient of x
  RopeStrides sx, sdy, sy;
  int H;
  int norm;  // RMSNorm in front of the rotation
  const void* w;  // [D] or NULL (ones)
  int w_f32;
  float eps;
};

struct RopeParams {
  RopeAxes axes;
  RopePos pos;
  int B, S, D;
  int half;      // pairs (p, p + D / 2) instead of (2 p, 2 p + 1)
  int f32;       // x and y are fp32 (bf16 otherwise)
  float sign;    // 1, or -1: rotated back
  RopeHeads t[2];  // q, k (H 0: none)
  float* wpart;  // backward: [q's blocks, then k's][D] sums of d xhat, NULL = not needed
};

hipError_t launch_rope_forward(const RopeParams& p, hipStream_t stream);
void rope_bwd_blocks(const RopeParams& p, int blocks[2]);  // of q, of k
// the gradients of x (in t[].y); wpart where it is given
hipError_t launch_rope_backward(const RopeParams& p, hipStream_t stream);
// gw[i] (i: q, k; NULL = not wanted) = sum over the tensor's blocks of wpart
hipError_t launch_rope_wgrad(const float* wpart, const int blocks[2], int D, void* const gw[2], const int gw_f32[2],
                             hipStream_t stream);
// (cos, sin) of every pair's angle: out[token][pair], the tokens of B batches of S one after the other
struct RopeTable {
  RopeAxes axes;
  RopePos pos;
  int S, pairs;
  int64_t tokens;
  float2* out;
};
hipError_t launch_rope_table(const RopeTable& t, hipStream_t stream);

// ---------------------------------------------------------------------------
// Low-rank adapters
// ---------------------------------------------------------------------------
constexpr int kMaxRank = 128;
constexpr int kMaxSets = 3;  // q, k, v

inline int rank_pad(int r) { return (r + 15) / 16 * 16; }

// Which tokens are whose: request i (0 <= i < count) is tokens offsets[i] ..
// offsets[i + 1] - 1 and takes adapter index[i] (none where that is not one of
// 0 .. n - 1).  offsets NULL: every request is len tokens.
struct Requests {
  const void* index;
  const void* offsets;
  int index64, offsets64;
  int count;
  int len;
  int tokens;
  int n;  // adapters
};

// t[m][0 .. rp - 1] = scale * x A^T of token m's adapter (zeros behind rank r;
// rows without an adapter are not written), as fp32 (t), and as a bf16 value
// with the bf16 rounding of what it left out (pairs: [rp high parts | rp low
// parts] of each token); either may be NULL.  Up to three sets; one read of an x that they share.
struct ShrinkSet {
  const void* a;       // bf16 [n, r, K]
  const float* scale;  // [n] or NULL (ones)
  const void* x;       // bf16 [tokens, K], row stride ldx
  int64_t ldx;
  float* t;  // row stride ldt
  void* pairs;  // bf16, row stride 2 rp
};
struct ShrinkParams {
  Requests req;
  int K, r, rp;
  int64_t ldt;
  int sets;
  int apart;  // the sets have an x each
  ShrinkSet set[kMaxSets];
};
// (table: written as well, by blocks of the same launch or by a launch in front; or NULL)
hipError_t launch_shrink(const ShrinkParams& p, const RopeTable* table, hipStream_t stream);

// out[m][j] = base[m][j] + sum over ranks t[m][.] B[j][.]
struct ExpandParams {
  Requests req;
  const float* t;  // [tokens, rp], row stride ldt
  int64_t ldt;
  const void* b;  // bf16 [n, N, r]
  const void* base;  // [tokens, N] or NULL (zeros)
  int64_t ld_base;
  void* out;
  int64_t ld_out;
  int base_f32, out_f32;  // (bf16 otherwise); an fp32 result has an fp32 base
  int N, r, rp;
};
hipError_t launch_expand(const ExpandParams& p, hipStream_t stream);

// Both of the above in one launch, for few tokens to a request: t is formed from x
// and A (as ShrinkSet's) where it is needed, and written if it is wanted.
struct FewParams {
  const void* a;
  const float* scale;
  const void* x;
  int64_t ldx;
  int K;
  float* t;  // row stride ldt of the other parameters, or NULL
};
bool few_tokens(const ExpandParams& p, int K);  // whether it is for this call
hipError_t launch_few(const ExpandParams& p, const FewParams& q, hipStream_t stream);

// For each adapter a the sum over its tokens m of v[m][j] x[m][c]: out [n, r, C],
// or [n, C, r] with `cols_first`, bf16.  Up to six such sums in one launch.
struct GradPart {
  const void* x;  // bf16 [tokens, C]
  int64_t ldx;
  const float* v;  // [tokens, rp]
  int64_t ldv;
  int C;
  int cols_first;
  void* out;
};
constexpr int kMaxGradParts = 2 * kMaxSets;
struct GradParams {
  Requests req;
  int r, rp;
  int parts;
  GradPart part[kMaxGradParts];
  int splits;   // each request's tokens in so many parts (grad_splits)
  float* work;  // [splits] of all outputs, one after the other, where splits > 1
};
int grad_splits(const GradParams& p);
// values of all outputs
__host__ __device__ inline int64_t grad_values(const GradParams& p) {
  int64_t c = 0;
#pragma unroll
  for (int i = 0; i < kMaxGradParts; ++i)
    if (i < p.parts) c += p.part[i].C;
  return c * p.req.n * p.r;
}
hipError_t launch_adapter_grad(const GradParams& p, hipStream_t stream);

// dst[i][c][r] = src[i][r][c], bf16, n matrices of rows x cols, dst's rows ld
// values apart and zero from the source's rows up to `fill`
struct TransposePart {
  const void* src;
  void* dst;
  int rows, cols;
  int ld, fill;
};
struct TransposeParams {
  int n;
  int parts;
  TransposePart part[2 * kMaxSets];
};
hipError_t launch_transpose(const TransposeParams& p, hipStream_t stream);

}  // namespace harp_req
