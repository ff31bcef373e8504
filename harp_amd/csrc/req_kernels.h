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

// Pair p of a head (p < end[a], not before the axis) turns by
// 2^(c0[a] + c1[a] * p) turns per unit of its position along axis a.
struct RopeAxes {
  int n;
  int end[kMaxAxes];  // first pair behind the axis; the last one is D / 2
  double c0[kMaxAxes], c1[kMaxAxes];
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
// fp32 (cos, sin) pairs [B, S, D / 2, 2]
hipError_t launch_rope_table(const RopeAxes& axes, const RopePos& pos, int B, int S, int D, float* out,
                             hipStream_t stream);

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
// rows without an adapter are not written), as fp32 or as a bf16 value and the
// bf16 rounding of what it left out: [high part (rp) | low part (rp)].
struct ShrinkSet {
  const void* a;       // bf16 [n, r, K]
  const float* scale;  // [n] or NULL (ones)
  void* t;
};
struct ShrinkParams {
  Requests req;
  const void* x;  // bf16 [tokens, K]
  int64_t ldx;
  int K, r, rp;
  int64_t ldt;  // elements (fp32, or bf16 with pairs)
  int pairs;
  int sets;
  ShrinkSet set[kMaxSets];
};
hipError_t launch_shrink(const ShrinkParams& p, hipStream_t stream);

// out[m][j] = base[m][j] + sum over ranks t[m][.] B[j][.]
struct ExpandParams {
  Requests req;
  const float* t;  // [tokens, rp]
  int64_t ldt;
  const void* b;  // bf16 [n, N, r]
  const void* base;  // [tokens, N] or NULL (zeros)
  int64_t ld_base;
  void* out;
  int64_t ld_out;
  int f32;  // base and out are fp32 (bf16 otherwise)
  int N, r, rp;
};
hipError_t launch_expand(const ExpandParams& p, hipStream_t stream);

// ga[a][j][c] = sum over the tokens m of adapter a of v[m][j] x[m][c]; stored [n, r, C]
// (or [n, C, r] with `cols_first`), bf16.  Two such sums run in one launch.
struct GradPart {
  const void* x;  // bf16 [tokens, C]
  int64_t ldx;
  const float* v;  // fp32 [tokens, rp]
  int64_t ldv;
  int C;
  int cols_first;
  void* out;  // bf16, NULL = not wanted
};
struct GradParams {
  Requests req;
  int r, rp;
  GradPart part[2];
  int splits;   // each request's tokens in so many parts (grad_splits)
  float* work;  // [splits][n][r][C of both parts] partial sums where splits > 1
};
int grad_splits(const GradParams& p);
hipError_t launch_adapter_grad(const GradParams& p, hipStream_t stream);

// dst[i][c][r] = src[i][r][c], bf16, n matrices of rows x cols; two in one launch
struct TransposePart {
  const void* src;
  void* dst;
  int rows, cols;
};
struct TransposeParams {
  int n;
  TransposePart part[2];
};
hipError_t launch_transpose(const TransposeParams& p, hipStream_t stream);

}  // namespace harp_req
