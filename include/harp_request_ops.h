/*
 * harp_request_ops.h — C ABI of the MI355X (gfx950) kernels that give every
 * request of a batch its own positions and its own adapter: the RMSNorm of
 * queries and keys with a rotary embedding of several axes (forward and
 * backward, and the embedding's table), and low-rank adapters beside a
 * projection (forward and backward, and inside the q/k/v producer).
 *
 * HARP's model rotates each head's features by the (time, height, width) of a
 * token: its RopeEmbedder gathers a table of exp(i angle) for each axis
 * (src/models/z_image/standalone_transformer.py), which the RoPE operators of
 * async_rt/csrc/rope.cc read.  Here the angles are formed where they are used.
 * The adapters have no reference counterpart.  libharp_ra.so exports the
 * functions declared here next to those of harp_ring_attn.h,
 * harp_qk_norm_rope.h and harp_block_ops.h.
 *
 * Conventions (as there): plain device pointers of the current device, strides
 * in elements, unit stride along a row, asynchronous on the given HIP stream
 * (NULL = default stream), int status (HARP_REQ_OK = 0) and
 * harp_req_last_error() for the message.  Nothing is allocated; arguments are
 * checked on the host before any device call.  No call waits for the GPU or
 * clears memory: all of them can be captured into a HIP graph.
 */
#ifndef HARP_REQUEST_OPS_H
#define HARP_REQUEST_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "harp_qk_norm_rope.h"

#ifndef HARP_REQ_API
#define HARP_REQ_API __attribute__((visibility("default")))
#endif

#ifdef __cplusplus
extern "C" {
#endif

enum {
  HARP_REQ_OK = 0,
  HARP_REQ_EINVAL = 1,       /* bad pointer, size, stride, alignment or dtype */
  HARP_REQ_EUNSUPPORTED = 2, /* valid request that the library does not handle */
  HARP_REQ_ENOMEM = 3,       /* workspace too small */
  HARP_REQ_ELAUNCH = 4       /* HIP launch or runtime error */
};

enum { HARP_REQ_F32 = 0, HARP_REQ_BF16 = 1, HARP_REQ_I32 = 2, HARP_REQ_I64 = 3 };

enum { HARP_REQ_MAX_AXES = 4, HARP_REQ_MAX_RANK = 128 };

/*
 * The axes of a rotary embedding of heads of sum(width) features: axis a takes
 * the next width[a] / 2 pairs, and pair j of it turns by
 * position[a] * theta[a]^(-2 j / width[a]) radians.  Pairs are (2 p, 2 p + 1), or
 * (p, p + D / 2) with half.  Angles are off by 2^-22 of a turn at most up
 * to positions of 2^31, for theta of 1 and more; a position that is not finite makes its
 * pairs NaN.
 */
typedef struct {
  int n;                            /* 1 to HARP_REQ_MAX_AXES */
  int width[HARP_REQ_MAX_AXES];     /* even, positive */
  double theta[HARP_REQ_MAX_AXES];  /* positive, finite */
  int half;
} harp_req_axes_t;

/* positions[b][s][a]: I32, I64 or F32, any strides (0 repeats) */
typedef struct {
  const void* p;
  int dtype;
  int64_t stride_b, stride_s, stride_a;
} harp_req_positions_t;

/* one of q and k: [B, heads, S, D] views, strides {b, h, s} */
typedef struct {
  const void* x;
  int64_t x_stride[3];
  void* y; /* forward: the result; backward: the gradient of x */
  int64_t y_stride[3];
  int heads; /* 0: no such tensor */
  int norm;  /* RMSNorm in front of the rotation */
  const void* weight; /* [D] of weight_dtype (F32 or BF16), or NULL for ones */
  int weight_dtype;
  float eps;
  const void* dy; /* backward: the gradient of y */
  int64_t dy_stride[3];
  void* grad_weight; /* backward: [D] of weight_dtype, or NULL */
} harp_req_heads_t;

/*
 * y = rotate(x / sqrt(mean(x^2) + eps) * weight) of q and k (heads[0], heads[1]) in
 * one launch, or y = rotate(x) where norm is 0.  dtype (of x, y, dy): F32 or
 * BF16; arithmetic is fp32, each result rounded once.  D = sum(width) a multiple
 * of 8, 8 to 256.  x, y and dy 16-byte aligned, strides multiples of 8 with the h and
 * s strides below 2^31 (x and dy may repeat); no two elements of y at one address,
 * y apart from x.  batch * seq * heads up to 2^31.
 */
HARP_REQ_API int harp_req_qk_norm_rope_forward(const harp_req_axes_t* axes, const harp_req_positions_t* positions,
                                               const harp_req_heads_t* heads, int batch, int seq, int dtype,
                                               void* stream);

/*
 * The gradients: of x (y of the structs) and of the weights, from dy.  x is read
 * where norm is set.  workspace: harp_req_qk_backward_workspace_bytes, 16-byte
 * aligned, for weight gradients only (NULL without them); it is free again when
 * the launches behind this call have run.
 */
HARP_REQ_API int harp_req_qk_norm_rope_backward(const harp_req_axes_t* axes, const harp_req_positions_t* positions,
                                                const harp_req_heads_t* heads, int batch, int seq, int dtype,
                                                void* workspace, size_t workspace_bytes, void* stream);
HARP_REQ_API size_t harp_req_qk_backward_workspace_bytes(int batch, int seq, int d, int q_heads, int k_heads);

/* table[b][s][p] = (cos, sin) of pair p's angle, fp32, contiguous [B, S, D / 2, 2], 8-byte aligned */
HARP_REQ_API int harp_req_rope_table(const harp_req_axes_t* axes, const harp_req_positions_t* positions, int batch,
                                     int seq, float* table, void* stream);

/*
 * Which tokens are whose: request i is tokens offsets[i] .. offsets[i + 1] - 1
 * (offsets: count + 1 values, never falling) and takes adapter index[i]; one that
 * is not 0 .. n - 1 takes none, nor do the tokens in front of the first request and
 * behind the last.  offsets NULL: each request is tokens / count tokens.  Both I32
 * or I64, each its own.  Values outside 0 .. tokens are read as the nearest of them.
 * An infinity or a NaN in one adapter reaches its own requests' tokens only (and from
 * b may come out as NaN).
 */
typedef struct {
  const void* index;
  int index_dtype;
  const void* offsets;
  int offsets_dtype;
  int count;
} harp_req_requests_t;

/* n adapters of one rank: a bf16 [n, rank, K], b bf16 [n, N, rank], contiguous; scales [n] fp32 or NULL for ones */
typedef struct {
  const void* a;
  const void* b;
  const float* scales;
  int n, rank;
} harp_req_adapters_t;

/* fp32 values that `t` of the calls below holds for each token: the rank rounded up to 16 */
HARP_REQ_API int harp_req_adapter_columns(int rank);

/*
 * out[m] = base[m] + scale x[m] A^T B^T of token m's adapter (out[m] = base[m]
 * without one).  x bf16 [tokens, K]; base and out [tokens, N] of dtype F32 or BF16;
 * out may be base itself, and no other input.  t: fp32 [tokens,
 * harp_req_adapter_columns(rank)] contiguous, 16-byte aligned: written with scale x A^T
 * for the tokens that have an adapter, to be kept for the backward call.  rank 1 to
 * 128; K and N 1 to 2^22, tokens up to 2^25, count up to 2^20, n up to 2^14.
 */
HARP_REQ_API int harp_req_add_adapters_forward(const void* x, int64_t ld_x, const void* base, int64_t ld_base,
                                               void* out, int64_t ld_out, int dtype,
                                               const harp_req_adapters_t* adapters,
                                               const harp_req_requests_t* requests, float* t, int tokens, int k_dim,
                                               int n_dim, void* stream);

/*
 * The gradients of one to three projections of one x, each with adapters of one n
 * and one rank: from dy bf16 [tokens, N] and the forward's t of each, da and db of a's
 * and b's shapes (zeros for adapters without a token; NULL = not wanted), and dx bf16
 * [tokens, K], the sum of all of them plus dx_base (NULL: zeros), or NULL.  (The
 * gradient of base is dy.)  dx_base: fp32 [tokens, K], written over where the ranks (rounded up
 * to 16) of all sets exceed 128 together; such calls with more than one set need it.  workspace:
 * harp_req_adapter_backward_workspace_bytes, 16-byte aligned, free again when the launches
 * behind this call have run.
 */
typedef struct {
  harp_req_adapters_t adapters;
  const float* t;
  const void* dy;
  int64_t ld_dy;
  void* da;
  void* db;
} harp_req_backward_set_t;

HARP_REQ_API int harp_req_add_adapters_backward(const harp_req_backward_set_t* sets, int n_sets, const void* x,
                                                int64_t ld_x, const harp_req_requests_t* requests, float* dx_base,
                                                int64_t ld_dx_base, void* dx, int64_t ld_dx, int tokens, int k_dim,
                                                int n_dim, void* workspace, size_t workspace_bytes, void* stream);
HARP_REQ_API size_t harp_req_adapter_backward_workspace_bytes(int tokens, int k_dim, int n_dim, int n, int rank,
                                                              int count, int n_sets);

/*
 * harp_qkv_project (harp_qk_norm_rope.h) with low-rank adapters beside its
 * projections, in one launch behind the one for x A^T: adapters[i] goes with outs[i]
 * (a [n, rank, k_dim], b [n, n_out, rank]; one n and one rank, a multiple of 8 up to
 * 128).  Arithmetic is fp32 from the products to the result, rounded once, to nearest
 * (harp_qkv_project truncates behind the norm and the rotation); y_lin is the rounded
 * product with its adapter.  t (n_outs pointers, or NULL): each fp32 [tokens,
 * harp_req_adapter_columns(rank)], as for harp_req_add_adapters_forward.  workspace:
 * harp_req_qkv_workspace_bytes, 16-byte aligned.  batch * seq up to 2^25.
 *
 * The rotation: freqs as harp_qkv_project takes it, or NULL and positions along axes of
 * 128 features together, of neighbouring pairs; then table, fp32 [batch, seq, 64, 2] ([1, seq,
 * 64, 2] where stride_b is 0), 16-byte aligned, is written with their table.
 */
HARP_REQ_API int harp_req_qkv_project(const void* x, int64_t ld_x, int batch, int seq, int k_dim, int n_out,
                                      const float* freqs, int64_t f_stride_b, int64_t f_stride_s,
                                      const harp_req_axes_t* axes, const harp_req_positions_t* positions,
                                      float* table, const harp_qkv_out_t* outs,
                                      const harp_req_adapters_t* adapters, int n_outs,
                                      const harp_req_requests_t* requests, float* const* t, void* workspace,
                                      size_t workspace_bytes, void* stream);
HARP_REQ_API size_t harp_req_qkv_workspace_bytes(int tokens, int rank, int n_outs);

HARP_REQ_API const char* harp_req_last_error(void);

#ifdef __cplusplus
}
#endif
#endif
