// C ABI of the kernels for requests of one batch (rotary positions, low-rank
// adapters): argument validation and kernel sequencing.  See
// include/harp_request_ops.h.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <string>
#include <utility>

#include "../../include/harp_request_ops.h"
#include "proj_kernels.h"
#include "req_kernels.h"

using namespace harp_req;

static_assert(HARP_REQ_F32 == kF32 && HARP_REQ_BF16 == kBf16 && HARP_REQ_I32 == kI32 && HARP_REQ_I64 == kI64,
              "the kernels' element types");
static_assert(HARP_REQ_MAX_AXES == kMaxAxes && HARP_REQ_MAX_RANK == kMaxRank, "the kernels' limits");

namespace {

thread_local std::string g_last_error;

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return code;
}
int ok() {
  g_last_error.clear();
  return HARP_REQ_OK;
}
int launched(hipError_t e, const char* what) {
  if (e != hipSuccess) return fail(HARP_REQ_ELAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
  return ok();
}
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr int64_t kMaxRows = (int64_t)1 << 31;
// (tokens: the smallest tiles' grids stay below 2^32 threads)
constexpr int kMaxTokens = 1 << 25, kMaxDim = 1 << 22, kMaxCount = 1 << 20, kMaxAdapters = 1 << 14;

// ---------------------------------------------------------------------------
// Rope
// ---------------------------------------------------------------------------
int check_axes(const harp_req_axes_t* in, RopeAxes& ax, int& D) {
  if (!in) return fail(HARP_REQ_EINVAL, "axes is NULL");
  if (in->n < 1 || in->n > kMaxAxes) return fail(HARP_REQ_EINVAL, "%d axes: 1 to %d", in->n, kMaxAxes);
  ax = RopeAxes{};
  ax.n = in->n;
  int64_t pairs = 0;
  for (int a = 0; a < in->n; ++a) {
    const int w = in->width[a];
    if (w < 2 || w % 2 || w > kMaxRopeDim)
      return fail(HARP_REQ_EINVAL, "width[%d]=%d must be even, 2 to %d", a, w, kMaxRopeDim);
    if (!(in->theta[a] > 0.0) || !std::isfinite(in->theta[a]))
      return fail(HARP_REQ_EINVAL, "theta[%d] must be positive and finite", a);
    ax.c[a] = -2.0 / w * std::log2(in->theta[a]);  // theta^(-2 j / w) = 2^(c j)
    pairs += w / 2;
    ax.end[a] = (int)pairs;
  }
  D = (int)(2 * pairs);
  if (D % 8 || D > kMaxRopeDim)
    return fail(HARP_REQ_EUNSUPPORTED, "heads of %d features: the axes' widths must add up to a multiple of 8, at most %d",
                D, kMaxRopeDim);
  return HARP_REQ_OK;
}
int check_positions(const harp_req_positions_t* in, RopePos& pos) {
  if (!in || !in->p) return fail(HARP_REQ_EINVAL, "positions is NULL");
  if (in->dtype != kI32 && in->dtype != kI64 && in->dtype != kF32)
    return fail(HARP_REQ_EINVAL, "positions dtype must be I32, I64 or F32");
  if (!aligned(in->p, in->dtype == kI64 ? 8 : 4)) return fail(HARP_REQ_EINVAL, "positions must be aligned to its elements");
  pos = RopePos{in->p, in->dtype, in->stride_b, in->stride_s, in->stride_a};
  return HARP_REQ_OK;
}
int check_batch(int batch, int seq) {
  if (batch < 0 || seq < 0) return fail(HARP_REQ_EINVAL, "batch=%d and seq=%d must not be negative", batch, seq);
  if ((int64_t)batch * seq > kMaxRows) return fail(HARP_REQ_EUNSUPPORTED, "batch * seq > 2^31");
  return HARP_REQ_OK;
}
int check_view(const void* p, const int64_t (&st)[3], const char* t, const char* name, RopeStrides& out) {
  if (!p || !aligned(p, 16)) return fail(HARP_REQ_EINVAL, "%s.%s must be a 16-byte aligned device pointer", t, name);
  for (int i = 0; i < 3; ++i)
    if (st[i] < 0 || st[i] % 8 || (i && st[i] > INT32_MAX))
      return fail(HARP_REQ_EINVAL, "%s.%s strides (%lld, %lld, %lld) must be multiples of 8, not negative, the last two below 2^31",
                  t, name, (long long)st[0], (long long)st[1], (long long)st[2]);
  out = RopeStrides{st[0], (int)st[1], (int)st[2]};
  return HARP_REQ_OK;
}
// no two elements at one address: sorted by stride, each covers what lies inside it
bool overlaps(const int64_t (&st)[3], int B, int H, int S, int D) {
  int64_t stride[3] = {st[0], st[1], st[2]}, size[3] = {B, H, S};
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 3; ++j)
      if (stride[j] < stride[i]) {
        std::swap(stride[i], stride[j]);
        std::swap(size[i], size[j]);
      }
  __int128 extent = D;
  for (int i = 0; i < 3; ++i) {
    if (size[i] == 1) continue;
    if (stride[i] < extent) return true;
    extent += (__int128)stride[i] * (size[i] - 1);
  }
  return false;
}
int check_heads(const harp_req_heads_t* in, RopeParams& p, bool backward) {
  if (!in) return fail(HARP_REQ_EINVAL, "heads is NULL");
  static const char* const names[2] = {"q", "k"};
  int64_t all = 0;
  for (int i = 0; i < 2; ++i) {
    const harp_req_heads_t& h = in[i];
    RopeHeads& t = p.t[i];
    int rc;
    if (h.heads < 0) return fail(HARP_REQ_EINVAL, "%s.heads=%d must not be negative", names[i], h.heads);
    all += h.heads;
    if (!h.heads) continue;
    t.H = h.heads;
    t.norm = h.norm != 0;
    if (!backward || h.norm) {
      if ((rc = check_view(h.x, h.x_stride, names[i], "x", t.sx))) return rc;
      t.x = h.x;
    }
    if ((rc = check_view(h.y, h.y_stride, names[i], "y", t.sy))) return rc;
    t.y = h.y;
    if (overlaps(h.y_stride, p.B, h.heads, p.S, p.D))
      return fail(HARP_REQ_EINVAL, "%s.y has two elements at one address", names[i]);
    if (backward) {
      if ((rc = check_view(h.dy, h.dy_stride, names[i], "dy", t.sdy))) return rc;
      t.dy = h.dy;
    }
    if (h.norm) {
      if (!(h.eps >= 0.f)) return fail(HARP_REQ_EINVAL, "%s.eps must be a non-negative number", names[i]);
      t.eps = h.eps;
      if (h.weight) {
        if (h.weight_dtype != kF32 && h.weight_dtype != kBf16)
          return fail(HARP_REQ_EINVAL, "%s.weight dtype must be F32 or BF16", names[i]);
        if (!aligned(h.weight, h.weight_dtype == kF32 ? 4 : 2))
          return fail(HARP_REQ_EINVAL, "%s.weight must be aligned to its elements", names[i]);
        t.w = h.weight;
        t.w_f32 = h.weight_dtype == kF32;
      }
    } else if (h.weight || h.grad_weight) {
      return fail(HARP_REQ_EINVAL, "%s has a weight without a norm", names[i]);
    }
    if (backward && h.grad_weight && (!h.weight || !aligned(h.grad_weight, h.weight_dtype == kF32 ? 4 : 2)))
      return fail(HARP_REQ_EINVAL, "%s.grad_weight needs a weight and its alignment", names[i]);
  }
  if ((int64_t)p.B * p.S * all > kMaxRows) return fail(HARP_REQ_EUNSUPPORTED, "batch * seq * heads > 2^31");
  return HARP_REQ_OK;
}
int rope_inputs(RopeParams& p, const harp_req_axes_t* axes, const harp_req_positions_t* positions,
                const harp_req_heads_t* heads, int batch, int seq, int dtype, bool backward) {
  int rc;
  if ((rc = check_axes(axes, p.axes, p.D))) return rc;
  if ((rc = check_batch(batch, seq))) return rc;
  if (dtype != kF32 && dtype != kBf16) return fail(HARP_REQ_EINVAL, "dtype must be F32 or BF16");
  p.B = batch;
  p.S = seq;
  p.half = axes->half != 0;
  p.f32 = dtype == kF32;
  p.sign = backward ? -1.f : 1.f;
  if (!((int64_t)batch * seq)) return HARP_REQ_OK;
  if ((rc = check_positions(positions, p.pos))) return rc;
  return check_heads(heads, p, backward);
}

// ---------------------------------------------------------------------------
// Adapters
// ---------------------------------------------------------------------------
int check_adapters(const harp_req_adapters_t* a, int K, int N, bool pointers) {
  if (!a) return fail(HARP_REQ_EINVAL, "adapters is NULL");
  if (a->n < 1 || a->rank < 1) return fail(HARP_REQ_EINVAL, "n=%d and rank=%d must be positive", a->n, a->rank);
  if (a->n > kMaxAdapters) return fail(HARP_REQ_EUNSUPPORTED, "n=%d adapters > %d", a->n, kMaxAdapters);
  if (a->rank > kMaxRank) return fail(HARP_REQ_EUNSUPPORTED, "rank=%d > %d", a->rank, kMaxRank);
  if (K < 1 || N < 1) return fail(HARP_REQ_EINVAL, "k_dim=%d and n_dim=%d must be positive", K, N);
  if (K > kMaxDim || N > kMaxDim) return fail(HARP_REQ_EUNSUPPORTED, "k_dim=%d, n_dim=%d: more than 2^22", K, N);
  if (!pointers) return HARP_REQ_OK;
  if (!a->a || !aligned(a->a, 2) || !a->b || !aligned(a->b, 2))
    return fail(HARP_REQ_EINVAL, "a and b must be device pointers aligned to their elements");
  if (!aligned(a->scales, 4)) return fail(HARP_REQ_EINVAL, "scales must be 4-byte aligned");
  return HARP_REQ_OK;
}
int check_tokens(int tokens) {
  if (tokens < 0) return fail(HARP_REQ_EINVAL, "tokens=%d must not be negative", tokens);
  if (tokens > kMaxTokens) return fail(HARP_REQ_EUNSUPPORTED, "tokens=%d > 2^25", tokens);
  return HARP_REQ_OK;
}
int check_requests(const harp_req_requests_t* r, int tokens, int n, Requests& q) {
  if (!r) return fail(HARP_REQ_EINVAL, "requests is NULL");
  if (r->count < 1) return fail(HARP_REQ_EINVAL, "count=%d must be positive", r->count);
  if (r->count > kMaxCount) return fail(HARP_REQ_EUNSUPPORTED, "count=%d > 2^20", r->count);
  auto ints = [](const void* p, int dtype, const char* name) {
    if (dtype != kI32 && dtype != kI64) return fail(HARP_REQ_EINVAL, "%s dtype must be I32 or I64", name);
    if (!aligned(p, dtype == kI64 ? 8 : 4)) return fail(HARP_REQ_EINVAL, "%s must be aligned to its elements", name);
    return (int)HARP_REQ_OK;
  };
  int rc;
  if (!r->index) return fail(HARP_REQ_EINVAL, "index is NULL");
  if ((rc = ints(r->index, r->index_dtype, "index"))) return rc;
  if (r->offsets) {
    if ((rc = ints(r->offsets, r->offsets_dtype, "offsets"))) return rc;
  } else if (tokens % r->count) {
    return fail(HARP_REQ_EINVAL, "%d tokens are not %d requests of one length: offsets are needed", tokens, r->count);
  }
  q = Requests{r->index,         r->offsets, r->index_dtype == kI64, r->offsets && r->offsets_dtype == kI64, r->count,
               tokens / r->count, tokens,     n};
  return HARP_REQ_OK;
}
int check_matrix(const void* p, int64_t ld, int dtype, int cols, bool output, const char* name) {
  if (!p) return fail(HARP_REQ_EINVAL, "%s is NULL", name);
  if (!aligned(p, dtype == kF32 ? 4 : 2)) return fail(HARP_REQ_EINVAL, "%s must be aligned to its elements", name);
  if (output ? ld < cols : ld < 0)
    return fail(HARP_REQ_EINVAL, "%s row stride %lld must be %s", name, (long long)ld,
                output ? "at least its columns (rows may not overlap)" : "non-negative");
  return HARP_REQ_OK;
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// the backward's workspace: u of all sets, B and A transposed, partial gradients
struct BackwardPlan {
  bool together;  // the sets' parts of dx in one pass, their ranks one after the other
  size_t u, bt, at, part, total;  // offsets
};
BackwardPlan backward_plan(int tokens, int K, int N, int n, int rank, int count, int sets) {
  BackwardPlan w{};
  const size_t rp = rank_pad(rank);
  GradParams g{};
  g.req.count = count;
  g.req.tokens = tokens;
  g.req.n = n;
  g.r = rank;
  g.rp = (int)rp;
  g.parts = 2 * sets;
  for (int i = 0; i < sets; ++i) {
    g.part[2 * i].C = K;
    g.part[2 * i + 1].C = N;
  }
  w.together = (int)rp * sets <= kMaxRank;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t r = at;
    at += align256(bytes);
    return r;
  };
  w.u = take((size_t)tokens * rp * sets * 4);
  w.bt = take((size_t)sets * n * rank * N * 2);
  w.at = take((size_t)sets * n * rp * K * 2);
  const int splits = grad_splits(g);
  w.part = take(splits > 1 ? (size_t)splits * grad_values(g) * 4 : 0);
  w.total = at;
  return w;
}

}  // namespace

extern "C" {

const char* harp_req_last_error(void) { return g_last_error.c_str(); }

int harp_req_qk_norm_rope_forward(const harp_req_axes_t* axes, const harp_req_positions_t* positions,
                                  const harp_req_heads_t* heads, int batch, int seq, int dtype, void* stream) {
  RopeParams p{};
  const int rc = rope_inputs(p, axes, positions, heads, batch, seq, dtype, false);
  if (rc) return rc;
  if (!(p.t[0].H + p.t[1].H) || !((int64_t)batch * seq)) return ok();
  return launched(launch_rope_forward(p, (hipStream_t)stream), "QK norm and rotation");
}

size_t harp_req_qk_backward_workspace_bytes(int batch, int seq, int d, int q_heads, int k_heads) {
  if (check_batch(batch, seq)) return (size_t)-1;
  if (d < 8 || d % 8 || d > kMaxRopeDim || q_heads < 0 || k_heads < 0 ||
      (int64_t)batch * seq * ((int64_t)q_heads + k_heads) > kMaxRows) {
    fail(HARP_REQ_EINVAL, "d=%d, q_heads=%d, k_heads=%d: no such call", d, q_heads, k_heads);
    return (size_t)-1;
  }
  RopeParams p{};
  p.B = batch;
  p.S = seq;
  p.D = d;
  p.t[0].H = q_heads;
  p.t[1].H = k_heads;
  int n[2];
  rope_bwd_blocks(p, n);
  return ((size_t)n[0] + n[1]) * d * sizeof(float);
}

int harp_req_qk_norm_rope_backward(const harp_req_axes_t* axes, const harp_req_positions_t* positions,
                                   const harp_req_heads_t* heads, int batch, int seq, int dtype, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  RopeParams p{};
  int rc = rope_inputs(p, axes, positions, heads, batch, seq, dtype, true);
  if (rc) return rc;
  if (!(p.t[0].H + p.t[1].H) || !((int64_t)batch * seq)) return ok();
  // a tensor without a norm is turned back by the forward kernel, the others by the backward kernel
  RopeParams turn = p, back = p;
  void* gw[2] = {nullptr, nullptr};
  int gw_f32[2] = {0, 0};
  for (int i = 0; i < 2; ++i) {
    if (p.t[i].norm) {
      turn.t[i].H = 0;
      gw[i] = p.t[i].H ? heads[i].grad_weight : nullptr;
      gw_f32[i] = p.t[i].w_f32;
    } else {
      back.t[i].H = 0;
      turn.t[i].x = p.t[i].dy;
      turn.t[i].sx = p.t[i].sdy;
    }
  }
  int blocks[2];
  rope_bwd_blocks(back, blocks);
  if (gw[0] || gw[1]) {
    const size_t need = ((size_t)blocks[0] + blocks[1]) * p.D * sizeof(float);
    if (!workspace || workspace_bytes < need)
      return fail(HARP_REQ_ENOMEM, "workspace of %zu bytes is smaller than the %zu bytes needed",
                  workspace ? workspace_bytes : (size_t)0, need);
    if (!aligned(workspace, 16)) return fail(HARP_REQ_EINVAL, "workspace must be 16-byte aligned");
    back.wpart = (float*)workspace;
  }
  if (turn.t[0].H + turn.t[1].H &&
      (rc = launched(launch_rope_forward(turn, (hipStream_t)stream), "rotation backward")))
    return rc;
  if (back.t[0].H + back.t[1].H &&
      (rc = launched(launch_rope_backward(back, (hipStream_t)stream), "QK norm and rotation backward")))
    return rc;
  if (!back.wpart) return ok();
  return launched(launch_rope_wgrad(back.wpart, blocks, p.D, gw, gw_f32, (hipStream_t)stream),
                  "weight-gradient reduction");
}

int harp_req_rope_table(const harp_req_axes_t* axes, const harp_req_positions_t* positions, int batch, int seq,
                        float* table, void* stream) {
  RopeAxes ax;
  RopePos pos;
  int rc, D;
  if ((rc = check_axes(axes, ax, D))) return rc;
  if ((rc = check_batch(batch, seq))) return rc;
  if (!((int64_t)batch * seq)) return ok();
  if ((rc = check_positions(positions, pos))) return rc;
  if (!table || !aligned(table, 8)) return fail(HARP_REQ_EINVAL, "table must be an 8-byte aligned device pointer");
  return launched(launch_rope_table(RopeTable{ax, pos, seq, D / 2, (int64_t)batch * seq, (float2*)table}, (hipStream_t)stream),
                  "rotary table");
}

int harp_req_adapter_columns(int rank) {
  if (rank < 1 || rank > kMaxRank) {
    fail(HARP_REQ_EINVAL, "rank=%d: 1 to %d", rank, kMaxRank);
    return -1;
  }
  return rank_pad(rank);
}

int harp_req_add_adapters_forward(const void* x, int64_t ld_x, const void* base, int64_t ld_base, void* out,
                                  int64_t ld_out, int dtype, const harp_req_adapters_t* adapters,
                                  const harp_req_requests_t* requests, float* t, int tokens, int k_dim, int n_dim,
                                  void* stream) {
  int rc;
  Requests q;
  if (dtype != kF32 && dtype != kBf16) return fail(HARP_REQ_EINVAL, "dtype must be F32 or BF16");
  if ((rc = check_tokens(tokens))) return rc;
  if ((rc = check_adapters(adapters, k_dim, n_dim, tokens > 0))) return rc;
  if (tokens == 0) return ok();
  if ((rc = check_requests(requests, tokens, adapters->n, q))) return rc;
  if ((rc = check_matrix(x, ld_x, kBf16, k_dim, false, "x"))) return rc;
  if ((rc = check_matrix(base, ld_base, dtype, n_dim, base == out, "base"))) return rc;
  if ((rc = check_matrix(out, ld_out, dtype, n_dim, true, "out"))) return rc;
  if (base == out && ld_base != ld_out) return fail(HARP_REQ_EINVAL, "out in base's place needs base's row stride");
  if (!t || !aligned(t, 16)) return fail(HARP_REQ_EINVAL, "t must be a 16-byte aligned device pointer");
  ExpandParams e{};
  e.req = q;
  e.r = adapters->rank;
  e.rp = rank_pad(e.r);
  e.t = t;
  e.ldt = e.rp;
  e.b = adapters->b;
  e.base = base;
  e.ld_base = ld_base;
  e.out = out;
  e.ld_out = ld_out;
  e.base_f32 = e.out_f32 = dtype == kF32;
  e.N = n_dim;
  if (few_tokens(e, k_dim))
    return launched(launch_few(e, FewParams{adapters->a, adapters->scales, x, ld_x, k_dim, t}, (hipStream_t)stream),
                    "adapters (few tokens)");
  ShrinkParams s{};
  s.req = q;
  s.K = k_dim;
  s.r = e.r;
  s.rp = e.rp;
  s.ldt = e.rp;
  s.sets = 1;
  s.set[0] = ShrinkSet{adapters->a, adapters->scales, x, ld_x, t, nullptr};
  if ((rc = launched(launch_shrink(s, nullptr, (hipStream_t)stream), "adapters (x A^T)"))) return rc;
  return launched(launch_expand(e, (hipStream_t)stream), "adapters (t B^T)");
}

size_t harp_req_adapter_backward_workspace_bytes(int tokens, int k_dim, int n_dim, int n, int rank, int count,
                                                 int n_sets) {
  const harp_req_adapters_t a{nullptr, nullptr, nullptr, n, rank};
  if (check_tokens(tokens) || check_adapters(&a, k_dim, n_dim, false)) return (size_t)-1;
  if (count < 1 || count > kMaxCount || n_sets < 1 || n_sets > kMaxSets) {
    fail(HARP_REQ_EINVAL, "count=%d: 1 to 2^20, n_sets=%d: 1 to %d", count, n_sets, kMaxSets);
    return (size_t)-1;
  }
  return backward_plan(tokens, k_dim, n_dim, n, rank, count, n_sets).total;
}

int harp_req_add_adapters_backward(const harp_req_backward_set_t* sets, int n_sets, const void* x, int64_t ld_x,
                                   const harp_req_requests_t* requests, float* dx_base, int64_t ld_dx_base, void* dx,
                                   int64_t ld_dx, int tokens, int k_dim, int n_dim, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  int rc;
  Requests q;
  if (!sets || n_sets < 1 || n_sets > kMaxSets)
    return fail(HARP_REQ_EINVAL, "sets must hold 1 to %d projections (got %d)", kMaxSets, n_sets);
  if ((rc = check_tokens(tokens))) return rc;
  const int n = sets[0].adapters.n, r = sets[0].adapters.rank;
  bool any_da = false, any_db = false;
  for (int i = 0; i < n_sets; ++i) {
    const harp_req_backward_set_t& s = sets[i];
    if ((rc = check_adapters(&s.adapters, k_dim, n_dim, tokens > 0))) return rc;
    if (s.adapters.n != n || s.adapters.rank != r)
      return fail(HARP_REQ_EINVAL, "sets[%d]: %d adapters of rank %d, sets[0] has %d of rank %d", i, s.adapters.n,
                  s.adapters.rank, n, r);
    any_da |= s.da != nullptr;
    any_db |= s.db != nullptr;
  }
  if (tokens == 0 || (!dx && !any_da && !any_db)) return ok();  // (no token: da and db are the caller's zeros)
  if ((rc = check_requests(requests, tokens, n, q))) return rc;
  for (int i = 0; i < n_sets; ++i) {
    const harp_req_backward_set_t& s = sets[i];
    if ((rc = check_matrix(s.dy, s.ld_dy, kBf16, n_dim, false, "dy"))) return rc;
    if (!aligned(s.da, 2) || !aligned(s.db, 2)) return fail(HARP_REQ_EINVAL, "da and db must be aligned to their elements");
    if (s.db && (!s.t || !aligned(s.t, 16))) return fail(HARP_REQ_EINVAL, "t must be a 16-byte aligned device pointer");
  }
  if (any_da && (rc = check_matrix(x, ld_x, kBf16, k_dim, false, "x"))) return rc;
  if (dx && (rc = check_matrix(dx, ld_dx, kBf16, k_dim, true, "dx"))) return rc;
  if (dx && dx_base && (rc = check_matrix(dx_base, ld_dx_base, kF32, k_dim, true, "dx_base"))) return rc;
  const int rp = rank_pad(r);
  const BackwardPlan w = backward_plan(tokens, k_dim, n_dim, n, r, q.count, n_sets);
  if (dx && !dx_base && n_sets > 1 && !w.together)
    return fail(HARP_REQ_EINVAL, "%d sets of rank %d need a dx_base", n_sets, r);
  if (!workspace || workspace_bytes < w.total)
    return fail(HARP_REQ_ENOMEM, "workspace of %zu bytes is smaller than the %zu bytes needed",
                workspace ? workspace_bytes : (size_t)0, w.total);
  if (!aligned(workspace, 16)) return fail(HARP_REQ_EINVAL, "workspace must be 16-byte aligned");
  char* const ws = (char*)workspace;
  float* const u = (float*)(ws + w.u);
  const int64_t ldu = (int64_t)rp * n_sets;
  uint16_t* const bt = (uint16_t*)(ws + w.bt);
  uint16_t* const at = (uint16_t*)(ws + w.at);
  const size_t bt_set = (size_t)n * r * n_dim, at_set = (size_t)n * rp * k_dim;
  hipStream_t st = (hipStream_t)stream;
  if (dx || any_da) {
    TransposeParams tp{};
    ShrinkParams s{};
    tp.n = n;
    s.req = q;
    s.K = n_dim;
    s.r = r;
    s.rp = rp;
    s.ldt = ldu;
    s.sets = n_sets;
    s.apart = 1;
    for (int i = 0; i < n_sets; ++i) {
      const harp_req_backward_set_t& e = sets[i];
      tp.part[tp.parts++] = TransposePart{e.adapters.b, bt + i * bt_set, n_dim, r, n_dim, 0};
      if (dx) {
        // rows of all sets' ranks side by side, or a matrix for each set
        uint16_t* const to = w.together ? at + (size_t)i * rp : at + i * at_set;
        tp.part[tp.parts++] = TransposePart{e.adapters.a, to, r, k_dim, w.together ? rp * n_sets : rp, rp};
      }
      s.set[i] = ShrinkSet{bt + i * bt_set, e.adapters.scales, e.dy, e.ld_dy, u + (size_t)i * rp, nullptr};
    }
    if ((rc = launched(launch_transpose(tp, st), "adapters' transpose"))) return rc;
    if ((rc = launched(launch_shrink(s, nullptr, st), "adapters (dy B)"))) return rc;
  }
  if (dx) {
    ExpandParams e{};
    e.req = q;
    e.ldt = ldu;
    e.N = k_dim;
    const int passes = w.together ? 1 : n_sets;
    for (int i = 0; i < passes; ++i) {
      e.t = u + (size_t)i * rp;
      e.b = at + (w.together ? 0 : i * at_set);
      e.r = e.rp = w.together ? rp * n_sets : rp;
      e.base = dx_base;
      e.ld_base = ld_dx_base;
      e.base_f32 = 1;
      e.out_f32 = i < passes - 1;
      e.out = e.out_f32 ? (void*)dx_base : dx;
      e.ld_out = e.out_f32 ? ld_dx_base : ld_dx;
      if ((rc = launched(launch_expand(e, st), "adapters (u A)"))) return rc;
    }
  }
  if (!any_da && !any_db) return ok();
  GradParams g{};
  g.req = q;
  g.r = r;
  g.rp = rp;
  for (int i = 0; i < n_sets; ++i) {
    const harp_req_backward_set_t& e = sets[i];
    if (e.da) g.part[g.parts++] = GradPart{x, ld_x, u + (size_t)i * rp, ldu, k_dim, 0, e.da};
    if (e.db) g.part[g.parts++] = GradPart{e.dy, e.ld_dy, e.t, rp, n_dim, 1, e.db};
  }
  // (the plan's workspace is for all sums; fewer of them may be split into more parts where it holds those)
  const size_t room = w.total - w.part, one = (size_t)grad_values(g) * 4;
  g.splits = grad_splits(g);
  if ((size_t)g.splits * one > room) g.splits = room / one > 1 ? (int)(room / one) : 1;
  g.work = (float*)(ws + w.part);
  return launched(launch_adapter_grad(g, st), "adapters' gradients");
}

size_t harp_req_qkv_workspace_bytes(int tokens, int rank, int n_outs) {
  if (check_tokens(tokens)) return (size_t)-1;
  if (rank < 1 || rank > kMaxRank || n_outs < 1 || n_outs > kMaxSets) {
    fail(HARP_REQ_EINVAL, "rank=%d: 1 to %d, n_outs=%d: 1 to %d", rank, kMaxRank, n_outs, kMaxSets);
    return (size_t)-1;
  }
  return n_outs * align256((size_t)tokens * 2 * rank_pad(rank) * 2);
}

int harp_req_qkv_project(const void* x, int64_t ld_x, int batch, int seq, int k_dim, int n_out, const float* freqs,
                         int64_t f_stride_b, int64_t f_stride_s, const harp_req_axes_t* axes,
                         const harp_req_positions_t* positions, float* table, const harp_qkv_out_t* outs,
                         const harp_req_adapters_t* adapters, int n_outs, const harp_req_requests_t* requests,
                         float* const* t, void* workspace, size_t workspace_bytes, void* stream) {
  harp_proj::ProjParams p;
  static_assert(HARP_QK_EINVAL == HARP_REQ_EINVAL && HARP_QK_EUNSUPPORTED == HARP_REQ_EUNSUPPORTED, "status values");
  int rc;
  RopeTable tab{};
  if (positions) {
    int D;
    if (freqs) return fail(HARP_REQ_EINVAL, "one rotation: freqs or positions");
    if ((rc = check_axes(axes, tab.axes, D)) || (rc = check_batch(batch, seq)) || (rc = check_positions(positions, tab.pos)))
      return rc;
    if (D != 128 || axes->half)
      return fail(HARP_REQ_EUNSUPPORTED, "the axes' widths must add up to 128 (got %d), of neighbouring pairs", D);
    if (!table || !aligned(table, 16)) return fail(HARP_REQ_EINVAL, "table must be a 16-byte aligned device pointer");
    tab.S = seq;
    tab.pairs = D / 2;
    tab.tokens = tab.pos.sb ? (int64_t)batch * seq : seq;
    tab.out = (float2*)table;
    freqs = table;
    f_stride_s = D;
    f_stride_b = tab.pos.sb ? (int64_t)seq * D : 0;
  }
  rc = harp_proj::fill_params(p, x, ld_x, batch, seq, k_dim, n_out, freqs, f_stride_b, f_stride_s, outs, n_outs);
  if (rc) return fail(rc, "%s", harp_qk_last_error());
  if ((int64_t)batch * seq > kMaxTokens) return fail(HARP_REQ_EUNSUPPORTED, "batch * seq > 2^25");
  if (!adapters) return fail(HARP_REQ_EINVAL, "adapters is NULL");
  const int tokens = batch * seq, n = adapters[0].n, r = adapters[0].rank;
  for (int i = 0; i < n_outs; ++i) {
    if ((rc = check_adapters(&adapters[i], k_dim, n_out, true))) return rc;
    if (adapters[i].n != n || adapters[i].rank != r)
      return fail(HARP_REQ_EINVAL, "adapters[%d]: %d of rank %d, adapters[0] are %d of rank %d", i, adapters[i].n,
                  adapters[i].rank, n, r);
    if (r % 8 || !aligned(adapters[i].b, 16))
      return fail(HARP_REQ_EUNSUPPORTED, "rank=%d must be a multiple of 8, b 16-byte aligned", r);
    if (t && !aligned(t[i], 16)) return fail(HARP_REQ_EINVAL, "t[%d] must be 16-byte aligned", i);
  }
  Requests q;
  if ((rc = check_requests(requests, tokens, n, q))) return rc;
  const size_t need = harp_req_qkv_workspace_bytes(tokens, r, n_outs);
  if (!workspace || workspace_bytes < need)
    return fail(HARP_REQ_ENOMEM, "workspace of %zu bytes is smaller than the %zu bytes needed",
                workspace ? workspace_bytes : (size_t)0, need);
  if (!aligned(workspace, 16)) return fail(HARP_REQ_EINVAL, "workspace must be 16-byte aligned");
  const int rp = rank_pad(r);
  ShrinkParams s{};
  harp_proj::ProjLow low{};
  s.req = low.req = q;
  s.K = k_dim;
  s.r = low.r = r;
  s.rp = low.rp = rp;
  s.ldt = rp;
  s.sets = n_outs;
  for (int i = 0; i < n_outs; ++i) {
    uint16_t* const pairs = (uint16_t*)((char*)workspace + i * (need / n_outs));
    s.set[i] = ShrinkSet{adapters[i].a, adapters[i].scales, x, ld_x, t ? t[i] : nullptr, pairs};
    low.t[i] = pairs;
    low.b[i] = (const uint16_t*)adapters[i].b;
  }
  if ((rc = launched(launch_shrink(s, positions ? &tab : nullptr, (hipStream_t)stream), "adapters (x A^T)"))) return rc;
  return launched(harp_proj::launch_proj_low(p, low, (hipStream_t)stream), "qkv projection with adapters");
}

}  // extern "C"
