// Gated delta rule: C-ABI entry points of the chunked operator (forward, backward).
//
// Forward: the chunks' triangular matrices (delta_chunk.cuh), then one pass along the sequence (delta_scan.cuh, delta_team.cuh).
// Backward: the pass back along the sequence, then the gradients of every chunk by itself (delta_grad.cuh).  What the forward
// has made of a chunk is kept for it: the matrices, the scaled tiles of k and q (in the place of k and q themselves), the states
// and the prediction errors.
#include "delta_launch.cuh"

namespace slx {
namespace delta {

struct Dims {
  int64_t BH, NC, P16, PB, NT;
  int planes;  // of computed operands: one for bf16, two otherwise
};
static Dims dims_of(const slx_gated_delta_shape *s) {
  Dims d;
  d.BH = (int64_t)s->batch * s->heads;
  d.NC = ((int64_t)s->T + L - 1) / L;
  d.P16 = (s->P + 15) / 16 * 16;
  d.PB = d.P16 / 16;
  d.NT = s->N <= 64 ? 64 : 128;
  d.planes = s->dtype == SLX_BF16 ? 1 : 2;
  return d;
}
static size_t up(size_t n) { return (n + 255) / 256 * 256; }
static size_t record_bytes(const Dims &d) { return up((size_t)(d.BH * d.NC) * sizeof(Record)); }
static size_t keys_bytes(const slx_gated_delta_shape *s, const Dims &d) {
  return up((size_t)s->batch * s->key_heads * d.NC * 2 * (s->dtype == SLX_F32 ? 2 : 1) * L * (d.NT + 8) * 2);
}
static size_t state_bytes(const Dims &d) { return up((size_t)(d.BH * d.NC * d.planes * d.P16 * (d.NT + 8)) * 2); }
static size_t value_bytes(const Dims &d) { return up((size_t)(d.BH * d.NC * d.planes * ((d.P16 + 63) / 64) * kTile) * 2); }
static size_t exp_bytes(const Dims &d) { return up((size_t)(d.BH * d.NC * d.PB) * 4); }
static size_t share_bytes(const slx_gated_delta_shape *s) {
  return s->heads == s->key_heads ? 0 : up((size_t)s->batch * s->heads * s->T * s->N * 4);
}

static int check_shape(const slx_gated_delta_shape *s, const char *what) {
  SLX_REQUIRE(s, SLX_E_NULL, "%s: shape is NULL", what);
  SLX_REQUIRE(s->batch > 0 && s->heads > 0 && s->key_heads > 0 && s->T > 0 && s->P > 0 && s->N > 0, SLX_E_SHAPE,
              "%s: sizes must be positive (batch %d, heads %d, key_heads %d, T %d, P %d, N %d)", what, s->batch, s->heads,
              s->key_heads, s->T, s->P, s->N);
  SLX_REQUIRE(s->heads % s->key_heads == 0, SLX_E_SHAPE, "%s: heads (%d) must be a multiple of key_heads (%d)", what, s->heads,
              s->key_heads);
  SLX_REQUIRE(s->dtype == SLX_F32 || s->dtype == SLX_BF16 || s->dtype == SLX_F16, SLX_E_DTYPE, "%s: unknown dtype %d", what,
              s->dtype);
  SLX_REQUIRE((s->g_dtype == SLX_F32 || s->g_dtype == SLX_BF16 || s->g_dtype == SLX_F16) &&
                  (s->beta_dtype == SLX_F32 || s->beta_dtype == SLX_BF16 || s->beta_dtype == SLX_F16),
              SLX_E_DTYPE, "%s: unknown gate dtype", what);
  SLX_REQUIRE(s->N <= 128, SLX_E_UNSUPPORTED, "%s: key dim N must be at most 128, got %d", what, s->N);
  SLX_REQUIRE(s->P <= 256, SLX_E_UNSUPPORTED, "%s: value dim P must be at most 256, got %d", what, s->P);
  SLX_REQUIRE((int64_t)s->batch * s->heads <= 65535, SLX_E_UNSUPPORTED, "%s: batch * heads must be at most 65535", what);
  return SLX_OK;
}

static Rows rows_of(const void *p, const int64_t *st, const slx_gated_delta_shape *s, int heads, int width, int size) {
  Rows r;
  r.p = p;
  r.sb = s->batch > 1 ? st[0] : 0;  // (the stride of an axis of one element means nothing)
  r.sh = heads > 1 ? st[1] : 0;
  r.st = s->T > 1 ? st[2] : 0;
  const int v = 16 / size;
  r.vec = (reinterpret_cast<uintptr_t>(p) & 15) == 0 && r.sb % v == 0 && r.sh % v == 0 && r.st % v == 0 && width % v == 0;
  return r;
}
static Args args_of(const slx_gated_delta_shape *s, const Dims &d) {
  Args a{};
  a.batch = s->batch;
  a.heads = s->heads;
  a.key_heads = s->key_heads;
  a.T = s->T;
  a.P = s->P;
  a.N = s->N;
  a.NC = (int)d.NC;
  a.P16 = (int)d.P16;
  a.scale = s->scale;
  a.g_dtype = s->g_dtype;
  a.beta_dtype = s->beta_dtype;
  return a;
}

// Zero: teams of eight warps on 16 value channels, where each can have an SM to itself, or two rounds of teams fill the SMs well.
// Else the warps of a CTA that hold 16 channels each: as many as there are, up to four, which share a CTA's tiles.  Measured
// (T 2048, N 128, P 64, bf16, forward and training, us) with 128 blocks of 16 channels: teams 102 / 275, warps 176 / 444; with
// 256: 194 / 511 and 209 / 550; with 320: 270 / 700 and 231 / 617.  Between 148 and 222 blocks teams take what they take with
// 256, and the warps, whose time grows with the blocks, less.  Fewer than four warps a CTA are never faster (512 blocks: four
// 275 / 767, two 323 / 873, one 413 / 1065).
static int scan_warps(const Dims &d) {
  const int64_t blocks = d.BH * d.PB, two_rounds = 2 * kB200Sms;
  if (blocks <= kB200Sms || (4 * blocks >= 3 * two_rounds && blocks <= two_rounds)) return 0;
  return (int)(d.PB < 4 ? d.PB : 4);
}

}  // namespace delta
}  // namespace slx

using namespace slx;
using namespace slx::delta;

// what the forward keeps, in this order: records, tiles of k and q, states, errors, exponents of both
struct Kept {
  size_t keys, states, values, exps, bytes;
};
static Kept kept_of(const slx_gated_delta_shape *s, const Dims &d) {
  Kept k;
  k.keys = record_bytes(d);
  k.states = k.keys + keys_bytes(s, d);
  k.values = k.states + state_bytes(d);
  k.exps = k.values + value_bytes(d);
  k.bytes = k.exps + 2 * exp_bytes(d);
  return k;
}
static void place_kept(Args &a, const Kept &k, const Dims &d, const void *residual) {
  char *r = static_cast<char *>(const_cast<void *>(residual));
  a.rec = reinterpret_cast<Record *>(r);
  a.kq = reinterpret_cast<__half *>(r + k.keys);
  a.st = reinterpret_cast<__half *>(r + k.states);
  a.y = reinterpret_cast<__half *>(r + k.values);
  a.est = reinterpret_cast<int *>(r + k.exps);
  a.ey = reinterpret_cast<int *>(r + k.exps + exp_bytes(d));
}

extern "C" size_t slx_gated_delta_fwd_workspace_bytes(const slx_gated_delta_shape *s) {
  if (check_shape(s, "gated_delta") != SLX_OK) return 0;
  const Dims d = dims_of(s);
  return record_bytes(d) + keys_bytes(s, d);
}
extern "C" size_t slx_gated_delta_residual_bytes(const slx_gated_delta_shape *s) {
  return check_shape(s, "gated_delta") == SLX_OK ? kept_of(s, dims_of(s)).bytes : 0;
}
extern "C" size_t slx_gated_delta_bwd_workspace_bytes(const slx_gated_delta_shape *s) {
  if (check_shape(s, "gated_delta") != SLX_OK) return 0;
  const Dims d = dims_of(s);
  return state_bytes(d) + value_bytes(d) + 3 * exp_bytes(d) + 2 * share_bytes(s);
}

static int check_workspace(const char *what, const void *workspace, size_t have, size_t need) {
  SLX_REQUIRE(workspace, SLX_E_NULL, "%s: workspace is NULL", what);
  SLX_REQUIRE(have >= need, SLX_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, have, need);
  SLX_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, SLX_E_WORKSPACE, "%s: workspace must be 256-byte aligned",
              what);
  return SLX_OK;
}
static bool known(int dtype) { return dtype == SLX_F32 || dtype == SLX_BF16 || dtype == SLX_F16; }

// per activation dtype, each in a file of its own (the instances take the compiler minutes)
#define SLX_DELTA_DISPATCH(call_)                                     \
  do {                                                                \
    if (s->dtype == SLX_BF16) return call_##_as<__nv_bfloat16> ARGS_; \
    if (s->dtype == SLX_F16) return call_##_as<__half> ARGS_;         \
    return call_##_as<float> ARGS_;                                   \
  } while (0)

extern "C" int slx_gated_delta_fwd(const slx_gated_delta_shape *s, const void *q, const void *k, const void *v, const void *g,
                                   const void *beta, const void *initial_state, int32_t initial_dtype, void *o,
                                   float *final_state, void *residual, void *workspace, size_t workspace_bytes, void *stream) {
  if (const int rc = check_shape(s, "gated_delta_fwd")) return rc;
  SLX_REQUIRE(q && k && v && g && beta, SLX_E_NULL, "gated_delta_fwd: q, k, v, g and beta must not be NULL");
  SLX_REQUIRE(!initial_state || known(initial_dtype), SLX_E_DTYPE, "gated_delta_fwd: unknown initial_dtype %d", initial_dtype);
  const Dims d = dims_of(s);
  Args a = args_of(s, d);
  const int size = s->dtype == SLX_F32 ? 4 : 2;
  a.q = rows_of(q, s->q_stride, s, s->key_heads, s->N, size);
  a.k = rows_of(k, s->k_stride, s, s->key_heads, s->N, size);
  a.v = rows_of(v, s->v_stride, s, s->heads, s->P, size);
  a.g = rows_of(g, s->g_stride, s, s->heads, 1, 4);
  a.beta = rows_of(beta, s->beta_stride, s, s->heads, 1, 4);
  a.init = initial_state;
  a.init_dtype = initial_dtype;
  a.o = o;
  a.final_state = final_state;
  if (residual) {
    SLX_REQUIRE((reinterpret_cast<uintptr_t>(residual) & 255) == 0, SLX_E_WORKSPACE,
                "gated_delta_fwd: residual must be 256-byte aligned");
    place_kept(a, kept_of(s, d), d, residual);
  } else {
    if (const int rc = check_workspace("gated_delta_fwd", workspace, workspace_bytes, slx_gated_delta_fwd_workspace_bytes(s)))
      return rc;
    a.rec = static_cast<Record *>(workspace);
    a.kq = reinterpret_cast<__half *>(static_cast<char *>(workspace) + record_bytes(d));
  }
  const int warps = scan_warps(d);
  cudaStream_t st = as_stream(stream);
#define ARGS_ (a, (int)d.NT, warps, st)
  SLX_DELTA_DISPATCH(launch_fwd);
#undef ARGS_
}

extern "C" int slx_gated_delta_bwd(const slx_gated_delta_shape *s, const void *residual, const void *d_o, const void *d_final,
                                   int32_t d_final_dtype, void *dq, void *dk, void *dv, void *dg, void *dbeta, void *d_initial,
                                   int32_t d_initial_dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (const int rc = check_shape(s, "gated_delta_bwd")) return rc;
  SLX_REQUIRE(residual && d_o && dq && dk && dv && dg && dbeta, SLX_E_NULL, "gated_delta_bwd: a required pointer is NULL");
  SLX_REQUIRE(!d_final || known(d_final_dtype), SLX_E_DTYPE, "gated_delta_bwd: unknown d_final_dtype %d", d_final_dtype);
  SLX_REQUIRE(!d_initial || known(d_initial_dtype), SLX_E_DTYPE, "gated_delta_bwd: unknown d_initial_dtype %d", d_initial_dtype);
  const Dims d = dims_of(s);
  if (const int rc = check_workspace("gated_delta_bwd", workspace, workspace_bytes, slx_gated_delta_bwd_workspace_bytes(s)))
    return rc;
  SLX_REQUIRE((reinterpret_cast<uintptr_t>(residual) & 255) == 0, SLX_E_WORKSPACE,
              "gated_delta_bwd: residual must be 256-byte aligned");
  char *w = static_cast<char *>(workspace);
  Args a = args_of(s, d);
  place_kept(a, kept_of(s, d), d, residual);
  const int64_t o_stride[3] = {(int64_t)s->heads * s->T * s->P, (int64_t)s->T * s->P, s->P};
  a.dO = rows_of(d_o, o_stride, s, s->heads, s->P, s->dtype == SLX_F32 ? 4 : 2);
  a.ds = reinterpret_cast<__half *>(w);
  w += state_bytes(d);
  a.dx = reinterpret_cast<__half *>(w);
  w += value_bytes(d);
  a.eds = reinterpret_cast<int *>(w);
  a.edx = reinterpret_cast<int *>(w + exp_bytes(d));
  a.edo = reinterpret_cast<int *>(w + 2 * exp_bytes(d));
  w += 3 * exp_bytes(d);
  a.dq = s->heads == s->key_heads ? dq : w;
  a.dk = s->heads == s->key_heads ? dk : w + share_bytes(s);
  a.d_final = d_final;
  a.d_final_dtype = d_final_dtype;
  a.d_init = d_initial;
  a.d_init_dtype = d_initial_dtype;
  a.dv = dv;
  a.dg = dg;
  a.dbeta = dbeta;
  const int warps = scan_warps(d);
  cudaStream_t st = as_stream(stream);
#define ARGS_ (a, (int)d.NT, dq, dk, warps, st)
  SLX_DELTA_DISPATCH(launch_bwd);
#undef ARGS_
}
