// One token of the gated delta rule on carried states (decode):
//     S' = a S + d k^T,   d = beta (v - a S k),   o = scale S' q = scale (a S q + d (k.q))
// The state is read and written once, 8 P N bytes per head, and that is what the step costs: both dots of a state row are
// taken in one pass over it (k.q is known beforehand), so a row goes from memory through registers and back.  Sixteen lanes
// share a row of more than 32 values (E vectors of four each), fewer a shorter one: the rows side by side in a warp meet for
// their dots in one set of exchanges.  Batch 256, 32 heads, 64 x 128 states (536 MB): 90 us a call among others with other states
// (6030 GB/s), as a plain copy of the states takes; the kernel on one set of states 86, with 32 lanes a row 102, with eight 87.6;
// four groups of rows in flight 95 and 108.
#include "common.cuh"

namespace slx {

struct DeltaStepArgs {
  const void *q, *k, *v, *g, *beta;
  int64_t q_sb, q_sh, k_sb, k_sh, v_sb, v_sh, g_sb, g_sh, b_sb, b_sh;
  int heads, share, P, N, dtype, g_dtype, beta_dtype, rows;  // rows of a CTA
  float scale;
  const float *in;
  void *o;
  float *out;
};

constexpr int kStepThreads = 128, kStepGroups = 2;

template <int kLanes, int E, bool VEC>
__global__ void __launch_bounds__(kStepThreads) gated_delta_step_kernel(DeltaStepArgs a) {
  constexpr int kSide = 32 / kLanes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / kLanes, l = lane % kLanes;
  const int bh = blockIdx.x, b = bh / a.heads, h = bh % a.heads, kh = h / a.share;
  const int row0 = blockIdx.y * a.rows, row1 = min(a.P, row0 + a.rows);
  const size_t base = (size_t)bh * a.P * a.N;
  auto col = [&](int e) { return (e * kLanes + l) * 4; };

  float4 s[kStepGroups][E];
  auto fetch = [&](int p) {
#pragma unroll
    for (int i = 0; i < kStepGroups; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int r = p + i * kSide + sub, n = col(e);
        s[i][e] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (a.in && r < row1 && n < a.N) {
          const float *at = a.in + base + (size_t)r * a.N + n;
          if (VEC) s[i][e] = __ldcs(reinterpret_cast<const float4 *>(at));
          else {
            s[i][e].x = at[0];
            if (n + 1 < a.N) s[i][e].y = at[1];
            if (n + 2 < a.N) s[i][e].z = at[2];
            if (n + 3 < a.N) s[i][e].w = at[3];
          }
        }
      }
  };
  constexpr int step = (kStepThreads / 32) * kSide * kStepGroups;
  int p = row0 + warp * kSide * kStepGroups;
  fetch(p);  // (on its way while the vectors are read)
  float k[E][4], q[E][4], kq = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = col(e) + i;
      k[e][i] = n < a.N ? load_as_f(a.k, a.dtype, b * a.k_sb + kh * a.k_sh + n) : 0.f;
      q[e][i] = n < a.N ? load_as_f(a.q, a.dtype, b * a.q_sb + kh * a.q_sh + n) : 0.f;
      kq = fmaf(k[e][i], q[e][i], kq);
    }
  auto over_lanes = [](float x) {
#pragma unroll
    for (int d = 1; d < kLanes; d <<= 1) x += __shfl_xor_sync(~0u, x, d);
    return x;
  };
  kq = over_lanes(kq);
  const float decay = expf(load_as_f(a.g, a.g_dtype, b * a.g_sb + h * a.g_sh));
  const float beta = load_as_f(a.beta, a.beta_dtype, b * a.b_sb + h * a.b_sh);
  const size_t v0 = b * a.v_sb + h * a.v_sh;
  for (; p < row1; p += step) {
#pragma unroll
    for (int i = 0; i < kStepGroups; ++i) {
      const int r = p + i * kSide + sub;
      const float v = r < row1 ? load_as_f(a.v, a.dtype, v0 + r) : 0.f;
      float sk = 0.f, sq = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float4 x = s[i][e];
        sk = fmaf(x.x, k[e][0], fmaf(x.y, k[e][1], fmaf(x.z, k[e][2], fmaf(x.w, k[e][3], sk))));
        sq = fmaf(x.x, q[e][0], fmaf(x.y, q[e][1], fmaf(x.z, q[e][2], fmaf(x.w, q[e][3], sq))));
      }
      sk = over_lanes(sk);
      sq = over_lanes(sq);
      const float d = beta * (v - decay * sk);
      if (r < row1) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int n = col(e);
          if (n >= a.N) continue;
          const float4 x = make_float4(fmaf(d, k[e][0], decay * s[i][e].x), fmaf(d, k[e][1], decay * s[i][e].y),
                                       fmaf(d, k[e][2], decay * s[i][e].z), fmaf(d, k[e][3], decay * s[i][e].w));
          float *at = a.out + base + (size_t)r * a.N + n;
          if (VEC) __stcs(reinterpret_cast<float4 *>(at), x);
          else {
            at[0] = x.x;
            if (n + 1 < a.N) at[1] = x.y;
            if (n + 2 < a.N) at[2] = x.z;
            if (n + 3 < a.N) at[3] = x.w;
          }
        }
        if (l == 0) store_as(a.o, a.dtype, (size_t)bh * a.P + r, a.scale * fmaf(d, kq, decay * sq));
      }
    }
    if (p + step < row1) fetch(p + step);
  }
}

// rows of a CTA: one group of every warp where that is needed to give each SM four CTAs, up to the whole head otherwise
template <int kLanes, int E>
static int launch_step(DeltaStepArgs a, int64_t bh, bool vec, cudaStream_t st) {
  const int least = (kStepThreads / 32) * (32 / kLanes) * kStepGroups;
  a.rows = (a.P + least - 1) / least * least;
  while (a.rows > least && bh * ((a.P + a.rows - 1) / a.rows) < 4 * kB200Sms) a.rows -= least;
  const dim3 grid((unsigned)bh, (a.P + a.rows - 1) / a.rows);
  if (vec) gated_delta_step_kernel<kLanes, E, true><<<grid, kStepThreads, 0, st>>>(a);
  else gated_delta_step_kernel<kLanes, E, false><<<grid, kStepThreads, 0, st>>>(a);
  return check_launch("gated_delta_step_kernel");
}

}  // namespace slx

using namespace slx;

extern "C" int slx_gated_delta_step(const slx_gated_delta_shape *s, const void *q, const void *k, const void *v, const void *g,
                                    const void *beta, const float *state_in, void *o, float *state_out, void *stream) {
  SLX_REQUIRE(s, SLX_E_NULL, "gated_delta_step: shape is NULL");
  SLX_REQUIRE(q && k && v && g && beta && o && state_out, SLX_E_NULL, "gated_delta_step: a required pointer is NULL");
  SLX_REQUIRE(s->batch > 0 && s->heads > 0 && s->key_heads > 0 && s->P > 0 && s->N > 0 && s->T == 1, SLX_E_SHAPE,
              "gated_delta_step: sizes must be positive and T 1 (batch %d, heads %d, key_heads %d, T %d, P %d, N %d)", s->batch,
              s->heads, s->key_heads, s->T, s->P, s->N);
  SLX_REQUIRE(s->heads % s->key_heads == 0, SLX_E_SHAPE, "gated_delta_step: heads (%d) must be a multiple of key_heads (%d)",
              s->heads, s->key_heads);
  for (int dt : {s->dtype, s->g_dtype, s->beta_dtype})
    SLX_REQUIRE(dt == SLX_F32 || dt == SLX_BF16 || dt == SLX_F16, SLX_E_DTYPE, "gated_delta_step: unknown dtype %d", dt);
  SLX_REQUIRE(s->N <= 128, SLX_E_UNSUPPORTED, "gated_delta_step: key dim N must be at most 128, got %d", s->N);
  SLX_REQUIRE(s->P <= 256, SLX_E_UNSUPPORTED, "gated_delta_step: value dim P must be at most 256, got %d", s->P);
  const size_t bytes = (size_t)s->batch * s->heads * s->P * s->N * 4;
  const uintptr_t from = reinterpret_cast<uintptr_t>(state_in), to = reinterpret_cast<uintptr_t>(state_out);
  SLX_REQUIRE(!state_in || from == to || from + bytes <= to || to + bytes <= from, SLX_E_SHAPE,
              "gated_delta_step: state_in and state_out must be the same or not overlap");
  DeltaStepArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.g = g;
  a.beta = beta;
  const bool many = s->batch > 1, heads = s->heads > 1, keys = s->key_heads > 1;
  a.q_sb = many ? s->q_stride[0] : 0;
  a.q_sh = keys ? s->q_stride[1] : 0;
  a.k_sb = many ? s->k_stride[0] : 0;
  a.k_sh = keys ? s->k_stride[1] : 0;
  a.v_sb = many ? s->v_stride[0] : 0;
  a.v_sh = heads ? s->v_stride[1] : 0;
  a.g_sb = many ? s->g_stride[0] : 0;
  a.g_sh = heads ? s->g_stride[1] : 0;
  a.b_sb = many ? s->beta_stride[0] : 0;
  a.b_sh = heads ? s->beta_stride[1] : 0;
  a.heads = s->heads;
  a.share = s->heads / s->key_heads;
  a.P = s->P;
  a.N = s->N;
  a.dtype = s->dtype;
  a.g_dtype = s->g_dtype;
  a.beta_dtype = s->beta_dtype;
  a.scale = s->scale;
  a.in = state_in;
  a.o = o;
  a.out = state_out;
  const bool vec = s->N % 4 == 0 && ((reinterpret_cast<uintptr_t>(state_in) | reinterpret_cast<uintptr_t>(state_out)) & 15) == 0;
  const int64_t bh = (int64_t)s->batch * s->heads;
  SLX_REQUIRE(bh <= 0x7fffffff, SLX_E_UNSUPPORTED, "gated_delta_step: too many heads");
  cudaStream_t st = as_stream(stream);
  if (s->N > 64) return launch_step<16, 2>(a, bh, vec, st);
  if (s->N > 32) return launch_step<16, 1>(a, bh, vec, st);
  if (s->N > 16) return launch_step<8, 1>(a, bh, vec, st);
  return launch_step<4, 1>(a, bh, vec, st);
}
