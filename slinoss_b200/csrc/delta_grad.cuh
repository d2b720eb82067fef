// Gradients of one chunk of the gated delta rule, given the states before it (S0, from the forward), the gradient of the
// state after it (R) and dX, both from the backward pass along the sequence.  With Y, dec, gamma and closing as in delta.cuh:
//     Q_ts = scale dec_ts (dO_t.Y_s) (t >= s),   H_ts = dec_ts (dX_t.Y_s) (t > s)
//     dq = scale gamma (dO S0) + (Q beta) k
//     Z  = closing (Y R) + Q^T q - H^T k                      (all that reaches k_s through the row written at s, over beta_s)
//     dk = beta Z - gamma (dX S0) - (H beta) k                (the rest reaches k_t through the error at t)
//     dbeta_s = k_s.Z_s
//     dG_t = q_t.dq_t + k_t.dk_t - 2 beta_t dbeta_t,  dG_63 += <R, S1>,   dg_t = sum of dG over the chunk's tokens >= t
// (no product of 64 x 64 matrices with the decays is formed for dg: the row sums that it needs are dots of rows that are
// there).  One CTA of four warps per chunk and head; a warp owns 16 tokens, as t for dq and as s for Z, with its result rows
// in accumulators; Q and H are formed in both orientations, in registers, which costs 1/8 more products than passing them
// through shared memory would save barriers.
#pragma once

#include "delta.cuh"

namespace slx {
namespace delta {

constexpr int kGld = 72;  // halves per row of the token-major tiles of 64 value channels

template <int NT, int SI, int SC>
constexpr int grad_smem() {
  return 2 * SI * L * (NT + 8) * 2 + (SI + 2 * SC) * L * kGld * 2 + 2 * SC * 64 * (NT + 8) * 2;
}

// sum over n of the rows' accumulators times the operand tile's rows (16 of them from `tile`); both rows of the thread
template <int NT, int SI>
__device__ __forceinline__ float2 row_dots(const float (&c)[NT / 8][4], const __half *tile, int e) {
  constexpr int ld = NT + 8, plane = L * ld;
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  float x = 0.f, y = 0.f;
#pragma unroll
  for (int j = 0; j < NT / 8; ++j)
#pragma unroll
    for (int s = 0; s < SI; ++s) {
      const float2 u = __half22float2(*reinterpret_cast<const __half2 *>(tile + s * plane + g * ld + 8 * j + 2 * q));
      const float2 w = __half22float2(*reinterpret_cast<const __half2 *>(tile + s * plane + (g + 8) * ld + 8 * j + 2 * q));
      x = fmaf(c[j][0], u.x, fmaf(c[j][1], u.y, x));
      y = fmaf(c[j][2], w.x, fmaf(c[j][3], w.y, y));
    }
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    x += __shfl_xor_sync(~0u, x, d);
    y += __shfl_xor_sync(~0u, y, d);
  }
  const float f = pow2(e);
  return make_float2(x * f, y * f);
}

// a warp's 16 rows of dq or dk
template <int NT, typename TI>
__device__ __forceinline__ void store_grad(const Args &a, void *out, const float (&c)[NT / 8][4], int b, int h, int kh, int t0,
                                           int rows) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3, warp = threadIdx.x >> 5;
  const bool shared = a.heads != a.key_heads;
  const size_t row0 = ((size_t)(shared ? b * a.heads + h : b * a.key_heads + kh)) * a.T + t0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = 16 * warp + g + 8 * i;
    if (t >= rows) continue;
#pragma unroll
    for (int j = 0; j < NT / 8; ++j) {
      const int n = 8 * j + 2 * q;
      const float x = c[j][2 * i], y = c[j][2 * i + 1];
      const size_t at = (row0 + t) * a.N + n;
      if (shared) {
        float *o = static_cast<float *>(out) + at;
        if (n < a.N) o[0] = x;
        if (n + 1 < a.N) o[1] = y;
      } else {
        TI *o = static_cast<TI *>(out) + at;
        if (sizeof(TI) == 2 && (a.N & 1) == 0) {
          if (n < a.N) {
            const TI pair[2] = {from_f<TI>(x), from_f<TI>(y)};
            *reinterpret_cast<uint32_t *>(o) = *reinterpret_cast<const uint32_t *>(pair);
          }
        } else {
          if (n < a.N) o[0] = from_f<TI>(x);
          if (n + 1 < a.N) o[1] = from_f<TI>(y);
        }
      }
    }
  }
}

__device__ __forceinline__ void rescale8(__half *at, int diff) {  // eight halves times 2^diff, diff < 0
  const __half2 f = __float2half2_rn(pow2(diff));
  uint4 x = *reinterpret_cast<uint4 *>(at);
  __half2 *w = reinterpret_cast<__half2 *>(&x);
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __hmul2(w[i], f);
  *reinterpret_cast<uint4 *>(at) = x;
}
__device__ __forceinline__ int top_exp(const int *e, int n) {
  int m = __ldg(e);
  for (int i = 1; i < n; ++i) m = max(m, __ldg(e + i));
  return m;
}

template <int NT, int SI, int SC, typename TI>
__global__ void __launch_bounds__(kThreads) delta_grad_kernel(Args a) {
  using Op = Operand<TI, SI, NT>;
  using Oo = Operand<TI, SI, 64>;
  static_assert(Oo::ld == kGld, "tiles of value channels share one layout");
  constexpr int ld = NT + 8, xplane = L * kGld, splane = 64 * ld;
  extern __shared__ __align__(128) char smem[];
  __half *qs = reinterpret_cast<__half *>(smem), *ks = qs + SI * Op::plane;
  __half *os = ks + SI * Op::plane, *xs = os + SI * xplane, *ys = xs + SC * xplane;
  __half *ss = ys + SC * xplane, *rs = ss + SC * splane;
  __shared__ double G[L];
  __shared__ float gamma[L], closing[L], beta[L], dGs[L], dbs[L], wsum[L], dots[4];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int chunk = blockIdx.x, bh = blockIdx.y, b = bh / a.heads, h = bh % a.heads, kh = h / (a.heads / a.key_heads);
  const int t0 = chunk * L, rows = min(L, a.T - t0), PB = a.P16 / 16, tiles = (a.P16 + 63) / 64;
  const size_t at = (size_t)bh * a.NC + chunk;
  const Record *rec = a.rec + at;
  const int eq = rec->eq, ek = rec->ek;
  const int es = top_exp(a.est + at * PB, PB), er = top_exp(a.eds + at * PB, PB), ey = top_exp(a.ey + at * PB, PB),
            ex = top_exp(a.edx + at * PB, PB), eo = top_exp(a.edo + at * PB, PB);

  if (tid < L) {
    G[tid] = rec->G[tid];
    gamma[tid] = rec->gamma[tid];
    closing[tid] = rec->closing[tid];
    beta[tid] = rec->beta[tid];
  }
  Op::issue(qs, head_base<TI>(a.q, b, kh, t0), a.q.st, rows, a.N, a.q.vec, eq);
  Op::issue(ks, head_base<TI>(a.k, b, kh, t0), a.k.st, rows, a.N, a.k.vec, ek);

  // value channels 64 pt .. + 63: dO, dX and Y (tokens x channels), S0 and R (channels x N), each brought to one exponent
  bool first = true;
  auto load = [&](int pt) {
    const int w = min(64, a.P16 - 64 * pt);
    Oo::issue(os, head_base<TI>(a.dO, b, h, t0) + 64 * pt, a.dO.st, rows, a.P - 64 * pt, a.dO.vec, eo);
    for (int i = tid; i < SC * L * 8; i += kThreads) {
      const int pl = i / (L * 8), r = (i / 8) % L, c = (i % 8) * 8;
      const size_t src = ((at * SC + pl) * L + r) * a.P16 + 64 * pt + c;
      cp16(xs + pl * xplane + r * kGld + c, a.dx + (c < w ? src : 0), c < w);
      cp16(ys + pl * xplane + r * kGld + c, a.y + (c < w ? src : 0), c < w);
    }
    for (int i = tid; i < SC * 64 * (NT / 8); i += kThreads) {
      const int pl = i / (64 * (NT / 8)), r = (i / (NT / 8)) % 64, c = (i % (NT / 8)) * 8;
      const size_t src = ((at * SC + pl) * a.P16 + 64 * pt + r) * NT + c;
      cp16(ss + pl * splane + r * ld + c, a.st + (r < w ? src : 0), r < w);
      cp16(rs + pl * splane + r * ld + c, a.ds + (r < w ? src : 0), r < w);
    }
    cp_commit();
    cp_wait<0>();
    if (first) {
      Op::finish(qs, a.q.vec, eq);
      Op::finish(ks, a.k.vec, ek);
      first = false;
    }
    Oo::finish(os, a.dO.vec, eo);
    for (int i = tid; i < SC * L * 8; i += kThreads) {
      const int pl = i / (L * 8), r = (i / 8) % L, c = (i % 8) * 8;
      if (c < w) {
        const int dx = __ldg(a.edx + at * PB + 4 * pt + c / 16) - ex, dy = __ldg(a.ey + at * PB + 4 * pt + c / 16) - ey;
        if (dx) rescale8(xs + pl * xplane + r * kGld + c, dx);
        if (dy) rescale8(ys + pl * xplane + r * kGld + c, dy);
      }
    }
    for (int i = tid; i < SC * 64 * (NT / 8); i += kThreads) {
      const int pl = i / (64 * (NT / 8)), r = (i / (NT / 8)) % 64, c = (i % (NT / 8)) * 8;
      if (r < w) {
        const int d1 = __ldg(a.est + at * PB + 4 * pt + r / 16) - es, d2 = __ldg(a.eds + at * PB + 4 * pt + r / 16) - er;
        if (d1) rescale8(ss + pl * splane + r * ld + c, d1);
        if (d2) rescale8(rs + pl * splane + r * ld + c, d2);
      }
    }
    __syncthreads();
  };
  auto blocks = [&](int pt) { return min(64, a.P16 - 64 * pt) / 16; };
  const int r0 = 16 * warp + g, r1 = r0 + 8;
  const __half *qrow = qs + 16 * warp * ld, *krow = ks + 16 * warp * ld;
  auto load_a = [&](uint32_t (&r)[4], const __half *tile, int kb) { a_mk(r, tile + 16 * warp * kGld + 16 * kb, kGld); };

  float acc[NT / 8][4], dot = 0.f;
  float2 qdq;
  // ---- dq
  {
    float Q[8][4];
    zero(Q);
    zero(acc);
    for (int pt = 0; pt < tiles; ++pt) {
      if (pt) __syncthreads();
      load(pt);
      for (int kb = 0; kb < blocks(pt); ++kb) {
        Frag<SI> fo;
#pragma unroll
        for (int s = 0; s < SI; ++s) load_a(fo.r[s], os + s * xplane, kb);
        uint32_t bb[SC][4];
#pragma unroll
        for (int sb = 0; sb < 4; ++sb)
          if (sb <= warp) {
#pragma unroll
            for (int s = 0; s < SC; ++s) b_nk(bb[s], ys + s * xplane + 16 * sb * kGld + 16 * kb, kGld);
            mma_split<SI, SC>(Q[2 * sb], Q[2 * sb + 1], fo, bb);
          }
#pragma unroll
        for (int nb = 0; nb < NT / 16; ++nb) {
#pragma unroll
          for (int s = 0; s < SC; ++s) b_kn(bb[s], ss + s * splane + 16 * kb * ld + 16 * nb, ld);
          mma_split<SI, SC>(acc[2 * nb], acc[2 * nb + 1], fo, bb);
        }
      }
      for (int i = tid; i < blocks(pt) * 16 * (NT / 2); i += kThreads) {
        const int r = i / (NT / 2), c = (i % (NT / 2)) * 2;
        float2 x = make_float2(0.f, 0.f), y = x;
#pragma unroll
        for (int s = 0; s < SC; ++s) {
          const float2 u = __half22float2(*reinterpret_cast<const __half2 *>(ss + s * splane + r * ld + c));
          const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(rs + s * splane + r * ld + c));
          x.x += u.x;
          x.y += u.y;
          y.x += v.x;
          y.y += v.y;
        }
        dot = fmaf(x.x, y.x, fmaf(x.y, y.y, dot));
      }
    }
    const float f = a.scale * pow2(eo + ey);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i < 2 ? r0 : r1, c = 8 * j + 2 * q + (i & 1);
        Q[j][i] = j <= 2 * warp + 1 && c <= r ? Q[j][i] * f * expf((float)(G[r] - G[c])) * beta[c] : 0.f;
      }
    const float fs = a.scale * pow2(eo + es);
    times_rows(acc, gamma[r0] * fs, gamma[r1] * fs);
    const int e = floor_exp(warp_exp(Q), warp_exp(acc), ek);
    times(acc, pow2(-(e + ek)));
    const float s = pow2(-e);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
      if (kb <= warp) {
        Frag<SC> fq;
        frag_of<SC>(fq, Q[2 * kb], Q[2 * kb + 1], s);
#pragma unroll
        for (int nb = 0; nb < NT / 16; ++nb) {
          uint32_t bb[SI][4];
#pragma unroll
          for (int s2 = 0; s2 < SI; ++s2) b_kn(bb[s2], ks + s2 * Op::plane + 16 * kb * ld + 16 * nb, ld);
          mma_split<SC, SI>(acc[2 * nb], acc[2 * nb + 1], fq, bb);
        }
      }
    times(acc, pow2(e + ek));
    store_grad<NT, TI>(a, a.dq, acc, b, h, kh, t0, rows);
    qdq = row_dots<NT, SI>(acc, qrow, eq);
  }
  // ---- Z
  float2 w, db;
  {
    float Q[8][4], H[8][4];
    zero(Q);
    zero(H);
    zero(acc);
    for (int pt = 0; pt < tiles; ++pt) {
      if (tiles > 1) {
        __syncthreads();
        load(pt);
      }
      for (int kb = 0; kb < blocks(pt); ++kb) {
        Frag<SC> fy;
#pragma unroll
        for (int s = 0; s < SC; ++s) load_a(fy.r[s], ys + s * xplane, kb);
#pragma unroll
        for (int tb = 0; tb < 4; ++tb)
          if (tb >= warp) {
            uint32_t bo[SI][4], bx[SC][4];
#pragma unroll
            for (int s = 0; s < SI; ++s) b_nk(bo[s], os + s * xplane + 16 * tb * kGld + 16 * kb, kGld);
            mma_split<SC, SI>(Q[2 * tb], Q[2 * tb + 1], fy, bo);
#pragma unroll
            for (int s = 0; s < SC; ++s) b_nk(bx[s], xs + s * xplane + 16 * tb * kGld + 16 * kb, kGld);
            mma_split<SC, SC>(H[2 * tb], H[2 * tb + 1], fy, bx);
          }
#pragma unroll
        for (int nb = 0; nb < NT / 16; ++nb) {
          uint32_t bb[SC][4];
#pragma unroll
          for (int s = 0; s < SC; ++s) b_kn(bb[s], rs + s * splane + 16 * kb * ld + 16 * nb, ld);
          mma_split<SC, SC>(acc[2 * nb], acc[2 * nb + 1], fy, bb);
        }
      }
    }
    const float fr = pow2(ey + er);
    times_rows(acc, closing[r0] * fr, closing[r1] * fr);
    w = row_dots<NT, SI>(acc, krow, ek);
    const float fq = a.scale * pow2(ey + eo), fh = -pow2(ey + ex);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = i < 2 ? r0 : r1, t = 8 * j + 2 * q + (i & 1);
        const float dec = t >= s ? expf((float)(G[t] - G[s])) : 0.f;
        Q[j][i] = t >= s ? Q[j][i] * fq * dec : 0.f;
        H[j][i] = t > s ? H[j][i] * fh * dec : 0.f;
      }
    const int ec = warp_exp(acc), e1 = floor_exp(warp_exp(Q), ec, eq);
    const int e2 = floor_exp(warp_exp(H), max(ec, e1 + eq + 21) + 1, ek);
    times(acc, pow2(-(e1 + eq)));
    const float s1 = pow2(-e1), s2 = pow2(-e2);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
      if (kb >= warp) {
        Frag<SC> f;
        frag_of<SC>(f, Q[2 * kb], Q[2 * kb + 1], s1);
#pragma unroll
        for (int nb = 0; nb < NT / 16; ++nb) {
          uint32_t bb[SI][4];
#pragma unroll
          for (int s = 0; s < SI; ++s) b_kn(bb[s], qs + s * Op::plane + 16 * kb * ld + 16 * nb, ld);
          mma_split<SC, SI>(acc[2 * nb], acc[2 * nb + 1], f, bb);
        }
      }
    times(acc, pow2(e1 + eq - (e2 + ek)));
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
      if (kb >= warp) {
        Frag<SC> f;
        frag_of<SC>(f, H[2 * kb], H[2 * kb + 1], s2);
#pragma unroll
        for (int nb = 0; nb < NT / 16; ++nb) {
          uint32_t bb[SI][4];
#pragma unroll
          for (int s = 0; s < SI; ++s) b_kn(bb[s], ks + s * Op::plane + 16 * kb * ld + 16 * nb, ld);
          mma_split<SC, SI>(acc[2 * nb], acc[2 * nb + 1], f, bb);
        }
      }
    times(acc, pow2(e2 + ek));
    db = row_dots<NT, SI>(acc, krow, ek);
    times_rows(acc, beta[r0], beta[r1]);
  }
  // ---- dk = beta Z - gamma (dX S0) - (H beta) k
  {
    float H[8][4];
    zero(H);
    // -gamma dX as an operand: gamma (which exceeds one where gates do) and a small dX both enter its exponent
    const int top = __reduce_max_sync(~0u, max(mag(gamma[r0]), mag(gamma[r1])));
    const int e3 = floor_exp(max((top >> 23) - 127 + 1, 0) + ex, warp_exp(acc), es);
    times(acc, pow2(-(e3 + es)));
    const float f0 = -gamma[r0] * pow2(ex - e3), f1 = -gamma[r1] * pow2(ex - e3);
    for (int pt = 0; pt < tiles; ++pt) {
      if (tiles > 1) {
        __syncthreads();
        load(pt);
      }
      for (int kb = 0; kb < blocks(pt); ++kb) {
        Frag<SC> fx, fg;
#pragma unroll
        for (int s = 0; s < SC; ++s) load_a(fx.r[s], xs + s * xplane, kb);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float2 x = unpack(fx.r[0][i]);
          if constexpr (SC == 2) {
            const float2 y = unpack(fx.r[1][i]);
            x.x += y.x;
            x.y += y.y;
          }
          const float f = i & 1 ? f1 : f0;
          split<SC>(x.x * f, x.y * f, &fg.r[0][i], &fg.r[SC - 1][i]);
        }
        uint32_t bb[SC][4];
#pragma unroll
        for (int sb = 0; sb < 4; ++sb)
          if (sb <= warp) {
#pragma unroll
            for (int s = 0; s < SC; ++s) b_nk(bb[s], ys + s * xplane + 16 * sb * kGld + 16 * kb, kGld);
            mma_split<SC, SC>(H[2 * sb], H[2 * sb + 1], fx, bb);
          }
#pragma unroll
        for (int nb = 0; nb < NT / 16; ++nb) {
#pragma unroll
          for (int s = 0; s < SC; ++s) b_kn(bb[s], ss + s * splane + 16 * kb * ld + 16 * nb, ld);
          mma_split<SC, SC>(acc[2 * nb], acc[2 * nb + 1], fg, bb);
        }
      }
    }
    times(acc, pow2(e3 + es));
    const float f = -pow2(ex + ey);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i < 2 ? r0 : r1, c = 8 * j + 2 * q + (i & 1);
        H[j][i] = c < r ? H[j][i] * f * expf((float)(G[r] - G[c])) * beta[c] : 0.f;
      }
    const int e = floor_exp(warp_exp(H), warp_exp(acc), ek);
    times(acc, pow2(-(e + ek)));
    const float s = pow2(-e);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
      if (kb <= warp) {
        Frag<SC> fh;
        frag_of<SC>(fh, H[2 * kb], H[2 * kb + 1], s);
#pragma unroll
        for (int nb = 0; nb < NT / 16; ++nb) {
          uint32_t bb[SI][4];
#pragma unroll
          for (int s2 = 0; s2 < SI; ++s2) b_kn(bb[s2], ks + s2 * Op::plane + 16 * kb * ld + 16 * nb, ld);
          mma_split<SC, SI>(acc[2 * nb], acc[2 * nb + 1], fh, bb);
        }
      }
    times(acc, pow2(e + ek));
    store_grad<NT, TI>(a, a.dk, acc, b, h, kh, t0, rows);
  }
  const float2 kdk = row_dots<NT, SI>(acc, krow, ek);
  // ---- gates
  dot = dot * pow2(es + er);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(~0u, dot, d);
  if (lane == 0) dots[warp] = dot;
  if (q == 0) {
    dGs[r0] = qdq.x + kdk.x - 2.f * beta[r0] * db.x;
    dGs[r1] = qdq.y + kdk.y - 2.f * beta[r1] * db.y;
    dbs[r0] = db.x;
    dbs[r1] = db.y;
    wsum[r0] = beta[r0] * w.x;
    wsum[r1] = beta[r1] * w.y;
  }
  __syncthreads();
  if (warp == 0) {
    float last = wsum[lane] + wsum[lane + 32];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) last += __shfl_xor_sync(~0u, last, d);
    last = fmaf(gamma[L - 1], dots[0] + dots[1] + dots[2] + dots[3], last);  // <R, S1>
    const float y = dGs[2 * lane + 1], x = dGs[2 * lane] + y;
    float run = x;  // of this lane's tokens and all later ones
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const float o = __shfl_down_sync(~0u, run, d);
      if (lane + d < 32) run += o;
    }
    const size_t row = (size_t)bh * a.T + t0 + 2 * lane;
    const float after = last + run - x;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (2 * lane + i < rows) {
        store_as(a.dg, a.g_dtype, row + i, i == 0 ? after + x : after + y);
        store_as(a.dbeta, a.beta_dtype, row + i, dbs[2 * lane + i]);
      }
  }
}

// dq and dk of key heads that several value heads share: the sums of theirs, in the order of the heads
template <typename TI>
__global__ void __launch_bounds__(256) delta_share_kernel(const float *pq, const float *pk, TI *dq, TI *dk, int share, int64_t per,
                                                          int64_t total) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const float *src = (blockIdx.y ? pk : pq) + (i / per) * share * per + i % per;
    float s = 0.f;
    for (int h = 0; h < share; ++h) s += src[h * per];
    (blockIdx.y ? dk : dq)[i] = from_f<TI>(s);
  }
}

}  // namespace delta
}  // namespace slx
