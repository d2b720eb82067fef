// Gradients of one chunk of the gated delta rule, given the states before it (S0, from the forward), the gradient of the
// state after it (R) and dX, both from the backward pass along the sequence.  With Y, dec, gamma and closing as in delta.cuh:
//     Q_ts = scale dec_ts (dO_t.Y_s) (t >= s),   H_ts = dec_ts (dX_t.Y_s) (t > s)
//     dq = scale gamma (dO S0) + (Q beta) k
//     Z  = closing (Y R) + Q^T q - H^T k                      (all that reaches k_s through the row written at s, over beta_s)
//     dk = beta Z - gamma (dX S0) - (H beta) k                (the rest reaches k_t through the error at t)
// What the row written at s passes to a later t is beta_s C_ts, C_ts = Q_ts q_t.k_s - H_ts k_t.k_s, and with that
//     dbeta_s = closing_s Y_s.(R k_s) + sum of C_ts over t >= s
//     dg_t = gamma_63 <R, S0> + sum over r >= t of gamma_r (scale dO_r.(S0 q_r) - dX_r.(S0 k_r))
//            + sum over s < t of beta_s closing_s Y_s.(R k_s) + sum over s < t <= r of beta_s C_rs
// : all that crosses the gate at t, term by term with its decay, so that a gate which is nearly closed has a gradient as small
// and as exact as what it lets through.  (The suffix sum of q.dq + k.dk - 2 beta dbeta is the same in exact arithmetic, but its
// terms of order one cancel: with g = -5 throughout it was off by 0.3 of dg in fp32 and by 180 times dg in bf16.)
// One CTA of four warps per chunk and head; a warp owns 16 tokens, as t for dq and as s for Z, with its result rows in
// accumulators; Q and H are formed in both orientations, in registers, which costs 1/8 more products than passing them through
// shared memory would save barriers.
//
// 16384 chunks of one head each (N 128, P 64, bf16): 1058 us at two CTAs an SM (106 KB and 241 registers a thread), of which the
// gates' terms are 160; 160 KB a chunk through HBM would take 400.  1.5 instructions a clock and SM, the tensor pipe busy 23 %: a
// warp waits for its own products and for what it reads.  fp16 with 64 columns (900 chunks, 110 KB): 85 us at two CTAs an SM.
// Without the gates' terms: 898 and 74; then eight warps a CTA, four for dO, Q and dq and four for dX, H and dk, took 1123 (at 128
// registers they spill, with one CTA an SM nothing hides the loads), and fp16 at one CTA an SM 107, which a second plane of dO
// made it.
#pragma once

#include "delta.cuh"

namespace slx {
namespace delta {

template <int NT, int SI, int SC>
constexpr int grad_smem() {
  return 2 * Operand<SI, NT>::halves * 2 + (SI + 2 * SC) * kTile * 2 + 2 * SC * 64 * (NT + 8) * 2 + kVectorBytes;
}

__device__ __forceinline__ float over_quad(float x) {
  x += __shfl_xor_sync(~0u, x, 1);
  return x + __shfl_xor_sync(~0u, x, 2);
}
__device__ __forceinline__ float over_rows(float x) {  // of the eight quads
  x += __shfl_xor_sync(~0u, x, 4);
  x += __shfl_xor_sync(~0u, x, 8);
  return x + __shfl_xor_sync(~0u, x, 16);
}

// This thread's part of the sums over n of the rows' accumulators (n of 8 columns) times the operand tile's rows (16 of them from
// `tile`); both rows of the thread
template <int NT, int SI, int n>
__device__ __forceinline__ float2 row_dots(const float (&c)[n][4], const __half *tile) {
  constexpr int ld = NT + 8, plane = L * ld;
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  float x = 0.f, y = 0.f;
#pragma unroll
  for (int j = 0; j < n; ++j)
#pragma unroll
    for (int s = 0; s < SI; ++s) {
      const float2 u = __half22float2(*reinterpret_cast<const __half2 *>(tile + s * plane + g * ld + 8 * j + 2 * q));
      const float2 w = __half22float2(*reinterpret_cast<const __half2 *>(tile + s * plane + (g + 8) * ld + 8 * j + 2 * q));
      x = fmaf(c[j][0], u.x, fmaf(c[j][1], u.y, x));
      y = fmaf(c[j][2], w.x, fmaf(c[j][3], w.y, y));
    }
  return make_float2(x, y);
}

// A warp's 16 rows of dq or dk, from accumulators: half types through `buf` (16 x (NT + 8) halves of the warp's own) in
// 16-byte pieces, fp32 (also where heads share their keys and the sums are still to be added up) directly.
template <int NT, typename TO>
__device__ __forceinline__ void store_grad(TO *out, const float (&c)[NT / 8][4], int rows, int N, __half *buf) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  if constexpr (sizeof(TO) == 4) {
    const bool pairs = (N & 1) == 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = g + 8 * i;
      if (t >= rows) continue;
      TO *o = out + (size_t)t * N;
#pragma unroll
      for (int j = 0; j < NT / 8; ++j) {
        const int n = 8 * j + 2 * q;
        if (pairs) {
          if (n < N) *reinterpret_cast<float2 *>(o + n) = make_float2(c[j][2 * i], c[j][2 * i + 1]);
        } else {
          if (n < N) o[n] = c[j][2 * i];
          if (n + 1 < N) o[n + 1] = c[j][2 * i + 1];
        }
      }
    }
  } else {
    constexpr int ld = NT + 8;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NT / 8; j += 2) {
      uint32_t r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = c[j + (i >> 1)][(i & 1) * 2], y = c[j + (i >> 1)][(i & 1) * 2 + 1];
        if constexpr (std::is_same<TO, __half>::value) r[i] = pack(x, y);
        else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
          r[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
      }
      stsm(smem_addr(buf + (lane & 15) * ld + 8 * j + (lane >> 4) * 8), r);
    }
    __syncwarp();
    if ((N & 7) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
#pragma unroll
      for (int i = 0; i < NT / 16; ++i) {
        const int t = (i * 32 + lane) / (NT / 8), n = (i * 32 + lane) % (NT / 8) * 8;
        if (t < rows && n < N)
          *reinterpret_cast<uint4 *>(out + (size_t)t * N + n) = *reinterpret_cast<const uint4 *>(buf + t * ld + n);
      }
    } else {
      for (int i = lane; i < 16 * NT; i += 32) {
        const int t = i / NT, n = i % NT;
        if (t < rows && n < N) out[(size_t)t * N + n] = reinterpret_cast<const TO *>(buf)[t * ld + n];
      }
    }
    __syncwarp();
  }
}

// Where products join sums that are there already.  The matrix instructions cut off what they add below the accumulator's last
// bit, always towards zero: sixty steps onto one accumulator were 1.2e-6 of dk in fp32, and by product they are 6e-7.  So each
// product of fp32 tensors has accumulators of its own, which are added by themselves (fp16's rounding hides it: 2 % of its time).
template <int NT, int SI, int SC>
struct Onto {
  static constexpr bool apart = SI == 2;
  float (&sum)[NT / 8][4];
  float own[apart ? NT / 8 : 1][4];
  __device__ __forceinline__ Onto(float (&c)[NT / 8][4]) : sum(c) {
    if constexpr (apart) zero(own);
  }
  template <int SB>
  __device__ __forceinline__ void add(const Frag<SC> &f, const __half *tile, int plane, int kb) {
    if constexpr (apart) tile_cols<SC, SB, NT, 2>(own, f, tile, plane, kb);
    else tile_cols<SC, SB, NT>(sum, f, tile, plane, kb);
  }
  __device__ __forceinline__ void join() {
    if constexpr (apart) {
#pragma unroll
      for (int j = 0; j < NT / 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[j][i] += own[j][i];
    }
  }
};

template <int NT, int SI, int SC, typename TI>
__global__ void __launch_bounds__(kThreads) delta_grad_kernel(Args a) {
  using Op = Operand<SI, NT>;
  constexpr int ld = NT + 8, splane = 64 * ld;
  extern __shared__ __align__(128) char smem[];
  __half *ks = reinterpret_cast<__half *>(smem), *qs = ks + Op::halves;
  __half *os = qs + Op::halves, *xs = os + SI * kTile, *ys = xs + SC * kTile;  // tokens x channels: dO, dX, Y
  __half *ss = ys + SC * kTile, *rs = ss + SC * splane;                          // channels x N: S0, R
  float *gamma = reinterpret_cast<float *>(rs + SC * splane), *closing = gamma + L, *beta = closing + L;
  float *rise = beta + L + 32, *fall = rise + L, *near = fall + 96;
  // per token: what it reads of S0, dbeta, what its row passes on behind the chunk; what crosses its gate from the tokens of its
  // block of 16, and (by block) from each earlier block to it
  __shared__ float reads[L], dbs[L], wsum[L], dots[4];
  __shared__ __align__(8) float near_cross[L], far_cross[3][L];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int chunk = blockIdx.x, bh = blockIdx.y, b = bh / a.heads, h = bh % a.heads, kh = h / (a.heads / a.key_heads);
  const int t0 = chunk * L, rows = min(L, a.T - t0), PB = a.P16 / 16, tiles = (a.P16 + 63) / 64;
  const size_t at = (size_t)bh * a.NC + chunk;
  const Record *rec = a.rec + at;

  // Tiles of channels come with an exponent per 16 of them.  Where channels are summed over, the A operand of a block takes
  // what its two exponents lie below the largest such sum.  Lane l holds those of block l.
  const int none = -100000;
  int es = none, er = none, ey = none, ex = none, eo = none;
  if (lane < PB) {
    es = __ldg(a.est + at * PB + lane);
    er = __ldg(a.eds + at * PB + lane);
    ey = __ldg(a.ey + at * PB + lane);
    ex = __ldg(a.edx + at * PB + lane);
    eo = __ldg(a.edo + at * PB + lane);
  }
  const int eq = rec->eq, ek = rec->ek;
  const int eo_top = __reduce_max_sync(~0u, eo);  // (dO is brought to one exponent as it is read)
  copy_bytes<2 * Op::halves * 2>(ks, a.kq + ((size_t)(b * a.key_heads + kh) * a.NC + chunk) * 2 * Op::halves);
  copy_bytes<kVectorBytes>(gamma, rec->gamma);

  // value channels 64 pt .. + 63: dO, dX and Y (tokens x channels), S0 and R (channels x N)
  auto load = [&](int pt) {
    const int w = min(64, a.P16 - 64 * pt);
#pragma unroll
    for (int s = 0; s < SC; ++s) {
      const size_t tile = ((at * SC + s) * tiles + pt) * kTile, state = ((at * SC + s) * a.P16 + 64 * pt) * ld;
      copy_bytes<kTile * 2>(xs + s * kTile, a.dx + tile);
      copy_bytes<kTile * 2>(ys + s * kTile, a.y + tile);
#pragma unroll 1
      for (int i = tid * 8; i < w * ld; i += kThreads * 8) {
        cp16(ss + s * splane + i, a.st + state + i, true);
        cp16(rs + s * splane + i, a.ds + state + i, true);
      }
    }
    cp_commit();
    Pieces<TI, 64> o;
    o.load(head_base<TI>(a.dO, b, h, t0) + 64 * pt, a.dO.st, rows, a.P - 64 * pt, a.dO.vec, os);
    o.template store<SI, false>(os, nullptr, eo_top);
    cp_wait<0>();
    __syncthreads();
  };
  auto below = [&](int e, int top, int pt, int kb) { return __shfl_sync(~0u, e, 4 * pt + kb) - top; };
  const int r0 = 16 * warp + g, r1 = r0 + 8;
  const __half *krow = ks + 16 * warp * ld;
  auto load_a = [&](Frag<SC> &f, const __half *tile, int planes, int kb) {  // (dO may have one where dX has two)
#pragma unroll
    for (int s = 0; s < SC; ++s) {
      if (s < planes) a_mk(f.r[s], tile + s * kTile + 16 * warp * kTileLd + 16 * kb, kTileLd);
      else f.r[s][0] = f.r[s][1] = f.r[s][2] = f.r[s][3] = 0;
    }
  };
  auto load_b = [&](auto &f, const __half *tile, int rb, int kb) {
    constexpr int planes = sizeof(f) / 16;
#pragma unroll
    for (int s = 0; s < planes; ++s) b_nk(f[s], tile + s * kTile + 16 * rb * kTileLd + 16 * kb, kTileLd);
  };
  float acc[NT / 8][4];
  // ---- Z, this warp's tokens as s
  int unit;  // of acc
  float2 w, db;
  float dot = 0.f;
  {
    float Q[8][4], H[8][4];
    zero(Q);
    zero(H);
    zero(acc);
    const int yx = ey + ex, yr = ey + er, sr = es + er;
    const int y_top = __reduce_max_sync(~0u, ey), yx_top = __reduce_max_sync(~0u, yx), yr_top = __reduce_max_sync(~0u, yr),
              sr_top = __reduce_max_sync(~0u, sr);
#pragma unroll 1
    for (int pt = 0; pt < tiles; ++pt) {
      if (pt) __syncthreads();
      load(pt);
      const int blocks = min(4, PB - 4 * pt);
#pragma unroll 1
      for (int kb = 0; kb < blocks; ++kb) {
        Frag<SC> fy;
        load_a(fy, ys, SC, kb);
        const Frag<SC> f1 = scaled(fy, below(ey, y_top, pt, kb)), f2 = scaled(fy, below(yx, yx_top, pt, kb));
#pragma unroll
        for (int tb = 0; tb < 4; ++tb)
          if (tb >= warp) {
            uint32_t bo[SI][4], bx[SC][4];
            load_b(bo, os, tb, kb);
            load_b(bx, xs, tb, kb);
            mma_split<SC, SI>(Q[2 * tb], Q[2 * tb + 1], f1, bo);
            mma_split<SC, SC>(H[2 * tb], H[2 * tb + 1], f2, bx);
          }
        tile_cols<SC, SC, NT>(acc, scaled(fy, below(yr, yr_top, pt, kb)), rs, splane, kb);
      }
      // <R, S0>
#pragma unroll 1
      for (int n = 0; n < blocks * 16 * (NT / 8) / kThreads; ++n) {
        const int i = n * kThreads + tid, r = i / (NT / 8), c = i % (NT / 8) * 8;
        float x[8] = {0.f}, y[8] = {0.f}, d = 0.f;
#pragma unroll
        for (int s = 0; s < SC; ++s) {
          const uint4 u = *reinterpret_cast<const uint4 *>(ss + s * splane + r * ld + c);
          const uint4 v = *reinterpret_cast<const uint4 *>(rs + s * splane + r * ld + c);
          const uint32_t uu[4] = {u.x, u.y, u.z, u.w}, vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const float2 p = unpack(uu[m]), o = unpack(vv[m]);
            x[2 * m] += p.x;
            x[2 * m + 1] += p.y;
            y[2 * m] += o.x;
            y[2 * m + 1] += o.y;
          }
        }
#pragma unroll
        for (int m = 0; m < 8; ++m) d = fmaf(x[m], y[m], d);
        dot = fmaf(d, pow2(below(sr, sr_top, pt, r / 16)), dot);
      }
    }
    dot *= pow2(sr_top);
    const float fr = pow2(yr_top);
    w = row_dots<NT, SI>(acc, krow);
    w.x = over_quad(w.x) * pow2(ek) * (closing[r0] * fr);
    w.y = over_quad(w.y) * pow2(ek) * (closing[r1] * fr);
#pragma unroll
    for (int tb = 0; tb < 4; ++tb)
      if (tb >= warp) {
        const float f0 = tb > warp ? fall[fall_at(tb) + r0] : 1.f, f1 = tb > warp ? fall[fall_at(tb) + r1] : 1.f;
#pragma unroll
        for (int j = 2 * tb; j < 2 * tb + 2; ++j) {
          const int t = 8 * j + 2 * q;
          if (tb == warp) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int s = g + (i >> 1) * 8, tt = (t & 15) + (i & 1);
              const float dec = near[(warp * 16 + tt) * kNearLd + s];  // (zero where s comes later)
              Q[j][i] = tt >= s ? Q[j][i] * dec : 0.f;
              H[j][i] = tt > s ? H[j][i] * dec : 0.f;
            }
          } else {
            const float2 up = *reinterpret_cast<const float2 *>(rise + t);
            const float d[4] = {up.x * f0, up.y * f0, up.x * f1, up.y * f1};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              Q[j][i] *= d[i];
              H[j][i] *= d[i];
            }
          }
        }
      }
    // Q and H still lack a factor each, which joins their scaling; the sum takes closing and its unit in one
    const float fq = a.scale * pow2(y_top + eo_top), fh = -pow2(yx_top);
    {  // C, a block of 16 x 16 at a time: rows s, columns t
      const float fk = pow2(ek), fqk = pow2(eq), b0 = beta[r0], b1 = beta[r1];
      float later0 = 0.f, later1 = 0.f, own0 = 0.f, own1 = 0.f;  // row sums, over later blocks and over this one
      float c[2][4];
#pragma unroll
      for (int i = 3; i >= 0; --i) {
        if (i < warp) continue;
        const int tb = i;
        float qk[2][4], kk[2][4];
        zero(qk);
        zero(kk);
#pragma unroll 4
        for (int nb = 0; nb < NT / 16; ++nb) {
          Frag<SI> f;
          uint32_t bq[SI][4], bk[SI][4];
#pragma unroll
          for (int s = 0; s < SI; ++s) {
            a_mk(f.r[s], krow + s * Op::plane + 16 * nb, ld);
            b_nk(bq[s], qs + s * Op::plane + 16 * tb * ld + 16 * nb, ld);
            b_nk(bk[s], ks + s * Op::plane + 16 * tb * ld + 16 * nb, ld);
          }
          mma_split<SI, SI>(qk[0], qk[1], f, bq);
          mma_split<SI, SI>(kk[0], kk[1], f, bk);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            c[j][e] = Q[2 * tb + j][e] * fq * (qk[j][e] * fk * fqk) + H[2 * tb + j][e] * fh * (kk[j][e] * fk * fk);
        const float x0 = (c[0][0] + c[0][1]) + (c[1][0] + c[1][1]), x1 = (c[0][2] + c[0][3]) + (c[1][2] + c[1][3]);
        if (tb > warp) {
          later0 += x0;
          later1 += x1;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float u = over_rows(fmaf(b0, c[j][0], b1 * c[j][2])), v = over_rows(fmaf(b0, c[j][1], b1 * c[j][3]));
            if (g == 0) *reinterpret_cast<float2 *>(&far_cross[warp][16 * tb + 8 * j + 2 * q]) = make_float2(u, v);
          }
        } else {
          own0 = x0;
          own1 = x1;
        }
      }
      later0 = over_quad(later0);
      later1 = over_quad(later1);
      db.x = w.x + later0 + over_quad(own0);
      db.y = w.y + later1 + over_quad(own1);
      // c is the diagonal block: per row, sums over the columns from t on and over the later blocks; of these the rows before t
      float sum[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int s = g + 8 * n;
        const float later = n ? later1 : later0, be = n ? b1 : b0;
        float from[2];  // over this thread's columns of the tile and those to their right
#pragma unroll
        for (int j = 1; j >= 0; --j) {
          float run = c[j][2 * n] + c[j][2 * n + 1];
#pragma unroll
          for (int d = 1; d < 4; d <<= 1) {
            const float o = __shfl_down_sync(~0u, run, d, 4);
            if (q + d < 4) run += o;
          }
          float right = __shfl_down_sync(~0u, run, 1, 4);  // (taken from the neighbour: a difference would keep roundings)
          if (q == 3) right = 0.f;
          const float behind = j ? later : later + __shfl_sync(~0u, from[1], lane & ~3);
          if (j) from[1] = run;
          const int t = 8 * j + 2 * q;
          right += behind;
          const float at1 = c[j][2 * n + 1] + right, at0 = c[j][2 * n] + at1;
          if (s < t) sum[j][0] = fmaf(be, at0, sum[j][0]);
          if (s < t + 1) sum[j][1] = fmaf(be, at1, sum[j][1]);
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float u = over_rows(sum[j][0]), v = over_rows(sum[j][1]);
        if (g == 0) *reinterpret_cast<float2 *>(&near_cross[16 * warp + 8 * j + 2 * q]) = make_float2(u, v);
      }
    }
    const float top = __uint_as_float(__reduce_max_sync(~0u, max(mag(closing[r0]), mag(closing[r1]))));
    const int ec = warp_exp(acc) + yr_top + above(top), e1 = floor_exp(warp_exp(Q) + above(fq), ec, eq);
    const int e2 = floor_exp(warp_exp(H) + yx_top, max(ec, e1 + eq + 21) + 1, ek);
    {
      const float u = fr * pow2(-(e1 + eq));
      times_rows(acc, closing[r0] * u, closing[r1] * u);
    }
    const float s1 = fq * pow2(-e1), s2 = fh * pow2(-e2);
    {
      Onto<NT, SI, SC> to(acc);
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
        if (kb >= warp) {
          Frag<SC> f;
          frag_of<SC>(f, Q[2 * kb], Q[2 * kb + 1], s1);
          to.template add<SI>(f, qs, Op::plane, kb);
        }
      to.join();
    }
    times(acc, pow2(e1 + eq - (e2 + ek)));
    {
      Onto<NT, SI, SC> to(acc);
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
        if (kb >= warp) {
          Frag<SC> f;
          frag_of<SC>(f, H[2 * kb], H[2 * kb + 1], s2);
          to.template add<SI>(f, ks, Op::plane, kb);
        }
      to.join();
    }
    unit = e2 + ek;  // (acc is Z without its unit)
  }
  __syncthreads();  // (R is not read any more: its room takes results on their way out)
  __half *buf = rs + warp * 16 * ld;
  // ---- this warp's tokens as t: dk = beta Z + f gamma (dX S0) + f (H beta) k with f = -1, then the same with dO, Q and
  // f = scale: dq (whose sum starts at zero and has t itself)
  float2 read = make_float2(0.f, 0.f);  // of S0, by this warp's tokens
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    const bool is_q = part == 1;
    const __half *tile = is_q ? os : xs;
    const int ea = is_q ? (lane < PB ? eo_top : none) : ex;
    const float f = is_q ? a.scale : -1.f;
    float H[8][4];
    zero(H);
    const int ya = ey + ea, sa = es + ea;
    const int ya_top = __reduce_max_sync(~0u, ya), sa_top = __reduce_max_sync(~0u, sa);
    // The product with S0 has sums of its own, half of the columns at a time: times q or k they are what the gates let through
    // to this token, and times f gamma (in fp32: beside open gates a closed one would leave nothing in fp16) they join dq or dk.
    const float g0 = f * gamma[r0], g1 = f * gamma[r1];
    const int top = __reduce_max_sync(~0u, max(mag(g0), mag(g1)));
    float2 d = make_float2(0.f, 0.f);
    float b0 = 0.f, b1 = 0.f;  // dk takes beta Z over
    int held = kZeroExp;
    if (!is_q) {
      b0 = beta[r0];
      b1 = beta[r1];
      held = warp_exp(acc) + unit + above(__uint_as_float(__reduce_max_sync(~0u, max(mag(b0), mag(b1)))));
    }
    const int before = unit;
    unit = max(sa_top + max((top >> 23) - 127 + 1, 0), held - 40);
    {
      const float u = pow2(max(before - unit, -126));
      if (is_q) zero(acc);
      else times_rows(acc, b0 * u, b1 * u);
    }
#pragma unroll 1
    for (int pt = 0; pt < tiles; ++pt) {
      if (tiles > 1) {
        __syncthreads();
        load(pt);
      }
      const int blocks = min(4, PB - 4 * pt);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float sum[NT / 16][4];
        zero(sum);
#pragma unroll 1
        for (int kb = 0; kb < blocks; ++kb) {
          Frag<SC> fa;
          load_a(fa, tile, is_q ? SI : SC, kb);
          if (half == 0) {
            const Frag<SC> fh = scaled(fa, below(ya, ya_top, pt, kb));
#pragma unroll
            for (int sb = 0; sb < 4; ++sb)
              if (sb <= warp) {
                uint32_t bb[SC][4];
                load_b(bb, ys, sb, kb);
                mma_split<SC, SC>(H[2 * sb], H[2 * sb + 1], fh, bb);
              }
          }
          tile_cols<SC, SC, NT, NT == 128 && SC == 1 ? 4 : 2, NT / 2>(sum, scaled(fa, below(sa, sa_top, pt, kb)),
                                                                      ss + half * (NT / 2), splane, kb);
        }
        const float2 x = row_dots<NT, SI>(sum, (is_q ? qs : ks) + 16 * warp * ld + half * (NT / 2));
        d.x += x.x;
        d.y += x.y;
        const float u = pow2(sa_top - unit), f0 = g0 * u, f1 = g1 * u;
#pragma unroll
        for (int j = 0; j < NT / 16; ++j) {
          float(&to)[4] = acc[half * (NT / 16) + j];
          to[0] = fmaf(f0, sum[j][0], to[0]);
          to[1] = fmaf(f0, sum[j][1], to[1]);
          to[2] = fmaf(f1, sum[j][2], to[2]);
          to[3] = fmaf(f1, sum[j][3], to[3]);
        }
      }
    }
    {
      const float u = pow2(sa_top), v = pow2(is_q ? eq : ek);
      read.x = fmaf(over_quad(d.x) * u * v, g0, read.x);
      read.y = fmaf(over_quad(d.y) * u * v, g1, read.y);
    }
#pragma unroll
    for (int sb = 0; sb < 4; ++sb)
      if (sb <= warp) {
        const float f0 = sb < warp ? rise[r0] : 1.f, f1 = sb < warp ? rise[r1] : 1.f;
#pragma unroll
        for (int j = 2 * sb; j < 2 * sb + 2; ++j) {
          const int c = 8 * j + 2 * q;
          const float2 be = *reinterpret_cast<const float2 *>(beta + c);
          if (sb == warp) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = g + (i >> 1) * 8, cc = (c & 15) + (i & 1);
              const float dec = near[(warp * 16 + r) * kNearLd + cc] * (i & 1 ? be.y : be.x);
              H[j][i] = cc < r + part ? H[j][i] * dec : 0.f;
            }
          } else {
            const float2 fa = *reinterpret_cast<const float2 *>(fall + fall_at(warp) + c);
            const float x = fa.x * be.x, y = fa.y * be.y;
            const float d[4] = {f0 * x, f0 * y, f1 * x, f1 * y};
#pragma unroll
            for (int i = 0; i < 4; ++i) H[j][i] *= d[i];
          }
        }
      }
    const int e = floor_exp(warp_exp(H) + ya_top + above(f), warp_exp(acc) + unit, ek);
    times(acc, pow2(unit - (e + ek)));
    const float s = f * pow2(ya_top - e);
    {
      Onto<NT, SI, SC> to(acc);
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
        if (kb <= warp) {
          Frag<SC> fh2;
          frag_of<SC>(fh2, H[2 * kb], H[2 * kb + 1], s);
          to.template add<SI>(fh2, ks, Op::plane, kb);
        }
      to.join();
    }
    times(acc, pow2(e + ek));
    if (tiles > 1) __syncthreads();  // (the last tile's R has been loaded by all threads)
    const bool shared = a.heads != a.key_heads;
    const size_t row0 = ((size_t)(shared ? bh : b * a.key_heads + kh) * a.T + t0 + 16 * warp) * a.N;
    void *out = is_q ? a.dq : a.dk;
    if (shared) store_grad<NT, float>(static_cast<float *>(out) + row0, acc, rows - 16 * warp, a.N, buf);
    else store_grad<NT, TI>(static_cast<TI *>(out) + row0, acc, rows - 16 * warp, a.N, buf);
  }
  // ---- gates
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(~0u, dot, d);
  if (lane == 0) dots[warp] = dot;
  if (q == 0) {
    reads[r0] = read.x;
    reads[r1] = read.y;
    dbs[r0] = db.x;
    dbs[r1] = db.y;
    wsum[r0] = beta[r0] * w.x;
    wsum[r1] = beta[r1] * w.y;
  }
  __syncthreads();
  if (warp == 0) {  // tokens 2 lane and 2 lane + 1
    // sums over a pair's lane and all later ones, or all earlier ones; neighbours hand over what excludes the own
    auto from_here = [&](float x, float y, float &at_x, float &at_y) {
      float run = x + y;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const float o = __shfl_down_sync(~0u, run, d);
        if (lane + d < 32) run += o;
      }
      float rest = __shfl_down_sync(~0u, run, 1);
      if (lane == 31) rest = 0.f;
      at_y += y + rest;
      at_x += x + (y + rest);
    };
    const float state = gamma[L - 1] * (dots[0] + dots[1] + dots[2] + dots[3]);
    float x = state + near_cross[2 * lane], y = state + near_cross[2 * lane + 1];
    from_here(reads[2 * lane], reads[2 * lane + 1], x, y);
#pragma unroll
    for (int n = 0; n < 3; ++n) {  // from block n to the later ones
      const bool in = lane >= 8 * (n + 1);
      float u = 0.f, v = 0.f;
      from_here(in ? far_cross[n][2 * lane] : 0.f, in ? far_cross[n][2 * lane + 1] : 0.f, u, v);
      if (in) {
        x += u;
        y += v;
      }
    }
    float run = wsum[2 * lane] + wsum[2 * lane + 1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const float o = __shfl_up_sync(~0u, run, d);
      if (lane >= d) run += o;
    }
    float before = __shfl_up_sync(~0u, run, 1);
    if (lane == 0) before = 0.f;
    x += before;
    y += before + wsum[2 * lane];
    const size_t row = (size_t)bh * a.T + t0 + 2 * lane;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (2 * lane + i < rows) {
        store_as(a.dg, a.g_dtype, row + i, i ? y : x);
        store_as(a.dbeta, a.beta_dtype, row + i, dbs[2 * lane + i]);
      }
  }
}

// dq and dk of key heads that several value heads share: the sums of theirs, in the order of the heads.  per: values of a head,
// V of them a thread at a time (4, where they divide into fours: 3 heads of 1537 x 64 values, 12 key heads, 5 us; one at a time 12).
template <int V, typename TI>
__global__ void __launch_bounds__(256) delta_share_kernel(const float *pq, const float *pk, TI *dq, TI *dk, int share, int64_t per) {
  const float *src = (blockIdx.z ? pk : pq) + blockIdx.y * (share * per);
  TI *dst = (blockIdx.z ? dk : dq) + blockIdx.y * per;
  for (int64_t i = (blockIdx.x * 256 + threadIdx.x) * V; i < per; i += (int64_t)gridDim.x * 256 * V) {
    float s[V] = {0.f};
    for (int h = 0; h < share; ++h) {
      if constexpr (V == 4) {
        const float4 x = __ldcs(reinterpret_cast<const float4 *>(src + h * per + i));
        s[0] += x.x;
        s[1] += x.y;
        s[2] += x.z;
        s[3] += x.w;
      } else {
        s[0] += src[h * per + i];
      }
    }
    if constexpr (V == 4) {
      alignas(16) TI out[V];
#pragma unroll
      for (int n = 0; n < V; ++n) out[n] = from_f<TI>(s[n]);
      using Wide = std::conditional_t<sizeof(TI) == 4, uint4, uint2>;
      *reinterpret_cast<Wide *>(dst + i) = *reinterpret_cast<const Wide *>(out);
    } else {
      dst[i] = from_f<TI>(s[0]);
    }
  }
}

}  // namespace delta
}  // namespace slx
