// Per-chunk part of the gated delta rule: the two lower triangular 64 x 64 matrices of a chunk and head,
//     Tm = (I + M diag(beta))^-1,  M_ts = dec_ts k_t.k_s (s < t),   and   P_ts = dec_ts q_t.k_s (s <= t),
// with the vectors that later kernels need of the gates.  One CTA of four warps per (chunk, batch, key head); it goes through
// the value heads that share the key head, which differ in their gates only.
//
// The inverse is formed by blocks of 16: each warp inverts a diagonal block by forward substitution (fp32, one column per
// lane), then takes one block column downwards, T_ij = -T_ii sum_m A_im T_mj, on tf32 matrix instructions with operands in
// two parts (22 bits).  A column's blocks are kept transposed in accumulators, which are A operands of the next products as
// they lie, so that warps meet only at the diagonal blocks.  Decays are exponentials of differences of G held in 64 bits:
// a large |g| anywhere in the chunk costs the later, slowly decaying tokens no precision.
#pragma once

#include "delta.cuh"

namespace slx {
namespace delta {

constexpr int kAld = 72;  // floats per row of the fp32 tile: float2 accesses of a quarter warp meet no bank twice
// Below this an exponential is zero in fp32 whatever it is multiplied with; -inf, which would make differences of sums
// meaningless, is held here: the state is dropped.
constexpr double kLowestGate = -110.0;

template <int NT, int SI>
constexpr int chunk_smem() {
  return 2 * SI * L * (NT + 8) * 2 + L * kAld * 4 + 4 * kTri * 2 + 64;
}

__device__ __forceinline__ void split_tf32(float x, uint32_t &hi, uint32_t &lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
// c (16 x 16, two n8 tiles) += sign * A B^T for A in accumulator layout (two n8 tiles) and B rows (n) of row-major fp32.
// The contraction's index runs as the accumulators hold it: columns 2 q and 2 q + 1 of a tile take the instruction's k = q
// and k = q + 4.
__device__ __forceinline__ void block_product(float (&c)[2][4], const float (&a)[2][4], const float *b, float sign) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    uint32_t hi[4], lo[4];
    split_tf32(sign * a[ks][0], hi[0], lo[0]);
    split_tf32(sign * a[ks][2], hi[1], lo[1]);
    split_tf32(sign * a[ks][1], hi[2], lo[2]);
    split_tf32(sign * a[ks][3], hi[3], lo[3]);
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const float2 x = *reinterpret_cast<const float2 *>(b + (8 * nt + g) * kAld + 8 * ks + 2 * q);
      uint32_t bh0, bl0, bh1, bl1;
      split_tf32(x.x, bh0, bl0);
      split_tf32(x.y, bh1, bl1);
      mma_tf32(c[nt], lo, bh0, bh1);
      mma_tf32(c[nt], hi, bl0, bl1);
      mma_tf32(c[nt], hi, bh0, bh1);
    }
  }
}

template <int NT, int SI, typename TI>
__global__ void __launch_bounds__(kThreads) delta_chunk_kernel(Args a) {
  using Op = Operand<TI, SI, NT>;
  extern __shared__ __align__(128) char smem[];
  __half *qs = reinterpret_cast<__half *>(smem), *ks = qs + SI * Op::plane;
  float *A = reinterpret_cast<float *>(smem + 2 * Op::bytes);
  __half *tri = reinterpret_cast<__half *>(A + L * kAld);  // T hi, T lo, P hi, P lo
  unsigned *tops = reinterpret_cast<unsigned *>(tri + 4 * kTri);
  __shared__ double G[L];
  __shared__ float beta[L];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int chunk = blockIdx.x, b = blockIdx.y / a.key_heads, kh = blockIdx.y % a.key_heads;
  const int share = a.heads / a.key_heads, t0 = chunk * L, rows = min(L, a.T - t0);
  const TI *qp = head_base<TI>(a.q, b, kh, t0), *kp = head_base<TI>(a.k, b, kh, t0);

  int eq = 0, ek = 0;
  if constexpr (!std::is_same<TI, __half>::value) {
    const unsigned mq = __reduce_max_sync(~0u, tile_mag(qp, a.q.st, rows, a.N, a.q.vec, NT));
    const unsigned mk = __reduce_max_sync(~0u, tile_mag(kp, a.k.st, rows, a.N, a.k.vec, NT));
    if (lane == 0) {
      tops[warp] = mq;
      tops[4 + warp] = mk;
    }
    __syncthreads();
    eq = exp_of(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
    ek = exp_of(max(max(tops[4], tops[5]), max(tops[6], tops[7])));
  }
  Op::issue(qs, qp, a.q.st, rows, a.N, a.q.vec, eq);
  Op::issue(ks, kp, a.k.st, rows, a.N, a.k.vec, ek);
  cp_commit();
  cp_wait<0>();
  Op::finish(qs, a.q.vec, eq);
  Op::finish(ks, a.k.vec, ek);
  __syncthreads();

  // rows 16 warp .. + 15 of k k^T and q k^T, columns up to the diagonal block
  float kk[8][4], qk[8][4];
  zero(kk);
  zero(qk);
#pragma unroll 2
  for (int kb = 0; kb < NT / 16; ++kb) {
    Frag<SI> fk, fq;
#pragma unroll
    for (int s = 0; s < SI; ++s) {
      a_mk(fk.r[s], ks + s * Op::plane + 16 * warp * Op::ld + 16 * kb, Op::ld);
      a_mk(fq.r[s], qs + s * Op::plane + 16 * warp * Op::ld + 16 * kb, Op::ld);
    }
#pragma unroll
    for (int sb = 0; sb < 4; ++sb)
      if (sb <= warp) {
        uint32_t bb[SI][4];
#pragma unroll
        for (int s = 0; s < SI; ++s) b_nk(bb[s], ks + s * Op::plane + 16 * sb * Op::ld + 16 * kb, Op::ld);
        mma_split<SI, SI>(kk[2 * sb], kk[2 * sb + 1], fk, bb);
        mma_split<SI, SI>(qk[2 * sb], qk[2 * sb + 1], fq, bb);
      }
  }
  const float fkk = pow2(ek), fqk = pow2(eq);  // (two factors: their product may leave the range where the results do not)
  times(kk, fkk);
  times(kk, fkk);
  times(qk, fqk);
  times(qk, fkk);

  for (int hs = 0; hs < share; ++hs) {
    const int h = kh * share + hs;
    Record *rec = a.rec + (size_t)(b * a.heads + h) * a.NC + chunk;
    if (warp == 0) {  // two tokens per lane; past the end g = 0 and beta = 0
      double s0, s1;
      float be[2];
      double gg[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = 2 * lane + i;
        gg[i] = 0.0;
        be[i] = 0.f;
        if (t < rows) {
          const double x = load_as_f(a.g.p, a.g_dtype, b * a.g.sb + h * a.g.sh + (int64_t)(t0 + t) * a.g.st);
          gg[i] = x < kLowestGate ? kLowestGate : x;
          be[i] = load_as_f(a.beta.p, a.beta_dtype, b * a.beta.sb + h * a.beta.sh + (int64_t)(t0 + t) * a.beta.st);
        }
        beta[t] = be[i];
      }
      s0 = gg[0];
      s1 = gg[0] + gg[1];
      double run = s1;
      for (int d = 1; d < 32; d <<= 1) {
        const double o = __shfl_up_sync(~0u, run, d);
        if (lane >= d) run += o;
      }
      const double before = run - s1, last = __shfl_sync(~0u, run, 31);
      s0 += before;
      s1 += before;
      G[2 * lane] = s0;
      G[2 * lane + 1] = s1;
      rec->G[2 * lane] = s0;
      rec->G[2 * lane + 1] = s1;
      *reinterpret_cast<float2 *>(rec->gamma + 2 * lane) = make_float2(expf((float)s0), expf((float)s1));
      *reinterpret_cast<float2 *>(rec->closing + 2 * lane) = make_float2(expf((float)(last - s0)), expf((float)(last - s1)));
      *reinterpret_cast<float2 *>(rec->beta + 2 * lane) = make_float2(be[0], be[1]);
    }
    __syncthreads();

    float pp[8][4];
    zero(pp);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j <= 2 * warp + 1) {
        float m[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * warp + g + (i >> 1) * 8, c = 8 * j + 2 * q + (i & 1);
          const float dec = c <= r ? expf((float)(G[r] - G[c])) : 0.f;
          pp[j][i] = c <= r ? dec * qk[j][i] : 0.f;
          m[i] = c < r ? dec * kk[j][i] * beta[c] : 0.f;
        }
        *reinterpret_cast<float2 *>(A + (16 * warp + g) * kAld + 8 * j + 2 * q) = make_float2(m[0], m[1]);
        *reinterpret_cast<float2 *>(A + (16 * warp + g + 8) * kAld + 8 * j + 2 * q) = make_float2(m[2], m[3]);
      }
    const unsigned mp = __reduce_max_sync(~0u, max_mag(pp));
    if (lane == 0) tops[warp] = mp;
    __syncwarp();
    // this warp's diagonal block, inverted in place: column `lane` by forward substitution
    if (lane < 16) {
      float *D = A + 16 * warp * kAld + 16 * warp;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s = i == lane ? 1.f : 0.f;
#pragma unroll
        for (int m = 0; m < i; ++m) s = fmaf(-D[i * kAld + m], x[m], s);
        x[i] = i < lane ? 0.f : s;
      }
      __syncwarp(0xffffu);
#pragma unroll
      for (int i = 0; i < 16; ++i) D[i * kAld + lane] = x[i];
    }
    __syncthreads();

    // P, scaled by the chunk's largest
    const int eQ = exp_of(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
    {
      const float s = pow2(-eQ);
      const int ld = tri_ld(warp);
      __half *at = tri + 2 * kTri + tri_base(warp) + g * ld + 2 * q;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j <= 2 * warp + 1)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t hi, lo;
            split<2>(pp[j][2 * i] * s, pp[j][2 * i + 1] * s, &hi, &lo);
            *reinterpret_cast<uint32_t *>(at + i * 8 * ld + 8 * j) = hi;
            *reinterpret_cast<uint32_t *>(at + kTri + i * 8 * ld + 8 * j) = lo;
          }
    }

    // block column `warp` of Tm, transposed: x[m] rows are the column's 16 columns, columns its rows 16 m .. + 15
    float x[4][2][4];
#pragma unroll
    for (int m = 0; m < 4; ++m) zero(x[m]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i == warp) {
        const float *D = A + 16 * warp * kAld + 16 * warp;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[i][nt][e] = D[(8 * nt + 2 * q + (e & 1)) * kAld + g + (e >> 1) * 8];
      } else if (i > warp) {
        float r[2][4];
        zero(r);
#pragma unroll
        for (int m = 0; m < 4; ++m)
          if (m >= warp && m < i) block_product(r, x[m], A + 16 * i * kAld + 16 * m, 1.f);
        block_product(x[i], r, A + 16 * i * kAld + 16 * i, -1.f);
      }
    }
    unsigned mt = 0;
#pragma unroll
    for (int m = 0; m < 4; ++m) mt = max(mt, max_mag(x[m]));
    mt = __reduce_max_sync(~0u, mt);
    if (lane == 0) tops[4 + warp] = mt;
    __syncthreads();
    const int eT = exp_of(max(max(tops[4], tops[5]), max(tops[6], tops[7])));
    {
      const float s = pow2(-eT);
#pragma unroll
      for (int m = 0; m < 4; ++m)
        if (m >= warp)
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y = x[m][nt][e] * s;
              __half *at = tri + tri_base(m) + (8 * nt + 2 * q + (e & 1)) * tri_ld(m) + 16 * warp + g + (e >> 1) * 8;
              const __half hi = __float2half_rn(y);
              at[0] = hi;
              at[kTri] = __float2half_rn(y - __half2float(hi));
            }
    }
    __syncthreads();
    uint4 *dst = reinterpret_cast<uint4 *>(rec);
    const uint4 *src = reinterpret_cast<const uint4 *>(tri);
    for (int i = tid; i < 4 * kTri / 8; i += kThreads) dst[i] = src[i];
    if (tid == 0) *reinterpret_cast<int4 *>(&rec->eT) = make_int4(eT, eQ, eq, ek);
    __syncthreads();  // G, beta, A and tri are written again
  }
}

}  // namespace delta
}  // namespace slx
