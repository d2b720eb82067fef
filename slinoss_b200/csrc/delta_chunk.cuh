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
//
// 16384 chunks of one head each (N 128, bf16): 526 us, 1.1 GB written; 1.4 instructions a clock and SM at 16 warps, a
// quarter of the waiting at barriers (the first warp takes the gates' sums, the inverse of block column 0 is the longest).
// Letting the other warps convert k and q meanwhile gains 2 % there and loses 8 % with 64 columns, for registers.
#pragma once

#include "delta.cuh"

namespace slx {
namespace delta {

constexpr int kAld = 72;  // floats per row of the fp32 tile: float2 accesses of a quarter warp meet no bank twice
// Below this an exponential is zero in fp32 whatever it is multiplied with; -inf, which would make differences of sums
// meaningless, is held here: the state is dropped.
constexpr double kLowestGate = -110.0;

template <int NT, int SI>
constexpr int chunk_tiles() {  // bytes: k and q, then the four triangular tiles in their place
  return 2 * Operand<SI, NT>::halves > 4 * kTri ? 2 * Operand<SI, NT>::halves * 2 : 4 * kTri * 2;
}
template <int NT, int SI>
constexpr int chunk_smem() {
  return chunk_tiles<NT, SI>() + L * kAld * 4;
}

// The upper part is rounded to nearest: what is left is then at most 2^-11 of x and of either sign, and the product of two
// such parts, which is left out, 2^-22.  (Cut off, it would be 2^-20, always of the result's sign.)  A NaN stays one in lo.
__device__ __forceinline__ void split_tf32(float x, uint32_t &hi, uint32_t &lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
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
__global__ void __launch_bounds__(kThreads, NT == 64 || SI == 1 ? 4 : 1) delta_chunk_kernel(Args a) {
  using Op = Operand<SI, NT>;
  using In = Pieces<TI, NT>;
  extern __shared__ __align__(128) char smem[];
  __half *ks = reinterpret_cast<__half *>(smem), *qs = ks + Op::halves;
  __half *tri = reinterpret_cast<__half *>(smem);  // T hi, T lo, P hi, P lo
  float *A = reinterpret_cast<float *>(smem + chunk_tiles<NT, SI>());
  __shared__ double G[L];
  __shared__ float beta[L], rise[L], fall[96];
  __shared__ unsigned tops[8];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int chunk = blockIdx.x, b = blockIdx.y / a.key_heads, kh = blockIdx.y % a.key_heads;
  const int share = a.heads / a.key_heads, t0 = chunk * L, rows = min(L, a.T - t0);

  const bool train = a.st;  // (the backward reads the tables and the lower plane of P; with bf16 the forward reads neither)

  // near pairs of block w lie in a block of A above the diagonal
  auto near_at = [&](int w, int r, int c) -> float & { return A[((w < 3 ? 0 : 16) + r) * kAld + (w < 3 ? 16 * w + 16 : 32) + c]; };
  In kx, qx;  // (on their way while the gates are read)
  kx.load(head_base<TI>(a.k, b, kh, t0), a.k.st, rows, a.N, a.k.vec, ks);
  qx.load(head_base<TI>(a.q, b, kh, t0), a.q.st, rows, a.N, a.q.vec, qs);
  float kk[8][4], qk[8][4];  // rows 16 warp .. + 15 of k k^T and q k^T, columns up to the diagonal block
  int eq = 0, ek = 0;

  auto gates = [&](int h, Record *rec) {  // of one head, to shared memory and its record
    if (warp == 0) {  // two tokens per lane; past the end g = 0 and beta = 0
      double gg[2];
      float write[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = 2 * lane + i;
        gg[i] = 0.0;
        write[i] = 0.f;
        if (t < rows) {
          const double x = load_as_f(a.g.p, a.g_dtype, b * a.g.sb + h * a.g.sh + (int64_t)(t0 + t) * a.g.st);
          gg[i] = x < kLowestGate ? kLowestGate : x;
          write[i] = load_as_f(a.beta.p, a.beta_dtype, b * a.beta.sb + h * a.beta.sh + (int64_t)(t0 + t) * a.beta.st);
        }
      }
      const double pair = gg[0] + gg[1];
      double run = pair;
      for (int d = 1; d < 32; d <<= 1) {
        const double o = __shfl_up_sync(~0u, run, d);
        if (lane >= d) run += o;
      }
      *reinterpret_cast<double2 *>(G + 2 * lane) = make_double2(run - pair + gg[0], run);
      const double last = __shfl_sync(~0u, run, 31);
      unsigned bits[3] = {0, 0, 0};  // (of magnitudes: a NaN is the largest)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const double s = i ? run : run - gg[1];
        const float x[3] = {expf((float)s), write[i], write[i] * expf((float)(last - s))};
#pragma unroll
        for (int n = 0; n < 3; ++n) bits[n] = max(bits[n], mag(x[n]));
      }
#pragma unroll
      for (int n = 0; n < 3; ++n) {
        for (int d = 1; d < 8; d <<= 1) bits[n] = max(bits[n], __shfl_xor_sync(~0u, bits[n], d));
        if (lane % 8 == 0) rec->tops[n][lane / 8] = above(__uint_as_float(bits[n]));
      }
      *reinterpret_cast<float2 *>(rec->beta + 2 * lane) = make_float2(write[0], write[1]);
      *reinterpret_cast<float2 *>(beta + 2 * lane) = make_float2(write[0], write[1]);
    }
    __syncthreads();
    if (tid < L) {
      const float x = expf((float)(G[tid] - (tid < 16 ? 0.0 : G[(tid & ~15) - 1])));
      rise[tid] = x;
      if (train) rec->rise[tid] = x;
      rec->gamma[tid] = expf((float)G[tid]);
    } else {
      rec->closing[tid - L] = expf((float)(G[L - 1] - G[tid - L]));
    }
    if (tid < 96) {
      const int i = tid < 16 ? 1 : tid < 48 ? 2 : 3;
      const float x = expf((float)(G[16 * i - 1] - G[tid - fall_at(i)]));
      fall[tid] = x;
      if (train) rec->fall[tid] = x;
    }
#pragma unroll 4
    for (int i = lane; i < 256; i += 32) {  // this warp's block of near pairs
      const int r = i / 16, c = i % 16;
      const float x = c <= r ? expf((float)(G[16 * warp + r] - G[16 * warp + c])) : 0.f;
      near_at(warp, r, c) = x;
      if (train) rec->near[warp][r * kNearLd + c] = x;
    }
  };
  auto record_of = [&](int h) { return a.rec + (size_t)(b * a.heads + h) * a.NC + chunk; };
  gates(kh * share, record_of(kh * share));
  {
    if constexpr (!std::is_same<TI, __half>::value) {
      const unsigned mq = __reduce_max_sync(~0u, qx.max_bits()), mk = __reduce_max_sync(~0u, kx.max_bits());
      if (lane == 0) {
        tops[warp] = mq;
        tops[4 + warp] = mk;
      }
      __syncthreads();
      eq = exp_of(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
      ek = exp_of(max(max(tops[4], tops[5]), max(tops[6], tops[7])));
    }
    __half *copy = a.kq + ((size_t)blockIdx.y * a.NC + chunk) * 2 * Op::halves;
    kx.template store<SI, true>(ks, copy, ek);
    qx.template store<SI, true>(qs, copy + Op::halves, eq);
    __syncthreads();
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
  }
  __syncthreads();  // (the tables are there; k and q have been read)

#pragma unroll 1
  for (int hs = 0; hs < share; ++hs) {
    Record *rec = record_of(kh * share + hs);

    float pp[8][4];
    zero(pp);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j <= 2 * warp + 1) {
        float m[4];
        const int c = 8 * j + 2 * q;
        const float2 be = *reinterpret_cast<const float2 *>(beta + c);
        if (j >= 2 * warp) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = g + (i >> 1) * 8, cc = (c & 15) + (i & 1);
            const float dec = near_at(warp, r, cc);  // (zero above the diagonal)
            pp[j][i] = cc <= r ? dec * qk[j][i] : 0.f;
            m[i] = cc < r ? dec * kk[j][i] * (i & 1 ? be.y : be.x) : 0.f;
          }
        } else {
          const float2 fa = *reinterpret_cast<const float2 *>(fall + fall_at(warp) + c);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float dec = rise[16 * warp + g + (i >> 1) * 8] * (i & 1 ? fa.y : fa.x);
            pp[j][i] = dec * qk[j][i];
            m[i] = dec * kk[j][i] * (i & 1 ? be.y : be.x);
          }
        }
        *reinterpret_cast<float2 *>(A + (16 * warp + g) * kAld + c) = make_float2(m[0], m[1]);
        *reinterpret_cast<float2 *>(A + (16 * warp + g + 8) * kAld + c) = make_float2(m[2], m[3]);
      }
    const unsigned mp = __reduce_max_sync(~0u, max_mag(pp));
    if (lane == 0) tops[warp] = mp;
    __syncwarp();
    // this warp's diagonal block, inverted in place: a column per lane by forward substitution (two lanes do the same one)
    {
      float *D = A + 16 * warp * kAld + 16 * warp;
      const int col = lane & 15;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s = i == col ? 1.f : 0.f, s2 = 0.f;
#pragma unroll
        for (int m = 0; m < i; m += 4) {
          const float4 d = *reinterpret_cast<const float4 *>(D + i * kAld + m);
          s = fmaf(-d.x, x[m], s);
          if (m + 1 < i) s2 = fmaf(-d.y, x[m + 1], s2);
          if (m + 2 < i) s = fmaf(-d.z, x[m + 2], s);
          if (m + 3 < i) s2 = fmaf(-d.w, x[m + 3], s2);
        }
        x[i] = i < col ? 0.f : s + s2;
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = lane < 16 ? i : i + 8;
        D[r * kAld + col] = lane < 16 ? x[i] : x[i + 8];
      }
    }
    __syncthreads();

    // P, scaled by the chunk's largest
    const int eQ = exp_of(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
    {
      const float s = pow2(-eQ);
      const int ld = tri_ld(warp);
      __half *at = tri + 2 * kTri + tri_base(warp) + (lane & 15) * ld + (lane >> 4) * 8;
#pragma unroll
      for (int j = 0; j < 8; j += 2)
        if (j <= 2 * warp) {
          Frag<2> f;
          frag_of<2>(f, pp[j], pp[j + 1], s);
          stsm(smem_addr(at + 8 * j), f.r[0]);
          stsm(smem_addr(at + kTri + 8 * j), f.r[1]);
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
        if (m >= warp) {
          Frag<2> f;
          frag_of<2>(f, x[m][0], x[m][1], s);
          __half *at = tri + tri_base(m) + ((lane & 7) + (lane >> 4) * 8) * tri_ld(m) + 16 * warp + ((lane >> 3) & 1) * 8;
          stsm_t(smem_addr(at), f.r[0]);
          stsm_t(smem_addr(at + kTri), f.r[1]);
        }
    }
    __syncthreads();
    uint4 *dst = reinterpret_cast<uint4 *>(rec);
    const uint4 *src = reinterpret_cast<const uint4 *>(tri);
#pragma unroll
    for (int i = 0; i < 4 * kTri / 8 / kThreads; ++i)
      if (i < 3 * kTri / 8 / kThreads || train || !std::is_same<TI, __nv_bfloat16>::value) dst[tid + i * kThreads] = src[tid + i * kThreads];
    if (tid == 0) *reinterpret_cast<int4 *>(&rec->eT) = make_int4(eT, eQ, eq, ek);
    if (hs + 1 < share) {  // G, beta, A and tri are written again
      __syncthreads();
      gates(kh * share + hs + 1, record_of(kh * share + hs + 1));
      __syncthreads();
    }
  }
}

}  // namespace delta
}  // namespace slx
