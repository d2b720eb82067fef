// The two passes of the gated delta rule along the sequence: states forwards (with the outputs), gradients of the states
// backwards (with dV).
//
// Rows of a state (value channels) do not meet in the recurrence, so a warp owns 16 rows p for the whole sequence and keeps
// its (16, N) part of the state in accumulators.  Every product has the 16 rows on the M side: the state and all that is
// computed from it are A operands as they lie in registers, and the B operands (k, q, Tm, P) are tiles in shared memory
// which the warps of a CTA share.  Per chunk, forward:
//     X = v^T - gamma (S k^T)      Y = X Tm^T      o = gamma (S q^T) + (beta Y) P^T      S = Gam S + (closing beta Y) k
// backward (R = dL/dS after the chunk, going down):
//     dD = scale dO^T P + closing (R k^T)   dX = (beta dD) Tm   R = Gam R + (scale gamma dO)^T q - (gamma dX)^T k
// The tiles of the next chunk are on their way while this one is computed: k is double-buffered, the rest is loaded again
// as soon as its last reader is through.
//
// 256 heads of 4096 tokens (N 128, P 64, bf16): 466 us forwards, 513 back, at two CTAs an SM; the state, two results and their
// fp16 parts fill the registers.  With one warp a scheduler the tensor pipe is busy 35 to 40 %: the rest is the chain of products
// of one warp (11 thousand clocks a chunk alone, 14 with a second CTA beside it).
#pragma once

#include "delta.cuh"

namespace slx {
namespace delta {

template <int NT>
constexpr int warp_buf() {  // halves: 64 x 24 or 16 x (NT + 8)
  return 16 * (NT + 8) > 64 * 24 ? 16 * (NT + 8) : 64 * 24;
}
template <int NT, int SI, int SC, typename TI>
constexpr int scan_smem(bool backward) {
  return 3 * Operand<SI, NT>::halves * 2 + (2 + (backward ? 2 : SC)) * kTri * 2 + kHeadBytes + Raw<TI>::bytes +
         (kThreads / 32) * warp_buf<NT>() * 2;
}

// Columns c0 .. c0 + 15 of a raw tile, transposed: accumulators with rows p (the tile's columns) and columns t (its rows).
template <typename TI>
__device__ __forceinline__ void load_cols(float (&c)[8][4], const TI *tile, int c0) {
  constexpr int ld = Raw<TI>::ld;
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  if constexpr (sizeof(TI) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[j][i] = tile[(8 * j + 2 * q + (i & 1)) * ld + c0 + g + (i >> 1) * 8];
  } else {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      uint32_t r[4];
      a_km(r, reinterpret_cast<const __half *>(tile) + 8 * j * ld + c0, ld);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 x;
        if constexpr (std::is_same<TI, __half>::value) x = unpack(r[i]);
        else x = make_float2(__uint_as_float(r[i] << 16), __uint_as_float(r[i] & 0xffff0000u));
        c[j + (i >> 1)][(i & 1) * 2] = x.x;
        c[j + (i >> 1)][(i & 1) * 2 + 1] = x.y;
      }
    }
  }
}
// times the entries s[t] of a vector over the columns
__device__ __forceinline__ void times_cols(float (&c)[8][4], const float *s, float f) {
  const int q = threadIdx.x & 3;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float2 x = *reinterpret_cast<const float2 *>(s + 8 * j + 2 * q);
    c[j][0] *= x.x * f;
    c[j][1] *= x.y * f;
    c[j][2] *= x.x * f;
    c[j][3] *= x.y * f;
  }
}
__device__ __forceinline__ int max4(const int (&e)[4]) { return max(max(e[0], e[1]), max(e[2], e[3])); }
// a warp's 16 rows of a state from its buffer
template <int NT>
__device__ __forceinline__ void copy_state(__half *out, const __half *buf) {
  constexpr int ld = NT + 8;
#pragma unroll
  for (int i = threadIdx.x & 31; i < 16 * (NT / 8); i += 32)
    *reinterpret_cast<uint4 *>(out + (i / (NT / 8)) * ld + (i % (NT / 8)) * 8) =
        *reinterpret_cast<const uint4 *>(buf + (i / (NT / 8)) * ld + (i % (NT / 8)) * 8);
}
// v less c, times the entries s[t] of a vector over the columns
__device__ __forceinline__ void minus_cols(float (&c)[8][4], const float (&v)[8][4], const float *s, float f) {
  const int q = threadIdx.x & 3;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float2 x = *reinterpret_cast<const float2 *>(s + 8 * j + 2 * q);
    const float a = -x.x * f, b = -x.y * f;
    c[j][0] = fmaf(a, c[j][0], v[j][0]);
    c[j][1] = fmaf(b, c[j][1], v[j][1]);
    c[j][2] = fmaf(a, c[j][2], v[j][2]);
    c[j][3] = fmaf(b, c[j][3], v[j][3]);
  }
}
// c = f c + s d.  Where fp32 and fp16 results are wanted, sums over a chunk's tokens have accumulators of their own: the matrix
// instructions cut off what they add below an accumulator's last bit, and the state, which goes on for the whole sequence, would
// shrink by that at every step (d_initial of 700 tokens in fp32 2.2e-6, so 6e-7).  With bf16 it would not show, and the passes of
// the teams take 2 and 7 % longer; fp16's pass back by warps would take 25 % longer for its registers and goes without.
template <int n>
__device__ __forceinline__ void join(float (&c)[n][4], float f, const float (&d)[n][4], float s) {
#pragma unroll
  for (int j = 0; j < n; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) c[j][i] = fmaf(c[j][i], f, d[j][i] * s);
}
template <int S>
__device__ __forceinline__ void frags_of(Frag<S> (&f)[4], const float (&c)[8][4], int e) {
  const float s = pow2(-e);
#pragma unroll
  for (int kb = 0; kb < 4; ++kb) frag_of<S>(f[kb], c[2 * kb], c[2 * kb + 1], s);
}
__device__ __forceinline__ int4 exps_of(const Record *r) { return __ldg(reinterpret_cast<const int4 *>(&r->eT)); }

// c = f c + a B, over the 64 tokens of an operand tile B
template <bool own, int SI, int NT>
__device__ __forceinline__ void onto(float (&c)[NT / 8][4], float f, const Frag<2> (&a)[4], const __half *tile) {
  if constexpr (own) {
    float d[NT / 8][4];
    zero(d);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) tile_cols<2, SI, NT>(d, a[kb], tile, Operand<SI, NT>::plane, kb);
    join(c, f, d, 1.f);
  } else {
    times(c, f);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) tile_cols<2, SI, NT>(c, a[kb], tile, Operand<SI, NT>::plane, kb);
  }
}

template <int NT, int SI, int SC, typename TI>
__global__ void __launch_bounds__(kThreads) delta_fwd_kernel(Args a, int pw) {
  using Op = Operand<SI, NT>;
  using V = Raw<TI>;
  extern __shared__ __align__(128) char smem[];
  __half *ks = reinterpret_cast<__half *>(smem);  // two buffers
  __half *qs = ks + 2 * Op::halves;
  __half *Ts = qs + Op::halves;  // T hi, T lo, planes of P, the record's vectors
  __half *Ps = Ts + 2 * kTri;
  float *hd = reinterpret_cast<float *>(Ps + SC * kTri);
  const float *gamma = hd, *closing = hd + L, *beta = hd + 2 * L;
  const int(*tops)[4] = reinterpret_cast<const int(*)[4]>(hd + 3 * L);
  TI *vs = reinterpret_cast<TI *>(reinterpret_cast<char *>(hd) + kHeadBytes);

  const int warp = threadIdx.x >> 5;
  __half *buf = reinterpret_cast<__half *>(reinterpret_cast<char *>(vs) + V::bytes) + warp * warp_buf<NT>();
  const int bh = blockIdx.y, b = bh / a.heads, h = bh % a.heads, kh = h / (a.heads / a.key_heads);
  const int first = blockIdx.x * pw * 16, p0 = first + warp * 16;  // value channels of the CTA, of the warp
  const bool active = warp < pw && p0 < a.P16;
  const Record *rec = a.rec + (size_t)bh * a.NC;
  const int PB = a.P16 / 16, tiles = (a.P16 + 63) / 64;

  const __half *kq = a.kq + (size_t)(b * a.key_heads + kh) * a.NC * 2 * Op::halves;
  auto issue_k = [&](int c) { copy_bytes<Op::halves * 2>(ks + (c & 1) * Op::halves, kq + (size_t)c * 2 * Op::halves); };
  auto issue_rest = [&](int c) {
    copy_bytes<Op::halves * 2>(qs, kq + (size_t)(2 * c + 1) * Op::halves);
    copy_bytes<(2 + SC) * kTri * 2>(Ts, rec[c].T);
    copy_bytes<kHeadBytes>(hd, rec[c].gamma);
    V::issue(vs, head_base<TI>(a.v, b, h, c * L) + first, a.v.st, min(L, a.T - c * L), a.P - first, a.v.vec);
  };

  float S[NT / 8][4];  // times 2^unit
  int unit = 0;
  if (active && a.init) load_state<NT>(S, a.init, a.init_dtype, (size_t)bh * a.P * a.N, p0, a.P, a.N);
  else zero(S);
  int4 ex = exps_of(rec);
  issue_k(0);
  issue_rest(0);
  cp_commit();
  for (int c = 0; c < a.NC; ++c) {
    const bool more = c + 1 < a.NC;
    const int4 nx = more ? exps_of(rec + c + 1) : ex;
    const int eT = ex.x, eQ = ex.y, eq = ex.z, ek = ex.w;
    const __half *kt = ks + (c & 1) * Op::halves;
    cp_wait<0>();
    __syncthreads();
    if (more) issue_k(c + 1);
    cp_commit();
    Frag<2> fc[4];  // closing beta Y
    int eC = 0;
    float top = 0.f;  // Gam
    if (active) {
      const size_t at = (size_t)bh * a.NC + c;
      const int e0 = warp_exp(S), eS = e0 + unit;
      __half *const st = a.st ? a.st + (at * SC * a.P16 + p0) * (NT + 8) : nullptr;
      if (st && (threadIdx.x & 31) == 0) a.est[at * PB + p0 / 16] = eS;
      if (SC > 1 && st) store_state<SC, NT>(st, (int64_t)a.P16 * (NT + 8), S, e0, buf);
      float X[8][4], O[8][4];
      zero(X);
      zero(O);
      {
        const float s = pow2(-e0);
        const int lane = threadIdx.x & 31;
        if (SC == 1 && st) __syncwarp();
#pragma unroll
        for (int kb = 0; kb < NT / 16; ++kb) {
          Frag<2> f;
          frag_of<2>(f, S[2 * kb], S[2 * kb + 1], s);
          if (SC == 1 && st) stsm(smem_addr(buf + (lane & 15) * (NT + 8) + 16 * kb + (lane >> 4) * 8), f.r[0]);
          Frag<SC> fo;
#pragma unroll
          for (int pl = 0; pl < SC; ++pl)
#pragma unroll
            for (int i = 0; i < 4; ++i) fo.r[pl][i] = f.r[pl][i];
          tile_rows<2, SI, NT>(X, f, kt, kb);
          tile_rows<SC, SI, NT>(O, fo, qs, kb);
        }
        if (SC == 1 && st) {
          __syncwarp();
          copy_state<NT>(st, buf);
          __syncwarp();
        }
      }
      // X = v - gamma S k
      {
        float v[8][4];
        load_cols<TI>(v, vs, warp * 16);
        minus_cols(X, v, gamma, pow2(eS + ek));
      }
      int y;  // the unit of Y
      {
        const int eX = warp_exp(X);
        Frag<2> fx[4];
        frags_of<2>(fx, X, eX);
        zero(X);
        tri_rows<2, 2>(X, fx, Ts);
        y = eX + eT;
      }
      const int eY = warp_exp(X);
      if (a.y) {
        store_planes<SC>(a.y + (at * SC * tiles + p0 / 64) * kTile + p0 % 64, kTileLd, tiles * kTile, X, eY, buf);
        if ((threadIdx.x & 31) == 0) a.ey[at * PB + p0 / 16] = eY + y;
      }
      times_cols(X, beta, 1.f);
      if (a.o) {
        // (exponents from bounds: of beta Y by the largest beta, of S q by its operands')
        const int eD = floor_exp(eY + y + max4(tops[1]), eS + eq + 22 + max4(tops[0]), eQ);
        times_cols(O, gamma, pow2(eS + eq - (eD + eQ)));
        Frag<SC> fd[4];
        frags_of<SC>(fd, X, eD - y);
        tri_rows<SC, SC>(O, fd, Ps);
        times(O, a.scale * pow2(eD + eQ));
        store_rows<TI>(static_cast<TI *>(a.o) + ((size_t)bh * a.T + c * L) * a.P + p0, a.P, min(L, a.T - c * L), a.P - p0, O, buf);
      }
      times_cols(X, closing, 1.f);
      top = gamma[L - 1];
      eC = floor_exp(eY + y + max4(tops[2]), eS + above(top), ek);
      frags_of<2>(fc, X, eC - y);
    }
    __syncthreads();
    if (more) issue_rest(c + 1);
    cp_commit();
    if (active) {
      onto<SC == 2, SI, NT>(S, times_pow2(top, unit - (eC + ek)), fc, kt);
      unit = eC + ek;
    }
    ex = nx;
  }
  cp_wait<0>();
  if (active && a.final_state) {
    times(S, pow2(unit));
    write_state<NT>(a.final_state, SLX_F32, (size_t)bh * a.P * a.N, S, p0, a.P, a.N);
  }
}

template <int NT, int SI, int SC, typename TI>
__global__ void __launch_bounds__(kThreads) delta_bwd_kernel(Args a, int pw) {
  using Op = Operand<SI, NT>;
  using V = Raw<TI>;
  extern __shared__ __align__(128) char smem[];
  __half *ks = reinterpret_cast<__half *>(smem);  // two buffers
  __half *qs = ks + 2 * Op::halves;
  __half *Ts = qs + Op::halves;  // T hi, T lo, P hi, P lo, the record's vectors
  __half *Ps = Ts + 2 * kTri;
  float *hd = reinterpret_cast<float *>(Ps + 2 * kTri);
  const float *gamma = hd, *closing = hd + L, *beta = hd + 2 * L;
  const int(*tops)[4] = reinterpret_cast<const int(*)[4]>(hd + 3 * L);
  TI *os = reinterpret_cast<TI *>(reinterpret_cast<char *>(hd) + kHeadBytes);

  const int warp = threadIdx.x >> 5;
  __half *buf = reinterpret_cast<__half *>(reinterpret_cast<char *>(os) + V::bytes) + warp * warp_buf<NT>();
  const int bh = blockIdx.y, b = bh / a.heads, h = bh % a.heads, kh = h / (a.heads / a.key_heads);
  const int first = blockIdx.x * pw * 16, p0 = first + warp * 16;
  const bool active = warp < pw && p0 < a.P16;
  const Record *rec = a.rec + (size_t)bh * a.NC;
  const int PB = a.P16 / 16, tiles = (a.P16 + 63) / 64;

  const __half *kq = a.kq + (size_t)(b * a.key_heads + kh) * a.NC * 2 * Op::halves;
  auto issue_k = [&](int c) { copy_bytes<Op::halves * 2>(ks + (c & 1) * Op::halves, kq + (size_t)c * 2 * Op::halves); };
  auto issue_rest = [&](int c) {
    copy_bytes<4 * kTri * 2>(Ts, rec[c].T);
    copy_bytes<kHeadBytes>(hd, rec[c].gamma);
    V::issue(os, head_base<TI>(a.dO, b, h, c * L) + first, a.dO.st, min(L, a.T - c * L), a.P - first, a.dO.vec);
  };

  float R[NT / 8][4];  // times 2^unit
  int unit = 0;
  if (active && a.d_final) load_state<NT>(R, a.d_final, a.d_final_dtype, (size_t)bh * a.P * a.N, p0, a.P, a.N);
  else zero(R);
  int4 ex = exps_of(rec + a.NC - 1);
  issue_k(a.NC - 1);
  issue_rest(a.NC - 1);
  cp_commit();
  for (int c = a.NC - 1; c >= 0; --c) {
    const int4 nx = c > 0 ? exps_of(rec + c - 1) : ex;
    const int eT = ex.x, eQ = ex.y, eq = ex.z, ek = ex.w;
    const __half *kt = ks + (c & 1) * Op::halves;
    const int rows = min(L, a.T - c * L);
    cp_wait<0>();
    __syncthreads();
    copy_bytes<Op::halves * 2>(qs, kq + (size_t)(2 * c + 1) * Op::halves);
    cp_commit();
    if (c > 0) issue_k(c - 1);
    cp_commit();
    Frag<2> f1[4], f2[4];  // scale gamma dO, -gamma dX
    int e1 = 0, e2 = 0;
    float top = 0.f;
    if (active) {
      const size_t at = (size_t)bh * a.NC + c;
      const int e0 = warp_exp(R), eR = e0 + unit;
      __half *const st = a.ds + (at * SC * a.P16 + p0) * (NT + 8);
      if (SC > 1) store_state<SC, NT>(st, (int64_t)a.P16 * (NT + 8), R, e0, buf);
      float W[8][4], X[8][4], dO[8][4];
      zero(X);
      {
        const float s = pow2(-e0);
        const int lane = threadIdx.x & 31;
        if (SC == 1) __syncwarp();
#pragma unroll
        for (int kb = 0; kb < NT / 16; ++kb) {
          Frag<2> f;
          frag_of<2>(f, R[2 * kb], R[2 * kb + 1], s);
          if (SC == 1) stsm(smem_addr(buf + (lane & 15) * (NT + 8) + 16 * kb + (lane >> 4) * 8), f.r[0]);
          tile_rows<2, SI, NT>(X, f, kt, kb);
        }
        if (SC == 1) {
          __syncwarp();
          copy_state<NT>(st, buf);
          __syncwarp();
        }
      }
      load_cols<TI>(dO, os, warp * 16);
      const int eG = warp_exp(dO), eo = std::is_same<TI, __half>::value ? 0 : eG;
      zero(W);
      {
        Frag<SI> fo[4];
        frags_of<SI>(fo, dO, eo);
        tri_cols<SI, 2>(W, fo, Ps);
      }
      {  // beta dD
        const float fx = pow2(eR + ek), fw = a.scale * pow2(eo + eQ);
        const int q = threadIdx.x & 3;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 be = *reinterpret_cast<const float2 *>(beta + 8 * j + 2 * q);
          const float2 cl = *reinterpret_cast<const float2 *>(closing + 8 * j + 2 * q);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float b = i & 1 ? be.y : be.x, l = i & 1 ? cl.y : cl.x;
            X[j][i] = b * fmaf(l * fx, X[j][i], W[j][i] * fw);
          }
        }
      }
      {
        const int eX = warp_exp(X);
        Frag<2> fx[4];
        frags_of<2>(fx, X, eX);
        zero(W);
        tri_cols<2, 2>(W, fx, Ts);
        times(W, pow2(eX + eT));  // dX
      }
      store_rows<TI>(static_cast<TI *>(a.dv) + ((size_t)bh * a.T + c * L) * a.P + p0, a.P, rows, a.P - p0, W, buf);
      const int eW = warp_exp(W);
      store_planes<SC>(a.dx + (at * SC * tiles + p0 / 64) * kTile + p0 % 64, kTileLd, tiles * kTile, W, eW, buf);
      if ((threadIdx.x & 31) == 0) {
        a.eds[at * PB + p0 / 16] = eR;
        a.edx[at * PB + p0 / 16] = eW;
        a.edo[at * PB + p0 / 16] = eo;
      }
      // (exponents from bounds: by the largest gamma)
      times_cols(dO, gamma, a.scale);
      top = gamma[L - 1];
      const int eD = eR + above(top);  // of the decayed R
      e1 = floor_exp(eG + max4(tops[0]) + above(a.scale), eD, eq);
      frags_of<2>(f1, dO, e1);
      times_cols(W, gamma, -1.f);
      // (64 products of values below 2^15 join R between the two)
      e2 = floor_exp(eW + max4(tops[0]), max(eD, e1 + eq + 21) + 1, ek);
      frags_of<2>(f2, W, e2);
    }
    cp_wait<1>();
    __syncthreads();
    if (c > 0) issue_rest(c - 1);
    cp_commit();
    if (active) {
      onto<SI == 2, SI, NT>(R, times_pow2(top, unit - (e1 + eq)), f1, qs);
      onto<SI == 2, SI, NT>(R, pow2(e1 + eq - (e2 + ek)), f2, kt);
      unit = e2 + ek;
    }
    ex = nx;
  }
  cp_wait<0>();
  if (active && a.d_init) {
    times(R, pow2(unit));
    write_state<NT>(a.d_init, a.d_init_dtype, (size_t)bh * a.P * a.N, R, p0, a.P, a.N);
  }
}

}  // namespace delta
}  // namespace slx
