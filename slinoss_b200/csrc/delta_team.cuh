// The passes along the sequence for calls with few heads: a team of eight warps on 16 value channels.
//
// Where the channels of all heads together are fewer than the SMs have warps for, a chunk's time is that of one warp's chain of
// products (delta_scan.cuh), and three quarters of every SM stand idle.  Here four warps share the
// chain and four more do what does not lie on it.  The state lies by columns: warp w of the first four holds N / 4 of them for
// the 16 rows.  Products with the state are partial sums over the columns, added up through shared memory by 16 tokens a warp;
// what a warp computes for its 16 tokens the others need as operands comes back the same way, as fragments.  The other four
// warps copy the next chunk's tiles in, form the outputs (from the state's fragments, 16 tokens each) and write everything that
// goes to memory.  Four barriers a chunk.  All tiles are double-buffered: a CTA has its SM to itself.
//
// 32 heads of 32768 tokens (N 128, P 64, bf16): 1083 us forwards, 1178 back, 4100 clocks a chunk (11 thousand for a warp by
// itself).  What is left is the chain: partial sums, X, Tm X and the state's update, each behind a barrier; fragments fetched
// ahead of their barrier made it slower.
#pragma once

#include "delta_scan.cuh"

namespace slx {
namespace delta {

// 64 tokens x 16 columns in TI
template <typename TI>
struct RawTeam {
  static constexpr int ld = 16 + 16 / (int)sizeof(TI);
  static constexpr int size = L * ld;
  static __device__ __forceinline__ void issue(TI *dst, const TI *src, int64_t st, int rows, int cols, bool vec, int tid) {
    constexpr int V = 16 / (int)sizeof(TI), per = 16 / V;
    if (vec) {
#pragma unroll
      for (int n = 0; n < L * per / kThreads; ++n) {
        const int i = n * kThreads + tid, r = i / per, c = i % per * V;
        const bool ok = r < rows && c < cols;
        cp16(dst + r * ld + c, ok ? src + r * st + c : src, ok);
      }
    } else {
#pragma unroll 1
      for (int i = tid; i < L * 16; i += kThreads) {
        const int r = i / 16, c = i % 16;
        dst[r * ld + c] = r < rows && c < cols ? src[r * st + c] : from_f<TI>(0.f);
      }
    }
  }
  // rows 16 w .. + 15, transposed: accumulators with rows p and columns t
  static __device__ __forceinline__ void load(float (&c)[2][4], const TI *tile, int w) {
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    if constexpr (sizeof(TI) == 4) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[j][i] = tile[(16 * w + 8 * j + 2 * q + (i & 1)) * ld + g + (i >> 1) * 8];
    } else {
      uint32_t r[4];
      a_km(r, reinterpret_cast<const __half *>(tile) + 16 * w * ld, ld);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 x;
        if constexpr (std::is_same<TI, __half>::value) x = unpack(r[i]);
        else x = make_float2(__uint_as_float(r[i] << 16), __uint_as_float(r[i] & 0xffff0000u));
        c[i >> 1][(i & 1) * 2] = x.x;
        c[i >> 1][(i & 1) * 2 + 1] = x.y;
      }
    }
  }
};

template <int NT, int SI, int SP, typename TI>  // SP: planes of P
struct alignas(128) TeamStage {  // the tiles of a chunk
  __half k[Operand<SI, NT>::halves], q[Operand<SI, NT>::halves], T[2 * kTri], P[SP * kTri];
  float gamma[L], closing[L], beta[L];
  int tops[3][4], pad[20];
  TI v[RawTeam<TI>::size];
};
template <int NT, int SI, int SP, typename TI>
struct alignas(128) TeamShared {
  TeamStage<NT, SI, SP, TI> stage[2];
  float2 part[4][8][2][32];          // partial sums by warp, tile, row half, lane
  uint4 state[NT / 16][2][32];       // the state's fragments: columns, plane, lane
  uint4 frag[4][4][2][32];           // fragments: kind, warp, plane, lane
  int exps[2][5][4];                 // their exponents, and (4) the state's; two sets in turn
  __half buf[4][16 * (NT / 4 + 8) > 16 * 24 ? 16 * (NT / 4 + 8) : 16 * 24];
};
constexpr int kTeamThreads = 2 * kThreads;
__device__ __forceinline__ void team_barrier() { asm volatile("barrier.sync 1, %0;" ::"n"(kTeamThreads) : "memory"); }

template <int S>
__device__ __forceinline__ void put_frag(uint4 (&dst)[2][32], const Frag<S> &f) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int s = 0; s < S; ++s) dst[s][lane] = make_uint4(f.r[s][0], f.r[s][1], f.r[s][2], f.r[s][3]);
}
template <int S>
__device__ __forceinline__ Frag<S> get_frag(const uint4 (&src)[2][32], int diff) {  // times 2^diff, diff <= 0
  const int lane = threadIdx.x & 31;
  Frag<S> f;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const uint4 x = src[s][lane];
    f.r[s][0] = x.x;
    f.r[s][1] = x.y;
    f.r[s][2] = x.z;
    f.r[s][3] = x.w;
  }
  return scaled(f, diff);
}
// 16 tokens x 16 channels (accumulators: rows p, columns t) to rows t: in TO, or as planes of scaled fp16
template <typename TO>
__device__ __forceinline__ void store_rows16(TO *out, int64_t st, int rows, int cols, const float (&c)[2][4], __half *buf) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  if constexpr (sizeof(TO) == 4) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = 8 * j + 2 * q + (i & 1), p = g + (i >> 1) * 8;
        if (t < rows && p < cols) out[t * st + p] = c[j][i];
      }
  } else {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = c[i >> 1][(i & 1) * 2], y = c[i >> 1][(i & 1) * 2 + 1];
      if constexpr (std::is_same<TO, __half>::value) r[i] = pack(x, y);
      else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        r[i] = *reinterpret_cast<const uint32_t *>(&h);
      }
    }
    __syncwarp();
    stsm_t(smem_addr(buf + ((lane & 7) + (lane >> 4) * 8) * 24 + ((lane >> 3) & 1) * 8), r);
    __syncwarp();
    const int t = lane >> 1, p = (lane & 1) * 8;
    if (cols >= 16 && (st & 7) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
      if (t < rows) *reinterpret_cast<uint4 *>(out + t * st + p) = *reinterpret_cast<const uint4 *>(buf + t * 24 + p);
    } else {
#pragma unroll
      for (int n = 0; n < 8; ++n)
        if (t < rows && p + n < cols) out[t * st + p + n] = reinterpret_cast<const TO *>(buf)[t * 24 + p + n];
    }
  }
}
template <int S>
__device__ __forceinline__ void store_planes16(__half *out, int64_t plane, const Frag<S> &f, __half *buf) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    __syncwarp();
    stsm_t(smem_addr(buf + ((lane & 7) + (lane >> 4) * 8) * 24 + ((lane >> 3) & 1) * 8), f.r[s]);
    __syncwarp();
    *reinterpret_cast<uint4 *>(out + s * plane + (lane >> 1) * kTileLd + (lane & 1) * 8) =
        *reinterpret_cast<const uint4 *>(buf + (lane >> 1) * 24 + (lane & 1) * 8);
  }
}
// NT / 4 columns of 16 rows of a state, from its fragments
template <int S, int NT>
__device__ __forceinline__ void store_state16(__half *out, int64_t plane, const uint4 (*state)[2][32], __half *buf) {
  const int lane = threadIdx.x & 31;
  constexpr int W = NT / 4, ld = W + 8;
#pragma unroll
  for (int pl = 0; pl < S; ++pl) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < W / 16; ++j) {
      const uint4 x = state[j][pl][lane];
      const uint32_t r[4] = {x.x, x.y, x.z, x.w};
      stsm(smem_addr(buf + (lane & 15) * ld + 16 * j + (lane >> 4) * 8), r);
    }
    __syncwarp();
#pragma unroll
    for (int i = lane; i < 16 * (W / 8); i += 32)
      *reinterpret_cast<uint4 *>(out + pl * plane + (i / (W / 8)) * (NT + 8) + (i % (W / 8)) * 8) =
          *reinterpret_cast<const uint4 *>(buf + (i / (W / 8)) * ld + (i % (W / 8)) * 8);
  }
}
// c (16 x 64 tokens) += a (16 x 16 of n) B^T for columns n0 .. of an operand tile
template <int SA, int SB, int NT>
__device__ __forceinline__ void team_rows(float (&c)[8][4], const Frag<SA> &a, const __half *tile, int n0) {
  uint32_t b[4][SB][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int s = 0; s < SB; ++s)
      b_nk(b[i][s], tile + s * Operand<SB, NT>::plane + 16 * i * Operand<SB, NT>::ld + n0, Operand<SB, NT>::ld);
  mma_group<SA, SB, 4>(c, 0, a, b);
}
// c (16 x NT / 4) += a (16 x 16 tokens) B for rows 16 kb .. and columns n0 .. of an operand tile
template <int SA, int SB, int NT>
__device__ __forceinline__ void team_cols(float (&c)[NT / 32][4], const Frag<SA> &a, const __half *tile, int kb, int n0) {
  uint32_t b[NT / 64][SB][4];
#pragma unroll
  for (int i = 0; i < NT / 64; ++i)
#pragma unroll
    for (int s = 0; s < SB; ++s)
      b_kn(b[i][s], tile + s * Operand<SB, NT>::plane + 16 * kb * Operand<SB, NT>::ld + n0 + 16 * i, Operand<SB, NT>::ld);
  mma_group<SA, SB, NT / 64>(c, 0, a, b);
}
__device__ __forceinline__ void put_part(float2 (&dst)[8][2][32], const float (&c)[8][4]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    dst[j][0][lane] = make_float2(c[j][0], c[j][1]);
    dst[j][1][lane] = make_float2(c[j][2], c[j][3]);
  }
}
__device__ __forceinline__ void sum_parts(float (&c)[2][4], const float2 (&src)[4][8][2][32], int w) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float2 s = src[0][2 * w + j][i][lane];
#pragma unroll
      for (int n = 1; n < 4; ++n) {
        const float2 x = src[n][2 * w + j][i][lane];
        s.x += x.x;
        s.y += x.y;
      }
      c[j][2 * i] = s.x;
      c[j][2 * i + 1] = s.y;
    }
}
__device__ __forceinline__ void times_cols16(float (&c)[2][4], const float *s, float f) {
  const int q = threadIdx.x & 3;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float2 x = *reinterpret_cast<const float2 *>(s + 8 * j + 2 * q);
    c[j][0] *= x.x * f;
    c[j][1] *= x.y * f;
    c[j][2] *= x.x * f;
    c[j][3] *= x.y * f;
  }
}

template <int NT>
__device__ __forceinline__ void load_state16(float (&c)[NT / 32][4], const void *src, int dtype, size_t base, int p0, int n0, int P,
                                             int N) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
#pragma unroll
  for (int j = 0; j < NT / 32; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = p0 + g + (i >> 1) * 8, n = n0 + 8 * j + 2 * q + (i & 1);
      c[j][i] = p < P && n < N ? load_as_f(src, dtype, base + (size_t)p * N + n) : 0.f;
    }
}
template <int NT>
__device__ __forceinline__ void write_state16(void *dst, int dtype, size_t base, const float (&c)[NT / 32][4], int p0, int n0, int P,
                                              int N) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
#pragma unroll
  for (int j = 0; j < NT / 32; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = p0 + g + (i >> 1) * 8, n = n0 + 8 * j + 2 * q + (i & 1);
      if (p < P && n < N) store_as(dst, dtype, base + (size_t)p * N + n, c[j][i]);
    }
}

// hi + lo of a fragment as accumulators, times s
template <int S>
__device__ __forceinline__ void frag_values(float (&c)[2][4], const Frag<S> &f, float s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 x = unpack(f.r[0][i]);
    if constexpr (S == 2) {
      const float2 y = unpack(f.r[1][i]);
      x.x += y.x;
      x.y += y.y;
    }
    c[i >> 1][(i & 1) * 2] = x.x * s;
    c[i >> 1][(i & 1) * 2 + 1] = x.y * s;
  }
}

template <int NT, int SI, int SC, typename TI>
__global__ void __launch_bounds__(kTeamThreads) delta_fwd_team_kernel(Args a) {
  using Op = Operand<SI, NT>;
  using Shared = TeamShared<NT, SI, SC, TI>;
  extern __shared__ __align__(128) char smem[];
  Shared &sm = *reinterpret_cast<Shared *>(smem);
  const int w = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
  const bool chain = threadIdx.x < kThreads;
  const int bh = blockIdx.y, b = bh / a.heads, h = bh % a.heads, kh = h / (a.heads / a.key_heads);
  const int p0 = blockIdx.x * 16, n0 = w * (NT / 4), PB = a.P16 / 16, tiles = (a.P16 + 63) / 64;
  const Record *rec = a.rec + (size_t)bh * a.NC;
  // kinds of fragments and exponents: X, beta Y, closing beta Y, Y; the state's
  enum { kX, kD, kC, kY, kS };
  if (chain) {
    float S[NT / 32][4];
    if (a.init) load_state16<NT>(S, a.init, a.init_dtype, (size_t)bh * a.P * a.N, p0, n0, a.P, a.N);
    else zero(S);
    int4 nx = exps_of(rec);
    {
      const int e = warp_exp(S);
      if (lane == 0) sm.exps[0][kS][w] = e;
    }
    for (int c = 0; c < a.NC; ++c) {
      const int4 ex = nx;
      const int eT = ex.x, ek = ex.w;
      const auto &st = sm.stage[c & 1];
      int(&exps)[5][4] = sm.exps[c & 1];
      team_barrier();
      if (c + 1 < a.NC) nx = exps_of(rec + c + 1);
      const int eS = max4(exps[kS]);
      {  // over this warp's columns: S k^T
        float X[8][4];
        zero(X);
        const float s = pow2(-eS);
#pragma unroll
        for (int kb = 0; kb < NT / 64; ++kb) {
          Frag<2> f;
          frag_of<2>(f, S[2 * kb], S[2 * kb + 1], s);
          put_frag<2>(sm.state[w * (NT / 64) + kb], f);
          team_rows<2, SI, NT>(X, f, st.k, n0 + 16 * kb);
        }
        put_part(sm.part[w], X);
      }
      team_barrier();
      float x[2][4];  // this warp's 16 tokens
      {
        float v[2][4];
        RawTeam<TI>::load(v, st.v, w);
        sum_parts(x, sm.part, w);
        times_cols16(x, st.gamma + 16 * w, pow2(eS + ek));
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[j][i] = v[j][i] - x[j][i];
        const int e = warp_exp(x);
        Frag<2> f;
        frag_of<2>(f, x[0], x[1], pow2(-e));
        put_frag<2>(sm.frag[kX][w], f);
        if (lane == 0) exps[kX][w] = e;
      }
      team_barrier();
      {
        const int eX = max4(exps[kX]);
        float z[2][2][4];  // (two chains)
        zero(z[0]);
        zero(z[1]);
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
          if (kb <= w) {
            const Frag<2> f = get_frag<2>(sm.frag[kX][kb], exps[kX][kb] - eX);
            uint32_t bb[2][4];
            b_nk(bb[0], st.T + tri_base(w) + 16 * kb, tri_ld(w));
            b_nk(bb[1], st.T + kTri + tri_base(w) + 16 * kb, tri_ld(w));
            mma_split<2, 2>(z[kb & 1][0], z[kb & 1][1], f, bb);
          }
        const float s = pow2(eX + eT);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[j][i] = (z[0][j][i] + z[1][j][i]) * s;  // Y
        // (the exponents of beta Y and closing beta Y: Y's and the factors' largest)
        const int eY = warp_exp(x), eD = eY + st.tops[1][w], eC = eY + st.tops[2][w];
        if (a.y) {
          Frag<SC> f;
          frag_of<SC>(f, x[0], x[1], pow2(-eY));
          put_frag<SC>(sm.frag[kY][w], f);
          if (lane == 0) exps[kY][w] = eY;
        }
        times_cols16(x, st.beta + 16 * w, 1.f);
        Frag<SC> fd;
        frag_of<SC>(fd, x[0], x[1], pow2(-eD));
        put_frag<SC>(sm.frag[kD][w], fd);
        times_cols16(x, st.closing + 16 * w, 1.f);
        Frag<2> fc;
        frag_of<2>(fc, x[0], x[1], pow2(-eC));
        put_frag<2>(sm.frag[kC][w], fc);
        if (lane == 0) {
          exps[kD][w] = eD;
          exps[kC][w] = eC;
        }
      }
      team_barrier();
      const int eC = floor_exp(max4(exps[kC]), eS + above(st.gamma[L - 1]), ek);
      if constexpr (SC == 2) {
        float D[NT / 32][4];
        zero(D);
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
          team_cols<2, SI, NT>(D, get_frag<2>(sm.frag[kC][kb], exps[kC][kb] - eC), st.k, kb, n0);
        join(S, st.gamma[L - 1], D, pow2(eC + ek));
      } else {
        times(S, st.gamma[L - 1] * pow2(-(eC + ek)));
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
          team_cols<2, SI, NT>(S, get_frag<2>(sm.frag[kC][kb], exps[kC][kb] - eC), st.k, kb, n0);
        times(S, pow2(eC + ek));
      }
      const int e = warp_exp(S);
      if (lane == 0) sm.exps[(c + 1) & 1][kS][w] = e;
    }
    if (a.final_state) write_state16<NT>(a.final_state, SLX_F32, (size_t)bh * a.P * a.N, S, p0, n0, a.P, a.N);
  } else {
    const int tid = threadIdx.x - kThreads;
    __half *buf = sm.buf[w];
    const __half *kq = a.kq + (size_t)(b * a.key_heads + kh) * a.NC * 2 * Op::halves;
    auto issue = [&](int c) {
      auto &st = sm.stage[c & 1];
      copy_bytes<2 * Op::halves * 2>(st.k, kq + (size_t)c * 2 * Op::halves, tid);  // k, q
      copy_bytes<(2 + SC) * kTri * 2>(st.T, rec[c].T, tid);                        // T, P
      copy_bytes<kHeadBytes>(st.gamma, rec[c].gamma, tid);
      RawTeam<TI>::issue(st.v, head_base<TI>(a.v, b, h, c * L) + p0, a.v.st, min(L, a.T - c * L), a.P - p0, a.v.vec, tid);
      cp_commit();
    };
    issue(0);
    for (int c = 0; c < a.NC; ++c) {
      const int4 ex = exps_of(rec + c);
      const int eQ = ex.y, eq = ex.z;
      const auto &st = sm.stage[c & 1];
      int(&exps)[5][4] = sm.exps[c & 1];
      const size_t at = (size_t)bh * a.NC + c;
      cp_wait<0>();
      team_barrier();
      if (c + 1 < a.NC) issue(c + 1);
      const int eS = max4(exps[kS]);
      team_barrier();
      float o[2][4];
      {
        float z[2][2][4];
        zero(z[0]);
        zero(z[1]);
        if (a.o) {
#pragma unroll
          for (int kb = 0; kb < NT / 16; ++kb) {
            const Frag<SC> f = get_frag<SC>(sm.state[kb], 0);
            uint32_t bb[SI][4];
#pragma unroll
            for (int s = 0; s < SI; ++s) b_nk(bb[s], st.q + s * Op::plane + 16 * w * Op::ld + 16 * kb, Op::ld);
            mma_split<SC, SI>(z[kb & 1][0], z[kb & 1][1], f, bb);
          }
        }
        const float s = pow2(eS + eq);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[j][i] = (z[0][j][i] + z[1][j][i]) * s;
      }
      team_barrier();
      if (a.st) {
        store_state16<SC, NT>(a.st + (at * SC * a.P16 + p0) * (NT + 8) + n0, (int64_t)a.P16 * (NT + 8),
                              sm.state + w * (NT / 64), buf);
        if (tid == 0) a.est[at * PB + p0 / 16] = eS;
      }
      times_cols16(o, st.gamma + 16 * w, 1.f);
      const int eo = warp_exp(o);
      team_barrier();
      if (a.o) {
        const int eD = floor_exp(max4(exps[kD]), eo, eQ);
        times(o, pow2(-(eD + eQ)));
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
          if (kb <= w) {
            const Frag<SC> f = get_frag<SC>(sm.frag[kD][kb], exps[kD][kb] - eD);
            uint32_t bb[SC][4];
#pragma unroll
            for (int s = 0; s < SC; ++s) b_nk(bb[s], st.P + s * kTri + tri_base(w) + 16 * kb, tri_ld(w));
            mma_split<SC, SC>(o[0], o[1], f, bb);
          }
        times(o, a.scale * pow2(eD + eQ));
        store_rows16<TI>(static_cast<TI *>(a.o) + ((size_t)bh * a.T + c * L + 16 * w) * a.P + p0, a.P, a.T - c * L - 16 * w,
                         a.P - p0, o, buf);
      }
      if (a.y) {
        const int e = max4(exps[kY]);
        store_planes16<SC>(a.y + (at * SC * tiles + p0 / 64) * kTile + 16 * w * kTileLd + p0 % 64, (int64_t)tiles * kTile,
                           get_frag<SC>(sm.frag[kY][w], exps[kY][w] - e), buf);
        if (tid == 0) a.ey[at * PB + p0 / 16] = e;
      }
    }
    cp_wait<0>();
  }
}

template <int NT, int SI, int SC, typename TI>
__global__ void __launch_bounds__(kTeamThreads) delta_bwd_team_kernel(Args a) {
  using Op = Operand<SI, NT>;
  using Shared = TeamShared<NT, SI, 2, TI>;
  extern __shared__ __align__(128) char smem[];
  Shared &sm = *reinterpret_cast<Shared *>(smem);
  const int w = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
  const bool chain = threadIdx.x < kThreads;
  const int bh = blockIdx.y, b = bh / a.heads, h = bh % a.heads, kh = h / (a.heads / a.key_heads);
  const int p0 = blockIdx.x * 16, n0 = w * (NT / 4), PB = a.P16 / 16, tiles = (a.P16 + 63) / 64;
  const Record *rec = a.rec + (size_t)bh * a.NC;
  // kinds of fragments and exponents: dO, then beta dD in the same place; scale gamma dO; -gamma dX; dX; the state's
  enum { kO, kG, kN, kX, kR };
  if (chain) {
    float R[NT / 32][4];
    if (a.d_final) load_state16<NT>(R, a.d_final, a.d_final_dtype, (size_t)bh * a.P * a.N, p0, n0, a.P, a.N);
    else zero(R);
    int4 nx = exps_of(rec + a.NC - 1);
    {
      const int e = warp_exp(R);
      if (lane == 0) sm.exps[(a.NC - 1) & 1][kR][w] = e;
    }
    for (int c = a.NC - 1; c >= 0; --c) {
      const int4 ex = nx;
      const int eT = ex.x, eQ = ex.y, eq = ex.z, ek = ex.w;
      const auto &st = sm.stage[c & 1];
      int(&exps)[5][4] = sm.exps[c & 1];
      team_barrier();
      if (c > 0) nx = exps_of(rec + c - 1);
      const int eR = max4(exps[kR]);
      {  // over this warp's columns: R k^T
        float X[8][4];
        zero(X);
        const float s = pow2(-eR);
#pragma unroll
        for (int kb = 0; kb < NT / 64; ++kb) {
          Frag<2> f;
          frag_of<2>(f, R[2 * kb], R[2 * kb + 1], s);
          put_frag<2>(sm.state[w * (NT / 64) + kb], f);
          team_rows<2, SI, NT>(X, f, st.k, n0 + 16 * kb);
        }
        put_part(sm.part[w], X);
      }
      team_barrier();
      float x[2][4], y[2][4];
      {
        const int eo = max4(exps[kO]);
        zero(y);
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
          if (kb >= w) {
            const Frag<SI> f = get_frag<SI>(sm.frag[kO][kb], exps[kO][kb] - eo);
            uint32_t bb[2][4];
            b_kn(bb[0], st.P + tri_base(kb) + 16 * w, tri_ld(kb));
            b_kn(bb[1], st.P + kTri + tri_base(kb) + 16 * w, tri_ld(kb));
            mma_split<SI, 2>(y[0], y[1], f, bb);
          }
        sum_parts(x, sm.part, w);
        times_cols16(x, st.closing + 16 * w, pow2(eR + ek));
        const float s = a.scale * pow2(eo + eQ);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[j][i] = fmaf(y[j][i], s, x[j][i]);
        times_cols16(x, st.beta + 16 * w, 1.f);
        const int e = warp_exp(x);
        Frag<2> f;
        frag_of<2>(f, x[0], x[1], pow2(-e));
        put_frag<2>(sm.frag[kX][w], f);  // (beta dD, until dX takes the place)
        if (lane == 0) exps[kX][w] = e;
      }
      team_barrier();
      {
        const int eX = max4(exps[kX]);
        float z[2][2][4];  // (two chains)
        zero(z[0]);
        zero(z[1]);
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
          if (kb >= w) {
            const Frag<2> f = get_frag<2>(sm.frag[kX][kb], exps[kX][kb] - eX);
            uint32_t bb[2][4];
            b_kn(bb[0], st.T + tri_base(kb) + 16 * w, tri_ld(kb));
            b_kn(bb[1], st.T + kTri + tri_base(kb) + 16 * w, tri_ld(kb));
            mma_split<2, 2>(z[kb & 1][0], z[kb & 1][1], f, bb);
          }
        const float s = pow2(eX + eT);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[j][i] = (z[0][j][i] + z[1][j][i]) * s;  // dX
        const int eW = warp_exp(x), eN = eW + st.tops[0][w];
        Frag<2> f;
        frag_of<2>(f, x[0], x[1], pow2(-eW));
        put_frag<2>(sm.frag[kO][w], f);  // (dO's place: everybody has read it)
        times_cols16(x, st.gamma + 16 * w, -1.f);
        frag_of<2>(f, x[0], x[1], pow2(-eN));
        put_frag<2>(sm.frag[kN][w], f);
        if (lane == 0) {
          exps[kO][w] = eW;
          exps[kN][w] = eN;
        }
      }
      team_barrier();
      const int eD = eR + above(st.gamma[L - 1]);  // of the decayed R
      const int u1 = floor_exp(max4(exps[kG]), eD, eq);
      const int u2 = floor_exp(max4(exps[kN]), max(eD, u1 + eq + 21) + 1, ek);
      if constexpr (SC == 2) {
        float D[NT / 32][4], E[NT / 32][4];
        zero(D);
        zero(E);
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
          team_cols<2, SI, NT>(D, get_frag<2>(sm.frag[kG][kb], exps[kG][kb] - u1), st.q, kb, n0);
          team_cols<2, SI, NT>(E, get_frag<2>(sm.frag[kN][kb], exps[kN][kb] - u2), st.k, kb, n0);
        }
        join(R, st.gamma[L - 1], D, pow2(u1 + eq));
        join(R, 1.f, E, pow2(u2 + ek));
      } else {
        times(R, st.gamma[L - 1] * pow2(-(u1 + eq)));
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
          team_cols<2, SI, NT>(R, get_frag<2>(sm.frag[kG][kb], exps[kG][kb] - u1), st.q, kb, n0);
        times(R, pow2(u1 + eq - (u2 + ek)));
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
          team_cols<2, SI, NT>(R, get_frag<2>(sm.frag[kN][kb], exps[kN][kb] - u2), st.k, kb, n0);
        times(R, pow2(u2 + ek));
      }
      const int e = warp_exp(R);
      if (lane == 0) sm.exps[(c + 1) & 1][kR][w] = e;
    }
    if (a.d_init) write_state16<NT>(a.d_init, a.d_init_dtype, (size_t)bh * a.P * a.N, R, p0, n0, a.P, a.N);
  } else {
    const int tid = threadIdx.x - kThreads;
    __half *buf = sm.buf[w];
    const __half *kq = a.kq + (size_t)(b * a.key_heads + kh) * a.NC * 2 * Op::halves;
    auto issue = [&](int c) {
      auto &st = sm.stage[c & 1];
      copy_bytes<2 * Op::halves * 2>(st.k, kq + (size_t)c * 2 * Op::halves, tid);  // k, q
      copy_bytes<4 * kTri * 2>(st.T, rec[c].T, tid);                               // T, P
      copy_bytes<kHeadBytes>(st.gamma, rec[c].gamma, tid);
      RawTeam<TI>::issue(st.v, head_base<TI>(a.dO, b, h, c * L) + p0, a.dO.st, min(L, a.T - c * L), a.P - p0, a.dO.vec, tid);
      cp_commit();
    };
    issue(a.NC - 1);
    for (int c = a.NC - 1; c >= 0; --c) {
      const auto &st = sm.stage[c & 1];
      int(&exps)[5][4] = sm.exps[c & 1];
      const size_t at = (size_t)bh * a.NC + c;
      cp_wait<0>();
      team_barrier();
      const int eR = max4(exps[kR]);
      float d[2][4];
      RawTeam<TI>::load(d, st.v, w);
      {  // dO of 16 tokens
        const int e = std::is_same<TI, __half>::value ? 0 : warp_exp(d);
        Frag<SI> f;
        frag_of<SI>(f, d[0], d[1], pow2(-e));
        put_frag<SI>(sm.frag[kO][w], f);
        if (lane == 0) exps[kO][w] = e;
      }
      if (c > 0) issue(c - 1);
      team_barrier();
      if (tid == 0) {
        a.edo[at * PB + p0 / 16] = max4(exps[kO]);
        a.eds[at * PB + p0 / 16] = eR;
      }
      {
        times_cols16(d, st.gamma + 16 * w, a.scale);
        const int e = warp_exp(d);
        Frag<2> f;
        frag_of<2>(f, d[0], d[1], pow2(-e));
        put_frag<2>(sm.frag[kG][w], f);
        if (lane == 0) exps[kG][w] = e;
      }
      team_barrier();
      store_state16<SC, NT>(a.ds + (at * SC * a.P16 + p0) * (NT + 8) + n0, (int64_t)a.P16 * (NT + 8), sm.state + w * (NT / 64), buf);
      team_barrier();
      const int e = max4(exps[kO]);  // of dX by now
      const Frag<2> f = get_frag<2>(sm.frag[kO][w], exps[kO][w] - e);
      Frag<SC> fs;
#pragma unroll
      for (int s = 0; s < SC; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) fs.r[s][i] = f.r[s][i];
      store_planes16<SC>(a.dx + (at * SC * tiles + p0 / 64) * kTile + 16 * w * kTileLd + p0 % 64, (int64_t)tiles * kTile, fs, buf);
      float y[2][4];
      frag_values<2>(y, get_frag<2>(sm.frag[kO][w], 0), pow2(exps[kO][w]));
      store_rows16<TI>(static_cast<TI *>(a.dv) + ((size_t)bh * a.T + c * L + 16 * w) * a.P + p0, a.P, a.T - c * L - 16 * w,
                       a.P - p0, y, buf);
      if (tid == 0) a.edx[at * PB + p0 / 16] = e;
    }
    cp_wait<0>();
  }
}

}  // namespace delta
}  // namespace slx
