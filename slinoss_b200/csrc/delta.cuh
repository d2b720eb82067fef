// Shared pieces of the gated delta rule kernels: sizes, the per-chunk record, scaled fp16 operands and the matrix
// instructions.
//
// Recurrence of a head, a_t = exp(g_t), state S (P, N):
//     y_t = v_t - a_t S_{t-1} k_t,   S_t = a_t S_{t-1} + beta_t y_t k_t^T,   o_t = scale S_t q_t
// over chunks of 64 tokens.  With G the running sum of g inside a chunk, S0 the state before it,
// dec_ts = e^{G_t-G_s}, closing_s = e^{G_63-G_s}:
//     M_ts = dec_ts k_t.k_s (s < t),   Tm = (I + M diag(beta))^{-1},   Y = Tm (v - e^G S0 k)
//     P_ts = dec_ts q_t.k_s (s <= t),  o = scale (e^G S0 q + P beta Y),  S1 = e^{G_63} S0 + sum_s closing_s beta_s y_s k_s^T
//
// Operands.  Products run on the fp16 matrix instructions with fp32 sums.  bf16 and fp16 values are exact in fp16 once a
// power of two per tile has brought the tile's largest magnitude to [2^14, 2^15); a computed operand is one fp16 value
// (11 bits) where the result is rounded to bf16 anyway, and a pair hi + lo (22 bits) where it feeds an fp32 or fp16 result.
// A pair costs two or three products instead of one.  (bf16 pairs hold 16 bits: 3e-6 in the fp32 states, against 2e-7.)
#pragma once

#include <type_traits>

#include "common.cuh"

namespace slx {
namespace delta {

constexpr int L = 64;             // tokens of a chunk
constexpr int kTri = 128 * 4 * 4 + 256 * 4;  // elements of a lower triangular 64 x 64 tile, by row blocks of 16 (tri_at)
constexpr int kThreads = 128;
constexpr int kTileLd = 72, kTile = L * kTileLd;  // Y and dX: 64 tokens x up to 64 value channels

// What every later kernel needs of one chunk and value head, written once by delta_chunk_kernel.
struct Record {
  __half T[2][kTri];  // Tm, hi and lo
  __half Q[2][kTri];  // P, hi and lo
  float gamma[L], closing[L], beta[L];
  int tops[3][4];  // of gamma, beta and closing beta in each 16 tokens: least e with all magnitudes below 2^e
  int pad0[20];    // (what is copied whole keeps its neighbours on 128-byte lines)
  // dec_ts for t and s in the same block of 16 tokens is near[block][t][s]; for t in block i and s in an earlier one it is
  // rise[t] * fall[fall_at(i) + s]: both exponents from G at the end of block i - 1, so that neither factor leaves the range
  // where gates close
  float rise[L], fall[96], near[4][16 * 20];
  int eT, eQ, eq, ek;  // binary exponents: value = stored * 2^e
  int pad1[28];
};
static_assert(sizeof(Record) == 31360 && sizeof(Record) % 128 == 0, "record layout");
constexpr int kHeadBytes = 3 * L * 4 + 128;  // gamma, closing, beta, tops
constexpr int kVectorBytes = kHeadBytes + L * 4 + 96 * 4 + 4 * 16 * 20 * 4;  // gamma .. near
constexpr int kNearLd = 20;
__host__ __device__ constexpr int fall_at(int i) { return 8 * i * (i - 1); }

struct Rows {  // a (batch, head, token, :) tensor whose last axis is dense; strides in elements
  const void *p;
  int64_t sb, sh, st;
  int vec;  // 16-byte accesses are aligned
};

struct Args {
  int batch, heads, key_heads, T, P, N, NC;
  int P16;  // P rounded up to 16
  float scale;
  int g_dtype, beta_dtype;
  Rows q, k, v, g, beta, dO;
  Record *rec;              // (batch*heads, NC)
  __half *kq;               // (batch*key_heads, NC): k, then q, as Operand holds them in shared memory
  // forward
  const void *init;         // (batch, heads, P, N) or null
  int init_dtype;
  void *o;                  // (batch, heads, T, P) or null
  float *final_state;       // or null
  __half *st;               // states before every chunk: (BH, NC, planes, P16, NT + 8), or null
  __half *y;                // Y of every chunk: (BH, NC, planes, tiles of 64 channels, 64, 72), or null
  int *est, *ey;            // (BH, NC, P16 / 16)
  // backward
  const void *d_final;
  int d_final_dtype;
  void *d_init;
  int d_init_dtype;
  __half *ds, *dx;          // as st and y: gradients of the states after every chunk, dX
  int *eds, *edx, *edo;
  void *dv;                 // (batch, heads, T, P)
  void *dq, *dk;            // (batch, key_heads, T, N) in dtype, or fp32 per value head where heads share keys
  void *dg, *dbeta;         // (batch, heads, T)
};

// ---- 64 x 64 lower triangular tiles: row blocks of 16 rows, block i holds columns 0 .. 16 i + 15 and 8 of padding (an odd
// number of 16-byte units per row: ldmatrix meets no bank twice).  5/8 of the square's bytes.
__host__ __device__ constexpr int tri_base(int i) { return 128 * i * i + 256 * i; }
__host__ __device__ constexpr int tri_ld(int i) { return 16 * i + 24; }

// Row-major operand tiles of 64 tokens x W columns, SI fp16 planes one after another; rows are padded to an odd number of
// 16-byte units.
template <int SI, int W>
struct Operand {
  static constexpr int ld = W + 8;
  static constexpr int plane = L * ld;
  static constexpr int halves = SI * plane;
};

// ---- exponents -----------------------------------------------------------------------------------------------------
constexpr int kZeroExp = -100;  // of a tile of zeros
// Of a tile that holds an infinity or NaN.  pow2 of it, by which results are brought back to their unit, is NaN, so that all of
// them are NaN and not finite values that scaling by the infinity has wiped out.  (pow2 of its negative, by which the tile is
// brought to fp16, is zero.)
constexpr int kNanExp = 2000;
// (zero below the normal range)
__device__ __forceinline__ float pow2(int e) {
  return e > 1000 ? __int_as_float(0x7fc00000) : __int_as_float((min(max(e, -127), 127) + 127) << 23);
}
// e with max * 2^-e in [2^14, 2^15), from the bits of the largest magnitude
__device__ __forceinline__ int exp_of(unsigned bits) {
  return bits >= 0x7f800000u ? kNanExp : bits == 0u ? kZeroExp : max((int)(bits >> 23) - 127 - 14, kZeroExp);
}
// least e with |x| < 2^e (for the exponent of values times x)
__device__ __forceinline__ int above(float x) {
  const unsigned b = __float_as_uint(x) & 0x7fffffffu;
  return b >= 0x7f800000u ? kNanExp : (int)(b >> 23) - 126;
}
// x 2^e in two steps: e may pass the range where the product does not
__device__ __forceinline__ float times_pow2(float x, int e) { return x * pow2(e >> 1) * pow2(e - (e >> 1)); }
// an exponent for a product's operand such that an accumulator of exponent ec, brought to the product's unit e + eb, stays
// far inside the range (what the raising rounds away is 2^-40 of the accumulator), and the unit does too.  (ec: of what the
// accumulator will be when the product joins it, behind its decay: a state that a gate has closed on keeps what was written
// before the gate.)
constexpr int kLowestUnit = -100;
__device__ __forceinline__ int floor_exp(int e, int ec, int eb) { return max(e, max(ec - 40, kLowestUnit) - eb); }
__device__ __forceinline__ unsigned mag(float x) { return __float_as_uint(x) & 0x7fffffffu; }
template <int n>
__device__ __forceinline__ unsigned max_mag(const float (&c)[n][4]) {
  unsigned m[4] = {0, 0, 0, 0};  // (four short chains)
#pragma unroll
  for (int j = 0; j < n; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = max(m[i], mag(c[j][i]));
  return max(max(m[0], m[1]), max(m[2], m[3]));
}
template <int n>
__device__ __forceinline__ int warp_exp(const float (&c)[n][4]) {
  return exp_of(__reduce_max_sync(0xffffffffu, max_mag(c)));
}

// ---- matrix instructions -------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void stsm(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};"
               :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void stsm_t(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};"
               :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
// A 16 x 16 block of a row-major half tile at `tile` (leading dimension ld).  The four registers are
//   block_rows:  {rows 0-7, cols 0-7}, {rows 8-15, cols 0-7}, {rows 0-7, cols 8-15}, {rows 8-15, cols 8-15}
//   block_cols:  the same with rows and columns exchanged in the order: {0-7, 0-7}, {0-7, 8-15}, {8-15, 0-7}, {8-15, 8-15}
// read plainly or transposed.  As operands:
//   A (16 x 16) from [m][k]: block_rows plain;  from [k][m]: block_cols transposed
//   B (16 x 16, two n8 tiles b[0..1], b[2..3]) from [n][k]: block_cols plain;  from [k][n]: block_rows transposed
__device__ __forceinline__ uint32_t block_rows(const __half *tile, int ld) {
  const int lane = threadIdx.x & 31;
  return smem_addr(tile + (lane & 15) * ld + (lane >> 4) * 8);
}
__device__ __forceinline__ uint32_t block_cols(const __half *tile, int ld) {
  const int lane = threadIdx.x & 31;
  return smem_addr(tile + ((lane & 7) + (lane >> 4) * 8) * ld + ((lane >> 3) & 1) * 8);
}
__device__ __forceinline__ void a_mk(uint32_t (&r)[4], const __half *t, int ld) { ldsm(r, block_rows(t, ld)); }
__device__ __forceinline__ void a_km(uint32_t (&r)[4], const __half *t, int ld) { ldsm_t(r, block_cols(t, ld)); }
__device__ __forceinline__ void b_nk(uint32_t (&r)[4], const __half *t, int ld) { ldsm(r, block_cols(t, ld)); }
__device__ __forceinline__ void b_kn(uint32_t (&r)[4], const __half *t, int ld) { ldsm_t(r, block_rows(t, ld)); }

__device__ __forceinline__ uint32_t pack(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack(uint32_t r) { return __half22float2(*reinterpret_cast<const __half2 *>(&r)); }
// planes of two values, already scaled
template <int S>
__device__ __forceinline__ void split(float x, float y, uint32_t *hi, uint32_t *lo) {
  *hi = pack(x, y);
  if constexpr (S == 2) {
    const float2 h = unpack(*hi);
    *lo = pack(x - h.x, y - h.y);
  }
}

// An A operand: S planes of a 16 x 16 block.
template <int S>
struct Frag {
  uint32_t r[S][4];
};
// from the accumulators of two neighbouring n8 tiles, times s
template <int S>
__device__ __forceinline__ void frag_of(Frag<S> &f, const float (&c0)[4], const float (&c1)[4], float s) {
  uint32_t *lo = f.r[S - 1];
  split<S>(c0[0] * s, c0[1] * s, &f.r[0][0], lo + 0);
  split<S>(c0[2] * s, c0[3] * s, &f.r[0][1], lo + 1);
  split<S>(c1[0] * s, c1[1] * s, &f.r[0][2], lo + 2);
  split<S>(c1[2] * s, c1[3] * s, &f.r[0][3], lo + 3);
}
template <int S>
__device__ __forceinline__ Frag<S> scaled(const Frag<S> &f, int diff) {  // times 2^diff, diff <= 0
  const __half2 m = __float2half2_rn(pow2(diff));
  Frag<S> r;
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 x = __hmul2(*reinterpret_cast<const __half2 *>(&f.r[s][i]), m);
      r.r[s][i] = *reinterpret_cast<const uint32_t *>(&x);
    }
  return r;
}

// c0, c1 += A B for the two n8 tiles of B; planes of A and B whose product is below 2^-22 are left out
template <int SA, int SB>
__device__ __forceinline__ void mma_split(float (&c0)[4], float (&c1)[4], const Frag<SA> &a, const uint32_t (&b)[SB][4]) {
  mma(c0, a.r[0], b[0][0], b[0][1]);
  mma(c1, a.r[0], b[0][2], b[0][3]);
  if constexpr (SA == 2) {
    mma(c0, a.r[1], b[0][0], b[0][1]);
    mma(c1, a.r[1], b[0][2], b[0][3]);
  }
  if constexpr (SB == 2) {
    mma(c0, a.r[0], b[1][0], b[1][1]);
    mma(c1, a.r[0], b[1][2], b[1][3]);
  }
}
// The same for the n8 tiles 2 first .. 2 (first + n) - 1 of an accumulator and n blocks of B, plane by plane: neighbouring
// instructions add to different tiles, so that none waits for the one before it.
template <int SA, int SB, int n, int tiles>
__device__ __forceinline__ void mma_group(float (&c)[tiles][4], int first, const Frag<SA> &a, const uint32_t (&b)[n][SB][4]) {
#pragma unroll
  for (int i = 0; i < n; ++i) {
    mma(c[2 * (first + i)], a.r[0], b[i][0][0], b[i][0][1]);
    mma(c[2 * (first + i) + 1], a.r[0], b[i][0][2], b[i][0][3]);
  }
  if constexpr (SA == 2) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
      mma(c[2 * (first + i)], a.r[1], b[i][0][0], b[i][0][1]);
      mma(c[2 * (first + i) + 1], a.r[1], b[i][0][2], b[i][0][3]);
    }
  }
  if constexpr (SB == 2) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
      mma(c[2 * (first + i)], a.r[0], b[i][1][0], b[i][1][1]);
      mma(c[2 * (first + i) + 1], a.r[0], b[i][1][2], b[i][1][3]);
    }
  }
}
template <int n>
__device__ __forceinline__ void zero(float (&c)[n][4]) {
#pragma unroll
  for (int j = 0; j < n; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) c[j][i] = 0.f;
}
// c (16 x 64 tokens) += a (16 x 64) B^T for a lower triangular tile B: columns t take the blocks s <= t.
template <int SA, int SB, int kb>
__device__ __forceinline__ void tri_rows_step(float (&c)[8][4], const Frag<SA> (&a)[4], const __half *tile) {
  uint32_t b[4 - kb][SB][4];
#pragma unroll
  for (int i = 0; i < 4 - kb; ++i)
#pragma unroll
    for (int s = 0; s < SB; ++s) b_nk(b[i][s], tile + s * kTri + tri_base(kb + i) + 16 * kb, tri_ld(kb + i));
  mma_group<SA, SB, 4 - kb>(c, kb, a[kb], b);
}
template <int SA, int SB>
__device__ __forceinline__ void tri_rows(float (&c)[8][4], const Frag<SA> (&a)[4], const __half *tile) {
  tri_rows_step<SA, SB, 0>(c, a, tile);
  tri_rows_step<SA, SB, 1>(c, a, tile);
  tri_rows_step<SA, SB, 2>(c, a, tile);
  tri_rows_step<SA, SB, 3>(c, a, tile);
}
// c += a B: columns s take the blocks t >= s.
template <int SA, int SB, int kb>
__device__ __forceinline__ void tri_cols_step(float (&c)[8][4], const Frag<SA> (&a)[4], const __half *tile) {
  uint32_t b[kb + 1][SB][4];
#pragma unroll
  for (int i = 0; i <= kb; ++i)
#pragma unroll
    for (int s = 0; s < SB; ++s) b_kn(b[i][s], tile + s * kTri + tri_base(kb) + 16 * i, tri_ld(kb));
  mma_group<SA, SB, kb + 1>(c, 0, a[kb], b);
}
template <int SA, int SB>
__device__ __forceinline__ void tri_cols(float (&c)[8][4], const Frag<SA> (&a)[4], const __half *tile) {
  tri_cols_step<SA, SB, 3>(c, a, tile);
  tri_cols_step<SA, SB, 2>(c, a, tile);
  tri_cols_step<SA, SB, 1>(c, a, tile);
  tri_cols_step<SA, SB, 0>(c, a, tile);
}
// c (16 x 64 tokens) += a (16 x 16 of n) B^T for columns 16 kb .. of an operand tile [t][n]
template <int SA, int SB, int W>
__device__ __forceinline__ void tile_rows(float (&c)[8][4], const Frag<SA> &a, const __half *tile, int kb) {
  uint32_t b[4][SB][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int s = 0; s < SB; ++s)
      b_nk(b[i][s], tile + s * Operand<SB, W>::plane + 16 * i * Operand<SB, W>::ld + 16 * kb, Operand<SB, W>::ld);
  mma_group<SA, SB, 4>(c, 0, a, b);
}
// c (16 x W) += a (16 x 16 tokens) B for rows 16 kb .. of a row-major tile of W columns (planes `plane` apart)
// (group: blocks of B that are held at a time; cols: columns from `tile` on, all W of them or fewer)
template <int SA, int SB, int W, int group = 4, int cols = W>
__device__ __forceinline__ void tile_cols(float (&c)[cols / 8][4], const Frag<SA> &a, const __half *tile, int plane, int kb) {
#pragma unroll
  for (int n0 = 0; n0 < cols / 16; n0 += group) {
    uint32_t b[group][SB][4];
#pragma unroll
    for (int i = 0; i < group; ++i)
#pragma unroll
      for (int s = 0; s < SB; ++s) b_kn(b[i][s], tile + s * plane + 16 * kb * (W + 8) + 16 * (n0 + i), W + 8);
    mma_group<SA, SB, group>(c, n0, a, b);
  }
}
template <int n>
__device__ __forceinline__ void times(float (&c)[n][4], float s) {
#pragma unroll
  for (int j = 0; j < n; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) c[j][i] *= s;
}
template <int n>
__device__ __forceinline__ void times_rows(float (&c)[n][4], float s0, float s1) {  // rows lane / 4 and lane / 4 + 8
#pragma unroll
  for (int j = 0; j < n; ++j) {
    c[j][0] *= s0;
    c[j][1] *= s0;
    c[j][2] *= s1;
    c[j][3] *= s1;
  }
}

// ---- asynchronous copies -------------------------------------------------------------------------------------------
__device__ __forceinline__ void cp16(void *dst, const void *src, bool valid) {  // zeros where not valid
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(smem_addr(dst)), "l"(src), "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(n) : "memory"); }

template <typename TI>
__device__ __forceinline__ const TI *head_base(const Rows &r, int b, int h, int t) {
  return static_cast<const TI *>(r.p) + b * r.sb + h * r.sh + (int64_t)t * r.st;
}

// A tile of 64 tokens x W columns from global memory in 16-byte pieces, `per` of a thread, zeros outside rows and cols.
// (By the first kThreads threads of a CTA.)
template <typename TI, int W>
struct Pieces {
  static constexpr int V = 16 / (int)sizeof(TI), per = L * W / V / kThreads;
  uint4 x[per];
  static __device__ __forceinline__ int row(int i) { return (i * kThreads + (int)threadIdx.x) / (W / V); }
  static __device__ __forceinline__ int col(int i) { return (i * kThreads + (int)threadIdx.x) % (W / V) * V; }
  static __device__ __forceinline__ void meet() { asm volatile("barrier.sync 2, %0;" ::"n"(kThreads) : "memory"); }
  // (room: as many bytes of shared memory as the tile has, for rows that no 16-byte access fits)
  __device__ __forceinline__ void load(const TI *src, int64_t st, int rows, int cols, bool vec, void *room) {
    if (!vec) {
      TI *raw = static_cast<TI *>(room);
#pragma unroll 1
      for (int i = threadIdx.x; i < L * W; i += kThreads) {
        const int r = i / W, c = i % W;
        raw[i] = r < rows && c < cols ? src[r * st + c] : from_f<TI>(0.f);
      }
      meet();
    }
#pragma unroll
    for (int i = 0; i < per; ++i) {
      const int r = row(i), c = col(i);
      x[i] = make_uint4(0, 0, 0, 0);
      if (!vec) x[i] = static_cast<const uint4 *>(room)[i * kThreads + threadIdx.x];
      else if (r < rows && c < cols) x[i] = *reinterpret_cast<const uint4 *>(src + r * st + c);
    }
    if (!vec) meet();
  }
  __device__ __forceinline__ unsigned max_bits() const {  // of the largest magnitude, as fp32 (a NaN is the largest)
    if constexpr (sizeof(TI) == 4) {
      unsigned m = 0;
#pragma unroll
      for (int i = 0; i < per; ++i) m = max(max(max(m, x[i].x & 0x7fffffffu), max(x[i].y & 0x7fffffffu, x[i].z & 0x7fffffffu)), x[i].w & 0x7fffffffu);
      return m;
    } else {
      __nv_bfloat162 m[2] = {__float2bfloat162_rn(0.f), __float2bfloat162_rn(0.f)};
#pragma unroll
      for (int i = 0; i < per; ++i) {
        const __nv_bfloat162 *w = reinterpret_cast<const __nv_bfloat162 *>(&x[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j & 1] = __hmax2_nan(m[j & 1], __habs2(w[j]));
      }
      const __nv_bfloat162 r = __hmax2_nan(m[0], m[1]);
      const uint32_t bits = *reinterpret_cast<const uint32_t *>(&r);
      return max((bits << 16) & 0x7fffffffu, bits & 0x7fff0000u);
    }
  }
  // as scaled fp16, to an operand tile in shared memory and (COPY) to a copy of it in global memory
  template <int SI, bool COPY>
  __device__ __forceinline__ void store(__half *tile, __half *copy, int e) const {
    constexpr int ld = Operand<SI, W>::ld, plane = Operand<SI, W>::plane;
    const float s = pow2(-e);
#pragma unroll
    for (int i = 0; i < per; ++i) {
      const int at = row(i) * ld + col(i);
      if constexpr (sizeof(TI) == 4) {
        uint2 hi, lo;
        split<2>(__uint_as_float(x[i].x) * s, __uint_as_float(x[i].y) * s, &hi.x, &lo.x);
        split<2>(__uint_as_float(x[i].z) * s, __uint_as_float(x[i].w) * s, &hi.y, &lo.y);
        *reinterpret_cast<uint2 *>(tile + at) = hi;
        *reinterpret_cast<uint2 *>(tile + plane + at) = lo;
        if constexpr (COPY) {
          *reinterpret_cast<uint2 *>(copy + at) = hi;
          *reinterpret_cast<uint2 *>(copy + plane + at) = lo;
        }
      } else {
        uint4 h = x[i];
        if constexpr (!std::is_same<TI, __half>::value) {
          uint32_t *w = reinterpret_cast<uint32_t *>(&h);
          const __nv_bfloat162 s2 = __float2bfloat162_rn(s);
#pragma unroll
          for (int j = 0; j < 4; ++j) {  // (times a power of two: exact, but for what fp16 rounds to zero)
            const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162 *>(&w[j]), s2);
            const uint32_t b = *reinterpret_cast<const uint32_t *>(&y);
            w[j] = pack(__uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u));
          }
        }
        *reinterpret_cast<uint4 *>(tile + at) = h;
        if constexpr (COPY) *reinterpret_cast<uint4 *>(copy + at) = h;
      }
    }
  }
};

// A raw tile of 64 tokens x up to 64 columns, kept in TI.
template <typename TI>
struct Raw {
  static constexpr int ld = 64 + 16 / (int)sizeof(TI);
  static constexpr int bytes = L * ld * (int)sizeof(TI);
  static __device__ __forceinline__ void issue(TI *dst, const TI *src, int64_t st, int rows, int cols, bool vec) {
    constexpr int V = 16 / (int)sizeof(TI), per = 64 / V;
    if (vec) {
#pragma unroll
      for (int n = 0; n < L * per / kThreads; ++n) {
        const int i = n * kThreads + threadIdx.x, r = i / per, c = i % per * V;
        const bool ok = r < rows && c < cols;
        cp16(dst + r * ld + c, ok ? src + r * st + c : src, ok);
      }
    } else {
      for (int i = threadIdx.x; i < L * 64; i += kThreads) {
        const int r = i / 64, c = i % 64;
        dst[r * ld + c] = r < rows && c < cols ? src[r * st + c] : from_f<TI>(0.f);
      }
    }
  }
};

// asynchronous, a multiple of 16 bytes, by kThreads threads of which this is number `tid`
template <int bytes>
__device__ __forceinline__ void copy_bytes(void *dst, const void *src, int tid) {
  static_assert(bytes % 16 == 0, "copies of 16 bytes");
  char *d = static_cast<char *>(dst) + tid * 16;
  const char *s = static_cast<const char *>(src) + tid * 16;
#pragma unroll
  for (int i = 0; i < bytes / 16 / kThreads; ++i) cp16(d + i * kThreads * 16, s + i * kThreads * 16, true);
  constexpr int whole = bytes / 16 / kThreads * kThreads * 16;
  if (whole < bytes && tid * 16 < bytes - whole) cp16(d + whole, s + whole, true);
}
template <int bytes>
__device__ __forceinline__ void copy_bytes(void *dst, const void *src) {
  copy_bytes<bytes>(dst, src, threadIdx.x);
}

// A warp's (16 columns p, 64 tokens) result, held transposed in accumulators (rows p, columns t), to global rows of `out`
// at its column p0: through `buf` (64 x 24 halves of the warp's own) for half types, directly for fp32.
template <typename TO>
__device__ __forceinline__ void store_rows(TO *out, int64_t st, int rows, int cols, const float (&c)[8][4], __half *buf) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  if constexpr (sizeof(TO) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = 8 * j + 2 * q + (i & 1), p = g + (i >> 1) * 8;
        if (t < rows && p < cols) out[t * st + p] = c[j][i];
      }
  } else {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
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
      // matrices {p 0-7, t 0-7}, {p 8-15, t 0-7}, {p 0-7, t 8-15}, {p 8-15, t 8-15} of [p][t], stored as [t][p]
      stsm_t(smem_addr(buf + (8 * j + (lane & 7) + (lane >> 4) * 8) * 24 + ((lane >> 3) & 1) * 8), r);
    }
    __syncwarp();
    const bool wide = cols >= 16 && (st & 7) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    if (wide) {
#pragma unroll
      for (int i = lane; i < 128; i += 32)
        if ((i >> 1) < rows)
          *reinterpret_cast<uint4 *>(out + (i >> 1) * st + (i & 1) * 8) =
              *reinterpret_cast<const uint4 *>(buf + (i >> 1) * 24 + (i & 1) * 8);
    } else {
      for (int i = lane; i < 1024; i += 32)
        if ((i >> 4) < rows && (i & 15) < cols)
          out[(i >> 4) * st + (i & 15)] = reinterpret_cast<const TO *>(buf)[(i >> 4) * 24 + (i & 15)];
    }
  }
}

// Accumulators (rows p, columns t) as S planes of scaled fp16 rows [t][p] in global memory (leading dimension st, 64 rows,
// always whole), scaled by 2^-e.
template <int S>
__device__ __forceinline__ void store_planes(__half *out, int64_t st, int64_t plane, const float (&c)[8][4], int e, __half *buf) {
  const int lane = threadIdx.x & 31;
  const float s = pow2(-e);
#pragma unroll
  for (int pl = 0; pl < S; ++pl) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      Frag<S> f;
      frag_of<S>(f, c[j], c[j + 1], s);
      stsm_t(smem_addr(buf + (8 * j + (lane & 7) + (lane >> 4) * 8) * 24 + ((lane >> 3) & 1) * 8), f.r[pl]);
    }
    __syncwarp();
#pragma unroll
    for (int i = lane; i < 128; i += 32)
      *reinterpret_cast<uint4 *>(out + pl * plane + (i >> 1) * st + (i & 1) * 8) =
          *reinterpret_cast<const uint4 *>(buf + (i >> 1) * 24 + (i & 1) * 8);
  }
}

// A warp's 16 rows of a state (accumulators: rows p, columns n) as S planes of fp16 rows of NT columns (NT + 8 apart), scaled
// by 2^-e.
template <int S, int NT>
__device__ __forceinline__ void store_state(__half *out, int64_t plane, const float (&c)[NT / 8][4], int e, __half *buf) {
  const int lane = threadIdx.x & 31;
  const float s = pow2(-e);
  constexpr int ld = NT + 8;
#pragma unroll
  for (int pl = 0; pl < S; ++pl) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NT / 8; j += 2) {
      Frag<S> f;
      frag_of<S>(f, c[j], c[j + 1], s);
      stsm(smem_addr(buf + (lane & 15) * ld + 8 * j + (lane >> 4) * 8), f.r[pl]);
    }
    __syncwarp();
#pragma unroll
    for (int i = lane; i < 16 * (NT / 8); i += 32)
      *reinterpret_cast<uint4 *>(out + pl * plane + (i / (NT / 8)) * ld + (i % (NT / 8)) * 8) =
          *reinterpret_cast<const uint4 *>(buf + (i / (NT / 8)) * ld + (i % (NT / 8)) * 8);
  }
}

// rows p0 .. p0 + 15 of a (P, N) matrix in any dtype, as accumulators
template <int NT>
__device__ __forceinline__ void load_state(float (&c)[NT / 8][4], const void *src, int dtype, size_t base, int p0, int P, int N) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
#pragma unroll
  for (int j = 0; j < NT / 8; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = p0 + g + (i >> 1) * 8, n = 8 * j + 2 * q + (i & 1);
      c[j][i] = p < P && n < N ? load_as_f(src, dtype, base + (size_t)p * N + n) : 0.f;
    }
}
template <int NT>
__device__ __forceinline__ void write_state(void *dst, int dtype, size_t base, const float (&c)[NT / 8][4], int p0, int P, int N) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
#pragma unroll
  for (int j = 0; j < NT / 8; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = p0 + g + (i >> 1) * 8, n = 8 * j + 2 * q + (i & 1);
      if (p < P && n < N) store_as(dst, dtype, base + (size_t)p * N + n, c[j][i]);
    }
}

}  // namespace delta
}  // namespace slx
