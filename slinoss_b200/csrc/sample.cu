// Tokens from logits and given random numbers: temperature, top-k, top-p, min-p.
//
// Tokens are ranked by logit (ties: lower index first).  The first top_k stay; of these the shortest run that holds at least
// top_p of their mass; of these the ones with at least min_p of the largest mass.  The draw goes through what is left in the
// order of the indices and takes the first token at which the running mass exceeds u times the whole.
//
// A row is read once: a cluster of up to eight CTAs holds it in shared memory, and everything after that runs there.
//   * The border of a filter (k tokens, or a share of the mass) is narrowed down by a histogram over steps of the logit
//     (for masses of 1/16 in their logarithm), counted in 32-bit integers (masses relative to their bin's edge, 15 bits: all of
//     a CTA's tokens may fall into one): one bin holds the border.
//   * Where no more than a few thousand tokens lie above the bin's lower edge, CTA 0 gathers them and finishes the row, and
//     the other CTAs are done.  Otherwise only the bin's own tokens are gathered for the border (a bin with too many is
//     divided again by the integer keys of its logits, with exact sums of every part), and the draw sums the tokens that stay
//     where they are.
//   * Masses that decide anything are exponentials in 64 bits, held as integers of 2^-44 of the largest: their sums do not
//     depend on an order.  (A token 31 temperatures below the largest has none and is never drawn.)  The whole mass that top_p
//     refers to is a sum over every token, of which those below 2^-20 take exponentials in 32 bits, off by 2^-41 of the
//     largest each: an error of 10^-6 in it would move the border past a token in ten, every draw by that token's mass, and
//     one draw in a hundred into the neighbour, where ten thousand tokens stay.  Only the histogram is coarser; it names a bin,
//     and its neighbours are looked at too.
//   * What costs is instructions: two CTAs of an SM go through 32 to 64 logits a thread.  A filter touches few of them, so
//     warps first collect the values above a bound (a compare and a vote each) and then work on 32 at a time: the histogram
//     of 192 rows of 150001 bf16 logits takes 5 thousand clocks instead of 13, their gathering 5 instead of 11.
//     64 rows of 131072 fp32 logits with top_p 0.95 take 91 us (136 without), those 192 rows with all filters 86 (151).
#include <cooperative_groups.h>

#include <type_traits>
#include <utility>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace slx {

struct SampleArgs {
  const void *logits;
  int64_t stride;
  int V;
  const void *u;
  int u_bytes;
  const float *temperature, *top_p, *min_p;
  const void *top_k;
  int top_k_bytes;
  float temperature0, top_p0, min_p0;
  int64_t top_k0;
  int64_t *out;
};

typedef unsigned long long u64;
constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr int kBins = 512;      // of a histogram; one per thread
constexpr int kTail = 400;      // counting tokens: the bin of all masses below 2^-25 of the largest
constexpr int kMassTail = 320;  // adding masses: of all below 2^-20
constexpr int kList = 4096;     // tokens that are sorted and walked one by one
constexpr int kRuns = 1024;     // of indices, in the order of which tokens are drawn
constexpr int kQueue = 32 + 32 * 8;  // values of a warp that wait for their masses
constexpr int kMaxVecs = 17;     // of a thread: eight CTAs hold 262144 fp32 logits that begin inside a vector
constexpr int kMaxGroups = kMaxVecs * kSampleWarps;
constexpr int kMaxCluster = 8;
static_assert((u64)kMaxVecs * kSampleThreads * 8 << 15 < (u64)1 << 32, "a bin holds the 15-bit masses of all tokens of a CTA");
static_assert(kBins == kSampleThreads, "threads scan the bins one each");

struct alignas(16) SampleShared {  // (the row's vectors follow it)
  u64 list[kList];              // tokens: key and inverted index, so that descending order is the ranking
  u64 group[kMaxGroups];
  double table[64];             // kPowers
  double scan[kSampleWarps], scan2[kSampleWarps];
  u64 sums[kSampleWarps], sums2[kSampleWarps];
  unsigned hist[kBins];
  unsigned short waiting[kSampleWarps][64];
  // written by every CTA of the cluster into each, two sets in turn
  float gather_top[kMaxCluster], gather_bound[kMaxCluster];
  u64 gather_u[2][kMaxCluster], gather_v[2][kMaxCluster];
  double pick_before, pick_tokens;
  u64 start, border;
  int pick_bin, pick_upto, found;
  // of CTA 0
  int count;
  unsigned lowest, highest;
  float border_x;
  int border_i;
  unsigned maxima[kSampleWarps], bounds[kSampleWarps];
};
static_assert(kSampleWarps * kQueue * 4 <= kList * 8, "the queues lie in the list's place");

// Unsigned integers in the order of the values (zeros of both signs are one value).
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __float_as_uint(x == 0.f ? 0.f : x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// A 16-byte vector of logits.
template <typename TI>
struct Vec {
  static constexpr int n = 16 / sizeof(TI);
  uint4 raw;
  __device__ __forceinline__ float at(int e) const {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&raw);
    float x;
    if constexpr (sizeof(TI) == 4) x = __uint_as_float(w[e]);
    else if constexpr (std::is_same<TI, __half>::value)
      x = e & 1 ? __high2float(*reinterpret_cast<const __half2 *>(&w[e >> 1])) : __low2float(*reinterpret_cast<const __half2 *>(&w[e >> 1]));
    else x = __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
    return fmaxf(x, -INFINITY);  // (a NaN counts as -inf)
  }
  __device__ __forceinline__ float most() const {  // (NaN where all are)
    if constexpr (sizeof(TI) == 4) {
      return fmaxf(fmaxf(__uint_as_float(raw.x), __uint_as_float(raw.y)), fmaxf(__uint_as_float(raw.z), __uint_as_float(raw.w)));
    } else {
      using T2 = std::conditional_t<std::is_same<TI, __half>::value, __half2, __nv_bfloat162>;
      const T2 *w = reinterpret_cast<const T2 *>(&raw);
      const T2 m = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
      if constexpr (std::is_same<TI, __half>::value) return fmaxf(__low2float(m), __high2float(m));
      else return fmaxf(__bfloat162float(__low2bfloat16(m)), __bfloat162float(__high2bfloat16(m)));
    }
  }
};

// sum over the CTA
__device__ __forceinline__ u64 sum_over_cta(SampleShared &sm, u64 v) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  __syncthreads();
  if (lane == 0) sm.sums[warp] = v;
  __syncthreads();
  v = sm.sums[lane % kSampleWarps];
  for (int d = kSampleWarps / 2; d > 0; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  return v;
}
struct Pair {
  u64 x, y;
};
__device__ __forceinline__ Pair sum_over_cta(SampleShared &sm, Pair v) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int d = 16; d > 0; d >>= 1) {
    v.x += __shfl_xor_sync(~0u, v.x, d);
    v.y += __shfl_xor_sync(~0u, v.y, d);
  }
  __syncthreads();
  if (lane == 0) {
    sm.sums[warp] = v.x;
    sm.sums2[warp] = v.y;
  }
  __syncthreads();
  u64 s = (lane < kSampleWarps ? sm.sums : sm.sums2)[lane % kSampleWarps];  // one sum in each half of the warp
  for (int d = kSampleWarps / 2; d > 0; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
  return Pair{__shfl_sync(~0u, s, 0), __shfl_sync(~0u, s, 31)};
}
static_assert(kSampleWarps == 16, "the sums of the warps are taken by half a warp");
// sum of the CTA's threads before this one, and of all
__device__ __forceinline__ u64 scan_over_cta(SampleShared &sm, u64 v, u64 &whole) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  u64 run = v;
  for (int d = 1; d < 32; d <<= 1) {
    const u64 o = __shfl_up_sync(~0u, run, d);
    if (lane >= d) run += o;
  }
  __syncthreads();
  if (lane == 31) sm.sums[warp] = run;
  __syncthreads();
  u64 upto = sm.sums[lane % kSampleWarps];
  for (int d = 1; d < kSampleWarps; d <<= 1) {
    const u64 o = __shfl_up_sync(~0u, upto, d, kSampleWarps);
    if (lane % kSampleWarps >= d) upto += o;
  }
  whole = __shfl_sync(~0u, upto, kSampleWarps - 1);
  return (warp ? __shfl_sync(~0u, upto, warp - 1) : 0) + run - v;
}

// 2^(i/64), rounded
__device__ const double kPowers[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0,
};

// A token's mass: exp of a difference below zero by table (Tang 1989): 2^(i/64) and the series of e^r, |r| <= ln 2 / 128
// (r^6 / 720 < 2^-54); as an integer of 2^-44, zero from exp(-31) on.  Without branches: the chains of neighbours overlap.
struct Mass {
  const double *table;
  double per_unit;  // 1 / temperature
  float top;        // (where it is infinite, the largest share the mass)
  __device__ __forceinline__ u64 operator()(float v) const {
    const double y = fmax(((double)v - (double)top) * per_unit, -40.0);  // (also for NaN, from two infinities)
    constexpr double kLn2 = 0.693147180559945309417232121458;
    const double t = fma(y, 64.0 / kLn2, 6755399441055744.0);  // 1.5 * 2^52: the rounded integer in the low bits
    const int n = __double2loint(t);
    const double s = fma(t - 6755399441055744.0, -kLn2 / 64.0, y);
    const double e = fma(s, fma(s, fma(s, fma(s, fma(s, 1.0 / 120, 1.0 / 24), 1.0 / 6), 0.5), 1.0), 1.0);
    const double b = table[n & 63];
    const double f = e * __hiloint2double(__double2hiint(b) + ((n >> 6) << 20), __double2loint(b));
    const double q = fma(f, 17592186044416.0, 4503599627370496.0);  // 2^44 and 2^52
    const u64 m = ((u64)(unsigned)(__double2hiint(q) & 0xfffff) << 32) | (unsigned)__double2loint(q);
    return v == top ? 1ull << 44 : y > -31.0 ? m : 0;
  }
};

// The list's n entries in descending order: thread t gets the ranks per t .. per t + per - 1 (zeros behind the n).  Bitonic:
// steps within a thread, within a warp by shuffles, and across warps through the list's memory; as many as n needs.
template <int per>
__device__ __forceinline__ void sorted_list(SampleShared &sm, int n, u64 (&e)[per]) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int c = 0; c < per; ++c) e[c] = tid * per + c < n ? sm.list[tid * per + c] : 0;
  auto within = [&](int k, auto stride) {
    constexpr int J = decltype(stride)::value;
#pragma unroll
    for (int c = 0; c < per; ++c)
      if (!(c & J) && c + J < per) {
        const u64 x = e[c], y = e[c + J];
        const bool change = (x < y) == (((tid * per + c) & k) == 0);
        e[c] = change ? y : x;
        e[c + J] = change ? x : y;
      }
  };
#pragma unroll 1
  for (int k = 2; k < 2 * n; k <<= 1) {
    const bool down = (tid * per & k) == 0;
#pragma unroll 1
    for (int j = k >> 1; j >= 32 * per; j >>= 1) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < per; ++c) sm.list[c * kSampleThreads + tid] = e[c];
      __syncthreads();
      const int other = tid ^ (j / per);
#pragma unroll
      for (int c = 0; c < per; ++c) {
        const u64 o = sm.list[c * kSampleThreads + other];
        e[c] = (e[c] > o) == (down == (tid < other)) ? e[c] : o;
      }
    }
#pragma unroll 1
    for (int j = min(k >> 1, 16 * per); j >= per; j >>= 1) {
      const int mask = j / per;
      const bool larger = down == ((tid & mask) == 0);
#pragma unroll
      for (int c = 0; c < per; ++c) {
        const u64 o = __shfl_xor_sync(~0u, e[c], mask);
        e[c] = (e[c] > o) == larger ? e[c] : o;
      }
    }
    if (per > 4 && k > 4) within(k, std::integral_constant<int, 4>());
    if (per > 2 && k > 2) within(k, std::integral_constant<int, 2>());
    if (per > 1) within(k, std::integral_constant<int, 1>());
  }
  __syncthreads();  // (the list may be written again)
}

// Of the n entries of CTA 0's list, the one with which the weights (masses, or one each), from the largest entry down,
// reach `need`; the smallest where they do not.  In sm.border, which is read after a barrier.
// (per: entries of a thread that n needs at most)
template <int per>
__device__ __noinline__ void border_of(SampleShared &sm, Mass mass_of, int n, double need, bool masses) {
  u64 e[per], w[per], sum = 0, whole;
  sorted_list<per>(sm, n, e);
#pragma unroll
  for (int c = 0; c < per; ++c) {
    w[c] = !e[c] ? 0 : masses ? mass_of(value_of((unsigned)(e[c] >> 32))) : 1;
    sum += w[c];
  }
  u64 run = scan_over_cta(sm, sum, whole);
#pragma unroll
  for (int c = 0; c < per; ++c) {
    const int rank = threadIdx.x * per + c;
    if (rank < n && (rank == 0 || (double)run < need) && (rank == n - 1 || (double)(run + w[c]) >= need)) sm.border = e[c];
    run += w[c];
  }
}

// Steps below the largest logit (rounding is monotone); of 1/16 in the logarithm of the mass where masses are added up.
struct Steps {
  float top, per_logit;
  __device__ __forceinline__ float of(float v) const {
    return v == top ? 0.f : top == INFINITY ? INFINITY : (top - v) * per_logit;
  }
  // all values of fewer steps than `edge` are at least this (two roundings are 2^-23)
  __device__ __forceinline__ float floor(float edge) const {
    return fmaxf(__fsub_rd(top, edge * 1.0001f / per_logit), -INFINITY);
  }
};

// ---- CTA 0 by itself: n tokens in its list, all that may stay and some below them.
// The draw takes the first token with running > u z: of integers, running > its floor; below z, so that there is one.
__device__ __forceinline__ u64 target_in(double u, u64 z) { return min((u64)(u * (double)z), z - 1); }
struct Row {  // of one row, what its last steps need
  Steps step;
  int V;
  bool by_mass;
  int64_t k;
  float p;
  u64 least;
  double u;
  int64_t *out;
};
// n tokens are in CTA 0's list, all down to the bin `last`.  With masses top_p's border, at the mass `want`, is among them, in
// `bin` or near it; else `bin` is the last and holds top_k's, `above` tokens lying in the bins before.
template <int per>
__device__ __noinline__ void finish(SampleShared &sm, unsigned *runs, Mass mass_of, Row row, int n, int bin, int last,
                                    bool masses, double want, double above) {
  const int tid = threadIdx.x;
  u64 entry[per], m[per], z;
  int bins[per];
#pragma unroll
  for (int c = 0; c < per; ++c) {
    const int i = tid + c * kSampleThreads;
    entry[c] = m[c] = 0;
    bins[c] = -1;
    if (i < n) {
      entry[c] = sm.list[i];
      const float v = value_of((unsigned)(entry[c] >> 32));
      m[c] = mass_of(v);
      bins[c] = (int)row.step.of(v);
    }
  }
  // Of the entries of one bin, by themselves, what lies below the one that reaches `need` is dropped.
  auto cut = [&](int at_bin, double need, bool by) {
    u64 *const weight = sm.list + kList - kSampleThreads;
    __syncthreads();
    if (tid == 0) sm.count = 0;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < per; ++c)
      if (bins[c] == at_bin) sm.list[atomicAdd(&sm.count, 1)] = entry[c];
    __syncthreads();
    const int some = sm.count;
    if (some > kSampleThreads) border_of<kList / kSampleThreads>(sm, mass_of, some, need, by);
    else {  // each looks at the others
      int parts = 1;  // threads that share an entry's row of comparisons
      while (16 * parts < some && 2 * parts * some <= kSampleThreads) parts *= 2;
      const int at = tid / parts;
      const u64 mine = at < some ? sm.list[at] : 0;
      if (tid < some) weight[tid] = by ? mass_of(value_of((unsigned)(sm.list[tid] >> 32))) : 1;
      __syncthreads();
      u64 larger = 0;
      int below = 0;
      if (at < some)
#pragma unroll 4
        for (int o = tid % parts; o < some; o += parts) {
          const u64 other = sm.list[o];
          if (other > mine) larger += weight[o];
          below += other < mine;
        }
      for (int d = 1; d < parts; d <<= 1) {
        larger += __shfl_xor_sync(~0u, larger, d);
        below += __shfl_xor_sync(~0u, below, d);
      }
      if (at < some) {
        const bool reaches = (double)(larger + weight[at]) >= need;
        if (((double)larger < need || larger == 0) && (reaches || below == 0)) sm.border = mine;
      }
    }
    __syncthreads();
    const u64 border = sm.border;
#pragma unroll
    for (int c = 0; c < per; ++c)
      if (bins[c] == at_bin ? entry[c] < border : bins[c] > at_bin) {
        m[c] = 0;
        bins[c] = -1;
      }
  };
  auto around = [&](int at) {  // {mass of the bins before `at`, of this one}
    Pair s{0, 0};
#pragma unroll
    for (int c = 0; c < per; ++c) {
      s.x += bins[c] < at ? m[c] : 0;
      s.y += bins[c] == at ? m[c] : 0;
    }
    return sum_over_cta(sm, s);
  };
  if (!masses) {
    cut(bin, (double)row.k - above, false);
    if (row.by_mass) {  // top_p of what top_k has left: a histogram of rounded masses says where about
      unsigned *const rough = sm.hist;
      rough[tid] = 0;
      want = (double)row.p * (double)around(last + 1).x;
      if (tid == 0) sm.found = last;
#pragma unroll
      for (int c = 0; c < per; ++c)
        if (m[c]) atomicAdd(&rough[bins[c]], (unsigned)(m[c] >> 25));  // (4096 tokens of 2^19)
      __syncthreads();
      const u64 mine = rough[tid], before = scan_over_cta(sm, mine, z);
      if ((double)before < want * 0x1p-25 && want * 0x1p-25 <= (double)(before + mine)) sm.found = tid;
      __syncthreads();
      bin = min(sm.found, last);
    }
  }
  if (row.by_mass) {
    // the exact sums have the last word: bins below while they do not reach, above while they would do without this one
    Pair s = around(bin);
    while (bin < last && (double)(s.x + s.y) < want) s = around(++bin);
    while (bin > 0 && (double)s.x >= want) s = around(--bin);
    cut(bin, want - (double)s.x, true);
  }
  // (runs: the row's room, which is not needed any more)
#pragma unroll
  for (int i = 0; i < 2 * kRuns; i += kSampleThreads) runs[tid + i] = 0;
  if (tid == 0) sm.count = 0;
  __syncthreads();
  // The draw in the order of the indices: sums over 1024 runs of indices (at most 512 of one run, so that two halves of 22
  // bits fit 32 each), then the tokens of one run among themselves.
  int shift = 0;
  while ((row.V >> shift) >= kRuns) ++shift;
  unsigned *const upper = runs + kRuns;
  u64 *const masses_of_run = sm.list;
  int *const members = reinterpret_cast<int *>(sm.list + kList / 2);
#pragma unroll
  for (int c = 0; c < per; ++c) {
    if (m[c] < row.least) m[c] = 0;
    if (m[c]) {
      const int to = (int)~(unsigned)entry[c] >> shift;
      atomicAdd(&runs[to], (unsigned)m[c] & 0x3fffffu);
      atomicAdd(&upper[to], (unsigned)(m[c] >> 22));
    }
  }
  __syncthreads();
  const uint2 lo = reinterpret_cast<const uint2 *>(runs)[tid], hi = reinterpret_cast<const uint2 *>(upper)[tid];
  const u64 first = ((u64)hi.x << 22) + lo.x, second = ((u64)hi.y << 22) + lo.y;
  const u64 start = scan_over_cta(sm, first + second, z), target = target_in(row.u, z);
  if (start <= target && target < start + first + second) {
    const bool later = target >= start + first;
    sm.found = 2 * tid + later;
    sm.start = later ? start + first : start;
  }
  __syncthreads();
  const int hit = sm.found;
#pragma unroll
  for (int c = 0; c < per; ++c) {
    const int i = (int)~(unsigned)entry[c];
    if (m[c] && (i >> shift) == hit) {
      const int to = atomicAdd(&sm.count, 1);
      members[to] = i;
      masses_of_run[to] = m[c];
    }
  }
  __syncthreads();
  const int count = sm.count;
  if (tid < count) {
    u64 at = sm.start;
    const int i = members[tid];
    for (int o = 0; o < count; ++o)
      if (members[o] < i) at += masses_of_run[o];
    if (at <= target && target < at + masses_of_run[tid]) *row.out = i;
  }
}

template <typename TI>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(SampleArgs a, int NV) {  // NV vectors a thread
  constexpr int VEC = Vec<TI>::n;
  extern __shared__ __align__(16) char smem_[];
  SampleShared &sm = *reinterpret_cast<SampleShared *>(smem_);
  Vec<TI> *const row_data = reinterpret_cast<Vec<TI> *>(smem_ + sizeof(SampleShared)) + threadIdx.x;  // of this thread
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), C = (int)cluster.num_blocks();
  SampleShared &sm0 = *cluster.map_shared_rank(&sm, 0);
  auto started = cluster.barrier_arrive();  // (waited for before the first access to another CTA's memory)
  const int row = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const TI *x = static_cast<const TI *>(a.logits) + row * a.stride;
  const float temperature = a.temperature ? a.temperature[row] : a.temperature0;
  const float p = a.top_p ? a.top_p[row] : a.top_p0, minp = a.min_p ? a.min_p[row] : a.min_p0;
  int64_t k = a.top_k0;
  if (a.top_k) k = a.top_k_bytes == 8 ? static_cast<const int64_t *>(a.top_k)[row] : static_cast<const int *>(a.top_k)[row];
  if (k <= 0 || k > a.V) k = a.V;
  double u = a.u_bytes == 4 ? (double)static_cast<const float *>(a.u)[row] : static_cast<const double *>(a.u)[row];
  u = fmin(fmax(u, 0.0), 1.0);
  // index of a thread's value (j, e): vectors lie on 16-byte boundaries, the first of a row may begin before it
  const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(TI));
  auto first_of = [&](int j) { return ((rank * NV + j) * kSampleThreads + tid) * VEC - shift; };
  float top = -INFINITY;
  const double power = tid < 64 ? kPowers[tid] : 0.0;  // (on its way with the row)
#pragma unroll 4
  for (int j = 0; j < NV; ++j) {
    const int i = first_of(j);
    Vec<TI> v;
    if (i >= 0 && i + VEC <= a.V) v.raw = __ldcs(reinterpret_cast<const uint4 *>(x + i));
    else {
      TI w[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] = i + e >= 0 && i + e < a.V ? x[i + e] : from_f<TI>(-INFINITY);
      memcpy(&v.raw, w, 16);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) top = fmaxf(top, v.at(e));
    row_data[j * kSampleThreads] = v;
  }
  if (tid < 64) sm.table[tid] = power;
  sm.hist[tid] = 0;
  if (tid == 0) {
    sm.count = 0;
    sm.lowest = ~0u;
    sm.highest = 0;
  }
  int turn = 0;
  // the same value from every CTA to every CTA: read after the next cluster barrier
  auto spread_u = [&](u64 v) {
    if (tid < C) cluster.map_shared_rank(&sm, tid)->gather_u[turn][rank] = v;
  };
#define EACH_VECTOR(body_)                                              \
  _Pragma("unroll 1") for (int j = 0; j < NV; ++j) {                    \
    const int i0 = first_of(j);                                         \
    const Vec<TI> vec = row_data[j * kSampleThreads];                   \
    body_                                                               \
  }
#define EACH(body_)                                                     \
  EACH_VECTOR({                                                         \
    _Pragma("unroll") for (int e = 0; e < VEC; ++e) {                   \
      const float v = vec.at(e);                                        \
      const int i = i0 + e;                                             \
      body_                                                             \
    }                                                                   \
  })

  // ---- the largest logit, and (where k is small) a value that k tokens reach: of each warp's threads the largest logits are
  // the first k / warps at least this
  float bound = -INFINITY;
  {
    const unsigned key = key_of(top), m = __reduce_max_sync(~0u, key);
    const int64_t of_warp = (k + C * kSampleWarps - 1) / (C * kSampleWarps);
    unsigned least_of = k < a.V && of_warp == 1 ? m : 0;
    if (k < a.V && of_warp > 1 && of_warp <= 32) {
      int rank_of = 0;
#pragma unroll 8
      for (int l = 0; l < 32; ++l) {
        const unsigned o = __shfl_sync(~0u, key, l);
        rank_of += o > key || (o == key && l < lane);
      }
      least_of = __shfl_sync(~0u, key, __ffs(__ballot_sync(~0u, rank_of == (int)of_warp - 1)) - 1);
    }
    if (lane == 0) {
      sm.maxima[warp] = m;
      sm.bounds[warp] = least_of;
    }
    __syncthreads();
    top = value_of(__reduce_max_sync(~0u, sm.maxima[lane & (kSampleWarps - 1)]));
    least_of = __reduce_min_sync(~0u, sm.bounds[lane & (kSampleWarps - 1)]);
    if (least_of) bound = value_of(least_of);
    cluster.barrier_wait(std::move(started));
    if (C > 1) {
      if (tid < C) {
        SampleShared &to = *cluster.map_shared_rank(&sm, tid);
        to.gather_top[rank] = top;
        to.gather_bound[rank] = bound;
      }
      cluster.sync();
      for (int c = 0; c < C; ++c) {
        top = fmaxf(top, sm.gather_top[c]);
        bound = fminf(bound, sm.gather_bound[c]);
      }
    }
  }
  // (no CTA leaves while another may still write to it)
  auto leave = [&]() {
    if (C > 1) cluster.sync();
  };
  if (top == -INFINITY) {  // nothing can be drawn
    if (rank == 0 && tid == 0) a.out[row] = -1;
    leave();
    return;
  }

  // body(vec, i0, valid), by whole warps, for the vectors with a value of at least `floor` (few of them, mostly: a warp
  // collects their places and takes 32 at a time)
  auto each_above = [&](float floor, auto body) {
    unsigned short *const queue = sm.waiting[warp];
    int waiting = 0;
    auto take = [&](int n) {
      waiting -= n;
      const bool valid = lane < n;
      const int at = valid ? queue[waiting + lane] : lane, other = at % 32 - lane;
      body(row_data[at / 32 * kSampleThreads + other], first_of(at / 32) + other * VEC, valid);
    };
#pragma unroll 1
    for (int j = 0; j < NV; ++j) {
      const bool in = row_data[j * kSampleThreads].most() >= floor;
      const unsigned mask = __ballot_sync(~0u, in);
      if (in) queue[waiting + __popc(mask & ((1u << lane) - 1))] = (unsigned short)(32 * j + lane);
      waiting += __popc(mask);
      if (waiting >= 32) {
        __syncwarp();
        take(32);
        __syncwarp();
      }
    }
    __syncwarp();
    if (waiting) take(waiting);
  };

  // body(v, i, j, valid), by whole warps, for the values of at least `floor`, of which j is the thread's vector
  auto each_value = [&](float floor, auto body) {
    unsigned short *const queue = sm.waiting[warp];
    int waiting = 0;
    auto take = [&](int n) {
      waiting -= n;
      const bool valid = lane < n;
      const int at = valid ? queue[waiting + lane] : lane, other = at % 32 - lane, e = at / 32 % VEC, j = at / 32 / VEC;
      body(to_f(reinterpret_cast<const TI *>(&row_data[j * kSampleThreads + other])[e]), first_of(j) + other * VEC + e, j, valid);
    };
    EACH_VECTOR({
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const bool in = vec.at(e) >= floor;
        const unsigned mask = __ballot_sync(~0u, in);
        if (in) queue[waiting + __popc(mask & ((1u << lane) - 1))] = (unsigned short)((j * VEC + e) * 32 + lane);
        waiting += __popc(mask);
        if (waiting >= 32) {
          __syncwarp();
          take(32);
          __syncwarp();
        }
      }
    })
    __syncwarp();
    if (waiting) take(waiting);
  };

  auto cta_sum = [&](u64 v) { return sum_over_cta(sm, v); };
  auto cta_scan = [&](u64 v, u64 &whole) { return scan_over_cta(sm, v, whole); };

  // Sums over a warp's vectors j in the order of the indices: sm.group[j * warps + warp].
  auto fill_groups = [&](auto weights) {  // weights(vec, i0, w): of a vector's values
    EACH_VECTOR({
      u64 w[VEC];
      weights(vec, i0, w);
      u64 s = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += w[e];
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
      if (lane == 0) sm.group[j * kSampleWarps + warp] = s;
    })
  };
  // The first index at which the running sum of the weights (whose groups are filled) exceeds target(whole).
  auto locate = [&](auto target_of, auto weights, auto found) {
    __syncthreads();
    const u64 mine = tid < NV * kSampleWarps ? sm.group[tid] : 0;
    u64 total;
    u64 start = cta_scan(mine, total);
    u64 whole = total;
    if (C > 1) {
      spread_u(total);
      cluster.sync();
      whole = 0;
      for (int c = 0; c < C; ++c) {
        const u64 t = sm.gather_u[turn][c];
        if (c < rank) start += t;
        whole += t;
      }
      turn ^= 1;
    }
    const u64 target = target_of(whole);
    if (tid == 0) sm.found = -1;
    __syncthreads();
    if (start <= target && target < start + mine) {
      sm.found = tid;
      sm.start = start;
    }
    __syncthreads();
    const int g = sm.found;
    if (g < 0 || g % kSampleWarps != warp) return;
    const int j = g / kSampleWarps, i0 = first_of(j);
    u64 w[VEC], sum = 0;
    weights(row_data[j * kSampleThreads], i0, w);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum += w[e];
    u64 run = sum;
    for (int d = 1; d < 32; d <<= 1) {
      const u64 o = __shfl_up_sync(~0u, run, d);
      if (lane >= d) run += o;
    }
    u64 at = sm.start + run - sum;
    if (at <= target && target < at + sum) {
      int here = VEC - 1;
#pragma unroll
      for (int e = VEC - 2; e >= 0; --e) {  // (from behind: the first that exceeds stays)
        sum -= w[e + 1];
        if (target < at + sum) here = e;
      }
      found(i0 + here);
    }
  };

  if (!(temperature > 0.f) || k == 1 || !(p > 0.f) || !(minp <= 1.f)) {  // the first largest logit
    auto is_top = [&](const Vec<TI> &vec, int, u64 *w) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] = vec.at(e) == top;
    };
    fill_groups(is_top);
    locate([](u64) { return (u64)0; }, is_top, [&](int i) { a.out[row] = i; });
    leave();
    return;
  }
  const double per_unit = 1.0 / (double)temperature;
  const Mass mass_of{sm.table, per_unit, top};
  const double one = 17592186044416.0;
  const u64 least = minp > 0.f ? (u64)ceil((double)minp * one) : 0;  // of a mass that min_p keeps

  // ---- no border to find: the draw over everything, or over what min_p keeps
  // What stays: logits above border_x, and those at it up to index border_i.
  float border_x = -INFINITY;
  int border_i = 0x7fffffff;
  auto stays = [&](float v, int i) { return v > border_x || (v == border_x && i <= border_i && v > -INFINITY); };
  auto kept = [&](const Vec<TI> &vec, int i0, u64 *w) {
    bool any = false;
#pragma unroll
    for (int e = 0; e < VEC; ++e) any |= stays(vec.at(e), i0 + e);
#pragma unroll
    for (int e = 0; e < VEC; ++e) w[e] = 0;
    if (__any_sync(~0u, any)) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const u64 m = mass_of(vec.at(e));
        w[e] = stays(vec.at(e), i0 + e) && m >= least ? m : 0;
      }
    }
  };
  const bool by_rank = k < a.V, by_mass = p < 1.f;

  const Steps step{top, (float)(16.0 * 1.4426950408889634 * per_unit)};

  if (by_rank || by_mass) {
    auto part = [&](float t) {  // 2^(-t/16)
      float r;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t * (-1.f / 16)));
      return r;
    };
    auto weight15 = [&](float t) { return (unsigned)__float2int_rn(part(t) * 32768.f); };
    bool done = false;
    // ---- a border: the first token, from the top, with which the weights of the tokens that stay reach the target.
    // masses: weights are masses and the target p of their whole; else numbers of tokens and the target k.
    // Leaves the border, and with masses the sums of what stays in the groups (those with at least min_p of the largest).
    auto narrow = [&](auto kind) {
      constexpr bool masses = decltype(kind)::value;
      const int last = masses ? kMassTail : kTail;  // the bin of all that lies below the others
      // (numbers of tokens: any steps will do, and all that counts lies above the bound)
      const Steps scale = masses || bound == -INFINITY ? step : Steps{top, (float)(kTail - 1) / (top - bound)};
      auto step_of = [&](float v) { return scale.of(v); };
      auto bin_of = [&](float t) { return t < (float)last ? (int)t : last; };
      u64 mass = 0, beyond = 0;  // of all tokens, of those in the last bin
      unsigned tail = 0;
      if (masses) {
        // The many tokens below 2^-20 need no more than an exponential in 32 bits: off by 2^-21 of themselves, in no common
        // direction (the factor is held in two parts), which is 2^-41 of the largest mass each.  As integers of 2^-43 they
        // fit the mantissa of 2^23.  The others queue up, so that whole warps take the 64-bit exponentials.
        const double c = 1.4426950408889634 * per_unit;
        const float c0 = (float)c, c1 = (float)(c - (double)c0), least_heavy = fmaxf(scale.floor((float)last), -3.402823466e38f);
        float *const queue = reinterpret_cast<float *>(sm.list) + warp * kQueue;
        unsigned light = 0;
        auto weigh = [&](float v) {
          const float t = step_of(v);
          const int b = bin_of(t);
          const u64 m = mass_of(v);
          if (b < last) atomicAdd(&sm.hist[b], weight15(t - (float)b));
          else beyond += m;
          mass += m;
        };
        auto add_up = [&](auto all) {  // (all: no border lies before this one)
          int waiting = 0;
          EACH_VECTOR({
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const float v = vec.at(e);
              const bool in = decltype(all)::value || stays(v, i0 + e);
              const bool heavy = in && v >= least_heavy;
              const unsigned mask = __ballot_sync(~0u, heavy);
              if (heavy) queue[waiting + __popc(mask & ((1u << lane) - 1))] = v;
              waiting += __popc(mask);
              float r;
              asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaxf(fmaf(v - top, c1, fmaf(v - top, c0, 43.f)), -200.f)));
              if (in && !heavy) light += __float_as_uint(r + 8388608.f) - __float_as_uint(8388608.f);
            }
            if (waiting >= 32) {
              __syncwarp();
              do {
                waiting -= 32;
                weigh(queue[waiting + lane]);
              } while (waiting >= 32);
              __syncwarp();
            }
          })
          __syncwarp();
          if (lane < waiting) weigh(queue[lane]);
        };
        if (border_x == -INFINITY) add_up(std::true_type());
        else add_up(std::false_type());
        beyond += 2 * (u64)light;
        mass += 2 * (u64)light;
      } else {
        each_above(bound, [&](const Vec<TI> &vec, int, bool valid) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float v = vec.at(e);
            if (valid && v >= bound && v > -INFINITY) {
              const int b = bin_of(step_of(v));
              if (b < kTail) atomicAdd(&sm.hist[b], 1u);
              else ++tail;
            }
          }
        });
      }
      if (masses) {
        const Pair s = sum_over_cta(sm, Pair{mass, beyond});
        spread_u(s.x);
        if (tid < C) cluster.map_shared_rank(&sm, tid)->gather_v[turn][rank] = s.y;
      }
      else if ((tail = __reduce_add_sync(~0u, tail)) && lane == 0) atomicAdd(&sm.hist[kTail], tail);
      // Picks the bin: every CTA the same from everybody's histograms.  unit: of a bin's weights; above: what lies before the
      // first, then before the bin; upto: the bin by which the target is met whatever the histogram's rounding (2^-15 of a
      // weight); tokens: about how many lie above its lower edge; listed: the tokens of all bins but the last meet the target.
      double target = (double)k, above = 0.0, tokens = 0.0;
      int upto = 0;
      bool listed = false;
      auto pick = [&](double unit) {
        if (C > 1) cluster.sync();
        else __syncthreads();
        unsigned n[kMaxCluster];
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c) n[c] = c < C ? cluster.map_shared_rank(&sm, c)->hist[tid] : 0;
        double w = 0.0;
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c) w += (double)n[c];
        double few = masses ? w * (1.0 / 32768) : w;
        w *= unit;
        double run = w;
        for (int d = 1; d < 32; d <<= 1) {
          const double o = __shfl_up_sync(~0u, run, d), f = __shfl_up_sync(~0u, few, d);
          if (lane >= d) {
            run += o;
            few += f;
          }
        }
        __syncthreads();
        if (lane == 31) {
          sm.scan[warp] = run;
          sm.scan2[warp] = few;
        }
        if (tid == 0) sm.pick_bin = sm.pick_upto = kBins;
        __syncthreads();
        double passed = (lane < kSampleWarps ? sm.scan : sm.scan2)[lane % kSampleWarps];  // each in half of the warp
        for (int d = 1; d < kSampleWarps; d <<= 1) {
          const double o = __shfl_up_sync(~0u, passed, d, kSampleWarps);
          if (lane % kSampleWarps >= d) passed += o;
        }
        const double run_before = __shfl_sync(~0u, passed, max(warp - 1, 0)), few_before = __shfl_sync(~0u, passed, 16 + max(warp - 1, 0));
        const double start = above + (warp ? run_before : 0.0), all = above + __shfl_sync(~0u, passed, kSampleWarps - 1);
        few += warp ? few_before : 0.0;
        if (masses) {
          u64 whole = 0, left = 0;
          for (int c = 0; c < C; ++c) {
            whole += sm.gather_u[turn][c];
            left += sm.gather_v[turn][c];
          }
          target = (double)p * (double)whole * (1.0 / one);
          listed = (double)(whole - left) >= target * one;
        }
        const bool reached = start + run >= target;
        const unsigned votes = __ballot_sync(~0u, reached);
        if (reached && lane == __ffs(votes) - 1) atomicMin(&sm.pick_bin, tid);
        const bool surely = start + run >= (masses ? target * (1.0 + 1.0 / 8192) : target);
        const unsigned sure_votes = __ballot_sync(~0u, surely);
        if (surely && lane == __ffs(sure_votes) - 1) atomicMin(&sm.pick_upto, tid);
        __syncthreads();
        const int b = sm.pick_bin;
        if (b == tid || (b == kBins && tid == kBins - 1)) sm.pick_before = b == tid ? start + run - w : all;
        upto = sm.pick_upto;
        if (tid == min(upto, kBins - 1)) sm.pick_tokens = few;
        __syncthreads();
        above = sm.pick_before;
        tokens = sm.pick_tokens;
        return b;
      };
      // (bins' edges are powers of 2^(1/16), from the table of 2^(i/64): 2^(-b/16) = 2^(-b>>4) 2^((-b&15)/16))
      const int e16 = -tid;
      const double edge0 = masses ? sm.table[(e16 & 15) * 4] * __hiloint2double((1023 + (e16 >> 4)) << 20, 0) * (1.0 / 32768) : 1.0;
      int bin = pick(edge0);
      if (masses) turn ^= 1;
      if (!masses && bin == kBins) {  // fewer than k tokens above -inf: all of them stay
        if (C > 1) cluster.sync();
        else __syncthreads();
        sm.hist[tid] = 0;  // (everybody has read the histograms)
        __syncthreads();
        return;
      }
      if (bin > last) bin = last;
      // the tokens of CTA 0's list: those that stay and are `in`
      // (each CTA lists its own; the others' lists then join CTA 0's)
      auto gather = [&](float floor, auto in) {  // (floor: no value below it is in)
        each_above(floor, [&](const Vec<TI> &vec, int i0, bool valid) {
          unsigned hits = 0;
#pragma unroll
          for (int e = 0; e < VEC; ++e) hits |= (unsigned)(valid && stays(vec.at(e), i0 + e) && in(vec.at(e))) << e;
          int run = __popc(hits);
          for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(~0u, run, d);
            if (lane >= d) run += o;
          }
          int at = 0;
          if (lane == 31 && run) at = atomicAdd(&sm.count, run);
          at = __shfl_sync(~0u, at, 31) + run - __popc(hits);
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (hits >> e & 1) {
              if (at < kList) sm.list[at] = ((u64)key_of(vec.at(e)) << 32) | (unsigned)~(i0 + e);
              ++at;
            }
        });
        if (rank != 0) {
          __syncthreads();
          const int n = sm.count;
          if (n > 0) {
            if (tid == 0) sm.found = atomicAdd(&sm0.count, n);
            __syncthreads();
            const int base = sm.found;
            for (int i = tid; i < min(n, kList - base); i += kSampleThreads) sm0.list[base + i] = sm.list[i];
            __syncthreads();
            if (tid == 0) sm.count = 0;
          }
        }
      };
      // the lowest and the highest key of what is `in`, to CTA 0
      auto extremes = [&](auto in) {
        unsigned lo = ~0u, hi = 0;
        EACH({
          if (stays(v, i) && in(v)) {
            lo = min(lo, key_of(v));
            hi = max(hi, key_of(v));
          }
        })
        lo = __reduce_min_sync(~0u, lo);
        hi = __reduce_max_sync(~0u, hi);
        if (lane == 0 && hi) {
          atomicMin(&sm0.lowest, lo);
          atomicMax(&sm0.highest, hi);
        }
      };
      if ((upto < last || listed) && tokens * 1.05 < (double)kList) {  // (masses tell their tokens' number to within 2^(1/16))
        upto = min(upto, last - 1);
        const float edge = (float)(upto + 1);
        gather(scale.floor(edge), [&](float v) { return step_of(v) < edge; });
        done = true;
        if (C > 1) cluster.sync();
        else __syncthreads();
        if (rank == 0) {
          const Row rest{scale, a.V, by_mass, k, p, least, u, a.out + row};
          unsigned *const room = reinterpret_cast<unsigned *>(row_data - tid);
          const int n = min(sm.count, kList);
          if (n <= kSampleThreads) finish<1>(sm, room, mass_of, rest, n, min(bin, upto), upto, masses, target * one, above);
          else if (n <= 3 * kSampleThreads) finish<3>(sm, room, mass_of, rest, n, min(bin, upto), upto, masses, target * one, above);
          else finish<kList / kSampleThreads>(sm, room, mass_of, rest, n, min(bin, upto), upto, masses, target * one, above);
        }
        return;
      }
      // with masses: what lies above the bin, exactly.  The exact sums have the last word on the bin.
      u64 sure = 0;
      while (masses) {
        Pair mine{0, 0};
        each_value(bin < last ? scale.floor((float)(bin + 1)) : -INFINITY, [&](float v, int i, int, bool valid) {
          const int b = bin_of(step_of(v));
          const u64 m = valid && stays(v, i) ? mass_of(v) : 0;
          mine.x += b < bin ? m : 0;
          mine.y += b == bin ? m : 0;
        });
        Pair s = sum_over_cta(sm, mine);
        if (C > 1) {
          spread_u(s.x);
          if (tid < C) cluster.map_shared_rank(&sm, tid)->gather_v[turn][rank] = s.y;
          cluster.sync();
          s = Pair{0, 0};
          for (int c = 0; c < C; ++c) {
            s.x += sm.gather_u[turn][c];
            s.y += sm.gather_v[turn][c];
          }
          turn ^= 1;
        }
        sure = s.x;
        if (bin > 0 && (double)s.x >= target * one) --bin;
        else if (bin < last && (double)(s.x + s.y) < target * one) ++bin;
        else break;
      }
      // Gathers the bin's tokens; divides it while they are too many: by the keys of its logits, with sums that are exact in
      // every part.  (Rounded weights would be off alike for all tokens of one value, by as much as the whole of another.)
      const double goal = masses ? target * one : target;
      if (!masses) sure = (u64)above;
      unsigned low = 0, high = ~0u;  // keys
      auto inside = [&](float v) {
        const unsigned key = key_of(v);
        return key >= low && key <= high && bin_of(step_of(v)) == bin;
      };
      u64 *const parts = sm.list;  // of every CTA, between two gatherings
      int n;
      for (;;) {
        gather(bin < last ? scale.floor((float)(bin + 1)) : -INFINITY, inside);
        if (C > 1) cluster.sync();
        else __syncthreads();
        sm.hist[tid] = 0;  // (everybody has read the histograms)
        n = sm0.count;
        if (n > kList) {
          extremes(inside);
          if (C > 1) cluster.sync();
          else __syncthreads();
          low = sm0.lowest;
          high = sm0.highest;
        }
        if (C > 1) cluster.sync();
        else __syncthreads();
        if (rank == 0 && tid == 0) {
          sm.count = 0;
          sm.lowest = ~0u;
          sm.highest = 0;
        }
        if (n <= kList || low == high) break;
        const int cut = max(0, 32 - __clz(high - low) - 9);  // (at most kBins parts, the highest keys first)
        parts[tid] = 0;
        __syncthreads();
        each_value(value_of(low), [&](float v, int i, int, bool valid) {
          if (valid && stays(v, i) && inside(v)) atomicAdd(&parts[(high - key_of(v)) >> cut], masses ? mass_of(v) : (u64)1);
        });
        if (C > 1) cluster.sync();
        else __syncthreads();
        u64 w = 0, whole;
#pragma unroll 1
        for (int c = 0; c < C; ++c) w += cluster.map_shared_rank(&sm, c)->list[tid];
        const u64 before = sure + cta_scan(w, whole);
        // the first part that reaches the goal (the last one, should the sums' roundings keep the goal above them all)
        if (tid == 0) sm.pick_bin = (int)((high - low) >> cut);
        __syncthreads();
        if ((double)(before + w) >= goal) atomicMin(&sm.pick_bin, tid);
        __syncthreads();
        const int b = sm.pick_bin;
        if (tid == b) sm.start = before;
        if (C > 1) cluster.sync();  // (and nobody reads the parts any more)
        else __syncthreads();
        sure = sm.start;
        const unsigned from = high - ((unsigned)b << cut);
        low = max(low, cut ? from - ((1u << cut) - 1) : from);
        high = from;
      }
      if (n == 0) return;  // (a tail without tokens)
      if (n <= kList) {
        if (rank == 0) {
          const double need = goal - (double)sure;
          if (n <= kSampleThreads) border_of<1>(sm, mass_of, n, need, masses);
          else border_of<kList / kSampleThreads>(sm, mass_of, n, need, masses);
          __syncthreads();
          if (tid == 0) {
            sm.border_x = value_of((unsigned)(sm.border >> 32));
            sm.border_i = (int)~(unsigned)sm.border;
          }
        }
        if (C > 1) cluster.sync();
        else __syncthreads();
        border_x = sm0.border_x;
        border_i = sm0.border_i;
      } else {  // many tokens of one value: their number decides, and the index of the last
        const float value = value_of(high);
        const u64 m = mass_of(value);
        const double want = masses ? (m ? ceil((goal - (double)sure) / (double)m) : (double)n) : goal - (double)sure;
        const u64 ties = (u64)fmin(fmax(want, 1.0), (double)n);
        auto is_tie = [&](const Vec<TI> &vec, int i0, u64 *w) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) w[e] = vec.at(e) == value && stays(vec.at(e), i0 + e);
        };
        __syncthreads();
        fill_groups(is_tie);
        locate([&](u64) { return ties - 1; }, is_tie, [&](int i) { sm0.border_i = i; });
        if (C > 1) cluster.sync();
        else __syncthreads();
        border_i = sm0.border_i;
        border_x = value;
      }
      if (C > 1) cluster.sync();
      else __syncthreads();
    };
    if (by_rank) narrow(std::false_type());
    if (done) return;  // (nobody reads or writes another CTA's memory after the last barrier)
    if (by_mass) narrow(std::true_type());
    if (done) return;
    __syncthreads();
    if (tid < NV * kSampleWarps) sm.group[tid] = 0;
    __syncthreads();
    each_value(fmaxf(border_x, -3.402823466e38f), [&](float v, int i, int j, bool valid) {
      u64 m = valid && stays(v, i) ? mass_of(v) : 0;
      if (m < least) m = 0;
      unsigned left = __ballot_sync(~0u, m != 0);
      while (left) {  // (a warp's values come in the order of its vectors: two or three of them)
        const int lead = __ffs(left) - 1, one_of = __shfl_sync(~0u, j, lead);
        const bool same = m != 0 && j == one_of;
        const unsigned mask = __ballot_sync(~0u, same);
        const unsigned lo = __reduce_add_sync(~0u, same ? (unsigned)m & 0x3fffffu : 0);
        const unsigned hi = __reduce_add_sync(~0u, same ? (unsigned)(m >> 22) : 0);
        if (lane == lead) sm.group[one_of * kSampleWarps + warp] += ((u64)hi << 22) + lo;
        __syncwarp();
        left &= ~mask;
      }
    });
  } else {
    fill_groups(kept);
  }
  // ---- the draw
  locate([&](u64 z) { return target_in(u, z); }, kept, [&](int i) { a.out[row] = i; });
  leave();
#undef EACH
#undef EACH_VECTOR
}

// A row's cluster: few vectors a thread while two CTAs an SM have not been filled, then more, up to eight, so that rows take
// fewer CTAs; more than eight only where a row needs them.  Measured with top_p 0.95, us: 192 rows of 150001 bf16 logits 330 with
// up to two or four vectors, 270 with eight, 468 with 17 (too few CTAs an SM); 64 rows of 131072 fp32 111 with up to eight, 124 with
// 17.  (256 rows of 65536 bf16 are the other way round, 219 and 187: at eight the third CTA of a row holds its last vector alone.)
// Filling one CTA an SM or four in the place of two: 148 rows of 20000 fp32 logits 46 and 56 against 37, the others alike.
template <typename TI>
static int launch_sample(const SampleArgs &a, int rows, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(TI);
  const int vecs = (a.V + VEC - 1) / VEC + 1;  // (a row that begins inside a vector may reach into one more)
  auto ctas_for = [&](int nv) { return (vecs + kSampleThreads * nv - 1) / (kSampleThreads * nv); };
  int nv = 1;
  while (nv < kMaxVecs && (ctas_for(nv) > kMaxCluster ||
                           (nv < 8 && ctas_for(nv) > 1 && (int64_t)rows * ctas_for(nv) > 2 * kB200Sms)))
    ++nv;
  const int ctas = ctas_for(nv);
  SLX_REQUIRE(ctas <= kMaxCluster, SLX_E_UNSUPPORTED, "sample: vocab too large");
  auto kernel = sample_kernel<TI>;
  const size_t bytes = sizeof(SampleShared) + (size_t)nv * kSampleThreads * 16;
  if (const int rc = ensure_dyn_smem(kernel, bytes)) return rc;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(ctas, rows);
  c.blockDim = dim3(kSampleThreads);
  c.dynamicSmemBytes = bytes;
  c.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&c, kernel, a, nv);
  if (e != cudaSuccess) return fail((int)e, "sample_kernel: %s", cudaGetErrorString(e));
  return check_launch("sample_kernel");
}

}  // namespace slx

using namespace slx;

extern "C" int slx_sample(const slx_sample_shape *s, const void *logits, const void *u, const float *temperature,
                          const void *top_k, const float *top_p, const float *min_p, int64_t *out, void *stream) {
  SLX_REQUIRE(s, SLX_E_NULL, "sample: shape is NULL");
  SLX_REQUIRE(logits && u && out, SLX_E_NULL, "sample: a required pointer is NULL");
  SLX_REQUIRE(s->rows > 0 && s->vocab > 0, SLX_E_SHAPE, "sample: sizes must be positive (rows %d, vocab %d)", s->rows, s->vocab);
  SLX_REQUIRE(s->vocab <= 262144, SLX_E_UNSUPPORTED, "sample: vocab must be at most 262144, got %d", s->vocab);
  SLX_REQUIRE(s->rows <= 65535, SLX_E_UNSUPPORTED, "sample: rows must be at most 65535, got %d", s->rows);
  SLX_REQUIRE(s->dtype == SLX_F32 || s->dtype == SLX_BF16 || s->dtype == SLX_F16, SLX_E_DTYPE, "sample: unknown dtype %d", s->dtype);
  SLX_REQUIRE(!top_k || s->top_k_bytes == 4 || s->top_k_bytes == 8, SLX_E_DTYPE, "sample: top_k entries must have 4 or 8 bytes");
  SLX_REQUIRE(s->u_bytes == 4 || s->u_bytes == 8, SLX_E_DTYPE, "sample: u must be float or double");
  SampleArgs a;
  a.logits = logits;
  a.stride = s->row_stride;
  a.V = s->vocab;
  a.u = u;
  a.u_bytes = s->u_bytes;
  a.temperature = temperature;
  a.top_p = top_p;
  a.min_p = min_p;
  a.top_k = top_k;
  a.top_k_bytes = s->top_k_bytes;
  a.temperature0 = s->temperature;
  a.top_p0 = s->top_p;
  a.min_p0 = s->min_p;
  a.top_k0 = s->top_k;
  a.out = out;
  cudaStream_t st = as_stream(stream);
  if (s->dtype == SLX_BF16) return launch_sample<__nv_bfloat16>(a, s->rows, st);
  if (s->dtype == SLX_F16) return launch_sample<__half>(a, s->rows, st);
  return launch_sample<float>(a, s->rows, st);
}
