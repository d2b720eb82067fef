// Tokens from logits and given random numbers: temperature, top-k, top-p, min-p.
//
// Tokens are ranked by logit (ties: lower index first).  The first top_k stay; of these the shortest run that holds at least
// top_p of their mass; of these the ones with at least min_p of the largest mass.  The draw goes through what is left in the
// order of the indices and takes the first token at which the running mass exceeds u times the whole.
//
// A row is read once: a cluster of up to eight CTAs holds it in shared memory, and everything after that runs
// there.  What a pass costs is arithmetic, so the passes are kept cheap:
//   * The border of a filter (k tokens, or a share of the mass) is narrowed down by a histogram over steps of 1/16 in the
//     logarithm of the mass, counted in 32-bit integers (masses relative to their bin's edge, 15 bits: a CTA's
//     2^17 tokens may all fall into one): one bin holds the
//     border.  Its tokens, a few dozen to a few hundred, are gathered, sorted and walked one by one.  A bin with too many
//     is divided again by the integer keys of its logits until it is small enough or holds a single value.
//   * Masses that decide between tokens are exponentials in 64 bits, taken only for tokens that stay, as integers of 2^-44 of
//     the largest: their sums do not depend on an order, and a draw is decided as exact sums would decide it but for about
//     one in 10^7 (the whole mass that top_p refers to is summed in 32-bit exponentials).
#include <cooperative_groups.h>

#include <type_traits>

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
constexpr int kTail = 400;      // the bin of all masses below 2^-25 of the largest
constexpr int kList = 2048;     // tokens that are sorted one by one
constexpr int kMaxVecs = 17;     // of a thread: eight CTAs hold 262144 fp32 logits that begin inside a vector
constexpr int kMaxGroups = kMaxVecs * kSampleWarps;
constexpr int kMaxCluster = 8;
static_assert(kBins == kSampleThreads, "threads scan the bins one each");

struct alignas(16) SampleShared {  // (the row's vectors follow it)
  u64 list[kList];
  u64 group[kMaxGroups];
  double table[64];             // 2^(i/64)
  double scan[kSampleWarps];
  u64 sums[kSampleWarps];
  unsigned hist[kBins];
  // written by every CTA of the cluster into each, two sets in turn
  float gather_f[2][kMaxCluster];
  u64 gather_u[2][kMaxCluster];
  double pick_before;
  int pick_bin;
  // of CTA 0
  int count;
  unsigned lowest, highest;
  float border_x;
  int border_i;
  u64 border_mass;
  // of every CTA
  unsigned maxima[kSampleWarps];
};

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
};

template <typename TI>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(SampleArgs a, int NV) {  // NV vectors a thread
  constexpr int VEC = Vec<TI>::n;
  extern __shared__ __align__(16) char smem_[];
  SampleShared &sm = *reinterpret_cast<SampleShared *>(smem_);
  Vec<TI> *const row_data = reinterpret_cast<Vec<TI> *>(smem_ + sizeof(SampleShared)) + threadIdx.x;  // of this thread
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), C = (int)cluster.num_blocks();
  SampleShared &sm0 = *cluster.map_shared_rank(&sm, 0);
  const int row = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const TI *x = static_cast<const TI *>(a.logits) + row * a.stride;
  // index of a thread's value (j, e): vectors lie on 16-byte boundaries, the first of a row may begin before it
  const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(TI));
  auto first_of = [&](int j) { return ((rank * NV + j) * kSampleThreads + tid) * VEC - shift; };
  float top = -INFINITY;
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
  if (tid < 64) sm.table[tid] = exp2((double)tid / 64.0);
  sm.hist[tid] = 0;
  if (tid == 0) {
    sm.count = 0;
    sm.lowest = ~0u;
    sm.highest = 0;
  }
  int turn = 0;
  // the same value from every CTA to every CTA: read after the next cluster barrier
  auto spread_f = [&](float v) {
    if (tid < C) cluster.map_shared_rank(&sm, tid)->gather_f[turn][rank] = v;
  };
  auto spread_u = [&](u64 v) {
    if (tid < C) cluster.map_shared_rank(&sm, tid)->gather_u[turn][rank] = v;
  };
#define EACH(body_)                                                     \
  _Pragma("unroll 1") for (int j = 0; j < NV; ++j) {                    \
    const int i0_ = first_of(j);                                        \
    const Vec<TI> vec_ = row_data[j * kSampleThreads];                  \
    _Pragma("unroll") for (int e = 0; e < VEC; ++e) {                   \
      const float v = vec_.at(e);                                       \
      const int i = i0_ + e;                                            \
      body_                                                             \
    }                                                                   \
  }

  // ---- the largest logit
  {
    const unsigned m = __reduce_max_sync(~0u, key_of(top));
    if (lane == 0) sm.maxima[warp] = m;
    __syncthreads();
    top = value_of(__reduce_max_sync(~0u, sm.maxima[lane & (kSampleWarps - 1)]));
    spread_f(top);
    cluster.sync();
    for (int c = 0; c < C; ++c) top = fmaxf(top, sm.gather_f[turn][c]);
    turn ^= 1;
  }
  if (top == -INFINITY) {  // nothing can be drawn
    if (rank == 0 && tid == 0) a.out[row] = -1;
    cluster.sync();  // (no CTA leaves while another may still write to it)
    return;
  }
  const float temperature = a.temperature ? a.temperature[row] : a.temperature0;
  const float p = a.top_p ? a.top_p[row] : a.top_p0, minp = a.min_p ? a.min_p[row] : a.min_p0;
  int64_t k = a.top_k0;
  if (a.top_k) k = a.top_k_bytes == 8 ? static_cast<const int64_t *>(a.top_k)[row] : static_cast<const int *>(a.top_k)[row];
  if (k <= 0 || k > a.V) k = a.V;

  // Sums over groups of 32 threads' vectors in the order of the indices, sm.group[j * warps + warp]: the first index at
  // which the running sum of `weight` exceeds `target` (which has to be below the whole), written by the warp that finds it.
  auto group_scan = [&](u64 &before, u64 &whole) {  // -> what lies before this warp's groups j = 0, in `before`
    // every CTA's total
    __syncthreads();
    u64 mine = 0;
    for (int g = tid; g < NV * kSampleWarps; g += kSampleThreads) mine += sm.group[g];
    for (int d = 16; d > 0; d >>= 1) mine += __shfl_xor_sync(~0u, mine, d);
    if (lane == 0) sm.sums[warp] = mine;
    __syncthreads();
    u64 total = 0;
    for (int w = 0; w < kSampleWarps; ++w) total += sm.sums[w];
    spread_u(total);
    cluster.sync();
    before = 0;
    whole = 0;
    for (int c = 0; c < C; ++c) {
      const u64 t = sm.gather_u[turn][c];
      if (c < rank) before += t;
      whole += t;
    }
    turn ^= 1;
  };
  // (vectors of one j lie side by side over the CTA's threads: groups follow one another in the order of the indices)
  auto locate = [&](u64 before, u64 target, auto weight, auto found) {
    // groups before this warp's, j by j
    for (int j = 0; j < NV; ++j) {
      u64 start = before, here = 0;
      for (int w = 0; w < kSampleWarps; ++w) {
        const u64 s = sm.group[j * kSampleWarps + w];
        if (w < warp) start += s;
        if (w == warp) here = s;
        before += s;
      }
      if (start <= target && target < start + here) {
        u64 lanes[VEC], sum = 0;
        const Vec<TI> vec = row_data[j * kSampleThreads];
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum += lanes[e] = weight(vec.at(e), first_of(j) + e);
        u64 run = sum;
        for (int d = 1; d < 32; d <<= 1) {
          const u64 o = __shfl_up_sync(~0u, run, d);
          if (lane >= d) run += o;
        }
        run += start;
        u64 at = run - sum;
        if (at <= target && target < run) {
          int here_e = VEC - 1;
#pragma unroll
          for (int e = 0; e < VEC - 1; ++e) {
            at += lanes[e];
            if (target < at && here_e == VEC - 1) here_e = e;
          }
          found(first_of(j) + here_e);
        }
      }
    }
  };
  auto fill_groups = [&](auto weight) {
#pragma unroll 1
    for (int j = 0; j < NV; ++j) {
      u64 s = 0;
      const Vec<TI> vec = row_data[j * kSampleThreads];
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += weight(vec.at(e), first_of(j) + e);
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
      if (lane == 0) sm.group[j * kSampleWarps + warp] = s;
    }
  };

  if (!(temperature > 0.f) || k == 1 || !(p > 0.f) || !(minp <= 1.f)) {  // the first largest logit
    auto is_top = [&](float v, int) -> u64 { return v == top; };
    fill_groups(is_top);
    u64 before, whole;
    group_scan(before, whole);
    locate(before, 0, is_top, [&](int i) { a.out[row] = i; });
    cluster.sync();
    return;
  }
  const bool infinite = top == INFINITY;  // the largest share the mass
  const double per_unit = 1.0 / (double)temperature;
  // exp of a difference below zero by table: 2^(i/64) and the series of e^r, |r| <= ln 2 / 128 (r^6 / 720 < 2^-54); as an
  // integer of 2^-44, zero from exp(-31) on
  auto mass_of = [&](float v) -> u64 {
    if (v == top) return 1ull << 44;
    if (infinite) return 0;
    const double y = ((double)v - (double)top) * per_unit;
    if (!(y > -31.0)) return 0;
    constexpr double kLn2 = 0.693147180559945309417232121458;
    const double t = fma(y, 64.0 / kLn2, 6755399441055744.0);  // 1.5 * 2^52: the rounded integer in the low bits
    const int n = __double2loint(t);
    const double s = fma(t - 6755399441055744.0, -kLn2 / 64.0, y);
    const double e = fma(s, fma(s, fma(s, fma(s, fma(s, 1.0 / 120, 1.0 / 24), 1.0 / 6), 0.5), 1.0), 1.0);
    const double b = sm.table[n & 63];
    const double f = e * __hiloint2double(__double2hiint(b) + ((n >> 6) << 20), __double2loint(b));
    const double q = fma(f, 17592186044416.0, 4503599627370496.0);  // 2^44 and 2^52
    return ((u64)(unsigned)(__double2hiint(q) & 0xfffff) << 32) | (unsigned)__double2loint(q);
  };
  const float steps = (float)(16.0 * 1.4426950408889634 / (double)temperature);
  auto step_of = [&](float v) { return v == top ? 0.f : infinite ? INFINITY : (top - v) * steps; };  // (rounding is monotone)
  auto bin_of = [&](float t) { return t < (float)kTail ? (int)t : kTail; };

  // What stays: logits above border_x, and those at it up to index border_i.
  float border_x = -INFINITY;
  int border_i = 0x7fffffff;
  auto stays = [&](float v, int i) { return v > border_x || (v == border_x && i <= border_i); };

  // ---- a border: the first token, from the top, with which the weights of the tokens that stay reach the target
  // masses: weights are masses and the target p of their whole; else numbers of tokens and the target k.
  // Leaves the border, and with masses the sums of what stays in the groups (those with at least min_p of the largest mass).
  bool summed = false;
  auto weight15 = [&](float part) { return (unsigned)__float2int_rn(exp2f(part * (-1.f / 16)) * 32768.f); };
  const u64 least = minp > 0.f ? (u64)ceil((double)minp * 17592186044416.0) : 0;
  auto narrow = [&](bool masses) {
    float tail = 0.f;
    EACH({
      if (stays(v, i)) {
        const float t = step_of(v);
        const int b = bin_of(t);
        if (!masses) atomicAdd(&sm.hist[b], 1u);
        else if (b < kTail) atomicAdd(&sm.hist[b], weight15(t - (float)b));
        else tail += exp2f(t * (-1.f / 16));
      }
    })
    // picks the bin: every CTA the same from everybody's histograms; unit: of a bin's weights
    double target = (double)k, above = 0.0, whole = 0.0;
    auto pick = [&](auto unit, double rest, double base) {
      cluster.sync();
      double w = 0.0;
      for (int c = 0; c < C; ++c) w += (double)cluster.map_shared_rank(&sm, c)->hist[tid];
      w *= unit(tid);
      double run = w;
      for (int d = 1; d < 32; d <<= 1) {
        const double o = __shfl_up_sync(~0u, run, d);
        if (lane >= d) run += o;
      }
      if (lane == 31) sm.scan[warp] = run;
      __syncthreads();
      double start = base, all = base;
      for (int i = 0; i < kSampleWarps; ++i) {
        if (i < warp) start += sm.scan[i];
        all += sm.scan[i];
      }
      whole = all + rest;
      if (masses && base == 0.0 && rest >= 0.0) target = (double)p * whole;
      const bool reached = start + run >= target;
      const unsigned votes = __ballot_sync(~0u, reached);
      if (tid == 0) sm.pick_bin = kBins;
      __syncthreads();
      if (reached && lane == __ffs(votes) - 1) atomicMin(&sm.pick_bin, tid);
      __syncthreads();
      const int b = sm.pick_bin;
      if (b == tid) sm.pick_before = start + run - w;
      if (b == kBins && tid == 0) sm.pick_before = all;
      cluster.sync();  // (everybody has read the histograms)
      above = sm.pick_before;
      sm.hist[tid] = 0;
      __syncthreads();
      return b;
    };
    if (masses) {
      for (int d = 16; d > 0; d >>= 1) tail += __shfl_xor_sync(~0u, tail, d);
      if (lane == 0) sm.scan[warp] = tail;
      __syncthreads();
      tail = 0.f;
      for (int w = 0; w < kSampleWarps; ++w) tail += (float)sm.scan[w];
      spread_f(tail);
    }
    int bin;
    {
      const int t0 = turn;
      auto unit = [&](int b) { return masses ? exp2((double)b * (-1.0 / 16)) * (1.0 / 32768) : 1.0; };
      double rest = 0.0;
      if (masses) {
        cluster.sync();
        for (int c = 0; c < C; ++c) rest += (double)sm.gather_f[t0][c];
        turn ^= 1;
      }
      bin = pick(unit, rest, 0.0);
      if (bin > kTail) bin = kTail;
    }
    // gathers the bin's tokens; divides it while they are too many
    unsigned low = 0, high = ~0u;  // keys
    auto inside = [&](float v) {
      const unsigned key = key_of(v);
      return key >= low && key <= high && bin_of(step_of(v)) == bin;
    };
    int n;
    for (;;) {
      unsigned lo = ~0u, hi = 0;
      EACH({
        const bool in = v > -INFINITY && stays(v, i) && inside(v);
        if (in) {
          const int at = atomicAdd(&sm0.count, 1);
          const unsigned key = key_of(v);
          if (at < kList) sm0.list[at] = ((u64)key << 32) | (unsigned)~i;
          lo = min(lo, key);
          hi = max(hi, key);
        }
      })
      lo = __reduce_min_sync(~0u, lo);
      hi = __reduce_max_sync(~0u, hi);
      if (lane == 0 && hi) {
        atomicMin(&sm0.lowest, lo);
        atomicMax(&sm0.highest, hi);
      }
      cluster.sync();
      n = sm0.count;
      const unsigned all_lo = sm0.lowest, all_hi = sm0.highest;
      cluster.sync();
      if (rank == 0 && tid == 0) {
        sm.count = 0;
        sm.lowest = ~0u;
        sm.highest = 0;
      }
      if (n > 0) {
        low = all_lo;
        high = all_hi;
      }
      if (n <= kList || low == high) break;
      // by keys, the highest first
      const int cut = max(0, 32 - __clz(high - low) - 9);
      const float edge = step_of(value_of(high));
      EACH({
        if (v > -INFINITY && stays(v, i) && inside(v))
          atomicAdd(&sm.hist[(high - key_of(v)) >> cut], masses ? weight15(step_of(v) - edge) : 1u);
      })
      const double unit = masses ? exp2((double)edge * (-1.0 / 16)) * (1.0 / 32768) : 1.0;
      int b = pick([&](int) { return unit; }, -1.0, above);
      if (b == kBins) b = (int)((high - low) >> cut);  // (weights that rounded away: the lowest)
      const unsigned from = high - ((unsigned)b << cut);
      low = max(low, cut ? from - ((1u << cut) - 1) : from);
      high = from;
    }
    // what lies above the bin, exactly, and in the groups
    u64 sure = 0;
    if (masses) {
      const float highest = value_of(high);
      u64 mine = 0;
      fill_groups([&](float v, int i) -> u64 {
        if (!(v > -INFINITY) || !stays(v, i)) return 0;
        const int b = bin_of(step_of(v));
        if (n > 0 ? v <= highest : b >= bin) return 0;
        const u64 m = mass_of(v);
        mine += m;
        return m >= least ? m : 0;
      });
      for (int d = 16; d > 0; d >>= 1) mine += __shfl_xor_sync(~0u, mine, d);
      if (lane == 0) sm.sums[warp] = mine;
      __syncthreads();
      mine = 0;
      for (int w = 0; w < kSampleWarps; ++w) mine += sm.sums[w];
      spread_u(mine);
      cluster.sync();
      for (int c = 0; c < C; ++c) sure += sm.gather_u[turn][c];
      turn ^= 1;
    }
    const double one = 17592186044416.0;
    if (n == 0) {  // (a tail without tokens, or weights that rounded away)
      if (masses) summed = true;
      return;
    }
    if (n <= kList) {
      if (rank == 0) {
        int size = 32;
        while (size < n) size *= 2;
        for (int i = n + tid; i < size; i += kSampleThreads) sm.list[i] = 0;
        // descending by logit, ascending by index
        for (int len = 2; len <= size; len *= 2)
          for (int step = len / 2; step > 0; step /= 2) {
            __syncthreads();
            for (int i = tid; i < size / 2; i += kSampleThreads) {
              const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
              const u64 x0 = sm.list[lo], x1 = sm.list[hi];
              if (((lo & len) == 0) == (x0 < x1)) {
                sm.list[lo] = x1;
                sm.list[hi] = x0;
              }
            }
          }
        __syncthreads();
        if (warp == 0) {  // walks the list: 32 at a time
          const double need = masses ? target * one - (double)sure : target - above;
          u64 seen = 0;
          int last = n - 1;
          for (int i0 = 0; i0 < n; i0 += 32) {
            u64 w = 0;
            if (i0 + lane < n) w = masses ? mass_of(value_of((unsigned)(sm.list[i0 + lane] >> 32))) : 1;
            u64 run = w;
            for (int d = 1; d < 32; d <<= 1) {
              const u64 o = __shfl_up_sync(~0u, run, d);
              if (lane >= d) run += o;
            }
            const unsigned there = __ballot_sync(~0u, i0 + lane < n && (double)(seen + run) >= need);
            if (there) {
              last = i0 + __ffs(there) - 1;
              break;
            }
            seen += __shfl_sync(~0u, run, 31);
          }
          if (lane == 0) {
            sm.border_x = value_of((unsigned)(sm.list[last] >> 32));
            sm.border_i = (int)~(unsigned)sm.list[last];
          }
        }
      }
      cluster.sync();
      border_x = sm0.border_x;
      border_i = sm0.border_i;
      if (masses) {  // the list's tokens that stay join the groups
        EACH({
          if (v > -INFINITY && inside(v) && stays(v, i)) {
            const u64 m = mass_of(v);
            if (m >= least) atomicAdd(&sm.group[j * kSampleWarps + warp], m);
          }
        })
        summed = true;
      }
      cluster.sync();
    } else {  // many tokens of one value: their number decides, and the index of the last
      const float value = value_of(high);
      u64 m = mass_of(value);
      double want = masses ? (m ? ceil((target * one - (double)sure) / (double)m) : (double)n) : target - above;
      const u64 ties = (u64)fmin(fmax(want, 1.0), (double)n);
      auto is_tie = [&](float v, int i) -> u64 { return v == value && stays(v, i); };
      fill_groups(is_tie);
      u64 before, whole_ties;
      group_scan(before, whole_ties);
      locate(before, ties - 1, is_tie, [&](int i) { sm0.border_i = i; });
      cluster.sync();
      border_i = sm0.border_i;
      border_x = value;
      cluster.sync();
    }
  };
  if (k < a.V) narrow(false);
  if (p < 1.f) narrow(true);

  // ---- the draw
  auto kept = [&](float v, int i) -> u64 {
    if (!(v > -INFINITY) || !stays(v, i)) return 0;
    const u64 m = mass_of(v);
    return m >= least ? m : 0;
  };
  if (!summed) fill_groups(kept);
  u64 before, z;
  group_scan(before, z);
  double u = a.u_bytes == 4 ? (double)static_cast<const float *>(a.u)[row] : static_cast<const double *>(a.u)[row];
  u = fmin(fmax(u, 0.0), 1.0);
  // running > u z: of integers, running > its floor; below z, so that there always is such a token
  const u64 target = min((u64)(u * (double)z), z - 1);
  locate(before, target, kept, [&](int i) { a.out[row] = i; });
  cluster.sync();
#undef EACH
}

// A row's cluster: few vectors a thread where the rows leave SMs for more CTAs (two to an SM).
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
