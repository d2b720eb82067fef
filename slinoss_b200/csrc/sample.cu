// Tokens from logits and given random numbers: temperature, top-k, top-p, min-p.
//
// Tokens are ranked by logit (ties: lower index first).  The first top_k stay; of these the shortest run that holds at least
// top_p of their mass; of these the ones with at least min_p of the largest mass.  The draw goes through what is left in the
// order of the indices and takes the first token at which the running mass exceeds u times the whole.
//
// Both thresholds are found by radix selection over order-preserving integer keys of the logits: a histogram of one digit of
// the keys still undecided (numbers of tokens for top-k, masses for top-p), then the bin in which the border lies.  Masses
// are exponentials in 64 bits, held as integers of 2^-44 of the largest: integer sums do not depend on the order of the
// atomics, and a running mass that is off by 2^-45 a token decides differently from exact sums once in some 10^9 draws.
// One CTA per row.
#include "common.cuh"

namespace slx {

struct SampleArgs {
  const void *logits;
  int64_t stride;
  int V, dtype;
  const void *u;
  int u_dtype;  // SLX_F32, or 64 for double
  const float *temperature, *top_p, *min_p;
  const void *top_k;
  int top_k_size;  // bytes of an entry
  float temperature0, top_p0, min_p0;
  int64_t top_k0;
  int64_t *out;
};

constexpr int kSampleThreads = 1024, kSampleWarps = kSampleThreads / 32;
constexpr double kMassOne = 17592186044416.0;  // 2^44

// Keys: unsigned integers in the order of the values; a NaN counts as -inf.
template <typename TI> struct Key;
template <> struct Key<float> {
  static constexpr int bits = 32;
  static __device__ __forceinline__ unsigned of(float x) {
    const unsigned b = __float_as_uint(x != x ? -INFINITY : x == 0.f ? 0.f : x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
  }
  static __device__ __forceinline__ float value(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
};
template <typename TI> struct Key16 {
  static constexpr int bits = 16;
  static __device__ __forceinline__ unsigned of(TI v) {
    const float x = to_f(v);
    unsigned short b;
    const TI w = x != x ? from_f<TI>(-INFINITY) : x == 0.f ? from_f<TI>(0.f) : v;
    memcpy(&b, &w, 2);
    return b & 0x8000u ? (~b & 0xffffu) : b | 0x8000u;
  }
  static __device__ __forceinline__ float value(unsigned k) {
    const unsigned short b = k & 0x8000u ? k & 0x7fffu : ~k & 0xffffu;
    TI v;
    memcpy(&v, &b, 2);
    return to_f(v);
  }
};
template <> struct Key<__nv_bfloat16> : Key16<__nv_bfloat16> {};
template <> struct Key<__half> : Key16<__half> {};

template <typename TI>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(SampleArgs a) {
  using K = Key<TI>;
  typedef unsigned long long u64;
  __shared__ u64 hist[256], sums[kSampleWarps];
  __shared__ unsigned tops[kSampleWarps];
  __shared__ u64 shared_before, shared_in;
  __shared__ int shared_bin;
  const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = a.V;
  const TI *x = static_cast<const TI *>(a.logits) + row * a.stride;
  auto key_at = [&](int i) { return K::of(x[i]); };

  // the largest key
  unsigned top = 0;
  for (int i = tid; i < V; i += kSampleThreads) top = max(top, key_at(i));
  top = __reduce_max_sync(~0u, top);
  if (lane == 0) tops[warp] = top;
  __syncthreads();
  top = __reduce_max_sync(~0u, tops[lane]);
  const float largest = K::value(top);
  if (largest == -INFINITY) {  // nothing can be drawn
    if (tid == 0) a.out[row] = -1;
    return;
  }

  const float temperature = a.temperature ? a.temperature[row] : a.temperature0;
  const float p = a.top_p ? a.top_p[row] : a.top_p0, minp = a.min_p ? a.min_p[row] : a.min_p0;
  int64_t k = a.top_k0;
  if (a.top_k) k = a.top_k_size == 8 ? static_cast<const int64_t *>(a.top_k)[row] : static_cast<const int *>(a.top_k)[row];
  if (k <= 0 || k > V) k = V;
  const bool greedy = !(temperature > 0.f) || k == 1 || !(p > 0.f) || !(minp <= 1.f);

  auto mass_of = [&](unsigned key) -> double {
    return key == top ? 1.0 : exp(((double)K::value(key) - (double)largest) / (double)temperature);
  };
  auto fixed_of = [&](double m) -> u64 { return (u64)(m * kMassOne + 0.5); };

  // Kept: keys above `border` and the first `ties` tokens at it.
  unsigned border = top;
  u64 ties = 1;
  if (!greedy) {
    // Walks the digits from the highest: `weigh` adds the weights of a digit's bins, `target(before)` says whether the border
    // lies further down.  Leaves the border key, the weight above it and in it.
    u64 above = 0, inside = 0;
    auto select = [&](auto weigh, auto reached) {
      unsigned prefix = 0;
      above = 0;
      for (int shift = K::bits - 8; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kSampleThreads) hist[i] = 0;
        __syncthreads();
        weigh(prefix, shift);
        __syncthreads();
        if (warp == 0) {  // lane 0 holds the eight highest bins
          u64 mine = 0;
          for (int j = 0; j < 8; ++j) mine += hist[255 - 8 * lane - j];
          u64 run = mine;
          for (int d = 1; d < 32; d <<= 1) {
            const u64 o = __shfl_up_sync(~0u, run, d);
            if (lane >= d) run += o;
          }
          u64 before = above + run - mine;
          const unsigned here = __ballot_sync(~0u, reached(above + run));
          const int first = here ? __ffs(here) - 1 : 31;
          if (lane == first) {
            int j = 0;
            for (; j < 7; ++j) {
              const u64 w = hist[255 - 8 * lane - j];
              if (reached(before + w)) break;
              before += w;
            }
            shared_bin = 255 - 8 * lane - j;
            shared_before = before;
            shared_in = hist[255 - 8 * lane - j];
          }
        }
        __syncthreads();
        prefix |= (unsigned)shared_bin << shift;
        above = shared_before;
        inside = shared_in;
        __syncthreads();
      }
      return prefix;
    };
    auto undecided = [&](unsigned key, unsigned prefix, int shift) { return ((u64)(key ^ prefix) >> (shift + 8)) == 0; };

    unsigned kborder = 0;
    u64 kties = ~0ull;
    if (k < V) {
      kborder = select(
          [&](unsigned prefix, int shift) {
            for (int i = tid; i < V; i += kSampleThreads) {
              const unsigned key = key_at(i);
              if (undecided(key, prefix, shift)) atomicAdd(&hist[(key >> shift) & 255], 1ull);
            }
          },
          [&](u64 n) { return n >= (u64)k; });
      kties = k - above;
    }
    border = kborder;
    ties = kties;
    if (p < 1.f) {
      // the whole mass, then the border in it; tokens at the top-k border enter as one entry
      const u64 at_border = k < V ? kties * fixed_of(mass_of(kborder)) : 0;
      u64 z = 0;
      for (int i = tid; i < V; i += kSampleThreads) {
        const unsigned key = key_at(i);
        if (key > kborder || (k == V)) z += fixed_of(mass_of(key));
      }
      for (int d = 16; d > 0; d >>= 1) z += __shfl_xor_sync(~0u, z, d);
      if (lane == 0) sums[warp] = z;
      __syncthreads();
      z = at_border;
      for (int i = 0; i < kSampleWarps; ++i) z += sums[i];
      const double want = (double)p * (double)z;
      const unsigned pborder = select(
          [&](unsigned prefix, int shift) {
            for (int i = tid; i < V; i += kSampleThreads) {
              const unsigned key = key_at(i);
              if ((key > kborder || k == V) && undecided(key, prefix, shift)) {
                const u64 m = fixed_of(mass_of(key));
                if (m) atomicAdd(&hist[(key >> shift) & 255], m);
              }
            }
            if (tid == 0 && k < V && undecided(kborder, prefix, shift)) atomicAdd(&hist[(kborder >> shift) & 255], at_border);
          },
          [&](u64 m) { return (double)m >= want; });
      const u64 one = fixed_of(mass_of(pborder));
      u64 n = ~0ull;
      if (one) {
        const double r = ceil((want - (double)above) / (double)one);
        n = r < 1.0 ? 1 : (u64)r;
      }
      if (pborder > kborder || k == V) {
        border = pborder;
        ties = n;
      } else {
        ties = min(n, kties);
      }
    }
  }

  // Warps take the tokens in runs of the indices' order.
  const int per = ((V + kSampleWarps - 1) / kSampleWarps + 31) / 32 * 32;
  const int lo = min(V, warp * per), hi = min(V, lo + per);
  u64 skip = 0;  // tokens at the border before this warp's run
  {
    u64 n = 0;
    for (int i = lo + lane; i < hi; i += 32) n += key_at(i) == border;
    for (int d = 16; d > 0; d >>= 1) n += __shfl_xor_sync(~0u, n, d);
    __syncthreads();
    if (lane == 0) sums[warp] = n;
    __syncthreads();
    for (int i = 0; i < warp; ++i) skip += sums[i];
    __syncthreads();
  }
  if (greedy) {  // the first token at the largest key
    for (int i0 = lo; i0 < hi && skip == 0; i0 += 32) {
      const unsigned here = __ballot_sync(~0u, i0 + lane < hi && key_at(i0 + lane) == top);
      if (here) {
        if (lane == 0) a.out[row] = i0 + __ffs(here) - 1;
        return;
      }
    }
    return;
  }
  auto kept_mass = [&](int i, u64 &before) -> u64 {  // of 32 tokens in order; before: ties seen
    const unsigned key = i < hi ? key_at(i) : 0;
    const bool tie = i < hi && key == border;
    const unsigned all = __ballot_sync(~0u, tie);
    bool keep = i < hi && (key > border || (tie && before + __popc(all & ((1u << lane) - 1)) < ties));
    before += __popc(all);
    if (!keep) return 0;
    const double m = mass_of(key);
    return m >= (double)minp ? fixed_of(m) : 0;
  };
  u64 mine = 0, seen = skip;
  for (int i = lo; i < hi; i += 32) mine += kept_mass(i + lane, seen);
  for (int d = 16; d > 0; d >>= 1) mine += __shfl_xor_sync(~0u, mine, d);
  if (lane == 0) sums[warp] = mine;
  __syncthreads();
  u64 before = 0, z = 0;
  for (int i = 0; i < kSampleWarps; ++i) {
    if (i < warp) before += sums[i];
    z += sums[i];
  }
  double u = a.u_dtype == SLX_F32 ? (double)static_cast<const float *>(a.u)[row] : static_cast<const double *>(a.u)[row];
  u = fmin(fmax(u, 0.0), 1.0);
  // running > u z: of integers, running > its floor; below z, so that there always is such a token
  const u64 target = min((u64)(u * (double)z), z - 1);
  if (before > target || before + mine <= target) return;
  seen = skip;
  for (int i = lo; i < hi; i += 32) {
    u64 run = kept_mass(i + lane, seen);
    for (int d = 1; d < 32; d <<= 1) {
      const u64 o = __shfl_up_sync(~0u, run, d);
      if (lane >= d) run += o;
    }
    const unsigned here = __ballot_sync(~0u, before + run > target);
    if (here) {
      if (lane == 0) a.out[row] = i + __ffs(here) - 1;
      return;
    }
    before += __shfl_sync(~0u, run, 31);
  }
}

}  // namespace slx

using namespace slx;

extern "C" int slx_sample(const slx_sample_shape *s, const void *logits, const void *u, const float *temperature,
                          const void *top_k, const float *top_p, const float *min_p, int64_t *out, void *stream) {
  SLX_REQUIRE(s, SLX_E_NULL, "sample: shape is NULL");
  SLX_REQUIRE(logits && u && out, SLX_E_NULL, "sample: a required pointer is NULL");
  SLX_REQUIRE(s->rows > 0 && s->vocab > 0, SLX_E_SHAPE, "sample: sizes must be positive (rows %d, vocab %d)", s->rows, s->vocab);
  SLX_REQUIRE(s->vocab <= 262144, SLX_E_UNSUPPORTED, "sample: vocab must be at most 262144, got %d", s->vocab);
  SLX_REQUIRE(s->dtype == SLX_F32 || s->dtype == SLX_BF16 || s->dtype == SLX_F16, SLX_E_DTYPE, "sample: unknown dtype %d", s->dtype);
  SLX_REQUIRE(!top_k || s->top_k_bytes == 4 || s->top_k_bytes == 8, SLX_E_DTYPE, "sample: top_k entries must have 4 or 8 bytes");
  SLX_REQUIRE(s->u_bytes == 4 || s->u_bytes == 8, SLX_E_DTYPE, "sample: u must be float or double");
  SampleArgs a;
  a.logits = logits;
  a.stride = s->row_stride;
  a.V = s->vocab;
  a.dtype = s->dtype;
  a.u = u;
  a.u_dtype = s->u_bytes == 4 ? SLX_F32 : 64;
  a.temperature = temperature;
  a.top_p = top_p;
  a.min_p = min_p;
  a.top_k = top_k;
  a.top_k_size = s->top_k_bytes;
  a.temperature0 = s->temperature;
  a.top_p0 = s->top_p;
  a.min_p0 = s->min_p;
  a.top_k0 = s->top_k;
  a.out = out;
  cudaStream_t st = as_stream(stream);
  if (s->dtype == SLX_BF16) sample_kernel<__nv_bfloat16><<<s->rows, kSampleThreads, 0, st>>>(a);
  else if (s->dtype == SLX_F16) sample_kernel<__half><<<s->rows, kSampleThreads, 0, st>>>(a);
  else sample_kernel<float><<<s->rows, kSampleThreads, 0, st>>>(a);
  return check_launch("sample_kernel");
}
