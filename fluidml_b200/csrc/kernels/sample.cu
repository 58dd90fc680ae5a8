// One token per row of logits from given random numbers (fml_sample): temperature, top-k, top-p, min-p.
//
// A cluster of CTAs holds a row in shared memory, read once from HBM.  No sort: a cut through the order (logit, then index) is
// a logit and an index, found by histograms that narrow a range of logits, 1024 bins at a time.
//
//   1  largest logit
//   2  counts in bins linear in (largest - logit) / temperature: the logits of a vocabulary spread over all of them, where the
//      leading bits of their encoding would put most into a dozen and serialise the atomics
//   3  top-k: where the bins up to the k-th token hold few tokens (1024), these go to one CTA, which sorts them, cuts and draws.
//      Else the bin that holds the k-th token, as a range of keys (integers in the order of the logits), is binned by key
//      until a bin is one key; of equal logits the lowest indexes are kept
//   4  top-p: the counts bound every bin's weight, which leaves a few bins for the cut; one pass sums the weights of all
//      tokens and of those above these bins exactly and bins the rest by key, as in 3, with weights in place of counts
//   5  min-p, as a key; the draw: sums of the kept weights per warp, in the vocabulary's order (those above 4's bins are known),
//      then the warp that holds the token walks its part
//
// Measured: 256 rows of 131072 bf16 logits, half of them with top-k, the others with top-p and min-p 227 us (a row of the former 60
// instructions per 32 logits, of the latter 170: weights in 64 bits of every logit, for the sum that top-p is a share of); one row
// of 50304 16 us, some ten cluster barriers and two small sorts.
//
// Weights are integers, 2^44 for the largest: their sums are exact in any order, so neither the atomics nor the split over warps
// and CTAs changes a result, and a cumulative sum lies within 2^-27 of the largest weight of the real one however many tokens
// there are (a rounded half unit each, 2^18 tokens).  The exponential is evaluated in 64 bits: its fp32 error, 2^-23 of a
// weight, is as wide as the steps of the random numbers, and would move one token in some thousand draws.
#include "serving_common.cuh"
#include <algorithm>
#include <cooperative_groups.h>
#include <type_traits>

namespace cg = cooperative_groups;

namespace fml {
namespace {

using u64 = unsigned long long;
constexpr int kThreads = 256, kWarps = kThreads / 32, kBins = 1024, kPer = kBins / kThreads, kMaxCluster = 8;
constexpr int kList = 1024;  // candidates that one CTA sorts
constexpr double kOne = 17592186044416.0;  // 2^44: the weight of the largest logit
constexpr float kSpan = 32.0f;             // the bins reach e^-32, below which every weight is a unit

struct SampleArgs {
  const void *logits;
  int64_t row_stride, col_stride, rows;
  const float *uniform, *temperature, *top_p, *min_p;
  int64_t uniform_s, temperature_s, top_p_s, min_p_s;
  IndexView top_k;
  void *tokens;
  float *probabilities;
  int64_t tokens_s, probabilities_s;
  int vocab, slice, tokens_wide, vec;  // slice: tokens per CTA; vec: rows take 16-byte accesses
};

struct Shared {
  u64 hist[kBins], merged[kBins];  // (one of them also the list of candidates)
  uint32_t counts[kBins];
  double part[2 * kWarps];         // u64 or double
  u64 sums[2][kMaxCluster];        // of every CTA
  u64 exchange[2][kMaxCluster];
  u64 found[4];
  double roots[32];
  int listed;
};

// Integers in the order of the logits, as wide as the type; both zeros are one.  Shared memory holds these: cuts compare them.
template <typename T> struct Key {  // 16-bit types
  using Int = uint16_t;
  static constexpr uint32_t kInfinity = std::is_same<T, __half>::value ? 0xfc00u : 0xff80u, kNone = 0xffffu ^ kInfinity;  // of +, - infinity
  __device__ __forceinline__ static uint32_t of(uint32_t u) {
    return u == 0x8000u ? 0x8000u : u & 0x8000u ? ~u & 0xffffu : u | 0x8000u;
  }
  __device__ __forceinline__ static float value(uint32_t k) {
    const unsigned short u = (unsigned short)(k & 0x8000u ? k ^ 0x8000u : ~k);
    return to_f32(*reinterpret_cast<const T *>(&u));
  }
  // two at a time
  __device__ __forceinline__ static uint32_t of_pair(uint32_t u) {
    u = zeros_alike(u);
    return u ^ (0x80008000u | (u >> 15 & 0x00010001u) * 0x7fffu);
  }
  __device__ __forceinline__ static uint32_t zeros_alike(uint32_t u);  // -0 -> 0: adds 0
};
template <> __device__ __forceinline__ uint32_t Key<__half>::zeros_alike(uint32_t u) {
  const __half2 y = __hadd2(*reinterpret_cast<const __half2 *>(&u), __half2half2(__ushort_as_half(0)));
  return *reinterpret_cast<const uint32_t *>(&y);
}
template <> __device__ __forceinline__ uint32_t Key<__nv_bfloat16>::zeros_alike(uint32_t u) {
  const __nv_bfloat162 y = __hadd2(*reinterpret_cast<const __nv_bfloat162 *>(&u), __bfloat162bfloat162(__ushort_as_bfloat16(0)));
  return *reinterpret_cast<const uint32_t *>(&y);
}
template <> struct Key<float> {
  using Int = uint32_t;
  static constexpr uint32_t kInfinity = 0xff800000u, kNone = 0x007fffffu;
  // (on the bits as they were loaded: of a float's, the compiler makes setting the sign a negation, which loses a NaN's bits)
  __device__ __forceinline__ static uint32_t of(uint32_t u) { return u == 0x80000000u ? u : u & 0x80000000u ? ~u : u | 0x80000000u; }
  __device__ __forceinline__ static float value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
};

// e^x for |x| <= ln 2 / 64 by Taylor's series to the fifth power, 2.3e-15: what is left of 2^y besides a power of two and one of
// 2^(i / 32), i = 0 .. 31, which a CTA has in a table.
__device__ __forceinline__ double exp_small(double x) {
  double p = fma(x, 1.0 / 120.0, 1.0 / 24.0);
  p = fma(p, x, 1.0 / 6.0);
  p = fma(p, x, 0.5);
  p = fma(p, x, 1.0);
  return fma(p, x, 1.0);
}

struct Row {
  double top, rate;  // weight = 2^((z - top) * rate / 32)
  const double *roots;  // 2^(i / 32), in shared memory
  float topf, scale;  // bins: (topf - z) / 2 * scale
  double least;       // 32 log2 of min-p, -infinity when off
  uint32_t cut_key;   // kept: a key above cut_key, or equal and an index up to cut_index
  int cut_index;
};

__device__ __forceinline__ double exponent_of(const Row &r, float z) { return z == r.topf ? 0.0 : ((double)z - r.top) * r.rate; }
__device__ __forceinline__ u64 weight_of(const Row &r, float z) {
  const double t = exponent_of(r, z);
  if (!(t >= -45.0 * 32)) return t > -1075.0 * 32 ? 1ull : 0ull;  // (a weight that 64 bits hold; NaN, of an infinite rate: none)
  // adding 1.5 x 2^52 leaves the nearest integer in the low bits, adding 2^52 the rounded weight
  const double shifted = t + 6755399441055744.0;
  const int i = __double2loint(shifted);
  const double p = exp_small((t - (shifted - 6755399441055744.0)) * (0.6931471805599453 / 32)) * r.roots[i & 31];
  const double scaled = __hiloint2double(__double2hiint(p) + (((i >> 5) + 44) << 20), __double2loint(p));
  const u64 w = (u64)__double_as_longlong(scaled + 4503599627370496.0) & 0xfffffffffffffull;
  return w ? w : 1ull;
}
// The weight as a number, of the largest's 1.
__device__ __forceinline__ double share_of(const Row &r, float z) { return exp2(fmax(exponent_of(r, z), -1074.0 * 32) * (1.0 / 32)); }
__device__ __forceinline__ int bin_of(const Row &r, float z) {
  // (halves: the difference of two finite logits may not be finite; that of two infinite ones is NaN, whose integer is 0)
  return min((int)(fmaf(z, -0.5f, 0.5f * r.topf) * r.scale), kBins - 1);
}
__device__ __forceinline__ bool kept_by_cut(const Row &r, uint32_t key, int index) {
  return key > r.cut_key || (key == r.cut_key && index <= r.cut_index);
}

template <typename T> struct Sampler {
  static constexpr int V = 16 / sizeof(T);  // logits per access
  using Int = typename Key<T>::Int;
  const Int *data;
  Shared *sh;
  cg::cluster_group cluster;
  int rank, ranks, base, seg, warp, lane, phase;
  uint32_t top_key;

  // f(key, index in the vocabulary) over the warp's part, in order by lane; the part is whole accesses
  template <typename F> __device__ __forceinline__ void each(F f) const {
    for (int i = warp * seg + lane * V; i < (warp + 1) * seg; i += 32 * V) {
      const uint4 raw = *reinterpret_cast<const uint4 *>(data + i);
#pragma unroll
      for (int j = 0; j < V; ++j) f(key_in(raw, j), base + i + j);
    }
  }
  __device__ __forceinline__ static uint32_t key_in(const uint4 &raw, int j) {
    const uint32_t w = sizeof(T) == 4 ? 0u : j < 2 ? raw.x : j < 4 ? raw.y : j < 6 ? raw.z : raw.w;
    return sizeof(T) == 4 ? (j == 0 ? raw.x : j == 1 ? raw.y : j == 2 ? raw.z : raw.w) : j & 1 ? w >> 16 : w & 0xffffu;
  }
  __device__ __forceinline__ u64 *part() { return reinterpret_cast<u64 *>(sh->part); }
  __device__ __forceinline__ u64 warp_sum(u64 v) const {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  // Sum over the CTA.
  __device__ u64 block_sum(u64 v) {
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) part()[warp] = v;
    __syncthreads();
    u64 all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) all += part()[w];
    return all;
  }
  // Every CTA's `mine` (of its first threads) to all CTAs: exchange[phase][rank]; ends with a cluster barrier.
  __device__ __forceinline__ const u64 *to_all(u64 mine) {
    phase ^= 1;
    if (threadIdx.x < ranks) *cluster.map_shared_rank(&sh->exchange[phase][rank], threadIdx.x) = mine;
    cluster.sync();
    return sh->exchange[phase];
  }
  __device__ uint32_t largest(uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (lane == 0) part()[warp] = v;
    __syncthreads();
    u64 all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) all = max(all, part()[w]);
    const u64 *x = to_all(all);
    all = 0;
    for (int i = 0; i < ranks; ++i) all = max(all, x[i]);
    return (uint32_t)all;
  }
  __device__ void clear() {
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh->hist[i] = 0;
    __syncthreads();
  }
  // Two sums of every CTA into every CTA's sums, to be read behind the next merge().  Once per row: nothing keeps a CTA that is
  // ahead from writing here again while another still reads.
  __device__ void share_sums(u64 s0, u64 s1) {
    if (threadIdx.x < ranks) {
      *cluster.map_shared_rank(&sh->sums[0][rank], threadIdx.x) = s0;
      *cluster.map_shared_rank(&sh->sums[1][rank], threadIdx.x) = s1;
    }
  }
  // hist of all CTAs, added up, into every CTA's merged.  Each CTA adds up its share of the bins.
  __device__ void merge() {
    cluster.sync();
    const int share = kBins / ranks;
    for (int i = rank * share + threadIdx.x; i < (rank + 1) * share; i += kThreads) {
      u64 sum = 0;
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c)
        if (c < ranks) sum += *cluster.map_shared_rank(&sh->hist[i], c);
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c)
        if (c < ranks) *cluster.map_shared_rank(&sh->merged[i], c) = sum;
    }
    cluster.sync();
  }
  __device__ __forceinline__ u64 sum_of(int which) const {
    u64 s = 0;
    for (int c = 0; c < ranks; ++c) s += sh->sums[which][c];
    return s;
  }
  // v: a thread's total -> what the threads before it have (N totals at once); all: the CTA's.
  template <typename U, int N> __device__ __forceinline__ void before(const U (&v)[N], U (&start)[N], U (&all)[N]) {
    U run[N];
    U *p = reinterpret_cast<U *>(sh->part);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      run[n] = v[n];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const U up = __shfl_up_sync(0xffffffffu, run[n], o);
        if (lane >= o) run[n] += up;
      }
    }
    __syncthreads();
    if (lane == 31)
#pragma unroll
      for (int n = 0; n < N; ++n) p[n * kWarps + warp] = run[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      U s = 0, t = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w == warp) s = t;
        t += p[n * kWarps + w];
      }
      start[n] = s + run[n] - v[n];
      all[n] = t;
    }
  }
  // The first bin whose running sum, from `above` on, has reached(sum), and the sum before it; the last bin if none has.
  template <typename R> __device__ void first_bin(u64 above, R reached, int *bin, u64 *sum_before) {
    u64 v[kPer], own[1] = {0}, start[1], all[1];
#pragma unroll
    for (int i = 0; i < kPer; ++i) own[0] += v[i] = sh->merged[kPer * threadIdx.x + i];
    if (threadIdx.x == 0) sh->found[0] = kBins - 1;
    before<u64, 1>(own, start, all);
    u64 run = above + start[0];
    if (threadIdx.x == kThreads - 1 && !reached(run + own[0])) sh->found[1] = run + own[0] - v[kPer - 1];
    if (!reached(run) && reached(run + own[0])) {  // (sums of non-negative numbers: one thread; its first bin that reaches)
      int i = 0;
      while (i < kPer - 1 && !reached(run + v[i])) run += v[i++];
      sh->found[0] = kPer * threadIdx.x + i;
      sh->found[1] = run;
    } else if (threadIdx.x == 0 && reached(above)) {
      sh->found[0] = 0;
      sh->found[1] = above;
    }
    __syncthreads();
    *bin = (int)sh->found[0];
    *sum_before = sh->found[1];
    __syncthreads();
  }
  // The keys of bins [b1, b2]: bin_of is monotone, so they are an interval.  A warp asks 32 keys at a time for either end.
  __device__ void keys_of(const Row &r, int b1, int b2, uint32_t *lo, uint32_t *hi) const {
    const uint32_t top = top_key;
    uint32_t l = Key<T>::kNone + 1, h = top;  // the smallest key of a bin up to b2 is in [l, h]
    while (l < h) {
      const uint32_t step = (h - l) / 33 + 1, m = min(l + (lane + 1) * step - 1, h);
      const unsigned yes = __ballot_sync(0xffffffffu, bin_of(r, Key<T>::value(m)) <= b2);
      const int k = yes ? __ffs(yes) - 1 : 32;  // the first that is
      const uint32_t was = l;
      if (k > 0) l = min(was + (uint32_t)k * step, h);
      if (k < 32) h = min(was + (uint32_t)(k + 1) * step - 1, h);
    }
    *lo = l;
    h = top;  // the largest key of a bin from b1 on is in [l, h]
    while (l < h) {
      const uint32_t step = (h - l) / 33 + 1, m = min(l + (lane + 1) * step, h);
      const unsigned yes = __ballot_sync(0xffffffffu, bin_of(r, Key<T>::value(m)) >= b1);
      const int k = __popc(yes);  // the first k are
      const uint32_t was = l;
      if (k > 0) l = min(was + (uint32_t)k * step, h);
      if (k < 32) h = min(was + (uint32_t)(k + 1) * step - 1, h);
    }
    *hi = l;
  }
  // The smallest key whose weight is not below min-p: the exponent is monotone in the key.
  __device__ uint32_t least_key(const Row &r) const {
    uint32_t l = Key<T>::kNone + 1, h = top_key;
    while (l < h) {
      const uint32_t step = (h - l) / 33 + 1, m = min(l + (lane + 1) * step - 1, h);
      const unsigned yes = __ballot_sync(0xffffffffu, exponent_of(r, Key<T>::value(m)) >= r.least);
      const int k = yes ? __ffs(yes) - 1 : 32;
      const uint32_t was = l;
      if (k > 0) l = min(was + (uint32_t)k * step, h);
      if (k < 32) h = min(was + (uint32_t)(k + 1) * step - 1, h);
    }
    return l;
  }
  // One kept key of the range into the histogram.  A bin of one key counts them (a 32-bit atomic; equal logits, of which a 16-bit
  // type has thousands, meet there, and 64-bit ones would go round in turns); wider bins add up what they measure.
  template <typename W> __device__ __forceinline__ void put(uint32_t hi, int shift, uint32_t key, W unit) {
    if (shift == 0) atomicAdd(reinterpret_cast<uint32_t *>(&sh->hist[hi - key]), 1u);
    else atomicAdd(&sh->hist[(hi - key) >> shift], unit(key));
  }
  // After merge(): counts times what their key measures.
  template <typename W> __device__ void weigh(uint32_t lo, uint32_t hi, int shift, W unit) {
    if (shift) return;
    for (uint32_t i = threadIdx.x; i <= hi - lo; i += kThreads)
      if (sh->merged[i]) sh->merged[i] *= unit(hi - i);
    __syncthreads();
  }
  // Narrows the range of keys [lo, hi], above which lies `above` of the measure (unit(key) for kept(key, index)), to the one key at
  // which the running sum has reached(sum).  first: the histogram of the range is merged already.
  template <typename K, typename W, typename R>
  __device__ void narrow(uint32_t lo, uint32_t hi, u64 above, bool first, K kept, W unit, R reached, uint32_t *key, u64 *sum_before, u64 *ties) {
    for (;;) {
      const int shift = shift_of(lo, hi);
      if (!first) {
        clear();
        each([&](uint32_t k, int i) {
          if (k >= lo && k <= hi && kept(k, i)) put(hi, shift, k, unit);
        });
        merge();
      }
      first = false;
      weigh(lo, hi, shift, unit);
      int b;
      first_bin(above, reached, &b, &above);
      const u64 inside = sh->merged[b];
      hi = hi - min((uint32_t)b << shift, hi - lo);
      if (shift == 0) {
        *key = hi; *sum_before = above; *ties = inside;
        return;
      }
      lo = max(lo, hi - min(hi, (1u << shift) - 1u));
    }
  }
  __device__ __forceinline__ static int shift_of(uint32_t lo, uint32_t hi) { return max(0, 22 - __clz((int)((hi - lo) | 1u))); }

  // The first index, in the vocabulary's order, at which the running sum of measure(key, index) has reached(sum); -1: none.
  // known: what the warp has of it in keys above `below`, which are then left out of the first pass.
  template <typename M, typename R> __device__ int locate(M measure, R reached, u64 *total, u64 known = 0, uint32_t below = 0xffffffffu) {
    u64 mine = 0;
    each([&](uint32_t k, int i) {
      if (k <= below) mine += measure(k, i);
    });
    mine = warp_sum(mine) + known;
    __syncthreads();
    if (lane == 0) part()[warp] = mine;
    if (threadIdx.x == 0) sh->found[3] = ~0ull;
    __syncthreads();
    u64 start = 0, all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) start = all;
      all += part()[w];
    }
    const u64 *x = to_all(all);
    u64 sum = 0;
    for (int c = 0; c < ranks; ++c) {
      if (c == rank) start += sum;
      sum += x[c];
    }
    *total = sum;
    if (!reached(start, sum) && reached(start + mine, sum)) {  // (one warp of the cluster)
      bool done = false;
      for (int i = warp * seg + lane * V; i < (warp + 1) * seg && !done; i += 32 * V) {
        const uint4 raw = *reinterpret_cast<const uint4 *>(data + i);
        u64 m[V], own = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) own += m[j] = measure(key_in(raw, j), base + i + j);
        u64 run = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 up = __shfl_up_sync(0xffffffffu, run, o);
          if (lane >= o) run += up;
        }
        u64 at = start + run - own;
        if (!reached(at, sum) && reached(at + own, sum)) {
          int j = 0;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            at += m[k];
            if (!reached(at, sum)) j = k + 1;
          }
          for (int c = 0; c < ranks; ++c) *cluster.map_shared_rank(&sh->found[3], c) = (u64)(base + i + j);
        }
        start = __shfl_sync(0xffffffffu, start + run, 31);
        done = reached(start, sum);
      }
    }
    cluster.sync();
    const u64 got = sh->found[3];
    return got == ~0ull ? -1 : (int)got;
  }
  // Sorts n <= kList numbers of the CTA, the rest of the next power of two filled up with the largest number.
  __device__ void sort(u64 *list, int n) {
    int size = 32;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += kThreads) list[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j; j >>= 1) {
        for (int i = threadIdx.x; i < size / 2; i += kThreads) {
          const int a = 2 * i - (i & (j - 1)), b = a + j;
          const u64 x = list[a], y = list[b];
          if ((x > y) == ((a & k) == 0)) { list[a] = y; list[b] = x; }
        }
        __syncthreads();
      }
  }
};

// Top-k of at most kList candidates, gathered in one CTA: sorted, cut, and drawn there.
template <typename T>
__device__ int draw_listed(Sampler<T> &s, const Row &r, int n, int k, float p, float u, double *probability) {
  u64 *const list = s.sh->hist, *const weights = s.sh->merged;
  s.sort(list, n);  // by falling key, then index
  n = min(n, k);
  // a thread has kPer neighbours of the order
  u64 w[kPer], own[1] = {0}, start[1], all[1];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int at = kPer * threadIdx.x + i;
    w[i] = at < n ? weight_of(r, Key<T>::value(~(uint32_t)(list[at] >> 32))) : 0ull;
    own[0] += w[i];
  }
  s.template before<u64, 1>(own, start, all);
  const double want = (double)fmaxf(p, 0.0f) * (double)all[0];
  u64 run = start[0];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int at = kPer * threadIdx.x + i;
    const u64 sum_before = run;
    run += w[i];
    const bool kept = at < n && (!(p < 1.0f) || at == 0 || (double)sum_before < want) &&
                      exponent_of(r, Key<T>::value(~(uint32_t)(list[at] >> 32))) >= r.least;
    if (!kept) w[i] = 0;
  }
  __syncthreads();
  // back to the vocabulary's order: index above, place below
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int at = kPer * threadIdx.x + i;
    if (at < n) {
      weights[at] = w[i];
      list[at] = (list[at] & 0xffffffffull) << 32 | (u64)at;
    }
  }
  __syncthreads();
  s.sort(list, n);
  own[0] = 0;
  int index[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int at = kPer * threadIdx.x + i;
    index[i] = at < n ? (int)(list[at] >> 32) : -1;
    w[i] = at < n ? weights[list[at] & 0xffffffffull] : 0ull;
    own[0] += w[i];
  }
  s.template before<u64, 1>(own, start, all);
  const double target = (double)u * (double)all[0];
  if (threadIdx.x == 0) s.sh->found[0] = ~0ull;
  __syncthreads();
  run = start[0];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (!((double)run > target) && (double)(run + w[i]) > target) s.sh->found[0] = (u64)index[i];
    run += w[i];
  }
  __syncthreads();
  const int token = s.sh->found[0] == ~0ull ? -1 : (int)s.sh->found[0];
  *probability = (double)all[0];
  return token;
}

template <typename T> __global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  __shared__ Shared shared;
  using Int = typename Key<T>::Int;
  Sampler<T> s{reinterpret_cast<const Int *>(raw), &shared, cg::this_cluster()};
  s.rank = (int)s.cluster.block_rank();
  s.ranks = (int)s.cluster.num_blocks();
  s.warp = threadIdx.x >> 5; s.lane = threadIdx.x & 31;
  s.base = s.rank * a.slice; s.seg = a.slice / kWarps; s.phase = 0;
  const int64_t row = blockIdx.x / s.ranks;
  // Nobody writes to another CTA's shared memory before that CTA runs: everyone says so here and asks below, behind the loads
  s.cluster.barrier_arrive();
  pdl_prologue();
  float temperature = a.temperature ? a.temperature[row * a.temperature_s] : 1.0f;
  float p = a.top_p ? a.top_p[row * a.top_p_s] : 1.0f;
  const float m = a.min_p ? a.min_p[row * a.min_p_s] : 0.0f;
  const int64_t k = a.top_k.p ? index_at(a.top_k, row) : 0;
  float u = a.uniform[row * a.uniform_s];
  // ---- 1: the slice's keys into shared memory, -infinity behind its end and for NaN
  constexpr int V = Sampler<T>::V;
  Int *const data = reinterpret_cast<Int *>(raw);
  const T *const src = static_cast<const T *>(a.logits) + row * a.row_stride;
  uint32_t top = 0, bottom = 0xffffffffu;  // (16-bit types: of pairs)
#pragma unroll 4
  for (int i = threadIdx.x * V; i < a.slice; i += kThreads * V) {
    uint4 k;
    uint32_t *const w = reinterpret_cast<uint32_t *>(&k);
    if (a.vec && s.base + i + V <= a.vocab) {
      const uint4 x = __ldg(reinterpret_cast<const uint4 *>(src + s.base + i));
      const uint32_t *const y = reinterpret_cast<const uint32_t *>(&x);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 2) w[j] = Key<T>::of_pair(y[j]);
        else w[j] = Key<T>::of(y[j]);
      }
    } else {
      uint32_t y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = s.base + i + j < a.vocab ? Key<T>::of(reinterpret_cast<const Int *>(src)[(int64_t)(s.base + i + j) * a.col_stride]) : Key<T>::kNone;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = sizeof(T) == 4 ? y[j] : y[2 * j % V] | y[(2 * j + 1) % V] << 16;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      top = sizeof(T) == 2 ? __vmaxu2(top, w[j]) : max(top, w[j]);
      bottom = sizeof(T) == 2 ? __vminu2(bottom, w[j]) : min(bottom, w[j]);
    }
    *reinterpret_cast<uint4 *>(data + i) = k;
  }
  if (sizeof(T) == 2) {
    top = max(top >> 16, top & 0xffffu);
    bottom = min(bottom >> 16, bottom & 0xffffu);
  }
  if (top > Key<T>::kInfinity || bottom < Key<T>::kNone) {  // rare: NaN lies beyond the infinities
    top = 0;
    for (int i = threadIdx.x * V; i < a.slice; i += kThreads * V) {
      uint4 k = *reinterpret_cast<const uint4 *>(data + i);
      uint32_t *const w = reinterpret_cast<uint32_t *>(&k);
      for (int j = 0; j < V; ++j) {
        const uint32_t key = Sampler<T>::key_in(k, j);
        if (key <= Key<T>::kInfinity && key >= Key<T>::kNone) top = max(top, key);
        else if (sizeof(T) == 4) w[j] = Key<T>::kNone;
        else w[j >> 1] = j & 1 ? (w[j >> 1] & 0xffffu) | Key<T>::kNone << 16 : (w[j >> 1] & 0xffff0000u) | Key<T>::kNone;
      }
      *reinterpret_cast<uint4 *>(data + i) = k;
    }
  }
  if (threadIdx.x < 32) shared.roots[threadIdx.x] = exp2(threadIdx.x * (1.0 / 32));
  __syncwarp();
  s.cluster.barrier_wait();
  const uint32_t top_key = s.largest(top);  // (its barriers publish the slice too)
  s.top_key = top_key;
  if (temperature > 0.0f) temperature = fmaxf(temperature, 1e-30f);  // (the bins' scale stays finite)
  int token = -1;
  double probability = 0.0;
  if (top_key > Key<T>::kNone) {
    Row r;
    r.topf = Key<T>::value(top_key);
    r.top = (double)r.topf;
    r.rate = 32 * 1.4426950408889634 / (double)temperature;
    r.roots = shared.roots;
    r.scale = 2.0f * (float)kBins / kSpan / temperature;
    r.cut_key = Key<T>::kNone + 1; r.cut_index = a.vocab;
    r.least = m > 0.0f ? 32 * log2((double)fminf(m, 1.0f)) : -INFINITY;
    u = u >= 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    if (!(temperature > 0.0f)) {
      // the largest logit, lowest index
      u64 total;
      token = s.locate([&](uint32_t key, int) { return (u64)(key == top_key); }, [](u64 c, u64) { return c >= 1; }, &total);
      probability = 1.0;
    } else {
      const bool by_k = k > 0 && k < a.vocab, by_p = p < 1.0f;
      // ---- 2: counts by distance from the largest
      if (by_k || by_p) {
        uint32_t *h = reinterpret_cast<uint32_t *>(shared.hist);
        if (threadIdx.x == 0) shared.listed = 0;
        s.clear();
        s.each([&](uint32_t key, int) {
          if (key > Key<T>::kNone) atomicAdd(&h[2 * bin_of(r, Key<T>::value(key))], 1u);
        });
        s.merge();  // (64-bit words whose upper halves are zero)
        for (int i = threadIdx.x; i < kBins; i += kThreads) shared.counts[i] = (uint32_t)shared.merged[i];
        __syncthreads();
      }
      // ---- 3: top-k
      if (by_k) {
        const u64 want = (u64)k;
        int b;
        u64 above;
        s.first_bin(0ull, [&](u64 c) { return c >= want; }, &b, &above);
        if (above + shared.counts[b] <= (u64)kList && above + shared.counts[b] >= want) {
          // few enough candidates for one CTA's shared memory: the rest happens there
          u64 *const list = s.cluster.map_shared_rank(shared.hist, 0);
          int *const listed = s.cluster.map_shared_rank(&shared.listed, 0);
          uint32_t lo, hi;
          s.keys_of(r, 0, b, &lo, &hi);
          s.each([&](uint32_t key, int i) {
            if (key >= lo) list[atomicAdd(listed, 1)] = (u64)(uint32_t)~key << 32 | (uint32_t)i;
          });
          s.cluster.sync();
          if (s.rank != 0) return;
          double total;
          token = draw_listed(s, r, (int)above + (int)shared.counts[b], (int)want, p, u, &total);
          if (threadIdx.x == 0) {
            if (token >= 0) {
              const float z = to_f32(src[(int64_t)token * a.col_stride]);  // (perhaps another CTA's)
              probability = share_of(r, z) * kOne / total;
            }
            if (a.tokens_wide) static_cast<int64_t *>(a.tokens)[row * a.tokens_s] = token;
            else static_cast<int32_t *>(a.tokens)[row * a.tokens_s] = token;
            if (a.probabilities) a.probabilities[row * a.probabilities_s] = (float)probability;
          }
          return;
        }
        if (above + shared.counts[b] > want) {  // the cut is inside the bin
          uint32_t lo, hi, key;
          u64 sum_before, ties;
          s.keys_of(r, b, b, &lo, &hi);
          s.narrow(lo, hi, above, false, [](uint32_t, int) { return true; }, [](uint32_t) { return 1ull; }, [&](u64 c) { return c >= want; }, &key,
                   &sum_before, &ties);
          r.cut_key = key;
          if (sum_before + ties > want) {
            u64 total;
            r.cut_index = s.locate([&](uint32_t x, int) { return (u64)(x == key); }, [&](u64 c, u64) { return c >= want - sum_before; }, &total);
          }
        } else if (above + shared.counts[b] == want) {  // behind it
          uint32_t lo, hi;
          s.keys_of(r, b, b, &lo, &hi);
          r.cut_key = lo;
        }  // (fewer tokens than k: all)
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads)
          if (i > b) shared.counts[i] = 0;
          else if (i == b) shared.counts[i] = (uint32_t)min((u64)shared.counts[i], want - above);
        __syncthreads();
      }
      // ---- 4: top-p
      u64 known = 0;                  // this warp's weights of keys above `range`, all of which are kept
      uint32_t range = 0xffffffffu;
      if (by_p) {
        const double share = p > 0.0f ? (double)p : 0.0;  // (0: the first token alone)
        // A bin's weights, in units of the largest, are exp(-x) for x between its ends: sums of the most and of the least they can
        // be, with more than fp32's errors to spare.
        const float width = kSpan / kBins * 1.4426950408889634f;
        double own[2] = {0.0, 0.0}, start[2], all2[2], most[kPer], least[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const int i = kPer * threadIdx.x + j;
          const double count = (double)shared.counts[i];
          most[j] = count * ((double)exp2f(-(float)i * width * (1.0f - 1e-5f)) * 1.0001 + 1e-13);
          least[j] = i == kBins - 1 ? 0.0 : count * fmax(0.0, (double)exp2f(-(float)(i + 1) * width * (1.0f + 1e-5f)) * 0.9999 - 1e-13);
          own[0] += most[j];
          own[1] += least[j];
        }
        if (threadIdx.x == 0) reinterpret_cast<int *>(shared.found)[0] = reinterpret_cast<int *>(shared.found)[1] = kBins - 1;
        s.template before<double, 2>(own, start, all2);
        int *const ends = reinterpret_cast<int *>(shared.found);
        // the cut is no earlier than the first bin that the most can reach it in, and no later than the first that the least must
        const double early = share * all2[1] * (1 - 1e-9), late = share * all2[0] * (1 + 1e-9);
#pragma unroll
        for (int j = kPer - 1; j >= 0; --j) {
          double c0 = start[0], c1 = start[1];
          for (int i = 0; i <= j; ++i) { c0 += most[i]; c1 += least[i]; }
          if (c0 >= early) atomicMin(&ends[0], kPer * (int)threadIdx.x + j);
          if (c1 >= late) atomicMin(&ends[1], kPer * (int)threadIdx.x + j);
        }
        __syncthreads();
        const int b1 = ends[0], b2 = max(b1, ends[1]);
        __syncthreads();
        uint32_t lo, hi;
        s.keys_of(r, b1, b2, &lo, &hi);
        const int shift = Sampler<T>::shift_of(lo, hi);
        u64 all = 0, over = 0;
        s.clear();
        s.each([&](uint32_t key, int i) {
          if (kept_by_cut(r, key, i)) {
            const u64 w = weight_of(r, Key<T>::value(key));
            all += w;
            if (key > hi) over += w;
            else if (key >= lo) s.put(hi, shift, key, [&](uint32_t) { return w; });
          }
        });
        known = s.warp_sum(over);
        range = hi;
        all = s.block_sum(all);
        over = s.block_sum(over);
        s.share_sums(all, over);
        s.merge();
        all = s.sum_of(0);
        over = s.sum_of(1);
        const double want = share * (double)all;
        uint32_t key;
        u64 sum_before, ties;
        s.narrow(lo, hi, over, true, [&](uint32_t x, int i) { return kept_by_cut(r, x, i); },
                 [&](uint32_t x) { return weight_of(r, Key<T>::value(x)); }, [&](u64 c) { return (double)c >= want && c > 0; }, &key, &sum_before, &ties);
        const u64 w = weight_of(r, Key<T>::value(key));
        // of the tied tokens the first n: those before which less than `want` lies
        u64 n = w ? (u64)fmax(ceil((want - (double)sum_before) / (double)w), 1.0) : 1;
        while (n > 1 && !((double)(sum_before + (n - 1) * w) < want)) --n;
        while (w && (double)(sum_before + n * w) < want && n * w < ties) ++n;
        int index = r.cut_index;
        if (w && n * w < ties) {
          u64 total;
          index = s.locate([&](uint32_t x, int i) { return (u64)(x == key && kept_by_cut(r, x, i)); }, [&](u64 c, u64) { return c >= n; }, &total);
        } else if (key != r.cut_key) {
          index = a.vocab;
        }
        r.cut_key = key;
        r.cut_index = index;
      }
      // ---- 5: the draw
      if (m > 0.0f) {
        const uint32_t least = s.least_key(r);
        if (least > r.cut_key) {
          r.cut_key = least;
          r.cut_index = a.vocab;
          if (least > range) { known = 0; range = 0xffffffffu; }  // (some keys above the range are not kept)
        }
      }
      u64 total;
      token = s.locate([&](uint32_t key, int i) { return kept_by_cut(r, key, i) ? weight_of(r, Key<T>::value(key)) : 0ull; },
                       [&](u64 c, u64 sum) { return (double)c > (double)u * (double)sum; }, &total, known, range);
      if (token >= s.base && token < s.base + a.slice) {
        const uint4 k = *reinterpret_cast<const uint4 *>(data + (token - s.base) / V * V);
        const uint32_t *const w = reinterpret_cast<const uint32_t *>(&k);
        const int j = (token - s.base) % V;
        const float z = Key<T>::value(sizeof(T) == 4 ? w[j] : j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu);
        probability = share_of(r, z) * kOne / (double)total;
      }
    }
  }
  if (threadIdx.x == 0 && (token < 0 ? s.rank == 0 : token >= s.base && token < s.base + a.slice)) {
    if (a.tokens_wide) static_cast<int64_t *>(a.tokens)[row * a.tokens_s] = token;
    else static_cast<int32_t *>(a.tokens)[row * a.tokens_s] = token;
    if (a.probabilities) a.probabilities[row * a.probabilities_s] = (float)probability;
  }
}

template <typename T> int launch(SampleArgs &a, cudaStream_t s) {
  // Eight CTAs per row, fewer only where half as many hold the vocabulary in one access of every lane.  The number of rows does not
  // count: of clusters of four, 256 rows of 131072 take 329 us instead of 227.
  constexpr int kGrain = kWarps * 32 * Sampler<T>::V;  // whole accesses for every lane
  int ranks = kMaxCluster;
  while (ranks > 1 && a.vocab <= kGrain * (ranks / 2)) ranks >>= 1;
  a.slice = ((a.vocab + ranks - 1) / ranks + kGrain - 1) / kGrain * kGrain;
  const size_t smem = (size_t)a.slice * sizeof(T);
  static bool attr_set[64] = {false};
  int dev = 0;
  FML_CUDA(cudaGetDevice(&dev));
  if (!attr_set[dev & 63]) {
    FML_CUDA(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    attr_set[dev & 63] = true;
  }
  FML_REQUIRE(a.rows * ranks < (1ll << 31), FML_UNSUPPORTED, "fml_sample: too many rows");
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)(a.rows * ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  FML_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel<T>, a));
  return FML_OK;
}

}  // namespace
}  // namespace fml

using namespace fml;

extern "C" int fml_sample(const fml_tensor *logits, const fml_tensor *uniform, const fml_tensor *temperature, const fml_tensor *top_k,
                          const fml_tensor *top_p, const fml_tensor *min_p, const fml_tensor *tokens, const fml_tensor *probabilities,
                          void *stream) {
  FML_REQUIRE(data_tensor(logits, 2), FML_BAD_ARG, "fml_sample: logits must be [rows, vocabulary] of fp32, fp16 or bf16");
  const int64_t rows = logits->shape[0], vocab = logits->shape[1];
  auto per_row = [&](const fml_tensor *t) { return t->shape[0] == rows; };
  FML_REQUIRE(float_tensor(uniform, 1) && per_row(uniform), FML_BAD_ARG, "fml_sample: uniform must be [rows] of fp32");
  FML_REQUIRE(!temperature || (float_tensor(temperature, 1) && per_row(temperature)), FML_BAD_ARG, "fml_sample: temperature must be [rows] of fp32");
  FML_REQUIRE(!top_k || (index_tensor(top_k, 1) && per_row(top_k)), FML_BAD_ARG, "fml_sample: top_k must be [rows] of int32 or int64");
  FML_REQUIRE(!top_p || (float_tensor(top_p, 1) && per_row(top_p)), FML_BAD_ARG, "fml_sample: top_p must be [rows] of fp32");
  FML_REQUIRE(!min_p || (float_tensor(min_p, 1) && per_row(min_p)), FML_BAD_ARG, "fml_sample: min_p must be [rows] of fp32");
  FML_REQUIRE(index_tensor(tokens, 1) && per_row(tokens), FML_BAD_ARG, "fml_sample: tokens must be [rows] of int32 or int64");
  FML_REQUIRE(!probabilities || (float_tensor(probabilities, 1) && per_row(probabilities)), FML_BAD_ARG,
              "fml_sample: probabilities must be [rows] of fp32");
  FML_REQUIRE(elements_apart(tokens) && (!probabilities || elements_apart(probabilities)), FML_BAD_ARG, "fml_sample: an output has a stride of 0");
  FML_REQUIRE(vocab >= 1 && vocab <= (1 << 18), FML_UNSUPPORTED, "fml_sample: 1 to %d tokens", 1 << 18);
  if (rows == 0) return FML_OK;
  FML_REQUIRE(inputs_on_current_device({logits, uniform, temperature, top_k, top_p, min_p}), FML_BAD_ARG,
              "fml_sample: an input is not memory of the current device");
  FML_REQUIRE(on_current_device(tokens->data) && (!probabilities || on_current_device(probabilities->data)), FML_BAD_ARG,
              "fml_sample: an output is not memory of the current device");
  SampleArgs a;
  memset(&a, 0, sizeof(a));
  auto floats = [](const fml_tensor *t, const float **p, int64_t *s) { if (t) { *p = static_cast<const float *>(t->data); *s = t->stride[0]; } };
  floats(uniform, &a.uniform, &a.uniform_s);
  floats(temperature, &a.temperature, &a.temperature_s);
  floats(top_p, &a.top_p, &a.top_p_s);
  floats(min_p, &a.min_p, &a.min_p_s);
  a.top_k = index_view(top_k);
  a.logits = logits->data;
  a.rows = rows; a.row_stride = logits->stride[0]; a.col_stride = logits->stride[1];
  a.vocab = (int)vocab;
  a.tokens = tokens->data; a.tokens_s = tokens->stride[0]; a.tokens_wide = tokens->dtype == FML_I64;
  if (probabilities) { a.probabilities = static_cast<float *>(probabilities->data); a.probabilities_s = probabilities->stride[0]; }
  const int64_t v = 16 / (int64_t)data_size(logits->dtype);
  a.vec = a.col_stride == 1 && (rows == 1 || a.row_stride % v == 0) && aligned16(a.logits);
  if (logits->dtype == FML_F32) return launch<float>(a, as_stream(stream));
  if (logits->dtype == FML_F16) return launch<__half>(a, as_stream(stream));
  return launch<__nv_bfloat16>(a, as_stream(stream));
}
