// Attention on warp-wide matrix instructions, shared by attention_rules.cu and attention_tree.cu: a warp owns 16 rows, whose
// queries, running maximum, sum and context stay in its registers, and takes keys and values from tiles in shared memory.
//
//   s = q k^T;  p = 2^(s - m);  l = l + sum p;  o = o + p v;  l and o times 2^(m - m') where m moves to m'
//
// 16-bit types: m16n8k16 with fp32 sums; p is rounded to the type (half a step of a weight, as the values carry), its sum is
// not.  fp32: every operand is split into two TF32 numbers, hi + lo to 2^-22, and three products of four are kept.
#pragma once
#include "serving_common.cuh"
#include "tc_common.cuh"

namespace fml {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool valid) {  // zeros when not valid
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t *r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t *r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T> __device__ __forceinline__ void mma16(float *d, const uint32_t *a, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16<__half>(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16<__nv_bfloat16>(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8_tf32(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void split_tf32(float x, uint32_t &hi, uint32_t &lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  const float rest = x - __uint_as_float(hi);
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(rest));
}
// fp16 weights, and the sums with them, are 2^7 times as large: up to 2^15 (they reach 2^8, since the reference follows the maximum by
// steps of more than 8), so that a small one is held to 2^-32 of the largest where it would be to 2^-25, half a step of the smallest
// numbers.  That counts where small weights meet values far above the others'.  (bf16 has fp32's range.)
template <typename T> constexpr float kLiftOf = 0.0f;
template <> constexpr float kLiftOf<__half> = 7.0f;
template <typename T> __device__ __forceinline__ uint32_t pack2(float x, float y);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Tiles in shared memory and products with them.  DP: the head size the tiles are laid out for (features from the real one on
// are zeros).  at(row, chunk): byte offset of 16 bytes of a row of a K (or Q) tile; at_v: of a V tile.
// HELD (16-bit types): the queries stay in registers; else they are read again for every tile, which leaves room for twice the
// warps.
template <typename T, int DP, bool HELD> struct Flash {
  static constexpr int kChunk = 8, kChunks = DP / 8, kPitch = DP * 2 + 16, kPitchV = kPitch;
  static constexpr float kLift = kLiftOf<T>, kUnlift = kLift > 0.0f ? 1.0f / 128.0f : 1.0f;  // 2^-kLift
  struct Q { uint32_t r[HELD ? DP / 16 : 1][4]; };
  // rows are 16 bytes longer than their features: a matrix load of 8 rows meets 8 different bank groups
  __device__ __forceinline__ static uint32_t at(int row, int chunk) { return (uint32_t)(row * kPitch + (chunk << 4)); }
  __device__ __forceinline__ static uint32_t at_v(int row, int chunk) { return at(row, chunk); }
  __device__ __forceinline__ static void load_q(Q &q, uint32_t tile, int row0) {
    const int lane = threadIdx.x & 31;
    if (HELD)
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) ldmatrix4(tile + at(row0 + (lane & 15), 2 * k + (lane >> 4)), q.r[HELD ? k : 0]);
  }
  template <int NT> __device__ __forceinline__ static void scores(float (&s)[NT][4], const Q &q, uint32_t q_tile, int row0, uint32_t tile, int key0) {
    static_assert(NT % 2 == 0, "two groups of eight keys per matrix load");
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      uint32_t a[4];
      if (!HELD) ldmatrix4(q_tile + at(row0 + (lane & 15), 2 * k + (lane >> 4)), a);
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        uint32_t b[4];
        ldmatrix4(tile + at(key0 + n * 8 + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)), b);
        mma16<T>(s[n], HELD ? q.r[HELD ? k : 0] : a, b[0], b[1]);
        mma16<T>(s[n + 1], HELD ? q.r[HELD ? k : 0] : a, b[2], b[3]);
      }
    }
  }
  // o = o * keep + p v
  template <int NT>
  __device__ __forceinline__ static void context(float (&o)[DP / 8][4], const float (&keep)[2], const float (&p)[NT][4], uint32_t tile, int key0) {
    const int lane = threadIdx.x & 31;
    if (__any_sync(0xffffffffu, keep[0] != 1.0f || keep[1] != 1.0f)) {  // (most tiles leave the maximum as it is)
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) { o[n][0] *= keep[0]; o[n][1] *= keep[0]; o[n][2] *= keep[1]; o[n][3] *= keep[1]; }
    }
#pragma unroll
    for (int k = 0; k < NT / 2; ++k) {
      const uint32_t a[4] = {pack2<T>(p[2 * k][0], p[2 * k][1]), pack2<T>(p[2 * k][2], p[2 * k][3]), pack2<T>(p[2 * k + 1][0], p[2 * k + 1][1]),
                             pack2<T>(p[2 * k + 1][2], p[2 * k + 1][3])};
#pragma unroll
      for (int n = 0; n < DP / 8; n += 2) {
        uint32_t b[4];
        ldmatrix4_trans(tile + at(key0 + k * 16 + (lane & 15), n + (lane >> 4)), b);
        mma16<T>(o[n], a, b[0], b[1]);
        mma16<T>(o[n + 1], a, b[2], b[3]);
      }
    }
  }
};

template <int DP, bool HELD> struct Flash<float, DP, HELD> {
  // rows are padded so that the loads below meet every bank once: K by pairs of features, V by single ones
  static constexpr int kChunk = 4, kChunks = DP / 4, kPitch = (DP + 8) * 4, kPitchV = (DP + 4) * 4;
  static constexpr float kLift = kLiftOf<float>, kUnlift = 1.0f;
  struct Q {};  // (hi and lo of 16 x DP queries would fill the registers: read again for every tile)
  __device__ __forceinline__ static uint32_t at(int row, int chunk) { return (uint32_t)(row * kPitch + (chunk << 4)); }
  __device__ __forceinline__ static uint32_t at_v(int row, int chunk) { return (uint32_t)(row * kPitchV + (chunk << 4)); }
  __device__ __forceinline__ static void load_q(Q &, uint32_t, int) {}
  __device__ __forceinline__ static float2 pair(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
  }
  __device__ __forceinline__ static float one(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
  }
  // k index t of an instruction is feature 2 t of its eight, t + 4 is 2 t + 1 (the order of a sum is free).  The tensor cores cut what
  // they add to an accumulator, 2^-25 of it on average: products with a low half go to one of their own, which stays small, and those
  // of the high halves are summed 32 features at a time and added in rounded steps.  One accumulator for all was off by up to seven times
  // a plain fp32 form; this is 0.6 to 1.6 times as far off as that (one head of 128: 1.1e-6 -> 2.1e-7), in the same time.
  template <int NT>
  __device__ __forceinline__ static void scores(float (&s)[NT][4], const Q &, uint32_t q_tile, int row0, uint32_t tile, int key0) {
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
    const uint32_t qa = q_tile + (uint32_t)((row0 + g) * kPitch + t * 8), ka = tile + (uint32_t)((key0 + g) * kPitch + t * 8);
    float small[NT][4];  // products with a low half
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) small[n][i] = 0.0f;
#pragma unroll (DP == 64 ? 2 : 1)
    for (int k0 = 0; k0 < DP / 8; k0 += 4) {
      float sum[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[n][i] = 0.0f;
#pragma unroll
      for (int k = k0; k < k0 + 4; ++k) {
        const float2 q0 = pair(qa + k * 32), q1 = pair(qa + k * 32 + 8 * kPitch);
        uint32_t hi[4], lo[4];
        split_tf32(q0.x, hi[0], lo[0]);
        split_tf32(q1.x, hi[1], lo[1]);
        split_tf32(q0.y, hi[2], lo[2]);
        split_tf32(q1.y, hi[3], lo[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float2 b = pair(ka + n * 8 * kPitch + k * 32);
          uint32_t bh[2], bl[2];
          split_tf32(b.x, bh[0], bl[0]);
          split_tf32(b.y, bh[1], bl[1]);
          mma8_tf32(small[n], lo, bh[0], bh[1]);
          mma8_tf32(small[n], hi, bl[0], bl[1]);
          mma8_tf32(sum[n], hi, bh[0], bh[1]);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] += sum[n][i];
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] += small[n][i];
  }
  // o = o * keep + p v.  A tile's (half a tile's) products are summed apart and added in one rounded step: the tensor cores cut
  // what they add to an accumulator, and one accumulator over all keys was off by six times as much.
  template <int NT>
  __device__ __forceinline__ static void context(float (&o)[DP / 8][4], const float (&keep)[2], const float (&p)[NT][4], uint32_t tile, int key0) {
    constexpr int kPart = NT < 4 ? NT : 4;
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
    const uint32_t va = tile + (uint32_t)((key0 + 2 * t) * kPitchV + g * 4);
#pragma unroll
    for (int k0 = 0; k0 < NT; k0 += kPart) {
      uint32_t hi[kPart][4], lo[kPart][4];
#pragma unroll
      for (int k = 0; k < kPart; ++k) {
        split_tf32(p[k0 + k][0], hi[k][0], lo[k][0]);
        split_tf32(p[k0 + k][2], hi[k][1], lo[k][1]);
        split_tf32(p[k0 + k][1], hi[k][2], lo[k][2]);
        split_tf32(p[k0 + k][3], hi[k][3], lo[k][3]);
      }
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) {
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < kPart; ++k) {
          uint32_t bh[2], bl[2];
          split_tf32(one(va + (k0 + k) * 8 * kPitchV + n * 32), bh[0], bl[0]);
          split_tf32(one(va + (k0 + k) * 8 * kPitchV + n * 32 + kPitchV), bh[1], bl[1]);
          mma8_tf32(sum, lo[k], bh[0], bh[1]);
          mma8_tf32(sum, hi[k], bl[0], bl[1]);
          mma8_tf32(sum, hi[k], bh[0], bh[1]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = k0 == 0 ? fmaf(o[n][i], keep[i >> 1], sum[i]) : o[n][i] + sum[i];
      }
    }
  }
};

// The two rows of a thread: lane / 4 and lane / 4 + 8 of the warp's 16.
template <int DP> struct Running {
  float o[DP / 8][4], m[2], l[2];  // o and l times 2^kLift; m (what p refers to), and the scores, in units of ln 2; -infinity before the first visible key
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.0f;
  }
};

// One tile's keys key0 .. key0 + 8 NT - 1.  shape(s): scores in units of ln 2 in place of q . k, -infinity for keys not seen.
template <typename F, int DP, int NT, typename S>
__device__ __forceinline__ void flash_step(Running<DP> &r, const typename F::Q &q, uint32_t q_tile, int row0, uint32_t k_tile, uint32_t v_tile,
                                           int key0, S shape) {
  float s[NT][4];
  F::template scores<NT>(s, q, q_tile, row0, k_tile, key0);
  shape(s);
  float keeps[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float m = fmaxf(s[0][2 * h], s[0][2 * h + 1]);
#pragma unroll
    for (int n = 1; n < NT; ++n) m = fmaxf(m, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    // the reference moves only for a score that exceeds it by more than 8: weights reach 2^8, and the context is seldom rescaled
    float keep = 1.0f;
    if (m > (r.m[h] == -INFINITY ? -3.402823466e38f : r.m[h] + 8.0f)) {
      keep = ex2_approx(r.m[h] - m);
      r.m[h] = m;
    }
    const float base = (r.m[h] == -INFINITY ? 0.0f : r.m[h]) - F::kLift;  // (no key so far: every p below is 2^-infinity)
    float sum = 0.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      s[n][2 * h] = ex2_approx(s[n][2 * h] - base);
      s[n][2 * h + 1] = ex2_approx(s[n][2 * h + 1] - base);
      sum += s[n][2 * h] + s[n][2 * h + 1];
    }
    r.l[h] = r.l[h] * keep + sum;  // (this thread's keys: the four lanes of a row are added up at the end)
    keeps[h] = keep;
  }
  F::template context<NT>(r.o, keeps, s, v_tile, key0);
}

// cap * tanh(s / cap) in units of ln 2, s = x * inv_divisor.
struct Cap {
  float scale, cap;  // without a cap scale = log2(e) / divisor; with one scale = 1 / (divisor cap), cap in units of ln 2
  __host__ static Cap make(float divisor, float cap) {
    Cap c;
    c.cap = cap > 0.0f ? cap * kLog2e : 0.0f;
    c.scale = cap > 0.0f ? 1.0f / (divisor * cap) : kLog2e / divisor;
    return c;
  }
};
// Whether the kernels' factors are normal fp32 numbers (an overflow or a flush to zero would make every score the same, or NaN).  A cap
// within 2^64 of one leaves room for the factors that packed pairs put before it.
inline bool factors_in_range(float divisor, float cap) {
  auto normal = [](double x) { return x >= 1.1754943508222875e-38 && x <= 3.4028234663852886e38; };
  const double inv = 1.0 / (divisor < 0 ? -(double)divisor : (double)divisor);
  return normal(inv) && normal(inv * kLog2e) && (cap == 0.0f || (cap >= 0x1p-64f && cap <= 0x1p64f && normal(inv / cap)));
}
template <bool EXACT> __device__ __forceinline__ float tanh_of(float x) {
  if (EXACT) return tanhf(x);
  // 1 - 2 / (e^2x + 1): 1e-7 of the whole, where 16-bit weights carry 2^-9 and more
  return 1.0f - __fdividef(2.0f, ex2_approx(x * (2.0f * kLog2e)) + 1.0f);
}
// Products -> scores in units of ln 2, bias and mask apart.
template <bool EXACT, int NT> __device__ __forceinline__ void cap_scores(const Cap &cap, float (&s)[NT][4]) {
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) s[n][i] *= cap.scale;
  if (!(cap.cap > 0.0f)) return;
  float far = 0.0f;
  if (!EXACT) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) far = fmaxf(far, fabsf(s[n][i]));
  }
  if (!EXACT && __all_sync(0xffffffffu, far <= 1.0f)) {
    // tanh(x) = x P(x^2) on [-1, 1]: least squares reweighted to the smallest largest error, 2.4e-7
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = s[n][i], u = x * x;
        float p = fmaf(u, -0.00283947f, 0.01611418f);
        p = fmaf(u, p, -0.05097286f);
        p = fmaf(u, p, 0.13253525f);
        p = fmaf(u, p, -0.33324004f);
        p = fmaf(u, p, 0.99999685f);
        s[n][i] = p * (x * cap.cap);
      }
  } else {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = cap.cap * tanh_of<EXACT>(s[n][i]);
  }
}

// The context of one query over those of the keys [key0, key1) that it sees, by a warp which reads no others: for rows that what
// they do not see has made infinite or NaN.  `at`: key -> whether it is seen, its rows of k and v, what its score loses.  Eight lanes to a
// product, four products at a time; the features lane, lane + 32, ... of the context stay in o, undivided.  It stops once nothing
// but NaN can come of it (l is NaN then): 32 causal heads of 2048 x 128 full of NaN 1.1 ms, where finite ones take 0.1 and
// one infinity that all later rows do see takes 48.
template <typename T, typename F>
__device__ __forceinline__ void context_of_seen(const T *q, int64_t q_d, int64_t k_d, int64_t v_d, int D, const Cap &cap, int key0, int key1,
                                                const F &at, float (&o)[4], float &m, float &l) {
  const int lane = threadIdx.x & 31;
  m = -INFINITY;
  l = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = 0.0f;
  for (int from = key0; from < key1; from += 32) {
    const T *k = nullptr, *v = nullptr;
    float less = 0.0f, s = -INFINITY;
    const bool seen = from + lane < key1 && at(from + lane, &k, &v, &less);
    unsigned left = __ballot_sync(0xffffffffu, seen);
    if (!left) continue;
#pragma unroll 2
    for (int r = 0; r < 8; ++r) {
      const int of = 4 * r + (lane >> 3);
      const T *row = reinterpret_cast<const T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(k), of));
      float x = 0.0f;
      if (left >> of & 1u)
        for (int d = lane & 7; d < D; d += 8) x = fmaf(to_f32(q[d * q_d]), to_f32(row[d * k_d]), x);
#pragma unroll
      for (int w = 4; w; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
      const float got = __shfl_sync(0xffffffffu, x, (lane & 3) * 8);  // of key 4 r + lane % 4
      if (lane >> 2 == r) s = got;
    }
    s *= cap.scale;
    if (cap.cap > 0.0f) s = cap.cap * tanhf(s);
    s = seen ? s - less : -INFINITY;
    float top = s;
#pragma unroll
    for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    top = fmaxf(top, m);
    const float base = top == -INFINITY ? 0.0f : top, keep = ex2_approx(m - base), p = seen ? ex2_approx(s - base) : 0.0f;
    float sum = p;
#pragma unroll
    for (int w = 16; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    m = top;
    l = l * keep + sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] *= keep;
#pragma unroll 2
    for (; left; left &= left - 1) {
      const int of = __ffs(left) - 1;
      const T *row = reinterpret_cast<const T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(v), of));
      const float f = __shfl_sync(0xffffffffu, p, of);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < D) o[i] = fmaf(f, to_f32(row[(lane + 32 * i) * v_d]), o[i]);
    }
    bool lost = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) lost = lost && (lane + 32 * i >= D || o[i] != o[i]);
    if (__all_sync(0xffffffffu, lost)) l = NAN;
    if (l != l) break;
  }
}

}  // namespace fml
