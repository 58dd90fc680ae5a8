// fml_attention_rules on the fifth-generation tensor cores: fp16 and bf16, head sizes that are multiples of 16.
//
// One CTA per SM takes 256 queries of a head as two tiles of 128 rows, A and B, against the same tiles of 128 keys.  Scores and
// contexts are accumulators in tensor memory (all 512 columns of it); weights go back over their scores, in the operands' type, as
// the A operand of the second product.
//
//   warps 0-7, 8-15  softmax of tile A, B: thread = query = lane of tensor memory, and 64 of the 128 keys: two threads share a
//                    query, and tell each other its largest score
//   warp 16          loads (tensor maps, 128-byte swizzle): Q once, K and V tiles into two stages each (four at head size 64)
//   warp 17          products (weights apart, see TcShape: whichever can go next): while one tile's softmax runs, the tensor cores
//                    work for the other
//   (warps 18, 19    make up the last group of four, which gives registers to the softmax: 512 x 104 + 128 x 64 = 640 x 96, what the
//                    launch has)
//
// What bounds it.  A tile of 128 x 128 is 512 clocks of tensor core for either product at head size 128 (256 at 64) and 16384
// exponentials at 16 a clock, 1024: per pair of products as much as they take at head size 128, twice as much at 64.  A capped
// score by two more such instructions would triple that, so tanh is a polynomial on packed pairs (below).  Measured:
// 4 x 16 heads of 2048 x 64 (fp16, bias, prefix) 105 us, 375 TFLOP/s of visible pairs; 32 heads of 8191 x 128 in five documents (bf16,
// capped) 377 us, 432.  Neither pipe is full (tensor 20 to 30 %): a tile's softmax is a chain of phases that its eight warps go
// through together, and a CTA that sees four or five tiles of keys spends a fifth of its time beginning and ending.
//
// A context is one accumulator over all keys, and the tensor cores cut what they add, by 2^-25 of the context on average: 1.5e-5 of it
// over 8192 keys, 2.4e-4 over 131072, beside the half step of 2^-11 (2^-8) that each weight and the result are rounded by.
//
// The running maximum follows only when a tile's exceeds it by more than 8 (in units of ln 2): weights then reach 2^8, which the
// sums carry, and the context's correction, a round trip through registers, is rare.  The commit that publishes S(j) also covers
// PV(j - 1), issued before it, so that the correction needs no barrier of its own (weights apart, S(j) may come first: the softmax
// waits for PV(j - 1) before it writes the next weights or corrects).
#include "attention_rules.cuh"
#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

namespace fml {
namespace {

constexpr int kThreads = 640, kRows = 128, kKeys = 128, kHalf = 64, kMaxTiles = 2048;
constexpr uint32_t kColS = 0, kColO = 256;  // columns of tensor memory

struct TcBarriers {  // offsets of 8 bytes
  enum { kQ = 0, kKFull = 2, kKEmpty = 6, kVFull = 10, kVEmpty = 14, kS = 18, kSFree = 20, kP = 22, kPV = 24, kDone = 26, kDrain = 27, kCount = 28 };
};

template <int DP> struct TcShape {
  static constexpr int kTile = 128 * DP * 2;  // bytes of 128 rows
  static constexpr int kBoxes = DP / 64;      // of 64 features: 128 bytes, one swizzle row
  // Head sizes up to 64 leave room in tensor memory for weights beside the scores: the next tile's scores are then computed as
  // soon as the softmax has read these.
  static constexpr bool kApart = DP == 64;
  static constexpr uint32_t kStepO = kApart ? 64 : 128, kColP = kApart ? 384 : kColS, kStepP = kApart ? 64 : 128, kHalfP = kApart ? 32 : 64;
  static constexpr int kStages = kApart ? 4 : 2;
  static constexpr size_t kBytes = (2 + 2 * kStages) * kTile + 16 * kHalf * 4 + 8 * kRows * 4 + kMaxTiles + TcBarriers::kCount * 8 + 16 + 16 * 4;
};

__device__ __forceinline__ void tmem_ld32_start(uint32_t taddr, float *v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
        "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]),
        "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]),
        "=f"(v[30]), "=f"(v[31])
      : "r"(taddr) : "memory");
}
// The values pass through the wait, so that nothing that uses them is moved in front of it.
__device__ __forceinline__ void tmem_ld_tie(float *v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]),
                 "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]),
                 "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]),
                 "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
               :: "memory");
}

// Two fp32 operations per instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// The tiles of keys that a role works on, in order: f(tile, its views) for tiles whose views have a bit of `mask`, until f says
// false.  By whole warps: 32 tiles are looked at together (one by one, those that a late document skips took thousands of clocks).
template <typename F> __device__ __forceinline__ void each_tile(const uint8_t *views, int tiles, int mask, F f) {
  for (int first = 0; first < tiles; first += 32) {
    const int i = first + (int)(threadIdx.x & 31);
    const int mine = i < tiles ? views[i] : 0;
    unsigned left = __ballot_sync(0xffffffffu, (mine & mask) != 0);
    while (left) {
      const int j = __ffs(left) - 1;
      left &= left - 1;
      if (!f(first + j, __shfl_sync(0xffffffffu, mine, j))) return;
    }
  }
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Instruction descriptor of kind::f16 with fp32 sums: type 0 fp16, 1 bf16; M = 128; B along its columns (1) or along k (0).
__device__ __forceinline__ uint32_t instr_desc_16(uint32_t type, int n, uint32_t b_mn_major) {
  return (1u << 4) | (type << 7) | (type << 10) | (b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// x - base, cut to +-INT_MAX (where it no longer says which).
__device__ __forceinline__ int near_difference(int64_t x, int64_t base) {
  const int64_t d = (int64_t)((uint64_t)x - (uint64_t)base);
  const bool wraps = (x < base) != (d < 0);  // (further apart than 64 bits hold)
  if (wraps) return x < base ? -INT_MAX : INT_MAX;
  return d >= INT_MAX ? INT_MAX : d <= -INT_MAX ? -INT_MAX : (int)d;
}

template <typename T, int DP, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kThreads, 1)
attention_rules_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_o, const __grid_constant__ RulesArgs a) {
  using S = TcShape<DP>;
  using B = TcBarriers;
  extern __shared__ __align__(1024) uint8_t smem[];
  // [ Q of A | Q of B | K stages | V stages | documents of a tile, per softmax warp | largest scores | views | barriers ]
  const uint32_t q_s = smem_u32(smem), k_s = q_s + 2 * S::kTile, v_s = k_s + S::kStages * S::kTile;
  int *const documents = reinterpret_cast<int *>(smem + (2 + 2 * S::kStages) * S::kTile);
  float *const largest = reinterpret_cast<float *>(documents + 16 * kHalf);  // [parity][tile A, B][half of the keys][row]
  uint8_t *const views = reinterpret_cast<uint8_t *>(largest + 8 * kRows);   // [tile]: view of A | view of B << 2
  uint64_t *const bars = reinterpret_cast<uint64_t *>(views + kMaxTiles);
  const uint32_t bar = smem_u32(bars);
  uint32_t *const tmem_slot = reinterpret_cast<uint32_t *>(bars + B::kCount);
  volatile int *const abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  unsigned *const redo_rows = tmem_slot + 2;  // [softmax warp]: rows that are not finite
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const bool leader = elect_one();
  const int head = blockIdx.y, batch = blockIdx.z, kv = head / a.group;
  const int row0 = ((int)gridDim.x - 1 - (int)blockIdx.x) * 2 * kRows;  // (causal: the longest first)
  const bool two = row0 + kRows < a.Sq;

  if (threadIdx.x == 0) {
    tma_prefetch_map(&map_q);
    tma_prefetch_map(&map_k);
    tma_prefetch_map(&map_v);
    for (int i = 0; i < B::kCount; ++i) mbar_init(bar + 8u * i, (i >= B::kP && i < B::kP + 2) || (i >= B::kSFree && i < B::kSFree + 2) ? 8 : 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 17) tmem_alloc(smem_u32(tmem_slot), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();  // (only now: tensor memory)
  pdl_wait();

  if (warp == 16 && leader && g_drop_loads != 1) {
    for (int t = 0; t < (two ? 2 : 1); ++t) {
      mbar_expect_tx(bar + 8u * (B::kQ + t), S::kTile);
      for (int i = 0; i < S::kBoxes; ++i)
        tma_load_4d(q_s + (uint32_t)(t * S::kTile + i * 16384), &map_q, bar + 8u * (B::kQ + t), 64 * i, row0 + t * kRows, a.q_s[1] ? head : 0,
                    a.q_s[0] ? batch : 0);
    }
  }
  __syncwarp();
  // ---- what the two tiles see of each tile of keys
  TileRange ra, rb;
  const int a1 = min(row0 + kRows, a.Sq), b0 = two ? a1 : row0, b1 = two ? min(row0 + 2 * kRows, a.Sq) : a1;
  ra.first_key = last_key_of(a, batch, row0);
  ra.last_key = last_key_of(a, batch, a1 - 1);
  rb.first_key = last_key_of(a, batch, b0);
  rb.last_key = last_key_of(a, batch, b1 - 1);
  const int tiles = (max(ra.last_key, rb.last_key) + kKeys - 1) / kKeys;
  const bool narrow = !a.q_documents.wide && !a.k_documents.wide;
  if (!a.k_documents.p) {
    for (int i = threadIdx.x; i < tiles; i += kThreads)
      views[i] = (uint8_t)(tile_view(ra, i * kKeys, kKeys) | (two ? tile_view(rb, i * kKeys, kKeys) << 2 : 0));
  } else {
    // Documents in 32 bits: as they are, or as differences from the first query's.  All of a warp's loads are in flight together (its four tiles of
    // keys, and the queries), and one width at a time: a choice at every load would put them one after another.
    constexpr int kWarps = kThreads / 32, kAtOnce = 4, kPer = kKeys / 32;
    const int64_t base = narrow ? 0 : document_at(a.q_documents, a.q_documents_row, batch, row0);
    int q_low[2], q_high[2];
    auto scan = [&](auto *qp, auto *kp) {
      using Wide = decltype(*qp + *kp);  // (int for two narrow ones)
      auto cut = [&](Wide x) { return sizeof(Wide) == 4 ? (int)x : near_difference(x, base); };
      qp += batch * a.q_documents_row;
      kp += batch * a.k_documents_row;
      Wide x[2 * kPer];
#pragma unroll
      for (int j = 0; j < 2 * kPer; ++j) x[j] = qp[(j < kPer ? min(row0 + 32 * j + lane, a1 - 1) : min(b0 + 32 * (j - kPer) + lane, b1 - 1)) * a.q_documents.stride];
#pragma unroll 1
      for (int i0 = warp; i0 < tiles || i0 == warp; i0 += kWarps * kAtOnce) {
        Wide y[kAtOnce][kPer];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
#pragma unroll
          for (int j = 0; j < kPer; ++j) y[k][j] = a.Sk > 0 ? kp[min((i0 + k * kWarps) * kKeys + 32 * j + lane, a.Sk - 1) * a.k_documents.stride] : 0;
        if (i0 == warp) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            int low = INT_MAX, high = INT_MIN;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
              const int d = cut(x[t * kPer + j]);
              low = min(low, d);
              high = max(high, d);
            }
            q_low[t] = __reduce_min_sync(0xffffffffu, low);
            q_high[t] = __reduce_max_sync(0xffffffffu, high);
          }
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          const int i = i0 + k * kWarps;
          int low = INT_MAX, high = INT_MIN;
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            const int d = cut(y[k][j]);
            low = min(low, d);
            high = max(high, d);
          }
          low = __reduce_min_sync(0xffffffffu, low);
          high = __reduce_max_sync(0xffffffffu, high);
          auto view_of = [&](const TileRange &r, int t) {
            const int view = tile_view(r, i * kKeys, kKeys);
            if (view == kTileNone || low > q_high[t] || high < q_low[t]) return (int)kTileNone;
            // one document, and not one that the difference was cut at
            const bool same = low == high && q_low[t] == q_high[t] && (narrow || (low != INT_MAX && low != -INT_MAX));
            return !same ? (int)kTileSome : view == kTileAll ? (int)kTileAll : (int)kTileLast;
          };
          if (lane == 0 && i < tiles) views[i] = (uint8_t)(view_of(ra, 0) | (two ? view_of(rb, 1) << 2 : 0));
        }
      }
    };
    if (a.q_documents.wide && a.k_documents.wide) {
      scan(static_cast<const int64_t *>(a.q_documents.p), static_cast<const int64_t *>(a.k_documents.p));
    } else if (a.k_documents.wide) {
      scan(static_cast<const int32_t *>(a.q_documents.p), static_cast<const int64_t *>(a.k_documents.p));
    } else if (a.q_documents.wide) {
      scan(static_cast<const int64_t *>(a.q_documents.p), static_cast<const int32_t *>(a.k_documents.p));
    } else {
      scan(static_cast<const int32_t *>(a.q_documents.p), static_cast<const int32_t *>(a.k_documents.p));
    }
  }
  __syncthreads();

  bool ok = true;
  if (warp >= 16) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  if (warp == 16) {
    // ------------------------------------------------------------ loads
    if (g_drop_loads != 1) {
      int n = 0, n_k = 0;
      each_tile(views, tiles, 15, [&](int i, int) {
        const uint32_t s = (uint32_t)n % S::kStages, free_parity = ((uint32_t)(n / S::kStages) & 1u) ^ 1u;
        ok = mbar_wait_warp(bar + 8u * (B::kKEmpty + s), free_parity, abort_flag);
        if (!ok) return false;
        if (leader) {
          mbar_expect_tx(bar + 8u * (B::kKFull + s), S::kTile);
          for (int b = 0; b < S::kBoxes; ++b)
            tma_load_4d(k_s + s * S::kTile + b * 16384, &map_k, bar + 8u * (B::kKFull + s), 64 * b, i * kKeys, a.k_s[1] ? kv : 0, a.k_s[0] ? batch : 0);
        }
        ++n_k;
        ok = mbar_wait_warp(bar + 8u * (B::kVEmpty + s), free_parity, abort_flag);
        if (!ok) return false;
        if (leader) {
          mbar_expect_tx(bar + 8u * (B::kVFull + s), S::kTile);
          for (int b = 0; b < S::kBoxes; ++b)
            tma_load_4d(v_s + s * S::kTile + b * 16384, &map_v, bar + 8u * (B::kVFull + s), 64 * b, i * kKeys, a.v_s[1] ? kv : 0, a.v_s[0] ? batch : 0);
        }
        ++n;
        return true;
      });
      if (!ok) {  // bounded wait for the loads in flight
        volatile int never = 0;
        for (int t = 0; t < (two ? 2 : 1); ++t) mbar_wait_warp(bar + 8u * (B::kQ + t), 0u, &never);
        for (int j = max(0, n_k - S::kStages); j < n_k; ++j)
          mbar_wait_warp(bar + 8u * (B::kKFull + j % S::kStages), (uint32_t)(j / S::kStages) & 1u, &never);
        for (int j = max(0, n - S::kStages); j < n; ++j)
          mbar_wait_warp(bar + 8u * (B::kVFull + j % S::kStages), (uint32_t)(j / S::kStages) & 1u, &never);
      }
    }
  } else if (warp == 17) {
    // ------------------------------------------------------------ products
    const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    const uint32_t idesc_s = instr_desc_16(type, kKeys, 0u), idesc_o = instr_desc_16(type, a.D, 1u);
    const uint64_t desc_q = smem_desc(q_s, 16u, 1024u), desc_k = smem_desc(k_s, 16u, 1024u), desc_v = smem_desc(v_s, 16384u, 1024u);
    const int steps = a.D / 16;
    ok = mbar_wait_warp(bar + 8u * B::kQ, 0u, abort_flag) && (!two || mbar_wait_warp(bar + 8u * (B::kQ + 1), 0u, abort_flag));
    auto issue_scores = [&](int t, uint32_t stage, bool last) {  // last: nobody needs these keys any more
      if (leader) {
        const uint64_t dq = desc_q + (uint64_t)(t * S::kTile >> 4), dk = desc_k + (uint64_t)(stage * S::kTile >> 4);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          // 32 bytes of a swizzle row per step; four steps to a box
          const uint64_t off = (uint64_t)((k >> 2) * 16384 + (k & 3) * 32) >> 4;
          if (k < steps) umma_f16_ss(tmem + kColS + 128u * t, dq + off, dk + off, idesc_s, k ? 1u : 0u);
        }
        umma_commit(bar + 8u * (B::kS + t));
        if (last) umma_commit(bar + 8u * (B::kKEmpty + stage));
      }
      __syncwarp();
    };
    auto issue_context = [&](int t, uint32_t stage, bool first, bool last) {
      if (leader) {
        const uint64_t dv = desc_v + (uint64_t)(stage * S::kTile >> 4);
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)  // (each half of the keys has its weights in a place of its own)
          umma_f16_ts(tmem + kColO + S::kStepO * t, tmem + S::kColP + S::kStepP * t + S::kHalfP * (k >> 2) + 8u * (k & 3), dv + (uint64_t)(k * 2048 >> 4),
                      idesc_o, first && k == 0 ? 0u : 1u);
        if (S::kApart) umma_commit(bar + 8u * (B::kPV + t));
        if (last) umma_commit(bar + 8u * (B::kVEmpty + stage));
      }
      __syncwarp();
    };
    if constexpr (S::kApart) {
      // Whatever can go next goes next.  Of query tile t: the tile of keys whose scores (values) come next, its number among those that
      // either query tile sees (stages and their phases go by that), and how many there have been.  Tiles below both numbers are done
      // with; one kStages or more above the lower cannot have been loaded, and its stage's phase may be that of an earlier one.
      struct Front { int tile; uint32_t number, count; };
      Front s_at[2], v_at[2];
      auto move = [&](int t, Front &f, bool begin) {  // to the next tile that t sees, `tiles` behind the last
        if (!begin) { ++f.tile; ++f.number; ++f.count; }
        while (f.tile < tiles) {
          const int view = views[f.tile];
          if (view >> (2 * t) & 3) return;
          if (view) ++f.number;
          ++f.tile;
        }
      };
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s_at[t].tile = 0;
        s_at[t].number = s_at[t].count = 0u;
        move(t, s_at[t], true);  // (without a tile B its views are none: its number is behind the last at once)
        v_at[t] = s_at[t];
      }
      uint32_t idle = 0;
      const uint32_t limit = g_wait_limit;
      while (ok && (v_at[0].tile < tiles || v_at[1].tile < tiles)) {
        bool moved = false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (v_at[t].count < s_at[t].count) {  // weights that are awaited
            const uint32_t n = v_at[t].number, stage = n % S::kStages, count = v_at[t].count;
            if (n < min(v_at[0].number, v_at[1].number) + S::kStages && mbar_test_warp(bar + 8u * (B::kP + t), count & 1u) && mbar_test_warp(bar + 8u * (B::kVFull + stage), n / S::kStages & 1u)) {
              tc_fence_after();
              const bool last = !(views[v_at[t].tile] >> (2 * (t ^ 1)) & 3) || v_at[t ^ 1].tile > v_at[t].tile;  // nobody needs these values any more
              issue_context(t, stage, count == 0, last);
              move(t, v_at[t], false);
              moved = true;
            }
          }
          // scores, once the softmax has read the last ones
          const uint32_t count = s_at[t].count;
          if (s_at[t].tile < tiles && (count == 0 || mbar_test_warp(bar + 8u * (B::kSFree + t), (count - 1u) & 1u))) {
            const uint32_t n = s_at[t].number, stage = n % S::kStages;
            if (n < min(s_at[0].number, s_at[1].number) + S::kStages && mbar_test_warp(bar + 8u * (B::kKFull + stage), n / S::kStages & 1u)) {
              tc_fence_after();
              const bool last = !(views[s_at[t].tile] >> (2 * (t ^ 1)) & 3) || s_at[t ^ 1].tile > s_at[t].tile;
              issue_scores(t, stage, last);
              move(t, s_at[t], false);
              moved = true;
            }
          }
        }
        idle = moved ? 0u : idle + 1u;
        if (idle > limit || ((idle & 255u) == 255u && __any_sync(0xffffffffu, *abort_flag))) ok = false;
      }
    } else {
      // Weights over their scores: S_A(j)  PV_B(j-1)  S_B(j)  PV_A(j), one wait after another (asking what is ready, as above, took
      // 399 us for 378 where the order is given anyway).
      uint32_t n = 0, done[2] = {0u, 0u}, wait_b = 0;
      bool pending = false;  // B's product with V of the tile before
      auto context = [&](int t, uint32_t number, bool last) {
        const uint32_t stage = number % S::kStages;
        ok = mbar_wait_warp(bar + 8u * (B::kVFull + stage), number / S::kStages & 1u, abort_flag) &&
             mbar_wait_warp(bar + 8u * (B::kP + t), done[t] & 1u, abort_flag);
        if (!ok) return;
        tc_fence_after();
        issue_context(t, stage, done[t] == 0, last);
        ++done[t];
      };
      if (ok) each_tile(views, tiles, 15, [&](int, int view) {
        const uint32_t stage = n % S::kStages;
        ok = mbar_wait_warp(bar + 8u * (B::kKFull + stage), n / S::kStages & 1u, abort_flag);
        if (!ok) return false;
        tc_fence_after();
        if (view & 3) issue_scores(0, stage, !(view >> 2));
        if (pending) {
          context(1, wait_b, true);
          pending = false;
          if (!ok) return false;
        }
        if (view >> 2) issue_scores(1, stage, true);
        if (view & 3) context(0, n, !(view >> 2));
        if (!ok) return false;
        if (view >> 2) {
          pending = true;
          wait_b = n;
        }
        ++n;
        return true;
      });
      if (ok && pending) context(1, wait_b, true);
    }
    if (ok && leader) umma_commit(bar + 8u * B::kDone);
    if (!ok) *abort_flag = 1;
    if (leader) umma_drain(bar + 8u * B::kDrain);
    __syncwarp();
  }
  } else {
    // ------------------------------------------------------------ softmax: two threads = query
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    const int t = warp >> 3, half = warp >> 2 & 1, local = (warp & 3) * 32 + lane;
    const int i = row0 + t * kRows + local, row = min(i, a.Sq - 1);
    const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16), col_s = lane_addr + kColS + 128u * t + 64u * half,
                   col_p = S::kApart ? lane_addr + S::kColP + S::kStepP * t + S::kHalfP * half : col_s, col_o = lane_addr + kColO + S::kStepO * t;
    const RowRules r = row_rules(a, batch, head, row);
    // wide documents go by their differences from the warp's first, which fit 32 bits unless they are cut (then the keys' own are
    // asked)
    int *const docs = documents + warp * kHalf;
    RowRules r0 = r;
    r0.document = __shfl_sync(0xffffffffu, (long long)r.document, 0);
    const int r_near = narrow ? (int)r.document : near_difference(r.document, r0.document);
    const bool far_documents = __any_sync(0xffffffffu, !narrow && (r_near == INT_MAX || r_near == -INT_MAX));
    float m = -INFINITY, l = 0.0f;
    uint32_t n = 0;
    if (t == 0 || two) {
      // (a warp that gave up goes on through the barriers, so that none is left waiting)
      each_tile(views, tiles, 3 << (2 * t), [&](int tile, int both_views) {
        const int view = both_views >> (2 * t) & 3;
        const int key0 = tile * kKeys + half * kHalf;
        if (ok && view == kTileSome && a.k_documents.p) {
          __syncwarp();
          for (int j = lane; j < kHalf; j += 32) {
            const int64_t x = key0 + j < a.Sk ? document_at(a.k_documents, a.k_documents_row, batch, key0 + j) : r0.document;
            docs[j] = narrow ? (int)x : near_difference(x, r0.document);
          }
          __syncwarp();
        }
        if (ok) ok = mbar_wait_warp(bar + 8u * (B::kS + t), n & 1u, abort_flag);
        float v[kHalf];
        float scale = 1.0f, m_tile = -INFINITY;
        if (ok) {
          tc_fence_after();
          tmem_ld32_start(col_s, v);
          tmem_ld32_start(col_s + 32u, v + 32);
          tmem_ld_tie(v);
          tmem_ld_tie(v + 32);
          if (S::kApart) {  // the next scores may come
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar + 8u * (B::kSFree + t));
          }
          // scores in units of ln 2 (without cap and bias they stay products, scaled on the way into the exponential)
          if (CAP) {
            const float2 f = both(a.cap.scale);
            float far = 0.0f;
#pragma unroll
            for (int j = 0; j < kHalf; j += 2) {
              const float2 x = mul2(make_float2(v[j], v[j + 1]), f);
              v[j] = x.x;
              v[j + 1] = x.y;
              far = fmaxf(far, fmaxf(fabsf(x.x), fabsf(x.y)));
            }
            if (__all_sync(0xffffffffu, far <= 1.0f)) {
              // tanh(x) = x P(x^2) on [-1, 1]: least squares reweighted to the smallest largest error, 2.4e-7
#pragma unroll
              for (int j = 0; j < kHalf; j += 2) {
                const float2 x = make_float2(v[j], v[j + 1]), u = mul2(x, x);
                float2 p = fma2(u, both(-0.00283947f), both(0.01611418f));
                p = fma2(u, p, both(-0.05097286f));
                p = fma2(u, p, both(0.13253525f));
                p = fma2(u, p, both(-0.33324004f));
                p = fma2(u, p, both(0.99999685f));
                p = mul2(p, x);
                v[j] = p.x;
                v[j + 1] = p.y;
              }
            } else {
#pragma unroll
              for (int j = 0; j < kHalf; ++j) v[j] = tanh_of<false>(v[j]);
            }
          }
          scale = CAP ? a.cap.cap : a.cap.scale;
          if (BIAS) {
            const float at = (float)(r.at - key0);
            // a tile that lies on one side of the query: |at - j| is a line
            const bool before = r.at >= key0 + kHalf - 1;
            if (__all_sync(0xffffffffu, before || r.at <= key0)) {
              // (stepped by eight keys in four chains: pairs of constants would cost two moves each)
              const float slope = before ? r.slope : -r.slope, start = -slope * at;
              const float2 step = both(8.0f * slope);
              float2 bias[4];
#pragma unroll
              for (int c = 0; c < 4; ++c) bias[c] = make_float2(fmaf(slope, (float)(2 * c), start), fmaf(slope, (float)(2 * c + 1), start));
#pragma unroll
              for (int j = 0; j < kHalf; j += 2) {
                const float2 x = fma2(make_float2(v[j], v[j + 1]), both(scale), bias[(j >> 1) & 3]);
                v[j] = x.x;
                v[j + 1] = x.y;
                bias[(j >> 1) & 3] = add2(bias[(j >> 1) & 3], step);
              }
            } else {
#pragma unroll
              for (int j = 0; j < kHalf; ++j) v[j] = fmaf(-r.slope, fabsf(at - (float)j), v[j] * scale);
            }
            scale = 1.0f;
          } else if (!(scale > 0.0f)) {  // (a negative divisor: the largest score is the smallest product)
#pragma unroll
            for (int j = 0; j < kHalf; ++j) v[j] *= scale;
            scale = 1.0f;
          }
          if (view != kTileAll) {
            const int last = r.last - key0;
            if (view == kTileSome && a.k_documents.p) {
#pragma unroll
              for (int j = 0; j < kHalf; j += 4) {
                const int4 d = *reinterpret_cast<const int4 *>(docs + j);
                if (j >= last || d.x != r_near) v[j] = -INFINITY;
                if (j + 1 >= last || d.y != r_near) v[j + 1] = -INFINITY;
                if (j + 2 >= last || d.z != r_near) v[j + 2] = -INFINITY;
                if (j + 3 >= last || d.w != r_near) v[j + 3] = -INFINITY;
              }
              if (far_documents) {
#pragma unroll
                for (int j = 0; j < kHalf; ++j)
                  if (key0 + j < a.Sk && document_at(a.k_documents, a.k_documents_row, batch, key0 + j) != r.document) v[j] = -INFINITY;
              }
            } else {
#pragma unroll
              for (int j = 0; j < kHalf; ++j)
                if (j >= last) v[j] = -INFINITY;
            }
          }
          float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
          for (int j = 4; j < kHalf - 4; j += 8) {
#pragma unroll
            for (int c = 0; c < 4; ++c) top[c] = fmaxf(top[c], fmaxf(v[j + c], v[j + 4 + c]));
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) top[c] = fmaxf(top[c], v[kHalf - 4 + c]);
          m_tile = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
        }
        // the query's largest score of the tile, from both halves
        float *const exchange = largest + ((n & 1u) * 2 + t) * 2 * kRows + local;
        exchange[half * kRows] = m_tile;
        named_barrier_sync(1 + t, 256);
        // (with weights apart the last product may still read the weights, and add to the context)
        if (S::kApart && n > 0 && ok) ok = mbar_wait_warp(bar + 8u * (B::kPV + t), (n - 1u) & 1u, abort_flag);
        if (ok) {
          if (S::kApart) tc_fence_after();
          m_tile = fmaxf(m_tile, exchange[(half ^ 1) * kRows]);
          if (n == 0) {
            m = m_tile;
          } else if (__any_sync(0xffffffffu, m_tile > m + 8.0f)) {
            const float m_new = fmaxf(m, m_tile), f = m_new == -INFINITY ? 1.0f : ex2_approx(m - m_new);
            l *= f;
            m = m_new;
#pragma unroll 1
            for (int c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 16) {
              uint32_t o[16];
              tmem_ld16(col_o + (uint32_t)c, o);
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st16(col_o + (uint32_t)c, o);
            }
          }
          const float2 base = both((m == -INFINITY ? 0.0f : -m) + kLiftOf<T>), s2 = both(scale);
          float2 sum[2] = {both(0.0f), both(0.0f)};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t p[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float2 x = fma2(make_float2(v[32 * c + 2 * j], v[32 * c + 2 * j + 1]), s2, base);
              const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
              sum[j & 1] = add2(sum[j & 1], e);
              p[j] = pack2<T>(e.x, e.y);
            }
            tmem_st16(col_p + 16u * c, p);
          }
          const float2 all = add2(sum[0], sum[1]);
          l += all.x + all.y;
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar + 8u * (B::kP + t));
        } else {
          *abort_flag = 1;
        }
        ++n;
        return true;
      });
      // ---- out = O / l, half of the features each
      float *const exchange = largest + ((n & 1u) * 2 + t) * 2 * kRows + local;
      exchange[half * kRows] = l;
      named_barrier_sync(1 + t, 256);
      l += exchange[(half ^ 1) * kRows];
      if (ok) ok = mbar_wait_warp(bar + 8u * B::kDone, 0u, abort_flag);
      bool bad = false;
      if (ok) {
        tc_fence_after();
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (no key seen: zeros; a NaN of keys not seen is done again below)
        T *const dst = static_cast<T *>(a.out) + batch * a.o_s[0] + head * a.o_s[1] + (int64_t)row * a.o_s[2];
        uint8_t *const staged = smem + t * S::kTile;  // (its queries are done with)
#pragma unroll
        for (int c0 = 0; c0 < DP / 2; c0 += 32) {
          const int c = half * (DP / 2) + c0;
          float o[32];
          if (n > 0) {
            __syncwarp();
            tmem_ld32_start(col_o + (uint32_t)c, o);
            tmem_ld_tie(o);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = 0.0f;
          }
          uint32_t x[16] = {};
          float2 check = both(0.0f);  // 0, or NaN from an infinity or NaN on
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 y = mul2(make_float2(o[j], o[j + 1]), both(inv));
            if (j % 16 == 0 && c + j >= a.D) break;  // (columns that the products do not write)
            check = fma2(y, both(0.0f), check);
            x[j / 2] = pack2<T>(y.x, y.y);
          }
          bad = bad || !(check.x + check.y == 0.0f);
          if (a.o_tma) {
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
              const int chunk = (c + 2 * j) >> 3;  // of 8 features; eight to a box's row, permuted as the map's swizzle does
              *reinterpret_cast<uint4 *>(staged + (chunk >> 3) * 16384 + local * 128 + (((chunk & 7) ^ (local & 7)) << 4)) =
                  make_uint4(x[j], x[j + 1], x[j + 2], x[j + 3]);
            }
          } else if (i < a.Sq) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c + j < a.D) dst[(int64_t)(c + j) * a.o_s[3]] = reinterpret_cast<const T *>(x)[j];
          }
        }
        if (a.o_tma) fence_async_smem();
      }
      const unsigned mine = __ballot_sync(0xffffffffu, bad && i < a.Sq);
      if (lane == 0) redo_rows[warp] = mine;
      named_barrier_sync(1 + t, 256);
      unsigned any = 0u;
#pragma unroll
      for (int w = 0; w < 8; ++w) any |= redo_rows[8 * t + w];
      if (ok && a.o_tma && (warp & 7) == 0 && leader) {
        for (int b = 0; b < S::kBoxes; ++b)
          if (64 * b < a.D)
            asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
                         ::"l"(&map_o), "r"(q_s + (uint32_t)(t * S::kTile + b * 16384)), "r"(64 * b), "r"(row0 + t * kRows), "r"(head), "r"(batch)
                         : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        if (any) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        else asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      }
      if (any) named_barrier_sync(1 + t, 256);  // (both halves of a row are written before it is done again)
      unsigned redo = half == 0 ? redo_rows[warp] | redo_rows[warp + 4] : 0u;
      while (redo) {
        const int which = __ffs(redo) - 1;
        redo &= redo - 1;
        redo_rules_row<T>(a, batch, head, row0 + t * kRows + (warp & 3) * 32 + which);
      }
    }
  }
  if (!ok) {
    if (leader) atomicOr(a.status, kStatusTimeout);
    *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 17) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// [batch][head][row][feature] in boxes of 64 features x 128 rows, zeros outside; dims of stride 0 have extent 1.
int rules_map(CUtensorMap *map, const void *base, int dtype, int64_t d, int64_t rows, const int64_t *s, int64_t heads, int64_t batch) {
  EncodeTiledFn fn = encode_fn();
  FML_REQUIRE(fn, FML_CUDA_ERROR, "fml_attention_rules: cuTensorMapEncodeTiled is not available");
  const int64_t any = (d + 7) / 8 * 8;  // a stride that is valid where the extent is 1
  const bool h = s[1] != 0 && heads > 1, b = s[0] != 0 && batch > 1;
  cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)rows, (cuuint64_t)(h ? heads : 1), (cuuint64_t)(b ? batch : 1)};
  cuuint64_t strides[3] = {(cuuint64_t)(rows > 1 ? s[2] : any) * 2, (cuuint64_t)(h ? s[1] : any) * 2, (cuuint64_t)(b ? s[0] : any) * 2};
  cuuint32_t box[4] = {64, 128, 1, 1}, step[4] = {1, 1, 1, 1};
  CUresult r = fn(map, dtype == FML_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base), dims, strides,
                  box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  FML_REQUIRE(r == CUDA_SUCCESS, FML_CUDA_ERROR, "fml_attention_rules: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return FML_OK;
}

using TcKernel = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const CUtensorMap, const RulesArgs);
template <typename T, int DP> TcKernel tc_kernel(bool cap, bool bias) {
  return cap ? bias ? attention_rules_tc_kernel<T, DP, true, true> : attention_rules_tc_kernel<T, DP, true, false>
             : bias ? attention_rules_tc_kernel<T, DP, false, true> : attention_rules_tc_kernel<T, DP, false, false>;
}

}  // namespace

// Large enough, and laid out for tensor maps: rows of 16-byte multiples, unit stride along the head, strides that do not run
// backwards.
bool attention_rules_tc_eligible(const RulesArgs &a, int dtype) {
  if ((dtype != FML_F16 && dtype != FML_BF16) || a.D % 16 != 0 || !a.q_vec || !a.k_vec || !a.v_vec || a.Sk < 1 || a.Sk > kMaxTiles * kKeys) return false;
  for (const int64_t *s : {a.q_s, a.k_s, a.v_s})
    for (int i = 0; i < 3; ++i)
      if (s[i] < 0 || s[i] >= (1ll << 38) || (i == 2 && s[i] == 0)) return false;
  return a.Sq >= 128 && a.Sk >= 128;
}

int launch_attention_rules_tc(const RulesArgs &args, int dtype, cudaStream_t s) {
  RulesArgs a = args;
  CUtensorMap mq, mk, mv, mo;
  int st = rules_map(&mq, a.q, dtype, a.D, a.Sq, a.q_s, a.heads, a.batch);
  if (st == FML_OK) st = rules_map(&mk, a.k, dtype, a.D, a.Sk, a.k_s, a.heads / a.group, a.batch);
  if (st == FML_OK) st = rules_map(&mv, a.v, dtype, a.D, a.Sk, a.v_s, a.heads / a.group, a.batch);
  // the result leaves through shared memory and a tensor map where its layout allows (a thread's own row, 16 bytes at a time to
  // 32 rows per instruction, cost 9000 clocks of a CTA)
  a.o_tma = a.o_s[3] == 1 && aligned16(a.out);
  for (int i = 0; i < 3; ++i) {
    const int64_t n = i == 0 ? a.batch : i == 1 ? a.heads : a.Sq;
    a.o_tma = a.o_tma && (n == 1 || (a.o_s[i] > 0 && a.o_s[i] < (1ll << 38) && a.o_s[i] % 8 == 0));
  }
  mo = mq;
  if (st == FML_OK && a.o_tma) st = rules_map(&mo, a.out, dtype, a.D, a.Sq, a.o_s, a.heads, a.batch);
  if (st != FML_OK) return st;
  const bool cap = a.cap.cap > 0.0f, bias = a.slopes != nullptr;
  const int dp = a.D <= 64 ? 64 : 128;
  const TcKernel kernel = dtype == FML_F16 ? (dp == 64 ? tc_kernel<__half, 64>(cap, bias) : tc_kernel<__half, 128>(cap, bias))
                                           : (dp == 64 ? tc_kernel<__nv_bfloat16, 64>(cap, bias) : tc_kernel<__nv_bfloat16, 128>(cap, bias));
  // 512 columns of tensor memory: a second CTA on the SM would wait for them, so the kernel asks for most of shared memory
  const size_t smem = std::max<size_t>(dp == 64 ? TcShape<64>::kBytes : TcShape<128>::kBytes, 120 * 1024);
  static bool attr_set[64][16] = {};
  int dev = 0;
  FML_CUDA(cudaGetDevice(&dev));
  bool &set = attr_set[dev & 63][(dtype == FML_F16) * 8 + (dp == 64) * 4 + cap * 2 + bias];
  if (!set) {
    FML_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    set = true;
  }
  FML_CUDA(launch_kernel(kernel, dim3((unsigned)((a.Sq + 2 * kRows - 1) / (2 * kRows)), (unsigned)a.heads, (unsigned)a.batch), dim3(kThreads), smem, s,
                         mq, mk, mv, mo, a));
  return FML_OK;
}

}  // namespace fml
