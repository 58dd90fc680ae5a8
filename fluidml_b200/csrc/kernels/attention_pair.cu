// Attention core on pairs of half-precision numbers (gemm_pair.cu): out = softmax(Q K^T / divisor + mask) V
// for head size 64, one CTA per (head, 128 query rows), keys in blocks of 64 with a running softmax.  The
// scores never leave the SM.
//
// What bounds it: the exponentials and operand splits (about 14 instructions per score and 6 per element
// of K and V), not the MMAs (768 clocks per 128 x 64 block against some 1300 issue slots per scheduler), so
// the work is laid out to keep the schedulers busy: separate warps split K and V for the block ahead while
// the softmax warps work on this one, and two CTAs share an SM.  Measured, 192 heads of 384 x 384: 51 us a launch,
// where two batched 3xTF32 GEMMs around a softmax took 163; 64 causal heads of 512: 25 us against 87.
//
//   warp 0      loads (tensor maps, 128-byte swizzle): Q once, K and V of a block into one of two raw stages
//   warp 1      MMAs: S = Q K^T with Q from tensor memory, O += P V with P from tensor memory; order
//               S(0), S(1), PV(0), S(2), PV(1) ..., so that the scores of the next block are computed while
//               the softmax of this one runs
//   warps 2-5   softmax, thread = query row = TMEM lane: scores -> P = exp(s - m), split and written over them
//   warps 6-9   split K and V: unswizzled core matrices [8 k values][row][16 bytes] in shared memory, K as
//               (key, 8 of d), V transposed as (d, 8 keys), so that both are K-major B operands
//
// Scales (powers of two).  Q per row, K and V per block, all from exact finite maxima (largest in [2^14, 2^15):
// 22 bits down to 2^-17 of it, below that an absolute error of 2^-39 of it); Q's and K's are divided out with the attention scale.  P is exp(s - m) times 2^x, x = (scale of O) - (scale of
// this block's V): O is one accumulator.  O is rescaled, by a round trip through registers, only when a
// block's maximum exceeds the reference m of a row by more than 4 in log2 or V's scale moves by more than 3:
// the largest P of a row is then within 2^-3 .. 2^7, and what its pair leaves out is below 2^-22 of it.
#include "attention_rules.cuh"
#include "gemm_common.cuh"
#include "pair_common.cuh"
#include <algorithm>
#include <cfloat>

namespace fml {
namespace {

constexpr int kThreads = 320, kKeys = 64, kD = 64;
constexpr int kRawStage = 2 * kKeys * kD * 4;    // K and V of a block, fp32: 32 KiB (= Q of the tile)
constexpr int kSplit = kKeys * kD * 4;           // hi and lo of K or V: 16 KiB
constexpr int kHalfSplit = kSplit / 2;           // offset of lo
constexpr uint32_t kColS = 0, kColO = 128, kColQ = 192;  // tensor memory: two score buffers (P over S), O, Q
enum { kNoMask = 0, kKeyMask = 1, kFullMask = 2, kCausal = 3, kRules = 4 };
constexpr int kMaxBlocks = 2048;  // of keys, with rules
constexpr int kFold = 4;          // (rules) blocks of keys that one accumulator takes
// (rules) P and the sums are 2^8 times as large, up to 2^15: a weight is held to 2^-33 of the row's largest where it would be to 2^-25, half
// a step of the smallest half-precision numbers.  That counts where small weights meet values far above the others'.
constexpr int kLift = 8;
struct NoRules {};

struct AttnPairArgs {
  int Sq, Sk, nb0;
  int q_h, q_b, k_h, k_b, v_h, v_b;  // whether the operand varies over heads / batches
  const float *mask;
  int64_t m_s[4], o_s[4];
  float *out;
  float inv_divisor, cap;
  int *status;
};

// Contexts that wait in the output while their accumulator takes other keys (rules): of a warp's 32 rows, row0 on, out = out * keep +
// O * scale, and back, O = O + out * keep.  Where all 32 rows are there they wait in an order of their own, in which a warp's 16 bytes to a
// thread are two rows from end to end: with every thread in its own row, 4 bytes at a time, a fold of all rows of 4 x 16 x 512 took 20 us.
// Functions of their own, so that the loop over the keys keeps its registers.
struct Folded {
  float *at;
  int64_t step;  // from one 16 bytes to the next of a thread's (0: by single features)
  bool there;
};
__device__ __forceinline__ Folded folded_at(const AttnPairArgs &a, int b, int h, int row0) {
  const int lane = threadIdx.x & 31;
  Folded f;
  f.at = a.out + (int64_t)b * a.o_s[0] + (int64_t)h * a.o_s[1] + (int64_t)row0 * a.o_s[2];
  f.there = row0 + lane < a.Sq;
  const bool vec = a.o_s[3] == 1 && (a.o_s[2] & 3) == 0 && (reinterpret_cast<uintptr_t>(f.at) & 15) == 0;
  if (vec && row0 + 31 < a.Sq) {
    f.step = 2 * a.o_s[2];
    f.at += (lane >> 4) * a.o_s[2] + 4 * (lane & 15);
  } else {
    f.step = vec ? 4 : 0;
    f.at += (f.there ? lane : 0) * a.o_s[2];
  }
  return f;
}
// All of a thread's 64 features, whose loads are in flight together.
__device__ __forceinline__ void load_folded(const AttnPairArgs &a, const Folded &f, float (&x)[kD]) {
  if (f.step) {
#pragma unroll
    for (int i = 0; i < kD / 4; ++i) {
      const float4 y = f.there ? *reinterpret_cast<const float4 *>(f.at + i * f.step) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      x[4 * i] = y.x; x[4 * i + 1] = y.y; x[4 * i + 2] = y.z; x[4 * i + 3] = y.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kD; ++i) x[i] = f.there ? f.at[i * a.o_s[3]] : 0.0f;
  }
}
__device__ __noinline__ void fold_out(const AttnPairArgs &a, int b, int h, int row0, uint32_t col_o, bool more, float keep, float scale) {
  const Folded f = folded_at(a, b, h, row0);
  float x[kD];
  if (more) {
    load_folded(a, f, x);
  } else {
#pragma unroll
    for (int i = 0; i < kD; ++i) x[i] = 0.0f;
  }
  __syncwarp();
#pragma unroll
  for (int c = 0; c < kD; c += 16) {
    uint32_t o[16];
    tmem_ld16(col_o + (uint32_t)c, o);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[c + i] = fmaf(x[c + i], keep, __uint_as_float(o[i]) * scale);
  }
  if (!f.there) {
  } else if (f.step) {
#pragma unroll
    for (int i = 0; i < kD / 4; ++i)
      *reinterpret_cast<float4 *>(f.at + i * f.step) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < kD; ++i) f.at[i * a.o_s[3]] = x[i];
  }
  __syncwarp();
}
__device__ __noinline__ void fold_in(const AttnPairArgs &a, int b, int h, int row0, uint32_t col_o, float keep) {
  const Folded f = folded_at(a, b, h, row0);
  float x[kD];
  load_folded(a, f, x);
  __syncwarp();
#pragma unroll
  for (int c = 0; c < kD; c += 16) {
    uint32_t o[16];
    tmem_ld16(col_o + (uint32_t)c, o);
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(fmaf(x[c + i], keep, __uint_as_float(o[i])));
    tmem_st16(col_o + (uint32_t)c, o);
  }
  tmem_wait_st();
  __syncwarp();  // (the warp's rows are read: now they may be written)
}

// With rules (fml_attention_rules): the blocks of keys that some query of the tile sees are listed first, heads share keys and values
// in groups, scores are capped, biased and masked as attention_rules.cuh says, and rows that see nothing are zero.  The tensor
// cores cut what they add to an accumulator, 2^-25 of it on average by every instruction and always downwards: every kFold blocks the context
// moves to the output, in fp32, and begins anew.  4 x 16 heads of 512, prefix, against 64 bits (a plain fp32 form is off by 3.9e-7):
// 16 blocks 30 us, 1.18e-6; 4 blocks 32 us, 9.3e-7 (with the small products of scores first 8.5e-7); 2 blocks 37 us, 6.8e-7.  16 heads of 1500, every key seen (plain 7.5e-7): 16 blocks
// 72 us, 3.3e-6; 8 blocks 75 us, 2.0e-6; 4 blocks 83 us, 1.1e-6.
template <int MASK, typename Rules>
__global__ void __launch_bounds__(kThreads, 2)
attention_pair_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnPairArgs a,
                      const __grid_constant__ Rules rules) {
  extern __shared__ __align__(1024) uint8_t smem[];
  // [ raw stage 0 | raw stage 1 | split K | split V | mask | barriers ]
  const uint32_t raw0 = smem_u32(smem), split_k = raw0 + 2 * kRawStage, split_v = split_k + kSplit;
  uint8_t *const split_k_ptr = smem + 2 * kRawStage, *const split_v_ptr = split_k_ptr + kSplit;
  float *const mask_s = reinterpret_cast<float *>(split_v_ptr + kSplit);            // [2][64]
  int *const exp_s = reinterpret_cast<int *>(mask_s + 2 * kKeys);                   // [2][2]: scale exponents of K, V
  unsigned *const max_s = reinterpret_cast<unsigned *>(exp_s + 4);                  // [3][2]: their largest magnitudes
  uint64_t *const bars = reinterpret_cast<uint64_t *>(max_s + 8);
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t bar_raw_full = bar0, bar_raw_empty = bar0 + 16, bar_s = bar0 + 32, bar_q_full = bar0 + 48, bar_q_ready = bar0 + 56,
                 bar_k_ready = bar0 + 64, bar_k_free = bar0 + 72, bar_v_ready = bar0 + 80, bar_p_ready = bar0 + 88, bar_pv = bar0 + 104, bar_final = bar0 + 112;
  uint32_t *const tmem_slot = reinterpret_cast<uint32_t *>(bars + 15);
  volatile int *const abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const bool leader = elect_one();
  const int q0 = (MASK == kRules ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x) * kBM, h = blockIdx.y % a.nb0, b = blockIdx.y / a.nb0;
  uint16_t *const list = reinterpret_cast<uint16_t *>(tmem_slot + 4);  // (rules) [block that is seen]: its index | TileView << 12
  int n_blocks = (a.Sk + kKeys - 1) / kKeys;
  if (MASK == kCausal) n_blocks = min(n_blocks, (q0 + kBM + kKeys - 1) / kKeys);  // keys beyond the tile's last row

  if (threadIdx.x == 0) {
    tma_prefetch_map(&map_q);
    tma_prefetch_map(&map_k);
    tma_prefetch_map(&map_v);
    for (int s = 0; s < 2; ++s) { mbar_init(bar_raw_full + 8u * s, 1); mbar_init(bar_raw_empty + 8u * s, 4); mbar_init(bar_s + 8u * s, 1); mbar_init(bar_p_ready + 8u * s, 4); }
    mbar_init(bar_q_full, 1);
    mbar_init(bar_q_ready, 4);
    mbar_init(bar_k_ready, 4);
    mbar_init(bar_k_free, 1);
    mbar_init(bar_v_ready, 4);
    mbar_init(bar_pv, 1);
    mbar_init(bar_final, 1);
    *abort_flag = 0;
    for (int i = 0; i < 6; ++i) max_s[i] = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_slot), 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // Only now may the next kernel start (tensor memory: see gemm_tc.cu).
  pdl_launch_dependents();
  pdl_wait();
  int kv = h;
  if constexpr (MASK == kRules) {
    kv = h / rules.group;
    const TileRange range = tile_range(rules, b, q0, min(q0 + kBM, a.Sq));
    const int blocks = (range.last_key + kKeys - 1) / kKeys;
    for (int i = warp; i < blocks; i += kThreads / 32) {
      int view = tile_view(range, i * kKeys, kKeys);
      if (rules.k_documents.p) {
        int64_t low, high;
        tile_documents(rules, b, i * kKeys, min(i * kKeys + kKeys, a.Sk), &low, &high);
        view = document_view(view, range, low, high);
      }
      if (lane == 0) list[i] = (uint16_t)view;
    }
    __syncthreads();
    if (warp == 0) {  // (a block's place is not behind its index, and 32 are read before they are written)
      int n = 0;
      for (int i0 = 0; i0 < blocks; i0 += 32) {
        const int view = i0 + lane < blocks ? list[i0 + lane] : (int)kTileNone;
        const unsigned seen = __ballot_sync(0xffffffffu, view != kTileNone);
        __syncwarp();
        if (view != kTileNone) list[n + __popc(seen & ((1u << lane) - 1u))] = (uint16_t)(i0 + lane | view << 12);
        n += __popc(seen);
        __syncwarp();
      }
      if (lane == 0) tmem_slot[2] = (uint32_t)n;
    }
    __syncthreads();
    n_blocks = (int)tmem_slot[2];
  }
  auto block = [&](int j) { return MASK == kRules ? list[j] & 0xfff : j; };

  bool ok = true;
  if (warp == 0) {
    // ------------------------------------------------------------ loads: Q lands in raw stage 1, block j in stage j & 1
    if (g_drop_loads != 1) {
      if (leader) {
        mbar_expect_tx(bar_q_full, kRawStage);
        for (int i = 0; i < 2; ++i)
          tma_load_4d(raw0 + kRawStage + (uint32_t)i * (kBM * 128), &map_q, bar_q_full, 32 * i, q0, a.q_h ? h : 0, a.q_b ? b : 0);
      }
      int issued = 0;
      for (int j = 0; j < n_blocks && ok; ++j) {
        const uint32_t s = (uint32_t)j & 1u, ph = (uint32_t)(j >> 1) & 1u;
        if (j == 1) ok = mbar_wait_warp(bar_q_ready, 0u, abort_flag);  // Q has left its stage
        if (ok) ok = mbar_wait_warp(bar_raw_empty + 8u * s, ph ^ 1u, abort_flag);
        if (!ok) break;
        if (leader) {
          const uint32_t dst = raw0 + s * kRawStage, bar = bar_raw_full + 8u * s;
          mbar_expect_tx(bar, kRawStage);
          for (int i = 0; i < 2; ++i) {
            tma_load_4d(dst + (uint32_t)i * (kKeys * 128), &map_k, bar, 32 * i, block(j) * kKeys, a.k_h ? kv : 0, a.k_b ? b : 0);
            tma_load_4d(dst + (uint32_t)(2 + i) * (kKeys * 128), &map_v, bar, 32 * i, block(j) * kKeys, a.v_h ? kv : 0, a.v_b ? b : 0);
          }
        }
        ++issued;
      }
      if (!ok) {  // bounded drain of the loads in flight
        volatile int never = 0;
        mbar_wait_warp(bar_q_full, 0u, &never);
        for (int j = max(0, issued - 2); j < issued; ++j)
          mbar_wait_warp(bar_raw_full + 8u * ((uint32_t)j & 1u), (uint32_t)(j >> 1) & 1u, &never);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    const uint32_t idesc = instr_desc_f16(64);
    const uint64_t desc_k = smem_desc(split_k, kKeys * 16u, 128u, 0u), desc_v = smem_desc(split_v, kD * 16u, 128u, 0u);
    ok = mbar_wait_warp(bar_q_ready, 0u, abort_flag);
    for (int j = 0; j <= n_blocks && ok; ++j) {
      if (j < n_blocks) {  // scores of block j
        ok = mbar_wait_warp(bar_k_ready, (uint32_t)j & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          const uint32_t d = tmem_base + kColS + ((uint32_t)j & 1u) * 64u;
#pragma unroll
          for (int k = 0; k < kD / 16; ++k) {
            const uint32_t q_hi = tmem_base + kColQ + 8u * k, q_lo = q_hi + 32u;
            const uint64_t kh = desc_k + (uint64_t)(2 * k * (kKeys * 16) >> 4), kl = kh + (uint64_t)(kHalfSplit >> 4);
            umma_f16_ts(d, q_lo, kh, idesc, k ? 1u : 0u);
            umma_f16_ts(d, q_hi, kl, idesc, 1u);
            if (MASK != kRules) umma_f16_ts(d, q_hi, kh, idesc, 1u);
          }
          if (MASK == kRules) {  // (the small products first, while little of the sum is cut)
#pragma unroll
            for (int k = 0; k < kD / 16; ++k)
              umma_f16_ts(d, tmem_base + kColQ + 8u * k, desc_k + (uint64_t)(2 * k * (kKeys * 16) >> 4), idesc, 1u);
          }
          umma_commit(bar_s + 8u * ((uint32_t)j & 1u));
          umma_commit(bar_k_free);
        }
        __syncwarp();
      }
      if (j > 0) {  // context of block j - 1
        const uint32_t ph = (uint32_t)(j - 1) & 1u;
        ok = mbar_wait_warp(bar_v_ready, ph, abort_flag) && mbar_wait_warp(bar_p_ready + 8u * ph, (uint32_t)((j - 1) >> 1) & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          const uint32_t p = tmem_base + kColS + ph * 64u, d = tmem_base + kColO;
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k) {
            const uint32_t p_hi = p + 8u * k, p_lo = p_hi + 32u;
            const uint64_t vh = desc_v + (uint64_t)(2 * k * (kD * 16) >> 4), vl = vh + (uint64_t)(kHalfSplit >> 4);
            umma_f16_ts(d, p_lo, vh, idesc, ((j == 1 || (MASK == kRules && (j - 1) % kFold == 0)) && k == 0) ? 0u : 1u);
            umma_f16_ts(d, p_hi, vl, idesc, 1u);
            umma_f16_ts(d, p_hi, vh, idesc, 1u);
          }
          umma_commit(bar_pv);
        }
        __syncwarp();
      }
    }
    if (!ok) *abort_flag = 1;
    if (leader) umma_drain(bar_final);
    __syncwarp();
  } else if (warp < 6) {
    // ------------------------------------------------------------ softmax: thread = query row
    const int q = warp & 3, row = q * 32 + lane;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(q * 32) << 16);
    const int grow = q0 + row, row_in = min(grow, a.Sq - 1);
    int e_q = 0;
    ok = mbar_wait_warp(bar_q_full, 0u, abort_flag);
    if (ok) {
      float4 x[16];
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 *src = reinterpret_cast<const float4 *>(smem + kRawStage + i * (kBM * 128) + row * 128);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float4 y = src[c ^ (row & 7)];
          x[8 * i + c] = y;
          m = fmaxf(m, fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
        }
      }
      e_q = scale_exponent(m, 14);
      const float s = pow2(e_q);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          split_pair(x[8 * i + c].x, x[8 * i + c].y, s, hi[2 * c], lo[2 * c]);
          split_pair(x[8 * i + c].z, x[8 * i + c].w, s, hi[2 * c + 1], lo[2 * c + 1]);
        }
        tmem_st16(lane_addr + kColQ + 16u * i, hi);
        tmem_st16(lane_addr + kColQ + 32u + 16u * i, lo);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_q_ready);
    }
    float m_ref = 0.0f, l = 0.0f;
    int ev_ref = 0, ev_min = 0, ek_low = 126, ev_low = 126;  // (rules) the scales of the largest keys and values
    RowRules rr;
    if constexpr (MASK == kRules) {
      rr = row_rules(rules, b, h, row_in);
      rr.slope *= 1.0f / kLog2e;  // (scores are in natural units here)
    }
    float m_fold = 0.0f;  // (rules) the reference of the context that the output holds
    for (int j = 0; j < n_blocks && ok; ++j) {
      const uint32_t buf = (uint32_t)j & 1u;
      ok = mbar_wait_warp(bar_s + 8u * buf, (uint32_t)(j >> 1) & 1u, abort_flag);
      if (!ok) break;
      tc_fence_after();
      if constexpr (MASK == kRules) {
        if (j > 0 && j % kFold == 0) {  // out = out + O, and O begins anew with this block
          ok = mbar_wait_warp(bar_pv, (uint32_t)(j - 1) & 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const float keep = j > kFold ? exp2f((m_fold - m_ref) * kLog2e) : 0.0f;
          m_fold = m_ref;
          fold_out(a, b, h, q0 + q * 32, lane_addr + kColO, j > kFold, keep, pow2(-ev_ref));
        }
      }
      const int ev = exp_s[2 * buf + 1];
      const float f = a.inv_divisor * pow2(max(-126, min(126, -(e_q + exp_s[2 * buf]))));
      const int key0 = block(j) * kKeys;
      float v[64];
      tmem_ld32(lane_addr + kColS + buf * 64u, v);
      tmem_ld32(lane_addr + kColS + buf * 64u + 32u, v + 32);
      float m_blk = -FLT_MAX;  // (finite, for blocks without a visible key)
      if constexpr (MASK == kRules) {
        const int view = list[j] >> 12, last = rr.last - key0;
        ek_low = min(ek_low, exp_s[2 * buf]);
        ev_low = min(ev_low, ev);
        if (a.cap > 0.0f) {
          const float g = f / a.cap;
#pragma unroll
          for (int i = 0; i < 64; ++i) v[i] = a.cap * tanhf(v[i] * g);
        } else {
#pragma unroll
          for (int i = 0; i < 64; ++i) v[i] *= f;
        }
        if (rules.slopes) {
          const float at = (float)(rr.at - key0);
#pragma unroll
          for (int i = 0; i < 64; ++i) v[i] = fmaf(-rr.slope, fabsf(at - (float)i), v[i]);
        }
        if (view != kTileAll) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i >= last) v[i] = -INFINITY;
          if (view == kTileSome && rules.k_documents.p) {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (document_at(rules.k_documents, rules.k_documents_row, b, min(key0 + i, a.Sk - 1)) != rr.document) v[i] = -INFINITY;
          }
        }
      } else if (MASK == kKeyMask) {
        const float *mk = mask_s + buf * kKeys;  // keys beyond the last one hold -infinity
#pragma unroll
        for (int i = 0; i < 64; ++i) v[i] = fmaf(v[i], f, mk[i]);
      } else if (MASK == kFullMask) {
        const float *mp = a.mask + (int64_t)b * a.m_s[0] + (int64_t)h * a.m_s[1] + row_in * a.m_s[2] + (int64_t)key0 * a.m_s[3];
#pragma unroll
        for (int i = 0; i < 64; ++i) v[i] = key0 + i < a.Sk ? fmaf(v[i], f, mp[i * a.m_s[3]]) : -INFINITY;
      } else {
        const int last = MASK == kCausal ? min(grow, a.Sk - 1) - key0 : a.Sk - 1 - key0;  // last visible key of the block
        if (__all_sync(0xffffffffu, last >= 63)) {
#pragma unroll
          for (int i = 0; i < 64; ++i) v[i] *= f;
        } else {
#pragma unroll
          for (int i = 0; i < 64; ++i) v[i] = i <= last ? v[i] * f : -INFINITY;
        }
      }
#pragma unroll
      for (int i = 0; i < 64; i += 4) m_blk = fmaxf(m_blk, fmaxf(fmaxf(v[i], v[i + 1]), fmaxf(v[i + 2], v[i + 3])));
      if (j == 0) {
        m_ref = m_blk;
        ev_ref = ev_min = ev;
      } else if (__any_sync(0xffffffffu, m_blk > m_ref + 4.0f / kLog2e) || abs(ev_ref - ev) > 3) {
        // rare: a new maximum out of reach, or a block of V far from those before it
        ok = mbar_wait_warp(bar_pv, (uint32_t)(j - 1) & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const float m_new = fmaxf(m_ref, m_blk), fac_l = exp2f((m_ref - m_new) * kLog2e);
        ev_min = min(ev_min, ev);
        const int ev_new = min(ev, ev_min + 60);  // (keeps O finite; V so small beside an earlier block adds nothing)
        const float fac = fac_l * pow2(max(-126, ev_new - ev_ref));
        l *= fac_l;
        m_ref = m_new;
        ev_ref = ev_new;
#pragma unroll
        for (int c = 0; c < 64; c += 16) {
          uint32_t o[16];
          tmem_ld16(lane_addr + kColO + (uint32_t)c, o);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fac);
          tmem_st16(lane_addr + kColO + (uint32_t)c, o);
        }
        tmem_wait_st();
      }
      const int xi = max(ev_ref - ev, -60);
      const float x = (float)(xi + (MASK == kRules ? kLift : 0));
      float sum = 0.0f;
      uint32_t hi[32], lo[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        // exp(s - m) 2^x; the difference is formed first: the rounding of m log2(e) would show in every score
        const float p0 = ex2_approx(fmaf(v[2 * i] - m_ref, kLog2e, x)), p1 = ex2_approx(fmaf(v[2 * i + 1] - m_ref, kLog2e, x));
        sum += p0 + p1;
        split_pair(p0, p1, 1.0f, hi[i], lo[i]);
      }
      l += sum * pow2(-xi);
      tmem_st32(lane_addr + kColS + buf * 64u, hi);
      tmem_st32(lane_addr + kColS + buf * 64u + 32u, lo);
      tmem_wait_st();
      tc_fence_before();
      // PV's phase must not be two behind at the wait after the loop: the last scores only say that PV(n - 3) is over
      if (j > 0 && j == n_blocks - 1) ok = mbar_wait_warp(bar_pv, (uint32_t)(j - 1) & 1u, abort_flag);
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(bar_p_ready + 8u * buf);  // (two barriers: the softmax may be a block ahead of PV)
    }
    // ---- out = O / l
    if (ok && (MASK != kRules || n_blocks > 0)) ok = mbar_wait_warp(bar_pv, (uint32_t)(n_blocks - 1) & 1u, abort_flag);
    if (ok) {
      tc_fence_after();
      const float inv = MASK == kRules && l == 0.0f ? 0.0f : pow2(-ev_ref) / l;
      bool bad = false;
      float largest = 0.0f;
      if constexpr (MASK == kRules) {
        if (n_blocks > kFold) fold_in(a, b, h, q0 + q * 32, lane_addr + kColO, exp2f((m_fold - m_ref) * kLog2e) * pow2(ev_ref));
      }
      float *dst = a.out + (int64_t)b * a.o_s[0] + (int64_t)h * a.o_s[1] + (int64_t)row_in * a.o_s[2];
      const bool vec = a.o_s[3] == 1 && (a.o_s[2] & 3) == 0 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        float o[32];
        __syncwarp();
        tmem_ld32(lane_addr + kColO + (uint32_t)c, o);
        if constexpr (MASK == kRules) {
          if (n_blocks == 0) {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.0f;
          }
          float check = 0.0f;  // 0, or NaN from an infinity or NaN on
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            check = fmaf(o[i] * inv, 0.0f, check);
            largest = fmaxf(largest, fabsf(o[i] * inv));
          }
          bad = bad || !(check == 0.0f);
        }
        if (grow >= a.Sq) {
        } else if (vec) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4 *>(dst + c + i) = make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) dst[(int64_t)(c + i) * a.o_s[3]] = o[i] * inv;
        }
      }
      if constexpr (MASK == kRules) {
        // A block's scale is that of its largest key and value, and some of them this row may not see.  Values are off by
        // 2^-39 of the largest, in [2^14, 2^15) 2^-ev_low: nothing to a context above 2^-16 of it (an average of N values of
        // random sign is some 2^-(log2 N) / 2).  A score is off by at most 64 |q| |k| 2^-39 / divisor: below 2^-19 where
        // that product of the largest is below 2^20.
        if (l > 0.0f) {
          const bool values = ev_low < 126 && largest < pow2(max(-126, -2 - ev_low));
          const bool keys = ek_low < 126 && 36.0f - (float)(e_q + ek_low) + log2f(fabsf(a.inv_divisor)) > 20.0f;
          bad = bad || values || keys;
        }
        unsigned redo = __ballot_sync(0xffffffffu, bad && grow < a.Sq);
        __syncwarp();
        while (redo) {
          const int which = __ffs(redo) - 1;
          redo &= redo - 1;
          redo_rules_row<float>(rules, b, h, q0 + q * 32 + which);
        }
      }
    }
  } else {
    // ------------------------------------------------------------ split of K and V
    const int t = threadIdx.x - 192, r = t & 63, half = t >> 6;
    for (int j = 0; j < n_blocks; ++j) {
      const uint32_t s = (uint32_t)j & 1u, slot = (uint32_t)j % 3u;
      float4 xk[8];
      float xv[32];
      if (ok) ok = mbar_wait_warp(bar_raw_full + 8u * s, (uint32_t)(j >> 1) & 1u, abort_flag);
      if (ok) {
        // K: key r, d in [32 half, 32 half + 32); V: d = r, keys in [32 half, 32 half + 32)
        const uint8_t *raw = smem + s * kRawStage;
        const float4 *src = reinterpret_cast<const float4 *>(raw + half * (kKeys * 128) + r * 128);
        float mk = 0.0f, mv = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          xk[c] = src[c ^ (r & 7)];
          mk = fmaxf(mk, fmaxf(fmaxf(fabsf(xk[c].x), fabsf(xk[c].y)), fmaxf(fabsf(xk[c].z), fabsf(xk[c].w))));
        }
        const uint8_t *rv = raw + (2 + (r >> 5)) * (kKeys * 128) + (r & 3) * 4;
        const int cv = (r & 31) >> 2;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int key = half * 32 + i;
          xv[i] = *reinterpret_cast<const float *>(rv + key * 128 + ((cv ^ (key & 7)) << 4));
          mv = fmaxf(mv, fabsf(xv[i]));
        }
        // (an infinity is in no maximum: it would flush the block's other keys and columns to zero)
        const unsigned wk = __reduce_max_sync(0xffffffffu, mk <= FLT_MAX ? __float_as_uint(mk) : 0u);
        const unsigned wv = __reduce_max_sync(0xffffffffu, mv <= FLT_MAX ? __float_as_uint(mv) : 0u);
        if (lane == 0) { atomicMax(max_s + 2 * slot, wk); atomicMax(max_s + 2 * slot + 1, wv); }
        if (MASK == kKeyMask && t < kKeys) {
          const int key = j * kKeys + t;
          // finite even where the mask is the lowest float: a row whose keys are all masked stays uniform
          mask_s[s * kKeys + t] = key < a.Sk ? a.mask[(int64_t)b * a.m_s[0] + (int64_t)h * a.m_s[1] + (int64_t)key * a.m_s[3]] : -INFINITY;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_raw_empty + 8u * s);
      } else {
        *abort_flag = 1;
      }
      named_barrier_sync(1, 128);  // reached by all four warps in every round, failed or not, so nobody is left waiting
      if (!ok) continue;
      const int ek = scale_exponent(__uint_as_float(max_s[2 * slot]), 14), ev = scale_exponent(__uint_as_float(max_s[2 * slot + 1]), 14);
      if (t == 0) {
        exp_s[2 * s] = ek;
        exp_s[2 * s + 1] = ev;
        const uint32_t next = slot == 0 ? 2u : slot - 1u;  // slot of block j + 2: free since this barrier
        max_s[2 * next] = max_s[2 * next + 1] = 0u;
      }
      if (j > 0) ok = mbar_wait_warp(bar_k_free, (uint32_t)(j - 1) & 1u, abort_flag);
      if (!ok) continue;
      const float sk = pow2(ek), sv = pow2(ev);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t hi[4], lo[4];
        split_pair(xk[2 * c].x, xk[2 * c].y, sk, hi[0], lo[0]);
        split_pair(xk[2 * c].z, xk[2 * c].w, sk, hi[1], lo[1]);
        split_pair(xk[2 * c + 1].x, xk[2 * c + 1].y, sk, hi[2], lo[2]);
        split_pair(xk[2 * c + 1].z, xk[2 * c + 1].w, sk, hi[3], lo[3]);
        uint8_t *o = split_k_ptr + (half * 4 + c) * (kKeys * 16) + r * 16;
        *reinterpret_cast<uint4 *>(o) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4 *>(o + kHalfSplit) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_k_ready);
      if (j > 0) ok = mbar_wait_warp(bar_pv, (uint32_t)(j - 1) & 1u, abort_flag);
      if (!ok) continue;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) split_pair(xv[8 * c + 2 * i], xv[8 * c + 2 * i + 1], sv, hi[i], lo[i]);
        uint8_t *o = split_v_ptr + (half * 4 + c) * (kD * 16) + r * 16;
        *reinterpret_cast<uint4 *>(o) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4 *>(o + kHalfSplit) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_v_ready);
    }
  }
  if (!ok) {
    if (leader) atomicOr(a.status, kStatusTimeout);
    *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 256);
  }
}

// 4-D map over [batch][head][row][d]; boxes of 32 floats x `box_rows` rows, 128-byte swizzle.
int attention_map(CUtensorMap *map, const float *base, int64_t rows, int64_t row_stride, int64_t nh, int64_t h_stride, int64_t nb,
                  int64_t b_stride, int box_rows) {
  return make_gemm_map(map, base, kD, rows, row_stride, nh, h_stride, nb, b_stride, 32, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace

// What attention_tc_eligible accepts (operands with unit-stride d and 16-byte aligned rows, blocks that
// belong on tensor cores) with head size 64.
bool attention_pair_shape_ok(int64_t d, int64_t d_v) { return d == kD && d_v == kD; }

int launch_attention_pair(int64_t nb1, int64_t nb0, int64_t Sq, int64_t Sk, const float *q, const int64_t *q_s, const float *k,
                          const int64_t *k_s, const float *v, const int64_t *v_s, const float *mask, const int64_t *m_s, bool causal,
                          float divisor, float *out, const int64_t *o_s, cudaStream_t s) {
  AttnPairArgs a;
  a.Sq = (int)Sq; a.Sk = (int)Sk; a.nb0 = (int)nb0;
  for (int i = 0; i < 4; ++i) { a.m_s[i] = mask ? m_s[i] : 0; a.o_s[i] = o_s[i]; }
  a.mask = mask; a.out = out; a.inv_divisor = 1.0f / divisor; a.cap = 0.0f;
  a.q_h = q_s[1] != 0; a.q_b = q_s[0] != 0; a.k_h = k_s[1] != 0; a.k_b = k_s[0] != 0; a.v_h = v_s[1] != 0; a.v_b = v_s[0] != 0;
  a.status = device_status_word();
  FML_REQUIRE(a.status, FML_CUDA_ERROR, "fml_attention: no device status word");
  CUtensorMap mq, mk, mv;
  int st = attention_map(&mq, q, Sq, q_s[2], nb0, q_s[1], nb1, q_s[0], kBM);
  if (st == FML_OK) st = attention_map(&mk, k, Sk, k_s[3], nb0, k_s[1], nb1, k_s[0], kKeys);
  if (st == FML_OK) st = attention_map(&mv, v, Sk, v_s[2], nb0, v_s[1], nb1, v_s[0], kKeys);
  if (st != FML_OK) return st;
  const size_t smem = 2 * kRawStage + 2 * kSplit + 2 * kKeys * 4 + 4 * 4 + 8 * 4 + 15 * 8 + 16;
  using KernelFn = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const AttnPairArgs, const NoRules);
  static const KernelFn kernels[4] = {attention_pair_kernel<kNoMask, NoRules>, attention_pair_kernel<kKeyMask, NoRules>,
                                      attention_pair_kernel<kFullMask, NoRules>, attention_pair_kernel<kCausal, NoRules>};
  static bool attr_set[64] = {false};
  int dev = 0;
  FML_CUDA(cudaGetDevice(&dev));
  if (!attr_set[dev & 63]) {
    for (KernelFn f : kernels) FML_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    attr_set[dev & 63] = true;
  }
  const int kind = causal ? kCausal : !mask ? kNoMask : m_s[2] == 0 ? kKeyMask : kFullMask;
  const dim3 grid((unsigned)((Sq + kBM - 1) / kBM), (unsigned)(nb0 * nb1));
  FML_CUDA(launch_kernel(kernels[kind], grid, dim3(kThreads), smem, s, mq, mk, mv, a, NoRules()));
  return FML_OK;
}

// fml_attention_rules in fp32, head size 64, operands that tensor maps take.
bool attention_rules_pair_eligible(const RulesArgs &r) {
  if (r.D != kD || !r.q_vec || !r.k_vec || !r.v_vec || r.Sk < 1 || r.Sk > kMaxBlocks * kKeys || (int64_t)r.heads * r.batch > 65535) return false;
  for (const int64_t *s : {r.q_s, r.k_s, r.v_s})
    for (int i = 0; i < 3; ++i)
      if (s[i] < 0 || s[i] >= (1ll << 37) || s[i] % 4 != 0 || (i == 2 && s[i] == 0)) return false;
  return true;
}

int launch_attention_rules_pair(const RulesArgs &r, float divisor, float cap, cudaStream_t s) {
  AttnPairArgs a;
  memset(&a, 0, sizeof(a));
  a.Sq = r.Sq; a.Sk = r.Sk; a.nb0 = r.heads;
  for (int i = 0; i < 4; ++i) a.o_s[i] = r.o_s[i];
  a.out = static_cast<float *>(r.out); a.inv_divisor = 1.0f / divisor; a.cap = cap;
  const int64_t kv_heads = r.heads / r.group;
  // (a dim of one row, head or batch takes any stride: the map is told none)
  auto stride = [](int64_t s, int64_t n) { return n > 1 ? s : 0; };
  const int64_t q_h = stride(r.q_s[1], r.heads), q_b = stride(r.q_s[0], r.batch), k_h = stride(r.k_s[1], kv_heads), k_b = stride(r.k_s[0], r.batch),
                v_h = stride(r.v_s[1], kv_heads), v_b = stride(r.v_s[0], r.batch);
  a.q_h = q_h != 0; a.q_b = q_b != 0; a.k_h = k_h != 0; a.k_b = k_b != 0; a.v_h = v_h != 0; a.v_b = v_b != 0;
  a.status = r.status;
  CUtensorMap mq, mk, mv;
  int st = attention_map(&mq, static_cast<const float *>(r.q), r.Sq, r.Sq > 1 ? r.q_s[2] : kD, r.heads, q_h, r.batch, q_b, kBM);
  if (st == FML_OK) st = attention_map(&mk, static_cast<const float *>(r.k), r.Sk, r.Sk > 1 ? r.k_s[2] : kD, kv_heads, k_h, r.batch, k_b, kKeys);
  if (st == FML_OK) st = attention_map(&mv, static_cast<const float *>(r.v), r.Sk, r.Sk > 1 ? r.v_s[2] : kD, kv_heads, v_h, r.batch, v_b, kKeys);
  if (st != FML_OK) return st;
  const size_t smem = 2 * kRawStage + 2 * kSplit + 2 * kKeys * 4 + 4 * 4 + 8 * 4 + 15 * 8 + 16 + kMaxBlocks * 2;
  static bool attr_set[64] = {false};
  int dev = 0;
  FML_CUDA(cudaGetDevice(&dev));
  if (!attr_set[dev & 63]) {
    FML_CUDA(cudaFuncSetAttribute(attention_pair_kernel<kRules, RulesArgs>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    attr_set[dev & 63] = true;
  }
  const dim3 grid((unsigned)((r.Sq + kBM - 1) / kBM), (unsigned)(r.heads * r.batch));
  FML_CUDA(launch_kernel(attention_pair_kernel<kRules, RulesArgs>, grid, dim3(kThreads), smem, s, mq, mk, mv, a, r));
  return FML_OK;
}

}  // namespace fml
