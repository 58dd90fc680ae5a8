// Attention over a prompt by rules (fml_attention_rules): capped scores, a bias by distance, documents, a prefix, grouped heads.
//
// Here: argument checks, the choice of the kernel, and the kernel on warp-wide matrix instructions, which takes fp32 and every
// layout: a CTA has 64 queries of a head, 16 to a warp, and keys pass in tiles through two stages of shared memory.  Large
// 16-bit problems run on the fifth-generation tensor cores (attention_rules_tc.cu).
//
// Measured, fp32: 4 x 16 heads of 512 x 64 119 us, where fp32 of head size 64 on packed pairs (attention_pair.cu) takes 32; what
// bounds it is the split of every operand of every product into two TF32 numbers by each warp for itself.
//
// A tile of keys that no query of the CTA sees is not loaded: causal and prefix leave the tiles up to a last one, documents are
// compared as ranges (smallest to largest number of a tile), which for documents in a row, one after another, is exact.
#include "attention_rules.cuh"
#include <algorithm>
#include <cmath>

namespace fml {
namespace {

constexpr int kMaxTiles = 4096;

template <typename T, int DP> struct Shape {
  using F = Flash<T, DP, true>;
  // (fp32 in tiles of 128 rows took as long at 4 x 16 x 512 x 64, and 23 us instead of 18 at 16 x 77)
  static constexpr int kThreads = 128, kRows = 64;
  static constexpr int kKeys = sizeof(T) == 2 ? 64 : DP == 64 ? 64 : 32, kGroups = kKeys / 8;
  static constexpr int kTileK = kKeys * F::kPitch, kTileV = kKeys * F::kPitchV, kStage = kTileK + kTileV, kQ = kRows * F::kPitch;
  static constexpr size_t kBytes = kQ + 2 * kStage + kMaxTiles;
};

template <typename T, int DP>
__global__ void __launch_bounds__(Shape<T, DP>::kThreads) attention_rules_kernel(const __grid_constant__ RulesArgs a) {
  using S = Shape<T, DP>;
  using F = typename S::F;
  constexpr int kThreads = S::kThreads, kRows = S::kRows;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t *const visible = smem + S::kQ + 2 * S::kStage;  // [tile]: TileView
  const uint32_t q_tile = smem_u32(smem), data = q_tile + S::kQ;
  const int warp = warp_index(), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int head = blockIdx.y, batch = blockIdx.z, kv = head / a.group;
  const int row0 = ((int)gridDim.x - 1 - (int)blockIdx.x) * kRows;  // (causal: the longest first)
  pdl_prologue();
  const T *const q = static_cast<const T *>(a.q) + batch * a.q_s[0] + head * a.q_s[1];
  const T *const k = static_cast<const T *>(a.k) + batch * a.k_s[0] + kv * a.k_s[1];
  const T *const v = static_cast<const T *>(a.v) + batch * a.v_s[0] + kv * a.v_s[1];

  const TileRange range = tile_range(a, batch, row0, min(row0 + kRows, a.Sq));
  const int tiles = (range.last_key + S::kKeys - 1) / S::kKeys;
  for (int i = warp; i < min(tiles, kMaxTiles); i += kThreads / 32) {
    int view = tile_view(range, i * S::kKeys, S::kKeys);
    if (a.k_documents.p && view != kTileNone) {
      int64_t low, high;
      tile_documents(a, batch, i * S::kKeys, min(i * S::kKeys + S::kKeys, a.Sk), &low, &high);
      view = document_view(view, range, low, high);
    }
    if (lane == 0) visible[i] = (uint8_t)view;
  }
  // a tile's rows from global memory, zeros for rows from `rows` on and features from D on
  auto load = [&](uint32_t dst, const T *src, int64_t row_s, int64_t d_s, int first, int rows, int total, bool vec, bool of_v) {
    for (int i = threadIdx.x; i < total * F::kChunks; i += kThreads) {
      const int row = i / F::kChunks, c = i % F::kChunks;
      const uint32_t to = dst + (of_v ? F::at_v(row, c) : F::at(row, c));
      if (vec) {
        const bool in = first + row < rows && c * F::kChunk < a.D;
        cp_async16(to, src + (in ? (int64_t)(first + row) * row_s + c * F::kChunk : 0), in);
      } else {
        alignas(16) T e[F::kChunk];
#pragma unroll
        for (int b = 0; b < F::kChunk; ++b) {
          const int d = c * F::kChunk + b;
          e[b] = first + row < rows && d < a.D ? src[(int64_t)(first + row) * row_s + d * d_s] : from_f32<T>(0.0f);
        }
        const uint4 x = *reinterpret_cast<const uint4 *>(e);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
      }
    }
  };
  load(q_tile, q, a.q_s[2], a.q_s[3], row0, a.Sq, kRows, a.q_vec, false);
  cp_async_commit();
  __syncthreads();
  auto view_of = [&](int i) { return i < kMaxTiles ? (int)visible[i] : (int)kTileSome; };
  auto next_tile = [&](int i) {
    while (i < tiles && view_of(i) == kTileNone) ++i;
    return i;
  };
  auto fetch = [&](int tile, int stage) {
    const uint32_t dst = data + (uint32_t)stage * S::kStage;
    load(dst, k, a.k_s[2], a.k_s[3], tile * S::kKeys, a.Sk, S::kKeys, a.k_vec, false);
    load(dst + S::kTileK, v, a.v_s[2], a.v_s[3], tile * S::kKeys, a.Sk, S::kKeys, a.v_vec, true);
    cp_async_commit();
  };
  int tile = next_tile(0);
  if (tile < tiles) fetch(tile, 0);
  cp_async_wait<0>();
  __syncthreads();
  typename F::Q qf;
  F::load_q(qf, q_tile, 16 * warp);
  Running<DP> run;
  run.reset();
  RowRules row[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) row[h] = row_rules(a, batch, head, min(row0 + 16 * warp + g + 8 * h, a.Sq - 1));
  int stage = 0;
  while (tile < tiles) {
    const int next = next_tile(tile + 1);
    if (next < tiles) fetch(next, stage ^ 1);
    const uint32_t k_tile = data + (uint32_t)stage * S::kStage;
    const bool open = view_of(tile) == kTileAll;
    const int key_base = tile * S::kKeys;
    flash_step<F, DP, S::kGroups>(run, qf, q_tile, 16 * warp, k_tile, k_tile + S::kTileK, 0, [&](float (&s)[S::kGroups][4]) {
      cap_scores<sizeof(T) == 4>(a.cap, s);
      if (a.slopes) {
#pragma unroll
        for (int n = 0; n < S::kGroups; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][i] -= row[i >> 1].slope * (float)abs(row[i >> 1].at - (key_base + 8 * n + 2 * t + (i & 1)));
      }
      if (!open) {
#pragma unroll
        for (int n = 0; n < S::kGroups; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int key = key_base + 8 * n + 2 * t + c;
            const int64_t document = a.k_documents.p && key < a.Sk ? document_at(a.k_documents, a.k_documents_row, batch, key) : 0;
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (!key_seen(a, row[h], key, document)) s[n][2 * h + c] = -INFINITY;
          }
      }
    });
    cp_async_wait<0>();
    __syncthreads();
    stage ^= 1;
    tile = next;
  }
  // ---- out = o / l; a row that is not finite is done again over the keys it sees alone
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    run.l[h] += __shfl_xor_sync(0xffffffffu, run.l[h], 1);
    run.l[h] += __shfl_xor_sync(0xffffffffu, run.l[h], 2);
    const float inv = run.l[h] == 0.0f ? 0.0f : 1.0f / run.l[h];
    const int i = row0 + 16 * warp + g + 8 * h;
    T *dst = static_cast<T *>(a.out) + batch * a.o_s[0] + head * a.o_s[1] + (int64_t)i * a.o_s[2];
    bool bad = false;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int d = 8 * n + 2 * t + c;
        const float x = run.l[h] == 0.0f ? 0.0f : run.o[n][2 * h + c] * inv;
        bad = bad || !(fabsf(x) <= 3.402823466e38f);
        if (i < a.Sq && d < a.D) dst[d * a.o_s[3]] = from_f32<T>(x);
      }
    unsigned redo = __ballot_sync(0xffffffffu, bad && i < a.Sq);
    __syncwarp();
    while (redo) {
      const int r = (__ffs(redo) - 1) >> 2;  // row r of the eight
      redo &= ~(0xfu << (4 * r));
      redo_rules_row<T>(a, batch, head, row0 + 16 * warp + r + 8 * h);
    }
  }
}

template <typename T, int DP> int launch_mma(const RulesArgs &a, cudaStream_t s) {
  using S = Shape<T, DP>;
  static bool attr_set[64] = {false};
  int dev = 0;
  FML_CUDA(cudaGetDevice(&dev));
  if (!attr_set[dev & 63]) {
    FML_CUDA(cudaFuncSetAttribute(attention_rules_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kBytes));
    attr_set[dev & 63] = true;
  }
  FML_LAUNCH((attention_rules_kernel<T, DP>), dim3((unsigned)((a.Sq + S::kRows - 1) / S::kRows), (unsigned)a.heads, (unsigned)a.batch), S::kThreads,
             S::kBytes, s, a);
  return FML_OK;
}
template <typename T> int launch_mma(const RulesArgs &a, cudaStream_t s) {
  return a.D <= 64 ? launch_mma<T, 64>(a, s) : launch_mma<T, 128>(a, s);
}

}  // namespace
}  // namespace fml

using namespace fml;

extern "C" int fml_attention_rules(const fml_tensor *q, const fml_tensor *k, const fml_tensor *v, const fml_tensor *slopes,
                                   const fml_tensor *prefix, const fml_tensor *q_documents, const fml_tensor *k_documents,
                                   const fml_score_rules *rules, const fml_tensor *out, void *stream) {
  FML_REQUIRE(data_tensor(q, 4) && data_tensor(k, 4) && data_tensor(v, 4) && data_tensor(out, 4), FML_BAD_ARG,
              "fml_attention_rules: q, k, v, out must be [batch, heads, length, head size] of fp32, fp16 or bf16");
  FML_REQUIRE(k->dtype == q->dtype && v->dtype == q->dtype && out->dtype == q->dtype, FML_BAD_ARG, "fml_attention_rules: one type per call");
  FML_REQUIRE(rules && std::isfinite(rules->divisor) && rules->divisor != 0.0f && std::isfinite(rules->cap) && rules->cap >= 0.0f, FML_BAD_ARG,
              "fml_attention_rules: divisor must be finite and not zero, cap finite and not negative");
  FML_REQUIRE(factors_in_range(rules->divisor, rules->cap), FML_UNSUPPORTED,
              "fml_attention_rules: caps of 2^-64 to 2^64 (0: none), divisors with 1 / divisor and 1 / (divisor cap) in fp32's range");
  const int64_t batch = q->shape[0], heads = q->shape[1], sq = q->shape[2], d = q->shape[3], kv_heads = k->shape[1], sk = k->shape[2];
  for (int i = 0; i < 4; ++i) {
    FML_REQUIRE(out->shape[i] == q->shape[i], FML_BAD_ARG, "fml_attention_rules: shape of out");
    FML_REQUIRE(v->shape[i] == k->shape[i], FML_BAD_ARG, "fml_attention_rules: shapes of k and v differ");
  }
  FML_REQUIRE(elements_apart(out), FML_BAD_ARG, "fml_attention_rules: out has a stride of 0");
  FML_REQUIRE(k->shape[0] == batch && k->shape[3] == d, FML_BAD_ARG, "fml_attention_rules: batch or head size of k and v");
  FML_REQUIRE(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, FML_BAD_ARG, "fml_attention_rules: heads must be a multiple of the heads of k and v");
  FML_REQUIRE(d >= 4 && d <= 128 && d % 4 == 0, FML_UNSUPPORTED, "fml_attention_rules: head sizes that are multiples of 4 up to 128");
  FML_REQUIRE(!slopes || (float_tensor(slopes, 1) && slopes->shape[0] == heads), FML_BAD_ARG, "fml_attention_rules: slopes must be [heads] of fp32");
  FML_REQUIRE(!prefix || (index_tensor(prefix, 1) && prefix->shape[0] == batch), FML_BAD_ARG,
              "fml_attention_rules: prefix must be [batch] of int32 or int64");
  FML_REQUIRE(!q_documents == !k_documents, FML_BAD_ARG, "fml_attention_rules: documents of queries and of keys go together");
  FML_REQUIRE(!q_documents || (index_tensor(q_documents, 2) && q_documents->shape[0] == batch && q_documents->shape[1] == sq &&
                               index_tensor(k_documents, 2) && k_documents->shape[0] == batch && k_documents->shape[1] == sk),
              FML_BAD_ARG, "fml_attention_rules: documents must be [batch, length] of int32 or int64");
  FML_REQUIRE(batch <= 65535 && heads <= 65535 && sq < (1 << 30) && sk < (1 << 30), FML_UNSUPPORTED, "fml_attention_rules: too large");
  if (batch == 0 || sq == 0) return FML_OK;
  FML_REQUIRE(inputs_on_current_device({q, k, v, slopes, prefix, q_documents, k_documents}), FML_BAD_ARG,
              "fml_attention_rules: an input is not memory of the current device");
  FML_REQUIRE(on_current_device(out->data), FML_BAD_ARG, "fml_attention_rules: the output is not memory of the current device");
  RulesArgs a;
  memset(&a, 0, sizeof(a));
  a.q = q->data; a.k = k->data; a.v = v->data; a.out = out->data;
  for (int i = 0; i < 4; ++i) { a.q_s[i] = q->stride[i]; a.k_s[i] = k->stride[i]; a.v_s[i] = v->stride[i]; a.o_s[i] = out->stride[i]; }
  a.batch = (int)batch; a.heads = (int)heads; a.group = (int)(heads / kv_heads); a.Sq = (int)sq; a.Sk = (int)sk; a.D = (int)d;
  a.causal = rules->causal != 0;
  a.cap = Cap::make(rules->divisor, rules->cap);
  a.slopes = slopes ? static_cast<const float *>(slopes->data) : nullptr;
  a.slopes_s = slopes ? slopes->stride[0] : 0;
  if (prefix && a.causal) a.prefix = index_view(prefix);
  if (q_documents) {
    a.q_documents = index_view(q_documents); a.k_documents = index_view(k_documents);
    a.q_documents_row = q_documents->stride[0]; a.k_documents_row = k_documents->stride[0];
  }
  const int64_t per16 = 16 / (int64_t)data_size(q->dtype);
  auto vec = [&](const fml_tensor *t) {
    bool ok = t->stride[3] == 1 && d % per16 == 0 && aligned16(t->data);
    for (int i = 0; i < 3; ++i) ok = ok && (t->shape[i] == 1 || t->stride[i] % per16 == 0);
    return ok;
  };
  a.q_vec = vec(q); a.k_vec = vec(k); a.v_vec = vec(v);
  a.status = device_status_word();
  FML_REQUIRE(a.status, FML_CUDA_ERROR, "fml_attention_rules: no device status word");
  if (attention_rules_tc_eligible(a, q->dtype)) return launch_attention_rules_tc(a, q->dtype, as_stream(stream));
  if (q->dtype == FML_F32 && attention_rules_pair_eligible(a)) return launch_attention_rules_pair(a, rules->divisor, rules->cap, as_stream(stream));
  if (q->dtype == FML_F32) return launch_mma<float>(a, as_stream(stream));
  if (q->dtype == FML_F16) return launch_mma<__half>(a, as_stream(stream));
  return launch_mma<__nv_bfloat16>(a, as_stream(stream));
}
