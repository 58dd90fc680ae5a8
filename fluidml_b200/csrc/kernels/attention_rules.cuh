// Rules of fml_attention_rules that its two kernels share: which keys a query sees, which tiles of keys a tile of queries sees,
// and the repair of rows that are not finite.
#pragma once
#include "flash_mma.cuh"

namespace fml {

struct RulesArgs {
  const void *q, *k, *v;
  void *out;
  int64_t q_s[4], k_s[4], v_s[4], o_s[4];  // element strides
  const float *slopes;
  int64_t slopes_s;
  IndexView prefix, q_documents, k_documents;  // documents: p of batch 0, stride along the length
  int64_t q_documents_row, k_documents_row;    // element strides over the batch
  int batch, heads, group, Sq, Sk, D, causal;
  Cap cap;
  int q_vec, k_vec, v_vec;  // rows take 16-byte accesses
  int o_tma;                // the result leaves by tensor map (attention_rules_tc.cu)
  int *status;
};

// attention_rules_tc.cu: whether its kernel takes these operands, and its launch.
bool attention_rules_tc_eligible(const RulesArgs &a, int dtype);
int launch_attention_rules_tc(const RulesArgs &a, int dtype, cudaStream_t s);
// attention_pair.cu: the same in fp32.
bool attention_rules_pair_eligible(const RulesArgs &r);
int launch_attention_rules_pair(const RulesArgs &r, float divisor, float cap, cudaStream_t s);

__device__ __forceinline__ int64_t document_at(const IndexView &v, int64_t row, int batch, int i) {
  const int64_t e = batch * row + i * v.stride;
  return v.wide ? static_cast<const int64_t *>(v.p)[e] : (int64_t)static_cast<const int32_t *>(v.p)[e];
}

// What a query goes by: its position, the last key + 1 that causal and prefix leave it, its document and slope (units of ln 2).
struct RowRules {
  int at, last;
  int64_t document;
  float slope;
};
__device__ __forceinline__ int last_key_of(const RulesArgs &a, int batch, int row) {
  if (!a.causal) return a.Sk;
  int64_t last = (int64_t)row + a.Sk - a.Sq + 1;
  if (a.prefix.p) last = max(last, index_at(a.prefix, batch));
  return (int)max((int64_t)0, min(last, (int64_t)a.Sk));
}
__device__ __forceinline__ RowRules row_rules(const RulesArgs &a, int batch, int head, int row) {
  RowRules r;
  r.at = row + a.Sk - a.Sq;
  r.last = last_key_of(a, batch, row);
  r.document = a.q_documents.p ? document_at(a.q_documents, a.q_documents_row, batch, row) : 0;
  r.slope = a.slopes ? a.slopes[head * a.slopes_s] * kLog2e : 0.0f;
  return r;
}
__device__ __forceinline__ bool key_seen(const RulesArgs &a, const RowRules &r, int key, int64_t document) {
  return key < r.last && (!a.q_documents.p || document == r.document);
}

// What the queries [row0, row1) of a tile see of a tile of keys: none, all of them every key, or some (kTileLast: those up to
// the query's last, all of its document).
enum TileView { kTileNone = 0, kTileSome = 1, kTileAll = 2, kTileLast = 3 };
struct TileRange {
  int first_key, last_key;  // every query sees the keys below first_key, none those from last_key on (documents apart)
  int64_t low, high;        // the queries' smallest and largest document
};
__device__ __forceinline__ int64_t warp_min(int64_t v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = min(v, (int64_t)__shfl_xor_sync(0xffffffffu, (long long)v, o));
  return v;
}
// By a whole warp.
__device__ __forceinline__ TileRange tile_range(const RulesArgs &a, int batch, int row0, int row1) {
  TileRange t;
  t.first_key = last_key_of(a, batch, row0);  // (grows with the row)
  t.last_key = last_key_of(a, batch, row1 - 1);
  t.low = INT64_MAX;
  t.high = INT64_MIN;
  if (a.q_documents.p) {
    for (int i = row0 + (int)(threadIdx.x & 31); i < row1; i += 32) {
      const int64_t x = document_at(a.q_documents, a.q_documents_row, batch, i);
      t.low = min(t.low, x);
      t.high = max(t.high, x);
    }
    t.low = warp_min(t.low);
    t.high = ~warp_min(~t.high);
  }
  return t;
}
__device__ __forceinline__ int tile_view(const TileRange &t, int key0, int keys) {  // documents apart
  return key0 >= t.last_key ? kTileNone : key0 + keys <= t.first_key ? kTileAll : kTileSome;
}
// The smallest and largest document of the keys [key0, key1), by a whole warp.
__device__ __forceinline__ void tile_documents(const RulesArgs &a, int batch, int key0, int key1, int64_t *low, int64_t *high) {
  int64_t l = INT64_MAX, h = INT64_MIN;
  for (int i = key0 + (int)(threadIdx.x & 31); i < key1; i += 32) {
    const int64_t x = document_at(a.k_documents, a.k_documents_row, batch, i);
    l = min(l, x);
    h = max(h, x);
  }
  *low = warp_min(l);
  *high = ~warp_min(~h);
}
__device__ __forceinline__ int document_view(int view, const TileRange &t, int64_t low, int64_t high) {
  if (view == kTileNone || low > t.high || high < t.low) return kTileNone;
  return low == high && t.low == t.high ? (view == kTileAll ? kTileAll : kTileLast) : kTileSome;
}

// A row whose context came out as not finite: keys that it does not see may hold infinities or NaN, which weights of zero do
// not cancel (or, on packed pairs, values beside which its own have no bits left).  Done again by a warp over those it sees (one
// of them may be the cause: then it stays).
template <typename T> __device__ __noinline__ void redo_rules_row(const RulesArgs &a, int batch, int head, int row) {
  const int lane = threadIdx.x & 31, kv = head / a.group;
  const RowRules r = row_rules(a, batch, head, row);
  const T *q = static_cast<const T *>(a.q) + batch * a.q_s[0] + head * a.q_s[1] + (int64_t)row * a.q_s[2];
  const T *k0 = static_cast<const T *>(a.k) + batch * a.k_s[0] + kv * a.k_s[1], *v0 = static_cast<const T *>(a.v) + batch * a.v_s[0] + kv * a.v_s[1];
  float o[4], m, l;
  context_of_seen(q, a.q_s[3], a.k_s[3], a.v_s[3], a.D, a.cap, 0, r.last, [&](int key, const T **k, const T **v, float *less) {
    if (a.k_documents.p && document_at(a.k_documents, a.k_documents_row, batch, key) != r.document) return false;
    *k = k0 + (int64_t)key * a.k_s[2];
    *v = v0 + (int64_t)key * a.v_s[2];
    if (a.slopes) *less = r.slope * (float)abs(r.at - key);
    return true;
  }, o, m, l);
  T *dst = static_cast<T *>(a.out) + batch * a.o_s[0] + head * a.o_s[1] + (int64_t)row * a.o_s[2];
  for (int i = 0, d = lane; d < a.D; ++i, d += 32) dst[d * a.o_s[3]] = from_f32<T>(l == 0.0f ? 0.0f : o[i] / l);
}

}  // namespace fml
