// Attention of new tokens over a paged cache (fml_attention_tree): the ordinary decoding step, and drafted trees of tokens.
//
// The queries of a request that share a kv head (new tokens x heads of the group) are rows of one tile, so that a key is read
// once for all of them.  What bounds it: the keys' and values' bytes.  All tiles of keys of all requests, kv heads and row
// tiles are one line of units, cut into equal parts for a fixed number of CTAs: a long request is shared by many, short ones
// share a CTA, and no CTA waits for the longest.  A CTA writes a stretch that is all of a row's keys to the output and any
// other to the workspace (normalised context, maximum and sum), which a second kernel adds up in a fixed order.
//
// Keys and values come through shared memory by 16-byte asynchronous copies (rows of a page are contiguous, pages are not).  One
// bulk copy per row instead, which a warp issues lane by lane, took 289 us for 232 on 64 requests of one token.
//
// Measured (bf16, head size 128): 64 requests of one token over up to 8192, 32 kv heads 805 us, 5.0 TB/s; 8 kv heads 215 us, 4.7;
// 48 requests of up to 16 drafts, 32 heads on 8, capped 380 us, 2.2 TB/s: there the instructions of softmax and cap, and one
// barrier per tile for two CTAs of eight warps, bound it; one token over 1000 14 us, most of it the two launches' dependent loads.
#include "flash_mma.cuh"
#include <algorithm>
#include <cmath>

namespace fml {
namespace {

constexpr int kJoinThreads = 128;

struct TreeArgs {
  const void *q, *k, *v;
  void *out;
  const int32_t *table, *context, *query_start;
  const int64_t *tree;
  const float *slopes;
  int64_t q_t, q_h, q_d, o_t, o_h, o_d;                       // element strides
  int64_t k_page, k_pos, k_head, v_page, v_pos, v_head;
  int64_t table_r, table_c, context_s, start_s, tree_s, slopes_s;
  int64_t pages, tokens;
  int requests, columns, page, heads, kv_heads, group, D, q_vec, page_shift;  // page_shift: -1 when the page size is no power of two
  int alike;  // pages and positions of K and V lie alike: places are byte offsets, else page << 32 | position
  Cap cap;
  float *partial;       // [CTA][2][rows of a tile][DP + 2]
  long long *first;     // [requests + 1]: first unit of a request, then all units
  int *status;
};

// Request r: its first new token, their number and the cached tokens, cut to what the tensors hold.
struct Request { int start, fresh, context; };
__device__ __forceinline__ Request request_of(const TreeArgs &a, int r, bool report) {
  Request x;
  int lo = a.query_start[r * a.start_s], hi = a.query_start[(r + 1) * a.start_s], ctx = a.context[r * a.context_s];
  const int64_t room = (int64_t)a.columns * a.page;
  const int lo_c = (int)min((int64_t)max(lo, 0), a.tokens), hi_c = (int)min((int64_t)max(hi, lo_c), a.tokens);
  const int ctx_c = (int)min((int64_t)max(ctx, 0), room);
  x.start = lo_c;
  x.context = ctx_c;
  x.fresh = hi_c - lo_c;
  bool bad = lo_c != lo || hi_c != hi || ctx_c != ctx;
  if ((int64_t)ctx_c + x.fresh > room) bad = true;  // (new tokens without room are queries still, but no keys)
  if (bad && report) atomicOr(a.status, kStatusIndexRange);
  return x;
}
__device__ __forceinline__ int keys_of(const TreeArgs &a, const Request &x) {
  return x.fresh == 0 ? 0 : (int)min((int64_t)x.context + x.fresh, (int64_t)a.columns * a.page);
}
template <int MT, int TK> __device__ __forceinline__ long long units_of(const TreeArgs &a, const Request &x) {
  if (x.fresh == 0) return 0;
  const long long row_tiles = ((long long)x.fresh * a.group + MT - 1) / MT, key_tiles = max(1, (keys_of(a, x) + TK - 1) / TK);
  return row_tiles * key_tiles * a.kv_heads;
}

// What new token j of a request sees of its new tokens, as bits (64 and more: a chain's).
__device__ __forceinline__ unsigned long long mask_of(const TreeArgs &a, const Request &x, int j) {
  const unsigned long long all = x.fresh >= 64 ? ~0ull : (1ull << x.fresh) - 1ull;
  return (unsigned long long)a.tree[(int64_t)(x.start + j) * a.tree_s] & all;
}
__device__ __forceinline__ int position_of(const TreeArgs &a, const Request &x, int j) {
  return x.context + (a.tree ? __popcll(mask_of(a, x, j)) - 1 : j);
}
__device__ __forceinline__ bool sees(const TreeArgs &a, const Request &x, int j, int key) {  // key >= context
  const int i = key - x.context;
  return a.tree ? i < 64 && (mask_of(a, x, j) >> i & 1ull) : i <= j;
}
// The page that holds a key, -1 for one that is not there.
__device__ __forceinline__ int64_t page_of(const TreeArgs &a, int r, int key) {
  const int64_t page = a.table[r * a.table_r + (key / a.page) * a.table_c];
  return page >= 0 && page < a.pages ? page : -1;
}

// A row whose context came out as not finite: keys it does not see may hold infinities, which weights of zero do not cancel.
// Done again by a warp over the keys that it sees, from first to last (one of them may be the cause: then it stays).
template <typename T>
__device__ __noinline__ void redo_row(const TreeArgs &a, int r, const Request &x, int kv, int j, int head, int key0, int key1, float *ctx, float *stats) {
  const int lane = threadIdx.x & 31;
  const T *q = static_cast<const T *>(a.q) + (int64_t)(x.start + j) * a.q_t + (int64_t)head * a.q_h;
  const float slope = a.slopes ? a.slopes[head * a.slopes_s] * kLog2e : 0.0f;
  const int at = position_of(a, x, j);
  float o[4], m, l;
  context_of_seen(q, a.q_d, 1, 1, a.D, a.cap, key0, key1, [&](int key, const T **k, const T **v, float *less) {
    if (key >= x.context && !sees(a, x, j, key)) return false;
    const int64_t page = page_of(a, r, key);
    if (page < 0) return false;
    *k = static_cast<const T *>(a.k) + page * a.k_page + (key % a.page) * a.k_pos + kv * a.k_head;
    *v = static_cast<const T *>(a.v) + page * a.v_page + (key % a.page) * a.v_pos + kv * a.v_head;
    if (a.slopes) *less = slope * (float)abs(at - (key < x.context ? key : position_of(a, x, key - x.context)));
    return true;
  }, o, m, l);
  for (int i = 0, d = lane; d < a.D; ++i, d += 32) ctx[d] = l == 0.0f ? 0.0f : o[i] / l;
  if (lane == 0) { stats[0] = m; stats[1] = l; }
}

// Warps: WR of 16 rows each, times those that take different keys of a tile.  Tiles of up to 16 rows: four warps, queries in
// registers, three stages of 64 keys.  More rows: eight warps, which leaves each half of the registers, so the queries are read
// from shared memory again and again, and two stages.
template <typename T, int DP, int WR> struct Shape {
  static constexpr bool kHeld = WR == 1;
  using F = Flash<T, DP, kHeld>;
  static constexpr int kWarps = WR == 1 ? 4 : 8, kThreads = 32 * kWarps, kWarpsK = kWarps / WR, kRows = 16 * WR;
  static constexpr int kKeys = sizeof(T) == 2 ? 64 : DP == 64 ? 64 : 32;  // 32 KiB of keys and values for head size 128
  static constexpr int kWarpKeys = kKeys / kWarpsK, kGroups = kWarpKeys / 8;
  static constexpr int kTileK = kKeys * F::kPitch, kTileV = kKeys * F::kPitchV, kStage = kTileK + kTileV;
  static constexpr int kQ = kRows * F::kPitch, kMerge = kWarps * 16 * (DP + 4) * 4;
  // held queries move on to registers: their tile is where the third stage will be
  static constexpr bool kQInStage = kHeld && sizeof(T) == 2;
  static constexpr int kStagesUsed = kHeld ? 3 : 2;
  static constexpr int kData = kStagesUsed * kStage > kMerge ? kStagesUsed * kStage : kMerge;
  static constexpr int kOffsets = (kStagesUsed + 1) * kKeys * 8;
  static constexpr size_t kBytes = (kQInStage ? 0 : kQ) + kData + kOffsets + kWarps * 16 * 2 * 4 + 64 * 4 + 64;
  static constexpr int kPartial = kRows * (DP + 2);  // floats of a partial result
  static_assert((kQ <= kStage || !kQInStage) && 2 * (kBytes + 1024) <= 228 * 1024, "two CTAs per SM");
};

template <typename T, int DP, int WR>
__global__ void __launch_bounds__(Shape<T, DP, WR>::kThreads, 2) attention_tree_kernel(const __grid_constant__ TreeArgs a) {
  using S = Shape<T, DP, WR>;
  constexpr int kThreads = S::kThreads;
  using F = typename S::F;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t *const data_ptr = smem + (S::kQInStage ? 0 : S::kQ);
  long long *const places = reinterpret_cast<long long *>(data_ptr + S::kData);   // [stage + 1][key]: see a.alike; -1 none
  float *const stats = reinterpret_cast<float *>(places + (S::kStagesUsed + 1) * S::kKeys);  // [warp][16][2]: m, l of a warp's rows
  int *const redo = reinterpret_cast<int *>(stats + S::kWarps * 32);                  // [64]
  int *const missing = redo + 64;                                                    // [stage + 1]: a key of the tile has no page
  long long *const scan = reinterpret_cast<long long *>(stats);                      // [warp] (before the first tile)
  __shared__ long long sh_first;
  __shared__ int sh_request;
  const uint32_t data = smem_u32(data_ptr);
  const int warp = warp_index(), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int wr = warp % WR, wk = warp / WR;
  pdl_prologue();

  // ---- this CTA's part of the line: all units are counted (requests in rounds of kThreads), then the part's first is looked for
  // (in the last round's counts first: few requests are read once)
  long long passed = 0, own = 0, before = 0;
  int r0 = 0;
  auto count = [&](bool report) {  // units of request r0 + thread, of those before it, and of all up to this round's end
    const int r = r0 + threadIdx.x;
    own = r < a.requests ? units_of<S::kRows, S::kKeys>(a, request_of(a, r, report)) : 0;
    long long run = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    __syncthreads();
    if (lane == 31) scan[warp] = run;
    __syncthreads();
    before = passed + run - own;
#pragma unroll
    for (int w = 0; w < S::kWarps; ++w) {
      if (w < warp) before += scan[w];
      passed += scan[w];
    }
  };
  if (threadIdx.x == 0) sh_request = -1;
  for (;; r0 += kThreads) {
    count(blockIdx.x == 0);
    if (blockIdx.x == 0 && r0 + threadIdx.x < a.requests) a.first[r0 + threadIdx.x] = before;
    if (r0 + kThreads >= a.requests) break;
  }
  const long long total = passed, share = (total + gridDim.x - 1) / gridDim.x;
  long long unit = min(total, share * blockIdx.x);
  const long long end = min(total, unit + share);
  auto look = [&]() {
    if (unit >= before && unit < before + own) { sh_request = r0 + threadIdx.x; sh_first = before; }
  };
  look();
  __syncthreads();
  if (a.requests > kThreads) {
    passed = 0;
    for (r0 = 0; r0 + kThreads < a.requests; r0 += kThreads) {
      count(false);
      look();
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.first[a.requests] = total;
  int r = sh_request;
  long long first = r >= 0 ? sh_first : 0;

  bool front = true;  // the CTA's first stretch
  while (unit < end) {
    Request x = request_of(a, r, false);
    const long long here = units_of<S::kRows, S::kKeys>(a, x);
    if (unit >= first + here) { first += here; ++r; continue; }
    const int keys = keys_of(a, x), key_tiles = max(1, (keys + S::kKeys - 1) / S::kKeys);
    const int rows = x.fresh * a.group, row_tiles = (rows + S::kRows - 1) / S::kRows;
    const long long in = unit - first;
    const int tile0 = (int)(in % key_tiles), tile1 = (int)min((long long)key_tiles, tile0 + end - unit);
    const int rt = (int)(in / key_tiles % row_tiles), kv = (int)(in / key_tiles / row_tiles), row_base = rt * S::kRows;

    // ---- queries of the row tile (row = token * group + head of the group), features beyond D zero
    uint8_t *const q_ptr = S::kQInStage ? data_ptr + (tile0 + 2) % 3 * S::kStage : smem;
    const uint32_t q_tile = smem_u32(q_ptr);
    __syncthreads();
    for (int i = threadIdx.x; i < S::kRows * F::kChunks; i += kThreads) {
      const int row = i / F::kChunks, c = i % F::kChunks, gr = row_base + row;
      const T *src = static_cast<const T *>(a.q) + (int64_t)(x.start + gr / a.group) * a.q_t + (int64_t)(kv * a.group + gr % a.group) * a.q_h;
      uint4 e = make_uint4(0u, 0u, 0u, 0u);
      if (a.q_vec) {
        if (gr < rows && c * F::kChunk < a.D) e = *reinterpret_cast<const uint4 *>(src + c * F::kChunk);
      } else {
        alignas(16) T x[F::kChunk];
#pragma unroll
        for (int b = 0; b < F::kChunk; ++b) {
          const int d = c * F::kChunk + b;
          x[b] = gr < rows && d < a.D ? src[d * a.q_d] : from_f32<T>(0.0f);
        }
        memcpy(&e, x, 16);
      }
      *reinterpret_cast<uint4 *>(q_ptr + F::at(row, c)) = e;
    }
    if (threadIdx.x < 64) redo[threadIdx.x] = 0;
    if (threadIdx.x <= S::kStagesUsed) missing[threadIdx.x] = 0;
    __syncthreads();

    // ---- the pipeline of three (two) stages: places of tile i + 3 (i + 2), copies of tile i + 2 (i + 1), products of tile i
    auto find = [&](int tile) {
      const int slot = tile % (S::kStagesUsed + 1);
      for (int i = threadIdx.x; i < S::kKeys; i += kThreads) {
        const int key = tile * S::kKeys + i;
        long long w = -1;
        if (key < keys) {
          const int at = a.page_shift >= 0 ? key >> a.page_shift : key / a.page, pos = key - at * a.page;
          int64_t page = a.table[r * a.table_r + at * a.table_c];
          if (page >= a.pages) page = -1;
          if (page >= 0) w = a.alike ? (page * a.k_page + pos * a.k_pos) * (int)sizeof(T) : page << 32 | pos;
          else { missing[slot] = 1; atomicOr(a.status, kStatusIndexRange); }
        }
        places[slot * S::kKeys + i] = w;
      }
    };
    auto fetch = [&](int tile) {
      // Eight threads copy 128 bytes of a row at a time: a row's address is formed once for all of its parts.
      constexpr int kParts = F::kChunks / 8, kStep = kThreads / 8;
      static_assert(F::kChunks % 8 == 0 && S::kKeys % kStep == 0, "");
      const uint32_t dst = data + (uint32_t)(tile % S::kStagesUsed) * S::kStage;
      const int c = threadIdx.x % 8, row0 = threadIdx.x / 8;
      const long long *place = places + tile % (S::kStagesUsed + 1) * S::kKeys + row0;
      const char *const k = static_cast<const char *>(a.k) + 16 * c + kv * a.k_head * (int)sizeof(T);
      const char *const v = static_cast<const char *>(a.v) + 16 * c + kv * a.v_head * (int)sizeof(T);
#pragma unroll
      for (int i = 0; i < S::kKeys / kStep; ++i) {
        const long long w = place[i * kStep];
        int64_t kw = w >= 0 ? w : 0, vw = kw;
        if (!a.alike) {
          const int64_t page = kw >> 32, pos = kw & 0xffffffff;
          kw = (page * a.k_page + pos * a.k_pos) * (int)sizeof(T);
          vw = (page * a.v_page + pos * a.v_pos) * (int)sizeof(T);
        }
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          const bool valid = w >= 0 && (8 * part + c) * F::kChunk < a.D;
          const int64_t off = valid ? 128 * part : -16 * c;  // (an address within the row for what is not read)
          cp_async16(dst + F::at(row0 + i * kStep, 8 * part + c), k + kw + off, valid);
          cp_async16(dst + S::kTileK + F::at_v(row0 + i * kStep, 8 * part + c), v + vw + off, valid);
        }
      }
    };
    for (int i = tile0; i < min(tile1, tile0 + S::kStagesUsed); ++i) find(i);
    __syncthreads();
    for (int i = 0; i < S::kStagesUsed - 1; ++i) {
      if (tile0 + i < tile1) fetch(tile0 + i);
      cp_async_commit();
    }
    typename F::Q q;
    F::load_q(q, q_tile, 16 * wr);
    Running<DP> run;
    run.reset();
    // this thread's rows
    int row_j[2];
    unsigned long long row_mask[2] = {0, 0};
    float row_slope[2] = {0.0f, 0.0f};
    int row_at[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int gr = min(row_base + 16 * wr + g + 8 * h, rows - 1);
      row_j[h] = gr / a.group;
      if (a.tree) row_mask[h] = mask_of(a, x, row_j[h]);
      if (a.slopes) row_slope[h] = a.slopes[(int64_t)(kv * a.group + gr % a.group) * a.slopes_s] * kLog2e;
      row_at[h] = position_of(a, x, row_j[h]);
    }
    for (int tile = tile0; tile < tile1; ++tile) {
      cp_async_wait<S::kStagesUsed - 2>();
      __syncthreads();  // tile's copies are there, and everyone is done with the stage that the next copies fill
      if (tile + S::kStagesUsed - 1 < tile1) fetch(tile + S::kStagesUsed - 1);
      cp_async_commit();
      const int slot = tile % (S::kStagesUsed + 1);
      const bool holes = missing[slot] != 0;
      if (tile + S::kStagesUsed < tile1) {
        find(tile + S::kStagesUsed);  // (its slot was tile - 1's: nobody reads that after this round's barrier)
      }
      const uint32_t k_tile = data + (uint32_t)(tile % S::kStagesUsed) * S::kStage;
      const int key_base = tile * S::kKeys + wk * S::kWarpKeys;
      const bool open = tile * S::kKeys + S::kKeys <= x.context && !holes;  // every key is seen by every row
      if (row_base + 16 * wr < rows)  // (a request's last tile may leave warps without rows)
      flash_step<F, DP, S::kGroups>(run, q, q_tile, 16 * wr, k_tile, k_tile + S::kTileK, wk * S::kWarpKeys, [&](float (&s)[S::kGroups][4]) {
        cap_scores<sizeof(T) == 4>(a.cap, s);
        if (open) {
          if (a.slopes) {
#pragma unroll
            for (int n = 0; n < S::kGroups; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) s[n][i] -= row_slope[i >> 1] * (float)abs(row_at[i >> 1] - (key_base + 8 * n + 2 * t + (i & 1)));
          }
        } else {
#pragma unroll
          for (int n = 0; n < S::kGroups; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int key = key_base + 8 * n + 2 * t + c, fresh = key - x.context;
              const bool there = key < keys && !(holes && places[slot * S::kKeys + wk * S::kWarpKeys + 8 * n + 2 * t + c] < 0);
              const int at = !a.slopes || fresh < 0 || !there ? key : position_of(a, x, fresh);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const bool seen = there && (fresh < 0 || (a.tree ? fresh < 64 && (row_mask[h] >> fresh & 1ull) : fresh <= row_j[h]));
                float &v = s[n][2 * h + c];
                v = seen ? (a.slopes ? v - row_slope[h] * (float)abs(row_at[h] - at) : v) : -INFINITY;
              }
            }
          }
        }
      });
    }
    cp_async_wait<0>();
    __syncthreads();

    // ---- the warps' shares of the keys put together: [key group][row][DP + 4] over the stages
    float *const merge = reinterpret_cast<float *>(data_ptr);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      run.l[h] += __shfl_xor_sync(0xffffffffu, run.l[h], 1);
      run.l[h] += __shfl_xor_sync(0xffffffffu, run.l[h], 2);
      const int row = warp * 16 + g + 8 * h;  // = (wk * WR + wr) * 16 + g + 8 h
      if (t == 0) { stats[2 * row] = run.m[h]; stats[2 * row + 1] = run.l[h]; }
#pragma unroll
      for (int n = 0; n < DP / 8; ++n)
        *reinterpret_cast<float2 *>(merge + row * (DP + 4) + 8 * n + 2 * t) = make_float2(run.o[n][2 * h], run.o[n][2 * h + 1]);
    }
    __syncthreads();
    const int n_rows = min(S::kRows, rows - row_base);
    const bool whole = tile0 == 0 && tile1 == key_tiles;
    float *const part = a.partial + ((int64_t)blockIdx.x * 2 + (front && tile0 > 0 ? 0 : 1)) * S::kPartial;
    auto put = [&](int row, int d, float v) {  // normalised context
      if (whole) {
        const int gr = row_base + row;
        static_cast<T *>(a.out)[(int64_t)(x.start + gr / a.group) * a.o_t + (int64_t)(kv * a.group + gr % a.group) * a.o_h + d * a.o_d] = from_f32<T>(v);
      } else {
        part[row * (DP + 2) + d] = v;
      }
    };
    for (int i = threadIdx.x; i < n_rows * DP; i += kThreads) {
      const int row = i / DP, d = i % DP;
      float m = -INFINITY, l = 0.0f, o = 0.0f;
#pragma unroll
      for (int w = 0; w < S::kWarpsK; ++w) m = fmaxf(m, stats[2 * (w * S::kRows + row)]);
      const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int w = 0; w < S::kWarpsK; ++w) {
        const float f = ex2_approx(stats[2 * (w * S::kRows + row)] - base);
        l += stats[2 * (w * S::kRows + row) + 1] * f;
        o += merge[(w * S::kRows + row) * (DP + 4) + d] * f;
      }
      const float v = l == 0.0f ? 0.0f : o / l;  // (no key seen: zeros)
      if (!(fabsf(v) <= 3.402823466e38f)) redo[row] = 1;
      if (d < a.D) put(row, d, v);
      if (d == 0 && !whole) { part[row * (DP + 2) + DP] = m; part[row * (DP + 2) + DP + 1] = l * F::kUnlift; }
    }
    __syncthreads();
    for (int row = warp; row < n_rows; row += S::kWarps) {
      if (!redo[row]) continue;
      const int gr = row_base + row;
      float *ctx = merge + row * (DP + 4);
      redo_row<T>(a, r, x, kv, gr / a.group, kv * a.group + gr % a.group, tile0 * S::kKeys, min(keys, tile1 * S::kKeys), ctx, stats + 2 * row);
      __syncwarp();
      for (int d = lane; d < a.D; d += 32) put(row, d, ctx[d]);
      if (lane == 0 && !whole) { part[row * (DP + 2) + DP] = stats[2 * row]; part[row * (DP + 2) + DP + 1] = stats[2 * row + 1]; }
    }
    unit += tile1 - tile0;
    front = false;
  }
}

// Rows whose keys several CTAs had: their parts in the order of the keys.  One warp per row (token, head).
template <typename T, int DP, int WR>
__global__ void __launch_bounds__(kJoinThreads) attention_tree_join_kernel(const __grid_constant__ TreeArgs a, int ctas) {
  using S = Shape<T, DP, WR>;
  pdl_prologue();
  const int lane = threadIdx.x & 31;
  const int64_t rows = a.tokens * a.heads, step = (int64_t)gridDim.x * (kJoinThreads / 32);
  const long long total = a.first[a.requests], share = (total + ctas - 1) / ctas;
  for (int64_t row = (int64_t)blockIdx.x * (kJoinThreads / 32) + (threadIdx.x >> 5); row < rows; row += step) {
    const int token = (int)(row / a.heads), head = (int)(row % a.heads), kv = head / a.group;
    // the request that the token belongs to (none: the row stays as it is).  Ranges may be anything, so all are asked.
    for (int r0 = 0; r0 < a.requests; r0 += 32) {
      Request x = {0, 0, 0};
      if (r0 + lane < a.requests) x = request_of(a, r0 + lane, false);
      unsigned mine = __ballot_sync(0xffffffffu, token >= x.start && token < x.start + x.fresh);
      while (mine) {
        const int from = __ffs(mine) - 1, r = r0 + from;
        mine &= mine - 1;
        Request y;
        y.start = __shfl_sync(0xffffffffu, x.start, from);
        y.fresh = __shfl_sync(0xffffffffu, x.fresh, from);
        y.context = __shfl_sync(0xffffffffu, x.context, from);
        const int key_tiles = max(1, (keys_of(a, y) + S::kKeys - 1) / S::kKeys), row_tiles = (y.fresh * a.group + S::kRows - 1) / S::kRows;
        const int in = (token - y.start) * a.group + head % a.group, rt = in / S::kRows, at = in % S::kRows;
        const long long u0 = a.first[r] + ((long long)kv * row_tiles + rt) * key_tiles, u1 = u0 + key_tiles - 1;
        const int c0 = (int)(u0 / share), c1 = (int)(u1 / share);
        if (c0 == c1) continue;
        auto part = [&](int c) { return a.partial + ((int64_t)c * 2 + (c == c0 ? 1 : 0)) * S::kPartial + at * (DP + 2); };
        // (c0's stretch begins inside it unless it begins at its very first unit, which is a slot 1 as well: its tile0 is 0)
        // 32 parts' maxima and sums at a time, one to a lane; then their contexts, whose loads do not wait for one another
        float m = -INFINITY, l = 0.0f, o[DP / 32];
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) o[i] = 0.0f;
        for (int c = c0; c <= c1; c += 32) {
          const int n = min(32, c1 - c + 1);
          const float pm = lane < n ? part(c + lane)[DP] : -INFINITY, pl = lane < n ? part(c + lane)[DP + 1] : 0.0f;
          float top = pm;
#pragma unroll
          for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
          top = fmaxf(top, m);
          const float base = top == -INFINITY ? 0.0f : top, keep = ex2_approx(m - base), w = pl == 0.0f ? 0.0f : pl * ex2_approx(pm - base);
          float sum = w;
#pragma unroll
          for (int k = 16; k; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
          m = top;
          l = l * keep + sum;
#pragma unroll
          for (int i = 0; i < DP / 32; ++i) o[i] *= keep;
#pragma unroll 4
          for (int k = 0; k < n; ++k) {
            const float *p = part(c + k);
            const float f = __shfl_sync(0xffffffffu, w, k);
            float v[DP / 32];
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) v[i] = lane + 32 * i < a.D ? p[lane + 32 * i] : 0.0f;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) o[i] += f == 0.0f ? 0.0f : f * v[i];
          }
        }
        T *out = static_cast<T *>(a.out) + (int64_t)token * a.o_t + (int64_t)head * a.o_h;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
          if (lane + 32 * i < a.D) out[(lane + 32 * i) * a.o_d] = from_f32<T>(l == 0.0f ? 0.0f : o[i] / l);
      }
    }
  }
}

// CTAs: two per SM, what shared memory leaves room for.
constexpr int kCtas = 2 * kSms;

// Rows of a tile by the average a request has: a wider tile reads the keys once for more rows, a narrower one has more warps
// on different keys.
int row_warps(int64_t requests, int64_t tokens, int64_t group) {
  const int64_t rows = requests > 0 ? (tokens * group + requests - 1) / requests : 0;
  return rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
}

template <typename T, int DP, int WR> int launch(const TreeArgs &a, cudaStream_t s) {
  using S = Shape<T, DP, WR>;
  static bool attr_set[64] = {false};
  int dev = 0;
  FML_CUDA(cudaGetDevice(&dev));
  if (!attr_set[dev & 63]) {
    FML_CUDA(cudaFuncSetAttribute(attention_tree_kernel<T, DP, WR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kBytes));
    attr_set[dev & 63] = true;
  }
  FML_LAUNCH((attention_tree_kernel<T, DP, WR>), kCtas, S::kThreads, S::kBytes, s, a);
  FML_LAUNCH((attention_tree_join_kernel<T, DP, WR>), grid_for(a.tokens * a.heads, kJoinThreads / 32, 4 * kSms), kJoinThreads, 0, s, a, kCtas);
  return FML_OK;
}
template <typename T, int DP> int launch(const TreeArgs &a, int warps, cudaStream_t s) {
  return warps == 1 ? launch<T, DP, 1>(a, s) : warps == 2 ? launch<T, DP, 2>(a, s) : launch<T, DP, 4>(a, s);
}
template <typename T> int launch(const TreeArgs &a, int warps, cudaStream_t s) {
  return a.D <= 64 ? launch<T, 64>(a, warps, s) : launch<T, 128>(a, warps, s);
}

}  // namespace
}  // namespace fml

using namespace fml;

namespace {
// Bytes of the counts of requests, and of them and the partial results for tiles of 16 * warps rows.
size_t counts_bytes(int64_t requests) { return (size_t)((requests + 1) * 8 + 15) / 16 * 16; }
size_t workspace_bytes_for(int64_t requests, int warps, int64_t head_size) {
  return counts_bytes(requests) + (size_t)kCtas * 2 * 16 * warps * ((head_size <= 64 ? 64 : 128) + 2) * 4;
}
}  // namespace

// The bound of every call of up to so many requests and tokens: all tokens may be one request's, and the tile is as high as its rows.
extern "C" size_t fml_attention_tree_workspace(int64_t requests, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_size) {
  if (requests < 0 || tokens < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || head_size < 1 || head_size > 128) return 0;
  return workspace_bytes_for(requests, row_warps(1, tokens, heads / kv_heads), head_size);
}

extern "C" int fml_attention_tree(const fml_tensor *q, const fml_tensor *k_cache, const fml_tensor *v_cache, const fml_tensor *block_table,
                                  const fml_tensor *context, const fml_tensor *query_start, const fml_tensor *tree, const fml_tensor *slopes,
                                  const fml_score_rules *rules, const fml_tensor *out, void *workspace, size_t workspace_bytes, void *stream) {
  FML_REQUIRE(data_tensor(q, 3) && data_tensor(out, 3) && data_tensor(k_cache, 4) && data_tensor(v_cache, 4), FML_BAD_ARG,
              "fml_attention_tree: q and out must be [tokens, heads, head size], the caches [pages, page size, kv heads, head size], of fp32, fp16 or bf16");
  FML_REQUIRE(out->dtype == q->dtype && k_cache->dtype == q->dtype && v_cache->dtype == q->dtype, FML_BAD_ARG, "fml_attention_tree: one type per call");
  FML_REQUIRE(rules && std::isfinite(rules->divisor) && rules->divisor != 0.0f && std::isfinite(rules->cap) && rules->cap >= 0.0f, FML_BAD_ARG,
              "fml_attention_tree: divisor must be finite and not zero, cap finite and not negative");
  FML_REQUIRE(factors_in_range(rules->divisor, rules->cap), FML_UNSUPPORTED,
              "fml_attention_tree: caps of 2^-64 to 2^64 (0: none), divisors with 1 / divisor and 1 / (divisor cap) in fp32's range");
  const int64_t tokens = q->shape[0], heads = q->shape[1], d = q->shape[2], pages = k_cache->shape[0], page = k_cache->shape[1],
                kv_heads = k_cache->shape[2];
  for (int i = 0; i < 3; ++i) FML_REQUIRE(out->shape[i] == q->shape[i], FML_BAD_ARG, "fml_attention_tree: shape of out");
  FML_REQUIRE(elements_apart(out), FML_BAD_ARG, "fml_attention_tree: out has a stride of 0");
  for (int i = 0; i < 4; ++i) FML_REQUIRE(v_cache->shape[i] == k_cache->shape[i], FML_BAD_ARG, "fml_attention_tree: the caches' shapes differ");
  FML_REQUIRE(k_cache->shape[3] == d, FML_BAD_ARG, "fml_attention_tree: head size of the caches");
  FML_REQUIRE(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, FML_BAD_ARG, "fml_attention_tree: heads must be a multiple of the caches' heads");
  const int esize = (int)data_size(q->dtype), per16 = 16 / esize;
  FML_REQUIRE(d >= 1 && d <= 128 && d % per16 == 0, FML_UNSUPPORTED, "fml_attention_tree: head sizes that are multiples of %d up to 128", per16);
  FML_REQUIRE(page >= 1 && page < (1ll << 31) && pages < (1ll << 31), FML_BAD_ARG, "fml_attention_tree: shape of the caches");
  FML_REQUIRE(tokens < (1ll << 24) && heads < (1 << 16) && tokens * heads < (1ll << 31) - 256, FML_UNSUPPORTED, "fml_attention_tree: too many tokens or heads");
  FML_REQUIRE(block_table && block_table->dtype == FML_I32 && index_tensor(block_table, 2), FML_BAD_ARG,
              "fml_attention_tree: block_table must be [requests, pages of a request] of int32");
  const int64_t requests = block_table->shape[0], columns = block_table->shape[1];
  FML_REQUIRE(requests < (1 << 24) && columns * page < (1ll << 31) - 256, FML_UNSUPPORTED, "fml_attention_tree: too many requests, or too many tokens per request");
  FML_REQUIRE(context && context->dtype == FML_I32 && index_tensor(context, 1) && context->shape[0] == requests, FML_BAD_ARG,
              "fml_attention_tree: context must be [requests] of int32");
  FML_REQUIRE(query_start && query_start->dtype == FML_I32 && index_tensor(query_start, 1) && query_start->shape[0] == requests + 1, FML_BAD_ARG,
              "fml_attention_tree: query_start must be [requests + 1] of int32");
  FML_REQUIRE(!tree || (tree->dtype == FML_I64 && index_tensor(tree, 1) && tree->shape[0] == tokens), FML_BAD_ARG,
              "fml_attention_tree: tree must be [tokens] of int64");
  FML_REQUIRE(!slopes || (float_tensor(slopes, 1) && slopes->shape[0] == heads), FML_BAD_ARG, "fml_attention_tree: slopes must be [heads] of fp32");
  if (tokens == 0 || requests == 0) return FML_OK;
  for (const fml_tensor *t : {k_cache, v_cache}) {
    FML_REQUIRE(t->stride[3] == 1 || d == 1, FML_MISALIGNED, "fml_attention_tree: the caches need unit stride along the head");
    bool ok = aligned16(t->data);
    for (int i = 0; i < 3; ++i) ok = ok && (t->shape[i] == 1 || t->stride[i] % per16 == 0);
    FML_REQUIRE(ok, FML_MISALIGNED, "fml_attention_tree: the caches' rows must lie on 16-byte boundaries");
  }
  const int warps = row_warps(requests, tokens, heads / kv_heads);
  const size_t need = workspace_bytes_for(requests, warps, d);
  FML_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need, FML_BAD_ARG,
              "fml_attention_tree: a 16-byte aligned workspace of %zu bytes is needed", need);
  FML_REQUIRE(inputs_on_current_device({q, k_cache, v_cache, block_table, context, query_start, tree, slopes}), FML_BAD_ARG,
              "fml_attention_tree: an input is not memory of the current device");
  FML_REQUIRE(on_current_device(out->data) && on_current_device(workspace), FML_BAD_ARG,
              "fml_attention_tree: the output or the workspace is not memory of the current device");
  TreeArgs a;
  memset(&a, 0, sizeof(a));
  a.q = q->data; a.out = out->data;
  a.k = pages ? k_cache->data : q->data; a.v = pages ? v_cache->data : q->data;  // (copies of nothing name an address all the same)
  a.table = static_cast<const int32_t *>(block_table->data);
  a.context = static_cast<const int32_t *>(context->data);
  a.query_start = static_cast<const int32_t *>(query_start->data);
  a.tree = tree ? static_cast<const int64_t *>(tree->data) : nullptr;
  a.slopes = slopes ? static_cast<const float *>(slopes->data) : nullptr;
  a.q_t = q->stride[0]; a.q_h = q->stride[1]; a.q_d = q->stride[2];
  a.q_vec = a.q_d == 1 && aligned16(q->data) && (tokens == 1 || a.q_t % per16 == 0) && (heads == 1 || a.q_h % per16 == 0);
  a.o_t = out->stride[0]; a.o_h = out->stride[1]; a.o_d = out->stride[2];
  a.k_page = k_cache->stride[0]; a.k_pos = k_cache->stride[1]; a.k_head = k_cache->stride[2];
  a.v_page = v_cache->stride[0]; a.v_pos = v_cache->stride[1]; a.v_head = v_cache->stride[2];
  a.alike = a.k_page == a.v_page && a.k_pos == a.v_pos && a.k_page >= 0 && a.k_pos >= 0;
  a.table_r = block_table->stride[0]; a.table_c = block_table->stride[1];
  a.context_s = context->stride[0]; a.start_s = query_start->stride[0];
  a.tree_s = tree ? tree->stride[0] : 0; a.slopes_s = slopes ? slopes->stride[0] : 0;
  a.pages = pages; a.tokens = tokens;
  a.requests = (int)requests; a.columns = (int)columns; a.page = (int)page;
  a.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (page == (1ll << i)) a.page_shift = i;
  a.heads = (int)heads; a.kv_heads = (int)kv_heads; a.group = (int)(heads / kv_heads); a.D = (int)d;
  a.cap = Cap::make(rules->divisor, rules->cap);
  a.first = static_cast<long long *>(workspace);
  a.partial = reinterpret_cast<float *>(static_cast<char *>(workspace) + counts_bytes(requests));
  a.status = device_status_word();
  FML_REQUIRE(a.status, FML_CUDA_ERROR, "fml_attention_tree: no device status word");
  if (q->dtype == FML_F32) return launch<float>(a, warps, as_stream(stream));
  if (q->dtype == FML_F16) return launch<__half>(a, warps, as_stream(stream));
  return launch<__nv_bfloat16>(a, warps, as_stream(stream));
}
