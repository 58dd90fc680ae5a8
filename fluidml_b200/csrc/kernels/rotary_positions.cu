// Rotary positions with the append to a paged cache (fml_rotary_positions), and the frequencies of the usual scalings
// (fml_rotary_frequencies).
//
//   (x1, x2) -> (x1 c - x2 s, x2 c + x1 s),  c, s = magnitude * cos, sin(position * frequency)
//
// What bounds it: every feature is read and written once and nothing else moves.  The angle is formed and reduced in pairs
// of 64-bit numbers (a position of a million times a frequency of one radian leaves fp32 no digits below 0.06); the reduction
// happens in turns, so that the fraction is exact, and the functions are evaluated in fp32 on an argument of at most half a turn.  A CTA
// computes them once per token, into shared memory, for all the token's heads.  Measured: 8191 tokens of 32 + 2 x 8 heads of 128,
// bf16, into a cache 42 us, 4.8 TB/s (74 % of a measured copy); eight tokens of the fp32 decoder 3.5 us, a launch.
#include "serving_common.cuh"
#include <algorithm>
#include <cmath>

namespace fml {
namespace {

constexpr int kThreads = 256;

// n / d for n d < 2^32, by a multiplication (an integer division is some twenty instructions, of about a hundred for 16 bytes).
struct SmallDivisor {
  uint32_t m;
  __host__ explicit SmallDivisor(int d = 1) : m(d > 1 ? (uint32_t)(0x100000000ull / (uint32_t)d + (0x100000000ull % (uint32_t)d != 0)) : 0) {}
  __device__ __forceinline__ int operator()(int n) const { return m ? (int)__umulhi((uint32_t)n, m) : n; }
};

struct RotaryPart {  // q, k or v: [tokens, heads, head size] in, the same or a paged cache out
  const void *in;
  void *out;
  int64_t in_t, in_h, in_d;         // element strides
  int64_t out_t, out_h, out_d;      // out_t: of a token, or of a position in its page
  int64_t out_page;                 // of a page (paged)
  int heads, units, turned, paged;  // units of a head; of which `turned` are rotated
  SmallDivisor by_units;
};

struct RotaryPositionsArgs {
  RotaryPart part[3];
  IndexView positions, slots;
  const float *frequencies;
  int64_t freq_stride, tokens, capacity;  // capacity: pages * page size
  float magnitude;
  int page, half, interleaved, per_token, tokens_per_cta;  // per_token: units of a token
  int ends[2];                                             // units of q, of q and k
  SmallDivisor by_token, by_half;
  int *status;
};

template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T x[V]; };

// V features per access.  Halves: a unit turns V pairs (two accesses, rot / 2 apart).  Interleaved: a unit turns V / 2
// adjacent pairs of one access (V = 1: one pair, two accesses).  Units beyond the turned ones copy V features.
template <typename T, int V> __global__ void __launch_bounds__(kThreads) rotary_positions_kernel(const __grid_constant__ RotaryPositionsArgs a) {
  extern __shared__ float2 table[];  // [token of the CTA][pair]: cos, sin
  __shared__ int64_t where[kThreads];   // page << 32 | position in it; -1: no slot
  pdl_prologue();
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens_per_cta;
  const int n = (int)min((int64_t)a.tokens_per_cta, a.tokens - t0);
  for (int i = threadIdx.x; i < n * a.half; i += kThreads) {
    const int t = a.by_half(i), j = i - t * a.half;
    // position * frequency / 2 pi with what each product rounds away (1 / 2 pi as two numbers), and beyond 2^53 the position's low
    // bits apart, which a double does not hold: the fraction is good to 2^-40 for frequencies up to one radian and any position
    // that 64 bits hold, to 2^-50 below 2^53.  What was rounded away may be turns again, so the sum is reduced once more.
    const int64_t at = index_at(a.positions, t0 + t), low = at >= (1ll << 53) || at <= -(1ll << 53) ? at & 2047 : 0;
    const double pos = (double)(at - low), f = (double)a.frequencies[j * a.freq_stride];
    const double angle = pos * f, turns = angle * 0.15915494309189535;
    const double rest = fma(angle, 0.15915494309189535, -turns) + (angle * -9.839338337591243e-18 + fma(pos, f, -angle) * 0.15915494309189535) +
                        (double)low * f * 0.15915494309189535;
    const double part = (turns - rint(turns)) + rest;
    float s, c;
    sincospif((float)(2.0 * (part - rint(part))), &s, &c);
    table[i] = make_float2(a.magnitude * c, a.magnitude * s);
  }
  if (a.slots.p && threadIdx.x < n) {
    const int64_t slot = index_at(a.slots, t0 + threadIdx.x);
    where[threadIdx.x] = -1;
    if (slot >= 0 && slot < a.capacity) {
      const int64_t page = slot < (1ll << 31) ? (int64_t)((uint32_t)slot / (uint32_t)a.page) : slot / a.page;
      where[threadIdx.x] = page << 32 | (slot - page * a.page);
    }
    else if (slot >= 0) atomicOr(a.status, kStatusIndexRange);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n * a.per_token; i += kThreads) {
    const int t = a.by_token(i);
    int u = i - t * a.per_token;
    const int which = u < a.ends[0] ? 0 : u < a.ends[1] ? 1 : 2;
    if (which) u -= a.ends[which - 1];
    const RotaryPart &p = a.part[which];
    const int h = p.by_units(u);
    u -= h * p.units;
    const T *src = static_cast<const T *>(p.in) + (t0 + t) * p.in_t + h * p.in_h;
    T *dst = static_cast<T *>(p.out) + h * p.out_h;
    if (p.paged) {
      const int64_t w = where[t];
      if (w < 0) continue;
      dst += (w >> 32) * p.out_page + (w & 0xffffffff) * p.out_t;
    } else {
      dst += (t0 + t) * p.out_t;
    }
    const float2 *cs = table + t * a.half;
    using Access = Vec<T, V>;
    if (u >= p.turned) {  // behind the turned features (a pair is two of them when V = 1 turns adjacent ones)
      const int d = (a.interleaved && V == 1 ? u + p.turned : a.interleaved ? u * V : (u + p.turned) * V);
      if (V == 1) dst[d * p.out_d] = src[d * p.in_d];
      else *reinterpret_cast<Access *>(dst + d) = *reinterpret_cast<const Access *>(src + d);
    } else if (V == 1) {
      const int d1 = a.interleaved ? 2 * u : u, d2 = a.interleaved ? 2 * u + 1 : u + a.half;
      const float x1 = to_f32(src[d1 * p.in_d]), x2 = to_f32(src[d2 * p.in_d]);
      const float2 f = cs[u];
      dst[d1 * p.out_d] = from_f32<T>(x1 * f.x - x2 * f.y);
      dst[d2 * p.out_d] = from_f32<T>(x2 * f.x + x1 * f.y);
    } else if (a.interleaved) {
      Access x = *reinterpret_cast<const Access *>(src + u * V);
#pragma unroll
      for (int i2 = 0; i2 + 1 < V; i2 += 2) {
        const float2 f = cs[(u * V + i2) >> 1];
        const float x1 = to_f32(x.x[i2]), x2 = to_f32(x.x[i2 + 1]);
        x.x[i2] = from_f32<T>(x1 * f.x - x2 * f.y);
        x.x[i2 + 1] = from_f32<T>(x2 * f.x + x1 * f.y);
      }
      *reinterpret_cast<Access *>(dst + u * V) = x;
    } else {
      Access x = *reinterpret_cast<const Access *>(src + u * V), y = *reinterpret_cast<const Access *>(src + u * V + a.half);
#pragma unroll
      for (int i2 = 0; i2 < V; ++i2) {
        const float2 f = cs[u * V + i2];
        const float x1 = to_f32(x.x[i2]), x2 = to_f32(y.x[i2]);
        x.x[i2] = from_f32<T>(x1 * f.x - x2 * f.y);
        y.x[i2] = from_f32<T>(x2 * f.x + x1 * f.y);
      }
      *reinterpret_cast<Access *>(dst + u * V) = x;
      *reinterpret_cast<Access *>(dst + u * V + a.half) = y;
    }
  }
}

template <typename T> int launch(RotaryPositionsArgs &a, int v, int64_t head, cudaStream_t s) {
  const int rot = 2 * a.half;
  for (int i = 0, per = 0; i < 3; ++i) {
    RotaryPart &p = a.part[i];
    if (!p.in) p.heads = 0;
    const int r = i == 2 ? 0 : rot;  // values are not turned
    p.turned = a.interleaved ? (v == 1 ? r / 2 : r / v) : r / 2 / v;
    p.units = p.turned + (int)((head - r) / v);
    per += p.heads * p.units;
    a.per_token = per;
    if (i < 2) a.ends[i] = per;
    p.by_units = SmallDivisor(p.units);
    FML_REQUIRE((int64_t)per * std::max(p.units, 1) < (1ll << 32), FML_UNSUPPORTED, "fml_rotary_positions: too many features");
  }
  if (a.tokens == 0 || a.per_token == 0) return FML_OK;
  // a CTA takes as many tokens as give every thread a unit, and one when a token alone has more
  a.tokens_per_cta = std::max(1, std::min(kThreads / std::max(1, a.per_token), kThreads));
  // long prompts: two, so that fewer barriers wait for angles (8191 tokens of 32 + 2 x 8 heads of 128, bf16: 45 -> 42 us; four: 42)
  if (a.tokens_per_cta == 1 && a.tokens >= 2ll * kSms * 8 && 2ll * a.per_token * a.per_token < (1ll << 32)) a.tokens_per_cta = 2;
  a.by_token = SmallDivisor(a.per_token);
  a.by_half = SmallDivisor(a.half);
  FML_REQUIRE((int64_t)a.per_token * a.tokens_per_cta * a.per_token < (1ll << 32) || a.tokens_per_cta == 1, FML_UNSUPPORTED,
              "fml_rotary_positions: too many features");
  if (a.tokens_per_cta == 1 && (int64_t)a.per_token * a.per_token >= (1ll << 32)) a.by_token.m = 1u;  // (n / per_token is 0: so is n * 1 >> 32)
  const int64_t ctas = (a.tokens + a.tokens_per_cta - 1) / a.tokens_per_cta;
  const size_t smem = (size_t)a.tokens_per_cta * a.half * sizeof(float2);
  FML_REQUIRE(ctas < (1ll << 31) && smem <= 40 * 1024, FML_UNSUPPORTED, "fml_rotary_positions: too many tokens or features");
  if (sizeof(T) == 2 && v == 8) FML_LAUNCH((rotary_positions_kernel<T, sizeof(T) == 2 ? 8 : 1>), (unsigned)ctas, kThreads, smem, s, a);
  else if (v == 4) FML_LAUNCH((rotary_positions_kernel<T, 4>), (unsigned)ctas, kThreads, smem, s, a);
  else if (v == 2) FML_LAUNCH((rotary_positions_kernel<T, 2>), (unsigned)ctas, kThreads, smem, s, a);
  else FML_LAUNCH((rotary_positions_kernel<T, 1>), (unsigned)ctas, kThreads, smem, s, a);
  FML_CUDA(cudaGetLastError());
  return FML_OK;
}

}  // namespace
}  // namespace fml

using namespace fml;

extern "C" int fml_rotary_positions(const fml_tensor *q, const fml_tensor *k, const fml_tensor *v, const fml_tensor *positions,
                                    const fml_tensor *slots, const fml_tensor *frequencies, float magnitude, int layout,
                                    const fml_tensor *q_out, const fml_tensor *k_out, const fml_tensor *v_out, void *stream) {
  const fml_tensor *in[3] = {q, k, v}, *out[3] = {q_out, k_out, v_out};
  const fml_tensor *first = q ? q : k ? k : v;
  FML_REQUIRE(first, FML_BAD_ARG, "fml_rotary_positions: none of q, k, v");
  FML_REQUIRE(layout == FML_ROTARY_HALVES || layout == FML_ROTARY_INTERLEAVED, FML_BAD_ARG, "fml_rotary_positions: no such layout (%d)", layout);
  FML_REQUIRE(data_tensor(first, 3), FML_BAD_ARG, "fml_rotary_positions: q, k, v must be [tokens, heads, head size] of fp32, fp16 or bf16");
  const int64_t tokens = first->shape[0], head = first->shape[2];
  FML_REQUIRE(index_tensor(positions, 1) && positions->shape[0] == tokens, FML_BAD_ARG,
              "fml_rotary_positions: positions must be [tokens] of int32 or int64");
  FML_REQUIRE(!slots || (index_tensor(slots, 1) && slots->shape[0] == tokens), FML_BAD_ARG,
              "fml_rotary_positions: slots must be [tokens] of int32 or int64");
  FML_REQUIRE(float_tensor(frequencies, 1) && 2 * frequencies->shape[0] <= head && frequencies->shape[0] <= 2048, FML_BAD_ARG,
              "fml_rotary_positions: frequencies must be fp32, one per pair of rotated features (at most half of the head, at most 2048)");
  FML_REQUIRE(std::isfinite(magnitude), FML_BAD_ARG, "fml_rotary_positions: magnitude is not finite");
  FML_REQUIRE(!slots || k || v, FML_BAD_ARG, "fml_rotary_positions: slots without keys or values");
  RotaryPositionsArgs a;
  memset(static_cast<void *>(&a), 0, sizeof(a));
  a.positions = index_view(positions);
  a.slots = index_view(slots);
  a.frequencies = static_cast<const float *>(frequencies->data);
  a.freq_stride = frequencies->stride[0];
  a.tokens = tokens;
  a.magnitude = magnitude;
  a.half = (int)frequencies->shape[0];
  a.interleaved = layout == FML_ROTARY_INTERLEAVED;
  const int rot = 2 * a.half, esize = (int)data_size(first->dtype);
  int64_t features = 0;  // of a token
  // the widest access that rotated part, rest, strides and addresses allow
  int width = 16 / esize;
  auto fits = [&](int64_t x) { while (width > 1 && x % width != 0) width >>= 1; };
  fits(head);
  fits(a.interleaved ? rot : a.half);
  for (int i = 0; i < 3; ++i) {
    const char *name = i == 0 ? "q" : i == 1 ? "k" : "v";
    const bool paged = slots && i > 0;
    FML_REQUIRE(!in[i] == !out[i], FML_BAD_ARG, "fml_rotary_positions: %s without its output, or the other way round", name);
    if (!in[i]) continue;
    FML_REQUIRE(data_tensor(in[i], 3) && data_tensor(out[i], paged ? 4 : 3) && in[i]->dtype == first->dtype && out[i]->dtype == first->dtype,
                FML_BAD_ARG, "fml_rotary_positions: %s and its output must be of one type and rank 3 (a paged cache: 4)", name);
    FML_REQUIRE(in[i]->shape[0] == tokens && in[i]->shape[2] == head && in[i]->shape[1] < (1 << 20), FML_BAD_ARG,
                "fml_rotary_positions: shape of %s", name);
    features += in[i]->shape[1] * head;
    FML_REQUIRE(features < (1ll << 31), FML_UNSUPPORTED, "fml_rotary_positions: too many features");  // (units are counted in 32 bits)
    const int r = paged ? 2 : 1;
    FML_REQUIRE(out[i]->shape[r] == in[i]->shape[1] && out[i]->shape[r + 1] == head && (paged || out[i]->shape[0] == tokens), FML_BAD_ARG,
                "fml_rotary_positions: shape of %s's output", name);
    FML_REQUIRE(elements_apart(out[i]), FML_BAD_ARG, "fml_rotary_positions: %s's output has a stride of 0", name);
    RotaryPart &p = a.part[i];
    p.in = in[i]->data; p.out = out[i]->data;
    p.heads = (int)in[i]->shape[1]; p.paged = paged;
    p.in_t = in[i]->stride[0]; p.in_h = in[i]->stride[1]; p.in_d = in[i]->stride[2];
    p.out_page = paged ? out[i]->stride[0] : 0;
    p.out_t = out[i]->stride[r - 1]; p.out_h = out[i]->stride[r]; p.out_d = out[i]->stride[r + 1];
    // in place: every thread writes what it alone has read, so only the same places in the same order
    FML_REQUIRE(p.in != p.out || (!paged && p.in_t == p.out_t && p.in_h == p.out_h && p.in_d == p.out_d), FML_BAD_ARG,
                "fml_rotary_positions: %s in place needs the output's strides to be the input's", name);
    if (paged) {
      const int64_t pages = out[i]->shape[0], page = out[i]->shape[1];
      FML_REQUIRE(page < (1ll << 31) && pages < (1ll << 31), FML_BAD_ARG, "fml_rotary_positions: shape of the cache");
      FML_REQUIRE(!(i == 2 && k) || (pages * page == a.capacity && page == a.page), FML_BAD_ARG,
                  "fml_rotary_positions: the caches of k and v must have the same pages");
      a.capacity = pages * page; a.page = (int)std::max<int64_t>(page, 1);
    }
    if (tokens == 0 || p.heads == 0 || head == 0) { p.in = nullptr; continue; }
    if (paged && numel(out[i]) == 0) { p.out = nullptr; }  // no page: every slot is out of range
    if (p.in_d != 1 || p.out_d != 1) width = 1;
    for (const int64_t x : {p.in_t, p.in_h, p.out_t, p.out_h, p.out_page}) fits(x);
    fits((int64_t)(reinterpret_cast<uintptr_t>(p.in) / esize));
    fits((int64_t)(reinterpret_cast<uintptr_t>(p.out) / esize));
  }
  FML_REQUIRE(inputs_on_current_device({q, k, v, positions, slots, frequencies}), FML_BAD_ARG,
              "fml_rotary_positions: an input is not memory of the current device");
  for (const RotaryPart &p : a.part)
    FML_REQUIRE(!p.in || !p.out || on_current_device(p.out), FML_BAD_ARG, "fml_rotary_positions: an output is not memory of the current device");
  a.status = device_status_word();
  FML_REQUIRE(a.status, FML_CUDA_ERROR, "fml_rotary_positions: no device status word");
  if (first->dtype == FML_F32) return launch<float>(a, width, head, as_stream(stream));
  if (first->dtype == FML_F16) return launch<__half>(a, width, head, as_stream(stream));
  return launch<__nv_bfloat16>(a, width, head, as_stream(stream));
}

extern "C" int fml_rotary_frequencies(const fml_rotary_spec *spec, float *frequencies, float *magnitude) {
  FML_REQUIRE(spec && frequencies && magnitude, FML_BAD_ARG, "fml_rotary_frequencies: null argument");
  FML_REQUIRE(spec->rot >= 2 && (spec->rot & 1) == 0 && spec->rot <= 4096, FML_BAD_ARG, "fml_rotary_frequencies: rot must be even, 2 to 4096");
  FML_REQUIRE(std::isfinite(spec->base) && spec->base > 1.0, FML_BAD_ARG, "fml_rotary_frequencies: base must be above 1");
  FML_REQUIRE(spec->scaling >= FML_ROTARY_PLAIN && spec->scaling <= FML_ROTARY_RAMP, FML_BAD_ARG, "fml_rotary_frequencies: no such scaling (%d)",
              spec->scaling);
  const bool scaled = spec->scaling != FML_ROTARY_PLAIN, by_turns = spec->scaling == FML_ROTARY_BANDS || spec->scaling == FML_ROTARY_RAMP;
  FML_REQUIRE(!scaled || (std::isfinite(spec->factor) && spec->factor >= 1.0), FML_BAD_ARG, "fml_rotary_frequencies: factor must be at least 1");
  FML_REQUIRE(spec->scaling != FML_ROTARY_NTK || spec->rot > 2, FML_BAD_ARG, "fml_rotary_frequencies: a scaled base needs more than one pair");
  FML_REQUIRE(!by_turns || (std::isfinite(spec->trained_length) && spec->trained_length > 0 && std::isfinite(spec->turns_high) &&
                            spec->turns_low > 0 && spec->turns_high > spec->turns_low),
              FML_BAD_ARG, "fml_rotary_frequencies: trained_length above 0 and 0 < turns_low < turns_high are needed");
  const double pi = 3.14159265358979323846, rot = spec->rot, half = rot / 2;
  double base = spec->base;
  if (spec->scaling == FML_ROTARY_NTK) base *= std::pow(spec->factor, rot / (rot - 2.0));
  // the pair that turns `turns` times over the trained length, as a real number
  auto pair_of = [&](double turns) { return half * std::log(spec->trained_length / (turns * 2.0 * pi)) / std::log(spec->base); };
  double lo = 0, hi = 1;
  if (spec->scaling == FML_ROTARY_RAMP) {
    lo = std::max(std::floor(pair_of(spec->turns_high)), 0.0);
    hi = std::min(std::ceil(pair_of(spec->turns_low)), rot - 1.0);
    hi = std::max(hi, lo + 0.001);  // (a ramp without width is a step)
  }
  for (int i = 0; i < spec->rot / 2; ++i) {
    double f = std::pow(base, -2.0 * i / rot), keep = 1.0;
    if (spec->scaling == FML_ROTARY_LINEAR) keep = 0.0;
    if (spec->scaling == FML_ROTARY_BANDS)
      keep = (spec->trained_length * f / (2.0 * pi) - spec->turns_low) / (spec->turns_high - spec->turns_low);
    if (spec->scaling == FML_ROTARY_RAMP) keep = 1.0 - (i - lo) / (hi - lo);
    keep = std::min(std::max(keep, 0.0), 1.0);
    frequencies[i] = (float)(f * (keep + (scaled && spec->scaling != FML_ROTARY_NTK ? (1.0 - keep) / spec->factor : 1.0 - keep)));
  }
  *magnitude = spec->scaling == FML_ROTARY_RAMP ? (float)(0.1 * std::log(spec->factor) + 1.0) : 1.0f;
  return FML_OK;
}
