// What the operators of a decoder's serving step share (rotary_positions.cu, attention_rules.cu, attention_tree.cu,
// sample.cu): their element types, operand checks and small device helpers.
#pragma once
#include "common.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <initializer_list>

namespace fml {

// Bytes of an element of the types these operators take as data; 0: none of them.
inline size_t data_size(int dtype) { return dtype == FML_F32 ? 4 : dtype == FML_F16 || dtype == FML_BF16 ? 2 : 0; }

// A described tensor of `rank` dims with elements of `size` bytes (0: a type that is not taken) whose extents are not
// negative; data may be null only when it is empty, and lies on a multiple of an element.
inline bool described(const fml_tensor *t, int rank, size_t size) {
  if (!t || t->rank != rank || size == 0) return false;
  int64_t n = 1;
  for (int i = 0; i < rank; ++i) {
    if (t->shape[i] < 0 || t->shape[i] > (1ll << 40)) return false;
    n = t->shape[i] && n > (1ll << 50) / t->shape[i] ? (1ll << 51) : n * t->shape[i];
    if (n > (1ll << 50)) return false;
  }
  return n == 0 || (t->data != nullptr && reinterpret_cast<uintptr_t>(t->data) % size == 0);
}
inline bool data_tensor(const fml_tensor *t, int rank) { return t && described(t, rank, data_size(t->dtype)); }
inline bool index_tensor(const fml_tensor *t, int rank) { return t && described(t, rank, t->dtype == FML_I64 ? 8 : t->dtype == FML_I32 ? 4 : 0); }
inline bool float_tensor(const fml_tensor *t, int rank) { return t && described(t, rank, t->dtype == FML_F32 ? 4 : 0); }

// Whether an output's elements along each dim are apart: with a stride of 0 several results would go to one place.
inline bool elements_apart(const fml_tensor *t) {
  for (int i = 0; i < t->rank; ++i)
    if (t->shape[i] > 1 && t->stride[i] == 0) return false;
  return true;
}

// Whether memory of the current device (or memory every device sees) is at `p`: a launch on another device's memory would
// fault there.  Unregistered host memory is not.
inline bool on_current_device(const void *p) {
  cudaPointerAttributes at;
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaPointerGetAttributes(&at, p) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  return at.type == cudaMemoryTypeManaged || at.type == cudaMemoryTypeHost || (at.type == cudaMemoryTypeDevice && at.device == dev);
}

// The same of a call's inputs (null and empty ones are not read).  With one device they can only be its own, and are not asked:
// that is a call into the driver for each.
inline bool inputs_on_current_device(std::initializer_list<const fml_tensor *> inputs) {
  static const int devices = [] {
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    return n;
  }();
  if (devices == 1) return true;
  for (const fml_tensor *t : inputs)
    if (t && numel(t) > 0 && !on_current_device(t->data)) return false;
  return true;
}

// Integers of either width, read one by one.
struct IndexView {
  const void *p;
  int64_t stride;
  int wide;
};
inline IndexView index_view(const fml_tensor *t) {
  IndexView v = {nullptr, 0, 0};
  if (t) { v.p = t->data; v.stride = t->stride[t->rank - 1]; v.wide = t->dtype == FML_I64; }
  return v;
}
__device__ __forceinline__ int64_t index_at(const IndexView &v, int64_t i) {
  return v.wide ? static_cast<const int64_t *>(v.p)[i * v.stride] : (int64_t)static_cast<const int32_t *>(v.p)[i * v.stride];
}

// fp32 value of an element, and a value rounded to the type (to nearest, ties to even).
template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

}  // namespace fml
