// Shared by the recurrences over tokens (conv_kernels.cu, scan_*.cu): types, sequences of a batch, rows that share a slot.
#pragma once
#include "common.cuh"

namespace lasp {

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f(float x) { return x; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }

// Element i of a parameter that is kept in fp32 or in the type of the activations.
template <typename T>
__device__ __forceinline__ float param(const void* p, bool f32, int64_t i) {
  return f32 ? static_cast<const float*>(p)[i] : to_f(static_cast<const T*>(p)[i]);
}
template <typename T>
__device__ __forceinline__ void store_param(void* p, bool f32, int64_t i, float x) {
  if (f32)
    static_cast<float*>(p)[i] = x;
  else
    static_cast<T*>(p)[i] = from_f<T>(x);
}

// V neighbouring elements, by one access where V > 1 (the launcher has looked at addresses and pitches).
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&out)[V]) {
  const Vec<T, V> x = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = to_f(x.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[V]) {
  Vec<T, V> x;
#pragma unroll
  for (int i = 0; i < V; ++i) x.v[i] = from_f<T>(in[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = x;
}

__device__ __forceinline__ int64_t index_at(const void* p, int bits, int64_t i) {
  return bits == 64 ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int32_t*>(p)[i];
}

// Offsets come from the device and are taken as they are only within the row.
struct Sequences {
  const void* offsets;
  int bits, count, tokens;
  __device__ __forceinline__ int at(int i) const {
    const int64_t o = index_at(offsets, bits, i);
    return (int)(o < 0 ? 0 : o > tokens ? tokens : o);
  }
  __device__ __forceinline__ void bounds(int i, int* begin, int* end) const {
    *begin = at(i);
    const int e = at(i + 1);
    *end = e > *begin ? e : *begin;
  }
  // the last sequence that begins at or before token t, -1 where none does
  __device__ __forceinline__ int find(int t) const {
    int lo = 0, hi = count;   // (sequences [0, lo) begin at or before t)
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (at(mid) <= t)
        lo = mid + 1;
      else
        hi = mid;
    }
    return lo - 1;
  }
};

// Rows of a step that name the same slot are consecutive tokens: the first of them takes the others along.  Every thread of the
// block calls this.  Returns -1 where an earlier row has the slot, 1 where a later one has, else 0.
__device__ __forceinline__ int shared_slot(const void* slots, int bits, int rows, int row, int64_t slot) {
  if (!slots || rows == 1) return 0;
  int before = 0, after = 0;
  for (int j = threadIdx.x + threadIdx.y * blockDim.x; j < rows; j += blockDim.x * blockDim.y)
    if (j != row && index_at(slots, bits, j) == slot) (j < row ? before : after) = 1;
  before = __syncthreads_or(before);
  after = __syncthreads_or(after);
  return before ? -1 : after;
}

// x sigmoid(x) and its derivative; 1 / (1 + e^-x) by the fast exponential and division (2^-21 relative, where the result is
// rounded to fp32's 2^-24 at best): an infinite e^-x gives 0.
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }
__device__ __forceinline__ float silu(float x) { return x * sigmoid(x); }
__device__ __forceinline__ float d_silu(float x) {
  const float s = sigmoid(x);
  return s + x * s * (1.f - s);
}

inline bool vector_ok(const lasp_tokens& t, size_t item) {
  return !t.data || ((reinterpret_cast<uintptr_t>(t.data) | (size_t)(t.row_pitch * (int64_t)item) | (size_t)(t.token_pitch * (int64_t)item)) & 15) == 0;
}
inline bool vector_ok(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

cudaError_t conv_forward(const lasp_conv_args& a, cudaStream_t st);
cudaError_t conv_backward(const lasp_conv_args& a, cudaStream_t st);
size_t conv_workspace(const lasp_conv_args& a);
cudaError_t conv_step(const lasp_conv_step_args& a, cudaStream_t st);
cudaError_t scan_forward(const lasp_scan_args& a, cudaStream_t st);
cudaError_t scan_backward(const lasp_scan_args& a, cudaStream_t st);
size_t scan_kept(const lasp_scan_args& a);
size_t scan_workspace(const lasp_scan_args& a);
cudaError_t scan_step(const lasp_scan_step_args& a, cudaStream_t st);

}  // namespace lasp
