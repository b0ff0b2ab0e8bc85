// Shared by the recurrences over tokens (conv_kernels.cu, scan_*.cu): types, sequences of a batch, rows that share a slot.
#pragma once
#include <string.h>

#include <type_traits>

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
// Arithmetic on pairs, one instruction for two fp32 values.  A pair is kept as the 64 bits that those instructions take: taken apart
// and put together again it would cost a move each time (a third of all instructions, when it was).
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void apart(F2 p, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p.v)); }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}

// Two neighbouring 16-bit numbers are a word, which is taken apart and put together whole (two instructions and one).
template <typename T>
__device__ __forceinline__ F2 pair_from(const T* two) {
  if constexpr (sizeof(T) == 4) {
    return f2(two[0], two[1]);
  } else {
    uint32_t w;
    memcpy(&w, two, 4);
    if constexpr (std::is_same<T, __half>::value) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
      return f2(v.x, v.y);
    } else {
      return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
  }
}
template <typename T>
__device__ __forceinline__ void pair_to(T* two, float x, float y) {
  if constexpr (sizeof(T) == 4) {
    two[0] = x, two[1] = y;
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 v = __floats2half2_rn(x, y);
    memcpy(two, &v, 4);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    memcpy(two, &v, 4);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[V]) {
  Vec<T, V> x;
  if constexpr (V % 2) {
#pragma unroll
    for (int i = 0; i < V; ++i) x.v[i] = from_f<T>(in[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) pair_to(&x.v[i], in[i], in[i + 1]);
  }
  *reinterpret_cast<Vec<T, V>*>(p) = x;
}

// x sigmoid(x) and its derivative; 1 / (1 + e^-x) by the fast exponential and reciprocal (2^-21 relative, where the result is
// rounded to fp32's 2^-24 at best): an infinite e^-x gives 0.
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float sigmoid(float x) { return reciprocal(1.f + ex2(-kLog2e * x)); }
__device__ __forceinline__ float silu(float x) { return x * sigmoid(x); }
__device__ __forceinline__ float d_silu(float x) {
  const float s = sigmoid(x);
  return s + x * s * (1.f - s);
}

__device__ __forceinline__ F2 sigmoid(F2 p) {
  float x, y;
  apart(mul2(p, f2(-kLog2e, -kLog2e)), x, y);
  apart(add2(f2(ex2(x), ex2(y)), f2(1.f, 1.f)), x, y);
  return f2(reciprocal(x), reciprocal(y));
}
__device__ __forceinline__ F2 silu(F2 p) { return mul2(p, sigmoid(p)); }
// s + (s p - s (s p)): the difference, exactly zero where s is one, before the sum, since p may be so large that p + 1 is no fp32 number any more
__device__ __forceinline__ F2 d_silu(F2 p) {
  const F2 s = sigmoid(p), sp = mul2(s, p);
  return add2(s, fma2(mul2(s, f2(-1.f, -1.f)), sp, sp));
}

// V neighbouring channels as pairs; of a single channel the other half is zero.
template <int V>
struct Channels {
  static constexpr int kPairs = (V + 1) / 2;
  F2 p[kPairs];
  template <typename T>
  __device__ __forceinline__ void set(const Vec<T, V>& x) {
#pragma unroll
    for (int k = 0; k < kPairs; ++k)
      if constexpr (V > 1)
        p[k] = pair_from(&x.v[2 * k]);
      else
        p[k] = f2(to_f(x.v[0]), 0.f);
  }
  template <typename T>
  __device__ __forceinline__ void load(const T* from) { set(*reinterpret_cast<const Vec<T, V>*>(from)); }
  template <typename T>
  __device__ __forceinline__ void store(T* to) const {
    Vec<T, V> v;
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      float x, y;
      apart(p[k], x, y);
      if constexpr (V > 1)
        pair_to(&v.v[2 * k], x, y);
      else
        v.v[0] = from_f<T>(x);
    }
    *reinterpret_cast<Vec<T, V>*>(to) = v;
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < kPairs; ++k) p[k] = f2(0.f, 0.f);
  }
};
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

// Single tokens: a block takes some channels of kStepRows rows at most, so that what belongs to the channels is read once.  Rows that name
// the same slot are consecutive tokens: the first of them takes the others along.
constexpr int kStepRows = 32;
struct StepRows {
  int64_t slot[kStepRows];
  uint32_t before, after;   // a bit for each row: an earlier, a later row has its slot
  __device__ __forceinline__ bool first(int q) const { return !(before >> q & 1); }
  __device__ __forceinline__ bool shared(int q) const { return after >> q & 1; }
  // (every thread of the block calls it; the block has at least kStepRows)
  __device__ __forceinline__ void find(const void* slots, int bits, int rows, int row0, int n) {
    if (threadIdx.x == 0) before = after = 0;
    if (threadIdx.x < n) slot[threadIdx.x] = slots ? index_at(slots, bits, row0 + threadIdx.x) : row0 + threadIdx.x;
    __syncthreads();
    if (!slots || rows == 1) return;
    uint32_t seen = 0, comes = 0;
    for (int j = threadIdx.x; j < rows; j += blockDim.x) {
      const int64_t s = index_at(slots, bits, j);
      for (int q = 0; q < n; ++q)
        if (s == slot[q]) (j < row0 + q ? seen : comes) |= (uint32_t)(j != row0 + q) << q;
    }
    if (seen) atomicOr(&before, seen);
    if (comes) atomicOr(&after, comes);
    __syncthreads();
  }
};
// Rows of a block: as few as leave no more than `resident` blocks for each SM, all of them at work at once.
inline int step_rows(int rows, int tiles, int resident) {
  const int64_t blocks = std::max<int64_t>(1, (int64_t)resident * sm_count() / tiles);   // for the rows
  return (int)std::min<int64_t>(kStepRows, (rows + blocks - 1) / blocks);
}

// A tensor of tokens can be read and written by `bytes` at a time.
inline bool by(const lasp_tokens& t, size_t bytes, size_t item) {
  const uint64_t at = reinterpret_cast<uintptr_t>(t.data) | (uint64_t)t.row_pitch * item | (uint64_t)t.token_pitch * item | (uint64_t)t.group_pitch * item;
  return !t.data || (at & (bytes - 1)) == 0;
}

cudaError_t conv_forward(const lasp_conv_args& a, cudaStream_t st);
cudaError_t conv_backward(const lasp_conv_args& a, cudaStream_t st);
size_t conv_workspace(const lasp_conv_args& a);
cudaError_t conv_step(const lasp_conv_step_args& a, cudaStream_t st);
cudaError_t scan_forward(const lasp_scan_args& a, cudaStream_t st);
cudaError_t scan_backward(const lasp_scan_args& a, cudaStream_t st);
size_t scan_kept(const lasp_scan_args& a);
size_t scan_forward_workspace(const lasp_scan_args& a);
size_t scan_workspace(const lasp_scan_args& a);
cudaError_t scan_step(const lasp_scan_step_args& a, cudaStream_t st);

}  // namespace lasp
