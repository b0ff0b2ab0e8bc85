// Selective scan for single tokens: every row of a decoding batch reads the state of its sequence, takes it one token on and writes
// it back.  Memory bounds it, 8 bytes for every state; B, C and what belongs to a channel are small beside it.
#include <algorithm>

#include "scan_common.cuh"

namespace lasp {
namespace {

// A lane holds 4 states of CPL channels; LPC lanes side by side have those of a channel.
template <typename T, int LPC, int CPL>
__global__ void __launch_bounds__(128) k_scan_step(lasp_scan_step_args a) {
  constexpr int kChannels = 128 / LPC;   // of a block, CPL times
  const int row = blockIdx.y, i = threadIdx.x % LPC, n = 4 * i;
  const int64_t slot = a.slots ? index_at(a.slots, a.index_bits, row) : row;
  const int c0 = blockIdx.x * kChannels * CPL + threadIdx.x / LPC, in_group = a.channels / a.groups;
  const bool f32 = a.param_dtype == LASP_F32;
  if (slot < 0 || slot >= a.slot_count) {   // a row that stands for no sequence
    for (int k = 0; k < CPL; ++k)
      if (const int c = c0 + k * kChannels; i == 0 && c < a.channels) static_cast<T*>(a.y.data)[(int64_t)row * a.y.row_pitch + c] = from_f<T>(0.f);
    return;
  }
  float* state = a.state + slot * a.channels * a.states;
  const int shared = shared_slot(a.slots, a.index_bits, a.rows, row, slot);
  if (shared < 0) return;
  S4 h[CPL], rate[CPL];
#pragma unroll
  for (int k = 0; k < CPL; ++k) {
    const int c = c0 + k * kChannels;
    h[k] = c < a.channels ? s4(four_of(state + (int64_t)c * a.states, n, a.states)) : splat(0.f);
  }
#pragma unroll
  for (int k = 0; k < CPL; ++k) {
    const int c = c0 + k * kChannels;
    rate[k] = c < a.channels ? rates(a.A + (int64_t)c * a.states, n, a.states) : splat(0.f);
  }
  for (int r = row; r < a.rows; ++r) {
    if (r > row) {
      if (!shared) break;
      if (index_at(a.slots, a.index_bits, r) != slot) continue;
    }
    const auto rows = [&](const lasp_tokens& t) { return static_cast<T*>(t.data) + (int64_t)r * t.row_pitch; };
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      const int c = c0 + k * kChannels;
      const bool there = c < a.channels;
      float u = 0.f, dt = 0.f;
      float4 B = make_float4(0.f, 0.f, 0.f, 0.f), C = B;
      if (there) {
        u = to_f(rows(a.u)[c]);
        dt = to_f(rows(a.dt)[c]) + (a.dt_bias ? param<T>(a.dt_bias, f32, c) : 0.f);
        if (a.softplus) dt = softplus(dt);
        const T *pB = rows(a.B) + (int64_t)(c / in_group) * a.B.group_pitch + n, *pC = rows(a.C) + (int64_t)(c / in_group) * a.C.group_pitch + n;
        const auto at = [&](const T* p, int q) { return n + q < a.states ? to_f(p[q]) : 0.f; };
        B = make_float4(at(pB, 0), at(pB, 1), at(pB, 2), at(pB, 3));
        C = make_float4(at(pC, 0), at(pC, 1), at(pC, 2), at(pC, 3));
      }
      const float in = dt * u;
      h[k] = fma(exp2(mul(rate[k], f2(dt, dt))), h[k], mul(s4(B), f2(in, in)));
      float y = dot(h[k], s4(C));
#pragma unroll
      for (int m = 1; m < LPC; m *= 2) y += __shfl_xor_sync(~0u, y, m);
      if (there && i == 0) {
        if (a.D) y = fmaf(param<T>(a.D, f32, c), u, y);
        if (a.z.data) y *= silu(to_f(rows(a.z)[c]));
        rows(a.y)[c] = from_f<T>(y);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < CPL; ++k)
    if (const int c = c0 + k * kChannels; c < a.channels) store_four(state + (int64_t)c * a.states, n, a.states, f4(h[k]));
}

template <typename T, int LPC>
cudaError_t launch(const lasp_scan_step_args& a, cudaStream_t st) {
  constexpr int kChannels = 128 / LPC;
  k_scan_step<T, LPC, 1><<<dim3((a.channels + kChannels - 1) / kChannels, a.rows), 128, 0, st>>>(a);
  return cudaGetLastError();
}
template <typename T>
cudaError_t step_as(const lasp_scan_step_args& a, cudaStream_t st) {
  switch (padded_states(a.states)) {
    case 16: return launch<T, 4>(a, st);
    case 32: return launch<T, 8>(a, st);
    default: return launch<T, 16>(a, st);
  }
}

}  // namespace

cudaError_t scan_step(const lasp_scan_step_args& a, cudaStream_t st) {
  return a.dtype == LASP_F32 ? step_as<float>(a, st) : a.dtype == LASP_BF16 ? step_as<__nv_bfloat16>(a, st) : step_as<__half>(a, st);
}

}  // namespace lasp
