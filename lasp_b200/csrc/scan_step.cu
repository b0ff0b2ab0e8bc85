// Selective scan for single tokens: every row of a decoding batch reads the state of its sequence, takes it one token on and writes
// it back.  Memory bounds it, 8 bytes for every state; B, C and what belongs to a channel are small beside it.
#include "scan_common.cuh"

namespace lasp {
namespace {

constexpr int kStepThreads = 128, kOwn = 4;   // channels of a lane, side by side: that many reads of the state under way

// A lane holds 4 states of each of its channels; LPC lanes side by side have those of a channel.  wide: u, dt, B and C can be read by four.
template <typename T, int LPC>
__global__ void __launch_bounds__(kStepThreads) k_scan_step(lasp_scan_step_args a, bool wide) {
  constexpr int kSame = LPC / kOwn;   // lanes that are left with the same channel's sum
  const int row = blockIdx.y, lane = threadIdx.x % 32, i = threadIdx.x % LPC, n = 4 * i;
  const int c0 = (blockIdx.x * (kStepThreads / LPC) + threadIdx.x / LPC) * kOwn, mine = c0 + i / kSame;   // mine: whose output this lane finishes
  const bool f32 = a.param_dtype == LASP_F32, writes = i % kSame == 0 && mine < a.channels;
  const int64_t slot = a.slots ? index_at(a.slots, a.index_bits, row) : row;
  if (slot < 0 || slot >= a.slot_count) {   // a row that stands for no sequence
    if (writes) static_cast<T*>(a.y.data)[(int64_t)row * a.y.row_pitch + mine] = from_f<T>(0.f);
    return;
  }
  float* state = a.state + (slot * a.channels + c0) * a.states;
  const float* A = a.A + (int64_t)c0 * a.states;
  const int left = a.channels - c0;
  S4 h[kOwn], rate[kOwn];
#pragma unroll
  for (int k = 0; k < kOwn; ++k) h[k] = k < left ? s4(four_of(state + (int64_t)k * a.states, n, a.states)) : splat(0.f);
#pragma unroll
  for (int k = 0; k < kOwn; ++k) rate[k] = k < left ? rates(A + (int64_t)k * a.states, n, a.states) : splat(0.f);
  const int shared = shared_slot(a.slots, a.index_bits, a.rows, row, slot);   // (the state is on its way meanwhile)
  if (shared < 0) return;
  float bias[kOwn];
#pragma unroll
  for (int k = 0; k < kOwn; ++k) bias[k] = k < left && a.dt_bias ? param<T>(a.dt_bias, f32, c0 + k) : 0.f;
  const float skip = writes && a.D ? param<T>(a.D, f32, mine) : 0.f;
  const int in_group = a.channels / a.groups, group = (c0 < a.channels ? c0 : 0) / in_group;
  const bool one_group = left >= kOwn && (c0 + kOwn - 1) / in_group == group;
  for (int r = row; r < a.rows; ++r) {
    if (r > row) {
      if (!shared) break;
      if (index_at(a.slots, a.index_bits, r) != slot) continue;
    }
    const auto rows = [&](const lasp_tokens& t) { return static_cast<T*>(t.data) + (int64_t)r * t.row_pitch; };
    const auto four = [&](const lasp_tokens& t, int g) {   // this lane's states of B or C
      const T* p = rows(t) + (int64_t)g * t.group_pitch + n;
      float x[4] = {};
      if (wide && n + 4 <= a.states) {
        numbers<T, 4>(*reinterpret_cast<const Vec<T, 4>*>(p), x);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n + q < a.states) x[q] = to_f(p[q]);
      }
      return s4(make_float4(x[0], x[1], x[2], x[3]));
    };
    float u[kOwn] = {}, dt[kOwn] = {}, y[kOwn];
    if (wide && left >= kOwn) {
      numbers<T, kOwn>(*reinterpret_cast<const Vec<T, kOwn>*>(rows(a.u) + c0), u), numbers<T, kOwn>(*reinterpret_cast<const Vec<T, kOwn>*>(rows(a.dt) + c0), dt);
    } else {
#pragma unroll
      for (int k = 0; k < kOwn; ++k)
        if (k < left) u[k] = to_f(rows(a.u)[c0 + k]), dt[k] = to_f(rows(a.dt)[c0 + k]);
    }
    S4 B = four(a.B, group), C = four(a.C, group);
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      if (!one_group && k && k < left) B = four(a.B, (c0 + k) / in_group), C = four(a.C, (c0 + k) / in_group);
      float step = dt[k] + bias[k];
      if (a.softplus) step = softplus(step);
      const float in = step * u[k];
      h[k] = fma(exp2(mul(rate[k], f2(step, step))), h[k], mul(B, f2(in, in)));
      y[k] = dot(h[k], C);
    }
    sum_over<kOwn, LPC, 1>(y, lane);
    if (writes) {
      float out = a.D ? fmaf(skip, to_f(rows(a.u)[mine]), y[0]) : y[0];
      if (a.z.data) out *= silu(to_f(rows(a.z)[mine]));
      rows(a.y)[mine] = from_f<T>(out);
    }
  }
#pragma unroll
  for (int k = 0; k < kOwn; ++k)
    if (k < left) store_four(state + (int64_t)k * a.states, n, a.states, f4(h[k]));
}

template <typename T, int LPC>
cudaError_t launch(const lasp_scan_step_args& a, cudaStream_t st) {
  constexpr int channels = kStepThreads / LPC * kOwn;
  const bool wide = reads_by<T>(a.u, kOwn) && reads_by<T>(a.dt, kOwn) && reads_by<T>(a.B, 4) && reads_by<T>(a.C, 4);
  k_scan_step<T, LPC><<<dim3((a.channels + channels - 1) / channels, a.rows), kStepThreads, 0, st>>>(a, wide);
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
