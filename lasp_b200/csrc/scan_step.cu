// Selective scan for single tokens: every row of a decoding batch reads the state of its sequence, takes it one token on and writes
// it back.  Its floor is memory, 8 bytes for every state; B, C and what belongs to a channel are small beside it.  256 rows of 4096 channels and 16 states,
// bf16: 33 us, 66 % of the copy rate (with 55 % of the issue slots busy: latency, one row's state being under way a block); one row of 2048 channels: 7 us, a launch.
#include "scan_common.cuh"

namespace lasp {
namespace {

constexpr int kStepThreads = 128, kStepBlocks = 5;   // (blocks: of an SM)
constexpr int kOwn = 4;                              // channels of a lane, side by side: that many reads of the state under way

// A lane holds 4 states of each of its channels; LPC lanes side by side have those of a channel.  The state of the next row is sent for
// before this one's is worked on.  What belongs to a channel and token (step, input, gate) is worked out by one lane and handed round.
// WHOLE: every lane has four states of four channels of one group, reads the states, B and C by four, and numbers and pitches have 32
// bits; checks for less than that and 64-bit products were half of all instructions.  Other numbers of states than 16, 32 and 64 take the
// variant with the checks, which spills (36 to 64 bytes a thread): 256 rows of 4096 channels take 53 us with 8 states and 59 with 12, 35 with 16.
template <typename T, int LPC, bool WHOLE>
__global__ void __launch_bounds__(kStepThreads, kStepBlocks) k_scan_step(lasp_scan_step_args a, int per) {
  __shared__ StepRows rows;
  constexpr int kSame = LPC / kOwn;   // lanes that work on the same channel
  const int lane = threadIdx.x % 32, i = threadIdx.x % LPC, n = 4 * i, row0 = blockIdx.y * per, count = min(per, a.rows - row0);
  const int c0 = (blockIdx.x * (kStepThreads / LPC) + threadIdx.x / LPC) * kOwn, mine = c0 + i / kSame, length = WHOLE ? 4 * LPC : a.states;
  const int own = WHOLE ? (c0 < a.channels ? kOwn : 0) : min(kOwn, a.channels - c0);
  const bool f32 = a.param_dtype == LASP_F32, there = mine < a.channels, writes = there && i % kSame == 0;
  const int64_t pitch = (int64_t)a.channels * length;
  float* const state = a.state + (int64_t)c0 * length;
  const auto by_slot = [&](int64_t slot) { return WHOLE ? (uint64_t)(uint32_t)pitch * (uint32_t)slot : (uint64_t)(slot * pitch); };
  const auto get = [&](const float* p) { return WHOLE ? *reinterpret_cast<const float4*>(p + n) : four_of(p, n, length); };
  const int in_group = a.channels / a.groups, group = (own > 0 ? c0 : 0) / in_group;
  // row r of a tensor, from a place in its first row
  const auto at = [&](T* p, int64_t row_pitch, int r) {
    return WHOLE ? p + (uint64_t)(uint32_t)row_pitch * (uint32_t)r : p + row_pitch * r;
  };
  T *const pu = static_cast<T*>(a.u.data) + mine, *const pdt = static_cast<T*>(a.dt.data) + mine, *const pz = static_cast<T*>(a.z.data) + mine;
  T *const py = static_cast<T*>(a.y.data) + mine, *const pB = static_cast<T*>(a.B.data) + n, *const pC = static_cast<T*>(a.C.data) + n;
  T *const gB = pB + group * a.B.group_pitch, *const gC = pC + group * a.C.group_pitch;
  const auto four = [&](const T* p) {   // this lane's states of B or C
    if constexpr (WHOLE) {
      return *reinterpret_cast<const Vec<T, 4>*>(p);
    } else {
      Vec<T, 4> x;
#pragma unroll
      for (int m = 0; m < 4; ++m) x.v[m] = n + m < length ? p[m] : from_f<T>(0.f);
      return x;
    }
  };
  S4 h[kOwn], rate[kOwn], next[kOwn];
  Vec<T, 4> next_B, next_C;
  T next_u = from_f<T>(0.f), next_dt = next_u, next_z = next_u;
  const auto fetch_token = [&](int r) {
    next_B = four(at(gB, a.B.row_pitch, r)), next_C = four(at(gC, a.C.row_pitch, r));
    if (there) next_u = *at(pu, a.u.row_pitch, r), next_dt = *at(pdt, a.dt.row_pitch, r);
    if (there && a.z.data) next_z = *at(pz, a.z.row_pitch, r);
  };
  const auto fetch = [&](int r, int64_t slot) {
    if (slot < 0 || slot >= a.slot_count) return;
    const float* from = state + by_slot(slot);
#pragma unroll
    for (int k = 0; k < kOwn; ++k)
      if (k < own) next[k] = s4(get(from + k * length));
    fetch_token(r);
  };
#pragma unroll
  for (int k = 0; k < kOwn; ++k) next[k] = rate[k] = splat(0.f);
  fetch(row0, a.slots ? index_at(a.slots, a.index_bits, row0) : row0);
#pragma unroll
  for (int k = 0; k < kOwn; ++k)
    if (k < own) rate[k] = rates(a.A + (int64_t)(c0 + k) * length, n, length);
  const float bias = there && a.dt_bias ? param<T>(a.dt_bias, f32, mine) : 0.f, skip = there && a.D ? param<T>(a.D, f32, mine) : 0.f;
  rows.find(a.slots, a.index_bits, a.rows, row0, count);
  for (int q = 0; q < count; ++q) {
    const int64_t slot = rows.slot[q];
#pragma unroll
    for (int k = 0; k < kOwn; ++k) h[k] = next[k];
    Vec<T, 4> now_B = next_B, now_C = next_C;
    T now_u = next_u, now_dt = next_dt, now_z = next_z;
    const bool more = q + 1 < count && rows.first(q + 1);
    if (more) fetch(row0 + q + 1, rows.slot[q + 1]);
    if (slot < 0 || slot >= a.slot_count) {   // a row that stands for no sequence
      if (writes) *at(py, a.y.row_pitch, row0 + q) = from_f<T>(0.f);
      continue;
    }
    if (!rows.first(q)) continue;
    for (int r = row0 + q; r < a.rows; ++r) {
      if (r > row0 + q) {
        if (!rows.shared(q)) break;
        if (index_at(a.slots, a.index_bits, r) != slot) continue;
        now_B = four(at(gB, a.B.row_pitch, r)), now_C = four(at(gC, a.C.row_pitch, r));
        if (there) now_u = *at(pu, a.u.row_pitch, r), now_dt = *at(pdt, a.dt.row_pitch, r);
        if (there && a.z.data) now_z = *at(pz, a.z.row_pitch, r);
      }
      const auto s4_of = [](const Vec<T, 4>& v) { return S4{pair_from(&v.v[0]), pair_from(&v.v[2])}; };
      S4 B = s4_of(now_B), C = s4_of(now_C);
      const float u = to_f(now_u);
      float step = to_f(now_dt) + bias, y[kOwn];
      if (a.softplus) step = softplus(step);
      const float in = step * u;
#pragma unroll
      for (int k = 0; k < kOwn; ++k) {
        const float dt = __shfl_sync(~0u, step, k * kSame, LPC), x = __shfl_sync(~0u, in, k * kSame, LPC);
        if constexpr (!WHOLE)
          if (const int64_t g = (c0 + k) / in_group; k && k < own && (c0 + k) % in_group == 0)
            B = s4_of(four(at(pB + g * a.B.group_pitch, a.B.row_pitch, r))), C = s4_of(four(at(pC + g * a.C.group_pitch, a.C.row_pitch, r)));
        h[k] = fma(decay_of(rate[k], dt), h[k], mul(B, f2(x, x)));
        y[k] = dot(h[k], C);
      }
      sum_over<kOwn, LPC, 1>(y, lane);
      if (a.D) y[0] = fmaf(skip, u, y[0]);
      if (a.z.data) y[0] *= silu(to_f(now_z));
      if (writes) *at(py, a.y.row_pitch, r) = from_f<T>(y[0]);
    }
    float* to = state + by_slot(slot);
#pragma unroll
    for (int k = 0; k < kOwn; ++k)
      if (k < own) {
        if constexpr (WHOLE)
          store4(to + k * length + n, h[k]);
        else
          store_four(to + k * length, n, length, f4(h[k]));
      }
  }
}

template <typename T, int LPC>
cudaError_t launch(const lasp_scan_step_args& a, cudaStream_t st) {
  constexpr int channels = kStepThreads / LPC * kOwn;
  const auto small = [](int64_t n) { return n >= 0 && n <= INT32_MAX; };
  bool whole = small(a.slot_count) && small((int64_t)a.channels * a.states);
  for (const lasp_tokens* t : {&a.u, &a.dt, &a.z, &a.B, &a.C, &a.y}) whole = whole && small(t->row_pitch);
  whole = whole && a.states == 4 * LPC && a.channels / a.groups % kOwn == 0 && reads_by<T>(a.B, 4) && reads_by<T>(a.C, 4) &&
          (reinterpret_cast<uintptr_t>(a.state) | reinterpret_cast<uintptr_t>(a.A)) % 16 == 0;
  const int tiles = (a.channels + channels - 1) / channels, per = step_rows(a.rows, tiles, kStepBlocks);
  const dim3 grid(tiles, (a.rows + per - 1) / per);
  if (whole)
    k_scan_step<T, LPC, true><<<grid, kStepThreads, 0, st>>>(a, per);
  else
    k_scan_step<T, LPC, false><<<grid, kStepThreads, 0, st>>>(a, per);
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
