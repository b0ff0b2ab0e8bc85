// Selective scan, cut into segments: what a part of a sequence does to a state of zero, and the sum of its steps (scan_common.cuh says what for).
//
//   forward:   h = a_t h + dt_t u_t B_t, from the part's first token to its last
//   backward:  g = a_t (g + d_t C_t), from the last to the first, d_t = dy_t silu(z_t)
//
// Nothing else is left of a token, so that the exponentials bound it.  A block takes a tile of a part, four warps that hold the states as
// those of the main pass do; five blocks an SM cover one another's preparation of
// tokens.  6003 tokens of 1536 channels and 16 states, fp16: 45 us, where 33 would do for the exponentials (half of the issue
// slots are busy).
#include "scan_common.cuh"

namespace lasp {
namespace {

constexpr int kTake = 32;   // tokens prepared at a time

// WIDE: tokens' channels and states come by four, all or none of them there.  Every load is then made, and made without a condition (from a
// place that is there): behind a condition the warp waits for it on the spot (6003 tokens of 1536 channels, fp16: 70 us
// forward and 55 back, now 45 and 42).
template <typename T, int LPC, bool BACK, bool WIDE>
__global__ void __launch_bounds__(kGroup, 5) k_scan_parts(lasp_scan_args a, int tiles, Cuts cuts) {
  using TILE = Tile<LPC>;
  constexpr int kEach = TILE::kEach, kVecs = TILE::kVecs, kUnits = (kTake * kVecs + kGroup - 1) / kGroup, kFours = (kTake * LPC + kGroup - 1) / kGroup;   // of a thread
  __shared__ float2 step[2][kTake][TILE::kChannels];   // dt, and dt u or d
  __shared__ float4 four[2][kTake][LPC];               // B or C
  const int me = threadIdx.x, tile_index = blockIdx.x % tiles, slot = blockIdx.x / tiles;
  const TilePlace<TILE> tile(tile_index, a.channels, a.groups);
  const Stretch at(a, slot, cuts.part);
  const int behind = (at.count - 1) / kParts * kParts;   // parts from here on are the last segment's
  if (at.index == at.count || (BACK ? at.index < kParts : at.index >= behind)) return;
  const bool f32 = a.param_dtype == LASP_F32, gated = BACK && a.z.data;
  const int takes = (at.tokens + kTake - 1) / kTake;
  const auto rows = [&](const lasp_tokens& t) {
    return static_cast<const T*>(t.data) + (int64_t)at.row * t.row_pitch + (int64_t)at.begin * t.token_pitch;
  };
  const lasp_tokens &in = BACK ? a.dy : a.u, &vec = BACK ? a.C : a.B;
  Vec<T, kEach> raw_dt[kUnits], raw_in[kUnits], raw_z[kUnits];
  Vec<T, 4> raw_four[kFours];
  const auto get = [&](Vec<T, kEach>& to, const lasp_tokens& t, int64_t token, int c) {
    const T* p = rows(t) + token * t.token_pitch + tile.channel + (WIDE && c >= tile.left ? 0 : c);
    if constexpr (WIDE) {
      to = *reinterpret_cast<const Vec<T, kEach>*>(p);
    } else {
#pragma unroll
      for (int k = 0; k < kEach; ++k) to.v[k] = c + k < tile.left ? p[k] : from_f<T>(0.f);
    }
  };
  const auto fetch = [&](int take) {   // (behind the end: the last token, which is not used)
#pragma unroll
    for (int q = 0; q < kUnits; ++q) {
      const int v = me + q * kGroup, c = v % kVecs * kEach;
      const int64_t t = min(take * kTake + min(v / kVecs, kTake - 1), at.tokens - 1);
      get(raw_dt[q], a.dt, t, c), get(raw_in[q], in, t, c);
      if (BACK) get(raw_z[q], gated ? a.z : in, t, c);
    }
#pragma unroll
    for (int q = 0; q < kFours; ++q) {
      const int v = me + q * kGroup, n = v % LPC * 4;
      const T* p = rows(vec) + (int64_t)min(take * kTake + v / LPC, at.tokens - 1) * vec.token_pitch + (int64_t)tile.group * vec.group_pitch + (WIDE && n >= a.states ? 0 : n);
      if constexpr (WIDE) {
        raw_four[q] = *reinterpret_cast<const Vec<T, 4>*>(p);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) raw_four[q].v[k] = n + k < a.states ? p[k] : from_f<T>(0.f);
      }
    }
  };
  float bias[kEach];   // (a thread's units lie at the same channels)
  static_assert(kGroup % kVecs == 0 && kTake * LPC % kGroup == 0, "");
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int c = me % kVecs * kEach + k;
    bias[k] = a.dt_bias && c < tile.left ? param<T>(a.dt_bias, f32, tile.channel + c) : 0.f;
  }
  const auto prepare = [&](int take) {
    const int buf = take & 1;
#pragma unroll
    for (int q = 0; q < kUnits; ++q) {
      const int v = me + q * kGroup, row = v / kVecs, c = v % kVecs * kEach;
      if (row >= kTake) break;
      const bool there = take * kTake + row < at.tokens && c < tile.left;   // behind the end the step is zero
      float dt[kEach], x[kEach], z[kEach];
      numbers<T, kEach>(raw_dt[q], dt), numbers<T, kEach>(raw_in[q], x);
      if (BACK) numbers<T, kEach>(raw_z[q], z);
#pragma unroll
      for (int k = 0; k < kEach; k += 2) {
        F2 d = add2(f2(dt[k], dt[k + 1]), f2(bias[k], bias[k + 1]));
        if (a.softplus) d = softplus(d);
        F2 p = f2(x[k], x[k + 1]);
        if (!BACK)
          p = mul2(d, p);
        else if (gated)
          p = f2(x[k] * silu(z[k]), x[k + 1] * silu(z[k + 1]));
        float s0, s1, p0, p1;
        apart(d, s0, s1), apart(p, p0, p1);
        *reinterpret_cast<float4*>(&step[buf][row][c + k]) = there ? make_float4(s0, p0, s1, p1) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
#pragma unroll
    for (int q = 0; q < kFours; ++q) {
      const int v = me + q * kGroup;
      const bool there = take * kTake + v / LPC < at.tokens && v % LPC * 4 < a.states;
      float x[4];
      numbers<T, 4>(raw_four[q], x);
      four[buf][v / LPC][v % LPC] = there ? make_float4(x[0], x[1], x[2], x[3]) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  const int lane = me % 32, i = lane / TILE::kGroups, ch = me / 32 * TILE::kGroups + lane % TILE::kGroups;
  const S4 A = ch < tile.left ? rates(a.A + (int64_t)(tile.channel + ch) * a.states, 4 * i, a.states) : splat(0.f);
  S4 h = splat(0.f);
  float sum = 0.f;
  const auto number = [&](int k) { return BACK ? takes - 1 - k : k; };
  fetch(number(0));
  for (int k = 0; k < takes; ++k) {
    prepare(number(k));
    fetch(number(k + 1 < takes ? k + 1 : k));   // (once too often)
    __syncthreads();
    const int buf = number(k) & 1;
#pragma unroll 8
    for (int s = 0; s < kTake; ++s) {
      const int t = BACK ? kTake - 1 - s : s;
      const float2 x = step[buf][t][ch];
      const S4 decay = decay_of(A, x.x), v = load4(&four[buf][t][i]);
      sum += x.x;
      h = BACK ? mul(decay, fma(v, f2(x.y, x.y), h)) : fma(decay, h, mul(v, f2(x.y, x.y)));
    }
  }
  const int64_t to = (int64_t)slot * tiles + tile_index;
  cuts.ends[to * kGroup + me] = f4(h);
  if (i == 0) cuts.steps[to * TILE::kChannels + ch] = sum;
}

}  // namespace

template <typename T, int LPC>
cudaError_t scan_parts(const lasp_scan_args& a, const Cuts& cuts, int tiles, bool backward, cudaStream_t st) {
  using TILE = Tile<LPC>;
  const lasp_tokens &in = backward ? a.dy : a.u, &vec = backward ? a.C : a.B;
  const bool wide = (a.channels / a.groups) % TILE::kEach == 0 && a.states % 4 == 0 && reads_by<T>(vec, 4) && reads_by<T>(a.dt, TILE::kEach) &&
                    reads_by<T>(in, TILE::kEach) && (!backward || reads_by<T>(a.z, TILE::kEach));
  const auto kernel = backward ? wide ? k_scan_parts<T, LPC, true, true> : k_scan_parts<T, LPC, true, false>
                               : wide ? k_scan_parts<T, LPC, false, true> : k_scan_parts<T, LPC, false, false>;
  kernel<<<(unsigned)(tiles * cuts.parts), kGroup, 0, st>>>(a, tiles, cuts);
  return cudaGetLastError();
}
#define LASP_PARTS(T) \
  template cudaError_t scan_parts<T, 4>(const lasp_scan_args&, const Cuts&, int, bool, cudaStream_t); \
  template cudaError_t scan_parts<T, 8>(const lasp_scan_args&, const Cuts&, int, bool, cudaStream_t); \
  template cudaError_t scan_parts<T, 16>(const lasp_scan_args&, const Cuts&, int, bool, cudaStream_t);
LASP_PARTS(float)
LASP_PARTS(__half)
LASP_PARTS(__nv_bfloat16)
#undef LASP_PARTS

}  // namespace lasp
