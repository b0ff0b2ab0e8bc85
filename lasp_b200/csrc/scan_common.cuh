// The selective scan's tile: how a warp shares the channels and states of a token out among its lanes.
//
//   h_t[c][n] = exp(dt_t[c] A[c][n]) h_(t-1)[c][n] + dt_t[c] u_t[c] B_t[n],   y_t[c] = sum_n C_t[n] h_t[c][n] + D[c] u_t[c]
//
// A lane holds 4 neighbouring states of each of CPL neighbouring channels: LPC lanes side by side make the states of a group of
// CPL channels, and the 32 / LPC such groups of a warp kChannels channels in all.  So B and C are read by 4s, and a sum over
// states or channels is added up within lanes before it crosses them.  Sums over the states of kRound tokens at a time give each
// lane exactly one (token, channel): the one whose u, dt, z it loads and whose outputs it stores (`sum_over`).
#pragma once
#include "recurrent.cuh"

namespace lasp {

constexpr int kKeep = 64;   // the forward pass of a training call keeps the state ahead of every 64th token of a sequence
constexpr float kLog2e = 1.4426950408889634f;

template <int LPC, int CPL>
struct Tile {
  static_assert(CPL <= LPC && 32 % LPC == 0, "a lane's channels are at most the lanes of their states");
  static constexpr int kStates = 4 * LPC;
  static constexpr int kGroups = 32 / LPC;
  static constexpr int kChannels = kGroups * CPL;
  static constexpr int kRound = LPC / CPL;   // tokens x kChannels = 32
};

struct F2 {
  float x, y;
};
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

// 4 states of a channel
struct S4 {
  F2 a, b;
};
__device__ __forceinline__ S4 splat(float x) { return {{x, x}, {x, x}}; }
__device__ __forceinline__ S4 mul(S4 p, S4 q) { return {mul2(p.a, q.a), mul2(p.b, q.b)}; }
__device__ __forceinline__ S4 mul(S4 p, float f) { return {mul2(p.a, {f, f}), mul2(p.b, {f, f})}; }
__device__ __forceinline__ S4 fma(S4 p, S4 q, S4 r) { return {fma2(p.a, q.a, r.a), fma2(p.b, q.b, r.b)}; }
__device__ __forceinline__ S4 fma(S4 p, float f, S4 r) { return {fma2(p.a, {f, f}, r.a), fma2(p.b, {f, f}, r.b)}; }
__device__ __forceinline__ S4 s4(float4 v) { return {{v.x, v.y}, {v.z, v.w}}; }
__device__ __forceinline__ float4 f4(S4 v) { return make_float4(v.a.x, v.a.y, v.b.x, v.b.y); }
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ S4 exp2(S4 x) { return {{ex2(x.a.x), ex2(x.a.y)}, {ex2(x.b.x), ex2(x.b.y)}}; }
__device__ __forceinline__ float add_up(S4 v) { return (v.a.x + v.a.y) + (v.b.x + v.b.y); }

// v[k] summed over the LANES lanes that differ in the bits from STEP to STEP * LANES / 2; lane (bits / STEP) keeps that of index
// k = bits / STEP (COUNT = LANES), or COUNT / LANES neighbouring ones in v[0], v[1], ...: half of them change lanes at each step.
template <int COUNT, int LANES, int STEP>
__device__ __forceinline__ void sum_over(float (&v)[COUNT], int lane) {
  if constexpr (LANES > 1) {
    constexpr int m = LANES / 2 * STEP;
    const bool upper = lane & m;
    float half[COUNT / 2];
#pragma unroll
    for (int k = 0; k < COUNT / 2; ++k) {
      const float send = upper ? v[k] : v[k + COUNT / 2], keep = upper ? v[k + COUNT / 2] : v[k];
      half[k] = keep + __shfl_xor_sync(~0u, send, m);
    }
    sum_over<COUNT / 2, LANES / 2, STEP>(half, lane);
#pragma unroll
    for (int k = 0; k < COUNT / 2; ++k) v[k] = half[k];
  }
}

// log(1 + e^x) = max(x, 0) + log(1 + e), e = e^-|x| in (0, 1].  Small steps need it exact relative to e, not to 1: log(1 + e) =
// 2 atanh(s) with s = e / (2 + e) <= 1/3, whose series s + s^3/3 + s^5/5 ... is cut where it falls below 2^-26.
__device__ __forceinline__ float softplus(float x) {
  const float e = expf(-fabsf(x)), s = __fdividef(e, 2.f + e), q = s * s;
  float p = fmaf(q, 1.f / 13, 1.f / 11);
  p = fmaf(q, p, 1.f / 9), p = fmaf(q, p, 1.f / 7), p = fmaf(q, p, 1.f / 5), p = fmaf(q, p, 1.f / 3);
  return fmaxf(x, 0.f) + 2.f * fmaf(s * q, p, s);
}

// Of a 4 x states row of A, B or a state: 4 from state n on, zeros behind the last one.
__device__ __forceinline__ float4 four_of(const float* p, int n, int states) {
  if (n + 4 <= states && (reinterpret_cast<uintptr_t>(p + n) & 15) == 0) return *reinterpret_cast<const float4*>(p + n);
  return make_float4(n < states ? p[n] : 0.f, n + 1 < states ? p[n + 1] : 0.f, n + 2 < states ? p[n + 2] : 0.f, n + 3 < states ? p[n + 3] : 0.f);
}
__device__ __forceinline__ void store_four(float* p, int n, int states, float4 v) {
  if (n + 4 <= states && (reinterpret_cast<uintptr_t>(p + n) & 15) == 0) {
    *reinterpret_cast<float4*>(p + n) = v;
    return;
  }
  if (n < states) p[n] = v.x;
  if (n + 1 < states) p[n + 1] = v.y;
  if (n + 2 < states) p[n + 2] = v.z;
  if (n + 3 < states) p[n + 3] = v.w;
}
// A of 4 states times log2(e); infinities as fp32's largest number, so that a step of zero (every token behind a sequence's end)
// keeps the state
__device__ __forceinline__ S4 rates(const float* A, int n, int states) {
  const float4 v = four_of(A, n, states);
  const auto one = [](float x) { return isinf(x) ? copysignf(3.402823466e38f, x) : x * kLog2e; };
  return {{one(v.x), one(v.y)}, {one(v.z), one(v.w)}};
}

// Which channels a warp's tile is: tiles do not reach across groups, the last of a group may be cut short.
template <class TILE>
struct TilePlace {
  int group, channel, left;   // its group, its first channel, how many channels there are from it to the group's end
  __device__ __forceinline__ TilePlace(int tile, int channels, int groups) {
    const int in_group = channels / groups, tiles = (in_group + TILE::kChannels - 1) / TILE::kChannels;
    group = tile / tiles;
    const int first = (tile - group * tiles) * TILE::kChannels;
    channel = group * in_group + first;
    left = in_group - first;
  }
};
template <class TILE>
int tiles_of(int channels, int groups) {
  const int in_group = channels / groups;
  return groups * ((in_group + TILE::kChannels - 1) / TILE::kChannels);
}

// Where a sequence's tokens lie: row and first token, and the number of its first kept state.  A row of n tokens keeps
// ceil(n / kKeep) states; packed sequence i those from offsets[i] / kKeep + i on, which leaves room for each.
struct Stretch {
  int row, begin, tokens;
  int64_t kept;
};
__device__ __forceinline__ Stretch stretch_of(const lasp_scan_args& a, int seq) {
  if (!a.sequences) return {seq, 0, a.tokens, (int64_t)seq * ((a.tokens + kKeep - 1) / kKeep)};
  int begin, end;
  Sequences{a.offsets, a.index_bits, a.sequences, a.tokens}.bounds(seq, &begin, &end);
  return {0, begin, end - begin, (int64_t)begin / kKeep + seq};
}
inline int64_t kept_states(const lasp_scan_args& a) {
  return a.sequences ? (int64_t)a.tokens / kKeep + a.sequences + 1 : (int64_t)a.rows * ((a.tokens + kKeep - 1) / kKeep);
}
inline int padded_states(int states) { return states <= 16 ? 16 : states <= 32 ? 32 : 64; }

// Zeros for the tokens of a packed row that lie in no sequence.
template <typename T, class TILE>
__device__ void fill_outside(const lasp_scan_args& a, const lasp_tokens& y, const TilePlace<TILE>& tile) {
  if (!y.data) return;
  const Sequences s{a.offsets, a.index_bits, a.sequences, a.tokens};
  const int begin = s.at(0), end = max(begin, s.at(a.sequences));
  T* p = static_cast<T*>(y.data) + tile.channel;
  for (int64_t e = threadIdx.x; e < (int64_t)(a.tokens - (end - begin)) * TILE::kChannels; e += blockDim.x) {
    const int k = (int)(e / TILE::kChannels), c = (int)(e % TILE::kChannels), t = k < begin ? k : k + (end - begin);
    if (c < tile.left) p[(int64_t)t * y.token_pitch + c] = from_f<T>(0.f);
  }
}

}  // namespace lasp
