// Selective scan over prompts and training batches, forward.  The formulas, and how a warp holds a tile of channels and states, are
// in scan_common.cuh.
//
// A block owns one tile of channels of one sequence and walks along its tokens, W * NT at a time.  Warp w has the NT tokens from
// w * NT on: it turns their steps into decays once (the exponentials, which bound the kernel: one for every state of every channel
// and token, at 16 per clock and SM), and takes them along in registers: first from a state of zero, which with the product of the decays
// says what these tokens make of any state; then, when the states at the W places are known, for the outputs.
#include "scan_common.cuh"

namespace lasp {
namespace {

template <typename T, int LPC, int CPL, int W, int NT>
struct Shared {
  using TILE = Tile<LPC, CPL>;
  struct Tokens {   // of one warp
    float dt[NT][TILE::kChannels], dtu[NT][TILE::kChannels];
    float B[NT][TILE::kStates], C[NT][TILE::kStates];
  } tokens[W];
  float4 decay[W > 1 ? W : 1][CPL][32], state[W > 1 ? W : 1][CPL][32];
};

template <typename T, int LPC, int CPL, int W, int NT>
__global__ void __launch_bounds__(32 * W) k_scan_forward(lasp_scan_args a, int tiles) {
  using TILE = Tile<LPC, CPL>;
  constexpr int kRounds = NT / TILE::kRound, kFill = NT * TILE::kStates / 32;
  static_assert(NT % TILE::kRound == 0 && kKeep % NT == 0, "");
  extern __shared__ char raw_smem[];
  auto& sm = *reinterpret_cast<Shared<T, LPC, CPL, W, NT>*>(raw_smem);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, i = lane % LPC, g = lane / LPC;
  const TilePlace<TILE> tile(blockIdx.x % tiles, a.channels, a.groups);
  const int seq = blockIdx.x / tiles;
  if (a.sequences && seq == a.sequences) return fill_outside<T, TILE>(a, a.y, tile);
  const Stretch at = stretch_of(a, seq);
  // this lane's (token, channel) of a round
  const int own = g * CPL + i % CPL, sub = i / CPL;
  const bool own_ok = own < tile.left;
  const int64_t own_c = tile.channel + own;
  const auto rows = [&](const lasp_tokens& t) { return static_cast<T*>(t.data) + (int64_t)at.row * t.row_pitch + (int64_t)at.begin * t.token_pitch; };
  const T *pu = rows(a.u) + own_c, *pdt = rows(a.dt) + own_c, *pz = a.z.data ? rows(a.z) + own_c : nullptr;
  const T *pB = rows(a.B) + (int64_t)tile.group * a.B.group_pitch, *pC = rows(a.C) + (int64_t)tile.group * a.C.group_pitch;
  T* py = rows(a.y) + own_c;
  const bool f32 = a.param_dtype == LASP_F32;
  const float skip = own_ok && a.D ? param<T>(a.D, f32, own_c) : 0.f;
  const float bias = own_ok && a.dt_bias ? param<T>(a.dt_bias, f32, own_c) : 0.f;

  S4 rate[CPL];   // of channels g * CPL + c, states 4 i to 4 i + 3
#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    const int ch = g * CPL + c;
    rate[c] = ch < tile.left ? rates(a.A + (int64_t)(tile.channel + ch) * a.states, 4 * i, a.states) : splat(0.f);
  }
  // The running state: of one warp in its lanes' own layout (W = 1), else shared out for the scan over the warps.
  constexpr int kShare = W > 1 ? 128 * CPL / (32 * W) : 1;
  static_assert(W == 1 || kShare >= 1, "");
  S4 h[CPL];
  float carry[kShare];
  const auto state_at = [&](int e, int64_t* where) {   // element e of a tile's states: [channel][lane][4]
    const int c = e / 128, l = e % 128 / 4, ch = (l / LPC) * CPL + c, n = (l % LPC) * 4 + e % 4;
    *where = ((int64_t)seq * a.channels + tile.channel + ch) * a.states + n;
    return ch < tile.left && n < a.states;
  };
  if constexpr (W == 1) {
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      const int ch = g * CPL + c;
      h[c] = a.state_in && ch < tile.left ? s4(four_of(a.state_in + ((int64_t)seq * a.channels + tile.channel + ch) * a.states, 4 * i, a.states)) : splat(0.f);
    }
  } else {
#pragma unroll
    for (int k = 0; k < kShare; ++k) {
      int64_t where;
      carry[k] = state_at(threadIdx.x + k * 32 * W, &where) && a.state_in ? a.state_in[where] : 0.f;
    }
  }

  T u_next[kRounds], dt_next[kRounds], z_next[kRounds], B_next[kFill], C_next[kFill];
  const auto fetch = [&](int base) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int t = base + r * TILE::kRound + sub;
      if (t < at.tokens && own_ok) {
        u_next[r] = pu[(int64_t)t * a.u.token_pitch], dt_next[r] = pdt[(int64_t)t * a.dt.token_pitch];
        if (pz) z_next[r] = pz[(int64_t)t * a.z.token_pitch];
      }
    }
#pragma unroll
    for (int k = 0; k < kFill; ++k) {
      const int t = base + (lane + 32 * k) / TILE::kStates, n = (lane + 32 * k) % TILE::kStates;
      const bool there = t < at.tokens && n < a.states;
      B_next[k] = there ? pB[(int64_t)t * a.B.token_pitch + n] : from_f<T>(0.f);
      C_next[k] = there ? pC[(int64_t)t * a.C.token_pitch + n] : from_f<T>(0.f);
    }
  };
  fetch(warp * NT);

  auto& my = sm.tokens[warp];
  for (int chunk = 0; chunk < at.tokens; chunk += W * NT) {
    const int base = chunk + warp * NT;
    float u[kRounds], z[kRounds];
    __syncwarp();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int t = r * TILE::kRound + sub;
      const bool there = base + t < at.tokens && own_ok;   // behind the end the step is zero: the state stays
      u[r] = there ? to_f(u_next[r]) : 0.f;
      z[r] = there && pz ? to_f(z_next[r]) : 0.f;
      const float raw = there ? to_f(dt_next[r]) + bias : 0.f;
      const float dt = there ? (a.softplus ? softplus(raw) : raw) : 0.f;
      my.dt[t][own] = dt;
      my.dtu[t][own] = dt * u[r];
    }
#pragma unroll
    for (int k = 0; k < kFill; ++k) {
      const int t = (lane + 32 * k) / TILE::kStates, n = (lane + 32 * k) % TILE::kStates;
      my.B[t][n] = to_f(B_next[k]), my.C[t][n] = to_f(C_next[k]);
    }
    __syncwarp();
    if (chunk + W * NT < at.tokens) fetch(base + W * NT);

    S4 decay[NT][CPL];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < CPL; ++c) decay[t][c] = exp2(mul(rate[c], my.dt[t][g * CPL + c]));
    if constexpr (W > 1) {
      S4 p[CPL], s[CPL];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const S4 B = s4(*reinterpret_cast<const float4*>(&my.B[t][4 * i]));
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          const S4 in = mul(B, my.dtu[t][g * CPL + c]);
          s[c] = t ? fma(decay[t][c], s[c], in) : in;
          p[c] = t ? mul(p[c], decay[t][c]) : decay[t][c];
        }
      }
#pragma unroll
      for (int c = 0; c < CPL; ++c) sm.decay[warp][c][lane] = f4(p[c]), sm.state[warp][c][lane] = f4(s[c]);
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kShare; ++k) {
        const int e = threadIdx.x + k * 32 * W;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          float* local = reinterpret_cast<float*>(sm.state[w]) + e;
          const float in = carry[k];
          carry[k] = fmaf(reinterpret_cast<const float*>(sm.decay[w])[e], in, *local);
          *local = in;
        }
      }
      __syncthreads();
#pragma unroll
      for (int c = 0; c < CPL; ++c) h[c] = s4(sm.state[warp][c][lane]);
    }
    if (a.kept && base % kKeep == 0 && base < at.tokens) {
      float4* to = static_cast<float4*>(a.kept) + ((at.kept + base / kKeep) * a.channels + tile.channel) * LPC;
#pragma unroll
      for (int c = 0; c < CPL; ++c)
        if (g * CPL + c < tile.left) to[(int64_t)(g * CPL + c) * LPC + i] = f4(h[c]);
    }
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      float sums[LPC];
#pragma unroll
      for (int q = 0; q < TILE::kRound; ++q) {
        const int t = r * TILE::kRound + q;
        const S4 B = s4(*reinterpret_cast<const float4*>(&my.B[t][4 * i])), C = s4(*reinterpret_cast<const float4*>(&my.C[t][4 * i]));
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          h[c] = fma(decay[t][c], h[c], mul(B, my.dtu[t][g * CPL + c]));
          sums[q * CPL + c] = add_up(mul(C, h[c]));
        }
      }
      sum_over<LPC, LPC, 1>(sums, lane);
      const int t = base + r * TILE::kRound + sub;
      if (t < at.tokens && own_ok) {
        const float y = fmaf(skip, u[r], sums[0]);
        py[(int64_t)t * a.y.token_pitch] = from_f<T>(pz ? y * silu(z[r]) : y);
      }
    }
  }
  if (!a.state_out) return;
  if constexpr (W == 1) {
#pragma unroll
    for (int c = 0; c < CPL; ++c)
      if (g * CPL + c < tile.left) store_four(a.state_out + ((int64_t)seq * a.channels + tile.channel + g * CPL + c) * a.states, 4 * i, a.states, f4(h[c]));
  } else {
#pragma unroll
    for (int k = 0; k < kShare; ++k) {
      int64_t where;
      if (state_at(threadIdx.x + k * 32 * W, &where)) a.state_out[where] = carry[k];
    }
  }
}

template <typename T, int LPC, int CPL, int W, int NT>
cudaError_t launch(const lasp_scan_args& a, cudaStream_t st) {
  constexpr auto kernel = k_scan_forward<T, LPC, CPL, W, NT>;
  constexpr size_t smem = sizeof(Shared<T, LPC, CPL, W, NT>);
  const cudaError_t err = opt_in_smem<kernel>(smem);
  if (err != cudaSuccess) return err;
  const int tiles = tiles_of<Tile<LPC, CPL>>(a.channels, a.groups);
  const int sequences = a.sequences ? a.sequences + 1 : a.rows;   // (one more: what lies in none)
  kernel<<<(unsigned)(tiles * sequences), 32 * W, smem, st>>>(a, tiles);
  return cudaGetLastError();
}

template <typename T>
cudaError_t forward_as(const lasp_scan_args& a, cudaStream_t st) {
  switch (padded_states(a.states)) {
    case 16: return launch<T, 4, 2, 1, 8>(a, st);
    case 32: return launch<T, 8, 2, 1, 8>(a, st);
    default: return launch<T, 16, 2, 1, 8>(a, st);
  }
}

}  // namespace

cudaError_t scan_forward(const lasp_scan_args& a, cudaStream_t st) {
  return a.dtype == LASP_F32 ? forward_as<float>(a, st) : a.dtype == LASP_BF16 ? forward_as<__nv_bfloat16>(a, st) : forward_as<__half>(a, st);
}

}  // namespace lasp
