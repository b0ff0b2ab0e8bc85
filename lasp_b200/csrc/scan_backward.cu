// Selective scan, backward.  With d_t = dy_t silu(z_t) and the gradient g that reaches the state behind token t,
//
//   g_t = C_t d_t + a_(t+1) g_(t+1),   a_t = exp(dt_t A)
//   dC_t = sum_c d_t h_t,  dB_t = sum_c g_t dt_t u_t,  du_t = dt_t <g_t, B_t> + D d_t
//   e_t = a_t g_t h_(t-1):  d dt_t = u_t <g_t, B_t> + <e_t, A>,  dA = sum_t dt_t e_t
//
// A block owns a tile of channels of a sequence, as in the forward pass, and walks back along its tokens, kKeep at a time, from the
// states that the forward pass has kept.  Each warp takes its NT tokens once up to learn three things of them: the product of the
// decays, the state they leave from zero, and the gradient they pass on from zero (sum_t a_first ... a_t C_t d_t, which runs upwards
// like the other two).  One exchange between the warps then gives each both what comes from before and what comes from behind;
// it goes up again for the states and down for the gradients.  dB and dC are sums over channels: each tile leaves its own,
// and k_scan_sum_tokens adds them up in the order of the tiles, so that results do not depend on when blocks run.
#include "scan_common.cuh"

namespace lasp {
namespace {

template <typename T, int LPC, int CPL, int W, int NT>
struct Shared {
  using TILE = Tile<LPC, CPL>;
  struct Tokens {
    float dt[NT][TILE::kChannels], dtu[NT][TILE::kChannels], d[NT][TILE::kChannels];
    float B[NT][TILE::kStates], C[NT][TILE::kStates];
  } tokens[W];
  float4 decay[W][CPL][32], state[W][CPL][32], grad[W][CPL][32];
};

// What a backward pass writes beside its results, in the order of the workspace.
struct Partial {
  float* tokens;   // [tile][row * tokens + token][LPC][8]: of 4 states their 4 dB, 4 dC
  float* rates;    // [sequence][channel][kStates]: dA
  float* skips;    // [sequence][2][channel]: dD, ddt_bias
};

template <typename T, int LPC, int CPL, int W, int NT>
__global__ void __launch_bounds__(32 * W) k_scan_backward(lasp_scan_args a, int tiles, Partial out) {
  using TILE = Tile<LPC, CPL>;
  constexpr int kRounds = NT / TILE::kRound, kFill = NT * TILE::kStates / 32, kHalf = 128 * CPL, kShare = 2 * kHalf / (32 * W);
  constexpr int kLeft = 8 / TILE::kGroups;   // of 8 sums over a warp's channels, how many a lane is left with
  static_assert(W * NT == kKeep && kShare >= 1 && TILE::kGroups <= 8, "");
  extern __shared__ char raw_smem[];
  auto& sm = *reinterpret_cast<Shared<T, LPC, CPL, W, NT>*>(raw_smem);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, i = lane % LPC, g = lane / LPC;
  const int tile_index = blockIdx.x % tiles, seq = blockIdx.x / tiles;
  const TilePlace<TILE> tile(tile_index, a.channels, a.groups);
  if (a.sequences && seq == a.sequences) {
    fill_outside<T, TILE>(a, a.du, tile), fill_outside<T, TILE>(a, a.ddt, tile), fill_outside<T, TILE>(a, a.dz, tile);
    return;
  }
  const Stretch at = stretch_of(a, seq);
  const int own = g * CPL + i % CPL, sub = i / CPL;
  const bool own_ok = own < tile.left;
  const int64_t own_c = tile.channel + own;
  const auto rows = [&](const lasp_tokens& t) { return static_cast<T*>(t.data) + (int64_t)at.row * t.row_pitch + (int64_t)at.begin * t.token_pitch; };
  const T *pu = rows(a.u) + own_c, *pdt = rows(a.dt) + own_c, *pz = a.z.data ? rows(a.z) + own_c : nullptr, *pdy = rows(a.dy) + own_c;
  const T *pB = rows(a.B) + (int64_t)tile.group * a.B.group_pitch, *pC = rows(a.C) + (int64_t)tile.group * a.C.group_pitch;
  T *pdu = rows(a.du) + own_c, *pddt = rows(a.ddt) + own_c, *pdz = pz ? rows(a.dz) + own_c : nullptr;
  float* to_tokens = out.tokens + ((int64_t)tile_index * a.rows * a.tokens + (int64_t)at.row * a.tokens + at.begin) * (2 * TILE::kStates) + i * 8 + g * kLeft;
  const bool f32 = a.param_dtype == LASP_F32;
  const float skip = own_ok && a.D ? param<T>(a.D, f32, own_c) : 0.f;
  const float bias = own_ok && a.dt_bias ? param<T>(a.dt_bias, f32, own_c) : 0.f;

  S4 rate[CPL], drate[CPL];
#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    const int ch = g * CPL + c;
    rate[c] = ch < tile.left ? rates(a.A + (int64_t)(tile.channel + ch) * a.states, 4 * i, a.states) : splat(0.f);
    drate[c] = splat(0.f);
  }
  float dskip = 0.f, dbias = 0.f;
  // element e of a tile's states: [channel][lane][4]
  const auto state_at = [&](int e, int* ch, int* n) {
    const int l = e % 128 / 4;
    *ch = (l / LPC) * CPL + e / 128, *n = (l % LPC) * 4 + e % 4;
    return *ch < tile.left && *n < a.states;
  };
  // The exchange between the warps, shared out over the threads: items below kHalf are states, upwards from what the forward pass
  // has kept; those from kHalf on gradients, downwards from what reaches the last state of what is left.
  float carry[kShare];
#pragma unroll
  for (int k = 0; k < kShare; ++k) {
    const int e = threadIdx.x + k * 32 * W;
    int ch, n;
    carry[k] = e >= kHalf && state_at(e - kHalf, &ch, &n) && a.dstate_out
                   ? a.dstate_out[((int64_t)seq * a.channels + tile.channel + ch) * a.states + n] : 0.f;
  }

  auto& my = sm.tokens[warp];
  for (int chunk = (at.tokens - 1) / kKeep * kKeep; chunk >= 0 && at.tokens > 0; chunk -= kKeep) {
    const int base = chunk + warp * NT;
    float u[kRounds], z[kRounds], dy[kRounds], dts[kRounds], slope[kRounds];   // slope: of the step size to what it is made of
#pragma unroll
    for (int k = 0; k < kShare; ++k) {
      const int e = threadIdx.x + k * 32 * W;
      int ch, n;
      if (e < kHalf)
        carry[k] = state_at(e, &ch, &n) ? static_cast<const float*>(a.kept)[((at.kept + chunk / kKeep) * a.channels + tile.channel + ch) * TILE::kStates + n] : 0.f;
    }
    __syncwarp();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int t = r * TILE::kRound + sub;
      const bool there = base + t < at.tokens && own_ok;
      const int64_t tt = base + t;
      u[r] = there ? to_f(pu[tt * a.u.token_pitch]) : 0.f;
      z[r] = there && pz ? to_f(pz[tt * a.z.token_pitch]) : 0.f;
      dy[r] = there ? to_f(pdy[tt * a.dy.token_pitch]) : 0.f;
      const float raw = there ? to_f(pdt[tt * a.dt.token_pitch]) + bias : 0.f;
      dts[r] = there ? (a.softplus ? softplus(raw) : raw) : 0.f;
      slope[r] = a.softplus ? sigmoid(raw) : 1.f;
      my.dt[t][own] = dts[r];
      my.dtu[t][own] = dts[r] * u[r];
      my.d[t][own] = pz ? dy[r] * silu(z[r]) : dy[r];
    }
#pragma unroll
    for (int k = 0; k < kFill; ++k) {
      const int t = (lane + 32 * k) / TILE::kStates, n = (lane + 32 * k) % TILE::kStates;
      const int64_t tt = base + t;
      const bool there = tt < at.tokens && n < a.states;
      my.B[t][n] = there ? to_f(pB[tt * a.B.token_pitch + n]) : 0.f;
      my.C[t][n] = there ? to_f(pC[tt * a.C.token_pitch + n]) : 0.f;
    }
    __syncwarp();

    S4 decay[NT][CPL];
    {
      S4 p[CPL], s[CPL], q[CPL];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const S4 B = s4(*reinterpret_cast<const float4*>(&my.B[t][4 * i])), C = s4(*reinterpret_cast<const float4*>(&my.C[t][4 * i]));
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          const int ch = g * CPL + c;
          decay[t][c] = exp2(mul(rate[c], my.dt[t][ch]));
          const S4 in = mul(B, my.dtu[t][ch]), back = mul(C, my.d[t][ch]);
          s[c] = t ? fma(decay[t][c], s[c], in) : in;
          p[c] = t ? mul(p[c], decay[t][c]) : decay[t][c];
          q[c] = t ? fma(p[c], back, q[c]) : mul(p[c], back);
        }
      }
#pragma unroll
      for (int c = 0; c < CPL; ++c) sm.decay[warp][c][lane] = f4(p[c]), sm.state[warp][c][lane] = f4(s[c]), sm.grad[warp][c][lane] = f4(q[c]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kShare; ++k) {
      const int e = threadIdx.x + k * 32 * W;
      const int at_e = e < kHalf ? e : e - kHalf;
      float* local = reinterpret_cast<float*>(e < kHalf ? sm.state[0] : sm.grad[W - 1]) + at_e;
      const float* decay = reinterpret_cast<const float*>(e < kHalf ? sm.decay[0] : sm.decay[W - 1]) + at_e;
      const int step = e < kHalf ? kHalf : -kHalf;
#pragma unroll
      for (int w = 0; w < W; ++w, local += step, decay += step) {
        const float in = carry[k];
        carry[k] = fmaf(*decay, in, *local);
        *local = in;
      }
    }
    __syncthreads();
    S4 first[CPL], h[NT][CPL], grad[CPL];   // grad: a_(t+1) g_(t+1)
#pragma unroll
    for (int c = 0; c < CPL; ++c) first[c] = s4(sm.state[warp][c][lane]), grad[c] = s4(sm.grad[warp][c][lane]);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const S4 B = s4(*reinterpret_cast<const float4*>(&my.B[t][4 * i]));
#pragma unroll
      for (int c = 0; c < CPL; ++c) h[t][c] = fma(decay[t][c], t ? h[t - 1][c] : first[c], mul(B, my.dtu[t][g * CPL + c]));
    }
#pragma unroll
    for (int r = kRounds - 1; r >= 0; --r) {
      float sum_y[LPC], sum_b[LPC], sum_a[LPC];
#pragma unroll
      for (int q = TILE::kRound - 1; q >= 0; --q) {
        const int t = r * TILE::kRound + q;
        const S4 B = s4(*reinterpret_cast<const float4*>(&my.B[t][4 * i])), C = s4(*reinterpret_cast<const float4*>(&my.C[t][4 * i]));
        S4 dB = splat(0.f), dC = splat(0.f);
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          const int ch = g * CPL + c;
          const float d = my.d[t][ch];
          const S4 now = fma(C, d, grad[c]);
          sum_y[q * CPL + c] = add_up(mul(C, h[t][c]));
          sum_b[q * CPL + c] = add_up(mul(B, now));
          dB = fma(now, my.dtu[t][ch], dB);
          dC = fma(h[t][c], d, dC);
          grad[c] = mul(decay[t][c], now);
          const S4 e = mul(grad[c], t ? h[t - 1][c] : first[c]);
          sum_a[q * CPL + c] = add_up(mul(e, rate[c]));
          drate[c] = fma(e, my.dt[t][ch], drate[c]);
        }
        float v[8] = {dB.a.x, dB.a.y, dB.b.x, dB.b.y, dC.a.x, dC.a.y, dC.b.x, dC.b.y};
        sum_over<8, TILE::kGroups, LPC>(v, lane);
        if (base + t < at.tokens) {
          float* to = to_tokens + (int64_t)(base + t) * (2 * TILE::kStates);
#pragma unroll
          for (int k = 0; k < kLeft; ++k) to[k] = v[k];
        }
      }
      sum_over<LPC, LPC, 1>(sum_y, lane);
      sum_over<LPC, LPC, 1>(sum_b, lane);
      sum_over<LPC, LPC, 1>(sum_a, lane);
      const int64_t t = base + r * TILE::kRound + sub;
      if (t < at.tokens && own_ok) {
        float d = dy[r];
        if (pz) {
          pdz[t * a.dz.token_pitch] = from_f<T>(d * fmaf(skip, u[r], sum_y[0]) * d_silu(z[r]));
          d *= silu(z[r]);
        }
        const float ddt = fmaf(sum_b[0], u[r], sum_a[0] * (1.f / kLog2e)) * slope[r];
        pdu[t * a.du.token_pitch] = from_f<T>(fmaf(sum_b[0], dts[r], skip * d));
        pddt[t * a.ddt.token_pitch] = from_f<T>(ddt);
        dskip = fmaf(d, u[r], dskip), dbias += ddt;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kShare; ++k) {
    const int e = threadIdx.x + k * 32 * W;
    int ch, n;
    if (a.dstate_in && e >= kHalf && state_at(e - kHalf, &ch, &n)) a.dstate_in[((int64_t)seq * a.channels + tile.channel + ch) * a.states + n] = carry[k];
  }
  // what the warps have of dA, dD and ddt_bias, in their order
  __syncthreads();
#pragma unroll
  for (int c = 0; c < CPL; ++c) sm.state[warp][c][lane] = f4(drate[c]);
  reinterpret_cast<float*>(sm.decay[warp])[lane] = dskip, reinterpret_cast<float*>(sm.decay[warp])[32 + lane] = dbias;
  __syncthreads();
  for (int e = threadIdx.x; e < kHalf; e += 32 * W) {
    int ch, n;
    const bool there = state_at(e, &ch, &n);
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) s += reinterpret_cast<const float*>(sm.state[w])[e];
    if (there) out.rates[((int64_t)seq * a.channels + tile.channel + ch) * TILE::kStates + n] = s;
  }
  if (threadIdx.x < 2 * TILE::kChannels) {
    const int which = threadIdx.x / TILE::kChannels, ch = threadIdx.x % TILE::kChannels;
    float s = 0.f;
    for (int w = 0; w < W; ++w)
      for (int q = 0; q < TILE::kRound; ++q)   // the lanes that had this channel
        s += reinterpret_cast<const float*>(sm.decay[w])[32 * which + (ch / CPL) * LPC + q * CPL + ch % CPL];
    if (ch < tile.left) out.skips[((int64_t)seq * 2 + which) * a.channels + tile.channel + ch] = s;
  }
}

// dB, dC of a token: over the tiles of its group, in their order.
template <typename T>
__global__ void __launch_bounds__(256) k_scan_sum_tokens(lasp_scan_args a, const float* part, int tiles, int padded) {
  const int64_t all = (int64_t)a.rows * a.tokens, wide = 2 * padded, e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= all * wide) return;
  const int group = blockIdx.y, in_group = tiles / a.groups;
  const int64_t token = e / wide;
  const int at = (int)(e % wide), n = at / 8 * 4 + at % 4, row = (int)(token / a.tokens), t = (int)(token - (int64_t)row * a.tokens);
  if (n >= a.states) return;
  float s = 0.f;
  bool inside = true;
  if (a.sequences) {
    const Sequences q{a.offsets, a.index_bits, a.sequences, a.tokens};
    inside = t >= q.at(0) && t < q.at(a.sequences);
  }
  if (inside) {
    const float* p = part + (int64_t)group * in_group * all * wide + e;
#pragma unroll 8
    for (int k = 0; k < in_group; ++k) s += p[(int64_t)k * all * wide];
  }
  const lasp_tokens& to = at % 8 < 4 ? a.dB : a.dC;
  static_cast<T*>(to.data)[(int64_t)row * to.row_pitch + (int64_t)t * to.token_pitch + (int64_t)group * to.group_pitch + n] = from_f<T>(s);
}

// dA, dD, ddt_bias: over the sequences, in their order.
template <typename T>
__global__ void __launch_bounds__(256) k_scan_sum_sequences(lasp_scan_args a, Partial in, int padded, int sequences) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, width = padded + 2;
  if (e >= a.channels * width) return;
  const int64_t c = e / width;
  const int n = (int)(e % width);
  const bool f32 = a.param_dtype == LASP_F32;
  float s = 0.f;
  if (n < padded) {
    if (n >= a.states || !a.dA) return;
    for (int q = 0; q < sequences; ++q) s += in.rates[((int64_t)q * a.channels + c) * padded + n];
    a.dA[c * a.states + n] = s;
  } else {
    void* to = n == padded ? a.dD : a.ddt_bias;
    if (!to) return;
    for (int q = 0; q < sequences; ++q) s += in.skips[((int64_t)q * 2 + (n - padded)) * a.channels + c];
    store_param<T>(to, f32, c, s);
  }
}

struct Plan {
  int tiles, sequences, padded;
  size_t tokens, rates, skips;   // floats
};
template <class TILE>
Plan plan_as(const lasp_scan_args& a) {
  Plan p;
  p.tiles = tiles_of<TILE>(a.channels, a.groups), p.sequences = a.sequences ? a.sequences : a.rows, p.padded = TILE::kStates;
  p.tokens = (size_t)p.tiles * a.rows * a.tokens * 2 * p.padded;
  p.rates = (size_t)p.sequences * a.channels * p.padded, p.skips = (size_t)p.sequences * 2 * a.channels;
  return p;
}

template <typename T, int LPC, int CPL, int W, int NT>
cudaError_t launch(const lasp_scan_args& a, cudaStream_t st) {
  constexpr auto kernel = k_scan_backward<T, LPC, CPL, W, NT>;
  constexpr size_t smem = sizeof(Shared<T, LPC, CPL, W, NT>);
  const cudaError_t err = opt_in_smem<kernel>(smem);
  if (err != cudaSuccess) return err;
  const Plan p = plan_as<Tile<LPC, CPL>>(a);
  float* ws = static_cast<float*>(a.ws);
  const Partial out{ws, ws + p.tokens, ws + p.tokens + p.rates};
  kernel<<<(unsigned)(p.tiles * (p.sequences + (a.sequences ? 1 : 0))), 32 * W, smem, st>>>(a, p.tiles, out);
  const int64_t per_group = (int64_t)a.rows * a.tokens * 2 * p.padded, params = (int64_t)a.channels * (p.padded + 2);
  if (per_group) k_scan_sum_tokens<T><<<dim3((unsigned)((per_group + 255) / 256), a.groups), 256, 0, st>>>(a, out.tokens, p.tiles, p.padded);
  if (a.dA || a.dD || a.ddt_bias) k_scan_sum_sequences<T><<<(unsigned)((params + 255) / 256), 256, 0, st>>>(a, out, p.padded, p.sequences);
  return cudaGetLastError();
}

template <typename T>
cudaError_t backward_as(const lasp_scan_args& a, cudaStream_t st) {
  switch (padded_states(a.states)) {
    case 16: return launch<T, 4, 2, 16, 4>(a, st);
    case 32: return launch<T, 8, 2, 16, 4>(a, st);
    default: return launch<T, 16, 2, 8, 8>(a, st);
  }
}

}  // namespace

cudaError_t scan_backward(const lasp_scan_args& a, cudaStream_t st) {
  return a.dtype == LASP_F32 ? backward_as<float>(a, st) : a.dtype == LASP_BF16 ? backward_as<__nv_bfloat16>(a, st) : backward_as<__half>(a, st);
}
// The forward pass keeps states of as many numbers as its tiles have.
size_t scan_kept(const lasp_scan_args& a) { return (size_t)kept_states(a) * a.channels * padded_states(a.states) * sizeof(float); }
size_t scan_workspace(const lasp_scan_args& a) {
  const int padded = padded_states(a.states);
  const Plan p = padded <= 16 ? plan_as<Tile<4, 2>>(a) : padded == 32 ? plan_as<Tile<8, 2>>(a) : plan_as<Tile<16, 2>>(a);
  return (p.tokens + p.rates + p.skips) * sizeof(float);
}

}  // namespace lasp
