// Selective scan over prompts and training batches, forward.  How a block shares out its work is in scan_common.cuh.
//
// One barrier a chunk: while the first four warps take chunk j through the recurrence, the next four prepare chunk j + 2 (step sizes, inputs,
// B and C as numbers), and the last four finish chunk j - 1 (gate, output), send for chunk j + 5 and wait for chunk j + 3.  Measured, 16 states,
// bf16: 2 x 2048 x 4096 140 us (256 blocks on 148 SMs; 20 us of memory, 60 of exponentials), 1 x 16384 x 4096 598 (128 blocks; 82, 238).
#include "scan_common.cuh"

namespace lasp {
namespace {

constexpr int kResident = 2;   // blocks of an SM
constexpr int kStages = 8;   // chunks that are here, or on their way, as they are in global memory: j - 1 to j + 5
template <typename T, int LPC>
struct Shared {
  using TILE = Tile<LPC>;
  Vec<T, TILE::kEach> u[kStages][TILE::kUnits], dt[kStages][TILE::kUnits], z[kStages][TILE::kUnits];
  Vec<T, 4> B[kStages][TILE::kStateUnits], C[kStages][TILE::kStateUnits];
  float2 step[3][kChunk][TILE::kChannels];                                          // dt, dt u
  float4 B4[3][kChunk][LPC], C4[3][kChunk][LPC];
  float y[2][kChunk][TILE::kRow];                                                   // <C, h>
};

// wide: u, dt, z, y can be read and written by kEach, B and C by four.
template <typename T, int LPC>
__global__ void __launch_bounds__(kThreads, 2) k_scan_forward(lasp_scan_args a, int tiles, Cuts cuts, bool wide) {
  using TILE = Tile<LPC>;
  constexpr int kEach = TILE::kEach, kVecs = TILE::kVecs;
  extern __shared__ __align__(16) char raw_smem[];
  auto& sm = *reinterpret_cast<Shared<T, LPC>*>(raw_smem);
  const int role = threadIdx.x / kGroup, me = threadIdx.x % kGroup;
  const int tile_index = blockIdx.x % tiles, slot = blockIdx.x / tiles;
  const TilePlace<TILE> tile(tile_index, a.channels, a.groups);
  if (slot == cuts.slots) return fill_outside<T, TILE>(a, a.y, tile);
  const Stretch at(a, slot, cuts.length);
  if (at.index == at.count) return;
  const int chunks = (at.tokens + kChunk - 1) / kChunk;
  const bool f32 = a.param_dtype == LASP_F32, gated = a.z.data != nullptr, whole = wide && tile.left >= TILE::kChannels;
  const auto rows = [&](const lasp_tokens& t) {
    return static_cast<T*>(t.data) + (int64_t)at.row * t.row_pitch + (int64_t)at.begin * t.token_pitch + tile.channel;
  };
  // Barriers: chunks + 3 of them in every role.
  if (role == 0) {
    take_registers<144>();
    const int lane = me % 32, i = lane / TILE::kGroups, ch = me / 32 * TILE::kGroups + lane % TILE::kGroups;
    const bool mine = ch < tile.left;
    const int64_t state_row = ((int64_t)at.seq * a.channels + tile.channel + ch) * a.states;
    const S4 A = mine ? rates(a.A + (int64_t)(tile.channel + ch) * a.states, 4 * i, a.states) : splat(0.f);
    S4 h = mine && a.state_in ? s4(four_of(a.state_in + state_row, 4 * i, a.states)) : splat(0.f);
    if (at.index) h = carry<TILE>(a, cuts, at, 0, at.index * kParts, false, h, A, tiles, tile_index, me, ch);
    float4* kept = a.kept ? static_cast<float4*>(a.kept) + (at.chunk * tiles + tile_index) * kGroup + me : nullptr;
    constexpr int kTurn = 8, kRound = LPC < kTurn ? LPC : kTurn, kSame = LPC / kRound;   // tokens taken, and summed, at a time
    S4 decay[kTurn], state[kTurn];   // state: first what a token puts in, then the state behind it
    const auto ahead = [&](int buf, int t0, int t) {   // of token t0 + t
      const float2 step = sm.step[buf][t0 + t][ch];
      decay[t] = decay_of(A, step.x);
      state[t] = mul(load4(&sm.B4[buf][t0 + t][i]), f2(step.y, step.y));
    };
    __syncthreads();   // chunk 0 is here
    __syncthreads();   // chunk 0 is prepared
    __syncthreads();   // chunk 1
    if (chunks) {
#pragma unroll
      for (int t = 0; t < kTurn; ++t) ahead(0, 0, t);
    }
    int buf = 0;
    for (int chunk = 0; chunk < chunks; ++chunk) {
      if (kept) *kept = f4(h), kept += (int64_t)tiles * kGroup;
      const int next = buf == 2 ? 0 : buf + 1;
#pragma unroll
      for (int t0 = 0; t0 < kChunk; t0 += kTurn) {
        S4 now[kTurn];
#pragma unroll
        for (int t = 0; t < kTurn; ++t) h = now[t] = fma(decay[t], h, state[t]);
        // the next tokens' decays go on beside the sums over these: neither needs the other
#pragma unroll
        for (int t = 0; t < kTurn; ++t) ahead(t0 + kTurn < kChunk ? buf : next, (t0 + kTurn) % kChunk, t);
#pragma unroll
        for (int r = 0; r < kTurn; r += kRound) {
          float sums[kRound];
#pragma unroll
          for (int t = 0; t < kRound; ++t) sums[t] = dot(load4(&sm.C4[buf][t0 + r + t][i]), now[r + t]);
          sum_over<kRound, LPC, TILE::kGroups>(sums, lane);
          if (kSame == 1 || i % kSame == 0) sm.y[chunk & 1][t0 + r + i / kSame][ch] = sums[0];
        }
      }
      buf = next;
      __syncthreads();
    }
    if (a.state_out && mine && at.index == at.count - 1) store_four(a.state_out + state_row, 4 * i, a.states, f4(h));
  } else if (role == 1) {
    give_registers<48>();
    static_assert(TILE::kUnits <= kGroup, "a thread has at most one unit of each tensor");
    const int row = me / kVecs, c0 = me % kVecs * kEach;
    float bias[kEach];
    params_of<T>(a.dt_bias, f32, tile.channel + c0, tile.left - c0, bias);
    __syncthreads();
    for (int chunk = 0, buf = 0; chunk < chunks + 2; ++chunk, buf = buf == 2 ? 0 : buf + 1) {
      const int stage = chunk % kStages, t0 = chunk * kChunk;
      if (chunk < chunks) {
        if (me < TILE::kUnits) {
          const bool there = t0 + row < at.tokens;   // behind the end the step is zero: the state stays
          float dt[kEach], u[kEach];
          numbers<T, kEach>(sm.dt[stage][me], dt), numbers<T, kEach>(sm.u[stage][me], u);
#pragma unroll
          for (int k = 0; k < kEach; k += 2) {
            F2 d = add2(f2(dt[k], dt[k + 1]), f2(bias[k], bias[k + 1]));
            if (a.softplus) d = softplus(d);
            apart(mul2(d, f2(u[k], u[k + 1])), u[k], u[k + 1]), apart(d, dt[k], dt[k + 1]);
          }
          put_steps(&sm.step[buf][row][c0], dt, u, me, there);
        }
#pragma unroll
        for (int v = me; v < 2 * TILE::kStateUnits; v += kGroup) {   // (B's and C's for whole warps each)
          const int k = v % TILE::kStateUnits;
          const bool there = t0 + k / LPC < at.tokens;
          float x[4];
          numbers<T, 4>(v < TILE::kStateUnits ? sm.B[stage][k] : sm.C[stage][k], x);
          (v < TILE::kStateUnits ? sm.B4 : sm.C4)[buf][k / LPC][k % LPC] = there ? make_float4(x[0], x[1], x[2], x[3]) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
      __syncthreads();
    }
  } else {
    give_registers<48>();
    const int row = me / kVecs, c0 = me % kVecs * kEach, left = tile.left - c0;
    const bool unit = me < TILE::kUnits;
    float skip[kEach];
    params_of<T>(a.D, f32, tile.channel + c0, left, skip);
    const T *pu = rows(a.u) + c0, *pdt = rows(a.dt) + c0, *pz = gated ? rows(a.z) + c0 : nullptr;
    const auto state_rows = [&](const lasp_tokens& t) {
      return static_cast<const T*>(t.data) + (int64_t)at.row * t.row_pitch + (int64_t)at.begin * t.token_pitch + (int64_t)tile.group * t.group_pitch;
    };
    const T *pB = state_rows(a.B), *pC = state_rows(a.C);
    T* py = rows(a.y) + c0;
    const auto fetch = [&](int chunk) {   // (behind the end: the last token, which is not used)
      const int stage = chunk % kStages, t0 = chunk * kChunk;
      if (chunk < chunks) {
        if (unit) {
          const int64_t t = min(t0 + row, at.tokens - 1);
          bring<T, kEach>(&sm.u[stage][me], pu + t * a.u.token_pitch, whole, left);
          bring<T, kEach>(&sm.dt[stage][me], pdt + t * a.dt.token_pitch, whole, left);
          if (gated) bring<T, kEach>(&sm.z[stage][me], pz + t * a.z.token_pitch, whole, left);
        }
#pragma unroll
        for (int v = me; v < 2 * TILE::kStateUnits; v += kGroup) {
          const int k = v % TILE::kStateUnits, n = k % LPC * 4;
          const int64_t t = min(t0 + k / LPC, at.tokens - 1);
          if (v < TILE::kStateUnits)
            bring<T, 4>(&sm.B[stage][k], pB + t * a.B.token_pitch + n, wide && n + 4 <= a.states, a.states - n);
          else
            bring<T, 4>(&sm.C[stage][k], pC + t * a.C.token_pitch + n, wide && n + 4 <= a.states, a.states - n);
        }
      }
      commit_copies();
    };
    const auto finish = [&](int chunk) {
      const int stage = chunk % kStages, t = chunk * kChunk + row;
      if (!unit) return;
      float y[kEach], u[kEach], z[kEach];
      numbers<T, kEach>(sm.u[stage][me], u);
#pragma unroll
      for (int k = 0; k < kEach; ++k) y[k] = fmaf(skip[k], u[k], sm.y[chunk & 1][row][c0 + k]);
      if (gated) {
        numbers<T, kEach>(sm.z[stage][me], z);
#pragma unroll
        for (int k = 0; k < kEach; ++k) y[k] *= silu(z[k]);
      }
      if (t < at.tokens) put_some<T, kEach>(py + (int64_t)t * a.y.token_pitch, y, whole, left);
    };
    fetch(0), fetch(1), fetch(2);
    await_copies<2>();
    __syncthreads();
    for (int chunk = -2; chunk < chunks; ++chunk) {
      fetch(chunk + 5);
      if (chunk > 0) finish(chunk - 1);
      await_copies<2>();   // chunk + 3 is here
      __syncthreads();
    }
    if (chunks) finish(chunks - 1);
  }
}

template <typename T, int LPC>
cudaError_t launch(const lasp_scan_args& a, cudaStream_t st) {
  using TILE = Tile<LPC>;
  constexpr auto kernel = k_scan_forward<T, LPC>;
  constexpr size_t smem = sizeof(Shared<T, LPC>);
  static_assert(blocks_of_sm(smem) == kResident, "");
  const cudaError_t err = ready<kernel>(smem);
  if (err != cudaSuccess) return err;
  const int tiles = tiles_of<TILE>(a.channels, a.groups);
  const Cuts cuts = cuts_of<TILE>(a, tiles, false, kResident, static_cast<float*>(a.ws));
  const bool wide = (a.channels / a.groups) % TILE::kEach == 0 && reads_by<T>(a.u, TILE::kEach) && reads_by<T>(a.dt, TILE::kEach) &&
                    reads_by<T>(a.z, TILE::kEach) && reads_by<T>(a.y, TILE::kEach) && reads_by<T>(a.B, 4) && reads_by<T>(a.C, 4);
  if (cuts.length != kUncut)
    if (const cudaError_t e = scan_parts<T, LPC>(a, cuts, tiles, false, st); e != cudaSuccess) return e;
  // (one slot more: what lies in no sequence)
  kernel<<<(unsigned)(tiles * (cuts.slots + (a.sequences ? 1 : 0))), kThreads, smem, st>>>(a, tiles, cuts, wide);
  return cudaGetLastError();
}

template <typename T>
cudaError_t forward_as(const lasp_scan_args& a, cudaStream_t st) {
  switch (padded_states(a.states)) {
    case 16: return launch<T, 4>(a, st);
    case 32: return launch<T, 8>(a, st);
    default: return launch<T, 16>(a, st);
  }
}

template <int LPC>
size_t workspace_as(const lasp_scan_args& a) {
  const int tiles = tiles_of<Tile<LPC>>(a.channels, a.groups);
  return (size_t)floats_of<Tile<LPC>>(cuts_of<Tile<LPC>>(a, tiles, false, kResident, nullptr), tiles) * sizeof(float);
}

}  // namespace

size_t scan_forward_workspace(const lasp_scan_args& a) {
  const int padded = padded_states(a.states);
  return padded == 16 ? workspace_as<4>(a) : padded == 32 ? workspace_as<8>(a) : workspace_as<16>(a);
}
cudaError_t scan_forward(const lasp_scan_args& a, cudaStream_t st) {
  return a.dtype == LASP_F32 ? forward_as<float>(a, st) : a.dtype == LASP_BF16 ? forward_as<__nv_bfloat16>(a, st) : forward_as<__half>(a, st);
}

}  // namespace lasp
