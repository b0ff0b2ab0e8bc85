// Selective scan, backward.  With d_t = dy_t silu(z_t) and the gradient g that reaches the state behind token t,
//
//   g_t = C_t d_t + a_(t+1) g_(t+1),   a_t = exp(dt_t A)
//   dC_t = sum_c d_t h_t,  dB_t = sum_c g_t dt_t u_t,  du_t = dt_t <g_t, B_t> + D d_t
//   e_t = a_t g_t h_(t-1):  d dt_t = u_t <g_t, B_t> + <e_t, A>,  dA = sum_t dt_t e_t
//
// Blocks share out their work as in the forward pass (scan_common.cuh) and walk back along the tokens.  The warps that hold the states take a
// chunk up from the state that the forward pass has kept ahead of it, and then half a chunk at a time: up for the states, down for the
// gradients, with the decays and states of eight tokens in registers.  (Those of 16 do not fit, and a state kept for every eighth
// token would cost 32 bytes of memory for every eight tokens and state more than the 8 exponentials that the first half takes twice.)  dB and dC are sums over channels: each block leaves
// its tile's, and k_scan_sums adds those up in the order of the tiles, so that results do not depend on when blocks run.
//
// Measured, 2 x 2048 x 4096 bf16, 16 states: 420 us, of which k_scan_sums 12.  121 instructions for a warp's four states a lane and token (60 % of the issue slots;
// 28 of them the sums over channels) and 32 turns of shared memory (60 % of the clocks) bound it together; memory would take 50 us.
#include "scan_common.cuh"

namespace lasp {
namespace {

constexpr int kSumsOfToken = 8;   // numbers of a four of states: 4 dB, 4 dC
template <typename T, int LPC>
struct Shared {
  using TILE = Tile<LPC>;
  static constexpr int kStages = sizeof(T) == 4 ? 6 : 7;   // chunks that are here, or on their way, as they are in global memory
  Vec<T, TILE::kEach> u[kStages][TILE::kUnits], dt[kStages][TILE::kUnits], z[kStages][TILE::kUnits], dy[kStages][TILE::kUnits];
  Vec<T, 4> B[kStages][TILE::kStateUnits], C[kStages][TILE::kStateUnits];
  float2 step[3][kChunk][TILE::kChannels];          // dt, dt u
  float d[3][kChunk][TILE::kChannels];
  float4 B4[3][kChunk][LPC], C4[3][kChunk][LPC];
  float y[2][kChunk][TILE::kRow], gB[2][kChunk][TILE::kRow], eA[2][kChunk][TILE::kRow];   // <C, h>, <g, B>, <e, A>
  float4 sums[2][kChunk][4][kSumsOfToken * LPC / 4];   // of each warp
  alignas(16) float skip[TILE::kChannels], bias[TILE::kChannels];   // (in registers they would be spilled)
};

// What a backward pass writes beside its results, in the order of the workspace.
struct Partial {
  float4* tokens;   // [tile][row * tokens + token][LPC][8]: of each four of states its 4 dB, 4 dC
  float4* rates;    // [slot][tile][kGroup]: dA, as the lanes hold it
  float* skips;     // [slot][2][channel]: dD, ddt_bias
};

// wide: the tensors of tokens can be read and written by kEach, B and C by four.  GATED: there is a z, whose gradient takes <C, h>
// (2 x 1000 x 1536 fp32 of 32 states, no z, forward and backward: 242 us with those sums, 233 without).
template <typename T, int LPC, bool GATED>
__global__ void __launch_bounds__(kThreads, 2) k_scan_backward(lasp_scan_args a, int tiles, Partial out, Cuts cuts, bool wide) {
  using TILE = Tile<LPC>;
  using SHARED = Shared<T, LPC>;
  constexpr int kEach = TILE::kEach, kVecs = TILE::kVecs, kStages = SHARED::kStages, kLead = kStages - 3;
  extern __shared__ __align__(16) char raw_smem[];
  auto& sm = *reinterpret_cast<SHARED*>(raw_smem);
  const int role = threadIdx.x / kGroup, me = threadIdx.x % kGroup;
  const int tile_index = blockIdx.x % tiles, slot = blockIdx.x / tiles;
  const TilePlace<TILE> tile(tile_index, a.channels, a.groups);
  if (slot == cuts.slots) {
    fill_outside<T, TILE>(a, a.du, tile), fill_outside<T, TILE>(a, a.ddt, tile), fill_outside<T, TILE>(a, a.dz, tile);
    return;
  }
  const Stretch at(a, slot, cuts.length);
  if (at.index == at.count) {   // no segment: nothing to add to the sums
    if (threadIdx.x < kGroup) out.rates[((int64_t)slot * tiles + tile_index) * kGroup + threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int e = threadIdx.x; e < 2 * TILE::kChannels; e += kThreads)
      if (const int c = e % TILE::kChannels; c < tile.left) out.skips[((int64_t)slot * 2 + e / TILE::kChannels) * a.channels + tile.channel + c] = 0.f;
    return;
  }
  const int chunks = (at.tokens + kChunk - 1) / kChunk;   // number k of them is chunk chunks - 1 - k of the segment
  const bool f32 = a.param_dtype == LASP_F32, whole = wide && tile.left >= TILE::kChannels;
  for (int c = threadIdx.x; c < TILE::kChannels; c += kThreads) {
    const bool there = c < tile.left;
    sm.skip[c] = there && a.D ? param<T>(a.D, f32, tile.channel + c) : 0.f;
    sm.bias[c] = there && a.dt_bias ? param<T>(a.dt_bias, f32, tile.channel + c) : 0.f;
  }
  __syncthreads();
  const auto rows = [&](const lasp_tokens& t) {
    return static_cast<T*>(t.data) + (int64_t)at.row * t.row_pitch + (int64_t)at.begin * t.token_pitch + tile.channel;
  };
  // Barriers: chunks + 3 of them in every role.
  if (role == 0) {
    take_registers<152>();
    const int lane = me % 32, i = lane / TILE::kGroups, ch = me / 32 * TILE::kGroups + lane % TILE::kGroups;
    const bool mine = ch < tile.left;
    const int64_t state_row = ((int64_t)at.seq * a.channels + tile.channel + ch) * a.states;
    const S4 A = mine ? rates(a.A + (int64_t)(tile.channel + ch) * a.states, 4 * i, a.states) : splat(0.f);
    S4 grad = mine && a.dstate_out ? s4(four_of(a.dstate_out + state_row, 4 * i, a.states)) : splat(0.f);   // a_(t+1) g_(t+1)
    if (at.index < at.count - 1) grad = carry<TILE>(a, cuts, at, (at.index + 1) * kParts, (at.sequence_tokens - 1) / cuts.part + 1, true, grad, A, tiles, tile_index, me, ch);
    S4 dA = splat(0.f);
    const float4* kept = static_cast<const float4*>(a.kept) + ((at.chunk + chunks - 1) * tiles + tile_index) * kGroup + me;
    constexpr int kLeft = 8 / TILE::kGroups;   // of 8 sums over a warp's channels, how many a lane is left with
    constexpr int kHalf = kChunk / 2, kRound = 4, kSame = LPC / kRound;   // tokens whose sums are made together
    float4 first = chunks ? *kept : make_float4(0.f, 0.f, 0.f, 0.f);
    __syncthreads();   // the first chunk is here
    __syncthreads();   // it is prepared
    __syncthreads();   // the second
    for (int k = 0, buf = 0; k < chunks; ++k, buf = buf == 2 ? 0 : buf + 1) {
      const S4 start = s4(first);
      kept -= (int64_t)tiles * kGroup;
      if (k + 1 < chunks) first = *kept;
      S4 decay[kHalf], h[kHalf];
      const auto ahead = [&](int t0) {   // decays, and in h what the tokens put in
#pragma unroll
        for (int t = 0; t < kHalf; ++t) {
          const float2 step = sm.step[buf][t0 + t][ch];
          decay[t] = decay_of(A, step.x);
          h[t] = mul(load4(&sm.B4[buf][t0 + t][i]), f2(step.y, step.y));
        }
      };
      S4 middle = start, e_sum = splat(0.f);   // (dA of the chunk: added up by themselves, sums of many tokens lose half as many bits)
      ahead(0);
#pragma unroll
      for (int t = 0; t < kHalf; ++t) middle = fma(decay[t], middle, h[t]);
#pragma unroll
      for (int half = 1; half >= 0; --half) {
        const S4 before = half ? middle : start;
        ahead(half * kHalf);
#pragma unroll
        for (int t = 0; t < kHalf; ++t) h[t] = fma(decay[t], t ? h[t - 1] : before, h[t]);
#pragma unroll
        for (int r = kHalf - kRound; r >= 0; r -= kRound) {
          float y[kRound], gB[kRound], eA[kRound], over[kRound][kLeft];   // (all stored together: what lies in between could not be read ahead)
#pragma unroll
          for (int q = kRound - 1; q >= 0; --q) {
            const int t = half * kHalf + r + q;
            const float2 step = sm.step[buf][t][ch];
            const S4 B = load4(&sm.B4[buf][t][i]), C = load4(&sm.C4[buf][t][i]), &now = h[r + q];
            const F2 d = f2(sm.d[buf][t][ch], sm.d[buf][t][ch]);
            const S4 g = fma(C, d, grad), dB = mul(g, f2(step.y, step.y)), dC = mul(now, d);
            if constexpr (GATED) y[q] = dot(C, now);
            gB[q] = dot(B, g);
            grad = mul(decay[r + q], g);
            const S4 e = mul(grad, r + q ? h[r + q - 1] : before);
            eA[q] = dot(e, A);
            e_sum = fma(e, f2(step.x, step.x), e_sum);
            float v[8];
            apart(dB.a, v[0], v[1]), apart(dB.b, v[2], v[3]), apart(dC.a, v[4], v[5]), apart(dC.b, v[6], v[7]);
            sum_over<8, TILE::kGroups, 1>(v, lane);
#pragma unroll
            for (int x = 0; x < kLeft; ++x) over[q][x] = v[x];
          }
          if constexpr (GATED) sum_over<kRound, LPC, TILE::kGroups>(y, lane);
          sum_over<kRound, LPC, TILE::kGroups>(gB, lane), sum_over<kRound, LPC, TILE::kGroups>(eA, lane);
#pragma unroll
          for (int q = 0; q < kRound; ++q) store_vec<float, kLeft>(reinterpret_cast<float*>(sm.sums[k & 1][half * kHalf + r + q][me / 32]) + lane * kLeft, over[q]);
          if (kSame == 1 || i % kSame == 0) {
            const int t = half * kHalf + r + i / kSame;
            if constexpr (GATED) sm.y[k & 1][t][ch] = y[0];
            sm.gB[k & 1][t][ch] = gB[0], sm.eA[k & 1][t][ch] = eA[0];
          }
        }
      }
      dA = {add2(dA.a, e_sum.a), add2(dA.b, e_sum.b)};
      __syncthreads();
    }
    if (a.dstate_in && mine && at.index == 0) store_four(a.dstate_in + state_row, 4 * i, a.states, f4(grad));
    out.rates[((int64_t)slot * tiles + tile_index) * kGroup + me] = f4(dA);
  } else if (role == 1) {
    // while the states are at number k: prepare k + 2, send for k + kLead, add up k - 1
    give_registers<40>();
    const int row = me / kVecs, c0 = me % kVecs * kEach, left = tile.left - c0;
    const bool unit = me < TILE::kUnits;
    constexpr int kSums = kSumsOfToken * LPC / 4;
    float4* to_tokens = out.tokens + ((int64_t)tile_index * a.rows * a.tokens + (int64_t)at.row * a.tokens + at.begin) * kSums;
    const auto state_rows = [&](const lasp_tokens& t) {
      return static_cast<const T*>(t.data) + (int64_t)at.row * t.row_pitch + (int64_t)at.begin * t.token_pitch + (int64_t)tile.group * t.group_pitch;
    };
    const auto fetch = [&](int k) {   // (behind the end: the last token, which is not used)
      if (k < chunks) {
        const int stage = k % kStages, t0 = (chunks - 1 - k) * kChunk;
        if (unit) {
          const int64_t t = min(t0 + row, at.tokens - 1);
          bring<T, kEach>(&sm.u[stage][me], rows(a.u) + t * a.u.token_pitch + c0, whole, left);
          bring<T, kEach>(&sm.dt[stage][me], rows(a.dt) + t * a.dt.token_pitch + c0, whole, left);
          bring<T, kEach>(&sm.dy[stage][me], rows(a.dy) + t * a.dy.token_pitch + c0, whole, left);
          if constexpr (GATED) bring<T, kEach>(&sm.z[stage][me], rows(a.z) + t * a.z.token_pitch + c0, whole, left);
        }
#pragma unroll
        for (int v = me; v < 2 * TILE::kStateUnits; v += kGroup) {   // (B's and C's for whole warps each)
          const int q = v % TILE::kStateUnits, n = q % LPC * 4;
          const int64_t t = min(t0 + q / LPC, at.tokens - 1);
          if (v < TILE::kStateUnits)
            bring<T, 4>(&sm.B[stage][q], state_rows(a.B) + t * a.B.token_pitch + n, wide && n + 4 <= a.states, a.states - n);
          else
            bring<T, 4>(&sm.C[stage][q], state_rows(a.C) + t * a.C.token_pitch + n, wide && n + 4 <= a.states, a.states - n);
        }
      }
      commit_copies();
    };
    const auto add_up = [&](int k) {   // dB, dC of the tile
      const int t0 = (chunks - 1 - k) * kChunk;
#pragma unroll
      for (int v = me; v < kChunk * kSums; v += kGroup) {
        const int token = v / kSums, q = v % kSums;
        float4 s = sm.sums[k & 1][token][0][q];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
          const float4 x = sm.sums[k & 1][token][w][q];
          s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
        }
        if (t0 + token < at.tokens) to_tokens[(int64_t)(t0 + token) * kSums + q] = s;
      }
    };
#pragma unroll
    for (int k = 0; k < kLead - 2; ++k) fetch(k);
    __syncthreads();
    for (int k = -2, buf = 0; k < chunks; ++k, buf = buf == 2 ? 0 : buf + 1) {
      fetch(k + kLead);
      await_copies<kLead - 2>();   // k + 2 is here, as far as this thread has brought it
      const int stage = (k + 2) % kStages, t0 = (chunks - 3 - k) * kChunk;
      if (k + 2 < chunks) {
        if (unit) {
          const bool there = t0 + row < at.tokens;   // behind the end the step is zero: the state stays, and no gradient comes in
          float dt[kEach], u[kEach], d[kEach];
          numbers<T, kEach>(sm.dt[stage][me], dt), numbers<T, kEach>(sm.u[stage][me], u), numbers<T, kEach>(sm.dy[stage][me], d);
          if constexpr (GATED) {
            float z[kEach];
            numbers<T, kEach>(sm.z[stage][me], z);
#pragma unroll
            for (int q = 0; q < kEach; ++q) d[q] *= silu(z[q]);
          }
#pragma unroll
          for (int q = 0; q < kEach; q += 2) {
            F2 s = add2(f2(dt[q], dt[q + 1]), pair_of(&sm.bias[c0 + q]));
            if (a.softplus) s = softplus(s);
            apart(mul2(s, f2(u[q], u[q + 1])), u[q], u[q + 1]), apart(s, dt[q], dt[q + 1]);
          }
          put_steps(&sm.step[buf][row][c0], dt, u, me, there);
          *reinterpret_cast<float4*>(&sm.d[buf][row][c0]) = there ? make_float4(d[0], d[1], d[2], d[3]) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int v = me; v < 2 * TILE::kStateUnits; v += kGroup) {
          const int n = v % TILE::kStateUnits;
          const bool there = t0 + n / LPC < at.tokens;
          float x[4];
          numbers<T, 4>(v < TILE::kStateUnits ? sm.B[stage][n] : sm.C[stage][n], x);
          (v < TILE::kStateUnits ? sm.B4 : sm.C4)[buf][n / LPC][n % LPC] = there ? make_float4(x[0], x[1], x[2], x[3]) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
      if (k > 0) add_up(k - 1);
      __syncthreads();
    }
    if (chunks) add_up(chunks - 1);
  } else {
    give_registers<48>();
    const int row = me / kVecs, c0 = me % kVecs * kEach, left = tile.left - c0;
    const bool unit = me < TILE::kUnits;
    float dskip[kEach] = {}, dbias[kEach] = {};
    const auto finish = [&](int k) {
      const int stage = k % kStages, t = (chunks - 1 - k) * kChunk + row;
      if (!unit || t >= at.tokens) return;
      float u[kEach], dt[kEach], d[kEach], x[kEach];
      numbers<T, kEach>(sm.u[stage][me], u), numbers<T, kEach>(sm.dy[stage][me], d);
      if constexpr (GATED) {
        float z[kEach];
        numbers<T, kEach>(sm.z[stage][me], z);
#pragma unroll
        for (int q = 0; q < kEach; ++q) {
          const float s = sigmoid(z[q]), zs = z[q] * s;
          x[q] = d[q] * fmaf(sm.skip[c0 + q], u[q], sm.y[k & 1][row][c0 + q]) * fmaf(zs, 1.f - s, s);
          d[q] *= zs;
        }
        put_some<T, kEach>(rows(a.dz) + (int64_t)t * a.dz.token_pitch + c0, x, whole, left);
      }
      numbers<T, kEach>(sm.dt[stage][me], dt);
#pragma unroll
      for (int q = 0; q < kEach; q += 2) {
        F2 s = add2(f2(dt[q], dt[q + 1]), pair_of(&sm.bias[c0 + q]));
        float raw[2], step[2];
        apart(s, raw[0], raw[1]);
        if (a.softplus) s = softplus(s);
        apart(s, step[0], step[1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float gB = sm.gB[k & 1][row][c0 + q + e];
          float ddt = fmaf(gB, u[q + e], sm.eA[k & 1][row][c0 + q + e] * (1.f / kLog2e));
          if (a.softplus) ddt *= sigmoid(raw[e]);
          dskip[q + e] = fmaf(d[q + e], u[q + e], dskip[q + e]), dbias[q + e] += ddt;
          x[q + e] = fmaf(gB, step[e], sm.skip[c0 + q + e] * d[q + e]);
          dt[q + e] = ddt;
        }
      }
      put_some<T, kEach>(rows(a.du) + (int64_t)t * a.du.token_pitch + c0, x, whole, left);
      put_some<T, kEach>(rows(a.ddt) + (int64_t)t * a.ddt.token_pitch + c0, dt, whole, left);
    };
    __syncthreads();
    __syncthreads();
    __syncthreads();
    for (int k = 0; k < chunks; ++k) {
      if (k) finish(k - 1);
      __syncthreads();
    }
    if (chunks) finish(chunks - 1);
    // dD and ddt_bias of the tile: the rows of a chunk in their order (the other roles are past their last barrier)
    float* part = &sm.y[0][0][0];
    static_assert(sizeof(sm.y) >= 2 * kChunk * TILE::kChannels * sizeof(float), "");
    asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
    for (int q = 0; q < kEach; ++q)
      if (unit) part[row * TILE::kChannels + c0 + q] = dskip[q], part[(kChunk + row) * TILE::kChannels + c0 + q] = dbias[q];
    asm volatile("bar.sync 1, 128;" ::: "memory");
    for (int e = me; e < 2 * TILE::kChannels; e += kGroup) {
      const int which = e / TILE::kChannels, c = e % TILE::kChannels;
      float s = 0.f;
      for (int r = 0; r < kChunk; ++r) s += part[(which * kChunk + r) * TILE::kChannels + c];
      if (c < tile.left) out.skips[((int64_t)slot * 2 + which) * a.channels + tile.channel + c] = s;
    }
  }
}

// What the blocks have left is added up by one launch whose blocks are of three kinds, each in a fixed order: dB and dC over the tiles of a
// group (a block takes kSumFours fours of numbers and kSumRanges ranges of tiles at once), then dA, then dD and ddt_bias over the slots.
constexpr int kSumThreads = 256, kSumRanges = 8, kSumFours = kSumThreads / kSumRanges;
template <typename T, int LPC>
__global__ void __launch_bounds__(kSumThreads) k_scan_sums(lasp_scan_args a, Partial part, int tiles, int slots, int64_t token_blocks) {
  using TILE = Tile<LPC>;
  const int me = threadIdx.x;
  int64_t block = blockIdx.x;
  const auto add = [](float4& s, const float4& v) { s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w; };
  if (block < token_blocks * a.groups) {
    __shared__ float4 ranges[kSumRanges][kSumFours];
    constexpr int kFours = kSumsOfToken * LPC / 4;   // of a token
    const int group = (int)(block / token_blocks), in_group = tiles / a.groups, range = me / kSumFours;
    const int64_t all = (int64_t)a.rows * a.tokens * kFours, e = (block - group * token_blocks) * kSumFours + me % kSumFours, token = e / kFours;
    const int at = (int)(e % kFours), n = at / 2 * 4, row = (int)(token / a.tokens), t = (int)(token - (int64_t)row * a.tokens);
    bool inside = e < all;
    if (a.sequences) {
      const Sequences q{a.offsets, a.index_bits, a.sequences, a.tokens};
      inside = inside && t >= q.at(0) && t < q.at(a.sequences);
    }
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (inside) {
      const float4* p = part.tokens + (int64_t)group * in_group * all + e;
      const int each = (in_group + kSumRanges - 1) / kSumRanges, end = min(in_group, (range + 1) * each);
#pragma unroll 8
      for (int k = range * each; k < end; ++k) add(s, p[k * all]);
    }
    ranges[range][me % kSumFours] = s;
    __syncthreads();
    if (range || e >= all) return;
#pragma unroll
    for (int r = 1; r < kSumRanges; ++r) add(s, ranges[r][me]);
    const lasp_tokens& to = at % 2 ? a.dC : a.dB;
    T* out = static_cast<T*>(to.data) + (int64_t)row * to.row_pitch + (int64_t)t * to.token_pitch + (int64_t)group * to.group_pitch + n;
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (n + k < a.states) out[k] = from_f<T>(v[k]);
    return;
  }
  block -= token_blocks * a.groups;
  if (block < tiles) {   // dA: a thread for each lane of a tile
    const TilePlace<TILE> tile((int)block, a.channels, a.groups);
    const int lane = me % 32, i = lane / TILE::kGroups, ch = me / 32 * TILE::kGroups + lane % TILE::kGroups;
    if (!a.dA || me >= kGroup || ch >= tile.left) return;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int q = 0; q < slots; ++q) add(s, part.rates[((int64_t)q * tiles + block) * kGroup + me]);
    store_four(a.dA + (int64_t)(tile.channel + ch) * a.states, 4 * i, a.states, s);
    return;
  }
  const int64_t c = (block - tiles) / 2 * kSumThreads + me;
  const int which = (int)((block - tiles) % 2);
  void* to = which ? a.ddt_bias : a.dD;
  if (c >= a.channels || !to) return;
  float s = 0.f;
  for (int q = 0; q < slots; ++q) s += part.skips[((int64_t)q * 2 + which) * a.channels + c];
  store_param<T>(to, a.param_dtype == LASP_F32, c, s);
}

struct Plan {
  int tiles;
  Cuts cuts;
  size_t tokens, rates, skips, parts;   // floats
};
template <int LPC>
Plan plan_as(const lasp_scan_args& a) {
  using TILE = Tile<LPC>;
  Plan p;
  p.tiles = tiles_of<TILE>(a.channels, a.groups);
  // 90 KB of shared memory for 16-bit types, 115 (fp32, 16 states), 109 (32), 132 and 157 (64 states, 16 bits and fp32)
  const int resident = blocks_of_sm(a.dtype == LASP_F32 ? sizeof(Shared<float, LPC>) : sizeof(Shared<__half, LPC>));
  const Cuts cuts = cuts_of<TILE>(a, p.tiles, true, resident, nullptr);
  p.tokens = (size_t)p.tiles * a.rows * a.tokens * 8 * LPC;
  p.rates = (size_t)cuts.slots * p.tiles * kGroup * 4, p.skips = ((size_t)cuts.slots * 2 * a.channels + 3) / 4 * 4, p.parts = (size_t)floats_of<TILE>(cuts, p.tiles);
  p.cuts = cuts_of<TILE>(a, p.tiles, true, resident, static_cast<float*>(a.ws) + p.tokens + p.rates + p.skips);
  return p;
}

template <typename T, int LPC, bool GATED>
cudaError_t launch(const lasp_scan_args& a, cudaStream_t st) {
  using TILE = Tile<LPC>;
  constexpr auto kernel = k_scan_backward<T, LPC, GATED>;
  constexpr size_t smem = sizeof(Shared<T, LPC>);
  const cudaError_t err = ready<kernel>(smem);
  if (err != cudaSuccess) return err;
  const Plan p = plan_as<LPC>(a);
  float* ws = static_cast<float*>(a.ws);
  const Partial out{reinterpret_cast<float4*>(ws), reinterpret_cast<float4*>(ws + p.tokens), ws + p.tokens + p.rates};
  bool wide = (a.channels / a.groups) % TILE::kEach == 0 && reads_by<T>(a.B, 4) && reads_by<T>(a.C, 4);
  for (const lasp_tokens* t : {&a.u, &a.dt, &a.z, &a.dy, &a.du, &a.ddt, &a.dz}) wide = wide && reads_by<T>(*t, TILE::kEach);
  if (p.cuts.length != kUncut)
    if (const cudaError_t e = scan_parts<T, LPC>(a, p.cuts, p.tiles, true, st); e != cudaSuccess) return e;
  kernel<<<(unsigned)(p.tiles * (p.cuts.slots + (a.sequences ? 1 : 0))), kThreads, smem, st>>>(a, p.tiles, out, p.cuts, wide);
  const int64_t token_blocks = ((int64_t)a.rows * a.tokens * (kSumsOfToken * LPC / 4) + kSumFours - 1) / kSumFours;
  const int64_t blocks = token_blocks * a.groups + p.tiles + 2 * (((int64_t)a.channels + kSumThreads - 1) / kSumThreads);
  k_scan_sums<T, LPC><<<(unsigned)blocks, kSumThreads, 0, st>>>(a, out, p.tiles, (int)p.cuts.slots, token_blocks);
  return cudaGetLastError();
}

template <typename T>
cudaError_t backward_as(const lasp_scan_args& a, cudaStream_t st) {
  const bool gated = a.z.data != nullptr;
  switch (padded_states(a.states)) {
    case 16: return gated ? launch<T, 4, true>(a, st) : launch<T, 4, false>(a, st);
    case 32: return gated ? launch<T, 8, true>(a, st) : launch<T, 8, false>(a, st);
    default: return gated ? launch<T, 16, true>(a, st) : launch<T, 16, false>(a, st);
  }
}
Plan plan_of(const lasp_scan_args& a) {
  const int padded = padded_states(a.states);
  return padded == 16 ? plan_as<4>(a) : padded == 32 ? plan_as<8>(a) : plan_as<16>(a);
}

}  // namespace

cudaError_t scan_backward(const lasp_scan_args& a, cudaStream_t st) {
  return a.dtype == LASP_F32 ? backward_as<float>(a, st) : a.dtype == LASP_BF16 ? backward_as<__nv_bfloat16>(a, st) : backward_as<__half>(a, st);
}
// The forward pass keeps four states of each lane of each tile ahead of each chunk.
size_t scan_kept(const lasp_scan_args& a) { return (size_t)chunks_of(a) * plan_of(a).tiles * kGroup * sizeof(float4); }
size_t scan_workspace(const lasp_scan_args& a) {
  const Plan p = plan_of(a);
  return (p.tokens + p.rates + p.skips + p.parts) * sizeof(float);
}

}  // namespace lasp
