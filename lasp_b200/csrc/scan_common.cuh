// What the kernels of the selective scan have in common.
//
//   h_t[c][n] = exp(dt_t[c] A[c][n]) h_(t-1)[c][n] + dt_t[c] u_t[c] B_t[n],   y_t[c] = sum_n C_t[n] h_t[c][n] + D[c] u_t[c]
//
// A block owns a tile of channels of one sequence and walks along its tokens, kChunk at a time.  Four of its warps hold the states: a
// lane 4 neighbouring ones of one channel, LPC lanes those of a channel (lanes g, g + 32 / LPC, ...: what belongs to a state is then
// the same for neighbouring lanes, which shared memory serves at once), a warp 32 / LPC channels.  They do nothing but the recurrence and the sums over it:
// a warp that also brought, prepared and finished its tokens spent half its time on the latencies of those, which is what the other eight
// warps are for.  What bounds it then is the pipe of shared memory (2 x 2048 x 4096, 16 states, forward: 45 of the 58 clocks that a tile takes
// for a token where an SM has two blocks) and the chain of the warps that hold the states (68 clocks where it has one); the exponentials, one for every state,
// channel and token at 16 per clock and SM, take 32.
#pragma once
#include <algorithm>

#include "recurrent.cuh"

namespace lasp {

constexpr int kChunk = 16, kGroup = 128, kThreads = 3 * kGroup;   // warps come in groups of four
template <int LPC>
struct Tile {
  static constexpr int kStates = 4 * LPC;
  static constexpr int kGroups = 32 / LPC;            // channels of a warp
  static constexpr int kChannels = 4 * kGroups;
  // units in which a chunk's tokens are brought and prepared: kEach channels of a token, 4 numbers of B or of C
  static constexpr int kEach = 4, kVecs = kChannels / kEach, kUnits = kChunk * kVecs;
  static constexpr int kRow = kChannels + (LPC == 4 ? 8 : 4);   // of sums that the warps with the states leave: lanes write several rows at once
  static constexpr int kStateUnits = kChunk * LPC;
};
// Registers move from the warps that prepare and finish to those that hold the states.  A block is launched with 3 x 128 x kRegisters
// (two blocks an SM, where shared memory allows it); the shares add up to no more.
constexpr int kRegisters = 80;
template <int N>
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
// Shared memory and, because a warp that takes more registers than there are waits for good, the registers that a kernel is launched with:
// looked at until both are as they should be, once for each kernel and device.
template <auto kernel>
cudaError_t ready(size_t smem) {
  static PerDevice looked;
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess)
    err = looked.once(dev, [] {
      cudaFuncAttributes at;
      const cudaError_t e = cudaFuncGetAttributes(&at, (const void*)kernel);
      return e != cudaSuccess ? e : at.numRegs >= kRegisters ? cudaSuccess : cudaErrorInvalidConfiguration;
    });
  if (err == cudaSuccess) return opt_in_smem<kernel>(smem);
  g_failed_step = "cudaFuncGetAttributes(registers of a scan kernel)";
  return err;
}

// `BYTES` (4, 8, 16 or 32) from global to shared memory without a register in between.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
  if constexpr (BYTES > 16) {
    copy_async<16>(to, from);
    copy_async<BYTES - 16>(static_cast<char*>(to) + 16, static_cast<const char*>(from) + 16);
  } else if constexpr (BYTES == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(from) : "memory");
  } else {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(from), "n"(BYTES) : "memory");
  }
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void await_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
// N neighbouring numbers of a row to shared memory: by one asynchronous copy where that may be (`whole`), else those below `left`.
template <typename T, int N>
__device__ __forceinline__ void bring(Vec<T, N>* to, const T* from, bool whole, int left) {
  if (whole) {
    copy_async<N * (int)sizeof(T)>(to, from);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) to->v[k] = k < left ? from[k] : from_f<T>(0.f);
  }
}
template <typename T, int N>
__device__ __forceinline__ void numbers(const Vec<T, N>& from, float (&out)[N]) {
  const Vec<T, N> v = from;
#pragma unroll
  for (int k = 0; k < N; k += 2) apart(pair_from(&v.v[k]), out[k], out[k + 1]);
}

// 4 states
struct S4 {
  F2 a, b;
};
__device__ __forceinline__ S4 splat(float x) { return {f2(x, x), f2(x, x)}; }
__device__ __forceinline__ S4 mul(S4 p, S4 q) { return {mul2(p.a, q.a), mul2(p.b, q.b)}; }
__device__ __forceinline__ S4 mul(S4 p, F2 f) { return {mul2(p.a, f), mul2(p.b, f)}; }   // (f: the same number twice)
__device__ __forceinline__ S4 fma(S4 p, S4 q, S4 r) { return {fma2(p.a, q.a, r.a), fma2(p.b, q.b, r.b)}; }
__device__ __forceinline__ S4 fma(S4 p, F2 f, S4 r) { return {fma2(p.a, f, r.a), fma2(p.b, f, r.b)}; }
__device__ __forceinline__ S4 s4(float4 v) { return {f2(v.x, v.y), f2(v.z, v.w)}; }
__device__ __forceinline__ float4 f4(S4 s) {
  float4 v;
  apart(s.a, v.x, v.y), apart(s.b, v.z, v.w);
  return v;
}
__device__ __forceinline__ S4 load4(const void* p) {   // 16 aligned bytes
  const ulonglong2 v = *static_cast<const ulonglong2*>(p);
  return {{v.x}, {v.y}};
}
__device__ __forceinline__ F2 pair_of(const void* p) { return {*static_cast<const unsigned long long*>(p)}; }   // 8 aligned bytes
__device__ __forceinline__ void store4(void* p, S4 s) { *static_cast<ulonglong2*>(p) = make_ulonglong2(s.a.v, s.b.v); }
__device__ __forceinline__ F2 exp2(F2 p) {
  float x, y;
  apart(p, x, y);
  return f2(ex2(x), ex2(y));
}
// The decays of a step.  The hardware's exponential falls short: 2e-8 of a decay of 0.5 and more, on average, which a state of a hundred tokens'
// memory adds up.  With 2.5e-8 more of an exponent y of such rows of 1000 tokens is off by 4.6e-7 of its norm instead of 1.8e-6, dA by 9.9e-7
// instead of 4.8e-6; a step of zero still gives 1.
__device__ __forceinline__ S4 decay_of(S4 rate, float step) {
  const F2 s = f2(step, step), more = f2(2.5e-8f, 2.5e-8f);
  return {exp2(fma2(rate.a, s, more)), exp2(fma2(rate.b, s, more))};
}
__device__ __forceinline__ float dot(S4 p, S4 q) {
  float x, y;
  apart(fma2(p.b, q.b, mul2(p.a, q.a)), x, y);
  return x + y;
}

// v[k] summed over the LANES lanes that differ in the bits from STEP to STEP * LANES / 2.  COUNT = LANES: the lane of bits q * STEP is left
// with the sum of index q in v[0].  More: it is left with COUNT / LANES neighbouring ones; fewer: LANES / COUNT neighbouring lanes have
// the same one.  Half of the values change lanes at each step, so that LANES - 1 exchanges do for LANES sums.
template <int COUNT, int LANES, int STEP>
__device__ __forceinline__ void sum_over(float (&v)[COUNT], int lane) {
  if constexpr (LANES > 1) {
    constexpr int m = LANES / 2 * STEP;
    if constexpr (COUNT == 1) {
      v[0] += __shfl_xor_sync(~0u, v[0], m);
      sum_over<1, LANES / 2, STEP>(v, lane);
    } else {
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
}

// log(1 + e^x) = max(x, 0) + log(1 + e), e = e^-|x| in (0, 1].  Small steps need it exact relative to e, not to 1: log(1 + e) =
// 2 atanh(s) with s = e / (2 + e) <= 1/3, whose series s + s^3/3 + s^5/5 ... is cut where it falls below 2^-26.
__device__ __forceinline__ F2 softplus(F2 p) {
  float x, y;
  apart(p, x, y);
  const float ex = ex2(-fabsf(x) * kLog2e), ey = ex2(-fabsf(y) * kLog2e);
  const F2 s = f2(ex * reciprocal(2.f + ex), ey * reciprocal(2.f + ey)), q = mul2(s, s);
  const auto k = [](float c) { return f2(c, c); };
  F2 t = fma2(q, k(1.f / 13), k(1.f / 11));
  t = fma2(q, t, k(1.f / 9)), t = fma2(q, t, k(1.f / 7)), t = fma2(q, t, k(1.f / 5)), t = fma2(q, t, k(1.f / 3));
  t = fma2(mul2(s, q), t, s);
  return fma2(t, k(2.f), f2(fmaxf(x, 0.f), fmaxf(y, 0.f)));
}
__device__ __forceinline__ float softplus(float x) {
  float r, again;
  apart(softplus(f2(x, x)), r, again);
  return r;
}

// Of a row of A or of a state: 4 numbers from the n-th on, zeros behind the last one.
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
  const auto one = [](float x) { return x *= kLog2e, isinf(x) ? copysignf(3.402823466e38f, x) : x; };
  return {f2(one(v.x), one(v.y)), f2(one(v.z), one(v.w))};
}

// What a parameter of kEach channels is, zeros where there are none.
template <typename T, int N>
__device__ __forceinline__ void params_of(const void* p, bool f32, int channel, int left, float (&out)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) out[k] = p && k < left ? param<T>(p, f32, channel + k) : 0.f;
}
// Steps and inputs of a unit's four channels, two 16-byte words: every other four threads write the second word first, so that eight threads
// together reach every bank.
__device__ __forceinline__ void put_steps(float2* to, const float (&step)[4], const float (&in)[4], int thread, bool there) {
  const bool second = thread & 4;
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f), x = there ? make_float4(step[0], in[0], step[1], in[1]) : zero;
  const float4 y = there ? make_float4(step[2], in[2], step[3], in[3]) : zero;
  float4* p = reinterpret_cast<float4*>(to);
  p[second] = second ? y : x;
  p[!second] = second ? x : y;
}

// Which channels a block's tile is: tiles do not reach across groups, the last of a group may be cut short.
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

// Few channels and sequences leave SMs idle.  Their tokens are then cut into segments of `length`, one for a block; where a segment starts
// (forward: the state, backward: the gradient that comes in from behind) is put together from what the parts of the others, kParts to a
// segment, do to a state of zero (`ends`) and from the sums of their steps, whose exponentials are the parts' decays: a first pass over
// the tokens (scan_parts.cu) finds those.  It takes the exponentials once more, so segments come only where they are that many.
constexpr int kParts = 4, kUncut = 0x7ffffff0;
// Tokens of a segment; segments for which the first pass pays: two backward where an SM has two blocks, else three.  us of whole rows and of rows in
// segments, 16384 tokens of 4096 channels and 16 states (128 blocks): forward 600 and 793 (two); backward 2314 and 1978 (two) in bf16, in fp32,
// where an SM has one block, 2283 and 2416 (two: as long as whole rows, and the first pass).  In three (4096 tokens in 80 blocks): forward 160 and 142,
// backward, one block an SM, 553 and 414 (fp32, 16 states), 574 and 468 (bf16, 64).
constexpr int kLeast = 128, kLeastSegments = 3, kLeastOfTwoBlocks = 2;
// Blocks of an SM: it has 228 KB of shared memory, of which a block takes 1 KB more than it asks for.
constexpr int blocks_of_sm(size_t smem) { return 2 * (smem + 1024) <= 228 * 1024 ? 2 : 1; }
struct Cuts {
  int length, part;       // tokens of a segment, of a part: multiples of kChunk, or kUncut
  int64_t slots, parts;   // how many there may be
  float4* ends;           // [part][tile][kGroup]: four states of each lane
  float* steps;           // [part][tile][channel of the tile]
};

// Slots: a row of n tokens has ceil(n / length) of them, one at least; packed sequence i those from offsets[i] / length + i on, which
// leaves room for each.  Chunks, as the kept states are counted, are slots of kChunk.
__device__ __forceinline__ int64_t slot_of(const lasp_scan_args& a, int seq, int begin, int length) {
  return a.sequences ? (int64_t)(begin / length) + seq : (int64_t)seq * (a.tokens > 0 ? (a.tokens - 1) / length + 1 : 1);
}
inline int64_t slots_of(const lasp_scan_args& a, int length) {
  return a.sequences ? (int64_t)a.tokens / length + a.sequences : (int64_t)a.rows * (a.tokens > 0 ? (a.tokens - 1) / length + 1 : 1);
}
inline int64_t chunks_of(const lasp_scan_args& a) { return slots_of(a, kChunk); }

// What a slot holds: segment `index` of the `count` of a sequence (none: index = count), the row, the first and the number of its tokens and
// of the sequence's, and the number of its first chunk.
struct Stretch {
  int seq, index, count, row, begin, tokens, sequence_begin, sequence_tokens;
  int64_t chunk;
  __device__ __forceinline__ Stretch(const lasp_scan_args& a, int slot, int length) {
    int& all = sequence_tokens;
    all = a.tokens, sequence_begin = 0;
    if (!a.sequences) {
      count = a.tokens > 0 ? (a.tokens - 1) / length + 1 : 1;
      seq = row = slot / count;
    } else {
      const Sequences s{a.offsets, a.index_bits, a.sequences, a.tokens};
      int lo = 0, hi = a.sequences;   // (the slots of sequences [0, lo) begin at or before this one)
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s.at(mid) / length + mid <= slot)
          lo = mid + 1;
        else
          hi = mid;
      }
      seq = max(lo - 1, 0), row = 0;
      int end;
      s.bounds(seq, &sequence_begin, &end);
      all = end - sequence_begin;
      count = all > 0 ? (all - 1) / length + 1 : 1;
    }
    const int i = a.sequences ? slot - sequence_begin / length - seq : slot - seq * count;
    index = i < 0 || i >= count ? count : i;
    const int first = index < count ? index * length : 0;
    begin = sequence_begin + first, tokens = index < count ? min(length, all - first) : 0;
    chunk = slot_of(a, seq, sequence_begin, kChunk) + first / kChunk;
  }
};

// Four of a lane's states (`me` of the tile's lanes, channel ch) taken from one end of parts [lo, hi) of a sequence to the other: forwards, or back.
template <class TILE>
__device__ __forceinline__ S4 carry(const lasp_scan_args& a, const Cuts& cuts, const Stretch& at, int lo, int hi, bool back, S4 from, S4 A, int tiles, int tile, int me, int ch) {
  const int64_t first = slot_of(a, at.seq, at.sequence_begin, cuts.part);
#pragma unroll 4
  for (int p = lo; p < hi; ++p) {
    const int64_t k = (first + (back ? lo + hi - 1 - p : p)) * tiles + tile;
    const float half = 0.5f * cuts.steps[k * TILE::kChannels + ch];
    float d[4];   // the decay's root, taken twice: what is zero stays so where the decay itself is beyond fp32
    const float4 x = f4(decay_of(A, half));
    d[0] = x.x, d[1] = x.y, d[2] = x.z, d[3] = x.w;
#pragma unroll
    for (int n = 0; n < 4; ++n) d[n] = d[n] > 3.402823466e38f ? 3.402823466e38f : d[n];
    const S4 root = s4(make_float4(d[0], d[1], d[2], d[3]));
    from = fma(root, mul(root, from), s4(cuts.ends[k * kGroup + me]));
  }
  return from;
}

// n neighbouring numbers of a tensor of tokens can be read and written by accesses of all their bytes, or of 16.
template <typename T>
bool reads_by(const lasp_tokens& t, int n) { return by(t, std::min<size_t>(16, n * sizeof(T)), sizeof(T)); }
inline int padded_states(int states) { return states <= 16 ? 16 : states <= 32 ? 32 : 64; }

template <typename T, int N>
__device__ __forceinline__ void put_some(T* p, const float (&x)[N], bool whole, int left) {
  if (whole) {
    store_vec<T, N>(p, x);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k < left) p[k] = from_f<T>(x[k]);
  }
}

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

// Floats that the parts' ends and steps take.
template <class TILE>
int64_t floats_of(const Cuts& c, int tiles) { return c.length == kUncut ? 0 : c.parts * tiles * (4 * kGroup + TILE::kChannels); }
// resident: blocks of an SM
template <class TILE>
Cuts cuts_of(const lasp_scan_args& a, int tiles, bool backward, int resident, float* ws) {
  Cuts c{kUncut, kUncut, 0, 0, nullptr, nullptr};
  // Two blocks for each SM, no more (sequences of a packed row: as many tokens for each as if there were one), also where it has one at a time:
  // 4096 tokens in 64 blocks, fp32, take 330 us in four segments and 345 in two.  Back three segments, too, where whole sequences leave some SMs
  // twice as many blocks as the others: those are then 2/3 as long.  us without and with, 1000 tokens: 150 blocks 216 and 168, 197 blocks 220 and 192
  // (bf16, 16 states; 32 states the same), 262 and 204, 268 and 241 (fp32, 16 states); 8000 tokens: 1609 and 1233, 1613 and 1299; 1953 and 1470,
  // 1988 and 1704; 64 states 2200 and 1668 (160 blocks), 2235 and 1834 (196).
  const int64_t unit = kParts * kChunk, blocks = (int64_t)tiles * a.rows, sms = std::max(1, sm_count());
  const int64_t segments = backward && blocks > sms && 3 * blocks <= 4 * sms ? 3 : 2 * sms / blocks;
  if (segments >= 2) {
    const int64_t length = std::max<int64_t>(kLeast, ((a.tokens + segments - 1) / segments + unit - 1) / unit * unit);
    const int least = backward && resident == 2 ? kLeastOfTwoBlocks : kLeastSegments;
    if (a.tokens > (least - 1) * length) c.length = (int)length, c.part = c.length / kParts;
  }
  c.slots = slots_of(a, c.length), c.parts = slots_of(a, c.part);
  c.ends = reinterpret_cast<float4*>(ws), c.steps = ws + c.parts * tiles * 4 * kGroup;
  return c;
}
// The first pass: ends and steps of the parts that a segment needs.
template <typename T, int LPC>
cudaError_t scan_parts(const lasp_scan_args& a, const Cuts& cuts, int tiles, bool backward, cudaStream_t st);

}  // namespace lasp
