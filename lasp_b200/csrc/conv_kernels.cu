// Short causal convolution, channel by channel, over prompts and training batches, and for single tokens.
//
//   p_t = bias + sum_j w_j x_(t-W+1+j),  y_t = p_t or silu(p_t)
//   dp_t = dy_t silu'(p_t),  dx_t = sum_k w_(W-1-k) dp_(t+k),  dw_j = sum_t dp_t x_(t-W+1+j)
//
// A thread owns V neighbouring channels and a run of tokens: the last W - 1 inputs slide through its registers, so that every input is
// read once but for the W - 1 ahead of a run.  Nothing is staged.  The latency of loads bounds it, nothing is near its limit: 8 x 2048 x 4096
// bf16 takes 62 us forward (41 at the copy rate; DRAM 45 % busy, issue slots and the pipe of exponentials and conversions 53 %, 34 of 64 warps an SM)
// and 128 backward (62; 38, 53 and 26 %, 29 warps), fp16 62 and 148, fp32 with as many bytes (4 x 2048 x 4096) 55 and 92.  Registers for five and
// four blocks an SM are paid for with spills, in bytes stored and loaded by a thread: forward 32 and 64 (16 bits), 108 and 260 (fp32); backward
// 52 and 80 (bf16), 56 and 84 (fp16), 112 and 260 (fp32).
#include <algorithm>
#include <type_traits>

#include "recurrent.cuh"

namespace lasp {
namespace {

constexpr int kVecs = 32, kRuns = 8;   // a block: 32 vectors of channels times 8 runs of tokens
constexpr int kBatch = 8, kBatchBack = 4;   // tokens whose loads are under way together

template <typename T, int V, int W>
struct Taps {
  Channels<V> w[W], bias;
  template <class ARGS>
  __device__ __forceinline__ void load(const ARGS& a, int c) {
    const bool f32 = a.param_dtype == LASP_F32;
    float x[W + 1][2 * Channels<V>::kPairs] = {};
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (f32 && W == 4 && reinterpret_cast<uintptr_t>(a.weight) % 16 == 0) {
        const float4 w4 = reinterpret_cast<const float4*>(a.weight)[c + i];
        x[0][i] = w4.x, x[1][i] = w4.y, x[2 % W][i] = w4.z, x[3 % W][i] = w4.w;
      } else {
#pragma unroll
        for (int j = 0; j < W; ++j) x[j][i] = param<T>(a.weight, f32, (int64_t)(c + i) * W + j);
      }
      if (a.bias) x[W][i] = param<T>(a.bias, f32, c + i);
    }
#pragma unroll
    for (int k = 0; k < Channels<V>::kPairs; ++k) {
#pragma unroll
      for (int j = 0; j < W; ++j) w[j].p[k] = f2(x[j][2 * k], x[j][2 * k + 1]);
      bias.p[k] = f2(x[W][2 * k], x[W][2 * k + 1]);
    }
  }
  // of pair k: bias + the sum over the taps
  __device__ __forceinline__ F2 sum(const Channels<V> (&past)[W - 1], F2 now, int k) const {
    F2 p = fma2(w[W - 1].p[k], now, bias.p[k]);
#pragma unroll
    for (int m = 0; m < W - 1; ++m) p = fma2(w[m].p[k], past[m].p[k], p);
    return p;
  }
};
template <int V, int W>
__device__ __forceinline__ void move_on(Channels<V> (&past)[W], const Channels<V>& now) {
#pragma unroll
  for (int m = 0; m + 1 < W; ++m) past[m] = past[m + 1];
  past[W - 1] = now;
}

// x at token p of a sequence that begins at `begin`; what lies before is its state, or zero
template <typename T, int V, int W>
__device__ __forceinline__ Channels<V> input_at(const T* x, int64_t pitch, const T* state, int64_t c_total, int begin, int p) {
  Channels<V> out;
  if (p >= begin)
    out.load(x + (int64_t)p * pitch);
  else if (state && p - begin + W - 1 >= 0)
    out.load(state + (int64_t)(p - begin + W - 1) * c_total);
  else
    out.clear();
  return out;
}

// The sequence that a thread is in.  `state` is the address of its channels in the state of that sequence.
template <typename T, int W>
struct Place {
  Sequences seqs;
  int seq, begin, end;
  __device__ __forceinline__ void start(const lasp_conv_args& a, int row, int t) {
    seqs = {a.offsets, a.index_bits, a.sequences, a.tokens};
    if (!a.sequences) {
      seq = row, begin = 0, end = a.tokens;
      return;
    }
    seq = seqs.find(t);
    if (seq >= 0)
      seqs.bounds(seq, &begin, &end);
    else
      begin = end = 0;
  }
  __device__ __forceinline__ bool inside(int t) const { return t >= begin && t < end; }
  // t has left the sequence: to the one that holds it, if there is one
  __device__ __forceinline__ void advance(int t) {
    while (seq + 1 < seqs.count && seqs.at(seq + 1) <= t) ++seq, seqs.bounds(seq, &begin, &end);
  }
  __device__ __forceinline__ const T* state(const void* base, int64_t c_total, int c) const {
    return base && seq >= 0 ? static_cast<const T*>(base) + (int64_t)seq * (W - 1) * c_total + c : nullptr;
  }
};

// state_out of one sequence
template <typename T, int V, int W>
__device__ void write_state(const lasp_conv_args& a, int row, int seq, int c) {
  int begin = 0, end = a.tokens;
  if (a.sequences) Sequences{a.offsets, a.index_bits, a.sequences, a.tokens}.bounds(seq, &begin, &end);
  const T* x = static_cast<const T*>(a.x.data) + (int64_t)row * a.x.row_pitch + c;
  const T* from = a.state_in ? static_cast<const T*>(a.state_in) + (int64_t)seq * (W - 1) * a.channels + c : nullptr;
  T* to = static_cast<T*>(a.state_out) + (int64_t)seq * (W - 1) * a.channels + c;
#pragma unroll
  for (int m = 0; m < W - 1; ++m)
    input_at<T, V, W>(x, a.x.token_pitch, from, a.channels, begin, end - (W - 1) + m).store(to + (int64_t)m * a.channels);
}

template <typename T, int V, int W>
__global__ void __launch_bounds__(kVecs* kRuns, 5) k_conv_forward(lasp_conv_args a, int run, int blocks_of_runs) {
  constexpr int kPairs = Channels<V>::kPairs;
  const int c = (blockIdx.x * kVecs + threadIdx.x) * V, row = blockIdx.z;
  if (c >= a.channels) return;
  if ((int)blockIdx.y >= blocks_of_runs) {   // the states after the last tokens
    const int seq = a.sequences ? ((int)blockIdx.y - blocks_of_runs) * kRuns + threadIdx.y : row;
    if (a.sequences ? seq < a.sequences : threadIdx.y == 0) write_state<T, V, W>(a, row, seq, c);
    return;
  }
  const int64_t first = ((int64_t)blockIdx.y * kRuns + threadIdx.y) * run;
  if (first >= a.tokens) return;
  const int t0 = (int)first, t1 = first + run < a.tokens ? (int)first + run : a.tokens;
  const T* x = static_cast<const T*>(a.x.data) + (int64_t)row * a.x.row_pitch + c;
  T* y = static_cast<T*>(a.y.data) + (int64_t)row * a.y.row_pitch + c;
  Taps<T, V, W> taps;
  taps.load(a, c);
  Place<T, W> at;
  at.start(a, row, t0);
  Channels<V> past[W - 1];   // past[m]: x_(t-W+1+m)
  const auto look_back = [&](int t) {
#pragma unroll
    for (int m = 0; m < W - 1; ++m)
      past[m] = input_at<T, V, W>(x, a.x.token_pitch, at.state(a.state_in, a.channels, c), a.channels, at.begin, t - (W - 1) + m);
  };
  look_back(t0);
  // kBatch tokens from t on; `whole`: all of them in this run and, where sequences are packed, in one sequence
  const auto batch = [&](int t, auto whole) {
    constexpr bool kWhole = decltype(whole)::value;
    Vec<T, V> in[kBatch];
    const T* from = x + (int64_t)t * a.x.token_pitch;
    T* to = y + (int64_t)t * a.y.token_pitch;
#pragma unroll
    for (int j = 0; j < kBatch; ++j, from += a.x.token_pitch)
      if (kWhole || t + j < t1) in[j] = *reinterpret_cast<const Vec<T, V>*>(from);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (!kWhole && t + j >= t1) break;
      bool inside = true;
      if (!kWhole && a.sequences) {
        if (t + j >= at.end) {
          at.advance(t + j);
          if (t + j >= at.begin) look_back(t + j);
        }
        inside = at.inside(t + j);
      }
      Channels<V> now, out;
      now.set(in[j]);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const F2 p = taps.sum(past, now.p[k], k);
        out.p[k] = a.activation == LASP_ACT_SILU ? silu(p) : p;
      }
      if (!inside) out.clear();
      move_on(past, now);
      out.store(to);
      to += a.y.token_pitch;
    }
  };
  for (int t = t0; t < t1; t += kBatch) {
    if (t + kBatch <= t1 && (!a.sequences || (t >= at.begin && t + kBatch <= at.end)))
      batch(t, std::true_type());
    else
      batch(t, std::false_type());
  }
}

// dstate_in of one sequence: what its first tokens, and its state_out where it is shorter than the taps, pass on to what lies
// before it
template <typename T, int V, int W>
__device__ void write_dstate(const lasp_conv_args& a, int row, int seq, int c) {
  int begin = 0, end = a.tokens;
  if (a.sequences) Sequences{a.offsets, a.index_bits, a.sequences, a.tokens}.bounds(seq, &begin, &end);
  const T* x = static_cast<const T*>(a.x.data) + (int64_t)row * a.x.row_pitch + c;
  const T* dy = static_cast<const T*>(a.dy.data) + (int64_t)row * a.dy.row_pitch + c;
  const int64_t at = (int64_t)seq * (W - 1) * a.channels + c;
  const T* from = a.state_in ? static_cast<const T*>(a.state_in) + at : nullptr;
  constexpr int kPairs = Channels<V>::kPairs;
  Taps<T, V, W> taps;
  taps.load(a, c);
  Channels<V> sum[W - 1];
#pragma unroll
  for (int m = 0; m < W - 1; ++m) {
    const int kept = begin - end + m;   // its place in state_out, if it is there still
    sum[m].clear();
    if (a.dstate_out && kept >= 0) sum[m].load(static_cast<const T*>(a.dstate_out) + at + (int64_t)kept * a.channels);
  }
#pragma unroll
  for (int r = 0; r < W - 1; ++r) {   // token begin + r reaches back to state entries r, r + 1, ...
    if (begin + r >= end) break;
    Channels<V> d, past[W - 1];
    d.load(dy + (int64_t)(begin + r) * a.dy.token_pitch);
    if (a.activation == LASP_ACT_SILU) {
#pragma unroll
      for (int m = 0; m < W - 1; ++m) past[m] = input_at<T, V, W>(x, a.x.token_pitch, from, a.channels, begin, begin + r - (W - 1) + m);
      const Channels<V> now = input_at<T, V, W>(x, a.x.token_pitch, from, a.channels, begin, begin + r);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) d.p[k] = mul2(d.p[k], d_silu(taps.sum(past, now.p[k], k)));
    }
#pragma unroll
    for (int m = r; m < W - 1; ++m)
#pragma unroll
      for (int k = 0; k < kPairs; ++k) sum[m].p[k] = fma2(taps.w[m - r].p[k], d.p[k], sum[m].p[k]);
  }
#pragma unroll
  for (int m = 0; m < W - 1; ++m) sum[m].store(static_cast<T*>(a.dstate_in) + at + (int64_t)m * a.channels);
}

// partial: for each row and block of runs, W + 1 rows of `channels` sums (the taps' and the bias')
template <typename T, int V, int W>
__global__ void __launch_bounds__(kVecs* kRuns, 4) k_conv_backward(lasp_conv_args a, int run, int blocks_of_runs, float* partial) {
  __shared__ __align__(16) float part[kRuns][kVecs * V];
  const int c = (blockIdx.x * kVecs + threadIdx.x) * V, row = blockIdx.z;
  const bool mine = c < a.channels;
  if ((int)blockIdx.y >= blocks_of_runs) {
    const int seq = a.sequences ? ((int)blockIdx.y - blocks_of_runs) * kRuns + threadIdx.y : row;
    if (mine && (a.sequences ? seq < a.sequences : threadIdx.y == 0)) write_dstate<T, V, W>(a, row, seq, c);
    return;
  }
  constexpr int kPairs = Channels<V>::kPairs;
  Channels<V> dw[W + 1];
#pragma unroll
  for (int k = 0; k <= W; ++k) dw[k].clear();
  const int64_t first = ((int64_t)blockIdx.y * kRuns + threadIdx.y) * run;
  if (mine && first < a.tokens) {
    const int t0 = (int)first, t1 = first + run < a.tokens ? (int)first + run : a.tokens;
    const T* x = static_cast<const T*>(a.x.data) + (int64_t)row * a.x.row_pitch + c;
    const T* dy = static_cast<const T*>(a.dy.data) + (int64_t)row * a.dy.row_pitch + c;
    T* dx = static_cast<T*>(a.dx.data) + (int64_t)row * a.dx.row_pitch + c;
    Taps<T, V, W> taps;
    taps.load(a, c);
    // Token s completes dx_(s-W+1): a run stores those from its own first token's on, to which the W - 1 tokens ahead of it contribute; the
    // row's last run completes the row.
    const int ahead = t0 < W - 1 ? 0 : t0 - (W - 1);
    Place<T, W> at;
    at.start(a, row, ahead);
    Channels<V> past[W - 1], sum[W - 1];   // sum[m]: dx_(t-W+1+m) so far
    const auto look_back = [&](int t) {
#pragma unroll
      for (int m = 0; m < W - 1; ++m)
        past[m] = input_at<T, V, W>(x, a.x.token_pitch, at.state(a.state_in, a.channels, c), a.channels, at.begin, t - (W - 1) + m);
    };
    look_back(ahead);
#pragma unroll
    for (int m = 0; m < W - 1; ++m) sum[m].clear();
    // Tokens t to `stop`, kBatchBack at most.  `whole`: so many, in one sequence, W - 1 tokens or more behind its beginning, in this run
    // and before what state_out holds.
    const auto batch = [&](int t, int stop, auto whole) {
      constexpr bool kWhole = decltype(whole)::value;
      Vec<T, V> in[kBatchBack], din[kBatchBack];
      const T *from = x + (int64_t)t * a.x.token_pitch, *dfrom = dy + (int64_t)t * a.dy.token_pitch;
      T* to = dx + (int64_t)(t - (W - 1)) * a.dx.token_pitch;
#pragma unroll
      for (int j = 0; j < kBatchBack; ++j, from += a.x.token_pitch, dfrom += a.dy.token_pitch)
        if (kWhole || (t + j < stop && t + j < a.tokens)) {
          in[j] = *reinterpret_cast<const Vec<T, V>*>(from);
          din[j] = *reinterpret_cast<const Vec<T, V>*>(dfrom);
        }
#pragma unroll
      for (int j = 0; j < kBatchBack; ++j) {
        const int s = t + j;
        if (!kWhole && s >= stop) break;
        bool inside = kWhole || s < a.tokens;
        if (!kWhole && a.sequences && inside) {
          if (s >= at.end) {
            at.advance(s);
            if (s >= at.begin) look_back(s);
          }
          inside = at.inside(s);
        }
        const int reach = kWhole ? W : inside ? s - at.begin : -1;   // how far back in its sequence this token's gradient goes
        Channels<V> now, d, out;
        now.set(in[j]), d.set(din[j]);
        if (!inside) now.clear(), d.clear();
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
          if (inside && a.activation == LASP_ACT_SILU) d.p[k] = mul2(d.p[k], d_silu(taps.sum(past, now.p[k], k)));
          if (kWhole || (s >= t0 && inside)) {
#pragma unroll
            for (int m = 0; m < W - 1; ++m) dw[m].p[k] = fma2(d.p[k], past[m].p[k], dw[m].p[k]);
            dw[W - 1].p[k] = fma2(d.p[k], now.p[k], dw[W - 1].p[k]);
            dw[W].p[k] = add2(dw[W].p[k], d.p[k]);
          }
          F2 full[W];
#pragma unroll
          for (int m = 0; m < W - 1; ++m) full[m] = reach >= W - 1 - m ? fma2(taps.w[m].p[k], d.p[k], sum[m].p[k]) : sum[m].p[k];
          full[W - 1] = inside ? mul2(taps.w[W - 1].p[k], d.p[k]) : f2(0.f, 0.f);   // (no product: a weight may be infinite)
          out.p[k] = full[0];
#pragma unroll
          for (int m = 0; m < W - 1; ++m) sum[m].p[k] = full[m + 1];
        }
        move_on(past, now);
        const int done = s - (W - 1);
        if (kWhole || (s >= t0 && done >= 0)) {
          if (!kWhole && a.dstate_out) {   // the last tokens of a sequence are in its state_out as well
            int seq = row, end = a.tokens;
            if (a.sequences) {
              int begin = 0;
              seq = at.seqs.find(done);
              if (seq >= 0) at.seqs.bounds(seq, &begin, &end);
            }
            const int kept = done - end + W - 1;
            if (seq >= 0 && done < end && kept >= 0) {
              Channels<V> more;
              more.load(static_cast<const T*>(a.dstate_out) + ((int64_t)seq * (W - 1) + kept) * a.channels + c);
#pragma unroll
              for (int k = 0; k < kPairs; ++k) out.p[k] = add2(out.p[k], more.p[k]);
            }
          }
          out.store(to);
        }
        to += a.dx.token_pitch;
      }
    };
    if (ahead < t0) batch(ahead, t0, std::false_type());
    for (int t = t0; t < t1; t += kBatchBack) {
      if (t + kBatchBack <= t1 && t - at.begin >= W - 1 && t + kBatchBack <= at.end)
        batch(t, t + kBatchBack, std::true_type());
      else
        batch(t, min(t + kBatchBack, t1), std::false_type());
    }
    if (t1 == a.tokens) batch(t1, t1 + W - 1, std::false_type());
  }
  if (!partial) return;
  float* to = partial + ((int64_t)row * blocks_of_runs + blockIdx.y) * (W + 1) * a.channels;
  for (int k = 0; k <= W; ++k) {
    __syncthreads();
    Channels<V> v = dw[0];   // (dw[k], with indexes that are known)
#pragma unroll
    for (int q = 1; q <= W; ++q)
      if (k == q) v = dw[q];
    v.store(&part[threadIdx.y][threadIdx.x * V]);
    __syncthreads();
    for (int e = threadIdx.y * kVecs + threadIdx.x; e < kVecs * V; e += kVecs * kRuns) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < kRuns; ++r) s += part[r][e];
      const int ch = blockIdx.x * kVecs * V + e;
      if (ch < a.channels) to[(int64_t)k * a.channels + ch] = s;
    }
  }
}

// dweight, dbias: the partial sums in the order of their blocks.  blockIdx.y: the tap, or the bias.
template <typename T>
__global__ void __launch_bounds__(256) k_conv_params(lasp_conv_args a, const float* partial, int parts) {
  __shared__ float part[8][32];
  const int c = blockIdx.x * 32 + threadIdx.x, k = blockIdx.y;
  const int64_t all = (int64_t)(a.width + 1) * a.channels, i = (int64_t)k * a.channels + c;
  float s = 0.f;
  if (c < a.channels)
    for (int p = threadIdx.y; p < parts; p += 8) s += partial[p * all + i];
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y || c >= a.channels) return;
#pragma unroll
  for (int r = 1; r < 8; ++r) s += part[r][threadIdx.x];
  const bool f32 = a.param_dtype == LASP_F32;
  if (k < a.width) {
    if (a.dweight) store_param<T>(a.dweight, f32, (int64_t)c * a.width + k, s);
  } else if (a.dbias) {
    store_param<T>(a.dbias, f32, c, s);
  }
}

// Single tokens: the inputs before the next row's token, and that token, are sent for before this row is worked on.  256 rows of 4096 channels, bf16:
// 10 us (2.6 at the copy rate: a launch and three latencies one after the other, slot, state, output).
constexpr int kStepThreads = 128;
template <typename T, int V, int W>
__global__ void __launch_bounds__(kStepThreads) k_conv_step(lasp_conv_step_args a, int per) {
  __shared__ StepRows rows;
  const int row0 = blockIdx.y * per, count = min(per, a.rows - row0), c = (blockIdx.x * kStepThreads + threadIdx.x) * V;
  const bool mine = c < a.channels;
  const auto state = [&](int64_t slot) { return static_cast<T*>(a.state) + slot * (W - 1) * a.channels + c; };
  constexpr int kPairs = Channels<V>::kPairs;
  Channels<V> next[W - 1], x;
  const auto token = [&](int r) { return static_cast<const T*>(a.x.data) + (int64_t)r * a.x.row_pitch + c; };
  const auto fetch = [&](int r, int64_t slot) {
    if (slot < 0 || slot >= a.slot_count || !mine) return;
#pragma unroll
    for (int m = 0; m < W - 1; ++m) next[m].load(state(slot) + (int64_t)m * a.channels);
    x.load(token(r));
  };
  fetch(row0, a.slots ? index_at(a.slots, a.index_bits, row0) : row0);
  Taps<T, V, W> taps;
  if (mine) taps.load(a, c);
  rows.find(a.slots, a.index_bits, a.rows, row0, count);
  if (!mine) return;
  for (int q = 0; q < count; ++q) {
    const int64_t slot = rows.slot[q];
    Channels<V> past[W - 1], now = x;
#pragma unroll
    for (int m = 0; m < W - 1; ++m) past[m] = next[m];
    if (q + 1 < count && rows.first(q + 1)) fetch(row0 + q + 1, rows.slot[q + 1]);
    T* y = static_cast<T*>(a.y.data) + c;
    if (slot < 0 || slot >= a.slot_count) {   // a row that stands for no sequence
      Channels<V> none;
      none.clear();
      none.store(y + (int64_t)(row0 + q) * a.y.row_pitch);
      continue;
    }
    if (!rows.first(q)) continue;
    for (int r = row0 + q; r < a.rows; ++r) {
      if (r > row0 + q) {
        if (!rows.shared(q)) break;
        if (index_at(a.slots, a.index_bits, r) != slot) continue;
        now.load(token(r));
      }
      Channels<V> out;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const F2 p = taps.sum(past, now.p[k], k);
        out.p[k] = a.activation == LASP_ACT_SILU ? silu(p) : p;
      }
      move_on(past, now);
      out.store(y + (int64_t)r * a.y.row_pitch);
    }
#pragma unroll
    for (int m = 0; m < W - 1; ++m) past[m].store(state(slot) + (int64_t)m * a.channels);
  }
}

// Tokens of a run: long ones read fewer inputs twice and leave fewer partial sums, short ones give more threads.
int run_of(const lasp_conv_args& a, int v, int least) {
  const int64_t vecs = (a.channels + v - 1) / v, threads = (int64_t)sm_count() * 1024;
  const int64_t runs = std::max<int64_t>(1, threads / std::max<int64_t>(1, vecs * a.rows));
  int64_t run = (a.tokens + runs - 1) / runs;
  run = std::min<int64_t>(std::max<int64_t>(run, least), 64);
  run = std::max<int64_t>(run, (a.tokens + (int64_t)kRuns * 32768 - 1) / ((int64_t)kRuns * 32768));   // (the grid's second dimension)
  return (int)((run + kBatch - 1) / kBatch * kBatch);
}
int blocks_of_runs(const lasp_conv_args& a, int run) { return (int)(((int64_t)a.tokens + (int64_t)run * kRuns - 1) / ((int64_t)run * kRuns)); }

// V neighbouring channels of every tensor can be read and written by one access.
template <typename T>
bool wide(const lasp_conv_args& a, bool backward, int v) {
  const auto tokens = [v](const lasp_tokens& t) { return by(t, v * sizeof(T), sizeof(T)); };
  const auto states = [v](const void* p) { return reinterpret_cast<uintptr_t>(p) % (v * sizeof(T)) == 0; };
  if (a.channels % v || !tokens(a.x) || !states(a.state_in)) return false;
  return backward ? tokens(a.dy) && tokens(a.dx) && states(a.dstate_out) && states(a.dstate_in) : tokens(a.y) && states(a.state_out);
}

template <typename T, int V, int W>
cudaError_t forward_as(const lasp_conv_args& a, cudaStream_t st) {
  const int run = run_of(a, V, kBatch), blocks = blocks_of_runs(a, run);
  const int extra = !a.state_out ? 0 : a.sequences ? (a.sequences + kRuns - 1) / kRuns : 1;
  const dim3 grid((a.channels + kVecs * V - 1) / (kVecs * V), blocks + extra, a.rows);
  if (blocks + extra) k_conv_forward<T, V, W><<<grid, dim3(kVecs, kRuns), 0, st>>>(a, run, blocks);
  return cudaGetLastError();
}

template <typename T, int V, int W>
cudaError_t backward_as(const lasp_conv_args& a, cudaStream_t st) {
  const int run = run_of(a, V, 4 * kBatch), blocks = blocks_of_runs(a, run);
  const int extra = !a.dstate_in ? 0 : a.sequences ? (a.sequences + kRuns - 1) / kRuns : 1;
  const dim3 grid((a.channels + kVecs * V - 1) / (kVecs * V), blocks + extra, a.rows);
  const bool params = a.dweight || a.dbias;
  float* partial = params ? static_cast<float*>(a.ws) : nullptr;
  if (blocks + extra) k_conv_backward<T, V, W><<<grid, dim3(kVecs, kRuns), 0, st>>>(a, run, blocks, partial);
  if (params) k_conv_params<T><<<dim3((a.channels + 31) / 32, W + 1), dim3(32, 8), 0, st>>>(a, partial, blocks * a.rows);
  return cudaGetLastError();
}

template <typename T, int V>
cudaError_t forward_of(const lasp_conv_args& a, cudaStream_t st) {
  return a.width == 4 ? forward_as<T, V, 4>(a, st) : a.width == 3 ? forward_as<T, V, 3>(a, st) : forward_as<T, V, 2>(a, st);
}
template <typename T, int V>
cudaError_t backward_of(const lasp_conv_args& a, cudaStream_t st) {
  return a.width == 4 ? backward_as<T, V, 4>(a, st) : a.width == 3 ? backward_as<T, V, 3>(a, st) : backward_as<T, V, 2>(a, st);
}

// Channels of a thread.  Eight need 250 registers: 8 x 2048 x 4096 bf16 took 177 us forward and 552 backward, four 76 and 179, a pair (packed
// arithmetic, five and four blocks an SM) 62 and 128.
constexpr int kPair = 2;
template <typename T>
cudaError_t dispatch(const lasp_conv_args& a, bool backward, cudaStream_t st) {
  if (backward) return wide<T>(a, true, kPair) ? backward_of<T, kPair>(a, st) : backward_of<T, 1>(a, st);
  return wide<T>(a, false, kPair) ? forward_of<T, kPair>(a, st) : forward_of<T, 1>(a, st);
}

template <typename T, int V>
cudaError_t step_of(const lasp_conv_step_args& a, cudaStream_t st) {
  const int tiles = (a.channels + kStepThreads * V - 1) / (kStepThreads * V), per = step_rows(a.rows, tiles, 8);
  const dim3 grid(tiles, (a.rows + per - 1) / per);
  if (a.width == 4)
    k_conv_step<T, V, 4><<<grid, kStepThreads, 0, st>>>(a, per);
  else if (a.width == 3)
    k_conv_step<T, V, 3><<<grid, kStepThreads, 0, st>>>(a, per);
  else
    k_conv_step<T, V, 2><<<grid, kStepThreads, 0, st>>>(a, per);
  return cudaGetLastError();
}
template <typename T>
cudaError_t step_as(const lasp_conv_step_args& a, cudaStream_t st) {
  constexpr int v = 4;
  const auto fits = [](const lasp_tokens& t) { return by(t, v * sizeof(T), sizeof(T)); };
  const bool ok = a.channels % v == 0 && fits(a.x) && fits(a.y) && reinterpret_cast<uintptr_t>(a.state) % (v * sizeof(T)) == 0;
  return ok ? step_of<T, v>(a, st) : step_of<T, 1>(a, st);
}

}  // namespace

cudaError_t conv_forward(const lasp_conv_args& a, cudaStream_t st) {
  return a.dtype == LASP_F32 ? dispatch<float>(a, false, st) : a.dtype == LASP_BF16 ? dispatch<__nv_bfloat16>(a, false, st) : dispatch<__half>(a, false, st);
}
cudaError_t conv_backward(const lasp_conv_args& a, cudaStream_t st) {
  return a.dtype == LASP_F32 ? dispatch<float>(a, true, st) : a.dtype == LASP_BF16 ? dispatch<__nv_bfloat16>(a, true, st) : dispatch<__half>(a, true, st);
}
// (for either width of the accesses: it must not depend on the addresses, which the caller may not have yet)
size_t conv_workspace(const lasp_conv_args& a) {
  const int blocks = std::max(blocks_of_runs(a, run_of(a, kPair, 4 * kBatch)), blocks_of_runs(a, run_of(a, 1, 4 * kBatch)));
  return (size_t)a.rows * blocks * (a.width + 1) * a.channels * sizeof(float);
}
cudaError_t conv_step(const lasp_conv_step_args& a, cudaStream_t st) {
  return a.dtype == LASP_F32 ? step_as<float>(a, st) : a.dtype == LASP_BF16 ? step_as<__nv_bfloat16>(a, st) : step_as<__half>(a, st);
}

}  // namespace lasp
