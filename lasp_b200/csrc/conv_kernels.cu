// Short causal convolution, channel by channel, over prompts and training batches, and for single tokens.
//
//   p_t = bias + sum_j w_j x_(t-W+1+j),  y_t = p_t or silu(p_t)
//   dp_t = dy_t silu'(p_t),  dx_t = sum_k w_(W-1-k) dp_(t+k),  dw_j = sum_t dp_t x_(t-W+1+j)
//
// A thread owns V neighbouring channels (16 bytes) and a run of tokens: the last W - 1 inputs slide through its registers, so
// that every input is read once but for the W - 1 ahead of a run.  What bounds it is memory; nothing is staged.
#include <algorithm>

#include "recurrent.cuh"

namespace lasp {
namespace {

constexpr int kVecs = 32, kRuns = 8;   // a block: 32 vectors of channels times 8 runs of tokens
constexpr int kBatch = 8;              // tokens whose loads are under way together

struct Rows {   // where a thread's channels of a row of tokens lie
  int64_t row, token;
};

template <typename T, int V, int W>
struct Taps {
  float w[W][V];
  __device__ __forceinline__ void load(const lasp_conv_args& a, int c) {
    const bool f32 = a.param_dtype == LASP_F32;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) w[j][i] = param<T>(a.weight, f32, (int64_t)(c + i) * W + j);
  }
};

template <typename T, int V>
__device__ __forceinline__ void load_bias(const void* bias, int param_dtype, int c, float (&out)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = bias ? param<T>(bias, param_dtype == LASP_F32, c + i) : 0.f;
}

// x at token p of a sequence that begins at `begin`; what lies before is its state, or zero
template <typename T, int V, int W>
__device__ __forceinline__ void input_at(const T* x, int64_t pitch, const T* state, int64_t c_total, int begin, int p, float (&out)[V]) {
  if (p >= begin) {
    load_vec<T, V>(x + (int64_t)p * pitch, out);
  } else if (state && p - begin + W - 1 >= 0) {
    load_vec<T, V>(state + (int64_t)(p - begin + W - 1) * c_total, out);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = 0.f;
  }
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
  for (int m = 0; m < W - 1; ++m) {
    float v[V];
    input_at<T, V, W>(x, a.x.token_pitch, from, a.channels, begin, end - (W - 1) + m, v);
    store_vec<T, V>(to + (int64_t)m * a.channels, v);
  }
}

template <typename T, int V, int W>
__global__ void __launch_bounds__(kVecs* kRuns) k_conv_forward(lasp_conv_args a, int run, int blocks_of_runs) {
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
  float bias[V];
  load_bias<T, V>(a.bias, a.param_dtype, c, bias);
  Place<T, W> at;
  at.start(a, row, t0);
  float past[W - 1][V];   // past[m]: x_(t-W+1+m)
#pragma unroll
  for (int m = 0; m < W - 1; ++m)
    input_at<T, V, W>(x, a.x.token_pitch, at.state(a.state_in, a.channels, c), a.channels, at.begin, t0 - (W - 1) + m, past[m]);
  for (int t = t0; t < t1; t += kBatch) {
    Vec<T, V> in[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (t + j < t1) in[j] = *reinterpret_cast<const Vec<T, V>*>(x + (int64_t)(t + j) * a.x.token_pitch);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (t + j >= t1) break;
      bool inside = true;
      if (a.sequences) {
        if (t + j >= at.end) {
          at.advance(t + j);
          if (t + j >= at.begin) {
#pragma unroll
            for (int m = 0; m < W - 1; ++m)
              input_at<T, V, W>(x, a.x.token_pitch, at.state(a.state_in, a.channels, c), a.channels, at.begin, t + j - (W - 1) + m, past[m]);
          }
        }
        inside = at.inside(t + j);
      }
      float now[V], out[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        now[i] = to_f(in[j].v[i]);
        float p = fmaf(taps.w[W - 1][i], now[i], bias[i]);
#pragma unroll
        for (int m = 0; m < W - 1; ++m) p = fmaf(taps.w[m][i], past[m][i], p);
        out[i] = inside ? (a.activation == LASP_ACT_SILU ? silu(p) : p) : 0.f;
#pragma unroll
        for (int m = 0; m + 1 < W - 1; ++m) past[m][i] = past[m + 1][i];
        past[W - 2][i] = now[i];
      }
      store_vec<T, V>(y + (int64_t)(t + j) * a.y.token_pitch, out);
    }
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
  Taps<T, V, W> taps;
  taps.load(a, c);
  float bias[V], sum[W - 1][V];
  load_bias<T, V>(a.bias, a.param_dtype, c, bias);
#pragma unroll
  for (int m = 0; m < W - 1; ++m) {
    const int kept = begin - end + m;   // its place in state_out, if it is there still
#pragma unroll
    for (int i = 0; i < V; ++i) sum[m][i] = 0.f;
    if (a.dstate_out && kept >= 0) load_vec<T, V>(static_cast<const T*>(a.dstate_out) + at + (int64_t)kept * a.channels, sum[m]);
  }
#pragma unroll
  for (int r = 0; r < W - 1; ++r) {   // token begin + r reaches back to state entries r, r + 1, ...
    if (begin + r >= end) break;
    float d[V], p[V];
    load_vec<T, V>(dy + (int64_t)(begin + r) * a.dy.token_pitch, d);
    if (a.activation == LASP_ACT_SILU) {
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = bias[i];
#pragma unroll
      for (int j = 0; j < W; ++j) {
        float v[V];
        input_at<T, V, W>(x, a.x.token_pitch, from, a.channels, begin, begin + r - (W - 1) + j, v);
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = fmaf(taps.w[j][i], v[i], p[i]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] *= d_silu(p[i]);
    }
#pragma unroll
    for (int m = r; m < W - 1; ++m)
#pragma unroll
      for (int i = 0; i < V; ++i) sum[m][i] = fmaf(taps.w[m - r][i], d[i], sum[m][i]);
  }
#pragma unroll
  for (int m = 0; m < W - 1; ++m) store_vec<T, V>(static_cast<T*>(a.dstate_in) + at + (int64_t)m * a.channels, sum[m]);
}

// partial: for each row and block of runs, W + 1 rows of `channels` sums (the taps' and the bias')
template <typename T, int V, int W>
__global__ void __launch_bounds__(kVecs* kRuns) k_conv_backward(lasp_conv_args a, int run, int blocks_of_runs, float* partial) {
  __shared__ float part[kRuns][kVecs * V];
  const int c = (blockIdx.x * kVecs + threadIdx.x) * V, row = blockIdx.z;
  const bool mine = c < a.channels;
  if ((int)blockIdx.y >= blocks_of_runs) {
    const int seq = a.sequences ? ((int)blockIdx.y - blocks_of_runs) * kRuns + threadIdx.y : row;
    if (mine && (a.sequences ? seq < a.sequences : threadIdx.y == 0)) write_dstate<T, V, W>(a, row, seq, c);
    return;
  }
  float dw[W + 1][V] = {};
  const int64_t first = ((int64_t)blockIdx.y * kRuns + threadIdx.y) * run;
  if (mine && first < a.tokens) {
    const int t0 = (int)first, t1 = first + run < a.tokens ? (int)first + run : a.tokens;
    const T* x = static_cast<const T*>(a.x.data) + (int64_t)row * a.x.row_pitch + c;
    const T* dy = static_cast<const T*>(a.dy.data) + (int64_t)row * a.dy.row_pitch + c;
    T* dx = static_cast<T*>(a.dx.data) + (int64_t)row * a.dx.row_pitch + c;
    Taps<T, V, W> taps;
    taps.load(a, c);
    float bias[V];
    load_bias<T, V>(a.bias, a.param_dtype, c, bias);
    Place<T, W> at;
    at.start(a, row, t0);
    float past[W - 1][V], sum[W - 1][V];   // sum[m]: dx_(t-W+1+m) so far
#pragma unroll
    for (int m = 0; m < W - 1; ++m) {
      input_at<T, V, W>(x, a.x.token_pitch, at.state(a.state_in, a.channels, c), a.channels, at.begin, t0 - (W - 1) + m, past[m]);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[m][i] = 0.f;
    }
    // token t + W - 1 completes dx_t: a run looks W - 1 tokens beyond its end
    const int stop = t1 + W - 1;
    for (int t = t0; t < stop; t += kBatch) {
      Vec<T, V> in[kBatch], din[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (t + j < stop && t + j < a.tokens) {
          in[j] = *reinterpret_cast<const Vec<T, V>*>(x + (int64_t)(t + j) * a.x.token_pitch);
          din[j] = *reinterpret_cast<const Vec<T, V>*>(dy + (int64_t)(t + j) * a.dy.token_pitch);
        }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int s = t + j;
        if (s >= stop) break;
        bool inside = s < a.tokens;
        if (a.sequences && inside) {
          if (s >= at.end) {
            at.advance(s);
            if (s >= at.begin) {
#pragma unroll
              for (int m = 0; m < W - 1; ++m)
                input_at<T, V, W>(x, a.x.token_pitch, at.state(a.state_in, a.channels, c), a.channels, at.begin, s - (W - 1) + m, past[m]);
            }
          }
          inside = at.inside(s);
        }
        const int reach = inside ? s - at.begin : -1;   // how far back in its sequence this token's gradient goes
        float out[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float now = inside ? to_f(in[j].v[i]) : 0.f;
          float d = inside ? to_f(din[j].v[i]) : 0.f;
          if (a.activation == LASP_ACT_SILU) {
            float p = fmaf(taps.w[W - 1][i], now, bias[i]);
#pragma unroll
            for (int m = 0; m < W - 1; ++m) p = fmaf(taps.w[m][i], past[m][i], p);
            d = inside ? d * d_silu(p) : 0.f;
          }
          if (s < t1 && inside) {
#pragma unroll
            for (int m = 0; m < W - 1; ++m) dw[m][i] = fmaf(d, past[m][i], dw[m][i]);
            dw[W - 1][i] = fmaf(d, now, dw[W - 1][i]);
            dw[W][i] += d;
          }
          float full[W];
#pragma unroll
          for (int m = 0; m < W - 1; ++m) full[m] = reach >= W - 1 - m ? fmaf(taps.w[m][i], d, sum[m][i]) : sum[m][i];
          full[W - 1] = taps.w[W - 1][i] * d;
          out[i] = full[0];
#pragma unroll
          for (int m = 0; m < W - 1; ++m) sum[m][i] = full[m + 1];
#pragma unroll
          for (int m = 0; m + 1 < W - 1; ++m) past[m][i] = past[m + 1][i];
          past[W - 2][i] = now;
        }
        const int done = s - (W - 1);
        if (done >= t0) {
          if (a.dstate_out) {   // the last tokens of a sequence are in its state_out as well
            int seq = row, end = a.tokens;
            if (a.sequences) {
              int begin = 0;
              seq = at.seqs.find(done);
              if (seq >= 0) at.seqs.bounds(seq, &begin, &end);
            }
            const int kept = done - end + W - 1;
            if (seq >= 0 && done < end && kept >= 0) {
              float more[V];
              load_vec<T, V>(static_cast<const T*>(a.dstate_out) + ((int64_t)seq * (W - 1) + kept) * a.channels + c, more);
#pragma unroll
              for (int i = 0; i < V; ++i) out[i] += more[i];
            }
          }
          store_vec<T, V>(dx + (int64_t)done * a.dx.token_pitch, out);
        }
      }
    }
  }
  if (!partial) return;
  float* to = partial + ((int64_t)row * blocks_of_runs + blockIdx.y) * (W + 1) * a.channels;
  for (int k = 0; k <= W; ++k) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float v = dw[0][i];   // (dw[k], with indexes that are known)
#pragma unroll
      for (int q = 1; q <= W; ++q) v = k == q ? dw[q][i] : v;
      part[threadIdx.y][threadIdx.x * V + i] = v;
    }
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

// dweight, dbias: the partial sums in the order of their blocks
template <typename T>
__global__ void __launch_bounds__(256) k_conv_params(lasp_conv_args a, const float* partial, int parts) {
  __shared__ float part[8][32];
  const int i = blockIdx.x * 32 + threadIdx.x, all = (a.width + 1) * a.channels;
  float s = 0.f;
  if (i < all)
    for (int p = threadIdx.y; p < parts; p += 8) s += partial[(int64_t)p * all + i];
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y || i >= all) return;
#pragma unroll
  for (int r = 1; r < 8; ++r) s += part[r][threadIdx.x];
  const int k = i / a.channels, c = i - k * a.channels;
  const bool f32 = a.param_dtype == LASP_F32;
  if (k < a.width) {
    if (a.dweight) store_param<T>(a.dweight, f32, (int64_t)c * a.width + k, s);
  } else if (a.dbias) {
    store_param<T>(a.dbias, f32, c, s);
  }
}

template <typename T, int V, int W>
__global__ void __launch_bounds__(128) k_conv_step(lasp_conv_step_args a) {
  const int row = blockIdx.y, c = (blockIdx.x * blockDim.x + threadIdx.x) * V;
  const bool mine = c < a.channels;
  const int64_t slot = a.slots ? index_at(a.slots, a.index_bits, row) : row;
  T* y = static_cast<T*>(a.y.data) + c;
  if (slot < 0 || slot >= a.slot_count) {   // a row that stands for no sequence
    const float none[V] = {};
    if (mine) store_vec<T, V>(y + (int64_t)row * a.y.row_pitch, none);
    return;
  }
  const int shared = shared_slot(a.slots, a.index_bits, a.rows, row, slot);
  if (shared < 0 || !mine) return;
  T* state = static_cast<T*>(a.state) + slot * (W - 1) * a.channels + c;
  const bool f32 = a.param_dtype == LASP_F32;
  float past[W - 1][V], w[W][V], bias[V];
#pragma unroll
  for (int m = 0; m < W - 1; ++m) load_vec<T, V>(state + (int64_t)m * a.channels, past[m]);
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][i] = param<T>(a.weight, f32, (int64_t)(c + i) * W + j);
  }
  load_bias<T, V>(a.bias, a.param_dtype, c, bias);
  for (int r = row; r < a.rows; ++r) {
    if (r > row && (!shared || index_at(a.slots, a.index_bits, r) != slot)) {
      if (!shared) break;
      continue;
    }
    float now[V], out[V];
    load_vec<T, V>(static_cast<const T*>(a.x.data) + (int64_t)r * a.x.row_pitch + c, now);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float p = fmaf(w[W - 1][i], now[i], bias[i]);
#pragma unroll
      for (int m = 0; m < W - 1; ++m) p = fmaf(w[m][i], past[m][i], p);
      out[i] = a.activation == LASP_ACT_SILU ? silu(p) : p;
#pragma unroll
      for (int m = 0; m + 1 < W - 1; ++m) past[m][i] = past[m + 1][i];
      past[W - 2][i] = now[i];
    }
    store_vec<T, V>(y + (int64_t)r * a.y.row_pitch, out);
  }
#pragma unroll
  for (int m = 0; m < W - 1; ++m) store_vec<T, V>(state + (int64_t)m * a.channels, past[m]);
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

template <typename T>
bool wide(const lasp_conv_args& a, bool backward) {
  constexpr int v = 16 / sizeof(T);
  bool ok = a.channels % v == 0 && vector_ok(a.x, sizeof(T)) && vector_ok(a.state_in);
  if (backward)
    return ok && vector_ok(a.dy, sizeof(T)) && vector_ok(a.dx, sizeof(T)) && vector_ok(a.dstate_out) && vector_ok(a.dstate_in);
  return ok && vector_ok(a.y, sizeof(T)) && vector_ok(a.state_out);
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
  if (params) k_conv_params<T><<<((W + 1) * a.channels + 31) / 32, dim3(32, 8), 0, st>>>(a, partial, blocks * a.rows);
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

template <typename T>
cudaError_t dispatch(const lasp_conv_args& a, bool backward, cudaStream_t st) {
  constexpr int v = 16 / sizeof(T);
  if (wide<T>(a, backward)) return backward ? backward_of<T, v>(a, st) : forward_of<T, v>(a, st);
  return backward ? backward_of<T, 1>(a, st) : forward_of<T, 1>(a, st);
}

template <typename T, int V>
cudaError_t step_of(const lasp_conv_step_args& a, cudaStream_t st) {
  const dim3 grid((a.channels + 128 * V - 1) / (128 * V), a.rows);
  if (a.width == 4)
    k_conv_step<T, V, 4><<<grid, 128, 0, st>>>(a);
  else if (a.width == 3)
    k_conv_step<T, V, 3><<<grid, 128, 0, st>>>(a);
  else
    k_conv_step<T, V, 2><<<grid, 128, 0, st>>>(a);
  return cudaGetLastError();
}
template <typename T>
cudaError_t step_as(const lasp_conv_step_args& a, cudaStream_t st) {
  constexpr int v = 16 / sizeof(T);
  const bool ok = a.channels % v == 0 && vector_ok(a.x, sizeof(T)) && vector_ok(a.y, sizeof(T)) && vector_ok(a.state);
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
  const int v = a.dtype == LASP_F32 ? 4 : 8;
  const int blocks = std::max(blocks_of_runs(a, run_of(a, v, 4 * kBatch)), blocks_of_runs(a, run_of(a, 1, 4 * kBatch)));
  return (size_t)a.rows * blocks * (a.width + 1) * a.channels * sizeof(float);
}
cudaError_t conv_step(const lasp_conv_step_args& a, cudaStream_t st) {
  return a.dtype == LASP_F32 ? step_as<float>(a, st) : a.dtype == LASP_BF16 ? step_as<__nv_bfloat16>(a, st) : step_as<__half>(a, st);
}

}  // namespace lasp
