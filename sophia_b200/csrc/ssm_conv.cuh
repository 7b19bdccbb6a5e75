// Causal depthwise convolution over tokens, with an optional SiLU:
//   c[t] = bias + sum_{k<W} w[k] x[t - (W-1) + k],   y = silu(c) or c,
// per channel, 1 <= W <= 4.  Inputs before a sequence's first token are its initial
// state [W-1] (oldest first; zeros without one); the final state is its last
// W-1 inputs.  Backward, with dc = dy * silu'(c):
//   dx[t] = sum_k w[k] dc[t + (W-1) - k],  dw[k] = sum_t dc[t] x[t-(W-1)+k],
//   dbias = sum_t dc[t],
// the terms of positions before the first token going to the initial state.
//
// Memory bound: x is read once and y written once (forward), x and dy read and
// dx written once (backward, c is recomputed).  A thread owns V neighbouring
// channels and walks a run of tokens with the last three inputs (and the three
// pending dx) in registers; runs re-read a halo of three tokens.  W < 4 runs as
// four taps whose leading ones are left out (FULL = false): not multiplied by zero, so that
// an infinity beyond the taps' reach stays out of the sum.
#pragma once

#include "ssm_common.cuh"

namespace kda {

constexpr int CONV_THREADS = 256;
constexpr int CONV_UNROLL = 4;  // rows loaded ahead

struct ConvParams {
  RowView x, dy;        // [B, T, C]
  const float *w, *bias;  // [C][W], [C] or null
  const float* h0;      // [nseq][C][W-1] or null
  SeqMap seq;
  int B, T, C, W, run, runs;  // runs per row, of `run` tokens
  bool silu;
  void* y;              // [B, T, C] contiguous (forward)
  float* ht;            // [nseq][C][W-1] or null
  // backward
  const float* dht;
  void* dx;             // [B, T, C] contiguous
  float* dh0;           // or null
  float* partial;       // [B * runs][C][W + 1]: dw, dbias
};

template <int V>
__device__ __forceinline__ void conv_taps(const ConvParams& P, int c0, float (&w)[4][V], float (&bias)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = P.bias ? __ldg(P.bias + c0 + i) : 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k][i] = k >= 4 - P.W ? __ldg(P.w + (long long)(c0 + i) * P.W + k - (4 - P.W)) : 0.f;
  }
}

// The three inputs before a sequence's first token.
template <int V>
__device__ __forceinline__ void conv_enter(const ConvParams& P, int seq, int c0, float (&win)[3][V]) {
#pragma unroll
  for (int s = 0; s < 3; ++s)
#pragma unroll
    for (int i = 0; i < V; ++i)
      win[s][i] = P.h0 && s >= 4 - P.W
                      ? __ldg(P.h0 + ((long long)seq * P.C + c0 + i) * (P.W - 1) + s - (4 - P.W))
                      : 0.f;
}

template <int V>
__device__ __forceinline__ void conv_push(float (&win)[3][V], const float (&x)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    win[0][i] = win[1][i];
    win[1][i] = win[2][i];
    win[2][i] = x[i];
  }
}

template <int V, bool FULL>
__device__ __forceinline__ void conv_point(int W, const float (&w)[4][V], const float (&bias)[V],
                                           const float (&win)[3][V], const float (&x)[V], float (&c)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float v = bias[i];
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (FULL || k >= 4 - W) v = fmaf(w[k][i], win[k][i], v);
    c[i] = fmaf(w[3][i], x[i], v);
  }
}

// The window in front of token t0: the three tokens before it, walked so that a
// sequence that starts among them brings in its initial state.
template <typename T, int V>
__device__ __forceinline__ void conv_window(const ConvParams& P, int b, int t0, int c0, float (&win)[3][V]) {
#pragma unroll
  for (int s = 0; s < 3; ++s)
#pragma unroll
    for (int i = 0; i < V; ++i) win[s][i] = 0.f;
#pragma unroll
  for (int s = 3; s >= 1; --s) {
    const int t = t0 - s;
    if (t < 0) continue;
    const int q = seq_start_at(P.seq, b, t);
    if (q >= 0) conv_enter<V>(P, q, c0, win);
    float x[V];
    io_load<T, V>(row_ptr<T>(P.x, b, t) + c0, x);
    conv_push<V>(win, x);
  }
}

struct ConvItem {
  int b, t0, t1, c0;
  long long run;
  bool ok;
};
template <int V>
__device__ __forceinline__ ConvItem conv_item(const ConvParams& P) {
  ConvItem it;
  const int nvec = P.C / V;
  const long long idx = (long long)blockIdx.x * CONV_THREADS + threadIdx.x;
  it.run = idx / nvec;
  it.c0 = (int)(idx - it.run * nvec) * V;
  it.ok = it.run < (long long)P.B * P.runs;
  it.b = (int)(it.run / P.runs);
  it.t0 = (int)(it.run - (long long)it.b * P.runs) * P.run;
  it.t1 = min(it.t0 + P.run, P.T);
  return it;
}

template <typename T, int V, bool FULL>
__global__ void __launch_bounds__(CONV_THREADS) ssm_conv_fwd_kernel(ConvParams P) {
  const ConvItem it = conv_item<V>(P);
  if (!it.ok) return;
  float w[4][V], bias[V], win[3][V];
  conv_taps<V>(P, it.c0, w, bias);
  conv_window<T, V>(P, it.b, it.t0, it.c0, win);
  T* y = static_cast<T*>(P.y) + ((long long)it.b * P.T) * P.C + it.c0;
  for (int t = it.t0; t < it.t1; t += CONV_UNROLL) {
    float x[CONV_UNROLL][V];
#pragma unroll
    for (int u = 0; u < CONV_UNROLL; ++u)
      if (t + u < it.t1) io_load<T, V>(row_ptr<T>(P.x, it.b, t + u) + it.c0, x[u]);
#pragma unroll
    for (int u = 0; u < CONV_UNROLL; ++u) {
      if (t + u >= it.t1) break;
      const int q = seq_start_at(P.seq, it.b, t + u);
      if (q >= 0) conv_enter<V>(P, q, it.c0, win);
      float c[V];
      conv_point<V, FULL>(P.W, w, bias, win, x[u], c);
      if (P.silu) {
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = siluf_(c[i]);
      }
      io_store<T, V>(y + (long long)(t + u) * P.C, c);
      conv_push<V>(win, x[u]);
      if (P.ht) {
        const int e = seq_end_at(P.seq, it.b, t + u);
        if (e >= 0) {
#pragma unroll
          for (int s = 0; s < 3; ++s)
#pragma unroll
            for (int i = 0; i < V; ++i)
              if (s >= 4 - P.W) P.ht[((long long)e * P.C + it.c0 + i) * (P.W - 1) + s - (4 - P.W)] = win[s][i];
        }
      }
    }
  }
}

// A pending dx leaves three tokens after its own, when the last tap that reads
// its input has been seen.  Slots of positions before a sequence's first token
// leave into its initial state's gradient.
template <typename T, int V>
__device__ __forceinline__ void conv_emit(const ConvParams& P, const ConvItem& it, int pos, int first, int seq,
                                          const float (&v)[V]) {
  if (pos >= first) {
    if (pos >= it.t0 && pos < it.t1)
      io_store<T, V>(static_cast<T*>(P.dx) + ((long long)it.b * P.T + pos) * P.C + it.c0, v);
  } else if (P.dh0 && first >= it.t0 && first < it.t1) {
    const int s = pos - (first - 3) - (4 - P.W);  // slot of the W-1 inputs before `first`
    if (s >= 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) P.dh0[((long long)seq * P.C + it.c0 + i) * (P.W - 1) + s] = v[i];
    }
  }
}

template <typename T, int V, bool FULL>
__global__ void __launch_bounds__(CONV_THREADS) ssm_conv_bwd_kernel(ConvParams P) {
  const ConvItem it = conv_item<V>(P);
  if (!it.ok) return;
  float w[4][V], bias[V], win[3][V], pend[3][V], dw[5][V];
  conv_taps<V>(P, it.c0, w, bias);
  conv_window<T, V>(P, it.b, it.t0, it.c0, win);
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int s = 0; s < 3; ++s) pend[s][i] = 0.f;
#pragma unroll
    for (int k = 0; k < 5; ++k) dw[k][i] = 0.f;
  }
  // first token of the current sequence; before the run only its being at most t0 - 3 or
  // the run's own start matter, as slots before t0 belong to the run in front
  int first = it.t0 - 3, seq = -1;
  const int stop = min(it.t1 + 3, P.T);
  int t = it.t0;
  for (; t < stop; ++t) {
    const int q = seq_start_at(P.seq, it.b, t);
    if (q >= 0) {
      if (t > it.t0) {  // the sequence in front ends: its pending slots are complete
#pragma unroll
        for (int s = 0; s < 3; ++s) conv_emit<T, V>(P, it, t - 3 + s, first, seq, pend[s]);
      }
      if (t >= it.t1) break;
      conv_enter<V>(P, q, it.c0, win);
      first = t;
      seq = q;
#pragma unroll
      for (int s = 0; s < 3; ++s)
#pragma unroll
        for (int i = 0; i < V; ++i) pend[s][i] = 0.f;
    }
    float x[V], dc[V], c[V];
    io_load<T, V>(row_ptr<T>(P.x, it.b, t) + it.c0, x);
    io_load<T, V>(row_ptr<T>(P.dy, it.b, t) + it.c0, dc);
    if (P.silu) {
      conv_point<V, FULL>(P.W, w, bias, win, x, c);
#pragma unroll
      for (int i = 0; i < V; ++i) dc[i] *= silu_slopef_(c[i]);
    }
    if (t < it.t1) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        dw[0][i] = fmaf(dc[i], win[0][i], dw[0][i]);
        dw[1][i] = fmaf(dc[i], win[1][i], dw[1][i]);
        dw[2][i] = fmaf(dc[i], win[2][i], dw[2][i]);
        dw[3][i] = fmaf(dc[i], x[i], dw[3][i]);
        dw[4][i] += dc[i];
      }
    }
    float out[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      out[i] = FULL || P.W > 3 ? fmaf(w[0][i], dc[i], pend[0][i]) : pend[0][i];
      pend[0][i] = FULL || P.W > 2 ? fmaf(w[1][i], dc[i], pend[1][i]) : pend[1][i];
      pend[1][i] = FULL || P.W > 1 ? fmaf(w[2][i], dc[i], pend[2][i]) : pend[2][i];
      pend[2][i] = w[3][i] * dc[i];
    }
    conv_emit<T, V>(P, it, t - 3, first, seq, out);
    conv_push<V>(win, x);
    if (P.dht) {
      const int e = seq_end_at(P.seq, it.b, t);
      if (e >= 0) {
#pragma unroll
        for (int s = 0; s < 3; ++s)
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (s >= 4 - P.W)
              pend[s][i] += __ldg(P.dht + ((long long)e * P.C + it.c0 + i) * (P.W - 1) + s - (4 - P.W));
      }
    }
  }
  if (t == P.T) {  // the row's end completes what is pending
#pragma unroll
    for (int s = 0; s < 3; ++s) conv_emit<T, V>(P, it, t - 3 + s, first, seq, pend[s]);
  }
  float* part = P.partial + (it.run * P.C + it.c0) * (P.W + 1);
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int k = 0; k < 5; ++k)
      if (k >= 4 - P.W) part[i * (P.W + 1) + k - (4 - P.W)] = dw[k][i];
}

// One token for each of `rows` requests: the W-1 last inputs of its slot are read,
// used and rewritten.  slots[r] < 0 marks a padding row (y = 0, nothing else touched);
// a slot past the pool sets the device error 11 and is treated the same.
struct ConvStepParams {
  const void* x;
  long long sx;  // row stride of x (elements)
  const float *w, *bias;
  float* state;  // [pool][C][W-1]
  const int* slots;
  int rows, C, W, pool;
  bool silu;
  void* y;  // [rows][C]
  int* err;
};

template <typename T>
__global__ void __launch_bounds__(CONV_THREADS) ssm_conv_step_kernel(ConvStepParams P) {
  const int c = blockIdx.x * CONV_THREADS + threadIdx.x;
  if (c >= P.C) return;
  float w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = k >= 4 - P.W ? __ldg(P.w + (long long)c * P.W + k - (4 - P.W)) : 0.f;
  const float bias = P.bias ? __ldg(P.bias + c) : 0.f;
  const int skip = 4 - P.W;
  for (int r = blockIdx.y; r < P.rows; r += gridDim.y) {
    const int s = step_slot(P.slots, r, P.pool, P.err);
    float out = 0.f;
    if (s >= 0) {
      float* st = P.state + ((long long)s * P.C + c) * (P.W - 1);
      float win[3];
#pragma unroll
      for (int k = 0; k < 3; ++k) win[k] = k >= skip ? st[k - skip] : 0.f;
      const float x = io_to_f(static_cast<const T*>(P.x)[r * P.sx + c]);
      out = bias;
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (k >= skip) out = fmaf(w[k], win[k], out);
      out = fmaf(w[3], x, out);
      if (P.silu) out = siluf_(out);
      if (skip < 1) st[0] = win[1];
      if (skip < 2) st[1 - skip] = win[2];
      if (skip < 3) st[2 - skip] = x;
    }
    static_cast<T*>(P.y)[(long long)r * P.C + c] = io_from_f<T>(out);
  }
}

}  // namespace kda
