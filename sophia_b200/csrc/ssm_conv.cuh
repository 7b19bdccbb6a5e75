// Causal depthwise convolution over tokens, with an optional SiLU:
//   c[t] = bias + sum_{k<W} w[k] x[t - (W-1) + k],   y = silu(c) or c,
// per channel, 1 <= W <= 4.  Inputs before a sequence's first token are its initial
// state [W-1] (oldest first; zeros without one); the final state is its last
// W-1 inputs.  Backward, with dc = dy * silu'(c):
//   dx[t] = sum_k w[k] dc[t + (W-1) - k],  dw[k] = sum_t dc[t] x[t-(W-1)+k],
//   dbias = sum_t dc[t],
// the terms of positions before the first token going to the initial state.
//
// Memory bound by its bytes: x is read once and y written once (forward), x and dy read and
// dx written once (backward, c is recomputed).  A thread owns V = 2 neighbouring
// channels (1 where rows are not aligned for that) and walks a run of tokens with the last
// three inputs (and the three pending dx) in registers, rows fetched groups ahead through a ring in
// shared memory; runs re-read a halo of three tokens.  Two channels a thread rather than eight: the same bytes in
// flight from four times the threads at a third of the registers.  W < 4 runs as
// four taps whose leading ones are left out (FULL = false): not multiplied by zero, so that
// an infinity beyond the taps' reach stays out of the sum.
// Measured, bf16 [4, 4096, 2048] with SiLU: forward 36 us (3.7 TB/s of 134 MB), backward
// 64 us (3.2 TB/s of 201 MB) and 3 us to join dw.  No pipe is full by the counters of that size; warps wait for their
// own results.  Forward: 58 % of issue slots, 49 % of the pipe of ex2 and rcp, 31 % of HBM's time, 6.7 warps per
// scheduler of which 1.8 can issue, 1024 CTAs in 1.7 waves.  Backward: 53 %, 26 %, 31 %, 3.4 warps (114 registers) of
// which 1.0 can issue; of the 6.4 cycles between a warp's instructions 2.0 are fixed latency, 0.8 shared memory
// and special functions, 0.7 the fp32 pipe.
#pragma once

#include <type_traits>

#include "ssm_common.cuh"

namespace kda {

constexpr int CONV_THREADS = 256;
constexpr int CONV_BWD_GROUP = 4;
constexpr int CONV_GROUP = 8;  // rows a forward group (the ring holds four groups of 4-byte pieces, two of 8 bytes)

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
__device__ __forceinline__ void conv_taps(const ConvParams& P, int c0, Lane<V> (&w)[4], Lane<V>& bias) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias.set(i, P.bias ? __ldg(P.bias + c0 + i) : 0.f);
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k].set(i, k >= 4 - P.W ? __ldg(P.w + (long long)(c0 + i) * P.W + k - (4 - P.W)) : 0.f);
  }
}

// The three inputs before a sequence's first token.
template <int V>
__device__ __forceinline__ void conv_enter(const ConvParams& P, int seq, int c0, Lane<V> (&win)[3]) {
#pragma unroll
  for (int s = 0; s < 3; ++s)
#pragma unroll
    for (int i = 0; i < V; ++i)
      win[s].set(i, P.h0 && s >= 4 - P.W
                        ? __ldg(P.h0 + ((long long)seq * P.C + c0 + i) * (P.W - 1) + s - (4 - P.W))
                        : 0.f);
}

template <int V>
__device__ __forceinline__ void conv_push(Lane<V> (&win)[3], const Lane<V>& x) {
  win[0] = win[1];
  win[1] = win[2];
  win[2] = x;
}

template <int V, bool FULL>
__device__ __forceinline__ Lane<V> conv_point(int W, const Lane<V> (&w)[4], const Lane<V>& bias, const Lane<V> (&win)[3],
                                              const Lane<V>& x) {
  Lane<V> c = bias;
#pragma unroll
  for (int k = 0; k < 3; ++k)
    if (FULL || k >= 4 - W) c = fma(w[k], win[k], c);
  return fma(w[3], x, c);
}

// The window in front of token t0: the three tokens before it, walked so that a
// sequence that starts among them brings in its initial state.
template <typename T, int V>
__device__ __forceinline__ void conv_window(const ConvParams& P, int b, int t0, int c0, Lane<V> (&win)[3]) {
#pragma unroll
  for (int s = 0; s < 3; ++s) win[s] = Lane<V>::all(0.f);
#pragma unroll
  for (int s = 3; s >= 1; --s) {
    const int t = t0 - s;
    if (t < 0) continue;
    const int q = seq_start_at(P.seq, b, t);
    if (q >= 0) conv_enter<V>(P, q, c0, win);
    conv_push<V>(win, lane_from(*reinterpret_cast<const IoVec<T, V>*>(row_ptr<T>(P.x, b, t) + c0)));
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

// Rows on their way to a thread, STAGES - 1 groups ahead: by cp.async into a ring in shared memory
// of which every thread reads back only its own pieces (no barrier), so bytes in flight
// cost no registers.  Pieces under 4 bytes (single 16-bit channels) are loaded when needed.
template <typename T, int V, int TENSORS, int GROUP>
struct ConvRing {
  static constexpr bool ASYNC = sizeof(T) * V >= 4;
  static constexpr int STAGES = ASYNC ? 16 / (int)(sizeof(T) * V) : 1;  // 32 KB of ring
  typedef IoVec<T, V> Piece;
  struct Smem {
    Piece p[STAGES][TENSORS][GROUP][CONV_THREADS];
  };
  Smem& sm;
  const T* src[TENSORS];
  long long st[TENSORS];
  int next, last;  // token of the next fetch, end of the tokens
  int put, get;
  __device__ __forceinline__ ConvRing(Smem& s, int t0, int t1) : sm(s), next(t0), last(t1), put(0), get(0) {}
  __device__ __forceinline__ void fetch() {
#pragma unroll
    for (int q = 0; q < TENSORS; ++q) {
#pragma unroll
      for (int u = 0; u < GROUP; ++u)
        if (ASYNC && next + u < last) {
          const uint32_t d = smem_u32(&sm.p[put][q][u][threadIdx.x]);
          const void* g = src[q] + u * st[q];
          if (sizeof(Piece) == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d), "l"(g) : "memory");
          else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d), "l"(g) : "memory");
        }
      if (ASYNC) src[q] += GROUP * st[q];
    }
    if (ASYNC) {
      cp_async_commit();
      next += GROUP;
      put = put + 1 == STAGES ? 0 : put + 1;
    }
  }
  __device__ __forceinline__ void start() {
#pragma unroll
    for (int s = 0; s + 1 < STAGES; ++s) fetch();
  }
  __device__ __forceinline__ void take(Piece (&r)[TENSORS][GROUP]) {
    if (ASYNC) {
      fetch();
      cp_async_wait<STAGES - 1>();
#pragma unroll
      for (int q = 0; q < TENSORS; ++q)
#pragma unroll
        for (int u = 0; u < GROUP; ++u) r[q][u] = sm.p[get][q][u][threadIdx.x];
      get = get + 1 == STAGES ? 0 : get + 1;
    } else {
#pragma unroll
      for (int q = 0; q < TENSORS; ++q) {
#pragma unroll
        for (int u = 0; u < GROUP; ++u)
          if (next + u < last) r[q][u] = *reinterpret_cast<const Piece*>(src[q] + u * st[q]);
        src[q] += GROUP * st[q];
      }
      next += GROUP;
    }
  }
};

// Whether a sequence starts (or ends, with `ends`) among GROUP tokens from t (a multiple of 4;
// entries past the row's end may say yes).
template <int GROUP>
__device__ __forceinline__ bool conv_marks(const SeqMap& m, int t, bool ends) {
  if (!m.start) return t == 0 || (ends && t + GROUP >= m.T);
  bool any = false;
#pragma unroll
  for (int k = 0; k < GROUP; k += 4) {
    if (t + k >= m.T) break;
    const int4 f = __ldg(reinterpret_cast<const int4*>(m.start + t + k));
    any |= (f.x & f.y & f.z & f.w) >= 0;
    if (ends) {
      const int4 l = __ldg(reinterpret_cast<const int4*>(m.end + t + k));
      any |= (l.x & l.y & l.z & l.w) >= 0;
    }
  }
  return any;
}

template <typename T, int V, bool FULL>
__global__ void __launch_bounds__(CONV_THREADS, 4) ssm_conv_fwd_kernel(ConvParams P) {
  using Ring = ConvRing<T, V, 1, CONV_GROUP>;
  const ConvItem it = conv_item<V>(P);
  if (!it.ok) return;
  Lane<V> w[4], bias = Lane<V>::all(0.f), win[3];
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = bias;
  conv_taps<V>(P, it.c0, w, bias);
  conv_window<T, V>(P, it.b, it.t0, it.c0, win);
  T* y = static_cast<T*>(P.y) + ((long long)it.b * P.T + it.t0) * P.C + it.c0;
  __shared__ typename Ring::Smem ring_sm;
  Ring ring(ring_sm, it.t0, it.t1);
  ring.src[0] = row_ptr<T>(P.x, it.b, it.t0) + it.c0;
  ring.st[0] = P.x.st;
  ring.start();
  // EDGE: tokens past the run, or starts and ends of sequences among the group's
  auto group = [&](int t, auto edge) {
    constexpr bool EDGE = decltype(edge)::value;
    IoVec<T, V> raw[1][CONV_GROUP];
    ring.take(raw);
#pragma unroll
    for (int u = 0; u < CONV_GROUP; ++u) {
      if (EDGE && t + u >= it.t1) break;
      if (EDGE) {
        const int q = seq_start_at(P.seq, it.b, t + u);
        if (q >= 0) conv_enter<V>(P, q, it.c0, win);
      }
      const Lane<V> v = lane_from(raw[0][u]);
      Lane<V> c = conv_point<V, FULL>(P.W, w, bias, win, v);
      if (P.silu) c = c * lane_sigmoid(c);
      lane_store(y + (long long)u * P.C, c);
      conv_push<V>(win, v);
      if (EDGE && P.ht) {
        const int e = seq_end_at(P.seq, it.b, t + u);
        if (e >= 0) {
#pragma unroll
          for (int s = 0; s < 3; ++s)
#pragma unroll
            for (int i = 0; i < V; ++i)
              if (s >= 4 - P.W) P.ht[((long long)e * P.C + it.c0 + i) * (P.W - 1) + s - (4 - P.W)] = win[s].get(i);
        }
      }
    }
    y += (long long)CONV_GROUP * P.C;
  };
#pragma unroll 1
  for (int t = it.t0; t < it.t1; t += CONV_GROUP) {
    if (t + CONV_GROUP > it.t1 || conv_marks<CONV_GROUP>(P.seq, t, P.ht != nullptr)) group(t, std::true_type{});
    else group(t, std::false_type{});
  }
}

// A pending dx leaves three tokens after its own, when the last tap that reads
// its input has been seen.  Slots of positions before a sequence's first token
// leave into its initial state's gradient.
template <typename T, int V>
__device__ __forceinline__ void conv_emit(const ConvParams& P, const ConvItem& it, int pos, int first, int seq,
                                          const Lane<V>& v) {
  if (pos >= first) {
    if (pos >= it.t0 && pos < it.t1)
      lane_store(static_cast<T*>(P.dx) + ((long long)it.b * P.T + pos) * P.C + it.c0, v);
  } else if (P.dh0 && first >= it.t0 && first < it.t1) {
    const int s = pos - (first - 3) - (4 - P.W);  // slot of the W-1 inputs before `first`
    if (s >= 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) P.dh0[((long long)seq * P.C + it.c0 + i) * (P.W - 1) + s] = v.get(i);
    }
  }
}

template <typename T, int V, bool FULL>
__global__ void __launch_bounds__(CONV_THREADS, 2) ssm_conv_bwd_kernel(ConvParams P) {
  using Ring = ConvRing<T, V, 2, CONV_BWD_GROUP>;
  const ConvItem it = conv_item<V>(P);
  if (!it.ok) return;
  const Lane<V> zero = Lane<V>::all(0.f);
  Lane<V> w[4], bias = zero, win[3], pend[3] = {zero, zero, zero}, dw[5] = {zero, zero, zero, zero, zero};
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = zero;
  conv_taps<V>(P, it.c0, w, bias);
  conv_window<T, V>(P, it.b, it.t0, it.c0, win);
  // first token of the current sequence; before the run only its being at most t0 - 3 or
  // the run's own start matter, as slots before t0 belong to the run in front
  int first = it.t0 - 3, seq = -1;
  const int stop = min(it.t1 + 3, P.T);
  __shared__ typename Ring::Smem ring_sm;
  Ring ring(ring_sm, it.t0, stop);
  ring.src[0] = row_ptr<T>(P.x, it.b, it.t0) + it.c0;
  ring.src[1] = row_ptr<T>(P.dy, it.b, it.t0) + it.c0;
  ring.st[0] = P.x.st;
  ring.st[1] = P.dy.st;
  ring.start();
  T* dxr = static_cast<T*>(P.dx) + ((long long)it.b * P.T + it.t0 - 3) * P.C + it.c0;
  int t = it.t0;
  bool done = false;  // a sequence that starts behind the run ends it
  // EDGE: the first and last groups of the run (their dx are not all the run's), and groups with
  // starts or ends of sequences
  auto group = [&](int tg, auto edge) {
    constexpr bool EDGE = decltype(edge)::value;
    IoVec<T, V> raw[2][CONV_BWD_GROUP];
    ring.take(raw);
#pragma unroll
    for (int u = 0; u < CONV_BWD_GROUP; ++u) {
      if (EDGE && tg + u >= stop) break;
      t = tg + u;
      if (EDGE) {
        const int q = seq_start_at(P.seq, it.b, t);
        if (q >= 0) {
          if (t > it.t0) {  // the sequence in front ends: its pending slots are complete
#pragma unroll
            for (int s = 0; s < 3; ++s) conv_emit<T, V>(P, it, t - 3 + s, first, seq, pend[s]);
          }
          if (t >= it.t1) {
            done = true;
            return;
          }
          conv_enter<V>(P, q, it.c0, win);
          first = t;
          seq = q;
          pend[0] = pend[1] = pend[2] = zero;
        }
      }
      const Lane<V> x = lane_from(raw[0][u]);
      Lane<V> dc = lane_from(raw[1][u]);
      if (P.silu) {
        const Lane<V> c = conv_point<V, FULL>(P.W, w, bias, win, x), p = lane_sigmoid(c), one = Lane<V>::all(1.f);
        dc = dc * p * fma(c, fma(p, Lane<V>::all(-1.f), one), one);
      }
      if (!EDGE || t < it.t1) {
        dw[0] = fma(dc, win[0], dw[0]);
        dw[1] = fma(dc, win[1], dw[1]);
        dw[2] = fma(dc, win[2], dw[2]);
        dw[3] = fma(dc, x, dw[3]);
        dw[4] = dw[4] + dc;
      }
      const Lane<V> out = FULL || P.W > 3 ? fma(w[0], dc, pend[0]) : pend[0];
      pend[0] = FULL || P.W > 2 ? fma(w[1], dc, pend[1]) : pend[1];
      pend[1] = FULL || P.W > 1 ? fma(w[2], dc, pend[2]) : pend[2];
      pend[2] = w[3] * dc;
      if (EDGE) conv_emit<T, V>(P, it, t - 3, first, seq, out);
      else lane_store(dxr + (long long)u * P.C, out);
      conv_push<V>(win, x);
      if (EDGE && P.dht) {
        const int e = seq_end_at(P.seq, it.b, t);
        if (e >= 0) {
#pragma unroll
          for (int s = 0; s < 3; ++s)
#pragma unroll
            for (int i = 0; i < V; ++i)
              if (s >= 4 - P.W)
                pend[s].set(i, pend[s].get(i) + __ldg(P.dht + ((long long)e * P.C + it.c0 + i) * (P.W - 1) + s - (4 - P.W)));
        }
      }
    }
  };
#pragma unroll 1
  for (int tg = it.t0; tg < stop && !done; tg += CONV_BWD_GROUP) {
    // (the slots t - 3 of an inner group are tokens of the run and of the current sequence)
    const bool inner = tg - 3 >= it.t0 && tg - 3 >= first && tg + CONV_BWD_GROUP <= it.t1;
    if (!inner || conv_marks<CONV_BWD_GROUP>(P.seq, tg, P.dht != nullptr)) group(tg, std::true_type{});
    else group(tg, std::false_type{});
    dxr += (long long)CONV_BWD_GROUP * P.C;
  }
  if (ConvRing<T, V, 2, CONV_BWD_GROUP>::ASYNC) cp_async_wait<0>();
  if (!done) t = stop;
  if (t == P.T) {  // the row's end completes what is pending
#pragma unroll
    for (int s = 0; s < 3; ++s) conv_emit<T, V>(P, it, t - 3 + s, first, seq, pend[s]);
  }
  float* part = P.partial + (it.run * P.C + it.c0) * (P.W + 1);
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int k = 0; k < 5; ++k)
      if (k >= 4 - P.W) part[i * (P.W + 1) + k - (4 - P.W)] = dw[k].get(i);
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
