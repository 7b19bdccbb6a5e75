// C ABI of the state-space operators and of gradient clipping (declared in
// include/kda_b200.h): argument checks, buffer carving and kernel launches.
// No allocation, no host sync.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <string>

#include "../../include/kda_b200.h"
#include "grad_clip.cuh"
#include "kda_host.h"
#include "ssm_conv.cuh"
#include "ssm_scan_launch.cuh"

using namespace kda;

namespace {

size_t io_size(int dtype) { return dtype == KDA_IO_F32 ? 4 : 2; }

int check_dtype(int dtype) {
  if (dtype < KDA_IO_F32 || dtype > KDA_IO_F16)
    return fail(KDA_ERR_INVALID, "dtype must be KDA_IO_F32, KDA_IO_BF16 or KDA_IO_F16");
  return KDA_OK;
}

// Sequences of a call: B rows of T tokens, or (cu) one row of N packed ones.
int check_rows(long long B, long long T, int N, const int32_t* cu) {
  if (B < 1 || T < 0 || N < 1) return fail(KDA_ERR_INVALID, "B >= 1, T >= 0 and N >= 1 are required");
  if (cu && B != 1)
    return fail(KDA_ERR_INVALID, "The batch size is expected to be 1 rather than " + std::to_string(B) +
                                     " when using `cu_seqlens`.");
  if (!cu && N != B) return fail(KDA_ERR_INVALID, "N must equal B without cu_seqlens");
  if (B > 65535) return fail(KDA_ERR_UNSUPPORTED, "more than 65535 rows");
  if (T > INT32_MAX / 2) return fail(KDA_ERR_UNSUPPORTED, "too many tokens");
  return KDA_OK;
}

bool vec_rows(const void* p, long long sb, long long st, long long B, long long T, int elems, size_t esz) {
  return aligned(p, (size_t)elems * esz) && (B <= 1 || sb % elems == 0) && (T <= 1 || st % elems == 0);
}

size_t map_bytes(long long T, bool packed) { return packed ? 2 * align256((size_t)std::max(T, 1LL) * 4) : 0; }

// Sequence maps of a packed call, and the rows of empty sequences (dst <- src).
int build_map(SeqMap& m, Carver& cv, const int32_t* cu, int T, int N, const float* src, float* dst, long long per,
              cudaStream_t st) {
  m.start = m.end = nullptr;
  m.T = T;
  if (!cu) return KDA_OK;
  int* err = device_error_flag();
  if (!err) return fail(KDA_ERR_CUDA, "the device error flag has no address");
  int* start = cv.take<int>((size_t)T * 4);
  int* end = cv.take<int>((size_t)T * 4);
  SeqMapParams p{cu, N, T, start, end, src, dst, per, err};
  const int blocks = (T + SEQ_MAP_THREADS - 1) / SEQ_MAP_THREADS + std::min(N, 2 * sm_count());
  {
    TimedLaunch tl(K_TABLE, st);
    ssm_seq_map_kernel<<<blocks, SEQ_MAP_THREADS, 0, st>>>(p);
  }
  m.start = start;
  m.end = end;
  return launch_check("sequence map");
}

// T = 0: every sequence is empty, its state goes through.
int pass_state(const float* src, float* dst, long long elems, cudaStream_t st) {
  if (!dst || elems == 0) return KDA_OK;
  const cudaError_t e = src ? cudaMemcpyAsync(dst, src, (size_t)elems * 4, cudaMemcpyDeviceToDevice, st)
                            : cudaMemsetAsync(dst, 0, (size_t)elems * 4, st);
  return e == cudaSuccess ? KDA_OK : fail(KDA_ERR_CUDA, cudaGetErrorString(e));
}
int zero_floats(float* p, long long elems, cudaStream_t st) { return pass_state(nullptr, p, elems, st); }

// ---- convolution

int check_conv(const void* x, const float* w, long long B, long long T, int C, int W, int N, const int32_t* cu, int dtype) {
  int rc;
  if ((rc = check_dtype(dtype))) return rc;
  if ((rc = check_rows(B, T, N, cu))) return rc;
  if (W < 1 || W > 4) return fail(KDA_ERR_UNSUPPORTED, "the convolution has 1 to 4 taps, got " + std::to_string(W));
  if (C < 1) return fail(KDA_ERR_INVALID, "C >= 1 is required");
  if (!w || (!x && B * T > 0)) return fail(KDA_ERR_INVALID, "null input pointer");
  return KDA_OK;
}

constexpr int CONV_V = 2;  // channels per thread

// Tokens per thread: the longest run up to `longest` that leaves `threads` threads per SM (8 tokens at least).
// Long runs read the halo of three tokens and, backward, write partial sums of dw less often; short ones make
// enough threads for narrow or short problems.  Measured, us, forward with 512 threads and runs up to 64 against
// 1024 threads: [1, 2048, 2048] bf16 8.3 and 10.3, [4, 4096, 2048] 36 and 36 (runs up to 128: 38.5).  Backward
// and its sums with 256 threads and runs up to 256 against 1024 and 64: 17 and 37, 66 and 79.
int conv_run(long long B, long long T, long long lanes, int threads, int longest) {
  const long long want = (long long)threads * sm_count();
  for (int run = longest; run > 8; run >>= 1)
    if (B * ((T + run - 1) / run) * lanes >= want) return run;
  return 8;
}

template <typename T, int V>
int launch_conv_fwd(ConvParams& p, cudaStream_t st) {
  const long long lanes = p.C / V;
  p.run = conv_run(p.B, p.T, lanes, 512, 64);
  p.runs = (p.T + p.run - 1) / p.run;
  const long long blocks = ((long long)p.B * p.runs * lanes + CONV_THREADS - 1) / CONV_THREADS;
  if (blocks > INT32_MAX) return fail(KDA_ERR_UNSUPPORTED, "too many elements");
  {
    TimedLaunch tl(K_CONV_FWD, st);
    if (p.W == 4) ssm_conv_fwd_kernel<T, V, true><<<(unsigned)blocks, CONV_THREADS, 0, st>>>(p);
    else ssm_conv_fwd_kernel<T, V, false><<<(unsigned)blocks, CONV_THREADS, 0, st>>>(p);
  }
  return launch_check("short conv forward");
}

template <typename T>
int conv_fwd(ConvParams& p, cudaStream_t st) {
  constexpr int V = CONV_V;
  const bool vec = p.C % V == 0 && aligned(p.y, V * sizeof(T)) && vec_rows(p.x.p, p.x.sb, p.x.st, p.B, p.T, V, sizeof(T));
  return vec ? launch_conv_fwd<T, V>(p, st) : launch_conv_fwd<T, 1>(p, st);
}

template <typename T, int V>
int launch_conv_bwd(ConvParams& p, float* dw, float* dbias, cudaStream_t st) {
  const long long blocks = ((long long)p.B * p.runs * (p.C / V) + CONV_THREADS - 1) / CONV_THREADS;
  if (blocks > INT32_MAX) return fail(KDA_ERR_UNSUPPORTED, "too many elements");
  const long long cols = (long long)p.C * (p.W + 1);
  {
    TimedLaunch tl(K_CONV_BWD, st);
    if (p.W == 4) ssm_conv_bwd_kernel<T, V, true><<<(unsigned)blocks, CONV_THREADS, 0, st>>>(p);
    else ssm_conv_bwd_kernel<T, V, false><<<(unsigned)blocks, CONV_THREADS, 0, st>>>(p);
    ssm_reduce_kernel<<<(unsigned)((cols + SSM_REDUCE_COLS - 1) / SSM_REDUCE_COLS), SSM_REDUCE_COLS * SSM_REDUCE_SLICES,
                        0, st>>>(p.partial, (long long)p.B * p.runs, cols, p.W, p.W + 1, dw, dbias, nullptr);
  }
  return launch_check("short conv backward");
}

int conv_bwd_run(long long B, long long T, int C) { return conv_run(B, T, (C + CONV_V - 1) / CONV_V, 256, 256); }

template <typename T>
int conv_bwd(ConvParams& p, float* dw, float* dbias, cudaStream_t st) {
  constexpr int V = CONV_V;
  const bool vec = p.C % V == 0 && aligned(p.dx, V * sizeof(T)) &&
                   vec_rows(p.x.p, p.x.sb, p.x.st, p.B, p.T, V, sizeof(T)) &&
                   vec_rows(p.dy.p, p.dy.sb, p.dy.st, p.B, p.T, V, sizeof(T));
  return vec ? launch_conv_bwd<T, V>(p, dw, dbias, st) : launch_conv_bwd<T, 1>(p, dw, dbias, st);
}

template <typename T>
int conv_step(const ConvStepParams& p, cudaStream_t st) {
  const int gx = (p.C + CONV_THREADS - 1) / CONV_THREADS;
  const int gy = std::max(1, std::min(p.rows, (16 * sm_count() + gx - 1) / gx));
  {
    TimedLaunch tl(K_CONV_STEP, st);
    ssm_conv_step_kernel<T><<<dim3(gx, gy), CONV_THREADS, 0, st>>>(p);
  }
  return launch_check("short conv step");
}

// ---- scan

constexpr int SCAN_MAX_N = 64;

int check_scan(const kda_b200_scan_args* a, bool step) {
  int rc;
  if (!a) return fail(KDA_ERR_INVALID, "null arguments");
  if ((rc = check_dtype(a->dtype))) return rc;
  if (a->E < 1 || a->N < 1 || a->G < 1) return fail(KDA_ERR_INVALID, "E, N and G must be >= 1");
  if (a->E % a->G) return fail(KDA_ERR_INVALID, "the groups must divide the channels");
  if (a->N > SCAN_MAX_N) return fail(KDA_ERR_UNSUPPORTED, "more than 64 states per channel");
  if (step) {
    if ((long long)a->E * a->N > INT32_MAX) return fail(KDA_ERR_UNSUPPORTED, "too many channels");
    if (a->rows < 0 || a->pool < 0) return fail(KDA_ERR_INVALID, "rows >= 0 and pool >= 0 are required");
    if (!a->slots && a->rows > a->pool) return fail(KDA_ERR_INVALID, "more rows than states");
    if (a->rows > 0 && (!a->x || !a->dt || !a->A || !a->B_ || !a->C_ || !a->state || !a->y))
      return fail(KDA_ERR_INVALID, "null pointer");
    return KDA_OK;
  }
  if ((rc = check_rows(a->B, a->T, a->nseq, a->cu_seqlens))) return rc;
  if (!a->A) return fail(KDA_ERR_INVALID, "null input pointer");
  if (a->B * a->T > 0 && (!a->x || !a->dt || !a->B_ || !a->C_)) return fail(KDA_ERR_INVALID, "null input pointer");
  if ((long long)a->G * ((a->E / a->G + 15) / 16) > INT32_MAX / 4) return fail(KDA_ERR_UNSUPPORTED, "too many channels");
  return KDA_OK;
}

ScanParams scan_params(const kda_b200_scan_args* a) {
  ScanParams p{};
  p.x = {a->x, a->x_sb, a->x_st};
  p.dt = {a->dt, a->dt_sb, a->dt_st};
  p.z = {a->z, a->z_sb, a->z_st};
  p.Bm = a->B_; p.b_sb = a->B_sb; p.b_st = a->B_st; p.b_sg = a->B_sg;
  p.Cm = a->C_; p.c_sb = a->C_sb; p.c_st = a->C_st; p.c_sg = a->C_sg;
  p.A = a->A; p.D = a->D; p.dt_bias = a->dt_bias; p.h0 = a->h0;
  p.B = (int)a->B; p.T = (int)a->T; p.E = a->E; p.N = a->N; p.G = a->G;
  p.softplus = a->softplus != 0;
  const size_t esz = io_size(a->dtype);
  const int V = (int)(16 / esz);
  p.vec = a->E % V == 0 && (a->G == 1 || (a->E / a->G) % V == 0) &&
          vec_rows(a->x, a->x_sb, a->x_st, a->B, a->T, V, esz) && vec_rows(a->dt, a->dt_sb, a->dt_st, a->B, a->T, V, esz) &&
          (!a->z || vec_rows(a->z, a->z_sb, a->z_st, a->B, a->T, V, esz));
  const int VB = std::min(V, a->N);  // elements of a piece of B and C
  p.vec_bc = (a->N % V == 0 || a->N == 4) && vec_rows(a->B_, a->B_sb, a->B_st, a->B, a->T, VB, esz) &&
             vec_rows(a->C_, a->C_sb, a->C_st, a->B, a->T, VB, esz) &&
             (a->G == 1 || (a->B_sg % VB == 0 && a->C_sg % VB == 0));
  return p;
}

// The spans, and the room of their carries.
void cut_scan(ScanParams& p, Carver& cv, int dtype, bool backward) {
  const ScanCut cut = scan_cut(p.B, p.T, p.E, p.N, p.G, dtype != KDA_IO_F32, p.vec, backward);
  p.span = cut.span;
  p.spans = cut.spans(p.T);
  p.tile = cut.tile;
  p.carry = p.spans > 1 ? cv.take<float2>(scan_carry_bytes(p.B, p.spans, p.E, p.N)) : nullptr;
}

template <typename T, int LP, int Q>
int launch_scan_step(const ScanStepParams& p, cudaStream_t st) {
  const long long gx = ((long long)p.E * LP + STEP_THREADS - 1) / STEP_THREADS;
  const int gy = (int)std::max(1LL, std::min((long long)p.rows, (8LL * sm_count() + gx - 1) / gx));
  const size_t piece = 4 * sizeof(T);
  auto fours = [&](const void* q, long long sb, long long sg) {
    return aligned(q, piece) && (p.rows == 1 || sb % 4 == 0) && (p.G == 1 || sg % 4 == 0);
  };
  const bool vec = p.N % 4 == 0 && aligned(p.state, 16) && fours(p.Bm, p.b_sb, p.b_sg) && fours(p.Cm, p.c_sb, p.c_sg);
  {
    TimedLaunch tl(K_SCAN_STEP, st);
    if (vec) ssm_scan_step_kernel<T, LP, Q, true><<<dim3((unsigned)gx, gy), STEP_THREADS, 0, st>>>(p);
    else ssm_scan_step_kernel<T, LP, Q, false><<<dim3((unsigned)gx, gy), STEP_THREADS, 0, st>>>(p);
  }
  return launch_check("scan step");
}

template <typename T>
int scan_step(const ScanStepParams& p, cudaStream_t st) {
  const int quads = (p.N + 3) / 4;
  if (quads <= 1) return launch_scan_step<T, 1, 1>(p, st);
  if (quads <= 2) return launch_scan_step<T, 1, 2>(p, st);
  if (quads <= 4) return launch_scan_step<T, 2, 2>(p, st);
  if (quads <= 8) return launch_scan_step<T, 4, 2>(p, st);
  return launch_scan_step<T, 8, 2>(p, st);
}

// ---- gradient clipping

int grad_ctas() { return 16 * sm_count(); }

template <int M>
int grad_table(GradTable<M>& t, const kda_b200_grad_args* a, long long first, int n) {
  t.n = n;
  long long chunks = 0;
  for (int i = 0; i < n; ++i) {
    const long long k = first + i;
    t.in[i] = reinterpret_cast<const void*>(a->in[k]);
    t.out[i] = a->out ? reinterpret_cast<void*>(a->out[k]) : nullptr;
    t.numel[i] = a->numel[k];
    t.tin[i] = a->in_type[k];
    t.tout[i] = a->out ? a->out_type[k] : 0;
    t.chunk0[i] = (int)chunks;
    chunks += (a->numel[k] + GRAD_CHUNK - 1) / GRAD_CHUNK;
    if (chunks > INT32_MAX / 2) return fail(KDA_ERR_UNSUPPORTED, "too many gradient elements in one call");
  }
  t.chunk0[n] = (int)chunks;
  return KDA_OK;
}

template <int M>
int grad_run(const kda_b200_grad_args* a, double* partial, int parts, float* norm, bool scale, cudaStream_t st) {
  GradTable<M> t;
  const int ctas = grad_ctas();
  int launch = 0;
  for (long long first = 0; first < a->count; first += M, ++launch) {
    const int n = (int)std::min<long long>(M, a->count - first);
    int rc = grad_table(t, a, first, n);
    if (rc) return rc;
    if (scale) {
      const int grid = std::max(1, std::min(ctas, t.chunk0[n]));
      TimedLaunch tl(K_GRAD_SCALE, st);
      grad_scale_kernel<M><<<grid, GRAD_THREADS, 0, st>>>(t, partial, parts, a->max_norm, a->eps, norm);
    } else {
      TimedLaunch tl(K_GRAD_NORM, st);
      grad_norm_kernel<M><<<ctas, GRAD_THREADS, 0, st>>>(t, partial + (long long)launch * ctas);
    }
    if ((rc = launch_check(scale ? "gradient scaling" : "gradient norm"))) return rc;
  }
  return KDA_OK;
}

long long grad_launches(long long count) {
  return count <= GRAD_FEW_TENSORS ? 1 : (count + GRAD_MAX_TENSORS - 1) / GRAD_MAX_TENSORS;
}

}  // namespace

#define SSM_DISPATCH(dtype, fn, ...)                              \
  ((dtype) == KDA_IO_F32    ? fn<float>(__VA_ARGS__)              \
   : (dtype) == KDA_IO_BF16 ? fn<bf16>(__VA_ARGS__)               \
                            : fn<f16>(__VA_ARGS__))

extern "C" {

size_t kda_b200_short_conv_workspace_bytes(int64_t B, int64_t T, int C, int W, int packed, int backward) {
  if (B < 1 || T < 0 || C < 1 || W < 1 || W > 4) return 0;
  size_t b = map_bytes(T, packed != 0);
  if (backward) {
    const int run = conv_bwd_run(B, T, C);
    b += align256((size_t)B * ((T + run - 1) / run) * C * (W + 1) * 4);
  }
  return std::max<size_t>(b, 16);
}

int kda_b200_short_conv_fwd(const void* x, int64_t x_sb, int64_t x_st, const float* w, const float* bias,
                            const float* h0, const int32_t* cu_seqlens, int64_t B, int64_t T, int C, int W, int N,
                            int dtype, int silu, void* y, float* ht, void* workspace, size_t workspace_bytes,
                            void* stream) {
  int rc = check_conv(x, w, B, T, C, W, N, cu_seqlens, dtype);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) return pass_state(h0, ht, (long long)N * C * (W - 1), st);
  if (!y) return fail(KDA_ERR_INVALID, "null output pointer");
  if (!workspace || workspace_bytes < kda_b200_short_conv_workspace_bytes(B, T, C, W, cu_seqlens != nullptr, 0) ||
      !aligned(workspace, 16))
    return fail(KDA_ERR_INVALID, "workspace too small: kda_b200_short_conv_workspace_bytes() bytes are needed");
  ConvParams p{};
  p.x = {x, x_sb, x_st};
  p.w = w; p.bias = bias; p.h0 = h0;
  p.B = (int)B; p.T = (int)T; p.C = C; p.W = W;
  p.silu = silu != 0;
  p.y = y; p.ht = W > 1 ? ht : nullptr;
  Carver cv(workspace);
  if ((rc = build_map(p.seq, cv, cu_seqlens, p.T, N, h0, p.ht, (long long)C * (W - 1), st))) return rc;
  return SSM_DISPATCH(dtype, conv_fwd, p, st);
}

int kda_b200_short_conv_bwd(const void* x, int64_t x_sb, int64_t x_st, const float* w, const float* bias,
                            const float* h0, const int32_t* cu_seqlens, int64_t B, int64_t T, int C, int W, int N,
                            int dtype, int silu, const void* dy, int64_t dy_sb, int64_t dy_st, const float* dht,
                            void* dx, float* dw, float* dbias, float* dh0, void* workspace, size_t workspace_bytes,
                            void* stream) {
  int rc = check_conv(x, w, B, T, C, W, N, cu_seqlens, dtype);
  if (rc) return rc;
  if (!dw) return fail(KDA_ERR_INVALID, "null gradient pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {
    if ((rc = zero_floats(dw, (long long)C * W, st)) || (rc = zero_floats(dbias, C, st))) return rc;
    return pass_state(dht, dh0, (long long)N * C * (W - 1), st);
  }
  if (!dy || !dx) return fail(KDA_ERR_INVALID, "null gradient pointer");
  if (!workspace || workspace_bytes < kda_b200_short_conv_workspace_bytes(B, T, C, W, cu_seqlens != nullptr, 1) ||
      !aligned(workspace, 16))
    return fail(KDA_ERR_INVALID, "workspace too small: kda_b200_short_conv_workspace_bytes() bytes are needed");
  ConvParams p{};
  p.x = {x, x_sb, x_st};
  p.dy = {dy, dy_sb, dy_st};
  p.w = w; p.bias = bias; p.h0 = h0;
  p.B = (int)B; p.T = (int)T; p.C = C; p.W = W;
  p.silu = silu != 0;
  p.dht = W > 1 ? dht : nullptr; p.dx = dx; p.dh0 = W > 1 ? dh0 : nullptr;
  p.run = conv_bwd_run(B, T, C);
  p.runs = (p.T + p.run - 1) / p.run;
  Carver cv(workspace);
  if ((rc = build_map(p.seq, cv, cu_seqlens, p.T, N, dht, p.dh0, (long long)C * (W - 1), st))) return rc;
  p.partial = cv.take<float>((size_t)B * p.runs * C * (W + 1) * 4);
  return SSM_DISPATCH(dtype, conv_bwd, p, dw, dbias, st);
}

int kda_b200_short_conv_step(const void* x, int64_t x_sr, const float* w, const float* bias, float* state,
                             const int32_t* slots, int rows, int C, int W, int pool, int dtype, int silu, void* y,
                             void* stream) {
  int rc = check_dtype(dtype);
  if (rc) return rc;
  if (W < 1 || W > 4) return fail(KDA_ERR_UNSUPPORTED, "the convolution has 1 to 4 taps, got " + std::to_string(W));
  if (rows < 0 || C < 1 || pool < 0) return fail(KDA_ERR_INVALID, "rows >= 0, C >= 1 and pool >= 0 are required");
  if (!slots && rows > pool) return fail(KDA_ERR_INVALID, "more rows than states");
  if (rows == 0) return KDA_OK;
  if (!x || !w || !y || (!state && W > 1)) return fail(KDA_ERR_INVALID, "null pointer");
  int* err = device_error_flag();
  if (!err) return fail(KDA_ERR_CUDA, "the device error flag has no address");
  ConvStepParams p{x, x_sr, w, bias, state, slots, rows, C, W, pool, silu != 0, y, err};
  return SSM_DISPATCH(dtype, conv_step, p, static_cast<cudaStream_t>(stream));
}

int kda_b200_put_states(const float* src, const int32_t* slots, int rows, int64_t per, int pool, float* dst, void* stream) {
  if (rows < 0 || per < 0 || pool < 0) return fail(KDA_ERR_INVALID, "rows >= 0, per >= 0 and pool >= 0 are required");
  if (rows == 0 || per == 0) return KDA_OK;
  if (!src || !slots || (!dst && pool > 0)) return fail(KDA_ERR_INVALID, "null pointer");
  int* err = device_error_flag();
  if (!err) return fail(KDA_ERR_CUDA, "the device error flag has no address");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool vec = per % 4 == 0 && aligned(src, 16) && aligned(dst, 16);
  const long long elems = vec ? per / 4 : per;
  const dim3 grid((unsigned)std::min<long long>((elems + 255) / 256, 1024), std::min(rows, 65535));
  if (vec)
    ssm_put_states_kernel<<<grid, 256, 0, st>>>(reinterpret_cast<const float4*>(src), slots, rows, elems, pool,
                                                reinterpret_cast<float4*>(dst), err);
  else
    ssm_put_states_kernel<<<grid, 256, 0, st>>>(src, slots, rows, elems, pool, dst, err);
  return launch_check("states to their slots");
}

size_t kda_b200_scan_saved_bytes(int64_t B, int64_t T, int E, int N, int G) {
  if (B < 1 || T < 0 || E < 1 || N < 1 || N > SCAN_MAX_N || G < 1 || E % G) return 0;
  return std::max<size_t>(16, (size_t)B * ((T + SCAN_SEG - 1) / SCAN_SEG) * E * N * 4);
}

size_t kda_b200_scan_workspace_bytes(int64_t B, int64_t T, int E, int N, int G, int packed, int backward) {
  if (B < 1 || T < 0 || E < 1 || N < 1 || N > SCAN_MAX_N || G < 1 || E % G) return 0;
  size_t b = map_bytes(T, packed != 0);
  const int spans = T ? scan_most_spans(B, T, E, N, G, backward != 0) : 0;
  b += align256(scan_carry_bytes(B, spans, E, N));
  if (backward)
    b += align256((size_t)scan_part_floats(B, T, E, N, G) * 4) + align256((size_t)B * spans * E * (N + 2) * 4);
  return std::max<size_t>(b, 16);
}

int kda_b200_selective_scan_fwd(const kda_b200_scan_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_scan(a, false);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->T == 0) return pass_state(a->h0, a->ht, (long long)a->nseq * a->E * a->N, st);
  if (!a->y) return fail(KDA_ERR_INVALID, "null output pointer");
  if (!workspace || !aligned(workspace, 16) ||
      workspace_bytes < kda_b200_scan_workspace_bytes(a->B, a->T, a->E, a->N, a->G, a->cu_seqlens != nullptr, 0))
    return fail(KDA_ERR_INVALID, "workspace too small: kda_b200_scan_workspace_bytes() bytes are needed");
  if (a->saved && (!aligned(a->saved, 16) || a->saved_bytes < kda_b200_scan_saved_bytes(a->B, a->T, a->E, a->N, a->G)))
    return fail(KDA_ERR_INVALID, "saved buffer too small: kda_b200_scan_saved_bytes() bytes are needed");
  ScanParams p = scan_params(a);
  p.y = a->y;
  p.ht = a->ht;
  p.ckpt = static_cast<float*>(a->saved);
  p.vec = p.vec && aligned(a->y, 16);
  Carver cv(workspace);
  if ((rc = build_map(p.seq, cv, a->cu_seqlens, p.T, a->nseq, a->h0, a->ht, (long long)a->E * a->N, st))) return rc;
  cut_scan(p, cv, a->dtype, false);
  return SSM_DISPATCH(a->dtype, scan_fwd, p, st);
}

int kda_b200_selective_scan_bwd(const kda_b200_scan_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_scan(a, false);
  if (rc) return rc;
  if (!a->dA) return fail(KDA_ERR_INVALID, "null gradient pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->T == 0) {
    if ((rc = zero_floats(a->dA, (long long)a->E * a->N, st)) || (rc = zero_floats(a->dD, a->E, st)) ||
        (rc = zero_floats(a->ddt_bias, a->E, st)))
      return rc;
    return pass_state(a->dht, a->dh0, (long long)a->nseq * a->E * a->N, st);
  }
  if (!a->dy || !a->dx || !a->ddt || !a->dB || !a->dC || (a->z && !a->dz))
    return fail(KDA_ERR_INVALID, "null gradient pointer");
  if (!a->saved || !aligned(a->saved, 16) || a->saved_bytes < kda_b200_scan_saved_bytes(a->B, a->T, a->E, a->N, a->G))
    return fail(KDA_ERR_INVALID, "saved buffer missing or too small");
  if (!workspace || !aligned(workspace, 16) ||
      workspace_bytes < kda_b200_scan_workspace_bytes(a->B, a->T, a->E, a->N, a->G, a->cu_seqlens != nullptr, 1))
    return fail(KDA_ERR_INVALID, "workspace too small: kda_b200_scan_workspace_bytes() bytes are needed");
  ScanParams p = scan_params(a);
  p.dy = {a->dy, a->dy_sb, a->dy_st};
  p.ckpt = static_cast<float*>(a->saved);
  p.dht = a->dht; p.dh0 = a->dh0;
  p.dx = a->dx; p.ddt = a->ddt; p.dz = a->dz;
  const size_t esz = io_size(a->dtype);
  p.vec = p.vec && vec_rows(a->dy, a->dy_sb, a->dy_st, a->B, a->T, (int)(16 / esz), esz) && aligned(a->dx, 16) &&
          aligned(a->ddt, 16) && (!a->z || aligned(a->dz, 16));
  Carver cv(workspace);
  if ((rc = build_map(p.seq, cv, a->cu_seqlens, p.T, a->nseq, a->dht, a->dh0, (long long)a->E * a->N, st))) return rc;
  cut_scan(p, cv, a->dtype, true);
  p.bc_part = cv.take<float>((size_t)scan_part_floats(p.B, p.T, p.E, p.N, p.G) * 4);
  p.e_part = cv.take<float>((size_t)p.B * p.spans * p.E * (p.N + 2) * 4);
  const ScanGrads g{a->dA, a->dD, a->ddt_bias, a->dB, a->dC};
  return SSM_DISPATCH(a->dtype, scan_bwd, p, g, st);
}

int kda_b200_selective_scan_step(const kda_b200_scan_args* a, void* stream) {
  int rc = check_scan(a, true);
  if (rc) return rc;
  if (a->rows == 0) return KDA_OK;
  int* err = device_error_flag();
  if (!err) return fail(KDA_ERR_CUDA, "the device error flag has no address");
  ScanStepParams p{};
  p.x = a->x; p.dt = a->dt; p.z = a->z; p.Bm = a->B_; p.Cm = a->C_;
  p.sx = a->x_sb; p.sdt = a->dt_sb; p.sz = a->z_sb;
  p.b_sb = a->B_sb; p.b_sg = a->B_sg; p.c_sb = a->C_sb; p.c_sg = a->C_sg;
  p.A = a->A; p.D = a->D; p.dt_bias = a->dt_bias;
  p.state = a->state; p.slots = a->slots;
  p.rows = a->rows; p.E = a->E; p.N = a->N; p.G = a->G; p.pool = a->pool;
  p.softplus = a->softplus != 0;
  p.y = a->y; p.err = err;
  return SSM_DISPATCH(a->dtype, scan_step, p, static_cast<cudaStream_t>(stream));
}

size_t kda_b200_grad_workspace_bytes(int64_t count) {
  if (count < 0) return 0;
  return (size_t)std::max<long long>(1, grad_launches(count)) * grad_ctas() * sizeof(double);
}

int kda_b200_grad_clip(const kda_b200_grad_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (!a || a->count < 0) return fail(KDA_ERR_INVALID, "null arguments");
  if (a->count > 0 && (!a->in || !a->numel || !a->in_type || (a->out && !a->out_type)))
    return fail(KDA_ERR_INVALID, "null table pointer");
  if (!a->norm) return fail(KDA_ERR_INVALID, "null output pointer");
  for (long long i = 0; i < a->count; ++i) {
    if (a->numel[i] < 0) return fail(KDA_ERR_INVALID, "negative element count");
    if (a->in_type[i] > KDA_IO_F16 || (a->out && a->out_type[i] > KDA_IO_F16))
      return fail(KDA_ERR_INVALID, "dtype must be KDA_IO_F32, KDA_IO_BF16 or KDA_IO_F16");
    if (a->numel[i] > 0 && (!a->in[i] || (a->out && !a->out[i]))) return fail(KDA_ERR_INVALID, "null tensor pointer");
    if (a->in[i] % (a->in_type[i] == KDA_IO_F32 ? 4 : 2) ||
        (a->out && a->out[i] % (a->out_type[i] == KDA_IO_F32 ? 4 : 2)))
      return fail(KDA_ERR_INVALID, "a tensor's address is not a multiple of its element size");
  }
  if (!workspace || !aligned(workspace, 16) || workspace_bytes < kda_b200_grad_workspace_bytes(a->count))
    return fail(KDA_ERR_INVALID, "workspace too small: kda_b200_grad_workspace_bytes() bytes are needed");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->count == 0) return zero_floats(a->norm, 1, st);
  double* partial = static_cast<double*>(workspace);
  const int parts = (int)(grad_launches(a->count) * grad_ctas());
  const bool few = a->count <= GRAD_FEW_TENSORS;
  int rc = few ? grad_run<GRAD_FEW_TENSORS>(a, partial, parts, nullptr, false, st)
               : grad_run<GRAD_MAX_TENSORS>(a, partial, parts, nullptr, false, st);
  if (rc) return rc;
  if (!a->out) {
    grad_norm_finish_kernel<<<1, GRAD_THREADS, 0, st>>>(partial, parts, a->norm);
    return launch_check("gradient norm");
  }
  return few ? grad_run<GRAD_FEW_TENSORS>(a, partial, parts, a->norm, true, st)
             : grad_run<GRAD_MAX_TENSORS>(a, partial, parts, a->norm, true, st);
}

}  // extern "C"
