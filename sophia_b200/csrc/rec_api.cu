// C ABI of the gated linear recurrence (declared in include/kda_b200.h):
// argument checks, buffer carving and kernel launches.  No allocation, no host sync.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <string>

#include "../../include/kda_b200.h"
#include "gated_recurrence.cuh"
#include "kda_host.h"
#include "ssm_host.cuh"

using namespace kda;

namespace {

int rec_tokens(int dtype) { return dtype == KDA_IO_F32 ? rec_tile<float>() : rec_tile<bf16>(); }
long long rec_tiles(long long T, int dtype) { return (T + rec_tokens(dtype) - 1) / rec_tokens(dtype); }

// CTAs that share a row's tiles: as many as two CTAs per SM allow, never more than there are tiles.
int rec_cluster(long long B, long long T, int E, int dtype) {
  const long long lanes = B * ((E + REC_CH - 1) / REC_CH), tiles = rec_tiles(T, dtype), slots = (long long)REC_CTAS * sm_count();
  int c = 1;
  while (2 * c <= REC_MAX_CLUSTER && 2 * c * lanes <= slots && 2 * c <= tiles) c *= 2;
  return c;
}

int check_rec(const kda_b200_recurrence_args* a, bool step) {
  int rc;
  if (!a) return fail(KDA_ERR_INVALID, "null arguments");
  if ((rc = check_dtype(a->dtype))) return rc;
  if (a->E < 1) return fail(KDA_ERR_INVALID, "E >= 1 is required");
  if (!a->A) return fail(KDA_ERR_INVALID, "null input pointer");
  if (step) {
    if (a->rows < 0 || a->pool < 0) return fail(KDA_ERR_INVALID, "rows >= 0 and pool >= 0 are required");
    if (!a->slots && a->rows > a->pool) return fail(KDA_ERR_INVALID, "more rows than states");
    if (a->rows > 0 && (!a->x || !a->decay || !a->gate || !a->state || !a->y)) return fail(KDA_ERR_INVALID, "null pointer");
    return KDA_OK;
  }
  if ((rc = check_rows(a->B, a->T, a->nseq, a->cu_seqlens))) return rc;
  if (a->B * a->T > 0 && (!a->x || !a->decay || !a->gate)) return fail(KDA_ERR_INVALID, "null input pointer");
  if (a->E > INT32_MAX / (4 * REC_MAX_CLUSTER)) return fail(KDA_ERR_UNSUPPORTED, "too many channels");
  return KDA_OK;
}

RecParams rec_params(const kda_b200_recurrence_args* a) {
  RecParams p{};
  p.k = rec_const();
  p.x = {a->x, a->x_sb, a->x_st};
  p.decay = {a->decay, a->decay_sb, a->decay_st};
  p.gate = {a->gate, a->gate_sb, a->gate_st};
  p.z = {a->z, a->z_sb, a->z_st};
  p.A = a->A; p.decay_bias = a->decay_bias; p.gate_bias = a->gate_bias; p.h0 = a->h0;
  p.B = (int)a->B; p.T = (int)a->T; p.E = a->E;
  p.tiles = (int)rec_tiles(a->T, a->dtype);
  p.cluster = rec_cluster(a->B, a->T, a->E, a->dtype);
  p.ckpt = static_cast<float*>(a->saved);
  return p;
}

// 16-byte pieces: every row of every activation starts at a multiple of them.
bool rec_vec_ok(const RecParams& p, int dtype) {
  const size_t esz = io_size(dtype);
  const int V = (int)(16 / esz);
  auto ok = [&](const RowView& r) { return !r.p || vec_rows(r.p, r.sb, r.st, p.B, p.T, V, esz); };
  return p.E % V == 0 && ok(p.x) && ok(p.decay) && ok(p.gate) && ok(p.z) && ok(p.dy) && aligned(p.y, 16) &&
         aligned(p.dx, 16) && aligned(p.ddecay, 16) && aligned(p.dgate, 16) && aligned(p.dz, 16);
}

// The tensor maps of a call's activations: boxes of a tile's tokens x 64 channels of a row.  False where a layout has
// none (a row or token that is expanded has the stride 0): the kernels then copy by words.
bool rec_maps(RecParams& p, int dtype, bool backward) {
  const RowView fwd[4] = {p.decay, p.x, p.gate, p.z}, bwd[5] = {p.decay, p.x, p.gate, p.dy, p.z};
  const RowView* r = backward ? bwd : fwd;
  const int n = (backward ? 5 : 4) - (p.z.p ? 0 : 1);
  const size_t esz = io_size(dtype);
  for (int i = 0; i < n; ++i) {
    // (a stride that is never taken, of a single row or token, may be anything: give the encoder a legal one)
    const unsigned long long st = (p.T > 1 ? r[i].st : p.E) * esz, sb = (p.B > 1 ? r[i].sb : p.E) * esz;
    const unsigned long long dims[3] = {(unsigned long long)p.E, (unsigned long long)p.T, (unsigned long long)p.B};
    const unsigned long long strides[2] = {st, sb};
    const unsigned box[3] = {REC_CH, (unsigned)rec_tokens(dtype), 1u};
    if (!st || !sb || !encode_tiled_map(&p.map[i], r[i].p, dtype, 3, dims, strides, box)) return false;
  }
  return true;
}

// `smem`: the kernel's stages.
int launch_rec(void (*kernel)(RecParams), const RecParams& p, int smem, int id, const char* what, cudaStream_t st) {
  auto maps = [](int cluster) { return cluster > 1 ? 2 * cluster * 32 * (int)sizeof(float4) : 0; };  // of the cluster's CTAs
  // The kernel's limit is the same for every call: host threads with clusters of other sizes may be here too.
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem + maps(REC_MAX_CLUSTER));
  if (e != cudaSuccess) return fail(KDA_ERR_CUDA, std::string(what) + " smem: " + cudaGetErrorString(e));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((p.E + REC_CH - 1) / REC_CH * p.cluster), (unsigned)p.B);
  cfg.blockDim = dim3(REC_THREADS);
  cfg.dynamicSmemBytes = (size_t)(smem + maps(p.cluster));
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)p.cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  {
    TimedLaunch tl(id, st);
    e = cudaLaunchKernelEx(&cfg, kernel, p);
  }
  if (e != cudaSuccess) return fail(KDA_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  return launch_check(what);
}

template <typename T, bool VEC>
int rec_fwd_z(const RecParams& p, cudaStream_t st) {
  const int smem = rec_fwd_stages<VEC>() * (p.z.p ? 4 : 3) * rec_tensor_bytes<T, VEC>();
  return launch_rec(p.z.p ? rec_fwd_kernel<T, VEC, true> : rec_fwd_kernel<T, VEC, false>, p, smem, K_REC_FWD,
                    "recurrence forward", st);
}
template <typename T>
int rec_fwd(const RecParams& p, bool vec, cudaStream_t st) {
  return vec ? rec_fwd_z<T, true>(p, st) : rec_fwd_z<T, false>(p, st);
}

template <typename T, bool VEC>
int rec_bwd_z(const RecParams& p, cudaStream_t st) {
  const int smem = REC_BWD_STAGES * (p.z.p ? 5 : 4) * rec_tensor_bytes<T, VEC>();
  return launch_rec(p.z.p ? rec_bwd_kernel<T, VEC, true> : rec_bwd_kernel<T, VEC, false>, p, smem, K_REC_BWD,
                    "recurrence backward", st);
}
template <typename T>
int rec_bwd(const RecParams& p, bool vec, cudaStream_t st) {
  return vec ? rec_bwd_z<T, true>(p, st) : rec_bwd_z<T, false>(p, st);
}

template <typename T>
int rec_step(const RecStepParams& p, cudaStream_t st) {
  auto two = [&](const void* q, long long sr) { return aligned(q, 2 * sizeof(T)) && (p.rows == 1 || sr % 2 == 0); };
  const bool vec = p.E % 2 == 0 && two(p.x, p.sx) && two(p.decay, p.sd) && two(p.gate, p.sg) && two(p.z, p.sz) &&
                   aligned(p.y, 2 * sizeof(T)) && aligned(p.state, 8);
  const int per = REC_STEP_THREADS * (vec ? 2 : 1), gx = (p.E + per - 1) / per;
  const int gy = std::max(1, std::min(p.rows, (16 * sm_count() + gx - 1) / gx));
  {
    TimedLaunch tl(K_REC_STEP, st);
    if (vec) rec_step_kernel<T, true><<<dim3(gx, gy), REC_STEP_THREADS, 0, st>>>(p);
    else rec_step_kernel<T, false><<<dim3(gx, gy), REC_STEP_THREADS, 0, st>>>(p);
  }
  return launch_check("recurrence step");
}

}  // namespace

extern "C" {

size_t kda_b200_recurrence_saved_bytes(int64_t B, int64_t T, int E, int dtype) {
  if (B < 1 || T < 0 || E < 1 || dtype < KDA_IO_F32 || dtype > KDA_IO_F16) return 0;
  return std::max<size_t>(16, (size_t)B * rec_tiles(T, dtype) * E * 4);
}

size_t kda_b200_recurrence_workspace_bytes(int64_t B, int64_t T, int E, int dtype, int packed, int backward) {
  if (B < 1 || T < 0 || E < 1 || dtype < KDA_IO_F32 || dtype > KDA_IO_F16) return 0;
  size_t b = map_bytes(T, packed != 0);
  if (backward) b += align256((size_t)B * rec_cluster(B, T, E, dtype) * E * 3 * 4);
  return std::max<size_t>(b, 16);
}

int kda_b200_recurrence_fwd(const kda_b200_recurrence_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_rec(a, false);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->T == 0) return pass_state(a->h0, a->ht, (long long)a->nseq * a->E, st);
  if (!a->y) return fail(KDA_ERR_INVALID, "null output pointer");
  if (a->cu_seqlens &&  // (plain rows need none)
      (!workspace || !aligned(workspace, 16) ||
       workspace_bytes < kda_b200_recurrence_workspace_bytes(a->B, a->T, a->E, a->dtype, 1, 0)))
    return fail(KDA_ERR_INVALID, "workspace too small: kda_b200_recurrence_workspace_bytes() bytes are needed");
  if (a->saved && (!aligned(a->saved, 16) ||
                   a->saved_bytes < kda_b200_recurrence_saved_bytes(a->B, a->T, a->E, a->dtype)))
    return fail(KDA_ERR_INVALID, "saved buffer too small: kda_b200_recurrence_saved_bytes() bytes are needed");
  RecParams p = rec_params(a);
  if (!(p.err = device_error_flag())) return fail(KDA_ERR_CUDA, "the device error flag has no address");
  p.y = a->y;
  p.ht = a->ht;
  Carver cv(workspace);
  if ((rc = build_map(p.seq, cv, a->cu_seqlens, p.T, a->nseq, a->h0, a->ht, a->E, st))) return rc;
  const bool vec = rec_vec_ok(p, a->dtype) && rec_maps(p, a->dtype, false);
  return SSM_DISPATCH(a->dtype, rec_fwd, p, vec, st);
}

int kda_b200_recurrence_bwd(const kda_b200_recurrence_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_rec(a, false);
  if (rc) return rc;
  if (!a->dA) return fail(KDA_ERR_INVALID, "null gradient pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->T == 0) {
    if ((rc = zero_floats(a->dA, a->E, st)) || (rc = zero_floats(a->ddecay_bias, a->E, st)) ||
        (rc = zero_floats(a->dgate_bias, a->E, st)))
      return rc;
    return pass_state(a->dht, a->dh0, (long long)a->nseq * a->E, st);
  }
  if (!a->dy || !a->dx || !a->ddecay || !a->dgate || (a->z && !a->dz)) return fail(KDA_ERR_INVALID, "null gradient pointer");
  if (!a->saved || !aligned(a->saved, 16) ||
      a->saved_bytes < kda_b200_recurrence_saved_bytes(a->B, a->T, a->E, a->dtype))
    return fail(KDA_ERR_INVALID, "saved buffer missing or too small");
  if (!workspace || !aligned(workspace, 16) ||
      workspace_bytes < kda_b200_recurrence_workspace_bytes(a->B, a->T, a->E, a->dtype, a->cu_seqlens != nullptr, 1))
    return fail(KDA_ERR_INVALID, "workspace too small: kda_b200_recurrence_workspace_bytes() bytes are needed");
  RecParams p = rec_params(a);
  if (!(p.err = device_error_flag())) return fail(KDA_ERR_CUDA, "the device error flag has no address");
  p.dy = {a->dy, a->dy_sb, a->dy_st};
  p.dht = a->dht; p.dh0 = a->dh0;
  p.dx = a->dx; p.ddecay = a->ddecay; p.dgate = a->dgate; p.dz = a->z ? a->dz : nullptr;
  Carver cv(workspace);
  if ((rc = build_map(p.seq, cv, a->cu_seqlens, p.T, a->nseq, a->dht, a->dh0, a->E, st))) return rc;
  p.partial = cv.take<float>((size_t)p.B * p.cluster * p.E * 3 * 4);
  const bool vec = rec_vec_ok(p, a->dtype) && rec_maps(p, a->dtype, true);
  if ((rc = SSM_DISPATCH(a->dtype, rec_bwd, p, vec, st))) return rc;
  const long long cols = 3LL * p.E;
  {
    TimedLaunch tl(K_REC_BWD, st);
    ssm_reduce_kernel<<<(unsigned)((cols + SSM_REDUCE_COLS - 1) / SSM_REDUCE_COLS), SSM_REDUCE_COLS * SSM_REDUCE_SLICES, 0,
                        st>>>(p.partial, (long long)p.B * p.cluster, cols, 1, 3, a->dA, a->ddecay_bias, a->dgate_bias);
  }
  return launch_check("recurrence sums");
}

int kda_b200_recurrence_step(const kda_b200_recurrence_args* a, void* stream) {
  int rc = check_rec(a, true);
  if (rc) return rc;
  if (a->rows == 0) return KDA_OK;
  int* err = device_error_flag();
  if (!err) return fail(KDA_ERR_CUDA, "the device error flag has no address");
  RecStepParams p{rec_const(), a->x, a->decay, a->gate, a->z, a->x_sb, a->decay_sb, a->gate_sb, a->z_sb, a->A, a->decay_bias,
                  a->gate_bias, a->state, a->slots, a->rows, a->E, a->pool, a->y, err};
  return SSM_DISPATCH(a->dtype, rec_step, p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
