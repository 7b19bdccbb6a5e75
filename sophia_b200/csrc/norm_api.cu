// C ABI of the residual norm (declared in include/kda_b200.h): argument checks,
// buffer carving and kernel launches.  No allocation, no host sync.
#include <cuda_runtime.h>

#include <climits>
#include <cmath>

#include "../../include/kda_b200.h"
#include "norm_launch.cuh"
#include "ssm_host.cuh"

using namespace kda;

namespace {

int check_norm(const kda_b200_norm_args* a) {
  int rc;
  if (!a) return fail(KDA_ERR_INVALID, "null arguments");
  if ((rc = check_dtype(a->dtype)) || (rc = check_dtype(a->stream_dtype))) return rc;
  if (a->stream_dtype != a->dtype && a->stream_dtype != KDA_IO_F32)
    return fail(KDA_ERR_UNSUPPORTED, "the residual stream is float32 or of the branch's type");
  if (a->B < 0 || a->T < 0 || a->D < 1) return fail(KDA_ERR_INVALID, "B >= 0, T >= 0 and D >= 1 are required");
  if (a->D > RN_MAX_WIDTH) return fail(KDA_ERR_UNSUPPORTED, "more than 8192 channels");
  if (a->T > INT32_MAX) return fail(KDA_ERR_UNSUPPORTED, "too many tokens");
  if (!aligned(a->rstd, 8)) return fail(KDA_ERR_INVALID, "rstd must be 8-byte aligned");
  if (!(a->dropout_p >= 0.0 && a->dropout_p <= 1.0)) return fail(KDA_ERR_INVALID, "dropout_p must be in [0, 1]");
  if (a->B * a->T > 0 && (!a->x || !a->o)) return fail(KDA_ERR_INVALID, "null input pointer");
  return KDA_OK;
}

RnParams norm_params(const kda_b200_norm_args* a) {
  RnParams p{};
  p.x = {a->x, a->x_sb, a->x_st};
  p.o = {a->o, a->o_sb, a->o_st};
  p.g = {a->gate, a->gate_sb, a->gate_st};
  p.w = a->w; p.wb = a->wb; p.scale = a->scale;
  p.seed_ptr = reinterpret_cast<const long long*>(a->seed_ptr);
  p.seed = a->seed;
  p.offset = a->offset;
  const double below = std::nearbyint(a->dropout_p * 4294967296.0);
  p.drop_all = below >= 4294967296.0;
  p.drop = p.drop_all ? 0u : (unsigned)below;
  p.dropout = below > 0.0;
  p.keep_scale = a->dropout_p < 1.0 ? (float)(1.0 / (1.0 - a->dropout_p)) : 0.f;
  p.rstd = a->rstd;
  p.rows = a->B * a->T;
  p.T = (int)a->T;
  p.D = a->D;
  p.eps = a->eps;
  return p;
}

// Pieces: every row of every tensor starts at a multiple of 16 bytes, and the parameters do.
bool norm_vec(const RnParams& p, long long B, int dtype, int stream_dtype) {
  const int V = (int)(16 / io_size(dtype));
  auto ok = [&](const RowView& r, int type) {
    const size_t esz = io_size(type);
    return !r.p || vec_rows(r.p, r.sb, r.st, B, p.T, (int)(16 / esz), esz);
  };
  return p.D % V == 0 && ok(p.x, stream_dtype) && ok(p.o, dtype) && ok(p.g, dtype) && ok(p.dv, stream_dtype) &&
         ok(p.dn, dtype) && aligned(p.v, 16) && aligned(p.n, 16) && aligned(p.dx, 16) && aligned(p.d_o, 16) &&
         aligned(p.dg, 16) && aligned(p.w, 16) && aligned(p.wb, 16) && aligned(p.scale, 16);
}

// One stride over all rows?  And which tensors' rows lie end to end.
void norm_flatten(RnParams& p, long long B) {
  auto flat = [&](const RowView& r) { return !r.p || B <= 1 || r.sb == (long long)p.T * r.st; };
  const RowView* all[5] = {&p.x, &p.o, &p.g, &p.dv, &p.dn};
  for (int i = 0; i < 5; ++i)
    if (all[i]->st == p.D && flat(*all[i])) p.dense |= 1u << i;
  if (flat(p.x) && flat(p.o) && flat(p.g) && flat(p.dv) && flat(p.dn)) p.T = 0;
}

template <template <typename, typename> class F>
int by_type(int dtype, int stream_dtype, RnParams& p, bool vec, cudaStream_t st) {
  if (dtype == KDA_IO_F32) return F<float, float>::run(p, vec, st);
  if (dtype == KDA_IO_BF16)
    return stream_dtype == KDA_IO_F32 ? F<float, bf16>::run(p, vec, st) : F<bf16, bf16>::run(p, vec, st);
  return stream_dtype == KDA_IO_F32 ? F<float, f16>::run(p, vec, st) : F<f16, f16>::run(p, vec, st);
}
template <typename TX, typename TO>
struct Fwd {
  static int run(RnParams& p, bool vec, cudaStream_t st) { return rn_fwd<TX, TO>(p, vec, st); }
};
template <typename TX, typename TO>
struct Bwd {
  static int run(RnParams& p, bool vec, cudaStream_t st) { return rn_bwd<TX, TO>(p, vec, st); }
};

// The most CTAs that a backward call may have, whichever way its rows are read and whatever parts it has.
long long norm_parts(long long rows, int D, int dtype) {
  const size_t o = io_size(dtype);
  long long most = rn_plain_ctas(rows, rn_plain_shape(D));
  const RnShape s = rn_bwd_shape(D, o);
  for (size_t x : {o, (size_t)4})
    for (int parts = 0; parts < 8; ++parts)
      most = std::max(most, rn_fit(s, rows, rn_bwd_row(D, x, o, parts & 1, parts & 2, parts & 4), rn_fixed(D)).ctas);
  return most;
}

}  // namespace

extern "C" {

size_t kda_b200_norm_workspace_bytes(int64_t B, int64_t T, int D, int dtype) {
  if (B < 0 || T < 0 || D < 1 || D > RN_MAX_WIDTH || dtype < KDA_IO_F32 || dtype > KDA_IO_F16) return 0;
  const long long rows = B * T;
  return std::max<size_t>(16, (size_t)norm_parts(rows, D, dtype) * 3 * D * 4);
}

int kda_b200_norm_fwd(const kda_b200_norm_args* a, void* stream) {
  int rc = check_norm(a);
  if (rc) return rc;
  RnParams p = norm_params(a);
  if (p.rows == 0) return KDA_OK;
  if (!(p.err = device_error_flag())) return fail(KDA_ERR_CUDA, "the device error flag has no address");
  if (!a->v || (a->w && !a->n)) return fail(KDA_ERR_INVALID, "null output pointer");
  p.v = a->v;
  p.n = a->n;
  const bool vec = norm_vec(p, a->B, a->dtype, a->stream_dtype);
  norm_flatten(p, a->B);
  return by_type<Fwd>(a->dtype, a->stream_dtype, p, vec, static_cast<cudaStream_t>(stream));
}

int kda_b200_norm_bwd(const kda_b200_norm_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_norm(a);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  RnParams p = norm_params(a);
  if (p.rows == 0) {
    for (float* q : {a->dw, a->dwb, a->dscale})
      if ((rc = zero_floats(q, a->D, st))) return rc;
    return KDA_OK;
  }
  if (!(p.err = device_error_flag())) return fail(KDA_ERR_CUDA, "the device error flag has no address");
  p.dv = {a->dv, a->dv_sb, a->dv_st};
  if (a->w) p.dn = {a->dn, a->dn_sb, a->dn_st};
  p.dx = a->dx; p.d_o = a->d_o; p.dg = a->dgate;
  if (!p.dx || !p.d_o || (p.g.p && !p.dg)) return fail(KDA_ERR_INVALID, "null gradient pointer");
  if (!p.rstd) return fail(KDA_ERR_INVALID, "rstd of the forward is needed");
  if (!workspace || !aligned(workspace, 16) || workspace_bytes < kda_b200_norm_workspace_bytes(a->B, a->T, a->D, a->dtype))
    return fail(KDA_ERR_INVALID, "workspace too small: kda_b200_norm_workspace_bytes() bytes are needed");
  p.partial = static_cast<float*>(workspace);
  const bool vec = norm_vec(p, a->B, a->dtype, a->stream_dtype);
  norm_flatten(p, a->B);
  if ((rc = by_type<Bwd>(a->dtype, a->stream_dtype, p, vec, st))) return rc;
  if (!a->dw && !a->dwb && !a->dscale) return KDA_OK;
  {
    TimedLaunch tl(K_NORM_BWD, st);
    rn_reduce_kernel<<<dim3((a->D + RN_REDUCE_COLS - 1) / RN_REDUCE_COLS, 3), RN_REDUCE_COLS * RN_REDUCE_SLICES, 0, st>>>(
        p.partial, p.parts, a->D, a->dw, a->dwb, a->dscale);
  }
  return launch_check("residual norm sums");
}

}  // extern "C"
