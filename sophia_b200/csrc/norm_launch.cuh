// Shapes and launches of the residual norm's kernels, shared by the translation units of its two directions.
#pragma once

#include <algorithm>
#include <climits>
#include <string>

#include "kda_host.h"
#include "residual_norm.cuh"

namespace kda {

// How a row is laid over threads: `warps` of a group (or, of one, `lanes` lanes a row), k pieces of v channels a thread,
// `groups` of a CTA.
struct RnShape {
  int v, k, warps, groups, lanes;
};
// Rows that are read as they lie, element by element: 8 or 16 channels a thread.
inline RnShape rn_plain_shape(int D) {
  RnShape s{4, D <= 2048 ? 2 : 4, 0, 0, 32};
  s.warps = (D + 128 * s.k - 1) / (128 * s.k);
  s.groups = std::max(1, 8 / s.warps);
  return s;
}
// Rows in pieces of 16 bytes of the branch's type, `channels` of them a thread (8 where a row has no more than 256).
inline RnShape rn_ring_shape(int D, size_t branch_size, int channels) {
  RnShape s;
  s.v = (int)(16 / branch_size);
  s.k = (D <= 256 ? 8 : channels) / s.v;
  const int threads = (D + s.v * s.k - 1) / (s.v * s.k);
  s.warps = (threads + 31) / 32;
  s.groups = std::max(1, RN_MAX_WARPS / s.warps);
  s.lanes = 1;
  while (s.lanes < threads && s.lanes < 32) s.lanes *= 2;
  return s;
}
// The forward's channels a thread: 32, 24 or 16, whichever leaves the fewest threads idle, the most of them at a tie.  More
// channels a thread mean fewer warps a row that wait for one another.
inline RnShape rn_fwd_shape(int D, size_t branch_size) {
  RnShape best = rn_ring_shape(D, branch_size, 32);
  for (int channels : {24, 16}) {
    const RnShape s = rn_ring_shape(D, branch_size, channels);
    if (s.warps * s.k < best.warps * best.k) best = s;
  }
  return best;
}
inline RnShape rn_bwd_shape(int D, size_t branch_size) { return rn_ring_shape(D, branch_size, 16); }
inline long long rn_units(long long rows, int rows_a_cta) { return std::max(1LL, (rows + rows_a_cta - 1) / rows_a_cta); }

// An SM's shared memory, whose registers hold one CTA; up to 2 KB are static.
constexpr size_t RN_RING_SMEM = 227 * 1024 - 2 * 1024;
static_assert(sizeof(RnShared<3>) <= 2048, "what the kernels share beside the ring");
// The ring: rows of a stage, stages, and the CTAs of an SM.  A stage has 4 KB at least, unless that left groups
// without rows; two stages at least where the SM's shared memory has room for them, up to four.  No stage: the rows are
// too wide.
struct RnFit {
  int batch, stages, groups;
  long long ctas;
  size_t smem;
};
inline RnFit rn_fit(const RnShape& s, long long rows, size_t row_bytes, size_t fixed) {
  const size_t room = RN_RING_SMEM - fixed;
  const int per = s.warps > 1 ? 1 : 32 / s.lanes;
  RnFit f;
  // few rows: a group to an SM before the second
  f.groups = (int)std::max<long long>(1, std::min<long long>(s.groups, rows / ((long long)per * sm_count())));
  while (f.groups > 1 && 2 * f.groups * per * row_bytes > room) --f.groups;
  f.batch = 1;
  while (f.batch * per * row_bytes < 4096 && 4 * f.groups * f.batch * per * row_bytes <= room &&
         rows >= 4LL * f.batch * per * f.groups * sm_count()) f.batch *= 2;
  const size_t stage = (size_t)f.groups * f.batch * per * row_bytes;
  f.stages = (int)std::min<size_t>(RN_MAX_STAGES, room / stage);
  f.smem = f.stages * stage + fixed;
  f.ctas = std::min<long long>(rn_units(rows, f.groups * per * f.batch), sm_count());
  return f;
}
inline size_t rn_fixed(int D) { return (size_t)2 * D * 4; }  // the parameters
inline size_t rn_bwd_row(int D, size_t x, size_t o, bool g, bool dv, bool dn) {
  return (size_t)D * (x + o + (g ? o : 0) + (dv ? x : 0) + (dn ? o : 0));
}
template <typename TX, typename TO>
RnFit rn_fwd_fit(const RnParams& p, const RnShape& s) {
  return rn_fit(s, p.rows, (size_t)p.D * (sizeof(TX) + (p.g.p ? 2 : 1) * sizeof(TO)), rn_fixed(p.D));
}
template <typename TX, typename TO>
RnFit rn_bwd_fit(const RnParams& p, const RnShape& s) {
  return rn_fit(s, p.rows, rn_bwd_row(p.D, sizeof(TX), sizeof(TO), p.g.p, p.dv.p, p.dn.p), rn_fixed(p.D));
}
// (the backward: as many as the SMs hold at once, which is one of more than eight warps)
inline long long rn_plain_ctas(long long rows, const RnShape& s) {
  return std::min(rn_units(rows, s.groups), (long long)(s.warps <= 8 ? 2 : 1) * sm_count());
}

template <typename TX, typename TO>
int rn_fwd(RnParams& p, bool vec, cudaStream_t st);
template <typename TX, typename TO>
int rn_bwd(RnParams& p, bool vec, cudaStream_t st);

template <typename TX, typename TO, int K>
int launch_rn_fwd(const RnParams& p, const RnShape& s, cudaStream_t st) {
  {
    TimedLaunch tl(K_NORM_FWD, st);
    rn_fwd_kernel<TX, TO, K>
        <<<(unsigned)std::min(rn_units(p.rows, s.groups), 1LL << 20), s.warps * s.groups * 32, 0, st>>>(p);
  }
  return launch_check("residual norm forward");
}

// `most`: the kernel's limit, the same for every call, because host threads with other sizes may be here too.
template <typename K>
int rn_smem(K kernel, size_t smem, size_t most) {
  if (smem <= 40 * 1024) return KDA_OK;  // (48 KB go without asking, the static ones included)
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
  return e == cudaSuccess ? KDA_OK : fail(KDA_ERR_CUDA, std::string("residual norm smem: ") + cudaGetErrorString(e));
}

// The ring kernel for a call's parts: Kernel::get<FULL, GATE, DROP>().
template <typename Kernel>
auto rn_pick(bool full, bool gate, bool drop) {
  if (full)
    return gate ? (drop ? Kernel::template get<true, true, true>() : Kernel::template get<true, true, false>())
                : (drop ? Kernel::template get<true, false, true>() : Kernel::template get<true, false, false>());
  return gate ? (drop ? Kernel::template get<false, true, true>() : Kernel::template get<false, true, false>())
              : (drop ? Kernel::template get<false, false, true>() : Kernel::template get<false, false, false>());
}
template <typename Kernel>
int launch_rn_ring(RnParams& p, const RnShape& s, const RnFit& fit, int id, const char* what, cudaStream_t st) {
  p.stages = fit.stages;
  p.batch = fit.batch;
  p.parts = (int)fit.ctas;
  p.params = (long long)(fit.smem / 4) - 2LL * p.D;
  auto kernel = rn_pick<Kernel>(p.D == s.warps * 32 * s.v * s.k, p.g.p != nullptr, p.dropout);
  if (int rc = rn_smem(kernel, fit.smem, RN_RING_SMEM)) return rc;
  {
    TimedLaunch tl(id, st);
    kernel<<<(unsigned)fit.ctas, s.warps * fit.groups * 32, fit.smem, st>>>(p);
  }
  return launch_check(what);
}

template <typename TX, typename TO, int K>
int launch_rn_bwd(RnParams& p, const RnShape& s, cudaStream_t st) {
  const size_t smem = (size_t)s.groups * 2 * p.D * 4;
  auto kernel = rn_bwd_kernel<TX, TO, K>;
  if (int rc = rn_smem(kernel, smem, (size_t)2 * RN_MAX_WIDTH * 4)) return rc;  // (above 2048 channels one group)
  p.parts = (int)rn_plain_ctas(p.rows, s);
  {
    TimedLaunch tl(K_NORM_BWD, st);
    kernel<<<(unsigned)p.parts, s.warps * s.groups * 32, smem, st>>>(p);
  }
  return launch_check("residual norm backward");
}

}  // namespace kda
