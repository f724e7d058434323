// C-ABI entry points of the normed and rotated heads (declared in include/coalibi.h).  Arguments
// are checked before any device use; nothing here allocates or synchronises.
#include "heads.cuh"

#include <algorithm>

#include "serving_host.cuh"

using namespace coalibi;

namespace coalibi {
namespace {

// CTAs to an SM in all, at most.  Many short ones end together: with 12 / 48 the forward of 32,764 tokens of 48 heads of
// 128 takes 130 / 124 us, of 32,768 tokens of 36 heads of 64 54 / 52.  The backward leaves a row of sums for each CTA: 179 /
// 174 with 5 / 12 of adding them up, and 69 / 72 with 3 / 5.
constexpr int kHeadsForwardWaves = 48, kHeadsWaves = 12;

int heads_chunks(int H, int per) { return (H + per - 1) / per; }

int check_heads(const CoalibiHeadsArgs* a, bool backward) {
  if (a == nullptr || !a->qkv || !a->q || !a->k || !a->v) return COALIBI_ERR_NULL_POINTER;
  if (backward && !a->dqkv) return COALIBI_ERR_NULL_POINTER;
  if (a->D != 64 && a->D != 128) return COALIBI_ERR_HEAD_DIM;
  if (a->dtype != COALIBI_F16 && a->dtype != COALIBI_BF16) return COALIBI_ERR_DTYPE;
  if (a->weight_dtype != a->dtype && a->weight_dtype != COALIBI_F32) return COALIBI_ERR_DTYPE;
  if (a->B <= 0 || a->S <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq > 65535 || a->Hkv > 65535 ||
      (long long)a->B * a->S > 0x7fffffffLL)
    return COALIBI_ERR_SHAPE;
  if (a->rot < 0 || a->rot > a->D || a->rot % 16 != 0 || (a->rot > 0 && a->n_pos <= 0)) return COALIBI_ERR_SHAPE;
  if (a->rot > 0 && (!a->cos || !a->sin)) return COALIBI_ERR_NULL_POINTER;
  if (!row_strides(a->qkv_stride) || !row_strides(a->q_stride) || !row_strides(a->k_stride) || !row_strides(a->v_stride))
    return COALIBI_ERR_ALIGNMENT;
  if (!aligned(a->qkv, 16) || !aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->cos, 16) ||
      !aligned(a->sin, 16) || !aligned(a->dqkv, 16) || !aligned(a->q_weight, 4) || !aligned(a->k_weight, 4) ||
      !aligned(a->start, 4) || !aligned(a->positions, 4))
    return COALIBI_ERR_ALIGNMENT;
  return COALIBI_OK;
}

HeadsParams heads_params(const CoalibiHeadsArgs* a, int waves) {
  HeadsParams p{};
  p.qkv = a->qkv;
  p.weight[0] = a->q_weight;
  p.weight[1] = a->k_weight;
  p.cos = a->cos;
  p.sin = a->sin;
  p.start = a->start;
  p.positions = a->positions;
  p.status = a->status;
  copy3(p.xs, a->qkv_stride);
  copy3(p.hs[0], a->q_stride);
  copy3(p.hs[1], a->k_stride);
  copy3(p.hs[2], a->v_stride);
  p.tokens = a->B * a->S;
  p.Hq = a->Hq;
  p.Hkv = a->Hkv;
  p.S = a->S;
  // Chunks of heads: up to eight by the same angles, but no fewer CTAs than SMs (64 tokens of 36 heads of 64
  // under a profiler: 5.9 us with a head to a chunk, 7.8 with six).
  const int slots = kHeadsThreads / (a->D / 16), sms = std::min(device_sm_count(), kPagedMaxSms);
  p.groups = (p.tokens - 1) / slots + 1;
  int most = kHeadsChunk;
  while (most > 1 && (long long)p.groups * (heads_chunks(a->Hq, most) + 2 * heads_chunks(a->Hkv, most)) < sms) most /= 2;
  for (int i = 0; i < 2; ++i) {
    const int H = i ? a->Hkv : a->Hq;
    p.per[i] = (H + heads_chunks(H, most) - 1) / heads_chunks(H, most);
    p.chunks[i] = heads_chunks(H, p.per[i]);
  }
  const int chunks = p.chunks[0] + 2 * p.chunks[1];
  p.ctas = std::min(p.groups, std::max(1, waves * sms / chunks));
  p.per_cta = (p.groups - 1) / p.ctas + 1;
  p.ctas = (p.groups - 1) / p.per_cta + 1;
  p.rot = a->rot;
  p.n_pos = a->n_pos;
  p.weight_f32 = a->weight_dtype == COALIBI_F32;
  p.eps = a->eps;
  return p;
}

unsigned heads_grid(const HeadsParams& p) { return (unsigned)(p.ctas * (p.chunks[0] + 2 * p.chunks[1])); }

template <bool PAIRS>
auto heads_fwd_kernel(const CoalibiHeadsArgs* a) {
  const bool bf16 = a->dtype == COALIBI_BF16;
  return a->D == 128 ? (bf16 ? coalibi_heads_fwd_kernel<true, 128, PAIRS> : coalibi_heads_fwd_kernel<false, 128, PAIRS>)
                     : (bf16 ? coalibi_heads_fwd_kernel<true, 64, PAIRS> : coalibi_heads_fwd_kernel<false, 64, PAIRS>);
}
template <bool PAIRS>
auto heads_bwd_kernel(const CoalibiHeadsArgs* a) {
  const bool bf16 = a->dtype == COALIBI_BF16;
  return a->D == 128 ? (bf16 ? coalibi_heads_bwd_kernel<true, 128, PAIRS> : coalibi_heads_bwd_kernel<false, 128, PAIRS>)
                     : (bf16 ? coalibi_heads_bwd_kernel<true, 64, PAIRS> : coalibi_heads_bwd_kernel<false, 64, PAIRS>);
}

int heads_result(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return launched(what);
  set_last_error_detail(cudaGetErrorString(e));
  return COALIBI_ERR_LAUNCH;
}

}  // namespace
}  // namespace coalibi

extern "C" int coalibi_heads_fwd(const CoalibiHeadsArgs* a, void* stream) {
  if (int rc = check_heads(a, false)) return rc;
  CtxGuard guard;
  if (int rc = enter_device(a->qkv, stream)) return rc;
  HeadsParams p = heads_params(a, kHeadsForwardWaves);
  p.out[0] = a->q;
  p.out[1] = a->k;
  p.out[2] = a->v;
  auto kernel = a->interleaved ? heads_fwd_kernel<true>(a) : heads_fwd_kernel<false>(a);
  return heads_result(launch_pdl(kernel, dim3(heads_grid(p)), dim3(kHeadsThreads), HeadsRing<2>::BYTES,
                                 static_cast<cudaStream_t>(stream), p),
                      "heads launch");
}

// A row of sums for each CTA of the queries' and keys' chunks: at most those of kHeadsWaves to an SM, or one for
// each head.
extern "C" size_t coalibi_heads_bwd_workspace_bytes(int Hq, int Hkv, int D) {
  if (Hq <= 0 || Hkv <= 0 || Hq > 65535 || Hkv > 65535 || (D != 64 && D != 128)) return 0;
  return (size_t)std::max(kHeadsWaves * kPagedMaxSms, Hq + Hkv) * D * 4;
}

extern "C" int coalibi_heads_bwd(const CoalibiHeadsArgs* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_heads(a, true)) return rc;
  if (!aligned(a->dq_weight, 4) || !aligned(a->dk_weight, 4)) return COALIBI_ERR_ALIGNMENT;
  if (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < coalibi_heads_bwd_workspace_bytes(a->Hq, a->Hkv, a->D))
    return COALIBI_ERR_WORKSPACE;
  CtxGuard guard;
  if (int rc = enter_device(a->qkv, stream)) return rc;
  HeadsParams p = heads_params(a, kHeadsWaves);
  p.in[0] = a->q;
  p.in[1] = a->k;
  p.in[2] = a->v;
  p.dqkv = a->dqkv;
  p.partial = static_cast<float*>(workspace);
  p.dweight[0] = a->dq_weight;
  p.dweight[1] = a->dk_weight;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = a->dtype == COALIBI_BF16;
  auto kernel = a->interleaved ? heads_bwd_kernel<true>(a) : heads_bwd_kernel<false>(a);
  auto sum = a->D == 128 ? (bf16 ? coalibi_heads_sum_kernel<true, 128> : coalibi_heads_sum_kernel<false, 128>)
                         : (bf16 ? coalibi_heads_sum_kernel<true, 64> : coalibi_heads_sum_kernel<false, 64>);
  constexpr int ring = HeadsRing<4>::BYTES;
  static std::atomic<unsigned long long> ready[8];  // bit per device, of each kernel
  const int which = (a->D == 128) + 2 * bf16 + 4 * (a->interleaved != 0);
  int dev = 0;
  cudaGetDevice(&dev);
  cudaError_t e = cudaSuccess;
  if (!(ready[which].load(std::memory_order_relaxed) >> dev & 1)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ring);
    if (e == cudaSuccess) ready[which].fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  if (e == cudaSuccess) e = launch_pdl(kernel, dim3(heads_grid(p)), dim3(kHeadsThreads), ring, s, p);
  if (e == cudaSuccess && (a->dq_weight || a->dk_weight)) e = launch_pdl(sum, dim3(2 * a->D / 32), dim3(1024), 0, s, p);
  return heads_result(e, "heads backward launch");
}
