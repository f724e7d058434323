// C-ABI entry points of the serving operators (declared in include/coalibi.h): paged
// append, attention of drafted trees over a paged cache, and sampling.  Arguments are
// checked before any device use; nothing here allocates or synchronises.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cstdio>

#include "coalibi.h"
#include "ctx_guard.h"
#include "paged.cuh"
#include "sample.cuh"

namespace coalibi {

void set_last_error_detail(const char* msg);
int make_page_tmap(CUtensorMap* map, const void* base, int D, int page_size, int heads, int pages,
                   const long long* stride, bool bf16);

namespace {

bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// strides of 16-byte rows: multiples of 8 elements, not negative
bool row_strides(const long long* s) {
  for (int i = 0; i < 3; ++i)
    if (s[i] < 0 || s[i] % 8 != 0) return false;
  return true;
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return COALIBI_OK;
  char msg[160];
  snprintf(msg, sizeof(msg), "%s: %s", what, cudaGetErrorString(e));
  set_last_error_detail(msg);
  return COALIBI_ERR_LAUNCH;
}

void copy3(long long* dst, const long long* src) {
  for (int i = 0; i < 3; ++i) dst[i] = src[i];
}

int check_cache(int B, int Hkv, int D, int page_size, int max_pages, int n_pages, int dtype,
                const long long* k_page_stride, const long long* v_page_stride, long long table_stride) {
  if (D != 64 && D != 128) return COALIBI_ERR_HEAD_DIM;
  if (dtype != COALIBI_F16 && dtype != COALIBI_BF16) return COALIBI_ERR_DTYPE;
  if (B <= 0 || Hkv <= 0 || page_size <= 0 || page_size % 16 != 0 || max_pages <= 0 || n_pages <= 0)
    return COALIBI_ERR_SHAPE;
  // token numbers and lengths are 32-bit on the device
  if ((long long)max_pages * page_size > 0x7fffff00LL || table_stride < 0 || B > 65535 || Hkv > 65535)
    return COALIBI_ERR_SHAPE;
  if (!row_strides(k_page_stride) || !row_strides(v_page_stride)) return COALIBI_ERR_ALIGNMENT;
  const int sizes[3] = {n_pages, Hkv, page_size};
  for (int i = 0; i < 3; ++i) {
    const long long k = k_page_stride[i], v = v_page_stride[i];
    if (sizes[i] > 1 && (k == 0 || v == 0)) return COALIBI_ERR_SHAPE;  // entries on top of each other
    if (k >= 1LL << 39 || v >= 1LL << 39) return COALIBI_ERR_SHAPE;
  }
  return COALIBI_OK;
}

}  // namespace
}  // namespace coalibi

using namespace coalibi;

namespace coalibi {
namespace {
template <bool BF16, int D>
auto append_kernel(int turn) {
  return turn == kTurnNone    ? coalibi_paged_append_kernel<BF16, D, kTurnNone>
         : turn == kTurnPairs ? coalibi_paged_append_kernel<BF16, D, kTurnPairs>
                              : coalibi_paged_append_kernel<BF16, D, kTurnHalves>;
}
}  // namespace
}  // namespace coalibi

extern "C" int coalibi_paged_append(const CoalibiPagedAppendArgs* a, void* stream) {
  if (a == nullptr || !a->k || !a->v || !a->k_pages || !a->v_pages || !a->page_table || !a->start)
    return COALIBI_ERR_NULL_POINTER;
  if ((a->q != nullptr) != (a->q_out != nullptr)) return COALIBI_ERR_NULL_POINTER;
  int rc = check_cache(a->B, a->Hkv, a->D, a->page_size, a->max_pages, a->n_pages, a->dtype, a->k_page_stride,
                       a->v_page_stride, a->table_stride);
  if (rc) return rc;
  if (a->S <= 0 || (long long)a->B * a->S > 0x7fffffffLL || (a->q && (a->Hq <= 0 || a->Hq > 65535)))
    return COALIBI_ERR_SHAPE;
  if (a->rot < 0 || a->rot > a->D || a->rot % 16 != 0 || (a->rot > 0 && a->n_pos <= 0)) return COALIBI_ERR_SHAPE;
  if (a->rot > 0 && (!a->cos || !a->sin)) return COALIBI_ERR_NULL_POINTER;
  if (!row_strides(a->k_stride) || !row_strides(a->v_stride) ||
      (a->q && (!row_strides(a->q_stride) || !row_strides(a->q_out_stride))))
    return COALIBI_ERR_ALIGNMENT;
  if (!aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->q, 16) || !aligned(a->q_out, 16) ||
      !aligned(a->k_pages, 16) || !aligned(a->v_pages, 16) || !aligned(a->cos, 16) || !aligned(a->sin, 16))
    return COALIBI_ERR_ALIGNMENT;
  CtxGuard guard;
  if ((rc = enter_device(a->k_pages, stream))) return rc;
  AppendParams p{};
  p.k = a->k;
  p.v = a->v;
  p.q = a->q;
  p.q_out = a->q_out;
  p.k_pages = a->k_pages;
  p.v_pages = a->v_pages;
  p.page_table = a->page_table;
  p.start = a->start;
  p.count = a->count;
  p.positions = a->positions;
  p.cos = a->cos;
  p.sin = a->sin;
  p.status = a->status;
  copy3(p.ks, a->k_stride);
  copy3(p.vs, a->v_stride);
  copy3(p.qs, a->q_stride);
  copy3(p.qos, a->q_out_stride);
  copy3(p.kps, a->k_page_stride);
  copy3(p.vps, a->v_page_stride);
  p.table_stride = a->table_stride;
  p.Hq = a->q != nullptr ? a->Hq : 0;
  p.Hkv = a->Hkv;
  p.S = a->S;
  p.tokens = (long long)a->B * a->S;
  p.page_size = a->page_size;
  p.max_pages = a->max_pages;
  p.n_pages = a->n_pages;
  p.rot = a->rot;
  p.n_pos = a->n_pos;
  p.interleaved = a->interleaved;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Few tokens spread over the SMs, one to a CTA; a prompt's go in pairs, whose lookups overlap
  // (16,000 ragged prompt tokens of 48 heads: 49 us in groups of 8, 48 of 4, 46.6 of 2).
  p.group = p.tokens >= 8LL * kAppendGroup * device_sm_count() ? kAppendGroup : 1;
  const dim3 grid((unsigned)((p.tokens + p.group - 1) / p.group));
  const bool bf16 = a->dtype == COALIBI_BF16;
  const int turn = a->rot == 0 ? kTurnNone : a->interleaved ? kTurnPairs : kTurnHalves;
  auto kernel = a->D == 128 ? (bf16 ? append_kernel<true, 128>(turn) : append_kernel<false, 128>(turn))
                            : (bf16 ? append_kernel<true, 64>(turn) : append_kernel<false, 64>(turn));
  if (const cudaError_t e = launch_pdl(kernel, grid, dim3(kAppendThreads), 0, s, p); e != cudaSuccess) {
    set_last_error_detail(cudaGetErrorString(e));
    return COALIBI_ERR_LAUNCH;
  }
  return launched("paged append launch");
}

namespace coalibi {
namespace {

// The attention kernel of layout L and the kernel that joins its pieces.
template <int D, bool BF16, typename L, typename K>
int launch_paged(K kernel, std::atomic<unsigned long long>& ready, int threads, const CUtensorMap& tk,
                 const CUtensorMap& tv, PagedAttnParams& p, int sms, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(ready.load(std::memory_order_relaxed) >> dev & 1)) {  // bit per device (the library knows at most 64)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::BYTES);
    if (e == cudaSuccess) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  const int rows = p.Hq / p.Hkv * p.Sq;
  p.row_blocks = (rows + L::ROWS - 1) / L::ROWS;
  p.n_ctas = (sms < kPagedMaxSms ? sms : kPagedMaxSms) * L::CTAS;
  const long long most = ((long long)p.max_pages * p.page_size + L::UNIT - 1) / L::UNIT;
  const long long bound = (most + L::COST) * p.B * p.Hkv * p.row_blocks;  // if every table row were full
  if (bound > 0x7fffffffLL) return COALIBI_ERR_SHAPE;
  const long long items = (long long)p.B * p.Hkv * p.row_blocks;
  p.whole = most * L::UNIT <= L::WHOLE;
  if (p.whole)
    p.n_ctas = (int)items;
  else if (bound < p.n_ctas)
    p.n_ctas = (int)bound;
  if (e == cudaSuccess) e = launch_pdl(kernel, dim3(p.n_ctas), dim3(threads), L::BYTES, s, tk, tv, p);
  if (e == cudaSuccess && !p.whole)
    e = launch_pdl(coalibi_paged_join_kernel<D, BF16, L>, dim3(p.B * p.Hkv, (rows + 3) / 4), dim3(128), 0, s, p);
  if (e != cudaSuccess) set_last_error_detail(cudaGetErrorString(e));
  return e == cudaSuccess ? launched("paged attention launch") : COALIBI_ERR_LAUNCH;
}

template <int D, bool BF16, int RW, int XR, int WARPS>
int launch_narrow_of(const CUtensorMap& tk, const CUtensorMap& tv, PagedAttnParams& p, int sms, cudaStream_t s) {
  static std::atomic<unsigned long long> ready{0};
  return launch_paged<D, BF16, PagedLayout<D, RW, WARPS>>(coalibi_paged_attn_kernel<D, BF16, RW, XR, WARPS>, ready,
                                                          32 * WARPS, tk, tv, p, sms, s);
}

template <int D, bool BF16, int RW, int XR>
int launch_narrow(const CUtensorMap& tk, const CUtensorMap& tv, PagedAttnParams& p, int sms, cudaStream_t s) {
  // Four warps to an item where the tables hold little work, else RW to a CTA, measured (four / one,
  // us a call, 8 kv heads, 4 rows): 1 request of 500 keys 11 / 28, 32 of 500 21 / 29, 1 of 1000 11 / 15,
  // 8 of 1000 16 / 15, 8 of 1900 21 / 19, 8 of 8192 55 / 52, 64 of 500 46 / 31, 256 of 200 92 / 52,
  // 256 of 1000 230 / 170; 16 rows, 8 of 8192 63 / 55.  The host sees the tables' width alone, which
  // was the longest request's in all of these: under a table of 2048 or 8192 keys 1 request of 37
  // (12 heads of 64) takes 12.1 us a call, 9.4 under one of 48; 16 of 0 .. 8191 under one of 32768 the same 52.
  const int rows = p.Hq / p.Hkv * p.Sq;
  const long long items = (long long)p.B * p.Hkv * ((rows + 16 * RW - 1) / (16 * RW));
  const long long width = (long long)p.max_pages * p.page_size;
  if (items > 2LL * sms || (width > 512 && items * width > 32768))
    return launch_narrow_of<D, BF16, RW, XR, RW>(tk, tv, p, sms, s);
  return launch_narrow_of<D, BF16, RW, XR, 4>(tk, tv, p, sms, s);
}

template <int D, bool BF16, bool DUP>
int launch_wide(const CUtensorMap& tk, const CUtensorMap& tv, PagedAttnParams& p, int sms, cudaStream_t s) {
  static std::atomic<unsigned long long> ready{0};
  using L = WideLayout<D, DUP>;
  return launch_paged<D, BF16, L>(coalibi_paged_wide_kernel<D, BF16, DUP>, ready, L::THREADS, tk, tv, p, sms, s);
}

template <int D, bool BF16>
int launch_paged_rows(const CUtensorMap& tk, const CUtensorMap& tv, PagedAttnParams& p, int sms, cudaStream_t s) {
  const int rows = p.Hq / p.Hkv * p.Sq;
  // Warp-level MMAs up to 32 rows, tcgen05 from there, measured (warp level / tcgen05, us a call):
  // 32 rows, 8 requests of 8192 keys, 8 kv heads 68 / 67; 32 rows, 32 requests of 500 keys 33 / 37;
  // 24 rows of D = 64, 8 requests of 4000 keys, 12 heads 38 / 53; 16 rows, 8 of 8192 62 / 66;
  // 64 rows, 8 requests of 127 to 16383 keys 120 / 75.
  if (rows <= 8) return launch_narrow<D, BF16, 1, 1>(tk, tv, p, sms, s);
  if (rows <= 16) return launch_narrow<D, BF16, 1, 2>(tk, tv, p, sms, s);
  if (rows <= 32) return launch_narrow<D, BF16, 2, 2>(tk, tv, p, sms, s);
  if (rows <= 64) return launch_wide<D, BF16, true>(tk, tv, p, sms, s);
  return launch_wide<D, BF16, false>(tk, tv, p, sms, s);
}

template <int D>
size_t paged_ws_rows(int B, int rows) {
  if (rows <= 16) return std::max(paged_ws_bytes<PagedLayout<D, 1, 1>>(B), paged_ws_bytes<PagedLayout<D, 1, 4>>(B));
  if (rows <= 32) return std::max(paged_ws_bytes<PagedLayout<D, 2, 2>>(B), paged_ws_bytes<PagedLayout<D, 2, 4>>(B));
  if (rows <= 64) return paged_ws_bytes<WideLayout<D, true>>(B);
  return paged_ws_bytes<WideLayout<D, false>>(B);
}

}  // namespace
}  // namespace coalibi

extern "C" size_t coalibi_paged_attention_workspace_bytes(int B, int Hq, int Hkv, int Sq, int D) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq <= 0 || Sq > kTreeMaxSq || Hq % Hkv != 0 || (D != 64 && D != 128)) return 0;
  return D == 128 ? paged_ws_rows<128>(B, Hq / Hkv * Sq) : paged_ws_rows<64>(B, Hq / Hkv * Sq);
}

extern "C" int coalibi_paged_attention(const CoalibiPagedAttentionArgs* a, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  if (a == nullptr || !a->q || !a->o || !a->k_pages || !a->v_pages || !a->slopes || !a->page_table || !a->ctx_lens)
    return COALIBI_ERR_NULL_POINTER;
  int rc = check_cache(a->B, a->Hkv, a->D, a->page_size, a->max_pages, a->n_pages, a->dtype, a->k_page_stride,
                       a->v_page_stride, a->table_stride);
  if (rc) return rc;
  if (a->slopes_dtype != COALIBI_F16 && a->slopes_dtype != COALIBI_BF16 && a->slopes_dtype != COALIBI_F32)
    return COALIBI_ERR_DTYPE;
  if (a->Hq <= 0 || a->Hq % a->Hkv != 0 || a->Hq > 65535 || a->Sq <= 0 || a->Sq > kTreeMaxSq || a->mask_stride < 0)
    return COALIBI_ERR_SHAPE;
  if (!row_strides(a->q_stride) || !row_strides(a->o_stride)) return COALIBI_ERR_ALIGNMENT;
  if (!aligned(a->q, 16) || !aligned(a->o, 16) || !aligned(a->k_pages, 16) || !aligned(a->v_pages, 16) ||
      !aligned(a->tree_mask, 8))
    return COALIBI_ERR_ALIGNMENT;
  if (workspace == nullptr || !aligned(workspace, 16) ||
      workspace_bytes < coalibi_paged_attention_workspace_bytes(a->B, a->Hq, a->Hkv, a->Sq, a->D))
    return COALIBI_ERR_WORKSPACE;
  CtxGuard guard;
  if ((rc = enter_device(a->k_pages, stream))) return rc;
  PagedAttnParams p{};
  p.q = a->q;
  p.o = a->o;
  p.k_pages = a->k_pages;
  p.v_pages = a->v_pages;
  p.slopes = a->slopes;
  p.page_table = a->page_table;
  p.ctx_lens = a->ctx_lens;
  p.tree_mask = a->tree_mask;
  p.status = a->status;
  copy3(p.qs, a->q_stride);
  copy3(p.os, a->o_stride);
  copy3(p.kps, a->k_page_stride);
  copy3(p.vps, a->v_page_stride);
  p.table_stride = a->table_stride;
  p.mask_stride = a->mask_stride;
  p.B = a->B;
  p.Hq = a->Hq;
  p.Hkv = a->Hkv;
  p.Sq = a->Sq;
  p.page_size = a->page_size;
  p.max_pages = a->max_pages;
  p.n_pages = a->n_pages;
  p.slopes_dtype = a->slopes_dtype;
  p.sm_scale = a->sm_scale;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  p.ws = static_cast<float*>(workspace);
  p.page_shift = -1;
  for (int k = 4; k < 31; ++k)
    if (a->page_size == 1 << k) p.page_shift = k;
  const bool bf16 = a->dtype == COALIBI_BF16;
  const int sms = device_sm_count();
  CUtensorMap tk, tv;
  if ((rc = make_page_tmap(&tk, a->k_pages, a->D, a->page_size, a->Hkv, a->n_pages, a->k_page_stride, bf16))) return rc;
  if ((rc = make_page_tmap(&tv, a->v_pages, a->D, a->page_size, a->Hkv, a->n_pages, a->v_page_stride, bf16))) return rc;
  if (a->D == 128) return bf16 ? launch_paged_rows<128, true>(tk, tv, p, sms, s) : launch_paged_rows<128, false>(tk, tv, p, sms, s);
  return bf16 ? launch_paged_rows<64, true>(tk, tv, p, sms, s) : launch_paged_rows<64, false>(tk, tv, p, sms, s);
}

namespace coalibi {
namespace {

// A launch with clusters of p.cluster CTAs, one cluster per row, its set-up beside the end of the
// kernel before it on the stream.
template <typename K>
cudaError_t launch_rows(K kernel, int threads, size_t smem, const SampleParams& p, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.B * p.cluster));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // (the kernels wait before global memory)
  attr[1].val.programmaticStreamSerializationAllowed = COALIBI_PDL ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int DT>
int launch_sample(SampleParams& p, cudaStream_t s) {
  constexpr int kSize = DT == 2 ? 4 : 2, kChunk = 16 / kSize;
  constexpr int kMostBytes = 200 << 10, kRowBytes = 64 << 10;
  const int sms = device_sm_count();
  const long long chunks = (p.V + kChunk - 2) / kChunk + 1;  // of a row at any alignment, at most
  p.filters = p.top_k || p.top_p || (p.top_k_all > 0 && p.top_k_all < p.V) || !(p.top_p_all >= 1.f);
  if (!p.filters && !p.min_p && !(p.min_p_all > 0.f)) {
    // as many CTAs as run at once (four to an SM), while slices keep two rounds of loads: 256 rows
    // of 131072 tokens take 57 us with 2 per row (512 CTAs), 68 with 4, 83 with 8, 81 with 1
    int c = 1;
    while (c < kSampleMaxCluster && (long long)p.B * c * 2 <= 4LL * sms && chunks >= 4LL * c * kStreamThreads) c *= 2;
    p.cluster = c;
    const cudaError_t e = launch_rows(coalibi_sample_stream_kernel<DT>, kStreamThreads, 0, p, s);
    if (e != cudaSuccess) set_last_error_detail(cudaGetErrorString(e));
    return e == cudaSuccess ? COALIBI_OK : COALIBI_ERR_LAUNCH;
  }
  // CTAs per row: enough for slices of about 64 KB, and more while the SMs outnumber them
  int c = 1;
  while (c < kSampleMaxCluster && (chunks * 16 > (long long)c * kRowBytes || (long long)p.B * c * 2 <= sms) &&
         chunks >= 256LL * c)
    c *= 2;
  p.cluster = c;
  const long long per = (chunks + c - 1) / c;
  const size_t fixed = p.filters ? 8 * kSampleBins + 8 * kSampleListed : 4096;
  const size_t scratch = p.filters ? 5 * kSampleMaxK * 8 : 0;  // see coalibi_sample_kernel's top-k
  size_t slice = (size_t)per * 16;
  p.slice_chunks = slice + fixed <= kMostBytes ? (int)per : 0;
  if (p.slice_chunks == 0) slice = 0;
  const size_t bytes = fixed + (slice > scratch ? slice : scratch);
  cudaError_t e = cudaSuccess;
  static std::atomic<unsigned long long> ready{0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    e = cudaFuncSetAttribute(coalibi_sample_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostBytes);
    if (e == cudaSuccess) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  if (e == cudaSuccess) e = launch_rows(coalibi_sample_kernel<DT>, kSampleThreads, bytes, p, s);
  if (e != cudaSuccess) set_last_error_detail(cudaGetErrorString(e));
  return e == cudaSuccess ? COALIBI_OK : COALIBI_ERR_LAUNCH;
}

}  // namespace
}  // namespace coalibi

extern "C" int coalibi_sample(const CoalibiSampleArgs* a, void* stream) {
  if (a == nullptr || !a->logits || !a->noise || !a->tokens || !a->logprobs) return COALIBI_ERR_NULL_POINTER;
  if (a->dtype != COALIBI_F16 && a->dtype != COALIBI_BF16 && a->dtype != COALIBI_F32) return COALIBI_ERR_DTYPE;
  if (a->B <= 0 || a->B > 0x7fffffff / kSampleMaxCluster || a->V <= 0 || a->V > COALIBI_SAMPLE_MAX_VOCAB || a->logits_stride < 0 || a->noise_stride < 0)
    return COALIBI_ERR_SHAPE;
  if (!aligned(a->logits, a->dtype == COALIBI_F32 ? 4 : 2) || !aligned(a->noise, 4) || !aligned(a->tokens, 8) ||
      !aligned(a->logprobs, 4))
    return COALIBI_ERR_ALIGNMENT;
  CtxGuard guard;
  if (int rc = enter_device(a->logits, stream)) return rc;
  SampleParams p{};
  p.logits = a->logits;
  p.noise = a->noise;
  p.temperature = a->temperature;
  p.top_k = a->top_k;
  p.top_p = a->top_p;
  p.min_p = a->min_p;
  p.tokens = a->tokens;
  p.logprobs = a->logprobs;
  p.logits_stride = a->logits_stride;
  p.noise_stride = a->noise_stride;
  p.B = a->B;
  p.V = a->V;
  p.temperature_all = a->temperature_all;
  p.top_k_all = a->top_k_all;
  p.top_p_all = a->top_p_all;
  p.min_p_all = a->min_p_all;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = a->dtype == COALIBI_F32    ? launch_sample<2>(p, s)
                 : a->dtype == COALIBI_BF16 ? launch_sample<1>(p, s)
                                            : launch_sample<0>(p, s);
  return rc ? rc : launched("sampling launch");
}
