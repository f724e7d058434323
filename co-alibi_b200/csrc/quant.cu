// C-ABI entry points of the paged cache in 8 bits (declared in include/coalibi.h): append, read
// back, attention.  Arguments are checked before any device use; nothing here allocates or
// synchronises.
#include <cuda_runtime.h>

#include <algorithm>

#include "paged8_wide.cuh"
#include "serving_host.cuh"

using namespace coalibi;

namespace coalibi {
namespace {

// Codes stand in rows of 16-byte multiples; a scale for each block of each head of each page.
int check_codes(const CoalibiCacheScales* s, const void* k_pages, const void* v_pages, const long long* k_stride,
                const long long* v_stride, int n_pages, int heads) {
  for (int i = 0; i < 3; ++i)
    if (k_stride[i] % 16 != 0 || v_stride[i] % 16 != 0) return COALIBI_ERR_ALIGNMENT;
  if (!aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(s->k, 4) || !aligned(s->v, 4))
    return COALIBI_ERR_ALIGNMENT;
  const int sizes[2] = {n_pages, heads};
  for (int i = 0; i < 2; ++i)
    for (long long stride : {s->k_stride[i], s->v_stride[i]})
      if (stride < 0 || (sizes[i] > 1 && stride == 0)) return COALIBI_ERR_SHAPE;
  return COALIBI_OK;
}

// log2 of the page size, or -1.
int page_shift_of(int page_size) {
  for (int k = 4; k < 31; ++k)
    if (page_size == 1 << k) return k;
  return -1;
}

void copy2(long long* dst, const long long* src) { dst[0] = src[0], dst[1] = src[1]; }

template <bool BF16, int D>
auto append8_kernel(int turn) {
  return turn == kTurnNone    ? coalibi_paged_append8_kernel<BF16, D, kTurnNone>
         : turn == kTurnPairs ? coalibi_paged_append8_kernel<BF16, D, kTurnPairs>
                              : coalibi_paged_append8_kernel<BF16, D, kTurnHalves>;
}

template <bool BF16, int D>
auto queries_kernel(int turn) {
  return turn == kTurnNone    ? coalibi_paged_append_kernel<BF16, D, kTurnNone>
         : turn == kTurnPairs ? coalibi_paged_append_kernel<BF16, D, kTurnPairs>
                              : coalibi_paged_append_kernel<BF16, D, kTurnHalves>;
}

template <int D, bool BF16, int NT, int RW, int WARPS, bool HALF>
int launch_attention8(const CUtensorMap& tk, const CUtensorMap& tv, Paged8Params& p, int sms, cudaStream_t s) {
  static std::atomic<unsigned long long> ready{0};
  using L = Paged8Layout<D, NT, RW, WARPS>;
  // A CTA joins a row where items come in many pieces, a warp where they come in few.  With a warp / a CTA to a
  // row: contexts in some 50 pieces 15 / 6 us, a ragged decode batch 7.5 / 4.4, 4096 rows of 2 to 3 pieces (of
  // the wide kernel) 4.7 / 12.7.
  const auto join = [&p, s](int rows) {
    const PagedAttnParams& a = p;
    if ((long long)p.n_ctas > 8LL * p.B * p.Hkv * p.row_blocks)
      return launch_pdl(coalibi_paged8_join_kernel<D, BF16, L>, dim3(p.B * p.Hkv, rows), dim3(kJoinThreads), 0, s, a);
    return launch_pdl(coalibi_paged_join_kernel<D, BF16, L>, dim3(p.B * p.Hkv, (rows + 3) / 4), dim3(128), 0, s, a);
  };
  return launch_paged<L>(coalibi_paged8_attn_kernel<D, BF16, NT, RW, WARPS, HALF>, join, ready, 32 * WARPS, tk, tv, p, sms, s);
}

// Four warps to an item where the tables hold little work, else as many as its rows take (as in the
// 16-bit attention).  Items of up to 32 rows.
bool shares_items(const Paged8Params& p, int sms) {
  const long long items = (long long)p.B * p.Hkv, width = (long long)p.max_pages * p.page_size;
  return !(items > 2LL * sms || (width > 512 && items * width > 32768));
}
template <int D, bool BF16, int NT, int RW, bool HALF = false>
int launch_rows8(const CUtensorMap& tk, const CUtensorMap& tv, Paged8Params& p, int sms, cudaStream_t s) {
  return shares_items(p, sms) ? launch_attention8<D, BF16, NT, RW, 4, HALF>(tk, tv, p, sms, s)
                              : launch_attention8<D, BF16, NT, RW, RW, HALF>(tk, tv, p, sms, s);
}

template <int D, bool BF16>
int launch_wide8(const CUtensorMap& tk, const CUtensorMap& tv, Paged8Params& p, int sms, cudaStream_t s) {
  static std::atomic<unsigned long long> ready{0};
  using L = Wide8Layout<D>;
  const auto join = [&p, s](int rows) {
    return launch_pdl(coalibi_paged_join_kernel<D, BF16, L>, dim3(p.B * p.Hkv, (rows + 3) / 4), dim3(128), 0, s,
                      static_cast<const PagedAttnParams&>(p));
  };
  return launch_paged<L>(coalibi_paged8_wide_kernel<D, BF16>, join, ready, L::THREADS, tk, tv, p, sms, s);
}

template <int D, bool BF16>
int launch_paged8(const CUtensorMap& tk, const CUtensorMap& tv, Paged8Params& p, int sms, cudaStream_t s) {
  const int rows = p.Hq / p.Hkv * p.Sq;
  // Up to 4 rows lanes share what 8 columns leave over (4 rows of long contexts, without / with it: 127 / 124 us of kernel;
  // the shuffles it takes would buy nothing with more rows).  The wide kernel costs the same for 1 to 64 rows.  8 ragged
  // contexts up to 16k keys, narrow / wide: 16 rows 55 / 70 us, 20 rows 73 / 71, 32 rows 78 / 71 (bfloat16 81 / 71); 32 rows
  // of 64 contexts of 200 keys 27 / 58, of 1000 keys 89 / 98; 32 rows of D = 64 56 / 65.
  if (rows <= 4) return launch_rows8<D, BF16, 1, 1, true>(tk, tv, p, sms, s);
  if (rows <= 8) return launch_rows8<D, BF16, 1, 1>(tk, tv, p, sms, s);
  if (rows <= 16) return launch_rows8<D, BF16, 2, 1>(tk, tv, p, sms, s);
  if (rows <= 32) return launch_rows8<D, BF16, 2, 2>(tk, tv, p, sms, s);
  return launch_wide8<D, BF16>(tk, tv, p, sms, s);
}

template <int D>
size_t paged8_ws(int B, int rows) {
  if (rows <= 8) return std::max(paged_ws_bytes<Paged8Layout<D, 1, 1, 1>>(B), paged_ws_bytes<Paged8Layout<D, 1, 1, 4>>(B));
  if (rows <= 16) return std::max(paged_ws_bytes<Paged8Layout<D, 2, 1, 1>>(B), paged_ws_bytes<Paged8Layout<D, 2, 1, 4>>(B));
  if (rows <= 32) return std::max(paged_ws_bytes<Paged8Layout<D, 2, 2, 2>>(B), paged_ws_bytes<Paged8Layout<D, 2, 2, 4>>(B));
  return paged_ws_bytes<Wide8Layout<D>>(B);
}

}  // namespace
}  // namespace coalibi

extern "C" int coalibi_paged_append8(const CoalibiPagedAppendArgs* a, const CoalibiCacheScales* sc, void* stream) {
  if (a == nullptr || sc == nullptr || !sc->k || !sc->v || !a->k || !a->v || !a->k_pages || !a->v_pages ||
      !a->page_table || !a->start)
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
  if (!aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->q, 16) || !aligned(a->q_out, 16) || !aligned(a->cos, 16) ||
      !aligned(a->sin, 16))
    return COALIBI_ERR_ALIGNMENT;
  if ((rc = check_codes(sc, a->k_pages, a->v_pages, a->k_page_stride, a->v_page_stride, a->n_pages, a->Hkv))) return rc;
  Append8Params p{};
  p.blocks = (int)(((long long)a->S + kQuantBlock - 2) / kQuantBlock) + 1;
  // a head to a warp, up to eight warps to a CTA
  p.chunks = (a->Hkv + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
  const int threads = 32 * ((a->Hkv + p.chunks - 1) / p.chunks);
  const long long kv_ctas = (long long)a->B * p.blocks * 2 * p.chunks;
  if (kv_ctas > 0x7fffffffLL) return COALIBI_ERR_SHAPE;
  CtxGuard guard;
  if ((rc = enter_device(a->k_pages, stream))) return rc;
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
  p.k_scales = sc->k;
  p.v_scales = sc->v;
  copy2(p.kss, sc->k_stride);
  copy2(p.vss, sc->v_stride);
  p.page_shift = page_shift_of(a->page_size);
  p.kv_ctas = (int)kv_ctas;
  p.group = p.tokens >= 8LL * kAppendGroup * device_sm_count() ? kAppendGroup : 1;
  const long long q_ctas = a->q != nullptr ? (p.tokens + p.group - 1) / p.group : 0;
  if (p.kv_ctas + q_ctas > 0x7fffffffLL) return COALIBI_ERR_SHAPE;
  const bool bf16 = a->dtype == COALIBI_BF16;
  const int turn = a->rot == 0 ? kTurnNone : a->interleaved ? kTurnPairs : kTurnHalves;
  auto kernel = a->D == 128 ? (bf16 ? append8_kernel<true, 128>(turn) : append8_kernel<false, 128>(turn))
                            : (bf16 ? append8_kernel<true, 64>(turn) : append8_kernel<false, 64>(turn));
  // The queries of few tokens go in the same launch; those of many in one of their own (the 16-bit append's kernel
  // without keys), whose CTAs take half the registers.  8 kv and 32 query heads of 128, together / apart: 1000 tokens
  // 14 / 17 us, 4000 30 / 32, 8000 51 / 48, 16,000 92 / 81.
  const bool apart = q_ctas > 0 && p.tokens >= 40LL * device_sm_count();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = launch_pdl(kernel, dim3((unsigned)(p.kv_ctas + (apart ? 0 : q_ctas))), dim3(threads), 0, s, p);
  if (e == cudaSuccess && apart) {
    AppendParams q = p;
    q.Hkv = 0;
    auto queries = a->D == 128 ? (bf16 ? queries_kernel<true, 128>(turn) : queries_kernel<false, 128>(turn))
                               : (bf16 ? queries_kernel<true, 64>(turn) : queries_kernel<false, 64>(turn));
    e = launch_pdl(queries, dim3((unsigned)q_ctas), dim3(kAppendThreads), 0, s, q);
  }
  if (e != cudaSuccess) {
    set_last_error_detail(cudaGetErrorString(e));
    return COALIBI_ERR_LAUNCH;
  }
  return launched("paged append launch");
}

extern "C" int coalibi_paged_read8(const CoalibiPagedReadArgs* a, const CoalibiCacheScales* sc, void* stream) {
  if (a == nullptr || sc == nullptr || !sc->k || !sc->v || !a->k || !a->v || !a->k_pages || !a->v_pages ||
      !a->page_table || !a->positions)
    return COALIBI_ERR_NULL_POINTER;
  int rc = check_cache(a->B, a->Hkv, a->D, a->page_size, a->max_pages, a->n_pages, a->dtype, a->k_page_stride,
                       a->v_page_stride, a->table_stride);
  if (rc) return rc;
  if (a->S <= 0) return COALIBI_ERR_SHAPE;
  if (!aligned(a->k, 32) || !aligned(a->v, 32) || !aligned(a->positions, 4)) return COALIBI_ERR_ALIGNMENT;
  if ((rc = check_codes(sc, a->k_pages, a->v_pages, a->k_page_stride, a->v_page_stride, a->n_pages, a->Hkv))) return rc;
  Read8Params p{};
  const int tokens = kReadThreads / (a->D / 16);
  p.chunks = (a->S - 1) / tokens + 1;
  if ((long long)a->B * p.chunks > 0x7fffffffLL || a->Hkv > 32767) return COALIBI_ERR_SHAPE;
  CtxGuard guard;
  if ((rc = enter_device(a->k_pages, stream))) return rc;
  p.k_pages = a->k_pages;
  p.v_pages = a->v_pages;
  p.k_scales = sc->k;
  p.v_scales = sc->v;
  p.page_table = a->page_table;
  p.positions = a->positions;
  p.k = a->k;
  p.v = a->v;
  p.status = a->status;
  copy3(p.kps, a->k_page_stride);
  copy3(p.vps, a->v_page_stride);
  copy2(p.kss, sc->k_stride);
  copy2(p.vss, sc->v_stride);
  p.table_stride = a->table_stride;
  p.Hkv = a->Hkv;
  p.S = a->S;
  // All heads to a CTA where tokens are plenty, so that they are looked up once, else fewer, so that every SM has
  // some.  8 heads of 128, all / one to a CTA: 144 tokens 10 / 6 us, 2000 10 / 10 (four to a CTA 8), 16,000 23 / 35,
  // 65,536 72 / 123.
  p.per = 2 * a->Hkv;
  while (p.per > 1 && (long long)a->B * p.chunks * (2 * a->Hkv / p.per) < 2LL * device_sm_count()) p.per = (p.per + 1) / 2;
  p.page_size = a->page_size;
  p.max_pages = a->max_pages;
  p.n_pages = a->n_pages;
  p.page_shift = page_shift_of(a->page_size);
  const bool bf16 = a->dtype == COALIBI_BF16;
  auto kernel = a->D == 128 ? (bf16 ? coalibi_paged_read8_kernel<true, 128> : coalibi_paged_read8_kernel<false, 128>)
                            : (bf16 ? coalibi_paged_read8_kernel<true, 64> : coalibi_paged_read8_kernel<false, 64>);
  const dim3 grid((unsigned)(a->B * p.chunks), (2 * a->Hkv + p.per - 1) / p.per);
  if (const cudaError_t e = launch_pdl(kernel, grid, dim3(kReadThreads), 0, static_cast<cudaStream_t>(stream), p);
      e != cudaSuccess) {
    set_last_error_detail(cudaGetErrorString(e));
    return COALIBI_ERR_LAUNCH;
  }
  return launched("paged read launch");
}

extern "C" size_t coalibi_paged_attention8_workspace_bytes(int B, int Hq, int Hkv, int Sq, int D) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq <= 0 || Sq > kTreeMaxSq || Hq % Hkv != 0 || (D != 64 && D != 128)) return 0;
  return D == 128 ? paged8_ws<128>(B, Hq / Hkv * Sq) : paged8_ws<64>(B, Hq / Hkv * Sq);
}

extern "C" int coalibi_paged_attention8(const CoalibiPagedAttentionArgs* a, const CoalibiCacheScales* sc, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  if (a == nullptr || sc == nullptr || !sc->k || !sc->v || !a->q || !a->o || !a->k_pages || !a->v_pages || !a->slopes ||
      !a->page_table || !a->ctx_lens)
    return COALIBI_ERR_NULL_POINTER;
  int rc = check_cache(a->B, a->Hkv, a->D, a->page_size, a->max_pages, a->n_pages, a->dtype, a->k_page_stride,
                       a->v_page_stride, a->table_stride);
  if (rc) return rc;
  if (a->slopes_dtype != COALIBI_F16 && a->slopes_dtype != COALIBI_BF16 && a->slopes_dtype != COALIBI_F32)
    return COALIBI_ERR_DTYPE;
  if (a->Hq <= 0 || a->Hq % a->Hkv != 0 || a->Hq > 65535 || a->Sq <= 0 || a->Sq > kTreeMaxSq || a->mask_stride < 0)
    return COALIBI_ERR_SHAPE;
  if (!row_strides(a->q_stride) || !row_strides(a->o_stride)) return COALIBI_ERR_ALIGNMENT;
  if (!aligned(a->q, 16) || !aligned(a->o, 16) || !aligned(a->tree_mask, 8)) return COALIBI_ERR_ALIGNMENT;
  if ((rc = check_codes(sc, a->k_pages, a->v_pages, a->k_page_stride, a->v_page_stride, a->n_pages, a->Hkv))) return rc;
  if (workspace == nullptr || !aligned(workspace, 16) ||
      workspace_bytes < coalibi_paged_attention8_workspace_bytes(a->B, a->Hq, a->Hkv, a->Sq, a->D))
    return COALIBI_ERR_WORKSPACE;
  CtxGuard guard;
  if ((rc = enter_device(a->k_pages, stream))) return rc;
  Paged8Params p{};
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
  p.ws = static_cast<float*>(workspace);
  p.page_shift = page_shift_of(a->page_size);
  p.k_scales = sc->k;
  p.v_scales = sc->v;
  copy2(p.kss, sc->k_stride);
  copy2(p.vss, sc->v_stride);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = a->dtype == COALIBI_BF16;
  const int sms = device_sm_count();
  // Loads of 32 slots where a warp walks whole steps and no step crosses a page; the 16-slot form
  // serves the rest (its warps share an item, or pages end within a step).
  const bool narrow = a->Hq / a->Hkv * a->Sq <= 32;
  p.box = narrow && a->page_size % 32 == 0 && !shares_items(p, sms) ? 32 : 16;
  CUtensorMap tk, tv;
  if ((rc = make_page_tmap(&tk, a->k_pages, a->D, a->page_size, a->Hkv, a->n_pages, a->k_page_stride, COALIBI_E4M3, p.box))) return rc;
  if ((rc = make_page_tmap(&tv, a->v_pages, a->D, a->page_size, a->Hkv, a->n_pages, a->v_page_stride, COALIBI_E4M3, p.box))) return rc;
  if (a->D == 128) return bf16 ? launch_paged8<128, true>(tk, tv, p, sms, s) : launch_paged8<128, false>(tk, tv, p, sms, s);
  return bf16 ? launch_paged8<64, true>(tk, tv, p, sms, s) : launch_paged8<64, false>(tk, tv, p, sms, s);
}
