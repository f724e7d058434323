// What the C entries of the serving operators share: checks of arguments and the launch of the
// paged attention kernels.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstdio>

#include "coalibi.h"
#include "ctx_guard.h"
#include "paged.cuh"

namespace coalibi {

void set_last_error_detail(const char* msg);
int make_page_tmap(CUtensorMap* map, const void* base, int D, int page_size, int heads, int pages,
                   const long long* stride, int dtype, int slots);

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

// The attention kernel of layout L and the kernel that joins its pieces (join: launches it, for `rows` query
// rows that share a kv head).
template <typename L, typename K, typename P, typename J>
int launch_paged(K kernel, J join, std::atomic<unsigned long long>& ready, int threads, const CUtensorMap& tk,
                 const CUtensorMap& tv, P& p, int sms, cudaStream_t s) {
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
  if (e == cudaSuccess && !p.whole) e = join(rows);
  if (e != cudaSuccess) set_last_error_detail(cudaGetErrorString(e));
  return e == cudaSuccess ? launched("paged attention launch") : COALIBI_ERR_LAUNCH;
}

}  // namespace
}  // namespace coalibi
