// Paged key/value cache: appending new tokens (with the position rotation on the
// way) and Co-ALiBi attention of one token or of a tree of drafted tokens over it.
#pragma once

#include "sm100.cuh"
#include "fwd.cuh"

namespace coalibi {

constexpr int kStatusPage = 11;  // COALIBI_ERR_PAGE
constexpr int kTreeMaxSq = 64;   // COALIBI_TREE_MAX_SQ

__device__ __forceinline__ void report_page(int* status) {
  if (status != nullptr) atomicCAS(status, 0, kStatusPage);
}

// ---------------------------------------------------------------------------
// Append.  One CTA per (request, new token); a thread moves 16-byte pieces (8
// elements) of its heads.  A rotated piece also needs its partner's 8 elements (half
// layout) or none (interleaved); the partner is in the same row, so the second load hits L1.
// ---------------------------------------------------------------------------
struct AppendParams {
  const void* k;
  const void* v;
  const void* q;
  void* q_out;
  void* k_pages;
  void* v_pages;
  const int* page_table;
  const int* start;
  const int* count;
  const int* positions;
  const float* cos;
  const float* sin;
  int* status;
  long long ks[3], vs[3], qs[3], qos[3], kps[3], vps[3];
  long long table_stride;
  int Hq, Hkv, S, D;
  int page_size, max_pages, n_pages;
  int rot, n_pos, interleaved;
};

constexpr int kAppendThreads = 256;

// Rotate the 8 elements at column c of row x (rot columns take part).
template <bool BF16>
__device__ __forceinline__ uint4 rotate8(const uint16_t* x, int c, uint4 own, const float* cos, const float* sin,
                                         int rot, int interleaved) {
  uint32_t a[4] = {own.x, own.y, own.z, own.w};
  if (interleaved) {
    const float4 cs = *reinterpret_cast<const float4*>(cos + c / 2);
    const float4 sn = *reinterpret_cast<const float4*>(sin + c / 2);
    const float cc[4] = {cs.x, cs.y, cs.z, cs.w}, ss[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<BF16>(a[i]);
      a[i] = pack2<BF16>(f.x * cc[i] - f.y * ss[i], f.y * cc[i] + f.x * ss[i]);
    }
  } else {
    const int half = rot / 2;
    const bool low = c < half;
    const int j = low ? c : c - half;
    const uint4 other = *reinterpret_cast<const uint4*>(x + (low ? c + half : j));
    const uint32_t o[4] = {other.x, other.y, other.z, other.w};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 cs = *reinterpret_cast<const float4*>(cos + j + 4 * h);
      const float4 sn = *reinterpret_cast<const float4*>(sin + j + 4 * h);
      const float sg = low ? -1.f : 1.f;
      const float2 f0 = unpack2<BF16>(a[2 * h]), f1 = unpack2<BF16>(a[2 * h + 1]);
      const float2 g0 = unpack2<BF16>(o[2 * h]), g1 = unpack2<BF16>(o[2 * h + 1]);
      a[2 * h] = pack2<BF16>(f0.x * cs.x + sg * g0.x * sn.x, f0.y * cs.y + sg * g0.y * sn.y);
      a[2 * h + 1] = pack2<BF16>(f1.x * cs.z + sg * g1.x * sn.z, f1.y * cs.w + sg * g1.y * sn.w);
    }
  }
  return make_uint4(a[0], a[1], a[2], a[3]);
}

template <bool BF16>
__global__ void __launch_bounds__(kAppendThreads) coalibi_paged_append_kernel(const AppendParams p) {
  const int b = blockIdx.x / p.S, i = blockIdx.x - b * p.S;
  const int start = p.start[b];
  const bool fresh = i < (p.count != nullptr ? min(p.count[b], p.S) : p.S);
  const long long tok = (long long)start + i;
  const int pieces = p.D / 8, Hq = p.q != nullptr ? p.Hq : 0;
  bool stored = false;
  long long slot_k = 0, slot_v = 0;
  int pos = 0;
  bool turn = false;
  if (fresh) {
    int page = -1;
    const int at = (int)(tok / p.page_size);
    if (start >= 0 && tok < (long long)p.max_pages * p.page_size) page = p.page_table[(size_t)b * p.table_stride + at];
    stored = page >= 0 && page < p.n_pages;
    const int s = (int)(tok - (long long)at * p.page_size);
    slot_k = page * p.kps[0] + s * p.kps[2];
    slot_v = page * p.vps[0] + s * p.vps[2];
    pos = p.positions != nullptr ? p.positions[(size_t)b * p.S + i] : (int)tok;
    turn = p.rot > 0 && pos >= 0 && pos < p.n_pos;
    if (threadIdx.x == 0 && (!stored || (p.rot > 0 && !turn))) report_page(p.status);
  }
  const float* cos = turn ? p.cos + (size_t)pos * (p.rot / 2) : nullptr;
  const float* sin = turn ? p.sin + (size_t)pos * (p.rot / 2) : nullptr;
  const int items = (2 * p.Hkv + Hq) * pieces;
  for (int it = threadIdx.x; it < items; it += kAppendThreads) {
    const int row = it / pieces, c = (it - row * pieces) * 8;
    const int kind = row < Hq ? 0 : (row < Hq + p.Hkv ? 1 : 2);
    const int h = kind == 0 ? row : (kind == 1 ? row - Hq : row - Hq - p.Hkv);
    if (kind != 0 && !stored) continue;
    const long long* st = kind == 0 ? p.qs : (kind == 1 ? p.ks : p.vs);
    const void* src = kind == 0 ? p.q : (kind == 1 ? p.k : p.v);
    const uint16_t* x = static_cast<const uint16_t*>(src) + b * st[0] + h * st[1] + i * st[2];
    uint4 val = make_uint4(0u, 0u, 0u, 0u);
    if (fresh) {
      val = *reinterpret_cast<const uint4*>(x + c);
      if (kind != 2 && turn && c < p.rot) val = rotate8<BF16>(x, c, val, cos, sin, p.rot, p.interleaved);
    }
    uint16_t* y = kind == 0 ? static_cast<uint16_t*>(p.q_out) + b * p.qos[0] + h * p.qos[1] + i * p.qos[2]
                  : kind == 1 ? static_cast<uint16_t*>(p.k_pages) + slot_k + h * p.kps[1]
                              : static_cast<uint16_t*>(p.v_pages) + slot_v + h * p.vps[1];
    *reinterpret_cast<uint4*>(y + c) = val;
  }
}

// ---------------------------------------------------------------------------
// Attention.  One CTA per (request, query head, row): the keys right to left in
// blocks of 128, one key per thread; a block-wide suffix sum of the sigmoids gives z,
// then an online softmax and, one column per thread, the weighted sum of V.
// ---------------------------------------------------------------------------
struct PagedAttnParams {
  const void* q;
  void* o;
  const void* k_pages;
  const void* v_pages;
  const void* slopes;
  const int* page_table;
  const int* ctx_lens;
  const long long* tree_mask;
  int* status;
  long long qs[3], os[3], kps[3], vps[3];
  long long table_stride, mask_stride;
  int B, Hq, Hkv, Sq;
  int page_size, max_pages, n_pages;
  int slopes_dtype;
  float sm_scale;
};

template <int D, bool BF16>
__global__ void __launch_bounds__(128) coalibi_paged_attn_kernel(const PagedAttnParams p) {
  __shared__ float s_q[D], s_p[128], s_red[8];
  __shared__ long long s_v[128];
  const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, g = h / (p.Hq / p.Hkv);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint16_t* kp = static_cast<const uint16_t*>(p.k_pages) + g * p.kps[1];
  const uint16_t* vp = static_cast<const uint16_t*>(p.v_pages) + g * p.vps[1];
  if (tid < D / 2) {
    const float2 f = unpack2<BF16>(*reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p.q) + b * p.qs[0] +
                                                                      h * p.qs[1] + i * p.qs[2] + 2 * tid));
    s_q[2 * tid] = f.x;
    s_q[2 * tid + 1] = f.y;
  }
  const unsigned long long bits = p.tree_mask != nullptr ? (unsigned long long)p.tree_mask[b * p.mask_stride + i]
                                                         : (2ull << i) - 1;
  const long long room = (long long)p.max_pages * p.page_size;
  const int ctx = max(p.ctx_lens[b], 0);
  const unsigned long long mine = p.Sq < 64 ? bits & ((1ull << p.Sq) - 1) : bits;
  long long end = (long long)ctx + (64 - __clzll((long long)mine));
  if (end > room) {
    end = room;
    if (tid == 0) report_page(p.status);
  }
  const float slope = load_slope(p.slopes, p.slopes_dtype, h);
  float m = -INFINITY, l = 0.f, carry = 0.f, o = 0.f;
  __syncthreads();
  for (long long hi = end; hi > 0; hi -= 128) {
    // thread tid takes key hi - 1 - tid: the block's prefix sums are sums over the keys to the right
    const long long key = hi - 1 - tid;
    bool seen = key >= 0 && (key < ctx || (mine >> (key - ctx) & 1));
    long long ko = 0;
    s_v[tid] = -1;
    if (seen) {
      const int at = (int)(key / p.page_size), slot = (int)(key - (long long)at * p.page_size);
      const int page = p.page_table[(size_t)b * p.table_stride + at];
      seen = page >= 0 && page < p.n_pages;
      if (!seen) report_page(p.status);
      if (seen) {
        ko = page * p.kps[0] + slot * p.kps[2];
        s_v[tid] = page * p.vps[0] + slot * p.vps[2];
      }
    }
    float dot = 0.f;
    if (seen) {
      for (int c = 0; c < D; c += 8) {
        const uint4 u = *reinterpret_cast<const uint4*>(kp + ko + c);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = unpack2<BF16>(w[j]);
          dot = fmaf(f.x, s_q[c + 2 * j], dot);
          dot = fmaf(f.y, s_q[c + 2 * j + 1], dot);
        }
      }
    }
    const float x = dot * p.sm_scale;
    const float sg = seen ? 1.f / (1.f + expf(-x)) : 0.f;
    float inc = sg;
    for (int d = 1; d < 32; d <<= 1) {
      const float y = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += y;
    }
    if (lane == 31) s_red[warp] = inc;
    __syncthreads();
    float left = carry;
    for (int w = 0; w < 4; ++w) {
      if (w < warp) left += s_red[w];
      carry += s_red[w];
    }
    const float a = seen ? x - slope * (inc + left) : -INFINITY;
    float mx = a;
    for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    if (lane == 0) s_red[4 + warp] = mx;
    __syncthreads();
    const float m_new = fmaxf(fmaxf(fmaxf(s_red[4], s_red[5]), fmaxf(s_red[6], s_red[7])), m);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float fac = m == -INFINITY ? 0.f : expf(m - m_use);
    s_p[tid] = a == -INFINITY ? 0.f : expf(a - m_use);
    m = m_new;
    l *= fac;
    o *= fac;
    __syncthreads();
    for (int j = 0; j < 128; ++j) {
      const float w = s_p[j];
      l += w;
      if (s_v[j] < 0 || tid >= D) continue;
      const uint16_t e = vp[s_v[j] + tid];
      o = fmaf(w, BF16 ? __bfloat162float(__ushort_as_bfloat16(e)) : __half2float(__ushort_as_half(e)), o);
    }
    __syncthreads();
  }
  if (tid < D) {
    const float r = l > 0.f ? o / l : 0.f;
    uint16_t* y = static_cast<uint16_t*>(p.o) + b * p.os[0] + h * p.os[1] + i * p.os[2];
    y[tid] = BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(r)) : __half_as_ushort(__float2half_rn(r));
  }
}

}  // namespace coalibi
