// Paged key/value cache in 8 bits: e4m3 codes with one scale for each block of 16 tokens and
// head, a power of two.  Appending (with the position rotation on the way), reading back, and
// Co-ALiBi attention over it.
//
// With a power of two for a scale nothing but the exponent moves: a code keeps its three mantissa
// bits whatever the scale is, so raising a block's scale for a larger token that joins it later
// leaves the tokens before it as they are (only what falls below 2^-6 of the new scale rounds), and a
// token that is read back whole (in bfloat16) and appended again, under a scale that does not grow, gets the same code.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "paged.cuh"

namespace coalibi {

constexpr int kQuantBlock = 16;        // tokens that share a scale
constexpr float kE4m3Max = 448.f;
constexpr int kScaleMinExp = -100;     // its inverse is a normal float32 too
// Scales of V that are 0, negative or far from 1 take the attention's masked steps (below).
constexpr float kScaleHeldMin = 0x1p-100f, kScaleHeldMax = 0x1p126f;
__device__ __forceinline__ bool odd_scale(float s) {  // not within [2^-40, 2^40)
  return __float_as_uint(s) - (87u << 23) >= (80u << 23);
}

__device__ __forceinline__ uint32_t e4m3_to_f16x2(uint32_t two) {  // the low 16 bits
  uint32_t h;
  asm("{ .reg .b16 t; cvt.u16.u32 t, %1; cvt.rn.f16x2.e4m3x2 %0, t; }" : "=r"(h) : "r"(two));
  return h;
}
__device__ __forceinline__ void e4m3_to_f16x4(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{ .reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b; }"
      : "=r"(lo), "=r"(hi)
      : "r"(four));
}
// Four codes, the first in the low byte.  NaN gives the code of NaN.
__device__ __forceinline__ uint32_t e4m3_from(float a, float b, float c, float d) {
  uint32_t r;
  asm("{ .reg .b16 x, y; cvt.rn.satfinite.e4m3x2.f32 x, %2, %1; cvt.rn.satfinite.e4m3x2.f32 y, %4, %3; mov.b32 %0, {x, y}; }"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
__device__ __forceinline__ float2 f16x2_to_float2(uint32_t h) { return __half22float2(*reinterpret_cast<__half2*>(&h)); }

// The least power of two s >= 2^-100 with most <= 448 s; most >= 0 and finite.
__device__ __forceinline__ float quant_scale(float most) {
  const int bits = __float_as_int(most);
  // most = m 2^e, 1 <= m < 2, and 448 = 1.75 * 2^8 (a subnormal counts as 2^-127)
  const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000);
  return __int_as_float((max(e, kScaleMinExp) + 127) << 23);
}

// For a scale that is no power of two (only another program writes one; a block keeps it where it is large enough): a
// result in 24 bits towards zero, its last bit set where it is not exact, so that it rounds to a code as the exact one would.
__device__ __forceinline__ float to_odd(float x, float rest) {  // the exact value is x and something of rest's sign
  const uint32_t u = __float_as_uint(x), back = ((__float_as_uint(rest) ^ u) >> 31) & 1u;
  return rest == 0.f ? x : __uint_as_float((u - back) | 1u);
}
__device__ __forceinline__ float quotient_to_odd(float y, float s, float inv) {  // s > 0, inv = 1 / s
  float q = y * inv;
  q = fmaf(fmaf(-q, s, y), inv, q);
  return to_odd(q, fmaf(-q, s, y));
}
__device__ __forceinline__ float product_to_odd(float a, float b) {
  const float x = a * b;
  return to_odd(x, fmaf(a, b, -x));
}

// ---------------------------------------------------------------------------
// Append.  Of each block of 16 tokens and head, y the new tokens' values (keys turned by their angles, each product
// and sum rounded to float32 by itself):
//   s = max(the least 2^k, k >= -100, with max |y| <= 448 2^k; the scale of tokens that the block holds already),
//   code = e4m3(y / s), and where s grew, old codes = e4m3(old code * (old s / s)).
//
// Bound by the bytes where tokens are many (2 read for 1 written) and by the launch where they are few.  A
// warp has a block of one head, so that the largest value is a reduction of the warp and no block is written by two.  Its
// 16 rows stay in registers in 16 bits and are turned twice, for the largest and for the codes: in float32 they took
// twice the registers and half the warps (8 ragged prompts of up to 2000 tokens 62 us, 53 so, as keys, values and blocks also became CTAs of
// their own, whose warps share the angles).  Queries go on beside them or, where they are many, in a launch of
// their own.  Of those 53 us (the bytes take 38) the keys and values of 8 heads of 128 take 19 and the queries of 32
// heads 36, side by side at their ends; one token for each of 256 requests takes 6.3 us.
// ---------------------------------------------------------------------------
struct Append8Params : AppendParams {
  float* k_scales;
  float* v_scales;
  long long kss[2], vss[2];  // page, head
  int page_shift;            // log2(page_size), or -1
  int blocks;                // that a request's S tokens may touch
  int chunks;                // of the Hkv heads, one head to a warp
  int kv_ctas;               // B * blocks * 2 chunks
};

template <bool BF16, int D, int TURN>
__global__ void __launch_bounds__(kAppendThreads, 4) coalibi_paged_append8_kernel(const Append8Params p) {
  constexpr int PIECES = D / 8;
  __shared__ __align__(16) float s_angle[TURN == kTurnNone ? 1 : 2][TURN == kTurnNone ? 4 : kQuantBlock * D / 2];
  __shared__ bool s_turned[kQuantBlock];  // whether a token has angles
  grid_dep_wait();
  const int tid = threadIdx.x, half = p.rot / 2;
  if ((int)blockIdx.x >= p.kv_ctas) {  // ---- queries: a thread keeps its column, as in the 16-bit append
    const long long first = (long long)((int)blockIdx.x - p.kv_ctas) * p.group;
    const int n = (int)min((long long)p.group, p.tokens - first);
    const int step = blockDim.x / PIECES, r0 = tid / PIECES, c = (tid % PIECES) * 8;
    const int partner = c < half ? half : -half;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    for (int k = 0; k < n; ++k) {
      const int b = (int)(first + k) / p.S, i = (int)(first + k) - b * p.S;
      const bool fresh = i < (p.count != nullptr ? p.count[b] : p.S);
      const uint16_t* x = static_cast<const uint16_t*>(p.q) + b * p.qs[0] + i * p.qs[2] + r0 * p.qs[1] + c;
      uint16_t* y = static_cast<uint16_t*>(p.q_out) + b * p.qos[0] + i * p.qos[2] + r0 * p.qos[1] + c;
      const long long dx = step * p.qs[1], dy = step * p.qos[1];
      if (!fresh) {
        for (int row = r0; row < p.Hq; row += step, y += dy) *reinterpret_cast<uint4*>(y) = zero;
        continue;
      }
      bool turn = false;
      Angles<TURN> g;
      if (TURN != kTurnNone && c < p.rot) {
        const long long pos = p.positions != nullptr ? p.positions[(size_t)b * p.S + i] : (long long)p.start[b] + i;
        turn = pos >= 0 && pos < p.n_pos;
        if (turn) g.load(p.cos + (size_t)pos * half, p.sin + (size_t)pos * half, c, half);
      }
#pragma unroll 2
      for (int row = r0; row < p.Hq; row += step, x += dx, y += dy) {
        uint4 val = *reinterpret_cast<const uint4*>(x);
        if (turn)
          val = g.template turn<BF16>(val, TURN == kTurnHalves ? *reinterpret_cast<const uint4*>(x + partner) : zero);
        *reinterpret_cast<uint4*>(y) = val;
      }
    }
    return;
  }
  // ---- keys or values: a warp takes the 16 tokens of a block for one head.  Keys and values, and blocks, are
  // CTAs of their own, so that the warps of one share the tokens' angles.
  const int lane = tid & 31;
  const int at = blockIdx.x / (2 * p.chunks), part = blockIdx.x - at * 2 * p.chunks;
  const int b = at / p.blocks, j = at - b * p.blocks;
  const bool key = part < p.chunks;
  const int h = (key ? part : part - p.chunks) * (blockDim.x / 32) + (tid >> 5);
  const int start = p.start[b];
  const int fresh = min(p.count != nullptr ? p.count[b] : p.S, p.S);
  if (fresh <= 0) return;
  if (start < 0) {
    if (tid == 0) report_page(p.status);
    return;
  }
  const long long t0 = ((long long)(start / kQuantBlock) + j) * kQuantBlock;  // the block's first token
  // its tokens of this call
  const int lo = (int)max((long long)start - t0, 0ll), hi = (int)min((long long)start + fresh - t0, (long long)kQuantBlock);
  if (lo >= hi) return;
  constexpr int RPW = 32 / PIECES, N = kQuantBlock / RPW;  // rows of a pass of the warp, passes
  const int l = lane % PIECES, r0 = lane / PIECES;
  // A lane's 8 columns: where it turns in halves, 4 and their partners; else neighbours.
  const bool turns = TURN != kTurnNone && key && 8 * l < p.rot, split = TURN == kTurnHalves && turns;
  const int ca = split ? 4 * l : 8 * l, cb = split ? half + 4 * l : 8 * l + 4;
  uint4 raw[N];
  {
    const long long* xs = key ? p.ks : p.vs;
    const uint16_t* x = static_cast<const uint16_t*>(key ? p.k : p.v) + b * xs[0] + h * xs[1] + (t0 - start + r0) * xs[2];
    const long long step = RPW * xs[2];
#pragma unroll
    for (int i = 0; i < N; ++i, x += step) {
      const int r = r0 + i * RPW;
      raw[i] = make_uint4(0u, 0u, 0u, 0u);
      if (r >= lo && r < hi && h < p.Hkv) {
        if (split) {
          const uint2 u = *reinterpret_cast<const uint2*>(x + ca), v = *reinterpret_cast<const uint2*>(x + cb);
          raw[i] = make_uint4(u.x, u.y, v.x, v.y);
        } else {
          raw[i] = *reinterpret_cast<const uint4*>(x + ca);
        }
      }
    }
  }
  int page = -1, slot = 0;
  if (t0 < (long long)p.max_pages * p.page_size) {
    const int n = p.page_shift >= 0 ? (int)t0 >> p.page_shift : (int)t0 / p.page_size;
    slot = (int)t0 - n * p.page_size;
    page = p.page_table[(size_t)b * p.table_stride + n];
  }
  if (TURN != kTurnNone && key) {
    const int row4 = half / 4;  // pieces of a row
    for (int e = tid; e < kQuantBlock * row4; e += blockDim.x) {
      const int r = e / row4, c = (e - r * row4) * 4;
      if (r < lo || r >= hi) continue;
      const long long pos = p.positions != nullptr ? p.positions[(size_t)b * p.S + (t0 + r - start)] : t0 + r;
      const bool has = pos >= 0 && pos < p.n_pos;
      if (c == 0) s_turned[r] = has;
      if (has) {
        *reinterpret_cast<float4*>(&s_angle[0][r * half + c]) = *reinterpret_cast<const float4*>(p.cos + (size_t)pos * half + c);
        *reinterpret_cast<float4*>(&s_angle[1][r * half + c]) = *reinterpret_cast<const float4*>(p.sin + (size_t)pos * half + c);
      } else if (c == 0) {
        report_page(p.status);
      }
    }
    __syncthreads();
  }
  if (h >= p.Hkv) return;
  if (page < 0 || page >= p.n_pages) {
    if (lane == 0) report_page(p.status);
    return;
  }
  float* scale_at = (key ? p.k_scales + page * p.kss[0] + h * p.kss[1] : p.v_scales + page * p.vss[0] + h * p.vss[1]) +
                    slot / kQuantBlock;
  const float was = lo > 0 ? *scale_at : 0.f;  // the block holds tokens already
  // Row i: f[0], f[1] and f[2], f[3] are the a and the b of pairs (a, b); without a rotation, the columns in order.
  // Computed twice, for the block's largest and for the codes: the rows in float32 would take twice the registers
  // and leave half the warps.
  auto values = [&](int i, float2* f) {
    const float2 w[4] = {unpack2<BF16>(raw[i].x), unpack2<BF16>(raw[i].y), unpack2<BF16>(raw[i].z), unpack2<BF16>(raw[i].w)};
    if (TURN == kTurnPairs) {
      f[0] = make_float2(w[0].x, w[1].x), f[1] = make_float2(w[2].x, w[3].x);
      f[2] = make_float2(w[0].y, w[1].y), f[3] = make_float2(w[2].y, w[3].y);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = w[e];
    }
    const int r = r0 + i * RPW;
    if (!turns || r < lo || r >= hi || !s_turned[r]) return;
    const float4 c4 = *reinterpret_cast<const float4*>(&s_angle[0][r * half + 4 * l]);
    const float4 s4 = *reinterpret_cast<const float4*>(&s_angle[1][r * half + 4 * l]);
    // products and their sum rounded one by one: the same codes as plain float32 arithmetic gives
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float2 cs = e ? make_float2(c4.z, c4.w) : make_float2(c4.x, c4.y);
      const float2 sn = e ? make_float2(s4.z, s4.w) : make_float2(s4.x, s4.y);
      const float2 u = f[e], v = f[2 + e], vs = __fmul2_rn(v, sn);
      f[e] = __fadd2_rn(__fmul2_rn(u, cs), make_float2(-vs.x, -vs.y));
      f[2 + e] = __fadd2_rn(__fmul2_rn(v, cs), __fmul2_rn(u, sn));
    }
  };
  auto some = [&](int i) { return i * RPW < hi && (i + 1) * RPW > lo; };  // whether row i of any lane is new
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (!some(i)) continue;
    float2 f[4];
    values(i, f);
#pragma unroll
    for (int e = 0; e < 4; ++e) most = fmaxf(most, fmaxf(fabsf(f[e].x), fabsf(f[e].y)));  // (passes over NaN)
  }
  const bool infinite = __any_sync(0xffffffffu, most == INFINITY);
  if (infinite) {  // an infinity has no code: NaN, not the block's largest
    most = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float2 f[4];
      values(i, f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        most = fmaxf(most, fabsf(f[e].x) == INFINITY ? 0.f : fabsf(f[e].x));
        most = fmaxf(most, fabsf(f[e].y) == INFINITY ? 0.f : fabsf(f[e].y));
      }
    }
  }
  most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
  const float scale = fmaxf(quant_scale(most), was), inv = 1.f / scale;
  uint8_t* y = static_cast<uint8_t*>(key ? p.k_pages : p.v_pages) +
               (key ? page * p.kps[0] + h * p.kps[1] + (slot + r0) * p.kps[2] : page * p.vps[0] + h * p.vps[1] + (slot + r0) * p.vps[2]);
  const long long step = RPW * (key ? p.kps[2] : p.vps[2]);
  if (lo > 0 && scale != was) {  // the tokens that the block held: the same values by the new scale
    const float ratio = was / scale;
    uint8_t* at_old = y + 8 * l;
#pragma unroll 1
    for (int r = r0; r < lo; r += RPW, at_old += step) {
      const uint2 u = *reinterpret_cast<const uint2*>(at_old);
      uint32_t g[4];
      e4m3_to_f16x4(u.x, g[0], g[1]);
      e4m3_to_f16x4(u.y, g[2], g[3]);
      float2 v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 u = f16x2_to_float2(g[e]);
        v[e] = make_float2(product_to_odd(u.x, ratio), product_to_odd(u.y, ratio));
      }
      *reinterpret_cast<uint2*>(at_old) =
          make_uint2(e4m3_from(v[0].x, v[0].y, v[1].x, v[1].y), e4m3_from(v[2].x, v[2].y, v[3].x, v[3].y));
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)  // (so that nothing of the first pass is kept for the codes)
    asm volatile("" : "+r"(raw[i].x), "+r"(raw[i].y), "+r"(raw[i].z), "+r"(raw[i].w));
  auto store = [&](auto power_of_two) {
#pragma unroll
    for (int i = 0; i < N; ++i, y += step) {
      const int r = r0 + i * RPW;
      if (some(i) && r >= lo && r < hi) {
        float2 f[4];
        values(i, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (infinite && fabsf(f[e].x) == INFINITY) f[e].x = __int_as_float(0x7fc00000);
          if (infinite && fabsf(f[e].y) == INFINITY) f[e].y = __int_as_float(0x7fc00000);
          if (decltype(power_of_two)::value)
            f[e] = __fmul2_rn(f[e], make_float2(inv, inv));
          else
            f[e] = make_float2(quotient_to_odd(f[e].x, scale, inv), quotient_to_odd(f[e].y, scale, inv));
        }
        uint2 codes;
        if (TURN == kTurnPairs)
          codes = make_uint2(e4m3_from(f[0].x, f[2].x, f[0].y, f[2].y), e4m3_from(f[1].x, f[3].x, f[1].y, f[3].y));
        else
          codes = make_uint2(e4m3_from(f[0].x, f[0].y, f[1].x, f[1].y), e4m3_from(f[2].x, f[2].y, f[3].x, f[3].y));
        if (split) {
          *reinterpret_cast<uint32_t*>(y + ca) = codes.x;
          *reinterpret_cast<uint32_t*>(y + cb) = codes.y;
        } else {
          *reinterpret_cast<uint2*>(y + ca) = codes;
        }
      }
    }
  };
  if ((__float_as_uint(scale) & 0x7fffffu) == 0u)
    store(std::true_type{});
  else
    store(std::false_type{});
  if (lane == 0 && scale != was) *scale_at = scale;
}

// ---------------------------------------------------------------------------
// Read back: tokens at given positions of each request in 16 bits, code times scale, rounded once.  A value past
// the type's largest (its code rounded up) is that largest.
//
// Bound by the bytes (1 read, 2 written).  A thread takes 16 columns of a token, looks the token up once and goes over
// heads, eight rows of codes on their way; stores of 32 bytes fill whole sectors, where two of 16 left each half
// written until the next (4 prefixes of 16,384 tokens of 8 heads of 128 84 us, 68 so, 0.90 of
// the measured copy rate).
// ---------------------------------------------------------------------------
struct Read8Params {
  const void* k_pages;
  const void* v_pages;
  const float* k_scales;
  const float* v_scales;
  const int* page_table;
  const int* positions;  // [B, S] contiguous
  void* k;               // [B, Hkv, S, D] contiguous
  void* v;
  int* status;
  long long kps[3], vps[3], kss[2], vss[2];
  long long table_stride;
  int Hkv, S;
  int chunks;  // of the tokens that a CTA takes
  int per;     // of the 2 Hkv rows of heads that a CTA goes over
  int page_size, page_shift, max_pages, n_pages;  // page_shift: log2(page_size), or -1
};

constexpr int kReadThreads = 256;
constexpr int kReadUnroll = 8;  // heads whose codes a thread has on their way

// 32 bytes in one store: a whole sector, where two of 16 bytes would each write half of every one of the warp's.
__device__ __forceinline__ void store32(void* to, const uint32_t* y) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]),
               "r"(y[4]), "r"(y[5]), "r"(y[6]), "r"(y[7])
               : "memory");
}

template <bool BF16, int D>
__global__ void __launch_bounds__(kReadThreads, 4) coalibi_paged_read8_kernel(const Read8Params p) {
  constexpr int PIECES = D / 16, TOKENS = kReadThreads / PIECES;
  grid_dep_wait();
  const int b = blockIdx.x / p.chunks, t = (blockIdx.x - b * p.chunks) * TOKENS + threadIdx.x / PIECES;
  if (t >= p.S) return;
  const int c = (threadIdx.x % PIECES) * 16;
  const int pos = p.positions[(size_t)b * p.S + t];
  int page = -1, slot = 0;
  if (pos >= 0) {
    if (pos < p.max_pages * p.page_size) {
      const int n = p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size;
      slot = pos - n * p.page_size;
      page = p.page_table[(size_t)b * p.table_stride + n];
    }
    if (page < 0 || page >= p.n_pages) {
      if (c == 0) report_page(p.status);
      page = -1;
    }
  }
  const int row0 = blockIdx.y * p.per, row1 = min(row0 + p.per, 2 * p.Hkv);
  // (pointers of keys and values at head 0)
  const uint8_t* codes_at[2] = {static_cast<const uint8_t*>(p.k_pages) + page * p.kps[0] + slot * p.kps[2] + c,
                                static_cast<const uint8_t*>(p.v_pages) + page * p.vps[0] + slot * p.vps[2] + c};
  const float* scale_at[2] = {p.k_scales + page * p.kss[0] + slot / kQuantBlock, p.v_scales + page * p.vss[0] + slot / kQuantBlock};
  const size_t to = ((size_t)b * p.Hkv * p.S + t) * D + c, head = (size_t)p.S * D;
  // Codes times scale, rounded once.  A scale by which no code passes the type's largest needs no clamp; a
  // power of two within float16's range multiplies there, where the product is rounded once too.
  const float top = BF16 ? 3.38953139e38f : 65504.f;
  for (int row = row0; row < row1; row += kReadUnroll) {
    uint4 codes[kReadUnroll];
    float scale[kReadUnroll];
#pragma unroll
    for (int i = 0; i < kReadUnroll; ++i) {
      const bool key = row + i < p.Hkv;
      const int h = key ? row + i : row + i - p.Hkv;
      codes[i] = make_uint4(0u, 0u, 0u, 0u);
      scale[i] = 1.f;
      if (page >= 0 && row + i < row1) {
        codes[i] = *reinterpret_cast<const uint4*>(key ? codes_at[0] + h * p.kps[1] : codes_at[1] + h * p.vps[1]);
        scale[i] = key ? scale_at[0][h * p.kss[1]] : scale_at[1][h * p.vss[1]];
      }
    }
#pragma unroll
    for (int i = 0; i < kReadUnroll; ++i) {
      if (row + i >= row1) break;
      const uint32_t w[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
      uint32_t y[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) e4m3_to_f16x4(w[e], y[2 * e], y[2 * e + 1]);
      if (!BF16 && scale[i] <= 128.f && scale[i] >= 5.9604645e-8f && (__float_as_int(scale[i]) & 0x7fffff) == 0) {
        const __half2 s = __float2half2_rn(scale[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const __half2 v = __hmul2(*reinterpret_cast<__half2*>(&y[e]), s);
          y[e] = *reinterpret_cast<const uint32_t*>(&v);
        }
      } else {
        const bool clamps = !(fabsf(scale[i]) <= (BF16 ? 7e35f : 128.f));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float2 u = __fmul2_rn(f16x2_to_float2(y[e]), make_float2(scale[i], scale[i]));
          if (clamps) {  // (NaN stays)
            u.x = u.x > top ? top : u.x < -top ? -top : u.x;
            u.y = u.y > top ? top : u.y < -top ? -top : u.y;
          }
          y[e] = pack2<BF16>(u.x, u.y);
        }
      }
      const bool key = row + i < p.Hkv;
      store32(static_cast<uint16_t*>(key ? p.k : p.v) + to + (key ? row + i : row + i - p.Hkv) * head, y);
    }
  }
}

// ---------------------------------------------------------------------------
// Attention.  The formulas and the division of work are those of the 16-bit kernel (paged.cuh);
// with k_j = a_j kc_j and v_j = c_j vc_j (codes and the scales of their blocks)
//   x_j = (scale a_j) (q.kc_j),   o = sum_j (w_j c_j) vc_j / sum_j w_j.
// The codes go through the tensor cores as float16, which holds them exactly.  c_j enters the
// exponent of its weight: the running reference is the largest x_j - slope z_j + log2 c_j, so the largest
// *contribution* has a weight near 1, whatever the blocks' scales are, and a block whose values are
// small beside another's is rounded relative to what it adds; the sum of the weights is kept in
// float32 by the same reference, as sum (w_j c_j) / c_j.
// A block whose c_j is 0, negative or far from 1 (one of zeros that the append wrote, 2^-100; any that another program
// wrote) cannot give its weights back by that division.  Its step goes as a masked one, with c~_j = |c_j| held within
// 2^-100 .. 2^126 in the exponent and the product's weight times c_j / c~_j; what it adds to the sum is (h c~_j^-1/2)^2 with
// h the root of the weight, which does not flush to 0 where the weight does, and moves to other references by PieceFactor.
//
// The keys stand on the rows of the MMA and the queries on its 8 columns (S^T = K Q^T, O^T += V^T P^T):
// with at most 8 rows that share a key nothing of a product is wasted.  Both operands come out of
// ldmatrix bytewise: a 16-byte chunk of 8 keys gives a lane 4 neighbouring codes of a key,
// which are the two halves of an A fragment when Q's columns are taken in the same order; transposed, it
// gives 2 keys x 2 columns, and the columns of a pair go to rows g and g + 8 of the tile.
//
// What bounds it.  With 4 rows to a kv head, 4 contexts of 65,537 to 131,071 keys take 125 us, 0.98 of the measured copy
// rate: memory (130 to 138 a pass with 6 of joining, under the power cap, whose clock makes the instructions count).  With
// 64 columns a score costs the same for half the bytes: 126 us for 92 of reading at 12 heads.  16 contexts of up
// to 8191 keys take 28 us and 4.5 of joining against 20.5 of reading: the starts and
// ends of the items.  With 16 and 32 rows the instructions bound it (56 and 73 us where 8 rows take 31): a score costs a
// row the same whatever the codes' width is, so 8 bits gain little over 16 there.
// 16 or 32 rows are two blocks of columns of a warp, or of two warps that share the ring.
// ---------------------------------------------------------------------------
struct Paged8Params : PagedAttnParams {
  const float* k_scales;
  const float* v_scales;
  long long kss[2], vss[2];  // page, head
  int box;                   // slots of a load: 16, or 32 where a step lies in one page
};

template <int D, int NT, int RW, int WARPS>
struct Paged8Layout {
  static constexpr int THREADS = 32 * WARPS, KG = WARPS / RW;
  static constexpr int UNIT = kPagedStep * KG;
  static constexpr int COST = KG == 1 ? 4 : 256 / UNIT;
  static constexpr int WHOLE = 512;
  static constexpr int ROWS = 8 * NT * RW;
  static constexpr int TILE = kPagedStep * D;      // K or V of a step: [32 keys][D bytes], swizzled
  static constexpr int NBUF = KG > 1 ? 3 : (RW == 1 ? 2 : 3) + (D == 64 ? 1 : 0);
  static constexpr int RING = NBUF * 2 * TILE;     // per key group
  static constexpr int EXCHANGE = KG > 1 ? ROWS * D * 4 : 0;  // of a key group, over its ring
  static constexpr int GROUP = RING > EXCHANGE ? RING : EXCHANGE;
  static constexpr int BYTES = KG * GROUP + 1024;
  // resident per SM: by shared memory, and by 168 registers a thread
  static constexpr int FIT = 208 * 1024 / BYTES, CTAS = FIT < 384 / THREADS ? FIT : 384 / THREADS;
  static constexpr int RECORD = ROWS * (4 + D);
  static constexpr bool SPREAD_SUMS = true;
};

// Order of a step's 32 keys: lane group g (0 .. 7) holds keys 4 g .. 4 g + 3, so a row's suffix sum is
// additions in a lane and one scan over the groups; tile c (0 .. 3) takes one key of each group, rotated so
// that the eight rows of an ldmatrix hit all phases of the swizzle.
__device__ __forceinline__ int paged8_key(int c, int g) { return 4 * g + ((c + (g >> 1)) & 3); }

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// The float16 MMA with nothing to add to.
__device__ __forceinline__ void mma16816_zero(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Pairs in scalar arithmetic: packed instructions want both halves in neighbouring registers, and the moves
// that puts them there cost more than the issue slots they save.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return make_float2(a.x * b.x, a.y * b.y); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return make_float2(fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y)); }

// HALF: at most 4 rows.  The product leaves half of the lanes with columns of no row, so those lanes (tig 2 and 3) take
// the second rows of the others: a lane has one row of its 4 keys, in .x, and .y is dead.  The long contexts above took
// 127 us without it.
template <int D, bool BF16, int NT, int RW, int WARPS, bool HALF>
__global__ void __launch_bounds__(32 * WARPS, (Paged8Layout<D, NT, RW, WARPS>::CTAS))
    coalibi_paged8_attn_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                               const Paged8Params p) {
  using L = Paged8Layout<D, NT, RW, WARPS>;
  constexpr int KG = L::KG, KK = D / 16;
  constexpr int THREADS = 32 * RW;  // per key group
  extern __shared__ __align__(128) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t s_full[KG * L::NBUF];
  __shared__ int s_abort;
  __shared__ volatile int s_fail[KG], s_plain[KG][2];
  __shared__ int s_pre[128], s_warp[4], s_find;
  __shared__ float4 s_stat[KG > 1 ? KG * L::ROWS : 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gq = lane >> 2, tig = lane & 3;
  static_assert(!HALF || (NT == 1 && RW == 1), "four rows fit one block of columns");
  const int my_row = HALF ? 2 * (tig & 1) + (tig >> 1) : 2 * tig;  // in a block of columns
  auto other = [](float x) { return __shfl_xor_sync(0xffffffffu, x, 2); };
  const int rwarp = warp % RW, kg = warp / RW;
  const bool issuer = rwarp == 0 && lane == 0;  // of the group's loads
  const int G = p.Hq / p.Hkv, rows = G * p.Sq;
  const int heads = p.Hkv * p.row_blocks;  // items per request
  uint8_t* ring = smem + kg * L::GROUP;
  uint64_t* full = s_full + kg * L::NBUF;
  const CtaGuard guard{&s_abort, p.status, kPagedTimeoutNs};
  if (tid == 0) {
    for (int i = 0; i < KG * L::NBUF; ++i) mbar_init(&s_full[i], 1);
    s_abort = 0;
    for (int i = 0; i < KG; ++i) s_fail[i] = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  __syncthreads();
  grid_dep_wait();

  // ---- this CTA's run of units
  unsigned at = 0, stop;
  int b, span, item, v0 = 0;
  if (p.whole) {
    b = blockIdx.x / heads;
    item = blockIdx.x - b * heads;
    span = paged_span<L>(p, b);
    stop = span;
  } else {
    int* head = reinterpret_cast<int*>(p.ws);
    constexpr int NTH = L::THREADS < 128 ? L::THREADS : 128;
    const int per = (p.B + NTH - 1) / NTH;
    const unsigned total = (unsigned)paged_prefix<L>(p, s_pre, s_warp, per, blockIdx.x == 0 ? head : nullptr) * heads;
    const unsigned quota = (total + p.n_ctas - 1) / p.n_ctas;  // (the host bounds the total below 2^31)
    if (blockIdx.x == 0 && tid == 0) head[p.B + 1] = (int)quota;
    at = quota * blockIdx.x;
    stop = min(total, at + quota);
    if (at >= stop) return;
    paged_find<L>(p, s_pre, &s_find, per, heads, at, b, span, item, v0);
  }

  // this lane's ldmatrix row: key of tile lane / 8, row lane % 8; the chunk flips the swizzled bits
  const int key_ld = paged8_key(lane >> 3, lane & 7);
  const uint32_t off = D == 128 ? key_ld * 128 + ((key_ld & 7) << 4) : key_ld * 64 + ((key_ld >> 1 & 3) << 4);
  const int turn = gq >> 1;  // this lane's keys 4 gq + (c + turn) % 4 of tile c
  const int hf = gq >> 2;    // and their block of the step
  LoadRing<L::NBUF> loads;
  bool ok = true;  // no wait has run out

  while (at < stop) {
    // units [u0, u1) of the item; none if the run ends within its overhead
    const int v1 = (int)min((unsigned)span, v0 + (stop - at));
    const int u0 = max(v0 - L::COST, 0), u1 = v1 - L::COST, units = span - L::COST;
    if (u1 <= 0) break;
    const int g = item / p.row_blocks, r0 = (item - g * p.row_blocks) * L::ROWS + rwarp * 8 * NT;
    const int len = p.ctx_lens[b], room = p.max_pages * p.page_size, ctx = min(max(len, 0), room);

    // ---- drafted tokens that any row of the request sees
    unsigned long long seen_by_any = 0;
    if (p.tree_mask == nullptr) {
      seen_by_any = (2ull << (p.Sq - 1)) - 1;
    } else {
      for (int i = lane; i < p.Sq; i += 32) seen_by_any |= (unsigned long long)p.tree_mask[b * p.mask_stride + i];
#pragma unroll
      for (int d = 16; d; d >>= 1) seen_by_any |= __shfl_xor_sync(0xffffffffu, seen_by_any, d);
      if (p.Sq < 64) seen_by_any &= (1ull << p.Sq) - 1;
    }
    const int drafts = 64 - __clzll((long long)seen_by_any);
    if ((len > room || ctx + drafts > room) && tid == 0) report_page(p.status);

    // ---- this key group's keys: [lo, hi), lo a multiple of 16 (so a half step is one block of one page)
    const int s_lo = u0 * L::UNIT, s_hi = min(min(u1 * L::UNIT, room), ctx + drafts);
    const int sub = ((s_hi - s_lo + KG - 1) / KG + 15) & ~15;
    const int lo = s_lo + kg * sub, hi = min(s_hi, lo + sub);
    const int nsteps = hi > lo ? (hi - lo + kPagedStep - 1) / kPagedStep : 0;

    const int* table = p.page_table + (size_t)b * p.table_stride;
    int page_id[2], page_slot[2];  // of the next step to be loaded, per half; id -1: nothing there
    uint32_t gone_q = 0;           // two bits per ring slot: halves that were not loaded
    float ks_q[L::NBUF - 1], vs_q[L::NBUF - 1];  // scales of this lane's block in the steps under way
    auto lookup_half = [&](int key, int f) {
      page_id[f] = -1;
      page_slot[f] = 0;
      if (key >= lo && key < hi) {
        const int n = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
        page_id[f] = table[n];
        page_slot[f] = key - n * p.page_size;
        if ((unsigned)page_id[f] >= (unsigned)p.n_pages) {
          page_id[f] = -1;
          report_page(p.status);
        }
      }
    };
    auto lookup = [&](int st) {
      const int key = lo + st * kPagedStep;
      lookup_half(key, 0);
      if (KG == 1 && p.box == 32) {  // (steps begin at multiples of 32 here)
        page_id[1] = key + 16 < hi ? page_id[0] : -1;
        page_slot[1] = page_slot[0] + 16;
      } else {
        lookup_half(key + 16, 1);
      }
    };
    auto load = [&]() {
      const int slot = loads.fill;
      gone_q &= ~(3u << (2 * slot));
      gone_q |= ((page_id[0] < 0 ? 1u : 0u) | (page_id[1] < 0 ? 2u : 0u)) << (2 * slot);
      if (issuer) {
        const uint32_t dst = smem_u32(ring + slot * 2 * L::TILE);
        if (KG == 1 && p.box == 32) {  // (the second half may lie past the keys: it is loaded, and masked)
          mbar_arrive_expect_tx(&full[slot], page_id[0] >= 0 ? 2 * L::TILE : 0);
          if (page_id[0] >= 0) {
            tma_load_4d(dst, &tk, &full[slot], 0, page_slot[0], g, page_id[0]);
            tma_load_4d(dst + L::TILE, &tv, &full[slot], 0, page_slot[0], g, page_id[0]);
          }
        } else {
          mbar_arrive_expect_tx(&full[slot], ((page_id[0] >= 0) + (page_id[1] >= 0)) * L::TILE);
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            if (page_id[f] < 0) continue;
            tma_load_4d(dst + f * 16 * D, &tk, &full[slot], 0, page_slot[f], g, page_id[f]);
            tma_load_4d(dst + L::TILE + f * 16 * D, &tv, &full[slot], 0, page_slot[f], g, page_id[f]);
          }
        }
      }
      loads.issue();
    };
    auto load_scales = [&](float& ks, float& vs) {  // of the step whose pages were looked up
      const int page = hf ? page_id[1] : page_id[0], blk = (hf ? page_slot[1] : page_slot[0]) / kQuantBlock;
      ks = vs = 1.f;
      if (page >= 0) {
        ks = p.k_scales[page * p.kss[0] + g * p.kss[1] + blk];
        vs = p.v_scales[page * p.vss[0] + g * p.vss[1] + blk];
      }
    };
    auto group_sync = [&]() {
      if (RW == 1)
        __syncwarp();
      else
        asm volatile("bar.sync %0, %1;" ::"r"(1 + kg), "n"(THREADS) : "memory");
    };

    lookup(nsteps - 1);
#pragma unroll
    for (int a = 1; a < L::NBUF; ++a) {
      load_scales(ks_q[a - 1], vs_q[a - 1]);
      if (nsteps - a >= 0) load();
      lookup(nsteps - a - 1);
    }

    // ---- the rows: Q^T as B fragments, columns in the order of the codes; bfloat16 queries as float16
    // scaled by a power of two that puts a row's largest at 2^14 (the smallest that is kept whole then lies
    // 28 binades below it)
    uint32_t qb[NT][KK][2];
    float2 unit[NT];  // scale * log2 e over that power, of columns 2 tig and 2 tig + 1
    float2 slope2[NT];
    const float c_a = p.sm_scale * kLog2e;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = r0 + 8 * n + gq;
      const int rr = r < rows ? r : 0;
      const uint16_t* q = static_cast<const uint16_t*>(p.q) + b * p.qs[0] + (g * G + rr / p.Sq) * p.qs[1] + (rr % p.Sq) * p.qs[2];
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const uint2 u = r < rows ? *reinterpret_cast<const uint2*>(q + 16 * kk + 4 * tig) : make_uint2(0u, 0u);
        qb[n][kk][0] = u.x, qb[n][kk][1] = u.y;
      }
      unit[n] = make_float2(c_a, c_a);
      if (BF16) {
        uint32_t most = 0;  // largest exponent, as bits
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
          for (int e = 0; e < 2; ++e) most = max(most, max(qb[n][kk][e] << 16 & 0x7f800000u, qb[n][kk][e] & 0x7f800000u));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // 2^(14 - e); e kept where both this and its inverse are normal.  Rows with an infinity or NaN stay so.
        const int up = 14 - min(max((int)(most >> 23) - 127, -100), 127);
        const float f = __int_as_float((up + 127) << 23), down = __int_as_float((127 - up) << 23);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 u = unpack2<true>(qb[n][kk][e]);
            qb[n][kk][e] = pack2<false>(u.x * f, u.y * f);
          }
        unit[n].x *= __shfl_sync(0xffffffffu, down, 4 * my_row);
        if (!HALF) unit[n].y *= __shfl_sync(0xffffffffu, down, 4 * my_row + 4);
      }
      const int ra = min(r0 + 8 * n + my_row, rows - 1), rb = min(ra + 1, rows - 1);
      slope2[n] = make_float2(load_slope(p.slopes, p.slopes_dtype, g * G + ra / p.Sq) * kLog2e,
                              load_slope(p.slopes, p.slopes_dtype, g * G + rb / p.Sq) * kLog2e);
    }

    float o[KK][NT][4];
#pragma unroll
    for (int dm = 0; dm < KK; ++dm)
#pragma unroll
      for (int n = 0; n < NT; ++n) o[dm][n][0] = o[dm][n][1] = o[dm][n][2] = o[dm][n][3] = 0.f;
    float2 m_run[NT], l_part[NT], carry[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m_run[n] = make_float2(-INFINITY, -INFINITY);
      l_part[n] = carry[n] = make_float2(0.f, 0.f);
    }

    for (int st = nsteps - 1; st >= 0; --st) {
      if (ok && !mbar_wait(&full[loads.drain], loads.phase, guard)) s_fail[kg] = st + 1;
      // Whether every key is of the context and every scale plain.  One warp decides for the group, which meets again in
      // the other steps: were a page or scale written to meanwhile, its warps might disagree and wait for each other.
      auto plain = [&]() {
        return lo + (st + 1) * kPagedStep <= min(hi, ctx) && (gone_q >> (2 * loads.drain) & 3) == 0 &&
               !__any_sync(0xffffffffu, odd_scale(vs_q[0]));
      };
      if (RW > 1 && rwarp == 0) {
        const bool mine = plain();
        if (lane == 0) s_plain[kg][st & 1] = mine;
      }
      group_sync();  // all are done with step st + 1, whose slot is loaded next
      // the same for the group's warps, which meet again in the masked steps: a wait of this step or
      // of one before it ran out (one that a faster warp already meets in the next step counts there)
      ok = s_fail[kg] <= st;
      if (!ok) continue;
      const bool all = RW > 1 ? s_plain[kg][st & 1] != 0 : plain();
      const int slot = loads.drain;
      loads.landed();
      const float k_scale = ks_q[0], v_scale = vs_q[0];
#pragma unroll
      for (int i = 0; i + 1 < L::NBUF - 1; ++i) ks_q[i] = ks_q[i + 1], vs_q[i] = vs_q[i + 1];
      load_scales(ks_q[L::NBUF - 2], vs_q[L::NBUF - 2]);
      if (st - (L::NBUF - 1) >= 0) load();
      lookup(st - L::NBUF);
      const int kb = lo + st * kPagedStep;
      const uint32_t kt = smem_u32(ring + slot * 2 * L::TILE), vt = kt + L::TILE;
      // ---- S^T = K Q^T: rows of tile pair mt, columns of block n
      float sc[2][NT][4];
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        uint32_t w[4], a[2][4];
        ldsm_x4(kt + (off ^ (kk << 4)), w[0], w[1], w[2], w[3]);
#pragma unroll
        for (int c = 0; c < 4; ++c) e4m3_to_f16x4(w[c], a[c >> 1][c & 1], a[c >> 1][2 + (c & 1)]);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (kk == 0)
              mma16816_zero(sc[mt][n], a[mt], qb[n][kk][0], qb[n][kk][1]);
            else
              mma16816<false>(sc[mt][n], a[mt], qb[n][kk][0], qb[n][kk][1]);
          }
      }
      // ---- which of this lane's 4 keys each of its rows sees: bit 8 n + 4 x + c
      const uint32_t gone = gone_q >> (2 * slot) & 3;
      uint32_t vis = 0xffffu;
      if (!all) {
        vis = 0;
#pragma unroll 1
        for (int i = 0; i < (HALF ? 1 : 2 * NT); ++i) {
          const int r = r0 + 8 * (i >> 1) + my_row + (i & 1), row = r < rows ? r % p.Sq : 0;
          const unsigned long long word =
              p.tree_mask != nullptr ? (unsigned long long)p.tree_mask[b * p.mask_stride + row] : (2ull << row) - 1;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int key = kb + paged8_key(c, gq);
            if (!(gone >> hf & 1) && key < hi && (key < ctx || (word >> (key - ctx) & 1))) vis |= 1u << (4 * i + c);
          }
        }
      }
      // ---- sigmoids, suffix sums, logits (in log2 units), online softmax; both rows of a column
      // pair as float2
      uint32_t pb[NT][4];
      auto softmax = [&](auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        const bool odd = MASKED && odd_scale(v_scale);
        const float held = odd ? fminf(fmaxf(fabsf(v_scale), kScaleHeldMin), kScaleHeldMax) : v_scale;
        const float lv = lg2_approx(held), iv = rcp_approx(held);
        float2 mx[NT];
        float2 v[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float2 s[4];
          const float2 f = mul2(unit[n], make_float2(k_scale, k_scale));
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float2 d = make_float2(sc[c >> 1][n][2 * (c & 1)], sc[c >> 1][n][2 * (c & 1) + 1]);
            if (HALF) {
              const float y = other(d.y);
              d = make_float2(tig < 2 ? d.x : y, 0.f);
            }
            v[n][c] = mul2(d, f);
            const float2 e = add2(make_float2(ex2_approx(-v[n][c].x), ex2_approx(-v[n][c].y)), make_float2(1.f, 1.f));
            s[c] = make_float2(rcp_approx(e.x), rcp_approx(e.y));
            if (MASKED) {
              s[c].x = vis >> (8 * n + c) & 1 ? s[c].x : 0.f;
              s[c].y = vis >> (8 * n + 4 + c) & 1 ? s[c].y : 0.f;
            }
          }
          // sums of the tiles c and after it; tiles c >= 4 - turn hold the lane's first keys
          s[2] = add2(s[2], s[3]);
          s[1] = add2(s[1], s[2]);
          s[0] = add2(s[0], s[1]);
          float2 inc = s[0];
#pragma unroll
          for (int d = 4; d <= 16; d <<= 1) {
            const float2 y = make_float2(__shfl_down_sync(0xffffffffu, inc.x, d), HALF ? 0.f : __shfl_down_sync(0xffffffffu, inc.y, d));
            if (lane + d < 32) inc = add2(inc, y);
          }
          const float2 wrapped = turn == 0 ? make_float2(0.f, 0.f) : turn == 1 ? s[3] : turn == 2 ? s[2] : s[1];
          const float2 right = make_float2(inc.x - s[0].x, inc.y - s[0].y);
          const float2 last = make_float2(carry[n].x + (right.x - wrapped.x), carry[n].y + (right.y - wrapped.y));
          const float2 first = add2(last, s[0]);
          carry[n].x += __shfl_sync(0xffffffffu, inc.x, tig);
          if (!HALF) carry[n].y += __shfl_sync(0xffffffffu, inc.y, tig);
          mx[n] = make_float2(-INFINITY, -INFINITY);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float2 z = add2(c + turn >= 4 ? first : last, s[c]);
            v[n][c] = fma2(make_float2(-slope2[n].x, -slope2[n].y), z, v[n][c]);
            if (MASKED) {
              v[n][c].x = vis >> (8 * n + c) & 1 ? v[n][c].x : -INFINITY;
              v[n][c].y = vis >> (8 * n + 4 + c) & 1 ? v[n][c].y : -INFINITY;
            }
            mx[n].x = fmaxf(mx[n].x, v[n][c].x);
            mx[n].y = fmaxf(mx[n].y, v[n][c].y);
          }
          mx[n].x += lv;
          mx[n].y += lv;
        }
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mx[n].x = fmaxf(mx[n].x, __shfl_xor_sync(0xffffffffu, mx[n].x, d));
            if (!HALF) mx[n].y = fmaxf(mx[n].y, __shfl_xor_sync(0xffffffffu, mx[n].y, d));
          }
        }
        // the newest keys weigh most, so the maximum seldom moves after the first steps
        bool up = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) up |= mx[n].x > m_run[n].x || (!HALF && mx[n].y > m_run[n].y);
        if (__any_sync(0xffffffffu, up)) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float2 m = make_float2(fmaxf(m_run[n].x, mx[n].x), fmaxf(m_run[n].y, mx[n].y));
            const PieceFactor<L> px(m_run[n].x == -INFINITY ? -INFINITY : m_run[n].x - m.x);
            const PieceFactor<L> py(HALF || m_run[n].y == -INFINITY ? -INFINITY : m_run[n].y - m.y);
            const float fx = px.f, fy = HALF ? other(fx) : py.f;
            m_run[n] = m;
            l_part[n].x = px.of_sum(l_part[n].x);
            if (!HALF) l_part[n].y = py.of_sum(l_part[n].y);
#pragma unroll
            for (int dm = 0; dm < KK; ++dm) {
              o[dm][n][0] *= fx, o[dm][n][2] *= fx;
              o[dm][n][1] *= fy, o[dm][n][3] *= fy;
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float2 off2 = make_float2(lv - (m_run[n].x == -INFINITY ? 0.f : m_run[n].x),
                                          lv - (m_run[n].y == -INFINITY ? 0.f : m_run[n].y));
          float2 l2 = make_float2(0.f, 0.f);
          const float by = odd ? v_scale * iv : 1.f, root = odd ? ex2_approx(-0.5f * lv) : 1.f;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float2 x = add2(v[n][c], off2);
            float2 w;
            if (odd) {  // (masked keys: x is -inf, all 0)
              w = make_float2(ex2_approx(0.5f * x.x), HALF ? 0.f : ex2_approx(0.5f * x.y));
              const float2 u = mul2(w, make_float2(root, root));
              l2 = fma2(u, u, l2);
              w = mul2(mul2(w, w), make_float2(by, by));
            } else {
              w = make_float2(ex2_approx(x.x), ex2_approx(x.y));
            }
            if (MASKED) {  // (a block that nothing of is seen may have any scale)
              w.x = vis >> (8 * n + c) & 1 ? w.x : 0.f;
              w.y = vis >> (8 * n + 4 + c) & 1 ? w.y : 0.f;
            }
            if (HALF) w.y = 0.f;
            if (!odd) l2 = add2(l2, w);
            if (HALF)
              v[n][c].x = w.x;
            else
              pb[n][c] = pack2<false>(w.x, w.y);
          }
          if (HALF) {  // both rows of a column pair again
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
              const uint32_t mine = pack2<false>(v[n][c].x, v[n][c + 1].x), theirs = __shfl_xor_sync(0xffffffffu, mine, 2);
              pb[n][c] = __byte_perm(mine, theirs, 0x5410);
              pb[n][c + 1] = __byte_perm(mine, theirs, 0x7632);
            }
          }
          // the weights themselves: without the block's scale
          const float un = odd ? 1.f : iv;
          l_part[n] = fma2(l2, make_float2(un, un), l_part[n]);
        }
      };
      if (all)
        softmax(std::false_type{});
      else
        softmax(std::true_type{});
      // ---- V rows that no row sees (past the end, of no page, unseen drafts) may hold any code: zero
      // them, 0 * NaN is not 0.  A drafted token's V that has codes of NaN must not reach the rows that do not
      // see it either: it is added by hand, then zeroed.
      if (!all) {
        if (HALF) vis = (vis & 15u) | __shfl_xor_sync(0xffffffffu, vis & 15u, 2) << 4;
        const int key = kb + lane;
        uint8_t* vrow = ring + slot * 2 * L::TILE + L::TILE + lane * D;
        const bool used = !(gone >> (lane >> 4) & 1) && key < hi && (key < ctx || (seen_by_any >> (key - ctx) & 1));
        bool bad = false;
        if (used && key >= ctx && p.Sq > 1) {
#pragma unroll 4
          for (int c = 0; c < D / 16; ++c) {
            const uint4 u = reinterpret_cast<const uint4*>(vrow)[c];
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) bad |= __vcmpeq4(w[j] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0;
          }
        }
        for (uint32_t left = __ballot_sync(0xffffffffu, bad); left != 0; left &= left - 1) {
          const int at_key = __ffs(left) - 1, from = (at_key >> 2) * 4 + tig;  // the lane that holds its weights
          const int c = ((at_key & 3) - (at_key >> 3)) & 3;                    // in this tile
          const uint8_t* vb = ring + slot * 2 * L::TILE + L::TILE + at_key * D;
          const uint32_t phase = D == 128 ? at_key & 7 : at_key >> 1 & 3;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint32_t w2 = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (c == j) w2 = pb[n][j];
            w2 = __shfl_sync(0xffffffffu, w2, from);
            const uint32_t see = __shfl_sync(0xffffffffu, vis, from) >> (8 * n + c);
            const float2 w = f16x2_to_float2(w2);
#pragma unroll
            for (int dm = 0; dm < KK; ++dm) {
              const float2 f = f16x2_to_float2(
                  e4m3_to_f16x2(*reinterpret_cast<const uint16_t*>(vb + ((dm ^ phase) << 4) + 2 * gq)));
              if (see & 1) {
                o[dm][n][0] = fmaf(w.x, f.x, o[dm][n][0]);
                o[dm][n][2] = fmaf(w.x, f.y, o[dm][n][2]);
              }
              if (see >> 4 & 1) {
                o[dm][n][1] = fmaf(w.y, f.x, o[dm][n][1]);
                o[dm][n][3] = fmaf(w.y, f.y, o[dm][n][3]);
              }
            }
          }
        }
        group_sync();
        if (rwarp == 0 && (!used || bad)) {
#pragma unroll
          for (int c = 0; c < D / 16; ++c) reinterpret_cast<uint4*>(vrow)[c] = make_uint4(0u, 0u, 0u, 0u);
          fence_async_smem();  // ordered before the load that refills the slot
        }
        group_sync();
      }
      // ---- O^T += V^T P^T.  P goes to float16 (half an ulp of each weight, which averages out over the
      // keys, and nothing of one below 2^-25 of the largest contribution; the sum takes them unrounded), and from the accumulators' layout to the operand's by a transpose.
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) pb[n][c] = transpose8x8(pb[n][c]);
#pragma unroll
      for (int dm = 0; dm < KK; ++dm) {
        uint32_t w[4], a[2][4];
        ldsm_x4_t(vt + (off ^ (dm << 4)), w[0], w[1], w[2], w[3]);
#pragma unroll
        for (int c = 0; c < 4; ++c)
          e4m3_to_f16x4(__byte_perm(w[c], 0, 0x3120), a[c >> 1][2 * (c & 1)], a[c >> 1][2 * (c & 1) + 1]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma16816<false>(o[dm][n], a[0], pb[n][0], pb[n][1]);
          mma16816<false>(o[dm][n], a[1], pb[n][2], pb[n][3]);
        }
      }
    }
    if (!ok && issuer)  // a wait ran out: the loads already issued land before the CTA leaves, below
      for (; loads.in_flight(); loads.landed()) mbar_drain(&full[loads.drain], loads.phase, kPagedTimeoutNs);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int d = 4; d <= 16; d <<= 1) {
        l_part[n].x += __shfl_xor_sync(0xffffffffu, l_part[n].x, d);
        if (!HALF) l_part[n].y += __shfl_xor_sync(0xffffffffu, l_part[n].y, d);
      }
    if (HALF) carry[0].y = other(carry[0].x), m_run[0].y = other(m_run[0].x), l_part[0].y = other(l_part[0].x), slope2[0].y = other(slope2[0].x);

    // ---- the piece's result: the output if the item is whole, else a record
    const bool whole = u0 == 0 && u1 == units;
    float* rec = p.ws + paged_ws_head(p.B) + ((size_t)blockIdx.x * 2 + (u0 > 0 ? 0 : 1)) * L::RECORD;
    float4* stats = reinterpret_cast<float4*>(rec);
    float* orec = rec + 4 * L::ROWS;
    if (KG == 1) {
#pragma unroll
      for (int i = 0; i < 2 * NT; ++i) {
        const int n = i >> 1, x = i & 1;
        const int r = rwarp * 8 * NT + 8 * n + 2 * tig + x, rr = r0 + 8 * n + 2 * tig + x;
        if (rr >= rows) continue;
        const float l = x ? l_part[n].y : l_part[n].x;
        if (whole) {
          uint16_t* y = static_cast<uint16_t*>(p.o) + b * p.os[0] + (g * G + rr / p.Sq) * p.os[1] + (rr % p.Sq) * p.os[2];
          const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
          for (int dm = 0; dm < KK; ++dm)
            *reinterpret_cast<uint32_t*>(y + 16 * dm + 2 * gq) = pack2<BF16>(o[dm][n][x] * inv, o[dm][n][2 + x] * inv);
        } else {
          if (gq == 0) stats[r] = make_float4(x ? carry[n].y : carry[n].x, x ? m_run[n].y : m_run[n].x, l, 0.f);
#pragma unroll
          for (int dm = 0; dm < KK; ++dm)
            *reinterpret_cast<float2*>(orec + r * D + 16 * dm + 2 * gq) = make_float2(o[dm][n][x], o[dm][n][2 + x]);
        }
      }
    } else {
      // key groups join through shared memory (the rings are idle now)
      __syncthreads();
      float* xo = reinterpret_cast<float*>(smem + kg * L::GROUP);  // [ROWS][D] of each group
#pragma unroll
      for (int i = 0; i < 2 * NT; ++i) {
        const int n = i >> 1, x = i & 1, r = rwarp * 8 * NT + 8 * n + 2 * tig + x;
        if (gq == 0)
          s_stat[kg * L::ROWS + r] = make_float4(x ? carry[n].y : carry[n].x, x ? m_run[n].y : m_run[n].x,
                                                 x ? l_part[n].y : l_part[n].x, x ? slope2[n].y : slope2[n].x);
#pragma unroll
        for (int dm = 0; dm < KK; ++dm)
          *reinterpret_cast<float2*>(xo + r * D + 16 * dm + 2 * gq) = make_float2(o[dm][n][x], o[dm][n][2 + x]);
      }
      __syncthreads();
      const int rb = (item - g * p.row_blocks) * L::ROWS;
      const int n = min(L::ROWS, rows - rb);
      for (int e = tid; e < n * (D / 4); e += L::THREADS) {
        const int r = e / (D / 4), d = (e % (D / 4)) * 4;
        float right = 0.f, M = -INFINITY, w[KG];
#pragma unroll
        for (int c = KG - 1; c >= 0; --c) {
          const float4 s = s_stat[c * L::ROWS + r];
          w[c] = s.y == -INFINITY ? -INFINITY : s.y - s.w * right;
          M = fmaxf(M, w[c]);
          right += s.x;
        }
        const float m_use = M == -INFINITY ? 0.f : M;
        float l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int c = KG - 1; c >= 0; --c) {
          const PieceFactor<L> pf(w[c] - m_use);
          const float f = pf.f;
          l += pf.of_sum(s_stat[c * L::ROWS + r].z);
          const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + c * L::GROUP) + r * D + d);
          acc.x = fmaf(v.x, f, acc.x);
          acc.y = fmaf(v.y, f, acc.y);
          acc.z = fmaf(v.z, f, acc.z);
          acc.w = fmaf(v.w, f, acc.w);
        }
        if (whole) {
          const int rr = rb + r;
          uint16_t* y = static_cast<uint16_t*>(p.o) + b * p.os[0] + (g * G + rr / p.Sq) * p.os[1] + (rr % p.Sq) * p.os[2];
          const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
          *reinterpret_cast<uint2*>(y + d) =
              make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
        } else {
          if (d == 0) stats[r] = make_float4(right, M, l, 0.f);
          *reinterpret_cast<float4*>(orec + r * D + d) = acc;
        }
      }
    }
    if (KG > 1) fence_async_smem();
    __syncthreads();  // the rings are free for the next item
    if (s_abort != 0) return;

    // ---- next item of the run
    at += v1 - v0;
    v0 = 0;
    if (++item == heads) {
      item = 0;
      if (++b < p.B) span = paged_span<L>(p, b);
    }
  }
}

// Joins the pieces of the items that span runs, as the 16-bit attention's kernel does, but with a CTA for a
// query row: runs are a warp's here, so a long item comes in dozens of pieces.  A thread takes a piece's
// statistics, rightmost first, and a warp every fourth piece's O, the first ones on their way beside the statistics.
constexpr int kJoinThreads = 128;

template <int D, bool BF16, typename L>
__global__ void __launch_bounds__(kJoinThreads) coalibi_paged8_join_kernel(const PagedAttnParams p) {
  constexpr int V = D / 32, WARPS = kJoinThreads / 32, EARLY = 8;
  __shared__ float s_f[kJoinThreads], s_a[WARPS], s_b[WARPS], s_c[WARPS], s_o[WARPS][D];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = p.Hq / p.Hkv;
  const int b = blockIdx.x / p.Hkv, g = blockIdx.x - b * p.Hkv, r = blockIdx.y;
  grid_dep_wait();
  const int* head = reinterpret_cast<const int*>(p.ws);
  const int heads = p.Hkv * p.row_blocks, item = g * p.row_blocks + r / L::ROWS, rr = r % L::ROWS;
  const int span = head[b + 1] - head[b];
  const long long quota = head[p.B + 1];
  const long long start = (long long)head[b] * heads + (long long)item * span;
  const long long t0 = start + L::COST, t1 = start + span;
  const int c0 = (int)(t0 / quota), c1 = (int)((t1 - 1) / quota);
  if (c0 == c1) return;  // finished by the attention kernel
  const int h = g * G + r / p.Sq, i = r % p.Sq;
  const float slope2 = load_slope(p.slopes, p.slopes_dtype, h) * kLog2e;
  const float* recs = p.ws + paged_ws_head(p.B);
  auto record = [&](int c) { return recs + ((size_t)c * 2 + (t0 < c * quota ? 0 : 1)) * L::RECORD; };
  float M = -INFINITY, l = 0.f, right = 0.f, acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.f;
  for (int top = c1; top >= c0; top -= kJoinThreads) {
    const int n = min(kJoinThreads, top - c0 + 1);
    auto o_of = [&](int j, float* u) {
      const float* y = record(top - j) + 4 * L::ROWS + rr * D + lane * V;
      if (V == 4) {
        const float4 f = *reinterpret_cast<const float4*>(y);
        u[0] = f.x, u[1] = f.y, u[V - 2] = f.z, u[V - 1] = f.w;
      } else {
        const float2 f = *reinterpret_cast<const float2*>(y);
        u[0] = f.x, u[1] = f.y;
      }
    };
    float4 s = make_float4(0.f, -INFINITY, 0.f, 0.f);
    if (tid < n) s = reinterpret_cast<const float4*>(record(top - tid))[rr];
    float early[EARLY][V];
#pragma unroll
    for (int k = 0; k < EARLY; ++k) {
#pragma unroll
      for (int v = 0; v < V; ++v) early[k][v] = 0.f;
      if (warp + k * WARPS < n) o_of(warp + k * WARPS, early[k]);
    }
    float inc = s.x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const float y = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += y;
    }
    if (lane == 31) s_a[warp] = inc;
    __syncthreads();
    float before = right;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before += s_a[w];
      right += s_a[w];
    }
    const float m = s.y == -INFINITY ? -INFINITY : s.y - slope2 * (before + (inc - s.x));
    float mx = m;
#pragma unroll
    for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    if (lane == 0) s_b[warp] = mx;
    __syncthreads();
    float m_new = M;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m_new = fmaxf(m_new, s_b[w]);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const PieceFactor<L> fac(M == -INFINITY ? -INFINITY : M - m_use), f(m - m_use);
    M = m_new;
    s_f[tid] = f.f;
    float lw = f.of_sum(s.z);
#pragma unroll
    for (int d = 16; d; d >>= 1) lw += __shfl_xor_sync(0xffffffffu, lw, d);
    if (lane == 0) s_c[warp] = lw;
    __syncthreads();
    l = fac.of_sum(l);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) l += s_c[w];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] *= fac.f;
#pragma unroll
    for (int k = 0; k < EARLY; ++k) {
      const float w = s_f[warp + k * WARPS];  // 0 past the last piece
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = fmaf(w, early[k][v], acc[v]);
    }
#pragma unroll 4
    for (int j = warp + EARLY * WARPS; j < n; j += WARPS) {
      const float w = s_f[j];
      float u[V];
      o_of(j, u);
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = fmaf(w, u[v], acc[v]);
    }
    __syncthreads();  // s_a, s_b, s_c and s_f are written again
  }
#pragma unroll
  for (int v = 0; v < V; ++v) s_o[warp][lane * V + v] = acc[v];
  __syncthreads();
  if (tid >= D / 2) return;
  float2 sum = make_float2(0.f, 0.f);
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    sum.x += s_o[w][2 * tid];
    sum.y += s_o[w][2 * tid + 1];
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  uint16_t* y = static_cast<uint16_t*>(p.o) + b * p.os[0] + h * p.os[1] + i * p.os[2] + 2 * tid;
  *reinterpret_cast<uint32_t*>(y) = pack2<BF16>(sum.x * inv, sum.y * inv);
}

}  // namespace coalibi
