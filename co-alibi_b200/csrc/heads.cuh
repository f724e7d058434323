// Query, key and value heads out of a fused projection: queries and keys normed per head (root mean
// square, a weight for each column) and rotated by their position, values moved; with the backward.
//
// With x a row of D, r = 1 / sqrt(mean(x^2) + eps), n = r x, R the rotation of the row's position:
//   y = R (w n),   d = R^T dy,   dw = sum over rows of d n,   dx = r (w d - n mean(w d n)).
//
// Bound by the bytes: the projection read once and the heads written once (forward); the projection and
// the heads' gradients read, the projection's gradient written (backward; r is computed again rather than
// kept).  D / 8 lanes take a row, each two pieces of 4 columns: those of a lane that rotates are the
// two partners of each pair, so a rotation needs no exchange and half the angles.  A CTA takes a token at a
// time and its threads several heads of it by the same angles.
#pragma once

#include "sm100.cuh"

namespace coalibi {

struct HeadsParams {
  const void* qkv;        // [B, S, Hq + 2 Hkv, D] by stride
  void* dqkv;             // the same, contiguous
  const void* in[3];      // backward: gradients of q, k, v
  void* out[3];           // forward: q, k, v
  const void* weight[2];  // of queries and keys; NULL: ones
  const float* cos;
  const float* sin;
  const int* start;
  const int* positions;
  int* status;
  float* partial;         // backward: [gridDim][2][D]
  void* dweight[2];
  long long xs[3];        // batch, token, head
  long long hs[3][3];     // of q, k, v: batch, head, token
  long long tokens;       // B * S
  int Hq, Hkv, S;
  int rows;               // heads that a pass of the CTA covers
  int rot, n_pos, interleaved;
  int weight_f32;
  float eps;
};

constexpr int kHeadsThreads = 128;  // at most

// A weight of column c, as float.
template <bool BF16>
__device__ __forceinline__ float load_weight(const void* w, int f32, int c) {
  if (w == nullptr) return 1.f;
  if (f32) return static_cast<const float*>(w)[c];
  const uint32_t u = static_cast<const uint16_t*>(w)[c];
  return unpack2<BF16>(u).x;
}

// Where a lane's columns and angles are.  Piece l of a row: partners 4 l .. and R / 2 + 4 l .. of a rotation
// in halves, else columns 8 l .. 8 l + 7.
struct HeadsLane {
  int c0, c1;
  bool turns;
};
__device__ __forceinline__ HeadsLane heads_lane(int l, int rot, int interleaved) {
  HeadsLane t;
  t.turns = 8 * l < rot;
  const bool halves = t.turns && !interleaved;
  t.c0 = halves ? 4 * l : 8 * l;
  t.c1 = halves ? rot / 2 + 4 * l : 8 * l + 4;
  return t;
}

// The row of the angles of token i of request b, or -1.
__device__ __forceinline__ int heads_angle(const HeadsParams& p, int b, int i, bool reports) {
  if (p.rot == 0) return -1;
  const long long pos = p.positions != nullptr ? p.positions[(size_t)b * p.S + i]
                                               : (p.start != nullptr ? (long long)p.start[b] : 0) + i;
  if (pos >= 0 && pos < p.n_pos) return (int)pos;
  if (reports && p.status != nullptr) atomicCAS(p.status, 0, 11 /* COALIBI_ERR_PAGE */);
  return -1;
}

template <bool BF16>
__device__ __forceinline__ void heads_unpack(uint2 a, uint2 b, float* f) {
  const uint32_t w[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 u = unpack2<BF16>(w[e]);
    f[2 * e] = u.x, f[2 * e + 1] = u.y;
  }
}
template <bool BF16>
__device__ __forceinline__ void heads_store(uint16_t* y, const HeadsLane& t, const float* f) {
  *reinterpret_cast<uint2*>(y + t.c0) = make_uint2(pack2<BF16>(f[0], f[1]), pack2<BF16>(f[2], f[3]));
  *reinterpret_cast<uint2*>(y + t.c1) = make_uint2(pack2<BF16>(f[4], f[5]), pack2<BF16>(f[6], f[7]));
}

// f's pairs turned by angles (cs, sign * sn): pairs (f[e], f[e + 4]) in halves, (f[2 e], f[2 e + 1]) interleaved.
__device__ __forceinline__ void heads_turn(float* f, const float4& cs, const float4& sn, float sign, int interleaved) {
  const float c[4] = {cs.x, cs.y, cs.z, cs.w}, s[4] = {sign * sn.x, sign * sn.y, sign * sn.z, sign * sn.w};
  if (interleaved) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = f[2 * e], b = f[2 * e + 1];
      f[2 * e] = a * c[e] - b * s[e];
      f[2 * e + 1] = b * c[e] + a * s[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = f[e], b = f[e + 4];
      f[e] = a * c[e] - b * s[e];
      f[e + 4] = b * c[e] + a * s[e];
    }
  }
}

template <bool BF16, int D>
__global__ void __launch_bounds__(kHeadsThreads) coalibi_heads_fwd_kernel(const HeadsParams p) {
  constexpr int PIECES = D / 8, UNROLL = 3;
  __shared__ __align__(16) float s_w[2][D];
  grid_dep_wait();
  const int tid = threadIdx.x, l = tid % PIECES, r0 = tid / PIECES;
  for (int e = tid; e < 2 * D; e += blockDim.x) s_w[e / D][e % D] = load_weight<BF16>(p.weight[e / D], p.weight_f32, e % D);
  __syncthreads();
  const HeadsLane t = heads_lane(l, p.rot, p.interleaved);
  const int H = p.Hq + 2 * p.Hkv, Hn = p.Hq + p.Hkv;
  for (long long tok = blockIdx.x; tok < p.tokens; tok += gridDim.x) {
    const int b = (int)(tok / p.S), i = (int)(tok - (long long)b * p.S);
    const uint16_t* x = static_cast<const uint16_t*>(p.qkv) + b * p.xs[0] + i * p.xs[1];
    const int angle = heads_angle(p, b, i, tid == 0);
    float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool turns = t.turns && angle >= 0;
    if (turns) {
      cs = *reinterpret_cast<const float4*>(p.cos + (size_t)angle * (p.rot / 2) + 4 * l);
      sn = *reinterpret_cast<const float4*>(p.sin + (size_t)angle * (p.rot / 2) + 4 * l);
    }
    // (the same passes for all threads: the reductions take whole warps)
    for (int base = 0; base < H; base += UNROLL * p.rows) {
      uint2 u0[UNROLL], u1[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int row = base + u * p.rows + r0;
        u0[u] = u1[u] = make_uint2(0u, 0u);
        if (row < H && r0 < p.rows) {
          u0[u] = *reinterpret_cast<const uint2*>(x + row * p.xs[2] + t.c0);
          u1[u] = *reinterpret_cast<const uint2*>(x + row * p.xs[2] + t.c1);
        }
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        if (base + u * p.rows >= H) break;
        const int row = base + u * p.rows + r0;
        float f[8];
        heads_unpack<BF16>(u0[u], u1[u], f);
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
#pragma unroll
        for (int d = 1; d < PIECES; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        if (row >= H || r0 >= p.rows) continue;
        const int kind = row < p.Hq ? 0 : row < Hn ? 1 : 2;
        const int h = kind == 0 ? row : kind == 1 ? row - p.Hq : row - Hn;
        uint16_t* y = static_cast<uint16_t*>(p.out[kind]) + b * p.hs[kind][0] + h * p.hs[kind][1] + i * p.hs[kind][2];
        if (kind == 2) {
          *reinterpret_cast<uint2*>(y + t.c0) = u0[u];
          *reinterpret_cast<uint2*>(y + t.c1) = u1[u];
          continue;
        }
        const float r = rsqrtf(ss * (1.f / D) + p.eps);
        const float4 w0 = *reinterpret_cast<const float4*>(&s_w[kind][t.c0]), w1 = *reinterpret_cast<const float4*>(&s_w[kind][t.c1]);
        const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = f[e] * r * w[e];
        if (turns) heads_turn(f, cs, sn, 1.f, p.interleaved);
        heads_store<BF16>(y, t, f);
      }
    }
  }
}

template <bool BF16, int D>
__global__ void __launch_bounds__(kHeadsThreads) coalibi_heads_bwd_kernel(const HeadsParams p) {
  constexpr int PIECES = D / 8, UNROLL = 3;
  __shared__ __align__(16) float s_w[2][D];
  __shared__ __align__(16) float s_sum[kHeadsThreads / PIECES][D];
  grid_dep_wait();
  const int tid = threadIdx.x, l = tid % PIECES, r0 = tid / PIECES;
  for (int e = tid; e < 2 * D; e += blockDim.x) s_w[e / D][e % D] = load_weight<BF16>(p.weight[e / D], p.weight_f32, e % D);
  __syncthreads();
  const HeadsLane t = heads_lane(l, p.rot, p.interleaved);
  const int H = p.Hq + 2 * p.Hkv, Hn = p.Hq + p.Hkv;
  float dw[2][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[0][e] = dw[1][e] = 0.f;
  for (long long tok = blockIdx.x; tok < p.tokens; tok += gridDim.x) {
    const int b = (int)(tok / p.S), i = (int)(tok - (long long)b * p.S);
    const uint16_t* x = static_cast<const uint16_t*>(p.qkv) + b * p.xs[0] + i * p.xs[1];
    uint16_t* dx = static_cast<uint16_t*>(p.dqkv) + (size_t)tok * H * D;
    const int angle = heads_angle(p, b, i, tid == 0);
    float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool turns = t.turns && angle >= 0;
    if (turns) {
      cs = *reinterpret_cast<const float4*>(p.cos + (size_t)angle * (p.rot / 2) + 4 * l);
      sn = *reinterpret_cast<const float4*>(p.sin + (size_t)angle * (p.rot / 2) + 4 * l);
    }
    for (int base = 0; base < H; base += UNROLL * p.rows) {
      uint2 u0[UNROLL], u1[UNROLL], g0[UNROLL], g1[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int row = base + u * p.rows + r0;
        u0[u] = u1[u] = g0[u] = g1[u] = make_uint2(0u, 0u);
        if (row < H && r0 < p.rows) {
          const int kind = row < p.Hq ? 0 : row < Hn ? 1 : 2;
          const int h = kind == 0 ? row : kind == 1 ? row - p.Hq : row - Hn;
          const uint16_t* dy =
              static_cast<const uint16_t*>(p.in[kind]) + b * p.hs[kind][0] + h * p.hs[kind][1] + i * p.hs[kind][2];
          g0[u] = *reinterpret_cast<const uint2*>(dy + t.c0);
          g1[u] = *reinterpret_cast<const uint2*>(dy + t.c1);
          if (kind < 2) {
            u0[u] = *reinterpret_cast<const uint2*>(x + row * p.xs[2] + t.c0);
            u1[u] = *reinterpret_cast<const uint2*>(x + row * p.xs[2] + t.c1);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        if (base + u * p.rows >= H) break;
        const int row = base + u * p.rows + r0;
        const int kind = row < p.Hq ? 0 : 1;  // (a value's x is 0 here, and its sums are not used)
        float f[8], d[8];
        heads_unpack<BF16>(u0[u], u1[u], f);
        heads_unpack<BF16>(g0[u], g1[u], d);
        if (turns) heads_turn(d, cs, sn, -1.f, p.interleaved);
        const float4 w0 = *reinterpret_cast<const float4*>(&s_w[kind][t.c0]), w1 = *reinterpret_cast<const float4*>(&s_w[kind][t.c1]);
        const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
        float ss = 0.f, dot = 0.f, dn[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          ss = fmaf(f[e], f[e], ss);
          dn[e] = d[e] * f[e];
          dot = fmaf(dn[e], w[e], dot);
        }
#pragma unroll
        for (int s = 1; s < PIECES; s <<= 1) {
          ss += __shfl_xor_sync(0xffffffffu, ss, s);
          dot += __shfl_xor_sync(0xffffffffu, dot, s);
        }
        if (row >= H || r0 >= p.rows) continue;
        uint16_t* y = dx + row * D;
        if (row >= Hn) {
          *reinterpret_cast<uint2*>(y + t.c0) = g0[u];
          *reinterpret_cast<uint2*>(y + t.c1) = g1[u];
          continue;
        }
        const float r = rsqrtf(ss * (1.f / D) + p.eps), m = r * r * dot * (1.f / D);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (kind == 0)
            dw[0][e] = fmaf(dn[e], r, dw[0][e]);
          else
            dw[1][e] = fmaf(dn[e], r, dw[1][e]);
          f[e] = r * (d[e] * w[e] - f[e] * m);
        }
        heads_store<BF16>(y, t, f);
      }
    }
  }
  // ---- the CTA's sums of the weights' gradients, in a fixed order
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    __syncthreads();
    *reinterpret_cast<float4*>(&s_sum[r0][t.c0]) = make_float4(dw[k][0], dw[k][1], dw[k][2], dw[k][3]);
    *reinterpret_cast<float4*>(&s_sum[r0][t.c1]) = make_float4(dw[k][4], dw[k][5], dw[k][6], dw[k][7]);
    __syncthreads();
    for (int c = tid; c < D; c += blockDim.x) {
      float sum = 0.f;
      for (int r = 0; r < p.rows; ++r) sum += s_sum[r][c];
      p.partial[((size_t)blockIdx.x * 2 + k) * D + c] = sum;
    }
  }
}

// The CTAs' sums added up, one warp for a column (grid: 2 D / 8, of 8 warps each).
template <bool BF16, int D>
__global__ void __launch_bounds__(256) coalibi_heads_sum_kernel(const HeadsParams p, int n) {
  grid_dep_wait();
  const int lane = threadIdx.x & 31, col = blockIdx.x * 8 + (threadIdx.x >> 5);
  float sum = 0.f;
  for (int i = lane; i < n; i += 32) sum += p.partial[(size_t)i * 2 * D + col];
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  void* y = p.dweight[col / D];
  if (lane != 0 || y == nullptr) return;
  if (p.weight_f32)
    static_cast<float*>(y)[col % D] = sum;
  else
    static_cast<uint16_t*>(y)[col % D] = (uint16_t)pack2<BF16>(sum, 0.f);
}

}  // namespace coalibi
