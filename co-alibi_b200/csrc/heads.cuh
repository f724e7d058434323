// Query, key and value heads out of a fused projection: queries and keys normed per head (root mean
// square, a weight for each column) and rotated by their position, values moved; with the backward.
//
// With x a row of D, r = 1 / sqrt(mean(x^2) + eps), n = r x, R the rotation of the row's position:
//   y = R (w n),   d = R^T dy,   dw = sum over rows of d n,   dx = r (w d - n mean(w d n)).
//
// Bound by the bytes: the projection read once and the heads written once (forward); the projection and
// the heads' gradients read, the projection's gradient written (backward; r is computed again rather than
// kept).  D / 16 lanes take a row, 16 columns each: those of a lane that rotates are both partners of its 8
// pairs, so a rotation needs no exchange.  A lane keeps its token and goes over a chunk of heads of one kind,
// with the token's angles in registers and the kind's weights in shared memory; the sums of a weight's gradient are a
// lane's own until the end.  With 8 columns to a lane, whose partners another lane had, forward and backward of 32,768
// tokens of 36 heads of 64 took 320 us, 157 with 16 and 128 with the ring of copies (below), where the bytes
// take 115; 32,764 tokens of 48 heads of 128 take 315 where the bytes take 306.
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
  float* partial;         // backward: [2][most CTAs of a kind][D]
  void* dweight[2];
  long long xs[3];        // batch, token, head
  long long hs[3][3];     // of q, k, v: batch, head, token
  int tokens;             // B * S
  int Hq, Hkv, S;
  int per[2];             // heads of a chunk: of queries, of keys and values
  int chunks[2];          // chunks of queries, of keys (and as many of values)
  int groups;             // token groups, one token to a slot of a CTA
  int per_cta;            // groups that a CTA goes over
  int ctas;               // for a chunk
  int rot, n_pos;
  int weight_f32;
  float eps;
};

constexpr int kHeadsThreads = 256;
constexpr int kHeadsChunk = 8;  // heads, at most

// A weight of column c, as float.
template <bool BF16>
__device__ __forceinline__ float load_weight(const void* w, int f32, int c) {
  if (w == nullptr) return 1.f;
  if (f32) return static_cast<const float*>(w)[c];
  const uint32_t u = static_cast<const uint16_t*>(w)[c];
  return unpack2<BF16>(u).x;
}

// A lane's 16 columns as the partners a and b of 8 pairs.  In halves (and where nothing turns) the pairs
// are (c0 + e, c1 + e), of two pieces of 8 columns; interleaved, neighbours.
struct HeadsRow {
  float2 a[4], b[4];
};
template <bool BF16, bool PAIRS>
__device__ __forceinline__ void heads_unpack(const uint4& p0, const uint4& p1, HeadsRow& x) {
  const uint32_t w0[4] = {p0.x, p0.y, p0.z, p0.w}, w1[4] = {p1.x, p1.y, p1.z, p1.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (PAIRS) {
      const float2 u = unpack2<BF16>(e < 2 ? w0[2 * e] : w1[2 * e - 4]), v = unpack2<BF16>(e < 2 ? w0[2 * e + 1] : w1[2 * e - 3]);
      x.a[e] = make_float2(u.x, v.x);
      x.b[e] = make_float2(u.y, v.y);
    } else {
      x.a[e] = unpack2<BF16>(w0[e]);
      x.b[e] = unpack2<BF16>(w1[e]);
    }
  }
}
template <bool BF16, bool PAIRS>
__device__ __forceinline__ void heads_pack(const HeadsRow& x, uint4& p0, uint4& p1) {
  uint32_t w0[4], w1[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (PAIRS) {
      (e < 2 ? w0[2 * e & 3] : w1[2 * e & 3]) = pack2<BF16>(x.a[e].x, x.b[e].x);
      (e < 2 ? w0[(2 * e & 3) + 1] : w1[(2 * e & 3) + 1]) = pack2<BF16>(x.a[e].y, x.b[e].y);
    } else {
      w0[e] = pack2<BF16>(x.a[e].x, x.a[e].y);
      w1[e] = pack2<BF16>(x.b[e].x, x.b[e].y);
    }
  }
  p0 = make_uint4(w0[0], w0[1], w0[2], w0[3]);
  p1 = make_uint4(w1[0], w1[1], w1[2], w1[3]);
}
__device__ __forceinline__ float2 splat(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 neg2(float2 x) { return make_float2(-x.x, -x.y); }

// Where a lane's two pieces of 8 columns are (lane l of D / 16 in a row): neighbouring lanes' lie side by side, so
// that a load or store of a row takes whole sectors.  In halves a lane that turns has the two partners of
// its pairs; interleaved, pairs lie within a piece, and each turns by itself.
struct HeadsLane {
  int c0, c1;
  int j0, j1;   // first angles of the pairs 0 .. 3 and 4 .. 7
  bool t0, t1;  // whether these turn
};
template <bool PAIRS, int D>
__device__ __forceinline__ HeadsLane heads_lane(int l, int rot) {
  HeadsLane t;
  if (PAIRS) {
    t.c0 = 8 * l, t.c1 = D / 2 + 8 * l;
    t.j0 = t.c0 / 2, t.j1 = t.c1 / 2;
    t.t0 = t.c0 < rot, t.t1 = t.c1 < rot;
  } else if (16 * l < rot) {
    t.c0 = 8 * l, t.c1 = rot / 2 + 8 * l;
    t.j0 = 8 * l, t.j1 = 8 * l + 4;
    t.t0 = t.t1 = true;
  } else {
    t.c0 = rot / 2 + 8 * l, t.c1 = D / 2 + 8 * l;  // rot + 8 (l - rot / 16), and (D - rot) / 2 after it
    t.j0 = t.j1 = 0;
    t.t0 = t.t1 = false;
  }
  return t;
}

// The weights of a kind in shared memory, in the order of each lane's pairs: piece e (a's first and last four,
// b's) of lane l at (e * LANES + l) * 4, so that a load takes every bank once.
template <bool BF16, bool PAIRS, int D>
__device__ __forceinline__ void heads_weights(const HeadsParams& p, int kind, float* s_w) {
  constexpr int LANES = D / 16;
  for (int at = threadIdx.x; at < D; at += kHeadsThreads) {
    const int e = at / (4 * LANES), l = at / 4 % LANES, i = e % 2 * 4 + at % 4;  // pair i, a or b of it
    const HeadsLane t = heads_lane<PAIRS, D>(l, p.rot);
    const int c = PAIRS ? (i < 4 ? t.c0 + 2 * i : t.c1 + 2 * i - 8) + e / 2 : (e < 2 ? t.c0 : t.c1) + i;
    s_w[at] = load_weight<BF16>(p.weight[kind], p.weight_f32, c);
  }
}
template <int LANES>
__device__ __forceinline__ float4 heads_weight(const float* s_w, int l, int e) {
  return *reinterpret_cast<const float4*>(s_w + (e * LANES + l) * 4);
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
// Cosines and sines of a lane's pairs.
struct HeadsAngles {
  float2 c[4], s[4];
};
// Whether the lane turns any pair of the row; if so, the angles.
__device__ __forceinline__ bool heads_angles(const HeadsParams& p, const HeadsLane& t, int l, int b, int i, bool valid, HeadsAngles& g) {
  if (!valid || !t.t0) return false;  // (t1 only with t0)
  const int row = heads_angle(p, b, i, l == 0);
  if (row < 0) return false;
  const float* c = p.cos + (size_t)row * (p.rot / 2);
  const float* s = p.sin + (size_t)row * (p.rot / 2);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float4 u = make_float4(1.f, 1.f, 1.f, 1.f), v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (e == 0 || t.t1) {
      u = *reinterpret_cast<const float4*>(c + (e ? t.j1 : t.j0));
      v = *reinterpret_cast<const float4*>(s + (e ? t.j1 : t.j0));
    }
    g.c[2 * e] = make_float2(u.x, u.y), g.c[2 * e + 1] = make_float2(u.z, u.w);
    g.s[2 * e] = make_float2(v.x, v.y), g.s[2 * e + 1] = make_float2(v.z, v.w);
  }
  return true;
}
// The pairs turned by the angles, or back by them.
template <bool BACK>
__device__ __forceinline__ void heads_turn(HeadsRow& x, const HeadsAngles& g, const HeadsLane& t) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (e >= 2 && !t.t1) break;  // (not by 1 and 0: 0 * infinity)
    const float2 a = x.a[e], b = x.b[e], s = BACK ? neg2(g.s[e]) : g.s[e];
    x.a[e] = __ffma2_rn(b, neg2(s), __fmul2_rn(a, g.c[e]));
    x.b[e] = __ffma2_rn(a, s, __fmul2_rn(b, g.c[e]));
  }
}

// What a CTA goes over: heads [h0, h0 + n) of a kind (0 queries, 1 keys, 2 values), token groups from `group`.
struct HeadsWork {
  int kind, h0, n, row0, group, end, index;  // row0: of the heads in the projection; index: of the CTA in its kind
};
__device__ __forceinline__ HeadsWork heads_work(const HeadsParams& p) {
  HeadsWork w;
  int chunk = blockIdx.x / p.ctas;
  const int at = blockIdx.x - chunk * p.ctas;
  w.index = chunk * p.ctas + at;
  w.kind = 0;
  if (chunk >= p.chunks[0]) {
    chunk -= p.chunks[0];
    w.index -= p.chunks[0] * p.ctas;
    w.kind = 1;
    if (chunk >= p.chunks[1]) {
      chunk -= p.chunks[1];
      w.kind = 2;
    }
  }
  const int per = p.per[w.kind > 0], H = w.kind == 0 ? p.Hq : p.Hkv;
  w.h0 = chunk * per;
  w.n = min(per, H - w.h0);
  w.row0 = (w.kind == 0 ? 0 : w.kind == 1 ? p.Hq : p.Hq + p.Hkv) + w.h0;
  w.group = at * p.per_cta;
  w.end = min(w.group + p.per_cta, p.groups);
  return w;
}

// Rows on their way: a thread's pieces of the next heads, copied to shared memory of its own (no other thread
// reads them, so nothing but its own copies is waited for).  A ring of registers holds less: the backward took
// 99 us with one head ahead in registers and no room for more.
constexpr int kHeadsStages = 4;
template <int N>  // pieces of a head
struct HeadsRing {
  static constexpr int BYTES = kHeadsStages * N * kHeadsThreads * 16;
  uint32_t base;
  int fill = 0, drain = 0;
  __device__ __forceinline__ explicit HeadsRing(void* smem) : base(smem_u32(smem) + threadIdx.x * 16) {}
  __device__ __forceinline__ void copy(int k, const uint16_t* from, bool valid) const {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(base + (fill * N + k) * kHeadsThreads * 16), "l"(from),
                 "r"(valid ? 16 : 0)
                 : "memory");
  }
  __device__ __forceinline__ void issued() {
    asm volatile("cp.async.commit_group;" ::: "memory");
    fill = fill + 1 == kHeadsStages ? 0 : fill + 1;
  }
  __device__ __forceinline__ void wait() const {  // for the oldest head
    asm volatile("cp.async.wait_group %0;" ::"n"(kHeadsStages - 1) : "memory");
  }
  __device__ __forceinline__ uint4 read(int k) const {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(base + (drain * N + k) * kHeadsThreads * 16));
    return v;
  }
  __device__ __forceinline__ void taken() { drain = drain + 1 == kHeadsStages ? 0 : drain + 1; }
};

// A token of the batch for a slot of a group.
struct HeadsToken {
  int tok, b, i;
  bool valid;
};
__device__ __forceinline__ HeadsToken heads_token(const HeadsParams& p, long long tok) {
  HeadsToken t;
  t.valid = tok < p.tokens;
  t.tok = t.valid ? (int)tok : 0;
  t.b = t.tok / p.S;
  t.i = t.tok - t.b * p.S;
  return t;
}

template <bool BF16, int D, bool PAIRS>
__global__ void __launch_bounds__(kHeadsThreads, 4) coalibi_heads_fwd_kernel(const HeadsParams p) {
  constexpr int LANES = D / 16, SLOTS = kHeadsThreads / LANES;
  extern __shared__ __align__(16) uint8_t s_ring[];
  __shared__ __align__(16) float s_w[D];
  grid_dep_wait();
  const int l = threadIdx.x % LANES, slot = threadIdx.x / LANES;
  const HeadsWork w = heads_work(p);
  const HeadsLane t = heads_lane<PAIRS, D>(l, p.rot);
  HeadsRing<2> ring(s_ring);
  int next_group = w.group, next_h = 0;
  const uint16_t* x = nullptr;
  bool next_valid = false;
  auto issue = [&]() {
    if (next_group < w.end) {
      if (next_h == 0) {
        const HeadsToken k = heads_token(p, (long long)next_group * SLOTS + slot);
        next_valid = k.valid;
        x = static_cast<const uint16_t*>(p.qkv) + k.b * p.xs[0] + k.i * p.xs[1] + w.row0 * p.xs[2];
      }
      ring.copy(0, x + t.c0, next_valid);
      ring.copy(1, x + t.c1, next_valid);
      x += p.xs[2];
      if (++next_h == w.n) next_h = 0, ++next_group;
    }
    ring.issued();
  };
#pragma unroll
  for (int k = 0; k < kHeadsStages - 1; ++k) issue();
  if (w.kind < 2) heads_weights<BF16, PAIRS, D>(p, w.kind, s_w);
  __syncthreads();
  for (int group = w.group; group < w.end; ++group) {
    const HeadsToken k = heads_token(p, (long long)group * SLOTS + slot);
    uint16_t* y = static_cast<uint16_t*>(p.out[w.kind]) + k.b * p.hs[w.kind][0] + w.h0 * p.hs[w.kind][1] + k.i * p.hs[w.kind][2];
    HeadsAngles g;
    const bool turns = w.kind < 2 && heads_angles(p, t, l, k.b, k.i, k.valid, g);
#pragma unroll 1
    for (int h = 0; h < w.n; ++h, y += p.hs[w.kind][1]) {
      issue();
      ring.wait();
      uint4 u0 = ring.read(0), u1 = ring.read(1);
      ring.taken();
      if (w.kind < 2) {
        HeadsRow f;
        heads_unpack<BF16, PAIRS>(u0, u1, f);
        float2 ss2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < 4; ++e) ss2 = __ffma2_rn(f.b[e], f.b[e], __ffma2_rn(f.a[e], f.a[e], ss2));
        float ss = ss2.x + ss2.y;
#pragma unroll
        for (int d = 1; d < LANES; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        const float2 r = splat(rsqrtf(ss * (1.f / D) + p.eps));
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float4 wa = heads_weight<LANES>(s_w, l, e / 2), wb = heads_weight<LANES>(s_w, l, 2 + e / 2);
          f.a[e] = __fmul2_rn(__fmul2_rn(f.a[e], r), make_float2(wa.x, wa.y));
          f.a[e + 1] = __fmul2_rn(__fmul2_rn(f.a[e + 1], r), make_float2(wa.z, wa.w));
          f.b[e] = __fmul2_rn(__fmul2_rn(f.b[e], r), make_float2(wb.x, wb.y));
          f.b[e + 1] = __fmul2_rn(__fmul2_rn(f.b[e + 1], r), make_float2(wb.z, wb.w));
        }
        if (turns) heads_turn<false>(f, g, t);
        heads_pack<BF16, PAIRS>(f, u0, u1);
      }
      if (k.valid) {
        *reinterpret_cast<uint4*>(y + t.c0) = u0;
        *reinterpret_cast<uint4*>(y + t.c1) = u1;
      }
    }
  }
}

template <bool BF16, int D, bool PAIRS>
__global__ void __launch_bounds__(kHeadsThreads, 2) coalibi_heads_bwd_kernel(const HeadsParams p) {
  constexpr int LANES = D / 16, SLOTS = kHeadsThreads / LANES;
  extern __shared__ __align__(16) uint8_t s_ring[];
  __shared__ __align__(16) float s_w[D], s_sum[kHeadsThreads / 32][D];
  grid_dep_wait();
  const int l = threadIdx.x % LANES, slot = threadIdx.x / LANES;
  const HeadsWork w = heads_work(p);
  const HeadsLane t = heads_lane<PAIRS, D>(l, p.rot);
  const int H = p.Hq + 2 * p.Hkv;
  HeadsRing<4> ring(s_ring);
  int next_group = w.group, next_h = 0;
  const uint16_t *x = nullptr, *dy = nullptr;
  bool next_valid = false;
  auto issue = [&]() {
    if (next_group < w.end) {
      if (next_h == 0) {
        const HeadsToken k = heads_token(p, (long long)next_group * SLOTS + slot);
        next_valid = k.valid;
        x = static_cast<const uint16_t*>(p.qkv) + k.b * p.xs[0] + k.i * p.xs[1] + w.row0 * p.xs[2];
        dy = static_cast<const uint16_t*>(p.in[w.kind]) + k.b * p.hs[w.kind][0] + w.h0 * p.hs[w.kind][1] + k.i * p.hs[w.kind][2];
      }
      ring.copy(0, dy + t.c0, next_valid);
      ring.copy(1, dy + t.c1, next_valid);
      if (w.kind < 2) {
        ring.copy(2, x + t.c0, next_valid);
        ring.copy(3, x + t.c1, next_valid);
      }
      x += p.xs[2];
      dy += p.hs[w.kind][1];
      if (++next_h == w.n) next_h = 0, ++next_group;
    }
    ring.issued();
  };
#pragma unroll
  for (int k = 0; k < kHeadsStages - 1; ++k) issue();
  if (w.kind < 2) heads_weights<BF16, PAIRS, D>(p, w.kind, s_w);
  __syncthreads();
  HeadsRow dw;
#pragma unroll
  for (int e = 0; e < 4; ++e) dw.a[e] = dw.b[e] = make_float2(0.f, 0.f);
  for (int group = w.group; group < w.end; ++group) {
    const HeadsToken k = heads_token(p, (long long)group * SLOTS + slot);
    uint16_t* dx = static_cast<uint16_t*>(p.dqkv) + ((size_t)k.tok * H + w.row0) * D;
    HeadsAngles g;
    const bool turns = w.kind < 2 && heads_angles(p, t, l, k.b, k.i, k.valid, g);
#pragma unroll 1
    for (int h = 0; h < w.n; ++h, dx += D) {
      issue();
      ring.wait();
      uint4 u0 = ring.read(0), u1 = ring.read(1);
      if (w.kind < 2) {
        HeadsRow f, d;
        heads_unpack<BF16, PAIRS>(u0, u1, d);
        heads_unpack<BF16, PAIRS>(ring.read(2), ring.read(3), f);
        if (turns) heads_turn<true>(d, g, t);
        float2 ss2 = make_float2(0.f, 0.f), dot2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 wa = heads_weight<LANES>(s_w, l, e / 2), wb = heads_weight<LANES>(s_w, l, 2 + e / 2);
          ss2 = __ffma2_rn(f.b[e], f.b[e], __ffma2_rn(f.a[e], f.a[e], ss2));
          dot2 = __ffma2_rn(__fmul2_rn(d.a[e], e & 1 ? make_float2(wa.z, wa.w) : make_float2(wa.x, wa.y)), f.a[e], dot2);
          dot2 = __ffma2_rn(__fmul2_rn(d.b[e], e & 1 ? make_float2(wb.z, wb.w) : make_float2(wb.x, wb.y)), f.b[e], dot2);
        }
        float ss = ss2.x + ss2.y, dot = dot2.x + dot2.y;
#pragma unroll
        for (int s = 1; s < LANES; s <<= 1) {
          ss += __shfl_xor_sync(0xffffffffu, ss, s);
          dot += __shfl_xor_sync(0xffffffffu, dot, s);
        }
        // a slot without a token (zeros) adds nothing, with an eps of 0 either; r times itself may overflow
        const float r = k.valid ? rsqrtf(ss * (1.f / D) + p.eps) : 0.f;
        const float2 r2 = splat(r), m2 = splat(-(r * (r * (dot * (1.f / D)))));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 wa = heads_weight<LANES>(s_w, l, e / 2), wb = heads_weight<LANES>(s_w, l, 2 + e / 2);
          dw.a[e] = __ffma2_rn(__fmul2_rn(d.a[e], f.a[e]), r2, dw.a[e]);
          dw.b[e] = __ffma2_rn(__fmul2_rn(d.b[e], f.b[e]), r2, dw.b[e]);
          d.a[e] = __fmul2_rn(d.a[e], e & 1 ? make_float2(wa.z, wa.w) : make_float2(wa.x, wa.y));
          d.b[e] = __fmul2_rn(d.b[e], e & 1 ? make_float2(wb.z, wb.w) : make_float2(wb.x, wb.y));
          f.a[e] = __fmul2_rn(__ffma2_rn(f.a[e], m2, d.a[e]), r2);
          f.b[e] = __fmul2_rn(__ffma2_rn(f.b[e], m2, d.b[e]), r2);
        }
        heads_pack<BF16, PAIRS>(f, u0, u1);
      }
      ring.taken();
      if (k.valid) {
        *reinterpret_cast<uint4*>(dx + t.c0) = u0;
        *reinterpret_cast<uint4*>(dx + t.c1) = u1;
      }
    }
  }
  if (w.kind == 2) return;
  // ---- the CTA's sums of the weight's gradient, in a fixed order: over a warp's tokens, then over the warps
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int s = LANES; s < 32; s <<= 1) {
      dw.a[e].x += __shfl_xor_sync(0xffffffffu, dw.a[e].x, s);
      dw.a[e].y += __shfl_xor_sync(0xffffffffu, dw.a[e].y, s);
      dw.b[e].x += __shfl_xor_sync(0xffffffffu, dw.b[e].x, s);
      dw.b[e].y += __shfl_xor_sync(0xffffffffu, dw.b[e].y, s);
    }
  if (lane < LANES) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = 2 * e + j;
        const int ca = PAIRS ? (i < 4 ? t.c0 + 2 * i : t.c1 + 2 * i - 8) : t.c0 + i, cb = PAIRS ? ca + 1 : t.c1 + i;
        s_sum[warp][ca] = j ? dw.a[e].y : dw.a[e].x;
        s_sum[warp][cb] = j ? dw.b[e].y : dw.b[e].x;
      }
  }
  __syncthreads();
  float* partial = p.partial + ((size_t)w.kind * p.ctas * p.chunks[0] + w.index) * D;  // (keys after all queries)
  for (int c = threadIdx.x; c < D; c += kHeadsThreads) {
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < kHeadsThreads / 32; ++r) sum += s_sum[r][c];
    partial[c] = sum;
  }
}

// The CTAs' sums added up: a CTA takes 32 columns of a kind (grid: 2 D / 32), its warps every 32nd row.
template <bool BF16, int D>
__global__ void __launch_bounds__(1024) coalibi_heads_sum_kernel(const HeadsParams p) {
  __shared__ float s_sum[32][33];
  grid_dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kind = blockIdx.x / (D / 32), col = (blockIdx.x % (D / 32)) * 32;
  const int n = p.ctas * p.chunks[kind];
  const float* x = p.partial + (size_t)kind * p.ctas * p.chunks[0] * D + col + lane;
  float sum = 0.f;
#pragma unroll 8
  for (int i = warp; i < n; i += 32) sum += x[(size_t)i * D];
  s_sum[warp][lane] = sum;
  __syncthreads();
  sum = s_sum[lane][warp];  // column `warp`, lane by lane
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  void* y = p.dweight[kind];
  if (lane != 0 || y == nullptr) return;
  if (p.weight_f32)
    static_cast<float*>(y)[col + warp] = sum;
  else
    static_cast<uint16_t*>(y)[col + warp] = (uint16_t)pack2<BF16>(sum, 0.f);
}

}  // namespace coalibi
