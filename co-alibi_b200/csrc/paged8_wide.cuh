// Attention over a paged cache in 8 bits for many rows per kv head (drafted trees): tcgen05.
//
// As in the 16-bit cache's kernel for such rows (paged.cuh), 64 rows stand twice in the 128 lanes of TMEM; two
// groups of warps work on keys of their own, 64 to a step, and the two halves of the lanes take the halves of a
// step, which come from two separate pieces of the item.  More rows go in blocks of 64.
//
// The tensor cores take the codes as float16, which holds them exactly, so each group has two warps that turn
// the codes of a step, as they arrive by TMA, into the swizzled tiles that the MMA reads; K's tile of the step after the next
// one is made as soon as the scores are out, V's as soon as its product is.  Scales enter the scores and the exponents of the
// weights as in the kernel for few rows (paged8.cuh).
//
// A group has eight softmax warps, 16 rows to each: four lanes share a row, 8 keys of its 32 to a lane.  The tiles' rows
// are in the order that makes those 8 consecutive keys (column 8 j + 2 q + e is key 8 q + 2 j + e), so that a row's suffix sum is
// additions in a lane and one scan over four, and a lane's keys have one scale.  With a row to a thread (four warps a group)
// the 32 keys of a step took a thread 2750 clocks, most of them its own latencies.
//
// Neither memory nor the tensor cores bound it but the softmax warps and the chain of a step: 8 trees of 16 tokens over
// 127 to 16,383 keys (64 rows to a kv head) take 73 us and 5 of joining, where the bytes take 21; twice the rows take
// 129 in all.  The warp-level products of few rows took 144 for the same trees.
#pragma once

#include "paged8.cuh"

namespace coalibi {

template <int D>
struct Wide8Layout {
  static constexpr int PIECES = 4;                 // of an item, per CTA
  static constexpr int STEP = 32;                  // keys of a piece per step
  static constexpr int UNIT = 128;
  static constexpr int COST = 10;                  // of starting and finishing an item, in units
  static constexpr int WHOLE = 1024;               // keys of a table that is not split
  static constexpr int ROWS = 64;
  static constexpr int TILE = 64 * D * 2;          // K or V of a step in float16: [D / 64][64 keys][128 bytes]
  static constexpr int BOX = 64 * 128;
  static constexpr int CODES = 64 * D;             // K or V of a step as codes: [64 keys][D], swizzled
  static constexpr int NCODE = 2, NTILE = 2;       // rings of steps
  static constexpr int GROUP = NTILE * 2 * TILE + NCODE * 2 * CODES;
  static constexpr int QBYTES = 128 * D * 2;       // [D / 64][128 rows][128 bytes]
  static constexpr int BYTES = QBYTES + 2 * GROUP + 1024;
  static constexpr int CTAS = 1;
  static constexpr int RECORD = ROWS * (4 + D);
  static constexpr bool SPREAD_SUMS = true;
  static constexpr int TM_S = 64, TM_O = 256;      // columns of an S buffer; O of group w at TM_O + w * D
  static constexpr int THREADS = 768;              // warps 0-15 softmax, 16 and 17 MMAs, 18 and 19 loads, 20-23 tiles
  // a group's part of the exchange (O in float, then statistics) reuses its rings
  static_assert(128 * D * 4 + 128 * 16 <= GROUP, "exchange fits the rings");
};

// Steps whose scales are kept: those of step n are written when K of step n - 2 is a tile, so the scores of step n - 4
// are out and the softmax warps past step n - 6.
constexpr int kWide8Meta = 6;

// 16 lanes of TMEM and 32 columns: register 4 j + 2 x + e holds row lane / 4 + 8 x, column 8 j + 2 (lane % 4) + e.
__device__ __forceinline__ void tmem_ld_quads(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : COALIBI_R8(0), COALIBI_R8(8)
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_quads(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      COALIBI_I8(0), COALIBI_I8(8)
      : "memory");
}
// 16 lanes and 16 columns: register 2 j + x holds row lane / 4 + 8 x, column 4 j + lane % 4.
__device__ __forceinline__ void tmem_st_quads16(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), COALIBI_I8(0) : "memory");
}
__device__ __forceinline__ float2 splat2(float x) { return make_float2(x, x); }

template <int D, bool BF16>
__global__ void __launch_bounds__(768, 1)
    coalibi_paged8_wide_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                               const Paged8Params p) {
  using L = Wide8Layout<D>;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t s_kc[2][2], s_kc_free[2][2], s_vc[2][2], s_vc_free[2][2];  // codes
  __shared__ uint64_t s_k[2][2], s_k_free[2][2], s_v[2][2], s_v_free[2][2];      // tiles
  __shared__ uint64_t s_scores[2][2], s_probs[2][2], s_meta[2][4], s_pv[2][2], s_idle[2];
  // of a step: the scales of its four blocks of 16 keys; which of them were not loaded (bits 0-3), and 16 where some
  // key of the step is not of the context, or a scale of V is one that odd_scale() names
  __shared__ __align__(16) float s_ks[2][kWide8Meta][4];
  __shared__ __align__(16) float s_vs[2][kWide8Meta][4];
  __shared__ unsigned char s_gone[2][kWide8Meta];
  __shared__ __align__(16) union {
    int pre[128];
    uint32_t nan[kTreeMaxSq][4];  // columns of a drafted token's V that are NaN
  } s_u;
  __shared__ int s_any_nan;
  __shared__ signed char s_up[128];  // exponents of the powers of two by which the queries' rows are scaled
  __shared__ int s_warp[4], s_find, s_abort;
  __shared__ uint32_t s_tmem;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool softmax = warp < 16, issues = warp == 16 || warp == 17, loads = warp == 18 || warp == 19;
  const int w = softmax ? warp >> 3 : warp < 20 ? warp & 1 : (warp - 20) >> 1;  // group
  const int G = p.Hq / p.Hkv, rows = G * p.Sq;
  const int heads = p.Hkv * p.row_blocks;
  const CtaGuard guard{&s_abort, p.status, kPagedTimeoutNs};
  if (tid == 0) {
    for (int g = 0; g < 2; ++g) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_kc[g][i], 1);
        mbar_init(&s_kc_free[g][i], 2);
        mbar_init(&s_vc[g][i], 1);
        mbar_init(&s_vc_free[g][i], 2);
        mbar_init(&s_k[g][i], 2);
        mbar_init(&s_k_free[g][i], 1);
        mbar_init(&s_v[g][i], 2);
        mbar_init(&s_v_free[g][i], 1);
        mbar_init(&s_scores[g][i], 1);
        mbar_init(&s_probs[g][i], 8);
        mbar_init(&s_pv[g][i], 1);
      }
      for (int i = 0; i < 4; ++i) mbar_init(&s_meta[g][i], 1);
      mbar_init(&s_idle[g], 1);
    }
    s_abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  if (warp == 16) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  grid_dep_wait();

  unsigned at = 0, stop;
  int b = 0, span = 1, item = 0, v0 = 0;
  if (p.whole) {
    b = blockIdx.x / heads;
    item = blockIdx.x - b * heads;
    span = paged_span<L>(p, b);
    stop = span;
  } else {
    int* head = reinterpret_cast<int*>(p.ws);
    const int per = (p.B + 127) / 128;
    const unsigned total = (unsigned)paged_prefix<L>(p, s_u.pre, s_warp, per, blockIdx.x == 0 ? head : nullptr) * heads;
    const unsigned quota = (total + p.n_ctas - 1) / p.n_ctas;
    if (blockIdx.x == 0 && tid == 0) head[p.B + 1] = (int)quota;
    at = quota * blockIdx.x;
    stop = min(total, at + quota);
    if (at < stop) paged_find<L>(p, s_u.pre, &s_find, per, heads, at, b, span, item, v0);
    __syncthreads();  // s_u is used otherwise from here on
  }

  uint8_t* const rings = smem + L::QBYTES + w * L::GROUP;
  uint8_t* const k_tiles = rings;
  uint8_t* const v_tiles = rings + L::NTILE * L::TILE;
  uint8_t* const codes = rings + 2 * L::NTILE * L::TILE;  // [slot][K, V]
  uint32_t seq = 0;  // steps of this group in earlier items: the barriers' phases go on
  bool ok = true;
  while (at < stop) {
    const int v1 = (int)min((unsigned)span, v0 + (stop - at));
    const int u0 = max(v0 - L::COST, 0), u1 = v1 - L::COST, units = span - L::COST;
    if (u1 <= 0) break;
    const int g = item / p.row_blocks, rb = (item - g * p.row_blocks) * L::ROWS;
    const int len = p.ctx_lens[b], room = p.max_pages * p.page_size, ctx = min(max(len, 0), room);
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
    // the pieces: `sub` keys each, the group's first at piece PIECES / 2 * w
    const int s_lo = u0 * L::UNIT, s_hi = min(min(u1 * L::UNIT, room), ctx + drafts);
    const int sub = ((max(s_hi - s_lo, 0) + L::PIECES - 1) / L::PIECES + 15) & ~15;
    auto piece_lo = [&](int q) { return s_lo + q * sub; };
    auto piece_hi = [&](int q) { return min(s_hi, s_lo + (q + 1) * sub); };
    auto piece_steps = [&](int q) { return max(0, (piece_hi(q) - piece_lo(q) + L::STEP - 1) / L::STEP); };
    const int q0 = L::PIECES / 2 * w;
    const int nsteps = max(piece_steps(q0), piece_steps(q0 + 1));
    // first key of half hf of step n (counted from the right); its piece's ends
    auto half_base = [&](int n, int hf) { return piece_lo(q0 + hf) + (piece_steps(q0 + hf) - 1 - n) * 32; };
    auto half_hi = [&](int hf) { return piece_hi(q0 + hf); };
    auto half_lo = [&](int hf) { return piece_lo(q0 + hf); };

    // ---- loads: step n of the group, by one warp; lane i < 4 looks up the step's block i
    int k_loaded = 0, v_loaded = 0;
    auto load = [&](int n) {
      const uint32_t k = seq + n;
      const int slot = k % L::NCODE, meta = k % kWide8Meta;
      int page = -1, at_slot = 0;
      bool inside = true;  // all keys of the block's half are of the context
      if (lane < 4) {
        const int base = half_base(n, lane >> 1), key = base + 16 * (lane & 1);
        inside = base + 32 <= min(half_hi(lane >> 1), ctx);
        if (key >= half_lo(lane >> 1) && key < half_hi(lane >> 1)) {
          const int t = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
          page = p.page_table[(size_t)b * p.table_stride + t];
          at_slot = key - t * p.page_size;
          if ((unsigned)page >= (unsigned)p.n_pages) {
            page = -1;
            report_page(p.status);
          }
        }
      }
      float ks = 1.f, vs = 1.f;
      if (page >= 0) {
        ks = p.k_scales[page * p.kss[0] + g * p.kss[1] + at_slot / kQuantBlock];
        vs = p.v_scales[page * p.vss[0] + g * p.vss[1] + at_slot / kQuantBlock];
      }
      const int gone = (int)(__ballot_sync(0xffffffffu, lane < 4 && page < 0) & 15u);
      const bool plain = gone == 0 && __all_sync(0xffffffffu, inside && !odd_scale(vs));
      const uint32_t dst = smem_u32(codes + slot * 2 * L::CODES), bytes = (4 - __popc(gone)) * 16 * D;
      if (!__all_sync(0xffffffffu, mbar_wait(&s_kc_free[w][slot], ((k / L::NCODE) & 1) ^ 1, guard))) return false;
      if (lane == 0) mbar_expect_tx(&s_kc[w][slot], bytes);
      __syncwarp();
      if (page >= 0) tma_load_4d(dst + lane * 16 * D, &tk, &s_kc[w][slot], 0, at_slot, g, page);
      if (lane < 4) s_ks[w][meta][lane] = ks, s_vs[w][meta][lane] = vs;
      if (lane == 0) s_gone[w][meta] = (unsigned char)(plain ? 0 : gone | 16);
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_kc[w][slot]);  // (the scales are in, too)
      ++k_loaded;
      if (!__all_sync(0xffffffffu, mbar_wait(&s_vc_free[w][slot], ((k / L::NCODE) & 1) ^ 1, guard))) return false;
      if (lane == 0) mbar_arrive_expect_tx(&s_vc[w][slot], bytes);
      __syncwarp();
      if (page >= 0) tma_load_4d(dst + L::CODES + lane * 16 * D, &tv, &s_vc[w][slot], 0, at_slot, g, page);
      ++v_loaded;
      return true;
    };
    const int ahead = min(nsteps, L::NCODE);  // the rings are free: these start beside the queries
    if (loads)
      for (int n = 0; n < ahead && ok; ++n) ok = load(n);
    if (softmax) {
      // ---- the queries, in the K-major 128-byte-swizzled form the MMA reads; bfloat16 ones as float16, scaled by
      // a power of two that puts a row's largest at 2^14
      for (int c = tid; c < 128 * (D / 8); c += 512) {
        const int r = c / (D / 8), ch = c % (D / 8), row = rb + (r & 63);
        uint4 val = make_uint4(0u, 0u, 0u, 0u);
        if (row < rows)
          val = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + b * p.qs[0] +
                                                (g * G + row / p.Sq) * p.qs[1] + (row % p.Sq) * p.qs[2] + ch * 8);
        if (BF16) {
          uint32_t x[4] = {val.x, val.y, val.z, val.w}, most = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) most = max(most, max(x[e] << 16 & 0x7f800000u, x[e] & 0x7f800000u));
#pragma unroll
          for (int d = 1; d < D / 8; d <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
          const int up = 14 - min(max((int)(most >> 23) - 127, -100), 127);
          const float by = __int_as_float((up + 127) << 23);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = unpack2<true>(x[e]);
            x[e] = pack2<false>(f.x * by, f.y * by);
          }
          val = make_uint4(x[0], x[1], x[2], x[3]);
          if (ch == 0) s_up[r] = (signed char)up;
        }
        *reinterpret_cast<uint4*>(smem + (ch >> 3) * (128 * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = val;
      }
      if (tid < kTreeMaxSq) *reinterpret_cast<uint4*>(s_u.nan[tid]) = make_uint4(0u, 0u, 0u, 0u);
      if (tid == 0) s_any_nan = 0;
      fence_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();

    if (loads) {
      for (int n = ahead; n < nsteps && ok; ++n) ok = load(n);
      // every issued copy lands before the item (and the CTA) ends
      if (lane == 0)
        for (int n = 0; n < L::NCODE; ++n) {
          const uint32_t kk = seq + k_loaded - 1 - n, kv = seq + v_loaded - 1 - n;
          if (n < k_loaded) mbar_drain(&s_kc[w][kk % L::NCODE], (kk / L::NCODE) & 1, guard.timeout_ns);
          if (n < v_loaded) mbar_drain(&s_vc[w][kv % L::NCODE], (kv / L::NCODE) & 1, guard.timeout_ns);
        }
      __syncwarp();
    } else if (warp >= 20) {
      // ---------------------------------------------------------- codes to tiles
      // A thread takes 16 codes at a time, of keys 16 apart.  The eight threads of a pass over shared memory take
      // chunks 0-3 of a key of even number and 4-7 of the next one (and then the others; with 64 columns, all four of
      // both), which hit all phases of both swizzles.
      const int t = (warp & 1) * 32 + lane, odd = t >> 2 & 1, key0 = 2 * (t >> 3) + odd, c0 = D == 128 ? (t & 3) + 4 * odd : t & 3;
      const uint32_t from0 = key0 * D + ((c0 ^ (D == 128 ? key0 & 7 : key0 >> 1 & 3)) << 4);
      const int row0 = 8 * (key0 >> 1 & 3) + 2 * (key0 >> 3) + odd;  // of key0; 16 keys on, 4 rows; 32 keys on, 32
      const uint32_t to0 = (c0 >> 2) * L::BOX + row0 * 128 + (((2 * c0 & 7) ^ row0 & 7) << 4);
      constexpr int OTHER = D / 64;  // chunks of a key that a thread takes
      auto convert = [&](const uint8_t* from, uint8_t* to, int i, int v, bool zero, bool takes_nan, uint32_t& nan) {
        const uint4 u = *reinterpret_cast<const uint4*>(from + (from0 ^ (v << 6)) + i * 16 * D);
        uint32_t x[4] = {u.x, u.y, u.z, u.w};
        if (zero) x[0] = x[1] = x[2] = x[3] = 0u;
        if (takes_nan) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t bad = __vcmpeq4(x[j] & 0x7f7f7f7fu, 0x7f7f7f7fu);  // a byte of ones each
            x[j] &= ~bad;
            nan |= ((bad & 1u) | (bad >> 7 & 2u) | (bad >> 14 & 4u) | (bad >> 21 & 8u)) << (4 * j);
          }
        }
        uint32_t h[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) e4m3_to_f16x4(x[j], h[2 * j], h[2 * j + 1]);
        const uint32_t at = ((to0 ^ (v * L::BOX)) + (i >> 1) * 4096 + (i & 1) * 512) ^ ((i & 1) << 6);
        *reinterpret_cast<uint4*>(to + at) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(to + (at ^ 16)) = make_uint4(h[4], h[5], h[6], h[7]);
      };
      auto convert_all = [&](const uint8_t* from, uint8_t* to) {
        uint32_t none = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int v = 0; v < OTHER; ++v) convert(from, to, i, v, false, false, none);
      };
      auto make_k = [&](int n) {
        const uint32_t k = seq + n;
        const int slot = k % L::NCODE, tile = k % L::NTILE;
        ok = mbar_wait(&s_kc[w][slot], (k / L::NCODE) & 1, guard) && mbar_wait(&s_k_free[w][tile], ((k / L::NTILE) & 1) ^ 1, guard);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        if (t == 0) mbar_arrive(&s_meta[w][k & 3]);  // the scales, to the softmax warps
        convert_all(codes + slot * 2 * L::CODES, k_tiles + tile * L::TILE);
        fence_async_smem();
        __syncwarp();  // (one arrival for the warp: those of its threads would be taken one by one)
        if (lane == 0) {
          mbar_arrive(&s_k[w][tile]);
          mbar_arrive(&s_kc_free[w][slot]);
        }
      };
      auto make_v = [&](int n) {
        const uint32_t k = seq + n;
        const int slot = k % L::NCODE, tile = k % L::NTILE;
        ok = mbar_wait(&s_vc[w][slot], (k / L::NCODE) & 1, guard) && mbar_wait(&s_v_free[w][tile], ((k / L::NTILE) & 1) ^ 1, guard);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        const uint8_t* from = codes + slot * 2 * L::CODES + L::CODES;
        uint8_t* to = v_tiles + tile * L::TILE;
        const int gone = s_gone[w][k % kWide8Meta];
        if (gone == 0) {
          convert_all(from, to);
        } else {
          // V rows that no row sees (past the end, of no page, unseen drafts) may hold any code: zeros, 0 * NaN
          // is not 0.  What is NaN of a drafted token must not reach the rows that do not see it: zeros too, and
          // the rows that do get their NaN at the end.
#pragma unroll 1
          for (int e = 0; e < 4 * OTHER; ++e) {
            const int i = e / OTHER, v = e % OTHER, key = key0 + 16 * i, c = c0 ^ (4 * v);
            const int hf = key >> 5, base = half_base(n, hf), pos = base + (key & 31);
            const bool used = base >= half_lo(hf) && !(gone >> (key >> 4) & 1) && pos < half_hi(hf) &&
                              (pos < ctx || (seen_by_any >> (pos - ctx) & 1));
            uint32_t nan = 0;
            convert(from, to, i, v, !used, used && pos >= ctx, nan);
            if (nan != 0) {
              atomicOr(&s_u.nan[pos - ctx][c >> 1], nan << (16 * (c & 1)));
              s_any_nan = 1;
            }
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&s_v[w][tile]);
          mbar_arrive(&s_vc_free[w][slot]);
        }
      };
      // K(0), K(1), V(0), K(2), V(1), ...: K's tile is free once the scores before the last are out
      if (nsteps > 0 && ok) make_k(0);
      for (int n = 0; n < nsteps && ok; ++n) {
        if (n + 1 < nsteps) make_k(n + 1);
        if (ok) make_v(n);
      }
    } else if (issues) {
      // ---------------------------------------------------------- MMAs (lane 0 issues)
      constexpr uint32_t idS = make_idesc_f16(false, 128, 64, false, false);
      constexpr uint32_t idPV = make_idesc_f16(false, 128, D, false, true);
      const uint32_t q_addr = smem_u32(smem), k_addr0 = smem_u32(k_tiles), v_addr0 = smem_u32(v_tiles);
      auto issue_scores = [&](int n) {
        const uint32_t k = seq + n;
        const int tile = k % L::NTILE;
        if (!__all_sync(0xffffffffu, mbar_wait(&s_k[w][tile], (k / L::NTILE) & 1, guard))) return false;
        if (lane == 0) {
          tc_fence_after();
          const uint32_t d = tmem + (2 * w + (k & 1)) * L::TM_S, k_addr = k_addr0 + tile * L::TILE;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_ss(d, make_sdesc_sw128(q_addr + (kk >> 2) * (128 * 128) + (kk & 3) * 32, 16, 1024),
                    make_sdesc_sw128(k_addr + (kk >> 2) * L::BOX + (kk & 3) * 32, 16, 1024), idS, kk > 0 ? 1u : 0u);
          umma_commit(&s_scores[w][k & 1]);
          umma_commit(&s_k_free[w][tile]);
        }
        __syncwarp();
        return true;
      };
      // S(0), S(1), PV(0), S(2), PV(1), ...: S(n + 2) overwrites the buffer that PV(n), issued
      // before it by this thread, has read P from
      for (int n = 0; n < 2 && n < nsteps && ok; ++n) ok = issue_scores(n);
      for (int n = 0; n < nsteps && ok; ++n) {
        const uint32_t k = seq + n;
        const int tile = k % L::NTILE;
        ok = mbar_wait(&s_probs[w][k & 1], (k >> 1) & 1, guard) && mbar_wait(&s_v[w][tile], (k / L::NTILE) & 1, guard);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        if (lane == 0) {
          tc_fence_after();
          const uint32_t pa = tmem + (2 * w + (k & 1)) * L::TM_S, v_addr = v_addr0 + tile * L::TILE;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_ts(tmem + L::TM_O + w * D, pa + kk * 8, make_sdesc_sw128(v_addr + kk * 16 * 128, L::BOX, 1024), idPV,
                    n > 0 || kk > 0 ? 1u : 0u);
          umma_commit(&s_pv[w][k & 1]);
          umma_commit(&s_v_free[w][tile]);
        }
        __syncwarp();
        if (n + 2 < nsteps) ok = issue_scores(n + 2);
      }
      if (!ok && lane == 0) {  // what was issued must have finished before TMEM is released
        umma_commit(&s_idle[w]);
        mbar_drain(&s_idle[w], 0, guard.timeout_ns);
      }
      __syncwarp();
    } else {
      // ---------------------------------------------------------- softmax: two rows of 8 keys to a lane
      const int t0 = (warp & 3) * 32 + (warp >> 2 & 1) * 16, hf = t0 >> 6, q = lane & 3;
      const uint32_t lane_base = tmem + ((uint32_t)t0 << 16);
      const uint32_t o_base = lane_base + L::TM_O + w * D;
      int row_of[2];       // of the request's drafted tokens
      float slope2[2], c_a[2], m[2], l[2], carry[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int t = t0 + (lane >> 2) + 8 * x, r = rb + (t & 63), rr = r < rows ? r : rb;
        row_of[x] = rr % p.Sq;
        slope2[x] = load_slope(p.slopes, p.slopes_dtype, g * G + rr / p.Sq) * kLog2e;
        c_a[x] = p.sm_scale * kLog2e * (BF16 ? __int_as_float((127 - s_up[t]) << 23) : 1.f);
        m[x] = -INFINITY;
        l[x] = carry[x] = 0.f;
      }
      bool left = false;
      for (int n = 0; n < nsteps; ++n) {
        const uint32_t k = seq + n;
        const int meta = k % kWide8Meta;
        const uint32_t s_base = lane_base + (2 * w + (k & 1)) * L::TM_S;
        if (ok) ok = mbar_wait(&s_meta[w][k & 3], (k >> 2) & 1, guard);
        if (ok) ok = mbar_wait(&s_scores[w][k & 1], (k >> 1) & 1, guard);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          left = true;
          break;
        }
        const int gone = s_gone[w][meta];
        uint32_t pk[8];
        float alpha[2] = {1.f, 1.f};
        bool rescale = false;
        tc_fence_after();
        uint32_t s[16];
        tmem_ld_quads(s_base + 32 * hf, s);
        const float k_scale = s_ks[w][meta][2 * hf + (q >> 1)], v_scale = s_vs[w][meta][2 * hf + (q >> 1)];
        const float held = fminf(fmaxf(fabsf(v_scale), kScaleHeldMin), kScaleHeldMax);  // (v_scale itself, unless odd)
        const float lv = lg2_approx(held), iv = rcp_approx(held);
        uint32_t seen[2] = {0xffu, 0xffu};  // of this lane's 8 keys
        if (gone != 0) {
          const int base = half_base(n, hf), in = min(half_hi(hf), ctx) - base, end = half_hi(hf) - base;
          const uint32_t context = in >= 32 ? 0xffffffffu : in > 0 ? (1u << in) - 1u : 0u;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            uint32_t v = context;
            if (end > in && end > 0) {  // drafted tokens, up to `end`
              const unsigned long long word = p.tree_mask != nullptr
                                                  ? (unsigned long long)p.tree_mask[b * p.mask_stride + row_of[x]]
                                                  : (2ull << row_of[x]) - 1;
              const int d = base - ctx;
              const uint32_t bits = d >= 0 ? (d < 64 ? (uint32_t)(word >> d) : 0u) : d > -32 ? (uint32_t)word << -d : 0u;
              v |= bits & (end >= 32 ? 0xffffffffu : (1u << end) - 1u) & ~context;
            }
            if (base < half_lo(hf)) v = 0u;  // this piece has ended
            if (gone >> (2 * hf) & 1) v &= 0xffff0000u;
            if (gone >> (2 * hf + 1) & 1) v &= 0x0000ffffu;
            seen[x] = v >> (8 * q) & 0xffu;
          }
        }
        // pair j of row x: keys 8 q + 2 j and the next one
        auto pair = [&](int j, int x) { return make_float2(__uint_as_float(s[4 * j + 2 * x]), __uint_as_float(s[4 * j + 2 * x + 1])); };
        auto keep = [&](int j, int x, float2 v) { s[4 * j + 2 * x] = __float_as_uint(v.x), s[4 * j + 2 * x + 1] = __float_as_uint(v.y); };
        auto step = [&](auto masked) {
          constexpr bool MASKED = decltype(masked)::value;
          auto mask = [&](int j, int x, float2 v, float none) {
            return make_float2(seen[x] >> (2 * j) & 1 ? v.x : none, seen[x] >> (2 * j + 1) & 1 ? v.y : none);
          };
          float tot[2], inc[2], mx[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float run = 0.f;
            const float2 f = splat2(c_a[x] * k_scale);
#pragma unroll
            for (int j = 3; j >= 0; --j) {
              const float2 y = __fmul2_rn(pair(j, x), f);
              const float2 dn = __fadd2_rn(make_float2(ex2_approx(-y.x), ex2_approx(-y.y)), splat2(1.f));
              float2 sg = make_float2(rcp_approx(dn.x), rcp_approx(dn.y));
              if (MASKED) sg = mask(j, x, sg, 0.f);
              const float z1 = run + sg.y;
              run = z1 + sg.x;
              keep(j, x, __ffma2_rn(splat2(-slope2[x]), make_float2(run, z1), y));
            }
            tot[x] = inc[x] = run;
          }
#pragma unroll
          for (int d = 1; d <= 2; ++d)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float y = __shfl_down_sync(0xffffffffu, inc[x], d);
              if (q + d < 4) inc[x] += y;
            }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float2 sh = splat2(-slope2[x] * (carry[x] + (inc[x] - tot[x])));
            carry[x] += __shfl_sync(0xffffffffu, inc[x], lane & ~3);
            mx[x] = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float2 v = __fadd2_rn(pair(j, x), sh);
              if (MASKED) v = mask(j, x, v, -INFINITY);
              keep(j, x, v);
              mx[x] = fmaxf(mx[x], fmaxf(v.x, v.y));
            }
            mx[x] += lv;
          }
#pragma unroll
          for (int d = 1; d <= 2; ++d)
#pragma unroll
            for (int x = 0; x < 2; ++x) mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], d));
          // the reference moves only when a contribution passes it by 2^8: weights stay below 256, and
          // O needs rescaling rarely
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (mx[x] > m[x] + 8.f || (m[x] == -INFINITY && mx[x] > -INFINITY)) {
              const PieceFactor<L> f(m[x] - mx[x]);
              rescale |= m[x] != -INFINITY;
              alpha[x] = m[x] != -INFINITY ? f.f : 1.f;
              l[x] = f.of_sum(l[x]);
              m[x] = mx[x];
            }
            const float ref = m[x] == -INFINITY ? 0.f : m[x];
            const float2 sh = splat2(lv - ref);
            const bool odd = MASKED && odd_scale(v_scale);  // (paged8.cuh)
            float2 ls = splat2(0.f);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 v = __fadd2_rn(pair(j, x), sh);
              float2 e = make_float2(ex2_approx(v.x), ex2_approx(v.y));
              if (odd) {  // (exponentials of their own for the sum: the roots, as there, cost the plain steps 1%)
                const float2 y = pair(j, x);
                ls = __fadd2_rn(ls, mask(j, x, make_float2(ex2_approx(y.x - ref), ex2_approx(y.y - ref)), 0.f));
                e = __fmul2_rn(e, splat2(v_scale * iv));
              }
              if (MASKED) e = mask(j, x, e, 0.f);  // (a block that nothing of is seen may have any scale)
              if (!odd) ls = __fadd2_rn(ls, e);
              pk[2 * j + x] = pack2<false>(e.x, e.y);
            }
            // the weights themselves: without the block's scale
            l[x] = fmaf(ls.x + ls.y, odd ? 1.f : iv, l[x]);
          }
        };
        if (gone == 0)
          step(std::false_type{});
        else
          step(std::true_type{});
        if (__any_sync(0xffffffffu, rescale)) {
          // every PV before this step's must have added its part
          if (n > 0) ok = mbar_wait(&s_pv[w][(k - 1) & 1], ((k - 1) >> 1) & 1, guard);
          ok = __all_sync(0xffffffffu, ok);
          if (ok && n > 0) {
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[16];
              tmem_ld_quads(o_base + c, o);
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha[j >> 1 & 1]);
              tmem_st_quads(o_base + c, o);
            }
          }
        }
        // ---- P over this step's scores
        if (!ok) {
          left = true;
          break;
        }
        __syncwarp();  // (the loads and stores of TMEM take converged warps)
        const uint32_t none[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
        tmem_st_quads16(s_base + 16 * hf, pk);
        tmem_st_quads16(s_base + 16 * (1 - hf), none);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_probs[w][k & 1]);
      }
      // ---- this group's pieces to the exchange: O, swizzled by row, and the statistics
      // (the last scores imply every PV but the last two, each of which has a barrier of its own: on one barrier
      // both might complete between two looks at it, and its parity be what it was)
      for (int n = max(nsteps - 2, 0); n < nsteps && ok && !left; ++n)
        ok = mbar_wait(&s_pv[w][(seq + n) & 1], ((seq + n) >> 1) & 1, guard);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after();
        float* xo = reinterpret_cast<float*>(rings);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
          l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
          if (q == 0) reinterpret_cast<float4*>(xo + 128 * D)[t0 + (lane >> 2) + 8 * x] = make_float4(carry[x], m[x], l[x], slope2[x]);
        }
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = 0u;
          if (nsteps > 0) tmem_ld_quads(o_base + c, o);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int t = t0 + (lane >> 2) + 8 * x, col = c + 8 * j + 2 * q;
              *reinterpret_cast<uint2*>(xo + t * D + (((col >> 2) ^ (t & (D / 4 - 1))) << 2) + (col & 3)) =
                  make_uint2(o[4 * j + 2 * x], o[4 * j + 2 * x + 1]);
            }
        }
      }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (*static_cast<volatile int*>(&s_abort) != 0) break;

    // ---- pieces join, right to left
    const bool whole = u0 == 0 && u1 == units;
    float* rec = p.ws + paged_ws_head(p.B) + ((size_t)blockIdx.x * 2 + (u0 > 0 ? 0 : 1)) * L::RECORD;
    const int n_rows = min(L::ROWS, rows - rb);
    for (int e = tid; e < n_rows * (D / 4); e += L::THREADS) {
      const int r = e / (D / 4), ch = e % (D / 4);
      float right = 0.f, M = -INFINITY, wt[L::PIECES];
#pragma unroll
      for (int q = L::PIECES - 1; q >= 0; --q) {
        const int lane_row = r + 64 * (q & 1), grp = q >> 1;
        const float* xo = reinterpret_cast<const float*>(smem + L::QBYTES + grp * L::GROUP);
        const float4 st = reinterpret_cast<const float4*>(xo + 128 * D)[lane_row];
        wt[q] = st.y == -INFINITY ? -INFINITY : st.y - st.w * right;
        M = fmaxf(M, wt[q]);
        right += st.x;
      }
      const float m_use = M == -INFINITY ? 0.f : M;
      float l = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int q = L::PIECES - 1; q >= 0; --q) {
        const int lane_row = r + 64 * (q & 1), grp = q >> 1;
        const float* xo = reinterpret_cast<const float*>(smem + L::QBYTES + grp * L::GROUP);
        const PieceFactor<L> pf(wt[q] - m_use);
        const float f = pf.f;
        l += pf.of_sum(reinterpret_cast<const float4*>(xo + 128 * D)[lane_row].z);
        const float4 v = *reinterpret_cast<const float4*>(xo + lane_row * D + ((ch ^ (lane_row & (D / 4 - 1))) << 2));
        acc.x = fmaf(v.x, f, acc.x);
        acc.y = fmaf(v.y, f, acc.y);
        acc.z = fmaf(v.z, f, acc.z);
        acc.w = fmaf(v.w, f, acc.w);
      }
      if (s_any_nan != 0) {  // a drafted token that the row sees
        const int row_of = (rb + r) % p.Sq;
        unsigned long long word =
            p.tree_mask != nullptr ? (unsigned long long)p.tree_mask[b * p.mask_stride + row_of] : (2ull << row_of) - 1;
        if (p.Sq < 64) word &= (1ull << p.Sq) - 1;
        uint32_t bad = 0;
        for (; word != 0; word &= word - 1) bad |= s_u.nan[__ffsll((long long)word) - 1][ch >> 3] >> (4 * (ch & 7));
        const float nan = __int_as_float(0x7fc00000);
        if (bad & 1) acc.x = nan;
        if (bad & 2) acc.y = nan;
        if (bad & 4) acc.z = nan;
        if (bad & 8) acc.w = nan;
      }
      if (whole) {
        const int rr = rb + r;
        uint16_t* y = static_cast<uint16_t*>(p.o) + b * p.os[0] + (g * G + rr / p.Sq) * p.os[1] + (rr % p.Sq) * p.os[2];
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        *reinterpret_cast<uint2*>(y + 4 * ch) =
            make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
      } else {
        if (ch == 0) reinterpret_cast<float4*>(rec)[r] = make_float4(right, M, l, 0.f);
        *reinterpret_cast<float4*>(rec + 4 * L::ROWS + r * D + 4 * ch) = acc;
      }
    }
    fence_async_smem();  // the exchange before the loads that refill the rings
    __syncthreads();

    seq += nsteps;
    at += v1 - v0;
    v0 = 0;
    if (++item == heads) {
      item = 0;
      if (++b < p.B) span = paged_span<L>(p, b);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace coalibi
