// Paged key/value cache: appending new tokens (with the position rotation on the
// way) and Co-ALiBi attention of one token or of a tree of drafted tokens over it.
#pragma once

#include <type_traits>

#include "sm100.cuh"
#include "decode.cuh"
#include "fwd.cuh"
#include "load_ring.h"

namespace coalibi {

constexpr int kStatusPage = 11;  // COALIBI_ERR_PAGE
constexpr int kTreeMaxSq = 64;   // COALIBI_TREE_MAX_SQ

__device__ __forceinline__ void report_page(int* status) {
  if (status != nullptr) atomicCAS(status, 0, kStatusPage);
}

// ---------------------------------------------------------------------------
// Append: key (a, b) of a rotated pair becomes (a cos - b sin, b cos + a sin), everything
// else is moved.  Bound by the bytes, each read and written once, for prompts (16,000 ragged
// tokens of 48 heads of 128: 264 MB in 46.6 us, 5.7 TB/s, 0.87 of the measured copy rate), and
// by latency (start -> page table -> store) for single tokens.  A CTA takes `group` consecutive
// tokens of the batch; its first threads look up where they go, then all threads move 16-byte
// pieces (8 elements).  A thread keeps its column, so it loads a token's angles once for all
// heads and needs no division per piece (with one the same prompts took 77 us); 32 registers
// leave 8 CTAs to an SM (at 4: 60 us).  A rotated piece also needs its partner's 8 elements
// (half layout) or none (interleaved); the partner is in the same row and hits L1.  The half
// layout's partners and second set of angles take 40 registers and leave 6: prompts whose whole
// heads turn so take 55 us (floor 41), the same without rotation, keys and values alone, 17.
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
  int Hq, Hkv, S;  // Hq 0: no queries
  long long tokens;  // B * S
  int group;         // tokens per CTA
  int page_size, max_pages, n_pages;
  int rot, n_pos, interleaved;
};

constexpr int kAppendThreads = 256;
constexpr int kAppendGroup = 2;  // most tokens of a CTA

enum { kTurnNone, kTurnHalves, kTurnPairs };

// A thread's angles of a token: 8 of them for 8 elements and their partners in the half layout
// (sn has the sign of the partner's share), 4 for 8 interleaved elements.
template <int TURN>
struct Angles {
  static constexpr int N = TURN == kTurnHalves ? 8 : 4;
  float cs[N], sn[N];
  __device__ __forceinline__ void load(const float* cos, const float* sin, int c, int half) {
    const int j = TURN == kTurnPairs ? c / 2 : (c < half ? c : c - half);
    const float sign = TURN == kTurnHalves && c < half ? -1.f : 1.f;
#pragma unroll
    for (int h = 0; h < N; h += 4) {
      const float4 a = *reinterpret_cast<const float4*>(cos + j + h), b = *reinterpret_cast<const float4*>(sin + j + h);
      cs[h] = a.x, cs[h + 1] = a.y, cs[h + 2] = a.z, cs[h + 3] = a.w;
      sn[h] = sign * b.x, sn[h + 1] = sign * b.y, sn[h + 2] = sign * b.z, sn[h + 3] = sign * b.w;
    }
  }
  template <bool BF16>
  __device__ __forceinline__ uint4 turn(uint4 own, uint4 other) const {
    uint32_t a[4] = {own.x, own.y, own.z, own.w};
    const uint32_t o[4] = {other.x, other.y, other.z, other.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<BF16>(a[i]);
      if (TURN == kTurnPairs) {
        a[i] = pack2<BF16>(f.x * cs[i] - f.y * sn[i], f.y * cs[i] + f.x * sn[i]);
      } else {
        const float2 h = unpack2<BF16>(o[i]);
        a[i] = pack2<BF16>(f.x * cs[2 * i % N] + h.x * sn[2 * i % N], f.y * cs[(2 * i + 1) % N] + h.y * sn[(2 * i + 1) % N]);
      }
    }
    return make_uint4(a[0], a[1], a[2], a[3]);
  }
};

template <bool BF16, int D, int TURN>
__global__ void __launch_bounds__(kAppendThreads, TURN == kTurnHalves ? 6 : 8) coalibi_paged_append_kernel(const AppendParams p) {
  struct Token {
    long long slot_k, slot_v;
    int b, i, angle;  // angle: row of the tables, or -1
    bool fresh, stored;
  };
  __shared__ Token s_tok[kAppendGroup];
  constexpr int PIECES = D / 8;
  const long long first = (long long)blockIdx.x * p.group;
  const int n = (int)min((long long)p.group, p.tokens - first);
  grid_dep_wait();
  if (threadIdx.x < n) {
    Token t;
    t.b = (int)((first + threadIdx.x) / p.S);
    t.i = (int)(first + threadIdx.x - (long long)t.b * p.S);
    const int start = p.start[t.b];
    const long long tok = (long long)start + t.i;
    t.fresh = t.i < (p.count != nullptr ? p.count[t.b] : p.S);
    t.stored = false;
    t.slot_k = t.slot_v = 0;
    t.angle = -1;
    if (t.fresh) {
      int page = -1;
      const int at = (int)(tok / p.page_size), slot = (int)(tok - (long long)at * p.page_size);
      if (start >= 0 && tok < (long long)p.max_pages * p.page_size)
        page = p.page_table[(size_t)t.b * p.table_stride + at];
      t.stored = page >= 0 && page < p.n_pages;
      t.slot_k = page * p.kps[0] + slot * p.kps[2];
      t.slot_v = page * p.vps[0] + slot * p.vps[2];
      if (p.rot > 0) {
        const long long pos = p.positions != nullptr ? p.positions[(size_t)t.b * p.S + t.i] : tok;
        if (pos >= 0 && pos < p.n_pos) t.angle = (int)pos;
      }
      if (!t.stored || (p.rot > 0 && t.angle < 0)) report_page(p.status);
    }
    s_tok[threadIdx.x] = t;
  }
  __syncthreads();
  constexpr int STEP = kAppendThreads / PIECES;  // heads that a pass of the threads covers
  const int r0 = threadIdx.x / PIECES, c = (threadIdx.x % PIECES) * 8, half = p.rot / 2;
  const int partner = c < half ? half : -half;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int k = 0; k < n; ++k) {
    const Token& t = s_tok[k];
    const bool turn = TURN != kTurnNone && c < p.rot && t.angle >= 0;
    Angles<TURN> g;
    if (turn) g.load(p.cos + (size_t)t.angle * half, p.sin + (size_t)t.angle * half, c, half);
    if (t.stored) {  // keys, then values
      for (int row = r0; row < 2 * p.Hkv; row += STEP) {
        const bool key = row < p.Hkv;
        const int h = key ? row : row - p.Hkv;
        const uint16_t* x = (key ? static_cast<const uint16_t*>(p.k) + t.b * p.ks[0] + t.i * p.ks[2] + h * p.ks[1]
                                 : static_cast<const uint16_t*>(p.v) + t.b * p.vs[0] + t.i * p.vs[2] + h * p.vs[1]) + c;
        uint16_t* y = (key ? static_cast<uint16_t*>(p.k_pages) + t.slot_k + h * p.kps[1]
                           : static_cast<uint16_t*>(p.v_pages) + t.slot_v + h * p.vps[1]) + c;
        uint4 val = *reinterpret_cast<const uint4*>(x);
        if (turn && key)
          val = g.template turn<BF16>(val, TURN == kTurnHalves ? *reinterpret_cast<const uint4*>(x + partner) : zero);
        *reinterpret_cast<uint4*>(y) = val;
      }
    }
    if (p.Hq > 0) {
      const uint16_t* x = static_cast<const uint16_t*>(p.q) + t.b * p.qs[0] + t.i * p.qs[2] + r0 * p.qs[1] + c;
      uint16_t* y = static_cast<uint16_t*>(p.q_out) + t.b * p.qos[0] + t.i * p.qos[2] + r0 * p.qos[1] + c;
      const long long dx = STEP * p.qs[1], dy = STEP * p.qos[1];
      if (t.fresh) {
#pragma unroll 2
        for (int row = r0; row < p.Hq; row += STEP, x += dx, y += dy) {
          uint4 val = *reinterpret_cast<const uint4*>(x);
          if (turn)
            val = g.template turn<BF16>(val, TURN == kTurnHalves ? *reinterpret_cast<const uint4*>(x + partner) : zero);
          *reinterpret_cast<uint4*>(y) = val;
        }
      } else {
        for (int row = r0; row < p.Hq; row += STEP, y += dy) *reinterpret_cast<uint4*>(y) = zero;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Attention.  Per row i and key j, keys in cache order:
//   x_j = scale q.k_j,  s_j = 1 / (1 + e^-x_j),  z_j = sum of s over the seen keys >= j,
//   o = sum_j e^(x_j - slope z_j) v_j / sum_j e^(x_j - slope z_j).
// A piece [lo, hi) of the keys, walked right to left with z restarted at 0, gives
// (T, m, l, O): its sigmoid total, largest logit, weight sum and weighted V.  The keys
// right of it add the constant R (their total) to every z in it, that is -slope R to
// every logit, so pieces join exactly: m' = m - slope R, then the usual log-sum-exp merge.
//
// What must move is K and V, once per kv head: the G * Sq rows that share them go
// through the tensor cores together.  Up to 32 rows, 16 to a warp with warp-level MMAs (a
// 128-lane tcgen05 tile would be mostly empty); a CTA has WARPS warps, RW of them side by side
// over the rows and KG = WARPS / RW over the keys.  Each RW warps are a CTA of their own, whose
// starts and ends overlap the others' reads; four warps share an item where there is little
// work.  Bound by the reads: 4 requests of 65 to 131 thousand keys, 4 rows each, 1.61 GB, take
// 254 us, 0.97 of the measured copy rate (237 of them here, 10 the joining).
//
// The work is cut evenly, whatever the lengths: items (request, kv head, block of RW *
// 16 rows) are laid end to end in units of 32 * KG keys, and each of a grid of resident
// CTAs takes an equal run of units.  An item inside one run is finished there; the
// pieces of one that spans runs go to the workspace and a second kernel joins them.
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
  float* ws;
  long long qs[3], os[3], kps[3], vps[3];
  long long table_stride, mask_stride;
  int B, Hq, Hkv, Sq;
  int page_size, page_shift, max_pages, n_pages;  // page_shift: log2(page_size), or -1
  int slopes_dtype;
  int row_blocks;  // blocks of RW * 16 rows per kv head
  int n_ctas;      // of the attention kernel
  int whole;       // one item to a CTA, none split
  float sm_scale;
};

constexpr int kPagedStep = 32;  // keys per step of a warp

template <int D, int RW, int WARPS>
struct PagedLayout {
  static constexpr int THREADS = 32 * WARPS, KG = WARPS / RW;
  static constexpr int UNIT = kPagedStep * KG;
  // What starting and finishing an item costs, in units: lengths, queries and the first load's
  // latency before its keys, the results after them.  Ragged decoding of 16 requests of 0 .. 8191
  // keys with four warps: 81 us without, 60 / 62 / 65 / 69 us with 2 / 3 / 5 / 8 units of 128
  // keys; with one warp, beside others on its SM, 4 units of 32 do (8: 1% slower).
  static constexpr int COST = KG == 1 ? 4 : 256 / UNIT;
  // Up to this many keys an item is not worth splitting: the joining costs a launch.
  static constexpr int WHOLE = 512;
  static constexpr int ROWS = 16 * RW;
  static constexpr int TILE = kPagedStep * D * 2;  // K or V of one step: [D / 64][32 keys][128 bytes], swizzled
  // Ring of steps.  Six CTAs of one warp with one step in flight each read faster than four with
  // two: long contexts 254 / 280 us, a ragged decode batch 52 / 56 us.
  static constexpr int NBUF = KG == 1 ? 2 : 3;
  static constexpr int RING = NBUF * 2 * TILE;     // per key group
  static constexpr int BYTES = KG * RING + 1024;   // (the ring starts at a multiple of 1024)
  // resident per SM: by shared memory, and by 256 registers a thread
  static constexpr int FIT = 200 * 1024 / BYTES, CTAS = FIT < 256 / THREADS ? FIT : 256 / THREADS;
  static constexpr int RECORD = ROWS * (4 + D);    // floats of one piece: stats, then O
  // the joining of the key groups reuses the ring
  static_assert(16 * RW * D * 4 <= RING, "exchange fits the ring");
};

constexpr int kPagedMaxSms = 160;
constexpr uint64_t kPagedTimeoutNs = 2000000000ull;  // bound on every wait for a load

// Workspace: B + 2 ints (prefix of the requests' spans, units per run), then two records per CTA.
template <typename L>
inline size_t paged_ws_bytes(int B) {
  const size_t head = ((size_t)(B + 2) * 4 + 255) / 256 * 256;
  return head + (size_t)kPagedMaxSms * L::CTAS * 2 * L::RECORD * 4;
}
__host__ __device__ inline size_t paged_ws_head(int B) { return ((size_t)(B + 2) * 4 + 255) / 256 * 64; }  // in floats

__device__ __forceinline__ int paged_keys(const PagedAttnParams& p, int b) {
  const int room = p.max_pages * p.page_size;  // at most 2^31 - 256
  return min(min(max(p.ctx_lens[b], 0), room) + p.Sq, room);
}

// Units of an item of request b, with its overhead.
template <typename L>
__device__ __forceinline__ int paged_span(const PagedAttnParams& p, int b) {
  return (paged_keys(p, b) + L::UNIT - 1) / L::UNIT + L::COST;
}

// One thread per request range: exclusive prefix sums of the requests' spans.  Returns
// the total; s_pre[t] is the prefix at the first request of thread t's range.
template <typename L>
__device__ __forceinline__ int paged_prefix(const PagedAttnParams& p, int* s_pre, int* s_warp, int per, int* out) {
  constexpr int NT = L::THREADS < 128 ? L::THREADS : 128;  // (the others only meet at the barriers)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool takes = tid < NT;
  int sum = 0;
  if (takes)
    for (int b = tid * per; b < min(p.B, (tid + 1) * per); ++b) sum += paged_span<L>(p, b);
  int inc = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  if (takes && lane == 31) s_warp[warp] = inc;
  __syncthreads();
  int left = 0, total = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) left += s_warp[w];
    total += s_warp[w];
  }
  int at = left + inc - sum;
  if (takes) {
    s_pre[tid] = at;
    if (out != nullptr) {
      for (int b = tid * per; b < min(p.B, (tid + 1) * per); ++b) {
        out[b] = at;
        at += paged_span<L>(p, b);
      }
      if (tid == 0) out[p.B] = total;
    }
  }
  __syncthreads();
  return total;
}

// The request, item and unit of it (after its overhead's) that stand at `at`.  All threads.
template <typename L>
__device__ __forceinline__ void paged_find(const PagedAttnParams& p, const int* s_pre, int* s_find, int per, int heads,
                                           unsigned at, int& b, int& span, int& item, int& v0) {
  constexpr int NT = L::THREADS < 128 ? L::THREADS : 128;
  const int tid = threadIdx.x;
  if (tid < NT && (unsigned)s_pre[tid] * heads <= at && (tid == NT - 1 || (unsigned)s_pre[tid + 1] * heads > at))
    *s_find = tid;
  __syncthreads();
  b = *s_find * per;
  int pre = s_pre[*s_find];
  span = paged_span<L>(p, b);
  while ((unsigned)(pre + span) * heads <= at) {
    pre += span;
    ++b;
    span = paged_span<L>(p, b);
  }
  item = (int)((at - (unsigned)pre * heads) / (unsigned)span);
  v0 = (int)((at - (unsigned)pre * heads) - (unsigned)item * span);
}

// A 4-D tile load (column, slot, head, page) of the page pool.
__device__ __forceinline__ void tma_load_4d(uint32_t smem_dst, const void* tmap, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(smem_dst),
      "l"(tmap), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// Order of a step's 32 keys in the score fragments.  Lane t of a quad holds keys
// 8 t .. 8 t + 7, so a row's suffix sum is additions in a lane and one scan over the
// quad; key tile n of the MMA takes the pair (n + t) % 4 of them, which spreads the
// eight rows of a tile over all eight phases of the 128-byte swizzle (no bank conflicts).
// Key of row j (0 .. 7) of tile n:
__device__ __forceinline__ int paged_tile_key(int n, int j) {
  const int t = j >> 1;
  return 8 * t + 2 * ((n + t) & 3) + (j & 1);
}

template <int D, bool BF16, int RW, int XR, int WARPS>
__global__ void __launch_bounds__(32 * WARPS)
    coalibi_paged_attn_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                              const PagedAttnParams p) {
  using L = PagedLayout<D, RW, WARPS>;
  constexpr int KG = L::KG, KK = D / 16;
  constexpr int THREADS = 32 * RW;  // per key group
  extern __shared__ __align__(128) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t s_full[KG * L::NBUF];
  __shared__ int s_abort;
  __shared__ volatile int s_fail[KG];
  __shared__ int s_pre[128], s_warp[4], s_find;
  __shared__ float4 s_stat[KG > 1 ? KG * L::ROWS : 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gq = lane >> 2, tig = lane & 3;
  const int rwarp = warp % RW, kg = warp / RW;
  const bool issuer = rwarp == 0 && lane == 0;  // of the group's loads
  const int G = p.Hq / p.Hkv, rows = G * p.Sq;
  const int heads = p.Hkv * p.row_blocks;  // items per request
  uint8_t* ring = smem + kg * L::RING;
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
    constexpr int NT = L::THREADS < 128 ? L::THREADS : 128;
    const int per = (p.B + NT - 1) / NT;
    const unsigned total = (unsigned)paged_prefix<L>(p, s_pre, s_warp, per, blockIdx.x == 0 ? head : nullptr) * heads;
    const unsigned quota = (total + p.n_ctas - 1) / p.n_ctas;  // (the host bounds the total below 2^31)
    if (blockIdx.x == 0 && tid == 0) head[p.B + 1] = (int)quota;
    at = quota * blockIdx.x;
    stop = min(total, at + quota);
    if (at >= stop) return;
    paged_find<L>(p, s_pre, &s_find, per, heads, at, b, span, item, v0);
  }

  // shared-memory offsets (within a tile) of this lane's ldmatrix rows; the k-step and the
  // tile pair only flip bits of them: columns 32 * (kk % 4), pair 1 moves the key by 4
  const int mat = lane >> 3, row8 = lane & 7;
  const int key_k = paged_tile_key(mat >> 1, row8), key_v = paged_tile_key(mat & 1, row8);
  const uint32_t off_k = key_k * 128 + (((mat & 1) ^ (key_k & 7)) << 4);
  const uint32_t off_v = key_v * 128 + (((mat >> 1) ^ (key_v & 7)) << 4);
  constexpr uint32_t kPair = 4 * 128 | 4 << 4;
  LoadRing<L::NBUF> loads;
  bool ok = true;  // no wait has run out

  while (at < stop) {
    // units [u0, u1) of the item; none if the run ends within its overhead
    const int v1 = (int)min((unsigned)span, v0 + (stop - at));
    const int u0 = max(v0 - L::COST, 0), u1 = v1 - L::COST, units = span - L::COST;
    if (u1 <= 0) break;
    const int g = item / p.row_blocks, r0 = (item - g * p.row_blocks) * L::ROWS + rwarp * 16;
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

    // ---- this key group's keys: [lo, hi), lo a multiple of 16 (so a half step lies in one page)
    const int s_lo = u0 * L::UNIT, s_hi = min(min(u1 * L::UNIT, room), ctx + drafts);
    const int sub = ((s_hi - s_lo + KG - 1) / KG + 15) & ~15;
    const int lo = s_lo + kg * sub, hi = min(s_hi, lo + sub);
    const int nsteps = hi > lo ? (hi - lo + kPagedStep - 1) / kPagedStep : 0;

    const int* table = p.page_table + (size_t)b * p.table_stride;
    int page_id[2], page_slot[2];  // of the next step to be loaded, per half; id -1: nothing there
    uint32_t gone_q = 0;           // two bits per ring slot: halves that were not loaded
    auto lookup = [&](int st) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int key = lo + st * kPagedStep + 16 * hf;
        page_id[hf] = -1;
        page_slot[hf] = 0;
        if (st >= 0 && key < hi) {
          const int n = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
          page_id[hf] = table[n];
          page_slot[hf] = key - n * p.page_size;
          if ((unsigned)page_id[hf] >= (unsigned)p.n_pages) {
            page_id[hf] = -1;
            report_page(p.status);
          }
        }
      }
    };
    // the half steps are 16 keys of one page: a box of 64 columns x 16 slots each
    auto load = [&]() {
      const int slot = loads.fill;
      gone_q &= ~(3u << (2 * slot));
      gone_q |= ((page_id[0] < 0 ? 1u : 0u) | (page_id[1] < 0 ? 2u : 0u)) << (2 * slot);
      if (issuer) {
        const uint32_t dst = smem_u32(ring + slot * 2 * L::TILE);
        const int halves = (page_id[0] >= 0) + (page_id[1] >= 0);
        mbar_arrive_expect_tx(&full[slot], halves * L::TILE);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          if (page_id[hf] < 0) continue;
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            tma_load_4d(dst + c * 4096 + hf * 2048, &tk, &full[slot], 64 * c, page_slot[hf], g, page_id[hf]);
            tma_load_4d(dst + L::TILE + c * 4096 + hf * 2048, &tv, &full[slot], 64 * c, page_slot[hf], g, page_id[hf]);
          }
        }
      }
      loads.issue();
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
      if (nsteps - a >= 0) load();
      lookup(nsteps - a - 1);
    }

    // ---- the rows: visibility words, slopes, queries as A fragments
    unsigned long long word[XR];
    float slope2[XR];
    const uint16_t* qrow[XR];
    bool rok[XR];
#pragma unroll
    for (int x = 0; x < XR; ++x) {
      const int r = r0 + gq + 8 * x;
      rok[x] = r < rows;
      const int rr = rok[x] ? r : 0;
      const int h = g * G + rr / p.Sq, i = rr % p.Sq;
      word[x] = p.tree_mask != nullptr ? (unsigned long long)p.tree_mask[b * p.mask_stride + i] : (2ull << i) - 1;
      slope2[x] = load_slope(p.slopes, p.slopes_dtype, h) * kLog2e;
      qrow[x] = static_cast<const uint16_t*>(p.q) + b * p.qs[0] + h * p.qs[1] + i * p.qs[2];
    }
    uint32_t qa[KK][4];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          qa[kk][2 * hf + x] = x < XR && rok[x % XR]
                                   ? *reinterpret_cast<const uint32_t*>(qrow[x % XR] + 16 * kk + 8 * hf + 2 * tig)
                                   : 0u;

    float o[2 * KK][4];
#pragma unroll
    for (int dn = 0; dn < 2 * KK; ++dn) o[dn][0] = o[dn][1] = o[dn][2] = o[dn][3] = 0.f;
    float m_run[XR], l_part[XR], carry[XR];
#pragma unroll
    for (int x = 0; x < XR; ++x) m_run[x] = -INFINITY, l_part[x] = 0.f, carry[x] = 0.f;

    const float c_a = p.sm_scale * kLog2e;
    for (int st = nsteps - 1; st >= 0; --st) {
      if (ok && !mbar_wait(&full[loads.drain], loads.phase, guard)) s_fail[kg] = st + 1;
      group_sync();  // all are done with step st + 1, whose slot is loaded next
      // the same for the group's warps, which meet again in the masked steps: a wait of this step or
      // of one before it ran out (one that a faster warp already meets in the next step counts there)
      ok = s_fail[kg] <= st;
      if (!ok) continue;
      const int slot = loads.drain;
      loads.landed();
      if (st - (L::NBUF - 1) >= 0) load();
      lookup(st - L::NBUF);
      const int kb = lo + st * kPagedStep;
      const uint32_t kt = smem_u32(ring + slot * 2 * L::TILE), vt = kt + L::TILE;
      // ---- S = Q K^T
      float sc[4][4];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
        for (int np = 0; np < 2; ++np) {
          uint32_t b0, b1, b2, b3;
          ldsm_x4(kt + (off_k ^ (32 * (kk & 3)) ^ (np * kPair)) + (kk >> 2) * 4096, b0, b1, b2, b3);
          mma16816<BF16>(sc[2 * np], qa[kk], b0, b1);
          mma16816<BF16>(sc[2 * np + 1], qa[kk], b2, b3);
        }
      }
      // ---- which of this lane's 8 keys each row sees: bit 2 n + e for element e of tile n
      const uint32_t gone = gone_q >> (2 * slot) & 3;
      const bool all = kb + kPagedStep <= min(hi, ctx) && gone == 0;
      uint32_t vis[XR];
#pragma unroll
      for (int x = 0; x < XR; ++x) vis[x] = 0xffu;
      // ---- sigmoids, suffix sums, logits (in log2 units), online softmax.  The rows go
      // through each stage together (their chains overlap), pairs of keys as float2.
      auto softmax = [&](auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        float2 sg[XR][4];                 // sigmoids of a pair: x first key, y second
        float pr[XR][4], tot[XR], inc[XR];
#pragma unroll
        for (int x = 0; x < XR; ++x) {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            float2 v = __fmul2_rn(make_float2(sc[n][2 * x], sc[n][2 * x + 1]), make_float2(c_a, c_a));
            sc[n][2 * x] = v.x;
            sc[n][2 * x + 1] = v.y;
            v = __fadd2_rn(make_float2(ex2_approx(-v.x), ex2_approx(-v.y)), make_float2(1.f, 1.f));
            sg[x][n] = make_float2(rcp_approx(v.x), rcp_approx(v.y));
            if (MASKED) {
              sg[x][n].x = vis[x] >> (2 * n) & 1 ? sg[x][n].x : 0.f;
              sg[x][n].y = vis[x] >> (2 * n + 1) & 1 ? sg[x][n].y : 0.f;
            }
            pr[x][n] = sg[x][n].x + sg[x][n].y;
          }
          tot[x] = ((pr[x][0] + pr[x][1]) + (pr[x][2] + pr[x][3]));
          inc[x] = tot[x];
        }
#pragma unroll
        for (int d = 1; d <= 2; ++d) {
#pragma unroll
          for (int x = 0; x < XR; ++x) {
            const float y = __shfl_down_sync(0xffffffffu, inc[x], d);
            if (tig + d < 4) inc[x] += y;
          }
        }
        float mx[XR];
#pragma unroll
        for (int x = 0; x < XR; ++x) {
          // tiles n >= 4 - t hold the lane's first pairs: their suffix also takes in all the
          // others, whose own suffix stops at tile 3 - t
          const float r2 = pr[x][3], r1 = r2 + pr[x][2], r0 = r1 + pr[x][1];
          const float wrapped = tig == 0 ? 0.f : tig == 1 ? r2 : tig == 2 ? r1 : r0;
          const float b_last = carry[x] + ((inc[x] - tot[x]) - wrapped), b_first = b_last + tot[x];
          carry[x] += __shfl_sync(0xffffffffu, inc[x], lane & ~3);
          const float after[4] = {b_last + r0, (tig == 3 ? b_first : b_last) + r1,
                                  (tig >= 2 ? b_first : b_last) + r2, tig >= 1 ? b_first : b_last};
          float m4[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const float2 z = __fadd2_rn(make_float2(pr[x][n], sg[x][n].y), make_float2(after[n], after[n]));
            float2 v = __ffma2_rn(make_float2(-slope2[x], -slope2[x]), z,
                                  make_float2(sc[n][2 * x], sc[n][2 * x + 1]));
            if (MASKED) {
              v.x = vis[x] >> (2 * n) & 1 ? v.x : -INFINITY;
              v.y = vis[x] >> (2 * n + 1) & 1 ? v.y : -INFINITY;
            }
            sc[n][2 * x] = v.x;
            sc[n][2 * x + 1] = v.y;
            m4[n] = fmaxf(v.x, v.y);
          }
          mx[x] = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        }
#pragma unroll
        for (int d = 1; d <= 2; ++d) {
#pragma unroll
          for (int x = 0; x < XR; ++x) mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], d));
        }
        // the newest keys weigh most, so the maximum seldom moves after the first steps
        bool up = mx[0] > m_run[0];
        if (XR > 1) up |= mx[XR - 1] > m_run[XR - 1];
        if (__any_sync(0xffffffffu, up)) {
#pragma unroll
          for (int x = 0; x < XR; ++x) {
            const float m_new = fmaxf(m_run[x], mx[x]);
            const float fac = m_run[x] == -INFINITY ? 0.f : ex2_approx(m_run[x] - m_new);
            m_run[x] = m_new;
            l_part[x] *= fac;
#pragma unroll
            for (int dn = 0; dn < 2 * KK; ++dn) {
              o[dn][2 * x] *= fac;
              o[dn][2 * x + 1] *= fac;
            }
          }
        }
#pragma unroll
        for (int x = 0; x < XR; ++x) {
          const float m_use = m_run[x] == -INFINITY ? 0.f : m_run[x];
          float2 l2 = make_float2(0.f, 0.f);
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const float2 v =
                __fadd2_rn(make_float2(sc[n][2 * x], sc[n][2 * x + 1]), make_float2(-m_use, -m_use));
            const float2 w = make_float2(ex2_approx(v.x), ex2_approx(v.y));
            l2 = __fadd2_rn(l2, w);
            sc[n][2 * x] = w.x;
            sc[n][2 * x + 1] = w.y;
          }
          l_part[x] += l2.x + l2.y;
        }
      };
      if (!all) {
#pragma unroll 1
        for (int x = 0; x < XR; ++x) {
          uint32_t v = 0;
#pragma unroll 1
          for (int j = 0; j < 8; ++j) {
            const int key = kb + 8 * tig + 2 * (((j >> 1) + tig) & 3) + (j & 1);
            if (!(gone >> (tig >> 1) & 1) && key < hi && (key < ctx || ((x ? word[XR - 1] : word[0]) >> (key - ctx) & 1)))
              v |= 1u << j;
          }
          if (x)
            vis[XR - 1] = v;
          else
            vis[0] = v;
        }
      }
      // with one row to a lane a second copy for the steps without masks costs more in
      // instruction fetches than it saves (long contexts 281 us with, 269 without); with two
      // rows it pays (16 rows, 8 requests of 8192 keys 62 us with, 65 without)
      if (XR == 1 || !all)
        softmax(std::true_type{});
      else
        softmax(std::false_type{});
      // ---- V rows that no row sees (past the end, of no page, unseen drafts) may hold
      // anything: zero them, 0 * NaN is not 0.  A drafted token's V that is not finite must
      // not reach the rows that do not see it either: it is added by hand, then zeroed.
      if (!all) {
        const int key = kb + lane;
        uint8_t* vrow = ring + slot * 2 * L::TILE + L::TILE + lane * 128;
        const bool used = !(gone >> (lane >> 4) & 1) && key < hi && (key < ctx || (seen_by_any >> (key - ctx) & 1));
        bool bad = false;
        if (used && key >= ctx && p.Sq > 1) {
#pragma unroll 4
          for (int c = 0; c < D / 8; ++c) {
            const uint4 u = *reinterpret_cast<const uint4*>(vrow + (c >> 3) * 4096 + ((c & 7) << 4));
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = unpack2<BF16>(w[j]);
              bad |= !(fabsf(f.x) < INFINITY) || !(fabsf(f.y) < INFINITY);
            }
          }
        }
        for (uint32_t left = __ballot_sync(0xffffffffu, bad); left != 0; left &= left - 1) {
          const int off = __ffs(left) - 1, t = off >> 3;
          const int el = 2 * ((((off & 7) >> 1) - t) & 3) + (off & 1);  // 2 n + e in the lanes t
          const uint8_t* vb = ring + slot * 2 * L::TILE + L::TILE + off * 128;
#pragma unroll
          for (int x = 0; x < XR; ++x) {
            float w = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (el == j) w = sc[j >> 1][2 * x + (j & 1)];
            uint32_t see = vis[x] >> el & 1;
            w = __shfl_sync(0xffffffffu, w, (lane & ~3) | t);
            see = __shfl_sync(0xffffffffu, see, (lane & ~3) | t);
            if (see) {
#pragma unroll
              for (int dn = 0; dn < 2 * KK; ++dn) {
                const float2 f = unpack2<BF16>(*reinterpret_cast<const uint32_t*>(
                    vb + (dn >> 3) * 4096 + (((dn & 7) ^ (off & 7)) << 4) + 4 * tig));
                o[dn][2 * x] = fmaf(w, f.x, o[dn][2 * x]);
                o[dn][2 * x + 1] = fmaf(w, f.y, o[dn][2 * x + 1]);
              }
            }
          }
        }
        group_sync();
        if (rwarp == 0 && (!used || bad)) {
#pragma unroll
          for (int c = 0; c < D / 8; ++c)
            *reinterpret_cast<uint4*>(vrow + (c >> 3) * 4096 + ((c & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
          fence_async_smem();  // ordered before the load that refills the slot
        }
        group_sync();
      }
      // ---- O += P V: the C fragments of two key tiles are the A fragment of one k-step.
      // P is rounded to the inputs' type, which the MMA takes; l sums it unrounded (half an ulp of
      // each weight, averaging out over the keys).
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        uint32_t pa[4];
        pa[0] = pack2<BF16>(sc[2 * k2][0], sc[2 * k2][1]);
        pa[1] = XR > 1 ? pack2<BF16>(sc[2 * k2][2], sc[2 * k2][3]) : 0u;
        pa[2] = pack2<BF16>(sc[2 * k2 + 1][0], sc[2 * k2 + 1][1]);
        pa[3] = XR > 1 ? pack2<BF16>(sc[2 * k2 + 1][2], sc[2 * k2 + 1][3]) : 0u;
#pragma unroll
        for (int dp = 0; dp < KK; ++dp) {
          uint32_t b0, b1, b2, b3;
          ldsm_x4_t(vt + (off_v ^ (32 * (dp & 3)) ^ (k2 * kPair)) + (dp >> 2) * 4096, b0, b1, b2, b3);
          mma16816<BF16>(o[2 * dp], pa, b0, b1);
          mma16816<BF16>(o[2 * dp + 1], pa, b2, b3);
        }
      }
    }
    if (!ok && issuer)  // a wait ran out: the loads already issued land before the CTA leaves, below
      for (; loads.in_flight(); loads.landed()) mbar_drain(&full[loads.drain], loads.phase, kPagedTimeoutNs);
#pragma unroll
    for (int x = 0; x < XR; ++x) {
      l_part[x] += __shfl_xor_sync(0xffffffffu, l_part[x], 1);
      l_part[x] += __shfl_xor_sync(0xffffffffu, l_part[x], 2);
    }

    // ---- the piece's result: the output if the item is whole, else a record
    const bool whole = u0 == 0 && u1 == units;
    float* rec = p.ws + paged_ws_head(p.B) + ((size_t)blockIdx.x * 2 + (u0 > 0 ? 0 : 1)) * L::RECORD;
    float4* stats = reinterpret_cast<float4*>(rec);
    float* orec = rec + 4 * L::ROWS;
    if (KG == 1) {
#pragma unroll
      for (int x = 0; x < XR; ++x) {
        const int r = rwarp * 16 + gq + 8 * x, rr = r0 + gq + 8 * x;
        if (!rok[x]) continue;
        if (whole) {
          uint16_t* y = static_cast<uint16_t*>(p.o) + b * p.os[0] + (g * G + rr / p.Sq) * p.os[1] + (rr % p.Sq) * p.os[2];
          const float inv = l_part[x] > 0.f ? 1.f / l_part[x] : (l_part[x] == 0.f ? 0.f : l_part[x]);
#pragma unroll
          for (int dn = 0; dn < 2 * KK; ++dn)
            *reinterpret_cast<uint32_t*>(y + 8 * dn + 2 * tig) = pack2<BF16>(o[dn][2 * x] * inv, o[dn][2 * x + 1] * inv);
        } else {
          if (tig == 0) stats[r] = make_float4(carry[x], m_run[x], l_part[x], 0.f);
#pragma unroll
          for (int dn = 0; dn < 2 * KK; ++dn)
            *reinterpret_cast<float2*>(orec + r * D + 8 * dn + 2 * tig) = make_float2(o[dn][2 * x], o[dn][2 * x + 1]);
        }
      }
    } else {
      // key groups join through shared memory (the rings are idle now)
      float* xo = reinterpret_cast<float*>(smem);  // [KG][ROWS][D]
      __syncthreads();
#pragma unroll
      for (int x = 0; x < XR; ++x) {
        const int r = rwarp * 16 + gq + 8 * x;
        if (tig == 0) s_stat[kg * L::ROWS + r] = make_float4(carry[x], m_run[x], l_part[x], slope2[x]);
#pragma unroll
        for (int dn = 0; dn < 2 * KK; ++dn)
          *reinterpret_cast<float2*>(xo + ((size_t)kg * L::ROWS + r) * D + 8 * dn + 2 * tig) =
              make_float2(o[dn][2 * x], o[dn][2 * x + 1]);
      }
      __syncthreads();
      const int rb = (item - g * p.row_blocks) * L::ROWS;
      const int n = min(XR == 1 ? 8 : L::ROWS, rows - rb);
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
          const float f = ex2_approx(w[c] - m_use);
          l = fmaf(s_stat[c * L::ROWS + r].z, f, l);
          const float4 v = *reinterpret_cast<const float4*>(xo + ((size_t)c * L::ROWS + r) * D + d);
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

// ---------------------------------------------------------------------------
// More than 32 rows per kv head (trees): tcgen05.  64 or 128 rows as the 128 lanes of TMEM,
// one row to a thread, so a row's scan over its keys is additions in a register file and
// needs no shuffles, fragments or ldmatrix (per score about a third of the instructions of
// the warp-level kernel above, which stays for fewer rows: there a 128-lane tile would be
// mostly empty).  Two groups of four softmax warps work on their own keys, each with a
// warp that issues its MMAs and one that issues its loads; per step of a group
//   S [128 x 64 keys] = Q K^T into one of two TMEM buffers, P = softmax weights written over
//   it as 16-bit, O [128 x D] += P V.
// With at most 64 rows (DUP) the rows stand twice in the tile: lanes 0 .. 63 take the first 32
// keys of a step, lanes 64 .. 127 the other 32, with zeros in P for each other's, so all four
// warps of a group are busy; those 32 keys come from two separate pieces of the item, and no
// step needs an exchange between threads.  Pieces join at the item's end as above.  Bound by
// the reads in long items (8 requests of 8192 keys, 64 rows, 268 MB: 63 us, 4.3 TB/s; each
// further 1000 keys per SM cost 13 us, 5.8 TB/s) and by an item's start and end, about 10 us.
// More rows share the reads but not the exponentials: 8 requests of 127 to 16383 keys, 8 kv heads,
// take 76 us with 64 rows, 104 with 128 and 184 with 256 (two blocks of rows, each reading all keys).
//
// P is 16-bit, as the MMA takes it, while l sums the weights unrounded: an error of half an ulp of
// each weight that averages out over the keys, at half the bytes of TMEM and of the instruction's
// operands.  Where the reference moves between the halves of a step, the right half's weights, rounded
// already, are scaled and rounded again (only when a logit passes it by 8 in log2 units, and the other way is to hold
// 32 floats more); the drafts that are added by hand take the weight as rounded, like the others of their row.
// ---------------------------------------------------------------------------
template <int D, bool DUP>
struct WideLayout {
  static constexpr int PIECES = DUP ? 4 : 2;       // of an item, per CTA
  static constexpr int STEP = DUP ? 32 : 64;       // keys of a piece per step
  static constexpr int UNIT = 128;
  // As above: trees of 16 drafts over 127 .. 16383 keys took 132 us with 3 units, 79 with 7, 70 with
  // 9 to 11, 71 with 14, in one run on one GPU (an item's queries, first loads, exchange and joining take
  // about 10 us; 75 to 76 is usual).
  static constexpr int COST = 10;
  static constexpr int WHOLE = 1024;  // 32 requests of 500 / 1000 keys, 8 kv heads: 43 / 52 us, split 50 / 59
  static constexpr int ROWS = DUP ? 64 : 128;
  static constexpr int TILE = 64 * D * 2;          // K or V of a group's step: [D / 64][64 keys][128 bytes]
  static constexpr int BOX = 64 * 128;
  static constexpr int NBUF = 3;
  static constexpr int RING = NBUF * 2 * TILE;     // per group
  static constexpr int QBYTES = 128 * D * 2;       // [D / 64][128 rows][128 bytes]
  static constexpr int BYTES = QBYTES + 2 * RING + 1024;
  static constexpr int CTAS = 1;
  static constexpr int RECORD = ROWS * (4 + D);
  static constexpr int TM_S = 64, TM_O = 256;      // columns of an S buffer; O of group w at TM_O + w * D
  static constexpr int THREADS = 384;
  // a group's part of the exchange (O in float, then statistics) reuses its ring
  static_assert(128 * D * 4 + 128 * 16 <= RING, "exchange fits the ring");
};

template <int D, bool BF16, bool DUP>
__global__ void __launch_bounds__(384, 1)
    coalibi_paged_wide_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                              const PagedAttnParams p) {
  using L = WideLayout<D, DUP>;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t s_full[2][L::NBUF], s_empty[2][L::NBUF], s_scores[2][2], s_probs[2][2], s_pv[2], s_idle[2];
  // four bits: 16-key quarters of the step that were not loaded; 16: some key of it is not of the context
  __shared__ int s_gone[2][L::NBUF];
  __shared__ int s_pre[128], s_warp[4], s_find, s_abort;
  __shared__ uint32_t s_tmem;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool softmax = warp < 8, issues = warp == 8 || warp == 9;
  const int w = softmax ? warp >> 2 : warp & 1;  // group
  const int G = p.Hq / p.Hkv, rows = G * p.Sq;
  const int heads = p.Hkv * p.row_blocks;
  const CtaGuard guard{&s_abort, p.status, kPagedTimeoutNs};
  if (tid == 0) {
    for (int g = 0; g < 2; ++g) {
      for (int i = 0; i < L::NBUF; ++i) {
        mbar_init(&s_full[g][i], 1);
        mbar_init(&s_empty[g][i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_scores[g][i], 1);
        mbar_init(&s_probs[g][i], 4);
      }
      mbar_init(&s_pv[g], 1);
      mbar_init(&s_idle[g], 1);
    }
    s_abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  if (warp == 8) {
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
    constexpr int NT = L::THREADS < 128 ? L::THREADS : 128;
    const int per = (p.B + NT - 1) / NT;
    const unsigned total = (unsigned)paged_prefix<L>(p, s_pre, s_warp, per, blockIdx.x == 0 ? head : nullptr) * heads;
    const unsigned quota = (total + p.n_ctas - 1) / p.n_ctas;
    if (blockIdx.x == 0 && tid == 0) head[p.B + 1] = (int)quota;
    at = quota * blockIdx.x;
    stop = min(total, at + quota);
    if (at < stop) paged_find<L>(p, s_pre, &s_find, per, heads, at, b, span, item, v0);
  }

  uint8_t* ring = smem + L::QBYTES + w * L::RING;
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
    const int nsteps = DUP ? max(piece_steps(q0), piece_steps(q0 + 1)) : piece_steps(q0);
    // first key of half hf of step n (counted from the right); its piece's end
    auto half_base = [&](int n, int hf) {
      if (DUP) return piece_lo(q0 + hf) + (piece_steps(q0 + hf) - 1 - n) * 32;
      return piece_lo(q0) + (nsteps - 1 - n) * 64 + 32 * hf;
    };
    auto half_hi = [&](int hf) { return piece_hi(DUP ? q0 + hf : q0); };
    auto half_lo = [&](int hf) { return piece_lo(DUP ? q0 + hf : q0); };

    // whether some row sees key `lane` of half hf of step n; whether it is a drafted one of those
    auto used = [&](int n, int hf, int gone) {
      const int base = half_base(n, hf), key = base + lane;
      return base >= half_lo(hf) && !(gone >> (2 * hf + (lane >> 4)) & 1) && key < half_hi(hf) &&
             (key < ctx || (seen_by_any >> (key - ctx) & 1));
    };
    auto drafted = [&](int n, int hf, int gone) { return used(n, hf, gone) && half_base(n, hf) + lane >= ctx; };
    auto not_finite = [&](const uint8_t* vrow) {  // a row of V in shared memory
      bool bad = false;
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        const uint4 u = *reinterpret_cast<const uint4*>(vrow + (c >> 3) * L::BOX + ((c & 7) << 4));
        const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = unpack2<BF16>(x[j]);
          bad |= !(fabsf(f.x) < INFINITY) || !(fabsf(f.y) < INFINITY);
        }
      }
      return bad;
    };
    auto is_plain = [&](int n, int gone) {  // all 64 keys loaded and of the context
      bool plain = gone == 0;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) plain = plain && half_base(n, hf) + 32 <= min(half_hi(hf), ctx);
      return plain;
    };
    int loaded = 0;
    auto load = [&](int n) {  // step n of the group (one lane of its loading warp)
      const uint32_t k = seq + n;
      const int slot = k % L::NBUF;
      const int* table = p.page_table + (size_t)b * p.table_stride;
      int page[4], at_slot[4], gone = 0, bytes = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = half_base(n, i >> 1) + 16 * (i & 1);
        page[i] = -1;
        at_slot[i] = 0;
        if (key >= half_lo(i >> 1) && key < half_hi(i >> 1)) {
          const int t = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
          page[i] = table[t];
          at_slot[i] = key - t * p.page_size;
          if ((unsigned)page[i] >= (unsigned)p.n_pages) {
            page[i] = -1;
            report_page(p.status);
          }
        }
        if (page[i] < 0)
          gone |= 1 << i;
        else
          bytes += 16 * D * 2 * 2;
      }
      if (!mbar_wait(&s_empty[w][slot], ((k / L::NBUF) & 1) ^ 1, guard)) return false;
      s_gone[w][slot] = is_plain(n, gone) ? 0 : gone | 16;
      mbar_arrive_expect_tx(&s_full[w][slot], bytes);
      const uint32_t dst = smem_u32(ring + slot * 2 * L::TILE);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (page[i] < 0) continue;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          tma_load_4d(dst + c * L::BOX + i * 2048, &tk, &s_full[w][slot], 64 * c, at_slot[i], g, page[i]);
          tma_load_4d(dst + L::TILE + c * L::BOX + i * 2048, &tv, &s_full[w][slot], 64 * c, at_slot[i], g, page[i]);
        }
      }
      ++loaded;
      return true;
    };
    const int ahead = min(nsteps, L::NBUF);  // the rings are free: these start beside the queries
    if (warp >= 10) {
      if (lane == 0)
        for (int n = 0; n < ahead && ok; ++n) ok = load(n);
      __syncwarp();
    }
    if (softmax) {
      // ---- the queries, in the K-major 128-byte-swizzled form the MMA reads
      for (int c = tid; c < 128 * (D / 8); c += 256) {
        const int r = c / (D / 8), ch = c % (D / 8), row = rb + (DUP ? r & 63 : r);
        uint4 val = make_uint4(0u, 0u, 0u, 0u);
        if (row < rows)
          val = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + b * p.qs[0] +
                                                (g * G + row / p.Sq) * p.qs[1] + (row % p.Sq) * p.qs[2] + ch * 8);
        *reinterpret_cast<uint4*>(smem + (ch >> 3) * (128 * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = val;
      }
      // O starts at zero
      const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16);
      uint32_t zero[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) zero[j] = 0u;
#pragma unroll
      for (int c = 0; c < D; c += 32) tmem_st32(mine + L::TM_O + w * D + c, zero);
      tmem_st_wait();
      fence_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();

    if (warp >= 10) {
      // ---------------------------------------------------------- loads
      if (lane == 0) {
        for (int n = ahead; n < nsteps && ok; ++n) ok = load(n);
        const int n_issued = loaded;
        // every issued copy lands before the item (and the CTA) ends
        for (int n = max(n_issued - L::NBUF, 0); n < n_issued; ++n)
          mbar_drain(&s_full[w][(seq + n) % L::NBUF], ((seq + n) / L::NBUF) & 1, guard.timeout_ns);
      }
      __syncwarp();
    } else if (issues) {
      // ---------------------------------------------------------- MMAs (lane 0 issues)
      constexpr uint32_t idS = make_idesc_f16(BF16, 128, 64, false, false);
      constexpr uint32_t idPV = make_idesc_f16(BF16, 128, D, false, true);
      const uint32_t q_addr = smem_u32(smem), ring_addr = smem_u32(ring);
      auto issue_scores = [&](int n) {
        const uint32_t k = seq + n;
        const int slot = k % L::NBUF;
        if (!__all_sync(0xffffffffu, mbar_wait(&s_full[w][slot], (k / L::NBUF) & 1, guard))) return false;
        if (lane == 0) {
          tc_fence_after();
          const uint32_t d = tmem + (2 * w + (k & 1)) * L::TM_S, k_addr = ring_addr + slot * 2 * L::TILE;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_ss(d, make_sdesc_sw128(q_addr + (kk >> 2) * (128 * 128) + (kk & 3) * 32, 16, 1024),
                    make_sdesc_sw128(k_addr + (kk >> 2) * L::BOX + (kk & 3) * 32, 16, 1024), idS, kk > 0 ? 1u : 0u);
          umma_commit(&s_scores[w][k & 1]);
        }
        __syncwarp();
        return true;
      };
      // S(0), S(1), PV(0), S(2), PV(1), ...: S(n + 2) overwrites the buffer that PV(n), issued
      // before it by this thread, has read P from
      for (int n = 0; n < 2 && n < nsteps && ok; ++n) ok = issue_scores(n);
      for (int n = 0; n < nsteps && ok; ++n) {
        const uint32_t k = seq + n;
        const int slot = k % L::NBUF;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&s_probs[w][k & 1], (k >> 1) & 1, guard)))) break;
        const int gone = s_gone[w][slot];
        if (gone != 0) {
          // V rows that no row sees (past the end, of no page, unseen drafts) may hold anything: zero
          // them, 0 * NaN is not 0; the drafts that the softmax warps have added by hand too
#pragma unroll 1
          for (int hf = 0; hf < 2; ++hf) {
            uint8_t* vrow = ring + slot * 2 * L::TILE + L::TILE + (32 * hf + lane) * 128;
            const bool mine = used(n, hf, gone);
            if (!mine || (p.Sq > 1 && half_base(n, hf) + lane >= ctx && not_finite(vrow))) {
#pragma unroll
              for (int c = 0; c < D / 8; ++c)
                *reinterpret_cast<uint4*>(vrow + (c >> 3) * L::BOX + ((c & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          fence_async_smem();
          __syncwarp();
        }
        if (lane == 0) {
          tc_fence_after();
          const uint32_t pa = tmem + (2 * w + (k & 1)) * L::TM_S, v_addr = ring_addr + slot * 2 * L::TILE + L::TILE;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_ts(tmem + L::TM_O + w * D, pa + kk * 8, make_sdesc_sw128(v_addr + kk * 16 * 128, L::BOX, 1024), idPV, 1u);
          umma_commit(&s_pv[w]);
          umma_commit(&s_empty[w][slot]);
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
      // ---------------------------------------------------------- softmax: one row to a thread
      const int t = (warp & 3) * 32 + lane, r = DUP ? t & 63 : t, my_half = t >> 6;
      const bool rok = rb + r < rows;
      const float slope2 = load_slope(p.slopes, p.slopes_dtype, g * G + (rok ? rb + r : rb) / p.Sq) * kLog2e, c_a = p.sm_scale * kLog2e;
      const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
      const uint32_t o_base = lane_base + L::TM_O + w * D;
      float m = -INFINITY, l = 0.f, carry = 0.f;
      bool left = false;
      for (int n = 0; n < nsteps; ++n) {
        const uint32_t k = seq + n;
        const int slot = k % L::NBUF;
        const uint32_t s_base = lane_base + (2 * w + (k & 1)) * L::TM_S;
        if (ok) ok = mbar_wait(&s_full[w][slot], (k / L::NBUF) & 1, guard);
        if (ok) ok = mbar_wait(&s_scores[w][k & 1], (k >> 1) & 1, guard);
        ok = __all_sync(0xffffffffu, ok);
        const int gone = s_gone[w][slot];
        const bool plain = gone == 0;
        uint32_t pk[DUP ? 1 : 2][16];
        float alpha = 1.f;
        bool rescale = false;
        uint32_t vis[2] = {0xffffffffu, 0xffffffffu};
        if (!plain) {
          const int row_of = (rok ? rb + r : rb) % p.Sq;
          const unsigned long long word =
              p.tree_mask != nullptr ? (unsigned long long)p.tree_mask[b * p.mask_stride + row_of] : (2ull << row_of) - 1;
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const int base = half_base(n, hf), in = min(half_hi(hf), ctx) - base, end = half_hi(hf) - base;
            uint32_t v = in >= 32 ? 0xffffffffu : in > 0 ? (1u << in) - 1u : 0u;  // of the context
            if (end > in && end > 0) {  // drafted tokens, up to `end`
              const int d = base - ctx;
              const uint32_t bits = d >= 0 ? (d < 64 ? (uint32_t)(word >> d) : 0u) : d > -32 ? (uint32_t)word << -d : 0u;
              const uint32_t upto = end >= 32 ? 0xffffffffu : (1u << end) - 1u;
              v |= bits & upto & ~(in > 0 ? (in >= 32 ? 0xffffffffu : (1u << in) - 1u) : 0u);
            }
            if (base < half_lo(hf)) v = 0u;  // this piece has ended
            if (gone >> (2 * hf) & 1) v &= 0xffff0000u;
            if (gone >> (2 * hf + 1) & 1) v &= 0x0000ffffu;
            vis[hf] = v;
          }
        }
        if (ok) {
          tc_fence_after();
#pragma unroll
          for (int x = 0; x < (DUP ? 1 : 2); ++x) {  // (the right half first)
            const int hf = DUP ? my_half : 1 - x;
            uint32_t s[32];
            tmem_ld32_sync(s_base + 32 * hf, s);
            const uint32_t seen = hf ? vis[1] : vis[0];
            auto scan = [&](auto masked) {
              constexpr bool MASKED = decltype(masked)::value;
              // sub-chunks of 8 keys: short chains of additions that overlap
              float tot[4];
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                float run = 0.f;
#pragma unroll
                for (int j = 7; j >= 0; j -= 2) {
                  const int e = 8 * c + j - 1;  // the pair (e, e + 1)
                  const float2 y = __fmul2_rn(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])),
                                              make_float2(c_a, c_a));
                  const float2 dn = __fadd2_rn(make_float2(ex2_approx(-y.x), ex2_approx(-y.y)), make_float2(1.f, 1.f));
                  float2 sg = make_float2(rcp_approx(dn.x), rcp_approx(dn.y));
                  if (MASKED) {
                    sg.x = seen >> e & 1 ? sg.x : 0.f;
                    sg.y = seen >> (e + 1) & 1 ? sg.y : 0.f;
                  }
                  const float z1 = run + sg.y, z0 = z1 + sg.x;
                  run = z0;
                  const float2 v = __ffma2_rn(make_float2(-slope2, -slope2), make_float2(z0, z1), y);
                  s[e] = __float_as_uint(v.x);
                  s[e + 1] = __float_as_uint(v.y);
                }
                tot[c] = run;
              }
              // sums right of each sub-chunk shift its logits
              float off[4];
              off[3] = carry;
              off[2] = off[3] + tot[3];
              off[1] = off[2] + tot[2];
              off[0] = off[1] + tot[1];
              carry = off[0] + tot[0];
              float mx = -INFINITY;
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const float sh = -slope2 * off[c];
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                  const int e = 8 * c + j;
                  float2 v = __fadd2_rn(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), make_float2(sh, sh));
                  if (MASKED) {
                    v.x = seen >> e & 1 ? v.x : -INFINITY;
                    v.y = seen >> (e + 1) & 1 ? v.y : -INFINITY;
                  }
                  s[e] = __float_as_uint(v.x);
                  s[e + 1] = __float_as_uint(v.y);
                  mx = fmaxf(mx, fmaxf(v.x, v.y));
                }
              }
              return mx;
            };
            const float mx = plain ? scan(std::false_type{}) : scan(std::true_type{});
            // the reference moves only when a logit passes it by 2^8: weights stay below 256, and
            // O needs rescaling rarely
            if (mx > m + 8.f || (m == -INFINITY && mx > -INFINITY)) {
              const float f = m == -INFINITY ? 0.f : ex2_approx(m - mx);
              if (m != -INFINITY) {
                rescale = true;
                alpha *= f;
                if (!DUP && x == 1) {  // the right half's weights of this step move too
                  const float2 f2 = make_float2(f, f);
#pragma unroll
                  for (int j = 0; j < 16; ++j) {
                    const float2 u = __fmul2_rn(unpack2<BF16>(pk[0][j]), f2);
                    pk[0][j] = pack2<BF16>(u.x, u.y);
                  }
                }
              }
              l *= f;
              m = mx;
            }
            const float m_use = m == -INFINITY ? 0.f : m;
            float2 ls = make_float2(0.f, 0.f);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float2 v = __fadd2_rn(make_float2(__uint_as_float(s[2 * j]), __uint_as_float(s[2 * j + 1])),
                                          make_float2(-m_use, -m_use));
              const float2 e = make_float2(ex2_approx(v.x), ex2_approx(v.y));
              ls = __fadd2_rn(ls, e);
              pk[DUP ? 0 : x][j] = pack2<BF16>(e.x, e.y);
            }
            l += ls.x + ls.y;
          }
          if (__any_sync(0xffffffffu, rescale)) {
            // every PV before this step's must have added its part
            if (k > 0) ok = mbar_wait(&s_pv[w], (k - 1) & 1, guard);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
              tc_fence_after();
#pragma unroll
              for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                tmem_ld32_sync(o_base + c, o);
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                tmem_st32(o_base + c, o);
              }
            }
          }
        }
        // ---- P over this step's scores
        if (!ok) {
          left = true;
          break;
        }
        if (DUP) {
          const uint32_t none[16] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
          tmem_st16(s_base + 16 * my_half, pk[0]);
          tmem_st16(s_base + 16 * (1 - my_half), none);
        } else {
          tmem_st16(s_base + 16, pk[0]);
          tmem_st16(s_base, pk[DUP ? 0 : 1]);
        }
        tmem_st_wait();
        if (!plain && p.Sq > 1) {
          // ---- a drafted token's V that is not finite must not reach the rows that do not see it
          // through 0 * V: it is added by hand, and the issuing warp zeroes it
#pragma unroll 1
          for (int hf = 0; hf < 2; ++hf) {
            const uint8_t* vt = ring + slot * 2 * L::TILE + L::TILE + 32 * hf * 128;
            const bool bad = drafted(n, hf, gone) && not_finite(vt + lane * 128);
            const uint32_t bads = __ballot_sync(0xffffffffu, bad);
            if (bads != 0 && (!DUP || hf == my_half)) {
              if (k > 0) ok = mbar_wait(&s_pv[w], (k - 1) & 1, guard);
              ok = __all_sync(0xffffffffu, ok);
              if (!ok) break;
              tc_fence_after();
              for (uint32_t rest = bads; rest != 0; rest &= rest - 1) {
                const int j = __ffs(rest) - 1;
                const float2 w2 = unpack2<BF16>(__float_as_uint(tmem_ld1_sync(s_base + 16 * hf + (j >> 1))));
                const float wj = j & 1 ? w2.y : w2.x;
                const bool see = (hf ? vis[1] : vis[0]) >> j & 1;
                const uint8_t* vj = vt + j * 128;
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                  uint32_t o[16];
                  tmem_ld16_sync(o_base + c, o);
#pragma unroll
                  for (int q = 0; q < 8; ++q) {
                    const int ch = (c + 2 * q) >> 3;
                    const float2 f = unpack2<BF16>(*reinterpret_cast<const uint32_t*>(
                        vj + (ch >> 3) * L::BOX + (((ch & 7) ^ (j & 7)) << 4) + ((2 * q) & 7) * 2));
                    if (see) {
                      o[2 * q] = __float_as_uint(fmaf(wj, f.x, __uint_as_float(o[2 * q])));
                      o[2 * q + 1] = __float_as_uint(fmaf(wj, f.y, __uint_as_float(o[2 * q + 1])));
                    }
                  }
                  tmem_st16(o_base + c, o);
                  tmem_st_wait();
                }
              }
            }
          }
        }
        if (!ok) {
          left = true;
          break;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_probs[w][k & 1]);
      }
      // ---- this group's pieces to the exchange: O, swizzled by row, and the statistics
      // (the last scores imply every PV but the last two: a wait on the last one's parity alone would
      // pass while the one before it is under way)
      if (!left && nsteps > 1) ok = mbar_wait(&s_pv[w], (seq + nsteps - 2) & 1, guard);
      if (ok && !left && nsteps > 0) ok = mbar_wait(&s_pv[w], (seq + nsteps - 1) & 1, guard);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after();
        float* xo = reinterpret_cast<float*>(ring);
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_ld32_sync(o_base + c, o);
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const int ch = (c + j) >> 2;
            *reinterpret_cast<uint4*>(xo + t * D + ((ch ^ (t & (D / 4 - 1))) << 2)) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
          }
        }
        reinterpret_cast<float4*>(xo + 128 * D)[t] = make_float4(carry, m, l, slope2);
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
        const int lane_row = DUP ? r + 64 * (q & 1) : r, grp = DUP ? q >> 1 : q;
        const float* xo = reinterpret_cast<const float*>(smem + L::QBYTES + grp * L::RING);
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
        const int lane_row = DUP ? r + 64 * (q & 1) : r, grp = DUP ? q >> 1 : q;
        const float* xo = reinterpret_cast<const float*>(smem + L::QBYTES + grp * L::RING);
        const float f = ex2_approx(wt[q] - m_use);
        l = fmaf(reinterpret_cast<const float4*>(xo + 128 * D)[lane_row].z, f, l);
        const float4 v = *reinterpret_cast<const float4*>(xo + lane_row * D + ((ch ^ (lane_row & (D / 4 - 1))) << 2));
        acc.x = fmaf(v.x, f, acc.x);
        acc.y = fmaf(v.y, f, acc.y);
        acc.z = fmaf(v.z, f, acc.z);
        acc.w = fmaf(v.w, f, acc.w);
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
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the pieces of the items that span runs.  One warp per query row; lanes hold the
// statistics of up to 32 pieces at a time, rightmost first.
template <int D, bool BF16, typename L>
__global__ void __launch_bounds__(128) coalibi_paged_join_kernel(const PagedAttnParams p) {
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31;
  const int G = p.Hq / p.Hkv, rows = G * p.Sq;
  const int r = blockIdx.y * 4 + (threadIdx.x >> 5);
  const int b = blockIdx.x / p.Hkv, g = blockIdx.x - b * p.Hkv;
  grid_dep_wait();
  if (r >= rows) return;
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
  constexpr int EARLY = 8;  // pieces whose O is on its way beside the statistics (4: 1% slower)
  for (int top = c1; top >= c0; top -= 32) {
    const int n = min(32, top - c0 + 1);
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
    if (lane < n) s = reinterpret_cast<const float4*>(record(top - lane))[rr];
    float early[EARLY][V];
#pragma unroll
    for (int j = 0; j < EARLY; ++j) {
#pragma unroll
      for (int v = 0; v < V; ++v) early[j][v] = 0.f;
      if (j < n) o_of(j, early[j]);
    }
    float inc = s.x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const float y = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += y;
    }
    float m = s.y == -INFINITY ? -INFINITY : s.y - slope2 * (right + (inc - s.x));
    right += __shfl_sync(0xffffffffu, inc, 31);
    float mx = m;
#pragma unroll
    for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    const float m_new = fmaxf(M, mx), m_use = m_new == -INFINITY ? 0.f : m_new;
    const float fac = M == -INFINITY ? 0.f : ex2_approx(M - m_use);
    M = m_new;
    const float f = ex2_approx(m - m_use);
    float lw = f * s.z;
#pragma unroll
    for (int d = 16; d; d >>= 1) lw += __shfl_xor_sync(0xffffffffu, lw, d);
    l = l * fac + lw;
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] *= fac;
#pragma unroll
    for (int j = 0; j < EARLY; ++j) {
      const float w = __shfl_sync(0xffffffffu, f, j);  // 0 past the last piece
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = fmaf(w, early[j][v], acc[v]);
    }
#pragma unroll 4
    for (int j = EARLY; j < n; ++j) {
      const float w = __shfl_sync(0xffffffffu, f, j);
      float u[V];
      o_of(j, u);
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = fmaf(w, u[v], acc[v]);
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  uint16_t* y = static_cast<uint16_t*>(p.o) + b * p.os[0] + h * p.os[1] + i * p.os[2] + lane * V;
#pragma unroll
  for (int v = 0; v < V; v += 2) *reinterpret_cast<uint32_t*>(y + v) = pack2<BF16>(acc[v] * inv, acc[v + 1] * inv);
}

}  // namespace coalibi
