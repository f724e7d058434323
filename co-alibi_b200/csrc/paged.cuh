// Paged key/value cache: appending new tokens (with the position rotation on the
// way) and Co-ALiBi attention of one token or of a tree of drafted tokens over it.
#pragma once

#include <type_traits>

#include "sm100.cuh"
#include "decode.cuh"
#include "fwd.cuh"

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
// (half layout) or none (interleaved); the partner is in the same row and hits L1.
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
// through the tensor cores together, 16 to a warp.  A CTA has four warps: RW of them
// side by side over the rows and KG = 4 / RW over the keys.  Up to 64 rows the kernel
// is bound by the reads; the warp-level MMA is enough for that, and its fragments can be
// scanned in registers.
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
  float sm_scale;
};

constexpr int kPagedStep = 32;  // keys per step of a warp

template <int D, int RW>
struct PagedLayout {
  static constexpr int KG = 4 / RW;
  static constexpr int UNIT = kPagedStep * KG;
  // What starting and finishing an item costs, in units (256 keys' worth): lengths,
  // queries and the first load's latency before its keys, the results after them.  Ragged
  // decoding of 16 requests of 0 .. 8191 keys: 81 us without, 60 / 62 / 65 / 69 us with 2 / 3
  // / 5 / 8 units of 128 keys; trees of 16 over 127 .. 16383: 166 us, with 2 / 3 / 5 / 8 units
  // of 32 keys 135 / 123 / 121 / 120 us.
  static constexpr int COST = 256 / UNIT;
  static constexpr int ROWS = 16 * RW;
  static constexpr int TILE = kPagedStep * D * 2;  // K or V of one step: [D / 64][32 keys][128 bytes], swizzled
  static constexpr int NBUF = RW == 4 ? 4 : 3;     // all but one of the steps in flight
  static constexpr int RING = NBUF * 2 * TILE;     // per key group
  static constexpr int BYTES = KG * RING + 1024;   // (the ring starts at a multiple of 1024)
  static constexpr int CTAS = D == 128 ? (RW == 1 ? 1 : 2) : RW == 1 ? 2 : RW == 2 ? 3 : 4;  // resident per SM
  static constexpr int RECORD = ROWS * (4 + D);    // floats of one piece: stats, then O
  // the joining of the key groups reuses the ring
  static_assert(KG * 16 * RW * D * 4 <= KG * RING || KG == 1, "exchange fits the ring");
};

constexpr int kPagedMaxSms = 160;
constexpr uint64_t kPagedTimeoutNs = 2000000000ull;  // bound on every wait for a load

// Workspace: B + 2 ints (prefix of the requests' spans, units per run), then two records per CTA.
template <int D, int RW>
inline size_t paged_ws_bytes(int B) {
  using L = PagedLayout<D, RW>;
  const size_t head = ((size_t)(B + 2) * 4 + 255) / 256 * 256;
  return head + (size_t)kPagedMaxSms * L::CTAS * 2 * L::RECORD * 4;
}
__host__ __device__ inline size_t paged_ws_head(int B) { return ((size_t)(B + 2) * 4 + 255) / 256 * 64; }  // in floats

// Row warps for `rows` query rows per kv head.
inline int paged_row_warps(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

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
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int sum = 0;
  for (int b = tid * per; b < min(p.B, (tid + 1) * per); ++b) sum += paged_span<L>(p, b);
  int inc = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  int left = 0, total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < warp) left += s_warp[w];
    total += s_warp[w];
  }
  int at = left + inc - sum;
  s_pre[tid] = at;
  if (out != nullptr) {
    for (int b = tid * per; b < min(p.B, (tid + 1) * per); ++b) {
      out[b] = at;
      at += paged_span<L>(p, b);
    }
    if (tid == 0) out[p.B] = total;
  }
  __syncthreads();
  return total;
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

template <int D, bool BF16, int RW, int XR>
__global__ void __launch_bounds__(128)
    coalibi_paged_attn_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                              const PagedAttnParams p) {
  using L = PagedLayout<D, RW>;
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
  grid_dep_wait();

  // ---- this CTA's run of units
  int* head = reinterpret_cast<int*>(p.ws);
  const int per = (p.B + 127) / 128;
  const long long total = (long long)paged_prefix<L>(p, s_pre, s_warp, per, blockIdx.x == 0 ? head : nullptr) * heads;
  const long long quota = (total + p.n_ctas - 1) / p.n_ctas;
  if (blockIdx.x == 0 && tid == 0) head[p.B + 1] = (int)quota;
  long long at = quota * blockIdx.x;
  const long long stop = min(total, at + quota);
  if (at >= stop) return;
  // the request that holds unit `at`
  if ((long long)s_pre[tid] * heads <= at && (tid == 127 || (long long)s_pre[tid + 1] * heads > at)) s_find = tid;
  __syncthreads();
  int b = s_find * per, pre = s_pre[s_find];
  int span = paged_span<L>(p, b);
  while ((long long)(pre + span) * heads <= at) {
    pre += span;
    ++b;
    span = paged_span<L>(p, b);
  }
  int item = (int)((at - (long long)pre * heads) / span);
  int v0 = (int)((at - (long long)pre * heads) - (long long)item * span);

  // shared-memory offsets (within a tile) of this lane's ldmatrix rows; the k-step and the
  // tile pair only flip bits of them: columns 32 * (kk % 4), pair 1 moves the key by 4
  const int mat = lane >> 3, row8 = lane & 7;
  const int key_k = paged_tile_key(mat >> 1, row8), key_v = paged_tile_key(mat & 1, row8);
  const uint32_t off_k = key_k * 128 + (((mat & 1) ^ (key_k & 7)) << 4);
  const uint32_t off_v = key_v * 128 + (((mat >> 1) ^ (key_v & 7)) << 4);
  constexpr uint32_t kPair = 4 * 128 | 4 << 4;
  int fill = 0, drain = 0;            // ring slots of the next load and of the next step
  uint32_t fill_n = 0, drain_n = 0;   // loads issued, steps awaited
  uint32_t phase = 0;                 // parity of the next step's barrier
  bool ok = true;                     // no wait has run out

  while (at < stop) {
    // units [u0, u1) of the item; none if the run ends within its overhead
    const int v1 = (int)min((long long)span, v0 + (stop - at));
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
      gone_q &= ~(3u << (2 * fill));
      gone_q |= ((page_id[0] < 0 ? 1u : 0u) | (page_id[1] < 0 ? 2u : 0u)) << (2 * fill);
      if (issuer) {
        const uint32_t dst = smem_u32(ring + fill * 2 * L::TILE);
        const int halves = (page_id[0] >= 0) + (page_id[1] >= 0);
        mbar_arrive_expect_tx(&full[fill], halves * L::TILE);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          if (page_id[hf] < 0) continue;
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            tma_load_4d(dst + c * 4096 + hf * 2048, &tk, &full[fill], 64 * c, page_slot[hf], g, page_id[hf]);
            tma_load_4d(dst + L::TILE + c * 4096 + hf * 2048, &tv, &full[fill], 64 * c, page_slot[hf], g, page_id[hf]);
          }
        }
      }
      fill = fill + 1 == L::NBUF ? 0 : fill + 1;
      ++fill_n;
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
      if (ok && !mbar_wait(&full[drain], phase, guard)) s_fail[kg] = 1;
      group_sync();  // all are done with step st + 1, whose slot is loaded next
      ok = s_fail[kg] == 0;  // the same for the group's warps, which meet again in the masked steps
      const int slot = drain;
      drain = drain + 1 == L::NBUF ? 0 : drain + 1;
      if (drain == 0) phase ^= 1;
      ++drain_n;
      if (!ok) continue;
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
      if (all) {
        softmax(std::false_type{});
      } else {
#pragma unroll
        for (int x = 0; x < XR; ++x) {
          uint32_t v = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int key = kb + 8 * tig + 2 * (((j >> 1) + tig) & 3) + (j & 1);
            if (!(gone >> (tig >> 1) & 1) && key < hi && (key < ctx || (word[x] >> (key - ctx) & 1))) v |= 1u << j;
          }
          vis[x] = v;
        }
        softmax(std::true_type{});
      }
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
      // P is rounded to the inputs' type for the product; l sums it unrounded.
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
    if (!ok && issuer) {  // a wait ran out: let the loads already issued land before leaving
      for (; drain_n < fill_n; ++drain_n) {
        mbar_drain(&full[drain], phase, kPagedTimeoutNs);
        drain = drain + 1 == L::NBUF ? 0 : drain + 1;
        if (drain == 0) phase ^= 1;
      }
    }
    if (!ok) drain_n = fill_n;
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
        const int r = rwarp * 16 + gq + 8 * x;
        if (!rok[x]) continue;
        if (whole) {
          const int rr = r0 + gq + 8 * x;
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
      for (int e = tid; e < n * (D / 4); e += 128) {
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

// Joins the pieces of the items that span runs.  One warp per query row; lanes hold the
// statistics of up to 32 pieces at a time, rightmost first.
template <int D, bool BF16, int RW>
__global__ void __launch_bounds__(128) coalibi_paged_join_kernel(const PagedAttnParams p) {
  using L = PagedLayout<D, RW>;
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
  for (int top = c1; top >= c0; top -= 32) {
    const int n = min(32, top - c0 + 1);
    float4 s = make_float4(0.f, -INFINITY, 0.f, 0.f);
    if (lane < n) s = reinterpret_cast<const float4*>(record(top - lane))[rr];
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
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const float w = __shfl_sync(0xffffffffu, f, j);
      const float* y = record(top - j) + 4 * L::ROWS + rr * D + lane * V;
      if (V == 4) {
        const float4 u = *reinterpret_cast<const float4*>(y);
        acc[0] = fmaf(w, u.x, acc[0]);
        acc[1] = fmaf(w, u.y, acc[1]);
        acc[V - 2] = fmaf(w, u.z, acc[V - 2]);
        acc[V - 1] = fmaf(w, u.w, acc[V - 1]);
      } else {
        const float2 u = *reinterpret_cast<const float2*>(y);
        acc[0] = fmaf(w, u.x, acc[0]);
        acc[1] = fmaf(w, u.y, acc[1]);
      }
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  uint16_t* y = static_cast<uint16_t*>(p.o) + b * p.os[0] + h * p.os[1] + i * p.os[2] + lane * V;
#pragma unroll
  for (int v = 0; v < V; v += 2) *reinterpret_cast<uint32_t*>(y + v) = pack2<BF16>(acc[v] * inv, acc[v + 1] * inv);
}

}  // namespace coalibi
