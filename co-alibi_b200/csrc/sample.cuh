// Drawing tokens from logits: temperature, top-k, top-p, min-p and a race of given
// exponential random numbers.
//
// With the tokens ranked by (logit descending, index ascending) every filter keeps a
// prefix of the ranking, so a row needs one threshold, and no sort of the vocabulary.
// What must move is the logits, once (and the random numbers of the kept tokens); the
// rest is latency.  A cluster of CTAs takes a row, each CTA a slice that it holds in
// shared memory, so that the passes after the first read no memory:
//
//   maximum    of the slice, then of the row;
//   top-k      (k <= kSampleMaxK) each CTA lists what can be among its k largest: what is not
//              below the k-th largest of its threads' maxima, or the bins of a histogram
//              down to rank k; the first CTA sorts the few hundred listed and works on those;
//   top-p      2048 bins of the weight's logarithm collect the weights; tokens above the bin
//              in which their sum crosses top_p race at once, its own are compared one by one;
//   the race   largest w / noise.
//
// Histograms use 32-bit shared-memory atomics alone: they run at the rate of plain
// stores, 64-bit and float ones are loops of compare-and-swap (48 adds of 1024 threads:
// 11 thousand cycles against 41 to 340 thousand).  Weights are 2^-31 fixed point in two
// 16-bit halves there, so sums are exact integers and the order of atomics is irrelevant.
// Measured, us a call: one row of 50304 with top-k 50 9.8; 64 rows of 50304, each with its own
// parameters, 22.7 (floor of the reads 2); 300 rows of 32001 with top-p 60 (floor 3: per row 7 us
// are the bins' atomics, 5 the random numbers' latency, and 300 rows are four more than run at
// once); 256 rows of 131072 without filters 55 (floor 41, the streaming kernel below); 64 rows of
// 50304 with top-p 25, with min-p alone 10, greedy 14.
//
// Rows that the bins do not separate (masses of equal logits, infinite ones, k above
// kSampleMaxK, slices over 65536 tokens) take a radix descent in one CTA, up to eight passes over
// the row in global memory for each filter: one row of 50304 with k = 1025 takes 165 us, 64 such
// rows 245 (k = 12576: 255), 64 of 131072 560 (k = 32768: 710), and 64 rows of 50304 whose tokens but
// 20 are masked by the type's lowest value, k = 50, 468: the masked ones share the last bin.
#pragma once

#include <cooperative_groups.h>

#include "fwd.cuh"
#include "sm100.cuh"

namespace coalibi {

struct SampleParams {
  const void* logits;
  const float* noise;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  long long* tokens;
  float* logprobs;
  long long logits_stride, noise_stride;
  int B, V;
  float temperature_all;
  int top_k_all;
  float top_p_all, min_p_all;
  int cluster;       // CTAs per row
  int slice_chunks;  // 16-byte chunks per CTA; 0: the slices stay in global memory
  int filters;       // whether any row may ask for top-k or top-p
};

constexpr int kSampleThreads = 512;
constexpr int kSampleMaxCluster = 8;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 2048;
constexpr int kSampleMaxK = 1024;
constexpr int kSampleListed = 2048;       // tokens a CTA may list
constexpr int kSampleQuickK = 384;        // of 512 threads: the bound by their maxima stays tight
constexpr int kSampleTies = 1024;         // tokens of the crossing bin that are compared one by one
constexpr int kSampleMaxSlice = 65536;    // 16-bit halves of the weights then sum within 32 bits
constexpr float kSampleBinsPerLogit = 64.f;
constexpr float kSampleBinsPerLog2 = 44.f;  // 2048 bins reach down to 2^-46, below half of 2^-31

template <int DT>
__device__ __forceinline__ float load_logit(const void* base, long long i) {
  if (DT == 2) return static_cast<const float*>(base)[i];
  if (DT == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
  return __half2float(static_cast<const __half*>(base)[i]);
}

// NaN counts as -inf.
__device__ __forceinline__ float clean_logit(float x) { return fmaxf(x, -INFINITY); }

// The same for a 32-bit word of logits, and the larger of two clean words' elements.
template <int DT>
__device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b) {
  if (DT == 2) return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  uint32_t r;
  if (DT == 1)
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <int DT>
__device__ __forceinline__ uint32_t clean_word(uint32_t a) {  // (max takes the operand that is a number)
  return max_word<DT>(a, DT == 2 ? 0xff800000u : DT == 1 ? 0xff80ff80u : 0xfc00fc00u);
}

// Integer of the same order as a clean logit (-0 as +0), and back.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// Rank of a token: larger is earlier.
__device__ __forceinline__ unsigned long long rank_key(float x, int i) {
  return ((unsigned long long)order_key(x) << 32) | (uint32_t)~i;
}

struct SampleShared {
  unsigned int* hist;  // [2][kSampleBins], dynamic shared memory
  unsigned int warp_u[kSampleWarps];
  unsigned long long warp_ull[kSampleWarps];
  float warp_f[kSampleWarps];
  double warp_d[kSampleWarps];
  int warp_i[kSampleWarps];
  // results that all threads, or the other CTAs of the cluster, read
  unsigned long long best_key;  // of this CTA's slice
  unsigned long long floor_key, target, base;
  unsigned int found_bin, found_count, n_list;
  unsigned int bound;  // bits of the best score so far
  int first, overflow;
  // in the first CTA, an entry from each
  unsigned int sent[kSampleMaxCluster];  // listed tokens; ~0: more than fit, or +inf among them
  float score[kSampleMaxCluster];
  int token[kSampleMaxCluster];
  double rest[kSampleMaxCluster];
};

__device__ __forceinline__ unsigned long long block_max(unsigned long long v, SampleShared& s) {
  // the high words' maximum, then the low words' among the threads that hold it
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto warp_max = [](unsigned long long x) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(x >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(x >> 32) == hi ? (uint32_t)x : 0u);
    return ((unsigned long long)hi << 32) | lo;
  };
  v = warp_max(v);
  if (lane == 0) s.warp_ull[warp] = v;
  __syncthreads();
  v = warp_max(lane < kSampleWarps ? s.warp_ull[lane] : 0ull);
  __syncthreads();
  return v;
}

__device__ __forceinline__ uint32_t block_max(uint32_t v, SampleShared& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = __reduce_max_sync(0xffffffffu, v);
  if (lane == 0) s.warp_u[warp] = v;
  __syncthreads();
  v = __reduce_max_sync(0xffffffffu, lane < kSampleWarps ? s.warp_u[lane] : 0u);
  __syncthreads();
  return v;
}

template <typename T>
__device__ __forceinline__ T block_exclusive(T v, T* warp_sums, T& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T inc = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  T left = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSampleWarps; ++w) {
    const T y = warp_sums[w];
    if (w < warp) left += y;
    total += y;
  }
  __syncthreads();
  return left + inc - v;
}

// 1 / T, held to normal numbers: 0 * infinity would be NaN, for the largest logit at the smallest
// temperatures and for masked ones at an infinite one.
__device__ __forceinline__ float inverse_temperature(float t) { return fminf(fmaxf(1.f / t, 0x1p-126f), 0x1p126f); }

// Weights and distances of a row.
struct SampleScale {
  float mx, inv_t, k2;
  __device__ __forceinline__ float dist(float x) const { return x == mx ? 0.f : (x - mx) * inv_t; }
  // of a finite maximum only; the passes over a slice use it with an approximate 2^x, whose error
  // of about 2^-22 a weight goes into the log-probability's sum
  __device__ __forceinline__ float log2w(float x) const { return (x - mx) * k2; }
  __device__ __forceinline__ unsigned fixed(float l2) const { return __float2uint_rn(ex2_approx(l2 + 31.f)); }
};

// The winner of the block's race and the weights beside the first token's, in thread 0.
__device__ __forceinline__ void block_race(float& score, int& token, double& rest, SampleShared& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float ys = __shfl_xor_sync(0xffffffffu, score, o);
    const int yi = __shfl_xor_sync(0xffffffffu, token, o);
    if (ys > score || (ys == score && yi < token)) score = ys, token = yi;
    rest += __shfl_xor_sync(0xffffffffu, rest, o);
  }
  if (lane == 0) s.warp_f[warp] = score, s.warp_i[warp] = token, s.warp_d[warp] = rest;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kSampleWarps; ++w) {
      if (s.warp_f[w] > score || (s.warp_f[w] == score && s.warp_i[w] < token)) score = s.warp_f[w], token = s.warp_i[w];
      rest += s.warp_d[w];
    }
  }
}

// The radix descent, by one CTA over the whole row: 8 bits of the rank key per level, a
// histogram of the counts or of the weights (three parts of 11 bits: 2^21 of them fit 32
// bits) of the keys that share the prefix, and the bin in which the target is reached.
template <int DT>
__device__ void sample_general(const SampleParams& p, SampleShared& s, int b, const void* lrow, const float* nrow,
                               const SampleScale& sc, int first, int top_k, float top_p, float min_p) {
  const int tid = threadIdx.x;
  auto weight = [&](float x) { return expf(sc.dist(x)); };
  auto fixed = [&](float x) { return (unsigned)__float2uint_rn(weight(x) * 2147483648.f); };
  unsigned long long floor_key = ((unsigned long long)(order_key(-INFINITY) + 1)) << 32;
  unsigned int* h = s.hist;  // [4][256]: counts, then the parts of the weights
  for (int filter = 0; filter < 2; ++filter) {
    const bool by_mass = filter == 1;
    if (by_mass ? top_p >= 1.f : (top_k <= 0 || top_k >= p.V)) continue;
    unsigned long long target = top_k;
    if (by_mass) {
      unsigned long long sum = 0, total;
      for (int i = tid; i < p.V; i += kSampleThreads) {
        const float x = clean_logit(load_logit<DT>(lrow, i));
        if (rank_key(x, i) >= floor_key) sum += fixed(x);
      }
      block_exclusive(sum, s.warp_ull, total);
      target = (unsigned long long)fmax(1.0, ceil((double)fmaxf(top_p, 0.f) * (double)total));
    }
    unsigned long long prefix = 0, acc = 0;
    int done = 0;
    for (int shift = 56; shift >= 0 && done == 0; shift -= 8) {
      for (int i = tid; i < 1024; i += kSampleThreads) h[i] = 0;
      __syncthreads();
      for (int i = tid; i < p.V; i += kSampleThreads) {
        const float x = clean_logit(load_logit<DT>(lrow, i));
        const unsigned long long ck = rank_key(x, i);
        if (ck < floor_key || (shift < 56 && (ck >> (shift + 8)) != (prefix >> (shift + 8)))) continue;
        const int bin = (int)(ck >> shift) & 255;
        atomicAdd(&h[bin], 1u);
        if (by_mass) {
          const unsigned w = fixed(x);
          atomicAdd(&h[256 + bin], w & 2047u);
          atomicAdd(&h[512 + bin], w >> 11 & 2047u);
          atomicAdd(&h[768 + bin], w >> 22);
        }
      }
      __syncthreads();
      if (tid == 0) {
        int bin = 255, last = -1;
        for (; bin >= 0; --bin) {
          if (h[bin] == 0) continue;
          last = bin;
          const unsigned long long v =
              by_mass ? h[256 + bin] + ((unsigned long long)h[512 + bin] << 11) + ((unsigned long long)h[768 + bin] << 22)
                      : h[bin];
          if (acc + v >= target) break;
          acc += v;
        }
        s.overflow = 0;
        if (bin < 0) s.overflow = 2, bin = last;  // fewer than the target: all stay
        s.base = acc;
        s.floor_key = prefix | ((unsigned long long)bin << shift);
        if (s.overflow == 0 && (h[bin] == 1 || (!by_mass && acc + h[bin] == target))) s.overflow = 1;
      }
      __syncthreads();
      done = s.overflow;
      acc = s.base;
      prefix = s.floor_key;
      __syncthreads();
    }
    if (done != 2 && prefix > floor_key) floor_key = prefix;
  }
  float score = -1.f;
  int token = first;
  double rest = 0.0;
  for (int i = tid; i < p.V; i += kSampleThreads) {
    const float x = clean_logit(load_logit<DT>(lrow, i));
    const float w = weight(x);
    if (i != first) {
      if (rank_key(x, i) < floor_key || w < min_p || w == 0.f) continue;
      rest += (double)w;
    }
    const float y = w / nrow[i];
    if (y > score || (y == score && i < token)) score = y, token = i;
  }
  block_race(score, token, rest, s);
  if (tid == 0) {
    p.tokens[b] = token;
    p.logprobs[b] = sc.dist(clean_logit(load_logit<DT>(lrow, token))) - log1pf((float)rest);
  }
}

// Top-k, in the first CTA: the n listed tokens of the cluster (rank keys, key_at(i)) sorted
// as far as rank k, then the other filters and the race on the sorted list.  `binned` and
// `sorted` are scratch; done_reading() follows the last key_at.  Returns false if the bins
// do not separate the tokens.
template <typename KeyAt, typename Done>
__device__ bool sample_topk(const SampleParams& p, SampleShared& s, int b, const float* nrow, SampleScale sc, int n,
                            KeyAt&& key_at, Done&& done_reading, unsigned long long* binned,
                            unsigned long long* sorted, int k, float top_p, float min_p) {
  const int tid = threadIdx.x;
  unsigned int* hist = s.hist;
  unsigned int* off = s.hist + kSampleBins;
  constexpr int PER = kSampleBins / kSampleThreads;
  unsigned long long best = 0;
  for (int i = tid; i < kSampleBins; i += kSampleThreads) hist[i] = 0;
  for (int i = tid; i < n; i += kSampleThreads) {
    const unsigned long long key = key_at(i);
    best = key > best ? key : best;
  }
  if (tid == 0) s.found_count = 0;
  best = block_max(best, s);
  if (best == 0) {  // nothing but -inf
    done_reading();
    if (tid == 0) p.tokens[b] = -1, p.logprobs[b] = -INFINITY;
    return true;
  }
  sc.mx = key_logit((uint32_t)(best >> 32));
  auto bin_of = [&](unsigned long long key) {
    return min(kSampleBins - 1, __float2int_rz((sc.mx - key_logit((uint32_t)(key >> 32))) * kSampleBinsPerLogit));
  };
  for (int i = tid; i < n; i += kSampleThreads) atomicAdd(&hist[bin_of(key_at(i))], 1u);
  __syncthreads();
  unsigned v[PER], sum = 0, total;
#pragma unroll
  for (int j = 0; j < PER; ++j) v[j] = hist[tid * PER + j], sum += v[j];
  unsigned at = block_exclusive(sum, s.warp_u, total);
  const int kk = min(k, (int)total);
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    off[tid * PER + j] = at;
    hist[tid * PER + j] = at;  // where the bin's next key goes
    at += v[j];
    if (v[j] > 0 && (int)(at - v[j]) < kk && (int)at >= kk) s.found_count = at;  // keys of the bins down to rank kk - 1
  }
  __syncthreads();
  const int m = s.found_count;
  if (m > 2 * kSampleMaxK) {
    done_reading();
    return false;
  }
  for (int i = tid; i < n; i += kSampleThreads) {
    const unsigned long long key = key_at(i);
    const int bin = bin_of(key);
    if ((int)off[bin] < kk) binned[atomicAdd(&hist[bin], 1u)] = key;
  }
  done_reading();  // (a barrier)
  for (int i = tid; i < m; i += kSampleThreads) {
    const unsigned long long key = binned[i];
    const int bin = bin_of(key), from = off[bin], to = hist[bin];
    int place = from;
    for (int j = from; j < to; ++j) place += binned[j] > key;
    if (place < kk) sorted[place] = key;
  }
  __syncthreads();
  // ranks 2 tid and 2 tid + 1
  float w[2] = {0.f, 0.f};
  int index[2] = {0, 0};
  unsigned long long f[2] = {0, 0}, mass;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = 2 * tid + j;
    if (r < kk) {
      w[j] = expf(sc.dist(key_logit((uint32_t)(sorted[r] >> 32))));
      index[j] = (int)~(uint32_t)sorted[r];
      f[j] = __float2uint_rn(w[j] * 2147483648.f);
    }
  }
  const unsigned long long before = block_exclusive(f[0] + f[1], s.warp_ull, mass);
  const unsigned long long target =
      top_p >= 1.f ? ~0ull : (unsigned long long)fmax(1.0, ceil((double)fmaxf(top_p, 0.f) * (double)mass));
  float score = -1.f;
  int token = 2 * tid < kk ? index[0] : 0x7fffffff;
  double rest = 0.0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = 2 * tid + j;
    if (r >= kk || before + (j ? f[0] : 0) >= target) continue;
    if (r > 0) {
      if (w[j] < min_p || w[j] == 0.f) continue;
      rest += (double)w[j];
    }
    const float y = w[j] / nrow[index[j]];
    if (y > score || (y == score && index[j] < token)) score = y, token = index[j];
  }
  block_race(score, token, rest, s);
  if (tid == 0) {
    if (score < 0.f) token = (int)~(uint32_t)best;  // no number won: the first of the ranking
    s.token[0] = token;
    s.rest[0] = rest;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = 2 * tid + j;
    if (r < kk && index[j] == s.token[0]) {
      p.tokens[b] = index[j];
      p.logprobs[b] = sc.dist(key_logit((uint32_t)(sorted[r] >> 32))) - log1pf((float)s.rest[0]);
    }
  }
  return true;
}

template <int DT>
__global__ void __launch_bounds__(kSampleThreads, 2) coalibi_sample_kernel(const SampleParams p) {
  namespace cg = cooperative_groups;
  constexpr int SIZE = DT == 2 ? 4 : 2, EPC = 16 / SIZE;  // elements per 16-byte chunk
  constexpr int PER = kSampleBins / kSampleThreads;
  __shared__ SampleShared s;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  // histograms, listed tokens (or the row's bin masses), the slice; without filters the
  // first are 4 KB for the descent and there is no list
  unsigned int* hist = reinterpret_cast<unsigned int*>(smem_raw);
  unsigned long long* list = reinterpret_cast<unsigned long long*>(smem_raw + 8 * kSampleBins);
  uint4* data = reinterpret_cast<uint4*>(smem_raw + (p.filters ? 8 * kSampleBins + 8 * kSampleListed : 4096));
  cg::cluster_group cluster = cg::this_cluster();
  const int C = p.cluster, rank = C > 1 ? (int)cluster.block_rank() : 0, b = blockIdx.x / C;
  const int tid = threadIdx.x;
  SampleShared& s0 = C > 1 ? *cluster.map_shared_rank(&s, 0) : s;  // the first CTA's
  unsigned long long* list0 = C > 1 ? cluster.map_shared_rank(list, 0) : list;
  auto meet = [&]() {
    if (C > 1)
      cluster.sync();
    else
      __syncthreads();
  };
  const char* lrow = static_cast<const char*>(p.logits) + (size_t)b * p.logits_stride * SIZE;
  const float* nrow = p.noise + (size_t)b * p.noise_stride;
  grid_dep_wait();
  const float t = p.temperature ? p.temperature[b] : p.temperature_all;
  const float top_p = p.top_p ? p.top_p[b] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[b] : p.min_p_all;
  const int top_k = p.top_k ? p.top_k[b] : p.top_k_all;
  const bool greedy = !(t > 0.f), by_k = top_k > 0 && top_k < p.V;
  SampleScale sc;
  sc.inv_t = greedy ? 0.f : inverse_temperature(t);
  sc.k2 = sc.inv_t * kLog2e;

  if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  // before the first access to another CTA's memory: all of the cluster have started
  auto started = [&]() {
    if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  };
  if (p.filters)
    for (int i = tid; i < 2 * kSampleBins; i += kSampleThreads) hist[i] = 0;
  if (tid == 0) {
    s.hist = hist;
    s.n_list = 0, s.overflow = 0, s.found_bin = kSampleBins - 1, s.found_count = 0, s.first = 0x7fffffff, s.bound = 0;
  }

  // ---- the slice: chunks [c0, c1) of the 16-byte chunks that the row touches.  Elements of a
  // chunk outside the row, and NaN, become -inf.
  const int skip = (int)(reinterpret_cast<uintptr_t>(lrow) & 15) / SIZE;
  const char* base = lrow - (size_t)skip * SIZE;
  const int chunks = (p.V + skip + EPC - 1) / EPC, per = (chunks + C - 1) / C;
  const int c0 = min(rank * per, chunks), c1 = min(c0 + per, chunks);
  const bool cached = p.slice_chunks > 0;
  auto fetch = [&](int c) {
    const int i0 = c * EPC - skip;
    uint32_t w[4];
    if (i0 >= 0 && i0 + EPC <= p.V) {
      const uint4 u = *reinterpret_cast<const uint4*>(base + (size_t)c * 16);
      w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (DT == 2) {
          w[j] = i0 + j >= 0 && i0 + j < p.V ? reinterpret_cast<const uint32_t*>(lrow)[i0 + j] : 0xff800000u;
        } else {
          const uint32_t none = DT == 1 ? 0xff80u : 0xfc00u;
          const uint16_t* h = reinterpret_cast<const uint16_t*>(lrow);
          const int a = i0 + 2 * j;
          const uint32_t lo = a >= 0 && a < p.V ? h[a] : none, hi = a + 1 >= 0 && a + 1 < p.V ? h[a + 1] : none;
          w[j] = lo | hi << 16;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = clean_word<DT>(w[j]);
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  auto unpack = [](uint4 u, float* x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (DT == 2) {
        x[j] = __uint_as_float(w[j]);
      } else {
        const float2 f = unpack2<DT == 1>(w[j]);
        x[2 * j % EPC] = f.x;
        x[(2 * j + 1) % EPC] = f.y;
      }
    }
  };
  // calls f(first index, EPC logits) for the chunks of this thread
  auto each = [&](auto&& f) {
    for (int c = c0 + tid; c < c1; c += kSampleThreads) {
      float x[EPC];
      unpack(cached ? data[c - c0] : fetch(c), x);
      f(c * EPC - skip, x);
    }
  };
  float tmax = -INFINITY;  // of this thread's elements
  {
    uint32_t m = DT == 2 ? 0xff800000u : DT == 1 ? 0xff80ff80u : 0xfc00fc00u;
#pragma unroll 4
    for (int c = c0 + tid; c < c1; c += kSampleThreads) {
      const uint4 u = fetch(c);
      if (cached) data[c - c0] = u;
      m = max_word<DT>(max_word<DT>(max_word<DT>(m, u.x), max_word<DT>(u.y, u.z)), u.w);
    }
    if (DT == 2) {
      tmax = __uint_as_float(m);
    } else {
      const float2 f = unpack2<DT == 1>(m);
      tmax = fmaxf(f.x, f.y);
    }
  }
  sc.mx = key_logit(block_max(order_key(tmax), s));

  if (by_k && !greedy && top_k <= kSampleMaxK) {
    // ---- top-k: list what can be among this slice's k largest
    const float mx = sc.mx;
    auto bin_of = [&](float x) { return min(kSampleBins - 1, __float2int_rz((mx - x) * kSampleBinsPerLogit)); };
    // the bin of rank `want` - 1 of the histogram, and the count down to its end
    auto find = [&](unsigned want) {
      __syncthreads();
      unsigned v[PER], sum = 0, total;
#pragma unroll
      for (int j = 0; j < PER; ++j) v[j] = hist[tid * PER + j], sum += v[j];
      unsigned at = block_exclusive(sum, s.warp_u, total);
      want = min(want, total);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (at < want && at + v[j] >= want) s.found_bin = tid * PER + j, s.found_count = at + v[j];
        at += v[j];
      }
      __syncthreads();
      return total;
    };
    unsigned n = 0;
    if (mx == INFINITY) {
      n = ~0u;
    } else if (mx > -INFINITY) {
      bool listed = false;
      if (top_k <= kSampleQuickK) {
        if (tmax > -INFINITY) atomicAdd(&hist[bin_of(tmax)], 1u);
        if (find(top_k) >= (unsigned)top_k) {
          // k threads have a maximum of at least this, so the k-th largest token is no less
          const bool in = tmax > -INFINITY && bin_of(tmax) <= (int)s.found_bin;
          const float least = key_logit(~block_max(in ? ~order_key(tmax) : 0u, s));
          each([&](int i0, const float* x) {
#pragma unroll
            for (int e = 0; e < EPC; ++e)
              if (x[e] >= least) {
                const unsigned at = atomicAdd(&s.n_list, 1u);
                if (at < kSampleListed) list[at] = rank_key(x[e], i0 + e);
              }
          });
          __syncthreads();
          n = s.n_list;
          listed = n <= kSampleListed;
        }
      }
      if (!listed) {
        __syncthreads();
        for (int i = tid; i < kSampleBins; i += kSampleThreads) hist[i] = 0;
        if (tid == 0) s.n_list = 0;
        __syncthreads();
        each([&](int, const float* x) {
#pragma unroll
          for (int e = 0; e < EPC; ++e)
            if (x[e] > -INFINITY) atomicAdd(&hist[bin_of(x[e])], 1u);
        });
        find(top_k);
        const int last = s.found_bin;
        n = s.found_count <= kSampleListed ? s.found_count : ~0u;
        if (n != ~0u) {
          each([&](int i0, const float* x) {
#pragma unroll
            for (int e = 0; e < EPC; ++e)
              if (x[e] > -INFINITY && bin_of(x[e]) <= last) list[atomicAdd(&s.n_list, 1u)] = rank_key(x[e], i0 + e);
          });
        }
      }
    }
    started();
    if (tid == 0) s0.sent[rank] = n;
    meet();
    if (rank != 0) {
      meet();  // the first CTA has read the list
      return;
    }
    int start[kSampleMaxCluster + 1], total = 0;
    bool fits = true;
#pragma unroll
    for (int r = 0; r < kSampleMaxCluster; ++r) {
      start[r] = total;
      if (r < C) {
        fits = fits && s.sent[r] != ~0u;
        total += (int)s.sent[r];
      }
    }
    if (fits) {
      auto remote = [&](int i) {
        int r = 0, from = 0;
#pragma unroll
        for (int q = 1; q < kSampleMaxCluster; ++q)
          if (q < C && i >= start[q]) r = q, from = start[q];
        return cluster.map_shared_rank(list, r)[i - from];
      };
      // scratch over the slice: [2048] binned, [1024] sorted, [2048] the cluster's listed tokens
      unsigned long long* scratch = reinterpret_cast<unsigned long long*>(data);
      unsigned long long* sorted = scratch + 2 * kSampleMaxK;
      unsigned long long* near_list = scratch + 3 * kSampleMaxK;
      bool done;
      if (C == 1 || total <= 2 * kSampleMaxK) {  // brought here once, the other CTAs leave
        if (C > 1) {
          for (int i = tid; i < total; i += kSampleThreads) near_list[i] = remote(i);
          meet();
        } else {
          near_list = list;
        }
        done = sample_topk(p, s, b, nrow, sc, total, [&](int i) { return near_list[i]; }, [] { __syncthreads(); },
                           scratch, sorted, top_k, top_p, min_p);
      } else {
        done = sample_topk(p, s, b, nrow, sc, total, remote, meet, scratch, sorted, top_k, top_p, min_p);
      }
      if (done) return;
    } else {
      meet();
    }
    __syncthreads();
    unsigned long long best = 0;
    for (int i = tid; i < p.V; i += kSampleThreads) {
      const unsigned long long key = rank_key(clean_logit(load_logit<DT>(lrow, i)), i);
      best = key > best ? key : best;
    }
    best = block_max(best, s);
    sc.mx = key_logit((uint32_t)(best >> 32));
    sample_general<DT>(p, s, b, lrow, nrow, sc, (int)~(uint32_t)best, top_k, top_p, min_p);
    return;
  }

  // ---- the row's first: the threads that hold the slice's maximum look for its lowest index
  if (sc.mx > -INFINITY && tmax == sc.mx) {
    int arg = 0x7fffffff;
    each([&](int i0, const float* x) {
#pragma unroll
      for (int e = EPC - 1; e >= 0; --e)
        if (x[e] == tmax && i0 + e < arg) arg = i0 + e;
    });
    atomicMin(&s.first, arg);
  }
  started();
  __syncthreads();
  unsigned long long best = sc.mx > -INFINITY ? rank_key(sc.mx, s.first) : 0ull;
  if (C > 1) {
    if (tid == 0) s.best_key = best;
    meet();
    for (int r = 0; r < C; ++r) {
      const unsigned long long y = cluster.map_shared_rank(&s, r)->best_key;
      best = y > best ? y : best;
    }
  }
  const int first = (int)~(uint32_t)best;
  sc.mx = best != 0 ? key_logit((uint32_t)(best >> 32)) : -INFINITY;
  const bool general = by_k || sc.mx == INFINITY || (top_p < 1.f && per * EPC > kSampleMaxSlice);
  if (best == 0 || greedy || general) {
    meet();  // the others have read this CTA's best_key
    if (rank != 0) return;
    if (best == 0 || greedy) {
      if (tid == 0) p.tokens[b] = best == 0 ? -1 : first, p.logprobs[b] = best == 0 ? -INFINITY : 0.f;
    } else {
      sample_general<DT>(p, s, b, lrow, nrow, sc, first, top_k, top_p, min_p);
    }
    return;
  }

  // ---- the race.  Only a token whose quick weight comes within 1e-4 of beating `bound`, the best
  // that its CTA has seen (the quick weight's error is below 2e-5), gets an exact weight and
  // division; the first token's own score is the bound to start from.  The bound stays finite: after
  // a random number of 0, tokens of another such number still enter, and the lowest index wins.
  float score = 0.f;
  int token = 0x7fffffff;
  double rest = 0.0;
  const float e_first = nrow[first];
  constexpr float kMost = 3.402823466e38f;
  float bound = e_first > 0.f ? fminf(1.f / e_first, kMost) : 0.f, near = bound * 0.9999f;
  auto enter = [&](int i, float x, float w, float e) {
    if (w > near * e) {
      const float y = expf(sc.dist(x)) / e;
      if (y > score || (y == score && i < token)) score = y, token = i;
    }
  };
  // one chunk per thread, with random numbers e and weights w, 0 for the tokens that stay out;
  // returns the weights' sum without the first token's own 1
  auto race = [&](int i0, const float* x, const float* w, const float* e) {
    float2 sum2 = make_float2(w[0], w[1]);
    bool any = false;
    bound = fmaxf(bound, __uint_as_float(*const_cast<volatile unsigned int*>(&s.bound)));
    near = bound * 0.9999f;
#pragma unroll
    for (int q = 0; q < EPC; q += 2) {
      if (q > 0) sum2 = __fadd2_rn(sum2, make_float2(w[q], w[q + 1]));
      const float2 lim = __fmul2_rn(make_float2(e[q], e[q + 1]), make_float2(near, near));
      any |= w[q] > lim.x || w[q + 1] > lim.y;
    }
    float sum = sum2.x + sum2.y;
    if ((unsigned)(first - i0) < (unsigned)EPC) {
      sum = 0.f;
#pragma unroll
      for (int q = 0; q < EPC; ++q) sum += i0 + q != first ? w[q] : 0.f;
    }
    if (__any_sync(0xffffffffu, any)) {
      if (any) {
#pragma unroll
        for (int q = 0; q < EPC; ++q) enter(i0 + q, x[q], w[q], e[q]);
      }
      __syncwarp();
      bound = fmaxf(bound, __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fminf(score, kMost)))));
      if ((tid & 31) == 0) atomicMax(&s.bound, __float_as_uint(bound));
      near = bound * 0.9999f;
    }
    return sum;
  };
  auto log2w2 = [&](float x0, float x1) {
    return __fmul2_rn(__fadd2_rn(make_float2(x0, x1), make_float2(-sc.mx, -sc.mx)), make_float2(sc.k2, sc.k2));
  };
  if (top_p < 1.f) {
    // ---- top-p: bins of the weights' logarithm
    const float to_bin = -kSampleBinsPerLog2;
    each([&](int i0, const float* x) {
      unsigned most = 0;
#pragma unroll
      for (int q = 0; q < EPC; q += 2) {
        const float2 l2 = log2w2(x[q], x[q + 1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const unsigned w = sc.fixed(j ? l2.y : l2.x);
          most = max(most, w);
          if (w == 0) continue;
          const int bin = min(kSampleBins - 1, __float2int_rz((j ? l2.y : l2.x) * to_bin));
          atomicAdd(&hist[bin], w & 0xffffu);
          if (w >> 16) atomicAdd(&hist[kSampleBins + bin], w >> 16);
        }
      }
      // the random numbers of tokens that are likely to stay, on their way while the bins are summed
      if (most >= 1u << 19) asm volatile("prefetch.global.L2 [%0];" ::"l"(nrow + max(i0, 0)));
    });
    meet();
    if (C > 1) {  // a stripe of the bins each, summed over the cluster
      for (int i = rank * kSampleThreads + tid; i < kSampleBins; i += C * kSampleThreads) {
        unsigned long long sum = 0;
        for (int r = 0; r < C; ++r) {
          const unsigned int* h = cluster.map_shared_rank(hist, r);
          sum += h[i] + ((unsigned long long)h[kSampleBins + i] << 16);
        }
        list0[i] = sum;
      }
      meet();
    }
    if (rank == 0) {
      unsigned long long v[PER], sum = 0, total;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int i = tid * PER + j;
        v[j] = C > 1 ? list[i] : hist[i] + ((unsigned long long)hist[kSampleBins + i] << 16);
        sum += v[j];
      }
      unsigned long long at = block_exclusive(sum, s.warp_ull, total);
      const unsigned long long target = (unsigned long long)fmax(1.0, ceil((double)fmaxf(top_p, 0.f) * (double)total));
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (at < target && at + v[j] >= target) s.found_bin = tid * PER + j, s.base = at, s.target = target;
        at += v[j];
      }
    }
    meet();
    // ---- the tokens of the bins above the crossing one race, its own are listed
    const float cross = (float)s0.found_bin;
    for (int cb = c0; cb < c1; cb += kSampleThreads) {  // (the warps stay together)
      const int c = cb + tid, i0 = c * EPC - skip;
      float x[EPC], w[EPC], e[EPC];
#pragma unroll
      for (int q = 0; q < EPC; ++q) w[q] = 0.f;
      if (c < c1) {
        unpack(cached ? data[c - c0] : fetch(c), x);
#pragma unroll
        for (int q = 0; q < EPC; q += 2) {
          const float2 l2 = log2w2(x[q], x[q + 1]), at = __fmul2_rn(l2, make_float2(to_bin, to_bin));
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float a = j ? at.y : at.x;
            if (a < cross) {
              const float y = ex2_approx(j ? l2.y : l2.x);
              w[q + j] = y >= min_p || i0 + q + j == first ? y : 0.f;
            } else if (a < cross + 1.f) {
              const unsigned n = atomicAdd(&s0.n_list, 1u);
              if (n < kSampleTies) list0[n] = rank_key(x[q + j], i0 + q + j);
            }
          }
        }
      }
#pragma unroll
      for (int q = 0; q < EPC; ++q) e[q] = w[q] > 0.f ? nrow[i0 + q] : 1.f;
      rest += (double)race(i0, x, w, e);
    }
    block_race(score, token, rest, s);
    if (tid == 0) s0.score[rank] = score, s0.token[rank] = token, s0.rest[rank] = rest;
    meet();
    if (rank != 0) return;
    const int n = s.n_list;
    if (n > kSampleTies) {
      __syncthreads();
      sample_general<DT>(p, s, b, lrow, nrow, sc, first, top_k, top_p, min_p);
      return;
    }
    for (int i = tid; i < n; i += kSampleThreads) hist[i] = sc.fixed(sc.log2w(key_logit((uint32_t)(list[i] >> 32))));
    score = 0.f, token = 0x7fffffff, rest = 0.0;
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += kSampleThreads / 4) {  // four lanes to a token
      const int i = i0 + tid / 4;
      unsigned long long before = 0;
      const unsigned long long key = i < n ? list[i] : 0ull;
      for (int j = tid & 3; j < n; j += 4) before += list[j] > key ? hist[j] : 0u;
      before += __shfl_xor_sync(0xffffffffu, before, 1);
      before += __shfl_xor_sync(0xffffffffu, before, 2);
      if (i >= n || (tid & 3) != 0 || s.base + before >= s.target) continue;
      const int at = (int)~(uint32_t)key;
      const float x = key_logit((uint32_t)(key >> 32)), w = ex2_approx(sc.log2w(x));
      if (at != first) {
        if (w < min_p) continue;
        rest += (double)w;  // exact in any order: at most 1024 floats of one bin, within 2^(1/44) of each other
      }
      enter(at, x, w, nrow[at]);
    }
    block_race(score, token, rest, s);
  } else if (min_p <= 0.f) {
    // ---- every token: the random numbers stream in beside the logits
    const bool wide = (reinterpret_cast<uintptr_t>(nrow - skip) & 15) == 0;
    constexpr int AHEAD = 16 / EPC;  // chunks whose numbers are in flight
    for (int cb = c0; cb < c1; cb += AHEAD * kSampleThreads) {
      float e[AHEAD][EPC];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int c = cb + a * kSampleThreads + tid, i0 = c * EPC - skip;
        if (c < c1 && wide && i0 >= 0 && i0 + EPC <= p.V) {
#pragma unroll
          for (int q = 0; q < EPC / 4; ++q)
            *reinterpret_cast<float4*>(&e[a][4 * q]) = __ldcs(reinterpret_cast<const float4*>(nrow + i0 + 4 * q));
        } else {
#pragma unroll
          for (int q = 0; q < EPC; ++q) e[a][q] = c < c1 && i0 + q >= 0 && i0 + q < p.V ? nrow[i0 + q] : 1.f;
        }
      }
      float sum = 0.f;
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int c = cb + a * kSampleThreads + tid;
        float x[EPC], w[EPC];
#pragma unroll
        for (int q = 0; q < EPC; ++q) w[q] = 0.f;
        if (c < c1) {
          unpack(cached ? data[c - c0] : fetch(c), x);
#pragma unroll
          for (int q = 0; q < EPC; q += 2) {
            const float2 l2 = log2w2(x[q], x[q + 1]);
            w[q] = ex2_approx(l2.x);
            w[q + 1] = ex2_approx(l2.y);
          }
        }
        sum += race(c * EPC - skip, x, w, e[a]);
      }
      rest += (double)sum;
    }
    block_race(score, token, rest, s);
  } else {
    // ---- min-p alone
    for (int cb = c0; cb < c1; cb += kSampleThreads) {
      const int c = cb + tid, i0 = c * EPC - skip;
      float x[EPC], w[EPC], e[EPC];
#pragma unroll
      for (int q = 0; q < EPC; ++q) w[q] = 0.f;
      if (c < c1) {
        unpack(cached ? data[c - c0] : fetch(c), x);
#pragma unroll
        for (int q = 0; q < EPC; ++q) {
          const float y = ex2_approx(sc.log2w(x[q]));
          w[q] = y >= min_p || i0 + q == first ? y : 0.f;
        }
      }
#pragma unroll
      for (int q = 0; q < EPC; ++q) e[q] = w[q] > 0.f ? nrow[i0 + q] : 1.f;
      rest += (double)race(i0, x, w, e);
    }
    block_race(score, token, rest, s);
  }

  // ---- the first CTA joins the results of all (after top-p its own last one is a further part)
  const bool more = top_p < 1.f;
  if (!more) {
    if (tid == 0) s0.score[rank] = score, s0.token[rank] = token, s0.rest[rank] = rest;
    meet();
  }
  if (rank == 0 && tid == 0) {
    for (int r = more ? 0 : 1; r < C; ++r) {
      if (s.score[r] > score || (s.score[r] == score && s.token[r] < token)) score = s.score[r], token = s.token[r];
      rest += s.rest[r];
    }
    if (token == 0x7fffffff) token = first;  // no number won
    p.tokens[b] = token;
    p.logprobs[b] = sc.dist(clean_logit(load_logit<DT>(lrow, token))) - log1pf((float)rest);
  }
}

// ---------------------------------------------------------------------------
// No filter at all: the race in one pass over logits and random numbers.  Weights are taken
// relative to the largest logit that the warp has met, sums are rescaled when that grows, and
// two tokens are compared by e^(x1 - x2) e2 / e1, which needs no maximum; so nothing waits
// before the last loads have been issued.  Bound by the bytes of the two arrays: 256 rows of
// 131072 float32 logits, 268 MB, take 55 us, 4.9 TB/s or 0.74 of the measured copy rate.
// ---------------------------------------------------------------------------
struct StreamPart {
  float m;      // largest logit (FLT_MAX for +inf, -infinity before any)
  double rest;  // sum of the weights relative to m, without that of one token of logit m
  float x, e;   // the race's leader
  int i;        // its index, or INT_MAX: nothing yet
  int first;    // lowest index of logit m (greedy rows)
};

// e^((x1 - x2) / T) / e1 > 1 / e2, ties to the lower index
__device__ __forceinline__ bool stream_beats(float x1, float e1, int i1, float x2, float e2, int i2, float inv_t) {
  if (i2 == 0x7fffffff) return true;
  if (i1 == 0x7fffffff) return false;
  const float a = expf((x1 - x2) * inv_t) * e2;
  return a > e1 || (a == e1 && i1 < i2);
}

__device__ __forceinline__ StreamPart stream_join(StreamPart a, const StreamPart& b, float inv_t, float k2, bool greedy) {
  const bool none_a = a.first == 0x7fffffff, none_b = b.first == 0x7fffffff;
  if (b.m > a.m || (b.m == a.m && b.first < a.first)) a.first = b.first;
  const float m = fmaxf(a.m, b.m);
  // each part's own token of weight 1 is left out of its rest: that of the smaller maximum comes
  // back in; a part that has met nothing (m = -FLT_MAX) has none
  const double fa = a.m == m ? 1.0 : (double)exp2f((a.m - m) * k2), fb = b.m == m ? 1.0 : (double)exp2f((b.m - m) * k2);
  a.rest = a.rest * fa + b.rest * fb;
  if (!none_a && !none_b) a.rest += a.m == m ? fb : fa;
  a.m = m;
  if (!greedy && stream_beats(b.x, b.e, b.i, a.x, a.e, a.i, inv_t)) a.x = b.x, a.e = b.e, a.i = b.i;
  return a;
}

constexpr int kStreamThreads = 256;

template <int DT>
__global__ void __launch_bounds__(kStreamThreads, 4) coalibi_sample_stream_kernel(const SampleParams p) {
  namespace cg = cooperative_groups;
  constexpr int SIZE = DT == 2 ? 4 : 2, EPC = 16 / SIZE;
  constexpr int AHEAD = 16 / EPC, N = AHEAD * EPC;  // chunks and tokens of a thread in flight
  constexpr int WARPS = kStreamThreads / 32;
  __shared__ StreamPart s_part[WARPS], s_row[kSampleMaxCluster];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = p.cluster, rank = C > 1 ? (int)cluster.block_rank() : 0, b = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  const char* lrow = static_cast<const char*>(p.logits) + (size_t)b * p.logits_stride * SIZE;
  const float* nrow = p.noise + (size_t)b * p.noise_stride;
  grid_dep_wait();
  const float t = p.temperature ? p.temperature[b] : p.temperature_all;
  const bool greedy = !(t > 0.f);
  const float inv_t = greedy ? 1.f : inverse_temperature(t), k2 = inv_t * kLog2e;
  const int skip = (int)(reinterpret_cast<uintptr_t>(lrow) & 15) / SIZE;
  const char* base = lrow - (size_t)skip * SIZE;
  const int chunks = (p.V + skip + EPC - 1) / EPC, per = (chunks + C - 1) / C;
  const int c0 = min(rank * per, chunks), c1 = min(c0 + per, chunks);
  const bool wide = (reinterpret_cast<uintptr_t>(nrow - skip) & 15) == 0;

  float m = -INFINITY, near = 0.f;  // of the warp
  bool inf = false;
  double rest = 0.0;                // of the lane
  float lx = 0.f, le = 1.f;
  int li = 0x7fffffff, first = 0x7fffffff;
  for (int cb = c0; cb < c1; cb += AHEAD * kStreamThreads) {
    float x[N], e[N];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int c = cb + a * kStreamThreads + tid, i0 = c * EPC - skip;
      if (c < c1 && wide && i0 >= 0 && i0 + EPC <= p.V) {
        const uint4 u = __ldcs(reinterpret_cast<const uint4*>(base + (size_t)c * 16));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int q = 0; q < EPC / 4; ++q)
          *reinterpret_cast<float4*>(&e[a * EPC + 4 * q]) = __ldcs(reinterpret_cast<const float4*>(nrow + i0 + 4 * q));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (DT == 2) {
            x[a * EPC + j] = __uint_as_float(clean_word<DT>(w[j]));
          } else {
            const float2 f = unpack2<DT == 1>(clean_word<DT>(w[j]));
            x[a * EPC + 2 * j % EPC] = f.x;
            x[a * EPC + (2 * j + 1) % EPC] = f.y;
          }
        }
      } else {
#pragma unroll
        for (int q = 0; q < EPC; ++q) {
          const bool in = c < c1 && i0 + q >= 0 && i0 + q < p.V;
          x[a * EPC + q] = in ? clean_logit(load_logit<DT>(lrow, i0 + q)) : -INFINITY;
          e[a * EPC + q] = in ? nrow[i0 + q] : 1.f;
        }
      }
    }
    auto index = [&](int n) { return (cb + n / EPC * kStreamThreads + tid) * EPC - skip + n % EPC; };
    float top = x[0];
#pragma unroll
    for (int n = 1; n < N; ++n) top = fmaxf(top, x[n]);
    if (!inf && __any_sync(0xffffffffu, top == INFINITY)) {  // all the weight is theirs
      inf = true;
      m = -INFINITY, near = 0.f, rest = 0.0, li = 0x7fffffff, first = 0x7fffffff;
    }
    if (inf) {
      top = -INFINITY;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        x[n] = x[n] == INFINITY ? 3.402823466e38f : -INFINITY;
        top = fmaxf(top, x[n]);
      }
    }
    bool mine = false;  // whether the token left out of `rest` is one of this lane's here
    if (__any_sync(0xffffffffu, top > m)) {
      const float up = key_logit(__reduce_max_sync(0xffffffffu, order_key(top)));
      const float f = m > -INFINITY ? ex2_approx((m - up) * k2) : 0.f;
      rest = rest * (double)f + (lane == 0 ? (double)f : 0.0);
      near *= f;
      m = up;
      mine = lane == __ffs(__ballot_sync(0xffffffffu, top == m)) - 1;
      int at = 0x7fffffff;
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (x[n] == m) at = min(at, index(n));
      first = __reduce_min_sync(0xffffffffu, at);
    }
    const float mc = fmaxf(m, -3.402823466e38f);
    float w[N];
    float2 sum2 = make_float2(0.f, 0.f);
    bool any = false;
#pragma unroll
    for (int n = 0; n < N; n += 2) {
      const float2 l2 = __fmul2_rn(__fadd2_rn(make_float2(x[n], x[n + 1]), make_float2(-mc, -mc)), make_float2(k2, k2));
      w[n] = ex2_approx(l2.x);
      w[n + 1] = ex2_approx(l2.y);
      sum2 = __fadd2_rn(sum2, make_float2(w[n], w[n + 1]));
      const float2 lim = __fmul2_rn(make_float2(e[n], e[n + 1]), make_float2(near, near));
      any |= w[n] > lim.x || w[n + 1] > lim.y;
    }
    float sum = sum2.x + sum2.y;
    if (mine) {
      bool out = false;
      sum = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const bool skip_it = !out && x[n] == m;
        out |= skip_it;
        sum += skip_it ? 0.f : w[n];
      }
    }
    rest += (double)sum;
    if (__any_sync(0xffffffffu, any)) {
      if (any) {
#pragma unroll
        for (int n = 0; n < N; ++n)
          if (w[n] > near * e[n] && stream_beats(x[n], e[n], index(n), lx, le, li, inv_t))
            lx = x[n], le = e[n], li = index(n);
      }
      __syncwarp();
      const float v = li == 0x7fffffff ? 0.f : ex2_approx((lx - mc) * k2) / le;
      near = 0.9999f * __uint_as_float(__reduce_max_sync(0xffffffffu, v > 0.f ? __float_as_uint(v) : 0u));
    }
  }
  // ---- lanes, warps, CTAs
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float ox = __shfl_xor_sync(0xffffffffu, lx, o), oe = __shfl_xor_sync(0xffffffffu, le, o);
    const int oi = __shfl_xor_sync(0xffffffffu, li, o);
    if (stream_beats(ox, oe, oi, lx, le, li, inv_t)) lx = ox, le = oe, li = oi;
    rest += __shfl_xor_sync(0xffffffffu, rest, o);
  }
  if (lane == 0) {
    s_part[warp] = StreamPart{m, rest, lx, le, li, first};
  }
  __syncthreads();
  if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (tid == 0) {
    StreamPart a = s_part[0];
    for (int w = 1; w < WARPS; ++w) a = stream_join(a, s_part[w], inv_t, k2, greedy);
    (C > 1 ? cluster.map_shared_rank(s_row, 0) : s_row)[rank] = a;
  }
  if (C > 1) cluster.sync();
  if (rank == 0 && tid == 0) {
    StreamPart a = s_row[0];
    for (int r = 1; r < C; ++r) a = stream_join(a, s_row[r], inv_t, k2, greedy);
    if (a.first == 0x7fffffff) {
      p.tokens[b] = -1;
      p.logprobs[b] = -INFINITY;
    } else if (greedy || a.i == 0x7fffffff) {  // (no number won: the first of the ranking)
      p.tokens[b] = a.first;
      p.logprobs[b] = greedy ? 0.f : -log1pf((float)a.rest);
    } else {
      p.tokens[b] = a.i;
      p.logprobs[b] = (a.x == a.m ? 0.f : (a.x - a.m) * inv_t) - log1pf((float)a.rest);
    }
  }
}

}  // namespace coalibi
