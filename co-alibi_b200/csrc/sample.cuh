// Drawing tokens from logits: temperature, top-k, top-p, min-p and a race of given
// exponential random numbers, one CTA per row.
//
// With the tokens ranked by (logit descending, index ascending) every filter keeps a
// prefix of the ranking, so a row needs one threshold: the lowest ranked key kept.
// It is found without sorting, by radix descent: 8 bits of the key per level, a
// histogram of the counts (top-k) or of the weights (top-p) of the keys that share
// the prefix so far, and the bin in which the wanted count or mass is reached.  The
// key is 64 bits, the logit mapped to an ordered integer and the inverted index
// below it, so equal logits are told apart by the same descent.
#pragma once

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
};

constexpr int kSampleThreads = 1024;
// Weights are summed as integers of 2^-42: the sum of up to 2^21 of them (each at most
// 1) fits 64 bits, integer addition makes the order of the atomics irrelevant, and
// the resolution is below float32's for every weight above 2^-18 of the largest.
constexpr float kWeightOne = 4398046511104.f;  // 2^42

template <int DT>
__device__ __forceinline__ float load_logit(const void* base, long long i) {
  if (DT == 2) return static_cast<const float*>(base)[i];
  if (DT == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
  return __half2float(static_cast<const __half*>(base)[i]);
}

// Logit -> integer of the same order; NaN ranks with -inf, -0 with +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

template <int DT>
__global__ void __launch_bounds__(kSampleThreads) coalibi_sample_kernel(const SampleParams p) {
  __shared__ unsigned int h_cnt[256];
  __shared__ unsigned long long h_mass[256];
  __shared__ float red_f[32];
  __shared__ int red_i[32];
  __shared__ unsigned long long red_u[32];
  __shared__ unsigned long long s_prefix, s_acc;
  __shared__ int s_done;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const char* lrow = static_cast<const char*>(p.logits) + (size_t)b * p.logits_stride * (DT == 2 ? 4 : 2);
  const float* nrow = p.noise + (size_t)b * p.noise_stride;
  const float t = p.temperature ? p.temperature[b] : p.temperature_all;
  const float top_p = p.top_p ? p.top_p[b] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[b] : p.min_p_all;
  const int top_k = p.top_k ? p.top_k[b] : p.top_k_all;
  const bool greedy = !(t > 0.f);
  const float inv_t = greedy ? 0.f : 1.f / t;

  // the first of the ranking: largest key, lowest index
  unsigned long long best = 0;
  for (int i = tid; i < p.V; i += kSampleThreads) {
    const unsigned long long ck = ((unsigned long long)order_key(load_logit<DT>(lrow, i)) << 32) | (uint32_t)~i;
    best = ck > best ? ck : best;
  }
  for (int o = 16; o; o >>= 1) {
    const unsigned long long y = __shfl_xor_sync(0xffffffffu, best, o);
    best = y > best ? y : best;
  }
  if (lane == 0) red_u[warp] = best;
  __syncthreads();
  for (int w = 0; w < 32; ++w) best = red_u[w] > best ? red_u[w] : best;
  __syncthreads();
  const int first = (int)~(uint32_t)best;
  const float mx = load_logit<DT>(lrow, first);
  if ((uint32_t)(best >> 32) == order_key(-INFINITY)) {
    if (tid == 0) {
      p.tokens[b] = -1;
      p.logprobs[b] = -INFINITY;
    }
    return;
  }
  if (greedy) {
    if (tid == 0) {
      p.tokens[b] = first;
      p.logprobs[b] = 0.f;
    }
    return;
  }
  auto dist = [&](float x) { return x == mx ? 0.f : (x != x ? -INFINITY : (x - mx) * inv_t); };

  // lowest key kept; the histogram descent below raises it
  unsigned long long floor_key = ((unsigned long long)(order_key(-INFINITY) + 1)) << 32;
  for (int filter = 0; filter < 2; ++filter) {
    const bool by_mass = filter == 1;
    if (by_mass ? top_p >= 1.f : (top_k <= 0 || top_k >= p.V)) continue;
    unsigned long long target;
    if (by_mass) {
      unsigned long long s = 0;
      for (int i = tid; i < p.V; i += kSampleThreads) {
        const float x = load_logit<DT>(lrow, i);
        const unsigned long long ck = ((unsigned long long)order_key(x) << 32) | (uint32_t)~i;
        if (ck >= floor_key) s += (unsigned long long)(expf(dist(x)) * kWeightOne);
      }
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) red_u[warp] = s;
      __syncthreads();
      s = 0;
      for (int w = 0; w < 32; ++w) s += red_u[w];
      __syncthreads();
      const double want = (double)fmaxf(top_p, 0.f) * (double)s;
      target = want < 1.0 ? 1ull : (unsigned long long)ceil(want);
    } else {
      target = top_k;
    }
    if (tid == 0) {
      s_prefix = 0;
      s_acc = 0;
      s_done = 0;
    }
    for (int shift = 56; shift >= 0; shift -= 8) {
      if (tid < 256) {
        h_cnt[tid] = 0;
        h_mass[tid] = 0;
      }
      __syncthreads();
      const unsigned long long prefix = s_prefix;
      for (int i = tid; i < p.V; i += kSampleThreads) {
        const float x = load_logit<DT>(lrow, i);
        const unsigned long long ck = ((unsigned long long)order_key(x) << 32) | (uint32_t)~i;
        if (ck < floor_key || (shift < 56 && (ck >> (shift + 8)) != (prefix >> (shift + 8)))) continue;
        const int bin = (int)(ck >> shift) & 255;
        atomicAdd(&h_cnt[bin], 1u);
        if (by_mass) atomicAdd(&h_mass[bin], (unsigned long long)(expf(dist(x)) * kWeightOne));
      }
      __syncthreads();
      if (tid == 0) {
        unsigned long long acc = s_acc;
        int bin = 255, last = -1;
        for (; bin >= 0; --bin) {
          if (h_cnt[bin] == 0) continue;
          last = bin;
          const unsigned long long v = by_mass ? h_mass[bin] : h_cnt[bin];
          if (acc + v >= target) break;
          acc += v;
        }
        if (bin < 0) bin = last, acc = 0, s_done = 2;  // fewer than the target: all stay
        s_acc = acc;
        s_prefix = prefix | ((unsigned long long)bin << shift);
        if (s_done == 0 && (h_cnt[bin] == 1 || (!by_mass && acc + h_cnt[bin] == target))) s_done = 1;
      }
      __syncthreads();
      if (s_done) break;
    }
    if (s_done != 2 && s_prefix > floor_key) floor_key = s_prefix;
    __syncthreads();
  }

  // the race among the kept, and the sum of their weights without the first's (exactly 1)
  float score = -1.f;
  int token = first;
  unsigned long long rest = 0;
  for (int i = tid; i < p.V; i += kSampleThreads) {
    const float x = load_logit<DT>(lrow, i);
    const unsigned long long ck = ((unsigned long long)order_key(x) << 32) | (uint32_t)~i;
    const float w = expf(dist(x));
    if (ck < floor_key || w < min_p || w == 0.f) {
      if (i != first) continue;
    }
    if (i != first) rest += (unsigned long long)(w * kWeightOne);
    const float sc = w / nrow[i];
    if (sc > score || (sc == score && i < token)) score = sc, token = i;
  }
  for (int o = 16; o; o >>= 1) {
    const float ys = __shfl_xor_sync(0xffffffffu, score, o);
    const int yi = __shfl_xor_sync(0xffffffffu, token, o);
    if (ys > score || (ys == score && yi < token)) score = ys, token = yi;
    rest += __shfl_xor_sync(0xffffffffu, rest, o);
  }
  if (lane == 0) red_f[warp] = score, red_i[warp] = token, red_u[warp] = rest;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < 32; ++w) {
      if (red_f[w] > score || (red_f[w] == score && red_i[w] < token)) score = red_f[w], token = red_i[w];
      rest += red_u[w];
    }
    p.tokens[b] = token;
    p.logprobs[b] = dist(load_logit<DT>(lrow, token)) - log1pf((float)((double)rest * (1.0 / (double)kWeightOne)));
  }
}

}  // namespace coalibi
