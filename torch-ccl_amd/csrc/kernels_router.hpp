// The router of a mixture of experts: softmax over the experts, the top-k of it, and the gradient (no
// kernel of the reference: the caller's step before the routing counts and the dispatch).
#pragma once

#include "kernels_common.hpp"

namespace {

constexpr int kRouterMaxExperts = 4096;
constexpr int kRouterMaxTopk = kWave;  // lane k keeps the k-th choice
constexpr int kRouterWaves = 4;

struct RouterArgs {
  const char* logits;
  int32_t* ids;
  float* weights;
  const float* grad_weights;
  const int32_t* chosen;
  char* grad_logits;
  uint32_t tokens;
  uint32_t experts;
  uint32_t topk;
  int normalize;
};

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint32_t o = __shfl_xor(v, d);
    v = o > v ? o : v;
  }
  return v;
}

__device__ __forceinline__ float wave_max_f32(float v) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const float o = __shfl_xor(v, d);
    v = o > v ? o : v;
  }
  return v;
}

__device__ __forceinline__ float wave_sum_f32(float v) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// A logit as an unsigned number of the same order; 0 where it cannot be chosen (-inf, NaN).  -0 and +0
// are equal, as they are as logits.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = f32_to_bits(f + 0.0f);
  const uint32_t k = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return f > -__builtin_inff() ? k : 0u;
}

// One wavefront per token.  Lane l holds the PER experts from l * PER on, so that the lowest index among
// equal logits is the lowest lane's first.
template <int DT, int PER>
__global__ __launch_bounds__(kRouterWaves * kWave) void router_kernel(const RouterArgs a) {
  using S = typename Elem<DT>::store_t;
  const uint32_t lane = threadIdx.x % kWave;
  for (uint32_t t = blockIdx.x * kRouterWaves + threadIdx.x / kWave; t < a.tokens; t += gridDim.x * kRouterWaves) {
    const S* row = (const S*)a.logits + (size_t)t * a.experts;
    float l[PER];
    uint32_t key[PER];
    bool nan = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t e = lane * PER + j;
      l[j] = e < a.experts ? Elem<DT>::load(row[e]) : -__builtin_inff();
      key[j] = order_key(l[j]);
      nan |= l[j] != l[j];
    }
    float top = -__builtin_inff();  // the largest logit
    float my_logit = -__builtin_inff();
    int32_t my_id = -1;
    for (uint32_t k = 0; k < a.topk; ++k) {
      uint32_t best = 0;
      int at = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (key[j] > best) { best = key[j]; at = j; }
      const uint32_t all = wave_max_u32(best);
      if (all == 0) break;  // nothing left to choose
      const int owner = __builtin_ctzll(__ballot(best == all));
      const int id = __shfl((int)(lane * PER) + at, owner);
      float value = 0.0f;
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (j == at) value = l[j];
      value = __shfl(value, owner);
      if ((int)lane == owner) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (j == at) key[j] = 0;
      }
      if (k == 0) top = value;
      if (lane == k) { my_id = id; my_logit = value; }
    }
    float e = my_id >= 0 ? expf(my_logit - top) : 0.0f;
    float total;
    if (a.normalize) {
      total = wave_sum_f32(e);
    } else {
      total = 0.0f;
#pragma unroll
      for (int j = 0; j < PER; ++j) total += (lane * PER + j < a.experts) ? expf(l[j] - top) : 0.0f;
      total = wave_sum_f32(total);
    }
    if (__ballot(nan)) total = __builtin_nanf("");  // the softmax of a row that holds a NaN
    if (lane < a.topk) {
      a.ids[(size_t)t * a.topk + lane] = my_id;
      a.weights[(size_t)t * a.topk + lane] = my_id >= 0 ? e / total : 0.0f;
    }
  }
}

// d_logits of sum_k grad_weights[k] * weights[k].  With p = softmax(logits) and s = sum_k g_k w_k:
//   not normalised (w = p):            d_e = p_e ([e chosen] g_e - s)
//   normalised (w = softmax of the chosen): d_e = [e chosen] w_e (g_e - s)
template <int DT, int PER>
__global__ __launch_bounds__(kRouterWaves * kWave) void router_grad_kernel(const RouterArgs a) {
  using S = typename Elem<DT>::store_t;
  const uint32_t lane = threadIdx.x % kWave;
  for (uint32_t t = blockIdx.x * kRouterWaves + threadIdx.x / kWave; t < a.tokens; t += gridDim.x * kRouterWaves) {
    const S* row = (const S*)a.logits + (size_t)t * a.experts;
    S* out = (S*)a.grad_logits + (size_t)t * a.experts;
    int32_t id = -1;
    float g = 0.0f, value = -__builtin_inff();
    if (lane < a.topk) {
      id = a.chosen[(size_t)t * a.topk + lane];
      if (id < 0 || (uint32_t)id >= a.experts) id = -1;
      if (id >= 0) {
        g = a.grad_weights[(size_t)t * a.topk + lane];
        value = Elem<DT>::load(row[id]);
      }
    }
    float l[PER];
    float top = value, total;
    if (a.normalize) {
      top = wave_max_f32(top);
      total = wave_sum_f32(id >= 0 ? expf(value - top) : 0.0f);
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const uint32_t e = lane * PER + j;
        l[j] = e < a.experts ? Elem<DT>::load(row[e]) : -__builtin_inff();
        top = l[j] > top ? l[j] : top;
      }
      top = wave_max_f32(top);
      total = 0.0f;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        l[j] = (lane * PER + j < a.experts) ? expf(l[j] - top) : 0.0f;
        total += l[j];
      }
      total = wave_sum_f32(total);
    }
    const float w = id >= 0 ? expf(value - top) / total : 0.0f;
    const float mean = wave_sum_f32(id >= 0 ? g * w : 0.0f);
    const bool none = top == -__builtin_inff();  // nothing could be chosen: no gradient
    float d[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) d[j] = (a.normalize || none) ? 0.0f : -(l[j] / total) * mean;
    for (uint32_t k = 0; k < a.topk; ++k) {
      const int idk = __shfl(id, (int)k);
      const float add = __shfl(a.normalize ? w * (g - mean) : w * g, (int)k);
      const int j0 = idk - (int)(lane * PER);
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (idk >= 0 && j0 == j && !none) d[j] += add;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t e = lane * PER + j;
      if (e < a.experts) out[e] = Elem<DT>::store(d[j]);
    }
  }
}

}  // namespace
