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

// Reductions over groups of LANES neighbouring lanes (16 or 64), in every lane of the group: neighbours, pairs,
// half rows and rows of 16 by the cross-lane modes of the vector instructions (no LDS), rows by a broadcast of
// the last lane's.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, ROWS, 0xf, false);
}

template <int LANES, typename OP>
__device__ __forceinline__ uint32_t group_reduce(uint32_t v, OP op) {
  v = op(v, dpp<0xb1>(v));   // lanes 1 0 3 2
  v = op(v, dpp<0x4e>(v));   // lanes 2 3 0 1
  v = op(v, dpp<0x141>(v));  // half rows mirrored
  v = op(v, dpp<0x140>(v));  // rows mirrored: now the same in all 16 lanes of a row
  if constexpr (LANES == 64) {
    const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)v, 0), b = (uint32_t)__builtin_amdgcn_readlane((int)v, 16);
    const uint32_t c = (uint32_t)__builtin_amdgcn_readlane((int)v, 32), d = (uint32_t)__builtin_amdgcn_readlane((int)v, 48);
    v = op(op(a, b), op(c, d));
  }
  return v;
}

template <int LANES>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  return group_reduce<LANES>(v, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
}

template <int LANES>
__device__ __forceinline__ float group_max(float v) {
  return bits_to_f32(group_reduce<LANES>(f32_to_bits(v), [](uint32_t x, uint32_t y) { return bits_to_f32(y) > bits_to_f32(x) ? y : x; }));
}

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
  return bits_to_f32(group_reduce<LANES>(f32_to_bits(v), [](uint32_t x, uint32_t y) { return f32_to_bits(bits_to_f32(x) + bits_to_f32(y)); }));
}

// A logit as an unsigned number of the same order; 0 where it cannot be chosen (-inf, NaN).  -0 and +0
// are equal, as they are as logits.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = f32_to_bits(f + 0.0f);
  const uint32_t k = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return f > -__builtin_inff() ? k : 0u;
}

// A lane's PER logits of a row, from column `first` on; -inf behind the row.  Rows begin at any element: the
// vectors are read at whatever alignment they have.
template <int DT, int PER>
__device__ __forceinline__ void load_logits(const typename Elem<DT>::store_t* row, uint32_t first, uint32_t experts, float (&l)[PER]) {
  using S = typename Elem<DT>::store_t;
  constexpr int VE = PER < vec_elems<DT>() ? PER : vec_elems<DT>();
  typedef S vec __attribute__((ext_vector_type(VE)));
  typedef vec vec_unaligned __attribute__((aligned(sizeof(S))));
  if (first + PER <= experts) {
    union { vec v; S e[VE]; } x[PER / VE];
#pragma unroll
    for (int b = 0; b < PER / VE; ++b) x[b].v = *(const vec_unaligned*)(row + first + b * VE);
#pragma unroll
    for (int j = 0; j < PER; ++j) l[j] = Elem<DT>::load(x[j / VE].e[j % VE]);
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) l[j] = first + j < experts ? Elem<DT>::load(row[first + j]) : -__builtin_inff();
  }
}

// LANES lanes per token, PER experts per lane: lane l of the group holds the experts from l * PER on, so that
// the lowest index among equal logits is the lowest lane's first.  A choice takes the largest key of the
// group; its owner is the lowest lane that has it, its place the first in that lane.  16 lanes per token
// serve four tokens with the instructions of one where a lane has room for its share.
template <int DT, int LANES, int PER>
__global__ __launch_bounds__(kRouterWaves * kWave) void router_kernel(const RouterArgs a) {
  using S = typename Elem<DT>::store_t;
  constexpr uint32_t kTokens = kWave / LANES;  // per wavefront
  const uint32_t lane = threadIdx.x % kWave, member = lane % LANES, group = lane / LANES;
  const uint64_t mine = LANES == 64 ? ~0ull : ((1ull << (LANES % 64)) - 1) << (group * LANES);
  const uint32_t step = gridDim.x * kRouterWaves * kTokens;
  for (uint32_t t0 = (blockIdx.x * kRouterWaves + threadIdx.x / kWave) * kTokens; t0 < a.tokens; t0 += step) {
    const uint32_t t = t0 + group < a.tokens ? t0 + group : a.tokens - 1;  // the last token again: not stored
    float l[PER];
    load_logits<DT, PER>((const S*)a.logits + (size_t)t * a.experts, member * PER, a.experts, l);
    uint32_t key[PER];
    bool nan = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      key[j] = order_key(l[j]);
      nan |= l[j] != l[j];
    }
    float top = -__builtin_inff();  // the largest logit that can be chosen
    float my_logit[64 / LANES], my_e[64 / LANES];
    int32_t my_id[64 / LANES];      // choices member, member + LANES, ...
#pragma unroll
    for (int x = 0; x < 64 / LANES; ++x) { my_id[x] = -1; my_logit[x] = 0.0f; }
    uint32_t best = 0;
    int at = 0;
#pragma unroll
    for (int j = PER - 1; j >= 0; --j) {
      const bool up = key[j] >= best;
      best = up ? key[j] : best;
      at = up ? j : at;
    }
    for (uint32_t k = 0; k < a.topk; ++k) {
      const uint32_t all = group_max<LANES>(best);
      const uint64_t have = __ballot(best == all) & mine;
      const uint32_t owner = (uint32_t)__builtin_ctzll(have);
      const bool owns = lane == owner && all;
      const int place = LANES == 64 ? __builtin_amdgcn_readlane(at, owner) : __shfl(at, (int)owner);
      const int32_t id = all ? (int32_t)((owner % LANES) * PER + place) : -1;
      // the key is the logit: turned back, it needs no look at the owner's registers
      const float value = bits_to_f32((all & 0x80000000u) ? all ^ 0x80000000u : ~all);
      if (k == 0 && all) top = value;
#pragma unroll
      for (int x = 0; x < 64 / LANES; ++x)
        if (k == member + x * LANES) { my_id[x] = id; my_logit[x] = value; }
      if (owns) {  // the owner's next best
#pragma unroll
        for (int j = 0; j < PER; ++j) key[j] = j == at ? 0u : key[j];
        best = 0;
#pragma unroll
        for (int j = PER - 1; j >= 0; --j) {
          const bool up = key[j] >= best;
          best = up ? key[j] : best;
          at = up ? j : at;
        }
      }
    }
    float total = 0.0f;
#pragma unroll
    for (int x = 0; x < 64 / LANES; ++x) {
      my_e[x] = my_id[x] >= 0 ? expf(my_logit[x] - top) : 0.0f;
      total += my_e[x];
    }
    if (!a.normalize) {
      total = 0.0f;
#pragma unroll
      for (int j = 0; j < PER; ++j) total += member * PER + j < a.experts ? expf(l[j] - top) : 0.0f;
    }
    total = group_sum<LANES>(total);
    if (__ballot(nan) & mine) total = __builtin_nanf("");  // the softmax of a row that holds a NaN
    if (t0 + group < a.tokens) {
#pragma unroll
      for (int x = 0; x < 64 / LANES; ++x) {
        const uint32_t k = member + x * LANES;
        if (k < a.topk) {
          a.ids[(size_t)t * a.topk + k] = my_id[x];
          a.weights[(size_t)t * a.topk + k] = my_id[x] >= 0 ? my_e[x] / total : 0.0f;
        }
      }
    }
  }
}

// d_logits of sum_k grad_weights[k] * weights[k].  With p = softmax(logits) and s = sum_k g_k w_k:
//   not normalised (w = p):            d_e = p_e ([e chosen] g_e - s)
//   normalised (w = softmax of the chosen): d_e = [e chosen] w_e (g_e - s)
// A wavefront per token; what the chosen experts get goes through LDS to the lanes that write them.
template <int DT, int PER>
__global__ __launch_bounds__(kRouterWaves * kWave) void router_grad_kernel(const RouterArgs a) {
  using S = typename Elem<DT>::store_t;
  __shared__ float space[kRouterWaves][kWave * PER];
  const uint32_t lane = threadIdx.x % kWave;
  float* chosen = space[threadIdx.x / kWave];
  for (uint32_t t = blockIdx.x * kRouterWaves + threadIdx.x / kWave; t < a.tokens; t += gridDim.x * kRouterWaves) {
    const S* row = (const S*)a.logits + (size_t)t * a.experts;
    S* out = (S*)a.grad_logits + (size_t)t * a.experts;
    int32_t id = -1;
    float g = 0.0f, value = -__builtin_inff();
    if (lane < a.topk) {
      id = a.chosen[(size_t)t * a.topk + lane];
      g = a.grad_weights[(size_t)t * a.topk + lane];
      if (id < 0 || (uint32_t)id >= a.experts) id = -1;
      if (id >= 0) value = Elem<DT>::load(row[id]);
    }
    if (id < 0) g = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) chosen[lane * PER + j] = 0.0f;
    float p[PER];
    float top, total;
    if (a.normalize) {
      top = group_max<64>(value);
      total = group_sum<64>(id >= 0 ? expf(value - top) : 0.0f);
    } else {
      load_logits<DT, PER>(row, lane * PER, a.experts, p);
      top = p[0];
#pragma unroll
      for (int j = 1; j < PER; ++j) top = p[j] > top ? p[j] : top;
      top = group_max<64>(top);
      total = 0.0f;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        p[j] = lane * PER + j < a.experts ? expf(p[j] - top) : 0.0f;
        total += p[j];
      }
      total = group_sum<64>(total);
    }
    const bool none = top == -__builtin_inff();  // nothing could be chosen: no gradient
    const float w = id >= 0 && !none ? expf(value - top) / total : 0.0f;
    const float mean = group_sum<64>(g * w);
    // an expert that is named more than once gets every share
    if (id >= 0) atomicAdd(&chosen[id], a.normalize ? w * (g - mean) : w * g);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    union { S e[PER]; } r;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const float own = chosen[lane * PER + j];
      r.e[j] = Elem<DT>::store(a.normalize || none ? own : own - (p[j] / total) * mean);
    }
    if (lane * PER + PER <= a.experts) {
      constexpr int VE = PER < vec_elems<DT>() ? PER : vec_elems<DT>();
      typedef S vec __attribute__((ext_vector_type(VE)));
      typedef vec vec_unaligned __attribute__((aligned(sizeof(S))));
#pragma unroll
      for (int b = 0; b < PER / VE; ++b) {
        vec v;
#pragma unroll
        for (int j = 0; j < VE; ++j) v[j] = r.e[b * VE + j];
        *(vec_unaligned*)(out + lane * PER + b * VE) = v;
      }
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (lane * PER + j < a.experts) out[lane * PER + j] = r.e[j];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

}  // namespace
