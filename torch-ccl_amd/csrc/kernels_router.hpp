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

// The same for a logit of 16 bits, in the upper half of the result with `low` behind it, and back.  `u`: the
// logit's bits in the upper half.
template <int DT>
__device__ __forceinline__ uint32_t order_key16(uint32_t u, uint32_t low) {
  constexpr uint32_t kInf = DT == MCCL_BF16 ? 0x7f800000u : 0x7c000000u;
  uint32_t k = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  k &= 0xffff0000u;
  if (k == 0x7fff0000u) k = 0x80000000u;                                 // -0
  constexpr uint32_t kLowest = 0xffff0000u & ~(0x80000000u | kInf);      // the key of -inf; NaNs lie below it and above +inf's
  return k - kLowest - 1u < (0x80000000u | kInf) - kLowest ? k | low : 0u;
}
template <int DT>
__device__ __forceinline__ float logit_of_key16(uint32_t key) {
  const uint32_t u = (key & 0x80000000u) ? key ^ 0x80000000u : ~key;
  if constexpr (DT == MCCL_BF16) return bits_to_f32(u & 0xffff0000u);
  else return Elem<DT>::load((uint16_t)(u >> 16));
}
template <int DT>
__device__ __forceinline__ uint32_t upper_half(float l) {  // of a value that is one of DT
  if constexpr (DT == MCCL_BF16) return f32_to_bits(l);
  else return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)l) << 16;
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

// LANES lanes per token, PER experts per lane: lane l of the group holds the experts from l * PER on; 16
// lanes per token serve four tokens with the instructions of one.  A choice takes the largest key of the
// group.  Logits of 16 bits have a key of 32 with the expert's index (the lower the larger) behind the logit:
// the largest key is the choice.  Keys of fp32 logits fill 32 bits; the choice is the lowest lane that has
// the largest, and in it the first.  The weights need no more than fp32 of the logits: one exp per choice (and
// per expert where they are not normalised), fp32 sums.
// Bound by the vector instructions of the selection, not by memory: 32768 tokens x 256 experts bf16, 8 choices,
// 11.4 us back to back and 13.1 alone, where reading them takes 2.8; fp32, with a ballot and a removal for every choice,
// 18.2 back to back; 16 tokens 3.5 us, one wavefront's time.
template <int DT, int LANES, int PER>
__global__ __launch_bounds__(kRouterWaves * kWave) void router_kernel(const RouterArgs a) {
  using S = typename Elem<DT>::store_t;
  constexpr bool kPacked = sizeof(S) == 2;
  constexpr uint32_t kTokens = kWave / LANES;  // per wavefront
  constexpr int kKept = kWave / LANES;         // choices a lane keeps: member, member + LANES, ...
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
      if constexpr (kPacked) {
        key[j] = order_key16<DT>(upper_half<DT>(l[j]), 0xffffu - (member * PER + j));
      } else {
        key[j] = order_key(l[j]);
      }
      nan |= l[j] != l[j];
    }
    float top = -__builtin_inff();  // the largest logit that can be chosen
    float my_logit[kKept], my_e[kKept];
    int32_t my_id[kKept];
#pragma unroll
    for (int x = 0; x < kKept; ++x) { my_id[x] = -1; my_logit[x] = 0.0f; }
    uint32_t all = 0;  // the key of the last choice
    for (uint32_t k = 0; k < a.topk; ++k) {
      // Packed keys are distinct: the next is the largest key below the last, which is the largest difference to it,
      // as those not below it do not wrap.  (all = 0 at first: the largest key.)
      uint32_t best = kPacked ? key[0] - all : key[0];
#pragma unroll
      for (int j = 1; j < PER; ++j) {
        const uint32_t next = kPacked ? key[j] - all : key[j];
        best = next > best ? next : best;
      }
      const uint32_t largest = group_max<LANES>(best) + (kPacked ? all : 0u);
      all = !kPacked || k == 0 || largest < all ? largest : 0u;
      int32_t id;
      float value;
      if constexpr (kPacked) {
        id = all ? (int32_t)(0xffffu - (all & 0xffffu)) : -1;
        value = logit_of_key16<DT>(all);
      } else {
        int at = 0;
#pragma unroll
        for (int j = PER - 1; j >= 0; --j) at = key[j] == all ? j : at;
        const uint64_t have = __ballot(best == all) & mine;
        const uint32_t owner = (uint32_t)__builtin_ctzll(have);
        const int place = LANES == 64 ? __builtin_amdgcn_readlane(at, owner) : __shfl(at, (int)owner);
        id = all ? (int32_t)((owner % LANES) * PER + place) : -1;
        value = bits_to_f32((all & 0x80000000u) ? all ^ 0x80000000u : ~all);
        const int gone = lane == owner ? at : -1;
#pragma unroll
        for (int j = 0; j < PER; ++j) key[j] = j == gone ? 0u : key[j];
      }
      if (k == 0 && all) top = value;
#pragma unroll
      for (int x = 0; x < kKept; ++x)
        if (k == member + x * LANES) { my_id[x] = id; my_logit[x] = value; }
    }
    float total = 0.0f;
#pragma unroll
    for (int x = 0; x < kKept; ++x) {
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
      for (int x = 0; x < kKept; ++x) {
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
// LANES lanes per token as in router_kernel; what the chosen experts get goes through LDS to the lanes that
// write it.  p is made again from the logits, which costs less than keeping it: 32768 tokens x 256 experts bf16
// 11.2 us back to back for 36 MB (3.2 TB/s) and 9.8 alone, not normalised fp32 14.1 us for 69 MB (4.9 TB/s).  Normalised,
// all logits are read for a NaN alone, which makes the weights NaN wherever it stands (10.2 us if only the chosen are).
template <int DT, int LANES, int PER>
__global__ __launch_bounds__(kRouterWaves * kWave) void router_grad_kernel(const RouterArgs a) {
  using S = typename Elem<DT>::store_t;
  constexpr uint32_t kTokens = kWave / LANES;
  constexpr int kKept = kWave / LANES;
  constexpr int VE = PER < vec_elems<DT>() ? PER : vec_elems<DT>();
  typedef S vec __attribute__((ext_vector_type(VE)));
  typedef vec vec_unaligned __attribute__((aligned(sizeof(S))));
  __shared__ float space[kRouterWaves][kWave * PER];
  const uint32_t lane = threadIdx.x % kWave, member = lane % LANES, group = lane / LANES;
  // Where expert j of a lane lies in its group's space: a lane's few in one vector, more of them across the
  // lanes, so that the lanes' accesses fall into different banks.
  constexpr bool kAcross = PER > 4;
  float* chosen = space[threadIdx.x / kWave] + group * (LANES * PER);
  const auto at = [](uint32_t who, uint32_t j) { return kAcross ? j * LANES + who : who * PER + j; };
  const uint32_t step = gridDim.x * kRouterWaves * kTokens;
  for (uint32_t t0 = (blockIdx.x * kRouterWaves + threadIdx.x / kWave) * kTokens; t0 < a.tokens; t0 += step) {
    const uint32_t t = t0 + group < a.tokens ? t0 + group : a.tokens - 1;  // the last token again: not stored
    const S* row = (const S*)a.logits + (size_t)t * a.experts;
    int32_t id[kKept];
    float g[kKept], value[kKept], w[kKept];
#pragma unroll
    for (int x = 0; x < kKept; ++x) {
      const uint32_t k = member + x * LANES;
      id[x] = -1;
      g[x] = 0.0f;
      value[x] = -__builtin_inff();
      if (k < a.topk) {
        id[x] = a.chosen[(size_t)t * a.topk + k];
        g[x] = a.grad_weights[(size_t)t * a.topk + k];
        if (id[x] < 0 || (uint32_t)id[x] >= a.experts) { id[x] = -1; g[x] = 0.0f; }
        if (id[x] >= 0) value[x] = Elem<DT>::load(row[id[x]]);
      }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) chosen[at(member, j)] = 0.0f;
    float p[PER];
    load_logits<DT, PER>(row, member * PER, a.experts, p);
    float top = -__builtin_inff(), total = 0.0f;
    if (a.normalize) {
#pragma unroll
      for (int x = 0; x < kKept; ++x) top = value[x] > top ? value[x] : top;
      top = group_max<LANES>(top);
#pragma unroll
      for (int x = 0; x < kKept; ++x) total += id[x] >= 0 ? expf(value[x] - top) : 0.0f;
      bool nan = false;
#pragma unroll
      for (int j = 0; j < PER; ++j) nan |= p[j] != p[j];
      if (nan) total = __builtin_nanf("");  // of a row that holds one the weights are NaN, whatever was chosen
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) top = p[j] > top ? p[j] : top;
      top = group_max<LANES>(top);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        p[j] = member * PER + j < a.experts ? expf(p[j] - top) : 0.0f;
        total += p[j];
      }
    }
    total = group_sum<LANES>(total);
    const bool none = top == -__builtin_inff();  // nothing could be chosen: no gradient
    float mean = 0.0f;
#pragma unroll
    for (int x = 0; x < kKept; ++x) {
      w[x] = id[x] >= 0 && !none ? expf(value[x] - top) / total : 0.0f;
      mean += g[x] * w[x];
    }
    mean = group_sum<LANES>(mean);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    // an expert that is named more than once gets every share
#pragma unroll
    for (int x = 0; x < kKept; ++x)
      if (id[x] >= 0) atomicAdd(&chosen[at((uint32_t)id[x] / PER, (uint32_t)id[x] % PER)], a.normalize ? w[x] * (g[x] - mean) : w[x] * g[x]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const float share = mean / total;
    S r[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const float own = chosen[at(member, j)];
      r[j] = Elem<DT>::store(a.normalize || none ? own : own - p[j] * share);
    }
    if (t0 + group < a.tokens) {
      S* out = (S*)a.grad_logits + (size_t)t * a.experts + member * PER;
      if (member * PER + PER <= a.experts) {
#pragma unroll
        for (int b = 0; b < PER; b += VE) {
          vec v;
#pragma unroll
          for (int j = 0; j < VE; ++j) v[j] = r[b + j];
          *(vec_unaligned*)(out + b) = v;
        }
      } else {
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (member * PER + j < a.experts) out[j] = r[j];
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

}  // namespace
