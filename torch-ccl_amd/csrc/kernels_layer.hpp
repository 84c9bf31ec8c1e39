// A whole mixture-of-experts layer for a few tokens (no kernel of the reference): every expert that a
// token of the batch was routed to is read once, for all of its tokens.
#pragma once

#include "kernels_common.hpp"

namespace {

constexpr int kLayerMaxTokens = 256;
constexpr int kLayerMaxPairs = 4096;
constexpr int kLayerWaves = 4;
constexpr int kLayerBlock = kLayerWaves * kWave;
constexpr int kLayerRows = 16;  // weight rows per matrix instruction, and tokens

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// 16 x 16 += (16 weight rows x 32) . (32 x 16 tokens): lane l holds 8 consecutive values of row (token)
// l % 16 from column 8 * (l / 16) on, and gets rows 4 * (l / 16) .. + 3 of token l % 16.
template <int DT>
__device__ __forceinline__ f32x4 mfma_16x16x32(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == MCCL_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

struct LayerArgs {
  const char* x;
  const char* w_in;     // [experts][2 * inter][hidden]: gate rows, then up rows
  const char* w_out;    // [experts][hidden][inter]
  const int32_t* ids;   // [tokens][topk]
  const float* weights; // [tokens][topk]
  char* h;              // workspace [pairs][inter]
  float* y;             // workspace [pairs][hidden]
  char* out;
  uint32_t tokens, topk, pairs, experts, hidden, inter;
  int64_t first_expert;
  int by_pair;          // the grid's second axis counts pairs (fewer than experts) instead of experts
  int activation;
};

__device__ __forceinline__ int local_expert(const LayerArgs& a, uint32_t pair) {
  const uint64_t e = (uint64_t)(int64_t)a.ids[pair] - (uint64_t)a.first_expert;
  return e < a.experts ? (int)e : -1;
}

// The expert of this workgroup's slot and the pairs routed to it, ascending; returns how many (0: nothing
// to do).  Where there are fewer pairs than experts a slot is a pair, and only the first pair of an
// expert works.
__device__ __forceinline__ uint32_t collect_pairs(const LayerArgs& a, uint32_t slot, uint16_t* list, uint32_t* counts, int* expert) {
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int e = a.by_pair ? local_expert(a, slot) : (int)slot;
  *expert = e;
  if (e < 0) return 0;
  uint32_t total = 0;
  for (uint32_t p0 = 0; p0 < a.pairs; p0 += kLayerBlock) {
    const uint32_t p = p0 + threadIdx.x;
    const bool mine = p < a.pairs && local_expert(a, p) == e;
    const uint64_t m = __ballot(mine);
    __syncthreads();
    if (lane == 0) counts[wave] = (uint32_t)__popcll(m);
    __syncthreads();
    uint32_t at = total;
    for (uint32_t w = 0; w < wave; ++w) at += counts[w];
    if (mine) list[at + __popcll(m & ((1ull << lane) - 1))] = (uint16_t)p;
    for (uint32_t w = 0; w < kLayerWaves; ++w) total += counts[w];
  }
  __syncthreads();
  if (total == 0 || (a.by_pair && list[0] != slot)) return 0;
  return total;
}

__device__ __forceinline__ float activate(float v, int activation) {
  if (activation == MCCL_ACT_SILU) return v / (1.0f + expf(-v));
  return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
}

// h[pair][i] = act(w_in[e][i] . x[t]) * (w_in[e][inter + i] . x[t]).  A wavefront takes 16 gate rows and
// their 16 up rows over the whole of hidden, 16 tokens at a time.
template <int DT>
__global__ __launch_bounds__(kLayerBlock) void layer_in_kernel(const LayerArgs a) {
  using S = typename Elem<DT>::store_t;
  __shared__ uint16_t list[kLayerMaxPairs];
  __shared__ uint32_t counts[kLayerWaves];
  int e;
  const uint32_t m = collect_pairs(a, blockIdx.y, list, counts, &e);
  if (m == 0) return;
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t r = lane % 16, q = lane / 16;
  const uint32_t i0 = (blockIdx.x * kLayerWaves + wave) * kLayerRows;
  if (i0 >= a.inter) return;
  const uint32_t row = i0 + r < a.inter ? i0 + r : a.inter - 1;
  const S* gate = (const S*)a.w_in + ((size_t)e * 2 * a.inter + row) * a.hidden;
  const S* up = gate + (size_t)a.inter * a.hidden;
  for (uint32_t m0 = 0; m0 < m; m0 += 16) {
    const uint32_t mine = m0 + r < m ? m0 + r : m - 1;
    const uint32_t pair = list[mine];
    const S* x = (const S*)a.x + (size_t)(pair / a.topk) * a.hidden;
    f32x4 cg = {0.0f, 0.0f, 0.0f, 0.0f}, cu = cg;
    for (uint32_t k0 = 0; k0 < a.hidden; k0 += 32) {
      const uint32_t k = k0 + q * 8;
      u32x4 ag = {0u, 0u, 0u, 0u}, au = ag, b = ag;
      if (k < a.hidden) {
        ag = *(const u32x4*)(gate + k);
        au = *(const u32x4*)(up + k);
        b = *(const u32x4*)(x + k);
      }
      cg = mfma_16x16x32<DT>(ag, b, cg);
      cu = mfma_16x16x32<DT>(au, b, cu);
    }
    if (m0 + r < m) {
      S* h = (S*)a.h + (size_t)pair * a.inter;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t i = i0 + q * 4 + c;
        if (i < a.inter) h[i] = Elem<DT>::store(activate(cg[c], a.activation) * cu[c]);
      }
    }
  }
}

// y[pair][c] = w_out[e][c] . h[pair]
template <int DT>
__global__ __launch_bounds__(kLayerBlock) void layer_out_kernel(const LayerArgs a) {
  using S = typename Elem<DT>::store_t;
  __shared__ uint16_t list[kLayerMaxPairs];
  __shared__ uint32_t counts[kLayerWaves];
  int e;
  const uint32_t m = collect_pairs(a, blockIdx.y, list, counts, &e);
  if (m == 0) return;
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t r = lane % 16, q = lane / 16;
  const uint32_t c0 = (blockIdx.x * kLayerWaves + wave) * kLayerRows;
  if (c0 >= a.hidden) return;
  const uint32_t row = c0 + r < a.hidden ? c0 + r : a.hidden - 1;
  const S* w = (const S*)a.w_out + ((size_t)e * a.hidden + row) * a.inter;
  for (uint32_t m0 = 0; m0 < m; m0 += 16) {
    const uint32_t mine = m0 + r < m ? m0 + r : m - 1;
    const uint32_t pair = list[mine];
    const S* h = (const S*)a.h + (size_t)pair * a.inter;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t k0 = 0; k0 < a.inter; k0 += 32) {
      const uint32_t k = k0 + q * 8;
      u32x4 av = {0u, 0u, 0u, 0u}, b = av;
      if (k < a.inter) {
        av = *(const u32x4*)(w + k);
        b = *(const u32x4*)(h + k);
      }
      acc = mfma_16x16x32<DT>(av, b, acc);
    }
    if (m0 + r < m) {
      float* y = a.y + (size_t)pair * a.hidden;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (c0 + q * 4 + c < a.hidden) y[c0 + q * 4 + c] = acc[c];
    }
  }
}

// out[t] = sum_k weights[t][k] * y[t * topk + k], ascending k.
template <int DT>
__global__ __launch_bounds__(256) void layer_join_kernel(const LayerArgs a) {
  using S = typename Elem<DT>::store_t;
  const uint32_t t = blockIdx.y, c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.hidden) return;
  float acc = 0.0f;
  for (uint32_t k = 0; k < a.topk; ++k) {
    const uint32_t p = t * a.topk + k;
    if (local_expert(a, p) >= 0) acc += a.weights[p] * a.y[(size_t)p * a.hidden + c];
  }
  ((S*)a.out)[(size_t)t * a.hidden + c] = Elem<DT>::store(acc);
}

}  // namespace
