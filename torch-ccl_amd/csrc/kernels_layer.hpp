// A whole mixture-of-experts layer for a few tokens (no kernel of the reference): every expert that a token of
// the batch was routed to is read once for up to 32 of its tokens (its second product: 16), or for up to 128 where
// tokens go through LDS.
#pragma once

#include "kernels_common.hpp"

namespace {

constexpr int kLayerMaxTokens = 256;
constexpr int kLayerMaxPairs = 4096;
constexpr uint32_t kFewMaxPairs = 2048;  // of layer_in_kernel and layer_out_kernel

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// 16 x 16 += (16 x 32) . (32 x 16): lane l holds 8 values of row (column) l % 16, from 8 * (l / 16) on of the
// 32, and gets rows 4 * (l / 16) .. + 3 of column l % 16.
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
  char* h;              // workspace [2][pairs][inter]: the high, then the low parts
  float* y;             // workspace [parts][pairs][hidden], where the products of a pair meet in memory
  char* out;
  uint32_t tokens, topk, pairs, experts, hidden, inter;
  int64_t first_expert;
  int by_pair;          // the slots of layer_in_kernel are pairs (fewer than experts) instead of experts
  int activation;
  uint32_t parts;       // the second product: parts of inter that are work of their own
};

// The wavefront's number in its workgroup, as a value that the compiler knows to be the same for all lanes.
__device__ __forceinline__ uint32_t wave_index() { return (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave)); }

// The expert of a pair among this rank's, or -1.
__device__ __forceinline__ int local_expert(const LayerArgs& a, uint32_t pair) {
  const uint64_t e = (uint64_t)(int64_t)a.ids[pair] - (uint64_t)a.first_expert;
  return e < a.experts ? (int)(uint32_t)e : -1;
}

__device__ __forceinline__ float activate(float v, int activation) {
  if (activation == MCCL_ACT_SILU) return v / (1.0f + expf(-v));
  return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
}

// ------------------------------------------------------------------------------------------
// what the second product takes
// ------------------------------------------------------------------------------------------
// h = act(gate) * up is an fp32 value, and the second product's matrix instructions take 16 bits.  Rounded to the
// layer's type, it made the result's error 1.4 times that of its own last rounding (0.0024 against 0.0017 in bf16), and
// in f16 infinite above 65504.  So h is kept as the sum of two bf16: its upper 8 significant bits as they are, and what they leave,
// rounded: 2^-16 of h at the most, over fp32's range.  The second product adds the products of both parts.
// Where nothing is left (h has 8 bits, or is infinite) the low part is the smallest normal number of h's sign, 2^-126, so
// that an infinite weight meets no zero that h does not have; from 2^-110 on that is below 2^-16 of h as well, and
// smaller ones are left as they are.
// That costs nothing for up to 4 pairs of an expert (1 token 36.4 us for the layer with and without, 32 tokens on an
// expert-parallel shard 213 and 212) and up to a tenth for more in bf16 (64 tokens on 128 experts 322 and 302, 160 on 8
// wide ones 307 and 287); the f16 weights' split a few percent more.
struct Parts {
  uint16_t high, low;
};
__device__ __forceinline__ Parts split(float h) {
  const uint32_t bits = f32_to_bits(h), high = bits >> 16;
  const float rest = h - bits_to_f32(high << 16);
  const uint32_t least = (high & 0x8000u) | ((high & 0x7fffu) >= (127u - 110u) << 7 ? 0x0080u : 0u);
  return {(uint16_t)high, rest < 0.0f || rest > 0.0f ? Elem<MCCL_BF16>::store(rest) : (uint16_t)least};
}

// f16 weights for the products with such parts: 8 values as the sum of two bf16, exactly (8 and 3 significant bits).
// An infinite weight leaves 256 instead of infinity - infinity.
__device__ __forceinline__ uint32_t bf16_pair(f16x2 v) {  // of values that bf16 has
  return __builtin_amdgcn_perm(f32_to_bits((float)v[1]), f32_to_bits((float)v[0]), 0x07060302u);
}
__device__ __forceinline__ void split_f16(const u32x4& w, u32x4& high, u32x4& low) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t pair = w[i], upper_bits = pair & 0xfff8fff8u;
    const f16x2 all = __builtin_bit_cast(f16x2, pair), upper = __builtin_bit_cast(f16x2, upper_bits);
    high[i] = bf16_pair(upper);
    low[i] = bf16_pair(__builtin_elementwise_min(all - upper, (f16x2){(_Float16)256.0f, (_Float16)256.0f}));
  }
}

// c += weights . parts
template <int DT>
__device__ __forceinline__ f32x4 mfma_parts(u32x4 w, u32x4 parts, f32x4 c) {
  if constexpr (DT == MCCL_BF16) {
    return mfma_16x16x32<MCCL_BF16>(w, parts, c);
  } else {
    u32x4 high, low;
    split_f16(w, high, low);
    return mfma_16x16x32<MCCL_BF16>(high, parts, mfma_16x16x32<MCCL_BF16>(low, parts, c));
  }
}

// ------------------------------------------------------------------------------------------
// products of 8 weight rows with 8 tokens
// ------------------------------------------------------------------------------------------
// The matrix instruction takes 16 rows of 32 columns: given 16 weight rows, a load would read 64 bytes
// of each, half a cache line, with every lane in another row than its neighbours.  Here its rows are 8
// weight rows twice, the odd ones for other columns than the even ones, and its columns 8 tokens twice
// likewise: a load reads 128 bytes of each of 8 rows, two lanes next to each other at a time.  Of each
// 2 x 2 block of the result the diagonal is used, the products of the two halves, and the rest is not:
// twice the matrix instructions, of which these kernels have far too few to matter.
constexpr int kSetRows = 8;
constexpr int kStepCols = 64;

// This lane's weight row, and token, of a set of 8, and where in a step's 64 columns its 8 values lie.
__device__ __forceinline__ uint32_t lane_member() { return (threadIdx.x % 16) / 2; }
__device__ __forceinline__ uint32_t lane_column() { return (threadIdx.x % 2 + (threadIdx.x % kWave) / 16 * 2) * 8; }

// Where the sums are, once add_halves has been called: rows lane_row() and lane_row() + 1 of token
// lane_member(), in even lanes.
__device__ __forceinline__ uint32_t lane_row() { return (threadIdx.x % kWave) / 16 * 2; }
__device__ __forceinline__ bool lane_holds() { return threadIdx.x % 2 == 0; }
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <int CTRL = 0xb1>  // lanes 1 0 3 2
__device__ __forceinline__ float from_neighbour(float v) {
  return bits_to_f32((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f32_to_bits(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ f32x2 add_halves(f32x4 v) { return (f32x2){v[0] + from_neighbour(v[1]), v[2] + from_neighbour(v[3])}; }

// Rows and tokens are read through buffer descriptors: the base is the same for all lanes, a lane has a
// 32-bit offset, and an offset with kOutside added reads zeros without touching memory, which is how columns
// that do not exist are left out without a branch.  A matrix and what the last turn of a loop asks for behind
// it stay below kOutside, so that no sum of offsets passes 32 bits.
constexpr uint32_t kOutside = 0x80000000u;
constexpr size_t kLayerMaxColumns = 1u << 17;          // hidden and inter: 4096 pairs of a part of h are 1 GiB
constexpr size_t kLayerMaxExpert = kOutside - 65536u;  // bytes of an expert's w_in
constexpr int kStreamed = 2;  // non-temporal: weights are not read again soon

__device__ __forceinline__ __amdgpu_buffer_rsrc_t matrix_at(const char* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, (int)bytes, 0x00020000);
}

// acc[w][t] += rows . tokens over the steps [s0, s1) below column `depth`: this lane's rows lie w[...] bytes into
// `rows`, its tokens b[...] into `tokens`, both at the lane's column.  The loads of STEPS steps are issued
// before the first product.
// PARTS: the tokens are rows of h.
template <int DT, bool PARTS, int NW, int NT, int STEPS>
__device__ __forceinline__ void multiply_sets(__amdgpu_buffer_rsrc_t rows, const uint32_t (&w)[NW], __amdgpu_buffer_rsrc_t tokens,
                                              const uint32_t (&b)[NT], uint32_t s0, uint32_t s1, uint32_t depth, f32x4 (&acc)[NW][NT]) {
  const uint32_t end = s1 * kStepCols < depth ? s1 * kStepCols : depth, col = lane_column();
  for (uint32_t s = s0; s < s1; s += STEPS) {
    u32x4 wv[STEPS][NW], bv[STEPS][NT];
#pragma unroll
    for (int u = 0; u < STEPS; ++u) {
      const uint32_t k = (s + u) * kStepCols;
      const uint32_t out = k + col < end ? 0 : kOutside;  // columns, depth: multiples of 8, so all 8 or none
#pragma unroll
      for (int n = 0; n < NT; ++n) bv[u][n] = __builtin_amdgcn_raw_buffer_load_b128(tokens, b[n] | out, k * 2, 0);
#pragma unroll
      for (int n = 0; n < NW; ++n) wv[u][n] = __builtin_amdgcn_raw_buffer_load_b128(rows, w[n] | out, k * 2, kStreamed);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < STEPS; ++u)
#pragma unroll
      for (int n = 0; n < NW; ++n)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[n][t] = PARTS ? mfma_parts<DT>(wv[u][n], bv[u][t], acc[n][t]) : mfma_16x16x32<DT>(wv[u][n], bv[u][t], acc[n][t]);
  }
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t w_in_of(const LayerArgs& a, int e) {
  const uint32_t bytes = 4 * a.inter * a.hidden;  // at most kLayerMaxExpert
  return matrix_at(a.w_in + (size_t)e * bytes, bytes);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t w_out_of(const LayerArgs& a, int e) {
  const uint32_t bytes = 2 * a.inter * a.hidden;
  return matrix_at(a.w_out + (size_t)e * bytes, bytes);
}

// The experts of all pairs into LDS: the lists are made from there, at an LDS round trip for every 64 pairs
// instead of one to memory.  Ends with a barrier.
__device__ __forceinline__ void stage_experts(const LayerArgs& a, int16_t* expert) {
  for (uint32_t p = threadIdx.x; p < a.pairs; p += blockDim.x) expert[p] = (int16_t)local_expert(a, p);
  __syncthreads();
}

// The next pairs of expert e in ascending order into `list`, from pair `from` on: at least kListPairs of them
// if there are as many, at most kListSpace; returns how many and leaves in `from` where to go on.  Every
// wavefront lists for itself (several that share the space write the same values).
constexpr uint32_t kListPairs = 64;
constexpr uint32_t kListSpace = kListPairs + kWave;

__device__ __forceinline__ uint32_t list_pairs(const int16_t* expert, uint32_t pairs, int e, uint32_t& from, uint16_t* list) {
  const uint32_t lane = threadIdx.x % kWave;
  uint32_t m = 0;
  for (; from < pairs && m < kListPairs; from += kWave) {
    const bool mine = from + lane < pairs && expert[from + lane] == e;
    const uint64_t set = __ballot(mine);
    if (mine) list[m + __popcll(set & ((1ull << lane) - 1))] = (uint16_t)(from + lane);
    m += (uint32_t)__popcll(set);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  return m;
}

// ------------------------------------------------------------------------------------------
// h[pair][i] = act(w_in[e][i] . x[t]) * (w_in[e][inter + i] . x[t])
// ------------------------------------------------------------------------------------------
// A workgroup takes 16 gate rows and their 16 up rows of one expert; its wavefronts share the columns, in fp32 until
// the gate is applied, and h leaves in two parts.
// Bound by reading the weights: 15.7 experts of 7168 x 2048, 32 tokens, 132 us, 7.0 TB/s; 8 experts of 4096 x 1024,
// 1 token, 23 us, 5.9 TB/s (a workgroup reads 256 KiB there, and its start and end are a fifth of its time).
// 8 and 16 wavefronts a workgroup, two halves of the loads in turns, and 4 workgroups a compute unit by fewer registers
// are no faster (1 token 36.0, 37.8, 36.4 and 36.0 us for the layer; 32 tokens 214, 228, 230 and 225 against 211).
constexpr int kInWaves = 4;
constexpr int kInRows = 2 * kSetRows;

template <int DT, int NT, int STEPS>
__device__ __forceinline__ void layer_in_tokens(const LayerArgs& a, int e, uint32_t i0, const uint16_t* list, uint32_t m0, uint32_t m,
                                                float (*sums)[4][NT][8][8]) {
  const uint32_t wave = wave_index();
  const uint32_t r = lane_member(), col = lane_column();
  uint32_t w[4], b[NT];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const uint32_t i = i0 + (n % 2) * kSetRows + r;
    w[n] = (((i < a.inter ? i : a.inter - 1) + (n / 2) * a.inter) * a.hidden + col) * 2;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const uint32_t mine = m0 + t * 8 + r;
    b[t] = ((list[mine < m ? mine : m - 1] / a.topk) * a.hidden + col) * 2;
  }
  f32x4 acc[4][NT];
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[n][t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  const uint32_t steps = (a.hidden + kStepCols - 1) / kStepCols, per = (steps + kInWaves - 1) / kInWaves;
  const uint32_t s0 = wave * per, s1 = s0 + per < steps ? s0 + per : steps;
  multiply_sets<DT, false, 4, NT, STEPS>(w_in_of(a, e), w, matrix_at(a.x, a.tokens * a.hidden * 2), b, s0, s1, a.hidden, acc);
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const f32x2 v = add_halves(acc[n][t]);
      if (lane_holds()) *(f32x2*)&sums[wave][n][t][r][lane_row()] = v;
    }
  __syncthreads();
  for (uint32_t o = threadIdx.x; o < NT * 8 * kInRows; o += kInWaves * kWave) {
    const uint32_t row = o % kInRows, token = o / kInRows;
    if (m0 + token >= m || i0 + row >= a.inter) continue;
    float g = 0.0f, u = 0.0f;
#pragma unroll
    for (int p = 0; p < kInWaves; ++p) {
      g += sums[p][row / 8][token / 8][token % 8][row % 8];
      u += sums[p][2 + row / 8][token / 8][token % 8][row % 8];
    }
    const Parts h = split(activate(g, a.activation) * u);
    uint16_t* at = (uint16_t*)a.h + (size_t)list[m0 + token] * a.inter + i0 + row;
    at[0] = h.high;
    at[(size_t)a.pairs * a.inter] = h.low;
  }
  __syncthreads();
}

// TOKENS bounds how many tokens one reading of the weights serves (and with it the registers).
template <int DT, int TOKENS>
__global__ __launch_bounds__(kInWaves * kWave) void layer_in_kernel(const LayerArgs a) {
  __shared__ int16_t expert[kFewMaxPairs];
  __shared__ uint16_t list[kListSpace];
  __shared__ float sums[kInWaves * 4 * (TOKENS / 8) * 64];
  stage_experts(a, expert);
  const int e = a.by_pair ? __builtin_amdgcn_readfirstlane(expert[blockIdx.y]) : (int)blockIdx.y;
  if (e < 0) return;
  const uint32_t i0 = blockIdx.x * kInRows;
  for (uint32_t from = 0; from < a.pairs;) {
    const bool begins = from == 0;
    const uint32_t m = list_pairs(expert, a.pairs, e, from, list);
    if (begins && a.by_pair && (m == 0 || list[0] != blockIdx.y)) return;  // of the pairs of an expert the first one works
    uint32_t m0 = 0;
    if constexpr (TOKENS >= 32)
      for (; m0 < m && m - m0 > 16; m0 += 32) layer_in_tokens<DT, 4, 1>(a, e, i0, list, m0, m, (float (*)[4][4][8][8])sums);
    if constexpr (TOKENS >= 16)
      for (; m0 < m && m - m0 > 8; m0 += 16) layer_in_tokens<DT, 2, 2>(a, e, i0, list, m0, m, (float (*)[4][2][8][8])sums);
    for (; m0 < m; m0 += 8) layer_in_tokens<DT, 1, 4>(a, e, i0, list, m0, m, (float (*)[4][1][8][8])sums);
  }
}

// ------------------------------------------------------------------------------------------
// out[t][c] = sum_k weights[t][k] * (w_out[e][c] . h[t * topk + k])
// ------------------------------------------------------------------------------------------
// A workgroup takes kSetRows * NW rows of w_out of every expert that was chosen and keeps the products of
// all pairs in LDS, so that the weighted sum needs no other workgroup: work of a wavefront is an expert
// and one of a.parts parts of inter.  Sums in fp32, the pairs of a token in ascending order, one rounding.
// Bound by reading the weights: 15.7 experts of 7168 x 2048, 32 tokens, 74 us, 6.3 TB/s; 8 of 4096 x 1024, 1 token,
// 14 us, 4.7 TB/s; from 5 pairs of an expert on h's reads, which every workgroup makes for its 8 or 16 rows, are as many as
// the weights'; below some 20 MB by its chain: ids, lists, h, products, sums (10 experts of 520 x 200 f16 6.2 us).
struct LayerOutLds {
  uint32_t weights, first, active, lists, y, bytes;
};
__host__ __device__ inline LayerOutLds layer_out_lds(uint32_t pairs, uint32_t experts, uint32_t parts, uint32_t rows, uint32_t waves) {
  LayerOutLds l;
  const uint32_t p8 = (pairs + 7) / 8 * 8;
  l.weights = p8 * 2;                           // the experts of the pairs come first, int16
  l.first = l.weights + p8 * 4;                 // their weights, fp32
  l.active = l.first + (experts + 3) / 4 * 16;  // first pair of every expert, uint32
  l.lists = l.active + p8 * 2;                  // first pairs of the chosen experts, uint16
  l.y = l.lists + waves * kListSpace * 2;       // a list per wavefront, uint16
  l.bytes = l.y + pairs * parts * rows * 4;
  return l;
}

// The 8 tokens of a set are the high and the low parts of 4 pairs, next to each other.
constexpr int kSetPairs = 4;

template <int DT, int NW, int NT, int STEPS>
__device__ __forceinline__ void layer_out_tokens(const LayerArgs& a, int e, uint32_t c0, uint32_t part, const uint16_t* list, uint32_t m0,
                                                 uint32_t m, float* y) {
  const uint32_t r = lane_member(), col = lane_column();
  uint32_t w[NW], b[NT];
#pragma unroll
  for (int n = 0; n < NW; ++n) {
    const uint32_t row = c0 + n * kSetRows + r;
    w[n] = ((row < a.hidden ? row : a.hidden - 1) * a.inter + col) * 2;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const uint32_t mine = m0 + t * kSetPairs + r / 2;
    b[t] = ((list[mine < m ? mine : m - 1] + r % 2 * a.pairs) * a.inter + col) * 2;
  }
  f32x4 acc[NW][NT];
#pragma unroll
  for (int n = 0; n < NW; ++n)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[n][t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  const uint32_t steps = (a.inter + kStepCols - 1) / kStepCols, per = (steps + a.parts - 1) / a.parts;
  const uint32_t s0 = part * per, s1 = s0 + per < steps ? s0 + per : steps;
  multiply_sets<DT, true, NW, NT, STEPS>(w_out_of(a, e), w, matrix_at(a.h, a.pairs * a.inter * 4), b, s0, s1, a.inter, acc);
#pragma unroll
  for (int n = 0; n < NW; ++n)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      f32x2 v = add_halves(acc[n][t]);
#pragma unroll
      for (int i = 0; i < 2; ++i) v[i] += from_neighbour<0x4e>(v[i]);  // lanes 2 3 0 1: the other part
      const uint32_t mine = m0 + t * kSetPairs + r / 2;
      if (threadIdx.x % 4 == 0 && mine < m)
        *(f32x2*)(y + (((size_t)list[mine] * a.parts + part) * NW + n) * kSetRows + lane_row()) = v;
    }
}

template <int DT, int NW, int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void layer_out_kernel(const LayerArgs a) {
  using S = typename Elem<DT>::store_t;
  constexpr uint32_t kRows = NW * kSetRows;
  extern __shared__ char lds[];
  const LayerOutLds l = layer_out_lds(a.pairs, a.experts, a.parts, kRows, WAVES);
  int16_t* expert = (int16_t*)lds;
  float* weight = (float*)(lds + l.weights);
  uint32_t* first = (uint32_t*)(lds + l.first);
  uint16_t* active = (uint16_t*)(lds + l.active);
  float* y = (float*)(lds + l.y);
  const uint32_t lane = threadIdx.x % kWave, wave = wave_index();
  uint16_t* list = (uint16_t*)(lds + l.lists) + wave * kListSpace;
  for (uint32_t p = threadIdx.x; p < a.pairs; p += WAVES * kWave) weight[p] = a.weights[p];
  for (uint32_t e = threadIdx.x; e < a.experts; e += WAVES * kWave) first[e] = ~0u;
  stage_experts(a, expert);
  for (uint32_t p = threadIdx.x; p < a.pairs; p += WAVES * kWave)
    if (expert[p] >= 0) atomicMin(&first[expert[p]], p);
  __syncthreads();
  uint32_t chosen = 0;  // every wavefront lists the first pairs, all with the same result
  for (uint32_t p0 = 0; p0 < a.pairs; p0 += kWave) {
    const uint32_t p = p0 + lane;
    const bool leads = p < a.pairs && expert[p] >= 0 && first[expert[p]] == p;
    const uint64_t set = __ballot(leads);
    if (leads) active[chosen + __popcll(set & ((1ull << lane) - 1))] = (uint16_t)p;
    chosen += (uint32_t)__popcll(set);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const uint32_t c0 = blockIdx.x * kRows, work = chosen * a.parts;
  for (uint32_t i = wave; i < work; i += WAVES) {
    const uint32_t part = i % a.parts;
    uint32_t from = __builtin_amdgcn_readfirstlane(active[i / a.parts]);
    const int e = __builtin_amdgcn_readfirstlane(expert[from]);
    from = from / kWave * kWave;
    while (from < a.pairs) {
      const uint32_t m = list_pairs(expert, a.pairs, e, from, list);
      uint32_t m0 = 0;
      for (; m0 < m && m - m0 > 8; m0 += 16) layer_out_tokens<DT, NW, 4, 2>(a, e, c0, part, list, m0, m, y);
      for (; m0 < m && m - m0 > 4; m0 += 8) layer_out_tokens<DT, NW, 2, 4>(a, e, c0, part, list, m0, m, y);
      for (; m0 < m; m0 += 4) layer_out_tokens<DT, NW, 1, 8 / NW>(a, e, c0, part, list, m0, m, y);
    }
  }
  __syncthreads();
  for (uint32_t o = threadIdx.x; o < a.tokens * kRows; o += WAVES * kWave) {
    const uint32_t t = o / kRows, c = o % kRows;
    if (c0 + c >= a.hidden) continue;
    float sum = 0.0f;
    for (uint32_t k = 0; k < a.topk; ++k) {
      const uint32_t p = t * a.topk + k;
      if (expert[p] < 0) continue;
      float v = 0.0f;
      for (uint32_t q = 0; q < a.parts; ++q) v += y[(p * a.parts + q) * kRows + c];
      sum += weight[p] * v;
    }
    ((S*)a.out)[(size_t)t * a.hidden + c0 + c] = Elem<DT>::store(sum);
  }
}

// ------------------------------------------------------------------------------------------
// many tokens per expert
// ------------------------------------------------------------------------------------------
// The same products where an expert has so many tokens that reading them again for every 16 rows costs
// more than the weights.  A tile is 8 wavefronts x 2 sets of rows of an expert, over all of hidden (first
// product: 64 gate rows and their up rows) or one part of inter (second product: 128 rows).  Its tokens go
// through LDS, a chunk of columns of 128 of them at a time.  While a chunk is multiplied, the rows and tokens of the
// next one are on their way into registers.
// 160 tokens on 8 experts of 4096 x 7168 f16, 40 each: 192 us for the first product (4.9 TB/s, 196 TFLOP/s) and 143 for
// the second (3.3 TB/s); 96 tokens on each of 2 experts of 4096 x 8192 bf16 122 us in all.  Two workgroups fit on a
// compute unit by registers (128) and LDS (80 KiB); with the products of few tokens, half of whose sums are not used,
// it was one and the layer took a tenth longer.
// What is lost is a workgroup's start and end, the join, and in the second product the turns, whose tokens are twice
// the bytes.  A workgroup that goes on to its next tile by itself, loads three chunks ahead, and 4 wavefronts instead of
// 8 were slower; a first product with tiles of 64 tokens is 1 or 2 percent faster or 4 slower below 64 tokens an
// expert and reads the weights twice above.
constexpr int kDenseWaves = 8;
constexpr int kDenseBlock = kDenseWaves * kWave;
constexpr uint32_t kDenseInRows = kDenseWaves * kSetRows, kDenseOutRows = 2 * kDenseInRows;

// With 16 tokens to a product the matrix instruction is used in full: its 16 rows are the wavefront's two sets of 8,
// the even ones of the first.  The rows are still loaded by lane pairs, 128 bytes of each, of which a lane has one
// 16-byte piece of a row of either set; the pair exchanges what the other's row needs, and each has two pieces of one
// row: columns of two products.
__device__ __forceinline__ void exchange_sets(const u32x4& first, const u32x4& second, u32x4& even, u32x4& odd) {
  const bool takes_first = threadIdx.x % 2 == 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t got = f32_to_bits(from_neighbour(bits_to_f32(takes_first ? second[i] : first[i])));
    even[i] = takes_first ? first[i] : got;
    odd[i] = takes_first ? got : second[i];
  }
}

// How the tokens of a turn, up to a barrier, lie in LDS: 32 KiB of them, twice.
//   first product            128 tokens of 128 columns
//   second, up to 64 pairs    64 pairs of 128 columns in both parts
//   second, more             128 pairs of 64 columns in both parts: a chunk of weights takes two turns
// The last form costs more where it is not needed (16 pairs on each of 8 experts of 4096 x 1792 81 us for the layer against
// 87): a turn is no shorter than a load of tokens takes, whatever it multiplies.  Tiles of 64 alone read the weights twice
// for 65 pairs (160 tokens on 8 experts of 4096 x 7168 356 us against 325).
constexpr int kDenseTokens = 128;  // of a tile
constexpr int kDenseSteps = 2;     // of 64 columns in a chunk of weights
constexpr int kDenseShare = 4;     // 16-byte pieces of tokens that one thread stages per turn

template <bool IN, int TOKENS>
struct Staging {
  static constexpr int kGroups = TOKENS / 16;                                    // of a product's tokens
  static constexpr int kParts = IN ? 1 : 2;                                      // of a token that are staged
  static constexpr int kSteps = 128 * kDenseSteps / (kParts * TOKENS);           // of a turn
  static constexpr int kTurns = kDenseSteps / kSteps;                            // of a chunk
  static constexpr int kPieces = kSteps * 8;                                     // of a token's row, side by side
  static constexpr int kApart = kDenseBlock / kPieces;                           // tokens from one of a thread's to its next
  static constexpr uint32_t kCols = kSteps * kStepCols, kRowBytes = kCols * 2 * kParts;
  static_assert(TOKENS * kRowBytes == 32 * 1024 && kDenseShare * kApart == TOKENS * kParts, "LDS and threads are filled");
};

template <int DT, bool IN>
__global__ __launch_bounds__(kDenseBlock, 4) void layer_dense_kernel(const LayerArgs a) {
  constexpr uint32_t kCols = kDenseSteps * kStepCols;
  __shared__ __align__(16) char space[2][32 * 1024];  // the tokens of two turns
  __shared__ int16_t expert[kLayerMaxPairs];
  __shared__ uint16_t list[kLayerMaxPairs];
  const uint32_t wave = wave_index(), r = lane_member(), col = lane_column();
  const uint32_t depth = IN ? a.hidden : a.inter, nrows = IN ? a.inter : a.hidden;
  const uint32_t chunks = (depth + kCols - 1) / kCols, per = IN ? chunks : (chunks + a.parts - 1) / a.parts;
  const uint32_t row_tiles = (nrows + (IN ? kDenseInRows : kDenseOutRows) - 1) / (IN ? kDenseInRows : kDenseOutRows);

  // The tile: neighbouring workgroups take neighbouring rows of one expert, which share its tokens.
  const uint32_t rest = blockIdx.x / row_tiles, part = IN ? 0 : rest / a.experts, e = rest - part * a.experts;
  const uint32_t row0 = (blockIdx.x - rest * row_tiles) * (IN ? kDenseInRows : kDenseOutRows) + wave * (IN ? 1 : 2) * kSetRows;
  uint32_t w[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const uint32_t row = row0 + (IN ? 0 : n * kSetRows) + r;
    w[n] = (((row < nrows ? row : nrows - 1) + (IN ? n * a.inter : 0)) * depth + col) * 2;
  }
  const uint32_t c0 = part * per, c1 = c0 + per < chunks ? c0 + per : chunks;
  const uint32_t end = c1 * kCols < depth ? c1 * kCols : depth;
  const __amdgpu_buffer_rsrc_t rows = IN ? w_in_of(a, (int)e) : w_out_of(a, (int)e);
  // Columns from `end` on (whole chunks too) are outside and not read.
  const auto load_rows = [&](uint32_t c, u32x4(&v)[kDenseSteps][2]) {
#pragma unroll
    for (int u = 0; u < kDenseSteps; ++u) {
      const uint32_t k = c * kCols + u * kStepCols, out = k + col < end ? 0 : kOutside;
#pragma unroll
      for (int n = 0; n < 2; ++n) v[u][n] = __builtin_amdgcn_raw_buffer_load_b128(rows, w[n] | out, k * 2, kStreamed);
    }
  };
  const uint32_t h_bytes = a.pairs * a.inter * 2;
  const __amdgpu_buffer_rsrc_t tokens[2] = {IN ? matrix_at(a.x, a.tokens * a.hidden * 2) : matrix_at(a.h, h_bytes), matrix_at(a.h + h_bytes, h_bytes)};
  const uint32_t token = threadIdx.x % 16;  // of 16, where the sums are too

  stage_experts(a, expert);
  uint32_t m = 0, turns = 0;
  for (uint32_t from = 0; from < a.pairs;) m += list_pairs(expert, a.pairs, (int)e, from, list + m);

  // The products of `used` tokens of the list, from m0 on.
  const auto multiply = [&](auto staging, uint32_t m0, uint32_t used) {
    using G = decltype(staging);
    // Staging: a thread's pieces of its tokens' rows.  The 8 pieces of 128 bytes are stored in an order turned by the
    // token so that the 8 tokens which a load from LDS takes at the same columns lie in different banks.
    uint32_t thread = threadIdx.x;
    asm("" : "+v"(thread));  // the addresses of either form are made where it begins: all of them at once do not fit the registers
    const uint32_t piece = thread % G::kPieces, staged = thread / G::kPieces;
    const uint32_t put = staged * G::kRowBytes + (piece / 8) * 128 + ((piece ^ staged) % 8) * 16;
    const uint32_t get = thread % 16 * G::kRowBytes + ((thread % kWave / 16 * 2) ^ (thread % 8)) * 16;  // its neighbour piece: ^ 16
    uint32_t from[kDenseShare / G::kParts];
#pragma unroll
    for (int i = 0; i < kDenseShare / G::kParts; ++i) {
      const uint32_t at = i * G::kApart + staged, pair = list[m0 + (at < used ? at : 0)];
      from[i] = at < used ? ((IN ? pair / a.topk : pair) * depth + piece * 8) * 2 : kOutside;
    }
    u32x4 wv[2][kDenseSteps][2], tv[kDenseShare];
    const auto load_tokens = [&](uint32_t turn) {
      const uint32_t k = turn * G::kCols, out = k + piece * 8 < end ? 0 : kOutside;
#pragma unroll
      for (int i = 0; i < kDenseShare; ++i) tv[i] = __builtin_amdgcn_raw_buffer_load_b128(tokens[i % G::kParts], from[i / G::kParts] | out, k * 2, 0);
    };
    const auto stage = [&]() {
      char* buf = space[turns & 1];
#pragma unroll
      for (int i = 0; i < kDenseShare; ++i)
        *(u32x4*)(buf + put + i / G::kParts * G::kApart * G::kRowBytes + i % G::kParts * (G::kCols * 2)) = tv[i];
      __syncthreads();
    };
    f32x4 acc[G::kGroups];
#pragma unroll
    for (int g = 0; g < G::kGroups; ++g) acc[g] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    const auto product = [&](const u32x4(&v)[kDenseSteps][2], int turn) {
      const char* buf = space[turns & 1];
      __builtin_amdgcn_sched_barrier(0);  // the loads go first
      // First product: the steps of a turn in turn for every 16 tokens; second: both parts, step by step, as f16 rows are split
      // for a step at a time (both steps at once take more registers than there are).
      constexpr int kAtOnce = IN ? G::kSteps : 1;
#pragma unroll
      for (int u0 = 0; u0 < G::kSteps; u0 += kAtOnce) {
        u32x4 rows_of[kAtOnce][2];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u)
          exchange_sets(v[turn * G::kSteps + u0 + u][0], v[turn * G::kSteps + u0 + u][1], rows_of[u][0], rows_of[u][1]);
#pragma unroll
        for (int g = 0; g < G::kGroups; ++g) {
          if (g * 16u >= used) break;
          u32x4 b[2][2];  // of a step or of a part, and the two pieces
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              b[n][i] = *(const u32x4*)(buf + g * 16 * G::kRowBytes + (IN ? n : n * G::kSteps + u0) * 128 + (get ^ (i * 16)));
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if constexpr (IN) acc[g] = mfma_16x16x32<DT>(rows_of[n][i], b[n][i], acc[g]);
              else acc[g] = mfma_parts<DT>(rows_of[0][i], b[n][i], acc[g]);
            }
        }
      }
      ++turns;
    };
    load_tokens(c0 * G::kTurns);
    load_rows(c0, wv[0]);
    for (uint32_t c = c0; c < c1; c += 2) {
#pragma unroll
      for (int turn = 0; turn < G::kTurns; ++turn) {
        stage();
        load_tokens(c * G::kTurns + turn + 1);
        if (turn == 0) load_rows(c + 1, wv[1]);
        product(wv[0], turn);
      }
#pragma unroll
      for (int turn = 0; turn < G::kTurns; ++turn) {
        if (c + 1 < c1) stage();
        load_tokens((c + 1) * G::kTurns + turn + 1);
        if (turn == 0) load_rows(c + 2, wv[0]);
        if (c + 1 < c1) product(wv[1], turn);
      }
    }
#pragma unroll
    for (int g = 0; g < G::kGroups; ++g) {
      if (g * 16 + token >= used) break;
      // rows 4 * (lane / 16) .. + 3 of the product: of either set two rows
      const f32x2 v0 = {acc[g][0], acc[g][2]}, v1 = {acc[g][1], acc[g][3]};
      const uint32_t pair = list[m0 + g * 16 + token], row = row0 + lane_row();
      if constexpr (IN) {
        if (row < a.inter) {  // inter is a multiple of 8: both rows or none
          uint32_t high = 0, low = 0;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const Parts h = split(activate(v0[c], a.activation) * v1[c]);
            high |= (uint32_t)h.high << (c * 16);
            low |= (uint32_t)h.low << (c * 16);
          }
          char* at = a.h + ((size_t)pair * a.inter + row) * 2;
          *(uint32_t*)at = high;
          *(uint32_t*)(at + h_bytes) = low;
        }
      } else {
        float* y = a.y + ((size_t)part * a.pairs + pair) * a.hidden + row;
        if (row < a.hidden) *(f32x2*)y = v0;
        if (row + kSetRows < a.hidden) *(f32x2*)(y + kSetRows) = v1;
      }
    }
  };

  for (uint32_t m0 = 0; m0 < m; m0 += kDenseTokens) {
    const uint32_t used = m - m0 < kDenseTokens ? m - m0 : kDenseTokens;
    if constexpr (IN) multiply(Staging<true, 128>{}, m0, used);
    else if (used <= 64) multiply(Staging<false, 64>{}, m0, used);
    else multiply(Staging<false, 128>{}, m0, used);
  }
}

// out[t] = sum_k weights[t][k] * (sum over the parts of y[t * topk + k]), ascending.  y comes from the caches: 160 tokens
// x 2 x 4096 5 us, two thirds of it the launch and the ids.
template <int DT>
__global__ __launch_bounds__(256) void layer_join_kernel(const LayerArgs a) {
  using S = typename Elem<DT>::store_t;
  const uint32_t t = blockIdx.y, c = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (c >= a.hidden) return;
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  // Pairs of other ranks' experts are read too (nobody has written their y) and left out: the loads of several
  // pairs are in flight together.
#pragma unroll 4
  for (uint32_t k = 0; k < a.topk; ++k) {
    const uint32_t p = t * a.topk + k;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t q = 0; q < a.parts; ++q) v += *(const f32x4*)(a.y + ((size_t)q * a.pairs + p) * a.hidden + c);
    v = a.weights[p] * v;
    if (local_expert(a, p) >= 0) sum += v;
  }
  union { S e[4]; uint2 v; } r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.e[i] = Elem<DT>::store(sum[i]);
  *(uint2*)((S*)a.out + (size_t)t * a.hidden + c) = r.v;
}

}  // namespace
