// Embedding lookup of a vocabulary shard, the sort of its tokens by row, and its gradient by sorted
// tokens (no kernel of the reference: the callers' steps before an all_reduce of vocabulary-sharded
// activations, and before and after the exchange of routed tokens).
#pragma once

#include "kernels_common.hpp"

namespace {

// ------------------------------------------------------------------------------------------
// rows of any length: a row is cut into 16-byte vectors of the storage type, the last one may be short
// ------------------------------------------------------------------------------------------
// Vectors are read and written at whatever alignment they have (legal for global memory on this
// target); `left` is how many elements of the row there are from this vector on.
template <int DT>
__device__ __forceinline__ void load_vec_f32(const typename Elem<DT>::store_t* p, uint32_t left, float (&f)[vec_elems<DT>()]) {
  constexpr int VE = vec_elems<DT>();
  VecU<DT> x;
  if (left >= VE) {
    x.v = *(const u32x4_unaligned*)p;
  } else {
    x.v = (u32x4){0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < VE; ++e)
      if ((uint32_t)e < left) x.e[e] = p[e];
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) f[e] = Elem<DT>::load(x.e[e]);
}

// Stores N values as elements of DT (N may be more than one 16-byte vector of it).
template <int DT, int N>
__device__ __forceinline__ void store_vec_f32(typename Elem<DT>::store_t* p, uint32_t left, const float (&f)[N]) {
  constexpr int VE = vec_elems<DT>();
  static_assert(N % VE == 0, "whole vectors");
  if (left >= N) {
#pragma unroll
    for (int b = 0; b < N; b += VE) {
      VecU<DT> x;
#pragma unroll
      for (int e = 0; e < VE; ++e) x.e[e] = Elem<DT>::store(f[b + e]);
      *(u32x4_unaligned*)(p + b) = x.v;
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if ((uint32_t)e < left) p[e] = Elem<DT>::store(f[e]);
  }
}

// ------------------------------------------------------------------------------------------
// lookup: out[i] = scale * table[ids[i] - first_row], zero where that row is not in the table
// ------------------------------------------------------------------------------------------
struct EmbeddingArgs {
  const char* table;
  const void* ids;
  char* out;
  uint32_t vecs;      // n * vecs_per_row; the host cuts longer lists
  uint32_t vecs_per_row;
  int64_t first_row;
  uint64_t rows;
  uint32_t hidden;
  float scale;
};

constexpr int kLookupVecs = 4;  // vectors per lane

// The output is one run of n * vecs_per_row vectors, of which a wavefront takes 64 * kLookupVecs in a row
// whatever the row length; every lane looks up the row of each of its vectors.
template <int DT, typename ID>
__global__ __launch_bounds__(256) void embedding_kernel(const EmbeddingArgs a) {
  using S = typename Elem<DT>::store_t;
  constexpr int VE = vec_elems<DT>();
  const S* table = (const S*)a.table;
  S* out = (S*)a.out;
  const ID* ids = (const ID*)a.ids;
  const uint32_t v0 = (blockIdx.x * 4 + threadIdx.x / kWave) * (uint32_t)(kWave * kLookupVecs) + threadIdx.x % kWave;
  float f[kLookupVecs][VE];
#pragma unroll
  for (int u = 0; u < kLookupVecs; ++u) {
    const uint32_t v = v0 + (uint32_t)u * kWave;
#pragma unroll
    for (int e = 0; e < VE; ++e) f[u][e] = 0.0f;
    if (v >= a.vecs) continue;
    const uint32_t i = v / a.vecs_per_row;
    const uint32_t c = (v - i * a.vecs_per_row) * VE;
    const uint64_t r = (uint64_t)(int64_t)ids[i] - (uint64_t)a.first_row;  // wraps: below the table is far above it
    if (r < a.rows) load_vec_f32<DT>(table + r * a.hidden + c, a.hidden - c, f[u]);
  }
#pragma unroll
  for (int u = 0; u < kLookupVecs; ++u) {
    const uint32_t v = v0 + (uint32_t)u * kWave;
    if (v >= a.vecs) break;
    const uint32_t i = v / a.vecs_per_row;
    const uint32_t c = (v - i * a.vecs_per_row) * VE;
#pragma unroll
    for (int e = 0; e < VE; ++e) f[u][e] = a.scale * f[u][e];
    store_vec_f32<DT>(out + (size_t)i * a.hidden + c, a.hidden - c, f[u]);
  }
}

// ------------------------------------------------------------------------------------------
// sort by row: order = stable argsort of the rows, offsets[v] = how many sorted tokens lie before row v
// ------------------------------------------------------------------------------------------
// The key of a token is its row, or `rows` where that is not in the table: those come last.
template <typename ID>
__device__ __forceinline__ uint32_t row_key(const ID* ids, uint64_t i, int64_t first_row, uint32_t rows) {
  const uint64_t r = (uint64_t)(int64_t)ids[i] - (uint64_t)first_row;
  return r < rows ? (uint32_t)r : rows;
}

// Few tokens (at most kSortSmall): all keys in LDS, and both results by counting, in one launch.  The
// first workgroups rank a token each (how many keys are smaller, or equal and earlier), the others
// count how many keys lie before a row.
constexpr int kSortSmall = 2048;
constexpr int kSortBlock = 256;

template <typename ID>
__global__ __launch_bounds__(kSortBlock) void sort_small_kernel(const ID* ids, uint32_t n, int64_t first_row, uint32_t rows,
                                                                uint32_t rank_groups, int64_t* order, int64_t* offsets) {
  __shared__ uint32_t key[kSortSmall];
  for (uint32_t i = threadIdx.x; i < n; i += kSortBlock) key[i] = row_key(ids, i, first_row, rows);
  __syncthreads();
  if (blockIdx.x < rank_groups) {
    const uint32_t i = blockIdx.x * kSortBlock + threadIdx.x;
    if (i >= n) return;
    const uint32_t mine = key[i];
    uint32_t before = 0;
    for (uint32_t j = 0; j < n; ++j) before += (key[j] < mine || (key[j] == mine && j < i)) ? 1u : 0u;
    order[before] = i;
  } else {
    const uint32_t v = (blockIdx.x - rank_groups) * kSortBlock + threadIdx.x;
    if (v > rows) return;
    uint32_t before = 0;
    for (uint32_t j = 0; j < n; ++j) before += key[j] < v ? 1u : 0u;
    offsets[v] = before;
  }
}

// More tokens: least-significant-digit radix sort, kSortDigits values a digit, three launches a pass.
constexpr int kSortBits = 8;
constexpr int kSortDigits = 1 << kSortBits;
constexpr int kSortSteps = 8;                                 // keys per lane
constexpr int kSortWaves = kSortBlock / kWave;
constexpr int kSortTile = kSortBlock * kSortSteps;            // keys per workgroup

struct SortArgs {
  const void* ids;         // first pass: the keys come from here
  const uint32_t* key_in;  // later passes
  const uint32_t* pos_in;
  uint32_t* key_out;       // null in the last pass but for the sorted keys the offsets are found in
  uint32_t* pos_out;
  int64_t* order;          // last pass
  uint32_t* counts;        // [kSortDigits][tiles]; after the scan: keys of the digit in earlier tiles
  uint32_t* totals;        // [kSortDigits]: keys of the digit in all tiles
  uint32_t n;
  uint32_t tiles;
  int64_t first_row;
  uint32_t rows;
  int shift;
};

template <typename ID, bool FIRST>
__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, uint32_t i) {
  if constexpr (FIRST) return row_key((const ID*)a.ids, i, a.first_row, a.rows);
  else return a.key_in[i];
}

template <typename ID, bool FIRST>
__global__ __launch_bounds__(kSortBlock) void sort_count_kernel(const SortArgs a) {
  __shared__ uint32_t hist[kSortDigits];
  for (int d = threadIdx.x; d < kSortDigits; d += kSortBlock) hist[d] = 0;
  __syncthreads();
  const uint32_t base = blockIdx.x * (uint32_t)kSortTile;
#pragma unroll
  for (int s = 0; s < kSortSteps; ++s) {
    const uint32_t i = base + (uint32_t)s * kSortBlock + threadIdx.x;
    if (i < a.n) atomicAdd(&hist[(sort_key<ID, FIRST>(a, i) >> a.shift) & (kSortDigits - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < kSortDigits; d += kSortBlock) a.counts[(size_t)d * a.tiles + blockIdx.x] = hist[d];
}

// One workgroup per digit: exclusive scan of its counts over the tiles, and their total.
__global__ __launch_bounds__(kSortBlock) void sort_scan_kernel(uint32_t* counts, uint32_t tiles, uint32_t* totals) {
  __shared__ uint32_t part[kSortBlock];
  uint32_t* row = counts + (size_t)blockIdx.x * tiles;
  uint32_t carry = 0;
  for (uint32_t t0 = 0; t0 < tiles; t0 += kSortBlock) {
    const uint32_t t = t0 + threadIdx.x;
    const uint32_t mine = t < tiles ? row[t] : 0;
    part[threadIdx.x] = mine;
    __syncthreads();
    for (int d = 1; d < kSortBlock; d <<= 1) {
      const uint32_t add = (int)threadIdx.x >= d ? part[threadIdx.x - d] : 0;
      __syncthreads();
      part[threadIdx.x] += add;
      __syncthreads();
    }
    if (t < tiles) row[t] = carry + part[threadIdx.x] - mine;
    carry += part[kSortBlock - 1];
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// A wavefront holds kSortSteps x 64 consecutive keys.  Within one step of 64, a key's rank among the
// equal digits is the number of lower lanes with the same digit, found by one ballot per bit; the
// digit's count so far is kept per wavefront in LDS, so equal digits stay in their order.
template <typename ID, bool FIRST, bool LAST>
__global__ __launch_bounds__(kSortBlock) void sort_scatter_kernel(const SortArgs a) {
  __shared__ uint32_t seen[kSortWaves][kSortDigits];
  __shared__ uint32_t start[kSortDigits];
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  for (int d = threadIdx.x; d < kSortWaves * kSortDigits; d += kSortBlock) (&seen[0][0])[d] = 0;
  if (threadIdx.x < kSortDigits) start[threadIdx.x] = a.totals[threadIdx.x];
  __syncthreads();
  // keys of smaller digits: scan of the totals
  for (int d = 1; d < kSortDigits; d <<= 1) {
    const uint32_t add = (int)threadIdx.x >= d && threadIdx.x < kSortDigits ? start[threadIdx.x - d] : 0;
    __syncthreads();
    if (threadIdx.x < kSortDigits) start[threadIdx.x] += add;
    __syncthreads();
  }
  const uint32_t base = blockIdx.x * (uint32_t)kSortTile + wave * (uint32_t)(kSortSteps * kWave) + lane;
  uint32_t key[kSortSteps], rank[kSortSteps];
#pragma unroll
  for (int s = 0; s < kSortSteps; ++s) {
    const uint32_t i = base + (uint32_t)s * kWave;
    key[s] = i < a.n ? sort_key<ID, FIRST>(a, i) : 0;
    rank[s] = 0;
  }
#pragma unroll
  for (int s = 0; s < kSortSteps; ++s) {
    const bool live = base + (uint32_t)s * kWave < a.n;
    const uint32_t digit = (key[s] >> a.shift) & (kSortDigits - 1);
    uint64_t same = __ballot(live);
#pragma unroll
    for (int b = 0; b < kSortBits; ++b) {
      const uint64_t set = __ballot((digit >> b) & 1u);
      same &= ((digit >> b) & 1u) ? set : ~set;
    }
    if (live) {
      const uint32_t before = __popcll(same & ((1ull << lane) - 1));
      rank[s] = seen[wave][digit] + before;
      // every lane of the group has read the count (one wavefront, in step); its first lane advances it
      if (before == 0) seen[wave][digit] += (uint32_t)__popcll(same);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  if (threadIdx.x < kSortDigits) {
    const uint32_t d = threadIdx.x;
    uint32_t at = start[d] - a.totals[d] + a.counts[(size_t)d * a.tiles + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = seen[w][d];
      seen[w][d] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < kSortSteps; ++s) {
    const uint32_t i = base + (uint32_t)s * kWave;
    if (i >= a.n) continue;
    const uint32_t at = seen[wave][(key[s] >> a.shift) & (kSortDigits - 1)] + rank[s];
    const uint32_t p = FIRST ? i : a.pos_in[i];
    a.key_out[at] = key[s];
    if constexpr (LAST) a.order[at] = p;
    else a.pos_out[at] = p;
  }
}

// offsets[v] = first position in the sorted keys whose key is not below v.
__global__ __launch_bounds__(kSortBlock) void sort_offsets_kernel(const uint32_t* key, uint32_t n, uint32_t rows, int64_t* offsets) {
  for (uint64_t v = (uint64_t)blockIdx.x * kSortBlock + threadIdx.x; v <= rows; v += (uint64_t)gridDim.x * kSortBlock) {
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (key[mid] < (uint32_t)v) lo = mid + 1; else hi = mid;
    }
    offsets[v] = lo;
  }
}

// ------------------------------------------------------------------------------------------
// gradient: d_table[v] = scale * sum of grad[order[j]], offsets[v] <= j < offsets[v + 1]
// ------------------------------------------------------------------------------------------
// A row with at most kGradPiece tokens is summed by one wavefront per column chunk, in ascending
// order.  A longer one (padding, a frequent word) is cut where the sorted tokens are cut into pieces of
// kGradPiece: every piece is summed on its own into the workspace and a second launch adds the pieces
// in ascending order.  A piece touches at most two such rows, the one it begins in (slot 0) and the
// one that begins inside it (slot 1), and at most one of them can begin in it.
constexpr int kGradPiece = 64;
constexpr int kGradWaves = 4;
constexpr int kGradLoads = 4;  // rows in flight per lane

struct EmbeddingGradArgs {
  const char* grad;
  const int64_t* order;
  const int64_t* offsets;
  char* out;
  float* partial;       // [pieces][2][hidden]
  uint32_t rows;
  uint32_t n;
  uint32_t piece_groups; // workgroups that take pieces: the first ones; 0 where no row can be longer than a piece
  uint32_t hidden;
  uint32_t chunk_waves_log2;  // 1, 2 or 4 wavefronts share a row (a piece), each a chunk of 64 vectors at a time
  float scale;
  int accumulate;
};

// An entry of offsets as 32 bits (the host keeps n below 2^31).  It comes from device memory: held to
// the order's length, whatever it is.
__device__ __forceinline__ uint32_t offset_at(const EmbeddingGradArgs& a, uint32_t v) {
  const uint64_t j = (uint64_t)a.offsets[v];
  const uint32_t low = (uint32_t)j, high = (uint32_t)(j >> 32);
  return high || low > a.n ? a.n : low;
}

// Sum of grad[order[j]] over j0 <= j < j1 in ascending j, one vector of columns per lane.
template <int DT>
__device__ __forceinline__ void sum_rows(const EmbeddingGradArgs& a, uint32_t j0, uint32_t j1, uint32_t col, float (&acc)[vec_elems<DT>()]) {
  constexpr int VE = vec_elems<DT>();
  const typename Elem<DT>::store_t* grad = (const typename Elem<DT>::store_t*)a.grad;
#pragma unroll
  for (int e = 0; e < VE; ++e) acc[e] = 0.0f;
  for (uint32_t j = j0; j < j1; j += kGradLoads) {
    float f[kGradLoads][VE];
#pragma unroll
    for (int u = 0; u < kGradLoads; ++u) {
#pragma unroll
      for (int e = 0; e < VE; ++e) f[u][e] = 0.0f;
      if (j + u < j1 && col < a.hidden) {
        const uint64_t i = (uint64_t)a.order[j + u];
        if (i < a.n) load_vec_f32<DT>(grad + i * a.hidden + col, a.hidden - col, f[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kGradLoads; ++u)
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[e] += f[u][e];
  }
}

template <int DT, int OUT>
__device__ __forceinline__ void write_row(const EmbeddingGradArgs& a, uint32_t v, uint32_t col, const float (&acc)[vec_elems<DT>()]) {
  constexpr int VE = vec_elems<DT>();
  if (col >= a.hidden) return;
  typename Elem<OUT>::store_t* out = (typename Elem<OUT>::store_t*)a.out + (size_t)v * a.hidden + col;
  float r[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) r[e] = a.scale * acc[e];
  if (a.accumulate) {
    constexpr int OE = vec_elems<OUT>();
#pragma unroll
    for (int b = 0; b < VE; b += OE) {
      if (col + b >= a.hidden) break;
      float old[OE];
      load_vec_f32<OUT>(out + b, a.hidden - col - b, old);
#pragma unroll
      for (int e = 0; e < OE; ++e) r[b + e] = old[e] + r[b + e];
    }
  }
  store_vec_f32<OUT>(out, a.hidden - col, r);
}

// The row that holds sorted position j: the largest v with offsets[v] <= j, by a search in which the
// 64 lanes probe at once (three round trips for 2^18 rows).  All lanes return the same row.
__device__ __forceinline__ uint32_t row_of_position(const EmbeddingGradArgs& a, uint32_t j) {
  uint32_t lo = 0, hi = a.rows;  // offsets[lo] <= j < offsets[hi]
  while (hi - lo > 1) {
    const uint32_t step = (hi - lo + kWave - 1) / kWave;
    const uint32_t probe = lo + step * (threadIdx.x % kWave);
    const uint64_t below = __ballot(probe < hi && offset_at(a, probe) <= j) | 1;  // lane 0 probes lo itself
    const uint32_t at = lo + step * (63u - (uint32_t)__builtin_clzll(below));
    if (at + step < hi) hi = at + step;
    lo = at;
  }
  return lo;
}

template <int DT, int OUT>
__global__ __launch_bounds__(kGradWaves * kWave) void embedding_grad_kernel(const EmbeddingGradArgs a) {
  constexpr int VE = vec_elems<DT>();
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t sharing = 1u << a.chunk_waves_log2;
  const uint32_t col0 = ((wave & (sharing - 1)) * kWave + lane) * VE, stride = sharing * kWave * VE;
  const uint32_t per_group_log2 = 2 - a.chunk_waves_log2;
  float acc[VE];
  if (blockIdx.x >= a.piece_groups) {
    const uint32_t step = (gridDim.x - a.piece_groups) << per_group_log2;
    for (uint32_t v = ((blockIdx.x - a.piece_groups) << per_group_log2) + (wave >> a.chunk_waves_log2); v < a.rows; v += step) {
      const uint32_t j0 = offset_at(a, v), j1 = offset_at(a, v + 1);
      if ((j1 > j0 && j1 - j0 > kGradPiece) || (a.accumulate && j1 <= j0)) continue;
      for (uint32_t col = col0; col - lane * VE < a.hidden; col += stride) {
        sum_rows<DT>(a, j0, j1, col, acc);
        write_row<DT, OUT>(a, v, col, acc);
      }
    }
  } else {
    const uint32_t piece = (blockIdx.x << per_group_log2) + (wave >> a.chunk_waves_log2);
    const uint32_t in_table = offset_at(a, a.rows);
    if (piece >= (in_table + kGradPiece - 1) / kGradPiece) return;
    const uint32_t p0 = piece * kGradPiece;
    const uint32_t p1 = p0 + kGradPiece < in_table ? p0 + kGradPiece : in_table;
    const uint32_t first = row_of_position(a, p0);
    const uint32_t last = row_of_position(a, p1 - 1);
    const uint32_t first_end = offset_at(a, first + 1), last_begin = offset_at(a, last);
    const bool first_long = first_end - offset_at(a, first) > kGradPiece;
    const bool last_long = last != first && offset_at(a, last + 1) - last_begin > kGradPiece;
    for (uint32_t col = col0; col - lane * VE < a.hidden; col += stride) {
      float* slot = a.partial + (size_t)piece * 2 * a.hidden + col;
      if (first_long) {
        sum_rows<DT>(a, p0, first_end < p1 ? first_end : p1, col, acc);
        if (col < a.hidden) store_vec_f32<MCCL_F32>(slot, a.hidden - col, acc);
      }
      if (last_long) {
        sum_rows<DT>(a, last_begin, p1, col, acc);
        if (col < a.hidden) store_vec_f32<MCCL_F32>(slot + a.hidden, a.hidden - col, acc);
      }
    }
  }
}

// Adds the pieces of the long row that begins in a workgroup's piece, a chunk of columns per workgroup:
// kJoinWaves wavefronts take every kJoinWaves-th piece each, and their sums are added in the order of the
// wavefronts.
constexpr int kJoinWaves = 8;

template <int DT, int OUT>
__global__ __launch_bounds__(kJoinWaves * kWave) void embedding_grad_join_kernel(const EmbeddingGradArgs a) {
  constexpr int VE = vec_elems<DT>();
  __shared__ float sum[kJoinWaves][kWave * VE];
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t in_table = offset_at(a, a.rows);
  const uint32_t piece = blockIdx.x, col = (blockIdx.y * kWave + lane) * VE;
  if (piece >= (in_table + kGradPiece - 1) / kGradPiece) return;
  const uint32_t p0 = piece * kGradPiece;
  const uint32_t p1 = p0 + kGradPiece < in_table ? p0 + kGradPiece : in_table;
  const uint32_t v = row_of_position(a, p1 - 1);  // of the rows of a piece only the last can begin in it and be long
  const uint32_t j0 = offset_at(a, v), j1 = offset_at(a, v + 1);
  if (j1 <= j0 || j1 - j0 <= kGradPiece || j0 < p0) return;
  const uint32_t last = (j1 - 1) / kGradPiece;
  float acc[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) acc[e] = 0.0f;
  for (uint32_t p = piece + wave; p <= last; p += kJoinWaves) {
    const float* from = a.partial + ((size_t)p * 2 + (p == piece && j0 != p0 ? 1 : 0)) * a.hidden + col;
#pragma unroll
    for (int e = 0; e < VE; ++e)
      if (col + e < a.hidden) acc[e] += from[e];
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) sum[wave][e * kWave + lane] = acc[e];
  __syncthreads();
  if (wave == 0) {
    for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[e] += sum[w][e * kWave + lane];
    write_row<DT, OUT>(a, v, col, acc);
  }
}

}  // namespace
