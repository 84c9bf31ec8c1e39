// Embedding lookup of a vocabulary shard, the sort of its tokens by row, and its gradient by sorted
// tokens (no kernel of the reference: the callers' steps before an all_reduce of vocabulary-sharded
// activations, and before and after the exchange of routed tokens).
#pragma once

#include <type_traits>

#include "kernels_common.hpp"

namespace {

// ------------------------------------------------------------------------------------------
// conversions
// ------------------------------------------------------------------------------------------
// Round to nearest even by the hardware's conversion, two elements an instruction (the exchange kernels'
// Elem::store makes every NaN the canonical one, at five instructions an element; here a NaN stays a NaN).
typedef float f32pair __attribute__((ext_vector_type(2)));
typedef __bf16 bf16pair __attribute__((ext_vector_type(2)));
typedef _Float16 f16pair __attribute__((ext_vector_type(2)));

template <int DT>
__device__ __forceinline__ uint32_t narrow_pair(float lo, float hi) {
  if constexpr (DT == MCCL_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32pair){lo, hi}, bf16pair));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32pair){lo, hi}, f16pair));
}

template <int DT>
__device__ __forceinline__ typename Elem<DT>::store_t narrow(float f) {
  if constexpr (DT == MCCL_F32) return f;
  else return (typename Elem<DT>::store_t)narrow_pair<DT>(f, 0.0f);
}

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

// Stores N values as elements of DT (N may be more than one 16-byte vector of it); STREAM: past the caches, for
// what is too large to be read from them again.
template <int DT, bool STREAM = false, int N>
__device__ __forceinline__ void store_vec_f32(typename Elem<DT>::store_t* p, uint32_t left, const float (&f)[N]) {
  constexpr int VE = vec_elems<DT>();
  static_assert(N % VE == 0, "whole vectors");
  if (left >= N) {
#pragma unroll
    for (int b = 0; b < N; b += VE) {
      VecU<DT> x;
      if constexpr (VE == 4) x.v = (u32x4){f32_to_bits(f[b]), f32_to_bits(f[b + 1]), f32_to_bits(f[b + 2]), f32_to_bits(f[b + 3])};
      else x.v = (u32x4){narrow_pair<DT>(f[b], f[b + 1]), narrow_pair<DT>(f[b + 2], f[b + 3]), narrow_pair<DT>(f[b + 4], f[b + 5]),
                         narrow_pair<DT>(f[b + 6], f[b + 7])};
      if constexpr (STREAM) __builtin_nontemporal_store(x.v, (u32x4_unaligned*)(p + b));
      else *(u32x4_unaligned*)(p + b) = x.v;
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if ((uint32_t)e < left) p[e] = narrow<DT>(f[e]);
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
constexpr int kLookupWaves = 4;

// The output is one run of n * vecs_per_row vectors, of which a wavefront takes 64 * kLookupVecs in a row
// whatever the row length; every lane looks up the row of each of its vectors.  All ids are loaded before
// the first row, all rows before the first store, and nothing in between depends on a branch: a vector
// behind the list reads the last one, an id outside the table reads row 0, and the last vector of a row
// that is no whole number of them begins early enough to be whole (its first elements are written twice,
// with the same values).  Rows shorter than a vector, and a table without rows, take the SHORT form.
// Bound by memory, the output's share by far the larger (a word's row is in the caches after its first use):
// 32768 rows of 7168 bf16 115 us (118 alone), 5.2 TB/s of what has to move; 8 rows of 4096 take 2.6 us, which is a launch and two
// loads that depend on each other.  Stores past the caches: rows of the table stay in them.
template <int DT, typename ID, bool SHORT>
__global__ __launch_bounds__(kLookupWaves * kWave) void embedding_kernel(const EmbeddingArgs a) {
  using S = typename Elem<DT>::store_t;
  constexpr int VE = vec_elems<DT>();
  const S* table = (const S*)a.table;
  S* out = (S*)a.out;
  const ID* ids = (const ID*)a.ids;
  const uint32_t v0 = (blockIdx.x * kLookupWaves + threadIdx.x / kWave) * (uint32_t)(kWave * kLookupVecs) + threadIdx.x % kWave;
  uint32_t i[kLookupVecs], c[kLookupVecs];
  uint64_t r[kLookupVecs];
#pragma unroll
  for (int u = 0; u < kLookupVecs; ++u) {
    const uint32_t v = v0 + (uint32_t)u * kWave < a.vecs ? v0 + (uint32_t)u * kWave : a.vecs - 1;
    i[u] = v / a.vecs_per_row;
    c[u] = (v - i[u] * a.vecs_per_row) * VE;
    if (!SHORT && c[u] + VE > a.hidden) c[u] = a.hidden - VE;
    r[u] = (uint64_t)(int64_t)ids[i[u]];
  }
  __builtin_amdgcn_sched_barrier(0);
  bool inside[kLookupVecs];
#pragma unroll
  for (int u = 0; u < kLookupVecs; ++u) {
    r[u] -= (uint64_t)a.first_row;  // wraps: below the table is far above it
    inside[u] = r[u] < a.rows;
    if (!inside[u]) r[u] = 0;
  }
  float f[kLookupVecs][VE];
  if constexpr (SHORT) {
#pragma unroll
    for (int u = 0; u < kLookupVecs; ++u) {
#pragma unroll
      for (int e = 0; e < VE; ++e) f[u][e] = 0.0f;
      if (inside[u]) load_vec_f32<DT>(table + r[u] * a.hidden + c[u], a.hidden - c[u], f[u]);
    }
  } else {
    VecU<DT> x[kLookupVecs];
#pragma unroll
    for (int u = 0; u < kLookupVecs; ++u) x[u].v = *(const u32x4_unaligned*)(table + r[u] * a.hidden + c[u]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < kLookupVecs; ++u)
#pragma unroll
      for (int e = 0; e < VE; ++e) f[u][e] = Elem<DT>::load(x[u].e[e]);
  }
#pragma unroll
  for (int u = 0; u < kLookupVecs; ++u) {
    if (v0 + (uint32_t)u * kWave >= a.vecs) break;
#pragma unroll
    for (int e = 0; e < VE; ++e) f[u][e] = inside[u] ? a.scale * f[u][e] : 0.0f;
    store_vec_f32<DT, true>(out + (size_t)i[u] * a.hidden + c[u], a.hidden - c[u], f[u]);
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

// Few tokens (at most kSortSmall): all keys in LDS, and both results by counting, in one launch.  A workgroup
// has 64 results, one a lane: the first workgroups rank a token each (how many keys are smaller, or equal and
// earlier), the others count how many keys lie before a row.  Its wavefronts share the keys, 64 in a row at a
// time, so that all keys of such a block lie before the 64 tokens, behind them, or are these.  Bound by the
// compares, n * (n + rows) of them, and by handing out the workgroups: 512 of them at most, which walk the
// results (2048 ids over 60000 rows 20 us against 23 with one for each 64).  Against the launches of the sort
// below: 2048 ids over 4000 rows 7.0 us against 17, over 60000 rows 20 against 17; 4096 over 4000 rows 11
// against 19, over 60000 rows 42 against 19.
constexpr int kSortSmall = 2048;
constexpr int kSortBlock = 256;

template <typename ID, int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void sort_small_kernel(const ID* ids, uint32_t n, int64_t first_row, uint32_t rows,
                                                                         uint32_t rank_groups, uint32_t groups, int64_t* order, int64_t* offsets) {
  __shared__ __align__(16) uint32_t key[kSortSmall];
  __shared__ uint32_t count[WAVES][kWave];
  const uint32_t lane = threadIdx.x % kWave, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
  const uint32_t blocks = (n + kWave - 1) / kWave;
  for (uint32_t i = threadIdx.x; i < blocks * kWave; i += WAVES * kWave) key[i] = i < n ? row_key(ids, i, first_row, rows) : ~0u;
  __syncthreads();
  for (uint32_t group = blockIdx.x; group < groups; group += gridDim.x) {
    const bool ranks = group < rank_groups;
    const uint32_t mine = (ranks ? group : group - rank_groups) * kWave + lane;
    const uint32_t limit = ranks ? key[mine] : mine;  // keys below it count; for a token, equal ones before it too
    uint32_t before = 0;
    for (uint32_t b = wave; b < blocks; b += WAVES) {
      const u32x4* four = (const u32x4*)(key + b * kWave);
      if (ranks && b == group) {
#pragma unroll
        for (uint32_t j = 0; j < kWave; ++j) before += four[j / 4][j % 4] < limit + (j < lane ? 1u : 0u) ? 1u : 0u;
      } else {
        const uint32_t below = limit + (ranks && b < group ? 1u : 0u);  // a row is below 2^31
#pragma unroll
        for (uint32_t j = 0; j < kWave; ++j) before += four[j / 4][j % 4] < below ? 1u : 0u;
      }
    }
    count[wave][lane] = before;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int w = 1; w < WAVES; ++w) before += count[w][lane];
      if (ranks) {
        if (mine < n) order[before] = mine;
      } else if (mine <= rows) {
        offsets[mine] = before;
      }
    }
    __syncthreads();
  }
}

// More tokens: least-significant-digit radix sort, kSortDigits values a digit, two launches a pass: the digits
// of every tile are counted, then every workgroup adds up the counts of the tiles before its own and of the
// smaller digits, ranks its keys and writes them where they belong.  Over kSortTilesAdded tiles a third
// launch in between does the adding up (two passes: 131072 ids, 64 tiles, 30.7 us with it and 27.6 without; 200000
// ids 32.5 and 33.2; three passes, 1048576 ids 75 and 110).  These launches move a few bytes a key: they are bound by their round trips
// (16384 ids over 32000 rows, two passes: 4.5 us a count, 5.8 and 5.4 the scatters, 4.8 the offsets).
constexpr int kSortBits = 8;
constexpr int kSortDigits = 1 << kSortBits;
constexpr int kSortWaves = 8;
constexpr int kSortThreads = kSortWaves * kWave;
constexpr int kSortSteps = 4;                                 // keys per lane
constexpr int kSortTile = kSortThreads * kSortSteps;          // keys per workgroup
constexpr uint32_t kSortTilesAdded = 96;

struct SortArgs {
  const void* ids;         // first pass: the keys come from here
  const uint32_t* key_in;  // later passes
  const uint32_t* pos_in;
  uint32_t* key_out;
  uint32_t* pos_out;
  int64_t* order;          // last pass
  uint32_t* counts;        // [tiles][kSortDigits]; once added up: keys of the digit in earlier tiles
  uint32_t* totals;        // [kSortDigits]: keys of the digit in all tiles, where they are added up by a launch
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
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const SortArgs a) {
  __shared__ uint32_t hist[kSortDigits];
  const uint32_t base = blockIdx.x * (uint32_t)kSortTile + threadIdx.x;
  uint32_t key[kSortSteps];
#pragma unroll
  for (int s = 0; s < kSortSteps; ++s) {
    const uint32_t i = base + (uint32_t)s * kSortThreads;
    key[s] = i < a.n ? sort_key<ID, FIRST>(a, i) : 0;
  }
  if (threadIdx.x < kSortDigits) hist[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int s = 0; s < kSortSteps; ++s)
    if (base + (uint32_t)s * kSortThreads < a.n) atomicAdd(&hist[(key[s] >> a.shift) & (kSortDigits - 1)], 1u);
  __syncthreads();
  if (threadIdx.x < kSortDigits) a.counts[(size_t)blockIdx.x * kSortDigits + threadIdx.x] = hist[threadIdx.x];
}

// Adds up the counts over the tiles, kAddDigits digits a workgroup, kAddParts parts of the tiles side by side.
constexpr uint32_t kAddDigits = 16, kAddParts = 64;

__global__ __launch_bounds__(kAddDigits * kAddParts) void sort_add_kernel(uint32_t* counts, uint32_t tiles, uint32_t* totals) {
  __shared__ uint32_t sum[kAddParts][kAddDigits];
  const uint32_t digit = threadIdx.x % kAddDigits, part = threadIdx.x / kAddDigits;
  const uint32_t per = (tiles + kAddParts - 1) / kAddParts;
  const uint32_t t0 = part * per, t1 = t0 + per < tiles ? t0 + per : tiles;
  uint32_t* column = counts + blockIdx.x * kAddDigits + digit;
  uint32_t mine = 0;
  for (uint32_t t = t0; t < t1; ++t) mine += column[(size_t)t * kSortDigits];
  sum[part][digit] = mine;
  __syncthreads();
  uint32_t before = 0, total = 0;
  for (uint32_t p = 0; p < kAddParts; ++p) {
    const uint32_t c = sum[p][digit];
    total += c;
    before += p < part ? c : 0;
  }
  if (part == 0) totals[blockIdx.x * kAddDigits + digit] = total;
  for (uint32_t t = t0; t < t1; ++t) {
    const uint32_t c = column[(size_t)t * kSortDigits];
    column[(size_t)t * kSortDigits] = before;
    before += c;
  }
}

// A wavefront holds kSortSteps x 64 consecutive keys.  Within one step of 64, a key's rank among the
// equal digits is the number of lower lanes with the same digit, found by one ballot per bit; the
// digit's count so far is kept per wavefront in LDS, so equal digits stay in their order.
template <typename ID, bool FIRST, bool LAST, bool ADDED>
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(const SortArgs a) {
  __shared__ uint32_t seen[kSortWaves][kSortDigits];
  __shared__ uint32_t below[kSortDigits / kWave];
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t base = blockIdx.x * (uint32_t)kSortTile + wave * (uint32_t)(kSortSteps * kWave) + lane;
  uint32_t key[kSortSteps], pos[kSortSteps], rank[kSortSteps];
#pragma unroll
  for (int s = 0; s < kSortSteps; ++s) {
    const uint32_t i = base + (uint32_t)s * kWave;
    key[s] = i < a.n ? sort_key<ID, FIRST>(a, i) : 0;
    pos[s] = FIRST ? i : i < a.n ? a.pos_in[i] : 0;
    rank[s] = 0;
  }
  // Where the digit of this thread begins: the keys of smaller digits, and its own in earlier tiles.
  uint32_t before = 0, total = 0, smaller = 0;
  if (threadIdx.x < kSortDigits) {
    if constexpr (ADDED) {
      before = a.counts[(size_t)blockIdx.x * kSortDigits + threadIdx.x];
      total = a.totals[threadIdx.x];
    } else {
#pragma unroll 8
      for (uint32_t t = 0; t < a.tiles; ++t) {
        const uint32_t c = a.counts[(size_t)t * kSortDigits + threadIdx.x];
        total += c;
        before += t < blockIdx.x ? c : 0;
      }
    }
    uint32_t scan = total;  // over the wavefront's 64 digits
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const uint32_t add = __shfl_up(scan, d);
      scan += (int)lane >= d ? add : 0;
    }
    smaller = scan - total;
    if (lane == kWave - 1) below[wave] = scan;
  }
  for (uint32_t d = threadIdx.x; d < kSortWaves * kSortDigits; d += kSortThreads) (&seen[0][0])[d] = 0;
  __syncthreads();
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
      const uint32_t lower = __popcll(same & ((1ull << lane) - 1));
      rank[s] = seen[wave][digit] + lower;
      // every lane of the group has read the count (one wavefront, in step); its first lane advances it
      if (lower == 0) seen[wave][digit] += (uint32_t)__popcll(same);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  if (threadIdx.x < kSortDigits) {
    uint32_t at = smaller + before;
    for (uint32_t w = 0; w < wave; ++w) at += below[w];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = seen[w][threadIdx.x];
      seen[w][threadIdx.x] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < kSortSteps; ++s) {
    if (base + (uint32_t)s * kWave >= a.n) continue;
    const uint32_t at = seen[wave][(key[s] >> a.shift) & (kSortDigits - 1)] + rank[s];
    a.key_out[at] = key[s];
    if constexpr (LAST) a.order[at] = pos[s];
    else a.pos_out[at] = pos[s];
  }
}

// offsets[v] = first position in the sorted keys whose key is not below v.  Every `every`-th key (a power of
// two, so that there are at most kSortSamples) goes into LDS and the search begins there: the round trips
// to memory that are left are those within `every` keys.
constexpr uint32_t kSortSamples = 1024;

__global__ __launch_bounds__(kSortBlock) void sort_offsets_kernel(const uint32_t* key, uint32_t n, uint32_t every_log2, uint32_t rows,
                                                                  int64_t* offsets) {
  __shared__ uint32_t sample[kSortSamples];
  const uint32_t samples = ((n - 1) >> every_log2) + 1;
  for (uint32_t i = threadIdx.x; i < samples; i += kSortBlock) sample[i] = key[i << every_log2];
  __syncthreads();
  const uint64_t v = (uint64_t)blockIdx.x * kSortBlock + threadIdx.x;
  if (v > rows) return;
  uint32_t lo = 0, hi = samples;  // the first sample that is not below v
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    if (sample[mid] < (uint32_t)v) lo = mid + 1; else hi = mid;
  }
  uint32_t end = lo < samples ? lo << every_log2 : n;
  uint32_t begin = lo ? ((lo - 1) << every_log2) + 1 : 0;
  while (begin < end) {
    const uint32_t mid = begin + (end - begin) / 2;
    if (key[mid] < (uint32_t)v) begin = mid + 1; else end = mid;
  }
  offsets[v] = begin;
}

// ------------------------------------------------------------------------------------------
// gradient: d_table[v] = scale * sum of grad[order[j]], offsets[v] <= j < offsets[v + 1]
// ------------------------------------------------------------------------------------------
// A row with at most kGradPiece tokens is summed by the wavefronts of its columns, in ascending order.  A
// longer one (padding, a frequent word) is cut where the sorted tokens are cut into pieces of kGradPiece:
// every piece is summed on its own into the workspace and a second launch adds the pieces in ascending
// order.  A piece touches at most two such rows, the one it begins in (slot 0) and the one that begins
// inside it (slot 1), and at most one of them can begin in it.  Nothing is added by atomics: the order, and
// with it every bit, depends on the offsets alone.
// Bound by memory: every gradient row is read once and every row of the result written once, both past the
// caches (with plain loads and stores 76 and 85 us instead of 70 in the first of these).  16384 tokens into
// 32000 x 4096 bf16: 65 us, 6.1 TB/s, and 4.8 for the join; 32768 tokens added to 16000 x 7168 fp32: 136 us,
// 5.2 TB/s (reads and writes of the same rows alternate), and 12 for the join.  Few tokens are bound by the chain of
// loads, offsets to indices to rows.  8 rows in flight a wavefront: 4 and 16 are no faster where memory binds,
// and 16 cost half as much again in registers (105 us in the first).
constexpr int kGradPiece = kWave;  // a lane holds the index of each
constexpr int kGradWaves = 4;
constexpr int kGradLoads = 8;      // gradient rows in flight
constexpr uint32_t kNoRow = ~0u;

struct EmbeddingGradArgs {
  const char* grad;
  const int64_t* order;
  const int64_t* offsets;
  char* out;
  float* partial;        // [pieces][2][hidden]
  uint32_t* long_row;    // [pieces][2]: the long rows whose sums the slots hold, kNoRow if none's
  uint32_t rows;
  uint32_t n;
  uint32_t piece_groups; // workgroups that take pieces: the first ones; 0 where no row can be longer than a piece
  uint32_t row_groups;   // and those that take rows
  uint32_t column_groups;// workgroups side by side that share a row (a piece): the grid's second axis
  uint32_t hidden;
  uint32_t sharing_log2; // 1, 2 or 4 wavefronts of each
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

// The columns of a lane: VL vectors, 64 vectors apart.  A vector that would end behind the row is read from
// further ahead, and `skip` of its elements belong to the lane before; `own` is how many are its own.
template <int DT, int VL, bool SHORT>
struct GradColumns {
  static constexpr int VE = vec_elems<DT>();
  uint32_t col[VL], skip[VL], own[VL];
  __device__ __forceinline__ GradColumns(uint32_t first, uint32_t hidden) {
#pragma unroll
    for (int x = 0; x < VL; ++x) {
      const uint32_t c = first + x * kWave * VE;
      own[x] = c < hidden ? (hidden - c < VE ? hidden - c : VE) : 0;
      col[x] = c;
      skip[x] = 0;
      if (!SHORT && own[x] < VE) {
        col[x] = hidden - VE;
        skip[x] = own[x] ? VE - own[x] : 0;
      }
    }
  }
};

// Sums of the gradient rows that lanes [l0, l1) hold the indices of, in ascending order.
template <int DT, int VL, bool SHORT>
__device__ __forceinline__ void sum_rows(const EmbeddingGradArgs& a, int index, uint32_t l0, uint32_t l1,
                                         const GradColumns<DT, VL, SHORT>& c, float (&acc)[VL][vec_elems<DT>()]) {
  constexpr int VE = vec_elems<DT>();
  using S = typename Elem<DT>::store_t;
  const S* grad = (const S*)a.grad;
#pragma unroll
  for (int x = 0; x < VL; ++x)
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[x][e] = 0.0f;
  uint32_t l = l0;
  if constexpr (!SHORT) {
    constexpr int G = kGradLoads / VL;
    const bool whole = __ballot(threadIdx.x % kWave >= l0 && threadIdx.x % kWave < l1 && index < 0) == 0;
    for (; whole && l + G <= l1; l += G) {
      VecU<DT> v[G][VL];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const S* row = grad + (size_t)(uint32_t)__builtin_amdgcn_readlane(index, l + g) * a.hidden;
#pragma unroll
        for (int x = 0; x < VL; ++x) v[g][x].v = __builtin_nontemporal_load((const u32x4_unaligned*)(row + c.col[x]));
      }
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int x = 0; x < VL; ++x)
#pragma unroll
          for (int e = 0; e < VE; ++e) acc[x][e] += Elem<DT>::load(v[g][x].e[e]);
    }
  }
  for (; l < l1; ++l) {
    const int i = __builtin_amdgcn_readlane(index, l);
    if (i < 0) continue;
    const S* row = grad + (size_t)(uint32_t)i * a.hidden;
#pragma unroll
    for (int x = 0; x < VL; ++x) {
      float f[VE];
      if constexpr (SHORT) {
#pragma unroll
        for (int e = 0; e < VE; ++e) f[e] = 0.0f;
        if (c.own[x]) load_vec_f32<DT>(row + c.col[x], c.own[x], f);
      } else {
        load_vec_f32<DT>(row + c.col[x], VE, f);
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[x][e] += f[e];
    }
  }
}

// What a lane's whole vectors of a row of the result hold, for the sums that are added to it: loaded before
// the sums are made.
template <int DT, int OUT, int VL, bool SHORT>
__device__ __forceinline__ void read_row(const EmbeddingGradArgs& a, uint32_t v, const GradColumns<DT, VL, SHORT>& c,
                                         VecU<OUT> (&old)[VL][vec_elems<DT>() / vec_elems<OUT>()]) {
  constexpr int VE = vec_elems<DT>(), OE = vec_elems<OUT>();
  if (!a.accumulate) return;
  const typename Elem<OUT>::store_t* row = (const typename Elem<OUT>::store_t*)a.out + (size_t)v * a.hidden;
#pragma unroll
  for (int x = 0; x < VL; ++x)
#pragma unroll
    for (int b = 0; b < VE / OE; ++b)
      if (c.own[x] == VE) old[x][b].v = __builtin_nontemporal_load((const u32x4_unaligned*)(row + c.col[x] + b * OE));
}

// Stores (or adds) a lane's columns of a row of the result, scaled and rounded once.
template <int DT, int OUT, int VL, bool SHORT>
__device__ __forceinline__ void write_row(const EmbeddingGradArgs& a, uint32_t v, const GradColumns<DT, VL, SHORT>& c,
                                          const VecU<OUT> (&old)[VL][vec_elems<DT>() / vec_elems<OUT>()],
                                          const float (&acc)[VL][vec_elems<DT>()]) {
  constexpr int VE = vec_elems<DT>(), OE = vec_elems<OUT>();
  typename Elem<OUT>::store_t* row = (typename Elem<OUT>::store_t*)a.out + (size_t)v * a.hidden;
#pragma unroll
  for (int x = 0; x < VL; ++x) {
    float r[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) r[e] = a.scale * acc[x][e];
    if (c.own[x] == VE) {
      if (a.accumulate) {
#pragma unroll
        for (int e = 0; e < VE; ++e) r[e] = Elem<OUT>::load(old[x][e / OE].e[e % OE]) + r[e];
      }
      store_vec_f32<OUT, true>(row + c.col[x], VE, r);
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if ((uint32_t)e >= c.skip[x] && (uint32_t)e < c.skip[x] + c.own[x]) {
          auto* p = row + c.col[x] + e;
          *p = narrow<OUT>(a.accumulate ? Elem<OUT>::load(*p) + r[e] : r[e]);
        }
    }
  }
}

template <int DT, int VL, bool SHORT>
__device__ __forceinline__ void write_partial(float* row, const GradColumns<DT, VL, SHORT>& c, const float (&acc)[VL][vec_elems<DT>()]) {
  constexpr int VE = vec_elems<DT>();
#pragma unroll
  for (int x = 0; x < VL; ++x) {
    if (!SHORT && c.own[x]) store_vec_f32<MCCL_F32>(row + c.col[x], VE, acc[x]);  // elements of two lanes are the same in both
    if (SHORT) store_vec_f32<MCCL_F32>(row + c.col[x], c.own[x], acc[x]);
  }
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

// The token at sorted position j, or -1 where there is none.
__device__ __forceinline__ int token_at(const EmbeddingGradArgs& a, uint32_t j, uint32_t end) {
  if (j >= end) return -1;
  const uint64_t i = (uint64_t)a.order[j];
  return i < a.n ? (int)(uint32_t)i : -1;
}

template <int DT, int OUT, int VL, bool SHORT>
__global__ __launch_bounds__(kGradWaves * kWave) void embedding_grad_kernel(const EmbeddingGradArgs a) {
  constexpr int VE = vec_elems<DT>();
  const uint32_t lane = threadIdx.x % kWave, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
  const uint32_t sharing = 1u << a.sharing_log2, per_group_log2 = 2 - a.sharing_log2;
  const uint32_t member = wave >> a.sharing_log2;
  const uint32_t first_col = ((blockIdx.y << a.sharing_log2) + (wave & (sharing - 1))) * (kWave * VL * VE);
  const uint32_t stride = (a.column_groups << a.sharing_log2) * (kWave * VL * VE);
  float acc[VL][VE];
  if (blockIdx.x >= a.piece_groups) {
    const uint32_t step = a.row_groups << per_group_log2;
    for (uint32_t v = ((blockIdx.x - a.piece_groups) << per_group_log2) + member; v < a.rows; v += step) {
      const uint32_t j0 = offset_at(a, v), j1 = offset_at(a, v + 1);
      const uint32_t count = j1 > j0 ? j1 - j0 : 0;
      if (count > kGradPiece || (a.accumulate && count == 0)) continue;
      const int index = token_at(a, j0 + lane, j1);
      for (uint32_t col = first_col; col < a.hidden; col += stride) {
        const GradColumns<DT, VL, SHORT> c(col + lane * VE, a.hidden);
        VecU<OUT> old[VL][VE / vec_elems<OUT>()];
        read_row<DT, OUT, VL, SHORT>(a, v, c, old);
        sum_rows<DT, VL, SHORT>(a, index, 0, count, c, acc);
        write_row<DT, OUT, VL, SHORT>(a, v, c, old, acc);
      }
    }
  } else {
    const uint32_t piece = (blockIdx.x << per_group_log2) + member;
    const uint32_t in_table = offset_at(a, a.rows);
    const uint32_t p0 = piece * kGradPiece;
    if (p0 >= a.n) return;
    uint32_t in_slot[2] = {kNoRow, kNoRow};
    if (p0 < in_table) {
      const uint32_t p1 = p0 + kGradPiece < in_table ? p0 + kGradPiece : in_table;
      const int index = token_at(a, p0 + lane, p1);
      const uint32_t first = row_of_position(a, p0), last = row_of_position(a, p1 - 1);
      const uint32_t first_begin = offset_at(a, first), first_end = offset_at(a, first + 1), last_begin = offset_at(a, last);
      // Before the first row begins (the offsets of a range of rows of a larger plan) the search returns it all the same.
      const bool first_long = first_begin <= p0 && first_end - first_begin > kGradPiece;
      const bool last_long = last_begin > p0 && last_begin < p1 && offset_at(a, last + 1) - last_begin > kGradPiece;
      if (first_long) in_slot[0] = first;
      if (last_long) in_slot[1] = last;
      for (uint32_t col = first_col; col < a.hidden; col += stride) {
        const GradColumns<DT, VL, SHORT> c(col + lane * VE, a.hidden);
        float* slot = a.partial + (size_t)piece * 2 * a.hidden;
        if (first_long) {
          sum_rows<DT, VL, SHORT>(a, index, 0, (first_end < p1 ? first_end : p1) - p0, c, acc);
          write_partial<DT, VL, SHORT>(slot, c, acc);
        }
        if (last_long) {
          sum_rows<DT, VL, SHORT>(a, index, last_begin - p0, p1 - p0, c, acc);
          write_partial<DT, VL, SHORT>(slot + a.hidden, c, acc);
        }
      }
    }
    if (lane < 2 && first_col == 0) a.long_row[piece * 2 + lane] = lane ? in_slot[1] : in_slot[0];
  }
}

// Adds the pieces of the long row that begins in a workgroup's piece, a chunk of columns per workgroup:
// kJoinWaves wavefronts take every kJoinWaves-th piece each, kJoinLoads of them at a time, and their sums
// are added in the order of the wavefronts.  Every piece of such a row but the one it begins in has it in slot 0; where
// offsets fall one may not, and is left out.
constexpr int kJoinWaves = 8;
constexpr int kJoinLoads = 4;

template <int DT, int OUT, bool SHORT>
__global__ __launch_bounds__(kJoinWaves * kWave) void embedding_grad_join_kernel(const EmbeddingGradArgs a) {
  constexpr int VE = vec_elems<DT>();
  __shared__ float sum[kJoinWaves][VE * kWave];
  const uint32_t lane = threadIdx.x % kWave, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
  const uint32_t piece = blockIdx.x;
  const uint32_t inside = a.long_row[piece * 2 + 1], v = inside != kNoRow ? inside : a.long_row[piece * 2];
  if (v == kNoRow) return;
  const uint32_t j0 = offset_at(a, v), j1 = offset_at(a, v + 1), last = (j1 - 1) / kGradPiece;
  if (j0 / kGradPiece != piece) return;  // it begins in an earlier piece
  const GradColumns<DT, 1, SHORT> c((blockIdx.y * kWave + lane) * VE, a.hidden);
  float acc[1][VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) acc[0][e] = 0.0f;
  const auto slot_of = [&](uint32_t p) { return (size_t)p * 2 + (p == piece && inside != kNoRow ? 1 : 0); };
  const auto add = [&](auto count, uint32_t p) {
    float f[count][VE];
    bool held[count];
#pragma unroll
    for (int g = 0; g < count; ++g) {
      const size_t slot = slot_of(p + g * kJoinWaves);
      const float* from = a.partial + slot * a.hidden + c.col[0];
      held[g] = a.long_row[slot] == v;
#pragma unroll
      for (int b = 0; b < VE; b += 4) {
        if constexpr (SHORT) {
#pragma unroll
          for (int e = b; e < b + 4; ++e) f[g][e] = (uint32_t)e < c.own[0] ? from[e] : 0.0f;
        } else {
          float four[4];
          load_vec_f32<MCCL_F32>(from + b, 4, four);
#pragma unroll
          for (int e = 0; e < 4; ++e) f[g][b + e] = four[e];
        }
      }
    }
#pragma unroll
    for (int g = 0; g < count; ++g)
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[0][e] += held[g] ? f[g][e] : 0.0f;
  };
  uint32_t p = piece + wave;
  for (; p + (kJoinLoads - 1) * kJoinWaves <= last; p += kJoinLoads * kJoinWaves) add(std::integral_constant<int, kJoinLoads>{}, p);
  for (; p <= last; p += kJoinWaves) add(std::integral_constant<int, 1>{}, p);
#pragma unroll
  for (int e = 0; e < VE; ++e) sum[wave][e * kWave + lane] = acc[0][e];
  __syncthreads();
  if (wave == 0) {
    for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[0][e] += sum[w][e * kWave + lane];
    VecU<OUT> old[1][VE / vec_elems<OUT>()];
    read_row<DT, OUT, 1, SHORT>(a, v, c, old);
    write_row<DT, OUT, 1, SHORT>(a, v, c, old, acc);
  }
}

}  // namespace
