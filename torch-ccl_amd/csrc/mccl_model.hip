// The C ABI of the operators around the collectives that compute: embedding lookup and gradient, the
// router, and the mixture-of-experts layer for a few tokens.  Device code: kernels_embedding.hpp,
// kernels_router.hpp, kernels_layer.hpp.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "mccl.h"

#include "host_checks.hpp"
#include "kernels_embedding.hpp"
#include "kernels_layer.hpp"
#include "kernels_router.hpp"

namespace {

constexpr size_t kMaxHidden = 1u << 23;       // grids of at most 65535 column chunks
constexpr size_t kMaxGradTokens = 1u << 28;   // and of at most 2^32 threads along their first axis
constexpr uint32_t kMaxGroups = 1u << 23;     // rows and tokens beyond that walk the grid
constexpr size_t kMaxDenseTiles = 1u << 22;   // of layer_dense_kernel, 512 threads each
constexpr uint32_t kMaxSmallGroups = 512;     // of the sort of few ids

size_t float_size(int dtype) {
  return dtype == MCCL_F32 ? 4 : (dtype == MCCL_BF16 || dtype == MCCL_F16) ? 2 : 0;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return mccl_report_error(MCCL_ERR_HIP, "%s launch failed: %s", what, hipGetErrorString(e));
  return MCCL_OK;
}

int check_ids(const void* ids, int id_dtype) {
  if (id_dtype != MCCL_I32 && id_dtype != MCCL_I64) return mccl_report_error(MCCL_ERR_UNSUPPORTED, "ids are int32 or int64");
  if (!ids) return mccl_report_error(MCCL_ERR_INVALID_ARG, "id pointer is null");
  if (misaligned(ids, id_dtype == MCCL_I32 ? 4 : 8)) return mccl_report_error(MCCL_ERR_INVALID_ARG, "ids not aligned to their element size");
  return MCCL_OK;
}

// The device counts an id's row modulo 2^64: with rows past the largest id, the smallest ones would come out inside.
int check_rows(int64_t first_row, size_t rows) {
  if (first_row > 0 && rows > (uint64_t)(INT64_MAX - first_row) + 1)
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "rows [%lld, +%zu) pass 2^63", (long long)first_row, rows);
  return MCCL_OK;
}

size_t up16(size_t b) { return (b + 15) & ~(size_t)15; }

int sort_passes(uint64_t rows) {
  int passes = 1;
  while (passes < 4 && (rows >> (kSortBits * passes))) ++passes;
  return passes;
}

// Workspace of the sort: two sets of keys and positions, the digit counts per tile, and their totals.
struct SortPlan {
  size_t tiles, keys, counts, bytes;
};

SortPlan plan_sort(size_t n) {
  SortPlan p{};
  if (n <= (size_t)kSortSmall) return p;
  p.tiles = (n + kSortTile - 1) / kSortTile;
  p.keys = up16(n * 4);
  p.counts = up16(p.tiles * kSortDigits * 4);
  p.bytes = 4 * p.keys + p.counts + kSortDigits * 4;
  return p;
}

template <typename ID>
int launch_sort(const ID* ids, size_t n, int64_t first_row, size_t rows, char* ws, int64_t* order, int64_t* offsets, hipStream_t s) {
  if (n <= (size_t)kSortSmall) {
    const unsigned rank_groups = (unsigned)((n + kWave - 1) / kWave), groups = rank_groups + (unsigned)(rows / kWave + 1);
    // 4 wavefronts share the keys, or 8 (16 ids over 32000 rows 3.5 us against 5.3, 512 over 60000 8.1 against 8.3,
    // 1000 over 900 6.3 against 4.7)
    const unsigned waves = n <= 512 ? 4 : 8;
    hipLaunchKernelGGL((waves == 4 ? sort_small_kernel<ID, 4> : sort_small_kernel<ID, 8>), dim3(std::min(groups, kMaxSmallGroups)),
                       dim3(waves * kWave), 0, s, ids, (uint32_t)n, first_row, (uint32_t)rows, rank_groups, groups, order, offsets);
    return launched("sort");
  }
  const SortPlan p = plan_sort(n);
  uint32_t* key[2] = {(uint32_t*)ws, (uint32_t*)(ws + p.keys)};
  uint32_t* pos[2] = {(uint32_t*)(ws + 2 * p.keys), (uint32_t*)(ws + 3 * p.keys)};
  SortArgs a{};
  a.ids = ids;
  a.order = order;
  a.counts = (uint32_t*)(ws + 4 * p.keys);
  a.totals = (uint32_t*)(ws + 4 * p.keys + p.counts);
  a.n = (uint32_t)n;
  a.tiles = (uint32_t)p.tiles;
  a.first_row = first_row;
  a.rows = (uint32_t)rows;
  const int passes = sort_passes(rows);
  const dim3 tiles((unsigned)p.tiles), threads(kSortThreads);
  const bool added = p.tiles > kSortTilesAdded;
  for (int pass = 0; pass < passes; ++pass) {
    const bool first = pass == 0, last = pass == passes - 1;
    a.shift = pass * kSortBits;
    a.key_in = key[(pass + 1) & 1];
    a.pos_in = pos[(pass + 1) & 1];
    a.key_out = key[pass & 1];
    a.pos_out = pos[pass & 1];
    hipLaunchKernelGGL((first ? sort_count_kernel<ID, true> : sort_count_kernel<ID, false>), tiles, threads, 0, s, a);
    if (added) hipLaunchKernelGGL(sort_add_kernel, dim3(kSortDigits / kAddDigits), dim3(kAddDigits * kAddParts), 0, s, a.counts, a.tiles, a.totals);
    auto scatter = added ? (first ? (last ? sort_scatter_kernel<ID, true, true, true> : sort_scatter_kernel<ID, true, false, true>)
                                  : (last ? sort_scatter_kernel<ID, false, true, true> : sort_scatter_kernel<ID, false, false, true>))
                         : (first ? (last ? sort_scatter_kernel<ID, true, true, false> : sort_scatter_kernel<ID, true, false, false>)
                                  : (last ? sort_scatter_kernel<ID, false, true, false> : sort_scatter_kernel<ID, false, false, false>));
    hipLaunchKernelGGL(scatter, tiles, threads, 0, s, a);
  }
  uint32_t every_log2 = 0;
  while (((a.n - 1) >> every_log2) + 1 > kSortSamples) ++every_log2;
  hipLaunchKernelGGL(sort_offsets_kernel, dim3((unsigned)(rows / kSortBlock + 1)), dim3(kSortBlock), 0, s, a.key_out, a.n, every_log2, a.rows, offsets);
  return launched("sort");
}

template <int DT>
void launch_embedding(const EmbeddingArgs& a, int id_dtype, hipStream_t s) {
  const unsigned per_group = kLookupWaves * kWave * kLookupVecs;
  const dim3 grid((a.vecs + per_group - 1) / per_group), block(kLookupWaves * kWave);
  const bool narrow = a.hidden < (uint32_t)vec_elems<DT>() || a.rows == 0;
  auto kernel = id_dtype == MCCL_I32 ? (narrow ? embedding_kernel<DT, int32_t, true> : embedding_kernel<DT, int32_t, false>)
                                     : (narrow ? embedding_kernel<DT, int64_t, true> : embedding_kernel<DT, int64_t, false>);
  hipLaunchKernelGGL(kernel, grid, block, 0, s, a);
}

// Below so many (row or piece, chunk of columns) pairs a wavefront has one pair and a row's chunks are spread over
// workgroups: then the time is that of the longest chain of loads (2000 tokens into 2000 x 7168 bf16 24 us
// against 38, 1500 into 600 x 4096 15 against 20).  From about there on it makes no difference (8192 tokens into
// 3000 x 4096 28 us both ways), and one wavefront takes two chunks, which halves the loads of indices.
constexpr uint32_t kGradSpread = 32768;
size_t grad_pieces(size_t n) { return n > (size_t)kGradPiece ? (n + kGradPiece - 1) / kGradPiece : 0; }

template <int DT, int OUT>
void launch_embedding_grad(EmbeddingGradArgs a, hipStream_t s) {
  constexpr uint32_t kChunk = kWave * vec_elems<DT>();
  const bool narrow = a.hidden < (uint32_t)vec_elems<DT>();
  const uint32_t chunks = (a.hidden + kChunk - 1) / kChunk, pieces = (uint32_t)grad_pieces(a.n);
  const bool spread = ((uint64_t)a.rows + pieces) * chunks < kGradSpread;
  const bool pairs = chunks > 4 && !spread;
  const uint32_t units = pairs ? (chunks + 1) / 2 : chunks;  // of one wavefront
  a.sharing_log2 = units >= 4 ? 2 : units >= 2 ? 1 : 0;
  const uint32_t per_group = kGradWaves >> a.sharing_log2;
  a.column_groups = spread ? (units + (1u << a.sharing_log2) - 1) >> a.sharing_log2 : 1;
  a.piece_groups = (pieces + per_group - 1) / per_group;
  a.row_groups = std::min(kMaxGroups, (a.rows + per_group - 1) / per_group);
  auto kernel = narrow ? embedding_grad_kernel<DT, OUT, 1, true> : pairs ? embedding_grad_kernel<DT, OUT, 2, false> : embedding_grad_kernel<DT, OUT, 1, false>;
  hipLaunchKernelGGL(kernel, dim3(a.piece_groups + a.row_groups, a.column_groups), dim3(kGradWaves * kWave), 0, s, a);
  auto join = narrow ? embedding_grad_join_kernel<DT, OUT, true> : embedding_grad_join_kernel<DT, OUT, false>;
  if (pieces) hipLaunchKernelGGL(join, dim3(pieces, chunks), dim3(kJoinWaves * kWave), 0, s, a);
}

template <int DT, bool GRAD, int LANES, int PER>
void launch_route(const RouterArgs& a, hipStream_t s) {
  const uint32_t per_group = kRouterWaves * (kWave / LANES);
  hipLaunchKernelGGL((GRAD ? router_grad_kernel<DT, LANES, PER> : router_kernel<DT, LANES, PER>),
                     dim3(std::min(kMaxGroups, (a.tokens + per_group - 1) / per_group)), dim3(kRouterWaves * kWave), 0, s, a);
}

// A batch takes 16 lanes per token, of 16 experts at most: 32768 tokens x 256 experts bf16 11.4 us and 11.2 for the
// gradient, against 18.4 and 13.0 with a wavefront per token; x 64 experts 6.2 and 5.3 against 13.6 and 9.2.  Few
// tokens are bound by one wavefront's time, which is shorter where it has one token and less per lane: 256 tokens x
// 256 experts 3.2 and 2.7 us against 3.9 and 3.7.  They meet at 4096 tokens (4.1 against 4.5, the gradient 4.1 against
// 3.5; 2048 tokens 4.0 against 3.6 and 3.9 against 2.9; 4096 x 128 experts 3.3 against 4.1).  16 experts of fp32 are a
// cache line's half per lane, which the gradient, reading and writing them, does slower than a wavefront per token (not
// normalised, 32768 x 256 18.7 us against 14.1), unlike 8 of them (x 128 10.1 against 11.7).
constexpr uint32_t kRouterBatch = 4096;

template <int DT, bool GRAD>
void launch_router(const RouterArgs& a, hipStream_t s) {
  constexpr bool kSixteen = !(GRAD && DT == MCCL_F32);  // experts per lane of 16 lanes, or at most 8
  if (a.tokens >= kRouterBatch && a.experts <= 16 * (kSixteen ? 16 : 8)) {
    if (a.experts <= 16) launch_route<DT, GRAD, 16, 1>(a, s);
    else if (a.experts <= 32) launch_route<DT, GRAD, 16, 2>(a, s);
    else if (a.experts <= 64) launch_route<DT, GRAD, 16, 4>(a, s);
    else if (a.experts <= 128) launch_route<DT, GRAD, 16, 8>(a, s);
    else if constexpr (kSixteen) launch_route<DT, GRAD, 16, 16>(a, s);
  } else if (a.experts <= 64) launch_route<DT, GRAD, 64, 1>(a, s);
  else if (a.experts <= 128) launch_route<DT, GRAD, 64, 2>(a, s);
  else if (a.experts <= 256) launch_route<DT, GRAD, 64, 4>(a, s);
  else if (a.experts <= 512) launch_route<DT, GRAD, 64, 8>(a, s);
  else if (a.experts <= 1024) launch_route<DT, GRAD, 64, 16>(a, s);
  else launch_route<DT, GRAD, 64, 64>(a, s);
}

int check_router(size_t tokens, size_t experts, int topk, int dtype) {
  if (!float_size(dtype)) return mccl_report_error(MCCL_ERR_UNSUPPORTED, "the router is defined for bf16, f16 and f32 logits");
  if (experts < 1 || experts > (size_t)kRouterMaxExperts)
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "expert count %zu outside [1, %d]", experts, kRouterMaxExperts);
  if (topk < 1 || topk > kRouterMaxTopk || (size_t)topk > experts)
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "topk %d outside [1, %d] or above the expert count %zu", topk, kRouterMaxTopk, experts);
  if (tokens > 0x7fffffffull) return mccl_report_error(MCCL_ERR_INVALID_ARG, "too many tokens");
  return MCCL_OK;
}

// How a layer is run, from its sizes alone (the routing is only known on the device).
struct LayerPlan {
  bool dense;      // layer_dense_kernel, or layer_in_kernel and layer_out_kernel
  uint32_t parts;  // of inter, in the second product
  size_t h_bytes, bytes;
};

// Pairs per expert above which the tokens go through LDS (layer_dense_kernel) instead of being read again by every
// workgroup.  Both ways, tokens spread evenly over experts that are all here: 8 experts of 4096 x 1792 with 8 / 12 / 16 / 24
// / 48 pairs each 76 / 76 / 89 / 112 / 202 us from memory and 75 / 79 / 81 / 90 / 109 through LDS; 32 experts of 2048 x 768
// with 8 / 12 / 16 / 24 pairs 68 / 84 / 98 / 136 and 69 / 72 / 76 / 87; 2 experts of 4096 x 8192 with 8 / 12 / 16 / 24 / 48
// pairs 69 / 75 / 79 / 98 / 180 and 86 / 91 / 88 / 89 / 95.  The pairs are those of all ranks: where only a part of the
// experts is here, the experts of this rank have fewer of them and the change comes too early.
constexpr size_t kDensePairs = 12;
LayerPlan plan_layer(size_t pairs, size_t experts, size_t hidden, size_t inter) {
  LayerPlan p{};
  p.dense = pairs > kDensePairs * experts || pairs > kFewMaxPairs;
  p.h_bytes = up16(pairs * inter * 4);
  p.bytes = p.h_bytes;
  if (p.dense) {
    const size_t groups = (hidden + kDenseOutRows - 1) / kDenseOutRows * experts;
    const size_t cols = kDenseSteps * kStepCols, chunks = (inter + cols - 1) / cols;
    // parts that give every compute unit the two workgroups it has room for; more are joined at a loss (24 pairs on each of
    // 32 experts of 2048 x 768 87 us, with twice the parts 92) or gain little (160 tokens on 8 of 4096 x 7168 325 and 314)
    const size_t wanted = std::min<size_t>({chunks, 8, (512 + groups - 1) / groups}), per = (chunks + wanted - 1) / wanted;
    p.parts = (uint32_t)((chunks + per - 1) / per);
    p.bytes += p.parts * pairs * hidden * sizeof(float);
  } else {
    // as many parts as give 16 wavefronts something to do, of 4 steps or more: where few experts can be chosen,
    // wavefronts would have nothing to do (8 tokens on one of 2 experts of 14336: 65 us against 88 with one part),
    // while parts of few steps only add joining (5 tokens x 3 experts, inter 200: 9.0 against 12.7)
    p.parts = (uint32_t)std::max<size_t>(1, std::min<size_t>((inter + kStepCols - 1) / kStepCols / 4, 16 / std::min(pairs, experts)));
  }
  return p;
}

template <int DT>
int launch_dense(const LayerArgs& a, hipStream_t s) {
  const uint32_t in_tiles = (a.inter + kDenseInRows - 1) / kDenseInRows * a.experts;
  const uint32_t out_tiles = (a.hidden + kDenseOutRows - 1) / kDenseOutRows * a.experts * a.parts;
  hipLaunchKernelGGL((layer_dense_kernel<DT, true>), dim3(in_tiles), dim3(kDenseBlock), 0, s, a);
  hipLaunchKernelGGL((layer_dense_kernel<DT, false>), dim3(out_tiles), dim3(kDenseBlock), 0, s, a);
  hipLaunchKernelGGL(layer_join_kernel<DT>, dim3((a.hidden / 4 + 255) / 256, a.tokens), dim3(256), 0, s, a);
  return launched("moe layer");
}

// Whether a workgroup of the second product takes 16 rows with 8 wavefronts, instead of 8 rows with 16: it
// reads the tokens half as often, if it fills the 256 compute units evenly (1 token, hidden 4096: 36.4 us
// against 38.9; 64 tokens x 128 experts 322 against 361; but hidden 5120, 320 workgroups, 244 against 237).
bool wide_out(size_t hidden, size_t pairs) {
  const size_t groups = (hidden + 15) / 16, rounds = (groups + 255) / 256;
  return pairs <= 1024 && groups * 5 >= rounds * 256 * 4;
}

template <int DT, int NW, int WAVES>
int launch_layer_out(const LayerArgs& a, hipStream_t s) {
  const uint32_t rows = NW * kSetRows, bytes = layer_out_lds(a.pairs, a.experts, a.parts, rows, WAVES).bytes;
  if (bytes > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)layer_out_kernel<DT, NW, WAVES>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != hipSuccess) return mccl_report_error(MCCL_ERR_HIP, "hipFuncSetAttribute failed: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL((layer_out_kernel<DT, NW, WAVES>), dim3((a.hidden + rows - 1) / rows), dim3(WAVES * kWave), bytes, s, a);
  return MCCL_OK;
}

template <int DT>
int launch_layer(const LayerArgs& a, bool dense, hipStream_t s) {
  if (dense) return launch_dense<DT>(a, s);
  const dim3 in_grid((a.inter + kInRows - 1) / kInRows, a.by_pair ? a.pairs : a.experts), in_block(kInWaves * kWave);
  // the fewest sums that serve all tokens of an expert at once (40 tokens, 10 on each of 23 experts of 4016 x 624: 115 us
  // with sums for 32 tokens, 117 for 16; 64 tokens, 4 on each of 128: 322 and 330)
  if (a.tokens <= 8) hipLaunchKernelGGL((layer_in_kernel<DT, 8>), in_grid, in_block, 0, s, a);
  else if (a.tokens <= 16) hipLaunchKernelGGL((layer_in_kernel<DT, 16>), in_grid, in_block, 0, s, a);
  else hipLaunchKernelGGL((layer_in_kernel<DT, 32>), in_grid, in_block, 0, s, a);
  const int rc = wide_out(a.hidden, a.pairs) ? launch_layer_out<DT, 2, 8>(a, s) : launch_layer_out<DT, 1, 16>(a, s);
  return rc != MCCL_OK ? rc : launched("moe layer");
}

}  // namespace

extern "C" {

int mccl_embedding(const void* table, size_t rows, const void* ids, int id_dtype, size_t n, int64_t first_row, size_t hidden,
                   float scale, int dtype, void* out, void* stream) {
  const size_t es = float_size(dtype);
  if (!es) return mccl_report_error(MCCL_ERR_UNSUPPORTED, "embedding is defined for bf16, f16 and f32");
  if (n == 0 || hidden == 0) return MCCL_OK;
  int rc = check_ids(ids, id_dtype);
  if (rc == MCCL_OK) rc = check_rows(first_row, rows);
  if (rc != MCCL_OK) return rc;
  if (!out || (rows && !table)) return mccl_report_error(MCCL_ERR_INVALID_ARG, "null pointer");
  if (misaligned(table, es) || misaligned(out, es)) return mccl_report_error(MCCL_ERR_INVALID_ARG, "table or output not aligned to its element size");
  if (hidden > kMaxHidden || n > 0x7fffffffull) return mccl_report_error(MCCL_ERR_INVALID_ARG, "row or id list too long");
  const size_t id_bytes = n * (id_dtype == MCCL_I32 ? 4 : 8);
  if (ranges_overlap(out, n * hidden * es, table, rows * hidden * es) || ranges_overlap(out, n * hidden * es, ids, id_bytes))
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "output overlaps the table or the ids");
  EmbeddingArgs a{};
  a.table = (const char*)table;
  a.first_row = first_row;
  a.rows = rows;
  a.hidden = (uint32_t)hidden;
  a.vecs_per_row = (uint32_t)((hidden * es + 15) / 16);
  a.scale = scale;
  // vectors are counted in 32 bits on the device: a longer list is looked up in parts
  const size_t most = 0x80000000ull / a.vecs_per_row;
  for (size_t i = 0; i < n; i += most) {
    const size_t part = std::min(most, n - i);
    a.ids = (const char*)ids + i * (id_dtype == MCCL_I32 ? 4 : 8);
    a.out = (char*)out + i * hidden * es;
    a.vecs = (uint32_t)(part * a.vecs_per_row);
    switch (dtype) {
      case MCCL_BF16: launch_embedding<MCCL_BF16>(a, id_dtype, (hipStream_t)stream); break;
      case MCCL_F16: launch_embedding<MCCL_F16>(a, id_dtype, (hipStream_t)stream); break;
      default: launch_embedding<MCCL_F32>(a, id_dtype, (hipStream_t)stream); break;
    }
  }
  return launched("embedding");
}

size_t mccl_sort_ids_workspace(size_t n) { return plan_sort(n).bytes; }

int mccl_sort_ids(const void* ids, int id_dtype, size_t n, int64_t first_row, size_t rows, void* workspace, size_t workspace_bytes,
                  int64_t* order, int64_t* offsets, void* stream) {
  if (id_dtype != MCCL_I32 && id_dtype != MCCL_I64) return mccl_report_error(MCCL_ERR_UNSUPPORTED, "ids are int32 or int64");
  if (n > 0x7fffffffull) return mccl_report_error(MCCL_ERR_INVALID_ARG, "too many ids");
  if (rows > 0x7fffffffull) return mccl_report_error(MCCL_ERR_INVALID_ARG, "too many rows");
  if (!offsets || misaligned(offsets, 8)) return mccl_report_error(MCCL_ERR_INVALID_ARG, "offsets pointer is null or misaligned");
  int rc = check_rows(first_row, rows);
  if (rc != MCCL_OK) return rc;
  if (n) {
    rc = check_ids(ids, id_dtype);
    if (rc != MCCL_OK) return rc;
    if (!order || misaligned(order, 8)) return mccl_report_error(MCCL_ERR_INVALID_ARG, "order pointer is null or misaligned");
  }
  const size_t id_bytes = n * (id_dtype == MCCL_I32 ? 4 : 8), need = plan_sort(n).bytes;
  if (need && (!workspace || misaligned(workspace, 16) || workspace_bytes < need))
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "workspace is null, not 16-byte aligned or smaller than %zu bytes", need);
  const void* part[] = {ids, order, offsets, workspace};
  const size_t bytes[] = {id_bytes, n * 8, (rows + 1) * 8, need};
  for (int i = 0; i < 4; ++i)
    for (int j = i + 1; j < 4; ++j)
      if (ranges_overlap(part[i], bytes[i], part[j], bytes[j]))
        return mccl_report_error(MCCL_ERR_INVALID_ARG, "ids, order, offsets and workspace must not overlap");
  hipStream_t s = (hipStream_t)stream;
  if (id_dtype == MCCL_I32) return launch_sort((const int32_t*)ids, n, first_row, rows, (char*)workspace, order, offsets, s);
  return launch_sort((const int64_t*)ids, n, first_row, rows, (char*)workspace, order, offsets, s);
}

size_t mccl_embedding_grad_workspace(size_t n, size_t hidden) { return grad_pieces(n) * 2 * (hidden * sizeof(float) + sizeof(uint32_t)); }

int mccl_embedding_grad(const void* grad, const int64_t* order, const int64_t* offsets, size_t n, size_t rows, size_t hidden,
                        float scale, int dtype, void* out, int out_dtype, int accumulate, void* workspace, size_t workspace_bytes,
                        void* stream) {
  const size_t es = float_size(dtype), os = float_size(out_dtype);
  if (!es || !os || (out_dtype != dtype && out_dtype != MCCL_F32))
    return mccl_report_error(MCCL_ERR_UNSUPPORTED, "embedding_grad takes bf16, f16 or f32 and writes the same type or f32");
  if (rows == 0 || hidden == 0) return MCCL_OK;
  if (hidden > kMaxHidden || n > kMaxGradTokens || rows > 0x7fffffffull)
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "row, id list or table too long");
  if (!offsets || !out || (n && (!grad || !order))) return mccl_report_error(MCCL_ERR_INVALID_ARG, "null pointer");
  if (misaligned(grad, es) || misaligned(out, os)) return mccl_report_error(MCCL_ERR_INVALID_ARG, "gradient or output not aligned to its element size");
  if (misaligned(order, 8) || misaligned(offsets, 8)) return mccl_report_error(MCCL_ERR_INVALID_ARG, "order or offsets misaligned");
  const size_t need = mccl_embedding_grad_workspace(n, hidden);
  if (need && (!workspace || misaligned(workspace, 16) || workspace_bytes < need))
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "workspace is null, not 16-byte aligned or smaller than %zu bytes", need);
  const size_t out_bytes = rows * hidden * os;
  const void* part[] = {grad, order, offsets};
  const size_t bytes[] = {n * hidden * es, n * 8, (rows + 1) * 8};
  for (int i = 0; i < 3; ++i)
    if (ranges_overlap(out, out_bytes, part[i], bytes[i]) || ranges_overlap(workspace, need, part[i], bytes[i]))
      return mccl_report_error(MCCL_ERR_INVALID_ARG, "output or workspace overlaps an input");
  if (ranges_overlap(out, out_bytes, workspace, need)) return mccl_report_error(MCCL_ERR_INVALID_ARG, "output overlaps the workspace");
  EmbeddingGradArgs a{};
  a.grad = (const char*)grad;
  a.order = order;
  a.offsets = offsets;
  a.out = (char*)out;
  a.partial = (float*)workspace;
  a.long_row = (uint32_t*)(a.partial + grad_pieces(n) * 2 * hidden);
  a.rows = (uint32_t)rows;
  a.n = (uint32_t)n;
  a.hidden = (uint32_t)hidden;
  a.scale = scale;
  a.accumulate = accumulate ? 1 : 0;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MCCL_F32) launch_embedding_grad<MCCL_F32, MCCL_F32>(a, s);
  else if (dtype == MCCL_BF16 && out_dtype == MCCL_BF16) launch_embedding_grad<MCCL_BF16, MCCL_BF16>(a, s);
  else if (dtype == MCCL_BF16) launch_embedding_grad<MCCL_BF16, MCCL_F32>(a, s);
  else if (out_dtype == MCCL_F16) launch_embedding_grad<MCCL_F16, MCCL_F16>(a, s);
  else launch_embedding_grad<MCCL_F16, MCCL_F32>(a, s);
  return launched("embedding gradient");
}

int mccl_moe_route(const void* logits, size_t tokens, size_t experts, int topk, int normalize, int dtype, int32_t* expert_ids,
                   float* weights, void* stream) {
  int rc = check_router(tokens, experts, topk, dtype);
  if (rc != MCCL_OK || tokens == 0) return rc;
  const size_t es = float_size(dtype), pairs = tokens * (size_t)topk;
  if (!logits || !expert_ids || !weights) return mccl_report_error(MCCL_ERR_INVALID_ARG, "null pointer");
  if (misaligned(logits, es) || misaligned(expert_ids, 4) || misaligned(weights, 4))
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "logits, ids or weights not aligned to their element size");
  if (ranges_overlap(expert_ids, pairs * 4, logits, tokens * experts * es) || ranges_overlap(weights, pairs * 4, logits, tokens * experts * es) ||
      ranges_overlap(expert_ids, pairs * 4, weights, pairs * 4))
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "ids, weights and logits must not overlap");
  RouterArgs a{};
  a.logits = (const char*)logits;
  a.ids = expert_ids;
  a.weights = weights;
  a.tokens = (uint32_t)tokens;
  a.experts = (uint32_t)experts;
  a.topk = (uint32_t)topk;
  a.normalize = normalize ? 1 : 0;
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case MCCL_BF16: launch_router<MCCL_BF16, false>(a, s); break;
    case MCCL_F16: launch_router<MCCL_F16, false>(a, s); break;
    default: launch_router<MCCL_F32, false>(a, s); break;
  }
  return launched("router");
}

int mccl_moe_route_grad(const float* grad_weights, const void* logits, const int32_t* expert_ids, size_t tokens, size_t experts, int topk,
                        int normalize, int dtype, void* grad_logits, void* stream) {
  int rc = check_router(tokens, experts, topk, dtype);
  if (rc != MCCL_OK || tokens == 0) return rc;
  const size_t es = float_size(dtype), pairs = tokens * (size_t)topk, bytes = tokens * experts * es;
  if (!logits || !expert_ids || !grad_weights || !grad_logits) return mccl_report_error(MCCL_ERR_INVALID_ARG, "null pointer");
  if (misaligned(logits, es) || misaligned(grad_logits, es) || misaligned(expert_ids, 4) || misaligned(grad_weights, 4))
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "logits, ids or gradients not aligned to their element size");
  if (ranges_overlap(grad_logits, bytes, logits, bytes) || ranges_overlap(grad_logits, bytes, expert_ids, pairs * 4) ||
      ranges_overlap(grad_logits, bytes, grad_weights, pairs * 4))
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "the gradient overlaps an input");
  RouterArgs a{};
  a.logits = (const char*)logits;
  a.chosen = expert_ids;
  a.grad_weights = grad_weights;
  a.grad_logits = (char*)grad_logits;
  a.tokens = (uint32_t)tokens;
  a.experts = (uint32_t)experts;
  a.topk = (uint32_t)topk;
  a.normalize = normalize ? 1 : 0;
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case MCCL_BF16: launch_router<MCCL_BF16, true>(a, s); break;
    case MCCL_F16: launch_router<MCCL_F16, true>(a, s); break;
    default: launch_router<MCCL_F32, true>(a, s); break;
  }
  return launched("router gradient");
}

size_t mccl_moe_layer_workspace(size_t tokens, int topk, size_t experts, size_t hidden, size_t inter) {
  if (topk < 1 || tokens == 0 || experts == 0 || hidden == 0 || inter == 0) return 0;
  return plan_layer(tokens * (size_t)topk, experts, hidden, inter).bytes;
}

int mccl_moe_layer(const void* x, const void* w_in, const void* w_out, const int32_t* expert_ids, const float* weights, size_t tokens,
                   int topk, size_t experts, int64_t first_expert, size_t hidden, size_t inter, int activation, int dtype, void* out,
                   void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != MCCL_BF16 && dtype != MCCL_F16) return mccl_report_error(MCCL_ERR_UNSUPPORTED, "moe_layer is defined for bf16 and f16");
  if (activation != MCCL_ACT_SILU && activation != MCCL_ACT_GELU) return mccl_report_error(MCCL_ERR_INVALID_ARG, "unknown activation %d", activation);
  if (tokens > (size_t)kLayerMaxTokens)
    return mccl_report_error(MCCL_ERR_UNSUPPORTED, "%zu tokens: moe_layer is for at most %d; dispatch larger batches", tokens, kLayerMaxTokens);
  if (topk < 1 || topk > kRouterMaxTopk || tokens * (size_t)topk > (size_t)kLayerMaxPairs)
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "topk %d outside [1, %d], or more than %d (token, expert) pairs", topk, kRouterMaxTopk, kLayerMaxPairs);
  if (experts < 1 || experts > (size_t)kRouterMaxExperts)
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "expert count %zu outside [1, %d]", experts, kRouterMaxExperts);
  if (tokens == 0 || hidden == 0) return MCCL_OK;
  if (hidden % 8 || inter % 8 || inter == 0) return mccl_report_error(MCCL_ERR_UNSUPPORTED, "moe_layer needs hidden and inter that are multiples of 8");
  if (hidden > kLayerMaxColumns || inter > kLayerMaxColumns || 4 * inter * hidden > kLayerMaxExpert)
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "hidden or inter above %zu, or an expert's w_in above %zu bytes", kLayerMaxColumns, kLayerMaxExpert);
  if (!x || !w_in || !w_out || !expert_ids || !weights || !out) return mccl_report_error(MCCL_ERR_INVALID_ARG, "null pointer");
  if (misaligned(x, 16) || misaligned(w_in, 16) || misaligned(w_out, 16) || misaligned(out, 16))
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "x, the weights or the output are not 16-byte aligned");
  if (misaligned(expert_ids, 4) || misaligned(weights, 4)) return mccl_report_error(MCCL_ERR_INVALID_ARG, "expert ids or weights misaligned");
  const size_t pairs = tokens * (size_t)topk, row = tokens * hidden * 2;
  const LayerPlan plan = plan_layer(pairs, experts, hidden, inter);
  if (plan.dense && std::max((inter + kDenseInRows - 1) / kDenseInRows, (hidden + kDenseOutRows - 1) / kDenseOutRows * plan.parts) * experts > kMaxDenseTiles)
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "%zu experts of %zu x %zu are too many rows for one launch", experts, hidden, inter);
  const size_t need = plan.bytes;
  if (!workspace || misaligned(workspace, 16) || workspace_bytes < need)
    return mccl_report_error(MCCL_ERR_INVALID_ARG, "workspace is null, not 16-byte aligned or smaller than %zu bytes", need);
  const void* part[] = {x, w_in, w_out, expert_ids, weights};
  const size_t bytes[] = {row, experts * 2 * inter * hidden * 2, experts * hidden * inter * 2, pairs * 4, pairs * 4};
  for (int i = 0; i < 5; ++i)
    if (ranges_overlap(out, row, part[i], bytes[i]) || ranges_overlap(workspace, need, part[i], bytes[i]))
      return mccl_report_error(MCCL_ERR_INVALID_ARG, "output or workspace overlaps an input");
  if (ranges_overlap(out, row, workspace, need)) return mccl_report_error(MCCL_ERR_INVALID_ARG, "output overlaps the workspace");
  LayerArgs a{};
  a.x = (const char*)x;
  a.w_in = (const char*)w_in;
  a.w_out = (const char*)w_out;
  a.ids = expert_ids;
  a.weights = weights;
  a.h = (char*)workspace;
  a.y = (float*)((char*)workspace + plan.h_bytes);
  a.out = (char*)out;
  a.parts = plan.parts;
  a.tokens = (uint32_t)tokens;
  a.topk = (uint32_t)topk;
  a.pairs = (uint32_t)pairs;
  a.experts = (uint32_t)experts;
  a.hidden = (uint32_t)hidden;
  a.inter = (uint32_t)inter;
  a.first_expert = first_expert;
  a.by_pair = pairs < experts ? 1 : 0;
  a.activation = activation;
  hipStream_t s = (hipStream_t)stream;
  return dtype == MCCL_BF16 ? launch_layer<MCCL_BF16>(a, plan.dense, s) : launch_layer<MCCL_F16>(a, plan.dense, s);
}

}  // extern "C"
