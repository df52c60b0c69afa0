// C ABI of the operators that route and move tokens (declared in include/avey_b200.h):
// argument checks, workspace layout and the launches of route_kernels.cuh,
// sort_kernels.cuh and rows_kernels.cuh.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstddef>
#include <mutex>

#include "avey_b200.h"
#include "host_api.h"
#include "launch_chain.h"
#include "rows_kernels.cuh"
#include "route_kernels.cuh"
#include "sort_kernels.cuh"

namespace {

using avey_host::Chain;

int fail(int code, const char* msg) { return avey_host::set_error(code, msg); }
int done(int rc) { return rc == AVEY_OK ? avey_host::clear_error() : rc; }

uint64_t up256(uint64_t x) { return (x + 255u) & ~uint64_t(255); }
uintptr_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }
int size_of(int dtype) { return dtype == AVEY_F32 ? 4 : 2; }
bool known(int dtype) { return dtype == AVEY_F32 || dtype == AVEY_F16 || dtype == AVEY_BF16; }

int check_workspace(const void* ws, uint64_t have, uint64_t need) {
  if (need == 0) return AVEY_OK;
  if (!ws || have < need) return fail(AVEY_ERR_ARGUMENT, "workspace is smaller than the call's workspace size");
  if ((address(ws) & 255u) != 0) return fail(AVEY_ERR_ARGUMENT, "workspace must be 256-byte aligned");
  return AVEY_OK;
}

unsigned blocks_for(int64_t items, int per) {
  return static_cast<unsigned>(
      std::max<int64_t>(1, std::min<int64_t>((items + per - 1) / per, avey_host::multiprocessors() * 32ll)));
}

// ------------------------------------------------------------------ routing

int validate(const AveyRouteParams* p, bool backward) {
  if (!p) return fail(AVEY_ERR_ARGUMENT, "params is NULL");
  if (p->struct_size != sizeof(AveyRouteParams))
    return fail(AVEY_ERR_ARGUMENT, "struct_size does not match sizeof(AveyRouteParams)");
  if (!known(p->dtype)) return fail(AVEY_ERR_ARGUMENT, "logits are f32, f16 or bf16");
  if (p->score != AVEY_SCORE_SOFTMAX && p->score != AVEY_SCORE_SIGMOID) return fail(AVEY_ERR_ARGUMENT, "unknown score");
  if (p->tokens < 0 || p->tokens > (1 << 30) || p->experts < 1 || p->experts > avey::kRtMaxExperts)
    return fail(AVEY_ERR_ARGUMENT, "tokens must be in [0, 2^30] and experts in [1, 1024]");
  if (p->groups < 1 || p->groups > avey::kRtMaxGroups || p->experts % p->groups != 0 || p->top_groups < 1 ||
      p->top_groups > p->groups || (p->group_best != 1 && p->group_best != 2))
    return fail(AVEY_ERR_ARGUMENT,
                "groups must divide the experts and be in [1, 32], top_groups in [1, groups], group_best 1 or 2");
  if (p->k < 1 || p->k > avey::kRtMaxK || p->k > p->experts / p->groups * p->top_groups)
    return fail(AVEY_ERR_ARGUMENT, "k must be in [1, 32] and no more than the experts of top_groups groups");
  if (!(p->scale > -1e30 && p->scale < 1e30)) return fail(AVEY_ERR_ARGUMENT, "scale must be finite");
  const uintptr_t element = size_of(p->dtype) - 1;
  if (((address(p->logits) | address(p->dlogits)) & element) != 0 ||
      ((address(p->bias) | address(p->weights) | address(p->chosen) | address(p->dweights)) & 3u) != 0)
    return fail(AVEY_ERR_ARGUMENT, "arrays must be aligned to their elements");
  if (p->tokens == 0) return AVEY_OK;
  if (!p->logits || !p->weights || !p->chosen) return fail(AVEY_ERR_ARGUMENT, "logits, weights and chosen are required");
  if (p->logits_ld < p->experts) return fail(AVEY_ERR_ARGUMENT, "strides must cover the rows");
  if (backward && (!p->dweights || !p->dlogits))
    return fail(AVEY_ERR_ARGUMENT, "dweights and dlogits are required");
  return AVEY_OK;
}

// Experts of a lane: `lanes` of a token's each take R of them.
template <typename T, int R>
int launch_route(const avey::RtArgs& q, bool backward, int lanes, Chain& chain) {
  const int64_t tokens = 32 * avey::kRtWarps / lanes;
  const dim3 grid(static_cast<unsigned>((q.tokens + tokens - 1) / tokens));
  if (backward)
    return chain.launch("route gradient", avey::route_backward<T, R>, grid, 32 * avey::kRtWarps,
                        avey::kRtWarps * 32 * (R + 1) * 4, 1, q, lanes);
  if (!q.bias && q.groups == 1)
    return chain.launch("route", avey::route_plain<T, R>, grid, 32 * avey::kRtWarps, 0, 1, q, lanes);
  const dim3 some(std::min<unsigned>(grid.x, avey_host::multiprocessors() * 8u));
  return chain.launch("route", avey::route_forward<T, R>, some, 32 * avey::kRtWarps, 0, 1, q);
}

template <typename T>
int route(const AveyRouteParams* p, bool backward, cudaStream_t stream) {
  avey::RtArgs q{};
  q.tokens = p->tokens;
  q.experts = static_cast<int>(p->experts);
  q.k = p->k;
  q.groups = p->groups;
  q.top_groups = p->top_groups;
  q.group_best = p->group_best;
  q.softmax = p->score == AVEY_SCORE_SOFTMAX;
  q.renormalize = p->renormalize != 0;
  q.scale = static_cast<float>(p->scale);
  q.logits = p->logits;
  q.ld = p->logits_ld;
  q.vec = ((address(p->logits) | static_cast<uint64_t>(p->logits_ld) * sizeof(T)) & 15u) == 0;
  q.bias = p->bias;
  q.weights = p->weights;
  q.chosen = p->chosen;
  q.dweights = p->dweights;
  q.dlogits = p->dlogits;
  q.dvec = ((address(p->dlogits) | static_cast<uint64_t>(p->experts) * sizeof(T)) & 15u) == 0;
  Chain chain{stream};
  // A whole warp for the choice by scores; else as many lanes as have 16 experts each, or
  // one of the chosen.
  int lanes = 32;
  if (backward || (!q.bias && q.groups == 1)) {
    lanes = 1;
    while (lanes < 32 && (lanes * 16 < q.experts || lanes < q.k)) lanes *= 2;
  }
  const int per = (q.experts + lanes - 1) / lanes;
  if (per <= 1) return launch_route<T, 1>(q, backward, lanes, chain);
  if (per <= 2) return launch_route<T, 2>(q, backward, lanes, chain);
  if (per <= 4) return launch_route<T, 4>(q, backward, lanes, chain);
  if (per <= 8) return launch_route<T, 8>(q, backward, lanes, chain);
  if (per <= 16) return launch_route<T, 16>(q, backward, lanes, chain);
  return launch_route<T, 32>(q, backward, lanes, chain);
}

int run_route(const AveyRouteParams* p, bool backward, void* stream) {
  int rc = validate(p, backward);
  if (rc != AVEY_OK) return rc;
  rc = avey_host::device_ok();
  if (rc != AVEY_OK || p->tokens == 0) return done(rc);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return done(p->dtype == AVEY_F32   ? route<float>(p, backward, s)
              : p->dtype == AVEY_F16 ? route<__half>(p, backward, s)
                                     : route<__nv_bfloat16>(p, backward, s));
}

// ------------------------------------------------------------------ sorting

// Blocks of a pass over n entries, and the entries of each (whole warps' steps).
int64_t sort_run(int64_t n) {
  if (n <= avey::kStOneBlock) return n;
  const int64_t share = (n + avey_host::multiprocessors() - 1) / avey_host::multiprocessors();
  return std::max<int64_t>(avey::kStRun, (share + 511) / 512 * 512);
}
int64_t sort_blocks(int64_t n) {
  const int64_t run = sort_run(n);
  return n ? (n + run - 1) / run : 1;
}
uint64_t count_bytes(int64_t n, int buckets) {
  const int64_t b = sort_blocks(n);
  return b > 1 ? up256(static_cast<uint64_t>(b) * buckets * 4) : 0;
}

// The kernels' shared memory, past what a launch has by itself, once per device.
int sort_opt_in() {
  constexpr int kMaxDevices = 64;
  static std::once_flag once[kMaxDevices];
  static cudaError_t err[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
    return fail(AVEY_ERR_CUDA, "no current device");
  std::call_once(once[dev], [dev] {
    err[dev] = cudaFuncSetAttribute(avey::st_count, cudaFuncAttributeMaxDynamicSharedMemorySize, avey::kStSmem);
    if (err[dev] == cudaSuccess)
      err[dev] = cudaFuncSetAttribute(avey::st_place, cudaFuncAttributeMaxDynamicSharedMemorySize, avey::kStSmem);
  });
  return err[dev] == cudaSuccess ? AVEY_OK : fail(AVEY_ERR_CUDA, cudaGetErrorString(err[dev]));
}

int sort_smem(int buckets) { return (avey::kStWarps + 1) * buckets * 4; }
// Blocks beside a sort's that write `bytes` of zeros.
int zero_blocks(int64_t bytes) {
  return static_cast<int>(std::min<int64_t>((bytes + 65535) / 65536, avey_host::multiprocessors() * 2ll));
}

// One pass over many blocks. `counted`: the pass before has counted for this one.
int launch_pass(avey::StArgs& q, Chain& chain, bool counted = false) {
  const int opted = sort_opt_in();
  if (opted != AVEY_OK) return opted;
  q.run = std::max<int64_t>(1, sort_run(q.n));
  q.blocks = static_cast<int>(sort_blocks(q.n));
  if (q.blocks > 1 && !counted) {
    const int rc = chain.launch("sort counts", avey::st_count, dim3(q.blocks), avey::kStThreads, sort_smem(q.buckets),
                                1, q);
    if (rc != AVEY_OK) return rc;
  }
  const dim3 grid(static_cast<unsigned>(q.blocks + zero_blocks(q.zero_bytes)));
  return chain.launch("sort", avey::st_place, grid, avey::kStThreads, sort_smem(q.buckets), 1, q);
}

int validate(const AveyArrangeParams* p) {
  if (!p) return fail(AVEY_ERR_ARGUMENT, "params is NULL");
  if (p->struct_size != sizeof(AveyArrangeParams))
    return fail(AVEY_ERR_ARGUMENT, "struct_size does not match sizeof(AveyArrangeParams)");
  if (p->index_bits != 32 && p->index_bits != 64) return fail(AVEY_ERR_ARGUMENT, "expert numbers have 32 or 64 bits");
  if (p->count < 0 || p->count > (1ll << 30) || p->experts < 1 || p->experts > avey::kRtMaxExperts)
    return fail(AVEY_ERR_ARGUMENT, "count must be in [0, 2^30] and experts in [1, 1024]");
  if ((address(p->chosen) & (p->index_bits / 8 - 1)) != 0 || ((address(p->slots) | address(p->offsets)) & 3u) != 0)
    return fail(AVEY_ERR_ARGUMENT, "arrays must be aligned to their elements");
  if (!p->offsets || (p->count > 0 && (!p->chosen || !p->slots)))
    return fail(AVEY_ERR_ARGUMENT, "chosen, slots and offsets are required");
  return AVEY_OK;
}

// ------------------------------------------------------------------ rows

int validate(const AveyRowsParams* p, int what) {
  if (!p) return fail(AVEY_ERR_ARGUMENT, "params is NULL");
  // (The block once ended before its workspace.)
  if (p->struct_size != sizeof(AveyRowsParams) && p->struct_size != offsetof(AveyRowsParams, workspace))
    return fail(AVEY_ERR_ARGUMENT, "struct_size does not match sizeof(AveyRowsParams)");
  if (!known(p->dtype)) return fail(AVEY_ERR_ARGUMENT, "rows are f32, f16 or bf16");
  if (p->tokens < 0 || p->k < 1 || p->k > avey::kRwMaxK || p->tokens > (1ll << 30) / p->k || p->width < 1 ||
      p->width > (1 << 22))
    return fail(AVEY_ERR_ARGUMENT, "k must be in [1, 32], tokens x k up to 2^30 and width in [1, 2^22]");
  const uintptr_t element = size_of(p->dtype) - 1;
  if (((address(p->x) | address(p->rows) | address(p->out) | address(p->drows)) & element) != 0 ||
      ((address(p->slots) | address(p->weights) | address(p->dweights)) & 3u) != 0)
    return fail(AVEY_ERR_ARGUMENT, "arrays must be aligned to their elements");
  if (p->tokens == 0) return AVEY_OK;
  if (!p->slots) return fail(AVEY_ERR_ARGUMENT, "slots is required");
  if ((p->x && p->x_ld < p->width) || (p->rows && p->rows_ld < p->width))
    return fail(AVEY_ERR_ARGUMENT, "strides must cover the rows");
  if (what == 0 && (!p->x || !p->rows)) return fail(AVEY_ERR_ARGUMENT, "x and rows are required");
  if (what == 1 && (!p->rows || !p->out)) return fail(AVEY_ERR_ARGUMENT, "rows and out are required");
  if (what == 2 && (!p->x || !p->weights || (p->dweights && !p->rows)))
    return fail(AVEY_ERR_ARGUMENT, "x (the gradient of out), weights and, for dweights, rows are required");
  return AVEY_OK;
}

// Whether places that no slot names are cleared (a block that ends before its workspace had no such
// field), and the workspace for it.
bool clears(const AveyRowsParams* p) { return p->struct_size == sizeof(AveyRowsParams) && p->clear != 0; }
uint64_t clear_bytes(const AveyRowsParams* p) {
  const int64_t places = p->tokens * p->k;
  return clears(p) && places > avey::kRwBlankPlaces ? static_cast<uint64_t>(places) * 4 : 0;
}

// Bytes of an access that all rows are whole multiples of.
int access_bytes(int size, int64_t width, std::initializer_list<const void*> bases,
                 std::initializer_list<int64_t> strides) {
  uint64_t all = static_cast<uint64_t>(width) * size;
  for (const void* b : bases) all |= address(b);
  for (int64_t s : strides) all |= static_cast<uint64_t>(s) * size;
  return (all & 15u) == 0 ? 16 : (all & 3u) == 0 ? 4 : size;
}

// Lanes that take a row: as many as it has accesses, up to a warp.
int part_lanes(int64_t width, int per) {
  int lanes = 1;
  while (lanes < 32 && lanes * per < width) lanes *= 2;
  return lanes;
}

template <typename T, int N, int HOLD>
int launch_combine(const avey::RwArgs& q, int what, int lanes, Chain& chain) {
  const int64_t tokens = avey::kRwThreads / lanes;
  const dim3 grid(static_cast<unsigned>(
      std::min<int64_t>((q.tokens + tokens - 1) / tokens,
                        avey_host::multiprocessors() * static_cast<int64_t>(avey::rw_blocks(HOLD))) + q.blanks));
  if (what == 1) return chain.launch("combine", avey::rw_combine<T, N, HOLD>, grid, avey::kRwThreads, 0, 1, q, lanes);
  return chain.launch("combine gradient", avey::rw_combine_backward<T, N, HOLD>, grid, avey::kRwThreads, 0, 1, q, lanes);
}

template <typename T, int N>
int launch_moves(const avey::RwArgs& q, int what, Chain& chain) {
  if (what == 0)
    return chain.launch("dispatch", avey::rw_dispatch<T, N>,
                        dim3(q.blanks + blocks_for(q.tokens * (q.width / N), 256)), 256, 0, 1, q);
  if constexpr (sizeof(T) * N == 16) {
    const int lanes = part_lanes(q.width, N);
    switch ((q.width / N + lanes - 1) / lanes) {
      case 1: return launch_combine<T, N, 1>(q, what, lanes, chain);
      case 3: return launch_combine<T, N, 3>(q, what, lanes, chain);
      case 4: return launch_combine<T, N, 4>(q, what, lanes, chain);
      default: return launch_combine<T, N, 2>(q, what, lanes, chain);
    }
  }
  return launch_combine<T, N, 2>(q, what, part_lanes(q.width, N), chain);
}

template <typename T, int N>
int launch_rows(const avey::RwArgs& q, int what, Chain& chain) {
  const int rc = launch_moves<T, N>(q, what, chain);
  if (rc != AVEY_OK || !q.namer) return rc;
  const int places = static_cast<int>(q.tokens * q.k);
  T* rows = static_cast<T*>(what == 0 ? q.rows : q.out);
  return chain.launch("clear places", avey::rw_clear<T, N>, dim3(blocks_for(places, 256)), 256, 0, 1, q.slots, q.namer,
                      places, rows, what == 0 ? q.rows_ld : static_cast<int64_t>(q.width), q.width);
}

// what: 0 dispatch, 1 combine, 2 combine's backward.
int run_rows(const AveyRowsParams* p, int what, void* stream) {
  int rc = validate(p, what);
  if (rc != AVEY_OK) return rc;
  // combine writes no places, and the gradient of rows may not be wanted.
  const bool clear = clears(p) && (what == 0 || (what == 2 && p->drows));
  const uint64_t need = clear ? clear_bytes(p) : 0;
  if (need) rc = check_workspace(p->workspace, p->workspace_bytes, need);
  if (rc != AVEY_OK) return rc;
  rc = avey_host::device_ok();
  if (rc != AVEY_OK || p->tokens == 0) return done(rc);
  avey::RwArgs q{};
  q.tokens = p->tokens;
  q.k = p->k;
  q.width = static_cast<int>(p->width);
  q.blanks = clear && need == 0;
  if (need) q.namer = static_cast<int32_t*>(p->workspace);
  q.slots = p->slots;
  q.x = p->x;
  q.x_ld = p->x_ld;
  q.rows = p->rows;
  q.rows_ld = p->rows_ld;
  q.weights = p->weights;
  q.out = what == 2 ? p->drows : p->out;
  q.dweights = p->dweights;
  Chain chain{static_cast<cudaStream_t>(stream)};
  const int size = size_of(p->dtype);
  const int bytes = access_bytes(size, p->width, {p->x, p->rows, q.out},
                                 {p->x ? p->x_ld : 0, p->rows ? p->rows_ld : 0});
  if (p->dtype == AVEY_F32)
    rc = bytes == 16 ? launch_rows<float, 4>(q, what, chain) : launch_rows<float, 1>(q, what, chain);
  else if (p->dtype == AVEY_F16)
    rc = bytes == 16  ? launch_rows<__half, 8>(q, what, chain)
         : bytes == 4 ? launch_rows<__half, 2>(q, what, chain)
                      : launch_rows<__half, 1>(q, what, chain);
  else
    rc = bytes == 16  ? launch_rows<__nv_bfloat16, 8>(q, what, chain)
         : bytes == 4 ? launch_rows<__nv_bfloat16, 2>(q, what, chain)
                      : launch_rows<__nv_bfloat16, 1>(q, what, chain);
  return done(rc);
}

// ------------------------------------------------------------------ embedding

int validate(const AveyEmbeddingParams* p, bool backward) {
  if (!p) return fail(AVEY_ERR_ARGUMENT, "params is NULL");
  if (p->struct_size != sizeof(AveyEmbeddingParams))
    return fail(AVEY_ERR_ARGUMENT, "struct_size does not match sizeof(AveyEmbeddingParams)");
  if (!known(p->dtype)) return fail(AVEY_ERR_ARGUMENT, "the table is f32, f16 or bf16");
  if (p->index_bits != 32 && p->index_bits != 64) return fail(AVEY_ERR_ARGUMENT, "tokens have 32 or 64 bits");
  if (p->count < 0 || p->count > (1 << 30) || p->width < 1 || p->width > (1 << 22) || p->vocab < 1 ||
      p->vocab > (1 << 30))
    return fail(AVEY_ERR_ARGUMENT, "count must be in [0, 2^30], width in [1, 2^22], vocab in [1, 2^30]");
  if (!(p->scale > -1e30 && p->scale < 1e30)) return fail(AVEY_ERR_ARGUMENT, "scale must be finite");
  const uintptr_t element = size_of(p->dtype) - 1;
  if (((address(p->table) | address(p->out) | address(p->dy) | address(p->dtable)) & element) != 0 ||
      (address(p->tokens) & (p->index_bits / 8 - 1)) != 0)
    return fail(AVEY_ERR_ARGUMENT, "arrays must be aligned to their elements");
  if (p->count > 0 && !p->tokens) return fail(AVEY_ERR_ARGUMENT, "tokens is required");
  if (!backward && p->count > 0 && (!p->table || !p->out || p->table_ld < p->width))
    return fail(AVEY_ERR_ARGUMENT, "table and out are required and strides must cover the rows");
  if (backward && (!p->dtable || (p->count > 0 && (!p->dy || p->dy_ld < p->width))))
    return fail(AVEY_ERR_ARGUMENT, "dy and dtable are required and strides must cover the rows");
  return AVEY_OK;
}

avey::EmArgs embedding_args(const AveyEmbeddingParams* p) {
  avey::EmArgs q{};
  q.n = p->count;
  q.width = static_cast<int>(p->width);
  q.vocab = p->vocab;
  q.tokens = p->tokens;
  q.tokens64 = p->index_bits == 64;
  q.table = p->table;
  q.table_ld = p->table_ld;
  q.scale = static_cast<float>(p->scale);
  q.out = p->out;
  q.dy = p->dy;
  q.dy_ld = p->dy_ld;
  q.dtable = p->dtable;
  return q;
}

// Places of a chunk of em_sum.
int64_t chunk_places(int64_t n) {
  int64_t chunk = avey::kEmChunk;
  while (chunk > avey::kEmSmallChunk && n < chunk * 4 * avey_host::multiprocessors()) chunk /= 2;
  return chunk;
}
// Workspace of the backward call: [keys, ids] twice, counts, edges, parts.
struct EmLayout {
  int passes = 0;
  uint64_t keys[2] = {}, ids[2] = {}, counts[2] = {}, edges = 0, parts = 0, total = 0;
};
EmLayout embedding_layout(const AveyEmbeddingParams* p) {
  EmLayout l;
  if (p->count == 0) return l;
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t o = at;
    at += up256(bytes);
    return o;
  };
  int bits = 1;
  while (bits < 31 && (1ll << bits) <= p->vocab) ++bits;  // keys up to vocab itself
  l.passes = (bits + 9) / 10;
  for (int i = 0; i < 2; ++i) {
    l.keys[i] = take(p->count * 4);
    l.ids[i] = take(p->count * 4);
  }
  l.counts[0] = take(count_bytes(p->count, 1024));
  // Zero before the first launch, where there is more than one block: the later passes'
  // counts and the number of edges.
  l.counts[1] = take(count_bytes(p->count, 1024) * (l.passes - 1));
  const uint64_t chunk = chunk_places(p->count), chunks = (p->count + chunk - 1) / chunk;
  l.edges = take((1 + chunks) * 4);
  l.parts = take(chunks * 2 * p->width * 4);
  l.total = at;
  return l;
}

template <typename T, int N>
int launch_sums(const avey::EmArgs& q, Chain& chain) {
  const int64_t columns = q.width / N;
  const int threads = static_cast<int>(std::min<int64_t>(256, (columns + 31) / 32 * 32));
  const unsigned slices = static_cast<unsigned>(std::min<int64_t>((columns + threads - 1) / threads, 64));
  int rc = chain.launch("embedding sums", avey::em_sum<T, N>, dim3(static_cast<unsigned>(q.chunks), slices), threads, 0,
                        1, q);
  if (rc != AVEY_OK || q.chunks < 2) return rc;
  constexpr int V = N > 1 && sizeof(T) * N == 16 ? 4 : 1;  // width is a multiple of 4
  const int slabs = (q.width + avey::kEmLanes * V - 1) / (avey::kEmLanes * V);
  const unsigned grid = static_cast<unsigned>(
      std::min<int64_t>(avey_host::multiprocessors() * 8ll, q.chunks * static_cast<int64_t>(slabs)));
  return chain.launch("embedding parts", avey::em_finish<T, V>, dim3(grid), avey::kEmGroups * avey::kEmLanes, 0, 1, q,
                      slabs);
}

int embedding_backward(const AveyEmbeddingParams* p, cudaStream_t stream) {
  const int size = size_of(p->dtype);
  if (p->count == 0) {
    const cudaError_t e = cudaMemsetAsync(p->dtable, 0, static_cast<size_t>(p->vocab) * p->width * size, stream);
    return e == cudaSuccess ? AVEY_OK : fail(AVEY_ERR_CUDA, cudaGetErrorString(e));
  }
  const EmLayout l = embedding_layout(p);
  int rc = check_workspace(p->workspace, p->workspace_bytes, l.total);
  if (rc != AVEY_OK) return rc;
  char* ws = static_cast<char*>(p->workspace);
  const uint64_t pass_bytes = count_bytes(p->count, 1024), table = static_cast<uint64_t>(p->vocab) * p->width * size;
  uint32_t* edges = reinterpret_cast<uint32_t*>(ws + l.edges);
  auto words = [&](uint64_t at) { return reinterpret_cast<uint32_t*>(ws + at); };
  const int last = (l.passes - 1) & 1;
  Chain chain{stream};
  avey::StArgs first{};
  first.n = p->count;
  first.buckets = 1024;
  first.mask = 1023;
  first.limit = p->vocab;
  first.skip = p->padding >= 0 ? p->padding : -1;
  first.raw = p->tokens;
  first.raw64 = p->index_bits == 64;
  if (pass_bytes == 0) {
    avey::StArgs q = first;
    q.blocks = static_cast<int>((p->count + avey::kStRankEntries - 1) / avey::kStRankEntries);
    q.keys_out = words(l.keys[last]);
    q.ids_out = words(l.ids[last]);
    q.clear = edges;
    q.zeros = static_cast<uint8_t*>(p->dtable);
    q.zero_bytes = static_cast<int64_t>(table);
    const dim3 grid(static_cast<unsigned>(q.blocks + zero_blocks(q.zero_bytes)));
    rc = chain.launch("sort", avey::st_rank, grid, avey::kStRankThreads, static_cast<int>(p->count) * 4, 1, q);
    if (rc != AVEY_OK) return rc;
  } else {
    const cudaError_t e = cudaMemsetAsync(ws + l.counts[1], 0, l.edges + 4 - l.counts[1], stream);
    if (e != cudaSuccess) return fail(AVEY_ERR_CUDA, cudaGetErrorString(e));
    for (int pass = 0; pass < l.passes; ++pass) {
      avey::StArgs q = first;
      q.shift = 10 * pass;
      if (pass > 0) {
        q.raw = nullptr;
        q.keys = words(l.keys[(pass - 1) & 1]);
        q.ids = words(l.ids[(pass - 1) & 1]);
      }
      q.counts = words(pass == 0 ? l.counts[0] : l.counts[1] + (pass - 1) * pass_bytes);
      if (pass + 1 < l.passes) q.next_counts = words(l.counts[1] + pass * pass_bytes);
      q.keys_out = words(l.keys[pass & 1]);
      q.ids_out = words(l.ids[pass & 1]);
      // A share of the table's zeros beside each pass, in whole 256 bytes. (With a share beside
      // the count as well the sort's launches took no longer and the call 5 us more.)
      const uint64_t share = table / l.passes / 256 * 256;
      const uint64_t z0 = share * pass, z1 = pass + 1 == l.passes ? table : share * (pass + 1);
      q.zeros = static_cast<uint8_t*>(p->dtable) + z0;
      q.zero_bytes = static_cast<int64_t>(z1 - z0);
      rc = launch_pass(q, chain, pass > 0);
      if (rc != AVEY_OK) return rc;
    }
  }
  avey::EmArgs q = embedding_args(p);
  q.keys = words(l.keys[last]);
  q.ids = words(l.ids[last]);
  q.parts = reinterpret_cast<float*>(ws + l.parts);
  q.edges = edges;
  q.chunk = static_cast<int>(chunk_places(p->count));
  q.chunks = (p->count + q.chunk - 1) / q.chunk;
  const int bytes = access_bytes(size, p->width, {p->dy, p->dtable}, {p->dy_ld});
  if (p->dtype == AVEY_F32) return bytes == 16 ? launch_sums<float, 4>(q, chain) : launch_sums<float, 1>(q, chain);
  if (p->dtype == AVEY_F16)
    return bytes == 16  ? launch_sums<__half, 8>(q, chain)
           : bytes == 4 ? launch_sums<__half, 2>(q, chain)
                        : launch_sums<__half, 1>(q, chain);
  return bytes == 16  ? launch_sums<__nv_bfloat16, 8>(q, chain)
         : bytes == 4 ? launch_sums<__nv_bfloat16, 2>(q, chain)
                      : launch_sums<__nv_bfloat16, 1>(q, chain);
}

template <typename T, int N>
int launch_lookup(const avey::EmArgs& q, Chain& chain) {
  const int lanes = part_lanes(q.width, N);
  const int64_t rows = avey::kRwThreads / lanes;
  return chain.launch("embedding", avey::em_forward<T, N>, dim3(static_cast<unsigned>((q.n + rows - 1) / rows)),
                      avey::kRwThreads, 0, 1, q, lanes);
}

int embedding_forward(const AveyEmbeddingParams* p, cudaStream_t stream) {
  if (p->count == 0) return AVEY_OK;
  const avey::EmArgs q = embedding_args(p);
  Chain chain{stream};
  const int bytes = access_bytes(size_of(p->dtype), p->width, {p->table, p->out}, {p->table_ld});
  if (p->dtype == AVEY_F32) return bytes == 16 ? launch_lookup<float, 4>(q, chain) : launch_lookup<float, 1>(q, chain);
  if (p->dtype == AVEY_F16)
    return bytes == 16  ? launch_lookup<__half, 8>(q, chain)
           : bytes == 4 ? launch_lookup<__half, 2>(q, chain)
                        : launch_lookup<__half, 1>(q, chain);
  return bytes == 16  ? launch_lookup<__nv_bfloat16, 8>(q, chain)
         : bytes == 4 ? launch_lookup<__nv_bfloat16, 2>(q, chain)
                      : launch_lookup<__nv_bfloat16, 1>(q, chain);
}

}  // namespace

extern "C" {

int avey_route_fwd_v1(const AveyRouteParams* p, void* stream) { return run_route(p, false, stream); }
int avey_route_bwd_v1(const AveyRouteParams* p, void* stream) { return run_route(p, true, stream); }

int avey_arrange_workspace_size(const AveyArrangeParams* p, uint64_t* bytes) {
  const int rc = validate(p);
  if (rc != AVEY_OK) return rc;
  if (!bytes) return fail(AVEY_ERR_ARGUMENT, "bytes is NULL");
  *bytes = count_bytes(p->count, static_cast<int>(p->experts) + 1);
  return avey_host::clear_error();
}

int avey_arrange_v1(const AveyArrangeParams* p, void* stream) {
  int rc = validate(p);
  if (rc != AVEY_OK) return rc;
  rc = avey_host::device_ok();
  if (rc != AVEY_OK) return rc;
  avey::StArgs q{};
  q.n = p->count;
  q.buckets = static_cast<int>(p->experts) + 1;  // the last: of no expert
  q.mask = -1;
  q.raw = p->chosen;
  q.raw64 = p->index_bits == 64;
  q.limit = p->experts;
  q.skip = -1;
  q.slots = p->slots;
  q.offsets = p->offsets;
  rc = check_workspace(p->workspace, p->workspace_bytes, count_bytes(q.n, q.buckets));
  if (rc != AVEY_OK) return rc;
  q.counts = static_cast<uint32_t*>(p->workspace);
  Chain chain{static_cast<cudaStream_t>(stream)};
  return done(launch_pass(q, chain));
}

int avey_rows_workspace_size(const AveyRowsParams* p, uint64_t* bytes) {
  if (!p || !bytes) return fail(AVEY_ERR_ARGUMENT, "params or bytes is NULL");
  AveyRowsParams sizes{};
  sizes.struct_size = p->struct_size;
  sizes.dtype = p->dtype;
  sizes.k = p->k;
  sizes.tokens = p->tokens;
  sizes.width = p->width;
  sizes.slots = p->slots;
  const int rc = validate(&sizes, 3);
  if (rc != AVEY_OK) return rc;
  *bytes = clear_bytes(p);
  return avey_host::clear_error();
}
int avey_dispatch_v1(const AveyRowsParams* p, void* stream) { return run_rows(p, 0, stream); }
int avey_combine_v1(const AveyRowsParams* p, void* stream) { return run_rows(p, 1, stream); }
int avey_combine_bwd_v1(const AveyRowsParams* p, void* stream) { return run_rows(p, 2, stream); }

int avey_embedding_workspace_size(const AveyEmbeddingParams* p, uint64_t* bytes) {
  const int rc = validate(p, true);
  if (rc != AVEY_OK) return rc;
  if (!bytes) return fail(AVEY_ERR_ARGUMENT, "bytes is NULL");
  *bytes = embedding_layout(p).total;
  return avey_host::clear_error();
}

int avey_embedding_fwd_v1(const AveyEmbeddingParams* p, void* stream) {
  int rc = validate(p, false);
  if (rc != AVEY_OK) return rc;
  rc = avey_host::device_ok();
  return done(rc == AVEY_OK ? embedding_forward(p, static_cast<cudaStream_t>(stream)) : rc);
}

int avey_embedding_bwd_v1(const AveyEmbeddingParams* p, void* stream) {
  int rc = validate(p, true);
  if (rc != AVEY_OK) return rc;
  rc = avey_host::device_ok();
  return done(rc == AVEY_OK ? embedding_backward(p, static_cast<cudaStream_t>(stream)) : rc);
}

}  // extern "C"
