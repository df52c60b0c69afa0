// C ABI of the cross entropy over a vocabulary (declared in include/avey_b200.h):
// argument checks, tile choice, workspace layout and the launches of tc_loss.cuh.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdio>
#include <mutex>

#include "avey_b200.h"
#include "host_api.h"
#include "launch_chain.h"
#include "tc_loss.cuh"
#include "linear_steps.cuh"

namespace {

using avey_host::Chain;

int fail(int code, const char* msg) { return avey_host::set_error(code, msg); }

constexpr int kMaxDevices = 64;

template <auto K>
cudaError_t smem_opt_in() {
  static std::once_flag once[kMaxDevices];
  static cudaError_t err[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [dev] {
    err[dev] = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, avey::kCeSmem);
  });
  return err[dev];
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool whole_rows(const void* p, int64_t ld) { return aligned16(p) && ld % 8 == 0; }
int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

float* saved_low(const AveyLossParams* p) { return p->struct_size == sizeof(AveyLossParams) ? p->saved_low : nullptr; }

int validate(const AveyLossParams* p, bool backward) {
  if (!p) return fail(AVEY_ERR_ARGUMENT, "params is NULL");
  // (The block once ended before saved_low.)
  if (p->struct_size != sizeof(AveyLossParams) && p->struct_size != offsetof(AveyLossParams, saved_low))
    return fail(AVEY_ERR_ARGUMENT, "struct_size does not match sizeof(AveyLossParams)");
  if (p->dtype != AVEY_BF16 && p->dtype != AVEY_F16)
    return fail(AVEY_ERR_ARGUMENT, "the cross entropy takes bf16 or f16 operands");
  if (p->target_bits != 32 && p->target_bits != 64) return fail(AVEY_ERR_ARGUMENT, "targets have 32 or 64 bits");
  if (p->reduction < AVEY_LOSS_NONE || p->reduction > AVEY_LOSS_MEAN)
    return fail(AVEY_ERR_ARGUMENT, "unknown reduction");
  if (p->rows < 0 || p->rows > (1 << 30) || p->width < 1 || p->width > (1 << 22) || p->vocab < 1 ||
      p->vocab > (1 << 30))
    return fail(AVEY_ERR_ARGUMENT, "rows must be in [0, 2^30], width in [1, 2^22], vocab in [1, 2^30]");
  if ((p->rows / 256 + 1) > (1ll << 30) / (p->vocab / 64 + 1) ||
      (std::max(p->rows, p->vocab) / 256 + 1) > (1ll << 30) / (p->width / 64 + 1))
    return fail(AVEY_ERR_ARGUMENT, "too many tiles");
  if (!(p->z_loss > -1e30 && p->z_loss < 1e30)) return fail(AVEY_ERR_ARGUMENT, "z_loss must be finite");
  uintptr_t odd = 0;
  for (const void* a : {p->x, p->weight, const_cast<const void*>(p->dx), const_cast<const void*>(p->dweight)})
    odd |= reinterpret_cast<uintptr_t>(a) & 1u;
  for (const void* a : {static_cast<const void*>(p->loss), static_cast<const void*>(p->saved),
                        static_cast<const void*>(saved_low(p)), static_cast<const void*>(p->dloss)})
    odd |= reinterpret_cast<uintptr_t>(a) & 3u;
  if (odd != 0 || (reinterpret_cast<uintptr_t>(p->targets) & (p->target_bits / 8 - 1)) != 0)
    return fail(AVEY_ERR_ARGUMENT, "arrays must be aligned to their elements");
  if (!backward && !p->loss && (p->rows > 0 || p->reduction != AVEY_LOSS_NONE))
    return fail(AVEY_ERR_ARGUMENT, "loss is required");
  if (p->rows > 0 && (!p->x || !p->targets)) return fail(AVEY_ERR_ARGUMENT, "x and targets are required");
  if (p->rows > 0 && !p->weight) return fail(AVEY_ERR_ARGUMENT, "weight is required");
  if (p->x_ld < p->width || p->weight_ld < p->width || p->target_stride < 0)
    return fail(AVEY_ERR_ARGUMENT, "strides must cover the rows");
  if (backward && p->rows > 0) {
    if (!p->saved || !p->dloss) return fail(AVEY_ERR_ARGUMENT, "saved and dloss are required");
    if ((p->dx && p->dx_ld < p->width) || p->dloss_stride < 0)
      return fail(AVEY_ERR_ARGUMENT, "strides must cover the rows");
  }
  return AVEY_OK;
}

int pairs() { return avey_host::multiprocessors() / 2; }

// Columns of a tile of the logits. A K block takes nearly as long for 64 columns as for
// 256 (33 rows, 32768 x 768: 49 us with tiles of 64, 31 of 128, 23 of 256), so narrower
// tiles are for smaller vocabularies only.
int logit_cols(int64_t n) { return n > 128 ? 256 : n > 64 ? 128 : 64; }
// Column tiles of a unit of logits: more than one where there are enough for the
// pairs to end together.
int unit_tiles(int64_t mt, int64_t nt) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(avey::kCeMaxSeg, mt * nt / (16 * pairs()))));
}
// Of a gradient's product over `width` columns (boxes of 64 for each CTA).
int grad_cols(int64_t width) { return width > 128 ? 256 : 128; }

// Rows up to which the statistics take the kernel for few rows (calls with W out of L2: 8 rows of 32768 x
// 768 25 us, where 9 by tiles take 27; of 131072 x 1024 74 and 76, of 50021 x 389 40 and 44; one row
// 23, 69 and 38. 16 rows in two passes of its products took longer than by tiles).
constexpr int64_t kFewRows = 8;
bool use_few(const AveyLossParams* p) { return p->rows <= kFewRows; }
// Its CTAs: a warp for 16 rows of W, up to four CTAs an SM.
int64_t few_grid(const AveyLossParams* p) {
  const int64_t groups = (p->vocab + 15) / 16;
  return std::min<int64_t>((groups + avey::kCfWarps - 1) / avey::kCfWarps, avey_host::multiprocessors() * 4ll);
}

// Workspace of a call, each part 256-byte aligned.
struct Layout {
  bool few = false, pack_x = false, pack_w = false;
  uint64_t x = 0, w = 0;
  // forward
  int bn = 0, seg = 0;
  int64_t n_nt = 0, segments = 0;
  uint64_t partial = 0, picked = 0, each = 0;
  // backward
  int64_t piece = 0, pieces = 0;  // columns of dz at a time
  uint64_t coef = 0, counters = 0, dirty = 0, copy = 0, dz = 0, dz_bytes = 0, sums = 0, parts = 0;
  uint64_t total = 0;
};

// Columns of dz kept at a time, twice where there is more than one piece: 256 MB, but
// 4096 at least (above 32768 rows), where reading and writing dx's fp32 sums for every
// piece takes a fourteenth of the time of its products.
int64_t piece_columns(const AveyLossParams* p) {
  const int64_t most = std::max<int64_t>((256ll << 20) / (2 * p->rows), 4096);
  const int64_t tiles = (p->vocab + 255) / 256, per = std::max<int64_t>(1, most / 256);
  if (2 * per >= tiles) return up(p->vocab, 16);
  const int64_t pieces = (tiles + per - 1) / per;
  return (tiles + pieces - 1) / pieces * 256;
}

int64_t tiles_of(int64_t m, int64_t n, int bn) { return (m + avey::kCeBM - 1) / avey::kCeBM * ((n + bn - 1) / bn); }

// K ranges of a tile of dX: more than one where a tile would last longer than a
// pair's share of the launch (with dW over `n` columns), of eight K blocks at least.
int dx_splits(const AveyLossParams* p, int64_t n) {
  const int bn = grad_cols(p->width);
  const int64_t nk = (n + 63) / 64, tiles = tiles_of(p->rows, p->width, bn);
  const int64_t dw = p->dweight ? tiles_of(n, p->width, bn) * ((p->rows + 63) / 64) : 0;
  const int64_t share = (tiles * nk + dw + pairs() - 1) / pairs();
  int64_t s = (nk + share - 1) / share;
  // Without dW's tiles to fill it, the last wave of dX's is cut finer too.
  if (!p->dweight && tiles % pairs() != 0 && tiles < 4 * pairs()) s = std::max<int64_t>(s, 4);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(s, nk / 8)));
}

Layout layout(const AveyLossParams* p, bool backward) {
  Layout l;
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t o = at;
    at += (bytes + 255u) & ~uint64_t(255);
    return o;
  };
  if (p->rows == 0) return l;
  l.few = !backward && use_few(p);
  l.pack_x = !l.few && !whole_rows(p->x, p->x_ld);
  l.pack_w = !l.few && !whole_rows(p->weight, p->weight_ld);
  const uint64_t row = up(p->width, 8) * 2;
  if (l.pack_x) l.x = take(p->rows * row);
  if (l.pack_w) l.w = take(p->vocab * row);
  if (!backward) {
    l.bn = logit_cols(p->vocab);
    l.n_nt = (p->vocab + l.bn - 1) / l.bn;
    const int64_t mt = (p->rows + avey::kCeBM - 1) / avey::kCeBM;
    l.seg = unit_tiles(mt, l.n_nt);
    l.segments = l.few ? few_grid(p) : (l.n_nt + l.seg - 1) / l.seg;
    l.partial = take(l.segments * p->rows * 8);
    l.picked = take(p->rows * 4);
    if (p->reduction != AVEY_LOSS_NONE) l.each = take(p->rows * 4);
  } else {
    l.piece = piece_columns(p);
    l.pieces = (p->vocab + l.piece - 1) / l.piece;
    l.coef = take(p->rows * 8);
    l.counters = take(4 * (l.pieces + 3));
    if (p->dweight) {
      l.dirty = take((p->rows + 63) / 64);
      l.copy = take(p->rows * row);
    }
    l.dz_bytes = (static_cast<uint64_t>(p->rows) * l.piece * 2 + 255) / 256 * 256;
    l.dz = take(l.dz_bytes * (l.pieces > 1 ? 2 : 1));
    if (p->dx) {
      if (l.pieces > 1) l.sums = take(p->rows * up(p->width, 4) * 4);
      const int bn = grad_cols(p->width);
      int splits = 1;
      for (int64_t n : {std::min(l.piece, p->vocab), p->vocab - (l.pieces - 1) * l.piece})
        splits = std::max(splits, dx_splits(p, n));
      if (splits > 1) l.parts = take(splits * tiles_of(p->rows, p->width, bn) * avey::kCeBM * bn * 4);
    }
  }
  l.total = at;
  return l;
}

int check_workspace(const AveyLossParams* p, const Layout& l) {
  if (l.total == 0) return AVEY_OK;
  if (!p->workspace || p->workspace_bytes < l.total)
    return fail(AVEY_ERR_ARGUMENT, "workspace is smaller than avey_loss_workspace_size");
  if ((reinterpret_cast<uintptr_t>(p->workspace) & 255u) != 0)
    return fail(AVEY_ERR_ARGUMENT, "workspace must be 256-byte aligned");
  return AVEY_OK;
}

struct Rows {
  const void* p;
  int64_t ld;
};

int pack_inputs(const AveyLossParams* p, const Layout& l, Rows* x, Rows* w, Chain& chain) {
  char* ws = static_cast<char*>(p->workspace);
  *x = {p->x, p->x_ld};
  *w = {p->weight, p->weight_ld};
  if (!l.pack_x && !l.pack_w) return AVEY_OK;
  avey::LnPack a{}, b{};
  a.ld = b.ld = up(p->width, 8);
  a.cols = b.cols = static_cast<int>(p->width);
  if (l.pack_x) {
    a.src = static_cast<const uint16_t*>(p->x);
    a.src_ld = p->x_ld;
    a.per = a.rows = p->rows;
    a.dst = reinterpret_cast<uint16_t*>(ws + l.x);
    *x = {a.dst, a.ld};
  }
  if (l.pack_w) {
    b.src = static_cast<const uint16_t*>(p->weight);
    b.src_ld = p->weight_ld;
    b.per = b.rows = p->vocab;
    b.dst = reinterpret_cast<uint16_t*>(ws + l.w);
    *w = {b.dst, b.ld};
  }
  const int64_t pieces = (a.rows + b.rows) * (a.ld / 8);
  const int64_t grid = std::min<int64_t>((pieces + 255) / 256, avey_host::multiprocessors() * 16ll);
  return chain.launch("row copy", avey::ln_pack_rows, dim3(static_cast<unsigned>(grid)), 256, 0, 1, a, b);
}

template <auto K>
int launch_product(const avey::CeMaps& m, avey::CeGeom& q, Chain& chain) {
  const cudaError_t attr = smem_opt_in<K>();
  if (attr != cudaSuccess) return fail(AVEY_ERR_CUDA, cudaGetErrorString(attr));
  q.units = 0;
  for (const avey::CeJob& j : q.job) q.units += j.units;
  const dim3 grid(2 * static_cast<unsigned>(std::min<int64_t>(q.units, pairs())));
  return chain.launch("cross entropy product", K, grid, avey::kCeThreads, avey::kCeSmem, 2, m, q);
}

avey::CeGeom geom(const AveyLossParams* p) {
  avey::CeGeom q{};
  q.rows = static_cast<int>(p->rows);
  q.vocab = static_cast<int>(p->vocab);
  q.targets = p->targets;
  q.target_stride = p->target_stride;
  q.target64 = p->target_bits == 64;
  q.ignore = p->ignore_index;
  q.test_stall = avey_host::test_stall();
  return q;
}

avey::CeJob job(int kind, int64_t m, int64_t n, int64_t k, int bn) {
  avey::CeJob j{};
  j.kind = kind;
  j.m = static_cast<int>(m);
  j.n = static_cast<int>(n);
  j.nk = static_cast<int>((k + avey::kLnBK - 1) / avey::kLnBK);
  j.bn = bn;
  j.n_mt = static_cast<int>((m + avey::kCeBM - 1) / avey::kCeBM);
  j.n_nt = static_cast<int>((n + bn - 1) / bn);
  j.seg = 1;
  j.units = j.n_mt * j.n_nt;
  return j;
}

// The ring of a launch: stages for its widest tiles.
void set_ring(avey::CeGeom& q) {
  int bn = 0;
  for (const avey::CeJob& j : q.job) bn = std::max(bn, j.units ? j.bn : 0);
  q.stage_bytes = avey::kCeHalfA + bn * avey::kLnBK;
  q.stages = std::min(avey::kCeMaxStages, avey::kCeRing / q.stage_bytes);
}

avey::CeRows rows_of(const AveyLossParams* p) {
  avey::CeRows q{};
  q.rows = static_cast<int>(p->rows);
  q.vocab = static_cast<int>(p->vocab);
  q.targets = p->targets;
  q.target_stride = p->target_stride;
  q.target64 = p->target_bits == 64;
  q.ignore = p->ignore_index;
  q.z_loss = static_cast<float>(p->z_loss);
  return q;
}

template <typename T>
int stats_few(const AveyLossParams* p, const Layout& l, Chain& chain) {
  char* ws = static_cast<char*>(p->workspace);
  auto vec = [](const void* base, int64_t ld) {
    const uint64_t all = reinterpret_cast<uintptr_t>(base) | static_cast<uint64_t>(ld) * 2;
    return all % 32 == 0 ? 2 : all % 16 == 0 ? 1 : 0;
  };
  avey::CeFew q{};
  q.rows = static_cast<int>(p->rows);
  q.vocab = static_cast<int>(p->vocab);
  q.width = static_cast<int>(p->width);
  q.x = static_cast<const uint16_t*>(p->x);
  q.w = static_cast<const uint16_t*>(p->weight);
  q.x_ld = p->x_ld;
  q.w_ld = p->weight_ld;
  q.x_vec = vec(p->x, p->rows > 1 ? p->x_ld : 0);
  q.w_vec = vec(p->weight, p->weight_ld);
  q.targets = p->targets;
  q.target_stride = p->target_stride;
  q.target64 = p->target_bits == 64;
  q.ignore = p->ignore_index;
  q.partial = reinterpret_cast<float2*>(ws + l.partial);
  q.picked = reinterpret_cast<float*>(ws + l.picked);
  const dim3 grid(static_cast<unsigned>(l.segments));
  return chain.launch("cross entropy of few rows", avey::ce_few<T>, grid, 32 * avey::kCfWarps, 0, 1, q);
}

template <typename T>
int stats_tiles(const AveyLossParams* p, const Layout& l, Chain& chain) {
  char* ws = static_cast<char*>(p->workspace);
  Rows x, w;
  int rc = pack_inputs(p, l, &x, &w, chain);
  if (rc != AVEY_OK) return rc;
  avey::CeGeom q = geom(p);
  q.job[0] = job(avey::kCeStats, p->rows, p->vocab, p->width, l.bn);
  q.job[0].seg = l.seg;
  q.job[0].units = static_cast<int>(l.segments) * q.job[0].n_mt;
  set_ring(q);
  q.partial = reinterpret_cast<float2*>(ws + l.partial);
  q.picked = reinterpret_cast<float*>(ws + l.picked);
  avey::CeMaps m{};
  rc = avey_host::encode_rows16(p->dtype, x.p, p->width, p->rows, 1, x.ld * 2, 0, 128, &m.x);
  if (rc == AVEY_OK) rc = avey_host::encode_rows16(p->dtype, w.p, p->width, p->vocab, 1, w.ld * 2, 0, l.bn / 2, &m.w);
  return rc == AVEY_OK ? launch_product<avey::ce_product<T, true>>(m, q, chain) : rc;
}

template <typename T>
int forward(const AveyLossParams* p, cudaStream_t stream) {
  const Layout l = layout(p, false);
  int rc = check_workspace(p, l);
  if (rc != AVEY_OK) return rc;
  char* ws = static_cast<char*>(p->workspace);
  Chain chain{stream};
  rc = l.few ? stats_few<T>(p, l, chain) : stats_tiles<T>(p, l, chain);
  if (rc != AVEY_OK) return rc;
  avey::CeRows r = rows_of(p);
  r.segments = static_cast<int>(l.segments);
  r.partial = reinterpret_cast<const float2*>(ws + l.partial);
  r.picked = reinterpret_cast<const float*>(ws + l.picked);
  const bool none = p->reduction == AVEY_LOSS_NONE;
  r.each = none ? p->loss : reinterpret_cast<float*>(ws + l.each);
  r.lse = p->saved;
  r.low = saved_low(p);
  r.per = 32;
  while (r.per > 1 && r.per / 2 >= p->rows) r.per /= 2;
  const dim3 blocks(static_cast<unsigned>((p->rows + r.per - 1) / r.per));
  rc = chain.launch("cross entropy rows", avey::ce_rows, blocks, 256, 0, 1, r);
  if (rc != AVEY_OK || none) return rc;
  return chain.launch("cross entropy total", avey::ce_total, dim3(1), 1024, 0, 1, r, p->reduction == AVEY_LOSS_MEAN ? 1 : 0,
                      p->loss, p->saved ? p->saved + p->rows : nullptr);
}

template <typename T>
int backward(const AveyLossParams* p, cudaStream_t stream) {
  const Layout l = layout(p, true);
  int rc = check_workspace(p, l);
  if (rc != AVEY_OK) return rc;
  char* ws = static_cast<char*>(p->workspace);
  Chain chain{stream};
  uint32_t* counters = reinterpret_cast<uint32_t*>(ws + l.counters);
  const cudaError_t zeroed = cudaMemsetAsync(counters, 0, 4 * (l.pieces + 3), stream);
  if (zeroed != cudaSuccess) return fail(AVEY_ERR_CUDA, cudaGetErrorString(zeroed));
  uint32_t* largest = counters + l.pieces + 1;
  Rows x, w;
  rc = pack_inputs(p, l, &x, &w, chain);
  if (rc != AVEY_OK) return rc;
  avey::CeCoef k{};
  k.rows = static_cast<int>(p->rows);
  k.vocab = static_cast<int>(p->vocab);
  k.width = static_cast<int>(p->width);
  k.targets = p->targets;
  k.target_stride = p->target_stride;
  k.target64 = p->target_bits == 64;
  k.ignore = p->ignore_index;
  k.lse = p->saved;
  k.low = saved_low(p);
  k.count = p->reduction == AVEY_LOSS_MEAN ? p->saved + p->rows : nullptr;
  k.dy = p->dloss;
  k.dy_stride = p->reduction == AVEY_LOSS_NONE ? p->dloss_stride : 0;
  k.z_loss = static_cast<float>(p->z_loss);
  k.coef = reinterpret_cast<float2*>(ws + l.coef);
  k.largest = largest;
  if (p->dweight) {
    k.x = static_cast<const uint16_t*>(x.p);
    k.x_ld = x.ld;
    k.copy = reinterpret_cast<uint16_t*>(ws + l.copy);
    k.copy_ld = up(p->width, 8);
    k.dirty = reinterpret_cast<uint8_t*>(ws + l.dirty);
  }
  const dim3 blocks(static_cast<unsigned>((p->rows + avey::kCeCoefRows - 1) / avey::kCeCoefRows));
  rc = chain.launch("cross entropy coefficients", avey::ce_coef<T>, blocks, 256, 0, 1, k);
  if (rc != AVEY_OK) return rc;
  const int64_t sums_ld = up(p->width, 4);
  float* sums = reinterpret_cast<float*>(ws + l.sums);
  float* parts = reinterpret_cast<float*>(ws + l.parts);
  const bool planes = l.pieces > 1;
  const int bn = grad_cols(p->width);
  // Launch i makes dz of piece i and the gradients' products of piece i - 1.
  for (int64_t i = 0; i <= l.pieces; ++i) {
    avey::CeGeom q = geom(p);
    avey::CeMaps m{};
    if (i > 0) q.claimed = counters + i;  // dz alone: units of one kind
    q.largest = largest;
    q.lse = p->saved;
    q.coef = k.coef;
    int jobs = 0, splits = 1;
    if (i > 0) {
      const int64_t v0 = (i - 1) * l.piece, n = std::min(l.piece, p->vocab - v0), ld = up(n, 16);
      const char* dz = ws + l.dz + (i - 1) % 2 * l.dz_bytes;
      const char* wp = static_cast<const char*>(w.p) + v0 * w.ld * 2;
      if (p->dx) {
        splits = dx_splits(p, n);
        avey::CeJob j = job(avey::kCeDx, p->rows, p->width, n, bn);
        j.seg = splits;
        j.units *= splits;
        q.job[jobs++] = j;
        q.dx = planes ? nullptr : p->dx;
        q.dx_ld = p->dx_ld;
        q.dx_vec = whole_rows(p->dx, p->dx_ld);
        q.dx_add = i > 1;
        rc = avey_host::encode_rows16(p->dtype, dz, n, p->rows, 1, ld * 2, 0, 128, &m.dz_x);
        if (rc == AVEY_OK) rc = avey_host::encode_rows16(p->dtype, wp, p->width, n, 1, w.ld * 2, 0, 64, &m.w_x);
        if (rc == AVEY_OK && splits > 1)
          rc = avey_host::encode_tiles(AVEY_F32, parts, bn, static_cast<uint64_t>(j.units) * avey::kCeBM, 1, bn * 4, 0,
                                       &m.parts);
        else if (rc == AVEY_OK && planes)
          rc = avey_host::encode_tiles(AVEY_F32, sums, p->width, p->rows, 1, sums_ld * 4, 0, &m.y_dx);
        else if (rc == AVEY_OK && q.dx_vec)
          rc = avey_host::encode_tiles(p->dtype, p->dx, p->width, p->rows, 1, p->dx_ld * 2, 0, &m.y_dx);
        if (rc != AVEY_OK) return rc;
      }
      if (p->dweight) {
        q.job[jobs++] = job(avey::kCeDw, n, p->width, p->rows, bn);
        char* dw = static_cast<char*>(p->dweight) + v0 * p->width * 2;
        q.dw = dw;
        q.dw_ld = p->width;
        q.dw_vec = whole_rows(dw, p->width);
        q.dirty = k.dirty;
        rc = avey_host::encode_rows16(p->dtype, dz, n, p->rows, 1, ld * 2, 0, 64, &m.dz_w);
        if (rc == AVEY_OK) rc = avey_host::encode_rows16(p->dtype, x.p, p->width, p->rows, 1, x.ld * 2, 0, 64, &m.x_w);
        if (rc == AVEY_OK)
          rc = avey_host::encode_rows16(p->dtype, k.copy, p->width, p->rows, 1, k.copy_ld * 2, 0, 64, &m.x2);
        if (rc == AVEY_OK && q.dw_vec)
          rc = avey_host::encode_tiles(p->dtype, dw, p->width, n, 1, p->width * 2, 0, &m.y_dw);
        if (rc != AVEY_OK) return rc;
        if (jobs == 2 && q.job[1].nk > q.job[0].nk / splits) std::swap(q.job[0], q.job[1]);  // the longest first
      }
    }
    if (i < l.pieces) {
      const int64_t v0 = i * l.piece, n = std::min(l.piece, p->vocab - v0), ld = up(n, 16);
      const int cols = logit_cols(n);
      q.job[jobs] = job(avey::kCeGrad, p->rows, n, p->width, cols);
      q.job[jobs].seg = unit_tiles(q.job[jobs].n_mt, q.job[jobs].n_nt);
      q.job[jobs].units = (q.job[jobs].n_nt + q.job[jobs].seg - 1) / q.job[jobs].seg * q.job[jobs].n_mt;
      ++jobs;
      q.col0 = static_cast<int>(v0);
      rc = avey_host::encode_rows16(p->dtype, x.p, p->width, p->rows, 1, x.ld * 2, 0, 128, &m.x);
      if (rc == AVEY_OK)
        rc = avey_host::encode_rows16(p->dtype, static_cast<const char*>(w.p) + v0 * w.ld * 2, p->width, n, 1, w.ld * 2,
                                      0, cols / 2, &m.w);
      q.dz = reinterpret_cast<uint16_t*>(ws + l.dz + i % 2 * l.dz_bytes);
      q.dz_ld = ld;
      if (rc != AVEY_OK) return rc;
    }
    set_ring(q);
    rc = launch_product<avey::ce_product<T, false>>(m, q, chain);
    if (rc != AVEY_OK) return rc;
    if (splits > 1) {
      avey::CeParts j{};
      j.parts = parts;
      j.m = static_cast<int>(p->rows);
      j.n = static_cast<int>(p->width);
      j.bn = bn;
      j.n_nt = static_cast<int>((p->width + bn - 1) / bn);
      j.tiles = static_cast<int>(tiles_of(p->rows, p->width, bn));
      j.splits = splits;
      j.largest = largest;
      j.out = planes ? static_cast<void*>(sums) : p->dx;
      j.out_ld = planes ? sums_ld : p->dx_ld;
      j.add = i > 1;
      const dim3 grid(static_cast<unsigned>(j.tiles * (avey::kCeBM / avey::kCeJoinRows)));
      rc = planes ? chain.launch("cross entropy parts", avey::ce_join_parts<T, true>, grid, 256, 0, 1, j)
                  : chain.launch("cross entropy parts", avey::ce_join_parts<T, false>, grid, 256, 0, 1, j);
      if (rc != AVEY_OK) return rc;
    }
  }
  if (p->dx && planes) {
    const int64_t quads = p->rows * (sums_ld / 4);
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((quads + 255) / 256, avey_host::multiprocessors() * 8ll)));
    rc = chain.launch("dx rounding", avey::ce_finish<T>, grid, 256, 0, 1, sums, sums_ld, p->rows, p->width, largest,
                      static_cast<T*>(p->dx), p->dx_ld);
  }
  return rc;
}

// Sum and mean of no row, and the gradient of a weight without rows.
int empty(const AveyLossParams* p, bool backward, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  if (!backward) {
    // 0, or the NaN of all ones for 0 / 0.
    if (p->reduction != AVEY_LOSS_NONE)
      e = cudaMemsetAsync(p->loss, p->reduction == AVEY_LOSS_MEAN ? 0xFF : 0, 4, stream);
    if (e == cudaSuccess && p->saved) e = cudaMemsetAsync(p->saved, 0, 4, stream);
  } else if (p->dweight) {
    e = cudaMemsetAsync(p->dweight, 0, static_cast<size_t>(p->vocab) * p->width * 2, stream);
  }
  return e == cudaSuccess ? AVEY_OK : fail(AVEY_ERR_CUDA, cudaGetErrorString(e));
}

int run(const AveyLossParams* p, bool back, void* stream) {
  int rc = validate(p, back);
  if (rc != AVEY_OK) return rc;
  rc = avey_host::device_ok();
  if (rc != AVEY_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p->rows == 0) rc = empty(p, back, s);
  else if (!back) rc = p->dtype == AVEY_BF16 ? forward<__nv_bfloat16>(p, s) : forward<__half>(p, s);
  else if (p->dx || p->dweight) rc = p->dtype == AVEY_BF16 ? backward<__nv_bfloat16>(p, s) : backward<__half>(p, s);
  return rc == AVEY_OK ? avey_host::clear_error() : rc;
}

}  // namespace

namespace avey_host {
int loss_flags(unsigned int* flags, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(flags, avey::g_devflags, sizeof(*flags));
  const unsigned int zero = 0;
  if (e == cudaSuccess && clear) e = cudaMemcpyToSymbol(avey::g_devflags, &zero, sizeof(zero));
  return e;
}
int loss_wait_limit(long long cycles) { return cudaMemcpyToSymbol(avey::g_wait_limit, &cycles, sizeof(cycles)); }
}  // namespace avey_host

extern "C" {

int avey_loss_workspace_size(const AveyLossParams* p, int backward, uint64_t* bytes) {
  const int rc = validate(p, backward != 0);
  if (rc != AVEY_OK) return rc;
  if (!bytes) return fail(AVEY_ERR_ARGUMENT, "bytes is NULL");
  *bytes = layout(p, backward != 0).total;
  return avey_host::clear_error();
}

int avey_loss_fwd_v1(const AveyLossParams* p, void* stream) { return run(p, false, stream); }
int avey_loss_bwd_v1(const AveyLossParams* p, void* stream) { return run(p, true, stream); }

}  // extern "C"
