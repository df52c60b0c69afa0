// C ABI of the linear layers (declared in include/avey_b200.h): argument checks,
// tile and kernel choice, workspace layout and the launches of tc_linear.cuh and
// linear_steps.cuh.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>
#include <mutex>

#include "avey_b200.h"
#include "host_api.h"
#include "tc_linear.cuh"
#include "linear_steps.cuh"

namespace {

int fail(int code, const char* msg) { return avey_host::set_error(code, msg); }

constexpr int kMaxDevices = 64;

// Opt kernel K into its shared memory, once per device; the outcome is kept.
template <auto K>
cudaError_t smem_opt_in(int bytes = avey::kLnSmem) {
  static std::once_flag once[kMaxDevices];
  static cudaError_t err[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [dev, bytes] {
    err[dev] = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  });
  return err[dev];
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    char buf[256];
    snprintf(buf, sizeof(buf), "%s launch: %s", what, cudaGetErrorString(e));
    return fail(AVEY_ERR_LAUNCH, buf);
  }
  avey_host::count_launches(1);
  return AVEY_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// Rows that TMA and 16-byte accesses can read in place.
bool whole_rows(const void* p, int64_t ld) { return aligned16(p) && ld % 8 == 0; }
int64_t up8(int64_t x) { return (x + 7) / 8 * 8; }
int64_t up16(int64_t x) { return (x + 15) / 16 * 16; }
uint64_t up256(uint64_t x) { return (x + 255u) & ~uint64_t(255); }

int validate(const AveyLinearParams* p, bool backward) {
  if (!p) return fail(AVEY_ERR_ARGUMENT, "params is NULL");
  if (p->struct_size != sizeof(AveyLinearParams))
    return fail(AVEY_ERR_ARGUMENT, "struct_size does not match sizeof(AveyLinearParams)");
  if (p->dtype != AVEY_BF16 && p->dtype != AVEY_F16)
    return fail(AVEY_ERR_ARGUMENT, "linear layers take bf16 or f16 operands");
  if (p->activation < 0 || p->activation > 4) return fail(AVEY_ERR_ARGUMENT, "unknown activation");
  if (p->kernel < AVEY_LINEAR_KERNEL_AUTO || p->kernel > AVEY_LINEAR_KERNEL_FEW)
    return fail(AVEY_ERR_ARGUMENT, "unknown linear kernel");
  if (p->rows < 0 || p->rows > (1 << 30) || p->d_in < 1 || p->d_in > (1 << 22) || p->d_out < 1 ||
      p->d_out > (1 << 22) || p->groups < 1 || p->groups > 65535)
    return fail(AVEY_ERR_ARGUMENT, "rows must be in [0, 2^30], d_in and d_out in [1, 2^22], groups in [1, 65535]");
  if (!p->offsets && p->groups != 1) return fail(AVEY_ERR_ARGUMENT, "more than one group needs offsets");
  if ((p->rows + 127) / 128 + p->groups > (1ll << 30) / ((std::max(p->d_in, p->d_out) + 63) / 64))
    return fail(AVEY_ERR_ARGUMENT, "too many output tiles");
  if (p->kernel == AVEY_LINEAR_KERNEL_FEW && p->offsets && std::min(p->groups, p->rows) > 65534)
    return fail(AVEY_ERR_ARGUMENT, "the kernel for few rows takes up to 65534 groups with rows");
  uintptr_t odd = 0;
  for (const void* a : {p->x, p->weight, p->bias, p->residual, p->dy, const_cast<const void*>(p->y),
                        const_cast<const void*>(p->dx), const_cast<const void*>(p->dweight),
                        const_cast<const void*>(p->dbias)})
    odd |= reinterpret_cast<uintptr_t>(a) & 1u;
  if (odd != 0 || (reinterpret_cast<uintptr_t>(p->offsets) & 3u) != 0)
    return fail(AVEY_ERR_ARGUMENT, "arrays must be aligned to their elements");
  if (p->rows == 0 && !backward) return AVEY_OK;
  if (p->rows > 0 && !p->x && (!backward || p->dweight)) return fail(AVEY_ERR_ARGUMENT, "x is required");
  if (!p->weight && (!backward || p->dx)) return fail(AVEY_ERR_ARGUMENT, "weight is required");
  if (p->x_ld < p->d_in || p->weight_ld < p->d_in || p->bias_group_stride < 0 ||
      (p->groups > 1 && p->weight_group_stride < (p->d_out - 1) * p->weight_ld + p->d_in))
    return fail(AVEY_ERR_ARGUMENT, "strides must cover the rows");
  if (!backward) {
    if (!p->y || p->y_ld < p->d_out || (p->residual && p->residual_ld < p->d_out))
      return fail(AVEY_ERR_ARGUMENT, "y is required and strides must cover the rows");
    if (p->deriv && p->activation == AVEY_ACT_IDENTITY)
      return fail(AVEY_ERR_ARGUMENT, "the identity has no derivative to keep");
  } else if (p->rows > 0) {
    if (!p->dy || p->dy_ld < p->d_out || (p->dx && p->dx_ld < p->d_in))
      return fail(AVEY_ERR_ARGUMENT, "dy is required and strides must cover the rows");
    if (!p->deriv && p->activation != AVEY_ACT_IDENTITY)
      return fail(AVEY_ERR_ARGUMENT, "the backward pass needs deriv from the forward pass");
  }
  if (p->deriv && (reinterpret_cast<uintptr_t>(p->deriv) & 31u) != 0)
    return fail(AVEY_ERR_ARGUMENT, "deriv must be 32-byte aligned");
  return AVEY_OK;
}

// Whether TMA can read x and the weights in place.
bool whole_x(const AveyLinearParams* p) { return whole_rows(p->x, p->x_ld); }
bool whole_w(const AveyLinearParams* p) {
  return whole_rows(p->weight, p->weight_ld) && (p->weight_group_stride % 8 == 0 || p->groups == 1);
}

// AUTO, dense layers: the kernel for few rows costs as its rows x d_in x d_out,
// tiles as their number. 8 rows at most finish sooner there at any size (768 ->
// 1536: 2.5 against 6.0 us, 8192 -> 16384: 43 against 50-70); up to 32 rows to 2^29
// (32 of 2048 -> 8192: 13.0 against 14.7; past it 16 of 4096 -> 14336: 29.8 against
// 27.3); up to 256 to 2^28 (64 of 1024 -> 4096: 8.1 against 9.2; 256 of 768 -> 768:
// 6.4 against 6.9; past it 64 of 1536 -> 6144: 15.6 against 12.3; 256 of 768 -> 1536:
// 11.1 against 8.5). Rows that are not whole 16-byte units it reads value by value,
// four times as dear (128 of 389 -> 771: 7.1 against 8.8; 256: 10.9 against 9.1).
// Grouped ones: up to 64 rows (of 16 experts, 1024 -> 2048: 14.3 against 18.4 us, of
// 64: 48.0 against 50.3; 64 rows of 16, 4096 -> 14336: 276 against 308), but those of
// more than 8 rows an expert to 2^28 (64 rows of 4, 2048 -> 2048: 12.1 against 15.3;
// past it 64 of 4, 2048 -> 8192: 33.7 against 28.7, 64 of 2, 4096 -> 14336: 90.8 against
// 46.1; odd rows alike to 2^27: 64 of 4, 1021 -> 2047: 18.7 against 19.7); more rows
// finish sooner here or there by the number of experts (128 rows of 32: 26.2 against
// 29.7; of 128, 768 -> 1536: 49.8 against 38.2) and take tiles.
bool use_few(const AveyLinearParams* p) {
  if (p->kernel != AVEY_LINEAR_KERNEL_AUTO) return p->kernel == AVEY_LINEAR_KERNEL_FEW;
  if (p->offsets)
    return p->rows <= 64 && (p->rows <= 8 * p->groups || p->rows * p->d_in * p->d_out <= 1ll << 28);
  if (p->rows <= 8) return true;
  const int64_t most = (p->rows <= 32 ? 1ll << 29 : 1ll << 28) / (whole_x(p) && whole_w(p) ? 1 : 4);
  return p->rows <= 256 && p->rows * p->d_in * p->d_out <= most;
}

// Row tiles of `tile` rows that the groups can come to.
int64_t row_tiles(const AveyLinearParams* p, int tile) {
  return p->offsets ? p->rows / tile + std::min(p->groups, p->rows) : (p->rows + tile - 1) / tile;
}

// Columns per tile: 256 wide tiles read the fewest bytes from shared memory for
// their products; narrower ones are taken where 256 would leave SMs without one.
int tile_cols(int64_t mt, int64_t n) {
  const int sms = avey_host::multiprocessors();
  for (int bn : {256, 128}) {
    if (n <= bn / 2) continue;
    if (mt * ((n + bn - 1) / bn) * 4 >= sms * 3) return bn;
  }
  return 64;
}

// K ranges per group of dW: as many as give every SM a tile, of four K blocks
// at least.
int dw_splits(const AveyLinearParams* p, int bn) {
  const int64_t tiles = p->groups * ((p->d_out + 127) / 128) * ((p->d_in + bn - 1) / bn);
  const int64_t blocks = (p->rows / p->groups + 63) / 64;
  return static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>({avey_host::multiprocessors() / tiles, blocks / 4, 64})));
}
int dw_cols(const AveyLinearParams* p) { return p->d_in <= 64 ? 64 : p->d_in <= 128 ? 128 : 256; }

// Workspace: [packed x | packed W | dpre | bias partials | dW partials], the
// parts that the call needs, each 256-byte aligned.
struct Layout {
  bool pack_x = false, pack_w = false, make_dpre = false, sums = false;
  int splits = 1;
  uint64_t x = 0, w = 0, dpre = 0, partial = 0, dw = 0, total = 0;
};

Layout layout(const AveyLinearParams* p, bool backward) {
  Layout l;
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t o = at;
    at += up256(bytes);
    return o;
  };
  if (p->rows == 0 || (!backward && use_few(p))) return l;
  const bool want_x = !backward || p->dweight, want_w = !backward || p->dx;
  l.pack_x = want_x && !whole_x(p);
  l.pack_w = want_w && !whole_w(p);
  if (l.pack_x) l.x = take(static_cast<uint64_t>(p->rows) * up8(p->d_in) * 2);
  if (l.pack_w) l.w = take(static_cast<uint64_t>(p->groups) * p->d_out * up8(p->d_in) * 2);
  if (backward) {
    l.make_dpre = (p->dx || p->dweight) &&
                  (p->activation != AVEY_ACT_IDENTITY || !whole_rows(p->dy, p->dy_ld));
    l.sums = p->dbias != nullptr;
    if (l.make_dpre) l.dpre = take(static_cast<uint64_t>(p->rows) * up8(p->d_out) * 2);
    if (l.sums) l.partial = take(static_cast<uint64_t>(row_tiles(p, avey::kLdRows)) * p->d_out * 4);
    if (p->dweight) {
      l.splits = dw_splits(p, dw_cols(p));
      if (l.splits > 1)
        l.dw = take(static_cast<uint64_t>(l.splits) * p->groups * p->d_out * ((p->d_in + 3) / 4 * 4) * 4);
    }
  }
  l.total = at;
  return l;
}

int check_workspace(const AveyLinearParams* p, const Layout& l) {
  if (l.total == 0) return AVEY_OK;
  if (!p->workspace || p->workspace_bytes < l.total)
    return fail(AVEY_ERR_ARGUMENT, "workspace is smaller than avey_linear_workspace_size");
  if ((reinterpret_cast<uintptr_t>(p->workspace) & 255u) != 0)
    return fail(AVEY_ERR_ARGUMENT, "workspace must be 256-byte aligned");
  return AVEY_OK;
}

// The operands as the tensor cores read them.
struct Rows {
  const void* p;
  int64_t ld, gs;
};

int pack_inputs(const AveyLinearParams* p, const Layout& l, Rows* x, Rows* w, cudaStream_t stream) {
  char* ws = static_cast<char*>(p->workspace);
  *x = {p->x, p->x_ld, 0};
  *w = {p->weight, p->weight_ld, p->weight_group_stride};
  if (!l.pack_x && !l.pack_w) return AVEY_OK;
  avey::LnPack a{}, b{};
  a.ld = b.ld = up8(p->d_in);
  a.cols = b.cols = static_cast<int>(p->d_in);
  if (l.pack_x) {
    a.src = static_cast<const uint16_t*>(p->x);
    a.src_ld = p->x_ld;
    a.per = a.rows = p->rows;
    a.dst = reinterpret_cast<uint16_t*>(ws + l.x);
    *x = {a.dst, a.ld, 0};
  }
  if (l.pack_w) {
    b.src = static_cast<const uint16_t*>(p->weight);
    b.src_ld = p->weight_ld;
    b.src_gs = p->weight_group_stride;
    b.per = p->d_out;
    b.rows = p->groups * p->d_out;
    b.dst = reinterpret_cast<uint16_t*>(ws + l.w);
    *w = {b.dst, b.ld, p->d_out * b.ld};
  }
  const int64_t pieces = (a.rows + b.rows) * (a.ld / 8);
  const int grid = static_cast<int>(std::min<int64_t>((pieces + 255) / 256, avey_host::multiprocessors() * 16ll));
  avey::ln_pack_rows<<<grid, 256, 0, stream>>>(a, b);
  return launched("row copy");
}

avey::LnGeom geom(const AveyLinearParams* p, int64_t n, int bn) {
  avey::LnGeom q{};
  q.groups = static_cast<int>(p->groups);
  q.offsets = p->offsets;
  q.rows = static_cast<int>(p->rows);
  q.n = static_cast<int>(n);
  q.bn = bn;
  q.n_nt = static_cast<int>((n + bn - 1) / bn);
  q.splits = 1;
  q.stage_bytes = avey::kLnABytes + bn * avey::kLnBK * 2;
  q.stages = avey::kLnRing / q.stage_bytes;
  q.test_stall = avey_host::test_stall();
  return q;
}

// Maps of a launch: the operands, and the output where it is stored by TMA.
struct Maps {
  CUtensorMap a{}, b{}, y{};
};

// `after`: the launch before this one on the stream is a step of the same call
// that lets its dependents start early.
template <auto K>
int launch_tc(const Maps& m, const avey::LnGeom& q, int64_t tiles, bool after, cudaStream_t stream) {
  const cudaError_t attr = smem_opt_in<K>();
  if (attr != cudaSuccess) return fail(AVEY_ERR_CUDA, cudaGetErrorString(attr));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(tiles, avey_host::multiprocessors())));
  cfg.blockDim = dim3(avey::kLnThreads);
  cfg.dynamicSmemBytes = avey::kLnSmem;
  cfg.stream = stream;
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = early;
  cfg.numAttrs = after ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, K, m.a, m.b, m.y, q);
  if (e != cudaSuccess) return fail(AVEY_ERR_LAUNCH, cudaGetErrorString(e));
  avey_host::count_launches(1);
  return AVEY_OK;
}

// CTAs that share a 128 x 64 tile's K blocks (1: the persistent kernel): enough
// for the SMs where such tiles are fewer than half of them, of two blocks each
// at least. 128 rows, 2048 -> 1024: 8.9 us (8 CTAs a tile) against 13.6 by
// one CTA a tile; 768 -> 1536: 6.9 (4 CTAs) against 7.7.
int split_ctas(const AveyLinearParams* p) {
  const int64_t tiles = (row_tiles(p, avey::kLnBM) + (p->offsets ? 1 : 0)) * ((p->d_out + avey::kLsBN - 1) / avey::kLsBN);
  const int64_t blocks = (p->d_in + avey::kLnBK - 1) / avey::kLnBK;
  int ctas = 1;
  while (ctas < 8 && tiles * ctas * 2 <= avey_host::multiprocessors() && blocks >= 4 * ctas) ctas *= 2;
  return ctas;
}

template <auto K>
int launch_split(const CUtensorMap& a, const CUtensorMap& b, avey::LnGeom q, int64_t tiles, int ctas, bool after,
                 cudaStream_t stream) {
  q.bn = avey::kLsBN;
  q.n_nt = (q.n + avey::kLsBN - 1) / avey::kLsBN;
  q.stages = std::min<int>(avey::kLnMaxStages, ((q.kc + avey::kLnBK - 1) / avey::kLnBK + ctas - 1) / ctas);
  const cudaError_t attr = smem_opt_in<K>(avey::ls_smem(avey::kLnMaxStages));
  if (attr != cudaSuccess) return fail(AVEY_ERR_CUDA, cudaGetErrorString(attr));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * ctas));
  cfg.blockDim = dim3(avey::kLsThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(avey::ls_smem(q.stages));
  cfg.stream = stream;
  cudaLaunchAttribute cluster[2];
  cluster[0].id = cudaLaunchAttributeClusterDimension;
  cluster[0].val.clusterDim.x = static_cast<unsigned>(ctas);
  cluster[0].val.clusterDim.y = 1;
  cluster[0].val.clusterDim.z = 1;
  cluster[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  cluster[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = cluster;
  cfg.numAttrs = after ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, K, a, b, q, ctas);
  if (e != cudaSuccess) return fail(AVEY_ERR_LAUNCH, cudaGetErrorString(e));
  avey_host::count_launches(1);
  return AVEY_OK;
}

template <typename T, int ACT>
int forward_tc(const AveyLinearParams* p, cudaStream_t stream) {
  const Layout l = layout(p, false);
  int rc = check_workspace(p, l);
  if (rc != AVEY_OK) return rc;
  Rows x, w;
  rc = pack_inputs(p, l, &x, &w, stream);
  if (rc != AVEY_OK) return rc;
  const int64_t mt = row_tiles(p, avey::kLnBM);
  const int ctas = split_ctas(p);
  avey::LnGeom q = geom(p, p->d_out, ctas > 1 ? avey::kLsBN : tile_cols(mt, p->d_out));
  q.kc = static_cast<int>(p->d_in);
  q.out = p->y;
  q.out_ld = p->y_ld;
  q.out_vec = whole_rows(p->y, p->y_ld);
  q.bias = p->bias;
  q.bias_gs = p->bias_group_stride;
  q.res = p->residual;
  q.res_ld = p->residual_ld;
  q.res_vec = p->residual && whole_rows(p->residual, p->residual_ld);
  q.deriv = static_cast<uint16_t*>(p->deriv);
  q.deriv_ld = up16(p->d_out);
  Maps m;
  rc = avey_host::encode_rows16(p->dtype, x.p, p->d_in, p->rows, 1, x.ld * 2, 0, avey::kLnBM, &m.a);
  if (rc == AVEY_OK)
    rc = avey_host::encode_rows16(p->dtype, w.p, p->d_in, p->d_out, p->groups, w.ld * 2, w.gs * 2, q.bn, &m.b);
  if (rc == AVEY_OK && q.out_vec)
    rc = avey_host::encode_tiles(p->dtype, p->y, p->d_out, p->rows, 1, p->y_ld * 2, 0, &m.y);
  if (rc != AVEY_OK) return rc;
  // One more row tile than the groups': the rows past the last group.
  const int64_t tiles = (mt + (p->offsets ? 1 : 0)) * q.n_nt;
  const bool packed = l.pack_x || l.pack_w;
  if (ctas > 1) {
    if constexpr (ACT != AVEY_ACT_IDENTITY)
      if (p->deriv) return launch_split<avey::tc_linear_split<T, ACT, true>>(m.a, m.b, q, tiles, ctas, packed, stream);
    return launch_split<avey::tc_linear_split<T, ACT, false>>(m.a, m.b, q, tiles, ctas, packed, stream);
  }
  if constexpr (ACT != AVEY_ACT_IDENTITY)
    if (p->deriv) return launch_tc<avey::tc_linear<T, avey::kLnForward, ACT, true>>(m, q, tiles, packed, stream);
  return launch_tc<avey::tc_linear<T, avey::kLnForward, ACT, false>>(m, q, tiles, packed, stream);
}

template <typename T, int ACT, bool DERIV, int NT>
int launch_few_rows(const avey::LnFew& q, int passes, cudaStream_t stream) {
  const dim3 grid((q.n + avey::kLfOut - 1) / avey::kLfOut, q.offsets ? std::min(q.groups, q.rows) + 1 : passes);
  const int64_t ctas = static_cast<int64_t>(grid.x) * (q.offsets ? grid.y - 1 : grid.y), sms = avey_host::multiprocessors();
  if (ctas <= sms && q.k >= 1024)
    avey::ln_few<T, ACT, DERIV, NT, 16><<<grid, 512, 0, stream>>>(q);
  else if (ctas < 3 * sms)
    avey::ln_few<T, ACT, DERIV, NT, 8><<<grid, 256, 0, stream>>>(q);
  else
    avey::ln_few<T, ACT, DERIV, NT, 4><<<grid, 128, 0, stream>>>(q);
  return launched("ln_few");
}

template <typename T, int ACT, bool DERIV>
int launch_few(const avey::LnFew& q, cudaStream_t stream) {
  // Rows of a pass over the weights: twice an expert's share, or the least that hold
  // all rows of a dense layer. Those share its rows among CTAs while there are no
  // more than two an SM: the weights come from L2 for all but one of them, and a CTA
  // takes in fewer rows of x, which is most of what it reads (48 rows of 2048 ->
  // 1024: 5.5 us by two passes, 7.2 by one; 64 of 768 -> 768: 3.2 by four, 5.2; with
  // up to three CTAs an SM 64 of 1536 -> 1536 take 8.0 us instead of 6.3).
  int passes = 1;
  if (!q.offsets)
    while (q.rows > 8 * passes && (q.n + avey::kLfOut - 1) / avey::kLfOut * passes <= avey_host::multiprocessors())
      passes *= 2;
  const int rows = q.offsets ? std::max(1, 2 * q.rows / q.groups) : (q.rows + passes - 1) / passes;
  if (rows <= 8) return launch_few_rows<T, ACT, DERIV, 1>(q, passes, stream);
  if (rows <= 16) return launch_few_rows<T, ACT, DERIV, 2>(q, passes, stream);
  if (rows <= 32) return launch_few_rows<T, ACT, DERIV, 4>(q, passes, stream);
  return launch_few_rows<T, ACT, DERIV, 8>(q, passes, stream);
}

template <typename T, int ACT>
int forward_few(const AveyLinearParams* p, cudaStream_t stream) {
  avey::LnFew q{};
  q.offsets = p->offsets;
  q.groups = static_cast<int>(p->groups);
  q.rows = static_cast<int>(p->rows);
  q.n = static_cast<int>(p->d_out);
  q.k = static_cast<int>(p->d_in);
  q.x = static_cast<const uint16_t*>(p->x);
  q.w = static_cast<const uint16_t*>(p->weight);
  q.bias = static_cast<const uint16_t*>(p->bias);
  q.res = static_cast<const uint16_t*>(p->residual);
  q.x_ld = p->x_ld;
  q.w_ld = p->weight_ld;
  q.w_gs = p->weight_group_stride;
  q.bias_gs = p->bias_group_stride;
  q.res_ld = p->residual_ld;
  q.y = static_cast<uint16_t*>(p->y);
  q.y_ld = p->y_ld;
  q.deriv = static_cast<uint16_t*>(p->deriv);
  q.deriv_ld = up16(p->d_out);
  auto vec = [](const void* base, int64_t ld, int64_t gs) {
    const uint64_t all = reinterpret_cast<uintptr_t>(base) | static_cast<uint64_t>(ld) * 2 | static_cast<uint64_t>(gs) * 2;
    return all % 32 == 0 ? 2 : all % 16 == 0 ? 1 : 0;
  };
  q.x_vec = vec(p->x, p->x_ld, 0);
  q.w_vec = vec(p->weight, p->weight_ld, p->groups > 1 ? p->weight_group_stride : 0);
  if constexpr (ACT != AVEY_ACT_IDENTITY)
    if (p->deriv) return launch_few<T, ACT, true>(q, stream);
  return launch_few<T, ACT, false>(q, stream);
}

template <typename T>
int forward(const AveyLinearParams* p, cudaStream_t stream) {
  const bool few = use_few(p);
  switch (p->activation) {
#define AVEY_CASE(A) \
  case A: return few ? forward_few<T, A>(p, stream) : forward_tc<T, A>(p, stream)
    AVEY_CASE(AVEY_ACT_RELU);
    AVEY_CASE(AVEY_ACT_RELU2);
    AVEY_CASE(AVEY_ACT_SILU);
    AVEY_CASE(AVEY_ACT_GELU);
    default: return few ? forward_few<T, AVEY_ACT_IDENTITY>(p, stream) : forward_tc<T, AVEY_ACT_IDENTITY>(p, stream);
#undef AVEY_CASE
  }
}

// The bias gradient is summed by 32 columns of a group at a time, in one of three
// places, with the same bits. An idle warp of each CTA of the dX kernel takes 1.2 us
// for one, 0.25 to walk past 32 groups and 1.5 for each 32 partial rows after the
// first; that is free where the CTA lasts as long: 5 us and 0.4 a K block. (Steps in
// a graph, with db in dX / by a launch of its own / without db: 4096 x 1024 -> 1024
// 46.0 / 48.1 / 45.7 us, 16 x 1024 -> 8192 50.8 / 53.2 / 50.5, 32768 x 768 -> 1536 324
// / 333 / 320; but 64 x 64 -> 4096 187.6 / 33.6 / 31.5, 65536 x 256 -> 256 128 / 92 / 84.)
bool bias_in_dx(const AveyLinearParams* p) {
  if (!p->dx) return false;
  const int64_t mt = row_tiles(p, avey::kLnBM), sms = avey_host::multiprocessors();
  const int64_t tiles = (mt + (p->offsets ? 1 : 0)) * ((p->d_in + tile_cols(mt, p->d_in) - 1) / tile_cols(mt, p->d_in));
  const int64_t ctas = std::min(tiles, sms), items = (p->d_out + 31) / 32 * p->groups;
  const int64_t partial = p->rows / p->groups / avey::kLdRows + 1;
  const double sums = static_cast<double>((items + ctas - 1) / ctas) *
                      (1.2 + 0.25 * static_cast<double>((p->groups + 31) / 32) + 1.5 * static_cast<double>(partial / 32));
  const double lasts = 5 + 0.4 * static_cast<double>((tiles + ctas - 1) / ctas) * static_cast<double>((p->d_out + 63) / 64);
  return sums <= lasts;
}

// A launch of its own: a CTA for 32 columns of a group, or a warp where that would
// be more than four CTAs an SM, of groups with up to 64 partial rows (steps in a graph:
// 512 rows of 16 experts, 768 -> 768: 31.2 against 30.0 us; 64 rows of 64, 64 -> 1536:
// 58.3 against 46.4; 1000 of 1000, 64 -> 512: 765 against 256; 4096 dense rows, 1024 ->
// 1024: 48.1 against 58.5).
template <typename T>
int launch_bias_sum(const AveyLinearParams* p, const float* partial, cudaStream_t stream) {
  const int groups = static_cast<int>(p->groups), rows = static_cast<int>(p->rows), n = static_cast<int>(p->d_out);
  T* db = static_cast<T*>(p->dbias);
  const int64_t cols = (p->d_out + 31) / 32, items = cols * p->groups;
  if (items > 4 * avey_host::multiprocessors() && p->rows / p->groups <= 64 * avey::kLdRows) {
    const dim3 grid(static_cast<unsigned>((items + avey::kLbWarps - 1) / avey::kLbWarps));
    avey::ln_bias_groups<T><<<grid, 32 * avey::kLbWarps, 0, stream>>>(p->offsets, groups, rows, n, partial, db);
  } else {
    const dim3 grid(static_cast<unsigned>(cols), static_cast<unsigned>(p->groups));
    avey::ln_bias_sum<T><<<grid, avey::kLbThreads, 0, stream>>>(p->offsets, groups, rows, n, partial, db);
  }
  return launched("bias sum");
}

template <typename T>
int launch_dpre(const avey::LnDpre& q, int activation, int64_t tiles, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(tiles), (q.n + avey::kLdCols - 1) / avey::kLdCols);
  switch (activation) {
    case AVEY_ACT_IDENTITY: avey::ln_dpre<T, 0><<<grid, avey::kLdThreads, 0, stream>>>(q); break;
    case AVEY_ACT_RELU2: avey::ln_dpre<T, 2><<<grid, avey::kLdThreads, 0, stream>>>(q); break;
    default: avey::ln_dpre<T, 1><<<grid, avey::kLdThreads, 0, stream>>>(q); break;  // one code for the bounded ones
  }
  return launched("ln_dpre");
}

template <typename T>
int backward(const AveyLinearParams* p, cudaStream_t stream) {
  const Layout l = layout(p, true);
  int rc = check_workspace(p, l);
  if (rc != AVEY_OK) return rc;
  char* ws = static_cast<char*>(p->workspace);
  Rows x, w, g{p->dy, p->dy_ld, 0};
  rc = pack_inputs(p, l, &x, &w, stream);
  if (rc != AVEY_OK) return rc;
  bool after = l.pack_x || l.pack_w;
  const bool sum_in_dx = l.sums && bias_in_dx(p);
  const float* partial = reinterpret_cast<const float*>(ws + l.partial);
  if (l.make_dpre || l.sums) {
    avey::LnDpre q{};
    q.offsets = p->offsets;
    q.groups = static_cast<int>(p->groups);
    q.rows = static_cast<int>(p->rows);
    q.n = static_cast<int>(p->d_out);
    q.dy = static_cast<const uint16_t*>(p->dy);
    q.dy_ld = p->dy_ld;
    q.dy_vec = whole_rows(p->dy, p->dy_ld);
    q.deriv = static_cast<const uint16_t*>(p->deriv);
    q.deriv_ld = up16(p->d_out);
    if (l.make_dpre) {
      q.dpre = reinterpret_cast<uint16_t*>(ws + l.dpre);
      q.dpre_ld = up8(p->d_out);
      g = {q.dpre, q.dpre_ld, 0};
    }
    if (l.sums) q.partial = reinterpret_cast<float*>(ws + l.partial);
    rc = launch_dpre<T>(q, p->activation, row_tiles(p, avey::kLdRows), stream);
    if (rc != AVEY_OK) return rc;
    after = true;
  }
  if (p->dx) {
    const int64_t mt = row_tiles(p, avey::kLnBM);
    avey::LnGeom q = geom(p, p->d_in, tile_cols(mt, p->d_in));
    q.kc = static_cast<int>(p->d_out);
    q.out = p->dx;
    q.out_ld = p->dx_ld;
    q.out_vec = whole_rows(p->dx, p->dx_ld);
    if (sum_in_dx) {
      q.bias_sums = partial;
      q.db = p->dbias;
    }
    Maps m;
    rc = avey_host::encode_rows16(p->dtype, g.p, p->d_out, p->rows, 1, g.ld * 2, 0, avey::kLnBM, &m.a);
    if (rc == AVEY_OK)
      rc = avey_host::encode_rows16(p->dtype, w.p, p->d_in, p->d_out, p->groups, w.ld * 2, w.gs * 2, 64, &m.b);
    if (rc == AVEY_OK && q.out_vec)
      rc = avey_host::encode_tiles(p->dtype, p->dx, p->d_in, p->rows, 1, p->dx_ld * 2, 0, &m.y);
    if (rc != AVEY_OK) return rc;
    const int64_t tiles = (mt + (p->offsets ? 1 : 0)) * q.n_nt;
    q.lets_next = p->dweight != nullptr;
    rc = launch_tc<avey::tc_linear<T, avey::kLnGradX, 0, false>>(m, q, tiles, after, stream);
    if (rc != AVEY_OK) return rc;
    after = true;
  }
  if (p->dweight) {
    avey::LnGeom q = geom(p, p->d_in, dw_cols(p));
    q.m = static_cast<int>(p->d_out);
    q.n_mt = (q.m + avey::kLnBM - 1) / avey::kLnBM;
    q.splits = l.splits;
    const bool parts = l.splits > 1;
    q.out = parts ? static_cast<void*>(ws + l.dw) : p->dweight;
    q.out_ld = parts ? (p->d_in + 3) / 4 * 4 : p->d_in;
    q.out_gs = p->d_out * q.out_ld;
    q.out_vec = !parts && whole_rows(p->dweight, p->d_in);
    Maps m;
    rc = avey_host::encode_rows16(p->dtype, g.p, p->d_out, p->rows, 1, g.ld * 2, 0, 64, &m.a);
    if (rc == AVEY_OK) rc = avey_host::encode_rows16(p->dtype, x.p, p->d_in, p->rows, 1, x.ld * 2, 0, 64, &m.b);
    if (rc == AVEY_OK && (parts || q.out_vec))
      rc = avey_host::encode_tiles(parts ? AVEY_F32 : p->dtype, q.out, p->d_in, p->d_out, q.splits * p->groups,
                                   q.out_ld * (parts ? 4 : 2), q.out_gs * (parts ? 4 : 2), &m.y);
    if (rc != AVEY_OK) return rc;
    const int64_t tiles = p->groups * q.n_mt * q.n_nt * q.splits;
    rc = parts ? launch_tc<avey::tc_linear<T, avey::kLnGradW, 0, true>>(m, q, tiles, after, stream)
               : launch_tc<avey::tc_linear<T, avey::kLnGradW, 0, false>>(m, q, tiles, after, stream);
    if (rc != AVEY_OK) return rc;
    if (parts) {
      const int64_t rows = p->groups * p->d_out, quads = rows * (q.out_ld / 4);
      const int grid = static_cast<int>(std::min<int64_t>((quads + 255) / 256, avey_host::multiprocessors() * 8ll));
      avey::ln_split_sum<T><<<grid, 256, 0, stream>>>(static_cast<const float*>(q.out), l.splits, rows,
                                                      static_cast<int>(p->d_in), q.out_ld,
                                                      static_cast<T*>(p->dweight));
      rc = launched("ln_split_sum");
      if (rc != AVEY_OK) return rc;
    }
  }
  if (l.sums && !sum_in_dx) {
    rc = launch_bias_sum<T>(p, partial, stream);
    if (rc != AVEY_OK) return rc;
  }
  return avey_host::clear_error();
}

}  // namespace

// The status word and the wait limit of this translation unit's kernels
// (ptx.cuh), for avey_device_status and avey_test_hooks_v1.
namespace avey_host {
int linear_flags(unsigned int* flags, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(flags, avey::g_devflags, sizeof(*flags));
  const unsigned int zero = 0;
  if (e == cudaSuccess && clear) e = cudaMemcpyToSymbol(avey::g_devflags, &zero, sizeof(zero));
  return e;
}
int linear_wait_limit(long long cycles) {
  return cudaMemcpyToSymbol(avey::g_wait_limit, &cycles, sizeof(cycles));
}
}  // namespace avey_host

extern "C" {

int avey_linear_workspace_size(const AveyLinearParams* p, int backward, uint64_t* bytes) {
  const int rc = validate(p, backward != 0);
  if (rc != AVEY_OK) return rc;
  if (!bytes) return fail(AVEY_ERR_ARGUMENT, "bytes is NULL");
  *bytes = layout(p, backward != 0).total;
  return avey_host::clear_error();
}

int avey_linear_fwd_v1(const AveyLinearParams* p, void* stream) {
  int rc = validate(p, false);
  if (rc != AVEY_OK) return rc;
  if (p->rows == 0) return avey_host::clear_error();
  rc = avey_host::device_ok();
  if (rc != AVEY_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  rc = p->dtype == AVEY_BF16 ? forward<__nv_bfloat16>(p, s) : forward<__half>(p, s);
  return rc == AVEY_OK ? avey_host::clear_error() : rc;
}

int avey_linear_bwd_v1(const AveyLinearParams* p, void* stream) {
  int rc = validate(p, true);
  if (rc != AVEY_OK) return rc;
  rc = avey_host::device_ok();
  if (rc != AVEY_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p->rows == 0) {
    // No rows: the weights' gradients are zero.
    cudaError_t e = cudaSuccess;
    if (p->dweight) e = cudaMemsetAsync(p->dweight, 0, static_cast<size_t>(p->groups) * p->d_out * p->d_in * 2, s);
    if (e == cudaSuccess && p->dbias)
      e = cudaMemsetAsync(p->dbias, 0, static_cast<size_t>(p->groups) * p->d_out * 2, s);
    return e == cudaSuccess ? avey_host::clear_error() : fail(AVEY_ERR_CUDA, cudaGetErrorString(e));
  }
  return p->dtype == AVEY_BF16 ? backward<__nv_bfloat16>(p, s) : backward<__half>(p, s);
}

}  // extern "C"
