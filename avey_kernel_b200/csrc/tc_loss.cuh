// Softmax cross entropy of z = x W^T over a vocabulary, and its gradients, on
// tcgen05 CTA pairs (avey_loss_*), without keeping z:
//
//   stats  (c, s) of every row over a segment of the vocabulary, where
//          s = sum_j 2^(z_j log2 e - c), and the target's z
//   grad   dz_ij = a_i 2^(z_ij log2 e - lse_i) - b_i [j = t_i] for a piece of the
//          vocabulary, z computed again
//   dX     dx (+)= dz W over the piece       dW    dW = dz^T x for the piece
//
// c is the running maximum, so every power is at most 1; lse_i = c + log2 s is
// kept in base 2, as the hardware's exponential takes it, with what its rounding left
// out, which goes into a_i. a_i and b_i hold the gradient that comes in, the z loss's factor and a scale that dX and dW divide by
// (CeScale). dz is rounded to the operand type once, as the tensor cores need it; all
// sums are fp32.
//
// Bounds: 2 M V d flops for the loss and 6 M V d for the gradients on the tensor
// cores. A cluster of two CTAs computes 256 x 256 tiles (cta_group::2): per K
// block of 64 a CTA takes in 32 KB for 512 cycles of products, just what an SM
// can (64 bytes a cycle); a CTA alone on a 128 x 256 tile would take in 48 KB.
// Warp 0 issues TMA, warp 1 of the even CTA tcgen05.mma into one of two TMEM
// accumulators, warps 4-19 of each CTA drain the other one. Every wait is bounded.
//
// The pairs claim units of work from a counter, the longest first, so that they end
// together: a unit is up to 4 column tiles of one row tile for the statistics and dz (a
// row's numbers stay in registers over it), else one tile. The gradients' launches
// hold three kinds: dX and dW of one piece and dz of the next (in the other half of
// dz), whose short units fill what the long ones leave of the last wave. (With a
// launch for each kind 48 tiles of dX on 74 pairs took 370 us instead of 150.) Who
// takes a unit does not change its result.
#pragma once

#include "linear_steps.cuh"

namespace avey {

constexpr int kCeThreads = kLnThreads;
constexpr int kCeBM = 256;                  // rows of a pair's tile
constexpr int kCeHalfA = 128 * kLnBK * 2;   // a CTA's 128 rows of A: 16 KB
constexpr int kCeMaxSeg = 4;                // column tiles of a unit
constexpr int kCeMaxStages = 8;
constexpr int kCeRing = 196608;
constexpr int kCeStaging = kLnEpiWarps * kLnStageTile;
constexpr int kCeCtrlBytes = 512;
constexpr int kCeSmem = 1024 + kCeRing + kCeStaging + kCeCtrlBytes;

enum CeKind { kCeStats = 0, kCeGrad = 1, kCeDx = 2, kCeDw = 3 };
template <int K>
using CeKindOf = std::integral_constant<int, K>;

// Units of one kind in a launch.
struct CeJob {
  int kind, units;
  int m, n, nk;            // output rows and columns, K blocks
  int bn, n_mt, n_nt;      // columns of a tile, tiles
  int seg;                 // stats, grad: column tiles of a unit; dX: K ranges of a tile
};
constexpr int kCeJobs = 3;

struct CeGeom {
  CeJob job[kCeJobs];
  int units;               // of all kinds
  int stages, stage_bytes;
  unsigned int* claimed;   // the next unit, zero before; or null
  int rows, vocab;
  int col0;                // grad: the piece's first column
  const void* targets;
  int64_t target_stride;
  int target64;
  int64_t ignore;
  float2* partial;         // stats: [segments][rows]
  float* picked;           // stats: the target's z, [rows]
  const float* lse;        // grad: [rows], base 2
  const float2* coef;      // grad: (a, b) of every row
  const uint32_t* largest; // bits of the largest |b| and |a|
  uint16_t* dz;            // grad: rows of dz_ld values, a multiple of 16
  int64_t dz_ld;
  void* dx;                // 16 bits; null: fp32 sums by map_dx
  int64_t dx_ld;
  int dx_vec, dx_add;      // rows stored by TMA; sums are added to
  void* dw;
  int64_t dw_ld;
  int dw_vec;
  const uint8_t* dirty;    // dW: K blocks whose rows come from the second map
  int test_stall;
};

// The target of a row: its column, -1 for a row that is ignored, -2 for a
// target outside the vocabulary.
__device__ __forceinline__ int ce_target(const void* targets, int64_t stride, int wide, int64_t ignore, int vocab,
                                         int row) {
  const int64_t t = wide ? __ldg(static_cast<const long long*>(targets) + row * stride)
                         : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(targets) + row * stride));
  if (t == ignore) return -1;
  return t >= 0 && t < vocab ? static_cast<int>(t) : -2;
}

// What dz is multiplied by before it is rounded, and its inverse. A row's b is its share
// of the gradient that comes in: divided by the largest |b| (largest[0]) it is exactly 1
// where all rows count alike, so that a target's dz, p - 1, keeps small p's to bf16's
// eight bits below 1 (dz = (p - 1) / rows, rounded, gave dx and dW twice the error). f16's
// range starts at 2^-14: the power of two brings the largest |a| and |b| (largest[1]: |a|)
// to between 2^12 and 2^13.
struct CeScale {
  float apply, undo;
};
__device__ __forceinline__ CeScale ce_scale(const uint32_t* largest) {
  // (Below 2^-100 the inverse would leave fp32's range: rows that small count less than 1.)
  const float b = fmaxf(__uint_as_float(__ldg(largest)), 0x1p-100f);
  const float ratio = fmaxf(1.f, __fdiv_rn(__uint_as_float(__ldg(largest + 1)), b));
  const int e = min(static_cast<int>(__float_as_uint(ratio) >> 23) - 127, 100);  // 2^e <= ratio < 2^(e + 1)
  const float up = __uint_as_float(static_cast<uint32_t>(127 + 12 - e) << 23);
  return {__fdiv_rn(up, b), __fdiv_rn(b, up)};
}

constexpr int kCeAhead = 4;  // units that the scheduler may be ahead of the last reader

struct CeCtrl {
  uint64_t full[kCeMaxStages], empty[kCeMaxStages];
  uint64_t unit_full[kCeAhead], unit_empty[kCeAhead];
  uint64_t want;               // the even CTA's TMA lane is near the end of its unit
  uint64_t acc_full[2], acc_empty[2];
  uint64_t met[4], joined[4];  // stats: a row quarter's parts have been written, and read
  uint64_t settled;
  int unit[kCeAhead];
  uint32_t failed;
  uint32_t tmem_base;
};
static_assert(sizeof(CeCtrl) <= kCeCtrlBytes, "control block too large");

// Arrive on an mbarrier of either CTA. Nothing in memory is handed over with it (the
// reads of tensor memory before it are ordered by their wait and fence), so it is
// relaxed: a release for the cluster makes each warp wait for a fence.
__device__ __forceinline__ void ce_arrive(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// The scheduler (a lane of the even CTA) hands unit u, the i-th of the pair, to every
// role of both CTAs: the store counts as 4 bytes on the barrier beside it.
__device__ __forceinline__ bool ce_hand(CeCtrl* ctrl, int i, int u) {
  const int slot = i % kCeAhead;
  if (i >= kCeAhead && !mbar_wait(smem_u32(&ctrl->unit_empty[slot]), (i / kCeAhead - 1) & 1)) return false;
#pragma unroll
  for (uint32_t cta = 0; cta < 2; ++cta)
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.u32 [%0], %1, [%2];" ::"r"(
                     mapa_shared(smem_u32(&ctrl->unit[slot]), cta)),
                 "r"(u), "r"(mapa_shared(smem_u32(&ctrl->unit_full[slot]), cta))
                 : "memory");
  return true;
}
// The pair's i-th unit (-1: none is left, or a wait gave up). Without a counter (units
// of one kind) a pair takes every pairs-th one.
__device__ __forceinline__ int ce_unit(const CeGeom& q, CeCtrl* ctrl, int i) {
  if (!q.claimed) {
    const int64_t u = (blockIdx.x >> 1) + static_cast<int64_t>(i) * (gridDim.x >> 1);
    return u < q.units ? static_cast<int>(u) : -1;
  }
  const int slot = i % kCeAhead;
  if (!mbar_wait(smem_u32(&ctrl->unit_full[slot]), (i / kCeAhead) & 1)) return -1;
  return *reinterpret_cast<volatile int*>(&ctrl->unit[slot]);
}
// By one lane of each role once it has been read.
__device__ __forceinline__ void ce_unit_read(const CeGeom& q, CeCtrl* ctrl, int i) {
  if (q.claimed) ce_arrive(mapa_shared(smem_u32(&ctrl->unit_empty[i % kCeAhead]), 0));
}
// The same for a whole warp.
__device__ __forceinline__ int ce_warp_unit(const CeGeom& q, CeCtrl* ctrl, int i) {
  const int u = __reduce_min_sync(0xFFFFFFFFu, ce_unit(q, ctrl, i));
  if (u >= 0 && (threadIdx.x & 31) == 0) ce_unit_read(q, ctrl, i);
  return u;
}

// A unit's tiles: `count` column tiles from (mt, nt) on, K blocks k0 to k1 of them.
struct CeUnit {
  int job, mt, nt, count, k0, k1;
  int part;  // stats: the segment; dX: where the sums of a cut tile go, or -1
};
template <bool STATS>
__device__ __forceinline__ CeUnit ce_set_unit(const CeGeom& q, int u) {
  CeUnit c;
  c.job = 0;
  if (!STATS) {
#pragma unroll
    for (int j = 0; j < kCeJobs - 1; ++j)
      if (c.job == j && u >= q.job[j].units) {
        u -= q.job[j].units;
        c.job = j + 1;
      }
  }
  const CeJob& b = q.job[c.job];
  c.k0 = 0;
  c.k1 = b.nk;
  c.count = 1;
  c.part = -1;
  if (STATS || b.kind == kCeGrad) {
    c.part = u / b.n_mt;  // rows first: the pairs at work share W's rows in L2
    c.mt = u - c.part * b.n_mt;
    c.nt = c.part * b.seg;
    c.count = min(b.seg, b.n_nt - c.nt);
  } else {
    const int tiles = b.n_mt * b.n_nt, split = u / tiles, t = u - split * tiles;
    c.mt = t / b.n_nt;
    c.nt = t - c.mt * b.n_nt;
    if (b.seg > 1) {
      c.k0 = static_cast<int>(static_cast<int64_t>(b.nk) * split / b.seg);
      c.k1 = static_cast<int>(static_cast<int64_t>(b.nk) * (split + 1) / b.seg);
      c.part = u;
    }
  }
  return c;
}

__device__ __forceinline__ void tma_reduce_add_3d(const void* tmap, uint32_t src, int x, int y, int z) {
  asm volatile(
      "cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
          reinterpret_cast<uint64_t>(tmap)),
      "r"(x), "r"(y), "r"(z), "r"(src)
      : "memory");
}

// What an epilogue lane holds of its row.
struct CeRow {
  int target;
  float lse, a, b;  // grad
  float c, s;       // stats
};

// (c, s) of two parts of a row.
__device__ __forceinline__ void ce_join(float& c, float& s, float c2, float s2) {
  const float top = fmaxf(c, c2);
  // A part without a column, or of infinite negative logits, has c = -inf and adds nothing.
  const float base = top == -INFINITY ? 0.f : top;
  s = s * ln_exp2(c - base) + s2 * ln_exp2(c2 - base);
  c = top;
}

// 32 columns of a row from column col on: the running maximum and sum.
template <bool EDGE>
__device__ __forceinline__ void ce_stats32(uint32_t (&o)[32], int left, CeRow& r) {
  constexpr float kLog2e = 1.4426950408889634f;
  if (EDGE) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j >= left) o[j] = 0xFF800000u;
  }
  float top = __uint_as_float(o[0]);
#pragma unroll
  for (int j = 1; j < 32; ++j) top = fmaxf(top, __uint_as_float(o[j]));
  const float c = fmaxf(r.c, top * kLog2e);
  const float base = c == -INFINITY ? 0.f : c;
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    s0 += ln_exp2(fmaf(__uint_as_float(o[j]), kLog2e, -base));
    s1 += ln_exp2(fmaf(__uint_as_float(o[j + 1]), kLog2e, -base));
  }
  r.s = r.s * ln_exp2(r.c - base) + (s0 + s1);
  r.c = c;
}

// 32 columns of a row of dz to global memory, from the lane's registers as whole 32-byte
// sectors: rows are padded to 16 columns. (Through shared memory and TMA, with a proxy
// fence a tile, the launch took 264,000 cycles instead of 261,000 at 4096 x 32768, width
// 768; without any epilogue 229,000.)
template <typename T, bool HIT>
__device__ __forceinline__ void ce_grad32(const uint32_t (&o)[32], int at, const CeRow& r, uint16_t* out, int left) {
  constexpr float kLog2e = 1.4426950408889634f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = 16 * h + 2 * j;
      float d0 = r.a * ln_exp2(fmaf(__uint_as_float(o[i]), kLog2e, -r.lse));
      float d1 = r.a * ln_exp2(fmaf(__uint_as_float(o[i + 1]), kLog2e, -r.lse));
      if (HIT) {
        if (i == at) d0 -= r.b;
        if (i + 1 == at) d1 -= r.b;
      }
      y[j] = r.target == -1 ? 0u : ln_pack<T>(d0, d1);
    }
    if (16 * h < left) ln_st32(out + 16 * h, y);
  }
}

struct CeMaps {
  CUtensorMap x, w;           // the logits' operands, K-major
  CUtensorMap y_dx;           // where dX goes (16 bits or fp32 sums)
  CUtensorMap dz_x, w_x;      // dX's operands
  CUtensorMap dz_w, x_w, x2;  // dW's operands, and the copy of x's blocks that hold ignored rows
  CUtensorMap y_dw, parts;
};

// Arrive on the barrier at this offset in both CTAs when the products issued so far are done.
__device__ __forceinline__ void ce_commit_both(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

// The ring as a producing or consuming lane walks it.
struct CeRingAt {
  int st = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++st == stages) {
      st = 0;
      ph ^= 1u;
    }
  }
};

// One CTA's loads for a unit (`half` columns of B a tile from bcol on). The next unit
// is asked for eight K blocks before the end: late, so that the pairs end together, and
// early enough for its number to arrive in time. The loops of the TMA and MMA lanes are
// compiled for each kind: with the kind looked up in them dX and dW of 4096 x 32768
// (width 768) took 689,000 cycles instead of 458,000.
template <int KIND>
__device__ __forceinline__ bool ce_load_unit(const CeMaps& maps, const CeGeom& q, const CeUnit& c, CeCtrl* ctrl,
                                             uint32_t base, bool leader, int arow, int bcol, int bn, int half,
                                             CeRingAt& at, int& fills, uint64_t keep) {
  const uint32_t bytes = 2u * (kCeHalfA + half * kLnBK * 2);
  const int stages = q.stages, stage_bytes = q.stage_bytes, k0 = c.k0, k1 = c.k1;
  const int count = KIND == kCeStats || KIND == kCeGrad ? c.count : 1;
  const int ask = max(k0, k1 - 8);
  for (int t = 0; t < count; ++t, bcol += bn) {
#pragma unroll 1
    for (int kk = k0; kk < k1; ++kk) {
      if (kk == ask && leader && t == count - 1 && q.claimed) mbar_arrive(smem_u32(&ctrl->want));
      if (fills >= stages && !mbar_wait(smem_u32(&ctrl->empty[at.st]), at.ph ^ 1u)) return false;
      const uint32_t mine = smem_u32(&ctrl->full[at.st]), full = mapa_shared(mine, 0);
      const uint32_t sa = base + at.st * stage_bytes, sb = sa + kCeHalfA;
      const int kx = kk * kLnBK;
      if (leader) mbar_arrive_expect_tx(mine, bytes);
      if constexpr (KIND == kCeStats || KIND == kCeGrad) {
        tma_load_3d_pair(sa, &maps.x, full, kx, arow, 0, keep);
        tma_load_3d_pair(sb, &maps.w, full, kx, bcol, 0, keep);
      } else if constexpr (KIND == kCeDx) {
        tma_load_3d_pair(sa, &maps.dz_x, full, kx, arow, 0, keep);
        tma_load_3d_pair(sb, &maps.w_x, full, bcol, kx, 0, keep);
        if (half > 64) tma_load_3d_pair(sb + kLnMnBox, &maps.w_x, full, bcol + 64, kx, 0, keep);
      } else {
        tma_load_3d_pair(sa, &maps.dz_w, full, arow, kx, 0, keep);
        tma_load_3d_pair(sa + kLnMnBox, &maps.dz_w, full, arow + 64, kx, 0, keep);
        const CUtensorMap* mb = __ldg(q.dirty + kk) ? &maps.x2 : &maps.x_w;
        tma_load_3d_pair(sb, mb, full, bcol, kx, 0, keep);
        if (half > 64) tma_load_3d_pair(sb + kLnMnBox, mb, full, bcol + 64, kx, 0, keep);
      }
      ++fills;
      at.next(stages);
    }
  }
  return true;
}

// The products of a unit.
template <int KIND, uint32_t FMT>
__device__ __forceinline__ bool ce_multiply_unit(const CeGeom& q, const CeUnit& c, CeCtrl* ctrl, uint32_t base,
                                                 uint32_t tmem, int bn, CeRingAt& at, int& it) {
  constexpr bool kAMn = KIND == kCeDw, kBMn = KIND == kCeDx || KIND == kCeDw;
  const uint32_t idesc = idesc_f16(FMT, kCeBM, static_cast<uint32_t>(bn), kAMn ? 1u : 0u, kBMn ? 1u : 0u);
  const uint64_t da0 = kAMn ? smem_desc_sw128(base, kLnMnBox, 1024) : smem_desc_sw128(base, 16, 1024);
  const uint64_t db0 =
      kBMn ? smem_desc_sw128(base + kCeHalfA, kLnMnBox, 1024) : smem_desc_sw128(base + kCeHalfA, 16, 1024);
  constexpr uint32_t ka = kAMn ? (2048u >> 4) : 2u, kb = kBMn ? (2048u >> 4) : 2u;
  const int stages = q.stages, stage_bytes = q.stage_bytes, blocks = c.k1 - c.k0;
  const int count = KIND == kCeStats || KIND == kCeGrad ? c.count : 1;
  for (int t = 0; t < count; ++t, ++it) {
    const int buf = it & 1;
    if (it >= 2) {
      if (!mbar_wait(smem_u32(&ctrl->acc_empty[buf]), ((it >> 1) - 1) & 1)) return false;
      tc_fence_after();
    }
    const uint32_t d_tmem = tmem + static_cast<uint32_t>(buf * 256);
#pragma unroll 1
    for (int kk = 0; kk < blocks; ++kk) {
      if (!mbar_wait(smem_u32(&ctrl->full[at.st]), at.ph)) return false;
      tc_fence_after();
      const uint32_t adv = static_cast<uint32_t>(at.st * stage_bytes) >> 4;
#pragma unroll
      for (int k = 0; k < kLnBK / 16; ++k)
        tc_mma_f16_pair(d_tmem, da0 + adv + ka * k, db0 + adv + kb * k, idesc, (kk != 0 || k != 0) ? 1u : 0u);
      ce_commit_both(smem_u32(&ctrl->empty[at.st]));
      at.next(stages);
    }
    ce_commit_both(smem_u32(&ctrl->acc_full[buf]));
  }
  return true;
}

// Store a warp's 32 x 32 fp32 sums (from TMEM) at column x, row y of a map.
__device__ __forceinline__ void ce_store_f32(uint32_t tb, uint32_t tile, int lane, const CUtensorMap* map, int x, int y,
                                             bool add, uint64_t policy) {
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    uint32_t o[16];
    ln_tmem_ld16(tb + 16 * hh, false, o);
    ln_tile_free(lane);
#pragma unroll
    for (int p = 0; p < 4; ++p) ln_sts(ln_piece(tile, lane, p), o[4 * p], o[4 * p + 1], o[4 * p + 2], o[4 * p + 3]);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (add) tma_reduce_add_3d(map, tile, x + 16 * hh, y, 0);
      else tma_store_3d(map, tile, x + 16 * hh, y, 0, policy);
      bulk_commit_group();
    }
  }
}

template <typename T, bool STATS>
__global__ void __launch_bounds__(kCeThreads, 1)
    ce_product(const __grid_constant__ CeMaps maps, const __grid_constant__ CeGeom q) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t staging = base + kCeRing;
  CeCtrl* ctrl = reinterpret_cast<CeCtrl*>(smem_raw + (base - raw) + kCeRing + kCeStaging);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  if (tid == 0) {
    for (int s = 0; s < q.stages; ++s) {
      mbar_init(smem_u32(&ctrl->full[s]), 1);
      mbar_init(smem_u32(&ctrl->empty[s]), 1);
    }
    for (int i = 0; i < kCeAhead; ++i) {
      mbar_init(smem_u32(&ctrl->unit_full[i]), 1);
      // Both CTAs' TMA lanes and epilogue warps, and the MMA lane.
      mbar_init(smem_u32(&ctrl->unit_empty[i]), 2 * (1 + kLnEpiWarps) + 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctrl->acc_full[i]), 1);
      mbar_init(smem_u32(&ctrl->acc_empty[i]), 2 * kLnEpiWarps);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(&ctrl->met[i]), 3);
      mbar_init(smem_u32(&ctrl->joined[i]), 1);
    }
    mbar_init(smem_u32(&ctrl->want), 1);
    mbar_init(smem_u32(&ctrl->settled), 1);
    ctrl->failed = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&ctrl->tmem_base), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers and tensor memory are set up
  tc_fence_after();
  const uint32_t tmem = ctrl->tmem_base;
  int fills = 0;
  // The set-up ran beside the end of the step before; what that wrote is read from here on.
  griddep_launch_dependents();
  griddep_wait();

  if (warp == 0) {
    // ============================================================ TMA producer (both CTAs)
    if (lane == 0) {
      const uint64_t keep = l2_policy_evict_last();
      CeRingAt at;
      bool alive = !q.test_stall;
      for (int i = 0; alive; ++i) {
        // The lane that expects the unit's four bytes.
        if (q.claimed) mbar_arrive_expect_tx(smem_u32(&ctrl->unit_full[i % kCeAhead]), 4);
        const int u = ce_unit(q, ctrl, i);
        if (u < 0) break;
        ce_unit_read(q, ctrl, i);
        const CeUnit c = ce_set_unit<STATS>(q, u);
        const CeJob& b = q.job[c.job];
        const int bn = b.bn, half = bn / 2, kind = b.kind;  // half: this CTA's columns of B
        const int arow = c.mt * kCeBM + static_cast<int>(rank) * 128;
        const int bcol = c.nt * bn + static_cast<int>(rank) * half;
        auto load = [&](auto k) {
          return ce_load_unit<decltype(k)::value>(maps, q, c, ctrl, base, leader, arow, bcol, bn, half, at, fills, keep);
        };
        if constexpr (STATS) alive = load(CeKindOf<kCeStats>{});
        else if (kind == kCeGrad) alive = load(CeKindOf<kCeGrad>{});
        else if (kind == kCeDx) alive = load(CeKindOf<kCeDx>{});
        else alive = load(CeKindOf<kCeDw>{});
      }
      // Until the leader's commits have released every stage that this CTA filled:
      // no signal of theirs may come after the CTA is gone.
      for (int f = max(0, fills - q.stages); alive && f < fills; ++f)
        alive = mbar_wait(smem_u32(&ctrl->empty[f % q.stages]), static_cast<uint32_t>(f / q.stages) & 1u);
      if (!alive) ctrl->failed = 1;
    }
  } else if (warp == 1) {
    // ============================================================ MMA issuer (even CTA)
    if (lane == 0 && leader) {
      constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      CeRingAt at;
      int it = 0, u;
      bool alive = true;
      for (int i = 0; alive && (u = ce_unit(q, ctrl, i)) >= 0; ++i) {
        ce_unit_read(q, ctrl, i);
        const CeUnit c = ce_set_unit<STATS>(q, u);
        const CeJob& b = q.job[c.job];
        const int bn = b.bn, kind = b.kind;
        auto multiply = [&](auto k) {
          return ce_multiply_unit<decltype(k)::value, fmt>(q, c, ctrl, base, tmem, bn, at, it);
        };
        if constexpr (STATS) alive = multiply(CeKindOf<kCeStats>{});
        else if (kind == kCeGrad) alive = multiply(CeKindOf<kCeGrad>{});
        else if (kind == kCeDx) alive = multiply(CeKindOf<kCeDx>{});
        else alive = multiply(CeKindOf<kCeDw>{});
      }
      if (!alive) ctrl->failed = 1;
    }
  } else if (warp == 3) {
    // ============================================================ scheduler (even CTA)
    if (lane == 0 && leader && q.claimed) {
      for (int i = 0, u = 0; u >= 0; ++i) {
        if (i > 0 && !mbar_wait(smem_u32(&ctrl->want), (i - 1) & 1)) break;
        const unsigned int claim = atomicAdd(q.claimed, 1u);
        u = claim < static_cast<unsigned int>(q.units) ? static_cast<int>(claim) : -1;
        if (!ce_hand(ctrl, i, u)) break;
      }
    }
  } else if (warp >= 4) {
    // ============================================================ epilogue (both CTAs)
    const int h = (warp - 4) >> 2;  // column part of the tile
    const int wq = warp & 3;        // TMEM lane quarter
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t tile = staging + static_cast<uint32_t>((warp - 4) * kLnStageTile);
    const uint32_t freed0 = mapa_shared(smem_u32(&ctrl->acc_empty[0]), 0);
    const uint32_t freed1 = mapa_shared(smem_u32(&ctrl->acc_empty[1]), 0);
    const uint64_t policy = l2_policy_evict_normal();
    const CeScale scale = STATS ? CeScale{1.f, 1.f} : ce_scale(q.largest);
    CeRow r{};
    bool alive = true;
    int it = 0, u;
    for (int i = 0; alive && (u = ce_warp_unit(q, ctrl, i)) >= 0; ++i) {
      const CeUnit c = ce_set_unit<STATS>(q, u);
      const CeJob b = q.job[c.job];
      const int part = max(32, b.bn >> 2);
      const int row0 = c.mt * kCeBM + static_cast<int>(rank) * 128 + wq * 32, row = row0 + lane;
      const bool logits = STATS || b.kind == kCeGrad;
      if (logits) {
        r.target = row < b.m ? ce_target(q.targets, q.target_stride, q.target64, q.ignore, q.vocab, row) : -1;
        if (!STATS) {
          const float2 ab = row < b.m ? __ldg(q.coef + row) : make_float2(0.f, 0.f);
          r.a = ab.x * scale.apply;
          r.b = ab.y * scale.apply;
          r.lse = row < b.m ? __ldg(q.lse + row) : 0.f;
        }
        r.c = -INFINITY;
        r.s = 0.f;
      }
      for (int t = 0; t < c.count; ++t, ++it) {
        const int buf = it & 1;
        const int col0 = (c.nt + t) * b.bn + h * part;
        const int nch = row0 < b.m && h * part < b.bn ? max(0, min(part, b.n - col0) + 31) / 32 : 0;
        if (alive && !ln_warp_wait(smem_u32(&ctrl->acc_full[buf]), (it >> 1) & 1)) {
          if (lane == 0) ctrl->failed = 1;
          alive = false;
        }
        if (!alive) break;
        tc_fence_after();
        const uint32_t tb = tmem + lane_off + static_cast<uint32_t>(buf * 256 + h * part);
#pragma unroll 1
        for (int ch = 0; ch < nch; ++ch) {
          const int col = col0 + ch * 32;
          if (logits) {
            uint32_t o[32];
            tmem_ld32(tb + ch * 32, o);
            tmem_wait_ld(o);
            const int at = r.target - q.col0 - col;  // the target's place among the 32
            const bool hit = __any_sync(0xFFFFFFFFu, r.target >= 0 && at >= 0 && at < 32);
            if constexpr (STATS) {
              if (hit) {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (j == at && r.target >= 0) q.picked[row] = __uint_as_float(o[j]);
              }
              if (col + 32 <= b.n) ce_stats32<false>(o, 32, r);
              else ce_stats32<true>(o, b.n - col, r);
            } else {
              if (row < b.m) {
                uint16_t* out = q.dz + static_cast<int64_t>(row) * q.dz_ld + col;
                if (hit) ce_grad32<T, true>(o, r.target >= 0 ? at : -1, r, out, b.n - col);
                else ce_grad32<T, false>(o, -1, r, out, b.n - col);
              }
            }
          } else if constexpr (!STATS) {
            if (c.part >= 0) {
              ce_store_f32(tb + ch * 32, tile, lane, &maps.parts, col - c.nt * b.bn,
                           c.part * kCeBM + (row0 - c.mt * kCeBM), false, policy);
            } else if (b.kind == kCeDx && !q.dx) {
              ce_store_f32(tb + ch * 32, tile, lane, &maps.y_dx, col, row0, q.dx_add, policy);
            } else {
              ln_tile_free(lane);
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                uint32_t o[16];
                ln_tmem_ld16(tb + ch * 32 + 16 * hh, false, o);
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                  uint32_t y[4];
#pragma unroll
                  for (int j = 0; j < 4; ++j)
                    y[j] = ln_pack<T>(__uint_as_float(o[8 * p + 2 * j]) * scale.undo,
                                      __uint_as_float(o[8 * p + 2 * j + 1]) * scale.undo);
                  ln_sts(ln_piece(tile, lane, 2 * hh + p), y[0], y[1], y[2], y[3]);
                }
              }
              const bool dx = b.kind == kCeDx;
              if (dx ? q.dx_vec : q.dw_vec) {
                ln_tma_tile(tile, lane, dx ? &maps.y_dx : &maps.y_dw, col, row0, 0, policy);
              } else {
                const LnLines l{row0 + (lane >> 2), b.m, col + (lane & 3) * 8, b.n};
                __syncwarp();
                ln_store_tile_by_column(tile, lane, static_cast<uint16_t*>(dx ? q.dx : q.dw), dx ? q.dx_ld : q.dw_ld, l);
                __syncwarp();
              }
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) ce_arrive(buf ? freed1 : freed0);
      }
      if constexpr (STATS) {
        if (!alive) break;
        // The four parts of a row meet in shared memory.
        const uint32_t meet = staging + static_cast<uint32_t>(wq * 32 + lane) * 8;
        if (h > 0) {
          alive = i == 0 || ln_warp_wait(smem_u32(&ctrl->joined[wq]), (i - 1) & 1);
          asm volatile("st.shared.v2.f32 [%0], {%1,%2};" ::"r"(meet + h * 1024), "f"(r.c), "f"(r.s) : "memory");
          __syncwarp();
          if (lane == 0 && alive) mbar_arrive(smem_u32(&ctrl->met[wq]));
        } else {
          alive = ln_warp_wait(smem_u32(&ctrl->met[wq]), i & 1);
#pragma unroll
          for (int j = 1; j < 4; ++j) {
            float c2, s2;
            asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(c2), "=f"(s2) : "r"(meet + j * 1024) : "memory");
            ce_join(r.c, r.s, c2, s2);
          }
          if (row < b.m && alive) q.partial[static_cast<int64_t>(c.part) * q.rows + row] = make_float2(r.c, r.s);
          __syncwarp();
          if (lane == 0 && alive) mbar_arrive(smem_u32(&ctrl->joined[wq]));
        }
        if (!alive && lane == 0) ctrl->failed = 1;
      }
    }
    if (lane == 0) bulk_wait_read_all();
  }

  // ---------------------------------------------------------------- teardown
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (ctrl->failed) {
    // The even CTA's barriers count the loads of both CTAs.
    if (tid == 0 && leader) ln_settle_loads(ctrl->full, q.stages, fills);
    if (tid == 32 && leader) {
      tc_commit_pair(smem_u32(&ctrl->settled));
      ln_settle(smem_u32(&ctrl->settled), 0);
    }
    __syncthreads();
  }
  cluster_sync();  // no signal goes to either CTA, and no product reads it, after this
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ---------------------------------------------------------------- few rows

// The statistics of a few rows: W is read once, straight from global memory into
// mma.sync fragments (16 rows of it by up to 8 of x; bound: its bytes). A lane takes 16
// consecutive k (32 bytes) of a 64-wide step for its fragments, so that four lanes read
// a whole line; the order of k inside a product is free as long as both operands agree. A
// warp takes 16 rows of W at a time and keeps (c, s) of the rows of x; a CTA's warps are
// joined at the end. 131072 x 1024: 49 us in calls in a row, 5.5 TB/s.
constexpr int kCfWarps = 8, kCfRows = 8;
struct CeFew {
  int rows, vocab, width;
  const uint16_t* x;
  const uint16_t* w;
  int64_t x_ld, w_ld;
  int x_vec, w_vec;
  const void* targets;
  int64_t target_stride;
  int target64;
  int64_t ignore;
  float2* partial;  // [gridDim.x][rows]
  float* picked;
};

template <typename T>
__global__ void __launch_bounds__(32 * kCfWarps) ce_few(const CeFew q) {
  constexpr float kLog2e = 1.4426950408889634f;
  __shared__ float2 meet[kCfWarps][kCfRows];
  griddep_launch_dependents();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tg = lane & 3;
  int target[2];
  float c[2], s[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = 2 * tg + j;
    target[j] = row < q.rows ? ce_target(q.targets, q.target_stride, q.target64, q.ignore, q.vocab, row) : -1;
    c[j] = -INFINITY;
    s[j] = 0.f;
  }
  const int groups = (q.vocab + 15) / 16;
  for (int group = blockIdx.x * kCfWarps + warp; group < groups; group += gridDim.x * kCfWarps) {
    const int v0 = group * 16 + g, v1 = v0 + 8;
    const uint16_t* w0 = q.w + v0 * q.w_ld;
    const uint16_t* w1 = q.w + v1 * q.w_ld;
    const bool in0 = v0 < q.vocab, in1 = v1 < q.vocab;
    float z[4] = {};
#pragma unroll 2
    for (int k0 = 0; k0 < q.width; k0 += 128) {
      LnOct2 a[2], b[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = k0 + 64 * h + 16 * tg, left = q.width - k;
        a[h] = ln_load16(w0 + k, in0 ? left : 0, q.w_vec);
        b[h] = ln_load16(w1 + k, in1 ? left : 0, q.w_vec);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = k0 + 64 * h + 16 * tg, left = q.width - k;
        const uint32_t wa[8] = {a[h].a.x, a[h].a.y, a[h].a.z, a[h].a.w, a[h].b.x, a[h].b.y, a[h].b.z, a[h].b.w};
        const uint32_t wb[8] = {b[h].a.x, b[h].a.y, b[h].a.z, b[h].a.w, b[h].b.x, b[h].b.y, b[h].b.z, b[h].b.w};
        const LnOct2 xv = ln_load16(q.x + g * q.x_ld + k, g < q.rows ? left : 0, q.x_vec);
        const uint32_t xw[8] = {xv.a.x, xv.a.y, xv.a.z, xv.a.w, xv.b.x, xv.b.y, xv.b.z, xv.b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          ln_mma<T>(z, wa[2 * i], wb[2 * i], wa[2 * i + 1], wb[2 * i + 1], xw[2 * i], xw[2 * i + 1]);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float z0 = in0 ? z[j] : -INFINITY, z1 = in1 ? z[j + 2] : -INFINITY;
      if (target[j] >= 0) {
        if (target[j] == v0) q.picked[2 * tg + j] = z0;
        if (target[j] == v1) q.picked[2 * tg + j] = z1;
      }
      const float top = fmaxf(c[j], fmaxf(z0, z1) * kLog2e), base = top == -INFINITY ? 0.f : top;
      s[j] = s[j] * ln_exp2(c[j] - base) + (ln_exp2(fmaf(z0, kLog2e, -base)) + ln_exp2(fmaf(z1, kLog2e, -base)));
      c[j] = top;
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) {
      const float c2 = __shfl_xor_sync(0xFFFFFFFFu, c[j], d), s2 = __shfl_xor_sync(0xFFFFFFFFu, s[j], d);
      ce_join(c[j], s[j], c2, s2);
    }
    if (g == 0) meet[warp][2 * tg + j] = make_float2(c[j], s[j]);
  }
  __syncthreads();
  const int row = threadIdx.x;
  if (row < q.rows) {
    float2 v = meet[0][row];
    for (int i = 1; i < kCfWarps; ++i) ce_join(v.x, v.y, meet[i][row].x, meet[i][row].y);
    q.partial[static_cast<int64_t>(blockIdx.x) * q.rows + row] = v;
  }
}

// ---------------------------------------------------------------- steps around the products

struct CeRows {
  int rows, vocab, segments;
  const void* targets;
  int64_t target_stride;
  int target64;
  int64_t ignore;
  const float2* partial;   // [segments][rows]
  const float* picked;
  float z_loss;
  float* each;             // losses of the rows
  float* lse;              // [rows], base 2
  float* low;              // [rows]: what its rounding left of it; or null
  int per;                 // rows of a block, a power of two up to 32
};

// The rows' log sums from their segments' parts, and their losses. A block takes
// `per` rows, 256 / per threads a row share its segments; parts are joined in a fixed
// order.
__global__ void __launch_bounds__(256) ce_rows(const CeRows q) {
  __shared__ float2 part[256];
  griddep_launch_dependents();
  griddep_wait();
  const int r = threadIdx.x & (q.per - 1), y = threadIdx.x / q.per, ny = 256 / q.per;
  const int row = blockIdx.x * q.per + r;
  float c = -INFINITY, s = 0.f;
  if (row < q.rows) {
    const float2* p = q.partial + row;
    int i = y;
    for (; i + 3 * ny < q.segments; i += 4 * ny) {
      float2 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __ldg(p + static_cast<int64_t>(i + j * ny) * q.rows);
#pragma unroll
      for (int j = 0; j < 4; ++j) ce_join(c, s, v[j].x, v[j].y);
    }
    for (; i < q.segments; i += ny) {
      const float2 v = __ldg(p + static_cast<int64_t>(i) * q.rows);
      ce_join(c, s, v.x, v.y);
    }
  }
  part[threadIdx.x] = make_float2(c, s);
  __syncthreads();
  for (int step = ny / 2; step > 0; step >>= 1) {
    if (y < step) {
      const float2 o = part[threadIdx.x + step * q.per];
      float2 mine = part[threadIdx.x];
      ce_join(mine.x, mine.y, o.x, o.y);
      part[threadIdx.x] = mine;
    }
    __syncthreads();
  }
  if (y != 0 || row >= q.rows) return;
  constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;
  const float2 v = part[threadIdx.x];
  const float log2s = log2f(v.y), lse2 = v.x + log2s, lse = lse2 * kLn2;
  const int t = ce_target(q.targets, q.target_stride, q.target64, q.ignore, q.vocab, row);
  float loss = 0.f;
  if (t >= 0) {
    // The maximum and the target's z are subtracted before the sum's logarithm is added: the
    // log sum is rounded at the logits' size (by 10^-5 at 400), the loss of a row that is sure of its
    // target is far below that. It is never negative, which the rounding of s may make it.
    loss = kLn2 * (fmaf(-q.picked[row], kLog2e, v.x) + log2s);
    if (loss < 0.f) loss = 0.f;
    if (q.z_loss != 0.f) loss = fmaf(q.z_loss * lse, lse, loss);
  } else if (t == -2) {
    loss = __int_as_float(0x7fc00000);
  }
  q.each[row] = loss;
  if (q.lse) q.lse[row] = lse2;
  if (q.low) {
    const float added = lse2 - v.x;
    q.low[row] = (v.x - (lse2 - added)) + (log2s - added);
  }
}

// The sum or mean of the rows' losses, in 64 bits and a fixed order; *count: the
// rows that are not ignored.
__global__ void __launch_bounds__(1024) ce_total(const CeRows q, int mean, float* loss, float* count) {
  __shared__ double sums[32];
  __shared__ int counts[32];
  griddep_launch_dependents();
  griddep_wait();
  double s = 0.0;
  int n = 0;
  for (int i = threadIdx.x; i < q.rows; i += 1024) {
    s += static_cast<double>(q.each[i]);
    n += ce_target(q.targets, q.target_stride, q.target64, q.ignore, q.vocab, i) != -1;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
    n += __shfl_xor_sync(0xFFFFFFFFu, n, d);
  }
  if ((threadIdx.x & 31) == 0) {
    sums[threadIdx.x >> 5] = s;
    counts[threadIdx.x >> 5] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    n = 0;
    for (int i = 0; i < 32; ++i) {
      s += sums[i];
      n += counts[i];
    }
    *loss = static_cast<float>(mean ? s / n : s);  // the mean of no row is 0 / 0
    if (count) *count = __int_as_float(n);
  }
}

struct CeCoef {
  int rows, vocab, width;
  const void* targets;
  int64_t target_stride;
  int target64;
  int64_t ignore;
  const float* lse;
  const float* low;        // the log sums' low parts, or null
  const float* count;      // mean: the bits of the number of rows, else null
  const float* dy;
  int64_t dy_stride;       // 0: one value
  float z_loss;
  float2* coef;
  uint32_t* largest;       // bits of the largest |b| and |a|, zero before
  const uint16_t* x;
  int64_t x_ld;
  uint16_t* copy;          // rows of ignored targets that are not finite, as zeros
  int64_t copy_ld;
  uint8_t* dirty;          // [ceil(rows / 64)], or null: dW is not wanted
};

constexpr int kCeCoefRows = kLnBK;

// a and b of 64 rows. dW multiplies every row of x by its dz, which is zero for
// an ignored row, but padding may hold infinities and NaN: a block of 64 rows
// with such a row is copied with those rows as zeros, and dW reads the copy there.
template <typename T>
__global__ void __launch_bounds__(256) ce_coef(const CeCoef q) {
  __shared__ uint8_t skip[kCeCoefRows];
  griddep_launch_dependents();
  griddep_wait();
  constexpr float kLn2 = 0.6931471805599453f;
  const int row0 = blockIdx.x * kCeCoefRows, tid = threadIdx.x, row = row0 + tid;
  const int here = min(kCeCoefRows, q.rows - row0);
  if (tid < kCeCoefRows) {
    float a = 0.f, b = 0.f;
    bool out = true;
    if (tid < here) {
      const int t = ce_target(q.targets, q.target_stride, q.target64, q.ignore, q.vocab, row);
      out = t == -1;
      if (!out) {
        float g = __ldg(q.dy + row * q.dy_stride);
        if (q.count) g /= static_cast<float>(__float_as_int(*q.count));
        if (t == -2) g = __int_as_float(0x7fc00000);
        b = g;
        a = q.z_loss != 0.f ? g * fmaf(2.f * q.z_loss, __ldg(q.lse + row) * kLn2, 1.f) : g;
        // The powers are relative to the rounded log sum, which is off by 10^-5 at logits of 400: a
        // row that is sure of its target has a gradient p - 1 far below that.
        if (q.low) a *= exp2f(-__ldg(q.low + row));
      }
      q.coef[row] = make_float2(a, b);
    }
    skip[tid] = out;
    // The largest finite ones; the order of the maxima does not matter.
    const float top_b = fabsf(b) < INFINITY ? fabsf(b) : 0.f, top_a = fabsf(a) < INFINITY ? fabsf(a) : 0.f;
    const uint32_t all_b = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top_b));
    const uint32_t all_a = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top_a));
    if ((tid & 31) == 0) {
      if (all_b) atomicMax(q.largest, all_b);
      if (all_a) atomicMax(q.largest + 1, all_a);
    }
  }
  if (!q.dirty) return;
  __syncthreads();
  // Rows of x are whole 16-byte units here; a warp looks at a row.
  constexpr uint32_t kTop = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  const int lane = tid & 31;
  bool bad = false;
#pragma unroll 4
  for (int i = tid >> 5; i < kCeCoefRows; i += 8) {
    if (!skip[i] || i >= here) continue;
    const uint16_t* p = q.x + static_cast<int64_t>(row0 + i) * q.x_ld;
    for (int j = lane * 8; j < q.width; j += 256) {
      const uint4 v = ln_load8(p + j, q.width - j, true);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) bad |= (w[k] & kTop) == kTop || (w[k] >> 16 & kTop) == kTop;
    }
  }
  bad = __syncthreads_or(bad);
  if (tid == 0) q.dirty[blockIdx.x] = bad;
  if (!bad) return;
  for (int i = 0; i < here; ++i) {
    const uint16_t* p = q.x + static_cast<int64_t>(row0 + i) * q.x_ld;
    uint16_t* o = q.copy + static_cast<int64_t>(row0 + i) * q.copy_ld;
    for (int j = tid; j < q.width; j += 256) o[j] = skip[i] ? static_cast<uint16_t>(0) : p[j];
  }
}

struct CeParts {
  const float* parts;      // [splits][tiles][256][bn]
  int m, n, bn, n_nt, tiles, splits;
  const uint32_t* largest;
  void* out;               // 16 bits, or fp32 sums to add to (`add`) or to set
  int64_t out_ld;
  int add;
};

// The sums of dX's tiles whose K blocks were shared, in the order of the blocks. A
// block takes 16 rows of a tile.
constexpr int kCeJoinRows = 16;
template <typename T, bool F32>
__global__ void __launch_bounds__(256) ce_join_parts(const CeParts q) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int kBlocks = kCeBM / kCeJoinRows;
  const int t = blockIdx.x / kBlocks, r0 = blockIdx.x % kBlocks * kCeJoinRows;
  const int mt = t / q.n_nt, nt = t - mt * q.n_nt;
  const float scale = F32 ? 1.f : ce_scale(q.largest).undo;
  const int per = q.bn / 4;
  for (int j = threadIdx.x; j < kCeJoinRows * per; j += 256) {
    const int r = r0 + j / per, c = j % per * 4;
    const int row = mt * kCeBM + r, col = nt * q.bn + c;
    if (row >= q.m || col >= q.n) continue;
    const float* p = q.parts + (static_cast<int64_t>(t) * kCeBM + r) * q.bn + c;
    const int64_t plane = static_cast<int64_t>(q.tiles) * kCeBM * q.bn;
    float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < q.splits; ++k) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(p + k * plane));
      z.x += v.x;
      z.y += v.y;
      z.z += v.z;
      z.w += v.w;
    }
    if constexpr (F32) {  // rows of whole 16 bytes
      float4* o = reinterpret_cast<float4*>(static_cast<float*>(q.out) + row * q.out_ld + col);
      if (q.add) {
        const float4 v = *o;
        z = make_float4(z.x + v.x, z.y + v.y, z.z + v.z, z.w + v.w);
      }
      *o = z;
    } else {
      const float f[4] = {z.x * scale, z.y * scale, z.z * scale, z.w * scale};
      T* o = static_cast<T*>(q.out) + row * q.out_ld + col;
      if (col + 4 <= q.n && (reinterpret_cast<uintptr_t>(o) & 7u) == 0) {
        *reinterpret_cast<uint2*>(o) = make_uint2(ln_pack<T>(f[0], f[1]), ln_pack<T>(f[2], f[3]));
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (col + k < q.n) o[k] = Elem<T>::from_f(f[k]);
      }
    }
  }
}

// dx from its fp32 sums over all pieces.
template <typename T>
__global__ void __launch_bounds__(256) ce_finish(const float* sums, int64_t ld, int rows, int width,
                                                 const uint32_t* largest, T* dx, int64_t dx_ld) {
  griddep_wait();
  const float scale = ce_scale(largest).undo;
  const int64_t per = ld / 4, total = rows * per;
  const bool vec = width % 4 == 0 && dx_ld % 4 == 0 && (reinterpret_cast<uintptr_t>(dx) & 7u) == 0;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / per;
    const int col = static_cast<int>(i - row * per) * 4;
    const float4 v = __ldcs(reinterpret_cast<const float4*>(sums + row * ld + col));
    T* o = dx + row * dx_ld + col;
    if (vec) {
      *reinterpret_cast<uint2*>(o) = make_uint2(ln_pack<T>(v.x * scale, v.y * scale), ln_pack<T>(v.z * scale, v.w * scale));
    } else {
      const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < width) o[j] = Elem<T>::from_f(f[j] * scale);
    }
  }
}

}  // namespace avey
