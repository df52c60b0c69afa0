// Linear layers on tcgen05, dense or grouped by expert (avey_linear_*):
//
//   forward   y  = act(x W_g^T + b_g) + r    (and a 16-bit code of act')
//   dX        dx = dpre W_g
//   dW        dW_g = dpre_g^T x_g            (fp32 partial sums when split over rows)
//
// where group g owns the rows [offsets[g], offsets[g + 1]) of x; a dense layer
// is one group of all rows. The groups' sizes are known on the device only:
// every role of the kernel walks the offsets itself, so nothing is read back to
// the host, and rows past the last group give zeros.
//
// Bounds: 2 M N K flops on the tensor cores against reading x, W, r and
// writing y once. Tiles are 128 rows x 256 columns (128 or 64 where 256 would
// leave SMs without a tile), K in blocks of 64 through a TMA ring (128-byte
// swizzle). Persistent CTAs, one per SM: warp 0 issues TMA, warp 1 issues
// tcgen05.mma into one of two TMEM accumulators, warps 4-19 drain the other one,
// so a tile's epilogue overlaps the next tile's products; warp 2 clears the
// rows of a neighbouring group out of dW's last K block. Every wait is bounded.
//
// The epilogue has as long as the products take: at d_in = 768 6144 cycles for
// 32768 elements, 24 issue slots each. silu and gelu take two special-function
// results each (4096 cycles a tile), so they are computed on pairs (packed
// fp32), with the code of act' by a magic-number sum, and sixteen warps cover one
// another's latencies: with eight warps and scalar sums the forward pass of
// 32768 x 768 x 1536 with silu, residual and codes took 185 us.
//
// Measured (bf16, one B200): 32768 x 768 x 1536 forward with bias and any
// activation 70-74 us (1,050-1,110 TFLOP/s; torch.matmul 62-64), with residual 88,
// for training with residual and codes 99-101 (350 MB moved, 3.5 TB/s); dX 66,
// dW 67-69 (77 with the set-up beside dX's end) and 4 for its partial sums; 8192 x 4096 x 4096 forward 183-191
// (1,440-1,500 TFLOP/s; torch.matmul 179-207). Tiles of 128 columns instead of 256:
// dX 89, dW 102 us, so what an SM takes in and reads back from shared memory for
// its products is the bound of the bare product.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"

namespace avey {

constexpr int kLnEpiWarps = 16;
constexpr int kLnThreads = 128 + 32 * kLnEpiWarps;
constexpr int kLnBM = 128, kLnBK = 64;
constexpr int kLnABytes = kLnBM * kLnBK * 2;  // 16 KB
constexpr int kLnMnBox = 64 * kLnBK * 2;      // one {64 (m or n), 64 (k)} box: 8 KB
constexpr int kLnStageTile = 2048;            // an epilogue warp's staging: 32 x 32 16-bit (or 32 x 16 32-bit) values
constexpr int kLnMaxStages = 8;
constexpr int kLnRowBlock = 12;  // row tiles of a block of tiles taken rows first,
constexpr int kLnMaxRow = 16;    // which starts above so many column tiles
constexpr int kLnCtrlBytes = 512;
constexpr int kLnRing = 196608;  // bytes of the TMA ring: 4, 6 or 8 stages by tile width
constexpr int kLnBiasBytes = 64;  // an epilogue warp's 32 bias values
constexpr int kLnSmem = 1024 + kLnRing + kLnEpiWarps * (kLnStageTile + kLnBiasBytes) + kLnCtrlBytes;

enum LnMode { kLnForward = 0, kLnGradX = 1, kLnGradW = 2 };

struct LnGeom {
  int groups;              // >= 1
  const int32_t* offsets;  // [groups + 1], or null: one group of all rows
  int rows;                // rows of x
  int n;                   // output columns
  int kc;                  // contraction length (forward, dX)
  int bn;                  // columns per tile
  int n_nt;                // column tiles
  int m, n_mt, splits;     // dW: output rows, row tiles, K ranges per group
  int stages, stage_bytes;
  void* out;               // y, dx or dW (T), or dW's partial sums (float)
  int64_t out_ld, out_gs;  // dW: group (and split) stride
  int out_vec;             // rows of `out` are 16-byte aligned: whole tiles go by TMA
  const void* bias;        // [groups][n], or null
  int64_t bias_gs;
  const void* res;         // residual rows, or null
  int64_t res_ld;
  int res_vec;
  uint16_t* deriv;         // codes of act' [rows][deriv_ld], or null
  int64_t deriv_ld;        // a multiple of 16
  const float* bias_sums;  // dX: partial sums of the bias gradient [tiles][kc], or null
  void* db;                // its [groups][kc]
  int lets_next;           // dX: dW is launched as its dependent
  int test_stall;          // tests: the TMA lane asks for nothing
};

// ---------------------------------------------------------------- activations

__device__ __forceinline__ float ln_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float ln_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 values in one 64-bit register.
typedef unsigned long long LnPair;
__device__ __forceinline__ LnPair ln_pair(float lo, float hi) {
  LnPair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ LnPair ln_pair(float x) { return ln_pair(x, x); }
__device__ __forceinline__ float2 ln_split(LnPair p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ LnPair ln_add2(LnPair a, LnPair b) {
  LnPair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ LnPair ln_mul2(LnPair a, LnPair b) {
  LnPair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ LnPair ln_fma2(LnPair a, LnPair b, LnPair c) {
  LnPair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// 1 / (1 + 2^t) by the hardware's base-2 exponential and reciprocal (about
// 2^-22 relative: far below a 16-bit result's rounding).
__device__ __forceinline__ float ln_sigmoid(float t) { return ln_rcp(__fadd_rn(1.f, ln_exp2(t))); }

// act(x) of a pair and, with D, its derivative. Operations between values are
// packed; those with a constant are scalar, where it is an immediate (a packed
// one takes two moves each time: 24 against 15 instructions an element).
template <int ACT, bool D>
__device__ __forceinline__ LnPair ln_act2(LnPair x, LnPair* d) {
  constexpr float kLog2e = 1.4426950408889634f;
  const float2 v = ln_split(x);
  if constexpr (ACT == 1) {
    if (D)
      *d = ln_pair(v.x > 0.f ? 1.f : (v.x <= 0.f ? 0.f : v.x), v.y > 0.f ? 1.f : (v.y <= 0.f ? 0.f : v.y));
    return ln_pair(v.x < 0.f ? 0.f : v.x, v.y < 0.f ? 0.f : v.y);
  } else if constexpr (ACT == 2) {
    const LnPair r = ln_pair(v.x < 0.f ? 0.f : v.x, v.y < 0.f ? 0.f : v.y);
    if (D) *d = ln_add2(r, r);
    return ln_mul2(r, r);
  } else if constexpr (ACT == 3) {
    const float s0 = ln_sigmoid(__fmul_rn(v.x, -kLog2e)), s1 = ln_sigmoid(__fmul_rn(v.y, -kLog2e));
    const LnPair s = ln_pair(s0, s1);
    const LnPair y = ln_mul2(x, s);
    if (D) *d = ln_fma2(y, ln_pair(__fsub_rn(1.f, s0), __fsub_rn(1.f, s1)), s);
    return y;
  } else if constexpr (ACT == 4) {
    // x sigmoid(2 t), t = sqrt(2 / pi) (x + 0.044715 x^3); x^2 is capped where
    // the sigmoid has long been 0 or 1, so that no infinity meets a zero.
    constexpr float c0 = 1.5957691216057308f, c1 = 0.07135481282754853f;
    const float2 q = ln_split(ln_mul2(x, x));
    const float u0 = fminf(q.x, 1e4f), u1 = fminf(q.y, 1e4f);
    const float2 t = ln_split(
        ln_mul2(x, ln_pair(fmaf(u0, -kLog2e * c1, -kLog2e * c0), fmaf(u1, -kLog2e * c1, -kLog2e * c0))));
    const float s0 = ln_sigmoid(t.x), s1 = ln_sigmoid(t.y);
    const LnPair s = ln_pair(s0, s1);
    const LnPair y = ln_mul2(x, s);
    if (D)
      *d = ln_fma2(ln_mul2(y, ln_pair(__fsub_rn(1.f, s0), __fsub_rn(1.f, s1))),
                   ln_pair(fmaf(u0, 3.f * c1, c0), fmaf(u1, 3.f * c1, c0)), s);
    return y;
  } else {
    if (D) *d = ln_pair(1.f);
    return x;
  }
}

// 16-bit codes of act' kept for the backward pass. relu, silu and gelu have
// derivatives in (-0.2, 1.2): fixed point in steps of 2^-14 from -1/4, which moves
// dpre by at most 2^-15 |dy|. That is an eighth of an f16 rounding where the
// derivative is near 1 (the pre-activation in 16 bits would add one or more of the
// operand type's own), and more of a small one: one below 2^-15, of a unit far on
// its flat side, becomes 0. relu2's (2 relu(x)) is unbounded and
// not negative: the fp32 bit pattern in equal steps from a base, which spreads
// 2^16 codes over 128 binades for bf16 (2^-62 .. 2^66, half steps of 2^-10) and
// over 25 for f16 (2^-15 .. 2^10, half steps of 2^-12.3); zero below. Both hold
// the derivative of every finite y: bf16's square leaves fp32's range at 2^64; f16's
// y is the square and a residual of -65504 at the least, rounded together, so
// the pre-activation stays below 362. The code 0xFFFF stands for a derivative that is
// not finite or out of range (a NaN gives it by itself in the fixed-point form).
template <typename T>
struct LnFloatCode {
  static constexpr uint32_t kBinades = std::is_same<T, __half>::value ? 25 : 128;
  static constexpr uint32_t kStep = kBinades * 128;  // 2^23 bit patterns a binade / 2^16 codes
  static constexpr uint32_t kBase = (std::is_same<T, __half>::value ? 112u : 65u) << 23;
};
template <typename T>
__device__ __forceinline__ uint32_t ln_float_code(float d) {
  using C = LnFloatCode<T>;
  if (!(d >= __uint_as_float(C::kBase + C::kStep))) return d >= 0.f ? 0u : 0xFFFFu;
  const uint32_t c = (__float_as_uint(d) - C::kBase + C::kStep / 2) / C::kStep;
  return c < 0xFFFFu ? c : 0xFFFFu;
}
// The codes of a pair, the first in the low half.
template <typename T, int ACT>
__device__ __forceinline__ uint32_t ln_encode2(LnPair d) {
  if constexpr (ACT == 2) {
    const float2 v = ln_split(d);
    return ln_float_code<T>(v.x) | (ln_float_code<T>(v.y) << 16);
  } else {
    // 2^23 + 2^22 + 2^12 + 2^14 d: the code is in the low 16 bits.
    const float2 v = ln_split(d);
    return __byte_perm(__float_as_uint(fmaf(v.x, 0x1p14f, 0x1.8p23f + 0x1p12f)),
                       __float_as_uint(fmaf(v.y, 0x1p14f, 0x1.8p23f + 0x1p12f)), 0x5410);
  }
}
template <typename T, int ACT>
__device__ __forceinline__ float ln_decode(uint32_t c) {
  if constexpr (ACT == 2) {
    using C = LnFloatCode<T>;
    if (c == 0xFFFFu) return __int_as_float(0x7f800000);
    return c ? __uint_as_float(c * C::kStep + C::kBase) : 0.f;
  } else {
    // (2^23 + c) 2^-14 - 2^9 - 1/4, exactly.
    const float d = fmaf(__uint_as_float(0x4B000000u | c), 0x1p-14f, -512.25f);
    return c == 0xFFFFu ? __int_as_float(0x7fc00000) : d;
  }
}

// ---------------------------------------------------------------- 16-bit pairs
template <typename T>
__device__ __forceinline__ uint32_t ln_pack(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ float2 ln_unpack(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  } else {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  }
}

__device__ __forceinline__ void ln_sts(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint4 ln_lds(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}

// ---------------------------------------------------------------- groups

struct LnTile {
  int g;           // group (== groups: rows past the last group, zeros)
  int lo, hi;      // its rows
  int mt, nt;      // row and column tile
  int row0;        // forward, dX: first row
  int split;       // dW
  int k0, nk;      // dW: first row of the K range; all: K blocks
  int last;        // dW: rows in the last K block (kLnBK: whole, or past the tensor's end)
};

// ---------------------------------------------------------------- groups, by a warp

struct LnSpan {
  int g, lo, hi;  // group and its rows
  int index;      // which of the group's tiles
  int base, cnt;  // the group's first tile and its tiles
};

// Every lane of the warp: walk the groups 32 at a time, a group counting
// count(lo, hi) items, and find the group that holds item t (t >= 0), or the
// items of group `want` (t < 0). False when there is none.
template <typename Count>
__device__ __forceinline__ bool ln_find(const int32_t* offsets, int groups, int rows, int t, int want, Count count,
                                        LnSpan& out) {
  const int lane = threadIdx.x & 31;
  int end_carry = 0, base = 0;
  for (int g0 = 0; g0 < groups; g0 += 32) {
    const int g = g0 + lane;
    int hi = g < groups ? (offsets ? min(max(__ldg(offsets + g + 1), 0), rows) : rows) : 0;
    hi = max(hi, end_carry);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xFFFFFFFFu, hi, d);
      if (lane >= d) hi = max(hi, o);
    }
    int lo = __shfl_up_sync(0xFFFFFFFFu, hi, 1);
    if (lane == 0) lo = end_carry;
    const int cnt = g < groups ? count(lo, hi) : 0;
    int incl = cnt;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xFFFFFFFFu, incl, d);
      if (lane >= d) incl += o;
    }
    const int excl = base + incl - cnt;
    const bool mine = t >= 0 ? (t >= excl && t < excl + cnt) : g == want;
    const unsigned hit = __ballot_sync(0xFFFFFFFFu, mine);
    if (hit) {
      const int src = __ffs(hit) - 1;
      out.g = g0 + src;
      out.lo = __shfl_sync(0xFFFFFFFFu, lo, src);
      out.hi = __shfl_sync(0xFFFFFFFFu, hi, src);
      out.base = __shfl_sync(0xFFFFFFFFu, excl, src);
      out.cnt = __shfl_sync(0xFFFFFFFFu, cnt, src);
      out.index = t - out.base;
      return true;
    }
    end_carry = __shfl_sync(0xFFFFFFFFu, hi, 31);
    base += __shfl_sync(0xFFFFFFFFu, incl, 31);
  }
  // Not found: the rows past the last group, and the items in all.
  out.g = groups;
  out.lo = end_carry;
  out.hi = rows;
  out.base = base;
  out.cnt = 0;
  out.index = t - base;
  return false;
}

// Row tiles of ln_dpre, which writes the bias gradient's partial sums by them.
constexpr int kLdRows = 64;
__device__ __forceinline__ int ln_dpre_tiles(int lo, int hi) { return (hi - lo + kLdRows - 1) / kLdRows; }

// db[g] for 32 columns from c0 by one warp: the sum of the group's partial rows in
// a fixed order (part i of 32 takes every 32nd row, then the parts in turn).
template <typename T>
__device__ __forceinline__ void ln_bias_columns(const int32_t* offsets, int groups, int rows, int n,
                                                const float* partial, T* db, int g, int c0) {
  LnSpan s;
  ln_find(offsets, groups, rows, -1, g, ln_dpre_tiles, s);
  const int c = c0 + (threadIdx.x & 31);
  if (c >= n) return;
  float part[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) part[j] = 0.f;
  const float* p = partial + static_cast<int64_t>(s.base) * n + c;
  for (int i = 0; i < s.cnt; i += 32) {
    float v[32];  // all on their way before the first sum: 1024 partial rows take 45 us instead of 85
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = i + j < s.cnt ? __ldcg(p + static_cast<int64_t>(i + j) * n) : 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) part[j] += v[j];
  }
  float z = 0.f;
#pragma unroll
  for (int j = 0; j < 32; ++j) z += part[j];
  db[static_cast<int64_t>(g) * n + c] = Elem<T>::from_f(z);
}

// Tiles of a group of the rows [lo, hi).
template <int MODE>
__device__ __forceinline__ int ln_tiles(const LnGeom& q, int lo, int hi) {
  return MODE == kLnGradW ? q.n_mt * q.n_nt * q.splits : (hi - lo + kLnBM - 1) / kLnBM * q.n_nt;
}

// Tile r of group g.
template <int MODE>
__device__ __forceinline__ void ln_set_tile(const LnGeom& q, LnTile& c, int g, int lo, int hi, int r) {
  c.g = g;
  c.lo = lo;
  c.hi = hi;
  if (MODE == kLnGradW) {
    c.split = r % q.splits;
    r /= q.splits;
    c.nt = r % q.n_nt;
    c.mt = r / q.n_nt;
    c.row0 = c.mt * kLnBM;
    const int blocks = (hi - lo + kLnBK - 1) / kLnBK;
    const int b0 = static_cast<int>(static_cast<int64_t>(blocks) * c.split / q.splits);
    const int b1 = static_cast<int>(static_cast<int64_t>(blocks) * (c.split + 1) / q.splits);
    c.k0 = lo + b0 * kLnBK;
    c.nk = b1 - b0;
    const int stop = c.k0 + c.nk * kLnBK;
    c.last = c.nk > 0 && stop > hi && hi < q.rows ? hi - (stop - kLnBK) : kLnBK;
  } else {
    // Column tiles first, so that the CTAs at work share rows of x; with more than 16
    // of them, blocks of 12 row tiles by all columns, rows first: for each k a wave of
    // 148 tiles then fetches 12 * 128 + 13 * 256 values from L2 instead of n_nt * 256
    // and more (8192^3: 982 -> 881-917 us; 8192 x 1536 -> 8192: 191 -> 179 us; 16
    // column tiles, 8192 x 4096 -> 4096: 203-206 us as they are, 208-216 in blocks).
    if (q.n_nt <= kLnMaxRow) {
      c.nt = r % q.n_nt;
      c.mt = r / q.n_nt;
    } else {
      const int mt = (hi - lo + kLnBM - 1) / kLnBM, block = r / (kLnRowBlock * q.n_nt);
      const int high = min(kLnRowBlock, mt - block * kLnRowBlock), k = r - block * kLnRowBlock * q.n_nt;
      c.nt = k / high;
      c.mt = block * kLnRowBlock + k - c.nt * high;
    }
    c.row0 = lo + c.mt * kLnBM;
    c.split = 0;
    c.k0 = 0;
    c.nk = g < q.groups ? (q.kc + kLnBK - 1) / kLnBK : 0;
    c.last = kLnBK;
  }
}

// Walks the groups' tiles in order (t must not decrease); every lane of a warp
// takes part. 32 groups are looked at together: a lane holds the rows and the
// tiles of one, from a running maximum of their ends (offsets out of order or
// out of range are pulled into [the group's start, rows], so no value of theirs
// leads out of the tensors) and a running sum of their tile counts. (One lane
// walking alone took 60 cycles a group: 20.6 us in all for 16 rows of 64
// experts, against 17.4 us.)
template <int MODE>
struct LnWalker {
  int g0 = -32, end = 0;     // first group of the window, and the end of the groups before it
  int base = 0, total = 0;   // tiles before the window, and in it
  int lo = 0, hi = 0, first = 0, cnt = 0;  // the lane's group: rows, first tile, tiles

  __device__ __forceinline__ bool seek(const LnGeom& q, int t, LnTile& c) {
    const int lane = threadIdx.x & 31;
    const int groups = MODE == kLnGradW ? q.groups : q.groups + 1;  // with the rows past the last group
    while (t >= base + total) {
      if (g0 + 32 >= groups) return false;
      g0 += 32;
      base += total;
      const int g = g0 + lane;
      hi = g < q.groups ? min(max(__ldg(q.offsets + g + 1), 0), q.rows) : (g < groups ? q.rows : 0);
      hi = max(hi, end);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xFFFFFFFFu, hi, d);
        if (lane >= d) hi = max(hi, o);
      }
      lo = __shfl_up_sync(0xFFFFFFFFu, hi, 1);
      if (lane == 0) lo = end;
      cnt = g < groups ? ln_tiles<MODE>(q, lo, hi) : 0;
      first = cnt;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xFFFFFFFFu, first, d);
        if (lane >= d) first += o;
      }
      total = __shfl_sync(0xFFFFFFFFu, first, 31);
      end = __shfl_sync(0xFFFFFFFFu, hi, 31);
      first += base - cnt;
    }
    const int src = __ffs(__ballot_sync(0xFFFFFFFFu, t >= first && t < first + cnt)) - 1;
    ln_set_tile<MODE>(q, c, g0 + src, __shfl_sync(0xFFFFFFFFu, lo, src), __shfl_sync(0xFFFFFFFFu, hi, src),
                      t - __shfl_sync(0xFFFFFFFFu, first, src));
    return true;
  }
};

constexpr int kLnAhead = 4;  // tiles that the scheduler may be ahead

struct LnCtrl {
  uint64_t full[kLnMaxStages], empty[kLnMaxStages];
  uint64_t sched_full[kLnAhead], sched_empty[kLnAhead];
  LnTile sched[kLnAhead];  // grouped layers: the CTA's next tiles (g < 0: none)
  uint64_t acc_full[2], acc_empty[2];
  uint64_t partial;  // dW: a last K block with rows of the next group has landed
  uint64_t cleared;  // dW: warp 2 has cleared them
  uint64_t settled;  // after a wait has given up: the products have ended
  uint32_t failed;   // a wait of this CTA has given up
  uint32_t tmem_base;
};
static_assert(sizeof(LnCtrl) <= kLnCtrlBytes, "control block too large");

// The i-th tile of this CTA (false: there is none, or a wait gave up): computed
// on the spot for a dense layer; for a grouped one warp 3 walks the groups and
// hands the tiles over in shared memory, so that the roles with one lane at
// work need no warp-wide step between their tiles.
template <int MODE>
__device__ __forceinline__ bool ln_tile(const LnGeom& q, LnCtrl* ctrl, int i, LnTile& c) {
  if (!q.offsets) {
    const int t = blockIdx.x + i * gridDim.x;
    if (t >= ln_tiles<MODE>(q, 0, q.rows)) return false;
    ln_set_tile<MODE>(q, c, 0, 0, q.rows, t);
    return true;
  }
  const int slot = i % kLnAhead;
  if (!mbar_wait(smem_u32(&ctrl->sched_full[slot]), (i / kLnAhead) & 1)) return false;
  c = ctrl->sched[slot];
  return c.g >= 0;
}
// After ln_tile, by one lane of each role: the slot may be filled again.
__device__ __forceinline__ void ln_tile_taken(const LnGeom& q, LnCtrl* ctrl, int i) {
  if (q.offsets) mbar_arrive(smem_u32(&ctrl->sched_empty[i % kLnAhead]));
}
// The same for a whole warp.
template <int MODE>
__device__ __forceinline__ bool ln_warp_tile(const LnGeom& q, LnCtrl* ctrl, int i, LnTile& c) {
  const bool ok = __all_sync(0xFFFFFFFFu, ln_tile<MODE>(q, ctrl, i, c));
  __syncwarp();  // every lane has read the slot
  if (ok && (threadIdx.x & 31) == 0) ln_tile_taken(q, ctrl, i);
  return ok;
}

// A wait by every lane of a warp: they go on, or give up, together.
__device__ __forceinline__ bool ln_warp_wait(uint32_t bar, uint32_t parity) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity));
}

// Once a wait has given up: what is still under way, the products issued so far
// and the TMA loads of the last `fills` K blocks, gets about a millisecond each to
// end before the CTA's tensor memory and shared memory go.
__device__ __forceinline__ void ln_settle(uint32_t bar, uint32_t parity) {
  const long long start = clock64();
  while (!mbar_try_wait(bar, parity) && clock64() - start < (1ll << 21)) {
  }
}
__device__ __forceinline__ void ln_settle_loads(const uint64_t* full, int stages, int fills) {
  for (int f = max(0, fills - stages); f < fills; ++f)
    ln_settle(smem_u32(full + f % stages), static_cast<uint32_t>(f / stages) & 1u);
}

// ---------------------------------------------------------------- epilogue

// A staging tile holds 32 rows of 64 bytes; 16-byte piece p of row r sits at
// piece p ^ (r / 2 mod 4), so rows (lane = row) and whole lines (4 lanes per
// row) are both read and written without bank conflicts.
__device__ __forceinline__ uint32_t ln_piece(uint32_t tile, int r, int p) {
  return tile + r * 64 + ((p ^ ((r >> 1) & 3)) << 4);
}

// Where a lane moves a tile's lines: rows row + 8 i, columns col..col + 7.
struct LnLines {
  int row, row_end, col, n;
  __device__ __forceinline__ bool in(int i) const { return row + 8 * i < row_end; }
};

// Address of element (r, column k) of a staging tile.
__device__ __forceinline__ uint32_t ln_element(uint32_t tile, int r, int k) {
  return ln_piece(tile, r, k >> 3) + 2 * (k & 7);
}

// Store a staged tile row by row, a lane to a column: rows that are not whole
// 16-byte units, and the last columns.
__device__ __forceinline__ void ln_store_tile_by_column(uint32_t tile, int lane, uint16_t* out, int64_t ld,
                                                        const LnLines& l) {
  const int row0 = l.row - (lane >> 2), col = l.col - (lane & 3) * 8 + lane;
  const int rows = min(32, l.row_end - row0);
  uint16_t* p = out + static_cast<int64_t>(row0) * ld + col;
  if (col < l.n) {
#pragma unroll 8
    for (int r = 0; r < rows; ++r) {
      uint16_t v;
      asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(ln_element(tile, r, lane)));
      p[r * ld] = v;
    }
  }
}

// Bring a tile into shared memory the same way (columns past the end: zeros).
__device__ __forceinline__ void ln_fetch_tile_by_column(uint32_t tile, int lane, const uint16_t* src, int64_t ld,
                                                        const LnLines& l) {
  const int row0 = l.row - (lane >> 2), col = l.col - (lane & 3) * 8 + lane;
  const int rows = min(32, l.row_end - row0);
  const uint16_t* p = src + static_cast<int64_t>(row0) * ld + col;
#pragma unroll 8
  for (int r = 0; r < rows; ++r) {
    const uint16_t v = col < l.n ? __ldg(p + r * ld) : static_cast<uint16_t>(0);
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(ln_element(tile, r, lane)), "h"(v) : "memory");
  }
}

// Store a staged 32 x 32 16-bit tile to `out`.
__device__ __forceinline__ void ln_store_tile(uint32_t tile, int lane, uint16_t* out, int64_t ld, const LnLines& l,
                                              bool vec) {
  // The decision is the warp's: lane 31 has the tile's last columns.
  if (vec && __shfl_sync(0xFFFFFFFFu, l.col, 31) + 8 <= l.n) {
    uint16_t* p = out + static_cast<int64_t>(l.row) * ld + l.col;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = ln_lds(ln_piece(tile, i * 8 + (lane >> 2), lane & 3));
      if (l.in(i)) *reinterpret_cast<uint4*>(p + 8 * i * ld) = v;
    }
  } else {
    ln_store_tile_by_column(tile, lane, out, ld, l);
  }
}

// Write a staged tile (32 rows of 64 bytes) at column x and row y of the
// mapped array (plane z) by TMA, which clips what is past its edges; the tile
// is free again once the store has read it. A store instruction per lane
// instead moves 8 half lines at a time through L1: 127 against 105 us for the
// forward pass with residual and codes at 32768 x 768 x 1536.
__device__ __forceinline__ void ln_tma_tile(uint32_t tile, int lane, const CUtensorMap* map, int x, int y, int z,
                                            uint64_t policy) {
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_3d(map, tile, x, y, z, policy);
    bulk_commit_group();
  }
}
// 32 bytes to 32-byte aligned global memory.
__device__ __forceinline__ void ln_st32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
// Before the staging tile is written again.
__device__ __forceinline__ void ln_tile_free(int lane) {
  if (lane == 0) bulk_wait_read_all();
  __syncwarp();
}

// 16 columns of this lane's accumulator row (zeros for an empty K range).
__device__ __forceinline__ void ln_tmem_ld16(uint32_t taddr, bool zero, uint32_t (&o)[16]) {
  if (zero) {
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = 0u;
    return;
  }
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]), "=r"(o[4]), "=r"(o[5]), "=r"(o[6]), "=r"(o[7]), "=r"(o[8]),
        "=r"(o[9]), "=r"(o[10]), "=r"(o[11]), "=r"(o[12]), "=r"(o[13]), "=r"(o[14]), "=r"(o[15])
      : "r"(taddr)
      : "memory");
}

// This lane's pieces of a 32 x 32 tile of 16-bit values in 16-byte aligned rows
// (outside: zeros; the last piece of a row may be cut).
__device__ __forceinline__ void ln_load_tile(const uint16_t* src, int64_t ld, const LnLines& l, uint4 (&v)[4]) {
  const uint16_t* p = src + static_cast<int64_t>(l.row) * ld + l.col;
  if (l.col + 8 <= l.n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (l.in(i)) v[i] = __ldg(reinterpret_cast<const uint4*>(p + 8 * i * ld));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (l.in(i) && l.col + j < l.n) w[j >> 1] |= static_cast<uint32_t>(__ldg(p + 8 * i * ld + j)) << (16 * (j & 1));
      v[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// What an epilogue warp reads ahead for a 32 x 32 chunk: its residual lines and
// the lane's bias value.
struct LnAhead {
  uint4 res[4];
  uint16_t bias;
};

// The columns of an epilogue warp in a tile, from its part h.
__device__ __forceinline__ int ln_part(const LnGeom& q) { return max(32, q.bn >> 2); }

template <int MODE>
__device__ __forceinline__ void ln_read_ahead(const LnGeom& q, const LnTile& c, int wq, int h, int ch, int lane,
                                              LnAhead& a) {
  if (MODE != kLnForward || c.g >= q.groups) return;
  const int col = c.nt * q.bn + h * ln_part(q) + ch * 32;
  if (q.res && q.res_vec) {
    const LnLines l{c.row0 + wq * 32 + (lane >> 2), c.hi, col + (lane & 3) * 8, q.n};
    ln_load_tile(static_cast<const uint16_t*>(q.res), q.res_ld, l, a.res);
  }
  a.bias = 0;
  if (q.bias && col + lane < q.n)
    a.bias = __ldg(static_cast<const uint16_t*>(q.bias) + static_cast<int64_t>(c.g) * q.bias_gs + col + lane);
}

// Drain this warp's 32 rows x max(32, bn / 4) columns of one accumulator and
// release it. FLAG: the forward pass writes act' as well, or dW writes partial
// sums. `a` holds the first chunk's residual and bias, and on return those of
// the next tile's (`next`, when there is one): the loads of a chunk are a whole
// chunk ahead of their use, across tiles too.
template <typename T, int MODE, int ACT, bool FLAG>
__device__ __forceinline__ bool ln_drain(const LnGeom& q, const CUtensorMap* map_y, uint64_t policy, const LnTile& c, const LnTile& next, bool has_next,
                                         uint32_t tb, int wq, int h, int lane, uint32_t tile, uint32_t bias_tile,
                                         uint32_t acc_full, uint32_t parity, uint32_t acc_empty, LnAhead& a) {
  constexpr bool F32 = MODE == kLnGradW && FLAG;
  constexpr bool DERIV = MODE == kLnForward && FLAG;
  const int row0 = c.row0 + wq * 32;
  const int row_end = MODE == kLnGradW ? q.m : c.hi;
  const int part = ln_part(q);
  const int col0 = c.nt * q.bn + h * part;
  const int nch = row0 < row_end && h * part < q.bn ? max(0, min(part, q.n - col0) + 31) / 32 : 0;
  const bool zero = c.nk == 0;
  const bool plain = MODE != kLnForward || c.g >= q.groups;  // no epilogue: the product (or zeros) itself
  const bool res = MODE == kLnForward && !plain && q.res;
  LnLines l{row0 + (lane >> 2), row_end, col0 + (lane & 3) * 8, q.n};
  // The maps end with the tensors: a tile that ends with its group inside the
  // tensor is stored by the lanes.
  const bool by_tma = q.out_vec && (MODE == kLnGradW || row0 + 32 <= row_end || row_end == q.rows);
  if (!ln_warp_wait(acc_full, parity)) return false;
  tc_fence_after();
  uint16_t* out16 = static_cast<uint16_t*>(q.out);
  if (MODE == kLnGradW) out16 += c.g * q.out_gs;
  if (nch == 0 && has_next) ln_read_ahead<MODE>(q, next, wq, h, 0, lane, a);
#pragma unroll 1
  for (int ch = 0; ch < nch; ++ch) {
    if constexpr (F32) {
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        uint32_t o[16];
        ln_tmem_ld16(tb + ch * 32 + 16 * hh, zero, o);
        ln_tile_free(lane);
#pragma unroll
        for (int p = 0; p < 4; ++p) ln_sts(ln_piece(tile, lane, p), o[4 * p], o[4 * p + 1], o[4 * p + 2], o[4 * p + 3]);
        ln_tma_tile(tile, lane, map_y, col0 + ch * 32 + 16 * hh, row0, c.split * q.groups + c.g, policy);
      }
    } else if (plain) {
      ln_tile_free(lane);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        uint32_t o[16];
        ln_tmem_ld16(tb + ch * 32 + 16 * hh, zero, o);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          uint32_t y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            y[j] = ln_pack<T>(__uint_as_float(o[8 * p + 2 * j]), __uint_as_float(o[8 * p + 2 * j + 1]));
          ln_sts(ln_piece(tile, lane, 2 * hh + p), y[0], y[1], y[2], y[3]);
        }
      }
      if (by_tma) {
        ln_tma_tile(tile, lane, map_y, col0 + ch * 32, row0, MODE == kLnGradW ? c.g : 0, policy);
      } else {
        __syncwarp();
        ln_store_tile(tile, lane, out16, q.out_ld, l, q.out_vec);
        __syncwarp();
      }
    } else {
      ln_tile_free(lane);
      // The residual's lines go through the staging tile to the lanes of their
      // rows, the bias to all lanes; the next chunk's are loaded meanwhile.
      if (res && q.res_vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          ln_sts(ln_piece(tile, i * 8 + (lane >> 2), lane & 3), a.res[i].x, a.res[i].y, a.res[i].z, a.res[i].w);
      } else if (res) {
        ln_fetch_tile_by_column(tile, lane, static_cast<const uint16_t*>(q.res), q.res_ld, l);
      }
      asm volatile("st.shared.b16 [%0], %1;" ::"r"(bias_tile + 2 * lane), "h"(a.bias) : "memory");
      __syncwarp();
      if (ch + 1 < nch) ln_read_ahead<MODE>(q, c, wq, h, ch + 1, lane, a);
      else if (has_next) ln_read_ahead<MODE>(q, next, wq, h, 0, lane, a);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        uint32_t o[16], dk[8];
        ln_tmem_ld16(tb + ch * 32 + 16 * hh, zero, o);
#pragma unroll
        for (int pp = 0; pp < 2; ++pp) {
          const int p = 2 * hh + pp;
          const uint4 bw = ln_lds(bias_tile + 16 * p);
          uint4 rw = make_uint4(0u, 0u, 0u, 0u);
          if (res) rw = ln_lds(ln_piece(tile, lane, p));
          const uint32_t b4[4] = {bw.x, bw.y, bw.z, bw.w}, r4[4] = {rw.x, rw.y, rw.z, rw.w};
          uint32_t y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = 8 * pp + 2 * j;
            const float2 bb = ln_unpack<T>(b4[j]);
            LnPair d;
            LnPair v = ln_act2<ACT, DERIV>(
                ln_add2(ln_pair(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), ln_pair(bb.x, bb.y)), &d);
            if (DERIV) dk[4 * pp + j] = ln_encode2<T, ACT>(d);
            if (res) {
              const float2 rr = ln_unpack<T>(r4[j]);
              v = ln_add2(v, ln_pair(rr.x, rr.y));
            }
            const float2 z = ln_split(v);
            y[j] = ln_pack<T>(z.x, z.y);
          }
          ln_sts(ln_piece(tile, lane, p), y[0], y[1], y[2], y[3]);
        }
        // The codes of 16 columns are one 32-byte sector of the lane's row.
        const int dcol = col0 + ch * 32 + 16 * hh;
        if (DERIV && row0 + lane < row_end && dcol < q.deriv_ld)
          ln_st32(q.deriv + static_cast<int64_t>(row0 + lane) * q.deriv_ld + dcol, dk);
      }
      if (by_tma) {
        ln_tma_tile(tile, lane, map_y, col0 + ch * 32, row0, 0, policy);
      } else {
        __syncwarp();
        ln_store_tile(tile, lane, out16, q.out_ld, l, q.out_vec);
        __syncwarp();
      }
    }
    l.col += 32;
  }
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(acc_empty);
  return true;
}

// ---------------------------------------------------------------- kernel

template <typename T, int MODE, int ACT, bool FLAG>
__global__ void __launch_bounds__(kLnThreads, 1)
    tc_linear(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
              const __grid_constant__ CUtensorMap map_y, const LnGeom q) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t staging = base + kLnRing;
  LnCtrl* ctrl =
      reinterpret_cast<LnCtrl*>(smem_raw + (base - raw) + kLnRing + kLnEpiWarps * (kLnStageTile + kLnBiasBytes));
  constexpr bool kAMn = MODE == kLnGradW, kBMn = MODE != kLnForward;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < q.stages; ++s) {
      mbar_init(smem_u32(&ctrl->full[s]), 1);
      mbar_init(smem_u32(&ctrl->empty[s]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctrl->acc_full[i]), 1);
      mbar_init(smem_u32(&ctrl->acc_empty[i]), kLnEpiWarps);
    }
    for (int i = 0; i < kLnAhead; ++i) {
      mbar_init(smem_u32(&ctrl->sched_full[i]), 1);
      // The TMA and MMA lanes and the epilogue warps, and warp 2 for dW.
      mbar_init(smem_u32(&ctrl->sched_empty[i]), 2 + kLnEpiWarps + (MODE == kLnGradW ? 1 : 0));
    }
    mbar_init(smem_u32(&ctrl->partial), 1);
    mbar_init(smem_u32(&ctrl->cleared), 1);
    mbar_init(smem_u32(&ctrl->settled), 1);
    ctrl->failed = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&ctrl->tmem_base), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctrl->tmem_base;
  int fills = 0;  // K blocks that the TMA lane has asked for

  if (warp == 0) {
    // ============================================================ TMA producer
    if (lane == 0) {
      const uint64_t keep = l2_policy_evict_last();  // operands are read again by other tiles
      // The CTA is set up beside the end of the step before (a copy of rows, dpre, dX),
      // and its operands are read after it. dW's too, though its operands are older
      // than dX: what an earlier grid has written is promised to a grid that waits for
      // the one before it, and to no other.
      griddep_wait();
      if (MODE == kLnGradX && q.lets_next) griddep_launch_dependents();
      LnTile c;
      int st = 0;
      uint32_t ph = 0;
      bool alive = !q.test_stall;
      for (int i = 0; alive && ln_tile<MODE>(q, ctrl, i, c); ++i) {
        ln_tile_taken(q, ctrl, i);
        for (int kk = 0; kk < c.nk; ++kk) {
          if (fills >= q.stages && !mbar_wait(smem_u32(&ctrl->empty[st]), ph ^ 1u)) {
            alive = false;
            break;
          }
          const uint32_t full = smem_u32(&ctrl->full[st]);
          const uint32_t sa = base + st * q.stage_bytes, sb = sa + kLnABytes;
          const int kx = c.k0 + kk * kLnBK;
          mbar_arrive_expect_tx(full, q.stage_bytes);
          if (!kAMn) {
            tma_load_3d_hint(sa, &map_a, full, kx, c.row0, 0, keep);
          } else {
            tma_load_3d_hint(sa, &map_a, full, c.row0, kx, 0, keep);
            tma_load_3d_hint(sa + kLnMnBox, &map_a, full, c.row0 + 64, kx, 0, keep);
          }
          if (!kBMn) {
            tma_load_3d_hint(sb, &map_b, full, kx, c.nt * q.bn, c.g, keep);
          } else {
            const int bz = MODE == kLnGradX ? c.g : 0;
            for (int j = 0; j < q.bn / 64; ++j)
              tma_load_3d_hint(sb + j * kLnMnBox, &map_b, full, c.nt * q.bn + j * 64, kx, bz, keep);
          }
          ++fills;
          if (++st == q.stages) {
            st = 0;
            ph ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ============================================================ MMA issuer
    if (lane == 0) {
      const uint32_t idesc = idesc_f16(std::is_same<T, __nv_bfloat16>::value ? 1u : 0u, kLnBM,
                                       static_cast<uint32_t>(q.bn), kAMn ? 1u : 0u, kBMn ? 1u : 0u);
      // K-major: 16 k (32 bytes) per MMA inside the 128-byte swizzled rows;
      // MN-major: 16 k rows (2 KB) per MMA, 64-wide m / n groups 8 KB apart.
      const uint64_t da0 = kAMn ? smem_desc_sw128(base, kLnMnBox, 1024) : smem_desc_sw128(base, 16, 1024);
      const uint64_t db0 = kBMn ? smem_desc_sw128(base + kLnABytes, kLnMnBox, 1024)
                                : smem_desc_sw128(base + kLnABytes, 16, 1024);
      constexpr uint32_t ka = kAMn ? (2048u >> 4) : 2u, kb = kBMn ? (2048u >> 4) : 2u;
      LnTile c;
      int st = 0;
      uint32_t ph = 0, cleared = 0;
      bool alive = true;
      for (int it = 0; alive && ln_tile<MODE>(q, ctrl, it, c); ++it) {
        ln_tile_taken(q, ctrl, it);
        const int buf = it & 1;
        if (it >= 2) {
          if (!mbar_wait(smem_u32(&ctrl->acc_empty[buf]), ((it >> 1) - 1) & 1)) {
            alive = false;
            break;
          }
          tc_fence_after();
        }
        const uint32_t d_tmem = tmem + static_cast<uint32_t>(buf * 256);
        for (int kk = 0; kk < c.nk; ++kk) {
          int steps = kLnBK / 16;
          bool ok = mbar_wait(smem_u32(&ctrl->full[st]), ph);
          if (MODE == kLnGradW && ok && kk == c.nk - 1 && c.last < kLnBK) {
            mbar_arrive(smem_u32(&ctrl->partial));
            ok = mbar_wait(smem_u32(&ctrl->cleared), cleared);
            cleared ^= 1u;
            steps = (c.last + 15) / 16;
          }
          if (!ok) {
            alive = false;
            break;
          }
          tc_fence_after();
          const uint32_t adv = static_cast<uint32_t>(st * q.stage_bytes) >> 4;
          if (MODE != kLnGradW || steps == kLnBK / 16) {
#pragma unroll
            for (int k = 0; k < kLnBK / 16; ++k)
              tc_mma_f16(d_tmem, da0 + adv + ka * k, db0 + adv + kb * k, idesc, (kk != 0 || k != 0) ? 1u : 0u);
          } else {
            for (int k = 0; k < steps; ++k)
              tc_mma_f16(d_tmem, da0 + adv + ka * k, db0 + adv + kb * k, idesc, (kk != 0 || k != 0) ? 1u : 0u);
          }
          tc_commit(smem_u32(&ctrl->empty[st]));
          if (++st == q.stages) {
            st = 0;
            ph ^= 1u;
          }
        }
        if (!alive) break;
        if (c.nk == 0)
          mbar_arrive(smem_u32(&ctrl->acc_full[buf]));  // empty K range: the tile is zero
        else
          tc_commit(smem_u32(&ctrl->acc_full[buf]));
      }
      if (!alive) ctrl->failed = 1;
    }
  } else if (warp == 2) {
    // ============================================================ dW: rows of the next group
    // The last K block of a group may hold rows of the next one. They are
    // cleared in both operands (not only one: theirs may be infinite), up to
    // the next multiple of 16 rows, where the products of the block stop.
    if (MODE == kLnGradX && q.bias_sums) {
      griddep_wait();
      // The bias gradient beside the products: a launch less.
      const int cols = (q.kc + 31) / 32;
      for (int64_t j = blockIdx.x; j < static_cast<int64_t>(cols) * q.groups; j += gridDim.x)
        ln_bias_columns<T>(q.offsets, q.groups, q.rows, q.kc, q.bias_sums, static_cast<T*>(q.db),
                           static_cast<int>(j / cols), static_cast<int>(j % cols) * 32);
    }
    if (MODE == kLnGradW) {
      LnTile c;
      int64_t filled = 0;  // K blocks of this CTA before the tile
      uint32_t turn = 0;
      for (int i = 0; ln_warp_tile<MODE>(q, ctrl, i, c); ++i) {
        if (c.nk > 0 && c.last < kLnBK) {
          const int64_t f = filled + c.nk - 1;
          const int st = static_cast<int>(f % q.stages);
          // The MMA warp has seen the block and waits: the stage holds it until then.
          if (!ln_warp_wait(smem_u32(&ctrl->partial), turn)) break;
          turn ^= 1u;
          if (!ln_warp_wait(smem_u32(&ctrl->full[st]), static_cast<uint32_t>(f / q.stages) & 1u)) break;
          const int r1 = (c.last + 15) / 16 * 16;
          const int boxes = (kLnBM + q.bn) / 64;
          const int pieces = (r1 - c.last) * 8;
          const uint32_t s0 = base + st * q.stage_bytes + c.last * 128;
          for (int j = lane; j < boxes * pieces; j += 32) {
            const int b = j / pieces, p = j - b * pieces;
            ln_sts(s0 + b * kLnMnBox + p * 16, 0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&ctrl->cleared));
        }
        filled += c.nk;
      }
    }
  } else if (warp == 3) {
    // ============================================================ scheduler
    if (q.offsets) {
      LnWalker<MODE> w;
      LnTile c;
      bool more = true;
      for (int i = 0; more; ++i) {
        more = w.seek(q, blockIdx.x + i * gridDim.x, c);
        const int slot = i % kLnAhead;
        if (i >= kLnAhead && !ln_warp_wait(smem_u32(&ctrl->sched_empty[slot]), (i / kLnAhead - 1) & 1)) break;
        if (lane == 0) {
          if (!more) c.g = -1;
          ctrl->sched[slot] = c;
          mbar_arrive(smem_u32(&ctrl->sched_full[slot]));
        }
        __syncwarp();
      }
    }
  } else if (warp >= 4) {
    // ============================================================ epilogue
    const int h = (warp - 4) >> 2;  // column part of the tile
    const int wq = warp & 3;        // TMEM lane quarter
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t stage = staging + static_cast<uint32_t>((warp - 4) * kLnStageTile);
    const uint32_t bias_tile = staging + kLnEpiWarps * kLnStageTile + static_cast<uint32_t>((warp - 4) * kLnBiasBytes);
    LnTile c, next;
    LnAhead ahead{};
    const uint64_t policy = l2_policy_evict_normal();
    bool more = ln_warp_tile<MODE>(q, ctrl, 0, c);
    if (more) ln_read_ahead<MODE>(q, c, wq, h, 0, lane, ahead);
    for (int it = 0; more; ++it) {
      const bool has_next = ln_warp_tile<MODE>(q, ctrl, it + 1, next);
      const int buf = it & 1;
      const uint32_t tb = tmem + lane_off + static_cast<uint32_t>(buf * 256 + h * ln_part(q));
      if (!ln_drain<T, MODE, ACT, FLAG>(q, &map_y, policy, c, next, has_next, tb, wq, h, lane, stage, bias_tile,
                                        smem_u32(&ctrl->acc_full[buf]), (it >> 1) & 1,
                                        smem_u32(&ctrl->acc_empty[buf]), ahead)) {
        if (lane == 0) ctrl->failed = 1;
        break;
      }
      more = has_next;
      c = next;
    }
    if (lane == 0) bulk_wait_read_all();
  }

  // ---------------------------------------------------------------- teardown
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (ctrl->failed) {
    if (tid == 0) ln_settle_loads(ctrl->full, q.stages, fills);
    if (tid == 32) {  // the lane that issued the products
      tc_commit(smem_u32(&ctrl->settled));
      ln_settle(smem_u32(&ctrl->settled), 0);
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ============================================================================
// The forward pass where 128 x 64 tiles are too few for the SMs: a cluster of 2,
// 4 or 8 CTAs shares one tile's K blocks. A CTA takes in only some 70 GB/s from
// L2, so a tile alone takes 0.35 us a K block; each CTA of a cluster
// accumulates its share in TMEM and lays it down in shared memory, and after a
// cluster barrier every CTA finishes a part of the tile from the sums of all
// (distributed shared memory, in the order of the CTAs). One tile a cluster.
constexpr int kLsThreads = 256;
constexpr int kLsBN = 64;
constexpr int kLsStageBytes = kLnABytes + kLsBN * kLnBK * 2;  // 24 KB
constexpr int kLsRow = kLsBN + 4;  // floats between rows of the sums: no bank conflicts
constexpr int kLsSums = kLnBM * kLsRow * 4;
constexpr int kLsCtrlBytes = 256;
// Dynamic shared memory for a ring of `stages`; the sums reuse it.
__host__ __device__ constexpr int ls_ring(int stages) {
  return stages * kLsStageBytes > kLsSums ? stages * kLsStageBytes : kLsSums;
}
__host__ __device__ constexpr int ls_smem(int stages) { return 1024 + ls_ring(stages) + kLsCtrlBytes; }

struct LsCtrl {
  uint64_t full[kLnMaxStages], empty[kLnMaxStages];
  uint64_t done;
  uint32_t failed, tmem_base;
};
static_assert(sizeof(LsCtrl) <= kLsCtrlBytes, "control block too large");

__device__ __forceinline__ float4 ls_peer_ld(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(mapa_shared(addr, rank)));
  return v;
}

template <typename T, int ACT, bool DERIV>
__global__ void __launch_bounds__(kLsThreads)
    tc_linear_split(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                    const LnGeom q, int ctas) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = static_cast<int>(blockIdx.x) % ctas;
  LnTile c;
  {
    const int t = static_cast<int>(blockIdx.x) / ctas;
    if (q.offsets) {
      LnWalker<kLnForward> w;
      if (!w.seek(q, t, c)) return;  // the cluster's CTAs agree
    } else {
      ln_set_tile<kLnForward>(q, c, 0, 0, q.rows, t);
    }
  }
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  LsCtrl* ctrl = reinterpret_cast<LsCtrl*>(smem_raw + (base - raw) + ls_ring(q.stages));
  const int k0 = c.nk * rank / ctas, nk = c.nk * (rank + 1) / ctas - k0;
  if (tid == 0) {
    for (int s = 0; s < q.stages; ++s) {
      mbar_init(smem_u32(&ctrl->full[s]), 1);
      mbar_init(smem_u32(&ctrl->empty[s]), 1);
    }
    mbar_init(smem_u32(&ctrl->done), 1);
    ctrl->failed = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&ctrl->tmem_base), kLsBN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctrl->tmem_base;
  int fills = 0;
  if (warp == 0 && lane == 0) {
    const uint64_t keep = l2_policy_evict_last();
    griddep_wait();  // for the copy of rows, if there is one
    for (int kk = 0; kk < nk && !q.test_stall; ++kk, ++fills) {
      const int st = kk % q.stages;
      if (kk >= q.stages && !mbar_wait(smem_u32(&ctrl->empty[st]), (kk / q.stages - 1) & 1)) break;
      const uint32_t full = smem_u32(&ctrl->full[st]);
      const uint32_t sa = base + st * kLsStageBytes;
      mbar_arrive_expect_tx(full, kLsStageBytes);
      tma_load_3d_hint(sa + kLnABytes, &map_b, full, (k0 + kk) * kLnBK, c.nt * kLsBN, c.g, keep);
      tma_load_3d_hint(sa, &map_a, full, (k0 + kk) * kLnBK, c.row0, 0, keep);
    }
  } else if (warp == 1 && lane == 0) {
    const uint32_t idesc = idesc_f16(std::is_same<T, __nv_bfloat16>::value ? 1u : 0u, kLnBM, kLsBN, 0u, 0u);
    const uint64_t da0 = smem_desc_sw128(base, 16, 1024), db0 = smem_desc_sw128(base + kLnABytes, 16, 1024);
    bool alive = true;
    for (int kk = 0; alive && kk < nk; ++kk) {
      const int st = kk % q.stages;
      alive = mbar_wait(smem_u32(&ctrl->full[st]), (kk / q.stages) & 1);
      if (!alive) break;
      tc_fence_after();
      const uint32_t adv = static_cast<uint32_t>(st * kLsStageBytes) >> 4;
#pragma unroll
      for (int k = 0; k < kLnBK / 16; ++k)
        tc_mma_f16(tmem, da0 + adv + 2 * k, db0 + adv + 2 * k, idesc, (kk != 0 || k != 0) ? 1u : 0u);
      tc_commit(smem_u32(&ctrl->empty[st]));
    }
    if (!alive) ctrl->failed = 1;
    if (nk > 0) tc_commit(smem_u32(&ctrl->done));  // when the products issued so far have ended
    else mbar_arrive(smem_u32(&ctrl->done));
  }
  __syncwarp();
  // Every product has read its operands when `done` completes: the ring is free.
  if (!ln_warp_wait(smem_u32(&ctrl->done), 0)) ln_settle(smem_u32(&ctrl->done), 0);
  if (tid == 0 && ctrl->failed) ln_settle_loads(ctrl->full, q.stages, fills);
  __syncwarp();
  tc_fence_after();
  const int wq = warp & 3, h = warp >> 2;
  if (c.row0 + wq * 32 < c.hi) {
    const uint32_t p = base + static_cast<uint32_t>((wq * 32 + lane) * kLsRow + h * 32) * 4;
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      uint32_t o[16];
      ln_tmem_ld16(tmem + (static_cast<uint32_t>(wq * 32) << 16) + static_cast<uint32_t>(h * 32 + hh * 16), nk == 0, o);
#pragma unroll
      for (int i = 0; i < 4; ++i) ln_sts(p + hh * 64 + i * 16, o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
    }
  }
  tc_fence_before();
  cluster_sync();  // all sums are in place (and this CTA's accumulator has been read)
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kLsBN);
  }
  const int rows = min(kLnBM, c.hi - c.row0);
  const bool zero = c.g >= q.groups;
  for (int i = rank * kLsThreads + tid; i < rows * (kLsBN / 4); i += ctas * kLsThreads) {
    const int r = i / (kLsBN / 4), tc = i % (kLsBN / 4) * 4;
    const int64_t row = c.row0 + r;
    const int col = c.nt * kLsBN + tc;
    if (col >= q.n) continue;
    const uint32_t at = base + static_cast<uint32_t>(r * kLsRow + tc) * 4;
    float z[4] = {0.f, 0.f, 0.f, 0.f};
    if (!zero) {
      for (int k = 0; k < ctas; ++k) {
        const float4 v = ls_peer_ld(at, static_cast<uint32_t>(k));
        z[0] += v.x;
        z[1] += v.y;
        z[2] += v.z;
        z[3] += v.w;
      }
      const T* bias = q.bias ? static_cast<const T*>(q.bias) + static_cast<int64_t>(c.g) * q.bias_gs + col : nullptr;
      const T* res = q.res ? static_cast<const T*>(q.res) + row * q.res_ld + col : nullptr;
      uint32_t codes[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bool one = col + 2 * j < q.n, two = col + 2 * j + 1 < q.n;
        if (bias) {
          if (one) z[2 * j] = __fadd_rn(z[2 * j], Elem<T>::to_f(bias[2 * j]));
          if (two) z[2 * j + 1] = __fadd_rn(z[2 * j + 1], Elem<T>::to_f(bias[2 * j + 1]));
        }
        LnPair d;
        const float2 y = ln_split(ln_act2<ACT, DERIV>(ln_pair(z[2 * j], z[2 * j + 1]), &d));
        if (DERIV) codes[j] = ln_encode2<T, ACT>(d);
        z[2 * j] = y.x;
        z[2 * j + 1] = y.y;
        if (res) {
          if (one) z[2 * j] = __fadd_rn(z[2 * j], Elem<T>::to_f(res[2 * j]));
          if (two) z[2 * j + 1] = __fadd_rn(z[2 * j + 1], Elem<T>::to_f(res[2 * j + 1]));
        }
      }
      if (DERIV)  // rows of codes are whole 32-byte units: past n lies padding
        *reinterpret_cast<uint2*>(q.deriv + row * q.deriv_ld + col) = make_uint2(codes[0], codes[1]);
    }
    T* out = static_cast<T*>(q.out) + row * q.out_ld + col;
    if (q.out_vec && col + 4 <= q.n) {
      *reinterpret_cast<uint2*>(out) = make_uint2(ln_pack<T>(z[0], z[1]), ln_pack<T>(z[2], z[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < q.n) out[j] = Elem<T>::from_f(z[j]);
    }
  }
  cluster_sync();  // the peers have read this CTA's sums
}

}  // namespace avey
