// The steps of the linear layers (avey_linear_*) around the products of
// tc_linear.cuh: the kernel for few rows, dpre = dy act' with the bias
// gradient's partial sums, the sums of partial results in a fixed order, and
// the copy that lays rows out in whole 16-byte units.
#pragma once

#include "tc_linear.cuh"

namespace avey {

// Eight 16-bit values at p as four words; values at `left` and beyond are zero.
__device__ __forceinline__ uint4 ln_load8(const uint16_t* p, int left, bool vec) {
  if (vec && left >= 8) return __ldg(reinterpret_cast<const uint4*>(p));
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) w[j >> 1] |= static_cast<uint32_t>(__ldg(p + j)) << (16 * (j & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

struct LnOct2 {
  uint4 a, b;  // 16 consecutive values
};
// Sixteen 16-bit values at p; values at `left` and beyond are zero. `vec`: 32-byte
// aligned (2), 16-byte aligned (1) or neither.
__device__ __forceinline__ LnOct2 ln_load16(const uint16_t* p, int left, int vec) {
  LnOct2 r;
  if (vec == 2 && left >= 16) {
    asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r.a.x), "=r"(r.a.y), "=r"(r.a.z), "=r"(r.a.w), "=r"(r.b.x), "=r"(r.b.y), "=r"(r.b.z),
                   "=r"(r.b.w)
                 : "l"(p));
  } else {
    r.a = ln_load8(p, left, vec != 0);
    r.b = ln_load8(p + 8, left - 8, vec != 0);
  }
  return r;
}

// ---------------------------------------------------------------- few rows

// y for a few rows per group: the weights are read once, straight from global
// memory into mma.sync fragments (bound: their bytes; the products are far
// below any tensor rate, and 128-row tiles would leave most SMs without
// work). W is the 16-row operand, up to 8 NT rows of x the 8-column one. The
// order of k inside a product is free as long as both operands agree, so a
// lane takes 16 consecutive k (32 bytes) of a 64-wide step for its fragments:
// four lanes read a whole line of a row (with 16 bytes a lane, half lines, 48
// rows of 2048 -> 1024 took 8.8 us).
// A CTA owns 16 outputs; its warps share the steps of K, and their sums are added
// in a fixed order: 8 warps; 16 where there are no more CTAs than SMs and K is
// long (48 rows of 2048 -> 1024 by 64 CTAs: 7.5 against 8.2 us); 4 where there are three CTAs
// an SM and more, which then come and go more evenly (16 rows of 16 experts, 1024
// -> 2048, from HBM: 11.2 against 13.9 us, 3.9 TB/s; 4 rows of 2048 -> 8192: 9.5
// against 10.3; but 384 CTAs of 1536 -> 6144: 7.0 against 6.3).
constexpr int kLfOut = 16;

struct LnFew {
  const int32_t* offsets;
  int groups, rows, n, k;
  const uint16_t *x, *w, *bias, *res;
  int64_t x_ld, w_ld, w_gs, bias_gs, res_ld, y_ld, deriv_ld;
  uint16_t *y, *deriv;
  int x_vec, w_vec;  // rows are 32-byte aligned (2), 16-byte aligned (1) or neither
};

template <typename T>
__device__ __forceinline__ void ln_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T, int ACT, bool DERIV, int NT, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) ln_few(const LnFew q) {
  constexpr int kThreads = 32 * WARPS;
  constexpr int kParts = WARPS < 8 ? WARPS : 8;
  __shared__ float red[kParts][8 * NT][kLfOut + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * kLfOut;
  LnSpan s{0, 0, q.rows, 0, 0, 1};
  if (q.offsets) {
    // Slot y: the y-th group that has rows; the slot after the last: the rest.
    ln_find(q.offsets, q.groups, q.rows, blockIdx.y, 0, [](int lo, int hi) { return hi > lo ? 1 : 0; }, s);
    if (s.g == q.groups && s.index != 0) return;
  }
  const bool zero = s.g == q.groups;
  const uint16_t* w0 = q.w + static_cast<int64_t>(s.g) * q.w_gs;
  const int o_lo = n0 + (lane >> 2), o_hi = o_lo + 8;
  const uint16_t* wl = w0 + static_cast<int64_t>(o_lo) * q.w_ld;
  const uint16_t* wh = w0 + static_cast<int64_t>(o_hi) * q.w_ld;
  // Dense layers: the passes of 8 NT rows are shared by the grid's second dimension.
  const int pass0 = q.offsets ? 0 : blockIdx.y, passes = q.offsets ? 1 : gridDim.y;
  for (int r0 = s.lo + pass0 * 8 * NT; r0 < s.hi; r0 += passes * 8 * NT) {
    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
    if (!zero) {
      constexpr int kUnroll = NT >= 4 ? 1 : 2;
      const int steps = (q.k + 63) / 64;
      for (int s0 = warp; s0 < steps; s0 += WARPS * kUnroll) {
        LnOct2 a[kUnroll], b[kUnroll], v[kUnroll][NT];
        const LnOct2 none{make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int k = (s0 + WARPS * u) * 64 + (lane & 3) * 16;
          const int left = q.k - k;
          a[u] = b[u] = none;
          if (left > 0 && o_lo < q.n) a[u] = ln_load16(wl + k, left, q.w_vec);
          if (left > 0 && o_hi < q.n) b[u] = ln_load16(wh + k, left, q.w_vec);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const int row = r0 + j * 8 + (lane >> 2);
            v[u][j] = none;
            if (left > 0 && row < s.hi)
              v[u][j] = ln_load16(q.x + static_cast<int64_t>(row) * q.x_ld + k, left, q.x_vec);
          }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            ln_mma<T>(acc[j], a[u].a.x, b[u].a.x, a[u].a.y, b[u].a.y, v[u][j].a.x, v[u][j].a.y);
            ln_mma<T>(acc[j], a[u].a.z, b[u].a.z, a[u].a.w, b[u].a.w, v[u][j].a.z, v[u][j].a.w);
            ln_mma<T>(acc[j], a[u].b.x, b[u].b.x, a[u].b.y, b[u].b.y, v[u][j].b.x, v[u][j].b.y);
            ln_mma<T>(acc[j], a[u].b.z, b[u].b.z, a[u].b.w, b[u].b.w, v[u][j].b.z, v[u][j].b.w);
          }
      }
    }
    // The upper warps of 16 hand their sums to the lower ones.
    auto put = [&](bool add) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float& z = red[warp % kParts][j * 8 + (lane & 3) * 2 + (i & 1)][(lane >> 2) + (i >> 1) * 8];
          z = add ? z + acc[j][i] : acc[j][i];
        }
    };
    __syncthreads();
    if (WARPS == 16) {
      if (warp >= 8) put(false);
      __syncthreads();
      if (warp < 8) put(true);
    } else {
      put(false);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * NT * kLfOut; i += kThreads) {
      const int r = i / kLfOut, o = i % kLfOut;
      const int row = r0 + r, col = n0 + o;
      if (row >= s.hi || col >= q.n) continue;
      float z = 0.f;
#pragma unroll
      for (int k = 0; k < kParts; ++k) z += red[k][r][o];
      float y = 0.f;
      if (!zero) {
        if (q.bias) z += Elem<T>::to_f(reinterpret_cast<const T*>(q.bias)[static_cast<int64_t>(s.g) * q.bias_gs + col]);
        LnPair d;
        y = ln_split(ln_act2<ACT, DERIV>(ln_pair(z), &d)).x;
        if (DERIV)
          q.deriv[static_cast<int64_t>(row) * q.deriv_ld + col] = static_cast<uint16_t>(ln_encode2<T, ACT>(d));
        if (q.res) y += Elem<T>::to_f(reinterpret_cast<const T*>(q.res)[static_cast<int64_t>(row) * q.res_ld + col]);
      }
      reinterpret_cast<T*>(q.y)[static_cast<int64_t>(row) * q.y_ld + col] = Elem<T>::from_f(y);
    }
  }
}

// ---------------------------------------------------------------- dpre

// dpre = dy act' in the operand type, and the fp32 sums of dpre (before that
// rounding) over every tile of 64 rows of a group. The rounding is what 16-bit
// operands of the two products take: it makes the error of dx and dW against 64
// bits 1.41 times that of an fp32 dpre (2.3 10^-3 of their norm in bf16, 2.9 10^-4 in
// f16; the results' own rounding is the rest), and a second 16-bit part for what it
// cuts off would double both products. Bound by HBM: 6 bytes an element. A warp reads rows of 512 bytes, a thread 8 columns of 8 rows at once,
// all loads before the first product (32768 x 1536: 54 us, 5.6 TB/s).
constexpr int kLdThreads = 256;
constexpr int kLdCols = 256;

struct LnDpre {
  const int32_t* offsets;
  int groups, rows, n;
  const uint16_t* dy;
  int64_t dy_ld;
  int dy_vec;
  const uint16_t* deriv;  // null: the identity
  int64_t deriv_ld;
  uint16_t* dpre;  // null: only the sums are wanted
  int64_t dpre_ld;
  float* partial;  // [tiles][n], or null
};

template <typename T, int ACT>
__global__ void __launch_bounds__(kLdThreads) ln_dpre(const LnDpre q) {
  __shared__ float red[8][kLdCols];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_launch_dependents();  // the products are set up meanwhile
  LnSpan s;
  if (!ln_find(q.offsets, q.groups, q.rows, blockIdx.x, 0, ln_dpre_tiles, s)) return;
  const int row0 = s.lo + s.index * kLdRows, row1 = min(s.hi, row0 + kLdRows);
  const int col = blockIdx.y * kLdCols + lane * 8;
  const int left = q.n - col;
  float sum[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) sum[j] = 0.f;
  if (left > 0) {
    uint4 g[8], d[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = row0 + warp + 8 * i;
      g[i] = d[i] = make_uint4(0u, 0u, 0u, 0u);
      if (row < row1) {
        g[i] = ln_load8(q.dy + static_cast<int64_t>(row) * q.dy_ld + col, left, q.dy_vec);
        if (ACT != 0) d[i] = ln_load8(q.deriv + static_cast<int64_t>(row) * q.deriv_ld + col, left, true);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = row0 + warp + 8 * i;
      if (row >= row1) break;
      const uint32_t gw[4] = {g[i].x, g[i].y, g[i].z, g[i].w}, dw[4] = {d[i].x, d[i].y, d[i].z, d[i].w};
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 v = ln_unpack<T>(gw[j]);
        if (ACT != 0) {
          v.x *= ln_decode<T, ACT>(dw[j] & 0xFFFFu);
          v.y *= ln_decode<T, ACT>(dw[j] >> 16);
        }
        sum[2 * j] += v.x;
        sum[2 * j + 1] += v.y;
        o[j] = ln_pack<T>(v.x, v.y);
      }
      if (q.dpre)  // rows of dpre are whole 16-byte units
        *reinterpret_cast<uint4*>(q.dpre + static_cast<int64_t>(row) * q.dpre_ld + col) =
            make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
  if (!q.partial) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) red[warp][lane * 8 + j] = sum[j];
  __syncthreads();
  const int c = blockIdx.y * kLdCols + threadIdx.x;
  if (c < q.n) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += red[i][threadIdx.x];
    q.partial[static_cast<int64_t>(blockIdx.x) * q.n + c] = t;
  }
}

// db where the dX kernel does not sum it: the same order as ln_bias_columns, by 32
// warps for 32 columns of a group (512 tiles of 1536 columns: 5.2 us; by 8 warps
// 7.6).
constexpr int kLbThreads = 1024;
template <typename T>
__global__ void __launch_bounds__(kLbThreads) ln_bias_sum(const int32_t* offsets, int groups, int rows, int n,
                                                          const float* partial, T* db) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  LnSpan s;
  ln_find(offsets, groups, rows, -1, blockIdx.y, ln_dpre_tiles, s);
  const int c = blockIdx.x * 32 + lane;
  float t = 0.f;
  if (c < n)
#pragma unroll 4
    for (int i = part; i < s.cnt; i += 32) t += partial[static_cast<int64_t>(s.base + i) * n + c];
  red[part][lane] = t;
  __syncthreads();
  if (part == 0 && c < n) {
    float z = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) z += red[i][lane];
    db[static_cast<int64_t>(blockIdx.y) * n + c] = Elem<T>::from_f(z);
  }
}

// The same for many groups of few tiles, where 32 warps each would mostly wait for
// the walk to their group: one warp for 32 columns of a group.
constexpr int kLbWarps = 8;
template <typename T>
__global__ void __launch_bounds__(32 * kLbWarps) ln_bias_groups(const int32_t* offsets, int groups, int rows, int n,
                                                                const float* partial, T* db) {
  const int cols = (n + 31) / 32;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * kLbWarps + (threadIdx.x >> 5);
  if (j < static_cast<int64_t>(cols) * groups)
    ln_bias_columns<T>(offsets, groups, rows, n, partial, db, static_cast<int>(j / cols),
                       static_cast<int>(j % cols) * 32);
}

// out[row][c] = sum over the splits of partial[split][row][c], in split order
// (four splits of 1536 x 768, out of L2: 4.2 us);
// rows of `partial` have `ld` floats (a multiple of 4), rows of `out` n values.
template <typename T>
__global__ void __launch_bounds__(256) ln_split_sum(const float* partial, int splits, int64_t rows, int n, int64_t ld,
                                                    T* out) {
  const int64_t per = ld / 4, total = rows * per, plane = rows * ld;
  const bool vec = (n & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 7u) == 0;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / per;
    const int c = static_cast<int>(i - row * per) * 4;
    const float* p = partial + row * ld + c;
    float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < splits; ++s) {
      const float4 v = *reinterpret_cast<const float4*>(p + s * plane);
      z.x += v.x;
      z.y += v.y;
      z.z += v.z;
      z.w += v.w;
    }
    T* o = out + row * n + c;
    if (c + 4 <= n && vec) {
      *reinterpret_cast<uint2*>(o) = make_uint2(ln_pack<T>(z.x, z.y), ln_pack<T>(z.z, z.w));
    } else {
      const float v[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < n) o[j] = Elem<T>::from_f(v[j]);
    }
  }
}

// Rows of `cols` 16-bit values (`per` rows of a group, groups gs apart) copied to
// rows of ld values (a multiple of 8), zeros at the end: what TMA can read. Two
// arrays a launch (rows 0: none). 1037 x 389 and 771 x 389 take 2.5 us.
struct LnPack {
  const uint16_t* src;
  int64_t src_ld, src_gs, per, rows, ld;
  int cols;
  uint16_t* dst;
};
static __global__ void __launch_bounds__(256) ln_pack_rows(const LnPack a, const LnPack b) {
  griddep_launch_dependents();  // the products are set up meanwhile
  griddep_wait();
  const int64_t na = a.rows * (a.ld / 8), nb = b.rows * (b.ld / 8);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < na + nb;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const LnPack& k = i < na ? a : b;
    const int64_t j = i < na ? i : i - na;
    const int64_t pieces = k.ld / 8, row = j / pieces, g = row / k.per;
    const int c = static_cast<int>(j - row * pieces) * 8;
    const uint16_t* p = k.src + g * k.src_gs + (row - g * k.per) * k.src_ld + c;
    *reinterpret_cast<uint4*>(k.dst + row * k.ld + c) = ln_load8(p, k.cols - c, false);
  }
}

}  // namespace avey
