// One AdamW step over many tensors (avey_adamw_v1), with states in fp32 or in
// float8 blocks of 256.
//
// Every element is read once and written once, so the step is bound by HBM:
// 28 bytes an element for fp32 weights with fp32 states (or 16-bit weights
// with fp32 masters), 22 for 16-bit weights, 10 with 8-bit states. 82 M bf16
// weights with masters take 365 us (6.3 TB/s, 0.96 of the copy rate); 0.7 M
// fp32 weights in 42 tensors 4.6 us.
//
// The tensors' pointers travel in the kernel's parameters (up to 400 tensors a
// launch), so a step is one launch, copies nothing to the device and keeps
// nothing between calls. Work is cut into chunks of 2048 elements of one tensor
// (8 warps, 256 elements each: a warp owns a block of the 8-bit states and
// finds its maximum with one reduction). A chunk's tensor is found by bisection
// of the chunk prefix at first and by walking forward after.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

namespace avey {

constexpr int kAwThreads = 256;
constexpr int kAwBlock = 256;                         // elements per warp and per 8-bit block
constexpr int kAwChunk = kAwBlock * kAwThreads / 32;  // elements per CTA and step

struct AwTensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* ms;
  float* vs;
  float* master;
  int64_t n;
  int64_t block0;  // number of the tensor's first block in the whole call
  int32_t chunk0;  // first chunk of the launch
  int32_t whole;   // 8-bit states: the first chunks that are whole and aligned
};

constexpr int kAwCtas8 = 3;   // CTAs per SM of the 8-bit step (at four, 64 registers a thread, it spills)
constexpr int kAwStages = 3;  // its blocks in flight per warp

template <int N>
struct AwTable {
  int count;
  int chunks;
  AwTensor t[N];
};

struct AwScalars {
  float b1, c1, b2, c2;  // beta, 1 - beta
  float decay;           // 1 - lr wd
  float step_size;       // lr / (1 - beta1^t)
  float inv_bc2;         // 1 / sqrt(1 - beta2^t)
  float eps;
  // The same as pairs, which packed instructions read from the parameters.
  float2 b1p, c1p, b2p, c2p, decayp, minus_stepp, inv_bc2p, epsp;
  float2 minus_zerop;  // -0 (see aw_prod2)
  uint32_t seed;
  uint32_t step;
  uint32_t key;          // aw_key of the first 2^32 elements
  const float* grad_scale;
};

// A 32-bit mix of two products, constants from C. Wellons, "Prospecting for hash
// functions" (2018).
__device__ __forceinline__ uint32_t aw_mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x7feb352du;
  x ^= x >> 15;
  x *= 0x846ca68bu;
  return x ^ (x >> 16);
}

__host__ __device__ __forceinline__ uint32_t aw_key(uint32_t seed, uint32_t step, uint32_t hi) {
  uint32_t x = seed + 0x9e3779b9u * (step + hi);
  x = (x ^ (x >> 16)) * 0x7feb352du;
  return (x ^ (x >> 16)) * 0x846ca68bu;
}

// N consecutive values of type T from / to memory aligned to the whole vector
// (at most 32 bytes), converted to fp32.
template <int BYTES>
struct AwRaw {
  uint32_t w[BYTES / 4];
};
template <int BYTES>
__device__ __forceinline__ AwRaw<BYTES> aw_ld(const void* p) {
  AwRaw<BYTES> r;
  if constexpr (BYTES == 32) {
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]),
                   "=r"(r.w[6]), "=r"(r.w[7])
                 : "l"(p));
  } else if constexpr (BYTES == 16) {
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3])
                 : "l"(p));
  } else {
    asm volatile("ld.global.L1::no_allocate.v2.b32 {%0,%1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "l"(p));
  }
  return r;
}
template <int BYTES>
__device__ __forceinline__ void aw_st(void* p, const AwRaw<BYTES>& r) {
  if constexpr (BYTES == 32) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]),
                 "r"(r.w[2]), "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7])
                 : "memory");
  } else if constexpr (BYTES == 16) {
    asm volatile("st.global.v4.b32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]),
                 "r"(r.w[3])
                 : "memory");
  } else {
    asm volatile("st.global.v2.b32 [%0], {%1,%2};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]) : "memory");
  }
}

template <typename T>
__device__ __forceinline__ float aw_to_f(T x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
  else return __bfloat162float(x);
}
template <typename T>
__device__ __forceinline__ T aw_from_f(float x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

// Eight values of T at element `at` of an array; lanes past `left` elements
// read zeros. `vec`: the array is aligned to eight elements.
template <typename T>
__device__ __forceinline__ void aw_load8(const void* base, int64_t at, int left, bool vec, float (&f)[8]) {
  const T* p = static_cast<const T*>(base) + at;
  if (vec && left >= 8) {
    const auto r = aw_ld<8 * sizeof(T)>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = aw_to_f<T>(reinterpret_cast<const T*>(&r)[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < left ? aw_to_f<T>(p[i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void aw_store8(void* base, int64_t at, int left, bool vec, const float (&f)[8]) {
  T* p = static_cast<T*>(base) + at;
  if (vec && left >= 8) {
    AwRaw<8 * sizeof(T)> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(&r)[i] = aw_from_f<T>(f[i]);
    aw_st<8 * sizeof(T)>(p, r);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = aw_from_f<T>(f[i]);
  }
}

// e4m3 codes, two to a 16-bit word.
__device__ __forceinline__ float2 aw_decode2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
  return __half22float2(__half2(h));
}
__device__ __forceinline__ uint32_t aw_encode2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// x / scale rounded to the e4m3 grid by adding `noise` (20 bits) below the
// last kept bit of the magnitude and cutting the rest off. Below 2^-6 the grid
// is even (steps of 2^-9): there the same is done to |r| + 2^-6.
__device__ __forceinline__ float aw_round_fast(float r, uint32_t noise) {
  return __uint_as_float((__float_as_uint(r) + noise) & 0xFFF00000u);
}
__device__ __forceinline__ float aw_round(float r, uint32_t noise) {
  const float a = fabsf(r);
  const bool small = a < 0x1p-6f;
  float t = __uint_as_float((__float_as_uint(small ? a + 0x1p-6f : a) + noise) & 0xFFF00000u);
  if (small) t -= 0x1p-6f;
  return copysignf(t, r);
}

// The scale of a block whose largest magnitude has the bits `top` (NaN above
// infinity, so a NaN stays visible).
__device__ __forceinline__ float aw_scale(uint32_t top) {
  const float s = __uint_as_float(top) * (1.f / 448.f);
  return s < 0x1p-126f ? 0x1p-126f : s;
}

// The warp's 256 elements from `at0` of tensor t (the last block of a tensor may
// be shorter; any alignment).
template <typename T, bool MASTER, bool Q8>
__device__ __forceinline__ void aw_block(const AwTensor& t, const AwScalars& c, float gs, int64_t at0) {
  const int lane = threadIdx.x & 31;
  const int64_t at = at0 + lane * 8;
  const int left = static_cast<int>(t.n - at < 8 ? (t.n - at < 0 ? 0 : t.n - at) : 8);
  constexpr uintptr_t kMask = 8 * sizeof(T) - 1;
  const bool vec = ((reinterpret_cast<uintptr_t>(t.p) | reinterpret_cast<uintptr_t>(t.g)) & kMask) == 0;
  const bool mvec = MASTER && (reinterpret_cast<uintptr_t>(t.master) & 31u) == 0;
  constexpr uintptr_t kStateMask = Q8 ? 7 : 31;
  const bool svec = ((reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v)) & kStateMask) == 0;
  float g[8], p[8], m[8], v[8];
  float ms = 0.f, vs = 0.f;
  AwRaw<8> mq{}, vq{};
  // Every load first, so that all are in flight together.
  aw_load8<T>(t.g, at, left, vec, g);
  if (MASTER) aw_load8<float>(t.master, at, left, mvec, p);
  else aw_load8<T>(t.p, at, left, vec, p);
  const int64_t block = at0 / kAwBlock;
  if constexpr (Q8) {
    ms = t.ms[block];
    vs = t.vs[block];
    const uint8_t* mp = static_cast<const uint8_t*>(t.m) + at;
    const uint8_t* vp = static_cast<const uint8_t*>(t.v) + at;
    if (svec && left == 8) {
      mq = aw_ld<8>(mp);
      vq = aw_ld<8>(vp);
    } else {
      for (int i = 0; i < left; ++i) {
        mq.w[i >> 2] |= static_cast<uint32_t>(mp[i]) << (8 * (i & 3));
        vq.w[i >> 2] |= static_cast<uint32_t>(vp[i]) << (8 * (i & 3));
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = aw_decode2((mq.w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
      const float2 b = aw_decode2((vq.w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
      m[2 * i] = a.x * ms;
      m[2 * i + 1] = a.y * ms;
      v[2 * i] = b.x * vs;
      v[2 * i + 1] = b.y * vs;
      v[2 * i] *= v[2 * i];
      v[2 * i + 1] *= v[2 * i + 1];
    }
  } else {
    aw_load8<float>(t.m, at, left, svec, m);
    aw_load8<float>(t.v, at, left, svec, v);
  }
  float root[8];
  uint32_t mtop = 0, vtop = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // Each product and sum of the states is rounded by itself, so that the
    // stochastic codes are the same bits as the formula's in plain fp32.
    const float gi = g[i] * gs;
    m[i] = __fadd_rn(__fmul_rn(m[i], c.b1), __fmul_rn(gi, c.c1));
    v[i] = __fadd_rn(__fmul_rn(v[i], c.b2), __fmul_rn(__fmul_rn(gi, gi), c.c2));
    root[i] = sqrtf(v[i]);
    const float upd = __fdividef(m[i], fmaf(root[i], c.inv_bc2, c.eps));
    p[i] = fmaf(p[i], c.decay, -c.step_size * upd);
    if (Q8) {
      mtop = max(mtop, __float_as_uint(m[i]) & 0x7FFFFFFFu);
      vtop = max(vtop, __float_as_uint(root[i]) & 0x7FFFFFFFu);
    }
  }
  if (MASTER) aw_store8<float>(t.master, at, left, mvec, p);
  aw_store8<T>(t.p, at, left, vec, p);
  if constexpr (Q8) {
    mtop = __reduce_max_sync(0xFFFFFFFFu, mtop);
    vtop = __reduce_max_sync(0xFFFFFFFFu, vtop);
    ms = aw_scale(mtop);
    vs = aw_scale(vtop);
    const float mi = 1.f / ms, vi = 1.f / vs;
    const uint64_t e0 = static_cast<uint64_t>(t.block0 + block) * kAwBlock;
    const uint32_t key = aw_key(c.seed, c.step, static_cast<uint32_t>(e0 >> 32));
    const uint32_t idx = static_cast<uint32_t>(e0) + lane * 8;
    AwRaw<8> mo{}, vo{};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t h = aw_mix((idx + i) ^ key);
      m[i] = aw_round(m[i] * mi, ((h << 4) & 0xFFFF0u) | 8u);
      root[i] = aw_round(root[i] * vi, ((h >> 12) & 0xFFFF0u) | 8u);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      mo.w[i >> 1] |= aw_encode2(m[2 * i], m[2 * i + 1]) << (16 * (i & 1));
      vo.w[i >> 1] |= aw_encode2(root[2 * i], root[2 * i + 1]) << (16 * (i & 1));
    }
    uint8_t* mp = static_cast<uint8_t*>(t.m) + at;
    uint8_t* vp = static_cast<uint8_t*>(t.v) + at;
    if (svec && left == 8) {
      aw_st<8>(mp, mo);
      aw_st<8>(vp, vo);
    } else {
      for (int i = 0; i < left; ++i) {
        mp[i] = static_cast<uint8_t>(mo.w[i >> 2] >> (8 * (i & 3)));
        vp[i] = static_cast<uint8_t>(vo.w[i >> 2] >> (8 * (i & 3)));
      }
    }
    if (lane == 0) {
      t.ms[block] = ms;
      t.vs[block] = vs;
    }
  } else {
    aw_store8<float>(t.m, at, left, svec, m);
    aw_store8<float>(t.v, at, left, svec, v);
  }
}

// The last tensor whose first chunk is at or before `chunk`.
template <int N>
__device__ __forceinline__ int aw_tensor_of(const AwTable<N>& tab, int chunk) {
  int lo = 0, hi = tab.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.t[mid].chunk0 <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

// States in fp32.
template <typename T, bool MASTER, int N>
__global__ void __launch_bounds__(kAwThreads) adamw_step(const __grid_constant__ AwTable<N> tab, const AwScalars c) {
  const float gs = c.grad_scale ? *c.grad_scale : 1.f;
  int ti = aw_tensor_of(tab, blockIdx.x);
  for (int64_t chunk = blockIdx.x; chunk < tab.chunks; chunk += gridDim.x) {
    while (ti + 1 < tab.count && tab.t[ti + 1].chunk0 <= chunk) ++ti;
    const AwTensor& t = tab.t[ti];
    const int64_t at0 = (chunk - t.chunk0) * kAwChunk + (threadIdx.x >> 5) * kAwBlock;
    if (at0 < t.n) aw_block<T, MASTER, false>(t, c, gs, at0);
  }
}

// ---------------------------------------------------------------- 8-bit states
//
// At 10 bytes an element HBM leaves about 55 instructions an element, so the
// whole blocks of aligned tensors take a loop of their own: two values to an
// instruction (f32x2), three-input minima and maxima, one square root step for
// a pair, and the next chunks' loads in flight (cp.async). 64 M bf16 parameters
// take 168 us (4.0 TB/s) with 65 instructions an element. Counters of that
// launch: issue slots 73% busy, the pipe of integer products and fp32 pairs 60%,
// the one of logic and comparisons 50%; of 6.9 warps a scheduler, 1.7 stand ready
// behind another, 1.6 wait out an instruction's latency, 1.1 for a pipe and 0.1 for
// memory. So the arithmetic bounds it, through no single pipe.

typedef unsigned long long AwPair;
__device__ __forceinline__ AwPair aw_pair(float lo, float hi) {
  AwPair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ AwPair aw_pair(float x) { return aw_pair(x, x); }
__device__ __forceinline__ AwPair aw_pair(float2 x) { return *reinterpret_cast<const AwPair*>(&x); }
__device__ __forceinline__ float2 aw_split(AwPair p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ AwPair aw_add2(AwPair a, AwPair b) {
  AwPair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ AwPair aw_mul2(AwPair a, AwPair b) {
  AwPair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ AwPair aw_fma2(AwPair a, AwPair b, AwPair c) {
  AwPair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// A product that is rounded by itself: the assembler joins mul.rn.f32x2 and a
// following add.rn.f32x2 into one operation (seen in the last bits of the
// states), but not a fused operation that adds a -0 it cannot see.
__device__ __forceinline__ AwPair aw_prod2(AwPair a, AwPair b, AwPair minus_zero) { return aw_fma2(a, b, minus_zero); }
// max(|a|, |b|, |c|), NaN if one is; min(|a|, |b|, |c|).
__device__ __forceinline__ float aw_max3(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float aw_min3(float a, float b, float c) {
  float r;
  asm("min.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float aw_rsqrt(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// sqrt(v) of a pair for v in [2^-100, 2^100]: with y about 1 / sqrt(v) and s = v y,
// the residual v - s^2 is exact in one fused operation and s + (residual) y / 2 is
// within 2^-20 of a unit in the last place before its rounding (P. Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor",
// 1990). That gives the nearest value but for the few mantissas whose root is as
// close to the middle of two (3.72775697 gives 1.93073797 for 1.93073809 unless y is
// the nearest value itself): far below the 20 bits that round it to a code.
__device__ __forceinline__ AwPair aw_sqrt2(AwPair v) {
  const float2 a = aw_split(v);
  const AwPair y = aw_pair(aw_rsqrt(a.x), aw_rsqrt(a.y));
  const AwPair s = aw_mul2(v, y);
  const AwPair e = aw_fma2(aw_mul2(s, aw_pair(-1.f)), s, v);
  return aw_fma2(e, aw_mul2(y, aw_pair(0.5f)), s);
}

__device__ __forceinline__ float aw_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The codes of eight m and sqrt(v) of the elements `idx` ^ 0..7 (element number
// and key). FAST: none is below 2^-6 of its scale, and none is zero.
template <bool FAST>
__device__ __forceinline__ void aw_codes(const AwPair (&m)[4], const AwPair (&u)[4], float mi, float vi, uint32_t idx,
                                         AwRaw<8>& mc, AwRaw<8>& vc) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 a = aw_split(aw_mul2(m[i], aw_pair(mi))), b = aw_split(aw_mul2(u[i], aw_pair(vi)));
    // aw_mix but for its last step, which leaves the upper half as it is.
    uint32_t h0 = idx ^ (2 * i), h1 = idx ^ (2 * i + 1);
    h0 = (h0 ^ (h0 >> 16)) * 0x7feb352du;
    h1 = (h1 ^ (h1 >> 16)) * 0x7feb352du;
    h0 = (h0 ^ (h0 >> 15)) * 0x846ca68bu;
    h1 = (h1 ^ (h1 >> 15)) * 0x846ca68bu;
    const uint32_t t0 = h0 >> 16, t1 = h1 >> 16;
    const uint32_t l0 = ((h0 ^ t0) & 0xFFFFu) * 16 + 8, l1 = ((h1 ^ t1) & 0xFFFFu) * 16 + 8;
    const uint32_t u0 = t0 * 16 + 8, u1 = t1 * 16 + 8;
    if (FAST) {
      a = make_float2(aw_round_fast(a.x, l0), aw_round_fast(a.y, l1));
      b = make_float2(aw_round_fast(b.x, u0), aw_round_fast(b.y, u1));
    } else {
      a = make_float2(aw_round(a.x, l0), aw_round(a.y, l1));
      b = make_float2(aw_round(b.x, u0), aw_round(b.y, u1));
    }
    mc.w[i >> 1] |= aw_encode2(a.x, a.y) << (16 * (i & 1));
    vc.w[i >> 1] |= aw_encode2(b.x, b.y) << (16 * (i & 1));
  }
}

// What the lanes of a CTA read of a chunk. Each thread copies and reads its own
// places only (cp.async), so stages need no barrier.
template <typename T, bool MASTER>
struct AwStage {
  static constexpr int kG = 8 * sizeof(T), kP = MASTER ? 32 : 8 * sizeof(T);
  uint4 g[kG / 16][kAwThreads];
  uint4 p[kP / 16][kAwThreads];
  uint2 m[kAwThreads], v[kAwThreads];
  float ms[kAwThreads], vs[kAwThreads];
};
template <int BYTES>
__device__ __forceinline__ void aw_copy(void* dst, const void* src) {
  const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(BYTES) : "memory");
}

template <typename T, bool MASTER, int N>
__global__ void __launch_bounds__(kAwThreads, kAwCtas8) adamw8_step(const __grid_constant__ AwTable<N> tab, const AwScalars c) {
  using Stage = AwStage<T, MASTER>;
  extern __shared__ __align__(16) uint8_t aw_smem[];
  Stage* stages = reinterpret_cast<Stage*>(aw_smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t off = threadIdx.x * 8;  // the lane's first element in a chunk
  const float gs = c.grad_scale ? *c.grad_scale : 1.f;
  // CTAs take chunks round robin, so that all work on neighbouring memory. The
  // copies run kAwStages - 1 chunks ahead, into the next tensor too.
  int ahead_ti = aw_tensor_of(tab, blockIdx.x);
  int ahead = blockIdx.x;
  auto copy = [&](int stage) {
    if (ahead < tab.chunks) {
      while (ahead_ti + 1 < tab.count && tab.t[ahead_ti + 1].chunk0 <= ahead) ++ahead_ti;
      const AwTensor& t = tab.t[ahead_ti];
      const int i = ahead - t.chunk0;
      if (i < t.whole) {
        Stage& d = stages[stage];
        const int64_t at = static_cast<int64_t>(i) * kAwChunk;
        const uint4* g = reinterpret_cast<const uint4*>(static_cast<const T*>(t.g) + at + off);
        const uint4* p = MASTER ? reinterpret_cast<const uint4*>(t.master + at + off)
                                : reinterpret_cast<const uint4*>(static_cast<const T*>(t.p) + at + off);
#pragma unroll
        for (int j = 0; j < Stage::kG / 16; ++j) aw_copy<16>(&d.g[j][threadIdx.x], g + j);
#pragma unroll
        for (int j = 0; j < Stage::kP / 16; ++j) aw_copy<16>(&d.p[j][threadIdx.x], p + j);
        aw_copy<8>(&d.m[threadIdx.x], static_cast<const uint8_t*>(t.m) + at + off);
        aw_copy<8>(&d.v[threadIdx.x], static_cast<const uint8_t*>(t.v) + at + off);
        aw_copy<4>(&d.ms[threadIdx.x], t.ms + at / kAwBlock + warp);
        aw_copy<4>(&d.vs[threadIdx.x], t.vs + at / kAwBlock + warp);
      }
    }
    ahead = min(ahead, tab.chunks) + gridDim.x;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kAwStages - 1; ++i) copy(i);
  int stage = 0, ti = aw_tensor_of(tab, blockIdx.x);
#pragma unroll 1
  for (int64_t chunk = blockIdx.x; chunk < tab.chunks; chunk += gridDim.x) {
    // The stage read last takes the chunk kAwStages - 1 ahead.
    copy(stage == 0 ? kAwStages - 1 : stage - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kAwStages - 1) : "memory");
    const Stage& in = stages[stage];
    stage = stage + 1 == kAwStages ? 0 : stage + 1;
    while (ti + 1 < tab.count && tab.t[ti + 1].chunk0 <= chunk) ++ti;
    const AwTensor& t = tab.t[ti];
    const int i = static_cast<int>(chunk) - t.chunk0;
    const int64_t at = static_cast<int64_t>(i) * kAwChunk;
    if (i >= t.whole) {
      if (at + warp * kAwBlock < t.n) aw_block<T, MASTER, true>(t, c, gs, at + warp * kAwBlock);
      continue;
    }
    const uint64_t e = static_cast<uint64_t>(t.block0) * kAwBlock + at;
    const uint32_t key = (e >> 32) == 0 ? c.key : aw_key(c.seed, c.step, static_cast<uint32_t>(e >> 32));
    const uint32_t idx = (static_cast<uint32_t>(e) + off) ^ key;
    const float ms0 = in.ms[threadIdx.x], vs0 = in.vs[threadIdx.x];
    uint4 graw[Stage::kG / 16], praw[Stage::kP / 16];
#pragma unroll
    for (int i = 0; i < Stage::kG / 16; ++i) graw[i] = in.g[i][threadIdx.x];
#pragma unroll
    for (int i = 0; i < Stage::kP / 16; ++i) praw[i] = in.p[i][threadIdx.x];
    const uint2 mq = in.m[threadIdx.x], vq = in.v[threadIdx.x];

    const AwPair mz = aw_pair(c.minus_zerop);
    AwPair m[4], v[4], u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = aw_decode2(((i < 2 ? mq.x : mq.y) >> (16 * (i & 1))) & 0xFFFFu);
      const float2 b = aw_decode2(((i < 2 ? vq.x : vq.y) >> (16 * (i & 1))) & 0xFFFFu);
      const T* gt = reinterpret_cast<const T*>(graw) + 2 * i;
      const AwPair g = aw_mul2(aw_pair(aw_to_f<T>(gt[0]), aw_to_f<T>(gt[1])), aw_pair(gs));
      const AwPair w = aw_mul2(aw_pair(b.x, b.y), aw_pair(vs0));
      m[i] = aw_add2(aw_prod2(aw_mul2(aw_pair(a.x, a.y), aw_pair(ms0)), aw_pair(c.b1p), mz),
                     aw_prod2(g, aw_pair(c.c1p), mz));
      v[i] = aw_add2(aw_prod2(aw_mul2(w, w), aw_pair(c.b2p), mz), aw_prod2(aw_mul2(g, g), aw_pair(c.c2p), mz));
    }
    float mmax = 0.f, vmax = 0.f, mmin = __int_as_float(0x7f800000), vmin = mmin;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = aw_split(m[i]), b = aw_split(v[i]);
      mmax = aw_max3(mmax, a.x, a.y);
      mmin = aw_min3(mmin, a.x, a.y);
      vmax = aw_max3(vmax, b.x, b.y);
      vmin = aw_min3(vmin, b.x, b.y);
    }
    // The block's maxima; a NaN's bits are above all others'.
    const uint32_t mtop = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(mmax) & 0x7FFFFFFFu);
    const uint32_t vtop = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(vmax) & 0x7FFFFFFFu);
    const bool plain = __all_sync(0xFFFFFFFFu, vmin >= 0x1p-100f && vmax <= 0x1p100f);
    if (plain) {
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = aw_sqrt2(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 b = aw_split(v[i]);
        u[i] = aw_pair(sqrtf(b.x), sqrtf(b.y));
      }
    }
    const float ms = aw_scale(mtop), vs = aw_scale(__float_as_uint(sqrtf(__uint_as_float(vtop))));
    const float mi = 1.f / ms, vi = 1.f / vs;
    // p = p decay - step_size m / (sqrt(v) inv_bc2 + eps)
    float pn[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 q = aw_split(aw_fma2(u[i], aw_pair(c.inv_bc2p), aw_pair(c.epsp)));
      const AwPair r = aw_pair(aw_rcp(q.x), aw_rcp(q.y));
      AwPair p0;
      if constexpr (MASTER) {
        const float* pt = reinterpret_cast<const float*>(praw) + 2 * i;
        p0 = aw_pair(pt[0], pt[1]);
      } else {
        const T* pt = reinterpret_cast<const T*>(praw) + 2 * i;
        p0 = aw_pair(aw_to_f<T>(pt[0]), aw_to_f<T>(pt[1]));
      }
      const float2 x = aw_split(aw_fma2(p0, aw_pair(c.decayp), aw_mul2(aw_mul2(m[i], r), aw_pair(c.minus_stepp))));
      pn[2 * i] = x.x;
      pn[2 * i + 1] = x.y;
    }
    if constexpr (MASTER) {
      AwRaw<32> o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o.w[i] = __float_as_uint(pn[i]);
      aw_st<32>(t.master + at + off, o);
    }
    AwRaw<8 * sizeof(T)> po;
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(&po)[i] = aw_from_f<T>(pn[i]);
    aw_st<8 * sizeof(T)>(static_cast<T*>(t.p) + at + off, po);
    // Codes. Values below 2^-6 (1 / 28672 of the block's maximum) and zeros are rare:
    // a block that has none takes the short rounding.
    AwRaw<8> mc{}, vc{};
    if (!__any_sync(0xFFFFFFFFu, mmin * mi < 0x1p-6f || sqrtf(vmin) * vi < 0x1p-6f))
      aw_codes<true>(m, u, mi, vi, idx, mc, vc);
    else
      aw_codes<false>(m, u, mi, vi, idx, mc, vc);
    aw_st<8>(static_cast<uint8_t*>(t.m) + at + off, mc);
    aw_st<8>(static_cast<uint8_t*>(t.v) + at + off, vc);
    if (lane == 0) {
      t.ms[at / kAwBlock + warp] = ms;
      t.vs[at / kAwBlock + warp] = vs;
    }
  }
}

}  // namespace avey
