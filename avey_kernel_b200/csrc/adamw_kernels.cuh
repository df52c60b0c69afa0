// One AdamW step over many tensors (avey_adamw_v1), with states in fp32 or in
// float8 blocks of 256.
//
// Every element is read once and written once, so the step is bound by HBM:
// 28 bytes an element for fp32 weights with fp32 states (or 16-bit weights
// with fp32 masters), 22 for 16-bit weights, 10 with 8-bit states.
//
// The tensors' pointers travel in the kernel's parameters (up to 400 tensors a
// launch), so a step is one launch, copies nothing to the device and keeps
// nothing between calls. Work is cut into chunks of 2048 elements of one tensor
// (8 warps, 256 elements each: a warp owns a block of the 8-bit states and
// finds its maximum with one reduction); CTAs take chunks round robin and
// find a chunk's tensor by bisection of the chunk prefix at first and by
// walking forward after.
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
  int64_t chunk0;  // first chunk of the launch
};

template <int N>
struct AwTable {
  int count;
  int64_t chunks;
  AwTensor t[N];
};

struct AwScalars {
  float b1, c1, b2, c2;  // beta, 1 - beta
  float decay;           // 1 - lr wd
  float step_size;       // lr / (1 - beta1^t)
  float inv_bc2;         // 1 / sqrt(1 - beta2^t)
  float eps;
  uint32_t seed;
  uint32_t step;
  const float* grad_scale;
};

__device__ __forceinline__ uint32_t aw_mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x7feb352du;
  x ^= x >> 15;
  x *= 0x846ca68bu;
  return x ^ (x >> 16);
}

__device__ __forceinline__ uint32_t aw_key(uint32_t seed, uint32_t step, uint32_t hi) {
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

template <typename T, bool MASTER, bool Q8, int N>
__global__ void __launch_bounds__(kAwThreads) adamw_step(const __grid_constant__ AwTable<N> tab, const AwScalars c) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t chunk = blockIdx.x;
  if (chunk >= tab.chunks) return;
  const float gs = c.grad_scale ? *c.grad_scale : 1.f;
  int ti = 0, hi = tab.count;  // the last tensor whose first chunk is at or before `chunk`
  while (hi - ti > 1) {
    const int mid = (ti + hi) >> 1;
    if (tab.t[mid].chunk0 <= chunk) ti = mid;
    else hi = mid;
  }
  for (; chunk < tab.chunks; chunk += gridDim.x) {
    while (ti + 1 < tab.count && tab.t[ti + 1].chunk0 <= chunk) ++ti;
    const AwTensor& t = tab.t[ti];
    const int64_t at0 = (chunk - t.chunk0) * kAwChunk + warp * kAwBlock;  // the warp's first element
    if (at0 >= t.n) continue;
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
    } else {
      aw_load8<float>(t.m, at, left, svec, m);
      aw_load8<float>(t.v, at, left, svec, v);
    }
    if constexpr (Q8) {
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
      float lowest = __int_as_float(0x7f800000);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        m[i] *= mi;
        root[i] *= vi;
        lowest = fminf(lowest, fminf(fabsf(m[i]), root[i]));
      }
      AwRaw<8> mo{}, vo{};
      // Values below 2^-6 (1 / 28672 of the block's maximum) are rare: a warp
      // that has none takes the short rounding.
      if (__any_sync(0xFFFFFFFFu, lowest < 0x1p-6f)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t h = aw_mix((idx + i) ^ key);
          m[i] = aw_round(m[i], ((h << 4) & 0xFFFF0u) | 8u);
          root[i] = aw_round(root[i], ((h >> 12) & 0xFFFF0u) | 8u);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t h = aw_mix((idx + i) ^ key);
          m[i] = aw_round_fast(m[i], ((h << 4) & 0xFFFF0u) | 8u);
          root[i] = aw_round_fast(root[i], ((h >> 12) & 0xFFFF0u) | 8u);
        }
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
}

}  // namespace avey
