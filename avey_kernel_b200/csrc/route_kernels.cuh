// Routing of tokens to experts (avey_route_*): the k best of each token's experts,
// their weights, and the gradient of the logits.
//
//   score  s = softmax(z) or sigmoid(z)
//   rank   z without a bias (its order is that of s), else s + bias; an expert whose
//          logit is -inf ranks below every other, one whose logit is NaN last
//   groups a group of experts ranks by the sum of its best one or two, and only the
//          experts of the best top_groups groups are chosen from; ties go to the lowest index
//   weight scale * s, or scale * s / (sum of s over the chosen)
//
// The renormalised weights are the softmax of log s over the chosen ones (log s = z up
// to a constant, or log sigmoid(z)), so they are right where s itself underflows. With
// all of the chosen at -inf the weights are zero.
//
// Scores in fp32 are off by some 10^-7 of themselves, and two experts may be closer than
// that. Where the order of two that matter is within the error, the token is done again
// in 64 bits, so the choice is the formula's. (Equal logits with equal biases are equal
// in any precision and need no second look.)
//
// Bound: the logits' bytes. A warp takes a token, a lane R consecutive experts in
// registers; a round of the choice is a maximum over the warp of 32-bit keys that are
// ordered like the ranks.
#pragma once

#include <math_constants.h>

#include "common.cuh"
#include "ptx.cuh"

namespace avey {

constexpr int kRtWarps = 8;
constexpr int kRtMaxExperts = 1024, kRtMaxK = 32, kRtMaxGroups = 32;

struct RtArgs {
  int64_t tokens;
  int experts, k, groups, top_groups, group_best;
  int softmax, renormalize;
  float scale;
  const void* logits;
  int64_t ld;
  int vec;            // rows of logits are read in whole 16 bytes (8 for two 32-bit or four 16-bit values)
  const float* bias;
  float* weights;     // forward: out
  int32_t* chosen;
  const float* dweights;
  void* dlogits;      // contiguous
  int dvec;
};

// A key in the order of the values; NaN below all (and above 0, which stands for "not there").
__device__ __forceinline__ uint32_t rt_key(float x) {
  if (x != x) return 1u;
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 as 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float rt_value(uint32_t key) {
  if (key <= 1u) return -CUDART_INF_F;
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// R consecutive logits of a row from e on; past the end: -inf.
template <typename T, int R>
__device__ __forceinline__ void rt_load(const T* row, int e, int experts, bool vec, float (&z)[R]) {
  constexpr int kBytes = R * sizeof(T) >= 16 ? 16 : R * sizeof(T), kPer = kBytes / sizeof(T);
  if (vec && kBytes >= 8 && e + R <= experts) {
#pragma unroll
    for (int i = 0; i < R; i += kPer) {
      T v[kPer];
      if constexpr (kBytes == 16) *reinterpret_cast<uint4*>(v) = __ldg(reinterpret_cast<const uint4*>(row + e + i));
      else if constexpr (kBytes == 8) *reinterpret_cast<uint2*>(v) = __ldg(reinterpret_cast<const uint2*>(row + e + i));
#pragma unroll
      for (int j = 0; j < kPer; ++j) z[i + j] = Elem<T>::to_f(v[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) z[i] = e + i < experts ? Elem<T>::load(row + e + i) : -CUDART_INF_F;
  }
}

template <typename S>
__device__ __forceinline__ S rt_exp(S x) {
  if constexpr (sizeof(S) == 8) return exp(x);
  else return expf(x);
}

// Scores of a lane's logits: the softmax needs the row's maximum and sum.
template <typename S, int R>
__device__ __forceinline__ void rt_scores(const float (&z)[R], bool softmax, S (&s)[R]) {
  if (softmax) {
    float top = z[0];
#pragma unroll
    for (int i = 1; i < R; ++i) top = fmaxf(top, z[i]);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    const S base = top == -CUDART_INF_F ? S(0) : S(top);
    S sum = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) sum += s[i] = rt_exp(S(z[i]) - base);
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    const S inv = sum > S(0) ? S(1) / sum : sum == S(0) ? S(0) : sum;  // no expert at all: zeros
#pragma unroll
    for (int i = 0; i < R; ++i) s[i] *= inv;
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) s[i] = S(1) / (S(1) + rt_exp(-S(z[i])));
  }
}

// The warp's best value and the lowest expert that has it; `there` marks what may be taken.
struct RtBest64 {
  double value;
  int expert;  // -1: none
};
template <int R>
__device__ __forceinline__ RtBest64 rt_best64(const double (&r)[R], uint32_t there, int e0) {
  RtBest64 b{-CUDART_INF, -1};
#pragma unroll
  for (int i = 0; i < R; ++i)
    if ((there >> i & 1u) && (b.expert < 0 || r[i] > b.value)) b = {r[i], e0 + i};
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const double v = __shfl_xor_sync(0xFFFFFFFFu, b.value, d);
    const int e = __shfl_xor_sync(0xFFFFFFFFu, b.expert, d);
    if (e >= 0 && (b.expert < 0 || v > b.value || (v == b.value && e < b.expert))) b = {v, e};
  }
  return b;
}

// Lane j's expert is the j-th chosen one. In 64 bits; of NaN and -inf ranks as the header says.
template <int R>
__device__ __noinline__ int rt_choose64(const RtArgs& q, const float (&z)[R], int lane) {
  const int e0 = lane * R;
  double r[R];
  if (q.bias || (q.groups > 1 && q.group_best == 2)) rt_scores<double, R>(z, q.softmax, r);
  double by[R];  // what groups rank by
  uint32_t there = 0, dead = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (e0 + i >= q.experts) continue;
    there |= 1u << i;
    if (q.bias) by[i] = r[i] += static_cast<double>(__ldg(q.bias + e0 + i));
    else if (q.groups > 1 && q.group_best == 2) by[i] = r[i], r[i] = z[i];
    else by[i] = r[i] = z[i];
    if (r[i] != r[i] || z[i] != z[i]) r[i] = by[i] = -CUDART_INF, dead |= 1u << i;
    else if (z[i] == -CUDART_INF_F) r[i] = by[i] = -CUDART_INF;
  }
  if (q.groups > 1) {
    const int size = q.experts / q.groups;
    double merit = -CUDART_INF;  // lane g: of group g
    for (int g = 0; g < q.groups; ++g) {
      uint32_t in = 0;
#pragma unroll
      for (int i = 0; i < R; ++i)
        if ((there >> i & 1u) && (e0 + i) / size == g) in |= 1u << i;
      const RtBest64 a = rt_best64<R>(by, in, e0);
      double m = a.value;
      if (q.group_best == 2 && a.value > -CUDART_INF) {
#pragma unroll
        for (int i = 0; i < R; ++i)
          if (e0 + i == a.expert) in &= ~(1u << i);
        const RtBest64 b = rt_best64<R>(by, in, e0);
        if (b.expert >= 0 && b.value > -CUDART_INF) m += b.value;
      }
      if (lane == g) merit = m;
    }
    uint32_t open = lane < q.groups, keep = 0;
    for (int n = 0; n < q.top_groups; ++n) {
      const double one[1] = {merit};
      const RtBest64 b = rt_best64<1>(one, open, lane);
      keep |= 1u << b.expert;
      if (lane == b.expert) open = 0;
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
      if ((there >> i & 1u) && !(keep >> ((e0 + i) / size) & 1u)) there &= ~(1u << i);
  }
  int mine = 0;
  for (int j = 0; j < q.k; ++j) {
    RtBest64 b = rt_best64<R>(r, there & ~dead, e0);
    if (b.expert < 0) b = rt_best64<R>(r, there, e0);  // only NaN are left
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (e0 + i == b.expert) there &= ~(1u << i);
    if (lane == j) mine = b.expert;
  }
  return mine;
}

// The warp's largest key, and the lowest expert that has it.
template <int R>
__device__ __forceinline__ uint32_t rt_best(const uint32_t (&key)[R], int e0, int& expert) {
  uint32_t top = key[0];
#pragma unroll
  for (int i = 1; i < R; ++i) top = max(top, key[i]);
  const uint32_t all = __reduce_max_sync(0xFFFFFFFFu, top);
  int at = 0;
#pragma unroll
  for (int i = R - 1; i >= 0; --i)
    if (key[i] == all) at = i;
  const int src = __ffs(__ballot_sync(0xFFFFFFFFu, top == all)) - 1;
  expert = __shfl_sync(0xFFFFFFFFu, e0 + at, src);
  return all;
}

// The same choice in 32 bits; false where two that matter are too near to tell.
template <int R>
__device__ __forceinline__ bool rt_choose(const RtArgs& q, const float (&z)[R], int lane, int& mine) {
  const int e0 = lane * R;
  const bool by_logit = !q.bias, sums = q.groups > 1 && q.group_best == 2;
  // Bounds of the errors of two ranks relative to their terms: the exponential and the
  // division (2^-22), the softmax's common sum of up to 32 + 5 additions (37 2^-24), the
  // addition of the bias (2^-24).
  const float tol = q.softmax ? 4e-6f : 1e-6f;
  uint32_t key[R];
  float s[R];
  if (!by_logit || sums) rt_scores<float, R>(z, q.softmax, s);
  bool sure = true;
  auto rank = [&](int i) {  // of this lane's i-th expert, where the choice is not by the logit
    const float r = q.bias ? s[i] + __ldg(q.bias + e0 + i) : s[i];
    return z[i] == -CUDART_INF_F ? -CUDART_INF_F : z[i] != z[i] ? z[i] : r;
  };
  if (sums || !by_logit) {
#pragma unroll
    for (int i = 0; i < R; ++i) key[i] = e0 + i < q.experts ? rt_key(rank(i)) : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) key[i] = e0 + i < q.experts ? rt_key(z[i]) : 0u;
  }
  if (q.groups > 1) {
    const int size = q.experts / q.groups;
    float merit = -CUDART_INF_F;  // lane g: of group g
    float bound = 0.f;            // of its terms' sizes
    for (int g = 0; g < q.groups; ++g) {
      uint32_t in[R];
#pragma unroll
      for (int i = 0; i < R; ++i) in[i] = (e0 + i) / size == g ? key[i] : 0u;
      int e;
      float m = rt_value(rt_best<R>(in, e0, e));
      float terms = fabsf(m) + (q.bias ? fabsf(__ldg(q.bias + e)) : 0.f);
      if (sums && m > -CUDART_INF_F) {
#pragma unroll
        for (int i = 0; i < R; ++i)
          if (e0 + i == e) in[i] = 0u;
        const float second = rt_value(rt_best<R>(in, e0, e));
        if (second > -CUDART_INF_F) {
          m += second;
          terms += fabsf(second) + (q.bias ? fabsf(__ldg(q.bias + e)) : 0.f);
        }
      }
      if (lane == g) {
        merit = m;
        bound = terms;
      }
    }
    const uint32_t one[1] = {lane < q.groups ? rt_key(merit) : 0u};
    uint32_t open[1] = {one[0]};
    uint32_t keep = 0;
    int last = 0;
    for (int n = 0; n < q.top_groups; ++n) {
      rt_best<1>(open, lane, last);
      keep |= 1u << last;
      if (lane == last) open[0] = 0u;
    }
    if (q.top_groups < q.groups && (sums || !by_logit)) {
      // The last group in and the first one out.
      int first = 0;
      const float out = rt_value(rt_best<1>(open, lane, first));
      const float in = __shfl_sync(0xFFFFFFFFu, merit, last);
      const float e = tol * (__shfl_sync(0xFFFFFFFFu, bound, last) + __shfl_sync(0xFFFFFFFFu, bound, first));
      sure = !(in - out <= e) || out == -CUDART_INF_F;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (by_logit && sums && key[i]) key[i] = rt_key(z[i]);
      if (!(keep >> ((e0 + i) / size) & 1u)) key[i] = 0u;
    }
  }
  // The chosen, and the next one, from the best on.
  uint32_t before = 0u;
  int before_e = 0;
  const int rounds = by_logit ? q.k : min(q.k + 1, q.top_groups * (q.experts / q.groups));
  for (int j = 0; j < rounds; ++j) {
    int e;
    const uint32_t top = rt_best<R>(key, e0, e);
    if (!by_logit && j > 0) {
      const float a = rt_value(before), b = rt_value(top);
      const float ba = __ldg(q.bias + before_e), bb = __ldg(q.bias + e);
      if (b > -CUDART_INF_F && a - b <= tol * (fabsf(a) + fabsf(b) + fabsf(ba) + fabsf(bb))) {
        // Too near, unless they are alike.
        float za = 0.f, zb = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
          if (e0 + i == before_e) za = z[i];
          if (e0 + i == e) zb = z[i];
        }
        za = __shfl_sync(0xFFFFFFFFu, za, before_e / R);
        zb = __shfl_sync(0xFFFFFFFFu, zb, e / R);
        sure = sure && za == zb && ba == bb;
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (e0 + i == e) key[i] = 0u;
    if (lane == j && j < q.k) mine = e;
    before = top;
    before_e = e;
  }
  return sure;
}

__device__ __forceinline__ float rt_log_sigmoid(float z) { return fminf(z, 0.f) - log1pf(expf(-fabsf(z))); }

__device__ __forceinline__ float rt_warp_sum(float x) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, d);
  return x;
}

// The chosen ones' weights without `scale`, a lane each (z: its logit; lanes from k on: 0).
__device__ __forceinline__ float rt_renormalized(float z, bool softmax, bool in) {
  const float l = !in ? -CUDART_INF_F : softmax ? z : rt_log_sigmoid(z);
  float top = l;
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
  const float e = top == -CUDART_INF_F && l == l ? 0.f : expf(l - top);
  const float sum = rt_warp_sum(e);
  return sum == 0.f ? 0.f : e / sum;
}

template <typename T, int R>
__global__ void __launch_bounds__(32 * kRtWarps) route_forward(const RtArgs q) {
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kRtWarps + (threadIdx.x >> 5);
  if (t >= q.tokens) return;
  const T* row = static_cast<const T*>(q.logits) + t * q.ld;
  float z[R];
  rt_load<T, R>(row, lane * R, q.experts, q.vec, z);
  int mine = 0;
  if (!rt_choose<R>(q, z, lane, mine)) mine = rt_choose64<R>(q, z, lane);
  const bool in = lane < q.k;
  const float mz = in ? Elem<T>::load(row + mine) : 0.f;
  float w;
  if (q.softmax) {
    // A NaN or +inf anywhere in the row makes the softmax NaN.
    float top = -CUDART_INF_F;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      top = fmaxf(top, z[i]);
      bad |= !(z[i] < CUDART_INF_F);
    }
    bad = __any_sync(0xFFFFFFFFu, bad);
    if (q.renormalize) {
      w = rt_renormalized(mz, true, in);
    } else {
#pragma unroll
      for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
      const float base = top == -CUDART_INF_F ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < R; ++i) sum += expf(z[i] - base);
      sum = rt_warp_sum(sum);
      w = sum == 0.f ? 0.f : expf(mz - base) / sum;
    }
    if (bad) w = CUDART_NAN_F;
  } else {
    w = q.renormalize ? rt_renormalized(mz, false, in) : 1.f / (1.f + expf(-mz));
  }
  if (in) {
    q.weights[t * q.k + lane] = w * q.scale;
    q.chosen[t * q.k + lane] = mine;
  }
}

// dlogits: for the softmax over all experts every logit has a gradient, p_e (h_e - sum h p)
// with h the gradient at the chosen ones' scores; else only the chosen ones have.
template <typename T, int R>
__global__ void __launch_bounds__(32 * kRtWarps) route_backward(const RtArgs q) {
  extern __shared__ float rows[];  // [warps][32 R]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kRtWarps + warp;
  if (t >= q.tokens) return;
  float* d = rows + warp * 32 * R;
  const T* row = static_cast<const T*>(q.logits) + t * q.ld;
  const bool in = lane < q.k, full = q.softmax && !q.renormalize;
  const int e = in ? min(max(__ldg(q.chosen + t * q.k + lane), 0), q.experts - 1) : 0;
  const float mz = in ? Elem<T>::load(row + e) : 0.f;
  const float g = in ? __ldg(q.dweights + t * q.k + lane) * q.scale : 0.f;
  const int e0 = lane * R;
#pragma unroll
  for (int i = 0; i < R; ++i) d[e0 + i] = 0.f;
  __syncwarp();
  if (!full) {
    float v;
    if (q.renormalize) {
      const float w = rt_renormalized(mz, q.softmax, in);
      v = w * (g - rt_warp_sum(in ? w * g : 0.f));
      if (!q.softmax) v *= 1.f / (1.f + expf(mz));  // 1 - s
      // A softmax over a row with a NaN or +inf was NaN.
      if (q.softmax && !(__ldg(q.weights + t * q.k) == __ldg(q.weights + t * q.k))) v = CUDART_NAN_F;
    } else {
      v = g / (1.f + expf(-mz)) / (1.f + expf(mz));
      if (mz == -CUDART_INF_F) v = 0.f;
    }
    if (in) d[e] = v;
    __syncwarp();
  } else {
    if (in) d[e] = g;
    __syncwarp();
    float z[R], s[R];
    rt_load<T, R>(row, e0, q.experts, q.vec, z);
    rt_scores<float, R>(z, true, s);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) dot += s[i] * d[e0 + i];
    dot = rt_warp_sum(dot);
#pragma unroll
    for (int i = 0; i < R; ++i) d[e0 + i] = s[i] * (d[e0 + i] - dot);
    __syncwarp();
  }
  T* out = static_cast<T*>(q.dlogits) + t * q.experts;
  constexpr int kPer = 16 / sizeof(T);
  if (q.dvec) {
    for (int i = lane * kPer; i < q.experts; i += 32 * kPer) {
      T v[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[j] = Elem<T>::from_f(d[i + j]);
      *reinterpret_cast<uint4*>(out + i) = *reinterpret_cast<const uint4*>(v);
    }
  } else {
    for (int i = lane; i < q.experts; i += 32) out[i] = Elem<T>::from_f(d[i]);
  }
}

}  // namespace avey
