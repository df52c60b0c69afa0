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
// that. Where the order of two that matter is within the error, a second look in 64 bits
// decides, so the choice is the formula's: at the chosen experts and the next one alone, a lane
// each, where no other is as near; else, and for groups, at all. (Equal logits with equal biases
// are equal in any precision and need none.) A few tokens of thousands need one, but the
// launch waits for them: with all ranks looked at again for each, 4093 tokens of 256 experts in 8
// groups took 20 us instead of 12.7 (and 11.8 without any such token).
//
// Bound: the logits' bytes, or instructions. Without a bias and groups (route_plain) and
// in the gradient a token takes as many lanes as give each 16 of its experts, so that a
// warp's shuffles serve several tokens: 65536 tokens of 128 experts, the best 4, 25 us
// forward and 18 backward from cold caches, where a warp for each token took 39 and 23. With them a warp
// takes a token; few tokens leave it latency-bound, many its instructions (65536 of 256 experts
// in 8 groups: 127 us; some 15% more with two blocks an SM for R = 8 instead of three).
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

// Scores of a lane's logits: the softmax needs the row's maximum and sum.
template <int R>
__device__ __forceinline__ void rt_scores(const float (&z)[R], bool softmax, float (&s)[R]) {
  if (softmax) {
    float top = z[0];
#pragma unroll
    for (int i = 1; i < R; ++i) top = fmaxf(top, z[i]);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    const float base = top == -CUDART_INF_F ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) sum += s[i] = expf(z[i] - base);
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;  // no expert at all: zeros
#pragma unroll
    for (int i = 0; i < R; ++i) s[i] *= inv;
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) s[i] = __fdividef(1.f, 1.f + expf(-z[i]));  // 0 below 2^-126
  }
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

// A warp's keys from the best on, ties by the lowest expert. Up to eight a lane are sorted
// first, so that a round compares one key of each lane (a round over eight unsorted ones
// takes 70 instructions, a sorted one 30 after 140 for the sort).
template <int R>
struct RtPool {
  static constexpr bool kSorted = R <= 8;
  uint32_t key[R];
  int index[R];

  __device__ __forceinline__ void fill(const uint32_t (&k)[R], int e0) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      key[i] = k[i];
      index[i] = e0 + i;
    }
    if constexpr (kSorted) {
      // Neighbours change places only for a larger key, so equal ones keep their order.
#pragma unroll
      for (int n = R - 1; n > 0; --n)
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const bool swap = key[i + 1] > key[i];
          const uint32_t hi = swap ? key[i + 1] : key[i], lo = swap ? key[i] : key[i + 1];
          const int hi_e = swap ? index[i + 1] : index[i], lo_e = swap ? index[i] : index[i + 1];
          key[i] = hi;
          key[i + 1] = lo;
          index[i] = hi_e;
          index[i + 1] = lo_e;
        }
    }
  }
  __device__ __forceinline__ uint32_t next(int lane, int& expert) {
    if constexpr (kSorted) {
      const uint32_t all = __reduce_max_sync(0xFFFFFFFFu, key[0]);
      const int src = __ffs(__ballot_sync(0xFFFFFFFFu, key[0] == all)) - 1;
      expert = __shfl_sync(0xFFFFFFFFu, index[0], src);
      if (lane == src) {
#pragma unroll
        for (int i = 0; i + 1 < R; ++i) {
          key[i] = key[i + 1];
          index[i] = index[i + 1];
        }
        key[R - 1] = 0u;
      }
      return all;
    } else {
      const uint32_t all = rt_best<R>(key, index[0], expert);
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (index[0] + i == expert) key[i] = 0u;
      return all;
    }
  }
};

// The same for 64-bit keys, which order doubles: NaN at 1, 0 stands for "not there".
__device__ __forceinline__ unsigned long long rt_key64(double x) {
  if (x != x) return 1ull;
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(x + 0.0));
  return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double rt_value64(unsigned long long key) {
  if (key <= 1ull) return -CUDART_INF;
  return __longlong_as_double(static_cast<long long>(key >> 63 ? key ^ (1ull << 63) : ~key));
}
template <int R>
__device__ __forceinline__ unsigned long long rt_best64(const unsigned long long (&key)[R], int e0, int& expert) {
  unsigned long long top = key[0];
#pragma unroll
  for (int i = 1; i < R; ++i) top = max(top, key[i]);
  const uint32_t hi = __reduce_max_sync(0xFFFFFFFFu, static_cast<uint32_t>(top >> 32));
  const uint32_t lo = __reduce_max_sync(0xFFFFFFFFu, top >> 32 == hi ? static_cast<uint32_t>(top) : 0u);
  const unsigned long long all = static_cast<unsigned long long>(hi) << 32 | lo;
  int at = 0;
#pragma unroll
  for (int i = R - 1; i >= 0; --i)
    if (key[i] == all) at = i;
  const int src = __ffs(__ballot_sync(0xFFFFFFFFu, top == all)) - 1;
  expert = __shfl_sync(0xFFFFFFFFu, e0 + at, src);
  return all;
}

// Which groups are chosen from: lane g has group g's merit. A group's place is the number
// of better ones (and of those as good before it). `in`, `out`: the last one kept and the
// first one not.
template <typename S>
__device__ __forceinline__ uint32_t rt_keep(const RtArgs& q, S merit, int lane, int& in, int& out) {
  int place = 0;
  for (int g = 0; g < q.groups; ++g) {
    const S other = __shfl_sync(0xFFFFFFFFu, merit, g);
    place += other > merit || (other == merit && g < lane);
  }
  const bool there = lane < q.groups;
  in = __ffs(__ballot_sync(0xFFFFFFFFu, there && place == q.top_groups - 1)) - 1;
  out = __ffs(__ballot_sync(0xFFFFFFFFu, there && place == q.top_groups)) - 1;
  return __ballot_sync(0xFFFFFFFFu, there && place < q.top_groups);
}

// The second looks, in 64 bits. They read the logits again: given them, they would have them kept
// in local memory by every token.
//
// The softmax's maximum and sum.
struct RtSoft {
  double base, inv;
};
template <typename T, int R>
__device__ __forceinline__ RtSoft rt_soft64(const RtArgs& q, const T* row, int lane) {
  if (!q.softmax) return {0.0, 1.0};
  float z[R];
  rt_load<T, R>(row, lane * R, q.experts, q.vec, z);
  float top = z[0];
#pragma unroll
  for (int i = 1; i < R; ++i) top = fmaxf(top, z[i]);
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
  const double base = top == -CUDART_INF_F ? 0.0 : top;
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < R; ++i) sum += exp(z[i] - base);
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
  return {base, sum > 0.0 ? 1.0 / sum : sum == 0.0 ? 0.0 : sum};
}
// An expert's rank, as a key.
__device__ __forceinline__ unsigned long long rt_rank64(const RtArgs& q, const RtSoft& soft, float z, int expert) {
  const double e = exp(q.softmax ? z - soft.base : -static_cast<double>(z));
  double rank = q.softmax ? e * soft.inv : 1.0 / (1.0 + e);
  if (q.bias) rank += static_cast<double>(__ldg(q.bias + expert));
  return z == -CUDART_INF_F ? rt_key64(-CUDART_INF) : z != z ? 1ull : rt_key64(rank);
}

// The groups to choose from. A group takes as many lanes, a power of two, as there are for each.
template <typename T, int R>
__device__ __noinline__ uint32_t rt_keep64(const RtArgs& q, int64_t t, int lane) {
  const T* row = static_cast<const T*>(q.logits) + t * q.ld;
  const RtSoft soft = rt_soft64<T, R>(q, row, lane);
  int lanes = 32;
  while (lanes * q.groups > 32) lanes >>= 1;
  const int size = q.experts / q.groups, group = lane / lanes, end = group < q.groups ? (group + 1) * size : 0;
  unsigned long long first = 0ull, second = 0ull;
#pragma unroll 4
  for (int e = group * size + lane % lanes; e < end; e += lanes) {
    const unsigned long long v = rt_rank64(q, soft, Elem<T>::load(row + e), e);
    second = max(second, min(first, v));
    first = max(first, v);
  }
  for (int d = lanes >> 1; d; d >>= 1) {
    const unsigned long long f = __shfl_xor_sync(0xFFFFFFFFu, first, d), s = __shfl_xor_sync(0xFFFFFFFFu, second, d);
    second = max(min(first, f), max(second, s));
    first = max(first, f);
  }
  const int src = min(lane * lanes, 31);
  const double best = rt_value64(__shfl_sync(0xFFFFFFFFu, first, src));
  const double next = rt_value64(__shfl_sync(0xFFFFFFFFu, second, src));
  int in, out;
  return rt_keep(q, q.group_best == 2 && next > -CUDART_INF ? best + next : best, lane, in, out);
}

// Lane j's expert is the j-th chosen one, of the groups in `keep`.
template <typename T, int R>
__device__ __noinline__ int rt_choose64(const RtArgs& q, int64_t t, int lane, uint32_t keep) {
  const int e0 = lane * R, size = q.experts / q.groups;
  const T* row = static_cast<const T*>(q.logits) + t * q.ld;
  const RtSoft soft = rt_soft64<T, R>(q, row, lane);
  float z[R];
  rt_load<T, R>(row, e0, q.experts, q.vec, z);
  unsigned long long key[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const bool there = e0 + i < q.experts && (keep >> min((e0 + i) / size, 31) & 1u);
    key[i] = there ? rt_rank64(q, soft, z[i], e0 + i) : 0ull;
  }
  int mine = 0;
  for (int j = 0; j < q.k; ++j) {
    int e;
    rt_best64<R>(key, e0, e);
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (e0 + i == e) key[i] = 0ull;
    if (lane == j) mine = e;
  }
  return mine;
}

// The order of the experts that lanes 0 to n - 1 hold, a score each.
template <typename T, int R>
__device__ __noinline__ int rt_order64(const RtArgs& q, int64_t t, int lane, int n, int expert) {
  const T* row = static_cast<const T*>(q.logits) + t * q.ld;
  const RtSoft soft = rt_soft64<T, R>(q, row, lane);
  const unsigned long long key = lane < n ? rt_rank64(q, soft, Elem<T>::load(row + expert), expert) : 0ull;
  int place = 0;
  for (int i = 0; i < n; ++i) {
    const unsigned long long other = __shfl_sync(0xFFFFFFFFu, key, i);
    const int other_e = __shfl_sync(0xFFFFFFFFu, expert, i);
    place += other > key || (other == key && other_e < expert);
  }
  int mine = 0;
  for (int i = 0; i < n; ++i) {
    const int e = __shfl_sync(0xFFFFFFFFu, expert, i);
    if (__shfl_sync(0xFFFFFFFFu, place, i) == lane) mine = e;
  }
  return mine;
}

// The choice: lane j's expert is the j-th chosen one, and mz its logit. `most`: the largest |bias|.
template <typename T, int R>
__device__ __forceinline__ void rt_choose(const RtArgs& q, int64_t t, const float (&z)[R], float most, int lane,
                                          int& mine, float& mz) {
  const T* row = static_cast<const T*>(q.logits) + t * q.ld;
  const int e0 = lane * R;
  uint32_t keep = 0xFFFFFFFFu;
  const bool by_logit = !q.bias, sums = q.groups > 1 && q.group_best == 2;
  // Bounds of the errors of two ranks relative to their terms: the exponential and the
  // division (2^-21), the softmax's common sum of up to 32 + 5 additions (37 2^-24) and
  // the difference to its maximum (2^-18, half a step below 128; a score further down is 0), the
  // addition of the bias (2^-24). And in all: scores below 2^-126 have fewer digits, or are 0.
  const float tol = q.softmax ? 7e-6f : 1e-6f, least = 0x1p-120f;
  float r[R];
  uint32_t key[R];
  if (by_logit && !sums) {
#pragma unroll
    for (int i = 0; i < R; ++i) r[i] = z[i];
  } else {
    rt_scores<R>(z, q.softmax, r);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (q.bias && e0 + i < q.experts) r[i] += __ldg(q.bias + e0 + i);
      if (z[i] == -CUDART_INF_F) r[i] = -CUDART_INF_F;
      if (z[i] != z[i]) r[i] = z[i];
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) key[i] = e0 + i < q.experts ? rt_key(by_logit ? z[i] : r[i]) : 0u;
  if (q.groups > 1) {
    const int size = q.experts / q.groups, span = size / R;
    const bool lanes = size % R == 0 && (span & (span - 1)) == 0;
    float first = -CUDART_INF_F, second = -CUDART_INF_F;  // lane g: of group g
    if (lanes) {
      // A group is `span` whole lanes, a power of two: all groups at once (and none has
      // lanes past the experts; a NaN counts as -inf).
      float a = -CUDART_INF_F, b = -CUDART_INF_F;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float v = e0 + i < q.experts ? fmaxf(r[i], -CUDART_INF_F) : -CUDART_INF_F;
        b = fmaxf(b, fminf(a, v));
        a = fmaxf(a, v);
      }
      for (int d = 1; d < span; d <<= 1) {
        const float a2 = __shfl_xor_sync(0xFFFFFFFFu, a, d), b2 = __shfl_xor_sync(0xFFFFFFFFu, b, d);
        b = fmaxf(fminf(a, a2), fmaxf(b, b2));
        a = fmaxf(a, a2);
      }
      const int src = min(lane * span, 31);
      first = __shfl_sync(0xFFFFFFFFu, a, src);
      second = __shfl_sync(0xFFFFFFFFu, b, src);
    } else {
      for (int g = 0; g < q.groups; ++g) {
        uint32_t in[R];
#pragma unroll
        for (int i = 0; i < R; ++i)
          in[i] = e0 + i >= g * size && e0 + i < (g + 1) * size ? rt_key(r[i]) : 0u;
        int e;
        const float a = rt_value(rt_best<R>(in, e0, e));
#pragma unroll
        for (int i = 0; i < R; ++i)
          if (e0 + i == e) in[i] = 0u;
        const float b = rt_value(rt_best<R>(in, e0, e));
        if (lane == g) {
          first = a;
          second = b;
        }
      }
    }
    const bool two = q.group_best == 2 && second > -CUDART_INF_F;
    const float merit = two ? first + second : first;
    int in, out;
    keep = rt_keep(q, merit, lane, in, out);
    if (q.top_groups < q.groups && !(by_logit && !sums)) {
      const float terms = fabsf(first) + (two ? fabsf(second) : 0.f) + 2.f * most;
      const float bound = tol * (__shfl_sync(0xFFFFFFFFu, terms, in) + __shfl_sync(0xFFFFFFFFu, terms, out)) + least;
      const float m_in = __shfl_sync(0xFFFFFFFFu, merit, in), m_out = __shfl_sync(0xFFFFFFFFu, merit, out);
      if (m_out > -CUDART_INF_F && m_in - m_out <= bound) keep = rt_keep64<T, R>(q, t, lane);
    }
    if (lanes) {
      if (!(keep >> min(lane / span, 31) & 1u)) {
#pragma unroll
        for (int i = 0; i < R; ++i) key[i] = 0u;
      }
    } else {
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (!(keep >> min((e0 + i) / size, 31) & 1u)) key[i] = 0u;
    }
  }
  // The chosen, and with a bias the next one, from the best on.
  RtPool<R> pool;
  pool.fill(key, e0);
  const int rounds = by_logit ? q.k : min(q.k + 1, q.top_groups * (q.experts / q.groups));
  uint32_t mine_key = 0u;
  float before = 0.f;
  int before_e = 0;
  // Near: two ranks whose order their errors may change. Alike: of equal logits and biases.
  auto near = [&](float a, float b) {
    return b > -CUDART_INF_F && a - b <= tol * (fabsf(a) + fabsf(b) + 2.f * most) + least;
  };
  auto alike = [&](int a, int b) {
    return Elem<T>::load(row + a) == Elem<T>::load(row + b) && __ldg(q.bias + a) == __ldg(q.bias + b);
  };
  bool order = false, last = false;  // near and not alike: any two, the last two
  for (int j = 0; j < rounds; ++j) {
    int e;
    const uint32_t top = pool.next(lane, e);
    if (!by_logit) {
      const float v = rt_value(top);
      last = j > 0 && near(before, v);
      order = order || (last && !alike(before_e, e));
      before = v;
      before_e = e;
    }
    if (lane == j) {
      mine = e;
      mine_key = top;
    }
  }
  if (!by_logit) {
    // Where the last one is near the one before it, others that are left may be too.
    bool full = false;
    if (last) {
      bool more = false;
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (near(before, rt_value(pool.key[i]))) more = more || order || !alike(before_e, pool.index[i]);
      full = __any_sync(0xFFFFFFFFu, more) || (order && rounds > 32);
    }
    if (full) mine = rt_choose64<T, R>(q, t, lane, keep);
    else if (order) mine = rt_order64<T, R>(q, t, lane, min(rounds, 32), mine);
  }
  if (lane < q.k) mz = by_logit ? (mine_key == 1u ? CUDART_NAN_F : rt_value(mine_key)) : Elem<T>::load(row + mine);
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
  return sum == 0.f ? 0.f : __fdividef(e, sum);  // a sum of up to 32 terms, of at most 1 each
}

// Lanes [first, first + lanes) of a warp take a token.
struct RtPart {
  int64_t t;
  int lane, first;
  unsigned mask;  // its lanes
};
__device__ __forceinline__ RtPart rt_part(int lanes) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 32 * kRtWarps + threadIdx.x;
  const int lane = static_cast<int>(threadIdx.x) & (lanes - 1), first = (threadIdx.x & 31) - lane;
  return {i / lanes, lane, first, (lanes == 32 ? 0xFFFFFFFFu : (1u << lanes) - 1) << first};
}
__device__ __forceinline__ float rt_part_sum(float x, int lanes) {
  for (int d = lanes >> 1; d; d >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, d);
  return x;
}

// Experts by their logits: no score decides, so 32 bits are exact. (lanes >= k: lane j has the
// j-th chosen one.)
template <typename T, int R>
__global__ void __launch_bounds__(32 * kRtWarps) route_plain(const __grid_constant__ RtArgs q, int lanes) {
  griddep_wait();
  const RtPart p = rt_part(lanes);
  const bool there = p.t < q.tokens;
  const int64_t t = there ? p.t : q.tokens - 1;  // (a part past the end goes along)
  const int e0 = p.lane * R;
  float z[R];
  rt_load<T, R>(static_cast<const T*>(q.logits) + t * q.ld, e0, q.experts, q.vec, z);
  uint32_t key[R];
#pragma unroll
  for (int i = 0; i < R; ++i) key[i] = e0 + i < q.experts ? rt_key(z[i]) : 0u;
  int mine = 0;
  uint32_t mine_key = 0u, best = 0u;
  for (int j = 0; j < q.k; ++j) {
    uint32_t top = key[0];
    int e = e0;
#pragma unroll
    for (int i = 1; i < R; ++i)
      if (key[i] > top) {
        top = key[i];
        e = e0 + i;
      }
    for (int d = lanes >> 1; d; d >>= 1) {
      const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, top, d);
      const int other_e = __shfl_xor_sync(0xFFFFFFFFu, e, d);
      if (other > top || (other == top && other_e < e)) {
        top = other;
        e = other_e;
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (e0 + i == e) key[i] = 0u;
    if (j == 0) best = top;
    if (p.lane == j) {
      mine = e;
      mine_key = top;
    }
  }
  const bool in = p.lane < q.k;
  const float mz = mine_key == 1u ? CUDART_NAN_F : rt_value(mine_key), top = rt_value(best);
  float w;
  if (q.softmax) {
    const float base = top == -CUDART_INF_F ? 0.f : top;
    float sum = 0.f;
    bool bad = false;  // a NaN or +inf anywhere in the row makes the softmax NaN
    if (q.renormalize) {
      sum = in ? expf(mz - base) : 0.f;
#pragma unroll
      for (int i = 0; i < R; ++i) bad |= !(z[i] < CUDART_INF_F);
      bad = (__ballot_sync(0xFFFFFFFFu, bad) & p.mask) != 0u;
    } else {
#pragma unroll
      for (int i = 0; i < R; ++i) sum += expf(z[i] - base);
    }
    sum = rt_part_sum(sum, lanes);
    w = sum == 0.f ? 0.f : __fdividef(expf(mz - base), sum);
    if (bad) w = CUDART_NAN_F;
  } else if (q.renormalize) {
    // The logarithms of the scores are in the logits' order: the first is the largest.
    const float l = in ? rt_log_sigmoid(mz) : -CUDART_INF_F;
    const float most = __shfl_sync(0xFFFFFFFFu, l, p.first);
    const float e = most == -CUDART_INF_F && l == l ? 0.f : expf(l - most);
    const float sum = rt_part_sum(e, lanes);
    w = sum == 0.f ? 0.f : __fdividef(e, sum);
  } else {
    w = 1.f / (1.f + expf(-mz));
  }
  if (there && in) {
    q.weights[t * q.k + p.lane] = w * q.scale;
    q.chosen[t * q.k + p.lane] = mine;
  }
}

template <typename T, int R>
__global__ void __launch_bounds__(32 * kRtWarps, R <= 4 ? 4 : R <= 8 ? 3 : 1)
    route_forward(const __grid_constant__ RtArgs q) {
  griddep_wait();
  const int lane = threadIdx.x & 31, e0 = lane * R;
  float most = 0.f;  // the largest |bias|
  if (q.bias) {
    for (int e = lane; e < q.experts; e += 32) most = fmaxf(most, fabsf(__ldg(q.bias + e)));
#pragma unroll
    for (int d = 16; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
  }
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRtWarps;
  int64_t t = static_cast<int64_t>(blockIdx.x) * kRtWarps + (threadIdx.x >> 5);
  float next[R];
  if (t < q.tokens) rt_load<T, R>(static_cast<const T*>(q.logits) + t * q.ld, e0, q.experts, q.vec, next);
  for (; t < q.tokens; t += step) {
    float z[R];
#pragma unroll
    for (int i = 0; i < R; ++i) z[i] = next[i];
    if (t + step < q.tokens)  // the next token's logits are under way meanwhile
      rt_load<T, R>(static_cast<const T*>(q.logits) + (t + step) * q.ld, e0, q.experts, q.vec, next);
    int mine = 0;
    float mz = 0.f;
    rt_choose<T, R>(q, t, z, most, lane, mine, mz);
    const bool in = lane < q.k;
    float w;
    if (q.softmax && !q.renormalize) {
      float top = z[0];
#pragma unroll
      for (int i = 1; i < R; ++i) top = fmaxf(top, z[i]);
      top = rt_value(__reduce_max_sync(0xFFFFFFFFu, rt_key(top)));
      const float base = top == -CUDART_INF_F ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < R; ++i) sum += expf(z[i] - base);
      sum = rt_warp_sum(sum);  // NaN where a logit is NaN or +inf
      w = sum == 0.f ? 0.f : __fdividef(expf(mz - base), sum);
    } else if (q.softmax) {
      // A NaN or +inf anywhere in the row makes the softmax NaN.
      bool bad = false;
#pragma unroll
      for (int i = 0; i < R; ++i) bad |= !(z[i] < CUDART_INF_F);
      w = rt_renormalized(mz, true, in);
      if (__any_sync(0xFFFFFFFFu, bad)) w = CUDART_NAN_F;
    } else {
      w = q.renormalize ? rt_renormalized(mz, false, in) : 1.f / (1.f + expf(-mz));
    }
    if (in) {
      q.weights[t * q.k + lane] = w * q.scale;
      q.chosen[t * q.k + lane] = mine;
    }
  }
}

// dlogits: for the softmax over all experts every logit has a gradient, p_e (h_e - sum h p)
// with h the gradient at the chosen ones' scores; else only the chosen ones have. (lanes >= k.)
template <typename T, int R>
__global__ void __launch_bounds__(32 * kRtWarps) route_backward(const __grid_constant__ RtArgs q, int lanes) {
  extern __shared__ float rows[];  // R values a thread and one of room, against bank conflicts
  griddep_wait();
  const RtPart p = rt_part(lanes);
  const bool there = p.t < q.tokens;
  const int64_t t = there ? p.t : q.tokens - 1;  // (a part past the end goes along)
  float* d = rows + (threadIdx.x - p.lane) * (R + 1);
  auto at = [](int expert) { return expert + expert / R; };  // a lane's: from e0 + lane on
  const T* row = static_cast<const T*>(q.logits) + t * q.ld;
  const bool in = p.lane < q.k, full = q.softmax && !q.renormalize;
  const int e = in ? min(max(__ldg(q.chosen + t * q.k + p.lane), 0), q.experts - 1) : 0;
  const float g = in ? __ldg(q.dweights + t * q.k + p.lane) * q.scale : 0.f;
  const int e0 = p.lane * R, d0 = p.lane * (R + 1);
#pragma unroll
  for (int i = 0; i < R; ++i) d[d0 + i] = 0.f;
  __syncwarp();
  if (!full) {
    const float mz = in ? Elem<T>::load(row + e) : 0.f;
    float v;
    if (q.renormalize) {
      const float l = !in ? -CUDART_INF_F : q.softmax ? mz : rt_log_sigmoid(mz);
      float top = l;
      for (int s = lanes >> 1; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
      const float x = top == -CUDART_INF_F && l == l ? 0.f : expf(l - top);
      const float sum = rt_part_sum(x, lanes), w = sum == 0.f ? 0.f : __fdividef(x, sum);
      v = w * (g - rt_part_sum(in ? w * g : 0.f, lanes));
      if (!q.softmax) v *= 1.f / (1.f + expf(mz));  // 1 - s
      // A softmax over a row with a NaN or +inf was NaN.
      const float first = __ldg(q.weights + t * q.k);
      if (q.softmax && first != first) v = CUDART_NAN_F;
    } else {
      v = g / (1.f + expf(-mz)) / (1.f + expf(mz));
      if (mz == -CUDART_INF_F) v = 0.f;
    }
    if (in) d[at(e)] = v;
  } else {
    if (in) d[at(e)] = g;
    __syncwarp();
    float z[R];
    rt_load<T, R>(row, e0, q.experts, q.vec, z);
    float top = z[0];
#pragma unroll
    for (int i = 1; i < R; ++i) top = fmaxf(top, z[i]);
    for (int s = lanes >> 1; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
    const float base = top == -CUDART_INF_F ? 0.f : top;
    float sum = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      z[i] = expf(z[i] - base);
      sum += z[i];
      dot = fmaf(z[i], d[d0 + i], dot);
    }
    sum = rt_part_sum(sum, lanes);  // NaN where a logit is NaN or +inf
    dot = rt_part_sum(dot, lanes);
    const float inv = sum == 0.f ? 0.f : __fdividef(1.f, sum);
    dot *= inv;
#pragma unroll
    for (int i = 0; i < R; ++i) d[d0 + i] = z[i] * inv * (d[d0 + i] - dot);
  }
  __syncwarp();
  if (!there) return;
  T* out = static_cast<T*>(q.dlogits) + t * q.experts;
  constexpr int kPer = 16 / sizeof(T);
  if (q.dvec) {
    for (int i = p.lane * kPer; i < q.experts; i += lanes * kPer) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
          w[j] = __float_as_uint(d[at(i + j)]);
        } else {
          const T lo = Elem<T>::from_f(d[at(i + 2 * j)]), hi = Elem<T>::from_f(d[at(i + 2 * j + 1)]);
          w[j] = *reinterpret_cast<const uint16_t*>(&lo) |
                 static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&hi)) << 16;
        }
      }
      *reinterpret_cast<uint4*>(out + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
    for (int i = p.lane; i < q.experts; i += lanes) out[i] = Elem<T>::from_f(d[at(i)]);
  }
}

}  // namespace avey
