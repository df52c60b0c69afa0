// Rows moved between tokens and the places that they are worked on or kept at:
//
//   dispatch   rows[slot_tj] = x_t                      (and the scaled form: the gradient
//                                                        of combine's rows, w_tj dout_t)
//   combine    out_t = residual_t + sum_j w_tj rows[slot_tj]   (w = 1: dispatch's gradient)
//   embedding  out_i = scale table[token_i]
//   and the embedding's gradient by sorted tokens.
//
// Bound: the rows' bytes, each read and written once; a thread moves 16 bytes of a row
// (less where rows are not whole 16-byte units), with all k rows of a token under way
// together. Sums are fp32, in the order of the choices, or of the tokens.
#pragma once

#include <math_constants.h>

#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"

namespace avey {

// N values of type T as one access.
template <typename T, int N>
struct alignas(sizeof(T) * N) RwVec {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ RwVec<T, N> rw_load(const T* p) {
  RwVec<T, N> r;
  constexpr int kBytes = sizeof(T) * N;
  if constexpr (kBytes == 16) *reinterpret_cast<uint4*>(&r) = __ldg(reinterpret_cast<const uint4*>(p));
  else if constexpr (kBytes == 8) *reinterpret_cast<uint2*>(&r) = __ldg(reinterpret_cast<const uint2*>(p));
  else if constexpr (kBytes == 4) *reinterpret_cast<uint32_t*>(&r) = __ldg(reinterpret_cast<const uint32_t*>(p));
  else *reinterpret_cast<uint16_t*>(&r) = __ldg(reinterpret_cast<const uint16_t*>(p));
  return r;
}
template <typename T, int N>
__device__ __forceinline__ void rw_store(T* p, const RwVec<T, N>& r) {
  *reinterpret_cast<RwVec<T, N>*>(p) = r;
}

constexpr int kRwMaxK = 32;

struct RwArgs {
  int64_t tokens;
  int k, width;
  const int32_t* slots;   // [tokens][k]: a value outside [0, tokens k) stands for no row
  const void* x;          // [tokens]: dispatch's input, combine's residual (or null), or dout
  int64_t x_ld;
  void* rows;             // [tokens k] rows
  int64_t rows_ld;
  const float* weights;   // [tokens][k], or null: 1
  void* out;              // [tokens], contiguous
  float* dweights;        // combine's backward, or null
};

template <typename T, int N>
__global__ void __launch_bounds__(256) rw_dispatch(const RwArgs q) {
  const int per = q.width / N;
  const int64_t total = q.tokens * per, places = q.tokens * q.k;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t t = i / per;
    const int c = static_cast<int>(i - t * per) * N;
    const RwVec<T, N> v = rw_load<T, N>(static_cast<const T*>(q.x) + t * q.x_ld + c);
    for (int j = 0; j < q.k; ++j) {
      const int64_t s = __ldg(q.slots + t * q.k + j);
      if (s >= 0 && s < places) rw_store<T, N>(static_cast<T*>(q.rows) + s * q.rows_ld + c, v);
    }
  }
}

template <typename T, int N>
__global__ void __launch_bounds__(256) rw_combine(const RwArgs q) {
  const int per = q.width / N;
  const int64_t total = q.tokens * per, places = q.tokens * q.k;
  const T* rows = static_cast<const T*>(q.rows);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t t = i / per;
    const int c = static_cast<int>(i - t * per) * N;
    float z[N];
    if (q.x) {
      const RwVec<T, N> v = rw_load<T, N>(static_cast<const T*>(q.x) + t * q.x_ld + c);
#pragma unroll
      for (int n = 0; n < N; ++n) z[n] = Elem<T>::to_f(v.v[n]);
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n) z[n] = 0.f;
    }
    for (int j0 = 0; j0 < q.k; j0 += 4) {
      RwVec<T, N> v[4];
      float w[4];
      bool in[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t s = j0 + j < q.k ? __ldg(q.slots + t * q.k + j0 + j) : -1;
        in[j] = s >= 0 && s < places;
        if (in[j]) {
          v[j] = rw_load<T, N>(rows + s * q.rows_ld + c);
          w[j] = q.weights ? __ldg(q.weights + t * q.k + j0 + j) : 1.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (in[j]) {
#pragma unroll
          for (int n = 0; n < N; ++n) z[n] = fmaf(w[j], Elem<T>::to_f(v[j].v[n]), z[n]);
        }
    }
    RwVec<T, N> o;
#pragma unroll
    for (int n = 0; n < N; ++n) o.v[n] = Elem<T>::from_f(z[n]);
    rw_store<T, N>(static_cast<T*>(q.out) + t * q.width + c, o);
  }
}

// combine's backward: a warp takes a token; drows[slot_tj] = w_tj dout_t (q.out: drows, contiguous)
// and dw_tj = <dout_t, rows[slot_tj]>. Lane j keeps the j-th sum.
constexpr int kRwWarps = 8;
template <typename T, int N>
__global__ void __launch_bounds__(32 * kRwWarps) rw_combine_backward(const RwArgs q) {
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kRwWarps + (threadIdx.x >> 5);
  if (t >= q.tokens) return;
  constexpr int kHold = 16 / (N * static_cast<int>(sizeof(T)) >= 16 ? 4 : N * static_cast<int>(sizeof(T)) >= 8 ? 2 : 1);
  const int64_t places = q.tokens * q.k;
  const T* dout = static_cast<const T*>(q.x) + t * q.x_ld;
  const int64_t my_slot = lane < q.k ? __ldg(q.slots + t * q.k + lane) : -1;
  const float my_weight = lane < q.k ? __ldg(q.weights + t * q.k + lane) : 0.f;
  float dw = 0.f;
  for (int c0 = 0; c0 < q.width; c0 += 32 * N * kHold) {
    RwVec<T, N> d[kHold];
#pragma unroll
    for (int h = 0; h < kHold; ++h) {
      const int c = c0 + (h * 32 + lane) * N;
      if (c < q.width) d[h] = rw_load<T, N>(dout + c);
    }
    for (int j = 0; j < q.k; ++j) {
      const int64_t s = __shfl_sync(0xFFFFFFFFu, my_slot, j);
      const float w = __shfl_sync(0xFFFFFFFFu, my_weight, j);
      if (s < 0 || s >= places) continue;
      if (q.out) {
        T* o = static_cast<T*>(q.out) + s * q.width;
#pragma unroll
        for (int h = 0; h < kHold; ++h) {
          const int c = c0 + (h * 32 + lane) * N;
          if (c >= q.width) continue;
          RwVec<T, N> y;
#pragma unroll
          for (int n = 0; n < N; ++n) y.v[n] = Elem<T>::from_f(w * Elem<T>::to_f(d[h].v[n]));
          rw_store<T, N>(o + c, y);
        }
      }
      if (q.dweights) {
        const T* r = static_cast<const T*>(q.rows) + s * q.rows_ld;
        RwVec<T, N> v[kHold];
#pragma unroll
        for (int h = 0; h < kHold; ++h) {
          const int c = c0 + (h * 32 + lane) * N;
          if (c < q.width) v[h] = rw_load<T, N>(r + c);
        }
        float sum = 0.f;
#pragma unroll
        for (int h = 0; h < kHold; ++h) {
          const int c = c0 + (h * 32 + lane) * N;
          if (c >= q.width) continue;
#pragma unroll
          for (int n = 0; n < N; ++n) sum = fmaf(Elem<T>::to_f(d[h].v[n]), Elem<T>::to_f(v[h].v[n]), sum);
        }
#pragma unroll
        for (int m = 16; m; m >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, m);
        if (lane == j) dw += sum;
      }
    }
  }
  if (q.dweights && lane < q.k) q.dweights[t * q.k + lane] = dw;
}

// ---------------------------------------------------------------- embedding

struct EmArgs {
  int64_t n;              // tokens
  int width;
  int64_t vocab;
  const void* tokens;
  int tokens64;
  const void* table;
  int64_t table_ld;
  float scale;
  void* out;              // [n], contiguous
  // backward
  const void* dy;         // [n] rows
  int64_t dy_ld;
  const uint32_t* keys;   // sorted tokens (vocab: no row of the table), and their numbers
  const uint32_t* ids;
  const uint8_t* seen;    // [vocab]
  float* parts;           // [chunks][2][width]
  int64_t chunks;
  void* dtable;           // [vocab], contiguous
};

// A token outside the vocabulary gives a row of NaN.
template <typename T, int N>
__global__ void __launch_bounds__(256) em_forward(const EmArgs q) {
  const int per = q.width / N;
  const int64_t total = q.n * per;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = i / per;
    const int c = static_cast<int>(i - r * per) * N;
    const int64_t t = q.tokens64 ? __ldg(static_cast<const long long*>(q.tokens) + r)
                                 : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(q.tokens) + r));
    RwVec<T, N> v;
    if (t >= 0 && t < q.vocab) {
      v = rw_load<T, N>(static_cast<const T*>(q.table) + t * q.table_ld + c);
      if (q.scale != 1.f) {
#pragma unroll
        for (int n = 0; n < N; ++n) v.v[n] = Elem<T>::from_f(Elem<T>::to_f(v.v[n]) * q.scale);
      }
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n) v.v[n] = Elem<T>::from_f(CUDART_NAN_F);
    }
    rw_store<T, N>(static_cast<T*>(q.out) + r * q.width + c, v);
  }
}

// The table's gradient. A block takes kEmChunk consecutive places of the sorted tokens
// and adds up the rows of each run of one token. A run inside the block's places is
// finished there; the parts of one that goes over their edge are kept: slot 0 of a
// chunk for the run that comes in, slot 1 for one that begins there and goes on. (A frequent
// token's rows are so shared by many blocks.) em_finish adds the parts up. Blocks past the
// chunks write the zeros of tokens that do not occur.
constexpr int kEmChunk = 32;
constexpr int kEmAhead = 8;  // rows under way for each thread
constexpr int kEmZeroRows = 32;

template <typename T, int N>
__device__ __forceinline__ void em_put(const EmArgs& q, uint32_t token, int c, const float (&z)[N]) {
  RwVec<T, N> o;
#pragma unroll
  for (int n = 0; n < N; ++n) o.v[n] = Elem<T>::from_f(z[n] * q.scale);
  rw_store<T, N>(static_cast<T*>(q.dtable) + static_cast<int64_t>(token) * q.width + c, o);
}

template <typename T, int N>
__global__ void __launch_bounds__(256) em_sum(const EmArgs q) {
  __shared__ uint32_t keys[kEmChunk + 1], ids[kEmChunk];
  griddep_launch_dependents();
  griddep_wait();
  const int threads = blockDim.x;
  if (blockIdx.x >= q.chunks) {
    const int64_t r0 = (blockIdx.x - q.chunks) * kEmZeroRows;
    RwVec<T, N> zero;
#pragma unroll
    for (int n = 0; n < N; ++n) zero.v[n] = Elem<T>::from_f(0.f);
    for (int64_t r = r0; r < min(r0 + kEmZeroRows, q.vocab); ++r) {
      if (q.seen[r]) continue;
      for (int c = threadIdx.x * N; c < q.width; c += threads * N)
        rw_store<T, N>(static_cast<T*>(q.dtable) + r * q.width + c, zero);
    }
    return;
  }
  const int64_t p0 = blockIdx.x * static_cast<int64_t>(kEmChunk);
  const int here = static_cast<int>(min(static_cast<int64_t>(kEmChunk), q.n - p0));
  for (int i = threadIdx.x; i <= here; i += threads) {
    keys[i] = p0 + i < q.n ? __ldg(q.keys + p0 + i) : 0xFFFFFFFFu;  // the last: the next chunk's first
    if (i < here) ids[i] = __ldg(q.ids + p0 + i);
  }
  __syncthreads();
  const bool enters = p0 > 0 && __ldg(q.keys + p0 - 1) == keys[0];
  for (int c = threadIdx.x * N; c < q.width; c += threads * N) {
    float z[N];
#pragma unroll
    for (int n = 0; n < N; ++n) z[n] = 0.f;
    bool came = enters;
    for (int i0 = 0; i0 < here; i0 += kEmAhead) {
      RwVec<T, N> v[kEmAhead];
#pragma unroll
      for (int j = 0; j < kEmAhead; ++j)
        if (i0 + j < here && keys[i0 + j] < q.vocab)
          v[j] = rw_load<T, N>(static_cast<const T*>(q.dy) + static_cast<int64_t>(ids[i0 + j]) * q.dy_ld + c);
#pragma unroll
      for (int j = 0; j < kEmAhead; ++j) {
        const int i = i0 + j;
        if (i >= here || keys[i] >= q.vocab) continue;
#pragma unroll
        for (int n = 0; n < N; ++n) z[n] += Elem<T>::to_f(v[j].v[n]);
        const bool on = i + 1 == here && keys[here] == keys[i];  // the run goes on in the next chunk
        if (keys[i + 1] != keys[i] || on) {
          if (!came && !on) {
            em_put<T, N>(q, keys[i], c, z);
          } else {
            float* o = q.parts + (blockIdx.x * 2ll + (came ? 0 : 1)) * q.width + c;
#pragma unroll
            for (int n = 0; n < N; ++n) o[n] = z[n];
          }
#pragma unroll
          for (int n = 0; n < N; ++n) z[n] = 0.f;
          came = false;
        }
      }
    }
  }
}

// The runs that go over a chunk's edge: the block of the chunk where one begins adds its
// parts up, eight groups of threads a share of the chunks each, then the groups in turn.
constexpr int kEmGroups = 8, kEmCols = 32;
template <typename T>
__global__ void __launch_bounds__(kEmGroups * kEmCols) em_finish(const EmArgs q) {
  __shared__ float sums[kEmGroups][kEmCols];
  __shared__ int64_t end;
  griddep_wait();
  const int64_t b = blockIdx.x, p0 = b * kEmChunk, next = p0 + kEmChunk;
  if (next >= q.n) return;
  const uint32_t token = __ldg(q.keys + next);
  if (token >= q.vocab || __ldg(q.keys + next - 1) != token) return;  // no run over this edge
  if (__ldg(q.keys + p0) == token && p0 > 0 && __ldg(q.keys + p0 - 1) == token) return;  // it began before
  // The first chunk after b that the run does not reach.
  if (threadIdx.x == 0) {
    int64_t lo = b + 1, hi = q.chunks;
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (__ldg(q.keys + mid * kEmChunk) == token) lo = mid + 1;
      else hi = mid;
    }
    end = lo;
  }
  __syncthreads();
  const int g = threadIdx.x / kEmCols, l = threadIdx.x % kEmCols;
  const int64_t count = end - (b + 1), share = (count + kEmGroups - 1) / kEmGroups;
  const int64_t c0 = b + 1 + g * share, c1 = min(end, c0 + share);
  for (int col0 = blockIdx.y * kEmCols; col0 < q.width; col0 += gridDim.y * kEmCols) {
    const int col = col0 + l;
    float z = 0.f;
    if (col < q.width) {
      if (g == 0) z = __ldcg(q.parts + (b * 2 + 1) * q.width + col);
#pragma unroll 8
      for (int64_t c = c0; c < c1; ++c) z += __ldcg(q.parts + c * 2 * q.width + col);
    }
    sums[g][l] = z;
    __syncthreads();
    if (g == 0 && col < q.width) {
#pragma unroll
      for (int j = 1; j < kEmGroups; ++j) z += sums[j][l];
      static_cast<T*>(q.dtable)[static_cast<int64_t>(token) * q.width + col] = Elem<T>::from_f(z * q.scale);
    }
    __syncthreads();
  }
}

}  // namespace avey
