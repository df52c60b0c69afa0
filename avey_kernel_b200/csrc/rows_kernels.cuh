// Rows moved between tokens and the places that they are worked on or kept at:
//
//   dispatch   rows[slot_tj] = x_t                      (and the scaled form: the gradient
//                                                        of combine's rows, w_tj dout_t)
//   combine    out_t = residual_t + sum_j w_tj rows[slot_tj]   (w = 1: dispatch's gradient)
//   embedding  out_i = scale table[token_i]
//   and the embedding's gradient by sorted tokens.
//
// Bound: the rows' bytes, each read and written once. A lane moves 16 bytes of a row at a
// time (less where rows are not whole 16-byte units); a token's rows belong to one warp
// (or a part of one, for narrow rows), which has up to 16 accesses a lane under way and
// the next token's slots read ahead. (32768 tokens, four rows of 768 in bf16: combine with
// a residual 71 us for 302 MB, its backward pass 84 for 453, dispatch 40 for 252; a
// bare sum over 268 MB takes 59 here, over 4.3 GB 666: what memory gives is 17 us and
// 6.6 TB/s.)
// Sums are fp32, in the order of the choices, or of the tokens.
#pragma once

#include <math_constants.h>

#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"

namespace avey {

// N values of type T as one access of 16, 4 or 2 bytes, held as words (as an array of T
// the compiler kept what is loaded under a condition in local memory: 101 -> 170 us for
// the sums of combine).
template <typename T, int N>
struct RwVec {
  static constexpr int kBytes = static_cast<int>(sizeof(T)) * N, kWords = kBytes < 4 ? 1 : kBytes / 4;
  uint32_t w[kWords];
};
template <typename T, int N>
__device__ __forceinline__ RwVec<T, N> rw_zero() {
  RwVec<T, N> r;
#pragma unroll
  for (int i = 0; i < RwVec<T, N>::kWords; ++i) r.w[i] = 0u;
  return r;
}
template <typename T, int N>
__device__ __forceinline__ RwVec<T, N> rw_load(const T* p) {
  RwVec<T, N> r;
  if constexpr (RwVec<T, N>::kBytes == 16) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    r.w[0] = v.x;
    r.w[1] = v.y;
    r.w[2] = v.z;
    r.w[3] = v.w;
  } else if constexpr (RwVec<T, N>::kBytes == 4) {
    r.w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  } else {
    r.w[0] = __ldg(reinterpret_cast<const uint16_t*>(p));
  }
  return r;
}
template <typename T, int N>
__device__ __forceinline__ void rw_store(T* p, const RwVec<T, N>& r) {
  if constexpr (RwVec<T, N>::kBytes == 16) *reinterpret_cast<uint4*>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
  else if constexpr (RwVec<T, N>::kBytes == 4) *reinterpret_cast<uint32_t*>(p) = r.w[0];
  else *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(r.w[0]);
}
// The n-th value, and values rounded to T.
template <typename T, int N>
__device__ __forceinline__ float rw_get(const RwVec<T, N>& r, int n) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(r.w[n]);
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return __uint_as_float((n & 1) ? r.w[n / 2] & 0xFFFF0000u : r.w[n / 2] << 16);
  } else {
    return __half2float(__ushort_as_half(static_cast<unsigned short>((n & 1) ? r.w[n / 2] >> 16 : r.w[n / 2])));
  }
}
template <typename T, int N>
__device__ __forceinline__ RwVec<T, N> rw_pack(const float (&z)[N]) {
  RwVec<T, N> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int n = 0; n < N; ++n) r.w[n] = __float_as_uint(z[n]);
  } else {
#pragma unroll
    for (int i = 0; i < RwVec<T, N>::kWords; ++i) {
      const float lo = z[2 * i], hi = 2 * i + 1 < N ? z[2 * i + 1] : 0.f;
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        r.w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(lo, hi);
        r.w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
  return r;
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
  int blanks;             // 1: the first block clears the places that no slot names (rw_blank)
  int32_t* namer;         // or: [tokens k], the choice that names a place, for rw_clear
};

// Rows that no slot names are zeros, not what memory held before. Up to kRwBlankPlaces places:
// a block ahead of the call's own reads the slots, marks the places that they name in a bit map in
// shared memory and clears the others, waiting for nothing (16 tokens of two: 1.7 us for the launch
// instead of 1.6). One block takes 60 us for 131072 slots beside the rows' own traffic, so more
// places take a launch of their own (rw_clear).
constexpr int kRwBlankPlaces = 8192;
template <typename T, int N>
__device__ __forceinline__ void rw_blank(const RwArgs& q, T* rows, int64_t ld) {
  __shared__ uint32_t named[kRwBlankPlaces / 32];
  const int places = static_cast<int>(q.tokens) * q.k, words = (places + 31) / 32;
  for (int i = threadIdx.x; i < words; i += blockDim.x) named[i] = 0u;
  __syncthreads();
#pragma unroll 8
  for (int i = threadIdx.x; i < places; i += blockDim.x) {
    const int32_t s = __ldg(q.slots + i);
    if (s >= 0 && s < places) atomicOr(named + (s >> 5), 1u << (s & 31));
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int w = threadIdx.x >> 5; w < words; w += static_cast<int>(blockDim.x >> 5)) {
    const int left = places - 32 * w;
    unsigned blank = ~named[w] & (left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1);
    for (; blank; blank &= blank - 1) {
      T* row = rows + static_cast<int64_t>(32 * w + __ffs(blank) - 1) * ld;
      for (int c = lane * N; c < q.width; c += 32 * N) rw_store<T, N>(row + c, rw_zero<T, N>());
    }
  }
}

// More places: the launch before has left in namer[p] the number of the choice that names p, and
// where none does, whatever was there: if that is a choice whose slot is p then p is named after all, so
// nothing has to be set up. A warp looks at 32 places. (131072 places: 4 us by itself, 2 of dispatch and of
// combine's backward pass each, as it is set up beside their ends.)
template <typename T, int N>
__global__ void __launch_bounds__(256) rw_clear(const int32_t* slots, const int32_t* namer, int places, T* rows,
                                                int64_t ld, int width) {
  griddep_wait();
  const int lane = threadIdx.x & 31, step = static_cast<int>(gridDim.x) * 256;
  for (int p0 = static_cast<int>(blockIdx.x) * 256 + threadIdx.x - lane; p0 < places; p0 += step) {
    const int p = p0 + lane;
    bool blank = false;
    if (p < places) {
      const int32_t i = __ldcg(namer + p);
      blank = i < 0 || i >= places || __ldg(slots + i) != p;
    }
    for (unsigned left = __ballot_sync(0xFFFFFFFFu, blank); left; left &= left - 1) {
      T* row = rows + static_cast<int64_t>(p0 + __ffs(left) - 1) * ld;
      for (int c = lane * N; c < width; c += 32 * N) rw_store<T, N>(row + c, rw_zero<T, N>());
    }
  }
}

template <typename T, int N>
__global__ void __launch_bounds__(256) rw_dispatch(const RwArgs q) {
  griddep_wait();
  const int block = static_cast<int>(blockIdx.x) - q.blanks, blocks = static_cast<int>(gridDim.x) - q.blanks;
  if (block < 0) {
    rw_blank<T, N>(q, static_cast<T*>(q.rows), q.rows_ld);
    return;
  }
  griddep_launch_dependents();
  const int per = q.width / N;
  const int64_t total = q.tokens * per, places = q.tokens * q.k;
  for (int64_t i = static_cast<int64_t>(block) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(blocks) * 256) {
    const int64_t t = i / per;
    const int c = static_cast<int>(i - t * per) * N;
    const RwVec<T, N> v = rw_load<T, N>(static_cast<const T*>(q.x) + t * q.x_ld + c);
    for (int j = 0; j < q.k; ++j) {
      const int64_t s = __ldg(q.slots + t * q.k + j);
      if (s < 0 || s >= places) continue;
      rw_store<T, N>(static_cast<T*>(q.rows) + s * q.rows_ld + c, v);
      if (c == 0 && q.namer) q.namer[s] = static_cast<int32_t>(t * q.k + j);
    }
  }
}

// A part of a warp for a token: 32 lanes, or the least power of two that holds a row.
// The parts take every gridDim-th token.
constexpr int kRwThreads = 256;
constexpr int kRwRows = 4;  // rows under way together; of each, HOLD accesses a lane: the row's
                            // own where those are up to four
constexpr int rw_blocks(int hold) { return hold == 1 ? 5 : hold == 2 ? 3 : 2; }  // of an SM
struct RwPart {
  int64_t t, step;
  int lane;
};
__device__ __forceinline__ RwPart rw_part(int lanes, int blanks = 0) {
  const int parts = kRwThreads / lanes;
  return {static_cast<int64_t>(blockIdx.x - blanks) * parts + threadIdx.x / lanes,
          static_cast<int64_t>(gridDim.x - blanks) * parts, static_cast<int>(threadIdx.x) & (lanes - 1)};
}
// Slots and weights of up to kRwRows choices of a token from j0 on (past its last: no row).
struct RwSlots {
  int32_t s[kRwRows];
  float w[kRwRows];
};
__device__ __forceinline__ RwSlots rw_slots(const RwArgs& q, int64_t t, int j0) {
  RwSlots r;
#pragma unroll
  for (int j = 0; j < kRwRows; ++j) {
    const bool in = t < q.tokens && j0 + j < q.k;
    r.s[j] = in ? __ldg(q.slots + t * q.k + j0 + j) : -1;
    r.w[j] = in && q.weights ? __ldg(q.weights + t * q.k + j0 + j) : 1.f;
  }
  return r;
}

template <typename T, int N, int HOLD>
__global__ void __launch_bounds__(kRwThreads, rw_blocks(HOLD)) rw_combine(const RwArgs q, int lanes) {
  griddep_wait();
  const RwPart at = rw_part(lanes);
  const int64_t places = q.tokens * q.k;
  const T* rows = static_cast<const T*>(q.rows);
  const int span = lanes * N;
  RwSlots ahead = rw_slots(q, at.t, 0);
  for (int64_t t = at.t; t < q.tokens; t += at.step) {
    const RwSlots first = ahead;
    ahead = rw_slots(q, t + at.step, 0);
    for (int c0 = at.lane * N; c0 < q.width; c0 += span * HOLD) {
      RwVec<T, N> r[HOLD];
#pragma unroll
      for (int h = 0; h < HOLD; ++h)
        r[h] = q.x && c0 + h * span < q.width ? rw_load<T, N>(static_cast<const T*>(q.x) + t * q.x_ld + c0 + h * span)
                                              : rw_zero<T, N>();
      float z[HOLD][N];
      for (int j0 = 0; j0 < q.k; j0 += kRwRows) {
        const RwSlots sl = j0 == 0 ? first : rw_slots(q, t, j0);
        RwVec<T, N> v[kRwRows][HOLD];
#pragma unroll
        for (int j = 0; j < kRwRows; ++j)
#pragma unroll
          for (int h = 0; h < HOLD; ++h)
            v[j][h] = sl.s[j] >= 0 && sl.s[j] < places && c0 + h * span < q.width
                          ? rw_load<T, N>(rows + static_cast<int64_t>(sl.s[j]) * q.rows_ld + c0 + h * span)
                          : rw_zero<T, N>();
        if (j0 == 0) {
#pragma unroll
          for (int h = 0; h < HOLD; ++h)
#pragma unroll
            for (int n = 0; n < N; ++n) z[h][n] = rw_get(r[h], n);
        }
#pragma unroll
        for (int j = 0; j < kRwRows; ++j)
          if (sl.s[j] >= 0 && sl.s[j] < places) {  // (its weight may be infinite where there is no row)
#pragma unroll
            for (int h = 0; h < HOLD; ++h)
#pragma unroll
              for (int n = 0; n < N; ++n) z[h][n] = fmaf(sl.w[j], rw_get(v[j][h], n), z[h][n]);
          }
      }
#pragma unroll
      for (int h = 0; h < HOLD; ++h) {
        if (c0 + h * span < q.width)
          rw_store<T, N>(static_cast<T*>(q.out) + t * q.width + c0 + h * span, rw_pack<T, N>(z[h]));
      }
    }
  }
}

// combine's backward: drows[slot_tj] = w_tj dout_t (q.out: drows, contiguous) and dw_tj =
// <dout_t, rows[slot_tj]>.
template <typename T, int N, int HOLD>
__global__ void __launch_bounds__(kRwThreads, rw_blocks(HOLD)) rw_combine_backward(const RwArgs q, int lanes) {
  griddep_wait();
  if (static_cast<int>(blockIdx.x) < q.blanks) {
    rw_blank<T, N>(q, static_cast<T*>(q.out), q.width);
    return;
  }
  griddep_launch_dependents();
  const RwPart at = rw_part(lanes, q.blanks);
  const unsigned mask = lanes == 32 ? 0xFFFFFFFFu : ((1u << lanes) - 1) << (threadIdx.x & 31 & ~(lanes - 1));
  const int64_t places = q.tokens * q.k;
  const T* rows = static_cast<const T*>(q.rows);
  const int span = lanes * N;
  RwSlots ahead = rw_slots(q, at.t, 0);
  for (int64_t t = at.t; t < q.tokens; t += at.step) {
    const T* dout = static_cast<const T*>(q.x) + t * q.x_ld;
    const RwSlots first = ahead;
    ahead = rw_slots(q, t + at.step, 0);
    for (int j0 = 0; j0 < q.k; j0 += kRwRows) {
      const RwSlots sl = j0 == 0 ? first : rw_slots(q, t, j0);
      float sum[kRwRows] = {};
      if (at.lane == 0 && q.namer) {
#pragma unroll
        for (int j = 0; j < kRwRows; ++j)
          if (sl.s[j] >= 0 && sl.s[j] < places) q.namer[sl.s[j]] = static_cast<int32_t>(t * q.k + j0 + j);
      }
      for (int c0 = at.lane * N; c0 < q.width; c0 += span * HOLD) {
        RwVec<T, N> d[HOLD], v[kRwRows][HOLD];
#pragma unroll
        for (int h = 0; h < HOLD; ++h)
          d[h] = c0 + h * span < q.width ? rw_load<T, N>(dout + c0 + h * span) : rw_zero<T, N>();
#pragma unroll
        for (int j = 0; j < kRwRows; ++j)
#pragma unroll
          for (int h = 0; h < HOLD; ++h)
            v[j][h] = q.dweights && sl.s[j] >= 0 && sl.s[j] < places && c0 + h * span < q.width
                          ? rw_load<T, N>(rows + static_cast<int64_t>(sl.s[j]) * q.rows_ld + c0 + h * span)
                          : rw_zero<T, N>();
#pragma unroll
        for (int j = 0; j < kRwRows; ++j) {
          if (sl.s[j] < 0 || sl.s[j] >= places) continue;
#pragma unroll
          for (int h = 0; h < HOLD; ++h) {
            if (q.out && c0 + h * span < q.width) {
              float y[N];
#pragma unroll
              for (int n = 0; n < N; ++n) y[n] = sl.w[j] * rw_get(d[h], n);
              rw_store<T, N>(static_cast<T*>(q.out) + static_cast<int64_t>(sl.s[j]) * q.width + c0 + h * span,
                             rw_pack<T, N>(y));
            }
            if (c0 + h * span < q.width) {
#pragma unroll
              for (int n = 0; n < N; ++n) sum[j] = fmaf(rw_get(d[h], n), rw_get(v[j][h], n), sum[j]);
            }
          }
        }
      }
      if (q.dweights) {
#pragma unroll
        for (int j = 0; j < kRwRows; ++j) {
          for (int m = lanes / 2; m; m >>= 1) sum[j] += __shfl_xor_sync(mask, sum[j], m);
          if (at.lane == 0 && j0 + j < q.k) q.dweights[t * q.k + j0 + j] = sum[j];
        }
      }
    }
  }
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
  float* parts;           // [chunks][2][width]
  int chunk;              // places of a chunk
  uint32_t* edges;        // chunks where a run begins that goes on: their number, zero before, and they
  int64_t chunks;
  void* dtable;           // [vocab], contiguous
};

// A token outside the vocabulary gives a row of NaN. A part of a warp takes a row.
template <typename T, int N>
__global__ void __launch_bounds__(kRwThreads) em_forward(const EmArgs q, int lanes) {
  griddep_wait();
  const RwPart at = rw_part(lanes);
  if (at.t >= q.n) return;
  const int64_t t = q.tokens64 ? __ldg(static_cast<const long long*>(q.tokens) + at.t)
                               : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(q.tokens) + at.t));
  const bool in = t >= 0 && t < q.vocab;
  const T* row = static_cast<const T*>(q.table) + t * q.table_ld;
  T* out = static_cast<T*>(q.out) + at.t * q.width;
  const int span = lanes * N;
  constexpr int kHold = 4;
  for (int c0 = at.lane * N; c0 < q.width; c0 += span * kHold) {
    RwVec<T, N> v[kHold];
#pragma unroll
    for (int h = 0; h < kHold; ++h)
      v[h] = in && c0 + h * span < q.width ? rw_load<T, N>(row + c0 + h * span) : rw_zero<T, N>();
#pragma unroll
    for (int h = 0; h < kHold; ++h) {
      if (c0 + h * span >= q.width) continue;
      if (!in || q.scale != 1.f) {
        float z[N];
#pragma unroll
        for (int n = 0; n < N; ++n) z[n] = in ? rw_get(v[h], n) * q.scale : CUDART_NAN_F;
        v[h] = rw_pack<T, N>(z);
      }
      rw_store<T, N>(out + c0 + h * span, v[h]);
    }
  }
}

// The table's gradient. A block takes kEmChunk consecutive places of the sorted tokens
// and adds up the rows of each run of one token. A run inside the block's places is
// finished there; the parts of one that goes over their edge are kept: slot 0 of a
// chunk for the run that comes in, slot 1 for one that begins there and goes on. (A frequent
// token's rows are so shared by many blocks.) em_finish adds the parts up: of the runs that
// em_sum lists, whose order does not matter. Zeros are written to the whole table before,
// beside the sort, which leaves most of the GPU idle. 32 places (64 halve em_finish's work,
// 18 to 11 us for 65536 tokens of 768, and cost the call 4 us elsewhere), or 16 or 8 where
// those would be too few blocks.
constexpr int kEmChunk = 32, kEmSmallChunk = 8;
constexpr int kEmAhead = 8;  // rows under way for each thread

template <typename T, int N>
__device__ __forceinline__ void em_put(const EmArgs& q, uint32_t token, int c, const float (&z)[N]) {
  float y[N];
#pragma unroll
  for (int n = 0; n < N; ++n) y[n] = z[n] * q.scale;
  rw_store<T, N>(static_cast<T*>(q.dtable) + static_cast<int64_t>(token) * q.width + c, rw_pack<T, N>(y));
}

template <typename T, int N>
__global__ void __launch_bounds__(256) em_sum(const EmArgs q) {
  __shared__ uint32_t keys[kEmChunk + 1], ids[kEmChunk];
  griddep_launch_dependents();
  griddep_wait();
  const int threads = blockDim.x;
  const int64_t p0 = blockIdx.x * static_cast<int64_t>(q.chunk);
  const int here = static_cast<int>(min(static_cast<int64_t>(q.chunk), q.n - p0));
  for (int i = threadIdx.x; i <= here; i += threads) {
    keys[i] = p0 + i < q.n ? __ldg(q.keys + p0 + i) : 0xFFFFFFFFu;  // the last: the next chunk's first
    if (i < here) ids[i] = __ldg(q.ids + p0 + i);
  }
  __syncthreads();
  const bool enters = p0 > 0 && __ldg(q.keys + p0 - 1) == keys[0];
  if (threadIdx.x == 0 && blockIdx.y == 0 && here == q.chunk && keys[here] == keys[here - 1] && keys[here] < q.vocab &&
      !(enters && keys[0] == keys[here]))
    q.edges[1 + atomicAdd(q.edges, 1u)] = blockIdx.x;
  for (int c = (blockIdx.y * threads + threadIdx.x) * N; c < q.width; c += gridDim.y * threads * N) {
    float z[N];
#pragma unroll
    for (int n = 0; n < N; ++n) z[n] = 0.f;
    bool came = enters;
    for (int i0 = 0; i0 < here; i0 += kEmAhead) {
      RwVec<T, N> v[kEmAhead];
#pragma unroll
      for (int j = 0; j < kEmAhead; ++j)
        v[j] = i0 + j < here && keys[i0 + j] < q.vocab
                   ? rw_load<T, N>(static_cast<const T*>(q.dy) + static_cast<int64_t>(ids[i0 + j]) * q.dy_ld + c)
                   : rw_zero<T, N>();
#pragma unroll
      for (int j = 0; j < kEmAhead; ++j) {
        const int i = i0 + j;
        if (i >= here || keys[i] >= q.vocab) continue;
#pragma unroll
        for (int n = 0; n < N; ++n) z[n] += rw_get(v[j], n);
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

// The runs that go over a chunk's edge. A block takes a run and 64 V of its columns: four
// groups of threads a share of its chunks each, then the groups in turn.
constexpr int kEmGroups = 4, kEmLanes = 64;
template <typename T, int V>
__global__ void __launch_bounds__(kEmGroups * kEmLanes) em_finish(const EmArgs q, int slabs) {
  __shared__ float sums[kEmGroups][kEmLanes * V];
  __shared__ int64_t last;
  griddep_wait();
  const int g = threadIdx.x / kEmLanes, l = threadIdx.x % kEmLanes;
  const int64_t items = static_cast<int64_t>(*q.edges) * slabs;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t b = q.edges[1 + item / slabs];
    const uint32_t token = __ldg(q.keys + (b + 1) * q.chunk);
    // The last chunk that the run reaches: looked at 256 at a time.
    if (threadIdx.x == 0) last = b;
    __syncthreads();
    for (int64_t c0 = b + 1;; c0 += kEmGroups * kEmLanes) {
      const int64_t c = c0 + threadIdx.x;
      const bool in = c < q.chunks && __ldg(q.keys + c * q.chunk) == token;
      const int n = __syncthreads_count(in);
      if (threadIdx.x == 0) last = c0 - 1 + n;
      if (n < kEmGroups * kEmLanes) break;
    }
    __syncthreads();
    const int64_t count = last - b, share = (count + kEmGroups - 1) / kEmGroups;
    const int64_t c0 = b + 1 + g * share, c1 = min(last + 1, c0 + share);
    const int col = static_cast<int>(item % slabs) * kEmLanes * V + l * V;
    float z[V];
#pragma unroll
    for (int n = 0; n < V; ++n) z[n] = 0.f;
    if (col < q.width) {
      if (g == 0) {
        const RwVec<float, V> v = rw_load<float, V>(q.parts + (b * 2 + 1) * q.width + col);
#pragma unroll
        for (int n = 0; n < V; ++n) z[n] = rw_get(v, n);
      }
#pragma unroll 8
      for (int64_t c = c0; c < c1; ++c) {
        const RwVec<float, V> v = rw_load<float, V>(q.parts + c * 2 * q.width + col);
#pragma unroll
        for (int n = 0; n < V; ++n) z[n] += rw_get(v, n);
      }
    }
#pragma unroll
    for (int n = 0; n < V; ++n) sums[g][l * V + n] = z[n];
    __syncthreads();
    if (g == 0 && col < q.width) {
#pragma unroll
      for (int n = 0; n < V; ++n) {
#pragma unroll
        for (int j = 1; j < kEmGroups; ++j) z[n] += sums[j][l * V + n];
        static_cast<T*>(q.dtable)[static_cast<int64_t>(token) * q.width + col + n] = Elem<T>::from_f(z[n] * q.scale);
      }
    }
    __syncthreads();
  }
}

}  // namespace avey
