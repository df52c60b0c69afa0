// A stable counting sort by a digit of whole-number keys: which choices of tokens go
// to which expert (avey_arrange_v1), and the tokens of an embedding's gradient in the order
// of the vocabulary (digits of 10 bits, the lowest first).
//
// Blocks take consecutive runs of the entries, warps consecutive parts of a run: so an
// entry's place is the number of entries with a lower digit, of those with its own in
// earlier blocks and warps, and of those before it in its warp (found 32 at a time by
// matching digits over the warp). No atomics but on counts, whose order does not matter:
// the same input gives the same order. Up to 4096 entries one block does it all; more
// take a launch that counts and one that places.
#pragma once

#include "ptx.cuh"

namespace avey {

constexpr int kStWarps = 8, kStThreads = 32 * kStWarps;
constexpr int kStMaxBuckets = 1025;
constexpr int kStRun = 2048;       // entries of a block at least
constexpr int kStOneBlock = 4096;  // entries that one block takes

struct StArgs {
  int64_t n;
  int64_t run;            // entries of a block
  int buckets;
  int shift;              // the digit: (key >> shift) & mask; mask -1: the key itself
  int mask;
  const void* raw;        // keys as they come (int32 or int64), or null: `keys`
  int raw64;
  int64_t limit, skip;    // a raw key outside [0, limit), or equal to skip, counts as limit
  const uint32_t* keys;
  const uint32_t* ids;    // entry numbers that go with keys; null: 0, 1, 2, ...
  uint8_t* seen;          // [limit + 1], or null: set for every key that occurs
  uint32_t* counts;       // [blocks][buckets]
  int blocks;
  uint32_t* keys_out;     // sorted keys and entry numbers, or
  uint32_t* ids_out;
  int32_t* slots;         // the place of every entry
  int32_t* offsets;       // [buckets]: entries with a lower digit; or null
};

__device__ __forceinline__ uint32_t st_key(const StArgs& q, int64_t i) {
  if (!q.raw) return __ldg(q.keys + i);
  const int64_t t = q.raw64 ? __ldg(static_cast<const long long*>(q.raw) + i)
                            : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(q.raw) + i));
  return static_cast<uint32_t>(t < 0 || t >= q.limit || t == q.skip ? q.limit : t);
}
__device__ __forceinline__ uint32_t st_digit(const StArgs& q, uint32_t key) {
  return (key >> q.shift) & static_cast<uint32_t>(q.mask);
}

// The digits of a block's entries, counted for each warp: hist [warps][buckets].
__device__ __forceinline__ void st_count_block(const StArgs& q, uint32_t* hist, int64_t lo, int64_t hi) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kStWarps * q.buckets; i += kStThreads) hist[i] = 0;
  __syncthreads();
  const int64_t part = (hi - lo + kStWarps * 32 - 1) / (kStWarps * 32) * 32;
  const int64_t w0 = lo + warp * part, w1 = min(hi, w0 + part);
  uint32_t* mine = hist + warp * q.buckets;
  for (int64_t i = w0; i < w1; i += 32) {
    const bool in = i + lane < w1;
    const uint32_t key = in ? st_key(q, i + lane) : 0u;
    const uint32_t d = in ? st_digit(q, key) : 0xFFFFFFFFu;
    if (in && q.seen) q.seen[key] = 1;
    const unsigned peers = __match_any_sync(0xFFFFFFFFu, d);
    if (in && (peers & ((1u << lane) - 1)) == 0) mine[d] += __popc(peers);
    __syncwarp();
  }
  __syncthreads();
}

__global__ void __launch_bounds__(kStThreads) st_count(const StArgs q) {
  extern __shared__ uint32_t hist[];
  griddep_launch_dependents();
  griddep_wait();
  const int64_t lo = blockIdx.x * q.run, hi = min(q.n, lo + q.run);
  st_count_block(q, hist, lo, hi);
  for (int d = threadIdx.x; d < q.buckets; d += kStThreads) {
    uint32_t sum = 0;
#pragma unroll
    for (int w = 0; w < kStWarps; ++w) sum += hist[w * q.buckets + d];
    q.counts[static_cast<int64_t>(blockIdx.x) * q.buckets + d] = sum;
  }
}

__global__ void __launch_bounds__(kStThreads) st_place(const StArgs q) {
  extern __shared__ uint32_t hist[];  // [warps][buckets], then [buckets]
  __shared__ uint32_t warp_sums[kStWarps];
  griddep_launch_dependents();
  griddep_wait();
  uint32_t* start = hist + kStWarps * q.buckets;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t lo = blockIdx.x * q.run, hi = min(q.n, lo + q.run);
  st_count_block(q, hist, lo, hi);
  // Entries with a lower digit: an exclusive sum over the digits' totals, `per`
  // consecutive digits a thread.
  constexpr int kPer = (kStMaxBuckets + kStThreads - 1) / kStThreads;
  uint32_t total[kPer], before[kPer], sum = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int d = tid * kPer + j;
    total[j] = before[j] = 0;
    if (d >= q.buckets) continue;
    if (q.blocks > 1) {
      const uint32_t* c = q.counts + d;
#pragma unroll 8
      for (int b = 0; b < q.blocks; ++b) {
        const uint32_t v = __ldcg(c + static_cast<int64_t>(b) * q.buckets);
        total[j] += v;
        if (b < static_cast<int>(blockIdx.x)) before[j] += v;
      }
    } else {
      for (int w = 0; w < kStWarps; ++w) total[j] += hist[w * q.buckets + d];
    }
    sum += total[j];
  }
  uint32_t incl = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(0xFFFFFFFFu, incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  uint32_t at = incl - sum;
  for (int w = 0; w < warp; ++w) at += warp_sums[w];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int d = tid * kPer + j;
    if (d >= q.buckets) continue;
    start[d] = at + before[j];
    if (q.offsets && blockIdx.x == 0) q.offsets[d] = static_cast<int32_t>(at);
    at += total[j];
  }
  __syncthreads();
  // The first place of each warp's entries of each digit.
  for (int d = tid; d < q.buckets; d += kStThreads) {
    uint32_t p = start[d];
#pragma unroll
    for (int w = 0; w < kStWarps; ++w) {
      const uint32_t c = hist[w * q.buckets + d];
      hist[w * q.buckets + d] = p;
      p += c;
    }
  }
  __syncthreads();
  const int64_t part = (hi - lo + kStWarps * 32 - 1) / (kStWarps * 32) * 32;
  const int64_t w0 = lo + warp * part, w1 = min(hi, w0 + part);
  uint32_t* mine = hist + warp * q.buckets;
  for (int64_t i = w0; i < w1; i += 32) {
    const bool in = i + lane < w1;
    const uint32_t key = in ? st_key(q, i + lane) : 0u;
    const uint32_t d = in ? st_digit(q, key) : 0xFFFFFFFFu;
    const unsigned peers = __match_any_sync(0xFFFFFFFFu, d);
    const unsigned lower = peers & ((1u << lane) - 1);
    uint32_t p = 0;
    if (in) p = mine[d] + __popc(lower);
    __syncwarp();
    if (in && lower == 0) mine[d] += __popc(peers);
    __syncwarp();
    if (!in) continue;
    if (q.slots) {
      q.slots[i + lane] = static_cast<int32_t>(p);
    } else {
      q.keys_out[p] = key;
      q.ids_out[p] = q.ids ? __ldg(q.ids + i + lane) : static_cast<uint32_t>(i + lane);
    }
  }
}

}  // namespace avey
