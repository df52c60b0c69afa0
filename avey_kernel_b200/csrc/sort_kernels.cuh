// A stable counting sort by a digit of whole-number keys: which choices of tokens go
// to which expert (avey_arrange_v1), and the tokens of an embedding's gradient in the order
// of the vocabulary (digits of 10 bits, the lowest first).
//
// Blocks take consecutive runs of the entries, warps consecutive parts of a run: so an
// entry's place is the number of entries with a lower digit, of those with its own in
// earlier blocks and warps, and of those before it in its warp (found 32 at a time by
// matching digits over the warp). No atomics but on counts: the same input gives the same
// order. Up to 8192 entries take one launch: of one block for one digit, or, for keys of more,
// of blocks that compare each key with all (st_rank). More take a launch that counts and one
// that places, which counts for the next digit. Blocks beside those, where the rest of the GPU
// would idle, write zeros (a table's gradient, of which most rows are zero).
//
// Bound: latency, of a few dependent reads a launch: so a warp's keys are loaded eight
// steps at a time, and the counts of all blocks 16 at a time.
#pragma once

#include "ptx.cuh"

namespace avey {

constexpr int kStWarps = 16, kStThreads = 32 * kStWarps;
constexpr int kStMaxBuckets = 1025;
// Entries of a block at least. (With 4096, 131072 choices of 64 experts and the training calls
// around them took 295 us instead of 288, an embedding's of 65536 tokens 138 instead of 129;
// with 1024: 288 and 132.)
constexpr int kStRun = 2048;
constexpr int kStOneBlock = 8192;  // entries that one block, or st_rank, takes
constexpr int kStSteps = 8;        // keys a lane holds
constexpr int kStSmem = (kStWarps + 1) * kStMaxBuckets * 4;

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
  uint32_t* counts;       // [blocks][buckets]
  int blocks;
  uint32_t* keys_out;     // sorted keys and entry numbers, or
  uint32_t* ids_out;
  int32_t* slots;         // the place of every entry
  int32_t* offsets;       // [buckets]: entries with a lower digit; or null
  uint32_t* next_counts;  // the next pass's [blocks][buckets], zero before: counted while placing; or null
  uint32_t* clear;        // st_rank: a word to be cleared
  // Blocks past `blocks` write zeros to these bytes.
  uint8_t* zeros;
  int64_t zero_bytes;
};

// Zeros by `blocks` blocks, 16 bytes an access but at the ends.
__device__ __forceinline__ void st_zero(uint8_t* p, int64_t bytes, int64_t block, int64_t blocks) {
  const int64_t head = min(bytes, static_cast<int64_t>(-reinterpret_cast<uintptr_t>(p) & 15u));
  const int64_t words = (bytes - head) / 16, tail = bytes - head - 16 * words;
  uint4* body = reinterpret_cast<uint4*>(p + head);
  for (int64_t i = block * blockDim.x + threadIdx.x; i < words; i += blocks * blockDim.x)
    body[i] = make_uint4(0u, 0u, 0u, 0u);
  if (block != 0) return;
  if (threadIdx.x < head) p[threadIdx.x] = 0;
  if (threadIdx.x < tail) p[bytes - tail + threadIdx.x] = 0;
}
__device__ __forceinline__ uint32_t st_key(const StArgs& q, int64_t i) {
  if (!q.raw) return __ldcg(q.keys + i);
  const int64_t t = q.raw64 ? __ldg(static_cast<const long long*>(q.raw) + i)
                            : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(q.raw) + i));
  return static_cast<uint32_t>(t < 0 || t >= q.limit || t == q.skip ? q.limit : t);
}
__device__ __forceinline__ uint32_t st_digit(const StArgs& q, uint32_t key) {
  return (key >> q.shift) & static_cast<uint32_t>(q.mask);
}

// A warp's part of a block's entries [lo, hi): whole steps of 32.
struct StPart {
  int64_t w0, w1;
};
__device__ __forceinline__ StPart st_part(int64_t lo, int64_t hi) {
  const int64_t part = (hi - lo + kStThreads - 1) / kStThreads * 32;
  const int64_t w0 = min(hi, lo + (threadIdx.x >> 5) * part);
  return {w0, min(hi, w0 + part)};
}
// Eight steps' keys from i0 on (past the end: none).
__device__ __forceinline__ void st_keys(const StArgs& q, int64_t i0, int64_t w1, uint32_t (&key)[kStSteps]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int s = 0; s < kStSteps; ++s) {
    const int64_t i = i0 + 32 * s + lane;
    key[s] = i < w1 ? st_key(q, i) : 0xFFFFFFFFu;
  }
}

// The digits of a block's entries, counted for each warp: hist [warps][buckets].
__device__ __forceinline__ void st_count_block(const StArgs& q, uint32_t* hist, const StPart& part) {
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kStWarps * q.buckets; i += kStThreads) hist[i] = 0;
  __syncthreads();
  uint32_t* mine = hist + (threadIdx.x >> 5) * q.buckets;
  for (int64_t i0 = part.w0; i0 < part.w1; i0 += 32 * kStSteps) {
    uint32_t key[kStSteps];
    st_keys(q, i0, part.w1, key);
#pragma unroll
    for (int s = 0; s < kStSteps; ++s) {
      if (i0 + 32 * s >= part.w1) break;
      const bool in = key[s] != 0xFFFFFFFFu;
      const uint32_t d = in ? st_digit(q, key[s]) : 0xFFFFFFFFu;
      const unsigned peers = __match_any_sync(0xFFFFFFFFu, d);
      if (in && (peers & ((1u << lane) - 1)) == 0) mine[d] += __popc(peers);
      __syncwarp();
    }
  }
  __syncthreads();
}

__global__ void __launch_bounds__(kStThreads) st_count(const StArgs q) {
  extern __shared__ uint32_t hist[];
  griddep_launch_dependents();
  griddep_wait();
  const int64_t lo = blockIdx.x * q.run, hi = min(q.n, lo + q.run);
  st_count_block(q, hist, st_part(lo, hi));
  for (int d = threadIdx.x; d < q.buckets; d += kStThreads) {
    uint32_t sum = 0;
#pragma unroll
    for (int w = 0; w < kStWarps; ++w) sum += hist[w * q.buckets + d];
    q.counts[static_cast<int64_t>(blockIdx.x) * q.buckets + d] = sum;
  }
}

// One pass of a block over its entries. hist: [warps][buckets], then [buckets].
__device__ __forceinline__ void st_place_block(const StArgs& q, uint32_t* hist, uint32_t* warp_sums) {
  uint32_t* totals = hist + kStWarps * q.buckets;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t lo = blockIdx.x * q.run, hi = min(q.n, lo + q.run);
  const StPart part = st_part(lo, hi);
  st_count_block(q, hist, part);
  // The digits' totals, and how many of them are in earlier blocks.
  constexpr int kPer = (kStMaxBuckets + kStThreads - 1) / kStThreads;
  uint32_t before[kPer];
  const int slices = q.blocks > 1 ? kStThreads / q.buckets : 0;
  if (slices > 1) {
    // Few digits: that many threads share the blocks of each.
    __shared__ uint2 shares[kStThreads];
    const int slice = tid / q.buckets, d = tid - slice * q.buckets;
    uint2 sum = make_uint2(0u, 0u);
    for (int b0 = slice; b0 < q.blocks && slice < slices; b0 += 16 * slices) {
      uint32_t v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int b = b0 + i * slices;
        v[i] = b < q.blocks ? __ldcg(q.counts + static_cast<int64_t>(b) * q.buckets + d) : 0u;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        sum.x += v[i];
        if (b0 + i * slices < static_cast<int>(blockIdx.x)) sum.y += v[i];
      }
    }
    shares[tid] = sum;
    __syncthreads();
    if (tid < q.buckets) {
      for (int i = 1; i < slices; ++i) {
        sum.x += shares[i * q.buckets + tid].x;
        sum.y += shares[i * q.buckets + tid].y;
      }
      totals[tid] = sum.x;
    }
    before[0] = sum.y;
#pragma unroll
    for (int j = 1; j < kPer; ++j) before[j] = 0;
  }
#pragma unroll
  for (int j = 0; j < kPer && slices <= 1; ++j) {
    const int d = j * kStThreads + tid;
    before[j] = 0;
    if (d >= q.buckets) continue;
    uint32_t total = 0;
    if (q.blocks > 1) {
      const uint32_t* c = q.counts + d;
      for (int b0 = 0; b0 < q.blocks; b0 += 16) {
        uint32_t v[16];
#pragma unroll
        for (int b = 0; b < 16; ++b)
          v[b] = b0 + b < q.blocks ? __ldcg(c + static_cast<int64_t>(b0 + b) * q.buckets) : 0u;
#pragma unroll
        for (int b = 0; b < 16; ++b) {
          total += v[b];
          if (b0 + b < static_cast<int>(blockIdx.x)) before[j] += v[b];
        }
      }
    } else {
#pragma unroll
      for (int w = 0; w < kStWarps; ++w) total += hist[w * q.buckets + d];
    }
    totals[d] = total;
  }
  __syncthreads();
  // Entries with a lower digit: an exclusive sum, kPer consecutive digits a thread.
  uint32_t mine[kPer], sum = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int d = tid * kPer + j;
    mine[j] = d < q.buckets ? totals[d] : 0u;
    sum += mine[j];
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
    totals[d] = at;
    if (q.offsets && blockIdx.x == 0) q.offsets[d] = static_cast<int32_t>(at);
    at += mine[j];
  }
  __syncthreads();
  // The first place of each warp's entries of each digit.
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int d = j * kStThreads + tid;
    if (d >= q.buckets) continue;
    uint32_t p = totals[d] + before[j];
#pragma unroll
    for (int w = 0; w < kStWarps; ++w) {
      const uint32_t c = hist[w * q.buckets + d];
      hist[w * q.buckets + d] = p;
      p += c;
    }
  }
  __syncthreads();
  uint32_t* place = hist + warp * q.buckets;
  for (int64_t i0 = part.w0; i0 < part.w1; i0 += 32 * kStSteps) {
    uint32_t key[kStSteps], id[kStSteps];
    st_keys(q, i0, part.w1, key);
#pragma unroll
    for (int s = 0; s < kStSteps; ++s) {
      const int64_t i = i0 + 32 * s + lane;
      id[s] = q.ids && i < part.w1 ? __ldcg(q.ids + i) : static_cast<uint32_t>(i);
    }
#pragma unroll
    for (int s = 0; s < kStSteps; ++s) {
      if (i0 + 32 * s >= part.w1) break;
      const bool in = key[s] != 0xFFFFFFFFu;
      const uint32_t d = in ? st_digit(q, key[s]) : 0xFFFFFFFFu;
      const unsigned peers = __match_any_sync(0xFFFFFFFFu, d);
      const unsigned lower = peers & ((1u << lane) - 1);
      uint32_t p = 0;
      if (in) p = place[d] + __popc(lower);
      __syncwarp();
      if (in && lower == 0) place[d] += __popc(peers);
      __syncwarp();
      if (q.next_counts) {
        // Lanes that count in one place (those of a frequent token) do so together.
        const uint32_t to =
            in ? p / static_cast<uint32_t>(q.run) * q.buckets + ((key[s] >> (q.shift + 10)) & static_cast<uint32_t>(q.mask))
               : 0xFFFFFFFFu;
        const unsigned same = __match_any_sync(0xFFFFFFFFu, to);
        if (in && (same & ((1u << lane) - 1)) == 0) atomicAdd(q.next_counts + to, static_cast<uint32_t>(__popc(same)));
      }
      if (!in) continue;
      if (q.slots) {
        q.slots[i0 + 32 * s + lane] = static_cast<int32_t>(p);
      } else {
        q.keys_out[p] = key[s];
        q.ids_out[p] = id[s];
      }
    }
  }
}

__global__ void __launch_bounds__(kStThreads) st_place(const StArgs q) {
  extern __shared__ uint32_t hist[];
  __shared__ uint32_t warp_sums[kStWarps];
  griddep_launch_dependents();
  griddep_wait();
  if (static_cast<int>(blockIdx.x) < q.blocks) st_place_block(q, hist, warp_sums);
  else st_zero(q.zeros, q.zero_bytes, blockIdx.x - q.blocks, gridDim.x - q.blocks);
}

// Up to kStOneBlock entries in one launch, whatever the keys: an entry's place is the number of
// lower keys and of equal ones before it, counted over all keys by a warp for kStEach
// entries. (The kernels of lookup and gradient, replayed from a graph: 8192 tokens of 768, vocabulary
// 32768: 39 us, with one block's passes by digits 57; 2047 of 389, 32003: 21 and 27; 64 of 64, 1000: 8.9 and
// 9.7. Calls as they come take longer up to 8192 tokens, 60 to 70 us: the autograd engine's time on the host.)
constexpr int kStRankThreads = 256, kStEach = 4, kStRankEntries = kStRankThreads / 32 * kStEach;
__global__ void __launch_bounds__(kStRankThreads) st_rank(const StArgs q) {
  extern __shared__ uint32_t hist[];  // the keys
  griddep_launch_dependents();
  griddep_wait();
  if (static_cast<int>(blockIdx.x) >= q.blocks) {
    st_zero(q.zeros, q.zero_bytes, blockIdx.x - q.blocks, gridDim.x - q.blocks);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 31, n = static_cast<int>(q.n);
  if (blockIdx.x == 0 && tid == 0) *q.clear = 0u;
#pragma unroll 4
  for (int i = tid; i < n; i += kStRankThreads) hist[i] = st_key(q, i);
  __syncthreads();
  const int i0 = blockIdx.x * kStRankEntries + (tid >> 5) * kStEach, split = min(i0, n);
  uint32_t mine[kStEach];
  int count[kStEach] = {};
#pragma unroll
  for (int e = 0; e < kStEach; ++e) {
    mine[e] = hist[min(i0 + e, n - 1)];
#pragma unroll
    for (int f = 0; f < e; ++f) count[e] += lane == 0 && mine[f] == mine[e];
  }
#pragma unroll 4
  for (int j = lane; j < split; j += 32) {
    const uint32_t k = hist[j];
#pragma unroll
    for (int e = 0; e < kStEach; ++e) count[e] += k <= mine[e];
  }
#pragma unroll 4
  for (int j = split + lane; j < n; j += 32) {
    const uint32_t k = hist[j];
#pragma unroll
    for (int e = 0; e < kStEach; ++e) count[e] += k < mine[e];
  }
#pragma unroll
  for (int e = 0; e < kStEach; ++e) {
    const int place = __reduce_add_sync(0xFFFFFFFFu, count[e]);
    if (lane != e || i0 + e >= n) continue;
    q.keys_out[place] = mine[e];
    q.ids_out[place] = static_cast<uint32_t>(i0 + e);
  }
}

}  // namespace avey
