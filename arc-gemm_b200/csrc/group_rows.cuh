// group_rows.cuh — the choices of a router, sorted by group, on the GPU.
//
//   ids       [slots] group of each choice (slots = tokens x top, row-major); an id outside
//             [0, E) chooses no group and is ordered behind the last one
//   offsets   [E + 1] where each group's choices begin in the sorted order
//   rows      [slots] the token (slot / top) at each place of that order
//   positions [slots] the place of each choice: the inverse permutation
//
// A stable counting sort: inside a group, choices keep their order, so the result is unique.
// Every block counts its contiguous share of the slots, then places it: a choice's place is
// the slots of lower groups + the same group's slots in earlier blocks + in earlier warps of
// this block + in earlier lanes (match_any). Ids are read once per kernel (the second time
// from L2) and nothing is sorted by comparison; no atomic decides an order. Bound by latency:
// the 16 bytes a slot needs pass in about a microsecond even for half a million slots, the
// chain of count, sum over blocks and placement takes a few.
//
// Up to kOneBlockSlots slots one block does it all in one launch; above, a counting kernel
// runs first and leaves every block's histogram in a workspace.
#pragma once

#include "sm100.cuh"

namespace arcb {
namespace rows {

constexpr uint32_t kThreads = 1024;
constexpr uint32_t kWarps = kThreads / 32;
constexpr uint32_t kMaxBuckets = 1025;  // up to 1024 groups and "no group"
constexpr uint32_t kOneBlockSlots = 8192;

struct Params {
  const void* ids;
  int32_t* offsets;
  int32_t* rows;
  int32_t* positions;
  uint32_t* counts;  // [blocks][buckets] or null (one block)
  uint32_t slots, top, groups, blocks;
  uint32_t per_block;  // slots of a block, a multiple of kThreads
};

constexpr size_t smem_bytes(uint32_t groups) { return size_t(kWarps + 1) * (groups + 1) * 4; }

template <typename Id>
__device__ __forceinline__ uint32_t bucket_of(const Params& p, uint32_t slot) {
  const Id v = __ldg(static_cast<const Id*>(p.ids) + slot);
  return v < 0 || v >= static_cast<Id>(p.groups) ? p.groups : static_cast<uint32_t>(v);
}

template <typename Id>
__global__ void __launch_bounds__(kThreads) count_rows_kernel(const Params p) {
  extern __shared__ uint32_t hist[];
  pdl_launch_dependents();
  const uint32_t buckets = p.groups + 1u;
  for (uint32_t i = threadIdx.x; i < buckets; i += kThreads) hist[i] = 0u;
  __syncthreads();
  pdl_wait();
  const uint32_t begin = blockIdx.x * p.per_block, end = min(p.slots, begin + p.per_block);
  for (uint32_t i = begin + threadIdx.x; i < end; i += kThreads) atomicAdd(&hist[bucket_of<Id>(p, i)], 1u);
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < buckets; i += kThreads) p.counts[size_t(blockIdx.x) * buckets + i] = hist[i];
}

template <typename Id>
__global__ void __launch_bounds__(kThreads) place_rows_kernel(const Params p) {
  extern __shared__ uint32_t smem[];
  __shared__ uint32_t warp_sums[kWarps];
  const uint32_t buckets = p.groups + 1u;
  uint32_t* base = smem;             // [buckets] first place of this block's slots of a bucket
  uint32_t* counts = smem + buckets;  // [kWarps][buckets]: counts, then running places
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  pdl_launch_dependents();
  for (uint32_t i = threadIdx.x; i < buckets * kWarps; i += kThreads) counts[i] = 0u;
  __syncthreads();
  pdl_wait();

  // Every warp counts its own contiguous share.
  const uint32_t per_warp = p.per_block / kWarps;
  const uint32_t begin = min(p.slots, blockIdx.x * p.per_block + warp * per_warp);
  const uint32_t end = min(p.slots, begin + per_warp);
  uint32_t* mine = counts + warp * buckets;
  for (uint32_t i = begin + lane; i < end; i += 32u) atomicAdd(&mine[bucket_of<Id>(p, i)], 1u);

  // Slots of each bucket in all blocks (total) and in the blocks before this one (before).
  // kThreads / buckets threads share a bucket's column of the histograms.
  __syncthreads();
  if (p.counts == nullptr) {
    for (uint32_t b = threadIdx.x; b < buckets; b += kThreads) {
      uint32_t total = 0;
      for (uint32_t w = 0; w < kWarps; ++w) total += counts[w * buckets + b];
      base[b] = total;
    }
  } else {
    for (uint32_t b = threadIdx.x; b < buckets; b += kThreads) base[b] = 0u;
    __syncthreads();
    const uint32_t share = buckets < kThreads ? kThreads / buckets : 1u;
    for (uint32_t i = threadIdx.x; i < buckets * share; i += kThreads) {
      const uint32_t b = i % buckets, part = i / buckets;
      uint32_t total = 0;
#pragma unroll 8
      for (uint32_t k = part; k < p.blocks; k += share) total += p.counts[size_t(k) * buckets + b];
      atomicAdd(&base[b], total);
    }
  }
  __syncthreads();

  // Exclusive sum over the buckets (at most kMaxBuckets: two per thread).
  const uint32_t b0 = 2u * threadIdx.x;
  const uint32_t v0 = b0 < buckets ? base[b0] : 0u, v1 = b0 + 1u < buckets ? base[b0 + 1u] : 0u;
  uint32_t incl = v0 + v1;
#pragma unroll
  for (uint32_t d = 1; d < 32u; d <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 31u) warp_sums[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    uint32_t v = warp_sums[lane];
#pragma unroll
    for (uint32_t d = 1; d < 32u; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += o;
    }
    warp_sums[lane] = v;
  }
  __syncthreads();
  const uint32_t excl = incl - v0 - v1 + (warp > 0u ? warp_sums[warp - 1u] : 0u);
  if (b0 < buckets) base[b0] = excl;
  if (b0 + 1u < buckets) base[b0 + 1u] = excl + v0;
  if (blockIdx.x == 0) {
    if (b0 < buckets) p.offsets[b0] = static_cast<int32_t>(excl);
    if (b0 + 1u < buckets) p.offsets[b0 + 1u] = static_cast<int32_t>(excl + v0);
  }
  __syncthreads();

  // Add the earlier blocks' slots, then turn the warps' counts into first places.
  if (p.counts != nullptr) {
    const uint32_t share = buckets < kThreads ? kThreads / buckets : 1u;
    for (uint32_t i = threadIdx.x; i < buckets * share; i += kThreads) {
      const uint32_t b = i % buckets, part = i / buckets;
      uint32_t before = 0;
#pragma unroll 8
      for (uint32_t k = part; k < blockIdx.x; k += share) before += p.counts[size_t(k) * buckets + b];
      atomicAdd(&base[b], before);
    }
    __syncthreads();
  }
  for (uint32_t b = threadIdx.x; b < buckets; b += kThreads) {
    uint32_t at = base[b];
#pragma unroll 8
    for (uint32_t w = 0; w < kWarps; ++w) {
      const uint32_t c = counts[w * buckets + b];
      counts[w * buckets + b] = at;
      at += c;
    }
  }
  __syncthreads();

  // Place the slots, 32 at a time in order.
  for (uint32_t i0 = begin; i0 < end; i0 += 32u) {
    const uint32_t i = i0 + lane;
    const bool valid = i < end;
    const uint32_t b = valid ? bucket_of<Id>(p, i) : 0xFFFFFFFFu;
    const uint32_t same = __match_any_sync(0xffffffffu, b);
    const uint32_t rank = __popc(same & ((1u << lane) - 1u));
    const uint32_t at = valid ? mine[b] + rank : 0u;
    __syncwarp();
    if (valid && rank == 0u) mine[b] = at + __popc(same);
    __syncwarp();
    if (valid && at < p.slots) {  // always, unless the ids change under the call
      p.positions[i] = static_cast<int32_t>(at);
      p.rows[at] = static_cast<int32_t>(i / p.top);
    }
  }
}

}  // namespace rows
}  // namespace arcb
