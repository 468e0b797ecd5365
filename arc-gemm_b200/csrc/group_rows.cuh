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
// this block + in earlier lanes (match_any). Ids are read once per kernel and nothing is sorted
// by comparison; no atomic decides an order. Bound by latency: the 16 bytes a slot needs pass in
// about a microsecond even for half a million slots, the chain of count, sum over blocks and
// placement takes the rest. Measured: 65536 x 8 int64 ids 14.4 us, 16 x 8 ids 3.9 us.
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
constexpr uint32_t kKept = 8;  // ids a lane keeps between counting and placing
constexpr uint32_t kNone = 0xFFFFFFFFu;

struct Params {
  const void* ids;
  int32_t* offsets;
  int32_t* rows;
  int32_t* positions;
  uint32_t* counts;  // [buckets][counts_ld(blocks)] or null (one block)
  uint32_t slots, top, groups, blocks;
  uint32_t per_block;  // slots of a block, a multiple of kThreads
};

// A bucket's counts of all blocks lie together, in whole 16-byte vectors.
__host__ __device__ constexpr uint32_t counts_ld(uint32_t blocks) { return (blocks + 3u) & ~3u; }

constexpr size_t smem_bytes(uint32_t groups) { return size_t(kWarps + 2) * (groups + 1) * 4; }

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
  for (uint32_t i0 = begin + threadIdx.x; i0 < end; i0 += kThreads * kKept) {
    uint32_t b[kKept];  // loads first
#pragma unroll
    for (uint32_t j = 0; j < kKept; ++j) {
      const uint32_t i = i0 + j * kThreads;
      b[j] = i < end ? bucket_of<Id>(p, i) : kNone;
    }
#pragma unroll
    for (uint32_t j = 0; j < kKept; ++j) {
      if (b[j] != kNone) atomicAdd(&hist[b[j]], 1u);
    }
  }
  __syncthreads();
  const uint32_t ld = counts_ld(p.blocks);
  for (uint32_t i = threadIdx.x; i < buckets; i += kThreads) {
    uint32_t* row = p.counts + size_t(i) * ld;
    row[blockIdx.x] = hist[i];
    if (blockIdx.x == 0) {
      for (uint32_t k = p.blocks; k < ld; ++k) row[k] = 0u;
    }
  }
}

template <typename Id>
__global__ void __launch_bounds__(kThreads) place_rows_kernel(const Params p) {
  extern __shared__ uint32_t smem[];
  __shared__ uint32_t warp_sums[kWarps];
  const uint32_t buckets = p.groups + 1u;
  uint32_t* base = smem;                  // [buckets] first place of this block's slots of a bucket
  uint32_t* before = smem + buckets;      // [buckets]
  uint32_t* counts = smem + 2 * buckets;  // [kWarps][buckets]: counts, then running places
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  pdl_launch_dependents();
  for (uint32_t i = threadIdx.x; i < buckets * (kWarps + 2); i += kThreads) smem[i] = 0u;
  __syncthreads();
  pdl_wait();

  // Every warp counts its own contiguous share; the first kKept ids of a lane stay in registers.
  const uint32_t per_warp = p.per_block / kWarps;
  const uint32_t begin = min(p.slots, blockIdx.x * p.per_block + warp * per_warp);
  const uint32_t end = min(p.slots, begin + per_warp);
  uint32_t* mine = counts + warp * buckets;
  uint32_t kept[kKept];
#pragma unroll
  for (uint32_t j = 0; j < kKept; ++j) {
    const uint32_t i = begin + j * 32u + lane;
    kept[j] = i < end ? bucket_of<Id>(p, i) : kNone;
  }
#pragma unroll
  for (uint32_t j = 0; j < kKept; ++j) {
    if (kept[j] != kNone) atomicAdd(&mine[kept[j]], 1u);
  }
  for (uint32_t i = begin + kKept * 32u + lane; i < end; i += 32u) atomicAdd(&mine[bucket_of<Id>(p, i)], 1u);

  // Slots of each bucket in all blocks (base) and in the blocks before this one (before).
  // One warp adds a bucket's counts.
  if (p.counts == nullptr) {
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < buckets; b += kThreads) {
      uint32_t total = 0;
#pragma unroll 8
      for (uint32_t w = 0; w < kWarps; ++w) total += counts[w * buckets + b];
      base[b] = total;
    }
  } else {
    const uint32_t vecs = counts_ld(p.blocks) / 4u;
#pragma unroll 8
    for (uint32_t b = warp; b < buckets; b += kWarps) {
      const uint4* column = reinterpret_cast<const uint4*>(p.counts) + size_t(b) * vecs;
      uint32_t total = 0, earlier = 0;
      for (uint32_t v = lane; v < vecs; v += 32u) {
        const uint4 c = column[v];
        const uint32_t k = 4u * v;
        total += c.x + c.y + c.z + c.w;
        earlier += (k < blockIdx.x ? c.x : 0u) + (k + 1u < blockIdx.x ? c.y : 0u) + (k + 2u < blockIdx.x ? c.z : 0u) +
                   (k + 3u < blockIdx.x ? c.w : 0u);
      }
      total = __reduce_add_sync(0xffffffffu, total);
      earlier = __reduce_add_sync(0xffffffffu, earlier);
      if (lane == 0) {
        base[b] = total;
        before[b] = earlier;
      }
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
  if (b0 < buckets) base[b0] = excl + before[b0];
  if (b0 + 1u < buckets) base[b0 + 1u] = excl + v0 + before[b0 + 1u];
  if (blockIdx.x == 0) {
    if (b0 < buckets) p.offsets[b0] = static_cast<int32_t>(excl);
    if (b0 + 1u < buckets) p.offsets[b0 + 1u] = static_cast<int32_t>(excl + v0);
  }
  __syncthreads();

  // The warps' counts become first places.
  for (uint32_t b = threadIdx.x; b < buckets; b += kThreads) {
    uint32_t at = base[b];
#pragma unroll
    for (uint32_t w0 = 0; w0 < kWarps; w0 += 8u) {
      uint32_t c[8];
#pragma unroll
      for (uint32_t w = 0; w < 8u; ++w) c[w] = counts[(w0 + w) * buckets + b];
#pragma unroll
      for (uint32_t w = 0; w < 8u; ++w) {
        counts[(w0 + w) * buckets + b] = at;
        at += c[w];
      }
    }
  }
  __syncthreads();

  // Place the slots, 32 at a time in order.
  const auto place = [&](uint32_t i, uint32_t b) {
    const bool valid = b != kNone;
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
  };
#pragma unroll
  for (uint32_t j = 0; j < kKept; ++j) {
    const uint32_t i0 = begin + j * 32u;
    if (i0 < end) place(i0 + lane, kept[j]);
  }
  for (uint32_t i0 = begin + kKept * 32u; i0 < end; i0 += 32u) {
    const uint32_t i = i0 + lane;
    place(i, i < end ? bucket_of<Id>(p, i) : kNone);
  }
}

}  // namespace rows
}  // namespace arcb
