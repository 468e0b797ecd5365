// lora.cuh — low-rank adapters of many requests beside a shared projection.
//
//   y[t] = act( x[t] w^T + bias + s_i (x[t] a_i^T) b_i^T ) + residual[t],   i = ids[t]
//
// lora_down_kernel writes u[t] = s_i (x[t] a_i^T), in bf16 (the tensor cores' operand type, one rounding), and for every
// row tile of the product which adapters occur in it. Then the product, with bias, activation and residual where they
// were; nothing of the output's size passes through memory twice.
//
// * Many rows (gemm_linear_pair.cuh): the adapters' part is a longer contraction. u follows x and b's rows follow w's, a
//   block of up to 64 of the rank for each adapter of a tile, whose products leave the rows of other adapters as they
//   are (tcgen05.mma's mask of output lanes). A prompt's tile has one adapter or two, which is what it pays.
// * Few rows (gemm_linear_stream.cuh), where rows bring an adapter each and the output's lanes are columns: warps
//   that wait for the stream of weights compute u b^T, adapter by adapter. As blocks of the contraction 25 rows
//   with 21 adapters cost 38 us beside the stream's 25.
//
// lora_down_kernel. An item is a block of 32 rows times as many of its adapters as have 64 rows together, the contraction
// split over a cluster of S blocks and eight warps each: warp i takes every eighth box of 64 by a ring slot
// of its own. All 32 rows are multiplied by all the adapters (the pipe idles either way) and a row's own part kept.
// Bound by latency for few rows, by the loads of x and the adapters from L2 for many. The partial sums are added over
// warps, then sent to the block of the cluster that owns the row, which adds them in rank order (with cluster barriers
// around reads of the peers' sums that took 4.3 us of the 8 of one token; sent, 1.5). (Straight from memory into registers, without the ring, 4096 rows of 4096
// by rank 64 took 59 us.)
#pragma once

#include "sm100.cuh"

namespace arcb {
namespace lora {

constexpr uint32_t kMaxAdapters = 1024;
constexpr uint32_t kMaxRank = 256;
constexpr uint32_t kNone = 0xFFFFFFFFu;

// The product's blocks start beside lora_down_kernel's, so what they read before they wait for it, ids and b, comes past
// the L1 cache, whose lines may be older.
__device__ __forceinline__ uint32_t id_at(const void* ids, uint32_t wide, uint32_t adapters, uint32_t row) {
  const int64_t v = wide ? static_cast<int64_t>(__ldcg(static_cast<const long long*>(ids) + row))
                         : static_cast<int64_t>(__ldcg(static_cast<const int32_t*>(ids) + row));
  return v < 0 || v >= static_cast<int64_t>(adapters) ? kNone : static_cast<uint32_t>(v);
}

// What the product needs of the adapters.
struct Extra {
  CUtensorMap tm_u;       // {rank, M, 1}, box {64, rows of a tile's operand, 1}, SW128
  CUtensorMap tm_b;       // {rank, N, adapters}, box {64, columns of a tile's operand, 1}, SW128
  const uint16_t* counts; // [row tiles]: adapters that occur
  const uint16_t* lists;  // [row tiles][cap]: which, in the order of their first rows
  const void* ids;        // [rows]
  uint32_t ids_wide, adapters, rows, rank, cap;
  // The streaming kernel's: u and b themselves, and where it leaves the adapters' sums.
  const uint16_t *u, *b;
  float* sums;  // [rows][N]
  uint64_t ldu, ldb, b_stride;
};

// The adapters of a row tile, as blocks of 64 of the rank. For use behind griddepcontrol.wait.
struct TileList {
  uint32_t blocks, per;
  const uint16_t* list;
  __device__ __forceinline__ TileList(const Extra& e, uint32_t tile)
      : per((e.rank + 63u) / 64u), list(e.lists + size_t(tile) * e.cap) {
    blocks = min(uint32_t(__ldcg(e.counts + tile)), e.cap) * per;
  }
  __device__ __forceinline__ uint32_t adapter(uint32_t i) const { return __ldcg(list + (per == 1u ? i : i / per)); }
  __device__ __forceinline__ uint32_t column(uint32_t i) const { return per == 1u ? 0u : i % per * 64u; }
};

// UMMA steps of 16 that block i of a list has.
__device__ __forceinline__ uint32_t steps_of(const Extra& e, uint32_t i) {
  const uint32_t per = (e.rank + 63u) / 64u;
  const uint32_t left = e.rank - (per == 1u ? 0u : i % per * 64u);
  return left >= 64u ? 4u : (left + 15u) / 16u;
}

// The adapters of ROWS rows from `row0` on, a row a lane at a time.
template <uint32_t ROWS>
struct RowAdapters {
  static constexpr uint32_t kSets = (ROWS + 31u) / 32u;
  uint32_t id[kSets];
  __device__ __forceinline__ RowAdapters(const Extra& e, uint32_t row0, uint32_t lane) {
#pragma unroll
    for (uint32_t i = 0; i < kSets; ++i) {
      const uint32_t r = i * 32u + lane;
      id[i] = r < ROWS && row0 + r < e.rows ? id_at(e.ids, e.ids_wide, e.adapters, row0 + r) : kNone;
    }
  }
  // One warp: the rows with another adapter or none, a bit each.
  __device__ __forceinline__ void others(uint32_t adapter, uint32_t (&mask)[kSets]) const {
#pragma unroll
    for (uint32_t i = 0; i < kSets; ++i) mask[i] = __ballot_sync(0xffffffffu, id[i] != adapter);
  }
};

__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Elements of a row by aligned vectors: where the row ends inside one, `keep` takes what lies behind it out (the vector
// itself has an element of the row, so it is there to be read).
template <uint32_t WORDS>
struct Keep {
  uint32_t mask[WORDS];
  __device__ __forceinline__ Keep(uint32_t k, uint32_t end) {
#pragma unroll
    for (uint32_t i = 0; i < WORDS; ++i) {
      mask[i] = (k + 2u * i < end ? 0x0000FFFFu : 0u) | (k + 2u * i + 1u < end ? 0xFFFF0000u : 0u);
    }
  }
};
__device__ __forceinline__ uint4 load8(const uint16_t* p, bool there, const Keep<4>& keep) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  // volatile: not to be moved behind a wait that it is meant to pass
  if (there) asm volatile("ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return make_uint4(v.x & keep.mask[0], v.y & keep.mask[1], v.z & keep.mask[2], v.w & keep.mask[3]);
}
__device__ __forceinline__ uint2 load4(const uint16_t* p, bool there, const Keep<2>& keep) {
  uint2 v = make_uint2(0u, 0u);
  if (there) asm volatile("ld.global.cg.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return make_uint2(v.x & keep.mask[0], v.y & keep.mask[1]);
}

// The lane of the n-th set bit (n < popc).
__device__ __forceinline__ uint32_t nth_bit(uint32_t mask, uint32_t n) {
  return mask == 0xFFFFFFFFu ? n : __fns(mask, 0, int(n) + 1);
}

// u b^T of a tile of ROWS rows and COLS columns, fp32, to `sums`, by four warps: an adapter each in turn, of the
// adapters in the order of their first rows those with index `part` modulo `parts`. The rows of one adapter are
// packed into tiles of 8, the columns are the 16 of mma.sync; operands go from memory straight into the registers, a
// lane takes 16 bytes of a row (8 where the rank is 16), the same elements for both. Beside a stream of weights a load takes
// microseconds, so what does not depend on u is under way before u is there. Contains griddepcontrol.wait. `added`: the
// rows that were written, a bit each.
template <uint32_t ROWS, uint32_t COLS>
__device__ __forceinline__ void adapter_sums(const Extra& e, uint32_t row0, uint32_t f0, uint32_t cols, uint32_t part,
                                             uint32_t parts, uint32_t warp, uint32_t lane, uint32_t (&added)[(ROWS + 31u) / 32u]) {
  constexpr uint32_t kSets = (ROWS + 31u) / 32u, kBlocks = COLS / 16u;
  const uint32_t g8 = lane >> 2, q = lane & 3u;
  const RowAdapters<ROWS> rows(e, row0, lane);
  // Rows that are the first with their adapter, a bit each.
  uint32_t firsts[kSets], n = 0;
#pragma unroll
  for (uint32_t k = 0; k < kSets; ++k) {
    const uint32_t same = __match_any_sync(0xffffffffu, rows.id[k]);  // of all lanes, those without an adapter too
    bool first = rows.id[k] != kNone && (same & ((1u << lane) - 1u)) == 0u;
    if (k > 0) {
#pragma unroll 1  // (an instruction that is not in the cache yet costs a short launch more than a loop does)
      for (uint32_t l = 0; l < 32u; ++l) {
#pragma unroll
        for (uint32_t j = 0; j < k; ++j) {
          const uint32_t earlier = __shfl_sync(0xffffffffu, rows.id[j], l);  // of all lanes, whatever `first` is
          if (earlier == rows.id[k]) first = false;
        }
      }
    }
    firsts[k] = __ballot_sync(0xffffffffu, first);
    n += __popc(firsts[k]);
  }
  // The adapter with index i, and its rows.
  const auto adapter_at = [&](uint32_t i, uint32_t (&own)[kSets]) {
    uint32_t adapter = 0, left = i;
#pragma unroll
    for (uint32_t k = 0; k < kSets; ++k) {
      const uint32_t here = __popc(firsts[k]);
      if (left < here) adapter = __shfl_sync(0xffffffffu, rows.id[k], nth_bit(firsts[k], left));
      left = left < here ? kNone : left == kNone ? kNone : left - here;
    }
    rows.others(adapter, own);
#pragma unroll
    for (uint32_t k = 0; k < kSets; ++k) own[k] = ~own[k];
    return adapter;
  };
  for (uint32_t i = part; i < n; i += parts) {
    uint32_t own[kSets];
    const uint32_t adapter = adapter_at(i, own);
#pragma unroll
    for (uint32_t k = 0; k < kSets; ++k) added[k] |= own[k];
    if ((i - part) / parts % 4u != warp) continue;
    for (uint32_t f = lane; f < COLS && f0 + f < cols; f += 32u) {
      const uint16_t* row = e.b + adapter * e.b_stride + size_t(f0 + f) * e.ldb;
      for (uint32_t r = 0; r < e.rank; r += 64u) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + r));
    }
  }
  const auto row_of = [&](const uint32_t (&own)[kSets], uint32_t c) {
    uint32_t r = 0, left = c;
#pragma unroll
    for (uint32_t k = 0; k < kSets; ++k) {
      const uint32_t here = __popc(own[k]);
      if (left < here) r = k * 32u + nth_bit(own[k], left);
      left = left < here ? kNone : left == kNone ? kNone : left - here;
    }
    return row0 + r;
  };
  // Sums of 8 rows from c0 on: this lane has two of them, in columns g8 and g8 + 8 of every 16.
  const auto store = [&](const uint32_t (&own)[kSets], uint32_t c0, uint32_t count, const float (&acc)[kBlocks][4]) {
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
      const uint32_t c = c0 + 2u * q + j;
      if (c >= count) continue;
      float* to = e.sums + size_t(row_of(own, c)) * cols + f0 + g8;
#pragma unroll
      for (uint32_t m = 0; m < kBlocks; ++m) {
        if (f0 + m * 16u + g8 < cols) to[m * 16u] = acc[m][j];
        if (f0 + m * 16u + g8 + 8u < cols) to[m * 16u + 8u] = acc[m][2 + j];
      }
    }
  };
  bool waited = false;
  if (e.rank <= 16u && n > 4u * parts) {
    // A rank of 16 is one step with four elements a lane, so that three adapters fit in the registers at once (32
    // rows by 14336 x 4096, 21 adapters: 33.2 us one by one, 28.7 so).
    constexpr uint32_t kAtOnce = 3;
    const Keep<2> keep(q * 4u, e.rank);
    const bool k_there = q * 4u < e.rank;
    for (uint32_t i0 = part + parts * warp; i0 < n; i0 += parts * 4u * kAtOnce) {
      uint32_t own[kAtOnce][kSets], count[kAtOnce];
      uint2 lo[kAtOnce][kBlocks], hi[kAtOnce][kBlocks];
#pragma unroll
      for (uint32_t h = 0; h < kAtOnce; ++h) {
        const uint32_t i = i0 + h * parts * 4u;
        count[h] = 0;
        if (i >= n) continue;
        const uint16_t* b = e.b + adapter_at(i, own[h]) * e.b_stride;
#pragma unroll
        for (uint32_t k = 0; k < kSets; ++k) count[h] += __popc(own[h][k]);
#pragma unroll
        for (uint32_t m = 0; m < kBlocks; ++m) {
          const uint32_t f = f0 + m * 16u + g8;
          lo[h][m] = load4(b + size_t(f) * e.ldb + q * 4u, k_there && f < cols, keep);
          hi[h][m] = load4(b + size_t(f + 8u) * e.ldb + q * 4u, k_there && f + 8u < cols, keep);
        }
      }
      if (!waited) {
        pdl_wait();
        waited = true;
      }
      uint2 v[kAtOnce];  // of the first 8 rows
      const auto load_u = [&](uint32_t h, uint32_t c0) {
        uint2 r = make_uint2(0u, 0u);
        if (c0 + g8 < count[h] && q * 4u < e.ldu) {
          r = __ldcg(reinterpret_cast<const uint2*>(e.u + size_t(row_of(own[h], c0 + g8)) * e.ldu + q * 4u));
        }
        return r;
      };
#pragma unroll
      for (uint32_t h = 0; h < kAtOnce; ++h) v[h] = load_u(h, 0u);
#pragma unroll
      for (uint32_t h = 0; h < kAtOnce; ++h) {
        for (uint32_t c0 = 0; c0 < count[h]; c0 += 8u) {
          if (c0 > 0u) v[h] = load_u(h, c0);
          float acc[kBlocks][4];
#pragma unroll
          for (uint32_t m = 0; m < kBlocks; ++m) {
            acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
            mma_16x8x16(acc[m], lo[h][m].x, hi[h][m].x, lo[h][m].y, hi[h][m].y, v[h].x, v[h].y);
          }
          store(own[h], c0, count[h], acc);
        }
      }
    }
  } else {
    for (uint32_t i = part + parts * warp; i < n; i += parts * 4u) {
      uint32_t own[kSets], count = 0;
      const uint16_t* b = e.b + adapter_at(i, own) * e.b_stride;
#pragma unroll
      for (uint32_t k = 0; k < kSets; ++k) count += __popc(own[k]);
      for (uint32_t c0 = 0; c0 < count; c0 += 8u) {
        const uint16_t* u = c0 + g8 < count ? e.u + size_t(row_of(own, c0 + g8)) * e.ldu : nullptr;
        float acc[kBlocks][4];
#pragma unroll
        for (uint32_t m = 0; m < kBlocks; ++m) acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
        for (uint32_t k = 0; k < e.rank; k += 32u) {
          uint4 lo[kBlocks], hi[kBlocks];
          const uint32_t kq = k + q * 8u;
          const Keep<4> keep(kq, e.rank);
#pragma unroll
          for (uint32_t m = 0; m < kBlocks; ++m) {
            const uint32_t f = f0 + m * 16u + g8;
            lo[m] = load8(b + size_t(f) * e.ldb + kq, kq < e.rank && f < cols, keep);
            hi[m] = load8(b + size_t(f + 8u) * e.ldb + kq, kq < e.rank && f + 8u < cols, keep);
          }
          if (!waited) {
            pdl_wait();
            waited = true;
          }
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          // Rows of u are padded to 16 bytes with zeros.
          if (u != nullptr && kq < e.rank) v = __ldcg(reinterpret_cast<const uint4*>(u + kq));
#pragma unroll
          for (uint32_t m = 0; m < kBlocks; ++m) {
            mma_16x8x16(acc[m], lo[m].x, hi[m].x, lo[m].y, hi[m].y, v.x, v.y);
            mma_16x8x16(acc[m], lo[m].z, hi[m].z, lo[m].w, hi[m].w, v.z, v.w);
          }
        }
        store(own, c0, count, acc);
      }
    }
  }
  if (!waited) pdl_wait();
}

// ---------------------------------------------------------------------------------
// lora_down_kernel
// ---------------------------------------------------------------------------------
constexpr uint32_t kDownWarps = 8;  // and one for the loads
constexpr uint32_t kDownThreads = 32 * (kDownWarps + 1);
constexpr uint32_t kDownRows = 32;  // rows of a block: one a lane
constexpr uint32_t kDownCols = 64;  // rows of adapters
constexpr uint32_t kDownXBytes = kDownRows * 128, kDownSlotBytes = kDownXBytes + kDownCols * 128;
constexpr uint32_t kDownGotBytes = kDownRows * kDownCols * 4;
constexpr uint32_t kDownSmem = kDownWarps * kDownSlotBytes + kDownGotBytes + 1024;
static_assert(kDownWarps * kDownRows * kDownCols * 4 <= kDownWarps * kDownSlotBytes, "the sums reuse the ring");

struct DownParams {
  CUtensorMap tm_x;     // {K, M}, box {64, 32}, SW128
  CUtensorMap tm_a;     // {K, rank, adapters}, box {64, RS, 1}, SW128
  const float* scales;  // [adapters] or null
  const void* ids;      // [M]
  uint16_t* u;          // [M][ldu]
  uint16_t *counts, *lists;  // null where the product streams
  uint64_t ldu;
  uint32_t ids_wide, adapters, M, K, rank;
  uint32_t row_blocks, sets;       // blocks of rows; clusters that share a block's adapters
  uint32_t rank_parts, splits;     // parts of 64 of the rank; blocks of a cluster
  uint32_t tile_rows, tiles, cap;  // row tiles of the product
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// Which adapters occur in row tile t, in the order of their first rows. One warp; `seen` has a bit an adapter.
__device__ __forceinline__ void list_tile(const DownParams& p, uint32_t t, uint32_t* seen, uint32_t lane) {
  constexpr uint32_t kSets = 8;  // tiles have 256 rows at most; their ids are loaded together
  const uint32_t first = t * p.tile_rows, end = min(p.M, first + p.tile_rows);
  uint32_t ids[kSets];
#pragma unroll
  for (uint32_t i = 0; i < kSets; ++i) {
    const uint32_t r = first + i * 32u + lane;
    ids[i] = r < end ? id_at(p.ids, p.ids_wide, p.adapters, r) : kNone;
  }
  seen[lane] = 0u;
  __syncwarp();
  uint32_t n = 0;
#pragma unroll
  for (uint32_t i = 0; i < kSets; ++i) {
    const uint32_t id = ids[i];
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    const bool is_new = id != kNone && (same & ((1u << lane) - 1u)) == 0u && ((seen[id >> 5] >> (id & 31u)) & 1u) == 0u;
    const uint32_t news = __ballot_sync(0xffffffffu, is_new);
    if (is_new) {
      p.lists[size_t(t) * p.cap + n + __popc(news & ((1u << lane) - 1u))] = static_cast<uint16_t>(id);
      atomicOr(&seen[id >> 5], 1u << (id & 31u));
    }
    n += __popc(news);
    __syncwarp();
  }
  if (lane == 0) p.counts[t] = static_cast<uint16_t>(n);
}

// Four elements of u, zeros behind the rank.
__device__ __forceinline__ void store_u(const DownParams& p, uint32_t row, uint32_t r, float scale, const float4& v) {
  if (r >= p.ldu) return;
  uint2 w;
  w.x = pack_bf16x2(r < p.rank ? scale * v.x : 0.f, r + 1u < p.rank ? scale * v.y : 0.f);
  w.y = pack_bf16x2(r + 2u < p.rank ? scale * v.z : 0.f, r + 3u < p.rank ? scale * v.w : 0.f);
  *reinterpret_cast<uint2*>(p.u + row * p.ldu + r) = w;
}

// RS: rows that an adapter has among the 64.
template <uint32_t RS>
__global__ void __launch_bounds__(kDownThreads, 2) lora_down_kernel(const __grid_constant__ DownParams p) {
  constexpr uint32_t kGroup = kDownCols / RS;  // adapters of an item
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ uint64_t full[kDownWarps], empty[kDownWarps], got_all;
  __shared__ uint32_t seen[kMaxAdapters / 32];
  __shared__ uint32_t abort_flag;
  uint8_t* ring = smem_raw + smem_align_pad(smem_raw);
  const uint32_t warp = warp_idx_sync(), lane = threadIdx.x & 31u;
  const uint32_t rank = p.splits > 1u ? cluster_ctarank() : 0u;
  volatile uint32_t* abort = &abort_flag;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&p.tm_x);
    tma_prefetch_desc(&p.tm_a);
    for (uint32_t i = 0; i < kDownWarps; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&got_all, 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  if (p.splits > 1u) cluster_arrive();  // this block is there, and its barriers
  // The product's weights do not wait for this grid, so it lets the product in at once, but only after what
  // precedes it has ended.
  pdl_wait();
  pdl_launch_dependents();

  const uint32_t cluster = blockIdx.x / p.splits;
  const uint32_t set = cluster % p.sets, rest = cluster / p.sets;
  const uint32_t r0 = rest % p.rank_parts * kDownCols, row0 = rest / p.rank_parts * kDownRows;
  const uint32_t id = row0 + lane < p.M ? id_at(p.ids, p.ids_wide, p.adapters, row0 + lane) : kNone;
  const uint32_t same = __match_any_sync(0xffffffffu, id);
  const uint32_t leaders = __ballot_sync(0xffffffffu, id != kNone && (same & ((1u << lane) - 1u)) == 0u);
  // This lane's row: the place of its adapter among the block's.
  const uint32_t place = id == kNone ? kNone : __popc(leaders & ((1u << (__ffs(same) - 1)) - 1u));
  const uint32_t distinct = __popc(leaders), boxes = (p.K + 63u) / 64u;
  const uint32_t b0 = boxes * rank / p.splits, own = boxes * (rank + 1u) / p.splits - b0;
  float* sums = reinterpret_cast<float*>(ring);  // [kDownWarps][kDownRows][kDownCols]
  // What the cluster's blocks send this one, for the rows rank, rank + S, ...: [S][kDownRows / S][kDownCols].
  float* got = reinterpret_cast<float*>(ring + kDownWarps * kDownSlotBytes);
  // A scale is on its way before it is needed. (A plain load: the launch in front may write the scales while this block is
  // there already, so they are not read-only to it.)
  const float scale = id != kNone && p.scales != nullptr ? p.scales[id] : 1.f;

  // The row tiles' lists are made by blocks that seldom have an adapter to work on.
  bool lists = p.lists != nullptr && warp == kDownWarps && rank == 0u && set + 1u == p.sets;
  const auto make_lists = [&]() {
    for (uint32_t t = rest; lists && t < p.tiles; t += p.row_blocks * p.rank_parts) list_tile(p, t, seen, lane);
    lists = false;
  };
  uint32_t parity = 0;
  uint32_t uses = 0;  // of the ring slot: a consumer's by its warp, a loader's by its lane
  bool ok = true;
  for (uint32_t g = set * kGroup; g < distinct; g += p.sets * kGroup) {
    const uint32_t adapters = min(kGroup, distinct - g);
    float acc[2][kDownCols / 8][4];
    if (warp == kDownWarps) {
      // ---------------------------------------------------------- loads: lane i for warp i
      uint32_t adapter[kGroup];
#pragma unroll
      for (uint32_t i = 0; i < kGroup; ++i) {
        adapter[i] = __shfl_sync(0xffffffffu, id, i < adapters ? nth_bit(leaders, g + i) : 0u);
      }
      if (lane < kDownWarps) {
        uint8_t* slot = ring + lane * kDownSlotBytes;
        for (uint32_t b = lane; ok && b < own; b += kDownWarps) {
          ok = mbar_wait(&empty[lane], (uses & 1u) ^ 1u, abort, kStatusTimeoutProducer);
          if (!ok) break;
          mbar_arrive_expect_tx(&full[lane], kDownXBytes + adapters * RS * 128u);
          const int32_t k = int32_t((b0 + b) * 64u);
          tma_load_2d(&p.tm_x, &full[lane], slot, k, int32_t(row0), kCacheEvictNormal);
#pragma unroll
          for (uint32_t i = 0; i < kGroup; ++i) {
            if (i < adapters) {
              tma_load_3d(&p.tm_a, &full[lane], slot + kDownXBytes + i * RS * 128u, k, int32_t(r0), int32_t(adapter[i]),
                          kCacheEvictNormal);
            }
          }
          ++uses;
        }
      }
      __syncwarp();
      make_lists();  // while the loads are on their way
      // Loads land before the ring is used for the sums, and before the block may exit.
      if (lane < kDownWarps && uses > 0u) mbar_drain(&full[lane], (uses - 1u) & 1u);
      __syncwarp();
    } else {
      // ---------------------------------------------------------- products
#pragma unroll
      for (uint32_t m = 0; m < 2; ++m) {
#pragma unroll
        for (uint32_t j = 0; j < kDownCols / 8; ++j) acc[m][j][0] = acc[m][j][1] = acc[m][j][2] = acc[m][j][3] = 0.f;
      }
      const uint32_t x_at = smem_u32(ring + warp * kDownSlotBytes), a_at = x_at + kDownXBytes;
      for (uint32_t b = warp; b < own; b += kDownWarps) {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[warp], uses & 1u, abort, kStatusTimeoutMma));
        ++uses;
        if (!ok) continue;
#pragma unroll
        for (uint32_t half = 0; half < 2; ++half) {  // 32 of the contraction
          uint32_t xa[2][2][4];
#pragma unroll
          for (uint32_t m = 0; m < 2; ++m) {
#pragma unroll
            for (uint32_t k = 0; k < 2; ++k) {
              const uint32_t row = m * 16u + (lane & 15u), chunk = half * 4u + k * 2u + (lane >> 4);
              ldmatrix_x4(x_at + row * 128u + ((chunk ^ (row & 7u)) << 4), xa[m][k]);
            }
          }
#pragma unroll
          for (uint32_t i = 0; i < kGroup; ++i) {
            if (i < adapters) {
#pragma unroll
              for (uint32_t j8 = 0; j8 < RS / 8; ++j8) {
                const uint32_t j = i * (RS / 8) + j8;
                uint32_t v[4];
                const uint32_t row = lane & 7u, chunk = half * 4u + (lane >> 3);
                ldmatrix_x4(a_at + (j * 8u + row) * 128u + ((chunk ^ row) << 4), v);
#pragma unroll
                for (uint32_t m = 0; m < 2; ++m) {
#pragma unroll
                  for (uint32_t k = 0; k < 2; ++k) {
                    mma_16x8x16(acc[m][j], xa[m][k][0], xa[m][k][1], xa[m][k][2], xa[m][k][3], v[2 * k], v[2 * k + 1]);
                  }
                }
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[warp]);
      }
    }
    __syncthreads();  // the ring is free
    if (warp < kDownWarps) {
#pragma unroll
      for (uint32_t m = 0; m < 2; ++m) {
#pragma unroll
        for (uint32_t j = 0; j < kDownCols / 8; ++j) {
          if (j < adapters * (RS / 8)) {
            float* to = sums + (warp * kDownRows + m * 16u + (lane >> 2)) * kDownCols + j * 8u + 2u * (lane & 3u);
            *reinterpret_cast<float2*>(to) = make_float2(acc[m][j][0], acc[m][j][1]);
            *reinterpret_cast<float2*>(to + 8 * kDownCols) = make_float2(acc[m][j][2], acc[m][j][3]);
          }
        }
      }
    }
    __syncthreads();
    // A row's own adapter, four of its rank a lane: the warps' sums are added and sent to the row's owner.
    constexpr uint32_t kLanes = RS / 4u, kRowsAtOnce = 32u / kLanes;
    const uint32_t r4 = lane % kLanes * 4u;
    const bool last = g + p.sets * kGroup >= distinct;
    const uint32_t per = kDownRows / p.splits;
    uint32_t mine = 0;  // rows of this block that others send sums for
    if (p.splits > 1u) {
      if (g == set * kGroup) cluster_wait();
      mine = __popc(__ballot_sync(0xffffffffu, place - g < adapters && lane % p.splits == rank));
      if (threadIdx.x == 0) mbar_arrive_expect_tx(&got_all, mine * RS * 4u * p.splits);
    }
    for (uint32_t first = warp * kRowsAtOnce; first < kDownRows; first += (kDownWarps + 1u) * kRowsAtOnce) {
      const uint32_t row = first + lane / kLanes;
      const uint32_t at = __shfl_sync(0xffffffffu, place, row) - g;  // wraps around for rows of other items
      const float row_scale = __shfl_sync(0xffffffffu, scale, row);
      if (at < adapters) {
        const float* from = sums + row * kDownCols + at * RS + r4;
        float4 v = *reinterpret_cast<const float4*>(from);
#pragma unroll
        for (uint32_t k = 1; k < kDownWarps; ++k) {
          const float4 o = *reinterpret_cast<const float4*>(from + k * kDownRows * kDownCols);
          v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
        }
        if (p.splits > 1u) {
          const uint32_t owner = row % p.splits;
          store_async(map_to_rank(got + (rank * per + row / p.splits) * kDownCols + r4, owner), v, map_to_rank(&got_all, owner));
        } else {
          store_u(p, row0 + row, r0 + r4, row_scale, v);
        }
      }
    }
    if (p.splits > 1u) {
      // All that is sent here lands before this block may exit, whatever has been abandoned: a peer's sums may come after
      // the limits of its own waits.
      if (mine > 0u || !last) mbar_drain(&got_all, parity, 4u * kWaitTimeoutNs);
      parity ^= 1u;
      for (uint32_t first = warp * kRowsAtOnce; first < per; first += (kDownWarps + 1u) * kRowsAtOnce) {
        const uint32_t i = first + lane / kLanes, row = i < per ? i * p.splits + rank : 0u;
        const uint32_t at = __shfl_sync(0xffffffffu, place, row) - g;
        const float row_scale = __shfl_sync(0xffffffffu, scale, row);
        if (i < per && at < adapters) {
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          for (uint32_t k = 0; k < p.splits; ++k) {
            const float4 o = *reinterpret_cast<const float4*>(got + (k * per + i) * kDownCols + r4);
            v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
          }
          store_u(p, row0 + row, r0 + r4, row_scale, v);
        }
      }
    }
    if (!last) {
      fence_proxy_async_smem();  // the next item's loads come behind these accesses
      if (p.splits > 1u) {
        cluster_sync_all();  // and its sums behind the reads of these
      } else {
        __syncthreads();
      }
    }
  }
  if (p.splits > 1u && set * kGroup >= distinct) cluster_wait();  // of the arrival above
  make_lists();  // where a block had no adapters
}

}  // namespace lora
}  // namespace arcb
