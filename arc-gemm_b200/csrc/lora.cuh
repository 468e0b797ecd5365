// lora.cuh — low-rank adapters of many requests beside a shared projection.
//
//   y[t] = act( x[t] w^T + bias + s_i (x[t] a_i^T) b_i^T ) + residual[t],   i = ids[t]
//
// The adapters' part is a longer contraction: row t's u[t] = s_i (x[t] a_i^T) follows x[t], and b_i's rows follow w's.
// lora_down_kernel writes u, in bf16 (the tensor cores' operand type, one rounding), and for every row tile of
// the product which adapters occur in it; the product (gemm_linear_stream.cuh, gemm_linear_pair.cuh) appends a block of
// up to 64 of the rank per such adapter, which leaves the rows of other adapters alone (the pair kernel's by
// tcgen05.mma's mask of output lanes, the streaming kernel's, whose lanes are columns, as zeros). So bias,
// activation and residual stay where they are, nothing of the output's size is written twice, and the price of a
// tile is its own adapters (a prompt's tile has one or two).
//
// lora_down_kernel. An item is one adapter of a block of 32 rows, the contraction split over a cluster of S
// blocks and eight warps each. The rows that have the adapter are packed into tiles of 16 (a decode batch has one or
// two per adapter), and both operands go from memory straight into the registers of mma.sync: a lane takes 16
// bytes of a row, the same 8 of 32 of the contraction for rows and adapter, so no layout has to be met
// in shared memory. Bound by the latency of those loads: a warp has one or two rounds of them. The partial sums
// are added over warps, then over the cluster in rank order.
#pragma once

#include "sm100.cuh"

namespace arcb {
namespace lora {

constexpr uint32_t kMaxAdapters = 1024;
constexpr uint32_t kMaxRank = 256;
constexpr uint32_t kNone = 0xFFFFFFFFu;

__device__ __forceinline__ uint32_t id_at(const void* ids, uint32_t wide, uint32_t adapters, uint32_t row) {
  const int64_t v = wide ? static_cast<int64_t>(__ldg(static_cast<const long long*>(ids) + row))
                         : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(ids) + row));
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

// One warp: zeros in the rows (128-byte lines) of an operand whose bit is set, whatever lies there.
template <uint32_t ROWS>
__device__ __forceinline__ void zero_rows(uint8_t* operand, const uint32_t (&mask)[(ROWS + 31u) / 32u], uint32_t lane) {
#pragma unroll
  for (uint32_t i = 0; i < (ROWS + 31u) / 32u; ++i) {
#pragma unroll
    for (uint32_t j = 0; j < 32u; j += 4u) {
      const uint32_t r = j + (lane >> 3);
      if (i * 32u + r < ROWS && ((mask[i] >> r) & 1u) != 0u) {
        *reinterpret_cast<uint4*>(operand + (i * 32u + r) * 128u + (lane & 7u) * 16u) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  }
}

// Rows of zeros keep other adapters' rows out of a product only if the adapter is finite: 0 times infinity is NaN, in
// rows of requests that have nothing to do with it. One warp looks through `rows` rows of an adapter's block (swizzled
// 128-byte lines, `cols` elements of each), sets what is not finite to zero, and notes in `spoilt` [row][words] that
// the rows of x in `own` get NaN there. Returns whether there was any.
template <uint32_t WORDS>
__device__ __forceinline__ bool take_out_nonfinite(uint8_t* operand, uint32_t rows, uint32_t cols, uint32_t (*spoilt)[WORDS],
                                                   const uint32_t (&own)[WORDS], uint32_t lane) {
  const uint32_t pieces = (cols + 7u) / 8u;  // 16 bytes each
  bool found = false;
  for (uint32_t i = lane; i < rows * pieces; i += 32u) {
    const uint32_t r = i / pieces, c = i % pieces;
    uint4* at = reinterpret_cast<uint4*>(operand + r * 128u + ((c ^ (r & 7u)) << 4));
    const uint4 v = *at;
    uint32_t word[4] = {v.x, v.y, v.z, v.w};
    bool bad = false;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      if ((word[k] & 0x7F80u) == 0x7F80u) word[k] &= 0xFFFF0000u, bad = true;
      if ((word[k] & 0x7F800000u) == 0x7F800000u) word[k] &= 0x0000FFFFu, bad = true;
    }
    if (bad) {
      *at = make_uint4(word[0], word[1], word[2], word[3]);
#pragma unroll
      for (uint32_t k = 0; k < WORDS; ++k) atomicOr(&spoilt[r][k], own[k]);
      found = true;
    }
  }
  return __any_sync(0xffffffffu, found);
}

// ---------------------------------------------------------------------------------
// lora_down_kernel
// ---------------------------------------------------------------------------------
constexpr uint32_t kDownWarps = 8;
constexpr uint32_t kDownThreads = 32 * kDownWarps;
constexpr uint32_t kDownRows = 32;  // rows of a block: one a lane

struct DownParams {
  const uint16_t* x;    // [M][ldx], 16-byte aligned rows
  const uint16_t* a;    // [adapters] x a_stride, [rank][lda], 16-byte aligned rows
  const float* scales;  // [adapters] or null
  const void* ids;      // [M]
  uint16_t* u;          // [M][ldu]
  uint16_t *counts, *lists;
  uint64_t ldx, lda, a_stride, ldu;
  uint32_t ids_wide, adapters, M, K, rank;
  uint32_t row_blocks, sets;       // blocks of rows; clusters that share a block's adapters
  uint32_t rank_parts, splits;     // parts of 8 RT of the rank; blocks of a cluster
  uint32_t tile_rows, tiles, cap;  // row tiles of the product
};

__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight elements of a row from k on, zeros behind the row's end and where there is no row.
__device__ __forceinline__ uint4 load8(const uint16_t* row, uint32_t k, uint32_t K) {
  if (row == nullptr || k >= K) return make_uint4(0u, 0u, 0u, 0u);
  if (k + 8u <= K) return __ldg(reinterpret_cast<const uint4*>(row + k));
  uint32_t v[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) {
    if (k + i < K) v[i >> 1] |= static_cast<uint32_t>(__ldg(row + k + i)) << ((i & 1u) * 16u);
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// The lane of the n-th set bit (n < popc).
__device__ __forceinline__ uint32_t nth_bit(uint32_t mask, uint32_t n) {
  return mask == 0xFFFFFFFFu ? n : __fns(mask, 0, int(n) + 1);
}

// Which adapters occur in row tile t, in the order of their first rows. One warp; `seen` has a bit an adapter.
__device__ __forceinline__ void list_tile(const DownParams& p, uint32_t t, uint32_t* seen, uint32_t lane) {
  seen[lane] = 0u;
  __syncwarp();
  uint32_t n = 0;
  const uint32_t end = min(p.M, (t + 1u) * p.tile_rows);
  for (uint32_t r0 = t * p.tile_rows; r0 < end; r0 += 32u) {
    const uint32_t id = r0 + lane < end ? id_at(p.ids, p.ids_wide, p.adapters, r0 + lane) : kNone;
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    const bool first = id != kNone && (same & ((1u << lane) - 1u)) == 0u && ((seen[id >> 5] >> (id & 31u)) & 1u) == 0u;
    const uint32_t firsts = __ballot_sync(0xffffffffu, first);
    if (first) {
      p.lists[size_t(t) * p.cap + n + __popc(firsts & ((1u << lane) - 1u))] = static_cast<uint16_t>(id);
      atomicOr(&seen[id >> 5], 1u << (id & 31u));
    }
    n += __popc(firsts);
    __syncwarp();
  }
  if (lane == 0) p.counts[t] = static_cast<uint16_t>(n);
}

// RT: tiles of 8 of the rank that a warp has; NW: groups of warps that share them out.
template <uint32_t RT, uint32_t NW>
__global__ void __launch_bounds__(kDownThreads) lora_down_kernel(const __grid_constant__ DownParams p) {
  constexpr uint32_t KW = kDownWarps / NW;   // warps along the contraction
  constexpr uint32_t kCols = RT * NW * 8;    // of the rank
  constexpr uint32_t kAhead = RT >= 4 ? 2 : 4;  // chunks of 32 whose loads are under way together
  __shared__ float sums[KW][kDownRows][kCols];
  __shared__ uint32_t seen[kMaxAdapters / 32];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t g8 = lane >> 2, q = lane & 3u;
  const uint32_t kw = warp % KW, nw = warp / KW;
  const uint32_t rank = p.splits > 1u ? cluster_ctarank() : 0u;
  // The product's weights do not wait for this grid, so it lets the product in at once, but only after what
  // precedes it has ended.
  pdl_wait();
  pdl_launch_dependents();

  const uint32_t cluster = blockIdx.x / p.splits;
  const uint32_t set = cluster % p.sets, rest = cluster / p.sets;
  const uint32_t r0 = rest % p.rank_parts * kCols, row0 = rest / p.rank_parts * kDownRows;
  const uint32_t id = row0 + lane < p.M ? id_at(p.ids, p.ids_wide, p.adapters, row0 + lane) : kNone;
  const uint32_t same = __match_any_sync(0xffffffffu, id);
  const uint32_t leaders = __ballot_sync(0xffffffffu, id != kNone && (same & ((1u << lane) - 1u)) == 0u);
  const uint32_t chunks = (p.K + 31u) / 32u;
  const uint32_t c0 = chunks * rank / p.splits, c1 = chunks * (rank + 1u) / p.splits;

  for (uint32_t n = set; n < uint32_t(__popc(leaders)); n += p.sets) {
    const uint32_t lead = nth_bit(leaders, n);
    const uint32_t adapter = __shfl_sync(0xffffffffu, id, lead), mask = __shfl_sync(0xffffffffu, same, lead);
    const uint32_t count = __popc(mask);
    // This lane's rows of x (g8 and 8 + g8 of up to two tiles) and of the adapter.
    const uint16_t *xr[4], *ar[RT];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t c = i * 8u + g8;
      xr[i] = c < count ? p.x + (row0 + nth_bit(mask, c)) * p.ldx : nullptr;
    }
#pragma unroll
    for (uint32_t i = 0; i < RT; ++i) {
      const uint32_t r = r0 + (nw * RT + i) * 8u + g8;
      ar[i] = r < p.rank ? p.a + adapter * p.a_stride + r * p.lda : nullptr;
    }
    float acc[2][RT][4];
#pragma unroll
    for (uint32_t m = 0; m < 2; ++m) {
#pragma unroll
      for (uint32_t i = 0; i < RT; ++i) acc[m][i][0] = acc[m][i][1] = acc[m][i][2] = acc[m][i][3] = 0.f;
    }
    const bool two = count > 16u;
    for (uint32_t c = c0 + kw; c < c1; c += KW * kAhead) {
      uint4 xv[kAhead][4], av[kAhead][RT];
#pragma unroll
      for (uint32_t h = 0; h < kAhead; ++h) {
        const uint32_t k = c + h * KW < c1 ? (c + h * KW) * 32u + q * 8u : p.K;
#pragma unroll
        for (uint32_t i = 0; i < RT; ++i) av[h][i] = load8(ar[i], k, p.K);
        xv[h][0] = load8(xr[0], k, p.K);
        xv[h][1] = load8(xr[1], k, p.K);
        xv[h][2] = two ? load8(xr[2], k, p.K) : make_uint4(0u, 0u, 0u, 0u);
        xv[h][3] = two ? load8(xr[3], k, p.K) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (uint32_t h = 0; h < kAhead; ++h) {
#pragma unroll
        for (uint32_t m = 0; m < 2; ++m) {
          if (m == 1 && !two) continue;
          const uint4 lo = xv[h][2 * m], hi = xv[h][2 * m + 1];
#pragma unroll
          for (uint32_t i = 0; i < RT; ++i) {
            mma_16x8x16(acc[m][i], lo.x, hi.x, lo.y, hi.y, av[h][i].x, av[h][i].y);
            mma_16x8x16(acc[m][i], lo.z, hi.z, lo.w, hi.w, av[h][i].z, av[h][i].w);
          }
        }
      }
    }
    // Warps, then blocks, in order.
#pragma unroll
    for (uint32_t m = 0; m < 2; ++m) {
#pragma unroll
      for (uint32_t i = 0; i < RT; ++i) {
        float* to = &sums[kw][m * 16u + g8][(nw * RT + i) * 8u + 2u * q];
        *reinterpret_cast<float2*>(to) = make_float2(acc[m][i][0], acc[m][i][1]);
        *reinterpret_cast<float2*>(to + 8 * kCols) = make_float2(acc[m][i][2], acc[m][i][3]);
      }
    }
    __syncthreads();
    float* mine = &sums[0][0][0];
    for (uint32_t o = threadIdx.x; o < count * kCols; o += kDownThreads) {
      float v = mine[o];
#pragma unroll
      for (uint32_t k = 1; k < KW; ++k) v += mine[k * kDownRows * kCols + o];
      mine[o] = v;
    }
    if (p.splits > 1u) {
      cluster_sync_all();
    } else {
      __syncthreads();
    }
    const float scale = p.scales != nullptr ? __ldg(p.scales + adapter) : 1.f;
    for (uint32_t o = threadIdx.x; o < count * kCols; o += kDownThreads) {
      const uint32_t row = o / kCols, r = r0 + o % kCols;
      if (row % p.splits != rank || r >= p.rank) continue;
      float v = 0.f;
      if (p.splits > 1u) {
        for (uint32_t i = 0; i < p.splits; ++i) v += ld_dsmem_f32(map_to_rank(mine + o, i));
      } else {
        v = mine[o];
      }
      p.u[(row0 + nth_bit(mask, row)) * p.ldu + r] = __bfloat16_as_ushort(__float2bfloat16_rn(scale * v));
    }
    if (p.splits > 1u) {
      cluster_sync_all();  // a peer may still be reading these sums
    } else {
      __syncthreads();
    }
  }
  for (uint32_t t = blockIdx.x; warp == 0 && t < p.tiles; t += gridDim.x) list_tile(p, t, seen, lane);
}

}  // namespace lora
}  // namespace arcb
