// gemm_linear_stream.cuh — out[t, f] = epilogue( sum_k x[t, k] w[e, f, k] ), bf16, for few rows.
//
// The rows are few (a decode batch, or an expert's share of one), so the weights are the
// traffic and the kernel is built to stream them: the 128 weight rows of a tile are the
// UMMA M operand and BN rows of x its N operand, so that a small batch costs a small N and
// not a padded M. One output tile per block, K split over a cluster of S blocks when there
// are fewer tiles than block slots; the partial sums meet in distributed shared memory and
// are added in rank order, so the result does not depend on timing.
//
// Bound by: HBM (weights, 2 bytes each, read once). Two blocks fit on an SM (about 110 KB of
// shared memory each), so one block's prologue and epilogue run under the other's stream and
// about 200 KB of loads are in flight per SM. Measured, one call after another on several sets of
// inputs: 16 rows, 14336 x 4096 with bias, GELU and residual 25.3 us, 4.6 TB/s of weights (one wave
// of blocks: some 7 us are the first bytes' way, the reduction and the epilogue); one row, 4096 x
// 4096 8.3 us.
//
// W_MN = false: w is [E][N][K], K contiguous: the forward product.
// W_MN = true:  the roles of N and K are exchanged: out[t, f] = sum_n dy[t, n] w[e, n, f], the
//               gradient of the rows. w is read as it lies, features contiguous (MN-major).
//
// Roles (192 threads): warp 0 TMA producer, warp 1 UMMA issuer and TMEM owner, warps 2-5
// epilogue (TMEM lane quarter = warp % 4). In the accumulator a lane is an output column and
// a TMEM column is a row of x.
#pragma once

#include "linear_common.cuh"
#include "lora.cuh"

namespace arcb {
namespace linstream {

using lin::BK;
using lin::kUmmaK;

constexpr uint32_t kRows = 128;  // weight rows (output columns) per tile
constexpr uint32_t kThreads = 192;
constexpr uint32_t kWBytes = kRows * BK * 2;

template <uint32_t BN>
struct Cfg {
  static_assert(BN == 16 || BN == 32 || BN == 64 || BN == 128, "row tile");
  static constexpr uint32_t kStages = BN == 16 ? 6 : BN == 32 ? 5 : BN == 64 ? 4 : 3;
  static constexpr uint32_t kXBytes = BN * BK * 2;
  static constexpr uint32_t kTmemCols = BN < 32 ? 32 : BN;
  static_assert(kStages * (kWBytes + kXBytes) >= BN * kRows * 4, "the partial sums reuse the ring");
};

template <uint32_t BN>
struct alignas(1024) Smem {
  union {
    struct {
      uint8_t w[Cfg<BN>::kStages][kWBytes];
      uint8_t x[Cfg<BN>::kStages][Cfg<BN>::kXBytes];
    };
    float part[BN][kRows];
    uint32_t prefix[lin::kMaxGroups + 1];  // only until the block knows its tile
  };
  uint64_t full[Cfg<BN>::kStages];
  uint64_t empty[Cfg<BN>::kStages];
  uint64_t done;
  uint32_t tmem_base;
  uint32_t abort;
};

template <uint32_t BN>
constexpr size_t smem_bytes() {
  return sizeof(Smem<BN>) + 1024;
}
// 228 KB of shared memory per SM, of which the system takes 1 KB per block.
constexpr size_t kHalfSm = (228 / 2 - 1) * 1024;
static_assert(smem_bytes<16>() <= kHalfSm && smem_bytes<32>() <= kHalfSm && smem_bytes<64>() <= kHalfSm &&
                  smem_bytes<128>() <= kHalfSm,
              "two blocks per SM");

struct Params {
  CUtensorMap tm_w;  // {K, N, E} box {64, 128, 1}; W_MN: {F, N, E} box {64, 64, 1}; SW128
  CUtensorMap tm_x;  // {K, rows} box {64, BN}, SW128
  uint16_t* out;
  uint64_t ldo;
  lin::Groups groups;
  lin::Epilogue epi;
  uint32_t cols;      // output columns (features)
  uint32_t tiles_n;   // ceil(cols / 128)
  uint32_t num_kb;    // contraction blocks of 64
  uint32_t splits;    // cluster size along the contraction
  uint32_t zero_others;  // zero the output rows of no group
};

// With adapters (LORA): see lora.cuh. The epilogue's warps compute the adapters' part of the tile while the weights
// stream, an adapter of the tile's list each in turn (a block of a cluster has every S-th), and leave it in memory,
// from where the block that has computed a row adds it to its own sums.
struct LoraParams : Params {
  lora::Extra extra;
};

// The rows rank, rank + S, ... of one output column: the cluster's partial sums in rank order, then
// the epilogue. 16 sums are on their way at once: row by row, each row waits for a round trip
// through the cluster (128 x 4096 x 4096 19.3 us against 14.8 without an epilogue); with 32 they
// come in no faster (64 x 4096 x 4096 11.9 and 12.2).
template <uint32_t BN, uint32_t S>
__device__ __forceinline__ void finish_rows(const Params& p, const float* part, uint32_t rank, uint32_t row0,
                                            uint32_t rows, uint32_t f, float bias) {
  constexpr uint32_t kAtOnce = 16u / S;
  uint32_t from[S];
#pragma unroll
  for (uint32_t i = 0; i < S; ++i) from[i] = map_to_rank(part, i);
#pragma unroll 1
  for (uint32_t c0 = rank; c0 < rows; c0 += kAtOnce * S) {
    float v[kAtOnce][S];
    uint16_t res[kAtOnce];
#pragma unroll
    for (uint32_t u = 0; u < kAtOnce; ++u) {
      // Behind the last row: its sums again, so that no branch lies between the loads.
      const uint32_t own = c0 + u * S, c = min(own, rows - 1u);
      res[u] = p.epi.residual != nullptr && own < rows ? p.epi.residual[(row0 + size_t(c)) * p.epi.ldr + f] : uint16_t(0);
#pragma unroll
      for (uint32_t i = 0; i < S; ++i) v[u][i] = ld_dsmem_f32(from[i] + c * (kRows * 4u));
    }
    float z[kAtOnce];
#pragma unroll
    for (uint32_t u = 0; u < kAtOnce; ++u) {
      const uint32_t c = c0 + u * S;
#pragma unroll
      for (uint32_t d = 1; d < S; d *= 2) {
#pragma unroll
        for (uint32_t i = 0; i + d < S; i += 2 * d) v[u][i] += v[u][i + d];
      }
      z[u] = v[u][0] + bias;
      if (p.epi.z != nullptr && c < rows) {
        p.epi.z[(row0 + size_t(c)) * p.epi.ldz + f] = __bfloat16_as_ushort(__float2bfloat16_rn(z[u]));
      }
    }
    lin::activate(z, p.epi.act);
#pragma unroll
    for (uint32_t u = 0; u < kAtOnce; ++u) {
      const uint32_t c = c0 + u * S;
      if (p.epi.residual != nullptr) z[u] += bf16_bits_to_float(res[u]);
      if (c < rows) p.out[(row0 + size_t(c)) * p.ldo + f] = __bfloat16_as_ushort(__float2bfloat16_rn(z[u]));
    }
  }
}

template <uint32_t BN, bool W_MN, bool LORA, typename P>
__device__ __forceinline__ void linear_stream(const P& p) {
  static_assert(!LORA || !W_MN, "adapters belong to the forward product");
  using C = Cfg<BN>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem<BN>& s = *reinterpret_cast<Smem<BN>*>(smem_raw + smem_align_pad(smem_raw));
  const uint32_t warp = warp_idx_sync();
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t rank = p.splits > 1u ? cluster_ctarank() : 0u;
  volatile uint32_t* abort = &s.abort;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&p.tm_w);
    tma_prefetch_desc(&p.tm_x);
    for (uint32_t i = 0; i < C::kStages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    mbar_init(&s.done, 1);
    s.abort = 0;
    fence_barrier_init();
  }
  __syncthreads();  // the barriers exist
  // TMEM is taken only after the preceding grid has ended, and the next grid is let in only after it
  // is taken: whatever kernels stand beside this one on the stream, none waits for columns that are
  // held by one that waits for it. The loads do not wait for it (of groups, they wait for the table).
  // What it costs: a second block that uses TMEM starts on an SM only when the first has given up its
  // right to allocate, so it starts some 0.6 us after the preceding grid's end (8 x 4096 x 4096, call
  // after call in a graph, 6.7 us with TMEM taken before the wait, 7.1 so).
  // With adapters the preceding grid is lora_down_kernel, which uses no TMEM and has waited for what came
  // before it: only what it writes, and the output, wait for its end.
  if (!LORA) pdl_wait();
  const bool grouped = p.groups.offsets != nullptr;
  if (warp == 1) {
    tmem_alloc(&s.tmem_base, C::kTmemCols);
    tmem_relinquish();
  }
  if (warp == 2 && grouped) lin::group_tiles_prefix(p.groups, BN, s.prefix);
  tc_fence_before_sync();
  if (grouped) {
    __syncthreads();
  } else if (warp != 0) {
    named_barrier_sync(1, kThreads - 32);
  }
  tc_fence_after_sync();
  if (!LORA && warp != 0) pdl_launch_dependents();
  const uint32_t tmem_base = warp != 0 ? s.tmem_base : 0u;
  if (p.zero_others) lin::zero_other_rows(p.groups, p.out, p.ldo, p.cols, blockIdx.x, gridDim.x);

  // This block's tile. The row tiles of a group lie next to one another, so that blocks that
  // read the same weights run together.
  const uint32_t item = blockIdx.x / p.splits;
  uint32_t e = 0, row0 = 0, row_end = 0, f0 = 0;
  bool live;
  if (p.groups.offsets == nullptr) {
    const uint32_t tiles_m = (p.groups.rows + BN - 1u) / BN;
    const uint32_t nt = item / tiles_m;
    row0 = (item - nt * tiles_m) * BN;
    row_end = p.groups.rows;
    f0 = nt * kRows;
    live = nt < p.tiles_n;
  } else {
    const uint32_t row_tiles = s.prefix[p.groups.num];
    live = item < row_tiles * p.tiles_n;
    if (live) {
      // Group e's items are [prefix[e], prefix[e+1]) x tiles_n.
      e = lin::group_of_tile(s.prefix, p.groups.num, item / p.tiles_n);
      const uint32_t own = s.prefix[e + 1] - s.prefix[e];
      const uint32_t rem = item - s.prefix[e] * p.tiles_n;
      const uint32_t nt = rem / own;
      const uint32_t first = lin::group_begin(p.groups, e);
      row0 = first + (rem - nt * own) * BN;
      row_end = first + lin::group_count(p.groups, e);
      f0 = nt * kRows;
    }
  }
  if (p.groups.offsets != nullptr) {
    // The table's bytes go to the TMA loads now: order the reads above before them.
    fence_proxy_async_smem();
    __syncthreads();
  }
  const uint32_t kb0 = p.num_kb * rank / p.splits, kb1 = p.num_kb * (rank + 1u) / p.splits;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0 && live) {
      uint32_t stage = 0, phase = 0, issued = 0;
      for (uint32_t kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&s.empty[stage], phase ^ 1u, abort, kStatusTimeoutProducer)) break;
        mbar_arrive_expect_tx(&s.full[stage], kWBytes + C::kXBytes);
        if (W_MN) {
          tma_load_3d(&p.tm_w, &s.full[stage], s.w[stage], int32_t(f0), int32_t(kb * BK), int32_t(e), kCacheEvictNormal);
          tma_load_3d(&p.tm_w, &s.full[stage], s.w[stage] + lin::kMnChunkBytes, int32_t(f0 + 64u), int32_t(kb * BK),
                      int32_t(e), kCacheEvictNormal);
        } else {
          tma_load_3d(&p.tm_w, &s.full[stage], s.w[stage], int32_t(kb * BK), int32_t(f0), int32_t(e), kCacheEvictNormal);
        }
        tma_load_2d(&p.tm_x, &s.full[stage], s.x[stage], int32_t(kb * BK), int32_t(row0), kCacheEvictLast);
        ++issued;
        if (++stage == C::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      const uint32_t n_drain = issued < C::kStages ? issued : C::kStages;
      for (uint32_t i = issued - n_drain; i < issued; ++i) {
        mbar_drain(&s.full[i % C::kStages], (i / C::kStages) & 1u);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ UMMA issuer
    if (lane == 0 && live) {
      constexpr uint32_t idesc = lin::idesc_of<W_MN, false>(kRows, BN);
      uint32_t stage = 0, phase = 0;
      for (uint32_t kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&s.full[stage], phase, abort, kStatusTimeoutMma)) break;
        tc_fence_after_sync();
        const uint64_t adesc = lin::operand_desc<W_MN>(s.w[stage]);
        const uint64_t bdesc = make_sw128_kmajor_desc(s.x[stage]);
#pragma unroll
        for (uint32_t k = 0; k < BK / kUmmaK; ++k) {
          umma_bf16(tmem_base, desc_advance(adesc, k * lin::operand_step<W_MN>()),
                    desc_advance(bdesc, k * kUmmaK * 2), idesc, (kb != kb0 || k != 0u) ? 1u : 0u);
        }
        umma_commit(&s.empty[stage]);
        if (++stage == C::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      // Covers every UMMA above: the accumulator is complete, the ring is free.
      umma_commit(&s.done);
      mbar_drain(&s.done, 0);
    }
  }
  __syncwarp();

  // LORA: which rows' adapters this block has computed.
  constexpr uint32_t kRowWords = (BN + 31u) / 32u;
  [[maybe_unused]] uint32_t added[kRowWords] = {};
  if constexpr (LORA) {
    if (warp >= 2u) {
      lora::adapter_sums<BN, kRows>(p.extra, row0, f0, p.cols, rank, p.splits, warp - 2u, lane, added);
      pdl_launch_dependents();
      named_barrier_sync(2, 128);
    }
  }
  // Adds what lora::adapter_sums has left to 16 rows from c0 on.
  [[maybe_unused]] const auto add_adapters = [&](float (&v)[16], uint32_t c0, uint32_t f, bool valid) {
    if constexpr (LORA) {
      uint32_t word = added[0];
#pragma unroll
      for (uint32_t k = 1; k < kRowWords; ++k) word = c0 / 32u == k ? added[k] : word;
      word = word >> (c0 % 32u) & 0xFFFFu;
      if (word == 0u) return;
      float d[16];
#pragma unroll
      for (uint32_t j = 0; j < 16; ++j) {
        d[j] = valid && ((word >> j) & 1u) != 0u ? __ldcg(p.extra.sums + size_t(row0 + c0 + j) * p.cols + f) : 0.f;
      }
#pragma unroll
      for (uint32_t j = 0; j < 16; ++j) v[j] += d[j];
    }
  };

  // ------------------------------------------------------------ epilogue
  const uint32_t q = warp & 3u;
  const uint32_t fl = q * 32u + lane;  // this thread's output column in the tile
  const uint32_t f = f0 + fl;
  const uint32_t rows = live ? min(BN, row_end - row0) : 0u;
  const uint32_t t_row = tmem_base + ((q * 32u) << 16);
  bool ok = false;
  if (warp >= 2u && live) {
    ok = __all_sync(0xffffffffu, mbar_wait(&s.done, 0, abort, kStatusTimeoutEpilogue));
    tc_fence_after_sync();
  }
  const bool mine = ok && f < p.cols;
  const float bias = mine && p.epi.bias != nullptr ? bf16_bits_to_float(p.epi.bias[f]) : 0.f;

  if (p.splits == 1u) {
    if (ok) {
#pragma unroll 1
      for (uint32_t c0 = 0; c0 < rows; c0 += 16u) {
        const size_t row = row0 + c0;
        uint32_t r[16], res[16];
        tmem_ld_32x32b_x16(t_row + c0, r);
        if (p.epi.residual != nullptr) {
          lin::load_columns_start(p.epi.residual + row * p.epi.ldr + f, p.epi.ldr, res, rows - c0, mine, p.epi.pair_residual);
        }
        tmem_ld_wait();
        float v[16];
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]) + bias;
        add_adapters(v, c0, f, mine);
        if (p.epi.z != nullptr) {
          lin::store_columns(p.epi.z + row * p.epi.ldz + f, p.epi.ldz, v, rows - c0, mine, p.epi.pair_z);
        }
        lin::activate(v, p.epi.act);
        if (p.epi.residual != nullptr) {
          float add[16];
          lin::load_columns_finish(res, add, p.epi.pair_residual);
#pragma unroll
          for (uint32_t j = 0; j < 16; ++j) v[j] += add[j];
        }
        lin::store_columns(p.out + row * p.ldo + f, p.ldo, v, rows - c0, mine, p.epi.pair_out);
        __syncwarp();
      }
    }
  } else {
    // Every rank leaves its partial sums in its own ring (all loads and UMMAs are done with
    // it); rank r then finishes the rows r, r + S, ... of the tile.
    if (ok) {
#pragma unroll 1
      for (uint32_t c0 = 0; c0 < rows; c0 += 16u) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(t_row + c0, r);
        tmem_ld_wait();
        float v[16];
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
        add_adapters(v, c0, f, mine);
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j) s.part[c0 + j][fl] = v[j];
      }
    }
    cluster_sync_all();
    if (mine) {
      if (p.splits == 2u) {
        finish_rows<BN, 2>(p, s.part[0] + fl, rank, row0, rows, f, bias);
      } else if (p.splits == 4u) {
        finish_rows<BN, 4>(p, s.part[0] + fl, rank, row0, rows, f, bias);
      } else {
        finish_rows<BN, 8>(p, s.part[0] + fl, rank, row0, rows, f, bias);
      }
    }
    cluster_sync_all();  // a peer may still be reading this block's sums
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

template <uint32_t BN, bool W_MN>
__global__ void __launch_bounds__(kThreads, 2) gemm_linear_stream_kernel(const __grid_constant__ Params p) {
  linear_stream<BN, W_MN, false>(p);
}

template <uint32_t BN>
__global__ void __launch_bounds__(kThreads, 2) lora_linear_stream_kernel(const __grid_constant__ LoraParams p) {
  linear_stream<BN, false, true>(p);
}

}  // namespace linstream
}  // namespace arcb
