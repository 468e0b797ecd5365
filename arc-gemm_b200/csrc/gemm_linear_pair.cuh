// gemm_linear_pair.cuh — the linear layer's large form and the weight gradients, on CTA pairs.
//
//   rows:               out[t, f]    = epilogue( sum_k a[t, k] b[f, k] )
//   contraction groups: out[e, i, j] = sum_{t in group e} a[t, i] b[t, j]     (weight gradient)
//
// Bound by the tensor pipe: a pair runs 256 x 256 x 16 UMMAs (cta_group::2), each CTA holding
// half of A's and half of B's rows, so that per 64 of the contraction a CTA's shared memory is
// written and read 32 KB each for 128 x 256 x 64 MACs (a single CTA with the same tile would
// move half as much again and stop near 70 % of the tensor peak). The accumulator is double
// buffered in TMEM; a tile's epilogue runs under the next tile's products. Measured: 4096 x 14336
// x 4096 with bias, GELU and residual 332 us in a short run (1450 TFLOP/s), 382 to 391 under the power
// cap; the gradient of 4096 x 8192 x 4096, from cold: rows 187, weights 195 us (both operands MN-major:
// each 64-row piece of them is two boxes, and the tensor pipe is busy 78 % against 90 % of the forward
// product's time).
//
// Operands are read as they lie in memory. A K-major operand has the contraction contiguous
// (the forward product); an MN-major one has the output index contiguous: w in the gradient
// of the rows, both operands in the gradient of the weights. No transposed copy is made.
//
// Contraction groups. The last block of a group may hold rows of the next one, which must not
// enter the sums, whatever they hold (infinities and NaN included, so one zeroed operand is not
// enough). The steps of 16 that lie wholly behind the group are not issued; the rows behind it
// inside the last step are overwritten with zeros in shared memory, in both operands, by a warp
// of each CTA between the load's arrival and the product.
//
// SPLIT: problems with fewer tiles than pairs. A cluster of two pairs takes one tile, its pairs
// half of the contraction each; each CTA then leaves its sums in its ring's shared memory, and
// pair i finishes the i-th half of the columns, adding the halves in order through distributed
// shared memory (the result does not depend on timing).
//
// TN: columns of a tile. 128 where tiles of 256 leave pairs without work or a last round mostly
// empty (with bias and GELU 256 x 4096 x 4096: 21.3 us with 256, 16.8 with 128; 512 x 4608 x 4096 30
// and 23; but 1024 x 4096 x 4096 31 to 35 and 43, since a stage's products then hardly cover its
// hand-offs).
//
// LORA: the blocks of a tile's adapters come behind the contraction's, as products that leave the rows of other
// adapters as they are.
//
// Roles (384 threads per CTA): warp 0 TMA producer, warp 1 UMMA issuer (rank 0), warp 2 TMEM
// owner, warp 3 zeroes a group's tail, warps 4-11 epilogue: two warpgroups take 32 columns in
// turn; a thread owns one output row, and a warp's 32 x 32 piece goes out by TMA through shared
// memory (the residual comes in the same way, one piece ahead).
#pragma once

#include "gemm_bf16_pair.cuh"
#include "linear_common.cuh"
#include "lora.cuh"

namespace arcb {
namespace linpair {

using lin::BK;
using lin::kUmmaK;

constexpr uint32_t kRowsPerCta = 128;
constexpr uint32_t kTile = 256;  // pair tile, rows; and columns unless TN is 128
constexpr uint32_t kEpiWarps = 8;
constexpr uint32_t kThreads = 32 * (4 + kEpiWarps);
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kBandM = 8;  // row tiles per raster band (L2 reuse)
constexpr uint32_t kOperandBytes = kRowsPerCta * BK * 2;
// A and B of one CTA, in as many stages as shared memory holds: narrow tiles are short of loads in
// flight rather than of tensor time (256 x 4096 x 14336 in two parts: 36.4 us with six stages, 34.8 with eight).
template <uint32_t TN>
struct Cfg {
  static constexpr uint32_t kStages = TN == 256 ? 6 : 8;
  static constexpr uint32_t kBBytes = TN / 2 * BK * 2;
  static constexpr uint32_t kStageBytes = kOperandBytes + kBBytes;
  static_assert(kStages * kStageBytes >= TN * kRowsPerCta * 4, "a CTA's sums fit in its ring");
};

template <uint32_t TN>
struct alignas(1024) Smem {
  static constexpr uint32_t kStages = Cfg<TN>::kStages;
  uint8_t a[kStages][kOperandBytes];
  uint8_t b[kStages][Cfg<TN>::kBBytes];
  uint8_t piece[kEpiWarps][2][lin::kWarpTileBytes];
  uint64_t full[kStages];        // rank 0: both CTAs' bytes of a stage
  uint64_t empty[kStages];       // each CTA: the pair's UMMAs consumed its stage
  uint64_t tail_full[kStages];   // each CTA: its own bytes of a group's tail block
  uint64_t tail_fixed[kStages];  // rank 0: rank 1's tail block is zeroed
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint64_t drain;
  uint64_t piece_in[kEpiWarps][2];  // a residual piece landed
  uint32_t tmem_base;
  uint32_t abort;
};
template <uint32_t TN>
constexpr size_t kSmemBytes = sizeof(Smem<TN>) + 1024;
static_assert(kSmemBytes<256> <= 232448 && kSmemBytes<128> <= 232448, "shared memory fits in 227 KB");

struct Params {
  CUtensorMap tm_a;  // 3-D, SW128: K-major {K, M, E} box {64, 128, 1}; MN-major {M, K, E} box {64, 64, 1}
  CUtensorMap tm_b;  // likewise, with N in the place of M
  // Pieces of 32 x 32, 3-D {N, M, E}, SW64, where tma_* says so.
  CUtensorMap tm_out, tm_z, tm_res;
  uint32_t tma_out, tma_z, tma_res;
  uint16_t* out;
  uint64_t ldo;        // elements between output rows
  uint64_t out_group;  // contraction mode: elements between the groups' outputs
  lin::Groups groups;  // contraction groups (rows: unused)
  lin::Epilogue epi;
  uint32_t M, N;       // output rows (of a group) and columns
  uint32_t tiles_m, tiles_n, num_kb;
};

// With adapters (LORA): see lora.cuh. The blocks of the tile's adapters follow those of the contraction.
struct LoraParams : Params {
  lora::Extra extra;
};

// One tile of the walk.
struct Tile {
  uint32_t e;           // group
  uint32_t m0, n0;
  uint32_t k0;          // first contraction row
  uint32_t num_kb;      // blocks of 64
  uint32_t kb0, kb1;    // this pair's
  uint32_t last_steps;  // UMMA steps of the last block (4 unless a group ends inside it)
  uint32_t tail_rows;   // valid rows of the last block if it needs zeroing, else 0
};

// `part`: this pair's half of the contraction (SPLIT).
template <bool ALONG_K, bool SPLIT, uint32_t TN>
__device__ __forceinline__ bool tile_at(const Params& p, uint32_t t, uint32_t part, Tile& w) {
  const uint32_t per = p.tiles_m * p.tiles_n;
  w.e = 0;
  w.k0 = 0;
  w.num_kb = p.num_kb;
  w.last_steps = BK / kUmmaK;
  w.tail_rows = 0;
  if (ALONG_K) {
    w.e = t / per;
    if (w.e >= p.groups.num) return false;
    t -= w.e * per;
    w.k0 = lin::group_begin(p.groups, w.e);
    const uint32_t cnt = lin::group_count(p.groups, w.e);
    w.num_kb = (cnt + BK - 1u) / BK;
    const uint32_t last = cnt - (w.num_kb == 0u ? 0u : (w.num_kb - 1u) * BK);
    w.last_steps = (last + kUmmaK - 1u) / kUmmaK;
    // Rows past the matrix are zero as TMA fills them.
    if ((last % kUmmaK) != 0u && w.k0 + cnt < p.groups.rows) w.tail_rows = last;
  } else if (t >= per) {
    return false;
  }
  const uint32_t band = t / (kBandM * p.tiles_n);
  const uint32_t rem = t - band * kBandM * p.tiles_n;
  const uint32_t m_first = band * kBandM;
  const uint32_t m_cnt = min(kBandM, p.tiles_m - m_first);
  w.m0 = (m_first + rem % m_cnt) * kTile;
  w.n0 = rem / m_cnt * TN;
  w.kb0 = SPLIT && part == 1u ? w.num_kb / 2u : 0u;
  w.kb1 = SPLIT && part == 0u ? w.num_kb / 2u : w.num_kb;
  return true;
}

// The limit of a wait for a tile's whole contraction, which the rows of a weight gradient can make
// long: 2^23 blocks of 64 rows take 2.2 s. A block takes 0.27 us; 2 are allowed.
__device__ __forceinline__ uint64_t products_limit(const Tile& w) {
  return kWaitTimeoutNs + uint64_t(w.kb1 - w.kb0) * 2000u;
}

// One warp's way to memory: its two pieces in turn.
struct Pieces {
  uint8_t (*buf)[lin::kWarpTileBytes];
  uint64_t* in;     // barriers of residual loads
  uint32_t next;    // piece to use next
  uint32_t phases;  // parity of each piece's next residual load
  bool asked;       // the residual's piece is on its way into `next`
};

// The piece to use next is free once all stores but the last have read theirs.
__device__ __forceinline__ void piece_claim(uint32_t lane) {
  if (lane == 0) tma_store_wait_read<1>();
  __syncwarp();
}

// A 32 x 32 piece (row `lane` in v) from the registers to rows m.., columns n.. of a matrix.
__device__ __forceinline__ void piece_store(Pieces& b, const float (&v)[32], const CUtensorMap* map, uint32_t tma,
                                            uint16_t* p, uint64_t ld, uint32_t rows, uint32_t cols, uint32_t n,
                                            uint32_t m, uint32_t e, uint32_t lane) {
  uint32_t packed[16];
#pragma unroll
  for (uint32_t i = 0; i < 16; ++i) packed[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
  uint8_t* tile = b.buf[b.next];
  lin::warp_tile_put(tile, packed);
  if (tma) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_3d(map, tile, int32_t(n), int32_t(m), int32_t(e));
      tma_store_commit();
    }
  } else {
    __syncwarp();
    lin::warp_tile_to_rows(tile, p, ld, rows, cols);
    fence_proxy_async_smem();  // a residual's load may be the next to write here
    __syncwarp();
    if (lane == 0) tma_store_commit();  // an empty group: every piece counts as one
  }
  b.next ^= 1u;
}

// Ask for the residual's piece at (m, n), which the piece to use next will hold.
__device__ __forceinline__ void piece_ask(const Params& p, Pieces& b, uint32_t n, uint32_t m, uint32_t lane) {
  piece_claim(lane);
  if (lane == 0) {
    mbar_arrive_expect_tx(&b.in[b.next], lin::kWarpTileBytes);
    tma_load_3d(&p.tm_res, &b.in[b.next], b.buf[b.next], int32_t(n), int32_t(m), 0, kCacheEvictNormal);
  }
  b.asked = true;
}

// 32 x 32 sums of a warp (lane = output row m + lane) from column n on, through the epilogue and
// out. False if a wait was abandoned.
template <bool ALONG_K>
__device__ __forceinline__ bool finish_piece(const Params& p, Pieces& b, float (&v)[32], uint32_t m, uint32_t n,
                                             uint32_t e, volatile uint32_t* abort, uint32_t lane) {
  const uint32_t rows = min(32u, p.M - m), cols = min(32u, p.N - n);
  // A TMA store writes whole 16-byte pieces, zeros behind a matrix's last column: where that column
  // ends inside one, the piece goes out element by element and what lies beside the matrix stays.
  const uint32_t whole = cols % 8u == 0u ? 1u : 0u;
  if (!ALONG_K) {
    if (p.epi.bias != nullptr) {
      uint32_t c[16];
      lin::load_row32(p.epi.bias + n, c, cols, p.epi.wide_bias);
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) {
        v[2 * i] += __uint_as_float(c[i] << 16);
        v[2 * i + 1] += __uint_as_float(c[i] & 0xFFFF0000u);
      }
    }
    if (p.epi.z != nullptr) {
      piece_claim(lane);
      piece_store(b, v, &p.tm_z, p.tma_z & whole, p.epi.z + size_t(m) * p.epi.ldz + n, p.epi.ldz, rows, cols, n, m, 0, lane);
    }
    lin::activate(v, p.epi.act);
  }
  if (!ALONG_K && p.epi.residual != nullptr) {
    uint32_t c[16];
    if (p.tma_res) {
      if (!b.asked) piece_ask(p, b, n, m, lane);
      if (!__all_sync(0xffffffffu, mbar_wait(&b.in[b.next], (b.phases >> b.next) & 1u, abort, kStatusTimeoutEpilogue))) {
        return false;
      }
      b.asked = false;
      b.phases ^= 1u << b.next;
    } else {
      piece_claim(lane);
      lin::warp_tile_from_rows(b.buf[b.next], p.epi.residual + size_t(m) * p.epi.ldr + n, p.epi.ldr, rows, cols);
      __syncwarp();
    }
    lin::warp_tile_get(b.buf[b.next], c);
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
      v[2 * i] += __uint_as_float(c[i] << 16);
      v[2 * i + 1] += __uint_as_float(c[i] & 0xFFFF0000u);
    }
  } else {
    piece_claim(lane);
  }
  piece_store(b, v, &p.tm_out, p.tma_out & whole, p.out + (ALONG_K ? size_t(e) * p.out_group : 0u) + size_t(m) * p.ldo + n,
              p.ldo, rows, cols, n, m, e, lane);
  return true;
}

template <bool A_MN, bool B_MN, bool ALONG_K, bool SPLIT, uint32_t TN, bool LORA, typename P>
__device__ __forceinline__ void linear_pair(const P& p) {
  static_assert(TN == 256 || (TN == 128 && !ALONG_K), "columns of a tile");
  static_assert(!LORA || (!A_MN && !B_MN && !ALONG_K), "adapters belong to the forward product");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  constexpr uint32_t kStages = Cfg<TN>::kStages;
  Smem<TN>& s = *reinterpret_cast<Smem<TN>*>(smem_raw + smem_align_pad(smem_raw));
  const uint32_t warp = warp_idx_sync();
  const uint32_t lane = threadIdx.x & 31u;
  // rank: CTA of the pair; lead: the pair's first CTA in the cluster. Without SPLIT a cluster is a pair
  // that walks over tiles, with it a cluster takes one tile.
  const uint32_t rank = cluster_ctarank() & 1u;
  const uint32_t lead = SPLIT ? cluster_ctarank() - rank : 0u, part = lead >> 1;
  constexpr uint32_t per_cluster = SPLIT ? 4u : 2u;
  const uint32_t pair = blockIdx.x / per_cluster, num_pairs = gridDim.x / per_cluster;
  const uint16_t both = static_cast<uint16_t>(0x3u << lead);
  volatile uint32_t* abort = &s.abort;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&p.tm_a);
    tma_prefetch_desc(&p.tm_b);
    for (uint32_t i = 0; i < kStages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
      mbar_init(&s.tail_full[i], 1);
      mbar_init(&s.tail_fixed[i], 1);
    }
    for (uint32_t i = 0; i < 2; ++i) {
      mbar_init(&s.tmem_full[i], 1);
      mbar_init(&s.tmem_empty[i], 2 * kEpiWarps);  // of both CTAs
    }
    mbar_init(&s.drain, 1);
    for (uint32_t i = 0; i < 2 * kEpiWarps; ++i) mbar_init(&s.piece_in[i >> 1][i & 1u], 1);
    s.abort = 0;
    fence_barrier_init();
  }
  // TMEM is taken only after the preceding grid has ended, and the next grid is let in only
  // after it is taken: two grids of the stream never hold each other's columns up. With adapters the preceding
  // grid is lora_down_kernel, which uses no TMEM and has waited for what came before it: only what it
  // writes, and the output, wait for its end.
  if (!LORA) pdl_wait();
  if (warp == 2) {
    tmem_alloc_pair(&s.tmem_base, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before any remote arrive or TMA
  tc_fence_after_sync();
  if (!LORA) pdl_launch_dependents();
  const uint32_t tmem_base = s.tmem_base;

  const uint32_t epi_warp = warp >= 4 ? warp - 4u : 0u;
  Pieces pieces = {s.piece[epi_warp], s.piece_in[epi_warp], 0u, 0u, false};
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, issued = 0;
      uint32_t is_tail = 0, tail_parity = 0;  // per stage: last block was a tail; its barrier's next parity
      const uint32_t row0 = rank * kRowsPerCta;
      Tile w;
      bool ok = true;
      for (uint32_t t = pair; ok && (tile_at<ALONG_K, SPLIT, TN>(p, t, part, w)); t += num_pairs) {
        for (uint32_t kb = w.kb0; kb < w.kb1; ++kb) {
          if (!mbar_wait(&s.empty[stage], phase ^ 1u, abort, kStatusTimeoutProducer)) {
            ok = false;
            break;
          }
          const bool tail = ALONG_K && w.tail_rows != 0u && kb + 1u == w.num_kb;
          uint32_t bar;
          if (tail) {
            bar = map_to_rank(&s.tail_full[stage], lead + rank);
            mbar_arrive_expect_tx(&s.tail_full[stage], Cfg<TN>::kStageBytes);
            is_tail |= 1u << stage;
            tail_parity ^= 1u << stage;
          } else {
            bar = map_to_rank(&s.full[stage], lead);
            if (rank == 0) mbar_arrive_expect_tx(&s.full[stage], 2 * Cfg<TN>::kStageBytes);
            is_tail &= ~(1u << stage);
          }
          const int32_t k = int32_t(w.k0 + kb * BK), m = int32_t(w.m0 + row0),
                        n = int32_t(w.n0 + rank * (TN / 2u));
          if (A_MN) {
            tma_load_3d_pair(&p.tm_a, bar, s.a[stage], m, k, 0, kCacheEvictNormal);
            tma_load_3d_pair(&p.tm_a, bar, s.a[stage] + lin::kMnChunkBytes, m + 64, k, 0, kCacheEvictNormal);
          } else {
            tma_load_3d_pair(&p.tm_a, bar, s.a[stage], k, m, 0, kCacheEvictNormal);
          }
          if (B_MN) {
            tma_load_3d_pair(&p.tm_b, bar, s.b[stage], n, k, 0, kCacheEvictNormal);
            if (TN == 256) {
              tma_load_3d_pair(&p.tm_b, bar, s.b[stage] + lin::kMnChunkBytes, n + 64, k, 0, kCacheEvictNormal);
            }
          } else {
            tma_load_3d_pair(&p.tm_b, bar, s.b[stage], k, n, 0, kCacheEvictNormal);
          }
          ++issued;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if constexpr (LORA) {
          if (SPLIT && part == 0u) continue;
          pdl_wait();
          const lora::TileList list(p.extra, w.m0 / kTile);
          for (uint32_t i = 0; ok && i < list.blocks; ++i) {
            if (!mbar_wait(&s.empty[stage], phase ^ 1u, abort, kStatusTimeoutProducer)) {
              ok = false;
              break;
            }
            const uint32_t bar = map_to_rank(&s.full[stage], lead);
            if (rank == 0) mbar_arrive_expect_tx(&s.full[stage], 2 * Cfg<TN>::kStageBytes);
            const int32_t r = int32_t(list.column(i));
            tma_load_3d_pair(&p.extra.tm_u, bar, s.a[stage], r, int32_t(w.m0 + row0), 0, kCacheEvictNormal);
            tma_load_3d_pair(&p.extra.tm_b, bar, s.b[stage], r, int32_t(w.n0 + rank * (TN / 2u)), int32_t(list.adapter(i)),
                             kCacheEvictNormal);
            ++issued;
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
      }
      // Loads in flight must land before the CTA may exit: tails on this CTA's own barriers,
      // the others on rank 0's, which rank 0 waits for (the closing cluster barrier keeps
      // rank 1's shared memory alive until then).
      const uint32_t n_drain = issued < kStages ? issued : kStages;
      for (uint32_t i = issued - n_drain; i < issued; ++i) {
        const uint32_t st = i % kStages;
        if ((is_tail >> st) & 1u) {
          mbar_drain(&s.tail_full[st], ((tail_parity >> st) & 1u) ^ 1u);
        } else if (rank == 0) {
          mbar_drain(&s.full[st], (i / kStages) & 1u);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ UMMA issuer (rank 0)
    // The whole warp walks (uniform values stay in uniform registers, fewer instructions per
    // stage), one lane issues.
    if (rank == 0) {
      const bool leader = elect_one();
      constexpr uint32_t idesc = lin::idesc_of<A_MN, B_MN>(kTile, TN);
      uint32_t stage = 0, phase = 0, local = 0;
      bool ok = true;
      Tile w;
      for (uint32_t t = pair; ok && (tile_at<ALONG_K, SPLIT, TN>(p, t, part, w)); t += num_pairs) {
        if (w.kb0 == w.kb1) continue;  // nothing to multiply: the epilogue takes zeros
        const uint32_t acc = local & 1u;
        const uint32_t acc_phase = (local >> 1) & 1u;
        ++local;
        if (!__all_sync(0xffffffffu, mbar_wait(&s.tmem_empty[acc], acc_phase ^ 1u, abort, kStatusTimeoutMma))) break;
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * TN;
        for (uint32_t kb = w.kb0; kb < w.kb1; ++kb) {
          if (!__all_sync(0xffffffffu, mbar_wait(&s.full[stage], phase, abort, kStatusTimeoutMma))) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint64_t adesc = lin::operand_desc<A_MN>(s.a[stage]);
          const uint64_t bdesc = lin::operand_desc<B_MN>(s.b[stage]);
          const uint32_t steps = kb + 1u == w.num_kb ? w.last_steps : BK / kUmmaK;
#pragma unroll
          for (uint32_t k = 0; k < BK / kUmmaK; ++k) {
            if (leader && (!ALONG_K || k < steps)) {
              umma_bf16_pair(d_tmem, desc_advance(adesc, k * lin::operand_step<A_MN>()),
                             desc_advance(bdesc, k * lin::operand_step<B_MN>()), idesc, kb != w.kb0 || k != 0u ? 1u : 0u);
            }
          }
          if (leader) umma_commit_pair(&s.empty[stage], both);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if constexpr (LORA) {
          pdl_wait();
          const lora::TileList list(p.extra, w.m0 / kTile);
          const lora::RowAdapters<kTile> rows(p.extra, w.m0, lane);
          const uint32_t blocks = !SPLIT || part == 1u ? list.blocks : 0u;
          for (uint32_t i = 0; ok && i < blocks; ++i) {
            uint32_t keep[kTile / 32];
            rows.others(list.adapter(i), keep);
            ok = __all_sync(0xffffffffu, mbar_wait(&s.full[stage], phase, abort, kStatusTimeoutMma));
            if (!ok) break;
            tc_fence_after_sync();
            const uint64_t adesc = lin::operand_desc<A_MN>(s.a[stage]);
            const uint64_t bdesc = lin::operand_desc<B_MN>(s.b[stage]);
            const uint32_t steps = lora::steps_of(p.extra, i);
#pragma unroll
            for (uint32_t k = 0; k < BK / kUmmaK; ++k) {
              if (leader && k < steps) {
                umma_bf16_pair_masked(d_tmem, desc_advance(adesc, k * lin::operand_step<A_MN>()),
                                      desc_advance(bdesc, k * lin::operand_step<B_MN>()), idesc, 1u, keep);
              }
            }
            if (leader) umma_commit_pair(&s.empty[stage], both);
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
        if (ok && leader) umma_commit_pair(&s.tmem_full[acc], both);
      }
      // Every pair UMMA must retire before either CTA releases TMEM or exits.
      if (leader) {
        umma_commit_pair(&s.drain, static_cast<uint16_t>(0x1u << lead));
        mbar_drain(&s.drain, 0);
      }
      __syncwarp();
    }
  } else if (warp == 2) {
    if (ALONG_K && p.groups.offsets != nullptr && blockIdx.x == 0) {
      for (uint32_t e = lane; e < p.groups.num; e += 32u) lin::group_check(p.groups, e);
    }
    __syncwarp();
  } else if (warp == 3) {
    // ------------------------------------------------------------ a group's tail
    if (ALONG_K) {
      uint32_t stage = 0, parity = 0;  // parity: per stage, of its next tail
      Tile w;
      bool ok = true;
      for (uint32_t t = pair; ok && (tile_at<ALONG_K, SPLIT, TN>(p, t, part, w)); t += num_pairs) {
        if (w.kb0 == w.kb1) continue;
        const uint32_t st = (stage + w.kb1 - w.kb0 - 1u) % kStages;
        stage = (stage + w.kb1 - w.kb0) % kStages;
        if (w.tail_rows == 0u || w.kb1 != w.num_kb) continue;
        const uint32_t par = (parity >> st) & 1u;
        ok = __all_sync(0xffffffffu, mbar_wait(&s.tail_full[st], par, abort, kStatusTimeoutScales, products_limit(w)));
        if (!ok) break;
        // Rows tail_rows .. end of their step, both chunks of both operands; a row of a chunk
        // is one 128-byte line whatever the swizzle does inside it.
        const uint32_t first = w.tail_rows, last = w.last_steps * kUmmaK;
        for (uint32_t i = lane; i < (last - first) * 32u; i += 32u) {
          const uint32_t row = first + (i >> 5), c = i & 31u;  // c: operand, chunk, 16-byte piece
          uint8_t* base = (c & 16u) ? s.b[st] : s.a[st];
          *reinterpret_cast<uint4*>(base + ((c >> 3) & 1u) * lin::kMnChunkBytes + row * 128u + (c & 7u) * 16u) =
              make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (rank == 1) {
            mbar_arrive_cluster(map_to_rank(&s.tail_fixed[st], lead));
          } else if (mbar_wait_cluster(&s.tail_fixed[st], par, abort, kStatusTimeoutScales)) {
            mbar_arrive(&s.full[st]);
          }
        }
        __syncwarp();
        parity ^= 1u << st;
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const uint32_t q = warp & 3u;
    const uint32_t wg = (warp - 4u) >> 2;
    const uint32_t row = q * 32 + lane;
    const uint32_t empty0[2] = {map_to_rank(&s.tmem_empty[0], lead), map_to_rank(&s.tmem_empty[1], lead)};
    if (LORA) {
      pdl_wait();
      pdl_launch_dependents();
    }
    uint32_t local = 0;
    bool ok = true;
    Tile w;
    for (uint32_t t = pair; (tile_at<ALONG_K, SPLIT, TN>(p, t, part, w)); t += num_pairs) {
      const bool any = w.kb0 != w.kb1;
      const uint32_t acc = local & 1u;
      const uint32_t acc_phase = (local >> 1) & 1u;
      if (any) ++local;
      const uint32_t t_row = tmem_base + ((q * 32u) << 16) + acc * TN;
      if constexpr (SPLIT) {
        // This CTA's sums, column by column, into its ring: every load and product has ended.
        if (any) {
          ok = __all_sync(0xffffffffu, mbar_wait(&s.tmem_full[acc], acc_phase, abort, kStatusTimeoutEpilogue, products_limit(w)));
          if (!ok) break;
          tc_fence_after_sync();
        }
        float* sums = reinterpret_cast<float*>(s.a[0]) + row;
#pragma unroll 1
        for (uint32_t c = wg; c < TN / 32u; c += 2u) {
          uint32_t r[32];
          if (any) {
            tmem_ld_32x32b_x32(t_row + c * 32u, r);
            tmem_ld_wait();
          }
#pragma unroll
          for (uint32_t i = 0; i < 32; ++i) sums[(c * 32u + i) * kRowsPerCta] = any ? __uint_as_float(r[i]) : 0.f;
        }
        continue;
      }
      const uint32_t m = w.m0 + rank * kRowsPerCta + q * 32u;  // the warp's first row
      if (ALONG_K && !any) {  // a group without rows
        float zero[32];
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i) zero[i] = 0.f;
        for (uint32_t n = w.n0 + wg * 32u; m < p.M && n < min(w.n0 + TN, p.N); n += 64u) {
          finish_piece<ALONG_K>(p, pieces, zero, m, n, w.e, abort, lane);
        }
        continue;
      }
      // The residual comes from memory: its first piece is asked for before the wait, the next
      // ones while the present is worked on (a pre-activation that also goes out takes turns on
      // the same pieces, which leaves none to ask ahead for).
      const bool ahead = !ALONG_K && p.epi.residual != nullptr && p.tma_res && p.epi.z == nullptr && m < p.M;
      if (ahead && w.n0 + wg * 32u < p.N) piece_ask(p, pieces, w.n0 + wg * 32u, m, lane);
      ok = __all_sync(0xffffffffu, mbar_wait(&s.tmem_full[acc], acc_phase, abort, kStatusTimeoutEpilogue, products_limit(w)));
      if (!ok) break;
      tc_fence_after_sync();
#pragma unroll 1
      for (uint32_t c = wg; c < TN / 32u; c += 2u) {
        const uint32_t n = w.n0 + c * 32u;
        uint32_t r[32];
        tmem_ld_32x32b_x32(t_row + c * 32u, r);
        tmem_ld_wait();
        if (c + 2u >= TN / 32u) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(empty0[acc]);
        }
        if (m < p.M && n < p.N && ok) {
          float v[32];
#pragma unroll
          for (uint32_t i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
          ok = finish_piece<ALONG_K>(p, pieces, v, m, n, w.e, abort, lane);
          if (ok && ahead && c + 2u < TN / 32u && n + 64u < p.N) piece_ask(p, pieces, n + 64u, m, lane);
        }
      }
      if (!ok) break;
    }
  }

  if constexpr (SPLIT) {
    __syncwarp();
    cluster_sync_all();  // every part's sums are in its shared memory
    Tile w;
    if (warp >= 4 && (tile_at<ALONG_K, SPLIT, TN>(p, pair, part, w)) && *abort == 0u) {
      const uint32_t row = (warp & 3u) * 32u + lane;
      const uint32_t m = w.m0 + rank * kRowsPerCta + (warp & 3u) * 32u;  // the warp's first row
      const uint32_t first = TN / 2u * part, last = first + TN / 2u;
      bool ok = m < p.M;
#pragma unroll 1
      for (uint32_t c = first + ((warp - 4u) >> 2) * 32u; c < last && w.n0 + c < p.N && ok; c += 64u) {
        float v[32];
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i) v[i] = 0.f;
        const float* sums = reinterpret_cast<const float*>(s.a[0]) + c * kRowsPerCta + row;
#pragma unroll 1
        for (uint32_t j = 0; j < 2u; ++j) {
          const uint32_t from = map_to_rank(sums, 2u * j + rank);
#pragma unroll
          for (uint32_t i = 0; i < 32; ++i) v[i] += ld_dsmem_f32(from + i * (kRowsPerCta * 4u));
        }
        ok = finish_piece<ALONG_K>(p, pieces, v, m, w.n0 + c, w.e, abort, lane);
      }
    }
    __syncwarp();
  }

  // Pieces on their way in have landed and those on their way out are written before the CTA may
  // exit (a load is under way here only if a wait was abandoned).
  if (warp >= 4 && lane == 0) {
    if (pieces.asked) mbar_drain(&pieces.in[pieces.next], (pieces.phases >> pieces.next) & 1u);
    tma_store_wait_all<0>();
  }
  __syncwarp();
  // Both CTAs stay resident until the pair's last UMMA retired (rank 0's drain) and both
  // epilogues finished with TMEM; then each frees its TMEM columns.
  tc_fence_before_sync();
  cluster_sync_all();
  if (warp == 2) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

template <bool A_MN, bool B_MN, bool ALONG_K, bool SPLIT, uint32_t TN>
__global__ void __launch_bounds__(kThreads, 1) gemm_linear_pair_kernel(const __grid_constant__ Params p) {
  linear_pair<A_MN, B_MN, ALONG_K, SPLIT, TN, false>(p);
}

template <bool SPLIT, uint32_t TN>
__global__ void __launch_bounds__(kThreads, 1) lora_linear_pair_kernel(const __grid_constant__ LoraParams p) {
  linear_pair<false, false, false, SPLIT, TN, true>(p);
}

}  // namespace linpair
}  // namespace arcb
