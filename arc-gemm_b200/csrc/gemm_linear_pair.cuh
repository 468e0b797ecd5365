// gemm_linear_pair.cuh — the linear layer's large form and the weight gradients, on CTA pairs.
//
//   rows:               out[t, f]    = epilogue( sum_k a[t, k] b[f, k] )
//   contraction groups: out[e, i, j] = sum_{t in group e} a[t, i] b[t, j]     (weight gradient)
//
// Bound by the tensor pipe: a pair runs 256 x 256 x 16 UMMAs (cta_group::2), each CTA holding
// half of A's and half of B's rows, so that per 64 of the contraction a CTA's shared memory is
// written and read 32 KB each for 128 x 256 x 64 MACs (a single CTA with the same tile would
// move half as much again and stop near 70 % of the tensor peak). The accumulator is double
// buffered in TMEM; a tile's epilogue runs under the next tile's products.
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
// Roles (384 threads per CTA): warp 0 TMA producer, warp 1 UMMA issuer (rank 0), warp 2 TMEM
// owner, warp 3 zeroes a group's tail, warps 4-11 epilogue: two warpgroups take 32 columns in
// turn, a thread owns one output row and stores 32 columns as two 32-byte sectors.
#pragma once

#include "gemm_bf16_pair.cuh"
#include "linear_common.cuh"

namespace arcb {
namespace linpair {

using lin::BK;
using lin::kUmmaK;

constexpr uint32_t kRowsPerCta = 128;
constexpr uint32_t kTile = 256;  // pair tile, both directions
constexpr uint32_t kStages = 6;
constexpr uint32_t kEpiWarps = 8;
constexpr uint32_t kThreads = 32 * (4 + kEpiWarps);
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kBandM = 8;  // row tiles per raster band (L2 reuse)
constexpr uint32_t kOperandBytes = kRowsPerCta * BK * 2;
constexpr uint32_t kStageBytes = 2 * kOperandBytes;  // A + B of one CTA

struct alignas(1024) Smem {
  uint8_t a[kStages][kOperandBytes];
  uint8_t b[kStages][kOperandBytes];
  uint64_t full[kStages];        // rank 0: both CTAs' bytes of a stage
  uint64_t empty[kStages];       // each CTA: the pair's UMMAs consumed its stage
  uint64_t tail_full[kStages];   // each CTA: its own bytes of a group's tail block
  uint64_t tail_fixed[kStages];  // rank 0: rank 1's tail block is zeroed
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  uint32_t abort;
};
constexpr size_t kSmemBytes = sizeof(Smem) + 1024;
static_assert(kSmemBytes <= 232448, "shared memory fits in 227 KB");

struct Params {
  CUtensorMap tm_a;  // 3-D, SW128: K-major {K, M, E} box {64, 128, 1}; MN-major {M, K, E} box {64, 64, 1}
  CUtensorMap tm_b;  // likewise, with N in the place of M
  uint16_t* out;
  uint64_t ldo;        // elements between output rows
  uint64_t out_group;  // contraction mode: elements between the groups' outputs
  lin::Groups groups;  // contraction groups (rows: unused)
  lin::Epilogue epi;
  uint32_t M, N;       // output rows (of a group) and columns
  uint32_t tiles_m, tiles_n, num_kb;
};

// One tile of the walk.
struct Tile {
  uint32_t e;           // group
  uint32_t m0, n0;
  uint32_t k0;          // first contraction row
  uint32_t num_kb;      // blocks of 64
  uint32_t last_steps;  // UMMA steps of the last block (4 unless a group ends inside it)
  uint32_t tail_rows;   // valid rows of the last block if it needs zeroing, else 0
};

template <bool ALONG_K>
__device__ __forceinline__ bool tile_at(const Params& p, uint32_t t, Tile& w) {
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
  w.n0 = rem / m_cnt * kTile;
  return true;
}

template <bool A_MN, bool B_MN, bool ALONG_K>
__global__ void __launch_bounds__(kThreads, 1) gemm_linear_pair_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>(smem_raw + smem_align_pad(smem_raw));
  const uint32_t warp = warp_idx_sync();
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t rank = cluster_ctarank();
  const uint32_t pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
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
    s.abort = 0;
    fence_barrier_init();
  }
  // TMEM is taken only after the preceding grid has ended, and the next grid is let in only
  // after it is taken: two grids of the stream never hold each other's columns up.
  pdl_wait();
  if (warp == 2) {
    tmem_alloc_pair(&s.tmem_base, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before any remote arrive or TMA
  tc_fence_after_sync();
  pdl_launch_dependents();
  const uint32_t tmem_base = s.tmem_base;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, issued = 0;
      uint32_t is_tail = 0, tail_parity = 0;  // per stage: last block was a tail; its barrier's next parity
      const uint32_t row0 = rank * kRowsPerCta;
      Tile w;
      bool ok = true;
      for (uint32_t t = pair; ok && tile_at<ALONG_K>(p, t, w); t += num_pairs) {
        for (uint32_t kb = 0; kb < w.num_kb; ++kb) {
          if (!mbar_wait(&s.empty[stage], phase ^ 1u, abort, kStatusTimeoutProducer)) {
            ok = false;
            break;
          }
          const bool tail = ALONG_K && w.tail_rows != 0u && kb + 1u == w.num_kb;
          uint32_t bar;
          if (tail) {
            bar = map_to_rank(&s.tail_full[stage], rank);
            mbar_arrive_expect_tx(&s.tail_full[stage], kStageBytes);
            is_tail |= 1u << stage;
            tail_parity ^= 1u << stage;
          } else {
            bar = map_to_rank(&s.full[stage], 0);
            if (rank == 0) mbar_arrive_expect_tx(&s.full[stage], 2 * kStageBytes);
            is_tail &= ~(1u << stage);
          }
          const int32_t k = int32_t(w.k0 + kb * BK), m = int32_t(w.m0 + row0), n = int32_t(w.n0 + row0);
          if (A_MN) {
            tma_load_3d_pair(&p.tm_a, bar, s.a[stage], m, k, 0, kCacheEvictNormal);
            tma_load_3d_pair(&p.tm_a, bar, s.a[stage] + lin::kMnChunkBytes, m + 64, k, 0, kCacheEvictNormal);
          } else {
            tma_load_3d_pair(&p.tm_a, bar, s.a[stage], k, m, 0, kCacheEvictNormal);
          }
          if (B_MN) {
            tma_load_3d_pair(&p.tm_b, bar, s.b[stage], n, k, 0, kCacheEvictNormal);
            tma_load_3d_pair(&p.tm_b, bar, s.b[stage] + lin::kMnChunkBytes, n + 64, k, 0, kCacheEvictNormal);
          } else {
            tma_load_3d_pair(&p.tm_b, bar, s.b[stage], k, n, 0, kCacheEvictNormal);
          }
          ++issued;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
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
      constexpr uint32_t idesc = lin::idesc_of<A_MN, B_MN>(kTile, kTile);
      uint32_t stage = 0, phase = 0, local = 0;
      bool ok = true;
      Tile w;
      for (uint32_t t = pair; ok && tile_at<ALONG_K>(p, t, w); t += num_pairs) {
        if (w.num_kb == 0u) continue;  // a group without rows: the epilogue stores zeros
        const uint32_t acc = local & 1u;
        const uint32_t acc_phase = (local >> 1) & 1u;
        ++local;
        if (!__all_sync(0xffffffffu, mbar_wait(&s.tmem_empty[acc], acc_phase ^ 1u, abort, kStatusTimeoutMma))) break;
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * kTile;
        for (uint32_t kb = 0; kb < w.num_kb; ++kb) {
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
                             desc_advance(bdesc, k * lin::operand_step<B_MN>()), idesc, (kb | k) != 0u ? 1u : 0u);
            }
          }
          if (leader) umma_commit_pair(&s.empty[stage], 0x3);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok && leader) umma_commit_pair(&s.tmem_full[acc], 0x3);
      }
      // Every pair UMMA must retire before either CTA releases TMEM or exits.
      if (leader) {
        umma_commit_pair(&s.drain, 0x1);
        mbar_drain(&s.drain, 0);
      }
      __syncwarp();
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------ a group's tail
    if (ALONG_K) {
      uint32_t stage = 0, parity = 0;  // parity: per stage, of its next tail
      Tile w;
      bool ok = true;
      for (uint32_t t = pair; ok && tile_at<ALONG_K>(p, t, w); t += num_pairs) {
        if (w.num_kb == 0u) continue;
        const uint32_t st = (stage + w.num_kb - 1u) % kStages;
        stage = (stage + w.num_kb) % kStages;
        if (w.tail_rows == 0u) continue;
        const uint32_t par = (parity >> st) & 1u;
        ok = __all_sync(0xffffffffu, mbar_wait(&s.tail_full[st], par, abort, kStatusTimeoutScales));
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
            mbar_arrive_cluster(map_to_rank(&s.tail_fixed[st], 0));
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
    const uint32_t empty0[2] = {map_to_rank(&s.tmem_empty[0], 0), map_to_rank(&s.tmem_empty[1], 0)};
    uint32_t local = 0;
    Tile w;
    for (uint32_t t = pair; tile_at<ALONG_K>(p, t, w); t += num_pairs) {
      const uint32_t m = w.m0 + rank * kRowsPerCta + row;
      const bool valid = m < p.M;
      uint16_t* out = p.out + (ALONG_K ? size_t(w.e) * p.out_group : 0u) + size_t(valid ? m : 0u) * p.ldo;
      if (ALONG_K && w.num_kb == 0u) {
        const uint32_t zero[16] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
#pragma unroll 1
        for (uint32_t n = w.n0 + wg * 32u; n < min(w.n0 + kTile, p.N) && valid; n += 64u) {
          lin::store_row32(out + n, zero, p.N - n, p.epi.vec_out);
        }
        __syncwarp();
        continue;
      }
      const uint32_t acc = local & 1u;
      const uint32_t acc_phase = (local >> 1) & 1u;
      ++local;
      // The residual comes from memory: its first columns are asked for before the wait, the
      // next ones while the present are worked on.
      const bool with_residual = !ALONG_K && p.epi.residual != nullptr && valid;
      const uint16_t* residual = p.epi.residual + (with_residual ? size_t(m) * p.epi.ldr : 0u);
      uint32_t res[16];
      if (with_residual && w.n0 + wg * 32u < p.N) {
        lin::load_row32(residual + w.n0 + wg * 32u, res, p.N - (w.n0 + wg * 32u), p.epi.vec_residual);
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&s.tmem_full[acc], acc_phase, abort, kStatusTimeoutEpilogue))) break;
      tc_fence_after_sync();
      const uint32_t t_row = tmem_base + ((q * 32u) << 16) + acc * kTile;
#pragma unroll 1
      for (uint32_t c = wg; c < kTile / 32u; c += 2u) {
        const uint32_t n = w.n0 + c * 32u;
        const uint32_t cols = n < p.N ? p.N - n : 0u;  // columns in range (more than 32: all)
        uint32_t r[32];
        tmem_ld_32x32b_x32(t_row + c * 32u, r);
        const bool live = valid && cols != 0u;
        tmem_ld_wait();
        if (c + 2u >= kTile / 32u) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(empty0[acc]);
        }
        if (live) {
          uint32_t packed[16];
          if (!ALONG_K) {
            if (p.epi.bias != nullptr) {
              uint32_t b[16];
              lin::load_row32(p.epi.bias + n, b, cols, p.epi.vec_bias);
#pragma unroll
              for (uint32_t i = 0; i < 16; ++i) {
                r[2 * i] = __float_as_uint(__uint_as_float(r[2 * i]) + __uint_as_float(b[i] << 16));
                r[2 * i + 1] = __float_as_uint(__uint_as_float(r[2 * i + 1]) + __uint_as_float(b[i] & 0xFFFF0000u));
              }
            }
            if (p.epi.z != nullptr) {
#pragma unroll
              for (uint32_t i = 0; i < 16; ++i) {
                packed[i] = pack_bf16x2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
              }
              lin::store_row32(p.epi.z + size_t(m) * p.epi.ldz + n, packed, cols, p.epi.vec_z);
            }
            float v[32];
#pragma unroll
            for (uint32_t i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
            lin::activate(v, p.epi.act);
#pragma unroll
            for (uint32_t i = 0; i < 32; ++i) r[i] = __float_as_uint(v[i]);
            if (with_residual) {
#pragma unroll
              for (uint32_t i = 0; i < 16; ++i) {
                r[2 * i] = __float_as_uint(__uint_as_float(r[2 * i]) + __uint_as_float(res[i] << 16));
                r[2 * i + 1] = __float_as_uint(__uint_as_float(r[2 * i + 1]) + __uint_as_float(res[i] & 0xFFFF0000u));
              }
              const uint32_t n2 = n + 64u;
              if (c + 2u < kTile / 32u && n2 < p.N) {
                lin::load_row32(residual + n2, res, p.N - n2, p.epi.vec_residual);
              }
            }
          }
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) {
            packed[i] = pack_bf16x2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
          }
          lin::store_row32(out + n, packed, cols, p.epi.vec_out);
        }
        __syncwarp();
      }
    }
  }

  // Both CTAs stay resident until the pair's last UMMA retired (rank 0's drain) and both
  // epilogues finished with TMEM; then each frees its TMEM columns.
  tc_fence_before_sync();
  cluster_sync_all();
  if (warp == 2) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

}  // namespace linpair
}  // namespace arcb
