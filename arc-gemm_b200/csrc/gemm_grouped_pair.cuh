// gemm_grouped_pair.cuh — grouped products for groups of many rows, on CTA pairs.
//
//   out[t, f] = sum_k x[t, k] w[e(t), f, k]        bf16 weights, or int4 codes with scales
//
// Orientation: 256 weight rows are the UMMA M operand (128 per CTA of the pair), a group's rows
// the N operand. A group ends anywhere, and the tensor pipe's time is proportional to N, so the
// last tile of a group is issued with N rounded up to 32 only; with the rows on the M side it
// would cost a full 256 (at 512 rows per group a quarter of all work). Bound by the tensor pipe.
// The accumulator is double buffered in TMEM (2 x 256 columns), the epilogue of a tile runs
// under the next tile's products. Measured: 8190 rows in 16 groups of 113 to 1101, 4096 x 4096,
// 233 us in a short run (1180 TFLOP/s), 274 to 281 under the power cap; 16 groups of 512 take 203. Row tiles of equal
// size within a group (200 + 200 for 256 + 144) measured the same there, 1 to 2 % slower with W_MN.
// W4: 4093 rows in 8 groups of 106 to 1255, 14336 x 4096, 400 to 410 us (1190 TFLOP/s), 455 to 485 under
// the cap.
//
// W_MN: w is read MN-major ([E][contraction][features]): the gradient of the rows.
//
// W4: w holds int4 codes c and bf16 scales per group of 128 along K, x int8 values widened to
// fp16 by a pass in front. The scales cannot wait for the accumulator (they change every 128
// products, and reading it out that often is what bounds the int32 kernel), so they are applied
// to the operand: c * s has at most 11 significant bits (3 of |c| <= 7, or the power of two 8,
// times 8 of a bf16 scale), which an fp16 holds exactly. What fp16 lacks is range: every weight
// row is multiplied by a power of two that takes its largest scale to [2^11, 2^12) (8 times that
// still fits), and the result is divided by it again in fp32. A weight is inexact only where
// its scale is less than 2^-24 of its row's largest, and then by at most 2^-29 of that one, below
// what an fp32 sum over the row resolves. Products of two fp16 are exact in fp32.
//
// Roles: warp 0 TMA producer, warp 1 UMMA issuer (rank 0), warp 2 TMEM owner and tile table (the
// producer and the issuer look the next tile up while the present one is under way),
// warps 4-11 epilogue (two warpgroups on alternate 32 columns). W4: warps 12-27 expand codes,
// warp 2 loads the codes, warp 3 tells rank 0 when rank 1's are expanded.
#pragma once

#include <cuda_fp16.h>

#include "linear_common.cuh"

namespace arcb {
namespace grouppair {

using lin::kUmmaK;

constexpr uint32_t kRowsPerCta = 128;  // weight rows
constexpr uint32_t kTileF = 256;       // weight rows per pair
constexpr uint32_t kTileT = 256;       // most rows of a group per tile
constexpr uint32_t kSubK = 64;         // one 128-byte swizzle row
constexpr uint32_t kSubBytes = kRowsPerCta * kSubK * 2;
constexpr uint32_t kEpiWarps = 8;
constexpr uint32_t kBandF = 8;  // weight tiles per raster band
// W4: the expanding warps work in sets of four on alternate stages: what a stage costs a warp is
// mostly waiting (for the slot, for its stores to be visible to the tensor core), about twice a
// stage's products. None of them shares a scheduler with the UMMA issuer (warp 1, and so every
// warp = 1 mod 4): the issuer has a few dozen instructions per stage in sequence, and beside busy
// warps they took it 1000 cycles instead of the products' 512 (4096 x 4096 x 4096: 162 us with
// sixteen expanding warps on all four schedulers, 124 us with twelve on three).
constexpr uint32_t kExpandSets = 3;
constexpr uint32_t kSetThreads = 128;
constexpr uint32_t kExpandWarps = 16;  // launched; those of the issuer's scheduler stay idle
constexpr uint32_t kTmemCols = 512;
// A group's last tile is loaded with the smaller of two boxes that holds its rows (several small
// boxes in their place cost more issue than the spared bytes: 16-row boxes took the tile from
// under 1.0 to 1.7 of a full one's time).
constexpr uint32_t kBox = kTileT / 2, kSmallBox = kTileT / 4;
constexpr uint32_t kScaleGroup = 128;  // W4: contraction elements per scale

constexpr uint32_t kStages = 6;
// W4: the codes have a ring of their own, one scale group (two stages) per slot, so that their
// way from memory is not part of the chain expand - multiply - reuse of an operand slot.
constexpr uint32_t kCodeSlots = 3;
constexpr uint32_t kCodeBytes = kRowsPerCta * kScaleGroup / 2;

template <bool W4>
constexpr uint32_t threads() {
  return 32 * (4 + kEpiWarps) + (W4 ? 32 * kExpandWarps : 0);
}

template <bool W4>
struct alignas(1024) Smem {
  uint8_t a[kStages][kSubBytes];  // weights
  uint8_t b[kStages][kSubBytes];  // rows
  uint8_t codes[kCodeSlots][W4 ? kCodeBytes : 16];
  uint64_t full[kStages];            // rank 0: both CTAs' bytes of a stage (W4: and rank 1's signal)
  uint64_t empty[kStages];           // each CTA: the pair's UMMAs consumed its stage
  uint64_t codes_full[kCodeSlots];   // W4, each CTA: its own codes landed
  uint64_t codes_empty[kCodeSlots];  // W4, each CTA: its expanding warps have read them
  uint64_t expanded[kStages];        // W4, each CTA: its expanding warps wrote the operand
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  uint32_t abort;
  uint32_t prefix[lin::kMaxGroups + 1];
};

template <bool W4>
constexpr size_t smem_bytes() {
  return sizeof(Smem<W4>) + 1024;
}
static_assert(smem_bytes<false>() <= 232448 && smem_bytes<true>() <= 232448, "shared memory fits in 227 KB");

struct Params {
  CUtensorMap tm_w;   // {K, N, E} box {64, 128, 1}; W_MN {F, N, E} box {64, 64, 1}; W4 {K/2 bytes, N, E} box {64, 128, 1}
  CUtensorMap tm_x;   // {K, rows} box {64, 128}, 16-bit
  CUtensorMap tm_xs;  // the same, box {64, kSmallBox}
  uint16_t* out;
  uint64_t ldo;
  const float* sa;     // W4: scale of each row
  const uint16_t* sb;  // W4: [E][cols][G] bf16
  lin::Groups groups;
  uint32_t cols;       // output columns (weight rows of a group)
  uint32_t tiles_f, num_kb;
  uint32_t G;          // W4: scales per weight row
  uint32_t split;      // W4: codes in the pre-packed layout
  uint32_t pair_store; // output rows take 4-byte stores
  uint32_t zero_others;
};

struct Tile {
  uint32_t e, f0, row0, rows, n;  // n: rows rounded up to the UMMA's granularity
};

__device__ __forceinline__ bool tile_at(const Params& p, const uint32_t* prefix, uint32_t t, Tile& w) {
  if (t >= prefix[p.groups.num] * p.tiles_f) return false;
  w.e = lin::group_of_tile(prefix, p.groups.num, t / p.tiles_f);
  const uint32_t own = prefix[w.e + 1] - prefix[w.e];
  const uint32_t rem = t - prefix[w.e] * p.tiles_f;
  // Bands of eight weight tiles: the pairs that run together share both operands in L2 (one group
  // of 8192 rows, 4096 x 4096: 191 us with a group's row tiles first, 177 in bands).
  const uint32_t band = rem / (kBandF * own);
  const uint32_t in_band = rem - band * kBandF * own;
  const uint32_t width = min(kBandF, p.tiles_f - band * kBandF);
  w.f0 = (band * kBandF + in_band % width) * kTileF;
  const uint32_t at = in_band / width * kTileT;
  w.row0 = lin::group_begin(p.groups, w.e) + at;
  w.rows = min(kTileT, lin::group_count(p.groups, w.e) - at);
  w.n = (w.rows + 31u) & ~31u;
  return true;
}

// Power of two that takes the largest scale of a weight row into [2^11, 2^12), as an exponent.
__device__ __forceinline__ int32_t row_shift(const uint16_t* sb_row, uint32_t G) {
  uint32_t m = 0;
  uint32_t g = 0;
  if ((reinterpret_cast<uintptr_t>(sb_row) & 15u) == 0u) {
    for (; g + 8u <= G; g += 8u) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(sb_row + g));
      // Two bf16 magnitudes per word: non-negative 16-bit integers in value order.
      m = __vmaxu2(m, __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu),
                               __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu)));
    }
  }
  for (; g < G; ++g) m = __vmaxu2(m, __ldg(sb_row + g) & 0x7FFFu);
  m = max(m & 0xFFFFu, m >> 16);
  return min(138 - static_cast<int32_t>(m >> 7), 127);
}

__device__ __forceinline__ float exp2i(int32_t e) {  // 2^e, -127 <= e <= 127 (2^-127 is subnormal)
  return e > -127 ? __uint_as_float(static_cast<uint32_t>(e + 127) << 23) : __uint_as_float(0x00400000u);
}

__device__ __forceinline__ uint32_t h2_sub_mul(uint32_t v, uint32_t c, uint32_t s) {
  uint32_t r;
  asm("{\n\t.reg .b32 d;\n\tsub.rn.f16x2 d, %1, %2;\n\tmul.rn.f16x2 %0, d, %3;\n\t}" : "=r"(r) : "r"(v), "r"(c), "r"(s));
  return r;
}

// 32 codes -> 32 fp16 values c * s, k ascending. A nibble, offset by 8, becomes the low bits of
// an fp16 1024 + n (from the low nibble of a byte) or 1024 + 16 n (from the high one): the
// subtraction leaves c or 16 c exactly, and the scales of high nibbles are s / 16.
__device__ __forceinline__ void expand_codes(const uint4& x, uint32_t split, uint32_t s_lo, uint32_t s_hi,
                                             uint32_t (&out)[16]) {
  const uint32_t w[4] = {x.x ^ 0x88888888u, x.y ^ 0x88888888u, x.z ^ 0x88888888u, x.w ^ 0x88888888u};
  constexpr uint32_t kMagic = 0x64646464u;
  constexpr uint32_t kLo = 0x6408u, kHi = 0x6480u;  // 1024 + 8, 1024 + 128
  if (split) {
    // Byte j: code j | code j + 16 << 4.
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint32_t v = __byte_perm(w[i >> 1], kMagic, (i & 1u) ? 0x4342u : 0x4140u);
      out[i] = h2_sub_mul(v & 0xFF0FFF0Fu, kLo | (kLo << 16), (s_lo & 0xFFFFu) | (s_lo << 16));
      out[i + 8] = h2_sub_mul(v & 0xFFF0FFF0u, kHi | (kHi << 16), (s_hi & 0xFFFFu) | (s_hi << 16));
    }
  } else {
    // Byte j: code 2j | code 2j + 1 << 4.
    const uint32_t s = s_lo | (s_hi << 16);
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
      const uint32_t v = __byte_perm(w[i >> 2], kMagic, 0x4040u | ((i & 3u) << 8) | (i & 3u));
      out[i] = h2_sub_mul(v & 0xFFF0FF0Fu, kLo | (kHi << 16), s);
    }
  }
}

template <bool W_MN, bool W4>
__global__ void __launch_bounds__(threads<W4>(), 1) gemm_grouped_pair_kernel(const __grid_constant__ Params p) {
  static_assert(!(W_MN && W4), "codes are K-major");
  static_assert(kStages % kExpandSets == 0, "a set returns to the same operand slots");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem<W4>& s = *reinterpret_cast<Smem<W4>*>(smem_raw + smem_align_pad(smem_raw));
  const uint32_t warp = warp_idx_sync();
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t rank = cluster_ctarank();
  const uint32_t pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  volatile uint32_t* abort = &s.abort;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&p.tm_w);
    tma_prefetch_desc(&p.tm_x);
    tma_prefetch_desc(&p.tm_xs);
    for (uint32_t i = 0; i < kStages; ++i) {
      mbar_init(&s.full[i], W4 ? 2 : 1);
      mbar_init(&s.empty[i], 1);
      mbar_init(&s.expanded[i], kSetThreads / 32);
    }
    for (uint32_t i = 0; i < kCodeSlots; ++i) {
      mbar_init(&s.codes_full[i], 1);
      mbar_init(&s.codes_empty[i], 2 * kSetThreads / 32);  // two stages read a slot
    }
    for (uint32_t i = 0; i < 2; ++i) {
      mbar_init(&s.tmem_full[i], 1);
      mbar_init(&s.tmem_empty[i], 2 * kEpiWarps);
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
    lin::group_tiles_prefix(p.groups, kTileT, s.prefix);
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before any remote arrive or TMA
  tc_fence_after_sync();
  pdl_launch_dependents();
  const uint32_t tmem_base = s.tmem_base;
  if (p.zero_others) lin::zero_other_rows(p.groups, p.out, p.ldo, p.cols, blockIdx.x, gridDim.x);

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, issued = 0;
      Tile w, next;
      bool ok = true;
      bool more = tile_at(p, s.prefix, pair, next);
      for (uint32_t t = pair; ok && more; t += num_pairs) {
        w = next;
        const uint32_t own_rows = w.n / 2u;  // rows of x in this CTA's half of the N operand
        const uint32_t box = own_rows > kSmallBox ? kBox : kSmallBox;
        const CUtensorMap* tm_x = own_rows > kSmallBox ? &p.tm_x : &p.tm_xs;
        const int32_t f = int32_t(w.f0 + rank * kRowsPerCta), row = int32_t(w.row0 + rank * own_rows);
        for (uint32_t kb = 0; kb < p.num_kb; ++kb) {
          if (!mbar_wait(&s.empty[stage], phase ^ 1u, abort, kStatusTimeoutProducer)) {
            ok = false;
            break;
          }
          const uint32_t full0 = map_to_rank(&s.full[stage], 0);
          if (rank == 0) {
            mbar_arrive_expect_tx(&s.full[stage], 2u * ((W4 ? 0u : kSubBytes) + box * kSubK * 2u));
          }
          const int32_t k = int32_t(kb * kSubK);
          if constexpr (W_MN) {
            tma_load_3d_pair(&p.tm_w, full0, s.a[stage], f, k, int32_t(w.e), kCacheEvictNormal);
            tma_load_3d_pair(&p.tm_w, full0, s.a[stage] + lin::kMnChunkBytes, f + 64, k, int32_t(w.e),
                             kCacheEvictNormal);
          } else if constexpr (!W4) {
            tma_load_3d_pair(&p.tm_w, full0, s.a[stage], k, f, int32_t(w.e), kCacheEvictNormal);
          }
          tma_load_2d_pair(tm_x, full0, s.b[stage], k, row, kCacheEvictNormal);
          ++issued;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
          if (kb == 0u) more = tile_at(p, s.prefix, t + num_pairs, next);
        }
      }
      // Loads in flight must land before the CTA may exit: all on rank 0's barriers, which rank 0
      // waits for (the closing cluster barrier keeps rank 1's shared memory alive until then).
      if (rank == 0) {
        for (uint32_t i = issued - min(issued, kStages); i < issued; ++i) {
          mbar_drain(&s.full[i % kStages], (i / kStages) & 1u);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ UMMA issuer (rank 0)
    // The whole warp walks (uniform values stay in uniform registers, fewer instructions per
    // stage), one lane issues.
    if (rank == 0) {
      const bool leader = elect_one();
      uint32_t stage = 0, phase = 0, local = 0;
      uint32_t full = 0, expanded = 0;  // the stage was seen complete by an early test
      bool ok = true;
      Tile w, next;
      bool more = tile_at(p, s.prefix, pair, next);
      for (uint32_t t = pair; ok && more; t += num_pairs, ++local) {
        w = next;
        const uint32_t idesc = W4 ? make_idesc(1, 0, 0, kTileF, w.n) : lin::idesc_of<W_MN, false>(kTileF, w.n);
        const uint32_t acc = local & 1u;
        const uint32_t acc_phase = (local >> 1) & 1u;
        if (!__all_sync(0xffffffffu, mbar_wait(&s.tmem_empty[acc], acc_phase ^ 1u, abort, kStatusTimeoutMma))) break;
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * kTileT;
        for (uint32_t kb = 0; kb < p.num_kb; ++kb) {
          if constexpr (W4) {
            // `full` also stands for the weights that rank 1 has expanded into its shared memory.
            ok = __all_sync(0xffffffffu,
                            (full != 0u || mbar_wait_relaxed(&s.full[stage], phase, abort, kStatusTimeoutMma)) &&
                                (expanded != 0u || mbar_wait(&s.expanded[stage], phase, abort, kStatusTimeoutMma)));
            fence_acquire_cluster_smem();
          } else {
            ok = __all_sync(0xffffffffu, full != 0u || mbar_wait(&s.full[stage], phase, abort, kStatusTimeoutMma));
          }
          if (!ok) break;
          tc_fence_after_sync();
          const uint64_t adesc = lin::operand_desc<W_MN>(s.a[stage]);
          const uint64_t bdesc = make_sw128_kmajor_desc(s.b[stage]);
#pragma unroll
          for (uint32_t k = 0; k < kSubK / kUmmaK; ++k) {
            if (leader) {
              umma_bf16_pair(d_tmem, desc_advance(adesc, k * lin::operand_step<W_MN>()),
                             desc_advance(bdesc, k * kUmmaK * 2), idesc, (kb | k) != 0u ? 1u : 0u);
            }
          }
          if (leader) umma_commit_pair(&s.empty[stage], 0x3);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
          // A test takes about 180 cycles to answer, a third of a stage's products: the next
          // stage's are asked together, and early.
          full = W4 ? mbar_test_relaxed(&s.full[stage], phase) : mbar_test(&s.full[stage], phase);
          if (W4) expanded = mbar_test(&s.expanded[stage], phase);
          if (kb == 0u) more = tile_at(p, s.prefix, t + num_pairs, next);
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
  } else if (W4 && warp == 2) {
    // ------------------------------------------------------------ TMA producer of the codes
    // A warp of its own: as a part of the other producer it would ask for a group's codes only
    // when the operand slot is free, and their way from memory would be waited for.
    if (lane == 0) {
      uint32_t slot = 0, phase = 0, issued = 0;
      bool ok = true;
      Tile w;
      for (uint32_t t = pair; ok && tile_at(p, s.prefix, t, w); t += num_pairs) {
        for (uint32_t g = 0; g < p.G; ++g) {
          if (!mbar_wait(&s.codes_empty[slot], phase ^ 1u, abort, kStatusTimeoutProducer)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&s.codes_full[slot], kCodeBytes);
          tma_load_3d(&p.tm_w, &s.codes_full[slot], s.codes[slot], int32_t(g * (kScaleGroup / 2)),
                      int32_t(w.f0 + rank * kRowsPerCta), int32_t(w.e), kCacheEvictNormal);
          ++issued;
          if (++slot == kCodeSlots) {
            slot = 0;
            phase ^= 1u;
          }
        }
      }
      for (uint32_t i = issued - min(issued, kCodeSlots); i < issued; ++i) {
        mbar_drain(&s.codes_full[i % kCodeSlots], (i / kCodeSlots) & 1u);
      }
    }
    __syncwarp();
  } else if (W4 && warp == 3) {
    // ------------------------------------------------------------ rank 1: "expanded" to rank 0
    if (rank == 1 && lane == 0) {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      Tile w;
      for (uint32_t t = pair; ok && tile_at(p, s.prefix, t, w); t += num_pairs) {
        for (uint32_t kb = 0; kb < p.num_kb && ok; ++kb) {
          ok = mbar_wait_poll(&s.expanded[stage], phase, abort, kStatusTimeoutUnpack);
          // The expanding warps made their writes visible to the tensor core (fence.proxy.async) in front
          // of "expanded"; this passes them on to the thread of rank 0 that issues the product.
          if (ok) {
            fence_release_cluster_smem();
            mbar_arrive_cluster_relaxed(map_to_rank(&s.full[stage], 0));
          }
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp >= 4 && warp < 4 + kEpiWarps) {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const uint32_t q = warp & 3u;
    const uint32_t wg = (warp - 4u) >> 2;
    const uint32_t fl = rank * kRowsPerCta + q * 32u + lane;  // column in the pair's tile
    const uint32_t empty0[2] = {map_to_rank(&s.tmem_empty[0], 0), map_to_rank(&s.tmem_empty[1], 0)};
    uint32_t local = 0;
    Tile w;
    for (uint32_t t = pair; tile_at(p, s.prefix, t, w); t += num_pairs, ++local) {
      const uint32_t f = w.f0 + fl;
      const bool valid = f < p.cols;
      float unscale = 1.f;
      if (W4 && valid) unscale = exp2i(-row_shift(p.sb + (size_t(w.e) * p.cols + f) * p.G, p.G));
      const uint32_t acc = local & 1u;
      const uint32_t acc_phase = (local >> 1) & 1u;
      if (!__all_sync(0xffffffffu, mbar_wait(&s.tmem_full[acc], acc_phase, abort, kStatusTimeoutEpilogue))) break;
      tc_fence_after_sync();
      const uint32_t t_row = tmem_base + ((q * 32u) << 16) + acc * kTileT;
#pragma unroll 1
      for (uint32_t c0 = wg * 32u; c0 < w.rows; c0 += 64u) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(t_row + c0, r);
        tmem_ld_wait();
        if (W4) {
          const uint32_t row = w.row0 + c0;
          const float sa = c0 + lane < w.rows ? __ldg(p.sa + row + lane) : 0.f;
#pragma unroll
          for (uint32_t j = 0; j < 32; ++j) {
            // In this order: the two scales' product may leave fp32 where the result does not.
            r[j] = __float_as_uint(__uint_as_float(r[j]) * unscale * __shfl_sync(0xffffffffu, sa, j));
          }
        }
        float v[32];
#pragma unroll
        for (uint32_t j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
        lin::store_columns(p.out + size_t(w.row0 + c0) * p.ldo + f, p.ldo, v, w.rows - c0, valid, p.pair_store);
        __syncwarp();
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(empty0[acc]);
    }
  } else if (W4 && warp >= 4 + kEpiWarps && (warp & 3u) != 1u) {
    // ------------------------------------------------------------ codes -> fp16 weights
    // Set j takes the stages c = j (mod kExpandSets) of the CTA's walk; stage c is half c & 1 of
    // scale group c / 2 (a tile has two stages per scale group). Thread (row, low) of a set
    // expands the 16-byte piece low of the rows row and row + 64, 32 codes each. Eight lanes write
    // four rows' 16-byte chunks, which the swizzle spreads over all banks.
    const uint32_t nth = ((warp - (4u + kEpiWarps)) >> 2) * 3u + ((warp & 3u) > 1u ? (warp & 3u) - 1u : 0u);
    const uint32_t xt = (nth & 3u) * 32u + lane;
    const uint32_t set = nth >> 2;
    const uint32_t row = xt >> 1, low = xt & 1u;
    uint32_t c0 = 0;  // stages of the walk before this tile
    Tile w;
    bool ok = true;
    for (uint32_t t = pair; ok && tile_at(p, s.prefix, t, w); t += num_pairs, c0 += p.num_kb) {
      const uint16_t* sb_row[2];
      float up[2];
      uint32_t next[2];
      // The set's first stage of this tile. A set must take every kExpandSets-th stage of the whole
      // walk (and so the same operand slots each time round): a parity wait tells a barrier's
      // phase only from the one before, which its waiter must have seen.
      uint32_t kb = (set + kExpandSets - c0 % kExpandSets) % kExpandSets;
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t f = w.f0 + rank * kRowsPerCta + row + 64u * i;
        sb_row[i] = p.sb + (size_t(w.e) * p.cols + (f < p.cols ? f : 0u)) * p.G;
        up[i] = exp2i(row_shift(sb_row[i], p.G));
        next[i] = kb < p.num_kb ? __ldg(sb_row[i] + kb / 2u) : 0u;
      }
      for (; kb < p.num_kb; kb += kExpandSets) {
        const uint32_t c = c0 + kb, slot = (c / 2u) % kCodeSlots, stage = c % kStages;
        float scale[2];
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
          scale[i] = bf16_bits_to_float(static_cast<uint16_t>(next[i])) * up[i];
          if (kb + kExpandSets < p.num_kb) next[i] = __ldg(sb_row[i] + (kb + kExpandSets) / 2u);
        }
        ok = __all_sync(0xffffffffu, mbar_wait_poll(&s.codes_full[slot], (c / 2u / kCodeSlots) & 1u, abort,
                                                    kStatusTimeoutUnpack));
        if (!ok) break;
        const uint8_t* src = s.codes[slot] + row * (kScaleGroup / 2) + (c & 1u) * 32u + low * 16u;
        const uint4 x[2] = {*reinterpret_cast<const uint4*>(src),
                            *reinterpret_cast<const uint4*>(src + 64u * (kScaleGroup / 2))};
        // The slot's next codes arrive by TMA: order this warp's reads before the release.
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.codes_empty[slot]);
        // The products that read this operand slot last have retired.
        ok = __all_sync(0xffffffffu,
                        mbar_wait_poll(&s.empty[stage], ((c / kStages) & 1u) ^ 1u, abort, kStatusTimeoutUnpack));
        if (!ok) break;
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
          uint32_t v[16];
          expand_codes(x[i], p.split, __half_as_ushort(__float2half_rn(scale[i])),
                       __half_as_ushort(__float2half_rn(scale[i] * 0.0625f)), v);
          uint8_t* dst = s.a[stage] + (row + 64u * i) * 128u;
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j) {
            *reinterpret_cast<uint4*>(dst + (((low * 4u + j) ^ (row & 7u)) << 4)) =
                make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.expanded[stage]);
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

// int8 rows -> fp16 (exact), the W4 kernel's N operand. HBM-bound: 3 bytes per element (the result
// mostly stays in L2 for the product). A thread has kWidenAhead 16-byte loads in flight and stores
// whole 32-byte sectors.
constexpr uint32_t kWidenThreads = 256;
constexpr uint32_t kWidenAhead = 4;
__global__ void __launch_bounds__(kWidenThreads) widen_rows_kernel(const uint4* src, uint4* dst, uint64_t pieces) {
  pdl_launch_dependents();
  pdl_wait();
  const uint64_t first = uint64_t(blockIdx.x) * (kWidenThreads * kWidenAhead) + threadIdx.x;
  uint4 x[kWidenAhead];
#pragma unroll
  for (uint32_t u = 0; u < kWidenAhead; ++u) {
    const uint64_t i = first + u * kWidenThreads;
    if (i < pieces) x[u] = __ldg(src + i);
  }
#pragma unroll
  for (uint32_t u = 0; u < kWidenAhead; ++u) {
    const uint64_t i = first + u * kWidenThreads;
    if (i >= pieces) break;
    const uint32_t w[4] = {x[u].x ^ 0x80808080u, x[u].y ^ 0x80808080u, x[u].z ^ 0x80808080u, x[u].w ^ 0x80808080u};
    uint32_t v[8];
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      // 1024 + (x + 128) - 1152 = x
      const uint32_t h = __byte_perm(w[j >> 1], 0x64646464u, (j & 1u) ? 0x4342u : 0x4140u);
      asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(v[j]) : "r"(h), "r"(0x64806480u));
    }
    if ((reinterpret_cast<uintptr_t>(dst) & 31u) == 0u) {
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + 2 * i), "r"(v[0]), "r"(v[1]),
                   "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                   : "memory");
    } else {
      dst[2 * i] = make_uint4(v[0], v[1], v[2], v[3]);
      dst[2 * i + 1] = make_uint4(v[4], v[5], v[6], v[7]);
    }
  }
}

}  // namespace grouppair
}  // namespace arcb
