// expert_layer.cuh — the expert layer of a few tokens, in two launches of one kernel.
//
//   FIRST   h[s] = act(x[t] g_e^T) * (x[t] u_e^T)   or act(x[t] w_e^T) without a gate
//   SECOND  y[t] = sum over t's choices s of weights[s] (h[s] w_e^T)
//   for the choices s = (t, j) of tokens t, e = ids[t, j]. An id outside [0, E) chooses nobody; an
//   expert chosen twice by a token counts with the sum of its weights.
//
// A few tokens choose most of the experts with a few rows each: the weights are the traffic, each read
// once, and everything else has to stay out of their way.
//
// * No sorting launch, no gathered copies. Every block sorts the choices in shared memory by itself (a
//   microsecond, in SECOND under the first launch), and the rows of x and h that belong to an expert
//   come by TMA gather, four rows an instruction.
// * Blocks walk over (expert, column tile) and their ring of loads runs on from one to the next, so the
//   stream of weights pauses only at a launch's ends. SECOND loads its first weights under FIRST's last tiles.
// * A tile is 32 WR weight rows; the eight warps are WR groups of rows times WK = 8 / WR parts of the
//   contraction. 32 rows make tiles fine enough to share evenly (one token, 8 experts, 2048 columns: 1024
//   tiles); wider tiles read the tokens' rows less often, which counts once an expert has many.
// * Products are mma.sync from registers: with at most 32 columns an operand byte is used for so little
//   arithmetic that the pipe idles either way, int4 codes pass through registers in any case, and
//   accumulators of 16 x 8 fit tiles of 16 columns, where UMMA's 128 lanes would cut the work into
//   pieces too coarse to share out.
// * SECOND keeps a column tile's sums of all tokens in shared memory and adds the experts in their order:
//   no atomics, no partial results in memory; where tiles are few a cluster shares the contraction and adds
//   its blocks' sums in rank order. The result does not depend on timing.
//
// Sums are fp32. h is rounded to bf16, the tensor cores' operand type, and the weights of the choices multiply
// fp32 sums. Codes of int4 weights are exact bf16; a group of 128 products is summed before its scale is
// applied in fp32.
#pragma once

#include "linear_common.cuh"

namespace arcb {
namespace experts {

constexpr uint32_t kConsumers = 8;  // warps
constexpr uint32_t kThreads = 32 * (kConsumers + 1);
constexpr uint32_t kRowBytes = 128;  // of a box: 64 bf16 or 256 codes
constexpr uint32_t kScaleGroup = 128;
constexpr uint32_t kMaxStages = 24;
constexpr uint16_t kNoExpert = 0xFFFFu;

struct Params {
  CUtensorMap tm_w;  // {K, columns, 2 or 1, E}, box {128 bytes, 16 WR, 2, 1} with a gate, else {.., 32 WR, 1, 1}; SW128
  CUtensorMap tm_x;  // {K, rows}, box {64, 1}, SW128
  const uint16_t* sb;   // int4: scales [E][weight rows][groups]
  const void* ids;      // [tokens][top]
  const void* weights;  // SECOND: [tokens][top], fp32 or bf16
  uint16_t* out;        // FIRST: h [slots][ldo]; SECOND: y [tokens][ldo]
  uint64_t ldo;
  uint32_t ids_wide, weights_bf16;  // int64 ids; bf16 weights
  uint32_t tokens, top, experts, slots;
  uint32_t cols, tiles;  // output columns, tiles of them
  uint32_t num_kb;       // boxes along the contraction
  uint32_t groups;       // scale groups along it
  uint32_t gated, act;
  uint32_t stages;       // of the ring, a multiple of WK
  uint32_t splits;       // SECOND: blocks of a cluster, which share the contraction
};

template <uint32_t NT, uint32_t WR, bool INT4>
struct Cfg {
  static_assert(NT == 8 || NT == 16 || NT == 32, "columns of a pass");
  static constexpr uint32_t kParts = kConsumers / WR;  // WK
  static_assert(kParts >= 2, "parts of the contraction");
  static constexpr uint32_t kRows = 32 * WR;
  static constexpr uint32_t kSub = INT4 ? 4 : 1;  // boxes of tokens per box of weights
  static constexpr uint32_t kWBytes = kRows * kRowBytes;
  static constexpr uint32_t kXBytes = NT * kRowBytes;  // a box of tokens
  static constexpr uint32_t kStageBytes = kWBytes + kSub * kXBytes;
  static constexpr uint32_t kSumBytes = kParts * kRows * NT * 4;
};

// One pass over an expert's weights, for up to NT of its choices.
struct Pass {
  uint16_t expert, first, count, unused;
};

// Shared memory behind the ring, in bytes from its end.
struct Layout {
  uint32_t sums, y, passes, list, ids, share, total;
};
__host__ __device__ inline Layout layout_of(uint32_t sum_bytes, uint32_t rows, uint32_t nt, uint32_t tokens,
                                            uint32_t slots, uint32_t experts, bool second) {
  const auto up = [](uint32_t v) { return (v + 15u) & ~15u; };
  Layout l;
  l.sums = 0;
  l.y = l.sums + sum_bytes;
  l.passes = l.y + (second ? tokens * rows * 4u : 0u);
  const uint32_t live = experts < slots ? experts : slots;
  l.list = l.passes + up((live + slots / nt) * 8u);
  l.ids = l.list + up(slots * 2u);
  l.share = l.ids + up(slots * 2u);
  l.total = l.share + (second ? up(slots * 4u) : 0u);
  return l;
}

// ---------------------------------------------------------------------------------
// Instructions
// ---------------------------------------------------------------------------------
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void lds_128(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four rows of a matrix, 128 bytes each from column x on; a row outside it comes as zeros.
__device__ __forceinline__ void tma_gather4(const CUtensorMap* map, uint64_t* bar, void* dst, int32_t x, int32_t r0,
                                            int32_t r1, int32_t r2, int32_t r3, uint64_t cache_hint) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1, {%3, %4, %5, %6, %7}], [%2], %8;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3),
      "l"(cache_hint)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(const CUtensorMap* map, uint64_t* bar, void* dst, int32_t x, int32_t y,
                                            int32_t z, int32_t w, uint64_t cache_hint) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "l"(cache_hint)
      : "memory");
}

// Eight int4 codes (k = 0..7 from the low nibble up) as bf16 pairs (0, 4), (1, 5), (2, 6), (3, 7). 0x4300 | m is
// the bf16 128 + m; a code's nibble with its sign bit turned over is code + 8, so 136 is taken off again, exactly.
__device__ __forceinline__ void codes_to_bf16(uint32_t w, uint32_t (&v)[4]) {
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    uint32_t m;
    asm("lop3.b32 %0, %1, 0x000F000F, 0x43084308, 0x6A;" : "=r"(m) : "r"(w >> (4 * i)));  // (a & b) ^ c
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(v[i]) : "r"(m), "r"(0x43084308u));
  }
}

// ---------------------------------------------------------------------------------
// The choices, sorted by expert in shared memory by the whole block: `list` holds the choices of
// every expert in their order, `passes` which of them a pass takes. Returns the number of passes.
// Every block must find the same, so the order is that of the choices: one warp counts
// 32 of them at a time.
// ---------------------------------------------------------------------------------
template <uint32_t NT>
__device__ __forceinline__ uint32_t sort_choices(const Params& p, Pass* passes, uint16_t* list, uint16_t* ids,
                                                 uint16_t* count /* [experts], scratch */, uint32_t* totals) {
  const uint32_t tid = threadIdx.x, lane = tid & 31u;
  for (uint32_t s = tid; s < p.slots; s += kThreads) {
    uint16_t id = kNoExpert;
    if (p.ids_wide) {
      const int64_t v = __ldg(static_cast<const long long*>(p.ids) + s);
      if (v >= 0 && v < static_cast<int64_t>(p.experts)) id = static_cast<uint16_t>(v);
    } else {
      const int32_t v = __ldg(static_cast<const int32_t*>(p.ids) + s);
      if (v >= 0 && v < static_cast<int32_t>(p.experts)) id = static_cast<uint16_t>(v);
    }
    ids[s] = id;
  }
  for (uint32_t e = tid; e < p.experts; e += kThreads) count[e] = 0;
  __syncthreads();
  // A choice that repeats an earlier one of its token adds nothing of its own. `list` notes it for now.
  for (uint32_t s = tid; s < p.slots; s += kThreads) {
    uint16_t id = ids[s];
    for (uint32_t i = s - s % p.top; i < s; ++i) {
      if (ids[i] == id) id = kNoExpert;
    }
    list[s] = id;
  }
  __syncthreads();
  if (tid < 32u) {
    // Counts, first choice and first pass of each expert.
    for (uint32_t s0 = 0; s0 < p.slots; s0 += 32u) {
      const uint32_t id = s0 + lane < p.slots ? list[s0 + lane] : kNoExpert;
      const uint32_t same = __match_any_sync(0xffffffffu, id);
      if (id != kNoExpert && (same >> lane) == 1u) count[id] = static_cast<uint16_t>(count[id] + __popc(same));
      __syncwarp();
    }
    uint32_t base = 0;  // choices in the lower half, passes in the upper
    for (uint32_t e0 = 0; e0 < p.experts; e0 += 32u) {
      const uint32_t e = e0 + lane;
      const uint32_t c = e < p.experts ? count[e] : 0u;
      const uint32_t own = c | (c + NT - 1u) / NT << 16;
      uint32_t incl = own;
#pragma unroll
      for (uint32_t d = 1; d < 32u; d <<= 1) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
      }
      const uint32_t at = base + incl - own;
      const uint32_t first = at & 0xFFFFu;
      for (uint32_t i = 0; i * NT < c; ++i) {
        passes[(at >> 16) + i] = {static_cast<uint16_t>(e), static_cast<uint16_t>(first + i * NT),
                                  static_cast<uint16_t>(min(NT, c - i * NT)), 0};
      }
      if (e < p.experts) count[e] = static_cast<uint16_t>(first);  // from here on the place of its next choice
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) *totals = base >> 16;
    __syncwarp();
    // `ids` takes over which choices count; then every choice goes to its place.
    for (uint32_t s = lane; s < p.slots; s += 32u) ids[s] = list[s];
    __syncwarp();
    for (uint32_t s0 = 0; s0 < p.slots; s0 += 32u) {
      const uint32_t id = s0 + lane < p.slots ? ids[s0 + lane] : kNoExpert;
      const uint32_t same = __match_any_sync(0xffffffffu, id);
      const uint32_t before = __popc(same & ((1u << lane) - 1u));
      if (id != kNoExpert) list[count[id] + before] = static_cast<uint16_t>(s0 + lane);
      __syncwarp();
      if (id != kNoExpert && (same >> lane) == 1u) count[id] = static_cast<uint16_t>(count[id] + before + 1u);
      __syncwarp();
    }
  }
  __syncthreads();
  return *totals;
}

// The weight of choice s: with those of its token's later choices of the same expert.
__device__ __forceinline__ float share_of(const Params& p, uint32_t s) {
  float sum = 0.f;
  const uint32_t end = s - s % p.top + p.top;
  int64_t own = 0;
  for (uint32_t i = s; i < end; ++i) {
    const int64_t id = p.ids_wide ? static_cast<int64_t>(__ldg(static_cast<const long long*>(p.ids) + i))
                                  : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(p.ids) + i));
    if (i == s) own = id;
    if (id == own) {
      sum += p.weights_bf16 ? bf16_bits_to_float(__ldg(static_cast<const uint16_t*>(p.weights) + i))
                            : __ldg(static_cast<const float*>(p.weights) + i);
    }
  }
  return sum;
}

template <uint32_t NT, uint32_t WR, bool INT4, bool SECOND>
__global__ void __launch_bounds__(kThreads, 2) expert_layer_kernel(const __grid_constant__ Params p) {
  using C = Cfg<NT, WR, INT4>;
  constexpr uint32_t WK = C::kParts;
  constexpr uint32_t kTiles8 = NT / 8;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages];
  __shared__ uint32_t abort_flag, num_passes;
  uint8_t* ring = smem_raw + smem_align_pad(smem_raw);
  uint8_t* rest = ring + p.stages * C::kStageBytes;
  const Layout l = layout_of(C::kSumBytes, C::kRows, NT, p.tokens, p.slots, p.experts, SECOND);
  float* sums = reinterpret_cast<float*>(rest + l.sums);  // [WK][kTiles8][kRows][8]
  float* y = reinterpret_cast<float*>(rest + l.y);        // SECOND: [tokens][kRows]
  Pass* passes = reinterpret_cast<Pass*>(rest + l.passes);
  uint16_t* list = reinterpret_cast<uint16_t*>(rest + l.list);
  uint16_t* ids = reinterpret_cast<uint16_t*>(rest + l.ids);
  float* share = reinterpret_cast<float*>(rest + l.share);  // SECOND: weights in the order of `list`

  const uint32_t warp = warp_idx_sync();
  const uint32_t lane = threadIdx.x & 31u;
  volatile uint32_t* abort = &abort_flag;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&p.tm_w);
    tma_prefetch_desc(&p.tm_x);
    for (uint32_t i = 0; i < p.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], WR);
    }
    abort_flag = 0;
    fence_barrier_init();
  }
  // The choices and their weights are older than the first launch, which has waited for them before it
  // lets the second one in.
  if (!SECOND) {
    pdl_wait();
    pdl_launch_dependents();
  }
  const uint32_t passes_n = sort_choices<NT>(p, passes, list, ids, reinterpret_cast<uint16_t*>(ring), &num_passes);
  if (SECOND) {
    for (uint32_t i = threadIdx.x; i < p.tokens * C::kRows; i += kThreads) y[i] = 0.f;
    const uint32_t listed = passes_n == 0u ? 0u : passes[passes_n - 1u].first + passes[passes_n - 1u].count;
    for (uint32_t i = threadIdx.x; i < listed; i += kThreads) share[i] = share_of(p, list[i]);
  }
  // The ring held scratch of the sorting: order its writes before the loads.
  fence_proxy_async_smem();
  __syncthreads();

  // This block's walk: items of (pass, column tile), each a run of boxes along the contraction.
  const uint32_t rank = SECOND && p.splits > 1u ? cluster_ctarank() : 0u;
  const uint32_t kb0 = SECOND ? p.num_kb * rank / p.splits : 0u;
  const uint32_t nkb = SECOND ? p.num_kb * (rank + 1u) / p.splits - kb0 : p.num_kb;
  const uint32_t tile_cols = p.gated ? C::kRows / 2u : C::kRows;
  uint32_t item0, item_step, item_end;
  if (SECOND) {  // one tile, every pass
    item0 = 0;
    item_step = 1;
    item_end = passes_n;
  } else {  // tiles of a pass side by side
    item0 = blockIdx.x;
    item_step = gridDim.x;
    item_end = passes_n * p.tiles;
  }
  const uint32_t my_tile = SECOND ? blockIdx.x / p.splits : 0u;

  if (warp == kConsumers) {
    // ------------------------------------------------------------ producer
    uint32_t stage = 0, phase = 0, issued = 0;
    bool ok = true;
    const auto coords = [&](uint32_t item, Pass& ps, uint32_t& f0) {
      const uint32_t pi = SECOND ? item : item / p.tiles;
      ps = passes[pi];
      f0 = (SECOND ? my_tile : item - pi * p.tiles) * tile_cols;
    };
    const auto load_weights = [&](const Pass& ps, uint32_t f0, uint32_t kb, uint32_t st) {
      const uint32_t quads = (ps.count + 3u) / 4u;
      mbar_arrive_expect_tx(&full[st], C::kWBytes + C::kSub * quads * 4u * kRowBytes);
      tma_load_4d(&p.tm_w, &full[st], ring + st * C::kStageBytes, int32_t(kb * (INT4 ? kRowBytes : kRowBytes / 2u)),
                  int32_t(f0), 0, ps.expert, kCacheEvictNormal);
    };
    const auto load_rows = [&](const Pass& ps, uint32_t kb, uint32_t st) {
      const uint32_t quads = (ps.count + 3u) / 4u;
      for (uint32_t g = lane; g < quads * C::kSub; g += 32u) {
        const uint32_t sub = g / quads, quad = g - sub * quads;
        int32_t r[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          const uint32_t c = quad * 4u + i;
          const uint32_t s = list[ps.first + min(c, ps.count - 1u)];
          r[i] = c < ps.count ? int32_t(SECOND ? s : s / p.top) : int32_t(SECOND ? p.slots : p.tokens);
        }
        tma_gather4(&p.tm_x, &full[st], ring + st * C::kStageBytes + C::kWBytes + sub * C::kXBytes + quad * 4u * kRowBytes,
                    int32_t((kb * C::kSub + sub) * 64u), r[0], r[1], r[2], r[3], kCacheEvictLast);
      }
    };
    uint32_t ahead = 0;  // boxes whose weights are on their way
    if (SECOND) {
      // The first weights do not wait for the first launch.
      ahead = min(p.stages, item_end * nkb);
      if (lane == 0) {
        for (uint32_t b = 0; b < ahead; ++b) {
          Pass ps;
          uint32_t f0;
          coords(b / nkb, ps, f0);
          load_weights(ps, f0, kb0 + b % nkb, b);
        }
      }
      __syncwarp();
      pdl_wait();
      pdl_launch_dependents();
    }
    for (uint32_t item = item0; ok && item < item_end; item += item_step) {
      Pass ps;
      uint32_t f0;
      coords(item, ps, f0);
      for (uint32_t kb = 0; kb < nkb; ++kb) {
        if (issued >= ahead) {
          if (lane == 0) {
            ok = mbar_wait(&empty[stage], phase ^ 1u, abort, kStatusTimeoutProducer);
            if (ok) load_weights(ps, f0, kb0 + kb, stage);
          }
          ok = __shfl_sync(0xffffffffu, ok ? 1u : 0u, 0) != 0u;
          if (!ok) break;
        }
        load_rows(ps, kb0 + kb, stage);
        ++issued;
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // Copies in flight land before the block may exit (of every box both parts are on their way: the
    // only wait that can be abandoned comes behind the boxes loaded ahead).
    if (lane == 0) {
      const uint32_t n = min(issued, p.stages);
      for (uint32_t i = issued - n; i < issued; ++i) mbar_drain(&full[i % p.stages], (i / p.stages) & 1u);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ consumers
    if (SECOND) pdl_wait();
    const uint32_t wr = warp % WR, part = warp / WR;
    const uint32_t g8 = lane >> 2, q = lane & 3u;
    uint32_t stage = part, phase = 0;  // of this part's next box
    uint32_t done = 0;                 // boxes of the items before
    bool ok = true;
    for (uint32_t item = item0; item < item_end; item += item_step) {
      const uint32_t pi = SECOND ? item : item / p.tiles;
      const Pass ps = passes[pi];
      const uint32_t f0 = (SECOND ? my_tile : item - pi * p.tiles) * tile_cols;
      float acc[2][kTiles8][4];
#pragma unroll
      for (uint32_t m = 0; m < 2; ++m) {
#pragma unroll
        for (uint32_t j = 0; j < kTiles8; ++j) {
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
        }
      }
      // The boxes whose running number is `part` modulo WK.
      for (uint32_t kb = (part + WK - done % WK) % WK; kb < nkb; kb += WK) {
        uint32_t scale_bits[2][2];  // int4: of the box's two groups, per block of rows: rows g8 and g8 + 8
        if constexpr (INT4) {
          const uint32_t g0 = (kb0 + kb) * 2u;
#pragma unroll
          for (uint32_t m = 0; m < 2; ++m) {
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
              const uint32_t f = f0 + (p.gated ? wr * 16u : (m * WR + wr) * 16u) + i * 8u + g8;
              const uint32_t row = f + (p.gated ? m * p.cols : 0u);
              uint32_t bits = 0;
              if (f < p.cols) {
                const uint16_t* at = p.sb + (size_t(ps.expert) * (p.gated ? 2u * p.cols : p.cols) + row) * p.groups + g0;
                bits = __ldg(at);
                if (g0 + 1u < p.groups) bits |= static_cast<uint32_t>(__ldg(at + 1)) << 16;
              }
              scale_bits[m][i] = bits;
            }
          }
        }
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, abort, kStatusTimeoutMma));
        const uint32_t w_at = smem_u32(ring + stage * C::kStageBytes), x_at = w_at + C::kWBytes;
        if (ok) {
          if constexpr (!INT4) {
#pragma unroll
            for (uint32_t half = 0; half < 2; ++half) {  // 32 of the contraction
              uint32_t b[kTiles8][4];
#pragma unroll
              for (uint32_t j = 0; j < kTiles8; ++j) {
                if (j * 8u < ps.count) {
                  const uint32_t row = lane & 7u, chunk = half * 4u + (lane >> 3);
                  ldmatrix_x4(x_at + (j * 8u + row) * kRowBytes + ((chunk ^ row) << 4), b[j]);
                }
              }
#pragma unroll
              for (uint32_t m = 0; m < 2; ++m) {
#pragma unroll
                for (uint32_t k = 0; k < 2; ++k) {
                  uint32_t a[4];
                  const uint32_t row = (m * WR + wr) * 16u + (lane & 15u), chunk = half * 4u + k * 2u + (lane >> 4);
                  ldmatrix_x4(w_at + row * kRowBytes + ((chunk ^ (row & 7u)) << 4), a);
#pragma unroll
                  for (uint32_t j = 0; j < kTiles8; ++j) {
                    if (j * 8u < ps.count) mma_bf16(acc[m][j], a[0], a[1], a[2], a[3], b[j][2 * k], b[j][2 * k + 1]);
                  }
                }
              }
            }
          } else {
#pragma unroll
            for (uint32_t g = 0; g < 2; ++g) {  // scale groups
              float part_sum[2][kTiles8][4];
#pragma unroll
              for (uint32_t m = 0; m < 2; ++m) {
#pragma unroll
                for (uint32_t j = 0; j < kTiles8; ++j) {
#pragma unroll
                  for (uint32_t i = 0; i < 4; ++i) part_sum[m][j][i] = 0.f;
                }
              }
#pragma unroll
              for (uint32_t c4 = 0; c4 < 4; ++c4) {  // 32 codes of a row, 16 bytes
                const uint32_t c = g * 4u + c4;
                uint32_t a[4];  // rows 0-7 and 8-15 of the two blocks of rows
                {
                  const uint32_t row = ((lane >> 4) * WR + wr) * 16u + (lane & 15u);
                  ldmatrix_x4(w_at + row * kRowBytes + ((c ^ (row & 7u)) << 4), a);
                }
                uint32_t v[4][4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) codes_to_bf16(a[i], v[i]);
#pragma unroll
                for (uint32_t j = 0; j < kTiles8; ++j) {
                  if (j * 8u < ps.count) {
                    // Lanes of column n take row n / 2 + 4 (n % 2), so that a quarter of a warp reads all banks.
                    const uint32_t row = (g8 >> 1) | (g8 & 1u) << 2, chunk = (c & 1u) * 4u + q;
                    uint32_t x[4];  // k = 8 q .. 8 q + 7 of the 32
                    lds_128(x_at + (c >> 1) * C::kXBytes + (j * 8u + row) * kRowBytes + ((chunk ^ row) << 4), x);
                    const uint32_t b0 = __byte_perm(x[0], x[2], 0x5410), b1 = __byte_perm(x[0], x[2], 0x7632);
                    const uint32_t b2 = __byte_perm(x[1], x[3], 0x5410), b3 = __byte_perm(x[1], x[3], 0x7632);
#pragma unroll
                    for (uint32_t m = 0; m < 2; ++m) {
                      mma_bf16(part_sum[m][j], v[2 * m][0], v[2 * m + 1][0], v[2 * m][1], v[2 * m + 1][1], b0, b1);
                      mma_bf16(part_sum[m][j], v[2 * m][2], v[2 * m + 1][2], v[2 * m][3], v[2 * m + 1][3], b2, b3);
                    }
                  }
                }
              }
#pragma unroll
              for (uint32_t m = 0; m < 2; ++m) {
                const float s0 = __uint_as_float(g == 0 ? scale_bits[m][0] << 16 : scale_bits[m][0] & 0xFFFF0000u);
                const float s1 = __uint_as_float(g == 0 ? scale_bits[m][1] << 16 : scale_bits[m][1] & 0xFFFF0000u);
#pragma unroll
                for (uint32_t j = 0; j < kTiles8; ++j) {
                  if (j * 8u < ps.count) {
                    acc[m][j][0] = fmaf(s0, part_sum[m][j][0], acc[m][j][0]);
                    acc[m][j][1] = fmaf(s0, part_sum[m][j][1], acc[m][j][1]);
                    acc[m][j][2] = fmaf(s1, part_sum[m][j][2], acc[m][j][2]);
                    acc[m][j][3] = fmaf(s1, part_sum[m][j][3], acc[m][j][3]);
                  }
                }
              }
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[stage]);
        }
        stage += WK;
        if (stage >= p.stages) {
          stage -= p.stages;
          phase ^= 1u;
        }
      }
      done += nkb;

      // The parts' sums meet in shared memory.
      named_barrier_sync(1, kConsumers * 32);  // the last item's have been read
#pragma unroll
      for (uint32_t j = 0; j < kTiles8; ++j) {
        if (j * 8u < ps.count) {
#pragma unroll
          for (uint32_t m = 0; m < 2; ++m) {
            float* at = sums + ((part * kTiles8 + j) * C::kRows + (m * WR + wr) * 16u + g8) * 8u;
            if constexpr (INT4) {
              at[q] = acc[m][j][0];
              at[q + 4] = acc[m][j][1];
              at[64 + q] = acc[m][j][2];
              at[64 + q + 4] = acc[m][j][3];
            } else {
              *reinterpret_cast<float2*>(at + 2 * q) = make_float2(acc[m][j][0], acc[m][j][1]);
              *reinterpret_cast<float2*>(at + 64 + 2 * q) = make_float2(acc[m][j][2], acc[m][j][3]);
            }
          }
        }
      }
      named_barrier_sync(1, kConsumers * 32);
      const auto total = [&](uint32_t row, uint32_t c) {
        float v = 0.f;
#pragma unroll
        for (uint32_t k = 0; k < WK; ++k) v += sums[((k * kTiles8 + (c >> 3)) * C::kRows + row) * 8u + (c & 7u)];
        return v;
      };
      for (uint32_t o = threadIdx.x; o < tile_cols * ps.count; o += kConsumers * 32u) {
        const uint32_t f = o % tile_cols, c = o / tile_cols;
        if (f0 + f >= p.cols) continue;
        const uint32_t s = list[ps.first + c];
        if (SECOND) {
          float* at = y + (s / p.top) * C::kRows + f;
          *at = fmaf(share[ps.first + c], total(f, c), *at);
        } else {
          float v[2] = {total(f, c), 0.f};
          lin::activate(v, p.act);
          if (p.gated) v[0] *= total(C::kRows / 2u + f, c);
          p.out[size_t(s) * p.ldo + f0 + f] = __bfloat16_as_ushort(__float2bfloat16_rn(v[0]));
        }
      }
    }
    if (SECOND) named_barrier_sync(1, kConsumers * 32);  // all experts are in y
  }

  if (SECOND) {
    const uint32_t f0 = my_tile * C::kRows, cols = min(C::kRows, p.cols - f0);
    if (p.splits > 1u) {
      __syncthreads();
      cluster_sync_all();
      // Block r of the cluster finishes the tokens r, r + S, ...
      for (uint32_t o = threadIdx.x; o < p.tokens * C::kRows; o += kThreads) {
        const uint32_t f = o % C::kRows, t = o / C::kRows;
        if (t % p.splits != rank || f >= cols) continue;
        float v = 0.f;
        for (uint32_t i = 0; i < p.splits; ++i) v += ld_dsmem_f32(map_to_rank(y + o, i));
        p.out[size_t(t) * p.ldo + f0 + f] = __bfloat16_as_ushort(__float2bfloat16_rn(v));
      }
      cluster_sync_all();
    } else if (warp < kConsumers) {
      for (uint32_t o = threadIdx.x; o < p.tokens * C::kRows; o += kConsumers * 32u) {
        const uint32_t f = o % C::kRows, t = o / C::kRows;
        if (f < cols) p.out[size_t(t) * p.ldo + f0 + f] = __bfloat16_as_ushort(__float2bfloat16_rn(y[o]));
      }
    }
  }
}

}  // namespace experts
}  // namespace arcb
