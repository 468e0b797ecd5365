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
// * No sorting launch. Every block sorts the choices in shared memory by itself (a microsecond or two, in SECOND under the
//   first launch), and the rows of x and h that belong to an expert come by TMA gather, four rows an instruction. Where
//   experts have many rows gathers hold the stream up (128 tokens, 64 experts of 2048 x 4096: loads alone 711 us,
//   508 without the rows), so h lies in the sorted order, eight rows a load, and a small launch in front puts the
//   rows of x there as well (expert_rows_kernel).
// * Blocks walk over (expert, column tile) and their ring of loads runs on from one to the next, so the
//   stream of weights pauses only at a launch's ends. SECOND loads its first weights under FIRST's last tiles.
// * A tile is WR groups of MR blocks of 16 weight rows; the eight warps are the WR groups times WK = 8 / WR parts of the
//   contraction. 64 rows make tiles fine enough to share evenly (one token, 8 experts, 2048 gated columns: 512
//   tiles); wider tiles read the tokens' rows less often, which counts once an expert has many.
// * Products are mma.sync from registers: with at most 32 columns an operand byte is used for so little
//   arithmetic that the pipe idles either way, int4 codes pass through registers in any case, and
//   accumulators of 16 x 8 fit tiles of 16 columns, where UMMA's 128 lanes would cut the work into
//   pieces too coarse to share out.
// * SECOND keeps a column tile's sums of all tokens in shared memory and adds the experts in their order:
//   no atomics, no partial results in memory; where tiles are few a cluster shares the passes' boxes and adds
//   its blocks' sums in rank order. The result does not depend on timing, but a token's last bits do on the other tokens: the
//   boxes of all passes are shared evenly, so where its sums are cut is a matter of what the others chose. (Cuts that
//   depend on the expert alone leave parts of a short contraction idle where the parts' sums meet: int4, 32 tokens, 198 us so
//   and 255 with them.)
//
// Bound by HBM with bf16 weights (16 tokens, 64 experts of 4096 x 2048, 8 a token: 334 us for 339 at the measured copy
// rate; one token 69 for 62). With int4 ones 32 tokens (60 passes over 48 experts) take 189 to 207 us for 96: the products alone
// take 149, the loads alone 134, and two stages a warp do not hide all of either under the other.
//
// Sums are fp32. h is rounded to bf16, the tensor cores' operand type, and the weights of the choices multiply
// fp32 sums. Codes of int4 weights enter as code + 8, exactly, and 8 times the group's sum of x, which the tensor cores give
// beside it, is taken off in fp32 before the scale is applied: the sum of a group is off by what 256 products of up to
// (16 + code) |x| leave, more than |code x| would where a large x has small codes.
#pragma once

#include "linear_common.cuh"

namespace arcb {
namespace experts {

constexpr uint32_t kConsumers = 8;  // warps
constexpr uint32_t kThreads = 32 * (kConsumers + 1);
constexpr uint32_t kRowBytes = 128;  // of a box of 64 bf16; one of 128 codes, a scale group, has 64
constexpr uint32_t kScaleGroup = 128;
constexpr uint32_t kMaxStages = 32;
constexpr uint16_t kNoExpert = 0xFFFFu;
constexpr uint16_t kRepeat = 0x8000u;  // beside an id: an earlier choice of the token is the same

struct Params {
  // {K or K / 2 bytes, columns, 2 or 1, E}: a box is 64 of a row (bf16 SW128, codes SW64) of a tile's rows, with a gate
  // half of them gate and half up.
  CUtensorMap tm_w;
  CUtensorMap tm_x;  // {K, rows}, SW128, box {64, 8}, of rows in the sorted order; else, of tokens, {64, 1}
  const uint16_t* sb;   // int4: scales [E][weight rows][groups]
  const void* ids;      // [tokens][top]
  const void* weights;  // SECOND: [tokens][top], fp32 or bf16
  uint16_t* out;        // FIRST: h [slots][ldo], sorted by expert; SECOND: y [tokens][ldo]
  uint64_t ldo;
  uint32_t ids_wide, weights_bf16;  // int64 ids; bf16 weights
  uint32_t tokens, top, experts, slots;
  uint32_t top_inverse;  // ceil(2^32 / top), for choices below 2^16; 0 for one choice a token
  uint32_t cols, tiles;  // output columns, tiles of them
  uint32_t num_kb;       // boxes along the contraction
  uint32_t groups;       // scale groups along it
  uint32_t gated, act;
  uint32_t sorted;       // FIRST: rows of x lie in the order of the sorted choices
  uint32_t stages;       // of the ring, a multiple of WK
  uint32_t splits;       // SECOND: blocks of a cluster, which share the passes' boxes
  uint32_t own_y;        // SECOND: see Layout
};

// NT columns of a pass; a tile is WR groups of MR blocks of 16 weight rows.
template <uint32_t NT, uint32_t MR, uint32_t WR, bool INT4>
struct Cfg {
  static_assert(NT == 8 || NT == 16 || NT == 32, "columns of a pass");
  static_assert(MR == 2 || MR == 4, "blocks of rows: half of them gate, half of them up");
  static constexpr uint32_t kParts = kConsumers / WR;  // WK
  static_assert(kParts >= 2, "parts of the contraction");
  static constexpr uint32_t kRows = 16 * MR * WR;
  static constexpr uint32_t kSub = INT4 ? 2 : 1;  // boxes of tokens per box of weights
  static constexpr uint32_t kWRow = INT4 ? 64 : kRowBytes;
  static constexpr uint32_t kWBytes = kRows * kWRow;
  static constexpr uint32_t kXBytes = NT * kRowBytes;  // a box of tokens
  static constexpr uint32_t kStageBytes = kWBytes + kSub * kXBytes;
  static constexpr uint32_t kSumBytes = kParts * kRows * NT * 4;
  static constexpr uint32_t kBatch = kParts < 4 ? kParts : 4;  // boxes loaded at a time
};

// One pass over an expert's weights, for up to NT of its choices.
struct Pass {
  uint16_t expert, first, count, unused;
};

// Shared memory behind the ring, in bytes from its end. SECOND with `own_y`: every part of the contraction adds
// to sums of y of its own, and the parts' sums of an item are not exchanged.
struct Layout {
  uint32_t sums, y, passes, list, ids, share, total;
};
__host__ __device__ inline Layout layout_of(uint32_t sum_bytes, uint32_t parts, uint32_t rows, uint32_t nt,
                                            uint32_t tokens, uint32_t slots, uint32_t experts, bool second, bool own_y) {
  const auto up = [](uint32_t v) { return (v + 15u) & ~15u; };
  Layout l;
  l.sums = 0;
  l.y = l.sums + (own_y ? 0u : sum_bytes);
  l.passes = l.y + (second ? tokens * rows * 4u * (own_y ? parts : 1u) : 0u);
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
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four rows of a matrix, 128 bytes each from column x on; a row outside it comes as zeros.
__device__ __forceinline__ void tma_gather4(const CUtensorMap* map, uint64_t* bar, void* dst, int32_t x, int32_t r0,
                                            int32_t r1, int32_t r2, int32_t r3, uint64_t cache_hint) {
  asm(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1, {%3, %4, %5, %6, %7}], [%2], %8;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3),
      "l"(cache_hint)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(const CUtensorMap* map, uint64_t* bar, void* dst, int32_t x, int32_t y,
                                            int32_t z, int32_t w, uint64_t cache_hint) {
  asm(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "l"(cache_hint)
      : "memory");
}

// The same with sums that start from others.
__device__ __forceinline__ void mma_bf16_from(float (&d)[4], const float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// And from zero.
__device__ __forceinline__ void mma_bf16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Eight int4 codes (k = 0..7 from the low nibble up) as bf16 pairs (0, 4), (1, 5), (2, 6), (3, 7). A nibble with its sign
// bit turned over is code + 8, and as the lowest bits of a bf16 it is that many units of 2^-133: below 2^-125 the bits
// of a bf16 are an integer. So a mask is all that the even pairs cost; the odd ones, four bits further up, come as 16 times as
// much, for which their x is 16 times smaller. (Nibbles moved to a place of their own in the mantissa of 128 + n took two
// instructions more for eight codes, 7 instead of 5, on the pipe that bounds the kernel.)
__device__ __forceinline__ void codes_to_bf16(uint32_t w, uint32_t (&v)[4]) {
  const uint32_t u = w >> 8;
  asm("lop3.b32 %0, %1, 0x000F000F, 0x00080008, 0x6A;" : "=r"(v[0]) : "r"(w));  // (a & b) ^ c
  asm("lop3.b32 %0, %1, 0x00F000F0, 0x00800080, 0x6A;" : "=r"(v[1]) : "r"(w));
  asm("lop3.b32 %0, %1, 0x000F000F, 0x00080008, 0x6A;" : "=r"(v[2]) : "r"(u));
  asm("lop3.b32 %0, %1, 0x00F000F0, 0x00800080, 0x6A;" : "=r"(v[3]) : "r"(u));
}
// Minus the eights that come with the codes.
constexpr uint32_t kEightEven = 0x80088008u, kEightOdd = 0x80808080u;  // -8 and -128 units
// x is multiplied by 2^64 (even pairs) and 2^60, so that products of codes are normal fp32 numbers, and the sums are in
// units of 2^-69. |x| must be below 2^63; what a group's sum loses to the end of fp32's range is below 2^-80 a product.
constexpr uint32_t kScaleEven = 0x5F805F80u, kScaleOdd = 0x5D805D80u;  // two bf16 each
constexpr float kCodeUnit = 590295810358705651712.f;                   // 2^69
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// ---------------------------------------------------------------------------------
// The choices, sorted by expert in shared memory by the whole block: `list` holds the choices of
// every expert in their order, `passes` which of them a pass takes. Returns the number of passes.
// Every block must find the same, so the order is that of the choices: eight warps have a contiguous share each, which
// they count, and place behind the shares before, 32 choices at a time (one warp alone took 15 us for 1024). `ids` keeps
// all choices' experts, repeats marked.
// ---------------------------------------------------------------------------------
constexpr uint32_t kSortWarps = 8;
__host__ __device__ constexpr uint32_t sort_scratch(uint32_t experts) { return kSortWarps * experts * 2u; }

// Choices and their weights are read past the L1 cache: a block that does not wait for the launch in front may start
// beside lines that are older than they are.
__device__ __forceinline__ int64_t id_at(const Params& p, uint32_t s) {
  return p.ids_wide ? static_cast<int64_t>(__ldcg(static_cast<const long long*>(p.ids) + s))
                    : static_cast<int64_t>(__ldcg(static_cast<const int32_t*>(p.ids) + s));
}

template <uint32_t NT>
__device__ __forceinline__ uint32_t sort_choices(const Params& p, Pass* passes, uint16_t* list, uint16_t* ids,
                                                 uint16_t* counts /* [kSortWarps][experts], scratch */, uint32_t* totals) {
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  const auto id_of = [&](uint32_t s) {
    const int64_t v = id_at(p, s);
    return v >= 0 && v < static_cast<int64_t>(p.experts) ? static_cast<uint16_t>(v) : kNoExpert;
  };
  if (p.slots <= 32u) {
    // A choice a lane, experts in the order of their first choices, one barrier (one token of 8 experts, 4096 x 2048: 73.3 us
    // with the general way, 69.2 so).
    if (warp == 0u) {
      uint32_t id = lane < p.slots ? id_of(lane) : kNoExpert;
      if (lane < p.slots) ids[lane] = static_cast<uint16_t>(id);
      const uint32_t below = (1u << lane) - 1u;
      const uint32_t first_of_token = lane - lane % p.top;
      const uint32_t repeats = __match_any_sync(0xffffffffu, id) & below & ~((1u << first_of_token) - 1u);
      if (repeats != 0u) id = kNoExpert;
      const uint32_t same = __match_any_sync(0xffffffffu, id);
      const bool first = id != kNoExpert && (same & below) == 0u;
      const uint32_t c = first ? __popc(same) : 0u;
      uint32_t incl = c | (c + NT - 1u) / NT << 16;
      const uint32_t own = incl;
#pragma unroll
      for (uint32_t d = 1; d < 32u; d <<= 1) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
      }
      const uint32_t at = incl - own;
      for (uint32_t i = 0; i * NT < c; ++i) {
        passes[(at >> 16) + i] = {static_cast<uint16_t>(id), static_cast<uint16_t>((at & 0xFFFFu) + i * NT),
                                  static_cast<uint16_t>(min(NT, c - i * NT)), 0};
      }
      const uint32_t begin = __shfl_sync(0xffffffffu, at & 0xFFFFu, __ffs(same) - 1);  // of this lane's expert
      if (id != kNoExpert) list[begin + __popc(same & below)] = static_cast<uint16_t>(lane);
      if (lane == 31u) *totals = incl >> 16;
    }
    __syncthreads();
    return *totals;
  }
  for (uint32_t s = tid; s < p.slots; s += kThreads) ids[s] = id_of(s);
  for (uint32_t i = tid; i < kSortWarps * p.experts; i += kThreads) counts[i] = 0;
  __syncthreads();
  // A choice that repeats an earlier one of its token has no place of its own. `list` notes it for now.
  for (uint32_t s = tid; s < p.slots; s += kThreads) {
    uint16_t id = ids[s];
    bool repeats = false;
    for (uint32_t i = s - s % p.top; i < s; ++i) repeats |= ids[i] == id;
    if (repeats && id != kNoExpert) id |= kRepeat;
    list[s] = id;
  }
  __syncthreads();
  const uint32_t share = ((p.slots + kSortWarps - 1u) / kSortWarps + 31u) & ~31u;
  const uint32_t begin = warp * share, end = warp < kSortWarps ? min(p.slots, begin + share) : 0u;
  uint16_t* mine = counts + (warp < kSortWarps ? warp : 0u) * p.experts;
  for (uint32_t s0 = begin; s0 < end; s0 += 32u) {
    const uint32_t s = s0 + lane, id = s < end ? list[s] : kNoExpert;
    if (s < end) ids[s] = static_cast<uint16_t>(id);
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    if ((id & kRepeat) == 0u && (same >> lane) == 1u) mine[id] = static_cast<uint16_t>(mine[id] + __popc(same));
    __syncwarp();
  }
  __syncthreads();
  if (warp == 0u) {
    // First choice and first pass of each expert; the counts become the places of the shares' next choices.
    uint32_t base = 0;  // choices in the lower half, passes in the upper
    for (uint32_t e0 = 0; e0 < p.experts; e0 += 32u) {
      const uint32_t e = e0 + lane;
      uint32_t of[kSortWarps], c = 0;
#pragma unroll
      for (uint32_t w = 0; w < kSortWarps; ++w) {
        of[w] = e < p.experts ? counts[w * p.experts + e] : 0u;
        c += of[w];
      }
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
      uint32_t place = first;
#pragma unroll
      for (uint32_t w = 0; w < kSortWarps; ++w) {
        if (e < p.experts) counts[w * p.experts + e] = static_cast<uint16_t>(place);
        place += of[w];
      }
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) *totals = base >> 16;
  }
  __syncthreads();
  for (uint32_t s0 = begin; s0 < end; s0 += 32u) {
    const uint32_t s = s0 + lane, id = s < end ? ids[s] : kNoExpert;
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    const uint32_t before = __popc(same & ((1u << lane) - 1u));
    if ((id & kRepeat) == 0u) list[mine[id] + before] = static_cast<uint16_t>(s);
    __syncwarp();
    if ((id & kRepeat) == 0u && (same >> lane) == 1u) mine[id] = static_cast<uint16_t>(mine[id] + before + 1u);
    __syncwarp();
  }
  __syncthreads();
  return *totals;
}

__device__ __forceinline__ uint32_t token_of(const Params& p, uint32_t s) {
  return p.top_inverse == 0u ? s : __umulhi(s, p.top_inverse);
}

// The weight of choice s, the first of its expert: with those of its token's later choices of the same.
__device__ __forceinline__ float share_of(const Params& p, const uint16_t* ids, uint32_t s) {
  float sum = 0.f;
  const uint32_t end = s - s % p.top + p.top, own = ids[s];
  for (uint32_t i = s; i < end; ++i) {
    if ((ids[i] & ~uint32_t(kRepeat)) == own) {
      sum += p.weights_bf16 ? bf16_bits_to_float(__ldcg(static_cast<const uint16_t*>(p.weights) + i))
                            : __ldcg(static_cast<const float*>(p.weights) + i);
    }
  }
  return sum;
}

// One warp's share of a box of weights times the J tiles of eight columns of its rows of x.
template <uint32_t MR, uint32_t WR, uint32_t XBYTES, bool INT4, uint32_t J, uint32_t N>
__device__ __forceinline__ void multiply_box(float (&acc)[MR][N][4], uint32_t w_at, uint32_t x_at,
                                             const uint32_t (&sc)[MR / 2], uint32_t wr, uint32_t lane) {
  if constexpr (!INT4) {
#pragma unroll
    for (uint32_t half = 0; half < 2; ++half) {  // 32 of the contraction
      uint32_t b[J][4];
#pragma unroll
      for (uint32_t j = 0; j < J; ++j) {
        const uint32_t row = lane & 7u, chunk = half * 4u + (lane >> 3);
        ldmatrix_x4(x_at + (j * 8u + row) * kRowBytes + ((chunk ^ row) << 4), b[j]);
      }
#pragma unroll
      for (uint32_t m = 0; m < MR; ++m) {
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k) {
          uint32_t a[4];
          const uint32_t row = (m * WR + wr) * 16u + (lane & 15u), chunk = half * 4u + k * 2u + (lane >> 4);
          ldmatrix_x4(w_at + row * kRowBytes + ((chunk ^ (row & 7u)) << 4), a);
#pragma unroll
          for (uint32_t j = 0; j < J; ++j) mma_bf16(acc[m][j], a[0], a[1], a[2], a[3], b[j][2 * k], b[j][2 * k + 1]);
        }
      }
    }
  } else {
    const uint32_t g8 = lane >> 2, q = lane & 3u;
    // A lane's codes are k = 8 q .. 8 q + 7 of 32, so it takes the same of x, 16 bytes of a row. Lanes of a quarter warp
    // take the rows r and r + 4, whose halves of 128 swizzled bytes lie in different banks; so column n of a
    // product is row perm(n).
    const uint32_t perm = (g8 >> 1) | (g8 & 1u) << 2;
    // Pairs of k: (0, 4), (1, 5), (2, 6), (3, 7) of a lane's eight, as the codes come; 32 codes of a row are 16 bytes.
    const auto load_x = [&](uint32_t c, uint32_t j, uint32_t (&b)[4]) {
      uint32_t x[4];
      lds_128(x_at + (c >> 1) * XBYTES + (j * 8u + perm) * kRowBytes + ((((c & 1u) * 4u + q) ^ perm) << 4), x);
      b[0] = mul_bf16x2(__byte_perm(x[0], x[2], 0x5410), kScaleEven);
      b[1] = mul_bf16x2(__byte_perm(x[0], x[2], 0x7632), kScaleOdd);
      b[2] = mul_bf16x2(__byte_perm(x[1], x[3], 0x5410), kScaleEven);
      b[3] = mul_bf16x2(__byte_perm(x[1], x[3], 0x7632), kScaleOdd);
    };
    // Over the group: -8 x, which the sums of (code + 8) x start from (32 tokens 200 us; sums from zero and 8 x
    // taken off each 201).
    float part_sum[MR][J][4], x_sum[J][4];
    uint32_t b[4][J][4];
#pragma unroll
    for (uint32_t j = 0; j < J; ++j) {
#pragma unroll
      for (uint32_t c = 0; c < 4; ++c) {
        load_x(c, j, b[c][j]);
        if (c == 0) {
          mma_bf16_first(x_sum[j], kEightEven, kEightEven, kEightOdd, kEightOdd, b[c][j][0], b[c][j][1]);
        } else {
          mma_bf16(x_sum[j], kEightEven, kEightEven, kEightOdd, kEightOdd, b[c][j][0], b[c][j][1]);
        }
        mma_bf16(x_sum[j], kEightEven, kEightEven, kEightOdd, kEightOdd, b[c][j][2], b[c][j][3]);
      }
    }
#pragma unroll
    for (uint32_t c = 0; c < 4; ++c) {
#pragma unroll
      for (uint32_t m2 = 0; m2 < MR; m2 += 2) {
        uint32_t a[4];  // rows 0-7 and 8-15 of two blocks of rows
        const uint32_t row = ((m2 + (lane >> 4)) * WR + wr) * 16u + (lane & 15u);
        ldmatrix_x4(w_at + row * 64u + ((c ^ ((row >> 1) & 3u)) << 4), a);
#pragma unroll
        for (uint32_t m = 0; m < 2; ++m) {
          uint32_t lo[4], hi[4];
          codes_to_bf16(a[2 * m], lo);
          codes_to_bf16(a[2 * m + 1], hi);
#pragma unroll
          for (uint32_t j = 0; j < J; ++j) {
            if (c == 0) {
              mma_bf16_from(part_sum[m2 + m][j], x_sum[j], lo[0], hi[0], lo[1], hi[1], b[c][j][0], b[c][j][1]);
            } else {
              mma_bf16(part_sum[m2 + m][j], lo[0], hi[0], lo[1], hi[1], b[c][j][0], b[c][j][1]);
            }
            mma_bf16(part_sum[m2 + m][j], lo[2], hi[2], lo[3], hi[3], b[c][j][2], b[c][j][3]);
          }
        }
      }
    }
#pragma unroll
    for (uint32_t m = 0; m < MR; ++m) {
      const float s0 = __uint_as_float(__shfl_sync(0xffffffffu, sc[m / 2], (m & 1u) * 16u + g8));
      const float s1 = __uint_as_float(__shfl_sync(0xffffffffu, sc[m / 2], (m & 1u) * 16u + 8u + g8));
#pragma unroll
      for (uint32_t j = 0; j < J; ++j) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          acc[m][j][i] = fmaf(i < 2 ? s0 : s1, part_sum[m][j][i], acc[m][j][i]);
        }
      }
    }
  }
}

// The rows of x in the order of the sorted choices, for batches whose experts have many: xs [choices][ldxs]. (Plain loads:
// the launch in front may write x while this one's blocks are there already, so it is not read-only to them.)
template <uint32_t NT>
__global__ void __launch_bounds__(kThreads) expert_rows_kernel(const __grid_constant__ Params p, uint16_t* xs, uint64_t ldxs,
                                                               const uint16_t* x, uint64_t ldx, uint32_t inner) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ uint32_t num_passes;
  const Layout l = layout_of(0, 1, 0, NT, p.tokens, p.slots, p.experts, false, true);
  Pass* passes = reinterpret_cast<Pass*>(smem_raw + l.passes);
  uint16_t* list = reinterpret_cast<uint16_t*>(smem_raw + l.list);
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t n = sort_choices<NT>(p, passes, list, reinterpret_cast<uint16_t*>(smem_raw + l.ids),
                                      reinterpret_cast<uint16_t*>(smem_raw + l.total), &num_passes);
  const uint32_t listed = n == 0u ? 0u : passes[n - 1u].first + passes[n - 1u].count;
  for (uint32_t i = blockIdx.x; i < listed; i += gridDim.x) {
    const uint16_t* from = x + token_of(p, list[i]) * ldx;
    uint16_t* to = xs + i * ldxs;
    for (uint32_t v = threadIdx.x; v < inner / 8u; v += kThreads) {
      reinterpret_cast<uint4*>(to)[v] = reinterpret_cast<const uint4*>(from)[v];
    }
    for (uint32_t k = inner / 8u * 8u + threadIdx.x; k < inner; k += kThreads) to[k] = from[k];
  }
}

template <uint32_t NT, uint32_t MR, uint32_t WR, bool INT4, bool SECOND>
__global__ void __launch_bounds__(kThreads, 2) expert_layer_kernel(const __grid_constant__ Params p) {
  using C = Cfg<NT, MR, WR, INT4>;
  constexpr uint32_t WK = C::kParts;
  constexpr uint32_t kTiles8 = NT / 8;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages];
  __shared__ uint32_t abort_flag, num_passes;
  uint8_t* ring = smem_raw + smem_align_pad(smem_raw);
  uint8_t* rest = ring + p.stages * C::kStageBytes;
  const Layout l =
      layout_of(C::kSumBytes, WK, C::kRows, NT, p.tokens, p.slots, p.experts, SECOND, SECOND && p.own_y != 0u);
  float* sums = reinterpret_cast<float*>(rest + l.sums);  // [WK][kTiles8][kRows][8]
  float* y = reinterpret_cast<float*>(rest + l.y);        // SECOND: [own_y ? WK : 1][tokens][kRows]
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
  // A launch of this layer in front of this one has waited for the choices and their weights before it let
  // this one in: they and the layer's weights can be read at once, its results (`tm_x`'s) after the wait.
  const bool early = SECOND || p.sorted != 0u;
  if (!early) {
    pdl_wait();
    pdl_launch_dependents();
  }
  const uint32_t passes_n = sort_choices<NT>(p, passes, list, ids, reinterpret_cast<uint16_t*>(ring), &num_passes);
  const uint32_t y_size = p.tokens * C::kRows;
  if (SECOND) {
    for (uint32_t i = threadIdx.x; i < y_size * (p.own_y ? WK : 1u); i += kThreads) y[i] = 0.f;
    const uint32_t listed = passes_n == 0u ? 0u : passes[passes_n - 1u].first + passes[passes_n - 1u].count;
    for (uint32_t i = threadIdx.x; i < listed; i += kThreads) share[i] = share_of(p, ids, list[i]);
  }
  // The ring held scratch of the sorting: order its writes before the loads.
  fence_proxy_async_smem();
  __syncthreads();

  // This block's walk: items of (pass, column tile), each a run of boxes along the contraction. FIRST: tiles of a
  // pass side by side over the blocks, whole items. SECOND: one tile, all passes; the blocks of a cluster share
  // the passes' boxes evenly, so an item may be cut at either end.
  const uint32_t rank = SECOND && p.splits > 1u ? cluster_ctarank() : 0u;
  const uint32_t nkb = p.num_kb;
  const uint32_t tile_cols = p.gated ? C::kRows / 2u : C::kRows;
  const uint32_t my_tile = SECOND ? blockIdx.x / p.splits : 0u;
  const uint32_t item_step = SECOND ? 1u : gridDim.x;
  uint32_t item0, kb_first, boxes;
  if (SECOND) {
    const uint32_t all = passes_n * nkb;
    const uint32_t from = static_cast<uint32_t>(uint64_t(all) * rank / p.splits);
    boxes = static_cast<uint32_t>(uint64_t(all) * (rank + 1u) / p.splits) - from;
    item0 = from / nkb;
    kb_first = from - item0 * nkb;
  } else {
    const uint32_t items = passes_n * p.tiles;
    item0 = blockIdx.x;
    kb_first = 0;
    boxes = item0 < items ? (items - item0 + item_step - 1u) / item_step * nkb : 0u;
  }

  if (warp == kConsumers) {
    // ------------------------------------------------------------ producer
    // kBatch boxes at a time, lane i for the weights of the i-th: their waits, and the issue of their loads,
    // run side by side (box by box a block fetched 4 KB per 780 cycles, whatever was in flight).
    constexpr uint32_t kBatch = C::kBatch;
    uint32_t item = item0, kb = kb_first + lane;  // of this lane's box
    Pass ps = {0, 0, 1, 0};
    uint32_t f0 = 0;
    const auto locate = [&]() {
      while (kb >= nkb) {
        kb -= nkb;
        item += item_step;
      }
      const uint32_t pi = SECOND ? item : item / p.tiles;
      ps = passes[pi];
      f0 = (SECOND ? my_tile : item - pi * p.tiles) * tile_cols;
    };
    const auto load_weights = [&](uint32_t st) {
      const uint32_t rows = early ? (ps.count + 7u) & ~7u : (ps.count + 3u) & ~3u;
      mbar_arrive_expect_tx(&full[st], C::kWBytes + C::kSub * rows * kRowBytes);
      tma_load_4d(&p.tm_w, &full[st], ring + st * C::kStageBytes, int32_t(kb * 64u),
                  int32_t(f0), 0, ps.expert, kCacheEvictNormal);
    };
    uint32_t ahead = 0;  // boxes whose weights are on their way
    if (early) {
      // The first weights do not wait for the launch in front.
      ahead = min(p.stages, boxes);
      if (lane < kBatch) {
        for (uint32_t b = lane; b < ahead; b += kBatch) {
          locate();
          load_weights(b);
          kb += kBatch;
        }
      }
      item = item0, kb = kb_first + lane;
      __syncwarp();
      pdl_wait();
      pdl_launch_dependents();
    }
    uint32_t stage = lane % kBatch, phase = 0, issued = 0;  // of this lane's box; boxes it has loaded
    for (uint32_t b0 = 0; b0 < boxes; b0 += kBatch) {
      const bool mine = lane < kBatch && b0 + lane < boxes;
      bool go = mine;
      if (mine) {
        locate();
        if (b0 + lane >= ahead) {
          go = mbar_wait(&empty[stage], phase ^ 1u, abort, kStatusTimeoutProducer);
          if (go) load_weights(stage);
        }
      }
      const uint32_t going = __ballot_sync(0xffffffffu, go);
      // Rows of all boxes that go: eight a load where they lie in the order of `list`, else four a gather.
      constexpr uint32_t kQuads = NT / 4u, kPerBox = kQuads * C::kSub;
#pragma unroll
      for (uint32_t g0 = 0; g0 < kBatch * kPerBox; g0 += 32u) {
        const uint32_t g = g0 + lane, box = g / kPerBox, sub = g % kPerBox / kQuads, quad = g % kQuads;
        const uint32_t from = box < kBatch ? box : 0u;
        const uint32_t first = __shfl_sync(0xffffffffu, uint32_t(ps.first), from);
        const uint32_t count = __shfl_sync(0xffffffffu, uint32_t(ps.count), from);
        const uint32_t k = __shfl_sync(0xffffffffu, kb, from);
        const uint32_t st = __shfl_sync(0xffffffffu, stage, from);
        if (box < kBatch && ((going >> box) & 1u) != 0u && quad * 4u < count) {
          uint8_t* to = ring + st * C::kStageBytes + C::kWBytes + sub * C::kXBytes + quad * 4u * kRowBytes;
          const int32_t x = int32_t((k * C::kSub + sub) * 64u);
          if (early) {
            if ((quad & 1u) == 0u) tma_load_2d(&p.tm_x, &full[st], to, x, int32_t(first + quad * 4u), kCacheEvictLast);
          } else {
            int32_t r[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
              const uint32_t c = quad * 4u + i;
              r[i] = int32_t(c < count ? token_of(p, list[first + c]) : p.tokens);
            }
            tma_gather4(&p.tm_x, &full[st], to, x, r[0], r[1], r[2], r[3], kCacheEvictLast);
          }
        }
      }
      if (go) {
        ++issued;
        kb += kBatch;
        stage += kBatch;
        if (stage >= p.stages) {
          stage -= p.stages;
          phase ^= 1u;
        }
      }
      if (__any_sync(0xffffffffu, mine && !go)) break;
    }
    // Copies in flight land before the block may exit.
    if (lane < kBatch) {
      const uint32_t per_lane = p.stages / kBatch;
      for (uint32_t i = issued - min(issued, per_lane); i < issued; ++i) {
        const uint32_t b = i * kBatch + lane;
        mbar_drain(&full[b % p.stages], (b / p.stages) & 1u);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ consumers
    if (early) pdl_wait();
    const uint32_t wr = warp % WR, part = warp / WR;
    const uint32_t g8 = lane >> 2, q = lane & 3u;
    uint32_t stage = part, phase = 0;             // of this part's next box
    uint32_t box = part;                          // its running number
    uint32_t item = item0, kb = kb_first + part;  // and where it lies
    bool ok = true;

    const auto locate = [&](uint32_t& of_item, uint32_t& of_kb) {
      while (of_kb >= nkb) {
        of_kb -= nkb;
        of_item += item_step;
      }
    };
    // int4: the scales of a box, one a weight row, on their way two boxes ahead. Lane l has row l (and l + 32) of
    // this warp's rows (behind the last column: that one's again). Where an item's rows have theirs is computed once an item (for
    // every box 32 tokens took 201 us, so 191). Scales have fewer than 2^32 elements: their codes are 64 times as many bytes.
    // (Plain loads, as of x in expert_rows_kernel.)
    constexpr uint32_t kScaleRegs = MR / 2;
    uint32_t scales[2][kScaleRegs], scale_at[kScaleRegs];
    uint32_t scale_box = part, scale_item = item0, scale_kb = kb_first + part;
    const auto locate_scales = [&]() {
      const uint32_t pi = SECOND ? scale_item : scale_item / p.tiles;
      const uint32_t f0 = (SECOND ? my_tile : scale_item - pi * p.tiles) * tile_cols;
      const uint32_t rows0 = passes[pi].expert * (p.gated ? 2u * p.cols : p.cols);
#pragma unroll
      for (uint32_t i = 0; i < kScaleRegs; ++i) {
        const uint32_t m = i * 2u + (lane >> 4);
        const bool up = p.gated && m >= MR / 2;
        const uint32_t f = min(f0 + ((up ? m - MR / 2 : m) * WR + wr) * 16u + (lane & 15u), p.cols - 1u);
        scale_at[i] = (rows0 + f + (up ? p.cols : 0u)) * p.groups;
      }
    };
    const auto fetch_scales = [&](uint32_t (&to)[kScaleRegs]) {
      if constexpr (INT4) {
        if (scale_box >= boxes) return;
        if (scale_kb >= nkb) {
          locate(scale_item, scale_kb);
          locate_scales();
        }
#pragma unroll
        for (uint32_t i = 0; i < kScaleRegs; ++i) to[i] = p.sb[scale_at[i] + scale_kb];
        scale_box += WK;
        scale_kb += WK;
      }
    };
    if (INT4 && box < boxes) {
      locate(scale_item, scale_kb);
      locate_scales();
    }
    fetch_scales(scales[0]);
    fetch_scales(scales[1]);
    if (box < boxes) locate(item, kb);

    const uint32_t last = boxes == 0u ? 0u : kb_first + boxes;  // boxes from the first item's start to this block's last one
    for (uint32_t at = item0, before = 0; before < last; at += item_step, before += nkb) {
      const uint32_t pi = SECOND ? at : at / p.tiles;
      const Pass ps = passes[pi];
      const uint32_t f0 = (SECOND ? my_tile : at - pi * p.tiles) * tile_cols;
      float acc[MR][kTiles8][4];
#pragma unroll
      for (uint32_t m = 0; m < MR; ++m) {
#pragma unroll
        for (uint32_t j = 0; j < kTiles8; ++j) {
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
        }
      }
      bool any = false;
      while (box < boxes && item == at) {
        any = true;
        uint32_t sc[kScaleRegs];
#pragma unroll
        for (uint32_t i = 0; i < kScaleRegs; ++i) {
          sc[i] = scales[0][i] << 16;  // bf16 as fp32
          scales[0][i] = scales[1][i];
        }
        fetch_scales(scales[1]);
        box += WK;
        kb += WK;
        if (box < boxes) locate(item, kb);
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, abort, kStatusTimeoutMma));
        const uint32_t w_at = smem_u32(ring + stage * C::kStageBytes), x_at = w_at + C::kWBytes;
        if (ok) {
          // As many tiles of eight columns as the pass has (in steps of two above two).
          if (NT == 8 || ps.count <= 8u) {
            multiply_box<MR, WR, C::kXBytes, INT4, (1 < kTiles8 ? 1 : kTiles8)>(acc, w_at, x_at, sc, wr, lane);
          } else if (NT == 16 || ps.count <= 16u) {
            multiply_box<MR, WR, C::kXBytes, INT4, (2 < kTiles8 ? 2 : kTiles8)>(acc, w_at, x_at, sc, wr, lane);
          } else {
            multiply_box<MR, WR, C::kXBytes, INT4, (4 < kTiles8 ? 4 : kTiles8)>(acc, w_at, x_at, sc, wr, lane);
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

      // Columns of a product that this lane holds.
      const uint32_t col[2] = {INT4 ? q : 2u * q, INT4 ? q + 4u : 2u * q + 1u};
      if constexpr (INT4) {
#pragma unroll
        for (uint32_t m = 0; m < MR; ++m) {
#pragma unroll
          for (uint32_t j = 0; j < kTiles8; ++j) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) acc[m][j][i] *= kCodeUnit;
          }
        }
      }
      if (SECOND && p.own_y) {
        // Into this part's own sums of y: a pass holds a token once, so no two lanes meet.
        if (any) {
#pragma unroll
          for (uint32_t j = 0; j < kTiles8; ++j) {
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
              const uint32_t c = j * 8u + col[i];
              if (c < ps.count) {
                const float w = share[ps.first + c];
                float* to = y + part * y_size + token_of(p, list[ps.first + c]) * C::kRows + wr * 16u + g8;
#pragma unroll
                for (uint32_t m = 0; m < MR; ++m) {
                  to[m * WR * 16u] = fmaf(w, acc[m][j][i], to[m * WR * 16u]);
                  to[m * WR * 16u + 8u] = fmaf(w, acc[m][j][2 + i], to[m * WR * 16u + 8u]);
                }
              }
            }
          }
        }
        __syncwarp();  // another lane may hold the token in the next pass
        continue;
      }
      // The parts' sums meet in shared memory.
      named_barrier_sync(1, kConsumers * 32);  // the last item's have been read
#pragma unroll
      for (uint32_t j = 0; j < kTiles8; ++j) {
        if (j * 8u < ps.count) {
#pragma unroll
          for (uint32_t m = 0; m < MR; ++m) {
            float* to = sums + ((part * kTiles8 + j) * C::kRows + (m * WR + wr) * 16u + g8) * 8u;
            if constexpr (INT4) {
              to[q] = acc[m][j][0];
              to[q + 4] = acc[m][j][1];
              to[64 + q] = acc[m][j][2];
              to[64 + q + 4] = acc[m][j][3];
            } else {
              *reinterpret_cast<float2*>(to + 2 * q) = make_float2(acc[m][j][0], acc[m][j][1]);
              *reinterpret_cast<float2*>(to + 64 + 2 * q) = make_float2(acc[m][j][2], acc[m][j][3]);
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
        if (SECOND) {
          float* to = y + token_of(p, list[ps.first + c]) * C::kRows + f;
          *to = fmaf(share[ps.first + c], total(f, c), *to);
        } else {
          float v[2] = {total(f, c), 0.f};
          lin::activate(v, p.act);
          if (p.gated) v[0] *= total(C::kRows / 2u + f, c);
          p.out[size_t(ps.first + c) * p.ldo + f0 + f] = __bfloat16_as_ushort(__float2bfloat16_rn(v[0]));
        }
      }
    }
    if (SECOND) named_barrier_sync(1, kConsumers * 32);  // all experts are in y
  }

  if (SECOND) {
    const uint32_t f0 = my_tile * C::kRows, cols = min(C::kRows, p.cols - f0);
    const auto part_total = [&](uint32_t o) {
      float v = y[o];
      if (p.own_y) {
        for (uint32_t k = 1; k < WK; ++k) v += y[k * y_size + o];
      }
      return v;
    };
    if (p.splits > 1u) {
      __syncthreads();
      if (p.own_y) {
        for (uint32_t o = threadIdx.x; o < y_size; o += kThreads) y[o] = part_total(o);
      }
      cluster_sync_all();
      // Block r of the cluster finishes the tokens r, r + S, ...
      for (uint32_t o = threadIdx.x; o < y_size; o += kThreads) {
        const uint32_t f = o % C::kRows, t = o / C::kRows;
        if (t % p.splits != rank || f >= cols) continue;
        float v = 0.f;
        for (uint32_t i = 0; i < p.splits; ++i) v += ld_dsmem_f32(map_to_rank(y + o, i));
        p.out[size_t(t) * p.ldo + f0 + f] = __bfloat16_as_ushort(__float2bfloat16_rn(v));
      }
      cluster_sync_all();
    } else if (warp < kConsumers) {
      for (uint32_t o = threadIdx.x; o < y_size; o += kConsumers * 32u) {
        const uint32_t f = o % C::kRows, t = o / C::kRows;
        if (f < cols) p.out[size_t(t) * p.ldo + f0 + f] = __bfloat16_as_ushort(__float2bfloat16_rn(part_total(o)));
      }
    }
  }
}

}  // namespace experts
}  // namespace arcb
