// linear_common.cuh — what the linear and grouped product kernels share: the row groups, the
// epilogue's activation functions and the 16-bit row vectors of 32 columns.
#pragma once

#include "sm100.cuh"

namespace arcb {
namespace lin {

constexpr uint32_t BK = 64;  // contraction elements per block: one 128-byte swizzle row
constexpr uint32_t kUmmaK = 16;
constexpr uint32_t kMaxGroups = 1024;

// ---------------------------------------------------------------------------------
// Row groups: group e owns rows [offsets[e], offsets[e+1]) of a [rows] x ... matrix. The
// offsets live on the GPU, so the host knows only `rows`; every bound is clamped to it when
// it is read, which keeps all accesses in range whatever the offsets hold. A null `offsets`
// is one group of all rows.
// ---------------------------------------------------------------------------------
struct Groups {
  const int32_t* offsets;  // [num + 1] or null
  uint32_t num, rows;
};

__device__ __forceinline__ uint32_t group_bound(const Groups& g, uint32_t e) {
  if (g.offsets == nullptr) return e == 0u ? 0u : g.rows;
  const int32_t v = __ldg(g.offsets + e);
  return v < 0 ? 0u : min(static_cast<uint32_t>(v), g.rows);
}

__device__ __forceinline__ uint32_t group_begin(const Groups& g, uint32_t e) { return group_bound(g, e); }
__device__ __forceinline__ uint32_t group_count(const Groups& g, uint32_t e) {
  const uint32_t a = group_bound(g, e), b = group_bound(g, e + 1u);
  return b > a ? b - a : 0u;
}

// Offsets that decrease or leave [0, rows] set the status bit that arc_device_status reports.
__device__ __forceinline__ void group_check(const Groups& g, uint32_t e) {
  const int32_t a = __ldg(g.offsets + e), b = __ldg(g.offsets + e + 1u);
  if (a < 0 || b < a || static_cast<uint32_t>(b) > g.rows) atomicOr(&g_arc_status, kStatusBadOffsets);
}

// One warp: prefix[e] = tiles of the groups before e (each group has ceil(count / tile)
// row tiles), prefix[num] = all of them. Checks the offsets.
__device__ __forceinline__ void group_tiles_prefix(const Groups& g, uint32_t tile, uint32_t* prefix) {
  const uint32_t lane = threadIdx.x & 31u;
  uint32_t base = 0;
  for (uint32_t e0 = 0; e0 < g.num; e0 += 32u) {
    const uint32_t e = e0 + lane;
    uint32_t c = 0;
    if (e < g.num) {
      if (g.offsets != nullptr) group_check(g, e);
      c = (group_count(g, e) + tile - 1u) / tile;
    }
    uint32_t incl = c;
#pragma unroll
    for (uint32_t d = 1; d < 32u; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += o;
    }
    if (e < g.num) prefix[e] = base + incl - c;
    base += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) prefix[g.num] = base;
}

// The group that row tile t belongs to: the last e with prefix[e] <= t (t < prefix[num]), so
// that groups without rows, whose prefix equals their successor's, are passed over.
__device__ __forceinline__ uint32_t group_of_tile(const uint32_t* prefix, uint32_t num, uint32_t t) {
  uint32_t lo = 0, hi = num;
  while (hi - lo > 1u) {
    const uint32_t mid = (lo + hi) >> 1;
    if (prefix[mid] <= t) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  return lo;
}

// Zero the output rows that belong to no group (before the first and behind the last),
// striped over the blocks of the grid; every thread of the block takes part.
__device__ __forceinline__ void zero_other_rows(const Groups& g, uint16_t* out, size_t ldo, uint32_t cols,
                                                uint32_t block, uint32_t num_blocks) {
  const uint32_t first = group_bound(g, 0), last = group_bound(g, g.num);
  const uint32_t behind = last < g.rows ? g.rows - last : 0u;
  const bool wide = ((reinterpret_cast<uintptr_t>(out) | (ldo * 2)) & 15u) == 0u;
  for (uint32_t i = block; i < first + behind; i += num_blocks) {
    uint16_t* row = out + size_t(i < first ? i : last + (i - first)) * ldo;
    const uint32_t vecs = wide ? cols / 8u : 0u;
    for (uint32_t c = threadIdx.x; c < vecs; c += blockDim.x) {
      reinterpret_cast<uint4*>(row)[c] = make_uint4(0u, 0u, 0u, 0u);
    }
    for (uint32_t c = vecs * 8u + threadIdx.x; c < cols; c += blockDim.x) row[c] = 0;
  }
}

// ---------------------------------------------------------------------------------
// Activations (fp32). gelu is the erf form, gelu_tanh the tanh form.
// ---------------------------------------------------------------------------------
enum Act : uint32_t { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };

constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kSqrt2OverPi = 0.79788456080286536f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kGeluCubic = 0.044715f;

constexpr float kLog2E = 1.4426950408889634f;

// 1 / (1 + e^-z); e^-z overflows to infinity, whose reciprocal is the right 0.
__device__ __forceinline__ float sigmoidf(float z) { return rcp_ftz(1.f + ex2_ftz(-kLog2E * z)); }

// The tanh form's argument. 1 + tanh(u) = 2 sigmoid(2u), which keeps its relative accuracy
// in the lower tail, where 1 + tanh(u) would cancel.
__device__ __forceinline__ float gelu_tanh_arg(float z) {
  return 2.f * kSqrt2OverPi * (z + kGeluCubic * z * z * z);
}

// q(y) = 1 - erf(y / sqrt 2) = t R(t) exp(-y^2 / 2), t = 1 / (1 + p y): the form of formula 7.1.26 of
// Abramowitz and Stegun (Handbook of Mathematical Functions) with seven terms, fitted here for the
// least relative error (minimax by linear programming on 0 <= y <= 13.5, where q leaves fp32: 6e-7,
// and 9e-6 in fp32, through the exponential's argument). q's own accuracy is what the lower tail of
// the activation needs: with a formula of an absolute bound (7.1.28, 3e-7) gelu(-5) was off by 5 %.
constexpr float kTailP = 0.265f;
__device__ __forceinline__ constexpr float tail_term(int i) {
  constexpr float c[7] = {0.21120048617f, 0.21566298207f, 0.16594652836f, 0.28485278664f,
                          -0.13254834990f, 0.39042731883f, -0.13554236419f};
  return c[i];
}

// t R(t) of two values, with one reciprocal for both and packed products.
__device__ __forceinline__ uint64_t gelu_tail_pair(uint64_t y) {
  const auto both = [](float c) { return f32x2_pack(c, c); };
  float d0, d1;
  f32x2_unpack(f32x2_fma(y, both(kTailP), both(1.f)), d0, d1);
  const float r = rcp_ftz(d0 * d1);
  const uint64_t t = f32x2_pack(r * d1, r * d0);
  uint64_t q = f32x2_fma(t, both(tail_term(6)), both(tail_term(5)));
#pragma unroll
  for (int i = 4; i >= 0; --i) q = f32x2_fma(t, q, both(tail_term(i)));
  return f32x2_mul(t, q);
}

// exp(-y^2 / 2) of two values.
__device__ __forceinline__ uint64_t gauss_pair(uint64_t y) {
  float e0, e1;
  f32x2_unpack(f32x2_mul(f32x2_mul(y, f32x2_pack(-0.5f * kLog2E, -0.5f * kLog2E)), y), e0, e1);
  return f32x2_pack(ex2_ftz(e0), ex2_ftz(e1));
}

// The erf form, two values at once: z Phi(z) = max(z, 0) - |z| q(|z|) / 2, where nothing cancels.
// |z| stops at 16, where q is 0 in fp32.
__device__ __forceinline__ void gelu_pair(float& z0, float& z1) {
  const uint64_t y = f32x2_pack(fminf(fabsf(z0), 16.f), fminf(fabsf(z1), 16.f));
  const uint64_t h = f32x2_mul(f32x2_mul(gelu_tail_pair(y), y), gauss_pair(y));
  f32x2_unpack(f32x2_fma(h, f32x2_pack(-0.5f, -0.5f), f32x2_pack(relu_nan(z0), relu_nan(z1))), z0, z1);
}

// Its slope Phi(z) + z phi(z), two values at once (in their place): with e = exp(-z^2 / 2) and
// h = t R(t) / 2 it is e (h + z / sqrt(2 pi)) below zero and 1 - e (h - z / sqrt(2 pi)) above.
__device__ __forceinline__ void gelu_slope_pair(float& z0, float& z1) {
  const uint64_t y = f32x2_pack(fminf(fabsf(z0), 16.f), fminf(fabsf(z1), 16.f));
  const uint64_t e = gauss_pair(f32x2_pack(z0, z1));  // not y: a NaN stays one
  // |slope - (z > 0)| = e (h - |z| / sqrt(2 pi))
  const uint64_t d = f32x2_mul(e, f32x2_fma(gelu_tail_pair(y), f32x2_pack(0.5f, 0.5f),
                                            f32x2_mul(y, f32x2_pack(-kInvSqrt2Pi, -kInvSqrt2Pi))));
  float d0, d1;
  f32x2_unpack(d, d0, d1);
  z0 = z0 < 0.f ? d0 : 1.f - d0;
  z1 = z1 < 0.f ? d1 : 1.f - d1;
}

// The others, one value.
__device__ __forceinline__ float act_value(float z, uint32_t act) {
  switch (act) {
    case kActRelu:
      return relu_nan(z);
    case kActGeluTanh:
      return z * sigmoidf(gelu_tanh_arg(z));
    case kActSilu:
      return z * sigmoidf(z);
    default:
      return z;
  }
}

// d act / d z.
__device__ __forceinline__ float act_slope(float z, uint32_t act) {
  switch (act) {
    case kActRelu:
      return z > 0.f ? 1.f : 0.f;
    case kActGeluTanh: {
      const float s = sigmoidf(gelu_tanh_arg(z));
      // z^2 stops where s (1 - s) has long been 0: infinity times that 0 would be NaN.
      return s + z * s * (1.f - s) * (2.f * kSqrt2OverPi) * (1.f + 3.f * kGeluCubic * fminf(z * z, 1e8f));
    }
    case kActSilu: {
      const float s = sigmoidf(z);
      return s * (1.f + z * (1.f - s));
    }
    default:
      return 1.f;
  }
}

// The activation of N values, one branch for all.
template <uint32_t N>
__device__ __forceinline__ void activate(float (&v)[N], uint32_t act) {
  switch (act) {
#define ARC_ACT_CASE(A)                                                             \
  case A:                                                                           \
    _Pragma("unroll") for (uint32_t i = 0; i < N; ++i) v[i] = act_value(v[i], A);    \
    break;
    case kActGelu:
#pragma unroll
      for (uint32_t i = 0; i < N; i += 2) gelu_pair(v[i], v[i + 1]);
      break;
    ARC_ACT_CASE(kActRelu)
    ARC_ACT_CASE(kActGeluTanh)
    ARC_ACT_CASE(kActSilu)
#undef ARC_ACT_CASE
    default:
      break;
  }
}

// ---------------------------------------------------------------------------------
// Row-major access from the transposed side: a lane holds one column (lane l of the warp column
// f = f0 + l) of N consecutive rows, of which `rows` exist. With `paired` (whole column pairs,
// 4-byte aligned rows) neighbouring lanes exchange values, so that each moves two columns of
// every second row. All lanes of the warp take part; `valid` says whether this lane's column
// exists.
// ---------------------------------------------------------------------------------
template <uint32_t N>
__device__ __forceinline__ void store_columns(uint16_t* p, uint64_t ld, const float (&v)[N], uint32_t rows, bool valid,
                                              uint32_t paired) {
  if (paired) {
    const uint32_t odd = threadIdx.x & 1u;
    uint16_t* p2 = p - odd + odd * ld;
#pragma unroll
    for (uint32_t j = 0; j < N; j += 2) {
      const float got = __shfl_xor_sync(0xffffffffu, odd ? v[j] : v[j + 1], 1);
      if (valid && j + odd < rows) {
        *reinterpret_cast<uint32_t*>(p2 + size_t(j) * ld) = odd ? pack_bf16x2(got, v[j + 1]) : pack_bf16x2(v[j], got);
      }
    }
  } else {
#pragma unroll
    for (uint32_t j = 0; j < N; ++j) {
      if (valid && j < rows) p[size_t(j) * ld] = __bfloat16_as_ushort(__float2bfloat16_rn(v[j]));
    }
  }
}

// The raw words of a paired load, for load_columns_finish (so that other work can come between).
template <uint32_t N>
__device__ __forceinline__ void load_columns_start(const uint16_t* p, uint64_t ld, uint32_t (&raw)[N], uint32_t rows,
                                                   bool valid, uint32_t paired) {
  const uint32_t odd = threadIdx.x & 1u;
  const uint16_t* p2 = p - odd + odd * ld;
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) {
    raw[j] = 0u;
    if (paired) {
      if ((j & 1u) == 0u && valid && j + odd < rows) raw[j] = *reinterpret_cast<const uint32_t*>(p2 + size_t(j) * ld);
    } else if (valid && j < rows) {
      raw[j] = p[size_t(j) * ld];
    }
  }
}

template <uint32_t N>
__device__ __forceinline__ void load_columns_finish(const uint32_t (&raw)[N], float (&v)[N], uint32_t paired) {
  const uint32_t odd = threadIdx.x & 1u;
#pragma unroll
  for (uint32_t j = 0; j < N; j += 2) {
    if (paired) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, raw[j], 1);
      const uint32_t even_row = odd ? other : raw[j], odd_row = odd ? raw[j] : other;
      v[j] = odd ? __uint_as_float(even_row & 0xFFFF0000u) : __uint_as_float(even_row << 16);
      v[j + 1] = odd ? __uint_as_float(odd_row & 0xFFFF0000u) : __uint_as_float(odd_row << 16);
    } else {
      v[j] = __uint_as_float(raw[j] << 16);
      v[j + 1] = __uint_as_float(raw[j + 1] << 16);
    }
  }
}

// 32 consecutive bf16 values, the same for all lanes, of which `cols` exist; `wide`: 16-byte aligned.
__device__ __forceinline__ void load_row32(const uint16_t* p, uint32_t (&v)[16], uint32_t cols, uint32_t wide) {
  if (wide != 0u && cols >= 32u) {
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const uint4 x = reinterpret_cast<const uint4*>(p)[j];
      v[4 * j] = x.x;
      v[4 * j + 1] = x.y;
      v[4 * j + 2] = x.z;
      v[4 * j + 3] = x.w;
    }
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 16; ++j) v[j] = 0u;
#pragma unroll
    for (uint32_t j = 0; j < 32; ++j) {
      if (j < cols) v[j >> 1] |= static_cast<uint32_t>(p[j]) << ((j & 1u) * 16u);
    }
  }
}

// ---------------------------------------------------------------------------------
// A warp's 32 x 32 bf16 tile in shared memory (2 KB, 64-byte rows in the 64-byte swizzle of a
// TMA box {32, 32}): lane = row on the side of the registers; on the side of memory TMA moves
// it whole, or the warp row by row where the matrix has no 16-byte aligned rows. Straight from
// registers every lane would touch a line of its own, and the load-store unit would take longer
// than a short contraction's products.
// ---------------------------------------------------------------------------------
constexpr uint32_t kWarpTileBytes = 32 * 64;

__device__ __forceinline__ uint8_t* warp_tile_piece(uint8_t* tile, uint32_t row, uint32_t j) {
  return tile + row * 64u + ((j ^ ((row >> 1) & 3u)) << 4);
}

__device__ __forceinline__ void warp_tile_put(uint8_t* tile, const uint32_t (&v)[16]) {
  const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    *reinterpret_cast<uint4*>(warp_tile_piece(tile, lane, j)) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  }
}

__device__ __forceinline__ void warp_tile_get(const uint8_t* tile, uint32_t (&v)[16]) {
  const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    const uint4 x = *reinterpret_cast<const uint4*>(warp_tile_piece(const_cast<uint8_t*>(tile), lane, j));
    v[4 * j] = x.x;
    v[4 * j + 1] = x.y;
    v[4 * j + 2] = x.z;
    v[4 * j + 3] = x.w;
  }
}

// Row by row, a lane per column; `rows` and `cols` of the tile lie in the matrix.
__device__ __forceinline__ void warp_tile_to_rows(const uint8_t* tile, uint16_t* p, uint64_t ld, uint32_t rows,
                                                  uint32_t cols) {
  const uint32_t lane = threadIdx.x & 31u;
#pragma unroll 8
  for (uint32_t r = 0; r < 32u; ++r) {
    const uint8_t* at = warp_tile_piece(const_cast<uint8_t*>(tile), r, lane >> 3) + (lane & 7u) * 2u;
    if (r < rows && lane < cols) p[size_t(r) * ld + lane] = *reinterpret_cast<const uint16_t*>(at);
  }
}

__device__ __forceinline__ void warp_tile_from_rows(uint8_t* tile, const uint16_t* p, uint64_t ld, uint32_t rows,
                                                    uint32_t cols) {
  const uint32_t lane = threadIdx.x & 31u;
#pragma unroll 8
  for (uint32_t r = 0; r < 32u; ++r) {
    const uint16_t v = r < rows && lane < cols ? p[size_t(r) * ld + lane] : uint16_t(0);
    *reinterpret_cast<uint16_t*>(warp_tile_piece(tile, r, lane >> 3) + (lane & 7u) * 2u) = v;
  }
}

// What follows the product: bias, the activation and the residual, and where the value in
// front of the activation is kept for a backward pass.
struct Epilogue {
  const uint16_t* bias;      // [N] or null
  const uint16_t* residual;  // [M][ldr] or null
  uint16_t* z;               // [M][ldz] or null: x w^T + bias, bf16
  uint64_t ldr, ldz;
  uint32_t act;
  uint32_t wide_bias;                           // 16-byte aligned
  uint32_t pair_residual, pair_z, pair_out;     // column-wise access (store_columns)
};

// Shared-memory descriptor of an MN-major operand as a TMA load with the 128-byte swizzle
// leaves it: chunks of 64 M (or N) elements, each chunk 64 contraction rows of 128 bytes.
//   leading byte offset  between chunks (64 rows x 128 bytes = 8192)
//   stride byte offset   between groups of 8 contraction rows (1024)
// A step of 16 along the contraction is 16 rows, 2048 bytes.
constexpr uint32_t kMnChunkBytes = 64 * 128;
constexpr uint32_t kMnStepBytes = 16 * 128;
__device__ __forceinline__ uint64_t make_sw128_mnmajor_desc(const void* smem_tile) {
  const uint32_t addr = smem_u32(smem_tile);
  uint64_t desc = 0;
  desc |= static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
  desc |= static_cast<uint64_t>(kMnChunkBytes >> 4) << 16;
  desc |= static_cast<uint64_t>(1024u >> 4) << 32;
  desc |= static_cast<uint64_t>(1u) << 46;
  desc |= static_cast<uint64_t>(2u) << 61;
  return desc;
}

template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(const void* tile) {
  return MN ? make_sw128_mnmajor_desc(tile) : make_sw128_kmajor_desc(tile);
}
// Bytes from one contraction step of 16 to the next.
template <bool MN>
__host__ __device__ constexpr uint32_t operand_step() {
  return MN ? kMnStepBytes : kUmmaK * 2;
}

template <bool A_MN, bool B_MN>
__host__ __device__ constexpr uint32_t idesc_of(uint32_t m, uint32_t n) {
  return idesc_bf16_f32(m, n) | (A_MN ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u);
}

}  // namespace lin
}  // namespace arcb
