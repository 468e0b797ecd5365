// api_grouped.cuh — host side of the grouped A8W4 product and of the row grouping. Included by
// api.cu, whose helpers it uses.
#pragma once

#include "api_linear.cuh"
#include "group_rows.cuh"

namespace {

namespace GQ = arcb::a8w4;
namespace GR = arcb::rows;

// The grouped int32 kernel by token tile.
template <uint32_t BT, uint32_t EWG, uint32_t LSN, uint32_t UWG, uint32_t UNP>
struct A8w4Grouped {
  using Cfg = GQ::Cfg<BT, EWG, LSN, UWG, UNP>;
  static constexpr size_t kSmem = sizeof(GQ::GroupedSmem<BT, EWG, LSN, UWG, UNP>) + 1024;
  static_assert(kSmem <= 232448, "shared memory fits in 227 KB");
  static constexpr auto kKernel = GQ::gemm_a8w4_grouped_kernel<BT, EWG, LSN, UWG, UNP>;
};
using A8w4Grouped16 = A8w4Grouped<16, 1, 6, 2, 3>;
using A8w4Grouped32 = A8w4Grouped<32, 2, 4, 2, 3>;
using A8w4Grouped64 = A8w4Grouped<64, 2, 4, 2, 2>;
using A8w4Grouped128 = A8w4Grouped<128, 2, 3, 1, 2>;

// The register moves between warpgroups need exactly the launch count they were sized for.
template <typename V>
cudaError_t a8w4_grouped_attr(bool* regs_ok) {
  cudaError_t e = allow_smem(V::kKernel, V::kSmem);
  cudaFuncAttributes fa;
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&fa, V::kKernel);
  if (e == cudaSuccess && fa.numRegs != static_cast<int>(V::Cfg::kLaunchRegs)) *regs_ok = false;
  return e;
}

int grouped_init() {
  bool regs_ok = true;
  cudaError_t e = a8w4_grouped_attr<A8w4Grouped16>(&regs_ok);
  if (e == cudaSuccess) e = a8w4_grouped_attr<A8w4Grouped32>(&regs_ok);
  if (e == cudaSuccess) e = a8w4_grouped_attr<A8w4Grouped64>(&regs_ok);
  if (e == cudaSuccess) e = a8w4_grouped_attr<A8w4Grouped128>(&regs_ok);
  const int most = static_cast<int>(GR::smem_bytes(GR::kMaxBuckets - 1));
  for (const void* k : {reinterpret_cast<const void*>(GR::place_rows_kernel<int32_t>),
                        reinterpret_cast<const void*>(GR::place_rows_kernel<int64_t>)}) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();  // clear
    return cuda_fail(e, "cudaFuncSetAttribute (grouped A8W4 and row grouping kernels)");
  }
  if (!regs_ok) {
    return fail(ARC_ERR_UNSUPPORTED, "gemm_a8w4_grouped_kernel was compiled with an unexpected register count");
  }
  return ARC_OK;
}

// Int4 codes [groups][rows][bytes].
int encode_codes_3d(CUtensorMap* map, const void* ptr, uint64_t bytes, uint64_t rows, uint64_t groups) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return fail(ARC_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[3] = {bytes, rows, groups};
  const cuuint64_t strides[2] = {bytes, bytes * rows};
  const cuuint32_t box[3] = {GP::kScaleGroup / 2, GP::kRowsPerCta, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(ptr), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    return fail(ARC_ERR_CUDA, "cuTensorMapEncodeTiled(codes) failed with CUresult %d", static_cast<int>(r));
  }
  return ARC_OK;
}

// Whether a grouped A8W4 product takes the pair kernel (scales in the operand) rather than the
// int32 kernel (scales on the partial sums): groups of more than a row tile of the latter, 128 rows,
// on average. 8 groups, 4096 x 4096: of 128 rows 43 us against 57, of 160 rows 80 against 60; 32
// groups, 2048 x 1024: 39 against 43, 68 against 46. ARC_A8W4_GROUPED="wide" | "narrow" (tests and tuning) forces one.
bool a8w4_grouped_wide(uint32_t T, uint32_t E) {
  if (const char* env = getenv("ARC_A8W4_GROUPED")) {
    if (strcmp(env, "wide") == 0) return true;
    if (strcmp(env, "narrow") == 0) return false;
  }
  return ceil_div(T, E < T ? E : T) > 128;
}

template <typename V>
cudaError_t launch_a8w4_grouped(const GQ::GroupedParams& p, uint64_t tiles, uint32_t sms, cudaStream_t stream) {
  const uint32_t grid = tiles < sms ? static_cast<uint32_t>(tiles) : sms;
  return launch_ex(V::kKernel, p, grid, V::Cfg::kThreads, V::kSmem, 1, stream);
}

// Blocks of the row grouping: one up to kOneBlockSlots slots, else one per SM of the largest
// part (the workspace size must not depend on the device).
constexpr uint32_t kRowBlocks = 148;
uint32_t group_rows_blocks(uint32_t slots, uint32_t* per_block) {
  if (slots <= GR::kOneBlockSlots) {
    *per_block = GR::kOneBlockSlots;
    return 1;
  }
  *per_block = ceil_div(ceil_div(slots, kRowBlocks), GR::kThreads) * GR::kThreads;
  return ceil_div(slots, *per_block);
}
size_t group_rows_workspace(uint32_t blocks, uint32_t groups) {
  return blocks == 1 ? 0 : size_t(GR::counts_ld(blocks)) * (groups + 1) * sizeof(uint32_t);
}

}  // namespace

extern "C" {

int arc_a8w4_grouped_workspace_bytes(int T, int E, int K, size_t* bytes) {
  if (bytes == nullptr || T <= 0 || E <= 0 || K <= 0) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "arc_a8w4_grouped_workspace_bytes: bad argument");
  }
  *bytes = a8w4_grouped_wide(T, E) ? size_t(T) * K * 2 : 0;
  return ARC_OK;
}

int arc_a8w4_grouped_gemm(const int8_t* A, const float* sa, const uint8_t* Wp, const uint16_t* sb,
                          const int32_t* offsets, uint16_t* C, void* workspace, size_t workspace_bytes, int T, int E,
                          int N, int K, int group, unsigned flags, cudaStream_t stream) {
  const char* what = "arc_a8w4_grouped_gemm";
  g_last_error[0] = '\0';
  if (sa == nullptr || sb == nullptr || offsets == nullptr) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  }
  if (int st = grouped_check(what, A, Wp, C, offsets, T, E, N, K)) return st;
  if (flags & ~(ARC_A8W4_PREPACKED | ARC_GROUPED_ZERO_OTHERS)) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: unknown flags 0x%x", what, flags);
  }
  if (group != static_cast<int>(GQ::kGroupK) || K % group != 0 || N % 8 != 0) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: need group == 128, K %% 128 == 0 and N %% 8 == 0 (group=%d N=%d K=%d)", what,
                group, N, K);
  }
  if (!aligned16(A) || !aligned16(Wp) || !aligned16(C) || (reinterpret_cast<uintptr_t>(sa) & 3u) ||
      (reinterpret_cast<uintptr_t>(sb) & 1u)) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: A, Wp and C must be 16-byte aligned", what);
  }
  if (int64_t(E) * N > 0x7FFFFFFF) return fail(ARC_ERR_UNSUPPORTED, "%s: E * N must be below 2^31", what);
  int dev = 0;
  if (int st = current_device(&dev, &DeviceState::grouped_status)) return st;
  const uint32_t live = E < T ? E : T;  // groups that can have rows
  const uint32_t avg = ceil_div(T, live);
  const uint32_t BT = avg <= 16 ? 16u : avg <= 32 ? 32u : avg <= 64 ? 64u : 128u;
  const arcb::lin::Groups groups = {offsets, static_cast<uint32_t>(E), static_cast<uint32_t>(T)};
  const bool zero_others = (flags & ARC_GROUPED_ZERO_OTHERS) != 0;
  if (a8w4_grouped_wide(T, E)) {
    if (int st = current_device(&dev, &DeviceState::linear_status)) return st;
    if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < size_t(T) * K * 2) {
      return fail(ARC_ERR_INVALID_ARGUMENT, "%s: needs a 16-byte aligned workspace of %zu bytes", what,
                  size_t(T) * K * 2);
    }
    const uint32_t max_pairs = static_cast<uint32_t>(g_dev[dev].max_linear_pairs);
    if (max_pairs == 0) return fail(ARC_ERR_UNSUPPORTED, "%s: no CTA pair fits on this device", what);
    const uint64_t pieces = uint64_t(T) * K / 16;
    const uint64_t per_block = uint64_t(GP::kWidenThreads) * GP::kWidenAhead;
    const uint64_t blocks = (pieces + per_block - 1) / per_block;
    if (blocks > 0x7FFFFFFFu) return fail(ARC_ERR_UNSUPPORTED, "%s: too many rows for one launch", what);
    cudaError_t e = launch_grid(GP::widen_rows_kernel, dim3(static_cast<uint32_t>(blocks)), GP::kWidenThreads, 0, stream,
                                reinterpret_cast<const uint4*>(A), static_cast<uint4*>(workspace), pieces);
    if (e != cudaSuccess) return cuda_fail(e, "widen_rows_kernel launch");
    GP::Params p = {};
    if (int st = encode_codes_3d(&p.tm_w, Wp, K / 2, N, E)) return st;
    if (int st = encode_2d(&p.tm_x, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, workspace, K, T, K, GP::kSubK, GP::kBox,
                           CU_TENSOR_MAP_SWIZZLE_128B, "rows")) {
      return st;
    }
    if (int st = encode_2d(&p.tm_xs, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, workspace, K, T, K, GP::kSubK, GP::kSmallBox,
                           CU_TENSOR_MAP_SWIZZLE_128B, "rows")) {
      return st;
    }
    p.sa = sa;
    p.sb = sb;
    p.G = K / GP::kScaleGroup;
    p.num_kb = K / GP::kSubK;
    p.split = (flags & ARC_A8W4_PREPACKED) ? 1u : 0u;
    e = grouped_pair_launch(p, groups, C, N, N, zero_others, max_pairs, GP::gemm_grouped_pair_kernel<false, true>,
                            GP::threads<true>(), GP::smem_bytes<true>(), stream);
    if (e != cudaSuccess) return cuda_fail(e, "gemm_grouped_pair_kernel launch");
    return ARC_OK;
  }
  GQ::GroupedParams p = {};
  if (int st = encode_2d(&p.tm_tok, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, A, K, T, K, GQ::kGroupK, BT,
                         CU_TENSOR_MAP_SWIZZLE_128B, "A")) {
    return st;
  }
  if (int st = encode_2d(&p.tm_wp, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, Wp, K / 2, uint64_t(E) * N, K / 2,
                         GQ::kPackedRow * GQ::kGps, GQ::kRows, CU_TENSOR_MAP_SWIZZLE_128B, "Wp")) {
    return st;
  }
  p.sa = sa;
  p.sb = sb;
  p.out = C;
  p.partials = nullptr;
  p.M = T;
  p.N = N;
  p.K = K;
  p.G = K / GQ::kGroupK;
  p.ldsb = p.G;
  p.ldc = N;
  p.R = GQ::kRows;
  p.tiles_n = ceil_div(N, GQ::kRows);
  p.split = (flags & ARC_A8W4_PREPACKED) ? 1u : 0u;
  p.groups = groups;
  p.zero_others = zero_others ? 1u : 0u;
  const uint64_t tiles = uint64_t(live + T / BT) * p.tiles_n;
  const uint32_t sms = static_cast<uint32_t>(g_dev[dev].sms);
  const cudaError_t e = BT == 16   ? launch_a8w4_grouped<A8w4Grouped16>(p, tiles, sms, stream)
                        : BT == 32 ? launch_a8w4_grouped<A8w4Grouped32>(p, tiles, sms, stream)
                        : BT == 64 ? launch_a8w4_grouped<A8w4Grouped64>(p, tiles, sms, stream)
                                   : launch_a8w4_grouped<A8w4Grouped128>(p, tiles, sms, stream);
  if (e != cudaSuccess) return cuda_fail(e, "gemm_a8w4_grouped_kernel launch");
  return ARC_OK;
}

int arc_group_rows_workspace_bytes(int slots, int E, size_t* bytes) {
  if (bytes == nullptr || slots <= 0 || E <= 0 || E > static_cast<int>(arcb::lin::kMaxGroups)) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "arc_group_rows_workspace_bytes: bad argument");
  }
  uint32_t per_block = 0;
  const uint32_t blocks = group_rows_blocks(slots, &per_block);
  *bytes = group_rows_workspace(blocks, E);
  return ARC_OK;
}

int arc_group_rows(const void* ids, int id_bytes, int32_t* offsets, int32_t* rows, int32_t* positions, void* workspace,
                   size_t workspace_bytes, int slots, int top, int E, cudaStream_t stream) {
  const char* what = "arc_group_rows";
  g_last_error[0] = '\0';
  if (ids == nullptr || offsets == nullptr || rows == nullptr || positions == nullptr) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  }
  if (slots <= 0 || top <= 0 || E <= 0) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: sizes must be positive (slots=%d top=%d E=%d)", what, slots, top, E);
  }
  if (slots > 0x7FFFFFFF - (1 << 20)) return fail(ARC_ERR_UNSUPPORTED, "%s: too many slots (%d)", what, slots);
  if (E > static_cast<int>(arcb::lin::kMaxGroups)) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: at most %u groups (got %d)", what, arcb::lin::kMaxGroups, E);
  }
  if (id_bytes != 4 && id_bytes != 8) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: ids are 4- or 8-byte integers (got %d bytes)", what, id_bytes);
  }
  if ((reinterpret_cast<uintptr_t>(ids) & (id_bytes - 1)) || (reinterpret_cast<uintptr_t>(offsets) & 3u) ||
      (reinterpret_cast<uintptr_t>(rows) & 3u) || (reinterpret_cast<uintptr_t>(positions) & 3u)) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: misaligned pointer", what);
  }
  uint32_t per_block = 0;
  const uint32_t blocks = group_rows_blocks(slots, &per_block);
  const size_t need = group_rows_workspace(blocks, E);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: needs a 16-byte aligned workspace of %zu bytes", what, need);
  }
  int dev = 0;
  if (int st = current_device(&dev, &DeviceState::grouped_status)) return st;
  GR::Params p = {};
  p.ids = ids;
  p.offsets = offsets;
  p.rows = rows;
  p.positions = positions;
  p.counts = blocks == 1 ? nullptr : static_cast<uint32_t*>(workspace);
  p.slots = slots;
  p.top = top;
  p.groups = E;
  p.blocks = blocks;
  p.per_block = per_block;
  cudaError_t e;
  if (blocks > 1) {
    const size_t hist = size_t(E + 1) * 4;
    e = id_bytes == 4 ? launch_grid(GR::count_rows_kernel<int32_t>, dim3(blocks), GR::kThreads, hist, stream, p)
                      : launch_grid(GR::count_rows_kernel<int64_t>, dim3(blocks), GR::kThreads, hist, stream, p);
    if (e != cudaSuccess) return cuda_fail(e, "count_rows_kernel launch");
  }
  const size_t smem = GR::smem_bytes(E);
  e = id_bytes == 4 ? launch_grid(GR::place_rows_kernel<int32_t>, dim3(blocks), GR::kThreads, smem, stream, p)
                    : launch_grid(GR::place_rows_kernel<int64_t>, dim3(blocks), GR::kThreads, smem, stream, p);
  if (e != cudaSuccess) return cuda_fail(e, "place_rows_kernel launch");
  return ARC_OK;
}

}  // extern "C"
