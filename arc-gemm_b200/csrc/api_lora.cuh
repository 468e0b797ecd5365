// api_lora.cuh — host side of the linear layer with adapters: argument checks, launches. Included by api.cu, whose
// helpers it uses.
#pragma once

#include "api_linear.cuh"

namespace {

namespace LO = arcb::lora;

int lora_init() {
  cudaError_t e = allow_smem(LP::lora_linear_pair_kernel<false, 256>, LP::kSmemBytes<256>);
  if (e == cudaSuccess) e = allow_smem(LP::lora_linear_pair_kernel<true, 256>, LP::kSmemBytes<256>);
  if (e == cudaSuccess) e = allow_smem(LP::lora_linear_pair_kernel<false, 128>, LP::kSmemBytes<128>);
  if (e == cudaSuccess) e = allow_smem(LP::lora_linear_pair_kernel<true, 128>, LP::kSmemBytes<128>);
  if (e == cudaSuccess) e = allow_smem(LS::lora_linear_stream_kernel<16>, LS::smem_bytes<16>());
  if (e == cudaSuccess) e = allow_smem(LS::lora_linear_stream_kernel<32>, LS::smem_bytes<32>());
  if (e == cudaSuccess) e = allow_smem(LS::lora_linear_stream_kernel<64>, LS::smem_bytes<64>());
  if (e == cudaSuccess) e = allow_smem(LS::lora_linear_stream_kernel<128>, LS::smem_bytes<128>());
  if (e == cudaSuccess) e = allow_smem(LO::lora_down_kernel<16>, LO::kDownSmem);
  if (e == cudaSuccess) e = allow_smem(LO::lora_down_kernel<32>, LO::kDownSmem);
  if (e == cudaSuccess) e = allow_smem(LO::lora_down_kernel<64>, LO::kDownSmem);
  if (e != cudaSuccess) {
    cudaGetLastError();  // clear
    return cuda_fail(e, "cudaFuncSetAttribute (linear layer with adapters)");
  }
  return ARC_OK;
}

// The workspace: u [M][ldu], the number of adapters of each row tile, their lists, and where the product streams the
// adapters' sums [M][N]. Row tiles have 16 rows at least, and a list has a place for each row of its tile.
struct LoraWorkspace {
  uint64_t ldu;
  size_t counts, lists, sums, bytes;  // offsets
};
LoraWorkspace lora_workspace(uint32_t M, uint32_t N, uint32_t rank, const LinearPlan& plan) {
  LoraWorkspace w;
  w.ldu = (uint64_t(rank) + 7) / 8 * 8;
  w.counts = (size_t(M) * w.ldu * 2 + 15) / 16 * 16;
  const size_t tiles = ceil_div(M, 16);
  w.lists = w.counts + (tiles * 2 + 15) / 16 * 16;
  w.sums = (w.lists + (size_t(M) + 256) * 2 + 15) / 16 * 16;  // row tiles x rows of a tile
  w.bytes = w.sums + (plan.pair ? 0 : size_t(M) * N * sizeof(float));
  return w;
}

// Rows that an adapter has among the 64 of an item.
uint32_t lora_rows(uint32_t rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : 64; }

// u and the row tiles' lists. Clusters share a block's adapters, of which a mixed batch has up to 32 and a prompt one, two
// where the next one begins: one cluster for both would make everyone wait for it (4096 rows of nine prompts, rank 64:
// 33 us). The contraction is split until the blocks fill the GPU or a warp has one box, but only in four
// from 5 blocks of rows on, so that a mixed batch finds clusters for its adapters.
int lora_down(LO::DownParams& p, uint32_t sms, cudaStream_t stream) {
  const uint32_t rows = lora_rows(p.rank), group = LO::kDownCols / rows;
  p.row_blocks = ceil_div(p.M, LO::kDownRows);
  p.rank_parts = ceil_div(p.rank, LO::kDownCols);
  const uint32_t adapters = p.adapters < p.M ? p.adapters : p.M;
  const uint32_t bound = ceil_div(adapters < LO::kDownRows ? adapters : LO::kDownRows, group);  // items of a block
  const uint32_t items = p.row_blocks * p.rank_parts, most = 2 * sms, boxes = ceil_div(p.K, 64);
  const uint32_t most_splits = p.row_blocks > 4 ? 4 : 8, least_sets = bound < 2 ? bound : 2;
  p.splits = 1;
  while (p.splits < most_splits && items * least_sets * p.splits * 2 <= most && boxes >= LO::kDownWarps * p.splits * 2) {
    p.splits *= 2;
  }
  p.sets = most / (items * p.splits);
  p.sets = p.sets < least_sets ? least_sets : p.sets < bound ? p.sets : bound;
  const uint64_t grid = uint64_t(items) * p.sets * p.splits;
  if (grid > 0x7FFFFFFFu) return fail(ARC_ERR_UNSUPPORTED, "too many rows for one launch");
  const auto kernel = rows == 16 ? LO::lora_down_kernel<16> : rows == 32 ? LO::lora_down_kernel<32> : LO::lora_down_kernel<64>;
  const cudaError_t e =
      launch_ex(kernel, p, static_cast<uint32_t>(grid), LO::kDownThreads, LO::kDownSmem, p.splits, stream);
  if (e != cudaSuccess) return cuda_fail(e, "lora_down_kernel launch");
  return ARC_OK;
}

template <bool SPLIT, uint32_t TN>
cudaError_t launch_lora_pair(const LP::LoraParams& p, uint64_t tiles, uint32_t max_pairs, cudaStream_t stream) {
  const uint32_t grid = SPLIT ? static_cast<uint32_t>(tiles) * 4 : 2 * static_cast<uint32_t>(tiles < max_pairs ? tiles : max_pairs);
  return launch_ex(LP::lora_linear_pair_kernel<SPLIT, TN>, p, grid, LP::kThreads, LP::kSmemBytes<TN>, SPLIT ? 4 : 2, stream);
}

template <uint32_t BN>
cudaError_t launch_lora_stream(const LS::LoraParams& p, uint32_t grid, cudaStream_t stream) {
  return launch_ex(LS::lora_linear_stream_kernel<BN>, p, grid, LS::kThreads, LS::smem_bytes<BN>(), p.splits, stream);
}

}  // namespace

extern "C" {

int arc_lora_linear_workspace_bytes(int M, int N, int K, int R, size_t* bytes) {
  if (bytes == nullptr || M <= 0 || N <= 0 || K <= 0 || R <= 0) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "arc_lora_linear_workspace_bytes: bad argument");
  }
  // The larger of the plans for aligned and for other output rows.
  *bytes = 0;
  int dev = 0;
  if (int st = current_device(&dev, &DeviceState::linear_status)) return st;
  for (bool aligned : {false, true}) {
    LinearPlan plan;
    if (int st = linear_plan(dev, M, 1, N, ceil_div(K, arcb::lin::BK), aligned, &plan)) return st;
    const size_t need = lora_workspace(M, N, R, plan).bytes;
    if (need > *bytes) *bytes = need;
  }
  return ARC_OK;
}

int arc_lora_linear(const uint16_t* x, const uint16_t* w, const uint16_t* a, const uint16_t* b, const void* ids,
                    int id_bytes, const float* scales, const uint16_t* bias, const uint16_t* residual, uint16_t* out,
                    void* workspace, size_t workspace_bytes, int M, int N, int K, int R, int L, int64_t ldx, int64_t ldw,
                    int64_t lda, int64_t a_stride, int64_t ldb, int64_t b_stride, int64_t ldr, int64_t ldo, int activation,
                    cudaStream_t stream) {
  const char* what = "arc_lora_linear";
  g_last_error[0] = '\0';
  if (x == nullptr || w == nullptr || a == nullptr || b == nullptr || ids == nullptr || out == nullptr) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  }
  if (M <= 0 || N <= 0 || K <= 0 || R <= 0 || L <= 0) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: sizes must be positive (M=%d N=%d K=%d R=%d L=%d)", what, M, N, K, R, L);
  }
  if (R > static_cast<int>(LO::kMaxRank) || L > static_cast<int>(LO::kMaxAdapters)) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: at most %u adapters of rank %u (got %d and %d)", what, LO::kMaxAdapters,
                LO::kMaxRank, L, R);
  }
  if (activation < ARC_ACT_NONE || activation > ARC_ACT_SILU) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", what, activation);
  }
  if (id_bytes != 4 && id_bytes != 8) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: ids are 4- or 8-byte integers (got %d bytes)", what, id_bytes);
  }
  if (int st = operand_check(what, "x", x, ldx, K)) return st;
  if (int st = operand_check(what, "w", w, ldw, K)) return st;
  if (int st = operand_check(what, "a", a, lda, K)) return st;
  if (int st = operand_check(what, "a's adapters", a, a_stride, int64_t(R - 1) * lda + K)) return st;
  if (int st = operand_check(what, "b", b, ldb, R)) return st;
  if (int st = operand_check(what, "b's adapters", b, b_stride, int64_t(N - 1) * ldb + R)) return st;
  if (int st = output_check(what, "out", out, ldo, N)) return st;
  if (residual != nullptr) {
    if (int st = output_check(what, "residual", residual, ldr, N)) return st;
  }
  if ((reinterpret_cast<uintptr_t>(bias) & 1u) || (reinterpret_cast<uintptr_t>(scales) & 3u) ||
      (reinterpret_cast<uintptr_t>(ids) & (id_bytes - 1))) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: bias, scales or ids are misaligned", what);
  }
  if (workspace == nullptr || !aligned16(workspace)) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: needs a 16-byte aligned workspace", what);
  }
  int dev = 0;
  if (int st = current_device(&dev, &DeviceState::linear_status)) return st;
  if (int st = current_device(&dev, &DeviceState::lora_status)) return st;
  const uint32_t num_kb = ceil_div(K, arcb::lin::BK), max_pairs = static_cast<uint32_t>(g_dev[dev].max_linear_pairs);
  LinearPlan plan;
  if (int st = linear_plan(dev, M, 1, N, num_kb, rows_aligned16(out, ldo), &plan)) return st;
  const LoraWorkspace ws = lora_workspace(M, N, R, plan);
  if (workspace_bytes < ws.bytes) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: needs a workspace of %zu bytes", what, ws.bytes);
  }
  const uint32_t tile_rows = plan.pair ? LP::kTile : plan.bn;

  uint8_t* const base = static_cast<uint8_t*>(workspace);
  LO::DownParams d = {};
  if (int st = encode_2d(&d.tm_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x, K, M, ldx, 64, LO::kDownRows,
                         CU_TENSOR_MAP_SWIZZLE_128B, "x")) {
    return st;
  }
  if (int st = encode_groups_3d(&d.tm_a, a, K, R, L, lda, a_stride, 64, lora_rows(R), "a")) return st;
  d.scales = scales;
  d.ids = ids;
  d.u = static_cast<uint16_t*>(workspace);
  if (plan.pair) {
    d.counts = reinterpret_cast<uint16_t*>(base + ws.counts);
    d.lists = reinterpret_cast<uint16_t*>(base + ws.lists);
  }
  d.ldu = ws.ldu;
  d.ids_wide = id_bytes == 8 ? 1 : 0;
  d.adapters = L;
  d.M = M;
  d.K = K;
  d.rank = R;
  d.tile_rows = tile_rows;
  d.tiles = ceil_div(M, tile_rows);
  d.cap = tile_rows;
  LO::Extra extra = {};
  if (plan.pair) {
    if (int st = encode_groups_3d(&extra.tm_u, workspace, R, M, 1, ws.ldu, 0, 64, LP::kRowsPerCta, "u")) return st;
    if (int st = encode_groups_3d(&extra.tm_b, b, R, N, L, ldb, b_stride, 64, plan.pair_cols / 2, "b")) return st;
  }
  extra.u = d.u;
  extra.b = b;
  extra.sums = reinterpret_cast<float*>(base + ws.sums);
  extra.ldu = ws.ldu;
  extra.ldb = ldb;
  extra.b_stride = b_stride;
  extra.counts = d.counts;
  extra.lists = d.lists;
  extra.ids = ids;
  extra.ids_wide = d.ids_wide;
  extra.adapters = L;
  extra.rows = M;
  extra.rank = R;
  extra.cap = d.cap;
  arcb::lin::Epilogue epi = {};
  epi.bias = bias;
  epi.residual = residual;
  epi.ldr = residual != nullptr ? ldr : 0;
  epi.act = static_cast<uint32_t>(activation);
  const uint64_t w_stride = uint64_t(N) * ldw;

  if (plan.pair) {
    LP::LoraParams p = {};
    if (int st = linear_pair_params(p, x, w, M, out, N, K, ldx, ldw, w_stride, ldo, epi, false, plan.pair_cols)) return st;
    p.extra = extra;
    if (int st = lora_down(d, static_cast<uint32_t>(g_dev[dev].sms), stream)) return st;
    const uint64_t tiles = uint64_t(p.tiles_m) * p.tiles_n;
    const bool narrow = plan.pair_cols == 128, split = plan.pair_splits > 1;
    const cudaError_t e = narrow ? (split ? launch_lora_pair<true, 128>(p, tiles, max_pairs, stream)
                                          : launch_lora_pair<false, 128>(p, tiles, max_pairs, stream))
                                 : (split ? launch_lora_pair<true, 256>(p, tiles, max_pairs, stream)
                                          : launch_lora_pair<false, 256>(p, tiles, max_pairs, stream));
    if (e != cudaSuccess) return cuda_fail(e, "lora_linear_pair_kernel launch");
    return ARC_OK;
  }
  LS::LoraParams p = {};
  uint32_t grid = 0;
  const arcb::lin::Groups groups = {nullptr, 1u, static_cast<uint32_t>(M)};
  if (int st = linear_stream_params(p, x, w, groups, out, N, K, ldx, ldw, w_stride, ldo, epi, false, plan, &grid)) return st;
  p.extra = extra;
  if (int st = lora_down(d, static_cast<uint32_t>(g_dev[dev].sms), stream)) return st;
  const cudaError_t e = plan.bn == 16   ? launch_lora_stream<16>(p, grid, stream)
                        : plan.bn == 32 ? launch_lora_stream<32>(p, grid, stream)
                        : plan.bn == 64 ? launch_lora_stream<64>(p, grid, stream)
                                        : launch_lora_stream<128>(p, grid, stream);
  if (e != cudaSuccess) return cuda_fail(e, "lora_linear_stream_kernel launch");
  return ARC_OK;
}

}  // extern "C"
