// api_linear.cuh — host side of the linear layer and the grouped products: argument checks,
// tensor maps, the choice between the streaming and the pair kernel, launches. Included by
// api.cu, whose helpers it uses.
#pragma once

#include "gemm_grouped_pair.cuh"
#include "gemm_linear_pair.cuh"
#include "gemm_linear_stream.cuh"
#include "linear_backward.cuh"

namespace {

namespace LS = arcb::linstream;
namespace LP = arcb::linpair;
namespace GP = arcb::grouppair;
namespace LB = arcb::linbwd;

// Row-major matrices [groups][rows][cols] (bf16), `ld` elements between rows and
// `group_stride` between groups.
int encode_groups_3d(CUtensorMap* map, const void* ptr, uint64_t cols, uint64_t rows, uint64_t groups, uint64_t ld,
                     uint64_t group_stride, uint32_t box_cols, uint32_t box_rows, const char* what,
                     CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return fail(ARC_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[3] = {cols, rows, groups};
  const cuuint64_t strides[2] = {ld * 2, (groups > 1 ? group_stride : ld) * 2};  // one group: never used
  const cuuint32_t box[3] = {box_cols, box_rows, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    return fail(ARC_ERR_CUDA, "cuTensorMapEncodeTiled(%s) failed with CUresult %d", what, static_cast<int>(r));
  }
  return ARC_OK;
}

// Whether TMA (or a 16-byte access) reaches every row of a bf16 matrix.
bool rows_aligned16(const void* p, uint64_t ld, uint64_t group_stride = 0) {
  return ((reinterpret_cast<uintptr_t>(p) | (ld * 2) | (group_stride * 2)) & 15u) == 0;
}

// The map of an epilogue matrix's 32 x 32 pieces, where TMA reaches it.
int encode_pieces(CUtensorMap* map, uint32_t* tma, const void* ptr, uint64_t cols, uint64_t rows, uint64_t groups,
                  uint64_t ld, uint64_t group_stride, const char* what) {
  *tma = ptr != nullptr && rows_aligned16(ptr, ld, groups > 1 ? group_stride : 0) ? 1u : 0u;
  if (!*tma) return ARC_OK;
  return encode_groups_3d(map, ptr, cols, rows, groups, ld, group_stride, 32, 32, what, CU_TENSOR_MAP_SWIZZLE_64B);
}

// Whether column pairs of a row-major bf16 matrix can be moved as 4-byte words.
uint32_t column_pairs(const void* p, uint64_t ld, uint32_t cols) {
  return cols % 2 == 0 && ld % 2 == 0 && (reinterpret_cast<uintptr_t>(p) & 3u) == 0 ? 1u : 0u;
}

// The pair kernel's parts of the contraction: two where the clusters of all tiles run at once, which
// are fewer than half the pairs (32 tiles: 512 x 4096 x 4096 30 us whole, 22 in two parts; 36 tiles:
// 512 x 4608 x 4096 30 and 41).
uint32_t pair_splits(uint64_t tiles, uint32_t num_kb, int dev) {
  return tiles <= static_cast<uint64_t>(g_dev[dev].max_linear_quads) && num_kb >= 8 ? 2 : 1;
}

// The kernel for a product of rows, in one group or several.
struct LinearPlan {
  bool pair;
  uint32_t pair_splits;            // pair kernel: 1 or 2
  uint32_t pair_cols;              // its tile's columns: 256 or 128
  uint32_t bn, splits, row_tiles;  // streaming kernel: row tile, parts of the contraction
};

// Estimated time of one group's product in microseconds: what a launch costs, and per round of
// blocks what a tile costs besides its contraction blocks of 64 and with them. The constants are a
// fit to the measured times of all plans of 500 products (1 to 4096 rows, 64 to 8192 columns,
// contractions of 64 to 6400). The plan it picks is 1.2 % behind the best one, geometric mean over
// those, and 1.4 % over 200 others; fixed thresholds on rows and tiles were 14 %.
double stream_cost(uint32_t rows, uint32_t cols, uint32_t num_kb, uint32_t bn, uint32_t splits, uint32_t sms) {
  // Two blocks fit on an SM; clusters of four and eight leave some slots empty. Counted on one B200,
  // by the blocks of a long launch that began before any ended: 296, 296, 284 and 264 blocks in
  // clusters of 1, 2, 4 and 8; a little less is assumed, since it depends on which SMs a part has.
  // (The driver's own count says one block per SM for any kernel that takes TMEM.)
  const double slots = 2.0 * sms * (splits == 8 ? 256.0 / 296 : splits == 4 ? 280.0 / 296 : 1.0);
  const double cluster = splits > 1 ? 1.36 : 0.0;
  const double blocks = static_cast<double>(ceil_div(rows, bn)) * ceil_div(cols, LS::kRows) * splits;
  const double load = blocks < 2.0 * sms ? blocks / (2.0 * sms) : 1.0;
  const double per_kb = 0.16 + 0.008 * (16 + bn / 8.0) * load;  // latency, and a share of the bandwidth
  const double epilogue = bn / 16.0 * (1.035 / splits + 0.48) + 0.95;
  return 1.3 + ceil(blocks / slots) * (ceil_div(num_kb, splits) * per_kb + epilogue) + cluster;
}

double pair_cost(uint32_t rows, uint32_t cols, uint32_t num_kb, uint32_t tile_cols, uint32_t splits, bool aligned,
                 uint32_t max_pairs) {
  const double tiles = static_cast<double>(ceil_div(rows, LP::kTile)) * ceil_div(cols, tile_cols);
  const double products = ceil_div(num_kb, splits) * (tile_cols == 128 ? 0.185 : 0.265) + 0.53;
  const double epilogue = (aligned ? 3.4 : 9.5) * tile_cols / 256;  // output rows by TMA, or element by element
  return 5.9 + ceil(tiles * splits / max_pairs) * (products > epilogue ? products : epilogue) + epilogue / splits +
         (splits > 1 ? 1.5 : 0.0);
}

// One group: the plan of the least estimated time. Several groups, of which the host knows only the
// average: the pair kernel's row tile fits itself to the group, so it takes all but the smallest
// groups (more than 16 rows; 64 groups, 2048 x 1024: at 32 rows 51 us against the streaming
// kernel's 70, at 128 57 against 116; 16 groups of 8 rows, 4096 x 4096: 93 against 85) where
// there are tiles for half of the pairs. Else the streaming kernel, its row tile the smallest that
// holds an average group's rows, with the contraction split over a cluster until the two block
// slots of every SM have work (four blocks of 64 each at least).
//
// ARC_LINEAR_PLAN="pair:S" | "pair128:S" | "BN:S" (tests and tuning) forces the choice where it is valid.
int linear_plan(int dev, uint32_t rows, uint32_t groups, uint32_t cols, uint32_t num_kb, bool aligned, LinearPlan* plan) {
  const uint32_t sms = static_cast<uint32_t>(g_dev[dev].sms);
  const uint32_t max_pairs = static_cast<uint32_t>(g_dev[dev].max_linear_pairs);
  const uint32_t live = groups < rows ? groups : rows;  // groups that can have rows
  const uint32_t avg = ceil_div(rows, live);
  *plan = {false, 1, LP::kTile, 16, 1, 0};
  if (const char* env = getenv("ARC_LINEAR_PLAN")) {
    unsigned bn = 0, s = 0;
    const bool narrow = sscanf(env, "pair128:%u", &s) == 1;
    if ((narrow || sscanf(env, "pair:%u", &s) == 1) && max_pairs > 0 && (s == 1 || s == 2)) {
      plan->pair = true;
      if (narrow) plan->pair_cols = 128;
      plan->pair_splits = s <= num_kb ? s : 1;
    } else if (sscanf(env, "%u:%u", &bn, &s) == 2 && (bn == 16 || bn == 32 || bn == 64 || bn == 128) &&
               (s == 1 || s == 2 || s == 4 || s == 8)) {
      plan->bn = bn;
      plan->splits = s <= num_kb ? s : 1;
    } else {
      return fail(ARC_ERR_INVALID_ARGUMENT, "ARC_LINEAR_PLAN must be 'pair:S', 'pair128:S' or 'BN:S' (got '%s')", env);
    }
  } else if (groups == 1) {
    double best = 1e30;
    for (uint32_t bn : {16u, 32u, 64u, 128u}) {
      for (uint32_t s : {1u, 2u, 4u, 8u}) {
        if (s > num_kb) break;
        const double t = stream_cost(rows, cols, num_kb, bn, s, sms);
        if (t < best) {
          best = t;
          plan->bn = bn;
          plan->splits = s;
        }
      }
    }
    for (uint32_t tile_cols : {256u, 128u}) {
      const uint64_t tiles = uint64_t(ceil_div(rows, LP::kTile)) * ceil_div(cols, tile_cols);
      for (uint32_t s = 1; max_pairs > 0 && s <= pair_splits(tiles, num_kb, dev); ++s) {
        const double t = pair_cost(rows, cols, num_kb, tile_cols, s, aligned, max_pairs);
        if (t < best) {
          best = t;
          plan->pair = true;
          plan->pair_splits = s;
          plan->pair_cols = tile_cols;
        }
      }
    }
  } else {
    const uint64_t pair_tiles = uint64_t(ceil_div(avg, GP::kTileT)) * live * ceil_div(cols, GP::kTileF);
    plan->pair = max_pairs > 0 && avg > 16 && pair_tiles * 2 > max_pairs;
    plan->bn = avg <= 16 ? 16 : avg <= 32 ? 32 : avg <= 64 ? 64 : 128;
    for (;; plan->bn /= 2) {
      const uint64_t tiles = uint64_t(live + rows / plan->bn) * ceil_div(cols, LS::kRows);
      plan->splits = 1;
      for (uint32_t s : {8u, 4u, 2u}) {
        if (tiles * s <= 2 * sms && num_kb >= 4 * s) {
          plan->splits = s;
          break;
        }
      }
      if (plan->bn == 16 || tiles * plan->splits >= sms) break;
    }
  }
  // With several groups the host knows only a bound: a group of c rows has at most c / bn + 1 tiles.
  plan->row_tiles = groups == 1 ? ceil_div(rows, plan->bn) : live + rows / plan->bn;
  return ARC_OK;
}

// The kernel of arc_linear_bf16 as ncu lists it (16-byte aligned output rows assumed).
int linear_kernel_name(int dev, uint32_t M, uint32_t N, uint32_t K, char* name, int len) {
  if (int st = current_device(&dev, &DeviceState::linear_status)) return st;
  LinearPlan plan;
  if (int st = linear_plan(dev, M, 1, N, ceil_div(K, arcb::lin::BK), true, &plan)) return st;
  if (plan.pair) {
    snprintf(name, static_cast<size_t>(len), "gemm_linear_pair_kernel<0, 0, 0, %d, %u>",
             plan.pair_splits > 1 ? 1 : 0, plan.pair_cols);
  } else {
    snprintf(name, static_cast<size_t>(len), "gemm_linear_stream_kernel<%u, 0>", plan.bn);
  }
  return ARC_OK;
}

// The pair kernel, one cluster of two pairs per tile if the contraction is split.
template <bool A_MN, bool B_MN, bool ALONG_K, uint32_t TN>
cudaError_t launch_linear_pair(const LP::Params& p, uint64_t tiles, uint32_t splits, uint32_t max_pairs, cudaStream_t stream) {
  if (splits > 1) {
    return launch_ex(LP::gemm_linear_pair_kernel<A_MN, B_MN, ALONG_K, true, TN>, p, static_cast<uint32_t>(tiles) * 4,
                     LP::kThreads, LP::kSmemBytes<TN>, 4, stream);
  }
  const uint32_t grid = 2 * static_cast<uint32_t>(tiles < max_pairs ? tiles : max_pairs);
  return launch_ex(LP::gemm_linear_pair_kernel<A_MN, B_MN, ALONG_K, false, TN>, p, grid, LP::kThreads, LP::kSmemBytes<TN>, 2,
                   stream);
}

template <uint32_t BN, bool W_MN>
cudaError_t launch_stream(const LS::Params& p, uint32_t grid, cudaStream_t stream) {
  return launch_ex(LS::gemm_linear_stream_kernel<BN, W_MN>, p, grid, LS::kThreads, LS::smem_bytes<BN>(), p.splits,
                   stream);
}

template <bool W_MN>
cudaError_t launch_stream_bn(const LS::Params& p, uint32_t bn, uint32_t grid, cudaStream_t stream) {
  return bn == 16   ? launch_stream<16, W_MN>(p, grid, stream)
         : bn == 32 ? launch_stream<32, W_MN>(p, grid, stream)
         : bn == 64 ? launch_stream<64, W_MN>(p, grid, stream)
                    : launch_stream<128, W_MN>(p, grid, stream);
}

#define ARC_LINEAR_STREAM_VARIANTS(X) X(16, false) X(32, false) X(64, false) X(128, false) \
  X(16, true) X(32, true) X(64, true) X(128, true)

// How many clusters of `size` CTAs of a kernel fit at once (0 where the query fails: no plan uses them).
template <typename Kern>
int clusters_at_once(Kern kernel, const DeviceState& st, uint32_t size, uint32_t threads, size_t smem) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(size * (st.sms / size), 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    cudaGetLastError();  // clear
    n = 0;
  }
  return n;
}

int linear_init(DeviceState& st) {
  cudaError_t e = cudaSuccess;
#define ARC_SET_ATTR(BN, MN) \
  if (e == cudaSuccess) e = allow_smem(LS::gemm_linear_stream_kernel<BN, MN>, LS::smem_bytes<BN>());
  ARC_LINEAR_STREAM_VARIANTS(ARC_SET_ATTR)
#undef ARC_SET_ATTR
#define ARC_SET_ATTR(SPLIT)                                                                                         \
  if (e == cudaSuccess) e = allow_smem(LP::gemm_linear_pair_kernel<false, false, false, SPLIT, 256>, LP::kSmemBytes<256>); \
  if (e == cudaSuccess) e = allow_smem(LP::gemm_linear_pair_kernel<false, true, false, SPLIT, 256>, LP::kSmemBytes<256>);  \
  if (e == cudaSuccess) e = allow_smem(LP::gemm_linear_pair_kernel<false, false, false, SPLIT, 128>, LP::kSmemBytes<128>); \
  if (e == cudaSuccess) e = allow_smem(LP::gemm_linear_pair_kernel<false, true, false, SPLIT, 128>, LP::kSmemBytes<128>);  \
  if (e == cudaSuccess) e = allow_smem(LP::gemm_linear_pair_kernel<true, true, true, SPLIT, 256>, LP::kSmemBytes<256>);
  ARC_SET_ATTR(false)
  ARC_SET_ATTR(true)
#undef ARC_SET_ATTR
  if (e == cudaSuccess) e = allow_smem(GP::gemm_grouped_pair_kernel<false, false>, GP::smem_bytes<false>());
  if (e == cudaSuccess) e = allow_smem(GP::gemm_grouped_pair_kernel<true, false>, GP::smem_bytes<false>());
  if (e == cudaSuccess) e = allow_smem(GP::gemm_grouped_pair_kernel<false, true>, GP::smem_bytes<true>());
  if (e != cudaSuccess) {
    cudaGetLastError();  // clear
    return cuda_fail(e, "cudaFuncSetAttribute (linear and grouped kernels)");
  }
  // Pairs of the largest of these kernels, and clusters of two pairs of the linear one.
  st.max_linear_pairs =
      clusters_at_once(GP::gemm_grouped_pair_kernel<false, true>, st, 2, GP::threads<true>(), GP::smem_bytes<true>());
  st.max_linear_quads = clusters_at_once(LP::gemm_linear_pair_kernel<false, false, false, true, 256>, st, 4, LP::kThreads,
                                         LP::kSmemBytes<256>);
  return ARC_OK;
}

// The walk's fields and the launch of the grouped pair kernel (its maps are set by the caller).
cudaError_t grouped_pair_launch(GP::Params& p, const arcb::lin::Groups& groups, uint16_t* out, uint64_t ldo,
                                uint32_t cols, bool zero_others, uint32_t max_pairs, void (*kernel)(GP::Params),
                                uint32_t threads, size_t smem, cudaStream_t stream) {
  p.out = out;
  p.ldo = ldo;
  p.groups = groups;
  p.cols = cols;
  p.tiles_f = ceil_div(cols, GP::kTileF);
  p.pair_store = column_pairs(out, ldo, cols);
  p.zero_others = zero_others ? 1u : 0u;
  // The host knows only a bound: a group of c rows has at most c / kTileT + 1 row tiles.
  const uint64_t tiles = uint64_t((groups.num < groups.rows ? groups.num : groups.rows) + groups.rows / GP::kTileT) *
                         p.tiles_f;
  const uint32_t grid = 2 * static_cast<uint32_t>(tiles < max_pairs ? tiles : max_pairs);
  return launch_ex(kernel, p, grid, threads, smem, 2, stream);
}

// The pair kernel's operands, epilogue and walk for one group of rows.
int linear_pair_params(LP::Params& p, const uint16_t* a, const uint16_t* w, uint32_t rows, uint16_t* out, uint32_t cols,
                       uint32_t inner, uint64_t lda, uint64_t ldw, uint64_t w_stride, uint64_t ldo,
                       const arcb::lin::Epilogue& epi, bool grad, uint32_t tile_cols) {
  const uint64_t w_rows = grad ? inner : cols, w_cols = grad ? cols : inner;
  if (int st = encode_groups_3d(&p.tm_a, a, inner, rows, 1, lda, 0, 64, LP::kRowsPerCta, "rows")) return st;
  if (int st = encode_groups_3d(&p.tm_b, w, w_cols, w_rows, 1, ldw, w_stride, 64, grad ? 64 : tile_cols / 2, "weights")) {
    return st;
  }
  p.out = out;
  p.ldo = ldo;
  p.epi = epi;
  p.epi.wide_bias = aligned16(epi.bias) ? 1u : 0u;
  if (int st = encode_pieces(&p.tm_out, &p.tma_out, out, cols, rows, 1, ldo, 0, "out")) return st;
  if (int st = encode_pieces(&p.tm_z, &p.tma_z, epi.z, cols, rows, 1, epi.ldz, 0, "z")) return st;
  if (int st = encode_pieces(&p.tm_res, &p.tma_res, epi.residual, cols, rows, 1, epi.ldr, 0, "residual")) return st;
  p.M = rows;
  p.N = cols;
  p.tiles_m = ceil_div(rows, LP::kTile);
  p.tiles_n = ceil_div(cols, tile_cols);
  p.num_kb = ceil_div(inner, arcb::lin::BK);
  if (uint64_t(p.tiles_m) * p.tiles_n * 4 > 0x7FFFFFFFu) {
    return fail(ARC_ERR_UNSUPPORTED, "the product has too many tiles for one launch");
  }
  return ARC_OK;
}

// The same of the streaming kernel, and its grid.
int linear_stream_params(LS::Params& p, const uint16_t* a, const uint16_t* w, const arcb::lin::Groups& groups,
                         uint16_t* out, uint32_t cols, uint32_t inner, uint64_t lda, uint64_t ldw, uint64_t w_stride,
                         uint64_t ldo, const arcb::lin::Epilogue& epi, bool grad, const LinearPlan& plan, uint32_t* grid) {
  const uint64_t w_rows = grad ? inner : cols, w_cols = grad ? cols : inner;
  if (int st = encode_groups_3d(&p.tm_w, w, w_cols, w_rows, groups.num, ldw, w_stride, 64, grad ? 64 : LS::kRows,
                                "weights")) {
    return st;
  }
  if (int st = encode_2d(&p.tm_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a, inner, groups.rows, lda, 64, plan.bn,
                         CU_TENSOR_MAP_SWIZZLE_128B, "rows")) {
    return st;
  }
  p.out = out;
  p.ldo = ldo;
  p.groups = groups;
  p.epi = epi;
  p.epi.pair_residual = column_pairs(epi.residual, epi.ldr, cols);
  p.epi.pair_z = column_pairs(epi.z, epi.ldz, cols);
  p.epi.pair_out = column_pairs(out, ldo, cols);
  p.cols = cols;
  p.tiles_n = ceil_div(cols, LS::kRows);
  p.num_kb = ceil_div(inner, arcb::lin::BK);
  p.splits = plan.splits;
  const uint64_t blocks = uint64_t(plan.row_tiles) * p.tiles_n * plan.splits;
  if (blocks > 0x7FFFFFFFu) return fail(ARC_ERR_UNSUPPORTED, "the product has too many tiles for one launch");
  *grid = static_cast<uint32_t>(blocks);
  return ARC_OK;
}

// out[rows][cols] = epilogue of a [rows][inner] times w, per group. grad = false: w is
// [E][cols][inner]; grad = true: w is [E][inner][cols] (the gradient of the rows).
int linear_rows(const uint16_t* a, const uint16_t* w, const arcb::lin::Groups& groups, uint16_t* out, uint32_t cols,
                uint32_t inner, uint64_t lda, uint64_t ldw, uint64_t w_stride, uint64_t ldo,
                const arcb::lin::Epilogue& epi, bool grad, bool zero_others, cudaStream_t stream) {
  int dev = 0;
  if (int st = current_device(&dev, &DeviceState::linear_status)) return st;
  const uint32_t num_kb = ceil_div(inner, arcb::lin::BK);
  LinearPlan plan;
  if (int st = linear_plan(dev, groups.rows, groups.num, cols, num_kb, rows_aligned16(out, ldo), &plan)) return st;
  const uint64_t w_rows = grad ? inner : cols, w_cols = grad ? cols : inner;
  cudaError_t e;
  const uint32_t max_pairs = static_cast<uint32_t>(g_dev[dev].max_linear_pairs);
  if (plan.pair && groups.offsets != nullptr) {
    GP::Params p = {};
    if (int st = encode_groups_3d(&p.tm_w, w, w_cols, w_rows, groups.num, ldw, w_stride, 64,
                                  grad ? 64 : GP::kRowsPerCta, "weights")) {
      return st;
    }
    if (int st = encode_2d(&p.tm_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a, inner, groups.rows, lda, GP::kSubK,
                           GP::kBox, CU_TENSOR_MAP_SWIZZLE_128B, "rows")) {
      return st;
    }
    if (int st = encode_2d(&p.tm_xs, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a, inner, groups.rows, lda, GP::kSubK,
                           GP::kSmallBox, CU_TENSOR_MAP_SWIZZLE_128B, "rows")) {
      return st;
    }
    p.num_kb = num_kb;
    e = grouped_pair_launch(p, groups, out, ldo, cols, zero_others, max_pairs,
                            grad ? GP::gemm_grouped_pair_kernel<true, false> : GP::gemm_grouped_pair_kernel<false, false>,
                            GP::threads<false>(), GP::smem_bytes<false>(), stream);
    if (e != cudaSuccess) return cuda_fail(e, "gemm_grouped_pair_kernel launch");
    return ARC_OK;
  }
  if (plan.pair) {
    LP::Params p = {};
    if (int st = linear_pair_params(p, a, w, groups.rows, out, cols, inner, lda, ldw, w_stride, ldo, epi, grad,
                                    plan.pair_cols)) {
      return st;
    }
    const uint64_t tiles = uint64_t(p.tiles_m) * p.tiles_n;
    const bool narrow = plan.pair_cols == 128;
    const auto launch = grad ? (narrow ? launch_linear_pair<false, true, false, 128> : launch_linear_pair<false, true, false, 256>)
                             : (narrow ? launch_linear_pair<false, false, false, 128> : launch_linear_pair<false, false, false, 256>);
    e = launch(p, tiles, plan.pair_splits, max_pairs, stream);
    if (e != cudaSuccess) return cuda_fail(e, "gemm_linear_pair_kernel launch");
    return ARC_OK;
  }
  LS::Params p = {};
  uint32_t grid = 0;
  if (int st = linear_stream_params(p, a, w, groups, out, cols, inner, lda, ldw, w_stride, ldo, epi, grad, plan, &grid)) {
    return st;
  }
  p.zero_others = zero_others ? 1u : 0u;
  e = grad ? launch_stream_bn<true>(p, plan.bn, grid, stream) : launch_stream_bn<false>(p, plan.bn, grid, stream);
  if (e != cudaSuccess) return cuda_fail(e, "gemm_linear_stream_kernel launch");
  return ARC_OK;
}

// dw[e][n][k] = sum over the rows t of group e of dy[t][n] x[t][k].
int linear_dw(const char* what, const uint16_t* dy, const uint16_t* x, const arcb::lin::Groups& groups, uint16_t* dw,
              uint32_t N, uint32_t K, uint64_t lddy, uint64_t ldx, uint64_t lddw, uint64_t dw_stride,
              cudaStream_t stream) {
  int dev = 0;
  if (int st = current_device(&dev, &DeviceState::linear_status)) return st;
  const uint32_t max_pairs = static_cast<uint32_t>(g_dev[dev].max_linear_pairs);
  if (max_pairs == 0) return fail(ARC_ERR_UNSUPPORTED, "%s: no CTA pair fits on this device", what);
  LP::Params p = {};
  if (int st = encode_groups_3d(&p.tm_a, dy, N, groups.rows, 1, lddy, 0, 64, 64, "dy")) return st;
  if (int st = encode_groups_3d(&p.tm_b, x, K, groups.rows, 1, ldx, 0, 64, 64, "x")) return st;
  p.out = dw;
  p.ldo = lddw;
  p.out_group = dw_stride;
  p.groups = groups;
  if (int st = encode_pieces(&p.tm_out, &p.tma_out, dw, K, N, groups.num, lddw, dw_stride, "dw")) return st;
  p.M = N;
  p.N = K;
  p.tiles_m = ceil_div(N, LP::kTile);
  p.tiles_n = ceil_div(K, LP::kTile);
  const uint64_t tiles = uint64_t(p.tiles_m) * p.tiles_n * groups.num;
  if (tiles * 4 > 0x7FFFFFFFu) return fail(ARC_ERR_UNSUPPORTED, "%s: too many tiles for one launch", what);
  // The host knows the contraction's length only for one group of all rows.
  const uint32_t splits =
      groups.offsets == nullptr ? pair_splits(tiles, ceil_div(groups.rows, arcb::lin::BK), dev) : 1;
  const cudaError_t e = launch_linear_pair<true, true, true, 256>(p, tiles, splits, max_pairs, stream);
  if (e != cudaSuccess) return cuda_fail(e, "gemm_linear_pair_kernel launch");
  return ARC_OK;
}

// Checks shared by the grouped entry points.
int grouped_check(const char* what, const void* a, const void* b, const void* c, const int32_t* offsets, int T, int E,
                  int N, int K) {
  if (a == nullptr || b == nullptr || c == nullptr) return fail(ARC_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (T <= 0 || E <= 0 || N <= 0 || K <= 0) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: sizes must be positive (T=%d E=%d N=%d K=%d)", what, T, E, N, K);
  }
  if (E > static_cast<int>(arcb::lin::kMaxGroups)) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: at most %u groups (got %d)", what, arcb::lin::kMaxGroups, E);
  }
  if (offsets == nullptr && E != 1) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: null offsets mean one group, got %d", what, E);
  }
  if (reinterpret_cast<uintptr_t>(offsets) & 3u) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: offsets must be 4-byte aligned", what);
  }
  return ARC_OK;
}

int operand_check(const char* what, const char* name, const void* p, int64_t ld, int64_t cols) {
  if (ld < cols) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: leading dimension of %s too small (%lld < %lld)", what, name,
                static_cast<long long>(ld), static_cast<long long>(cols));
  }
  if (!aligned16(p) || ld % 8 != 0) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: %s must be 16-byte aligned with a leading dimension that is a multiple of 8",
                what, name);
  }
  return ARC_OK;
}

int output_check(const char* what, const char* name, const void* p, int64_t ld, int64_t cols) {
  if (ld < cols) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: leading dimension of %s too small (%lld < %lld)", what, name,
                static_cast<long long>(ld), static_cast<long long>(cols));
  }
  if (reinterpret_cast<uintptr_t>(p) & 1u) return fail(ARC_ERR_UNSUPPORTED, "%s: %s is misaligned", what, name);
  return ARC_OK;
}

// Row blocks of the dz pass: the grid fills the GPU's block slots once, without a rest (a rest of
// a few blocks costs a whole round: 59 against 43 us at 4096 x 8192), at least 16 rows each.
// The workspace size must not depend on the device.
constexpr uint32_t kDzBlocks = 148 * LB::kBlocksPerSm;
uint32_t dz_row_blocks(uint32_t M, uint32_t N) {
  const uint32_t want = kDzBlocks / ceil_div(N, LB::kColsPerBlock), most = ceil_div(M, 16);
  return want < 1 ? 1 : want < most ? want : most;
}
// dz lies in the workspace with rows that TMA can read.
uint64_t dz_ld(uint32_t N) { return (uint64_t(N) + 7) / 8 * 8; }
size_t dz_bytes(uint32_t M, uint32_t N) { return (size_t(M) * dz_ld(N) * 2 + 255) / 256 * 256; }

}  // namespace

extern "C" {

int arc_linear_bf16(const uint16_t* x, const uint16_t* w, const uint16_t* bias, const uint16_t* residual,
                    uint16_t* out, uint16_t* z, int M, int N, int K, int64_t ldx, int64_t ldw, int64_t ldr,
                    int64_t ldo, int64_t ldz, int activation, cudaStream_t stream) {
  const char* what = "arc_linear_bf16";
  g_last_error[0] = '\0';
  if (x == nullptr || w == nullptr || out == nullptr) return fail(ARC_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (M <= 0 || N <= 0 || K <= 0) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: sizes must be positive (M=%d N=%d K=%d)", what, M, N, K);
  }
  if (activation < ARC_ACT_NONE || activation > ARC_ACT_SILU) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", what, activation);
  }
  if (int st = operand_check(what, "x", x, ldx, K)) return st;
  if (int st = operand_check(what, "w", w, ldw, K)) return st;
  if (int st = output_check(what, "out", out, ldo, N)) return st;
  if (residual != nullptr) {
    if (int st = output_check(what, "residual", residual, ldr, N)) return st;
  }
  if (z != nullptr) {
    if (int st = output_check(what, "z", z, ldz, N)) return st;
  }
  if (reinterpret_cast<uintptr_t>(bias) & 1u) return fail(ARC_ERR_UNSUPPORTED, "%s: bias is misaligned", what);
  arcb::lin::Epilogue epi = {};
  epi.bias = bias;
  epi.residual = residual;
  epi.z = z;
  epi.ldr = residual != nullptr ? ldr : 0;
  epi.ldz = z != nullptr ? ldz : 0;
  epi.act = static_cast<uint32_t>(activation);
  const arcb::lin::Groups groups = {nullptr, 1u, static_cast<uint32_t>(M)};
  return linear_rows(x, w, groups, out, N, K, ldx, ldw, uint64_t(N) * ldw, ldo, epi, false, false, stream);
}

int arc_linear_backward_workspace_bytes(int M, int N, int need_dz, int need_dbias, size_t* bytes) {
  if (bytes == nullptr || M <= 0 || N <= 0) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "arc_linear_backward_workspace_bytes: bad argument");
  }
  *bytes = (need_dz ? dz_bytes(M, N) : 0) +
           (need_dbias ? size_t(dz_row_blocks(M, N)) * N * sizeof(float) : 0);
  return ARC_OK;
}

int arc_linear_backward(const uint16_t* dy, const uint16_t* x, const uint16_t* w, const uint16_t* z, uint16_t* dx,
                        uint16_t* dw, uint16_t* dbias, void* workspace, size_t workspace_bytes, int M, int N, int K,
                        int64_t lddy, int64_t ldx, int64_t ldw, int64_t ldz, int64_t lddx, int64_t lddw,
                        int activation, cudaStream_t stream) {
  const char* what = "arc_linear_backward";
  g_last_error[0] = '\0';
  if (dy == nullptr || (dx == nullptr && dw == nullptr && dbias == nullptr) || (dx != nullptr && w == nullptr) ||
      (dw != nullptr && x == nullptr)) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  }
  if (M <= 0 || N <= 0 || K <= 0) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: sizes must be positive (M=%d N=%d K=%d)", what, M, N, K);
  }
  if (activation < ARC_ACT_NONE || activation > ARC_ACT_SILU) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", what, activation);
  }
  if (activation != ARC_ACT_NONE && z == nullptr) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: an activation's gradient needs z", what);
  }
  if (int st = output_check(what, "dy", dy, lddy, N)) return st;
  if (activation == ARC_ACT_NONE) {
    z = nullptr;
  } else if (int st = output_check(what, "z", z, ldz, N)) {
    return st;
  }
  if (dx != nullptr) {
    if (int st = operand_check(what, "w", w, ldw, K)) return st;
    if (int st = output_check(what, "dx", dx, lddx, K)) return st;
  }
  if (dw != nullptr) {
    if (int st = operand_check(what, "x", x, ldx, K)) return st;
    if (int st = output_check(what, "dw", dw, lddw, K)) return st;
  }
  if (reinterpret_cast<uintptr_t>(dbias) & 1u) return fail(ARC_ERR_UNSUPPORTED, "%s: dbias is misaligned", what);
  // The products read dy itself where there is nothing to multiply it by and TMA can read it.
  const bool products = dx != nullptr || dw != nullptr;
  const bool need_dz = products && (z != nullptr || !aligned16(dy) || lddy % 8 != 0);
  const uint32_t row_blocks = dz_row_blocks(M, N);
  const size_t dz_size = need_dz ? dz_bytes(M, N) : 0;
  const size_t need = dz_size + (dbias != nullptr ? size_t(row_blocks) * N * sizeof(float) : 0);
  if (need > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need)) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: needs a 16-byte aligned workspace of %zu bytes", what, need);
  }
  int dev = 0;
  if (int st = current_device(&dev, &DeviceState::linear_status)) return st;
  if (need_dz || dbias != nullptr) {
    LB::Params p = {};
    p.dy = dy;
    p.z = z;
    p.dz = need_dz ? static_cast<uint16_t*>(workspace) : nullptr;
    p.partial = dbias != nullptr ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + dz_size) : nullptr;
    p.lddy = lddy;
    p.ldz = ldz;
    p.lddz = dz_ld(N);
    p.M = M;
    p.N = N;
    p.act = static_cast<uint32_t>(activation);
    p.rows_per_block = ceil_div(M, row_blocks);
    const bool vec = N % 8 == 0 && rows_aligned16(dy, lddy) && (z == nullptr || rows_aligned16(z, ldz));
    const dim3 grid(ceil_div(N, LB::kColsPerBlock), row_blocks, 1);
    cudaError_t e = vec ? launch_grid(LB::linear_dz_kernel<true>, grid, LB::kThreads, 0, stream, p)
                        : launch_grid(LB::linear_dz_kernel<false>, grid, LB::kThreads, 0, stream, p);
    if (e != cudaSuccess) return cuda_fail(e, "linear_dz_kernel launch");
    if (dbias != nullptr) {
      e = launch_grid(LB::linear_dbias_kernel, dim3(ceil_div(N, LB::kThreads), 1, 1), LB::kThreads, 0, stream,
                      static_cast<const float*>(p.partial), dbias, uint32_t(N), row_blocks);
      if (e != cudaSuccess) return cuda_fail(e, "linear_dbias_kernel launch");
    }
    if (need_dz) {
      dy = p.dz;
      lddy = p.lddz;
    }
  }
  const arcb::lin::Groups groups = {nullptr, 1u, static_cast<uint32_t>(M)};
  if (dx != nullptr) {
    if (int st = linear_rows(dy, w, groups, dx, K, N, lddy, ldw, uint64_t(N) * ldw, lddx, arcb::lin::Epilogue{}, true,
                             false, stream)) {
      return st;
    }
  }
  return dw != nullptr ? linear_dw(what, dy, x, groups, dw, N, K, lddy, ldx, lddw, 0, stream) : ARC_OK;
}

int arc_grouped_matmul(const uint16_t* x, const uint16_t* w, const int32_t* offsets, uint16_t* out, int T, int E,
                       int N, int K, int64_t ldx, int64_t ldw, int64_t w_stride, int64_t ldo, unsigned flags,
                       cudaStream_t stream) {
  const char* what = "arc_grouped_matmul";
  g_last_error[0] = '\0';
  if (int st = grouped_check(what, x, w, out, offsets, T, E, N, K)) return st;
  if (flags & ~ARC_GROUPED_ZERO_OTHERS) return fail(ARC_ERR_INVALID_ARGUMENT, "%s: unknown flags 0x%x", what, flags);
  if (int st = operand_check(what, "x", x, ldx, K)) return st;
  if (int st = operand_check(what, "w", w, ldw, K)) return st;
  if (int st = operand_check(what, "w's groups", w, w_stride, int64_t(N - 1) * ldw + K)) return st;
  if (int st = output_check(what, "out", out, ldo, N)) return st;
  const arcb::lin::Groups groups = {offsets, static_cast<uint32_t>(E), static_cast<uint32_t>(T)};
  return linear_rows(x, w, groups, out, N, K, ldx, ldw, w_stride, ldo, arcb::lin::Epilogue{}, false,
                     (flags & ARC_GROUPED_ZERO_OTHERS) != 0 && offsets != nullptr, stream);
}

int arc_grouped_matmul_dx(const uint16_t* dy, const uint16_t* w, const int32_t* offsets, uint16_t* dx, int T, int E,
                          int N, int K, int64_t lddy, int64_t ldw, int64_t w_stride, int64_t lddx, unsigned flags,
                          cudaStream_t stream) {
  const char* what = "arc_grouped_matmul_dx";
  g_last_error[0] = '\0';
  if (int st = grouped_check(what, dy, w, dx, offsets, T, E, N, K)) return st;
  if (flags & ~ARC_GROUPED_ZERO_OTHERS) return fail(ARC_ERR_INVALID_ARGUMENT, "%s: unknown flags 0x%x", what, flags);
  if (int st = operand_check(what, "dy", dy, lddy, N)) return st;
  if (int st = operand_check(what, "w", w, ldw, K)) return st;
  if (int st = operand_check(what, "w's groups", w, w_stride, int64_t(N - 1) * ldw + K)) return st;
  if (int st = output_check(what, "dx", dx, lddx, K)) return st;
  const arcb::lin::Groups groups = {offsets, static_cast<uint32_t>(E), static_cast<uint32_t>(T)};
  return linear_rows(dy, w, groups, dx, K, N, lddy, ldw, w_stride, lddx, arcb::lin::Epilogue{}, true,
                     (flags & ARC_GROUPED_ZERO_OTHERS) != 0 && offsets != nullptr, stream);
}

int arc_grouped_matmul_dw(const uint16_t* dy, const uint16_t* x, const int32_t* offsets, uint16_t* dw, int T, int E,
                          int N, int K, int64_t lddy, int64_t ldx, int64_t lddw, int64_t dw_stride,
                          cudaStream_t stream) {
  const char* what = "arc_grouped_matmul_dw";
  g_last_error[0] = '\0';
  if (int st = grouped_check(what, dy, x, dw, offsets, T, E, N, K)) return st;
  if (int st = operand_check(what, "dy", dy, lddy, N)) return st;
  if (int st = operand_check(what, "x", x, ldx, K)) return st;
  if (int st = output_check(what, "dw", dw, lddw, K)) return st;
  if (int st = output_check(what, "dw's groups", dw, dw_stride, int64_t(N - 1) * lddw + K)) return st;
  const arcb::lin::Groups groups = {offsets, static_cast<uint32_t>(E), static_cast<uint32_t>(T)};
  return linear_dw(what, dy, x, groups, dw, N, K, lddy, ldx, lddw, dw_stride, stream);
}

}  // extern "C"
