// api_experts.cuh — host side of the expert layer: argument checks, the choice of the
// tiles, launches. Included by api.cu, whose helpers it uses.
#pragma once

#include "api_linear.cuh"
#include "expert_layer.cuh"

namespace {

namespace EX = arcb::experts;

// The instantiations the plan can choose: columns of a pass, blocks of 16 rows and row groups of a tile.
#define ARC_EXPERT_VARIANTS(X) X(8, 2, 1) X(8, 2, 2) X(8, 4, 1) X(8, 4, 2) X(16, 2, 2) X(16, 2, 4) X(16, 4, 1) X(16, 4, 2) X(32, 2, 2) X(32, 2, 4)

using ExpertKernel = void (*)(EX::Params);

struct ExpertVariant {
  uint32_t nt, mr, wr;
  ExpertKernel kernel[2][2];  // [int4][second]
  uint32_t stage_bytes[2], sum_bytes, rows;
};
constexpr ExpertVariant kExpertVariants[] = {
#define ARC_EXPERT_ENTRY(NT, MR, WR)                                                                             \
  {NT,                                                                                                           \
   MR,                                                                                                           \
   WR,                                                                                                           \
   {{EX::expert_layer_kernel<NT, MR, WR, false, false>, EX::expert_layer_kernel<NT, MR, WR, false, true>},       \
    {EX::expert_layer_kernel<NT, MR, WR, true, false>, EX::expert_layer_kernel<NT, MR, WR, true, true>}},        \
   {EX::Cfg<NT, MR, WR, false>::kStageBytes, EX::Cfg<NT, MR, WR, true>::kStageBytes},                            \
   EX::Cfg<NT, MR, WR, false>::kSumBytes,                                                                        \
   EX::Cfg<NT, MR, WR, false>::kRows},
    ARC_EXPERT_VARIANTS(ARC_EXPERT_ENTRY)
#undef ARC_EXPERT_ENTRY
};

// Dynamic shared memory of a block: what the system and the kernel's own barriers take is off.
constexpr uint32_t kExpertSmemHalf = 112 * 1024, kExpertSmemWhole = 226 * 1024;

int experts_init() {
  for (const ExpertVariant& v : kExpertVariants) {
    for (int i = 0; i < 4; ++i) {
      const cudaError_t e = allow_smem(v.kernel[i >> 1][i & 1], kExpertSmemWhole);
      if (e != cudaSuccess) {
        cudaGetLastError();  // clear
        return cuda_fail(e, "cudaFuncSetAttribute (expert layer)");
      }
    }
  }
  return ARC_OK;
}

struct ExpertPlan {
  const ExpertVariant* v;
  uint32_t stages, smem, blocks_per_sm;
  bool own_y;
};

const ExpertVariant* expert_variant(uint32_t nt, uint32_t mr, uint32_t wr) {
  for (const ExpertVariant& v : kExpertVariants) {
    if (v.nt == nt && v.mr == mr && v.wr == wr) return &v;
  }
  return nullptr;
}

// The ring of a launch: as many stages as half an SM holds if that keeps 48 KB of weights in flight, else
// as many as a whole one does.
void expert_ring(const ExpertVariant& v, bool int4, bool second, uint32_t tokens, uint32_t slots, uint32_t experts,
                 ExpertPlan* plan) {
  const uint32_t parts = EX::kConsumers / v.wr;
  const uint32_t stage = v.stage_bytes[int4 ? 1 : 0];
  plan->v = &v;
  plan->own_y = second && parts * v.rows * tokens * 4 <= 32 * 1024;
  const uint32_t rest =
      EX::layout_of(v.sum_bytes, parts, v.rows, v.nt, tokens, slots, experts, second, plan->own_y).total + 1024;
  const uint32_t unit = parts < 4 ? 4 : parts;  // a whole number of parts and of batches
  const auto stages = [&](uint32_t budget) {
    const uint32_t n = budget > rest ? (budget - rest) / stage : 0;
    return (n < EX::kMaxStages ? n : EX::kMaxStages) / unit * unit;
  };
  plan->blocks_per_sm = 2;
  plan->stages = stages(kExpertSmemHalf);
  if (plan->stages * v.rows * EX::kRowBytes < 32 * 1024) {
    plan->blocks_per_sm = 1;
    plan->stages = stages(kExpertSmemWhole);
  }
  plan->smem = rest + plan->stages * stage;
}

// Weights of E experts as {bytes or elements of a row, rows, 2 (gate and up) or 1, E}.
int encode_expert_weights(CUtensorMap* map, const void* w, bool int4, uint64_t inner, uint64_t cols, bool gated,
                          uint64_t experts, uint64_t ld_bytes, uint64_t stride_bytes, uint32_t rows) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return fail(ARC_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[4] = {inner, cols, gated ? 2u : 1u, experts};
  const cuuint64_t strides[3] = {ld_bytes, ld_bytes * cols, experts > 1 ? stride_bytes : ld_bytes * cols};
  const cuuint32_t box[4] = {int4 ? EX::kRowBytes : EX::kRowBytes / 2, gated ? rows / 2 : rows, gated ? 2u : 1u, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, int4 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                        const_cast<void*>(w), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    return fail(ARC_ERR_CUDA, "cuTensorMapEncodeTiled(expert weights) failed with CUresult %d", static_cast<int>(r));
  }
  return ARC_OK;
}

// Columns of a pass: those that an expert's choices fill on average, doubled, since they are uneven.
uint32_t expert_columns(uint32_t tokens, uint32_t slots, uint32_t experts) {
  const uint32_t live = experts < slots ? experts : slots;
  uint32_t want = 2 * ceil_div(slots, live);
  if (want > tokens) want = tokens;
  return want <= 8 ? 8 : want <= 16 ? 16 : 32;
}

// h lies in the workspace with rows that TMA can read.
uint64_t expert_ldh(uint32_t inner) { return (uint64_t(inner) + 7) / 8 * 8; }

}  // namespace

extern "C" {

int arc_moe_workspace_bytes(int T, int top, int I, size_t* bytes) {
  if (bytes == nullptr || T <= 0 || top <= 0 || I <= 0) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "arc_moe_workspace_bytes: bad argument");
  }
  *bytes = size_t(T) * top * expert_ldh(I) * 2;
  return ARC_OK;
}

int arc_moe(const uint16_t* x, const void* w_in, const uint16_t* s_in, const void* w_out, const uint16_t* s_out,
                     const void* ids, int id_bytes, const void* weights, int weight_bytes, uint16_t* out, void* workspace,
                     size_t workspace_bytes, int T, int top, int E, int K, int I, int N, int64_t ldx, int64_t ld_in,
                     int64_t stride_in, int64_t ld_out, int64_t stride_out, int64_t ldo, int gated, int activation,
                     cudaStream_t stream) {
  const char* what = "arc_moe";
  g_last_error[0] = '\0';
  if (x == nullptr || w_in == nullptr || w_out == nullptr || ids == nullptr || weights == nullptr || out == nullptr ||
      (s_in == nullptr) != (s_out == nullptr)) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  }
  if (T <= 0 || top <= 0 || E <= 0 || K <= 0 || I <= 0 || N <= 0) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: sizes must be positive (T=%d top=%d E=%d K=%d I=%d N=%d)", what, T, top,
                E, K, I, N);
  }
  if (T > ARC_MOE_MAX_TOKENS || int64_t(T) * top > ARC_MOE_MAX_CHOICES) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: at most %d tokens and %d choices (got %d x %d)", what,
                ARC_MOE_MAX_TOKENS, ARC_MOE_MAX_CHOICES, T, top);
  }
  if (E > static_cast<int>(arcb::lin::kMaxGroups)) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: at most %u experts (got %d)", what, arcb::lin::kMaxGroups, E);
  }
  if (activation < ARC_ACT_NONE || activation > ARC_ACT_SILU) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", what, activation);
  }
  if ((id_bytes != 4 && id_bytes != 8) || (weight_bytes != 2 && weight_bytes != 4)) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: ids are 4- or 8-byte integers, weights bf16 or fp32 (got %d and %d bytes)", what,
                id_bytes, weight_bytes);
  }
  const bool int4 = s_in != nullptr;
  const uint32_t group = EX::kScaleGroup;
  if (int4 && (K % group != 0 || I % group != 0)) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: int4 weights need K and I to be multiples of %u (K=%d I=%d)", what, group, K, I);
  }
  if (K > (1 << 30) || I > (1 << 29) || N > (1 << 30)) return fail(ARC_ERR_UNSUPPORTED, "%s: sizes too large", what);
  const int rows_in = gated ? 2 * I : I;
  if (int st = operand_check(what, "x", x, ldx, K)) return st;
  if (int4) {
    if (!aligned16(w_in) || !aligned16(w_out) || (reinterpret_cast<uintptr_t>(s_in) & 1u) ||
        (reinterpret_cast<uintptr_t>(s_out) & 1u)) {
      return fail(ARC_ERR_UNSUPPORTED, "%s: packed weights must be 16-byte aligned", what);
    }
    ld_in = K / 2;
    stride_in = ld_in * rows_in;
    ld_out = I / 2;
    stride_out = ld_out * N;
  } else {
    if (int st = operand_check(what, "w_in", w_in, ld_in, K)) return st;
    if (int st = operand_check(what, "w_in's experts", w_in, stride_in, int64_t(rows_in - 1) * ld_in + K)) return st;
    if (int st = operand_check(what, "w_out", w_out, ld_out, I)) return st;
    if (int st = operand_check(what, "w_out's experts", w_out, stride_out, int64_t(N - 1) * ld_out + I)) return st;
  }
  if (int st = output_check(what, "out", out, ldo, N)) return st;
  if ((reinterpret_cast<uintptr_t>(ids) & (id_bytes - 1)) || (reinterpret_cast<uintptr_t>(weights) & (weight_bytes - 1))) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: ids or weights are misaligned", what);
  }
  const uint32_t slots = static_cast<uint32_t>(T) * top;
  const uint64_t ldh = expert_ldh(I);
  const size_t need = size_t(slots) * ldh * 2;
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: needs a 16-byte aligned workspace of %zu bytes", what, need);
  }
  int dev = 0;
  if (int st = current_device(&dev, &DeviceState::experts_status)) return st;
  const uint32_t sms = static_cast<uint32_t>(g_dev[dev].sms);

  uint32_t nt = expert_columns(T, slots, E), mr1 = int4 && nt < 32 ? 4 : 2, mr2 = mr1, splits = 0, per_sm = 2;
  uint32_t wr1 = nt == 8 ? 2 : 4 * 2 / mr1, wr2 = 2;
  if (const char* env = getenv("ARC_EXPERT_PLAN")) {
    if (sscanf(env, "%u:%u:%u:%u:%u:%u:%u", &nt, &mr1, &wr1, &mr2, &wr2, &splits, &per_sm) < 5 ||
        expert_variant(nt, mr1, wr1) == nullptr || expert_variant(nt, mr2, wr2) == nullptr ||
        (splits & (splits - 1)) != 0 || splits > 8) {
      return fail(ARC_ERR_INVALID_ARGUMENT, "ARC_EXPERT_PLAN must be 'NT:MR:WR:MR:WR[:S]' (got '%s')", env);
    }
  }
  ExpertPlan first, second;
  expert_ring(*expert_variant(nt, mr1, wr1), int4, false, T, slots, E, &first);
  expert_ring(*expert_variant(nt, mr2, wr2), int4, true, T, slots, E, &second);
  if (first.stages == 0 || second.stages == 0) return fail(ARC_ERR_UNSUPPORTED, "%s: does not fit in shared memory", what);

  EX::Params p = {};
  p.ids = ids;
  p.weights = weights;
  p.ids_wide = id_bytes == 8;
  p.weights_bf16 = weight_bytes == 2;
  p.tokens = T;
  p.top = top;
  p.top_inverse = top == 1 ? 0 : static_cast<uint32_t>(((1ull << 32) + top - 1) / top);
  p.experts = E;
  p.slots = slots;
  const uint32_t elem = int4 ? 1 : 2;

  // FIRST: h [slots][I].
  const uint32_t box_k = int4 ? 2 * EX::kRowBytes : EX::kRowBytes / 2;
  if (int st = encode_expert_weights(&p.tm_w, w_in, int4, int4 ? K / 2 : K, I, gated, E, ld_in * elem, stride_in * elem, first.v->rows)) {
    return st;
  }
  if (int st = encode_2d(&p.tm_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x, K, T, ldx, 64, 1, CU_TENSOR_MAP_SWIZZLE_128B, "x")) {
    return st;
  }
  p.sb = s_in;
  p.out = static_cast<uint16_t*>(workspace);
  p.ldo = ldh;
  p.cols = I;
  p.tiles = ceil_div(I, gated ? first.v->rows / 2 : first.v->rows);
  p.num_kb = ceil_div(K, box_k);
  p.groups = K / group;
  p.gated = gated ? 1 : 0;
  p.act = activation;
  p.stages = first.stages;
  p.splits = 1;
  const uint64_t items = uint64_t((uint32_t(E) < slots ? E : slots) + slots / nt) * p.tiles;
  const uint64_t most = uint64_t(sms) * (first.blocks_per_sm < per_sm ? first.blocks_per_sm : per_sm);
  cudaError_t e = launch_ex(first.v->kernel[int4][0], p, static_cast<uint32_t>(items < most ? items : most), EX::kThreads,
                            first.smem, 1, stream);
  if (e != cudaSuccess) return cuda_fail(e, "expert_layer_kernel launch");

  // SECOND: y [T][N].
  if (int st = encode_expert_weights(&p.tm_w, w_out, int4, int4 ? I / 2 : I, N, false, E, ld_out * elem, stride_out * elem, second.v->rows)) {
    return st;
  }
  if (int st = encode_2d(&p.tm_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, workspace, I, slots, ldh, 64, 1,
                         CU_TENSOR_MAP_SWIZZLE_128B, "h")) {
    return st;
  }
  p.sb = s_out;
  p.out = out;
  p.ldo = ldo;
  p.cols = N;
  p.tiles = ceil_div(N, second.v->rows);
  p.num_kb = ceil_div(I, box_k);
  p.groups = I / group;
  p.gated = 0;
  p.act = ARC_ACT_NONE;
  p.stages = second.stages;
  if (splits == 0) {
    splits = 1;
    while (splits < 8 && p.tiles * splits * 2 <= sms * second.blocks_per_sm) splits *= 2;
  }
  p.splits = splits;
  p.own_y = second.own_y ? 1 : 0;
  e = launch_ex(second.v->kernel[int4][1], p, p.tiles * splits, EX::kThreads, second.smem, splits, stream);
  if (e != cudaSuccess) return cuda_fail(e, "expert_layer_kernel launch");
  return ARC_OK;
}

}  // extern "C"
