// api_experts.cuh — host side of the expert layer: argument checks, the choice of the
// tiles, launches. Included by api.cu, whose helpers it uses.
#pragma once

#include "api_linear.cuh"
#include "expert_layer.cuh"

namespace {

namespace EX = arcb::experts;

// The kernels by weights and columns of a pass. Tiles (blocks of 16 rows x row groups) as measured best, 4096 x 2048
// experts, microseconds: bf16 16 tokens of 64 experts (8 columns) 2x2 334, 2x1 389, 4x2 366; 64 tokens (16 columns)
// 2x4 both 495, 2x2 both 512; 128 tokens (32 columns) 2x4 and 2x2 659, 2x2 both 699; int4, one token (8 columns)
// 4x2 31, 2x2 41, 32 tokens 4x2 189, 2x2 248; 64 tokens (16 columns) 2x4 and 2x2 308, 2x2 both 321, 128 tokens 533 and 552.
using ExpertKernel = void (*)(EX::Params);
struct ExpertVariant {
  ExpertKernel kernel;
  uint32_t rows, parts, stage_bytes, weight_bytes, sum_bytes;
};
template <uint32_t NT, uint32_t MR, uint32_t WR, bool INT4, bool SECOND>
constexpr ExpertVariant expert_variant() {
  using C = EX::Cfg<NT, MR, WR, INT4>;
  return {EX::expert_layer_kernel<NT, MR, WR, INT4, SECOND>, C::kRows, C::kParts, C::kStageBytes, C::kWBytes, C::kSumBytes};
}
struct ExpertForm {
  bool int4;
  uint32_t columns;
  ExpertVariant first, second;
  ExpertVariant second_narrow;  // where the second's sums of all tokens do not fit
};
constexpr ExpertForm kExpertForms[] = {
    {false, 8, expert_variant<8, 2, 2, false, false>(), expert_variant<8, 2, 2, false, true>(),
     expert_variant<8, 2, 2, false, true>()},
    {false, 16, expert_variant<16, 2, 4, false, false>(), expert_variant<16, 2, 4, false, true>(),
     expert_variant<16, 2, 2, false, true>()},
    {false, 32, expert_variant<32, 2, 4, false, false>(), expert_variant<32, 2, 2, false, true>(),
     expert_variant<32, 2, 2, false, true>()},
    {true, 8, expert_variant<8, 4, 2, true, false>(), expert_variant<8, 4, 2, true, true>(),
     expert_variant<8, 2, 2, true, true>()},
    {true, 16, expert_variant<16, 2, 4, true, false>(), expert_variant<16, 2, 2, true, true>(),
     expert_variant<16, 2, 2, true, true>()},
};

// Dynamic shared memory of a block: what the system and the kernel's own barriers take is off.
constexpr uint32_t kExpertSmemHalf = 112 * 1024, kExpertSmemWhole = 226 * 1024;

int experts_init() {
  for (const ExpertForm& f : kExpertForms) {
    for (const ExpertVariant* v : {&f.first, &f.second, &f.second_narrow}) {
      const cudaError_t e = allow_smem(v->kernel, kExpertSmemWhole);
      if (e != cudaSuccess) {
        cudaGetLastError();  // clear
        return cuda_fail(e, "cudaFuncSetAttribute (expert layer)");
      }
    }
  }
  return ARC_OK;
}

// How a call runs: columns of a pass, blocks of a cluster of the second launch (0: as many as fit), and whether the
// rows of x are put in the sorted order first.
struct ExpertPlan {
  const ExpertForm* form;
  uint32_t splits;
  bool sorted;
};

// An expert's choices fill a pass on average half: they are uneven, and a second pass reads the weights again, while
// columns that stay empty cost shared memory. int4 weights stop at 16: the registers of 32 do not fit. Sorted rows
// pay from 8 choices an expert (8 experts of 4096 x 7168, two a token, 64 tokens: 333 us with gathers, 293 sorted; 32 tokens, 8 choices
// an expert, 277 and 274, int4 153 and 138; 64 experts of 4096 x 2048, 16 tokens of two choices an expert: 338 and 337). A
// layer of small experts loses the launch in front (32 experts of 2048 x 1024, 64 tokens: 101 and 104), and int4 would gain
// earlier (32 tokens, four choices an expert: 189 and 182).
//
// ARC_EXPERT_PLAN="columns:S:sorted" (tests and tuning) forces them.
int expert_plan(bool int4, uint32_t tokens, uint32_t slots, uint32_t experts, ExpertPlan* plan) {
  const uint32_t live = experts < slots ? experts : slots;
  uint32_t want = 2 * ceil_div(slots, live);
  if (want > tokens) want = tokens;
  uint32_t columns = want <= 8 ? 8 : want <= 16 || int4 ? 16 : 32, sorted = slots >= 8 * experts ? 1 : 0;
  plan->splits = 0;
  if (const char* env = getenv("ARC_EXPERT_PLAN")) {
    uint32_t s = 0;
    if (sscanf(env, "%u:%u:%u", &columns, &s, &sorted) != 3 || (s != 1 && s != 2 && s != 4 && s != 8) || sorted > 1) {
      return fail(ARC_ERR_INVALID_ARGUMENT, "ARC_EXPERT_PLAN must be 'columns:S:sorted' (got '%s')", env);
    }
    plan->splits = s;
  }
  plan->sorted = sorted != 0;
  for (const ExpertForm& f : kExpertForms) {
    plan->form = &f;
    if (f.int4 == int4 && f.columns == columns) return ARC_OK;
  }
  return fail(ARC_ERR_INVALID_ARGUMENT, "the expert layer has no form of %u columns", columns);
}

// The ring of a launch: as many stages as half an SM holds if that keeps 32 KB of weights in flight, else as many as
// a whole one does. In the second launch every part of the contraction has its own sums of y where they take 32 KB
// at most.
struct ExpertRing {
  uint32_t stages, smem, blocks_per_sm;
  bool own_y;
};
bool expert_ring(const ExpertVariant& v, bool second, uint32_t columns, uint32_t tokens, uint32_t slots, uint32_t experts,
                 ExpertRing* ring) {
  ring->own_y = second && v.parts * v.rows * tokens * 4 <= 32 * 1024;
  const uint32_t rest =
      EX::layout_of(v.sum_bytes, v.parts, v.rows, columns, tokens, slots, experts, second, ring->own_y).total + 1024;
  // A whole number of parts and of batches, so that a stage always has the same waiters: by its parity a wait tells a phase only from
  // the one before, and whoever skipped a phase may take an older one for its own.
  const uint32_t unit = v.parts < 4 ? 4 : v.parts;
  const auto stages = [&](uint32_t budget) {
    const uint32_t n = budget > rest ? (budget - rest) / v.stage_bytes : 0;
    return (n < EX::kMaxStages ? n : EX::kMaxStages) / unit * unit;
  };
  ring->blocks_per_sm = 2;
  ring->stages = stages(kExpertSmemHalf);
  if (ring->stages * v.weight_bytes < 32 * 1024) {
    ring->blocks_per_sm = 1;
    ring->stages = stages(kExpertSmemWhole);
  }
  ring->smem = rest + ring->stages * v.stage_bytes;
  return ring->stages > 0;
}

// Weights of E experts as {bytes or elements of a row, rows, 2 (gate and up) or 1, E}.
int encode_expert_weights(CUtensorMap* map, const void* w, bool int4, uint64_t inner, uint64_t cols, bool gated,
                          uint64_t experts, uint64_t ld_bytes, uint64_t stride_bytes, uint32_t rows) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return fail(ARC_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[4] = {inner, cols, gated ? 2u : 1u, experts};
  const cuuint64_t strides[3] = {ld_bytes, ld_bytes * cols, experts > 1 ? stride_bytes : ld_bytes * cols};
  const cuuint32_t box[4] = {64, gated ? rows / 2 : rows, gated ? 2u : 1u, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, int4 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                        const_cast<void*>(w), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        int4 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    return fail(ARC_ERR_CUDA, "cuTensorMapEncodeTiled(expert weights) failed with CUresult %d", static_cast<int>(r));
  }
  return ARC_OK;
}

// h, and the sorted rows of x, lie in the workspace with rows that TMA can read.
uint64_t expert_ld(uint32_t inner) { return (uint64_t(inner) + 7) / 8 * 8; }
size_t expert_workspace(size_t slots, uint32_t inner_in, uint32_t inner_out, bool sorted) {
  return slots * 2 * (expert_ld(inner_out) + (sorted ? expert_ld(inner_in) : 0));
}

}  // namespace

extern "C" {

int arc_moe_workspace_bytes(int T, int top, int E, int K, int I, size_t* bytes) {
  if (bytes == nullptr || T <= 0 || top <= 0 || E <= 0 || K <= 0 || I <= 0 ||
      T > ARC_MOE_MAX_TOKENS || int64_t(T) * top > ARC_MOE_MAX_CHOICES) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "arc_moe_workspace_bytes: bad argument");
  }
  ExpertPlan plan;
  if (int st = expert_plan(false, T, static_cast<uint32_t>(T) * top, E, &plan)) return st;
  *bytes = expert_workspace(size_t(T) * top, K, I, plan.sorted);
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
  // (The kernel counts a block's boxes in 32 bits.)
  if (K > ARC_MOE_MAX_WIDTH || I > ARC_MOE_MAX_WIDTH || N > ARC_MOE_MAX_WIDTH) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: K, I and N are at most %d (got %d, %d, %d)", what, ARC_MOE_MAX_WIDTH, K, I, N);
  }
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
  const uint64_t ldh = expert_ld(I);
  ExpertPlan plan;
  if (int st = expert_plan(int4, T, slots, E, &plan)) return st;
  const size_t need = expert_workspace(slots, K, I, plan.sorted);
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need) {
    return fail(ARC_ERR_INVALID_ARGUMENT, "%s: needs a 16-byte aligned workspace of %zu bytes", what, need);
  }
  const ExpertVariant& v1 = plan.form->first;
  const uint32_t columns = plan.form->columns;
  ExpertRing first, second;
  const bool narrow = !expert_ring(plan.form->second, true, columns, T, slots, E, &second);
  const ExpertVariant& v2 = narrow ? plan.form->second_narrow : plan.form->second;
  if ((narrow && !expert_ring(v2, true, columns, T, slots, E, &second)) ||
      !expert_ring(v1, false, columns, T, slots, E, &first)) {
    return fail(ARC_ERR_UNSUPPORTED, "%s: does not fit in shared memory", what);  // no sizes within the limits get here
  }
  int dev = 0;
  if (int st = current_device(&dev, &DeviceState::experts_status)) return st;
  const uint32_t sms = static_cast<uint32_t>(g_dev[dev].sms);

  EX::Params p = {};
  p.ids = ids;
  p.weights = weights;
  p.ids_wide = id_bytes == 8;
  p.weights_bf16 = weight_bytes == 2;
  p.tokens = T;
  p.top = top;
  p.sorted = plan.sorted ? 1 : 0;
  p.top_inverse = top == 1 ? 0 : static_cast<uint32_t>(((1ull << 32) + top - 1) / top);
  p.experts = E;
  p.slots = slots;
  const uint32_t elem = int4 ? 1 : 2;

  // FIRST: h [slots][I].
  const uint32_t box_k = int4 ? group : 64;
  if (int st = encode_expert_weights(&p.tm_w, w_in, int4, int4 ? K / 2 : K, I, gated, E, ld_in * elem, stride_in * elem, v1.rows)) {
    return st;
  }
  cudaError_t e;
  if (p.sorted) {
    uint16_t* xs = static_cast<uint16_t*>(workspace) + slots * ldh;
    const uint64_t ldxs = expert_ld(K);
    const uint32_t smem = EX::layout_of(0, 1, 0, columns, T, slots, E, false, true).total + EX::sort_scratch(E);
    e = launch_grid(columns == 8    ? EX::expert_rows_kernel<8>
                    : columns == 16 ? EX::expert_rows_kernel<16>
                                    : EX::expert_rows_kernel<32>,
                    dim3(slots < sms ? slots : sms), EX::kThreads, smem, stream, p, xs, ldxs, x, ldx, uint32_t(K));
    if (e != cudaSuccess) return cuda_fail(e, "expert_rows_kernel launch");
    if (int st = encode_2d(&p.tm_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, xs, K, slots, ldxs, 64, 8,
                           CU_TENSOR_MAP_SWIZZLE_128B, "sorted x")) {
      return st;
    }
  } else if (int st = encode_2d(&p.tm_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x, K, T, ldx, 64, 1,
                                CU_TENSOR_MAP_SWIZZLE_128B, "x")) {
    return st;
  }
  p.sb = s_in;
  p.out = static_cast<uint16_t*>(workspace);
  p.ldo = ldh;
  p.cols = I;
  p.tiles = ceil_div(I, gated ? v1.rows / 2 : v1.rows);
  p.num_kb = ceil_div(K, box_k);
  p.groups = K / group;
  p.gated = gated ? 1 : 0;
  p.act = activation;
  p.stages = first.stages;
  p.splits = 1;
  const uint64_t items = uint64_t((uint32_t(E) < slots ? E : slots) + slots / columns) * p.tiles;
  const uint64_t most = uint64_t(sms) * first.blocks_per_sm;
  e = launch_ex(v1.kernel, p, static_cast<uint32_t>(items < most ? items : most), EX::kThreads, first.smem, 1, stream);
  if (e != cudaSuccess) return cuda_fail(e, "expert_layer_kernel launch");

  // SECOND: y [T][N].
  if (int st = encode_expert_weights(&p.tm_w, w_out, int4, int4 ? I / 2 : I, N, false, E, ld_out * elem, stride_out * elem, v2.rows)) {
    return st;
  }
  if (int st = encode_2d(&p.tm_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, workspace, I, slots, ldh, 64, 8,
                         CU_TENSOR_MAP_SWIZZLE_128B, "h")) {
    return st;
  }
  p.sb = s_out;
  p.out = out;
  p.ldo = ldo;
  p.cols = N;
  p.tiles = ceil_div(N, v2.rows);
  p.num_kb = ceil_div(I, box_k);
  p.groups = I / group;
  p.gated = 0;
  p.act = ARC_ACT_NONE;
  p.stages = second.stages;
  // The cluster shares a tile's boxes until both block slots of every SM have work.
  uint32_t splits = plan.splits;
  if (splits == 0) {
    splits = 1;
    while (splits < 8 && p.tiles * splits * 2 <= sms * second.blocks_per_sm) splits *= 2;
  }
  p.splits = splits;
  p.own_y = second.own_y ? 1 : 0;
  e = launch_ex(v2.kernel, p, p.tiles * splits, EX::kThreads, second.smem, splits, stream);
  if (e != cudaSuccess) return cuda_fail(e, "expert_layer_kernel launch");
  return ARC_OK;
}

}  // extern "C"
