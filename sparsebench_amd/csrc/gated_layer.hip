// The MoE layer with gated experts, forward and backward, one host call each:
// routing, the gated product, DSD and combine enqueued on one stream; for
// training the forward pass keeps what the backward pass reads.

#include "gated.hpp"
#include "workspace.hpp"

namespace sb {
namespace {

constexpr int64_t kBlock = kBS;

// The routing's own buffers hold routing_blocks row blocks (the padding of every
// expert). At most a row block a copy holds rows, the first ones, so that the
// products' rows and grids go by max_row_blocks (max_rows): with 3 tokens and 256
// experts 3 instead of 254.
struct Problem {
  int64_t num_tokens, num_experts, d_model, ffn_dim;
  int32_t k;
  int64_t num_copies, routing_blocks, max_row_blocks, max_rows, counts;
};

int check_problem(int64_t num_tokens, int32_t k, int32_t num_experts, int64_t d_model, int64_t ffn_dim, Problem* p) {
  if (num_tokens <= 0 || k <= 0 || num_tokens > (kI32Limit - 1) / k)
    return fail(SB_ERR_INVALID, "expert_idx must be [T, k] with T, k > 0");
  if (num_experts <= 0) return fail(SB_ERR_INVALID, "gated experts: bad expert count");
  if (d_model <= 0 || d_model % 128 != 0 || ffn_dim <= 0 || ffn_dim % 128 != 0 || d_model >= kI32Limit ||
      ffn_dim >= kI32Limit)
    return fail(SB_ERR_INVALID, "gated experts: D (%lld) and F (%lld) must be multiples of 128",
                static_cast<long long>(d_model), static_cast<long long>(ffn_dim));
  // A chunk's rows (320 at most) of [P, 2F] and [P, D], W1[e] and W2[e] are
  // read with 32-bit buffer offsets.
  if (std::max(d_model, 2 * ffn_dim) * (32 * kGatedRmax * 2) >= kI32Limit)
    return fail(SB_ERR_INVALID, "gated experts: D or F too large for 32-bit buffer offsets");
  if (d_model * ffn_dim * 4 >= kI32Limit)
    return fail(SB_ERR_INVALID, "gated experts: one expert's weights too large for 32-bit buffer offsets");
  *p = Problem{num_tokens, num_experts, d_model, ffn_dim, k, num_tokens * k, 0, 0, 0, 0};
  if (int rc = sb_routing_sizes(p->num_copies, num_experts, static_cast<int32_t>(ffn_dim),
                                static_cast<int32_t>(kBlock), &p->routing_blocks, nullptr, &p->counts))
    return rc;
  p->max_row_blocks = std::min(p->routing_blocks, p->num_copies);
  p->max_rows = p->max_row_blocks * kBlock;
  if (p->max_row_blocks * (std::max(d_model, 2 * ffn_dim) / 128) >= kI32Limit || p->max_rows * (d_model / 8) >= kI32Limit)
    return fail(SB_ERR_INVALID, "problem too large");
  return SB_OK;
}

struct RoutingBuffers {
  int32_t *tokens_per_expert, *padded_offsets, *row_token, *copy_row, *row_block_expert, *row_offsets, *col_indices,
      *error;
};

RoutingBuffers carve_routing(Carver& ws, const Problem& p) {
  RoutingBuffers b;
  b.tokens_per_expert = ws.take<int32_t>(p.num_experts);
  b.padded_offsets = ws.take<int32_t>(p.num_experts + 1);
  b.row_token = ws.take<int32_t>(p.routing_blocks * kBlock);
  b.copy_row = ws.take<int32_t>(p.num_copies);
  b.row_block_expert = ws.take<int32_t>(p.routing_blocks);
  b.row_offsets = ws.take<int32_t>(p.routing_blocks + 1);
  b.col_indices = ws.take<int32_t>(p.routing_blocks * (p.ffn_dim / kBlock));
  b.error = ws.take<int32_t>(1);
  return b;
}

GatedLayout layout_of(const RoutingBuffers& r, const Problem& p) {
  return {r.row_token, r.row_block_expert, r.tokens_per_expert, r.padded_offsets,
          static_cast<int32_t>(p.num_experts), static_cast<int32_t>(p.max_row_blocks)};
}

// What sb_gated_train leaves for sb_gated_backward.
struct SavedBuffers {
  RoutingBuffers routing;
  uint16_t *gu, *y;
};

SavedBuffers carve_saved(Carver& ws, const Problem& p) {
  SavedBuffers b;
  b.routing = carve_routing(ws, p);
  b.gu = ws.take<uint16_t>(p.max_rows * 2 * p.ffn_dim);
  b.y = ws.take<uint16_t>(p.max_rows * p.d_model);
  return b;
}

// A split product's parts, if it is split.
float* take_parts(Carver& ws, const Problem& p, int64_t columns, int64_t k) {
  const GatedForm form = gated_form(p.max_row_blocks, p.num_experts, p.num_copies, columns, k, true);
  return ws.take<float>(form.parts > 1 ? form.parts * p.max_rows * columns : 0);
}

struct TrainBuffers {
  int32_t* counts;
  uint16_t* h;
  float* partial;
};

TrainBuffers carve_train(Carver& ws, const Problem& p) {
  TrainBuffers b;
  b.counts = ws.take<int32_t>(p.counts);
  b.h = ws.take<uint16_t>(p.max_rows * p.ffn_dim);
  b.partial = take_parts(ws, p, p.d_model, p.ffn_dim);
  return b;
}

struct LayerBuffers {
  RoutingBuffers routing;
  TrainBuffers train;
  uint16_t* y;
};

LayerBuffers carve_layer(Carver& ws, const Problem& p) {
  LayerBuffers b;
  b.routing = carve_routing(ws, p);
  b.train = carve_train(ws, p);
  b.y = ws.take<uint16_t>(p.max_rows * p.d_model);
  return b;
}

struct BackwardBuffers {
  float *row_gate, *partial;
  int32_t* expert_order;
  uint16_t *xg, *gog, *grad_gu, *wh, *dxr;
};

BackwardBuffers carve_backward(Carver& ws, const Problem& p) {
  BackwardBuffers b;
  b.row_gate = ws.take<float>(p.max_rows);
  b.expert_order = ws.take<int32_t>(p.num_experts);
  b.xg = ws.take<uint16_t>(p.max_rows * p.d_model);
  b.gog = ws.take<uint16_t>(p.max_rows * p.d_model);
  b.grad_gu = ws.take<uint16_t>(p.max_rows * 2 * p.ffn_dim);
  b.wh = ws.take<uint16_t>(p.max_rows * p.ffn_dim);
  b.dxr = ws.take<uint16_t>(p.max_rows * p.d_model);
  b.partial = take_parts(ws, p, p.d_model, 2 * p.ffn_dim);
  return b;
}

int check_operands(std::initializer_list<const void*> wide, std::initializer_list<const void*> others,
                   int32_t gate_dtype, int32_t act) {
  for (const void* p : wide) {
    if (!p) return fail(SB_ERR_INVALID, "gated experts: null buffer");
    if (!aligned16(p))
      return fail(SB_ERR_INVALID, "gated experts: activations, weights and gradients must be 16-byte aligned");
  }
  for (const void* p : others)
    if (!p) return fail(SB_ERR_INVALID, "gated experts: null buffer");
  if (gate_dtype != SB_DTYPE_BF16 && gate_dtype != SB_DTYPE_F16 && gate_dtype != SB_DTYPE_F32)
    return fail(SB_ERR_INVALID, "gated experts: unsupported gate dtype code %d", gate_dtype);
  if (act != SB_ACT_SILU && act != SB_ACT_GELU)
    return fail(SB_ERR_INVALID, "gated experts: unknown activation code %d", act);
  return SB_OK;
}

// Routing, G | U (kept when gu is given), H, y = H W2, combine.
int run_forward(const Problem& p, const RoutingBuffers& r, const TrainBuffers& t, uint16_t* gu, uint16_t* y,
                const void* x, const void* expert_idx, int32_t idx_is_i64, const void* gates, int32_t gate_dtype,
                const void* w1, const void* w2, void* out, int32_t act, const int32_t* valid_tokens, void* stream) {
  if (int rc = sb_routing(expert_idx, idx_is_i64, p.num_tokens, p.k, static_cast<int32_t>(p.num_experts),
                          static_cast<int32_t>(p.ffn_dim), static_cast<int32_t>(kBlock), valid_tokens, t.counts,
                          r.tokens_per_expert, r.padded_offsets, r.row_token, r.copy_row, r.row_block_expert,
                          r.row_offsets, r.col_indices, r.error, stream))
    return rc;
  if (int rc = launch_gated_up(x, w1, layout_of(r, p), t.h, gu, p.num_tokens, p.num_copies, p.d_model, p.ffn_dim, act,
                               as_stream(stream)))
    return rc;
  // The layer's DSD kernel where it takes the shape and its tiles have the CUs.
  const GatedForm form = gated_form(p.max_row_blocks, p.num_experts, p.num_copies, p.d_model, p.ffn_dim, true);
  const bool layer_dsd = p.d_model % 256 == 0 && p.max_rows * p.ffn_dim * 2 < kI32Limit && form.parts == 1;
  const int rc =
      layer_dsd ? dsd_experts(t.h, w2, r.tokens_per_expert, r.padded_offsets, r.row_block_expert, r.row_offsets,
                              r.col_indices, y, p.max_row_blocks, p.num_experts, p.num_copies,
                              valid_tokens ? 0 : p.num_copies, p.ffn_dim, p.d_model, stream)
                : launch_gated_down(t.h, w2, layout_of(r, p), y, t.partial, p.num_copies, p.d_model, p.ffn_dim,
                                    as_stream(stream));
  if (rc) return rc;
  return sb_combine(y, r.copy_row, gates, gate_dtype, out, p.num_tokens, p.k, p.d_model, p.max_rows, valid_tokens,
                    stream);
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_gated_sizes(int64_t num_tokens, int32_t k, int32_t num_experts, int64_t d_model, int64_t ffn_dim,
                              int64_t* layer_bytes, int64_t* saved_bytes, int64_t* train_bytes,
                              int64_t* backward_bytes) {
  Problem p;
  if (int rc = check_problem(num_tokens, k, num_experts, d_model, ffn_dim, &p)) return rc;
  auto size = [&](auto carve, int64_t* to) {
    Carver ws{nullptr};
    carve(ws, p);
    if (to) *to = ws.used;
  };
  size(carve_layer, layer_bytes);
  if (layer_bytes && few_copies(num_tokens, k)) *layer_bytes = few_workspace_floats(p.num_copies, d_model, ffn_dim) * 4;
  size(carve_saved, saved_bytes);
  size(carve_train, train_bytes);
  size(carve_backward, backward_bytes);
  return clear_ok();
}

extern "C" int sb_gated_layer(const void* x, const void* expert_idx, int32_t idx_is_i64, const void* gates,
                              int32_t gate_dtype, const void* w1, const void* w2, void* out, int32_t act,
                              void* workspace, int64_t workspace_bytes, int64_t num_tokens, int32_t k,
                              int32_t num_experts, int64_t d_model, int64_t ffn_dim, const int32_t* valid_tokens,
                              void* stream) {
  Problem p;
  if (int rc = check_problem(num_tokens, k, num_experts, d_model, ffn_dim, &p)) return rc;
  if (int rc = check_operands({x, w1, w2, out}, {expert_idx, gates}, gate_dtype, act)) return rc;
  if (few_copies(num_tokens, k)) {
    if (int rc = check_workspace(workspace, workspace_bytes, few_workspace_floats(p.num_copies, d_model, ffn_dim) * 4))
      return rc;
    const int rc = launch_few(x, expert_idx, idx_is_i64, gates, gate_dtype, w1, w2, out, static_cast<float*>(workspace),
                              num_tokens, k, num_experts, d_model, ffn_dim, act, valid_tokens, as_stream(stream));
    return rc ? rc : clear_ok();
  }
  Carver ws{static_cast<uint8_t*>(workspace)};
  const LayerBuffers b = carve_layer(ws, p);
  if (int rc = check_workspace(workspace, workspace_bytes, ws.used)) return rc;
  return run_forward(p, b.routing, b.train, nullptr, b.y, x, expert_idx, idx_is_i64, gates, gate_dtype, w1, w2, out,
                     act, valid_tokens, stream);
}

extern "C" int sb_gated_train(const void* x, const void* expert_idx, int32_t idx_is_i64, const void* gates,
                              int32_t gate_dtype, const void* w1, const void* w2, void* out, int32_t act, void* saved,
                              int64_t saved_bytes, void* workspace, int64_t workspace_bytes, int64_t num_tokens,
                              int32_t k, int32_t num_experts, int64_t d_model, int64_t ffn_dim,
                              const int32_t* valid_tokens, void* stream) {
  Problem p;
  if (int rc = check_problem(num_tokens, k, num_experts, d_model, ffn_dim, &p)) return rc;
  if (int rc = check_operands({x, w1, w2, out}, {expert_idx, gates}, gate_dtype, act)) return rc;
  Carver kept{static_cast<uint8_t*>(saved)}, ws{static_cast<uint8_t*>(workspace)};
  const SavedBuffers s = carve_saved(kept, p);
  const TrainBuffers t = carve_train(ws, p);
  if (int rc = check_workspace(saved, saved_bytes, kept.used)) return rc;
  if (int rc = check_workspace(workspace, workspace_bytes, ws.used)) return rc;
  return run_forward(p, s.routing, t, s.gu, s.y, x, expert_idx, idx_is_i64, gates, gate_dtype, w1, w2, out, act,
                     valid_tokens, stream);
}

extern "C" int sb_gated_backward(const void* grad_out, const void* x, const void* gates, int32_t gate_dtype,
                                 const void* w1, const void* w2, const void* saved, int64_t saved_bytes, void* grad_x,
                                 void* grad_gates, void* grad_w1, void* grad_w2, int32_t act, void* workspace,
                                 int64_t workspace_bytes, int64_t num_tokens, int32_t k, int32_t num_experts,
                                 int64_t d_model, int64_t ffn_dim, const int32_t* valid_tokens, void* stream) {
  Problem p;
  if (int rc = check_problem(num_tokens, k, num_experts, d_model, ffn_dim, &p)) return rc;
  if (int rc = check_operands({grad_out, x, w1, w2, grad_x, grad_w1, grad_w2}, {gates, grad_gates}, gate_dtype, act))
    return rc;
  Carver kept{static_cast<uint8_t*>(const_cast<void*>(saved))}, ws{static_cast<uint8_t*>(workspace)};
  const SavedBuffers s = carve_saved(kept, p);
  const BackwardBuffers b = carve_backward(ws, p);
  if (int rc = check_workspace(saved, saved_bytes, kept.used)) return rc;
  if (int rc = check_workspace(workspace, workspace_bytes, ws.used)) return rc;
  const GatedLayout l = layout_of(s.routing, p);
  const hipStream_t st = as_stream(stream);
  if (int rc = launch_grad_rows(x, grad_out, s.y, l, s.routing.copy_row, gates, gate_dtype, grad_gates, b.row_gate, b.xg,
                                b.gog, p.num_tokens, k, d_model, b.expert_order, valid_tokens, st))
    return rc;
  if (int rc = launch_gated_slope(b.gog, w2, s.gu, b.row_gate, l, b.grad_gu, b.wh, p.num_copies, d_model, ffn_dim, act,
                                  st))
    return rc;
  if (int rc = launch_rows_bt(b.grad_gu, w1, l, b.dxr, b.partial, p.num_copies, d_model, 2 * ffn_dim, st)) return rc;
  if (int rc = launch_sum_copies(b.dxr, s.routing.copy_row, grad_x, p.num_tokens, k, d_model, p.max_rows, valid_tokens,
                                 st))
    return rc;
  if (int rc = launch_expert_outers(b.xg, b.grad_gu, grad_w1, d_model, 2 * ffn_dim, b.wh, b.gog, grad_w2, ffn_dim,
                                    d_model, l, b.expert_order, st))
    return rc;
  return clear_ok();
}
