// A routed (mixture of experts) MLP block with 4-bit weights (no counterpart
// in megacu): the routing and 4-bit entry points called in a row on one
// workspace.
//   sort -> quantise the tokens' rows, to their experts -> act = silu(gate) * up by
//   expert -> quantise act -> down by expert -> weighted sum back
#include <cuda_runtime.h>

#include <cstdint>

#include <megacu_b200.h>

#include "status.h"

namespace {

using namespace megacu_b200;

constexpr std::int32_t kAlign = 128;  // rows of a product's tile

// Byte offsets of the workspace's parts, each 256-byte aligned.
struct mlp_layout {
  std::int64_t counts, offsets, row_of_slot, slot_of_row, sort, x_data, x_scales, act, act_data,
      act_scales, rows, total;
  std::int64_t capacity;  // rows of the sorted order
};

megacu_moe_problem routing(megacu_moe_mlp_problem const &p) {
  megacu_moe_problem r{};
  r.tokens = p.tokens;
  r.hidden = p.hidden;
  r.topk = p.topk;
  r.experts = p.experts;
  r.first_expert = p.first_expert;
  r.align = kAlign;
  r.dtype = p.dtype;
  r.id_bytes = p.id_bytes;
  return r;
}

megacu_fp4_matrix matrix(megacu_moe_mlp_problem const &p, std::int64_t rows, std::int64_t cols,
                         float scale) {
  megacu_fp4_matrix m{};
  m.rows = rows;
  m.cols = cols;
  m.format = p.format;
  m.dtype = p.dtype;
  m.scale = scale != 0.0f ? scale : 1.0f;
  return m;
}

megacu_fp4_gemm_problem product(megacu_moe_mlp_problem const &p, std::int64_t rows, std::int64_t n,
                                std::int64_t k, float alpha) {
  megacu_fp4_gemm_problem g{};
  g.m = rows;
  g.n = n;
  g.k = k;
  g.format = p.format;
  g.out_dtype = p.dtype;
  g.experts = p.experts;
  g.alpha = alpha;
  g.timeout_ns = p.timeout_ns;
  return g;
}

megacu_status make_layout(megacu_moe_mlp_problem const &p, mlp_layout &out) {
  if (p.inter < 1) return fail(MEGACU_INVALID_ARGUMENT, 1, "invalid problem");
  megacu_moe_problem const r = routing(p);
  std::int64_t sort[2] = {};
  megacu_status st = megacu_b200_moe_sizes(&r, sort);
  if (st.code != MEGACU_OK) return st;
  megacu_fp4_matrix const x = matrix(p, sort[0], p.hidden, p.x_scale);
  megacu_fp4_matrix const act = matrix(p, sort[0], p.inter, p.act_scale);
  std::int64_t xs[2] = {}, as[2] = {};
  st = megacu_b200_fp4_sizes(&x, xs);
  if (st.code == MEGACU_OK) st = megacu_b200_fp4_sizes(&act, as);
  if (st.code != MEGACU_OK) return st;
  std::int64_t const size = p.dtype == MEGACU_DTYPE_F32 ? 4 : 2;
  std::int64_t at = 0;
  auto take = [&at](std::int64_t bytes) {
    std::int64_t const here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  out.capacity = sort[0];
  out.counts = take(4 * static_cast<std::int64_t>(p.experts));
  out.offsets = take(4 * (static_cast<std::int64_t>(p.experts) + 1));
  out.row_of_slot = take(4 * p.tokens * p.topk);
  out.slot_of_row = take(4 * sort[0]);
  out.sort = take(sort[1]);
  out.x_data = take(xs[0]);
  out.x_scales = take(xs[1]);
  out.act = take(sort[0] * p.inter * size);
  out.act_data = take(as[0]);
  out.act_scales = take(as[1]);
  out.rows = take(sort[0] * p.hidden * size);
  out.total = at;
  return ok_status();
}

}  // namespace

extern "C" megacu_status megacu_b200_moe_mlp_workspace_bytes(megacu_moe_mlp_problem const *problem,
                                                             std::int64_t *bytes) {
  if (problem == nullptr || bytes == nullptr) {
    return fail(MEGACU_INVALID_ARGUMENT, 2, "missing problem or output");
  }
  mlp_layout l{};
  megacu_status const st = make_layout(*problem, l);
  if (st.code == MEGACU_OK) *bytes = l.total;
  return st;
}

extern "C" megacu_status megacu_cuda_moe_mlp_fp4(
    megacu_driver_view driver, void const *x, void const *expert_ids, void const *weights,
    void const *gate, void const *gate_scales, void const *up, void const *up_scales,
    void const *down, void const *down_scales, void const *up_alphas, void const *down_alphas,
    void *y, void *workspace, void *events, megacu_moe_mlp_problem const *problem) {
  if (problem == nullptr) return fail(MEGACU_INVALID_ARGUMENT, 2, "missing problem");
  megacu_moe_mlp_problem const &p = *problem;
  mlp_layout l{};
  megacu_status st = make_layout(p, l);
  if (st.code != MEGACU_OK) return st;
  if (p.tokens == 0) return ok_status();
  if (workspace == nullptr || weights == nullptr || x == nullptr || y == nullptr) {
    return fail(MEGACU_INVALID_ARGUMENT, 2, "missing storage");
  }
  if (!aligned_to(workspace, 256)) {
    return fail(MEGACU_INVALID_ARGUMENT, 21, "the workspace must be 256-byte aligned");
  }
  auto *const base = static_cast<char *>(workspace);
  auto part = [base](std::int64_t offset) -> void * { return base + offset; };

  megacu_moe_problem const route = routing(p);
  megacu_fp4_matrix x_matrix = matrix(p, l.capacity, p.hidden, p.x_scale);
  x_matrix.topk = p.topk;
  x_matrix.x_rows = p.tokens;
  x_matrix.scatter = 1;
  megacu_fp4_matrix const act_matrix = matrix(p, l.capacity, p.inter, p.act_scale);
  megacu_fp4_gemm_problem const gate_up =
      product(p, l.capacity, p.inter, p.hidden, p.up_alpha / x_matrix.scale);
  megacu_fp4_gemm_problem const project =
      product(p, l.capacity, p.hidden, p.inter, p.down_alpha / act_matrix.scale);

  // Everything is validated before anything is launched.
  megacu_driver_view check = driver;
  check.launch.stream = nullptr;
  for (megacu_driver_view const &d : {check, driver}) {
    st = megacu_cuda_moe_sort(d, expert_ids, part(l.counts), part(l.offsets), part(l.row_of_slot),
                              part(l.slot_of_row), part(l.sort), &route);
    if (st.code != MEGACU_OK) return st;
    st = megacu_cuda_fp4_quantize(d, x, part(l.row_of_slot), part(l.x_data), part(l.x_scales),
                                  &x_matrix);
    if (st.code != MEGACU_OK) return st;
    st = megacu_cuda_fp4_gemm_swiglu(d, part(l.x_data), part(l.x_scales), gate, gate_scales, up,
                                     up_scales, part(l.offsets), part(l.counts), up_alphas,
                                     part(l.act), events, &gate_up);
    if (st.code != MEGACU_OK) return st;
    st = megacu_cuda_fp4_quantize(d, part(l.act), part(l.slot_of_row), part(l.act_data),
                                  part(l.act_scales), &act_matrix);
    if (st.code != MEGACU_OK) return st;
    st = megacu_cuda_fp4_gemm(d, part(l.act_data), part(l.act_scales), down, down_scales,
                              part(l.offsets), part(l.counts), down_alphas, part(l.rows), events,
                              &project);
    if (st.code != MEGACU_OK) return st;
    st = megacu_cuda_moe_combine(d, part(l.rows), weights, part(l.row_of_slot), y, &route);
    if (st.code != MEGACU_OK || driver.launch.stream == nullptr) return st;
  }
  return ok_status();
}
