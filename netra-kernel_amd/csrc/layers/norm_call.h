// C entry points of the norm (included by netra_layers.hip): argument checks, choice of kernels
// and launches.
#pragma once
#include "layers_call.h"
#include "layers_plan.h"
#include "norm.hip"

namespace {

uint64_t row_bytes(uint32_t cols, uint32_t type) { return static_cast<uint64_t>(cols) * elem(type); }
Span rows_span(const void* p, uint32_t type, uint64_t stride, uint32_t rows, uint32_t cols) {
  return {p, stride * elem(type), row_bytes(cols, type), p ? rows : 0u};
}
bool same(const Span& a, const Span& b) { return a.p == b.p && a.stride == b.stride && a.row == b.row; }

bool bad_norm(uint32_t rows, uint32_t cols) { return rows > kMaxSize || cols == 0 || cols > nknorm::kMaxCols; }
bool bad_weight(const void* w, uint32_t type) { return !w || bad_type(type) || !aligned(w, elem(type)); }

// The launch of one of the kernels by the types and the row's length.
#define NETRA_NORM_ONE(KERNEL, X, R, W, C)                                          \
  do {                                                                              \
    if (once) launch(KERNEL##_##X##_##R##_w##W##c##C##_once_gfx950, grid, block, a); \
    else launch(KERNEL##_##X##_##R##_w##W##c##C##_gfx950, grid, block, a);          \
  } while (0)
#define NETRA_NORM_TYPES(KERNEL, W, C)                                                               \
  do {                                                                                               \
    if (first == NETRA_BF16 && second == NETRA_BF16) NETRA_NORM_ONE(KERNEL, bf16, bf16, W, C);       \
    else if (first == NETRA_BF16) NETRA_NORM_ONE(KERNEL, bf16, f32, W, C);                           \
    else if (second == NETRA_BF16) NETRA_NORM_ONE(KERNEL, f32, bf16, W, C);                          \
    else NETRA_NORM_ONE(KERNEL, f32, f32, W, C);                                                     \
  } while (0)
#define NETRA_NORM_SHAPES(KERNEL)                                            \
  if (plan.waves == 1u && plan.chunks == 1u) NETRA_NORM_TYPES(KERNEL, 1, 1); \
  else if (plan.waves == 1u) NETRA_NORM_TYPES(KERNEL, 1, 2);                 \
  else if (plan.waves == 4u) NETRA_NORM_TYPES(KERNEL, 4, 1);                 \
  else if (plan.waves == 8u) NETRA_NORM_TYPES(KERNEL, 8, 1);                 \
  else if (plan.chunks == 1u) NETRA_NORM_TYPES(KERNEL, 16, 1);               \
  else NETRA_NORM_TYPES(KERNEL, 16, 2)

}  // namespace

extern "C" uint64_t netra_norm_code_bytes(uint32_t rows, uint32_t cols, uint32_t layout) {
  return layout == NETRA_CODES_TILES ? code_bytes(rows, cols) : static_cast<uint64_t>(rows) * cols;
}
extern "C" uint64_t netra_norm_scale_count(uint32_t rows, uint32_t cols, uint32_t layout) {
  return static_cast<uint64_t>(layout == NETRA_CODES_TILES ? up(rows, 16u) : rows) * blocks(cols);
}

extern "C" int netra_norm_forward(const void* x, uint32_t x_type, uint64_t x_stride, const void* residual,
                                  uint32_t residual_type, uint64_t residual_stride, const void* weight,
                                  uint32_t weight_type, float offset, float eps, void* sum, uint64_t sum_stride,
                                  void* y, uint32_t y_type, uint64_t y_stride, uint8_t* codes, float* scales,
                                  uint32_t layout, uint32_t rows, uint32_t cols, hipStream_t stream) {
  const char* name = "netra_norm_forward";
  if (bad_norm(rows, cols)) return fail(-1, name, "rows have to be 0 .. 2^21, cols 1 .. 16384");
  if (!(eps >= 0.0f)) return fail(-1, name, "eps has to be 0 or more");
  if (rows == 0) {
    g_error.clear();
    return 0;
  }
  if (bad_matrix(x, x_type, x_stride, cols) || bad_weight(weight, weight_type) || !sum != !residual ||
      (residual && (bad_matrix(residual, residual_type, residual_stride, cols) ||
                    bad_matrix(sum, residual_type, sum_stride, cols))) ||
      (y && bad_matrix(y, y_type, y_stride, cols)))
    return fail(-1, name, "null or misaligned pointer, unknown type, or row stride below the row");
  if (!codes != !scales || (codes && layout != NETRA_CODES_ROWS && layout != NETRA_CODES_TILES) ||
      (codes && (!aligned(scales, 4) || (layout == NETRA_CODES_TILES && !aligned(codes, 16)))))
    return fail(-1, name, "codes and scales go together, aligned, in one of the two layouts");
  if (!codes && !y && !sum) return fail(-1, name, "no output");
  const uint64_t code_size = codes ? netra_norm_code_bytes(rows, cols, layout) : 0;
  const uint64_t scale_size = codes ? netra_norm_scale_count(rows, cols, layout) * 4u : 0;
  const Span in[] = {rows_span(x, x_type, x_stride, rows, cols),
                     rows_span(residual, residual_type, residual_stride, rows, cols),
                     {weight, row_bytes(cols, weight_type), row_bytes(cols, weight_type), 1}};
  const Span out[] = {rows_span(sum, residual_type, sum_stride, rows, cols), rows_span(y, y_type, y_stride, rows, cols),
                      {codes, code_size, code_size, codes ? 1u : 0u}, {scales, scale_size, scale_size, codes ? 1u : 0u}};
  for (int o = 0; o < 4; ++o) {
    for (int i = 0; i < 3; ++i)  // a row is read before it is written: in place is fine
      if (share(out[o], in[i]) && !(o < 2 && i < 2 && same(out[o], in[i])))
        return fail(-1, name, "an output shares memory with an input and is not in its place");
    for (int p = 0; p < o; ++p)
      if (share(out[o], out[p])) return fail(-1, name, "two outputs share memory");
  }
  nknorm::Norm a{};
  a.x = x;
  a.x_stride = x_stride;
  a.residual = residual;
  a.residual_stride = residual_stride;
  a.w = weight;
  a.w_bf16 = weight_type == NETRA_BF16;
  a.offset = offset;
  a.eps = eps;
  a.inv_cols = 1.0f / static_cast<float>(cols);
  a.sum = sum;
  a.sum_stride = sum_stride;
  a.y = y;
  a.y_bf16 = y_type == NETRA_BF16;
  a.y_stride = y_stride;
  a.codes = codes;
  a.scales = scales;
  a.layout = !codes ? nknorm::kNone : layout == NETRA_CODES_TILES ? nknorm::kTiles : nknorm::kRows;
  a.scales_ld = up(rows, 16u);
  a.rows = rows;
  a.cols = cols;
  a.all_rows = a.layout == nknorm::kTiles ? up(rows, 16u) : rows;
  const NormPlan plan = norm_plan(a.all_rows, cols);
  const uint32_t first = x_type, second = residual ? residual_type : x_type;
  const uint64_t row = row_bytes(cols, x_type) + (residual ? 2u * row_bytes(cols, residual_type) : 0u) +
                       (y ? row_bytes(cols, y_type) : 0u) + (codes ? cols : 0u);
  const bool once = row * rows > kInfinityCache;
  const dim3 grid(plan.groups), block(plan.threads);
  Launcher launch(stream);
  NETRA_NORM_SHAPES(netra_norm);
  return launch.result(name);
}

extern "C" uint64_t netra_norm_gradients_workspace(uint32_t rows, uint32_t cols) {
  if (rows == 0 || bad_norm(rows, cols)) return 0;
  const NormPlan plan = norm_gradients_plan(rows, cols);
  return 4u * static_cast<uint64_t>(plan.groups) * cols;
}

extern "C" int netra_norm_gradients(const void* dy, uint32_t dy_type, uint64_t dy_stride, const void* r, uint32_t r_type,
                                    uint64_t r_stride, const void* flow, uint64_t flow_stride, const void* weight,
                                    uint32_t weight_type, float offset, float eps, void* dr, uint64_t dr_stride,
                                    float* dw, uint32_t accumulate, uint32_t rows, uint32_t cols, void* workspace,
                                    uint64_t workspace_bytes, hipStream_t stream) {
  const char* name = "netra_norm_gradients";
  if (bad_norm(rows, cols)) return fail(-1, name, "rows have to be 0 .. 2^21, cols 1 .. 16384");
  if (!(eps >= 0.0f)) return fail(-1, name, "eps has to be 0 or more");
  if (bad_weight(weight, weight_type) || !dw || !aligned(dw, 4))
    return fail(-1, name, "null or misaligned pointer or unknown type");
  if (rows && (bad_matrix(dy, dy_type, dy_stride, cols) || bad_matrix(r, r_type, r_stride, cols) ||
               (flow && bad_matrix(flow, r_type, flow_stride, cols)) || bad_matrix(dr, r_type, dr_stride, cols)))
    return fail(-1, name, "null or misaligned pointer, unknown type, or row stride below the row");
  const Span in[] = {rows_span(dy, dy_type, dy_stride, rows, cols), rows_span(r, r_type, r_stride, rows, cols),
                     rows_span(flow, r_type, flow_stride, rows, cols),
                     {weight, row_bytes(cols, weight_type), row_bytes(cols, weight_type), 1}};
  const Span out[] = {rows_span(dr, r_type, dr_stride, rows, cols), {dw, cols * 4ull, cols * 4ull, 1}};
  for (int i = 0; i < 4; ++i)
    if ((share(out[0], in[i]) && !(i < 3 && same(out[0], in[i]))) || share(out[1], in[i]))
      return fail(-1, name, "an output shares memory with an input and is not in its place");
  if (share(out[0], out[1])) return fail(-1, name, "two outputs share memory");
  if (bad_workspace(workspace, workspace_bytes, netra_norm_gradients_workspace(rows, cols)))
    return fail(-1, name, "workspace too small, null or not 16-byte aligned");
  Launcher launch(stream);
  uint32_t parts = 0;
  if (rows) {
    const NormPlan plan = norm_gradients_plan(rows, cols);
    parts = plan.groups;
    nknorm::NormGradients a{};
    a.dy = dy;
    a.dy_stride = dy_stride;
    a.r = r;
    a.r_stride = r_stride;
    a.flow = flow;
    a.flow_stride = flow_stride;
    a.w = weight;
    a.w_bf16 = weight_type == NETRA_BF16;
    a.offset = offset;
    a.eps = eps;
    a.inv_cols = 1.0f / static_cast<float>(cols);
    a.dr = dr;
    a.dr_stride = dr_stride;
    a.partial = static_cast<float*>(workspace);
    a.rows = rows;
    a.cols = cols;
    const uint32_t first = dy_type, second = r_type;
    const bool once = (row_bytes(cols, dy_type) + (flow ? 3u : 2u) * row_bytes(cols, r_type)) * rows > kInfinityCache;
    const dim3 grid(plan.groups), block(plan.threads);
    NETRA_NORM_SHAPES(netra_norm_gradients);
  }
  if (rows || !accumulate)
    launch(netra_norm_sum_gfx950, dim3((cols + 63u) / 64u), dim3(1024), static_cast<const float*>(workspace), parts, cols,
           dw, accumulate ? 1u : 0u);
  return launch.result(name);
}
#undef NETRA_NORM_SHAPES
#undef NETRA_NORM_TYPES
#undef NETRA_NORM_ONE
