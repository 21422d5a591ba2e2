// C entry points of the routing to experts (included by netra_layers.hip): argument checks, choice
// of kernels and launches.
#pragma once
#include "layers_call.h"
#include "layers_plan.h"
#include "router_select.hip"

namespace {

bool bad_choice(uint32_t tokens, uint32_t experts, uint32_t k, uint32_t shared, uint32_t scoring, float scale) {
  return tokens > kMaxRouted || experts == 0 || experts > nkbal::kMaxExperts || k == 0 || k > nksel::kMost || k > experts ||
         shared > 1u || k + shared > nksel::kMost || scoring > NETRA_SIGMOID || !(scale == scale);
}
// Rows of 32-bit values with a stride in elements.
bool bad_words(const void* p, uint64_t stride, uint32_t cols) { return !p || !aligned(p, 4) || stride < cols; }

#define NETRA_SELECT_SHAPES(KERNEL)                                         \
  do {                                                                      \
    if (experts <= 64u) launch(KERNEL##_16x4_gfx950, grid, block, a);       \
    else if (experts <= 128u) launch(KERNEL##_16x8_gfx950, grid, block, a); \
    else if (experts <= 256u) launch(KERNEL##_16x16_gfx950, grid, block, a); \
    else if (experts <= 512u) launch(KERNEL##_16x32_gfx950, grid, block, a); \
    else launch(KERNEL##_64x16_gfx950, grid, block, a);                     \
  } while (0)

}  // namespace

extern "C" int netra_router_select(const void* logits, uint32_t logits_type, uint64_t logits_stride, const float* bias,
                                   const uint8_t* mask, uint32_t tokens, uint32_t experts, uint32_t k, uint32_t shared,
                                   uint32_t scoring, uint32_t groups, uint32_t top_groups, uint32_t group_score,
                                   uint32_t renormalise, float scale, int32_t* ids, uint64_t ids_stride, float* weights,
                                   uint64_t weights_stride, hipStream_t stream) {
  const char* name = "netra_router_select";
  if (bad_choice(tokens, experts, k, shared, scoring, scale))
    return fail(-1, name, "tokens up to 2^25, experts 1 .. 1024, k (with the shared expert) 1 .. 16 and at most the experts, a known scoring");
  if (groups == 0 || groups > nksel::kMost || experts % groups || top_groups == 0 || top_groups > groups ||
      k > top_groups * (experts / groups) || group_score > NETRA_GROUP_TOP2 ||
      (groups > 1u && group_score == NETRA_GROUP_TOP2 && experts / groups < 2u))
    return fail(-1, name, "groups 1 .. 16 that divide the experts, with k experts or more in the top groups, two in each for their sum");
  if (tokens == 0) {
    g_error.clear();
    return 0;
  }
  if (bad_matrix(logits, logits_type, logits_stride, experts + shared) || (bias && !aligned(bias, 4)) ||
      bad_words(ids, ids_stride, k + shared) || bad_words(weights, weights_stride, k + shared))
    return fail(-1, name, "null or misaligned pointer, unknown type, or row stride below the row");
  if (logits_stride >= (1u << 27)) return fail(-1, name, "the logits' row stride has to be below 2^27");
  const uint64_t slots = 4ull * (k + shared);
  const Span in = rows_span(logits, logits_type, logits_stride, tokens, experts + shared);
  const Span out[] = {{ids, ids_stride * 4u, slots, tokens}, {weights, weights_stride * 4u, slots, tokens}};
  const Span more[] = {{bias, experts * 4ull, experts * 4ull, bias ? 1u : 0u}, {mask, 1, 1, mask ? tokens : 0u}};
  for (const Span& o : out)
    if (share(in, o) || share(more[0], o) || share(more[1], o))
      return fail(-1, name, "an output shares memory with an input");
  if (share(out[0], out[1])) return fail(-1, name, "the outputs share memory");
  nksel::Select a{};
  a.z = logits;
  a.z_stride = logits_stride;
  a.bias = bias;
  a.mask = mask;
  a.tokens = tokens;
  a.experts = experts;
  a.k = k;
  a.shared = shared;
  a.scoring = scoring;
  a.groups = top_groups == groups ? 1u : groups;  // (all groups are kept)
  a.each = experts / groups;
  a.top_groups = top_groups;
  a.top2 = group_score == NETRA_GROUP_TOP2;
  a.renormalise = renormalise != 0;
  a.scale = scale;
  a.ids = ids;
  a.ids_stride = ids_stride;
  a.weights = weights;
  a.weights_stride = weights_stride;
  a.by_logits = !bias && (a.groups == 1u || !a.top2);
  Launcher launch(stream);
  const dim3 grid((tokens - 1u) / (experts <= 512u ? 16u : 4u) + 1u), block(256);
  if (logits_type == NETRA_BF16) {
    if (a.by_logits) NETRA_SELECT_SHAPES(netra_router_select_bf16);
    else NETRA_SELECT_SHAPES(netra_router_select_scored_bf16);
  } else {
    if (a.by_logits) NETRA_SELECT_SHAPES(netra_router_select_f32);
    else NETRA_SELECT_SHAPES(netra_router_select_scored_f32);
  }
  return launch.result(name);
}

extern "C" int netra_router_select_gradient(const float* dweights, uint64_t dweights_stride, const void* logits,
                                            uint32_t logits_type, uint64_t logits_stride, const int32_t* ids,
                                            uint64_t ids_stride, const uint8_t* mask, uint32_t tokens, uint32_t experts,
                                            uint32_t k, uint32_t shared, uint32_t scoring, uint32_t renormalise,
                                            float scale, void* grad, uint64_t grad_stride, uint32_t accumulate,
                                            hipStream_t stream) {
  const char* name = "netra_router_select_gradient";
  if (bad_choice(tokens, experts, k, shared, scoring, scale))
    return fail(-1, name, "tokens up to 2^25, experts 1 .. 1024, k (with the shared expert) 1 .. 16 and at most the experts, a known scoring");
  if (tokens == 0) {
    g_error.clear();
    return 0;
  }
  const uint32_t cols = experts + shared;
  if (bad_matrix(logits, logits_type, logits_stride, cols) || bad_matrix(grad, logits_type, grad_stride, cols) ||
      bad_words(dweights, dweights_stride, k + shared) || bad_words(ids, ids_stride, k))
    return fail(-1, name, "null or misaligned pointer, unknown type, or row stride below the row");
  if (logits_stride >= (1u << 27) || grad_stride >= (1u << 27))
    return fail(-1, name, "row strides of logits and grad have to be below 2^27");
  const Span out = rows_span(grad, logits_type, grad_stride, tokens, cols);
  if (share(out, rows_span(logits, logits_type, logits_stride, tokens, cols)) ||
      share(out, {dweights, dweights_stride * 4u, 4ull * (k + shared), tokens}) ||
      share(out, {ids, ids_stride * 4u, 4ull * k, tokens}) || share(out, {mask, 1, 1, mask ? tokens : 0u}))
    return fail(-1, name, "grad shares memory with an input");
  nksel::SelectGradient a{};
  a.dw = dweights;
  a.dw_stride = dweights_stride;
  a.z = logits;
  a.z_stride = logits_stride;
  a.ids = ids;
  a.ids_stride = ids_stride;
  a.mask = mask;
  a.tokens = tokens;
  a.experts = experts;
  a.k = k;
  a.shared = shared;
  a.scoring = scoring;
  a.renormalise = renormalise != 0;
  a.scale = scale;
  a.grad = grad;
  a.grad_stride = grad_stride;
  a.accumulate = accumulate != 0;
  Launcher launch(stream);
  const dim3 grid(select_groups(tokens, experts <= 512u ? 16u : 4u)), block(256);
  if (logits_type == NETRA_BF16) {
    NETRA_SELECT_SHAPES(netra_router_select_gradient_bf16);
  } else {
    NETRA_SELECT_SHAPES(netra_router_select_gradient_f32);
  }
  return launch.result(name);
}
#undef NETRA_SELECT_SHAPES
