// C entry points of the low-rank adapters (included by netra_layers.hip): argument checks,
// workspace layout, choice of kernels and launches.
#pragma once
#include "layers_call.h"
#include "layers_plan.h"
#include "adapters.hip"

namespace {

bool bad_adapters(uint32_t adapters, uint32_t rank, uint32_t n, uint32_t k) {
  return adapters == 0 || adapters > nkada::kMaxAdapters || rank == 0 || rank > nkada::kMaxRank || n == 0 || k == 0 ||
         n > kMaxSize || k > kMaxSize;
}
uint64_t u_bytes(const AdapterPlan& plan, uint32_t tokens, uint32_t rank) {
  return plan.fused ? 0 : 64ull * adapter_ranks(rank) * plan.splits * tokens;
}

}  // namespace

extern "C" uint64_t netra_adapters_packed_bytes(uint32_t adapters, uint32_t rank, uint32_t n, uint32_t k, uint32_t which) {
  const uint64_t part = 32ull * adapter_ranks(rank);
  return adapters * part * (which ? up(n, 64u) : up(k, 128u));
}

extern "C" int netra_adapters_pack(const void* a, const void* b, uint32_t type, void* packed_a, void* packed_b,
                                   uint32_t adapters, uint32_t rank, uint32_t n, uint32_t k, hipStream_t stream) {
  const char* name = "netra_adapters_pack";
  if (bad_adapters(adapters, rank, n, k))
    return fail(-1, name, "adapters have to be 1 .. 1024, the rank 1 .. 128, n and k 1 .. 2^21");
  if (!a || !b || bad_type(type) || !aligned(a, elem(type)) || !aligned(b, elem(type)) || !packed_a || !packed_b ||
      !aligned(packed_a, 16) || !aligned(packed_b, 16))
    return fail(-1, name, "null or misaligned pointer or unknown type");
  const uint64_t sizes[] = {static_cast<uint64_t>(adapters) * rank * k * elem(type),
                            static_cast<uint64_t>(adapters) * rank * n * elem(type),
                            netra_adapters_packed_bytes(adapters, rank, n, k, 0),
                            netra_adapters_packed_bytes(adapters, rank, n, k, 1)};
  const Span all[] = {{a, sizes[0], sizes[0], 1}, {b, sizes[1], sizes[1], 1}, {packed_a, sizes[2], sizes[2], 1}, {packed_b, sizes[3], sizes[3], 1}};
  for (int o = 2; o < 4; ++o)
    for (int i = 0; i < o; ++i)
      if (share(all[o], all[i])) return fail(-1, name, "an output shares memory with an input or the other output");
  const uint32_t nr = adapter_ranks(rank);
  const auto groups = [](uint64_t threads) { return static_cast<uint32_t>(threads / 256u < 65536u ? threads / 256u : 65536u); };
  const dim3 grid_a(groups(sizes[2] / 16u)), grid_b(groups(sizes[3] / 8u)), block(256);
  Launcher launch(stream);
  if (type == NETRA_BF16) {
    launch(netra_adapters_pack_a_bf16_gfx950, grid_a, block, static_cast<const uint16_t*>(a), static_cast<uint4*>(packed_a), adapters, rank, k, nr);
    launch(netra_adapters_pack_b_bf16_gfx950, grid_b, block, static_cast<const uint16_t*>(b), static_cast<uint2*>(packed_b), adapters, rank, n, nr);
  } else {
    launch(netra_adapters_pack_a_f32_gfx950, grid_a, block, static_cast<const float*>(a), static_cast<uint4*>(packed_a), adapters, rank, k, nr);
    launch(netra_adapters_pack_b_f32_gfx950, grid_b, block, static_cast<const float*>(b), static_cast<uint2*>(packed_b), adapters, rank, n, nr);
  }
  return launch.result(name);
}

extern "C" uint64_t netra_adapters_plan_bytes(uint32_t tokens, uint32_t adapters) {
  if (tokens == 0) return 0;
  return 4ull * nkada::kPlanHead + 4ull * up(tokens, 4u) + 16ull * adapter_tiles(tokens, adapters);
}

extern "C" int netra_adapters_plan(const int32_t* ids, uint32_t tokens, uint32_t adapters, void* plan,
                                   uint64_t plan_bytes, hipStream_t stream) {
  const char* name = "netra_adapters_plan";
  if (tokens > kMaxSize || adapters == 0 || adapters > nkada::kMaxAdapters)
    return fail(-1, name, "tokens have to be 0 .. 2^21, adapters 1 .. 1024");
  if (tokens == 0) {
    g_error.clear();
    return 0;
  }
  if (!ids || !aligned(ids, 4)) return fail(-1, name, "null or misaligned pointer");
  const uint64_t need = netra_adapters_plan_bytes(tokens, adapters);
  if (bad_workspace(plan, plan_bytes, need)) return fail(-1, name, "plan too small, null or not 16-byte aligned");
  if (share({ids, 4ull * tokens, 4ull * tokens, 1}, {plan, need, need, 1}))
    return fail(-1, name, "the plan shares memory with the ids");
  Launcher launch(stream);
  launch(netra_adapters_plan_gfx950, dim3(1), dim3(1024), ids, tokens, adapters, adapter_tile(tokens, adapters),
         static_cast<uint32_t*>(plan));
  return launch.result(name);
}

extern "C" uint64_t netra_adapters_add_workspace(uint32_t tokens, uint32_t adapters, uint32_t rank, uint32_t n, uint32_t k) {
  if (tokens == 0 || tokens > kMaxSize || bad_adapters(adapters, rank, n, k)) return 0;
  return u_bytes(adapter_plan(tokens, adapters, rank, n, k), tokens, rank);
}

extern "C" int netra_adapters_add(const void* x, uint32_t x_type, uint64_t x_stride, const void* packed_a,
                                  const void* packed_b, const float* scale, const void* plan, const uint16_t* y,
                                  uint64_t y_stride, uint16_t* out, uint64_t out_stride, uint32_t tokens,
                                  uint32_t adapters, uint32_t rank, uint32_t n, uint32_t k, void* workspace,
                                  uint64_t workspace_bytes, hipStream_t stream) {
  const char* name = "netra_adapters_add";
  if (tokens > kMaxSize || bad_adapters(adapters, rank, n, k))
    return fail(-1, name, "tokens have to be 0 .. 2^21, adapters 1 .. 1024, the rank 1 .. 128, n and k 1 .. 2^21");
  if (tokens == 0) {
    g_error.clear();
    return 0;
  }
  if (bad_matrix(x, x_type, x_stride, k) || bad_matrix(y, NETRA_BF16, y_stride, n) || bad_matrix(out, NETRA_BF16, out_stride, n) ||
      !packed_a || !packed_b || !aligned(packed_a, 16) || !aligned(packed_b, 16) || !scale || !aligned(scale, 4) || !plan ||
      !aligned(plan, 16))
    return fail(-1, name, "null or misaligned pointer, unknown type, or row stride below the row");
  const Span to = rows_span(out, NETRA_BF16, out_stride, tokens, n), from = rows_span(y, NETRA_BF16, y_stride, tokens, n);
  const AdapterPlan p = adapter_plan(tokens, adapters, rank, n, k);
  const uint64_t need = u_bytes(p, tokens, rank);
  if (bad_workspace(workspace, workspace_bytes, need))
    return fail(-1, name, "workspace too small, null or not 16-byte aligned");
  const auto bytes = [](const void* at, uint64_t size) { return Span{at, size, size, size ? 1u : 0u}; };
  const Span scratch = bytes(workspace, need);
  const Span read[] = {rows_span(x, x_type, x_stride, tokens, k),
                       bytes(packed_a, netra_adapters_packed_bytes(adapters, rank, n, k, 0)),
                       bytes(packed_b, netra_adapters_packed_bytes(adapters, rank, n, k, 1)), bytes(scale, 4ull * adapters),
                       bytes(plan, netra_adapters_plan_bytes(tokens, adapters))};
  for (const Span& r : read)
    if (share(to, r) || share(scratch, r))
      return fail(-1, name, "out or the workspace shares memory with x, the weights, the scales or the plan");
  if ((share(to, from) && !same(to, from)) || share(scratch, from) || share(scratch, to))
    return fail(-1, name, "out shares memory with y and is not in its place, or the workspace shares memory with one of them");
  nkada::Adapters a{};
  a.x = x;
  a.x_stride = x_stride;
  a.a = static_cast<const uint8_t*>(packed_a);
  a.b = static_cast<const uint8_t*>(packed_b);
  a.scale = scale;
  a.plan = static_cast<const uint32_t*>(plan);
  a.u = workspace;
  a.splits = p.splits;
  a.split_blocks = p.split_blocks;
  a.y = y;
  a.y_stride = y_stride;
  a.out = out;
  a.out_stride = out_stride;
  a.tokens = tokens;
  a.adapters = adapters;
  a.rank = rank;
  a.ranks = adapter_ranks(rank);
  a.n = n;
  a.k = k;
  a.in_place = out == y;
  a.wide = p.wide;
  const uint32_t width = p.fused ? 512u : 256u * p.wide;  // columns of a workgroup
  a.chunks = (n + width - 1u) / width;
  const uint64_t groups = static_cast<uint64_t>(a.chunks) * p.tiles;
  if (!launchable(groups, 512u)) return fail(-1, name, "more workgroups than one launch takes");
  Launcher launch(stream);
  if (p.fused) {
    const dim3 grid(static_cast<uint32_t>(groups)), block(512);
    if (x_type == NETRA_BF16) {
      if (a.ranks == 1u) launch(netra_adapters_fused_bf16_r1_gfx950, grid, block, a);
      else if (a.ranks == 2u) launch(netra_adapters_fused_bf16_r2_gfx950, grid, block, a);
      else if (a.ranks == 4u) launch(netra_adapters_fused_bf16_r4_gfx950, grid, block, a);
      else launch(netra_adapters_fused_bf16_r8_gfx950, grid, block, a);
    } else {
      if (a.ranks == 1u) launch(netra_adapters_fused_f32_r1_gfx950, grid, block, a);
      else if (a.ranks == 2u) launch(netra_adapters_fused_f32_r2_gfx950, grid, block, a);
      else if (a.ranks == 4u) launch(netra_adapters_fused_f32_r4_gfx950, grid, block, a);
      else launch(netra_adapters_fused_f32_r8_gfx950, grid, block, a);
    }
    return launch.result(name);
  }
  // (a rank over 64 in two parts of the first product: of one the operands do not fit the registers)
  const dim3 shrink(p.tiles, p.splits, a.ranks == 8u ? 2u : 1u), expand(static_cast<uint32_t>(groups));
  const bool once = adapter_once(tokens, adapters, rank, n);
#define NETRA_RUN(TT, NR, EXPAND_NR)                                                                        \
  do {                                                                                                      \
    if (x_type == NETRA_BF16) launch(netra_adapters_shrink_bf16_t##TT##r##NR##_gfx950, shrink, dim3(512), a); \
    else launch(netra_adapters_shrink_f32_t##TT##r##NR##_gfx950, shrink, dim3(512), a);                     \
    if (once) launch(netra_adapters_expand_t##TT##r##EXPAND_NR##_once_gfx950, expand, dim3(256), a);        \
    else launch(netra_adapters_expand_t##TT##r##EXPAND_NR##_gfx950, expand, dim3(256), a);                  \
  } while (0)
#define NETRA_RANKS(TT)                        \
  if (a.ranks == 1u) NETRA_RUN(TT, 1, 1);      \
  else if (a.ranks == 2u) NETRA_RUN(TT, 2, 2); \
  else if (a.ranks == 4u) NETRA_RUN(TT, 4, 4); \
  else NETRA_RUN(TT, 4, 8)
  if (adapter_tile(tokens, adapters) == 16u) {
    NETRA_RANKS(1);
  } else {
    NETRA_RANKS(2);
  }
#undef NETRA_RANKS
#undef NETRA_RUN
  return launch.result(name);
}
