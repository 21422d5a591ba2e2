// C entry points of libnetra_layers.so (include/netra_layers.h): argument
// checks, workspace layout, choice of kernels and launches.
#include "layers_call.h"
#include "layers_plan.h"
#include "linear_fp8.hip"
#include "router_balance.hip"

namespace {

using namespace nkplan;

// A quantised matrix in the workspace: codes of up(rows, 16) x up(cols, 128), then scales [blocks][up(rows, 16)].
uint64_t code_bytes(uint32_t rows, uint32_t cols) { return static_cast<uint64_t>(up(rows, 16u)) * up(cols, 128u); }
uint64_t matrix_bytes(uint32_t rows, uint32_t cols) {
  return code_bytes(rows, cols) + static_cast<uint64_t>(up(rows, 16u)) * blocks(cols) * 4u;
}

bool bad_sizes(uint32_t rows, uint32_t n, uint32_t k) {
  return n == 0 || k == 0 || rows > kMaxSize || n > kMaxSize || k > kMaxSize;
}
void quant_rows(const void* x, uint32_t type, uint64_t stride, uint8_t* q, float* s, uint32_t rows, uint32_t n,
                Launcher& launch) {
  const dim3 grid((rows + 15u) / 16u, (blocks(n) + 3u) / 4u), block(256);
  const uint32_t sld = up(rows, 16u);
  if (type == NETRA_BF16)
    launch(netra_linear_quant_rows_bf16_gfx950, grid, block, static_cast<const uint16_t*>(x), stride, q, s, rows, n,
           sld);
  else
    launch(netra_linear_quant_rows_f32_gfx950, grid, block, static_cast<const float*>(x), stride, q, s, rows, n, sld);
}

uint64_t product_workspace(uint32_t rows, uint32_t ni, uint32_t nc, uint32_t in_type) {
  if (rows == 0) return 0;
  const ProductPlan plan = product_plan(rows, ni, nc, in_type == NETRA_BF16);
  if (plan.form == kFused) return 0;
  const uint64_t partial = plan.splits > 1u ? 4u * static_cast<uint64_t>(plan.splits) * rows * up(ni, 4u) : 0u;
  return (matrix_bytes(rows, nc) + 15u) / 16u * 16u + partial;
}

template <typename X>
void product_fused(const nklin::Product& a, const ProductPlan& plan, const X* x, uint64_t stride, uint32_t nc,
                   Launcher& launch) {
  const dim3 grid(((a.ni + 15u) / 16u + plan.p - 1u) / plan.p), block(512);
#define NETRA_RUN(P, Q)                                                                                          \
  do {                                                                                                           \
    if constexpr (sizeof(X) == 2)                                                                                \
      launch(netra_linear_product_fused_bf16_p##P##q##Q##_gfx950, grid, block, a, x, stride, nc);                \
    else launch(netra_linear_product_fused_f32_p##P##q##Q##_gfx950, grid, block, a, x, stride, nc);              \
  } while (0)
  if (plan.q == 4u) {
    if constexpr (sizeof(X) == 2) launch(netra_linear_product_fused_bf16_p1q4_gfx950, grid, block, a, x, stride, nc);
  } else if (plan.q == 2u && plan.p == 2u) NETRA_RUN(2, 2);
  else if (plan.q == 2u) NETRA_RUN(1, 2);
  else if (plan.p == 2u) NETRA_RUN(2, 1);
  else NETRA_RUN(1, 1);
#undef NETRA_RUN
}

// An operand of the weight gradient as it is, or as bf16 with aligned rows in the workspace.
bool outer_ready(const void* m, uint32_t type, uint64_t stride, uint32_t cols) {
  return type == NETRA_BF16 && aligned(m, 4) && cols % 2u == 0 && stride % 2u == 0 && stride < (1u << 24);
}
uint64_t outer_bytes(const void* m, uint32_t type, uint64_t stride, uint32_t rows, uint32_t cols) {
  return outer_ready(m, type, stride, cols) ? 0 : static_cast<uint64_t>(rows) * up(cols, 8u) * 2u;
}
// Its pointer, and the copy that has to be made of it, if any.
const uint16_t* outer_operand(const void* m, uint32_t type, uint64_t& stride, uint32_t rows, uint32_t& cols,
                              uint8_t*& at, nklin::Copy& copy) {
  if (outer_ready(m, type, stride, cols)) return static_cast<const uint16_t*>(m);
  const uint32_t pitch = up(cols, 8u);
  uint16_t* out = reinterpret_cast<uint16_t*>(at);
  copy = {m, stride, out, type, cols, pitch, copy_groups(rows, pitch)};
  at += static_cast<uint64_t>(rows) * pitch * 2u;
  stride = cols = pitch;
  return out;
}

}  // namespace

extern "C" uint64_t netra_linear_packed_bytes(uint32_t n, uint32_t k, uint32_t transpose) {
  return transpose ? code_bytes(k, n) : code_bytes(n, k);
}

extern "C" int netra_linear_pack(const uint8_t* w, uint8_t* packed, uint32_t n, uint32_t k, uint32_t transpose,
                                 hipStream_t stream) {
  if (!w || !packed || w == packed || !aligned(packed, 16) || bad_sizes(0, n, k))
    return fail(-1, "netra_linear_pack", "null, aliased or misaligned pointers, or n / k not in 1 .. 2^21");
  Launcher launch(stream);
  if (transpose)
    launch(netra_linear_pack_transposed_gfx950, dim3((k + 63u) / 64u, blocks(n)), dim3(256), w, packed, n, k);
  else
    launch(netra_linear_pack_gfx950, dim3((n + 15u) / 16u, (blocks(k) + 3u) / 4u), dim3(256), w, packed, n, k);
  return launch.result("netra_linear_pack");
}

extern "C" uint64_t netra_linear_forward_workspace(uint32_t rows, uint32_t n, uint32_t k, uint32_t x_type) {
  return product_workspace(rows, n, k, x_type);
}
extern "C" uint64_t netra_linear_input_gradient_workspace(uint32_t rows, uint32_t n, uint32_t k, uint32_t dy_type) {
  return product_workspace(rows, k, n, dy_type);
}
static uint64_t partial_bytes(const OuterPlan& plan, uint32_t n, uint32_t k) {
  return plan.splits > 1u ? 4u * static_cast<uint64_t>(plan.splits) * n * k : 0;
}
extern "C" uint64_t netra_linear_weight_gradient_workspace(uint32_t rows, uint32_t n, uint32_t k, uint32_t in_place) {
  if (rows == 0) return 0;
  return partial_bytes(outer_plan(rows, n, k), n, k) +
         (in_place ? 0 : static_cast<uint64_t>(rows) * (static_cast<uint64_t>(up(n, 8u)) + up(k, 8u)) * 2u);
}

// One call of the product: in [rows, nc] times the packed matrix P [ni, nc] -> out [rows, ni].
struct ProductCall {
  const char* name;
  const void* in;
  uint32_t in_type;
  uint64_t in_stride;
  const uint8_t* packed;
  const float* scale;
  uint32_t sp_i, sp_b;
  uint16_t* out;
  uint64_t out_stride;
  uint32_t rows, ni, nc;
};

static int check(const ProductCall& c) {
  if (bad_matrix(c.in, c.in_type, c.in_stride, c.nc) || bad_matrix(c.out, NETRA_BF16, c.out_stride, c.ni) ||
      !c.packed || !aligned(c.packed, 16) || !c.scale || !aligned(c.scale, 4))
    return fail(-1, c.name, "null or misaligned pointer, unknown type, or row stride below the row");
  if (share({c.in, c.in_stride * elem(c.in_type), static_cast<uint64_t>(c.nc) * elem(c.in_type), c.rows},
            {c.out, c.out_stride * 2u, static_cast<uint64_t>(c.ni) * 2u, c.rows}))
    return fail(-1, c.name, "the output shares memory with the input");
  return 0;
}

static void set_up(const ProductCall& c, const ProductPlan& plan, uint8_t* workspace, nklin::Product& a) {
  a.p = c.packed;
  a.sp = c.scale;
  a.sp_i = c.sp_i;
  a.sp_b = c.sp_b;
  a.sp_bytes = blocks(c.ni) * blocks(c.nc) * 4u;
  a.out = c.out;
  a.ldo = c.out_stride;
  a.ni = c.ni;
  a.nq = c.rows;
  a.kb = blocks(c.nc);
  a.splits = plan.splits;
  a.split_blocks = plan.split_blocks;
  if (plan.form == kFused) return;
  a.q = workspace;
  a.sq = reinterpret_cast<float*>(workspace + code_bytes(c.rows, c.nc));
  a.sq_b = up(c.rows, 16u);
  a.partial = reinterpret_cast<float*>(workspace + (matrix_bytes(c.rows, c.nc) + 15u) / 16u * 16u);
}

static void quantise(const ProductCall& c, const ProductPlan& plan, uint8_t* workspace, Launcher& launch) {
  if (plan.form != kFused)
    quant_rows(c.in, c.in_type, c.in_stride, workspace, reinterpret_cast<float*>(workspace + code_bytes(c.rows, c.nc)),
               c.rows, c.nc, launch);
}

static uint64_t groups_of(const ProductCall& c, const ProductPlan& plan) {
  return tile_groups(c.ni, plan.p, c.rows, plan.q, plan.splits);
}
// Before anything is launched: whether the product's workgroups fit a launch. (Those that do not
// have outputs larger than the memory.)
static int check_grid(const ProductCall& c, const ProductPlan& plan) {
  if (plan.form == kTiles && !launchable(groups_of(c, plan), 512u))
    return fail(-1, c.name, "more workgroups than one launch takes");
  return 0;
}

static void run(const ProductCall& c, const nklin::Product& a, const ProductPlan& plan, Launcher& launch) {
  if (plan.form == kFused) {
    if (c.in_type == NETRA_BF16)
      return product_fused(a, plan, static_cast<const uint16_t*>(c.in), c.in_stride, c.nc, launch);
    return product_fused(a, plan, static_cast<const float*>(c.in), c.in_stride, c.nc, launch);
  }
  const dim3 block(512);
  if (plan.form == kStream) {
    const dim3 grid(((a.ni + 15u) / 16u + plan.p - 1u) / plan.p);
    if (plan.p == 2u) launch(netra_linear_product_stream_p2q4_gfx950, grid, block, a);
    else launch(netra_linear_product_stream_p1q4_gfx950, grid, block, a);
    return;
  }
  const dim3 grid(static_cast<uint32_t>(groups_of(c, plan)));
  if (plan.p == 256u && plan.q == 256u) launch(netra_linear_product_256x256_gfx950, grid, block, a);
  else if (plan.p == 256u) launch(netra_linear_product_256x128_gfx950, grid, block, a);
  else if (plan.q == 128u) launch(netra_linear_product_128x128_gfx950, grid, block, a);
  else if (plan.p == 128u) launch(netra_linear_product_128x64_gfx950, grid, block, a);
  else launch(netra_linear_product_64x64_gfx950, grid, block, a);
  if (plan.splits > 1u)
    launch(netra_linear_product_sum_gfx950, dim3((a.ni + 1023u) / 1024u, a.nq < 4096u ? a.nq : 4096u), dim3(256),
           a);
}

static int times_weights(const ProductCall& c, void* workspace, uint64_t workspace_bytes, hipStream_t stream) {
  if (bad_sizes(c.rows, c.ni, c.nc)) return fail(-1, c.name, "sizes have to be 1 .. 2^21 (rows may be 0)");
  if (c.rows == 0) {
    g_error.clear();
    return 0;
  }
  const int rc = check(c);
  if (rc != 0) return rc;
  if (bad_workspace(workspace, workspace_bytes, product_workspace(c.rows, c.ni, c.nc, c.in_type)))
    return fail(-1, c.name, "workspace too small, null or not 16-byte aligned");
  const ProductPlan plan = product_plan(c.rows, c.ni, c.nc, c.in_type == NETRA_BF16);
  if (check_grid(c, plan) != 0) return -1;
  nklin::Product a{};
  set_up(c, plan, static_cast<uint8_t*>(workspace), a);
  Launcher launch(stream);
  quantise(c, plan, static_cast<uint8_t*>(workspace), launch);
  run(c, a, plan, launch);
  return launch.result(c.name);
}

extern "C" int netra_linear_forward(const void* x, uint32_t x_type, uint64_t x_stride, const uint8_t* packed,
                                    const float* scale, uint16_t* y, uint64_t y_stride, uint32_t rows, uint32_t n,
                                    uint32_t k, void* workspace, uint64_t workspace_bytes, hipStream_t stream) {
  return times_weights({"netra_linear_forward", x, x_type, x_stride, packed, scale, blocks(k), 1u, y, y_stride, rows,
                        n, k},
                       workspace, workspace_bytes, stream);
}

extern "C" int netra_linear_input_gradient(const void* dy, uint32_t dy_type, uint64_t dy_stride,
                                           const uint8_t* packed_t, const float* scale, uint16_t* dx,
                                           uint64_t dx_stride, uint32_t rows, uint32_t n, uint32_t k, void* workspace,
                                           uint64_t workspace_bytes, hipStream_t stream) {
  return times_weights({"netra_linear_input_gradient", dy, dy_type, dy_stride, packed_t, scale, 1u, blocks(k), dx,
                        dx_stride, rows, k, n},
                       workspace, workspace_bytes, stream);
}

// Rows that come quantised (netra_norm_forward with NETRA_CODES_TILES).
extern "C" uint64_t netra_linear_forward_codes_workspace(uint32_t rows, uint32_t n, uint32_t k) {
  if (rows == 0) return 0;
  const ProductPlan plan = codes_plan(rows, n, k);
  return plan.splits > 1u ? 4u * static_cast<uint64_t>(plan.splits) * rows * up(n, 4u) : 0u;
}
extern "C" int netra_linear_forward_codes(const uint8_t* codes, const float* scales, const uint8_t* packed,
                                          const float* scale, uint16_t* y, uint64_t y_stride, uint32_t rows, uint32_t n,
                                          uint32_t k, void* workspace, uint64_t workspace_bytes, hipStream_t stream) {
  const char* name = "netra_linear_forward_codes";
  if (bad_sizes(rows, n, k)) return fail(-1, name, "sizes have to be 1 .. 2^21 (rows may be 0)");
  if (rows == 0) {
    g_error.clear();
    return 0;
  }
  if (!codes || !aligned(codes, 16) || !scales || !aligned(scales, 4) || !packed || !aligned(packed, 16) || !scale ||
      !aligned(scale, 4) || bad_matrix(y, NETRA_BF16, y_stride, n))
    return fail(-1, name, "null or misaligned pointer, or row stride below the row");
  const uint64_t bytes = code_bytes(rows, k), scale_bytes = 4ull * up(rows, 16u) * blocks(k);
  const Span out{y, y_stride * 2u, static_cast<uint64_t>(n) * 2u, rows};
  if (share(out, {codes, bytes, bytes, 1}) || share(out, {scales, scale_bytes, scale_bytes, 1}))
    return fail(-1, name, "the output shares memory with the codes or their scales");
  if (bad_workspace(workspace, workspace_bytes, netra_linear_forward_codes_workspace(rows, n, k)))
    return fail(-1, name, "workspace too small, null or not 16-byte aligned");
  const ProductCall c{name, codes, NETRA_BF16, k, packed, scale, blocks(k), 1u, y, y_stride, rows, n, k};
  const ProductPlan plan = codes_plan(rows, n, k);
  if (check_grid(c, plan) != 0) return -1;
  nklin::Product a{};
  set_up(c, plan, static_cast<uint8_t*>(workspace), a);
  a.q = codes;
  a.sq = scales;
  a.partial = static_cast<float*>(workspace);
  Launcher launch(stream);
  run(c, a, plan, launch);
  return launch.result(name);
}

// One call of the weight gradient.
struct OuterCall {
  const char* name;
  const void* dy;
  uint32_t dy_type;
  uint64_t dy_stride;
  const void* x;
  uint32_t x_type;
  uint64_t x_stride;
  float* dw;
  uint32_t accumulate, rows, n, k;
};

static int check(const OuterCall& c) {
  if (bad_matrix(c.dy, c.dy_type, c.dy_stride, c.n) || bad_matrix(c.x, c.x_type, c.x_stride, c.k))
    return fail(-1, c.name, "null or misaligned pointer, unknown type, or row stride below the row");
  const uint64_t bytes = static_cast<uint64_t>(c.n) * c.k * 4u;
  const Span out{c.dw, bytes, bytes, 1};
  if (share({c.dy, c.dy_stride * elem(c.dy_type), static_cast<uint64_t>(c.n) * elem(c.dy_type), c.rows}, out) ||
      share({c.x, c.x_stride * elem(c.x_type), static_cast<uint64_t>(c.k) * elem(c.x_type), c.rows}, out))
    return fail(-1, c.name, "dw shares memory with an input");
  return 0;
}

static uint64_t outer_workspace(const OuterCall& c, const OuterPlan& plan) {
  return outer_bytes(c.dy, c.dy_type, c.dy_stride, c.rows, c.n) + outer_bytes(c.x, c.x_type, c.x_stride, c.rows, c.k) +
         partial_bytes(plan, c.n, c.k);
}

static void set_up(const OuterCall& c, const OuterPlan& plan, uint8_t* workspace, nklin::Outer& a,
                   nklin::Copy (&copies)[2]) {
  a.dy_stride = c.dy_stride;
  a.dy_cols = c.n;
  a.dy = outer_operand(c.dy, c.dy_type, a.dy_stride, c.rows, a.dy_cols, workspace, copies[0]);
  a.x_stride = c.x_stride;
  a.x_cols = c.k;
  a.x = outer_operand(c.x, c.x_type, a.x_stride, c.rows, a.x_cols, workspace, copies[1]);
  a.dw = c.dw;
  a.rows = c.rows;
  a.n = c.n;
  a.k = c.k;
  a.accumulate = c.accumulate ? 1u : 0u;
  a.splits = plan.splits;
  a.split_rows = plan.split_rows;
  a.partial = reinterpret_cast<float*>(workspace);
}

// The operands' copies, with dy's quantisation (to `codes`, or null) in the same launch.
static void prepare(const OuterCall& c, const nklin::Copy (&copies)[2], uint8_t* codes, Launcher& launch) {
  const uint32_t quant = codes ? quant_groups(c.rows, c.n) : 0u;
  const dim3 grid(quant + copies[0].groups + copies[1].groups), block(256);
  float* s = codes ? reinterpret_cast<float*>(codes + code_bytes(c.rows, c.n)) : nullptr;
  const uint32_t sld = up(c.rows, 16u);
  if (c.dy_type == NETRA_BF16)
    launch(netra_linear_prepare_bf16_gfx950, grid, block, static_cast<const uint16_t*>(c.dy), c.dy_stride, codes,
           s, c.rows, c.n, sld, quant, copies[0], copies[1]);
  else
    launch(netra_linear_prepare_f32_gfx950, grid, block, static_cast<const float*>(c.dy), c.dy_stride, codes, s,
           c.rows, c.n, sld, quant, copies[0], copies[1]);
}

static uint64_t groups_of(const OuterCall& c, const OuterPlan& plan) {
  return tile_groups(c.k, plan.p, c.n, plan.q, plan.splits);
}
static int check_grid(const OuterCall& c, const OuterPlan& plan) {
  const uint64_t before = static_cast<uint64_t>(quant_groups(c.rows, c.n)) + copy_groups(c.rows, up(c.n, 8u)) +
                          copy_groups(c.rows, up(c.k, 8u));
  if (!launchable(groups_of(c, plan), 512u) || !launchable(before, 256u))
    return fail(-1, c.name, "more workgroups than one launch takes");
  return 0;
}

static void sum(const nklin::Outer& a, Launcher& launch) {
  if (a.splits == 1u) return;
  const uint64_t quads = (static_cast<uint64_t>(a.n) * a.k + 1023u) / 1024u;
  launch(netra_linear_outer_sum_gfx950, dim3(static_cast<uint32_t>(quads < 2048u ? quads : 2048u)), dim3(256), a);
}

static void run(const OuterCall& c, const nklin::Outer& a, const OuterPlan& plan, Launcher& launch) {
  const dim3 grid(static_cast<uint32_t>(groups_of(c, plan))), block(512);
  if (plan.p == 256u) launch(netra_linear_outer_256x256_gfx950, grid, block, a);
  else if (plan.q == 256u) launch(netra_linear_outer_128x256_gfx950, grid, block, a);
  else launch(netra_linear_outer_128x128_gfx950, grid, block, a);
  sum(a, launch);
}

// Sizes and dw, and the call without tokens: 0 or an error to return, or 1 to go on.
static int outer_start(const OuterCall& c, Launcher& launch) {
  if (bad_sizes(c.rows, c.n, c.k)) return fail(-1, c.name, "sizes have to be 1 .. 2^21 (rows may be 0)");
  if (!c.dw || !aligned(c.dw, 4)) return fail(-1, c.name, "null or misaligned dw");
  if (c.rows != 0) return 1;
  if (!c.accumulate)
    launch(netra_linear_zero_gfx950, dim3(1024), dim3(256), c.dw, static_cast<uint64_t>(c.n) * c.k);
  return launch.result(c.name);
}

extern "C" int netra_linear_weight_gradient(const void* dy, uint32_t dy_type, uint64_t dy_stride, const void* x,
                                            uint32_t x_type, uint64_t x_stride, float* dw, uint32_t accumulate,
                                            uint32_t rows, uint32_t n, uint32_t k, void* workspace,
                                            uint64_t workspace_bytes, hipStream_t stream) {
  const OuterCall c{"netra_linear_weight_gradient", dy, dy_type, dy_stride, x, x_type, x_stride, dw, accumulate, rows,
                    n, k};
  Launcher launch(stream);
  int rc = outer_start(c, launch);
  if (rc != 1) return rc;
  rc = check(c);
  if (rc != 0) return rc;
  const OuterPlan plan = outer_plan(rows, n, k);
  if (check_grid(c, plan) != 0) return -1;
  if (bad_workspace(workspace, workspace_bytes, outer_workspace(c, plan)))
    return fail(-1, c.name, "workspace too small, null or not 16-byte aligned");
  nklin::Outer a{};
  nklin::Copy copies[2] = {};
  set_up(c, plan, static_cast<uint8_t*>(workspace), a, copies);
  if (copies[0].groups + copies[1].groups) prepare(c, copies, nullptr, launch);
  run(c, a, plan, launch);
  return launch.result(c.name);
}

extern "C" uint64_t netra_linear_backward_workspace(uint32_t rows, uint32_t n, uint32_t k, uint32_t dy_type,
                                                    uint32_t in_place) {
  return (product_workspace(rows, k, n, dy_type) + 15u) / 16u * 16u +
         netra_linear_weight_gradient_workspace(rows, n, k, in_place);
}

extern "C" int netra_linear_backward(const void* dy, uint32_t dy_type, uint64_t dy_stride, const void* x,
                                     uint32_t x_type, uint64_t x_stride, const uint8_t* packed_t, const float* scale,
                                     uint16_t* dx, uint64_t dx_stride, float* dw, uint32_t accumulate, uint32_t rows,
                                     uint32_t n, uint32_t k, void* workspace, uint64_t workspace_bytes,
                                     hipStream_t stream) {
  const char* name = "netra_linear_backward";
  const OuterCall o{name, dy, dy_type, dy_stride, x, x_type, x_stride, dw, accumulate, rows, n, k};
  const ProductCall p{name, dy, dy_type, dy_stride, packed_t, scale, 1u, blocks(k), dx, dx_stride, rows, k, n};
  Launcher launch(stream);
  int rc = outer_start(o, launch);
  if (rc != 1) return rc;
  if ((rc = check(p)) != 0 || (rc = check(o)) != 0) return rc;
  const uint64_t dw_bytes = static_cast<uint64_t>(n) * k * 4u;
  if (share({dx, dx_stride * 2u, static_cast<uint64_t>(k) * 2u, rows}, {dw, dw_bytes, dw_bytes, 1}) ||
      share({dx, dx_stride * 2u, static_cast<uint64_t>(k) * 2u, rows},
            {x, x_stride * elem(x_type), static_cast<uint64_t>(k) * elem(x_type), rows}))
    return fail(-1, name, "dx shares memory with x or dw");
  ProductPlan product = product_plan(rows, k, n, dy_type == NETRA_BF16);
  const OuterPlan outer = outer_plan(rows, n, k);
  const uint64_t first = (product_workspace(rows, k, n, dy_type) + 15u) / 16u * 16u;
  if (bad_workspace(workspace, workspace_bytes, first + outer_workspace(o, outer)))
    return fail(-1, name, "workspace too small, null or not 16-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const bool small = backward_in_one(product, outer);
  if (small) product.p = product.q = 64u;
  if (check_grid(p, product) != 0 || check_grid(o, outer) != 0) return -1;
  const uint64_t outer_groups = groups_of(o, outer), groups = outer_groups + (small ? groups_of(p, product) : 0u);
  if (!launchable(groups, 512u)) return fail(-1, name, "more workgroups than one launch takes");
  nklin::Product a{};
  nklin::Outer b{};
  nklin::Copy copies[2] = {};
  set_up(p, product, ws, a);
  set_up(o, outer, ws + first, b, copies);
  if (copies[0].groups + copies[1].groups) prepare(o, copies, product.form == kFused ? nullptr : ws, launch);
  else quantise(p, product, ws, launch);
  if (small) {
    launch(netra_linear_backward_small_gfx950, dim3(static_cast<uint32_t>(groups)), dim3(512), a, b,
           static_cast<uint32_t>(outer_groups));
    sum(b, launch);
  } else {
    run(p, a, product, launch);
    run(o, b, outer, launch);
  }
  return launch.result(name);
}

// ---- router -------------------------------------------------------------------

static bool bad_router(uint32_t tokens, uint32_t slots, uint32_t experts) {
  return experts == 0 || experts > nkbal::kMaxExperts || static_cast<uint64_t>(tokens) * slots > 0x7fffffffull ||
         tokens > 0x7fffffffu;
}

static uint64_t parts_bytes(const CountPlan& plan, uint32_t experts) {
  return (4u * static_cast<uint64_t>(plan.groups) * (experts + 1u) + 15u) / 16u * 16u;
}

extern "C" uint64_t netra_router_counts_workspace(uint32_t tokens, uint32_t slots, uint32_t experts) {
  return parts_bytes(count_plan(tokens, kFewCounts, 256u), experts);
}

extern "C" int netra_router_counts(const int32_t* ids, uint64_t ids_stride, const uint8_t* mask, uint32_t tokens,
                                   uint32_t slots, uint32_t experts, int32_t* counts, uint32_t accumulate,
                                   void* workspace, uint64_t workspace_bytes, hipStream_t stream) {
  const char* name = "netra_router_counts";
  if (bad_router(tokens, slots, experts) || slots == 0)
    return fail(-1, name, "experts have to be 1 .. 1024, slots 1 or more, tokens * slots below 2^31");
  if (!counts || !aligned(counts, 4) || (tokens && (!ids || !aligned(ids, 4) || ids_stride < slots)))
    return fail(-1, name, "null or misaligned pointer, or ids' row stride below the slots");
  if (bad_workspace(workspace, workspace_bytes, netra_router_counts_workspace(tokens, slots, experts)))
    return fail(-1, name, "workspace too small, null or not 16-byte aligned");
  const CountPlan plan = count_plan(tokens, kFewCounts, 256u);
  Launcher launch(stream);
  if (plan.groups == 0) {
    launch(netra_router_counts_gfx950, dim3(1), dim3(1024), ids, ids_stride, mask, tokens, slots, experts, counts,
           accumulate ? 1u : 0u);
    return launch.result(name);
  }
  uint32_t* parts = static_cast<uint32_t*>(workspace);
  launch(netra_router_count_parts_gfx950, dim3(plan.groups), dim3(256), ids, ids_stride, mask, tokens, slots,
         experts, plan.each, parts, nullptr);
  launch(netra_router_count_sum_gfx950, dim3((experts + 15u) / 16u), dim3(256), parts, plan.groups, experts,
         counts, accumulate ? 1u : 0u);
  return launch.result(name);
}

extern "C" uint64_t netra_router_balance_workspace(uint32_t tokens, uint32_t slots, uint32_t experts) {
  const CountPlan plan = balance_plan(tokens, experts);
  return plan.groups ? 16u + 4u * kBalanceGrid + parts_bytes(plan, experts) : 0;
}

extern "C" int netra_router_balance(const void* logits, uint32_t logits_type, uint64_t logits_stride, const float* bias,
                                    const int32_t* ids, uint64_t ids_stride, uint32_t slots, const uint8_t* mask,
                                    uint32_t tokens, uint32_t experts, float coefficient, int32_t* counts,
                                    float* loss, void* grad, uint64_t grad_stride, void* workspace,
                                    uint64_t workspace_bytes, hipStream_t stream) {
  const char* name = "netra_router_balance";
  if (bad_router(tokens, slots, experts))
    return fail(-1, name, "experts have to be 1 .. 1024, tokens and tokens * slots below 2^31");
  if (bad_type(logits_type) || !counts || !aligned(counts, 4) || !loss || !aligned(loss, 4) ||
      (bias && !aligned(bias, 4)))
    return fail(-1, name, "null or misaligned pointer or unknown type");
  if (tokens && (bad_matrix(logits, logits_type, logits_stride, experts) ||
                 (slots && (!ids || !aligned(ids, 4) || ids_stride < slots)) ||
                 (grad && bad_matrix(grad, logits_type, grad_stride, experts))))
    return fail(-1, name, "null or misaligned pointer, or row stride below the row");
  // the kernel's offsets inside four rows have 31 bits
  if (tokens && (logits_stride >= (1u << 27) || (grad && grad_stride >= (1u << 27))))
    return fail(-1, name, "row strides of logits and grad have to be below 2^27");
  const uint64_t row = static_cast<uint64_t>(experts) * elem(logits_type);
  if (grad && share({logits, logits_stride * elem(logits_type), row, tokens},
                    {grad, grad_stride * elem(logits_type), row, tokens}))
    return fail(-1, name, "grad shares memory with logits");
  if (bad_workspace(workspace, workspace_bytes, netra_router_balance_workspace(tokens, slots, experts)))
    return fail(-1, name, "workspace too small, null or not 16-byte aligned");
  const CountPlan plan = balance_plan(tokens, experts);
  nkbal::Balance a{};
  a.z = logits;
  a.z_stride = logits_stride;
  a.bias = bias;
  a.ids = ids;
  a.ids_stride = ids_stride;
  a.slots = slots;
  a.mask = mask;
  a.tokens = tokens;
  a.experts = experts;
  a.coefficient = coefficient;
  a.counts = counts;
  a.loss = loss;
  a.grad = grad;
  a.grad_stride = grad_stride;
  Launcher launch(stream);
  uint32_t grid = 1;
  if (plan.groups) {
    uint32_t* words = static_cast<uint32_t*>(workspace);
    a.arrived = words;
    a.partial = reinterpret_cast<float*>(words + 4);
    uint32_t* parts = words + 4 + kBalanceGrid;
    a.parts = parts;
    a.groups = plan.groups;
    launch(netra_router_count_parts_gfx950, dim3(plan.groups), dim3(plan.each > 256u ? 1024 : 256), ids,
           ids_stride, mask, tokens, slots, experts, plan.each, parts, words);
    // Rows per pass of a workgroup. (Workgroups of 512 threads: 32768 x 256 bf16 26.8 us, of 1024 24.6.)
    const uint32_t rows = experts <= 256u ? 64u : 16u;
    grid = (tokens - 1u) / rows + 1u;
    grid = grid > kBalanceGrid ? kBalanceGrid : grid;
  }
#define NETRA_RUN(NAME, F) launch(netra_router_balance_##NAME##_##F##_gfx950, dim3(grid), dim3(1024), a)
#define NETRA_PICK(NAME)                       \
  if (experts <= 64u) NETRA_RUN(NAME, 16x4);   \
  else if (experts <= 128u) NETRA_RUN(NAME, 16x8);  \
  else if (experts <= 256u) NETRA_RUN(NAME, 16x16); \
  else if (experts <= 512u) NETRA_RUN(NAME, 64x8);  \
  else NETRA_RUN(NAME, 64x16)
  if (logits_type == NETRA_BF16) {
    NETRA_PICK(bf16);
  } else {
    NETRA_PICK(f32);
  }
#undef NETRA_PICK
#undef NETRA_RUN
  return launch.result(name);
}

extern "C" const char* netra_layers_last_error(void) { return g_error.c_str(); }

#include "norm_call.h"
#include "router_select_call.h"
#include "adapters_call.h"
