// C entry points of libnetra_layers.so (include/netra_layers.h): argument
// checks, workspace layout, choice of kernels and launches.
#include "../../../include/netra_layers.h"

#include <hip/hip_runtime.h>

#include <string>

#include "linear_fp8.hip"
#include "router_balance.hip"

namespace {

thread_local std::string g_error;

// No exception leaves a C entry point: a message there is no memory for is lost.
int fail(int code, const char* name, const char* text) noexcept {
  try {
    g_error = std::string(name) + ": " + text;
  } catch (...) {
    g_error.clear();
  }
  return code;
}

int launched(const char* name) noexcept {
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(static_cast<int>(err), name, hipGetErrorString(err));
  g_error.clear();
  return 0;
}

// Sizes up to 2^21 keep every grid dimension, tile count and scale index inside its type.
constexpr uint32_t kMaxSize = 1u << 21;

uint32_t up(uint32_t v, uint32_t m) { return (v + m - 1u) / m * m; }
uint32_t blocks(uint32_t v) { return (v + 127u) / 128u; }
uint32_t elem(uint32_t type) { return type == NETRA_BF16 ? 2u : 4u; }
bool aligned(const void* p, uint64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// A quantised matrix in the workspace: codes of up(rows, 16) x up(cols, 128), then scales [blocks][up(rows, 16)].
uint64_t code_bytes(uint32_t rows, uint32_t cols) { return static_cast<uint64_t>(up(rows, 16u)) * up(cols, 128u); }
uint64_t matrix_bytes(uint32_t rows, uint32_t cols) {
  return code_bytes(rows, cols) + static_cast<uint64_t>(up(rows, 16u)) * blocks(cols) * 4u;
}

bool bad_sizes(uint32_t rows, uint32_t n, uint32_t k) {
  return n == 0 || k == 0 || rows > kMaxSize || n > kMaxSize || k > kMaxSize;
}
bool bad_type(uint32_t type) { return type != NETRA_BF16 && type != NETRA_F32; }
// A matrix's base has to be aligned to its elements.
bool bad_matrix(const void* p, uint32_t type, uint64_t stride, uint32_t cols) {
  return !p || bad_type(type) || stride < cols || !aligned(p, elem(type));
}

void quant_rows(const void* x, uint32_t type, uint64_t stride, uint8_t* q, float* s, uint32_t rows, uint32_t n,
                hipStream_t stream) {
  const dim3 grid((rows + 15u) / 16u, (blocks(n) + 3u) / 4u), block(256);
  const bool vec = aligned(x, 16) && stride * elem(type) % 16u == 0;
  const uint32_t sld = up(rows, 16u);
  if (type == NETRA_BF16) {
    const uint16_t* p = static_cast<const uint16_t*>(x);
    if (vec) netra_linear_quant_rows_bf16_vec_gfx950<<<grid, block, 0, stream>>>(p, stride, q, s, rows, n, sld);
    else netra_linear_quant_rows_bf16_gfx950<<<grid, block, 0, stream>>>(p, stride, q, s, rows, n, sld);
  } else {
    const float* p = static_cast<const float*>(x);
    if (vec) netra_linear_quant_rows_f32_vec_gfx950<<<grid, block, 0, stream>>>(p, stride, q, s, rows, n, sld);
    else netra_linear_quant_rows_f32_gfx950<<<grid, block, 0, stream>>>(p, stride, q, s, rows, n, sld);
  }
}

// How a product runs: `stream` (quantising on the way) or tiles of p x q with splits of the contraction.
struct ProductPlan {
  bool stream;
  uint32_t p, q, splits, split_blocks;
};
ProductPlan product_plan(uint32_t rows, uint32_t ni, uint32_t nc) {
  if (rows <= 64u) return {true, 0, 0, 1, 0};
  auto tiles = [&](uint32_t p, uint32_t q) {
    return static_cast<uint64_t>((ni + p - 1u) / p) * ((rows + q - 1u) / q);
  };
  ProductPlan plan{false, 256, 256, 1, blocks(nc)};
  if (tiles(256, 256) < 200) plan.p = plan.q = 128;
  const uint64_t t = tiles(plan.p, plan.q);
  uint32_t splits = t >= 128 ? 1u : static_cast<uint32_t>(256 / t);
  const uint32_t most = (blocks(nc) + 3u) / 4u;  // 4 blocks at least
  splits = splits > most ? most : splits;
  plan.split_blocks = (blocks(nc) + splits - 1u) / splits;
  plan.splits = (blocks(nc) + plan.split_blocks - 1u) / plan.split_blocks;
  return plan;
}
uint64_t product_workspace(uint32_t rows, uint32_t ni, uint32_t nc) {
  if (rows == 0) return 0;
  const ProductPlan plan = product_plan(rows, ni, nc);
  if (plan.stream) return 0;
  const uint64_t partial = plan.splits > 1u ? 4u * static_cast<uint64_t>(plan.splits) * rows * up(ni, 4u) : 0u;
  return (matrix_bytes(rows, nc) + 15u) / 16u * 16u + partial;
}

template <typename X>
void product_stream(const nklin::Product& a, const X* x, uint64_t stride, uint32_t nc, hipStream_t stream) {
  const bool vec = aligned(x, 16) && stride * sizeof(X) % 16u == 0;
  const uint32_t pt = (a.ni + 15u) / 16u, q = (a.nq + 15u) / 16u;
  const bool wide = q > 1u || pt >= 512u;
  const dim3 grid(wide ? (pt + 1u) / 2u : pt), block(512);
#define NETRA_RUN(P, Q)                                                                                               \
  do {                                                                                                                \
    if constexpr (sizeof(X) == 2) {                                                                                   \
      if (vec) netra_linear_product_stream_bf16_vec_p##P##q##Q##_gfx950<<<grid, block, 0, stream>>>(a, x, stride, nc); \
      else netra_linear_product_stream_bf16_p##P##q##Q##_gfx950<<<grid, block, 0, stream>>>(a, x, stride, nc);        \
    } else {                                                                                                          \
      if (vec) netra_linear_product_stream_f32_vec_p##P##q##Q##_gfx950<<<grid, block, 0, stream>>>(a, x, stride, nc); \
      else netra_linear_product_stream_f32_p##P##q##Q##_gfx950<<<grid, block, 0, stream>>>(a, x, stride, nc);         \
    }                                                                                                                 \
  } while (0)
  if (q > 2u) NETRA_RUN(2, 4);
  else if (q == 2u) NETRA_RUN(2, 2);
  else if (wide) NETRA_RUN(2, 1);
  else NETRA_RUN(1, 1);
#undef NETRA_RUN
}

// An operand of the weight gradient as it is, or as bf16 with aligned rows in the workspace.
bool outer_ready(const void* m, uint32_t type, uint64_t stride, uint32_t cols) {
  return type == NETRA_BF16 && aligned(m, 16) && cols % 8u == 0 && stride % 8u == 0 && stride < (1u << 24);
}
const uint16_t* outer_operand(const void* m, uint32_t type, uint64_t& stride, uint32_t rows, uint32_t cols,
                              uint8_t*& at, hipStream_t stream) {
  if (outer_ready(m, type, stride, cols)) return static_cast<const uint16_t*>(m);
  const uint32_t pitch = up(cols, 8u);
  const dim3 grid((pitch + 511u) / 512u, rows < 4u * 4096u ? (rows + 3u) / 4u : 4096u);
  uint16_t* out = reinterpret_cast<uint16_t*>(at);
  if (type == NETRA_F32)
    netra_linear_to_bf16_f32_gfx950<<<grid, dim3(256), 0, stream>>>(static_cast<const float*>(m), stride, out, rows,
                                                                    cols, pitch);
  else
    netra_linear_to_bf16_bf16_gfx950<<<grid, dim3(256), 0, stream>>>(static_cast<const uint16_t*>(m), stride, out,
                                                                     rows, cols, pitch);
  at += static_cast<uint64_t>(rows) * pitch * 2u;
  stride = pitch;
  return out;
}

// Tile and split of the weight gradient.
struct OuterPlan {
  uint32_t p, q;  // columns of x and of dy per workgroup
  uint32_t splits, split_rows;
};
OuterPlan outer_plan(uint32_t rows, uint32_t n, uint32_t k) {
  auto tiles = [&](uint32_t p, uint32_t q) { return static_cast<uint64_t>((k + p - 1u) / p) * ((n + q - 1u) / q); };
  OuterPlan plan{256, 256, 1, 0};
  if (tiles(256, 256) < 200) plan = {128, 256, 1, 0};
  if (tiles(128, 256) < 200) plan = {128, 128, 1, 0};
  const uint64_t t = tiles(plan.p, plan.q);
  uint32_t splits = t >= 200 ? 1u : static_cast<uint32_t>(256 / t);
  const uint32_t most = (rows + 255u) / 256u;  // 256 tokens at least
  splits = splits < 1u ? 1u : splits > most ? most : splits;
  plan.split_rows = up((rows + splits - 1u) / splits, 64u);
  plan.splits = (rows + plan.split_rows - 1u) / plan.split_rows;
  return plan;
}

bool bad_workspace(const void* p, uint64_t bytes, uint64_t need) {
  return bytes < need || (need && (!p || !aligned(p, 16)));
}

}  // namespace

extern "C" uint64_t netra_linear_packed_bytes(uint32_t n, uint32_t k, uint32_t transpose) {
  return transpose ? code_bytes(k, n) : code_bytes(n, k);
}

extern "C" int netra_linear_pack(const uint8_t* w, uint8_t* packed, uint32_t n, uint32_t k, uint32_t transpose,
                                 hipStream_t stream) {
  if (!w || !packed || w == packed || !aligned(packed, 16) || bad_sizes(0, n, k))
    return fail(-1, "netra_linear_pack", "null, aliased or misaligned pointers, or n / k not in 1 .. 2^21");
  const uint32_t rows = transpose ? k : n, cols = transpose ? n : k;
  netra_linear_pack_gfx950<<<dim3((rows + 15u) / 16u, (blocks(cols) + 3u) / 4u), dim3(256), 0, stream>>>(
      w, packed, n, k, transpose ? 1u : 0u);
  return launched("netra_linear_pack");
}

extern "C" uint64_t netra_linear_forward_workspace(uint32_t rows, uint32_t n, uint32_t k) {
  return product_workspace(rows, n, k);
}
extern "C" uint64_t netra_linear_input_gradient_workspace(uint32_t rows, uint32_t n, uint32_t k) {
  return product_workspace(rows, k, n);
}
extern "C" uint64_t netra_linear_weight_gradient_workspace(uint32_t rows, uint32_t n, uint32_t k) {
  if (rows == 0) return 0;
  const OuterPlan plan = outer_plan(rows, n, k);
  return static_cast<uint64_t>(rows) * (up(n, 8u) + static_cast<uint64_t>(up(k, 8u))) * 2u +
         (plan.splits > 1u ? 4u * static_cast<uint64_t>(plan.splits) * n * k : 0u) + 16u;
}

// in [rows, nc] times the packed matrix P [ni, nc] -> out [rows, ni]
static int times_weights(const char* name, const void* in, uint32_t in_type, uint64_t in_stride, const uint8_t* packed,
                         const float* scale, uint32_t sp_i, uint32_t sp_b, uint16_t* out, uint64_t out_stride,
                         uint32_t rows, uint32_t ni, uint32_t nc, void* workspace,
                         uint64_t workspace_bytes, hipStream_t stream) {
  if (bad_sizes(rows, ni, nc)) return fail(-1, name, "sizes have to be 1 .. 2^21 (rows may be 0)");
  if (rows == 0) {
    g_error.clear();
    return 0;
  }
  if (bad_matrix(in, in_type, in_stride, nc) || bad_matrix(out, NETRA_BF16, out_stride, ni) || !packed ||
      !aligned(packed, 16) || !scale || !aligned(scale, 4))
    return fail(-1, name, "null or misaligned pointer, unknown type, or row stride below the row");
  if (bad_workspace(workspace, workspace_bytes, product_workspace(rows, ni, nc)))
    return fail(-1, name, "workspace too small, null or not 16-byte aligned");
  const ProductPlan plan = product_plan(rows, ni, nc);
  nklin::Product a{};
  a.p = packed;
  a.sp = scale;
  a.sp_i = sp_i;
  a.sp_b = sp_b;
  a.sp_bytes = blocks(ni) * blocks(nc) * 4u;
  a.out = out;
  a.ldo = out_stride;
  a.ni = ni;
  a.nq = rows;
  a.kb = blocks(nc);
  a.vec = aligned(out, 16) && out_stride % 8u == 0;
  a.splits = plan.splits;
  a.split_blocks = plan.split_blocks;
  if (plan.stream) {
    if (in_type == NETRA_BF16) product_stream(a, static_cast<const uint16_t*>(in), in_stride, nc, stream);
    else product_stream(a, static_cast<const float*>(in), in_stride, nc, stream);
    return launched(name);
  }
  uint8_t* q = static_cast<uint8_t*>(workspace);
  float* s = reinterpret_cast<float*>(q + code_bytes(rows, nc));
  quant_rows(in, in_type, in_stride, q, s, rows, nc, stream);
  a.q = q;
  a.sq = s;
  a.sq_b = up(rows, 16u);
  a.partial = reinterpret_cast<float*>(q + (matrix_bytes(rows, nc) + 15u) / 16u * 16u);
  const uint32_t items = ((ni + plan.p - 1u) / plan.p) * ((rows + plan.q - 1u) / plan.q) * plan.splits;
  const dim3 grid((items + 7u) / 8u * 8u), block(512);
  if (plan.p == 256u) netra_linear_product_256x256_gfx950<<<grid, block, 0, stream>>>(a);
  else netra_linear_product_128x128_gfx950<<<grid, block, 0, stream>>>(a);
  if (plan.splits > 1u)
    netra_linear_product_sum_gfx950<<<dim3((ni + 1023u) / 1024u, rows < 4096u ? rows : 4096u), dim3(256), 0, stream>>>(a);
  return launched(name);
}

extern "C" int netra_linear_forward(const void* x, uint32_t x_type, uint64_t x_stride, const uint8_t* packed,
                                    const float* scale, uint16_t* y, uint64_t y_stride, uint32_t rows, uint32_t n,
                                    uint32_t k, void* workspace, uint64_t workspace_bytes,
                                    hipStream_t stream) {
  return times_weights("netra_linear_forward", x, x_type, x_stride, packed, scale, blocks(k), 1u, y, y_stride,
                       rows, n, k, workspace, workspace_bytes, stream);
}

extern "C" int netra_linear_input_gradient(const void* dy, uint32_t dy_type, uint64_t dy_stride,
                                           const uint8_t* packed_t, const float* scale, uint16_t* dx, uint64_t dx_stride,
                                           uint32_t rows, uint32_t n, uint32_t k, void* workspace,
                                           uint64_t workspace_bytes, hipStream_t stream) {
  return times_weights("netra_linear_input_gradient", dy, dy_type, dy_stride, packed_t, scale, 1u, blocks(k), dx,
                       dx_stride, rows, k, n, workspace, workspace_bytes, stream);
}

extern "C" int netra_linear_weight_gradient(const void* dy, uint32_t dy_type, uint64_t dy_stride, const void* x,
                                            uint32_t x_type, uint64_t x_stride, float* dw, uint32_t accumulate,
                                            uint32_t rows, uint32_t n, uint32_t k, void* workspace,
                                            uint64_t workspace_bytes, hipStream_t stream) {
  const char* name = "netra_linear_weight_gradient";
  if (bad_sizes(rows, n, k)) return fail(-1, name, "sizes have to be 1 .. 2^21 (rows may be 0)");
  if (!dw || !aligned(dw, 4)) return fail(-1, name, "null or misaligned dw");
  if (rows == 0) {
    if (!accumulate)
      netra_linear_zero_gfx950<<<dim3(1024), dim3(256), 0, stream>>>(dw, static_cast<uint64_t>(n) * k);
    return launched(name);
  }
  if (bad_matrix(dy, dy_type, dy_stride, n) || bad_matrix(x, x_type, x_stride, k))
    return fail(-1, name, "null or misaligned pointer, unknown type, or row stride below the row");
  if (bad_workspace(workspace, workspace_bytes, netra_linear_weight_gradient_workspace(rows, n, k)))
    return fail(-1, name, "workspace too small, null or not 16-byte aligned");
  uint8_t* at = static_cast<uint8_t*>(workspace);
  const OuterPlan plan = outer_plan(rows, n, k);
  nklin::Outer a{};
  a.dy = outer_operand(dy, dy_type, dy_stride, rows, n, at, stream);
  a.dy_stride = dy_stride;
  a.x = outer_operand(x, x_type, x_stride, rows, k, at, stream);
  a.x_stride = x_stride;
  a.dw = dw;
  a.rows = rows;
  a.n = n;
  a.k = k;
  a.accumulate = accumulate ? 1u : 0u;
  a.splits = plan.splits;
  a.split_rows = plan.split_rows;
  a.partial = reinterpret_cast<float*>(at);
  const uint32_t items = ((k + plan.p - 1u) / plan.p) * ((n + plan.q - 1u) / plan.q) * plan.splits;
  const dim3 grid((items + 7u) / 8u * 8u), block(512);
  if (plan.p == 256u) netra_linear_outer_256x256_gfx950<<<grid, block, 0, stream>>>(a);
  else if (plan.q == 256u) netra_linear_outer_128x256_gfx950<<<grid, block, 0, stream>>>(a);
  else netra_linear_outer_128x128_gfx950<<<grid, block, 0, stream>>>(a);
  if (plan.splits > 1u) {
    const uint64_t quads = (static_cast<uint64_t>(n) * k + 1023u) / 1024u;
    netra_linear_outer_sum_gfx950<<<dim3(static_cast<uint32_t>(quads < 2048u ? quads : 2048u)), dim3(256), 0, stream>>>(
        a);
  }
  return launched(name);
}

// ---- router -------------------------------------------------------------------

static bool bad_router(uint32_t tokens, uint32_t slots, uint32_t experts) {
  return experts == 0 || experts > nkbal::kMaxExperts || static_cast<uint64_t>(tokens) * slots > 0x7fffffffull ||
         tokens > 0x7fffffffu;
}

// Counting is shared out over workgroups of 256 threads where one would take longer
// than a second launch; each counts `each` tokens.
struct CountPlan {
  uint32_t groups, each;
};
static CountPlan count_plan(uint32_t tokens, uint32_t few) {
  if (tokens <= few) return {0, tokens};
  const uint32_t groups = (tokens - 1u) / 256u + 1u;
  CountPlan plan{groups > 64u ? 64u : groups, 0};
  plan.each = (tokens + plan.groups - 1u) / plan.groups;
  return plan;
}
static constexpr uint32_t kFewCounts = 2048;   // tokens one workgroup counts
static constexpr uint32_t kFewBalance = 64;    // tokens one workgroup takes through the loss
static constexpr uint32_t kBalanceGrid = 256;

static uint64_t parts_bytes(const CountPlan& plan, uint32_t experts) {
  return (4u * static_cast<uint64_t>(plan.groups) * (experts + 1u) + 15u) / 16u * 16u;
}

extern "C" uint64_t netra_router_counts_workspace(uint32_t tokens, uint32_t slots, uint32_t experts) {
  return parts_bytes(count_plan(tokens, kFewCounts), experts);
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
  const CountPlan plan = count_plan(tokens, kFewCounts);
  if (plan.groups == 0) {
    netra_router_counts_gfx950<<<dim3(1), dim3(1024), 0, stream>>>(ids, ids_stride, mask, tokens, slots, experts,
                                                                   counts, accumulate ? 1u : 0u);
    return launched(name);
  }
  uint32_t* parts = static_cast<uint32_t*>(workspace);
  netra_router_count_parts_gfx950<<<dim3(plan.groups), dim3(256), 0, stream>>>(ids, ids_stride, mask, tokens, slots,
                                                                               experts, plan.each, parts, nullptr);
  netra_router_count_sum_gfx950<<<dim3((experts + 15u) / 16u), dim3(256), 0, stream>>>(
      parts, plan.groups, experts, counts, accumulate ? 1u : 0u);
  return launched(name);
}

extern "C" uint64_t netra_router_balance_workspace(uint32_t tokens, uint32_t slots, uint32_t experts) {
  const CountPlan plan = count_plan(tokens, kFewBalance);
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
  if (bad_workspace(workspace, workspace_bytes, netra_router_balance_workspace(tokens, slots, experts)))
    return fail(-1, name, "workspace too small, null or not 16-byte aligned");
  const CountPlan plan = count_plan(tokens, kFewBalance);
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
  uint32_t grid = 1;
  if (plan.groups) {
    uint32_t* words = static_cast<uint32_t*>(workspace);
    a.arrived = words;
    a.partial = reinterpret_cast<float*>(words + 4);
    uint32_t* parts = words + 4 + kBalanceGrid;
    a.parts = parts;
    a.groups = plan.groups;
    netra_router_count_parts_gfx950<<<dim3(plan.groups), dim3(256), 0, stream>>>(
        ids, ids_stride, mask, tokens, slots, experts, plan.each, parts, words);
    grid = (tokens + 15u) / 16u;
    grid = grid > kBalanceGrid ? kBalanceGrid : grid;
  }
  const uint32_t es = elem(logits_type);
  const bool vec = experts > 128u && experts % 4u == 0 && aligned(logits, 4u * es) && logits_stride % 4u == 0 &&
                   (!grad || (aligned(grad, 4u * es) && grad_stride % 4u == 0));
#define NETRA_RUN(NAME, V) netra_router_balance_##NAME##_v##V##_gfx950<<<dim3(grid), dim3(1024), 0, stream>>>(a)
#define NETRA_PICK(NAME)                                  \
  if (experts <= 64u) NETRA_RUN(NAME, 1x1);               \
  else if (experts <= 128u) NETRA_RUN(NAME, 2x1);         \
  else if (experts <= 256u && vec) NETRA_RUN(NAME, 4x4);  \
  else if (experts <= 256u) NETRA_RUN(NAME, 4x1);         \
  else if (experts <= 512u && vec) NETRA_RUN(NAME, 8x4);  \
  else if (experts <= 512u) NETRA_RUN(NAME, 8x1);         \
  else if (vec) NETRA_RUN(NAME, 16x4);                    \
  else NETRA_RUN(NAME, 16x1)
  if (logits_type == NETRA_BF16) {
    NETRA_PICK(bf16);
  } else {
    NETRA_PICK(f32);
  }
#undef NETRA_PICK
#undef NETRA_RUN
  return launched(name);
}

extern "C" const char* netra_layers_last_error(void) { return g_error.c_str(); }
