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

// Whether an output shares memory with an input: their byte ranges meet and they are
// not different columns of rows with one stride.
struct Span {
  const void* p;
  uint64_t stride, row, rows;  // bytes, bytes, count
};
bool share(const Span& a, const Span& b) {
  if (a.rows == 0 || b.rows == 0) return false;
  const uint64_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  if (pa + (a.rows - 1u) * a.stride + a.row <= pb || pb + (b.rows - 1u) * b.stride + b.row <= pa) return false;
  if (a.stride != b.stride) return true;
  const uint64_t d = pb >= pa ? (pb - pa) % a.stride : (a.stride - (pa - pb) % a.stride) % a.stride;
  return d < a.row || d + b.row > a.stride;
}

void quant_rows(const void* x, uint32_t type, uint64_t stride, uint8_t* q, float* s, uint32_t rows, uint32_t n,
                hipStream_t stream) {
  const dim3 grid((rows + 15u) / 16u, (blocks(n) + 3u) / 4u), block(256);
  const uint32_t sld = up(rows, 16u);
  if (type == NETRA_BF16)
    netra_linear_quant_rows_bf16_gfx950<<<grid, block, 0, stream>>>(static_cast<const uint16_t*>(x), stride, q, s, rows,
                                                                    n, sld);
  else
    netra_linear_quant_rows_f32_gfx950<<<grid, block, 0, stream>>>(static_cast<const float*>(x), stride, q, s, rows, n,
                                                                   sld);
}

// How a product runs: the streaming kernel, quantising on the way (kFused) or not
// (kStream), or tiles of p x q with splits of the contraction.
enum Form { kFused, kStream, kTiles };
struct ProductPlan {
  Form form;
  uint32_t p, q, splits, split_blocks;
};

// Tiles: time = rounds of workgroups over the 256 CUs x (steps x the step's time + what a
// workgroup takes besides), the step's time hardly depending on how many CUs work (us a step:
// 256x256 1.75, 256x128 1.18, 128x128 0.78, 128x64 0.58, 64x64 0.35, or 0.62 where two workgroups
// share a CU). Splits add a launch and the partial sums' way out and in. Measured as whole calls,
// best and next: T 333, N 2048, K 1024 64x64 10.0 us, 128x64 10.7, 128x128 11.0; T 700, N 2048, K
// 2048 128x64 13.8, 64x64 15.4; T 1500, N 1500, K 1500 128x128 17.3, 64x64 20.4; T 1500, N 4096, K
// 1024 256x128 16.4, 128x128 20.2; T 8192, N 512, K 4096 128x128 40.7, 256x128 in two splits 48.5;
// T 3000, N 6000, K 3000 256x256 81.3, 256x128 83.7, 128x128 92.5; T 4096, N 4096, K 2048 256x256
// 39.8, 256x128 45.9; T 200, N 500, K 8000 64x64 in eight splits 14.6, in two 19.5. The model misses
// by 7% at T 128, N 8192, K 8192: 128x64 in two splits 25.1, 64x64 26.8.
ProductPlan product_tiles(uint32_t rows, uint32_t ni, uint32_t nc) {
  struct Shape {
    uint32_t p, q;
    double step_us, group_us;
  };
  static const Shape shapes[] = {
      {256, 256, 1.75, 3.0}, {256, 128, 1.18, 2.0}, {128, 128, 0.78, 1.5}, {128, 64, 0.58, 1.2}, {64, 64, 0.35, 1.0}};
  const uint32_t kb = blocks(nc);
  ProductPlan best{kTiles, 256, 256, 1, kb};
  double best_us = 1e30;
  for (const Shape& s : shapes) {
    const uint64_t tiles = static_cast<uint64_t>((ni + s.p - 1u) / s.p) * ((rows + s.q - 1u) / s.q);
    for (uint32_t splits = 1; splits <= 8u && splits <= (kb + 3u) / 4u; splits *= 2u) {
      if (splits > 1u && tiles * splits > 512u) break;
      const uint32_t each = (kb + splits - 1u) / splits, n = (kb + each - 1u) / each;
      const bool pairs = s.p * s.q == 64u * 64u && tiles * n > 256u;
      const double rounds = static_cast<double>(pairs ? (tiles * n + 511u) / 512u : (tiles * n + 255u) / 256u);
      double us = rounds * (each * (pairs ? 0.62 : s.step_us) + s.group_us);
      if (n > 1u) us += 3.0 + static_cast<double>(rows) * ni * (8.0 * n) / 5e6;  // 5 TB/s
      if (us < best_us) {
        best_us = us;
        best = {kTiles, s.p, s.q, n, each};
      }
    }
  }
  return best;
}

ProductPlan product_plan(uint32_t rows, uint32_t ni, uint32_t nc, uint32_t in_type) {
  if (rows > 64u) return product_tiles(rows, ni, nc);
  // Quantising on the way saves a launch (10.7 us -> 6.7 at one row) and costs every
  // workgroup the quantisation of its waves' blocks: 16-row tiles x blocks per wave x
  // workgroups per CU, of which seven cost what the launch does (T 48, N 4096, K 2048, six:
  // 10.3 us against 10.7; T 64, eight: 11.7 against 10.8; T 32, N 8192, K 8192, sixteen: 23.5
  // against 17.5). One tile of rows always quantises on the way: at worst it costs 3% (T 16, N
  // 28672, K 8192: 50.5 us, with the launch 49.0), few rows gain most (T 1: 40.2 against 48.6).
  const uint32_t pt = (ni + 15u) / 16u, q = (rows + 15u) / 16u;
  const uint32_t groups = pt >= 512u ? (pt + 1u) / 2u : pt;
  const uint64_t cost = static_cast<uint64_t>((groups + 255u) / 256u) * q * ((blocks(nc) + 7u) / 8u);
  return {q == 1u || (cost < 8u && (q == 2u || in_type == NETRA_BF16)) ? kFused : kStream, 0, 0, 1, 0};
}
uint64_t product_workspace(uint32_t rows, uint32_t ni, uint32_t nc, uint32_t in_type) {
  if (rows == 0) return 0;
  const ProductPlan plan = product_plan(rows, ni, nc, in_type);
  if (plan.form == kFused) return 0;
  const uint64_t partial = plan.splits > 1u ? 4u * static_cast<uint64_t>(plan.splits) * rows * up(ni, 4u) : 0u;
  return (matrix_bytes(rows, nc) + 15u) / 16u * 16u + partial;
}

template <typename X>
void product_fused(const nklin::Product& a, const X* x, uint64_t stride, uint32_t nc, hipStream_t stream) {
  const uint32_t pt = (a.ni + 15u) / 16u, q = (a.nq + 15u) / 16u;
  // two tiles of columns per workgroup halve the quantisation (T 16, N 8192, K 8192: 21.7 us -> 16.2)
  const bool wide = q <= 2u && pt >= 512u;
  const dim3 grid(wide ? (pt + 1u) / 2u : pt), block(512);
#define NETRA_RUN(P, Q)                                                                                          \
  do {                                                                                                           \
    if constexpr (sizeof(X) == 2)                                                                                \
      netra_linear_product_fused_bf16_p##P##q##Q##_gfx950<<<grid, block, 0, stream>>>(a, x, stride, nc);         \
    else netra_linear_product_fused_f32_p##P##q##Q##_gfx950<<<grid, block, 0, stream>>>(a, x, stride, nc);       \
  } while (0)
  if (q > 2u) {
    if constexpr (sizeof(X) == 2) netra_linear_product_fused_bf16_p1q4_gfx950<<<grid, block, 0, stream>>>(a, x, stride, nc);
  } else if (q == 2u && wide) NETRA_RUN(2, 2);
  else if (q == 2u) NETRA_RUN(1, 2);
  else if (wide) NETRA_RUN(2, 1);
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
  const uint32_t pitch = up(cols, 8u), down = rows < 4u * 4096u ? (rows + 3u) / 4u : 4096u;
  uint16_t* out = reinterpret_cast<uint16_t*>(at);
  copy = {m, stride, out, type, cols, pitch, (pitch + 511u) / 512u * down};
  at += static_cast<uint64_t>(rows) * pitch * 2u;
  stride = cols = pitch;
  return out;
}

// Tile and split of the weight gradient, chosen as product_tiles' (steps of 64 tokens: 256x256
// 1.55 us, 128x256 0.93, 128x128 0.48, one workgroup per CU each). As whole calls, best and
// next: T 333, N 1024, K 2048 128x128 8.3 us, 128x256 11.8; T 4096, N 4096, K 2048 128x256 64,
// 128x128 82; T 4096, N 1024, K 1024 128x128 in four splits 21.3, in two 23.9; T 8192, N 4096,
// K 4096 256x256 216, 128x256 249.
struct OuterPlan {
  uint32_t p, q;  // columns of x and of dy per workgroup
  uint32_t splits, split_rows;
};
OuterPlan outer_plan(uint32_t rows, uint32_t n, uint32_t k) {
  struct Shape {
    uint32_t p, q;
    double step_us;
  };
  static const Shape shapes[] = {{256, 256, 1.55}, {128, 256, 0.93}, {128, 128, 0.48}};
  const uint32_t steps = (rows + 63u) / 64u;
  OuterPlan best{256, 256, 1, up(rows, 64u)};
  double best_us = 1e30;
  for (const Shape& s : shapes) {
    const uint64_t tiles = static_cast<uint64_t>((k + s.p - 1u) / s.p) * ((n + s.q - 1u) / s.q);
    for (uint32_t splits = 1; splits <= 16u && splits <= (steps + 3u) / 4u; splits *= 2u) {
      if (splits > 1u && tiles * splits > 512u) break;
      const uint32_t each = (steps + splits - 1u) / splits, count = (steps + each - 1u) / each;
      double us = static_cast<double>((tiles * count + 255u) / 256u) * each * s.step_us;
      if (count > 1u) us += 3.0 + static_cast<double>(n) * k * 4.0 * (2.0 * count + 1.0) / 6e6;  // 6 TB/s
      if (us < best_us) {
        best_us = us;
        best = {s.p, s.q, count, each * 64u};
      }
    }
  }
  return best;
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
  if (transpose)
    netra_linear_pack_transposed_gfx950<<<dim3((k + 63u) / 64u, blocks(n)), dim3(256), 0, stream>>>(w, packed, n, k);
  else
    netra_linear_pack_gfx950<<<dim3((n + 15u) / 16u, (blocks(k) + 3u) / 4u), dim3(256), 0, stream>>>(w, packed, n, k);
  return launched("netra_linear_pack");
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

static void quantise(const ProductCall& c, const ProductPlan& plan, uint8_t* workspace, hipStream_t stream) {
  if (plan.form != kFused)
    quant_rows(c.in, c.in_type, c.in_stride, workspace, reinterpret_cast<float*>(workspace + code_bytes(c.rows, c.nc)),
               c.rows, c.nc, stream);
}

static uint32_t groups_of(const nklin::Product& a, const ProductPlan& plan) {
  const uint32_t items = ((a.ni + plan.p - 1u) / plan.p) * ((a.nq + plan.q - 1u) / plan.q) * plan.splits;
  return (items + 7u) / 8u * 8u;
}

static void run(const ProductCall& c, const nklin::Product& a, const ProductPlan& plan, hipStream_t stream) {
  if (plan.form == kFused) {
    if (c.in_type == NETRA_BF16)
      return product_fused(a, static_cast<const uint16_t*>(c.in), c.in_stride, c.nc, stream);
    return product_fused(a, static_cast<const float*>(c.in), c.in_stride, c.nc, stream);
  }
  const dim3 block(512);
  if (plan.form == kStream) {
    const uint32_t pt = (a.ni + 15u) / 16u;
    const bool wide = pt >= 512u;  // the activations are read half as often (T 64, N 8192, K 8192: 24.1 us -> 20.3)
    const dim3 grid(wide ? (pt + 1u) / 2u : pt);
    if (wide) netra_linear_product_stream_p2q4_gfx950<<<grid, block, 0, stream>>>(a);
    else netra_linear_product_stream_p1q4_gfx950<<<grid, block, 0, stream>>>(a);
    return;
  }
  const dim3 grid(groups_of(a, plan));
  if (plan.p == 256u && plan.q == 256u) netra_linear_product_256x256_gfx950<<<grid, block, 0, stream>>>(a);
  else if (plan.p == 256u) netra_linear_product_256x128_gfx950<<<grid, block, 0, stream>>>(a);
  else if (plan.q == 128u) netra_linear_product_128x128_gfx950<<<grid, block, 0, stream>>>(a);
  else if (plan.p == 128u) netra_linear_product_128x64_gfx950<<<grid, block, 0, stream>>>(a);
  else netra_linear_product_64x64_gfx950<<<grid, block, 0, stream>>>(a);
  if (plan.splits > 1u)
    netra_linear_product_sum_gfx950<<<dim3((a.ni + 1023u) / 1024u, a.nq < 4096u ? a.nq : 4096u), dim3(256), 0, stream>>>(
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
  const ProductPlan plan = product_plan(c.rows, c.ni, c.nc, c.in_type);
  nklin::Product a{};
  set_up(c, plan, static_cast<uint8_t*>(workspace), a);
  quantise(c, plan, static_cast<uint8_t*>(workspace), stream);
  run(c, a, plan, stream);
  return launched(c.name);
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
static void prepare(const OuterCall& c, const nklin::Copy (&copies)[2], uint8_t* codes, hipStream_t stream) {
  const uint32_t quant = codes ? (c.rows + 15u) / 16u * ((blocks(c.n) + 3u) / 4u) : 0u;
  const dim3 grid(quant + copies[0].groups + copies[1].groups), block(256);
  float* s = codes ? reinterpret_cast<float*>(codes + code_bytes(c.rows, c.n)) : nullptr;
  const uint32_t sld = up(c.rows, 16u);
  if (c.dy_type == NETRA_BF16)
    netra_linear_prepare_bf16_gfx950<<<grid, block, 0, stream>>>(static_cast<const uint16_t*>(c.dy), c.dy_stride, codes,
                                                                 s, c.rows, c.n, sld, quant, copies[0], copies[1]);
  else
    netra_linear_prepare_f32_gfx950<<<grid, block, 0, stream>>>(static_cast<const float*>(c.dy), c.dy_stride, codes, s,
                                                                c.rows, c.n, sld, quant, copies[0], copies[1]);
}

static uint32_t groups_of(const nklin::Outer& a, const OuterPlan& plan) {
  const uint32_t items = ((a.k + plan.p - 1u) / plan.p) * ((a.n + plan.q - 1u) / plan.q) * plan.splits;
  return (items + 7u) / 8u * 8u;
}

static void sum(const nklin::Outer& a, hipStream_t stream) {
  if (a.splits == 1u) return;
  const uint64_t quads = (static_cast<uint64_t>(a.n) * a.k + 1023u) / 1024u;
  netra_linear_outer_sum_gfx950<<<dim3(static_cast<uint32_t>(quads < 2048u ? quads : 2048u)), dim3(256), 0, stream>>>(a);
}

static void run(const nklin::Outer& a, const OuterPlan& plan, hipStream_t stream) {
  const dim3 grid(groups_of(a, plan)), block(512);
  if (plan.p == 256u) netra_linear_outer_256x256_gfx950<<<grid, block, 0, stream>>>(a);
  else if (plan.q == 256u) netra_linear_outer_128x256_gfx950<<<grid, block, 0, stream>>>(a);
  else netra_linear_outer_128x128_gfx950<<<grid, block, 0, stream>>>(a);
  sum(a, stream);
}

// Sizes and dw, and the call without tokens: 0 or an error to return, or 1 to go on.
static int outer_start(const OuterCall& c, hipStream_t stream) {
  if (bad_sizes(c.rows, c.n, c.k)) return fail(-1, c.name, "sizes have to be 1 .. 2^21 (rows may be 0)");
  if (!c.dw || !aligned(c.dw, 4)) return fail(-1, c.name, "null or misaligned dw");
  if (c.rows != 0) return 1;
  if (!c.accumulate)
    netra_linear_zero_gfx950<<<dim3(1024), dim3(256), 0, stream>>>(c.dw, static_cast<uint64_t>(c.n) * c.k);
  return launched(c.name);
}

extern "C" int netra_linear_weight_gradient(const void* dy, uint32_t dy_type, uint64_t dy_stride, const void* x,
                                            uint32_t x_type, uint64_t x_stride, float* dw, uint32_t accumulate,
                                            uint32_t rows, uint32_t n, uint32_t k, void* workspace,
                                            uint64_t workspace_bytes, hipStream_t stream) {
  const OuterCall c{"netra_linear_weight_gradient", dy, dy_type, dy_stride, x, x_type, x_stride, dw, accumulate, rows,
                    n, k};
  int rc = outer_start(c, stream);
  if (rc != 1) return rc;
  rc = check(c);
  if (rc != 0) return rc;
  const OuterPlan plan = outer_plan(rows, n, k);
  if (bad_workspace(workspace, workspace_bytes, outer_workspace(c, plan)))
    return fail(-1, c.name, "workspace too small, null or not 16-byte aligned");
  nklin::Outer a{};
  nklin::Copy copies[2] = {};
  set_up(c, plan, static_cast<uint8_t*>(workspace), a, copies);
  if (copies[0].groups + copies[1].groups) prepare(c, copies, nullptr, stream);
  run(a, plan, stream);
  return launched(c.name);
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
  int rc = outer_start(o, stream);
  if (rc != 1) return rc;
  if ((rc = check(p)) != 0 || (rc = check(o)) != 0) return rc;
  const uint64_t dw_bytes = static_cast<uint64_t>(n) * k * 4u;
  if (share({dx, dx_stride * 2u, static_cast<uint64_t>(k) * 2u, rows}, {dw, dw_bytes, dw_bytes, 1}) ||
      share({dx, dx_stride * 2u, static_cast<uint64_t>(k) * 2u, rows},
            {x, x_stride * elem(x_type), static_cast<uint64_t>(k) * elem(x_type), rows}))
    return fail(-1, name, "dx shares memory with x or dw");
  ProductPlan product = product_plan(rows, k, n, dy_type);
  const OuterPlan outer = outer_plan(rows, n, k);
  const uint64_t first = (product_workspace(rows, k, n, dy_type) + 15u) / 16u * 16u;
  if (bad_workspace(workspace, workspace_bytes, first + outer_workspace(o, outer)))
    return fail(-1, name, "workspace too small, null or not 16-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  // Passes of small tiles run both products in one launch (T 333, N 1024, K 2048 13.3 us, in two
  // 16.9; T 3584, N 360, K 189 16.3, 20.7; T 1200, N 1000, K 1000 18.3, 24.5; T 3000, N 500, K 500
  // 21.3, 24.1); with larger tiles most lose by it (T 5000, N 600, K 1000 36.6, 33.5).
  const bool small = product.form == kTiles && product.p * product.q <= 128u * 64u && product.splits == 1u &&
                     outer.p * outer.q == 128u * 128u;
  if (small) product.p = product.q = 64u;
  nklin::Product a{};
  nklin::Outer b{};
  nklin::Copy copies[2] = {};
  set_up(p, product, ws, a);
  set_up(o, outer, ws + first, b, copies);
  if (copies[0].groups + copies[1].groups) prepare(o, copies, product.form == kFused ? nullptr : ws, stream);
  else quantise(p, product, ws, stream);
  if (small) {
    const uint32_t groups = groups_of(b, outer);
    netra_linear_backward_small_gfx950<<<dim3(groups + groups_of(a, product)), dim3(512), 0, stream>>>(a, b, groups);
    sum(b, stream);
  } else {
    run(p, a, product, stream);
    run(b, outer, stream);
  }
  return launched(name);
}

// ---- router -------------------------------------------------------------------

static bool bad_router(uint32_t tokens, uint32_t slots, uint32_t experts) {
  return experts == 0 || experts > nkbal::kMaxExperts || static_cast<uint64_t>(tokens) * slots > 0x7fffffffull ||
         tokens > 0x7fffffffu;
}

// Counting is shared out over workgroups of 256 threads where one would take longer
// than a second launch; each counts `each` tokens, one a thread while `most` workgroups reach (the
// loss kernel's workgroups all add up all parts: few of them, with more threads).
struct CountPlan {
  uint32_t groups, each;
};
static CountPlan count_plan(uint32_t tokens, uint32_t few, uint32_t most) {
  if (tokens <= few) return {0, tokens};
  const uint32_t groups = (tokens - 1u) / 256u + 1u;
  CountPlan plan{groups > most ? most : groups, 0};
  plan.each = (tokens + plan.groups - 1u) / plan.groups;
  return plan;
}
// Tokens one workgroup counts (1024 of 9 ids: 7.3 us, in two launches 9.5; 2048: 10.0, 9.5; 3500:
// 14.2, 9.6).
static constexpr uint32_t kFewCounts = 2048;
static constexpr uint32_t kBalanceGrid = 256;
// One workgroup takes 32768 logits through the loss, 256 tokens at most (128 x 256: 11.7 us, shared
// out 13.6; 256 x 16: 9.9, 13.6; 512 x 16: 13.3, 13.7; 64 x 512: 11.2, 13.6; 64 x 1024: 16.0, 13.6).
// More parts than 64 cost their summing up what they gain (32768 x 256 24.1 us with 128, 24.7 with
// 64; x 500 33.8, 32.3; with 32 27.7, 32.9).
static CountPlan balance_plan(uint32_t tokens, uint32_t experts) {
  const uint32_t few = 32768u / (experts ? experts : 1u);
  return count_plan(tokens, few < 256u ? few : 256u, 64u);
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
  uint32_t grid = 1;
  if (plan.groups) {
    uint32_t* words = static_cast<uint32_t*>(workspace);
    a.arrived = words;
    a.partial = reinterpret_cast<float*>(words + 4);
    uint32_t* parts = words + 4 + kBalanceGrid;
    a.parts = parts;
    a.groups = plan.groups;
    netra_router_count_parts_gfx950<<<dim3(plan.groups), dim3(plan.each > 256u ? 1024 : 256), 0, stream>>>(
        ids, ids_stride, mask, tokens, slots, experts, plan.each, parts, words);
    // Rows per pass of a workgroup. (Workgroups of 512 threads: 32768 x 256 bf16 26.8 us, of 1024 24.6.)
    const uint32_t rows = experts <= 256u ? 64u : 16u;
    grid = (tokens - 1u) / rows + 1u;
    grid = grid > kBalanceGrid ? kBalanceGrid : grid;
  }
#define NETRA_RUN(NAME, F) netra_router_balance_##NAME##_##F##_gfx950<<<dim3(grid), dim3(1024), 0, stream>>>(a)
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
  return launched(name);
}

extern "C" const char* netra_layers_last_error(void) { return g_error.c_str(); }
