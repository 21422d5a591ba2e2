// Root-mean-square norm with the residual's addition and an output in 8 bits, and its gradients.
//
//   r = x + residual (rounded to the residual's type), rstd = 1 / sqrt(mean(r^2) + eps),
//   y = r * rstd * (w + offset); codes and scales of y by the layer's 1x128 rule.
//   Gradients: g = dy (w + offset), xh = r rstd, c = mean(g xh):
//   dr = rstd (g - xh c) + (what flows into r besides),  dw = sum over the rows of dy xh.
//
// A row is held in registers by W waves (eight neighbouring columns a lane, C times), so it is
// read once; sums are fp32. y is quantised as it stands in fp32, not after its rounding to bf16:
// one rounding instead of two. Memory bounds both: T 16384, H 4096 with residual and codes 110 us
// (606 MB, 5.5 TB/s), its gradients 87 and 4.8 for dw's sum (537 MB); a large copy runs at 5.1. Few rows are a launch: T 1,
// H 2048 2.2 us, T 333 4.4 and 3.5.
#pragma once
#include "linear_fp8.hip"
#include "router_balance.hip"

namespace nknorm {

using nk::u32x2;
using nk::u32x4;

constexpr int kNowhere = (int)0x80000000u;
constexpr uint32_t kMaxCols = 16384;

// Eight neighbouring values of a row as they lie in memory.
template <typename X>
struct Eight;
template <>
struct Eight<uint16_t> {
  u32x4 w;
  uint32_t last;  // the row's last value where its length is odd
};
template <>
struct Eight<float> {
  u32x4 lo, hi;
};

// A row's descriptor: the range is checked per dword, so an odd bf16 row's last value is outside
// it and has a load and a store of its own. rows past the end have no bytes: loads give zeros.
template <typename X>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(const void* m, uint64_t stride, uint32_t row, uint32_t cols,
                                                           bool there) {
  return nk::buffer_rsrc(static_cast<const X*>(m) + (there ? (uint64_t)row * stride : 0u),
                         there ? cols * (uint32_t)sizeof(X) : 0u);
}

// kOnce: non-temporal loads and stores.
template <typename X, bool kOnce = false>
__device__ __forceinline__ Eight<X> load8(__amdgpu_buffer_rsrc_t r, uint32_t c, uint32_t cols) {
  constexpr int kAux = kOnce ? 2 : 0;
  Eight<X> v;
  if constexpr (sizeof(X) == 4) {
    v.lo = __builtin_amdgcn_raw_buffer_load_b128(r, (int)(c * 4u), 0, kAux);
    v.hi = __builtin_amdgcn_raw_buffer_load_b128(r, (int)(c * 4u + 16u), 0, kAux);
  } else {
    v.w = __builtin_amdgcn_raw_buffer_load_b128(r, (int)(c * 2u), 0, kAux);
    const bool mine = (cols & 1u) && c < cols && c + 8u > cols;
    v.last = (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, mine ? (int)((cols - 1u) * 2u) : kNowhere, 0, 0);
  }
  return v;
}

template <typename X>
__device__ __forceinline__ void values(const Eight<X>& v, uint32_t c, uint32_t cols, float (&f)[8]) {
  if constexpr (sizeof(X) == 4) {
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
      f[i] = __uint_as_float(v.lo[i]);
      f[4u + i] = __uint_as_float(v.hi[i]);
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
      f[2u * i] = nk::bf16_lo(c + 2u * i + 1u == cols ? v.last : v.w[i]);
      f[2u * i + 1u] = nk::bf16_hi(v.w[i]);
    }
  }
}

template <typename X, bool kOnce = false>
__device__ __forceinline__ void store8(__amdgpu_buffer_rsrc_t r, uint32_t c, uint32_t cols, const float (&f)[8]) {
  constexpr int kAux = kOnce ? 2 : 0;
  if constexpr (sizeof(X) == 4) {
    u32x4 lo, hi;
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
      lo[i] = __float_as_uint(f[i]);
      hi[i] = __float_as_uint(f[4u + i]);
    }
    __builtin_amdgcn_raw_buffer_store_b128(lo, r, (int)(c * 4u), 0, kAux);
    __builtin_amdgcn_raw_buffer_store_b128(hi, r, (int)(c * 4u + 16u), 0, kAux);
  } else {
    u32x4 w;
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) w[i] = nk::bf16x2_hw(f[2u * i], f[2u * i + 1u]);
    __builtin_amdgcn_raw_buffer_store_b128(w, r, (int)(c * 2u), 0, kAux);
    if (cols & 1u) {
      const uint32_t i = (cols - 1u - c) / 2u;  // the dword that the row's last value begins
#pragma unroll
      for (uint32_t j = 0; j < 4u; ++j)
        if (c < cols && i == j) __builtin_amdgcn_raw_buffer_store_b16((uint16_t)w[j], r, (int)((cols - 1u) * 2u), 0, 0);
    }
  }
}

// w + offset, eight columns from c; the type is an argument (both loads are made, one of them of
// nothing), as the weights are read once and not per row.
__device__ __forceinline__ void weights8(const void* w, bool bf16, float offset, uint32_t c, uint32_t cols,
                                         float (&f)[8]) {
  const Eight<uint16_t> h = load8<uint16_t>(nk::buffer_rsrc(w, bf16 ? cols * 2u : 0u), c, cols);
  const Eight<float> s = load8<float>(nk::buffer_rsrc(w, bf16 ? 0u : cols * 4u), c, cols);
  float a[8], b[8];
  values(h, c, cols, a);
  values(s, c, cols, b);
#pragma unroll
  for (uint32_t i = 0; i < 8u; ++i) f[i] = (bf16 ? a[i] : b[i]) + offset;
}

// The sum over a row's W waves in every lane, in one order. `part`: 2 W floats; the rows of a
// workgroup take its halves in turn, so one barrier a row is enough.
template <uint32_t W>
__device__ __forceinline__ float row_sum(float v, float* part, uint32_t turn) {
  v = nkbal::sum<64>(v);
  if constexpr (W == 1u) return v;
  const uint32_t wave = threadIdx.x >> 6;
  float* s = part + (turn & 1u) * W;
  if ((threadIdx.x & 63u) == 0u) s[wave] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (uint32_t i = 1; i < W; ++i) v += s[i];
  return v;
}

// Largest magnitude's bits over 16 lanes.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
#define NETRA_DPP(CTRL) (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false)
  v = max(v, NETRA_DPP(0xB1));
  v = max(v, NETRA_DPP(0x4E));
  v = max(v, NETRA_DPP(0x141));
  v = max(v, NETRA_DPP(0x140));
#undef NETRA_DPP
  return v;
}

enum Codes { kNone, kRows, kTiles };

struct Norm {
  const void* x;
  uint64_t x_stride;
  const void* residual;       // null: none
  uint64_t residual_stride;
  const void* w;
  uint32_t w_bf16;
  float offset, eps, inv_cols;
  void* sum;                  // r, of the residual's type; null where there is no residual
  uint64_t sum_stride;
  void* y;                    // null: none
  uint32_t y_bf16;
  uint64_t y_stride;
  uint8_t* codes;             // kRows: [rows, cols]; kTiles: tile16x128
  float* scales;              // kRows: [rows, blocks]; kTiles: [blocks, scales_ld]
  uint32_t layout, scales_ld;
  uint32_t rows, cols, all_rows;  // all_rows: with the last tile's empty ones
};

// Codes of eight columns, and their group's scale by its first lane.
template <bool kOnce>
__device__ __forceinline__ void quantise8(const Norm& a, uint32_t row, uint32_t c, const float (&y)[8]) {
  uint32_t m = 0u;
#pragma unroll
  for (uint32_t i = 0; i < 8u; ++i) m = max(m, __float_as_uint(y[i]) & 0x7fffffffu);
  m = max16(m);
  const uint32_t kb = (a.cols + 127u) / 128u, b = c / 128u;
  if (b >= kb) return;
  const float scale = nklin::group_scale(m), inv = 1.0f / scale;
  u32x2 q;
#pragma unroll
  for (uint32_t i = 0; i < 2u; ++i) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[4u * i] * inv, y[4u * i + 1u] * inv, 0, false);
    q[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4u * i + 2u] * inv, y[4u * i + 3u] * inv, lo, true);
  }
  const bool first = (threadIdx.x & 15u) == 0u;
  if (a.layout == kTiles) {
    const uint32_t in = c % 128u;
    uint8_t* tile = a.codes + ((size_t)(row / 16u) * kb + b) * 2048u;
    *reinterpret_cast<u32x2*>(tile + in % 32u / 16u * 1024u + ((row & 15u) + 16u * (in / 32u)) * 16u + in % 16u) = q;
    if (first) a.scales[(size_t)b * a.scales_ld + row] = scale;
    return;
  }
  const __amdgpu_buffer_rsrc_t r = nk::buffer_rsrc(a.codes + (uint64_t)row * a.cols, a.cols & ~3u);
  __builtin_amdgcn_raw_buffer_store_b64(q, r, (int)c, 0, kOnce ? 2 : 0);
  if (a.cols & 3u) {
    const uint32_t from = a.cols & ~3u;  // the last one to three columns, by the lane that has them
    if (from / 8u * 8u == c) {
      const uint32_t v = from & 4u ? q[1] : q[0];
      uint8_t* end = a.codes + (uint64_t)row * a.cols + from;
#pragma unroll
      for (uint32_t i = 0; i < 3u; ++i)
        if (from + i < a.cols) end[i] = (uint8_t)(v >> (8u * i));
    }
  }
  if (first) a.scales[(size_t)row * kb + b] = scale;
}

// Rows that a workgroup holds at once: with one wave a row, four.
template <uint32_t W>
struct Shape {
  static constexpr uint32_t kRows = W == 1u ? 4u : 1u, kThreads = W == 1u ? 256u : 64u * W;
};

// kOnce, where all that goes in and out is more than the 256 MiB behind the L2s hold: x and the residual are
// not kept there, nor the outputs. T 16384, H 4096 with residual and codes (606 MB): 117.3 us, with loads alone
// non-temporal 112.9, stores alone 113.9, both 110.3 (5.5 TB/s; a large copy 5.1); T 4096 (151 MB) 27.1, both 31.0.
template <typename X, typename R, uint32_t W, uint32_t C, bool kOnce>
__device__ __forceinline__ void forward(const Norm& a) {
  __shared__ float part[2u * W];
  constexpr uint32_t kRows = Shape<W>::kRows;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t at = (W == 1u ? threadIdx.x & 63u : threadIdx.x) * 8u, step = (W == 1u ? 64u : 64u * W) * 8u;
  float w[C][8];
  auto load = [&](uint32_t row, Eight<X> (&x)[C], Eight<R> (&res)[C]) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t rx = row_rsrc<X>(a.x, a.x_stride, row, a.cols, row < a.rows);
    const __amdgpu_buffer_rsrc_t rr =
        row_rsrc<R>(a.residual, a.residual_stride, row, a.cols, row < a.rows && a.residual != nullptr);
#pragma unroll
    for (uint32_t k = 0; k < C; ++k) {
      x[k] = load8<X, kOnce>(rx, at + k * step, a.cols);
      res[k] = load8<R, kOnce>(rr, at + k * step, a.cols);
    }
  };
  uint32_t row = blockIdx.x * kRows + (W == 1u ? wave : 0u), turn = 0u;
  Eight<X> x[C];
  Eight<R> res[C];
  load(row, x, res);
#pragma unroll
  for (uint32_t k = 0; k < C; ++k) weights8(a.w, a.w_bf16 != 0u, a.offset, at + k * step, a.cols, w[k]);
  for (; row < a.all_rows; row += gridDim.x * kRows) {
    float r[C][8], sum = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < C; ++k) {
      const uint32_t c = at + k * step;
      float f[8];
      values(x[k], c, a.cols, r[k]);
      values(res[k], c, a.cols, f);
      if (a.residual) {
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) {
          r[k][i] += f[i];
          if constexpr (sizeof(R) == 2) r[k][i] = nk::bf16_round_hw(r[k][i]);
        }
      }
#pragma unroll
      for (uint32_t i = 0; i < 8u; ++i) sum = fmaf(r[k][i], r[k][i], sum);
    }
    const uint32_t next = row + gridDim.x * kRows;
    load(next, x, res);  // rows past the end: no bytes
    sum = row_sum<W>(sum, part, turn++);
    const float rstd = 1.0f / sqrtf(fmaf(sum, a.inv_cols, a.eps));
    const bool there = row < a.rows;
    if (a.residual && there) {
      const __amdgpu_buffer_rsrc_t rs = row_rsrc<R>(a.sum, a.sum_stride, row, a.cols, true);
#pragma unroll
      for (uint32_t k = 0; k < C; ++k) store8<R, kOnce>(rs, at + k * step, a.cols, r[k]);
    }
#pragma unroll
    for (uint32_t k = 0; k < C; ++k)
#pragma unroll
      for (uint32_t i = 0; i < 8u; ++i) r[k][i] = there ? r[k][i] * rstd * w[k][i] : 0.0f;
    if (a.y && there) {
      if (a.y_bf16) {
        const __amdgpu_buffer_rsrc_t ry = row_rsrc<uint16_t>(a.y, a.y_stride, row, a.cols, true);
#pragma unroll
        for (uint32_t k = 0; k < C; ++k) store8<uint16_t, kOnce>(ry, at + k * step, a.cols, r[k]);
      } else {
        const __amdgpu_buffer_rsrc_t ry = row_rsrc<float>(a.y, a.y_stride, row, a.cols, true);
#pragma unroll
        for (uint32_t k = 0; k < C; ++k) store8<float, kOnce>(ry, at + k * step, a.cols, r[k]);
      }
    }
    if (a.layout != kNone) {
#pragma unroll
      for (uint32_t k = 0; k < C; ++k) quantise8<kOnce>(a, row, at + k * step, r[k]);
    }
  }
}

struct NormGradients {
  const void* dy;
  uint64_t dy_stride;
  const void* r;
  uint64_t r_stride;
  const void* flow;           // gradient that flows into r besides, of r's type; null: none
  uint64_t flow_stride;
  const void* w;
  uint32_t w_bf16;
  float offset, eps, inv_cols;
  void* dr;                   // of r's type
  uint64_t dr_stride;
  float* partial;             // [groups][cols]
  uint32_t rows, cols;
};

// kOnce as above, of the loads alone: T 16384, H 4096 (537 MB) 107.6 us, so 91.5 (5.9 TB/s), with stores too 98.5; T 4096
// (134 MB) 29.4 and 29.9.
template <typename G, typename X, uint32_t W, uint32_t C, bool kOnce>
__device__ __forceinline__ void gradients(const NormGradients& a) {
  __shared__ float part[4u * W];
  constexpr uint32_t kRows = Shape<W>::kRows;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t at = (W == 1u ? threadIdx.x & 63u : threadIdx.x) * 8u, step = (W == 1u ? 64u : 64u * W) * 8u;
  // The next row's values are under way during a row; of the longest rows there are no registers for them.
  constexpr bool kAhead = W * C <= 16u;
  auto load = [&](uint32_t row, Eight<X> (&x)[C], Eight<G> (&g)[C]) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t rx = row_rsrc<X>(a.r, a.r_stride, row, a.cols, row < a.rows);
    const __amdgpu_buffer_rsrc_t rg = row_rsrc<G>(a.dy, a.dy_stride, row, a.cols, row < a.rows);
#pragma unroll
    for (uint32_t k = 0; k < C; ++k) {
      x[k] = load8<X, kOnce>(rx, at + k * step, a.cols);
      g[k] = load8<G, kOnce>(rg, at + k * step, a.cols);
    }
  };
  auto load_flow = [&](uint32_t row, Eight<X> (&flow)[C]) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t rf =
        row_rsrc<X>(a.flow, a.flow_stride, row, a.cols, row < a.rows && a.flow != nullptr);
#pragma unroll
    for (uint32_t k = 0; k < C; ++k) flow[k] = load8<X, kOnce>(rf, at + k * step, a.cols);
  };
  const uint32_t first = blockIdx.x * kRows + (W == 1u ? wave : 0u);
  uint32_t row = first, turn = 0u;
  Eight<X> x[C], flow[C];
  Eight<G> g[C];
  if constexpr (kAhead) {
    load(row, x, g);
    load_flow(row, flow);
  }
  float w[C][8], dw[C][8];
#pragma unroll
  for (uint32_t k = 0; k < C; ++k) {
    weights8(a.w, a.w_bf16 != 0u, a.offset, at + k * step, a.cols, w[k]);
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) dw[k][i] = 0.0f;
  }
  for (; row < a.rows; row += gridDim.x * kRows) {
    float r[C][8], d[C][8], squares = 0.0f, dot = 0.0f;
    Eight<X> f[C];
    if constexpr (!kAhead) load(row, x, g);
#pragma unroll
    for (uint32_t k = 0; k < C; ++k) {
      const uint32_t c = at + k * step;
      values(x[k], c, a.cols, r[k]);
      values(g[k], c, a.cols, d[k]);
#pragma unroll
      for (uint32_t i = 0; i < 8u; ++i) {
        squares = fmaf(r[k][i], r[k][i], squares);
        dot = fmaf(d[k][i] * w[k][i], r[k][i], dot);
      }
    }
    if constexpr (kAhead) {
#pragma unroll
      for (uint32_t k = 0; k < C; ++k) f[k] = flow[k];
      load(row + gridDim.x * kRows, x, g);
      load_flow(row + gridDim.x * kRows, flow);
    } else {
      load_flow(row, f);
    }
    squares = nkbal::sum<64>(squares);
    dot = nkbal::sum<64>(dot);
    if constexpr (W > 1u) {
      float* s = part + (turn++ & 1u) * 2u * W;
      if ((threadIdx.x & 63u) == 0u) {
        s[wave] = squares;
        s[W + wave] = dot;
      }
      __syncthreads();
      squares = s[0];
      dot = s[W];
#pragma unroll
      for (uint32_t i = 1; i < W; ++i) {
        squares += s[i];
        dot += s[W + i];
      }
    }
    const float rstd = 1.0f / sqrtf(fmaf(squares, a.inv_cols, a.eps));
    const float c = dot * rstd * a.inv_cols;  // mean(g xh)
    const __amdgpu_buffer_rsrc_t rd = row_rsrc<X>(a.dr, a.dr_stride, row, a.cols, true);
#pragma unroll
    for (uint32_t k = 0; k < C; ++k) {
      float into[8];
      values(f[k], at + k * step, a.cols, into);
#pragma unroll
      for (uint32_t i = 0; i < 8u; ++i) {
        const float xh = r[k][i] * rstd;
        dw[k][i] = fmaf(d[k][i], xh, dw[k][i]);
        r[k][i] = fmaf(rstd, fmaf(-xh, c, d[k][i] * w[k][i]), into[i]);
      }
      store8<X>(rd, at + k * step, a.cols, r[k]);
    }
  }
  if constexpr (kRows > 1u) {  // the waves' rows together
    __shared__ float s_dw[kRows][C * 512u];
#pragma unroll
    for (uint32_t k = 0; k < C; ++k)
#pragma unroll
      for (uint32_t i = 0; i < 8u; ++i) s_dw[wave][(k * 8u + i) * 64u + (threadIdx.x & 63u)] = dw[k][i];
    __syncthreads();
    if (wave != 0u) return;
#pragma unroll
    for (uint32_t k = 0; k < C; ++k)
#pragma unroll
      for (uint32_t i = 0; i < 8u; ++i)
#pragma unroll
        for (uint32_t v = 1; v < kRows; ++v) dw[k][i] += s_dw[v][(k * 8u + i) * 64u + threadIdx.x];
  }
  const __amdgpu_buffer_rsrc_t rp = nk::buffer_rsrc(a.partial + (uint64_t)blockIdx.x * a.cols, a.cols * 4u);
#pragma unroll
  for (uint32_t k = 0; k < C; ++k) store8<float>(rp, at + k * step, a.cols, dw[k]);
}

// dw = the sum of `parts` partial sums, in one order: a workgroup takes 64 columns, its 16 waves
// every 16th part, eight loads at a time. (At most 512 parts: more of them, summed one load at
// a time, took 88 us where the gradients and their sum now take 10, at T 4943, H 538.)
__device__ __forceinline__ void sum_parts(const float* __restrict__ partial, uint32_t parts, uint32_t cols, float* dw,
                                          uint32_t accumulate) {
  __shared__ float s[16][64];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, c = blockIdx.x * 64u + lane;
  float v = 0.0f;
  if (c < cols)
    for (uint32_t p = wave; p < parts; p += 128u) {
      float f[8];
#pragma unroll
      for (uint32_t i = 0; i < 8u; ++i) f[i] = partial[(uint64_t)min(p + 16u * i, parts - 1u) * cols + c];
#pragma unroll
      for (uint32_t i = 0; i < 8u; ++i) v += p + 16u * i < parts ? f[i] : 0.0f;
    }
  s[wave][lane] = v;
  __syncthreads();
  if (wave != 0u || c >= cols) return;
#pragma unroll
  for (uint32_t p = 1; p < 16u; ++p) v += s[p][lane];
  dw[c] = accumulate ? dw[c] + v : v;
}

}  // namespace nknorm

// <type of x>_<type of the residual>, W waves a row, C times eight columns a lane
#define NETRA_NORM(X, R, XT, RT, W, C, NAME, ONCE)                                                             \
  extern "C" __global__                                                                                        \
      __launch_bounds__(nknorm::Shape<W>::kThreads) void netra_norm_##X##_##R##_w##W##c##C##NAME##_gfx950(nknorm::Norm a) { \
    nknorm::forward<XT, RT, W, C, ONCE>(a);                                                                    \
  }                                                                                                            \
  extern "C" __global__                                                                                        \
      __launch_bounds__(nknorm::Shape<W>::kThreads) void netra_norm_gradients_##X##_##R##_w##W##c##C##NAME##_gfx950( \
          nknorm::NormGradients a) {                                                                           \
    nknorm::gradients<XT, RT, W, C, ONCE>(a);                                                                  \
  }
#define NETRA_NORM_BOTH(X, R, XT, RT, W, C) \
  NETRA_NORM(X, R, XT, RT, W, C, , false)   \
  NETRA_NORM(X, R, XT, RT, W, C, _once, true)
#define NETRA_NORMS(W, C)                               \
  NETRA_NORM_BOTH(bf16, bf16, uint16_t, uint16_t, W, C) \
  NETRA_NORM_BOTH(bf16, f32, uint16_t, float, W, C)     \
  NETRA_NORM_BOTH(f32, bf16, float, uint16_t, W, C)     \
  NETRA_NORM_BOTH(f32, f32, float, float, W, C)
NETRA_NORMS(1, 1)
NETRA_NORMS(1, 2)
NETRA_NORMS(4, 1)
NETRA_NORMS(8, 1)
NETRA_NORMS(16, 1)
NETRA_NORMS(16, 2)

extern "C" __global__ __launch_bounds__(1024) void netra_norm_sum_gfx950(const float* partial, uint32_t parts,
                                                                        uint32_t cols, float* dw, uint32_t accumulate) {
  nknorm::sum_parts(partial, parts, cols, dw, accumulate);
}
