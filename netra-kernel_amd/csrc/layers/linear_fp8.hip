// Block-FP8 linear layer: quantisation into MFMA tiles, weight packing and the
// product. Both operands of every product are in the tile16x128 layout
// (moe_numerics.h): a matrix [rows, contraction] as row tiles of 16 x 128 codes,
// padded with zeros, so each half-operand wave load reads 1 KiB contiguous.
//
// One product serves forward and input gradient. It computes
//   out[q, i] = sum_b s_q[b, q] * s_p(i, b) * sum_{c in b} P[i, c] Q[q, c]
// with the rows i of P as the fast dimension of the output: an MFMA's D has
// rows i (four consecutive ones per lane) and columns q (one per lane), so a
// lane applies one activation scale per product and stores four neighbours.
//   forward          P = W        Q = x    s_p = s_w[i/128, b]
//   input gradient   P = W^T      Q = dy   s_p = s_w[b, i/128]
// The weight gradient is a bf16 product over the tokens (no scales).
#pragma once
#include "../kernels/moe_numerics.h"

namespace nklin {

using nk::u32x4;
using nk::v4f;
using nk::v8i;

// One activation value as fp32.
__device__ __forceinline__ float value(const uint16_t* p) { return nk::bf16_f32(*p); }
__device__ __forceinline__ float value(const float* p) { return *p; }

// Scale of a 128-group from the largest magnitude's bits (as an unsigned
// integer, a NaN's magnitude is above infinity's, so the maximum keeps it). A
// group with an infinity or NaN gets a NaN scale.
__device__ __forceinline__ float group_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return fmaxf(__uint_as_float(amax_bits), nk::kAmaxFloor) * nk::inv_e4m3_max();
}

// 32 consecutive values of one row from column c (zeros from column n on).
// kVec: 16-byte loads (base and row stride 16-byte aligned).
template <bool kVec>
__device__ __forceinline__ void load32(const uint16_t* row, uint32_t c, uint32_t n, float (&v)[32]) {
  if (kVec && c + 32u <= n) {
#pragma unroll
    for (uint32_t j = 0; j < 4u; ++j) {
      const uint4 u = *reinterpret_cast<const uint4*>(row + c + 8u * j);
      v[8 * j + 0] = nk::bf16_lo(u.x); v[8 * j + 1] = nk::bf16_hi(u.x);
      v[8 * j + 2] = nk::bf16_lo(u.y); v[8 * j + 3] = nk::bf16_hi(u.y);
      v[8 * j + 4] = nk::bf16_lo(u.z); v[8 * j + 5] = nk::bf16_hi(u.z);
      v[8 * j + 6] = nk::bf16_lo(u.w); v[8 * j + 7] = nk::bf16_hi(u.w);
    }
    return;
  }
#pragma unroll
  for (uint32_t j = 0; j < 32u; ++j) v[j] = c + j < n ? value(row + c + j) : 0.0f;
}
template <bool kVec>
__device__ __forceinline__ void load32(const float* row, uint32_t c, uint32_t n, float (&v)[32]) {
  if (kVec && c + 32u <= n) {
#pragma unroll
    for (uint32_t j = 0; j < 8u; ++j) {
      const float4 u = *reinterpret_cast<const float4*>(row + c + 4u * j);
      v[4 * j + 0] = u.x; v[4 * j + 1] = u.y; v[4 * j + 2] = u.z; v[4 * j + 3] = u.w;
    }
    return;
  }
#pragma unroll
  for (uint32_t j = 0; j < 32u; ++j) v[j] = c + j < n ? value(row + c + j) : 0.0f;
}

// The 32 values of each lane as MFMA operand bytes, with the scale of the
// 128-group that the lanes l, l ^ 16, l ^ 32, l ^ 48 hold together.
__device__ __forceinline__ float quantise32(const float (&v)[32], uint32_t (&q)[8]) {
  uint32_t m = 0u;
#pragma unroll
  for (uint32_t j = 0; j < 32u; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  m = max(m, (uint32_t)__shfl_xor((int)m, 16));
  m = max(m, (uint32_t)__shfl_xor((int)m, 32));
  const float scale = group_scale(m);
  const float inv = 1.0f / scale;
#pragma unroll
  for (uint32_t j = 0; j < 8u; ++j)
    q[j] = nk::e4m3x4(v[4 * j] * inv, v[4 * j + 1] * inv, v[4 * j + 2] * inv, v[4 * j + 3] * inv);
  return scale;
}

__device__ __forceinline__ void store_tile(uint8_t* tile, uint32_t lane, const uint32_t (&q)[8]) {
  *reinterpret_cast<uint4*>(tile + lane * 16u) = make_uint4(q[0], q[1], q[2], q[3]);
  *reinterpret_cast<uint4*>(tile + 1024u + lane * 16u) = make_uint4(q[4], q[5], q[6], q[7]);
}

// Rows: x [rows, n] -> tiles of 16 rows x 128 columns, scales s[b, row] with
// `sld` floats per block (sld = rows rounded up to 16 at least). One wave per tile; rows past
// the end are zeros.
template <typename X, bool kVec>
__device__ __forceinline__ void quant_rows(const X* __restrict__ x, uint64_t stride, uint8_t* __restrict__ q,
                                           float* __restrict__ s, uint32_t rows, uint32_t n, uint32_t sld) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t kb = (n + 127u) / 128u;
  const uint32_t rt = blockIdx.x, b = blockIdx.y * 4u + wave;
  if (b >= kb) return;
  const uint32_t r = rt * 16u + (lane & 15u), c = b * 128u + (lane >> 4) * 32u;
  float v[32];
  if (r < rows) {
    load32<kVec>(x + (uint64_t)r * stride, c, n, v);
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 32u; ++j) v[j] = 0.0f;
  }
  uint32_t code[8];
  const float scale = quantise32(v, code);
  store_tile(q + ((size_t)rt * kb + b) * 2048u, lane, code);
  if (lane < 16u) s[(size_t)b * sld + r] = scale;
}

__device__ __forceinline__ void store4(uint16_t* out, uint32_t left, bool vec, const float (&v)[4]) {
  if (vec && left >= 4u) {
    *reinterpret_cast<uint2*>(out) = make_uint2(nk::bf16_rne(v[0]) | ((uint32_t)nk::bf16_rne(v[1]) << 16),
                                                nk::bf16_rne(v[2]) | ((uint32_t)nk::bf16_rne(v[3]) << 16));
    return;
  }
#pragma unroll
  for (uint32_t j = 0; j < 4u; ++j)
    if (j < left) out[j] = nk::bf16_rne(v[j]);
}
__device__ __forceinline__ void store4(float* out, uint32_t left, bool vec, const float (&v)[4]) {
  if (vec && left >= 4u) {
    *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
    return;
  }
#pragma unroll
  for (uint32_t j = 0; j < 4u; ++j)
    if (j < left) out[j] = v[j];
}

struct Product {
  const uint8_t* p;       // tiles of P [ni, contraction]
  const float* sp;        // scale of (i, b) at (i / 128) * sp_i + b * sp_b
  uint32_t sp_i, sp_b;
  const uint8_t* q;       // tiles of Q [nq, contraction]
  const float* sq;        // scale of (b, q) at b * sq_b + q
  uint32_t sq_b;
  uint16_t* out;          // bf16 [nq, ni], row stride ldo elements
  uint64_t ldo;
  uint32_t ni, nq, kb;    // kb: 128-blocks of the contraction
  uint32_t vec;           // rows of out are aligned for four-element stores
};

// The simplest form: a wave computes 32 x 32 of the output, its operands read
// straight from memory.
__device__ __forceinline__ void product_direct(const Product& a) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t pt = (a.ni + 15u) / 16u, qt = (a.nq + 15u) / 16u;
  const uint32_t p0 = blockIdx.x * 4u + (wave & 1u) * 2u, q0 = blockIdx.y * 4u + (wave >> 1) * 2u;
  if (p0 >= pt || q0 >= qt) return;
  const uint32_t c = lane & 15u, r4 = (lane >> 4) * 4u;
  v4f acc[2][2];
#pragma unroll
  for (uint32_t i = 0; i < 2u; ++i)
#pragma unroll
    for (uint32_t j = 0; j < 2u; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t b = 0; b < a.kb; ++b) {
    v8i po[2], qo[2];
    float sp[2], sq[2];
#pragma unroll
    for (uint32_t i = 0; i < 2u; ++i) {
      const uint32_t t = min(p0 + i, pt - 1u);
      po[i] = nk::load_tile_operand(nk::tile_base(a.p, t, b, a.kb), lane);
      sp[i] = a.sp[(size_t)(t / 8u) * a.sp_i + (size_t)b * a.sp_b];
    }
#pragma unroll
    for (uint32_t j = 0; j < 2u; ++j) {
      const uint32_t t = min(q0 + j, qt - 1u);
      qo[j] = nk::load_tile_operand(nk::tile_base(a.q, t, b, a.kb), lane);
      sq[j] = a.sq[(size_t)b * a.sq_b + t * 16u + c];
    }
#pragma unroll
    for (uint32_t i = 0; i < 2u; ++i)
#pragma unroll
      for (uint32_t j = 0; j < 2u; ++j) {
        const v4f d = nk::mfma_e4m3_16x16x128(po[i], qo[j]);
        const float s = sq[j] * sp[i];
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) acc[i][j][e] = fmaf(s, d[e], acc[i][j][e]);
      }
  }
#pragma unroll
  for (uint32_t j = 0; j < 2u; ++j) {
    const uint32_t row = (q0 + j) * 16u + c;
#pragma unroll
    for (uint32_t i = 0; i < 2u; ++i) {
      const uint32_t col = (p0 + i) * 16u + r4;
      if (row >= a.nq || col >= a.ni) continue;
      const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
      store4(a.out + (uint64_t)row * a.ldo + col, a.ni - col, a.vec != 0u, v);
    }
  }
}

// ---- weight gradient ------------------------------------------------------------

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

struct Outer {
  const void* dy;   // [rows, n]
  uint64_t dy_stride;
  uint32_t dy_type;
  const void* x;    // [rows, k]
  uint64_t x_stride;
  uint32_t x_type;
  float* dw;        // [n, k]
  uint32_t rows, n, k;
  uint32_t accumulate;
};

// Eight tokens' values of one column as an MFMA operand, zeros past the end.
__device__ __forceinline__ v8bf column8(const void* m, uint64_t stride, uint32_t type, uint32_t c, uint32_t cols,
                                        uint32_t t, uint32_t rows) {
  v8bf v;
#pragma unroll
  for (uint32_t j = 0; j < 8u; ++j) {
    float f = 0.0f;
    if (c < cols && t + j < rows) {
      const uint64_t at = (uint64_t)(t + j) * stride + c;
      f = type == 0u ? value(static_cast<const uint16_t*>(m) + at) : value(static_cast<const float*>(m) + at);
    }
    v[j] = __builtin_bit_cast(__bf16, nk::bf16_rne(f));
  }
  return v;
}

// dw[n, k] = sum_t dy[t, n] x[t, k]: a wave computes 32 x 32, the columns read
// straight from memory.
__device__ __forceinline__ void outer_direct(const Outer& a) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t k0 = blockIdx.x * 64u + (wave & 1u) * 32u, n0 = blockIdx.y * 64u + (wave >> 1) * 32u;
  if (k0 >= a.k || n0 >= a.n) return;
  const uint32_t c = lane & 15u, g = lane >> 4;
  v4f acc[2][2];
#pragma unroll
  for (uint32_t i = 0; i < 2u; ++i)
#pragma unroll
    for (uint32_t j = 0; j < 2u; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t t = 0; t < a.rows; t += 32u) {
    v8bf po[2], qo[2];
#pragma unroll
    for (uint32_t i = 0; i < 2u; ++i) {
      po[i] = column8(a.x, a.x_stride, a.x_type, k0 + i * 16u + c, a.k, t + g * 8u, a.rows);
      qo[i] = column8(a.dy, a.dy_stride, a.dy_type, n0 + i * 16u + c, a.n, t + g * 8u, a.rows);
    }
#pragma unroll
    for (uint32_t i = 0; i < 2u; ++i)
#pragma unroll
      for (uint32_t j = 0; j < 2u; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(po[i], qo[j], acc[i][j], 0, 0, 0);
  }
#pragma unroll
  for (uint32_t j = 0; j < 2u; ++j) {
    const uint32_t row = n0 + j * 16u + c;
#pragma unroll
    for (uint32_t i = 0; i < 2u; ++i) {
      const uint32_t col = k0 + i * 16u + g * 4u;
      if (row >= a.n || col >= a.k) continue;
      float* o = a.dw + (uint64_t)row * a.k + col;
      float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
      if (a.accumulate) {
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e)
          if (col + e < a.k) v[e] += o[e];
      }
      store4(o, a.k - col, a.k % 4u == 0u && reinterpret_cast<uintptr_t>(a.dw) % 16u == 0u, v);
    }
  }
}

}  // namespace nklin

// Weights: w row-major e4m3 [n, k] -> tiles of w, or of w^T. One wave per tile;
// bytes past the matrix are zeros.
__global__ __launch_bounds__(256) void netra_linear_pack_gfx950(const uint8_t* __restrict__ w,
                                                                uint8_t* __restrict__ dst, uint32_t n, uint32_t k,
                                                                uint32_t transpose) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t rows = transpose ? k : n, cols = transpose ? n : k;
  const uint32_t cb = (cols + 127u) / 128u, b = blockIdx.y * 4u + wave;
  if (b >= cb) return;
  const uint32_t r = blockIdx.x * 16u + (lane & 15u), c = b * 128u + (lane >> 4) * 32u;
  uint32_t code[8];
#pragma unroll
  for (uint32_t j = 0; j < 8u; ++j) {
    code[j] = 0u;
#pragma unroll
    for (uint32_t e = 0; e < 4u; ++e) {
      const uint32_t cc = c + 4u * j + e;
      if (r < rows && cc < cols)
        code[j] |= (uint32_t)(transpose ? w[(size_t)cc * k + r] : w[(size_t)r * k + cc]) << (8u * e);
    }
  }
  nklin::store_tile(dst + ((size_t)blockIdx.x * cb + b) * 2048u, lane, code);
}

#define NETRA_QUANT_ROWS(NAME, X, VEC)                                                                       \
  __global__ __launch_bounds__(256) void netra_linear_quant_rows_##NAME##_gfx950(                            \
      const X* x, uint64_t stride, uint8_t* q, float* s, uint32_t rows, uint32_t n, uint32_t sld) {          \
    nklin::quant_rows<X, VEC>(x, stride, q, s, rows, n, sld);                                                \
  }
NETRA_QUANT_ROWS(bf16, uint16_t, false)
NETRA_QUANT_ROWS(bf16_vec, uint16_t, true)
NETRA_QUANT_ROWS(f32, float, false)
NETRA_QUANT_ROWS(f32_vec, float, true)

__global__ __launch_bounds__(256) void netra_linear_product_direct_gfx950(nklin::Product a) {
  nklin::product_direct(a);
}

__global__ __launch_bounds__(256) void netra_linear_outer_direct_gfx950(nklin::Outer a) { nklin::outer_direct(a); }

// dw of no tokens: zeros.
__global__ __launch_bounds__(256) void netra_linear_zero_gfx950(float* out, uint64_t n) {
  for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256u) out[i] = 0.0f;
}
