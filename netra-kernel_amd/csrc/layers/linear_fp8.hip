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
#include "lds_copy.h"

namespace nklin {

using nk::u32x4;
using nk::v4f;
using nk::v8i;

// Scale of a 128-group from the largest magnitude's bits (as an unsigned
// integer, a NaN's magnitude is above infinity's, so the maximum keeps it). A
// group with an infinity or NaN gets a NaN scale.
__device__ __forceinline__ float group_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return fmaxf(__uint_as_float(amax_bits), nk::kAmaxFloor) * nk::inv_e4m3_max();
}

// 32 consecutive values of a row as they lie in memory: bf16 pairs or fp32.
template <typename X>
struct Raw;
template <>
struct Raw<uint16_t> {
  uint32_t w[16];
};
template <>
struct Raw<float> {
  float w[32];
};

// 16 bytes from any element address: global loads need no alignment on this target.
struct __attribute__((packed, aligned(2))) Unaligned16 {
  uint32_t w[4];
};

// Values from column c of a row of n (zeros from column n on; nothing past it is read).
__device__ __forceinline__ void load32(const uint16_t* row, uint32_t c, uint32_t n, Raw<uint16_t>& v) {
  if (c + 32u <= n) {
#pragma unroll
    for (uint32_t j = 0; j < 4u; ++j) {
      const Unaligned16 u = *reinterpret_cast<const Unaligned16*>(row + c + 8u * j);
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) v.w[4u * j + i] = u.w[i];
    }
    return;
  }
#pragma unroll
  for (uint32_t j = 0; j < 4u; ++j) {
    const uint32_t e = c + 8u * j;
    if (e + 8u <= n) {
      const Unaligned16 u = *reinterpret_cast<const Unaligned16*>(row + e);
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) v.w[4u * j + i] = u.w[i];
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) {
        const uint32_t lo = e + 2u * i < n ? row[e + 2u * i] : 0u;
        const uint32_t hi = e + 2u * i + 1u < n ? row[e + 2u * i + 1u] : 0u;
        v.w[4u * j + i] = lo | hi << 16;
      }
    }
  }
}
__device__ __forceinline__ void load32(const float* row, uint32_t c, uint32_t n, Raw<float>& v) {
#pragma unroll
  for (uint32_t j = 0; j < 8u; ++j) {
    const uint32_t e = c + 4u * j;
    if (e + 4u <= n) {
      const Unaligned16 u = *reinterpret_cast<const Unaligned16*>(row + e);
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) v.w[4u * j + i] = __uint_as_float(u.w[i]);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) v.w[4u * j + i] = e + i < n ? row[e + i] : 0.0f;
    }
  }
}

// Largest magnitude's bits (fp32), and value j.
__device__ __forceinline__ uint32_t amax_bits(const Raw<uint16_t>& v) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 m = {0, 0};
#pragma unroll
  for (uint32_t j = 0; j < 16u; ++j) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v.w[j] & 0x7fff7fffu));
  return (uint32_t)max(m[0], m[1]) << 16;
}
__device__ __forceinline__ uint32_t amax_bits(const Raw<float>& v) {
  uint32_t m = 0u;
#pragma unroll
  for (uint32_t j = 0; j < 32u; ++j) m = max(m, __float_as_uint(v.w[j]) & 0x7fffffffu);
  return m;
}
__device__ __forceinline__ float at(const Raw<uint16_t>& v, uint32_t j) {
  return j & 1u ? nk::bf16_hi(v.w[j / 2u]) : nk::bf16_lo(v.w[j / 2u]);
}
__device__ __forceinline__ float at(const Raw<float>& v, uint32_t j) { return v.w[j]; }

// The 32 values of each lane as MFMA operand bytes, with the scale of the
// 128-group that the lanes l, l ^ 16, l ^ 32, l ^ 48 hold together. |v / scale| is
// at most 448 (1 + 4 * 2^-24), which rounds to 448 without the contract's clamp.
template <typename X>
__device__ __forceinline__ float quantise32(const Raw<X>& v, uint32_t (&q)[8]) {
  uint32_t m = amax_bits(v);
  const auto r16 = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  m = max((uint32_t)r16[0], (uint32_t)r16[1]);
  const auto r32 = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  m = max((uint32_t)r32[0], (uint32_t)r32[1]);
  const float scale = group_scale(m);
  const float inv = 1.0f / scale;
#pragma unroll
  for (uint32_t j = 0; j < 8u; ++j) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(at(v, 4 * j) * inv, at(v, 4 * j + 1) * inv, 0, false);
    q[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(at(v, 4 * j + 2) * inv, at(v, 4 * j + 3) * inv, lo, true);
  }
  return scale;
}

__device__ __forceinline__ void store_tile(uint8_t* tile, uint32_t lane, const uint32_t (&q)[8]) {
  *reinterpret_cast<uint4*>(tile + lane * 16u) = make_uint4(q[0], q[1], q[2], q[3]);
  *reinterpret_cast<uint4*>(tile + 1024u + lane * 16u) = make_uint4(q[4], q[5], q[6], q[7]);
}

// Rows: x [rows, n] -> tiles of 16 rows x 128 columns, scales s[b, row] with
// `sld` floats per block (sld = rows rounded up to 16 at least). One wave per tile; rows past
// the end are zeros. Bound by memory: a tile's loads, 64 bytes a lane, are one wave's whole
// work, so enough are under way. 8192 x 4096 bf16: 102 MB in and out, 20.5 us, 5.0 TB/s (a
// large copy: 5.1 to 5.2); 64 x 2048 bf16 2.9 us (a launch); 1001 x 1111 fp32 5.0 us, where a load
// instruction's lanes touch 64 lines for 16 bytes each.
template <typename X>
__device__ __forceinline__ void quant_rows(const X* __restrict__ x, uint64_t stride, uint8_t* __restrict__ q,
                                           float* __restrict__ s, uint32_t rows, uint32_t n, uint32_t sld,
                                           uint32_t rt, uint32_t b4) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t kb = (n + 127u) / 128u, b = b4 * 4u + wave;
  if (b >= kb) return;
  const uint32_t r = rt * 16u + (lane & 15u), c = b * 128u + (lane >> 4) * 32u;
  Raw<X> v = {};
  if (r < rows) load32(x + (uint64_t)r * stride, c, n, v);
  uint32_t code[8];
  const float scale = quantise32(v, code);
  store_tile(q + ((size_t)rt * kb + b) * 2048u, lane, code);
  if (lane < 16u) s[(size_t)b * sld + r] = scale;
}

// Stores at any element address, `left` values at most.
__device__ __forceinline__ void store4(uint16_t* out, uint32_t left, const float (&v)[4]) {
  struct __attribute__((packed, aligned(2))) Pair {
    uint32_t w[2];
  };
  const Pair p = {{nk::bf16x2_hw(v[0], v[1]), nk::bf16x2_hw(v[2], v[3])}};
  if (left >= 4u) {
    *reinterpret_cast<Pair*>(out) = p;
    return;
  }
#pragma unroll
  for (uint32_t j = 0; j < 3u; ++j)
    if (j < left) out[j] = (uint16_t)(p.w[j / 2u] >> (16u * (j & 1u)));
}
__device__ __forceinline__ void store4(float* out, uint32_t left, const float (&v)[4]) {
  struct __attribute__((packed, aligned(4))) Quad {
    float w[4];
  };
  if (left >= 4u) {
    *reinterpret_cast<Quad*>(out) = Quad{{v[0], v[1], v[2], v[3]}};
    return;
  }
#pragma unroll
  for (uint32_t j = 0; j < 3u; ++j)
    if (j < left) out[j] = v[j];
}

struct Product {
  const uint8_t* p;       // tiles of P [ni, contraction]
  const float* sp;        // scale of (i, b) at (i / 128) * sp_i + b * sp_b
  uint32_t sp_i, sp_b, sp_bytes;
  const uint8_t* q;       // tiles of Q [nq, contraction]
  const float* sq;        // scale of (b, q) at b * sq_b + q
  uint32_t sq_b;
  uint16_t* out;          // bf16 [nq, ni], row stride ldo elements
  uint64_t ldo;
  uint32_t ni, nq, kb;    // kb: 128-blocks of the contraction
  uint32_t splits, split_blocks;  // 128-blocks per split
  float* partial;         // [splits, nq, ni rounded up to 4] where splits > 1
};

// The same product with both operands staged through LDS.
//
// A workgroup of 8 waves (WP along P, WQ along Q) computes 16 WP NP rows of P by
// 16 WQ NQ rows of Q. Per 128-block ("step") it needs one tile row of each
// operand and the scales; they are copied global -> LDS, S - 1 steps ahead, into
// a ring of S stages. A step's single barrier, behind each wave's wait for its own
// copies of the step, both shows the step's data to all waves and tells them that
// the stage of the step before may be overwritten.
// Each wave holds its NQ operands of Q for the step and streams its NP operands of
// P past them: NQ products per operand, each scaled and added by VALU while the
// matrix core works on the next. (The scales differ per row of Q, so the sum over blocks
// cannot stay in the matrix core.) Copies spread over the products: in a burst at the head of
// a step they hold up the wave that issues them.
// What bounds it: no unit alone, but that all waves of the one workgroup on a CU go in step.
// 256x128 at T 2048, N 4096, K 4096: 35.9 us (1.9 PFLOP/s; the library's product without block
// scales 2.4 to 2.6 at 8192 x 8192 x 4096). A step takes 2180 cycles for 1024 of products: by
// counters the matrix cores are busy 47% of the waves' time, LDS 29%, and a wave spends 30% of it
// at the barrier or behind copies and 33% waiting to issue. 128x64 at T 1001, N 1500, K 1111: 8.2
// us, nine steps and one round.
template <uint32_t WP, uint32_t WQ, uint32_t NP, uint32_t NQ, uint32_t S>
struct Tile {
  static constexpr uint32_t kWaves = WP * WQ;
  static constexpr uint32_t kP = WP * NP, kQ = WQ * NQ;   // 16-row tiles of each operand
  static constexpr uint32_t kScaleAt = (kP + kQ) * 2048u; // 16 scales per tile of Q, then 64 words for P's
  static constexpr uint32_t kStage = kScaleAt + kQ * 64u + 256u;
  // A wave's copies per step: two for each of its whole tiles, one for a half of the rest, scales.
  static constexpr uint32_t kTiles = (kP + kQ) / kWaves, kHalves = (kP + kQ) % kWaves * 2u / kWaves;
  static constexpr uint32_t kCopies = 2u * kTiles + kHalves + 1u;
  // A row's pitch of the output's staging: 16 bytes over its NP tiles spread the writes over the banks.
  static constexpr uint32_t kPitch = NP * 32u + 16u;
  static constexpr uint32_t kOut = kWaves * 16u * NQ * kPitch;
  static constexpr uint32_t kLds = S * kStage > kOut ? S * kStage : kOut;
  static_assert(kWaves == 8u && (NP % 8u == 0u || 8u % NP == 0u) && (kP + kQ) % 4u == 0u && kQ % 4u == 0u && kQ <= 28u &&
                    kLds <= 160u * 1024u,
                "waves, scale blocks, copies and LDS");
};

// The tile of workgroup `group`: split, and first 16-row tiles of P and Q. False: none.
// The workgroups of an XCD (ids deal to the eight XCDs in turn) take neighbouring
// tiles, in bands of 4 along Q, so that they share operands in its L2 (T 4096, N 4096,
// K 2048: 43.4 us, in bands of 8 45.0, of 16 45.9).
__device__ __forceinline__ bool product_place(const Product& a, uint32_t group, uint32_t tiles_p, uint32_t tiles_q,
                                              uint32_t& split, uint32_t& p0, uint32_t& q0) {
  const uint32_t pt = (a.ni + 15u) / 16u, qt = (a.nq + 15u) / 16u;
  const uint32_t np = (pt + tiles_p - 1u) / tiles_p, nq = (qt + tiles_q - 1u) / tiles_q;
  const uint32_t total = np * nq * a.splits, per = (total + 7u) / 8u;
  const uint32_t item = (group % 8u) * per + group / 8u;
  if (group / 8u >= per || item >= total) return false;
  split = item / (np * nq);
  const uint32_t tile = item - split * np * nq;
  const uint32_t band = tile / (4u * np), in_band = tile - band * 4u * np;
  const uint32_t height = min(4u, nq - band * 4u);
  p0 = in_band / height * tiles_p;
  q0 = (band * 4u + in_band % height) * tiles_q;
  return true;
}

// A wave's NP x NQ tiles from row tile p of P and q of Q to the output, or, of a split, to the
// partial sums.
template <typename L, uint32_t NP, uint32_t NQ>
__device__ __forceinline__ void product_store(const Product& a, const v4f (&acc)[NP][NQ], uint32_t split, uint32_t p,
                                              uint32_t q, uint8_t* s_stage) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t c = lane & 15u, r4 = (lane >> 4) * 4u;
  const uint32_t col0 = p * 16u, row0 = q * 16u;
  if (a.splits > 1u) {  // fp32 partial sums, rows of a.ni rounded up to 4
    const uint32_t pitch = (a.ni + 3u) & ~3u;
    float* part = a.partial + (size_t)split * a.nq * pitch;
#pragma unroll
    for (uint32_t j = 0; j < NQ; ++j)
#pragma unroll
      for (uint32_t i = 0; i < NP; ++i) {
        const uint32_t row = row0 + j * 16u + c, col = col0 + i * 16u + r4;
        if (row < a.nq && col < pitch) *reinterpret_cast<v4f*>(part + (size_t)row * pitch + col) = acc[i][j];
      }
    return;
  }
  // Output: a wave's 16 NQ rows of 16 NP values through LDS, so that a row leaves as
  // whole lines. (A wave reads back only what it wrote itself.)
  __syncthreads();
  uint8_t* mine = s_stage + wave * 16u * NQ * L::kPitch;
#pragma unroll
  for (uint32_t j = 0; j < NQ; ++j)
#pragma unroll
    for (uint32_t i = 0; i < NP; ++i) {
      const v4f v = acc[i][j];
      *reinterpret_cast<uint2*>(mine + (j * 16u + c) * L::kPitch + (i * 16u + r4) * 2u) =
          make_uint2(nk::bf16x2_hw(v[0], v[1]), nk::bf16x2_hw(v[2], v[3]));
    }
  constexpr uint32_t kLanes = NP * 2u;  // lanes of 8 values per row
  for (uint32_t r = lane / kLanes; r < 16u * NQ; r += 64u / kLanes) {
    const uint32_t cc = (lane % kLanes) * 8u, row = row0 + r, col = col0 + cc;
    if (row >= a.nq || col >= a.ni) continue;
    const uint4 v = *reinterpret_cast<const uint4*>(mine + r * L::kPitch + cc * 2u);
    uint16_t* o = a.out + (uint64_t)row * a.ldo + col;
    const Unaligned16 w = {{v.x, v.y, v.z, v.w}};
    if (col + 8u <= a.ni) {
      *reinterpret_cast<Unaligned16*>(o) = w;
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 8u; ++e)
        if (col + e < a.ni) o[e] = (uint16_t)(w.w[e / 2u] >> (16u * (e & 1u)));
    }
  }
}

template <uint32_t WP, uint32_t WQ, uint32_t NP, uint32_t NQ, uint32_t S>
__device__ __forceinline__ void product_tile(const Product& a, uint32_t group, uint8_t* s_stage) {
  using L = Tile<WP, WQ, NP, NQ, S>;
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t pt = (a.ni + 15u) / 16u, qt = (a.nq + 15u) / 16u;
  uint32_t split, p0, q0;
  if (!product_place(a, group, L::kP, L::kQ, split, p0, q0)) return;
  const uint32_t wp = wave % WP, wq = wave / WP;
  const uint32_t b0 = split * a.split_blocks, b1 = min(a.kb, b0 + a.split_blocks);  // this split's blocks

  const uint32_t np_here = min(L::kP, pt - p0), nq_here = min(L::kQ, qt - q0);
  const u32x4 rp = nklds2::rsrc(a.p + (size_t)p0 * a.kb * 2048u, np_here * a.kb * 2048u);
  const u32x4 rq = nklds2::rsrc(a.q + (size_t)q0 * a.kb * 2048u, nq_here * a.kb * 2048u);
  // A wave copies one 64-word part of the scales: Q's by the first kQ / 4 waves, P's
  // (lane i: 128-block i of the tile) by the others, all of them alike.
  const bool q_scales = wave < L::kQ / 4u;
  const uint32_t sq_first = (q0 + wave * 4u) * 16u;
  const uint64_t s_base = (uint64_t)(q_scales ? a.sq + sq_first : a.sp);
  const uint32_t s_bytes = q_scales ? (sq_first < a.sq_b ? (a.sq_b - sq_first) * 4u : 0u) : a.sp_bytes;
  const uint32_t s_step = (q_scales ? a.sq_b : a.sp_b) * 4u, s_less = q_scales ? 0u : s_step;  // bytes per block
  const uint32_t s_at = q_scales ? wave * 256u : L::kQ * 64u;
  const uint32_t s_voff = q_scales ? lane * 4u
                          : lane * 8u < L::kP && (p0 / 8u + lane) * 128u < a.ni ? (p0 / 8u + lane) * a.sp_i * 4u
                                                                                 : 0x80000000u;
  const uint32_t voff = lane * 16u;
  const uint32_t lds0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)nklds2::lds_offset(&s_stage[0]));
  // This wave's tiles (of P's, then Q's), and then its half tile where they do not go round.
  // A tile past the matrix repeats its last one (its outputs are not stored).
  constexpr uint32_t kOwn = L::kTiles + L::kHalves;
  uint32_t own[kOwn], first[kOwn];
#pragma unroll
  for (uint32_t i = 0; i < kOwn; ++i) {
    own[i] = L::kWaves * i + (i < L::kTiles ? wave : wave >> 1);
    first[i] = (own[i] < L::kP ? min(own[i], np_here - 1u) : min(own[i] - L::kP, nq_here - 1u)) * a.kb * 2048u;
  }
  // Part i of a wave's copies for block b. Behind the split's last block a copy reads
  // nothing (an empty range) and leaves zeros that nobody looks at, so that a step's
  // code has no branch and always the same copies in flight.
  auto issue_part = [&](uint32_t b, uint32_t stage, uint32_t i) __attribute__((always_inline)) {
    const uint32_t st = lds0 + stage * L::kStage;
    const bool live = b < b1;
    if (i < kOwn) {
      u32x4 r = own[i] < L::kP ? rp : rq;
      r.z = live ? r.z : 0u;
      const uint32_t to = st + own[i] * 2048u, from = live ? first[i] + b * 2048u : 0u, half = (wave & 1u) * 1024u;
      if (i < L::kTiles) nklds2::copy_tile(to, r, voff, from);
      else nklds2::copy16(to + half, r, voff, from + half);
    } else {
      const uint32_t bytes = s_bytes - b * s_less;
      const u32x4 r = nklds2::rsrc((const void*)(s_base + (uint64_t)b * s_step), live ? bytes : 0u);
      nklds2::copy4(st + L::kScaleAt + s_at, r, s_voff, 0u);
    }
  };
  auto issue = [&](uint32_t b, uint32_t stage) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t i = 0; i <= kOwn; ++i) issue_part(b, stage, i);
  };

  v4f acc[NP][NQ];
#pragma unroll
  for (uint32_t i = 0; i < NP; ++i)
#pragma unroll
    for (uint32_t j = 0; j < NQ; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

#pragma unroll
  for (uint32_t i = 0; i + 1u < S; ++i) issue(b0 + i, i);
  uint32_t stage = 0u;
  for (uint32_t b = b0; b < b1; ++b) {
    nklds2::wait_copies<(S - 2u) * L::kCopies>();  // the copies of the steps behind this one may stay in flight
    nklds2::barrier();
    const uint32_t before = stage == 0u ? S - 1u : stage - 1u;
    const uint8_t* st = s_stage + stage * L::kStage;
    stage = stage + 1u == S ? 0u : stage + 1u;
    const uint8_t* sp_tiles = st + wp * NP * 2048u;
    const uint8_t* sq_tiles = st + (L::kP + wq * NQ) * 2048u;
    const float* scale = reinterpret_cast<const float*>(st + L::kScaleAt);
    v8i qo[NQ], po[2];
    float s[NQ];
    po[0] = nk::load_tile_operand(sp_tiles, lane);
    const float sp = scale[L::kQ * 16u + wp * NP / 8u];
#pragma unroll
    for (uint32_t j = 0; j < NQ; ++j) {
      qo[j] = nk::load_tile_operand(sq_tiles + j * 2048u, lane);
      s[j] = scale[(wq * NQ + j) * 16u + (lane & 15u)] * sp;
    }
    v4f d[2][NQ];
#pragma unroll
    for (uint32_t i = 0; i <= NP; ++i) {
      if (i + 1u < NP) po[(i + 1u) & 1u] = nk::load_tile_operand(sp_tiles + (i + 1u) * 2048u, lane);
#pragma unroll
      for (uint32_t j = 0; j < NQ; ++j) {
        if (i < NP) d[i & 1u][j] = nk::mfma_e4m3_16x16x128(po[i & 1u], qo[j]);
        if (i > 0u) {
#pragma unroll
          for (uint32_t e = 0; e < 4u; ++e)
            acc[i - 1u][j][e] = fmaf(s[j], d[(i - 1u) & 1u][j][e], acc[i - 1u][j][e]);
        }
      }
      // the copies of a later step, spread over this one's products
#pragma unroll
      for (uint32_t k = i * (kOwn + 1u) / (NP + 1u); k < (i + 1u) * (kOwn + 1u) / (NP + 1u); ++k)
        issue_part(b + S - 1u, before, k);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  nklds2::wait_copies<0>();

  product_store<L, NP, NQ>(a, acc, split, p0 + wp * NP, q0 + wq * NQ, s_stage);
}

// The product in tiles of 256 x 256, two groups of four waves taking turns: while one
// group's waves, one on each SIMD, multiply, the other's read their next operands from
// LDS and issue copies, so that neither an LDS latency nor a copy that waits for its turn
// holds the matrix cores up. A phase ends with a barrier; group 1 is one phase behind:
//   phase      2b          2b + 1        2b + 2
//   group 0    read b      multiply b    read b + 1
//   group 1    ..          read b        multiply b
// Group g owns half g of P's rows. Group 0 copies, while it reads block b, its half of P
// and all of Q for block b + 1, over block b - 1's: Q was last read by group 1 and the half
// of P by its own products, both a phase ago. Group 1 copies its own half of P, likewise.
// Copies are waited for at the end of the products of the same block, a phase and a half
// after they were issued, and needed by group 0 in the next phase (group 1: its own).
// T 8192, N 8192, K 4096: 230 us (2.4 PFLOP/s; the library's product without block scales 212 to
// 229 us), behind 20.5 of quantisation. A step takes 3320 cycles for 2048 of products: by counters
// the matrix cores are busy 62% of the waves' time, LDS 28%, and a wave spends 30% of it at a
// barrier or behind copies. All waves in step, product_tile's way, take 4% longer, without
// whole-tile copies 2%, with the copies spread over both groups' products 7%, with Q's operands
// straight from L2 to registers 18%. (256x128 in turns is slower, 47.8 us against 41.5 as calls at T
// 2048, N 4096, K 4096: its phases are 16 products long.) About 60 us go with the copies (timed
// without them).
__device__ __forceinline__ void product_turns(const Product& a, uint32_t index, uint8_t* s_stage) {
  using L = Tile<2, 4, 8, 4, 2>;
  constexpr uint32_t kStage = L::kScaleAt + 1024u + 512u;  // Q's scales, then P's for either group
  static_assert(2u * kStage <= L::kLds, "two stages");
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t g = wave >> 2, w = wave & 3u;  // group, wave in it
  const uint32_t pt = (a.ni + 15u) / 16u, qt = (a.nq + 15u) / 16u;
  uint32_t split, p0, q0;
  if (!product_place(a, index, 16u, 16u, split, p0, q0)) return;
  const uint32_t b0 = split * a.split_blocks, b1 = min(a.kb, b0 + a.split_blocks);
  const uint32_t np_here = min(16u, pt - p0), nq_here = min(16u, qt - q0);
  const u32x4 rp = nklds2::rsrc(a.p + (size_t)p0 * a.kb * 2048u, np_here * a.kb * 2048u);
  const u32x4 rq = nklds2::rsrc(a.q + (size_t)q0 * a.kb * 2048u, nq_here * a.kb * 2048u);
  const uint32_t sq_first = (q0 + w * 4u) * 16u;
  const uint32_t sq_bytes = sq_first < a.sq_b ? (a.sq_b - sq_first) * 4u : 0u;
  const uint32_t sp_voff = lane < 2u && (p0 / 8u + lane) * 128u < a.ni ? (p0 / 8u + lane) * a.sp_i * 4u : 0x80000000u;
  const uint32_t lds0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)nklds2::lds_offset(&s_stage[0]));
  // This wave's copies for block b (behind the last block: nothing, as product_tile's).
  auto issue = [&](uint32_t b) __attribute__((always_inline)) {
    const uint32_t st = lds0 + (b - b0) % 2u * kStage;
    const bool live = b < b1;
    auto tile = [&](const u32x4& from, uint32_t have, uint32_t t, uint32_t at) __attribute__((always_inline)) {
      u32x4 r = from;
      r.z = live ? r.z : 0u;
      nklds2::copy_tile(st + at, r, lane * 16u, live ? (min(t, have - 1u) * a.kb + b) * 2048u : 0u);
    };
#pragma unroll
    for (uint32_t i = 0; i < 2u; ++i) {  // half g of P
      const uint32_t t = g * 8u + i * 4u + w;
      tile(rp, np_here, t, t * 2048u);
    }
    const u32x4 rsp = nklds2::rsrc(a.sp + (size_t)b * a.sp_b, live ? a.sp_bytes - b * a.sp_b * 4u : 0u);
    nklds2::copy4(st + L::kScaleAt + 1024u + g * 256u, rsp, sp_voff, 0u);
    if (g == 0u) {
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) tile(rq, nq_here, i * 4u + w, 32768u + (i * 4u + w) * 2048u);
      const u32x4 rsq = nklds2::rsrc(a.sq + (size_t)b * a.sq_b + sq_first, live ? sq_bytes : 0u);
      nklds2::copy4(st + L::kScaleAt + w * 256u, rsq, lane * 4u, 0u);
    }
  };

  v4f acc[8][4];
#pragma unroll
  for (uint32_t i = 0; i < 8u; ++i)
#pragma unroll
    for (uint32_t j = 0; j < 4u; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  issue(b0);
  nklds2::wait_copies<0>();
  nklds2::barrier();
  if (g == 1u) nklds2::barrier();
  for (uint32_t b = b0; b < b1; ++b) {
    const uint8_t* st = s_stage + (b - b0) % 2u * kStage;
    const uint8_t* tp = st + g * 16384u;
    const float* scale = reinterpret_cast<const float*>(st + L::kScaleAt);
    // read
    v8i qo[4], po[3];
    float s[4];
    po[0] = nk::load_tile_operand(tp, lane);
    po[1] = nk::load_tile_operand(tp + 2048u, lane);
    const float sp = scale[256u + g * 64u + g];
#pragma unroll
    for (uint32_t j = 0; j < 4u; ++j) {
      qo[j] = nk::load_tile_operand(st + 32768u + (w * 4u + j) * 2048u, lane);
      s[j] = scale[(w * 4u + j) * 16u + (lane & 15u)] * sp;
    }
    __builtin_amdgcn_sched_barrier(0);
    issue(b + 1u);
    nklds2::barrier();
    __builtin_amdgcn_sched_barrier(0);
    // multiply
    __builtin_amdgcn_s_setprio(1);
    v4f d[4];
#pragma unroll
    for (uint32_t i = 0; i <= 8u; ++i) {
      if (i + 2u < 8u) po[(i + 2u) % 3u] = nk::load_tile_operand(tp + (i + 2u) * 2048u, lane);
#pragma unroll
      for (uint32_t j = 0; j < 4u; ++j) {
        if (i > 0u) {  // the tile before, one product of each row behind
#pragma unroll
          for (uint32_t e = 0; e < 4u; ++e) acc[i - 1u][j][e] = fmaf(s[j], d[j][e], acc[i - 1u][j][e]);
        }
        if (i < 8u) d[j] = nk::mfma_e4m3_16x16x128(po[i % 3u], qo[j]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    nklds2::wait_copies<0>();
    nklds2::barrier();
  }
  if (g == 0u) nklds2::barrier();
  nklds2::wait_copies<0>();
  product_store<L, 8u, 4u>(a, acc, split, p0 + g * 8u, q0 + w * 4u, s_stage);
}

// out = bf16 of the splits' sum, in split order. One row per blockIdx.y step. Memory.
__device__ __forceinline__ void product_sum(const Product& a) {
  const uint32_t pitch = (a.ni + 3u) & ~3u, col = (blockIdx.x * 256u + threadIdx.x) * 4u;
  if (col >= a.ni) return;
  for (uint32_t row = blockIdx.y; row < a.nq; row += gridDim.y) {
    v4f s = *reinterpret_cast<const v4f*>(a.partial + (size_t)row * pitch + col);
    for (uint32_t k = 1; k < a.splits; ++k)
      s += *reinterpret_cast<const v4f*>(a.partial + ((size_t)k * a.nq + row) * pitch + col);
    const float v[4] = {s[0], s[1], s[2], s[3]};
    store4(a.out + (uint64_t)row * a.ldo + col, a.ni - col, v);
  }
}

// Few rows: a workgroup computes 16 NP columns of the output for all 16 NQ rows,
// its 8 waves dealing the 128-blocks among them and adding up in LDS, in wave
// order. The weights go from memory to registers (each tile is read by one wave of
// the launch), one block ahead. Where kFused, the activations are quantised on the
// way, by every wave for its own blocks, so that a call is one launch: a wave's
// lanes hold a tile of 16 rows x 128 values exactly as an operand wants it, and the
// four lanes of a row find its scale with two exchanges. Else their tiles come from
// a.q. Bound by the weights' way from memory, or by a launch's length where they are few:
// T 1, N 28672, K 8192 (235 MB) 40.4 us, 5.8 TB/s; T 1, N 2048, K 2048 (4 MB, from the last
// level cache) 4.7 us, T 64, N 4096, K 2048 4.6 us behind 2.9 of quantisation.
template <uint32_t NP, uint32_t NQ, bool kFused, typename X>
__device__ __forceinline__ void product_stream(const Product& a, const X* __restrict__ x, uint64_t x_stride,
                                               uint32_t n) {
  __shared__ v4f s_part[8][NP * NQ][64];
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t pt = (a.ni + 15u) / 16u, qt = (a.nq + 15u) / 16u, p0 = blockIdx.x * NP;
  const uint32_t c = lane & 15u, g = lane >> 4;
  v4f acc[NP][NQ];
#pragma unroll
  for (uint32_t i = 0; i < NP; ++i)
#pragma unroll
    for (uint32_t j = 0; j < NQ; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const uint8_t* pb[NP];
  const float* spb[NP];
#pragma unroll
  for (uint32_t i = 0; i < NP; ++i) {
    const uint32_t t = min(p0 + i, pt - 1u);  // a tile past the end repeats the last one; not stored
    pb[i] = nk::tile_base(a.p, t, 0, a.kb);
    spb[i] = a.sp + (size_t)(t / 8u) * a.sp_i;
  }
  struct Block {  // what a block needs of memory
    v8i p[NP], q[kFused ? 1u : NQ];
    Raw<X> raw[kFused ? NQ : 1u];
    float sp[NP], sq[NQ];
  };
  auto load_p = [&](uint32_t b, Block& v) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t i = 0; i < NP; ++i) {
      v.p[i] = nk::load_tile_operand_once(pb[i] + (size_t)b * 2048u, lane);
      v.sp[i] = spb[i][(size_t)b * a.sp_b];
    }
  };
  auto load_q = [&](uint32_t b, Block& v) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t j = 0; j < NQ; ++j) {
      if constexpr (kFused) {
        // (a row past the end repeats the last one; not stored)
        load32(x + (uint64_t)min(j * 16u + c, a.nq - 1u) * x_stride, b * 128u + g * 32u, n, v.raw[j]);
      } else {
        const uint32_t t = min(j, qt - 1u);
        v.q[j] = nk::load_tile_operand(nk::tile_base(a.q, t, b, a.kb), lane);
        v.sq[j] = a.sq[(size_t)b * a.sq_b + t * 16u + c];
      }
    }
  };
  auto add = [&](Block& v) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t j = 0; j < NQ; ++j) {
      v8i qo;
      if constexpr (kFused) {
        uint32_t code[8];
        v.sq[j] = quantise32(v.raw[j], code);
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) qo[e] = (int)code[e];
      } else {
        qo = v.q[j];
      }
#pragma unroll
      for (uint32_t i = 0; i < NP; ++i) {
        const v4f d = nk::mfma_e4m3_16x16x128(v.p[i], qo);
        const float s = v.sq[j] * v.sp[i];
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) acc[i][j][e] = fmaf(s, d[e], acc[i][j][e]);
      }
    }
  };
  // The next block's loads are under way during a block (the activations' too, but for the
  // widest form: T 64, N 8192, K 8192 20.3 us, with them 21.9; T 16 15.2, without 16.2).
  constexpr bool kAhead = kFused || NP * NQ < 8u;
  if (wave < a.kb) {
    Block now;
    load_p(wave, now);
    if (kAhead) load_q(wave, now);
    for (uint32_t b = wave + 8u; b < a.kb; b += 8u) {
      Block next;
      if (!kAhead) load_q(b - 8u, now);
      load_p(b, next);
      if (kAhead) load_q(b, next);
      add(now);
      now = next;
    }
    if (!kAhead) load_q(wave + (a.kb - 1u - wave) / 8u * 8u, now);
    add(now);
  }
#pragma unroll
  for (uint32_t i = 0; i < NP; ++i)
#pragma unroll
    for (uint32_t j = 0; j < NQ; ++j) s_part[wave][i * NQ + j][lane] = acc[i][j];
  __syncthreads();
  for (uint32_t k = threadIdx.x; k < NP * NQ * 64u; k += 512u) {
    const uint32_t i = k / 64u / NQ, j = k / 64u % NQ, l = k & 63u;
    v4f s = s_part[0][i * NQ + j][l];
#pragma unroll
    for (uint32_t w = 1; w < 8u; ++w) s += s_part[w][i * NQ + j][l];
    const uint32_t row = j * 16u + (l & 15u), col = (p0 + i) * 16u + (l >> 4) * 4u;
    if (row >= a.nq || col >= a.ni) continue;
    const float v[4] = {s[0], s[1], s[2], s[3]};
    store4(a.out + (uint64_t)row * a.ldo + col, a.ni - col, v);
  }
}

// ---- weight gradient ------------------------------------------------------------

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

struct Outer {
  const uint16_t* dy;   // [rows, n] in rows of dy_cols readable elements (an even number)
  uint64_t dy_stride;
  uint32_t dy_cols;
  const uint16_t* x;    // [rows, k]
  uint64_t x_stride;
  uint32_t x_cols;
  float* dw;            // [n, k]
  uint32_t rows, n, k;
  uint32_t accumulate;
  uint32_t splits, split_rows;  // tokens per split (a multiple of 64)
  float* partial;               // [splits, n, k] where splits > 1
};

// dw[n, k] = sum_t dy[t, n] x[t, k], both operands staged through LDS, for bf16
// matrices whose rows are whole dwords (a copy's range ends with the last row, and
// ends are checked per dword). Both have the contraction (tokens) as their slow
// dimension, so their rows are copied as they are and the transposed LDS reads
// (ds_read_b64_tr_b16: among 16 lanes, lane i gets element i % 4 of the 8 bytes
// that lanes i / 4 + 0, 4, 8, 12 address) turn 4 tokens x 16 columns into operand
// rows. A stage holds 64 tokens; a token's row is kept in 32-byte groups (16
// columns) of which group c sits at c ^ f(t), f(t) = t % 4 + 4 (t / 8 % 2): the 16
// tokens of one read then meet every bank twice, which is what 512 bytes need.
// Workgroups, waves and the stage hand-over are product_tile's. Columns past the
// matrix read the next row and make outputs that are not stored; tokens past the
// end read zeros. 128x256 at T 4096, N 4096, K 2048: 61 us as a call of its own, 64 behind the
// input gradient (1.1 PFLOP/s; a library product of the same size 79 us, a large one 1.42
// PFLOP/s). A step takes 1950 cycles for 1024 of products: by counters the matrix cores are busy
// 52% of the waves' time, LDS 26%, and a wave spends 28% of it at the barrier or behind copies and 36%
// waiting to issue. Reading less from LDS, by waves of 64 x 128 over one half of a step's tokens each
// and a sum of the halves at the end, takes 62.5 us against 61.5, and 9.0 instead of 8.3 at T 333, N
// 1024, K 2048: the longer wait for a step's first operands costs as much. Two groups of waves in
// turn, product_turns' way, take 76 us, steps of 32 tokens in six stages 70, operands read two tiles
// ahead the same 62, non-temporal stores 64. 256x256 at T 8192, N 4096, K 4096: 206 us as a call (1.33
// PFLOP/s; with non-temporal stores 209), with its two stages' copies spread over the whole step
// 6% longer; about 30 are its stores, which nothing hides with one workgroup per CU, and with all
// copies from lines the cache holds it takes 40 less.
template <uint32_t WP, uint32_t WQ, uint32_t NP, uint32_t NQ, uint32_t S>
constexpr uint32_t outer_lds() {
  return S * 64u * 32u * (WP * NP + WQ * NQ);
}
template <uint32_t WP, uint32_t WQ, uint32_t NP, uint32_t NQ, uint32_t S>
__device__ __forceinline__ void outer_tile(const Outer& a, uint32_t group, uint8_t* s_stage) {
  constexpr uint32_t kP = WP * NP, kQ = WQ * NQ, kTokens = 64u;
  constexpr uint32_t kRowP = kP * 32u, kRowQ = kQ * 32u;  // bytes of a token's row
  constexpr uint32_t kStage = kTokens * (kRowP + kRowQ);
  constexpr uint32_t kCopies = kStage / 8192u;            // a wave's, per step
  static_assert(WP * WQ == 8u && (kRowP == 256u || kRowP == 512u) && (kRowQ == 256u || kRowQ == 512u) &&
                    S * kStage == outer_lds<WP, WQ, NP, NQ, S>() && S * kStage <= 160u * 1024u,
                "copies, swizzle and LDS");
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t np = (a.k + 16u * kP - 1u) / (16u * kP), nq = (a.n + 16u * kQ - 1u) / (16u * kQ);
  const uint32_t total = np * nq * a.splits, per = (total + 7u) / 8u;
  const uint32_t item = (group % 8u) * per + group / 8u;
  if (group / 8u >= per || item >= total) return;
  const uint32_t split = item / (np * nq), tile = item - split * np * nq;
  const uint32_t band = tile / (4u * np), in_band = tile - band * 4u * np;
  const uint32_t height = min(4u, nq - band * 4u);
  const uint32_t p0 = in_band / height * 16u * kP, q0 = (band * 4u + in_band % height) * 16u * kQ;  // first columns
  const uint32_t wp = wave % WP, wq = wave / WP;
  // this split's tokens
  const uint32_t t0 = split * a.split_rows, t1 = min(a.rows, t0 + a.split_rows);

  // lane's place in a copy of 1 KiB: row r of the 1024 / row bytes, 16-byte chunk
  auto lane_offset = [&](uint32_t row_bytes, uint64_t stride) __attribute__((always_inline)) {
    const uint32_t lanes = row_bytes / 16u, r = lane / lanes, chunk = lane % lanes;
    const uint32_t t = wave * (64u / lanes) + r;  // (rows 16 or 32 further have the same f)
    const uint32_t f = (t & 3u) | ((t >> 3) & 1u) << 2;
    return r * (uint32_t)stride * 2u + (chunk ^ (f << 1)) * 16u;
  };
  const uint32_t pv = lane_offset(kRowP, a.x_stride), qv = lane_offset(kRowQ, a.dy_stride);
  const uint32_t lds0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)nklds2::lds_offset(&s_stage[0]));
  // Copy i of a wave's kCopies for tokens t .. min(t1, t + 64) - 1 (x's, then dy's); from
  // t1 on it reads nothing and leaves zeros, so that a step's code has no branch.
  auto issue_part = [&](uint32_t t, uint32_t stage, uint32_t i) __attribute__((always_inline)) {
    constexpr uint32_t kCopiesP = kTokens * kRowP / 8192u;
    const bool is_p = i < kCopiesP, live = t < t1;
    const uint32_t row_bytes = is_p ? kRowP : kRowQ, each = 1024u / row_bytes;  // rows per copy
    const uint32_t row = ((is_p ? i : i - kCopiesP) * 8u + wave) * each;
    const uint64_t stride = is_p ? a.x_stride : a.dy_stride;
    const uint32_t c0 = is_p ? p0 : q0, cols = is_p ? a.x_cols : a.dy_cols;
    const uint32_t n = min(kTokens, t1 - min(t, t1 - 1u));
    const u32x4 r = nklds2::rsrc((is_p ? a.x : a.dy) + (uint64_t)t * stride + c0,
                                 live ? ((n - 1u) * (uint32_t)stride + (cols - c0)) * 2u : 0u);
    nklds2::copy16(lds0 + stage * kStage + (is_p ? 0u : kTokens * kRowP) + row * row_bytes, r, is_p ? pv : qv,
                   live ? row * (uint32_t)stride * 2u : 0u);
  };

  v4f acc[NP][NQ];
#pragma unroll
  for (uint32_t i = 0; i < NP; ++i)
#pragma unroll
    for (uint32_t j = 0; j < NQ; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const uint32_t c = lane & 15u, g = lane >> 4;
  const uint32_t f = (c >> 2) | (g & 1u) << 2;  // of the tokens this lane addresses
  // operand of column tile `tile` and tokens 32 h ..: tokens 32 h + 8 g .. + 7
  auto operand = [&](const uint8_t* m, uint32_t row_bytes, uint32_t tile, uint32_t h) __attribute__((always_inline)) {
    typedef short v4s __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4s* lds_v4s;
    const uint8_t* at = m + (h * 32u + g * 8u + (c >> 2)) * row_bytes + (tile ^ f) * 32u + (c & 3u) * 8u;
    const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)at);
    const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(at + 4u * row_bytes));
    typedef short v8s __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(v8bf, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
#pragma unroll
  for (uint32_t i = 0; i + 1u < S; ++i)
#pragma unroll
    for (uint32_t k = 0; k < kCopies; ++k) issue_part(t0 + i * kTokens, i, k);
  uint32_t stage = 0u;
  for (uint32_t t = t0; t < t1; t += kTokens) {
    nklds2::wait_copies<(S - 2u) * kCopies>();
    nklds2::barrier();
    const uint32_t before = stage == 0u ? S - 1u : stage - 1u;
    const uint8_t* px = s_stage + stage * kStage;
    const uint8_t* pq = px + kTokens * kRowP;
    stage = stage + 1u == S ? 0u : stage + 1u;
    v8bf qo[2][NQ], po[2];
    po[0] = operand(px, kRowP, wp * NP, 0u);
#pragma unroll
    for (uint32_t j = 0; j < NQ; ++j) qo[0][j] = operand(pq, kRowQ, wq * NQ + j, 0u);
    // tile i of the first 32 tokens, then of the second
#pragma unroll
    for (uint32_t i = 0; i < 2u * NP; ++i) {
      if (i + 1u < 2u * NP) po[(i + 1u) & 1u] = operand(px, kRowP, wp * NP + (i + 1u) % NP, (i + 1u) / NP);
      if (i == NP - 1u) {
#pragma unroll
        for (uint32_t j = 0; j < NQ; ++j) qo[1][j] = operand(pq, kRowQ, wq * NQ + j, 1u);
      }
#pragma unroll
      for (uint32_t j = 0; j < NQ; ++j)
        acc[i % NP][j] =
            __builtin_amdgcn_mfma_f32_16x16x32_bf16(po[i & 1u], qo[i / NP][j], acc[i % NP][j], 0, 0, 0);
      // the copies of a later step, spread over this one's products (with two stages, where
      // they are the next step's, over the first half of them)
      constexpr uint32_t kOver = S == 2u ? NP : 2u * NP;
#pragma unroll
      for (uint32_t k = min(kOver, i) * kCopies / kOver; k < min(kOver, i + 1u) * kCopies / kOver; ++k)
        issue_part(t + (S - 1u) * kTokens, before, k);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  nklds2::wait_copies<0>();
  float* dst = a.splits > 1u ? a.partial + (size_t)split * a.n * a.k : a.dw;
  const bool add = a.accumulate && a.splits == 1u;
#pragma unroll
  for (uint32_t j = 0; j < NQ; ++j) {
    const uint32_t row = q0 + (wq * NQ + j) * 16u + c;
#pragma unroll
    for (uint32_t i = 0; i < NP; ++i) {
      const uint32_t col = p0 + (wp * NP + i) * 16u + g * 4u;
      if (row >= a.n || col >= a.k) continue;
      float* o = dst + (uint64_t)row * a.k + col;
      float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
      if (add) {
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e)
          if (col + e < a.k) v[e] += o[e];
      }
      store4(o, a.k - col, v);
    }
  }
}

// dw = (dw +) the sum of the splits, in split order.
__device__ __forceinline__ void outer_sum(const Outer& a) {
  const uint64_t n = (uint64_t)a.n * a.k;
  for (uint64_t i = ((uint64_t)blockIdx.x * 256u + threadIdx.x) * 4u; i < n; i += (uint64_t)gridDim.x * 1024u) {
    if (i + 4u <= n && reinterpret_cast<uintptr_t>(a.dw) % 16u == 0u && n % 4u == 0u) {
      float4 s = *reinterpret_cast<const float4*>(a.partial + i);
      for (uint32_t k = 1; k < a.splits; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(a.partial + k * n + i);
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
      }
      float4* o = reinterpret_cast<float4*>(a.dw + i);
      if (a.accumulate) {
        const float4 v = *o;
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
      }
      *o = s;
    } else {
      for (uint64_t j = i; j < min(i + 4u, n); ++j) {
        float s = a.partial[j];
        for (uint32_t k = 1; k < a.splits; ++k) s += a.partial[k * n + j];
        a.dw[j] = a.accumulate ? a.dw[j] + s : s;
      }
    }
  }
}

// A matrix as bf16 with rows of `pitch` elements (a multiple of 8, zeros behind the columns), for
// operands that are fp32 or not aligned. Group g of `groups`: four rows and 512 columns at a time.
struct Copy {
  const void* m;
  uint64_t stride;
  uint16_t* out;
  uint32_t type, cols, pitch, groups;  // groups: a multiple of pitch / 512 rounded up, or 0
};
__device__ __forceinline__ void pack8(const uint16_t* p, uint32_t left, uint32_t (&w)[4]) {
  if (left >= 8u) {
    const Unaligned16 u = *reinterpret_cast<const Unaligned16*>(p);
#pragma unroll
    for (uint32_t e = 0; e < 4u; ++e) w[e] = u.w[e];
    return;
  }
#pragma unroll
  for (uint32_t e = 0; e < 8u; ++e)
    if (e < left) w[e / 2u] |= (uint32_t)p[e] << (16u * (e & 1u));
}
__device__ __forceinline__ void pack8(const float* p, uint32_t left, uint32_t (&w)[4]) {
  float v[8] = {};
  if (left >= 8u) {
    const Unaligned16 lo = *reinterpret_cast<const Unaligned16*>(p), hi = *reinterpret_cast<const Unaligned16*>(p + 4);
#pragma unroll
    for (uint32_t e = 0; e < 4u; ++e) {
      v[e] = __uint_as_float(lo.w[e]);
      v[e + 4u] = __uint_as_float(hi.w[e]);
    }
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 8u; ++e)
      if (e < left) v[e] = p[e];
  }
#pragma unroll
  for (uint32_t e = 0; e < 4u; ++e) w[e] = nk::bf16x2_hw(v[2u * e], v[2u * e + 1u]);
}
template <typename X>
__device__ __forceinline__ void to_bf16(const Copy& a, uint32_t rows, uint32_t g) {
  const uint32_t across = (a.pitch + 511u) / 512u, c = (g % across * 64u + (threadIdx.x & 63u)) * 8u;
  if (c >= a.pitch) return;
  for (uint32_t r = g / across * 4u + (threadIdx.x >> 6); r < rows; r += a.groups / across * 4u) {
    uint32_t w[4] = {};
    if (c < a.cols) pack8(static_cast<const X*>(a.m) + (uint64_t)r * a.stride + c, a.cols - c, w);
    *reinterpret_cast<uint4*>(a.out + (uint64_t)r * a.pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
__device__ __forceinline__ void to_bf16(const Copy& a, uint32_t rows, uint32_t g) {
  if (a.type == NETRA_F32) to_bf16<float>(a, rows, g);
  else to_bf16<uint16_t>(a, rows, g);
}

// What a backward pass needs made of dy and x, in one launch: dy quantised (`quant` workgroups,
// quant_rows's grid of row tiles first), then the copies.
template <typename X>
__device__ __forceinline__ void prepare(const X* dy, uint64_t stride, uint8_t* q, float* s, uint32_t rows, uint32_t n,
                                        uint32_t sld, uint32_t quant, const Copy& a, const Copy& b) {
  uint32_t g = blockIdx.x;
  const uint32_t tiles = (rows + 15u) / 16u;
  if (g < quant) return quant_rows(dy, stride, q, s, rows, n, sld, g % tiles, g / tiles);
  g -= quant;
  if (g < a.groups) to_bf16(a, rows, g);
  else to_bf16(b, rows, g - a.groups);
}

}  // namespace nklin

// Weights: w row-major e4m3 [n, k] -> tiles of w. One wave per tile; bytes past the
// matrix are zeros.
extern "C" __global__ __launch_bounds__(256) void netra_linear_pack_gfx950(const uint8_t* __restrict__ w,
                                                                           uint8_t* __restrict__ dst, uint32_t n,
                                                                           uint32_t k) {
  struct __attribute__((packed, aligned(1))) Bytes {
    uint32_t w[8];
  };
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t kb = (k + 127u) / 128u, b = blockIdx.y * 4u + wave;
  if (b >= kb) return;
  const uint32_t r = blockIdx.x * 16u + (lane & 15u), c = b * 128u + (lane >> 4) * 32u;
  uint32_t code[8] = {};
  if (r < n) {
    const uint8_t* at = w + (size_t)r * k + c;
    if (c + 32u <= k) {
      const Bytes v = *reinterpret_cast<const Bytes*>(at);
#pragma unroll
      for (uint32_t j = 0; j < 8u; ++j) code[j] = v.w[j];
    } else {
#pragma unroll
      for (uint32_t j = 0; j < 32u; ++j)
        if (c + j < k) code[j / 4u] |= (uint32_t)at[j] << (8u * (j % 4u));
    }
  }
  nklin::store_tile(dst + ((size_t)blockIdx.x * kb + b) * 2048u, lane, code);
}

// Tiles of w^T: a workgroup turns 128 rows x 64 columns of w through LDS into four
// tiles (16 columns by 128 rows). An LDS row of 64 bytes is followed by 4, so the
// four row groups of one read start 32 * 17 words apart and its 16 columns share
// four banks in each.
extern "C" __global__ __launch_bounds__(256) void netra_linear_pack_transposed_gfx950(const uint8_t* __restrict__ w,
                                                                                      uint8_t* __restrict__ dst,
                                                                                      uint32_t n, uint32_t k) {
  __shared__ uint32_t rows[128][17];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t nb = (n + 127u) / 128u, c0 = blockIdx.x * 64u, r0 = blockIdx.y * 128u;
#pragma unroll
  for (uint32_t i = 0; i < 8u; ++i) {  // 16 lanes of 4 bytes per row
    const uint32_t r = i * 16u + (threadIdx.x >> 4), c = c0 + (threadIdx.x & 15u) * 4u;
    uint32_t v = 0u;
    if (r0 + r < n) {
      const uint8_t* at = w + (size_t)(r0 + r) * k + c;
#pragma unroll
      for (uint32_t e = 0; e < 4u; ++e)
        if (c + e < k) v |= (uint32_t)at[e] << (8u * e);
    }
    rows[r][threadIdx.x & 15u] = v;
  }
  __syncthreads();
  const uint32_t tile = blockIdx.x * 4u + wave;
  if (tile >= (k + 15u) / 16u) return;
  const uint32_t c = wave * 16u + (lane & 15u), r = (lane >> 4) * 32u;
  uint32_t code[8];
#pragma unroll
  for (uint32_t j = 0; j < 8u; ++j) {
    code[j] = 0u;
#pragma unroll
    for (uint32_t e = 0; e < 4u; ++e)
      code[j] |= ((rows[r + 4u * j + e][c / 4u] >> (8u * (c & 3u))) & 0xffu) << (8u * e);
  }
  nklin::store_tile(dst + ((size_t)tile * nb + blockIdx.y) * 2048u, lane, code);
}

extern "C" __global__ __launch_bounds__(256) void netra_linear_quant_rows_bf16_gfx950(
    const uint16_t* x, uint64_t stride, uint8_t* q, float* s, uint32_t rows, uint32_t n, uint32_t sld) {
  nklin::quant_rows(x, stride, q, s, rows, n, sld, blockIdx.x, blockIdx.y);
}
extern "C" __global__ __launch_bounds__(256) void netra_linear_quant_rows_f32_gfx950(
    const float* x, uint64_t stride, uint8_t* q, float* s, uint32_t rows, uint32_t n, uint32_t sld) {
  nklin::quant_rows(x, stride, q, s, rows, n, sld, blockIdx.x, blockIdx.y);
}

#define NETRA_PRODUCT_TILE(P, Q, ...)                                                                             \
  extern "C" __global__ __launch_bounds__(512) void netra_linear_product_##P##x##Q##_gfx950(nklin::Product a) {    \
    __shared__ __align__(16) uint8_t lds[nklin::Tile<__VA_ARGS__>::kLds];                                         \
    nklin::product_tile<__VA_ARGS__>(a, blockIdx.x, lds);                                                         \
  }
extern "C" __global__ __launch_bounds__(512) void netra_linear_product_256x256_gfx950(nklin::Product a) {
  __shared__ __align__(16) uint8_t lds[nklin::Tile<2, 4, 8, 4, 2>::kLds];
  nklin::product_turns(a, blockIdx.x, lds);
}
NETRA_PRODUCT_TILE(256, 128, 4, 2, 4, 4, 3)
NETRA_PRODUCT_TILE(128, 128, 2, 4, 4, 2, 4)
NETRA_PRODUCT_TILE(128, 64, 4, 2, 2, 2, 4)
NETRA_PRODUCT_TILE(64, 64, 4, 2, 1, 2, 4)
extern "C" __global__ __launch_bounds__(256) void netra_linear_product_sum_gfx950(nklin::Product a) {
  nklin::product_sum(a);
}

#define NETRA_PRODUCT_FUSED(NAME, X, NP, NQ)                                                                 \
  extern "C" __global__ __launch_bounds__(512) void netra_linear_product_fused_##NAME##_p##NP##q##NQ##_gfx950( \
      nklin::Product a, const X* x, uint64_t x_stride, uint32_t n) {                                         \
    nklin::product_stream<NP, NQ, true, X>(a, x, x_stride, n);                                               \
  }
#define NETRA_PRODUCTS_FUSED(NP, NQ)           \
  NETRA_PRODUCT_FUSED(bf16, uint16_t, NP, NQ)  \
  NETRA_PRODUCT_FUSED(f32, float, NP, NQ)
NETRA_PRODUCTS_FUSED(1, 1)
NETRA_PRODUCTS_FUSED(2, 1)
NETRA_PRODUCTS_FUSED(1, 2)
NETRA_PRODUCTS_FUSED(2, 2)
NETRA_PRODUCT_FUSED(bf16, uint16_t, 1, 4)  // (fp32 rows of four tiles do not fit the registers)
#define NETRA_PRODUCT_STREAM(NP, NQ)                                                                                  \
  extern "C" __global__ __launch_bounds__(512) void netra_linear_product_stream_p##NP##q##NQ##_gfx950(nklin::Product a) { \
    nklin::product_stream<NP, NQ, false, uint16_t>(a, nullptr, 0, 0);                                                 \
  }
NETRA_PRODUCT_STREAM(1, 4)
NETRA_PRODUCT_STREAM(2, 4)

#define NETRA_OUTER_TILE(P, Q, ...)                                                                                \
  extern "C" __global__ __launch_bounds__(512) void netra_linear_outer_##P##x##Q##_gfx950(nklin::Outer a) {        \
    __shared__ __align__(16) uint8_t lds[nklin::outer_lds<__VA_ARGS__>()];                                         \
    nklin::outer_tile<__VA_ARGS__>(a, blockIdx.x, lds);                                                           \
  }
NETRA_OUTER_TILE(256, 256, 2, 4, 8, 4, 2)
NETRA_OUTER_TILE(128, 256, 2, 4, 4, 4, 3)
NETRA_OUTER_TILE(128, 128, 2, 4, 4, 2, 4)
// Both products of a small backward pass in one launch, the weight gradient's
// workgroups (the first `outer`, a multiple of 8) with their longer way first: neither
// fills the chip, and a launch is saved (T 333, N 1024, K 2048: a call 13.4 us, this kernel 9.6 at
// best and 11.0 in the middle; in two launches 16.9).
extern "C" __global__ __launch_bounds__(512) void netra_linear_backward_small_gfx950(nklin::Product a, nklin::Outer b,
                                                                                     uint32_t outer) {
  constexpr uint32_t kP = nklin::Tile<4, 2, 1, 2, 4>::kLds, kO = nklin::outer_lds<2, 4, 4, 2, 4>();
  __shared__ __align__(16) uint8_t lds[kP > kO ? kP : kO];
  if (blockIdx.x < outer) nklin::outer_tile<2, 4, 4, 2, 4>(b, blockIdx.x, lds);
  else nklin::product_tile<4, 2, 1, 2, 4>(a, blockIdx.x - outer, lds);
}
extern "C" __global__ __launch_bounds__(256) void netra_linear_outer_sum_gfx950(nklin::Outer a) { nklin::outer_sum(a); }

#define NETRA_PREPARE(NAME, X)                                                                                    \
  extern "C" __global__ __launch_bounds__(256) void netra_linear_prepare_##NAME##_gfx950(                        \
      const X* dy, uint64_t stride, uint8_t* q, float* s, uint32_t rows, uint32_t n, uint32_t sld, uint32_t quant, \
      nklin::Copy a, nklin::Copy b) {                                                                             \
    nklin::prepare(dy, stride, q, s, rows, n, sld, quant, a, b);                                                  \
  }
NETRA_PREPARE(bf16, uint16_t)
NETRA_PREPARE(f32, float)

// dw of no tokens: zeros.
extern "C" __global__ __launch_bounds__(256) void netra_linear_zero_gfx950(float* out, uint64_t n) {
  for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256u) out[i] = 0.0f;
}
