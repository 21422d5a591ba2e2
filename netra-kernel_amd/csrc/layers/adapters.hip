// Low-rank adapters of many requests beside a shared projection: out = y + s_l B_l (A_l x) for each
// token with its adapter l.
//
// A plan sorts the batch's tokens by adapter into tiles of one adapter each; every layer of a step
// uses the same one. Then two products: u = A x (contraction k, the ranks of a tile's tokens as
// fp32) and out = y + s B u (contraction of the rank). Operands are packed once so that a lane's
// operand bytes lie together:
//   A  [adapter][128-block of k][16 ranks][4][64 lanes][8]: lane l's operand j is rank l % 16,
//      columns 32 j + 8 (l / 16) .. + 7 of the block
//   B  [adapter][64 columns][32 ranks][4][64 lanes][8]: lane l's operand j is column 16 j + l % 16,
//      ranks 8 (l / 16) .. + 7; of a rank up to 16
//      [adapter][64 columns][2][64 lanes][2][4]: operands 2 h and 2 h + 1 of a lane, ranks 4 (l / 16) .. + 3
// u goes into the second product as the sum of two bf16 values (the rounded value and what the
// rounding left), each in matrix instructions of its own: 16 bits instead of 8, at no cost where memory is the bound.
// A rank up to 16 has both in one instruction, with B's operand twice.
//
// Memory bounds large batches: T 8192, N 8192, K 4096, rank 64 89 us, of which the first product takes 20 (67 MB of x)
// and the second 69 (269 MB of y and out, 3.9 TB/s); small ones are one launch (T 64, 32 adapters of rank 16, N = K = 2048:
// 6 us).
#pragma once
#include "linear_fp8.hip"

namespace nkada {

using nk::u32x2;
using nk::u32x4;
using nk::v4f;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kMaxAdapters = 1024, kMaxRank = 128;

// Plan words: tiles, tokens, adapters, 0; the tokens by adapter (those without one last, as
// adapter `adapters`); the tiles {adapter, first, tokens, 0}.
constexpr uint32_t kPlanHead = 4;
__device__ __forceinline__ const uint4* plan_tiles(const uint32_t* plan, uint32_t tokens) {
  return reinterpret_cast<const uint4*>(plan + kPlanHead + (tokens + 3u) / 4u * 4u);
}

// The plan by one workgroup: 16 waves count a run of the tokens each, then place them in order.
// Within 64 tokens a lane's place is the number of lanes before it with the same adapter, found one
// adapter at a time. Once for all layers of a step; in us, for one token 4.6, for 64 of 32 adapters 7.3, for 8192 of 8 in runs
// of 700 17 and of 64 in no order 51. A long batch waits for its one workgroup: 65536 tokens of one adapter 160, 2^21 5400
// (of 1024 in no order 17800).
__device__ __forceinline__ void make_plan(const int32_t* __restrict__ ids, uint32_t tokens, uint32_t adapters,
                                          uint32_t tile, uint32_t* plan) {
  __shared__ uint32_t count[16][kMaxAdapters + 1];
  __shared__ uint32_t scan[2][16], carry[2];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, parts = adapters + 1u;
  for (uint32_t i = threadIdx.x; i < 16u * (kMaxAdapters + 1u); i += 1024u) count[i / (kMaxAdapters + 1u)][i % (kMaxAdapters + 1u)] = 0u;
  if (threadIdx.x < 2u) carry[threadIdx.x] = 0u;
  __syncthreads();
  const uint32_t each = ((tokens + 15u) / 16u + 63u) / 64u * 64u, t0 = wave * each, t1 = min(tokens, t0 + each);
  auto adapter = [&](uint32_t t) __attribute__((always_inline)) { return min((uint32_t)ids[t], adapters); };
  for (uint32_t t = t0 + lane; t < t1; t += 64u) atomicAdd(&count[wave][adapter(t)], 1u);
  __syncthreads();
  // an adapter's tokens and tiles before it, 1024 adapters at a time
  uint4* tiles = const_cast<uint4*>(plan_tiles(plan, tokens));
  for (uint32_t first = 0; first < parts; first += 1024u) {
    const uint32_t l = first + threadIdx.x;
    uint32_t n = 0u;
    if (l < parts)
      for (uint32_t w = 0; w < 16u; ++w) n += count[w][l];
    uint32_t own[2] = {n, (n + tile - 1u) / tile}, before[2];
#pragma unroll
    for (uint32_t s = 0; s < 2u; ++s) {
      uint32_t v = own[s];
      for (uint32_t d = 1; d < 64u; d *= 2u) {
        const uint32_t o = (uint32_t)__shfl_up((int)v, d);
        if (lane >= d) v += o;
      }
      if (lane == 63u) scan[s][wave] = v;
      before[s] = v - own[s];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t s = 0; s < 2u; ++s) {
      before[s] += carry[s];
      for (uint32_t w = 0; w < wave; ++w) before[s] += scan[s][w];
    }
    __syncthreads();
    if (threadIdx.x == 1023u) {
      carry[0] = before[0] + own[0];
      carry[1] = before[1] + own[1];
    }
    if (l < parts) {
      uint32_t at = before[0];
      for (uint32_t w = 0; w < 16u; ++w) {
        const uint32_t c = count[w][l];
        count[w][l] = at;
        at += c;
      }
      for (uint32_t i = 0; i < own[1]; ++i)
        tiles[before[1] + i] = make_uint4(l, before[0] + i * tile, min(tile, n - i * tile), 0u);
    }
    __syncthreads();
  }
  if (threadIdx.x == 0u) {
    plan[0] = carry[1];
    plan[1] = tokens;
    plan[2] = adapters;
    plan[3] = 0u;
  }
  for (uint32_t b = t0; b < t1; b += 64u) {
    const uint32_t t = b + lane;
    const bool there = t < t1;
    const uint32_t l = there ? adapter(t) : 0u;
    uint64_t left = __ballot(there);
    while (left) {
      const uint32_t who = (uint32_t)__builtin_amdgcn_readlane((int)l, __ffsll((unsigned long long)left) - 1);
      const uint64_t with = __ballot(there && l == who);
      const uint32_t at = count[wave][who];
      if (there && l == who) plan[kPlanHead + at + __popcll(with & ((1ull << lane) - 1ull))] = t;
      if (lane == 0u) count[wave][who] = at + __popcll(with);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      left &= ~with;
    }
  }
}

// Packing: a thread per 8 values of A, 4 of B; zeros outside the matrices. Weights bf16 or fp32.
template <typename X>
__device__ __forceinline__ uint32_t bf16_at(const X* m, uint64_t i, bool there) {
  if (!there) return 0u;
  if constexpr (sizeof(X) == 2) return m[i];
  else return nk::bf16_rne(m[i]);
}
template <typename X>
__device__ __forceinline__ void pack_a(const X* __restrict__ a, uint4* __restrict__ out, uint32_t adapters, uint32_t rank,
                                       uint32_t k, uint32_t nr) {
  const uint32_t kb = (k + 127u) / 128u;
  const uint64_t all = (uint64_t)adapters * kb * nr * 256u;
  for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < all; i += (uint64_t)gridDim.x * 256u) {
    const uint32_t lane = (uint32_t)(i & 63u), j = (uint32_t)(i >> 6) & 3u;
    const uint64_t rest = i >> 8, block = rest / nr;
    const uint32_t r = (uint32_t)(rest % nr) * 16u + (lane & 15u), c = (uint32_t)(block % kb) * 128u + j * 32u + (lane >> 4) * 8u;
    const uint64_t row = ((block / kb) * rank + r) * (uint64_t)k;
    uint32_t w[4];
#pragma unroll
    for (uint32_t h = 0; h < 4u; ++h)
      w[h] = bf16_at(a, row + c + 2u * h, r < rank && c + 2u * h < k) |
             bf16_at(a, row + c + 2u * h + 1u, r < rank && c + 2u * h + 1u < k) << 16;
    out[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
template <typename X>
__device__ __forceinline__ void pack_b(const X* __restrict__ b, uint2* __restrict__ out, uint32_t adapters, uint32_t rank,
                                       uint32_t n, uint32_t nr) {
  const uint32_t nb = (n + 63u) / 64u;
  const uint64_t all = (uint64_t)adapters * nb * nr * 256u;
  for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < all; i += (uint64_t)gridDim.x * 256u) {
    const uint32_t lane = (uint32_t)(i >> 1) & 63u, odd = (uint32_t)i & 1u;
    const uint32_t j = nr == 1u ? ((uint32_t)(i >> 7) & 1u) * 2u + odd : (uint32_t)(i >> 7) & 3u;
    const uint64_t rest = i / (nr == 1u ? 256u : 512u), parts = nr == 1u ? 1u : nr / 2u, block = rest / parts;
    const uint32_t r = nr == 1u ? (lane >> 4) * 4u : (uint32_t)(rest % parts) * 32u + (lane >> 4) * 8u + odd * 4u;
    const uint32_t c = (uint32_t)(block % nb) * 64u + 16u * j + (lane & 15u);
    const uint64_t row = ((block / nb) * n + c) * (uint64_t)rank;
    uint32_t w[2];
#pragma unroll
    for (uint32_t h = 0; h < 2u; ++h)
      w[h] = bf16_at(b, row + r + 2u * h, c < n && r + 2u * h < rank) |
             bf16_at(b, row + r + 2u * h + 1u, c < n && r + 2u * h + 1u < rank) << 16;
    out[i] = make_uint2(w[0], w[1]);
  }
}

struct Adapters {
  const void* x;
  uint64_t x_stride;
  const uint8_t* a;
  const uint8_t* b;
  const float* scale;
  const uint32_t* plan;
  // A x by the plan's order of tokens: of one split scaled, rounded and what that left, bf16 [2][tokens][16 nr]; of
  // more fp32 [splits][tokens][16 nr]
  void* u;
  uint32_t splits, split_blocks;  // of k's 128-blocks
  const uint16_t* y;
  uint64_t y_stride;
  uint16_t* out;
  uint64_t out_stride;
  uint32_t tokens, adapters, rank, ranks, n, k, in_place;  // ranks: 16-rank parts
  uint32_t wide, chunks;      // wide: groups of 256 columns a workgroup takes; chunks: workgroups across the columns
};

__device__ __forceinline__ bool tile_of(const Adapters& a, uint32_t at, uint4& tile) {
  if (a.plan[1] != a.tokens || a.plan[2] != a.adapters || at >= a.plan[0]) return false;
  tile = plan_tiles(a.plan, a.tokens)[at];
  return true;
}

using nklin::Unaligned16;

// 8 neighbouring columns of a row as they lie in memory, from c on, and as bf16.
template <typename X>
struct Part {
  Unaligned16 w[sizeof(X) / 2u];
};
template <typename X>
__device__ __forceinline__ Part<X> part_whole(const X* row, uint32_t c) {
  Part<X> v;
#pragma unroll
  for (uint32_t h = 0; h < sizeof(X) / 2u; ++h) v.w[h] = *reinterpret_cast<const Unaligned16*>(row + c + 4u * h);
  return v;
}
// The same with zeros from column n on, of which nothing is read: the row's last eight, moved down. (Value by value, the
// lanes at a row's end hold up their whole wave for eight loads.)
template <typename X>
__device__ __forceinline__ Part<X> part_to(const X* row, uint32_t c, uint32_t n) {
  Part<X> v = {};
  if (n < 8u) {
#pragma unroll
    for (uint32_t i = 0; i < 7u; ++i)
      if (c + i < n) {
        if constexpr (sizeof(X) == 4) v.w[i / 4u].w[i & 3u] = __float_as_uint(row[c + i]);
        else v.w[0].w[i / 2u] |= (uint32_t)row[c + i] << (16u * (i & 1u));
      }
    return v;
  }
  const uint32_t at = min(c, n - 8u), by = min(c - at, 8u);
  v = part_whole(row, at);
  if constexpr (sizeof(X) == 4) {
    uint32_t w[8];
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) w[i] = v.w[i / 4u].w[i & 3u];
#pragma unroll
    for (uint32_t d = 1; d < 8u; d *= 2u)
#pragma unroll
      for (uint32_t i = 0; i < 8u; ++i) w[i] = by & d ? (i + d < 8u ? w[i + d] : 0u) : w[i];
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) v.w[i / 4u].w[i & 3u] = by < 8u ? w[i] : 0u;
  } else {
    const uint64_t lo = (uint64_t)v.w[0].w[1] << 32 | v.w[0].w[0], hi = (uint64_t)v.w[0].w[3] << 32 | v.w[0].w[2];
    const uint32_t bits = 16u * (by & 3u);
    const uint64_t up = hi >> bits, down = lo >> bits | (bits ? hi << (64u - bits) : 0u);
    const uint64_t first = by < 4u ? down : by < 8u ? up : 0u, second = by < 4u ? up : 0u;
    v.w[0].w[0] = (uint32_t)first;
    v.w[0].w[1] = (uint32_t)(first >> 32);
    v.w[0].w[2] = (uint32_t)second;
    v.w[0].w[3] = (uint32_t)(second >> 32);
  }
  return v;
}
template <typename X>
__device__ __forceinline__ bf16x8 operand(const Part<X>& v) {
  u32x4 w;
#pragma unroll
  for (uint32_t h = 0; h < 4u; ++h) {
    if constexpr (sizeof(X) == 2) w[h] = v.w[0].w[h];
    else w[h] = nk::bf16x2_hw(__uint_as_float(v.w[h / 2u].w[2u * (h & 1u)]), __uint_as_float(v.w[h / 2u].w[2u * (h & 1u) + 1u]));
  }
  return __builtin_bit_cast(bf16x8, w);
}

// Four ranks of u from r on, scaled, as a rounded and a left-over bf16 value each. Ranks past the last are zeros times
// what x holds, which is not 0 where that is an infinity.
__device__ __forceinline__ void split(v4f v, float scale, uint32_t r, uint32_t rank, u32x2& hi, u32x2& lo) {
  float h[4], l[4];
#pragma unroll
  for (uint32_t e = 0; e < 4u; ++e) {
    const float f = r + e < rank ? v[e] * scale : 0.0f;
    h[e] = nk::bf16_round_hw(f);
    l[e] = fabsf(h[e]) < __builtin_inff() ? f - h[e] : 0.0f;
  }
  hi = u32x2{nk::bf16x2_hw(h[0], h[1]), nk::bf16x2_hw(h[2], h[3])};
  lo = u32x2{nk::bf16x2_hw(l[0], l[1]), nk::bf16x2_hw(l[2], l[3])};
}

// The first product of a tile of TT times 16 tokens by 16 NR ranks from the 16-rank part r0 on: the eight waves of a
// workgroup share k's blocks out among them and leave their sums in LDS, to be joined in the order of the waves.
//
// A wave's loads are counted in the order in which they are issued, so waiting for A (from the L2) waits for all of
// x that was asked for before it (from memory). A block goes in two halves; a half's A is asked for before the next
// half's x. (Both a half further ahead takes 170 registers instead of 122, one workgroup on a CU instead of two: 39.5 us
// instead of 35.7 at T 8192, K 4096, rank 64 when it was tried, with tiles of 64 tokens; tiles of 32 take 20.)
template <typename X, uint32_t TT, uint32_t NR>
__device__ __forceinline__ void first_product(const Adapters& a, const uint4& tile, uint32_t split_at, uint32_t r0,
                                              v4f (&part)[8][TT * NR][64]) {
  constexpr uint32_t W = 8u;
  const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t kb = (a.k + 127u) / 128u, b1 = min(kb, (split_at + 1u) * a.split_blocks), c = (lane >> 4) * 8u;
  const X* row[TT];
#pragma unroll
  for (uint32_t t = 0; t < TT; ++t) {
    const uint32_t at = min(t * 16u + (lane & 15u), tile.z - 1u);  // (past the tile its last token again)
    row[t] = static_cast<const X*>(a.x) + (uint64_t)a.plan[kPlanHead + tile.y + at] * a.x_stride;
  }
  v4f acc[TT][NR];
#pragma unroll
  for (uint32_t t = 0; t < TT; ++t)
#pragma unroll
    for (uint32_t r = 0; r < NR; ++r) acc[t][r] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const u32x4* ab = reinterpret_cast<const u32x4*>(a.a) + ((uint64_t)tile.x * kb * a.ranks + r0) * 256u + lane;
  u32x4 wa[NR][2];    // A of a half
  Part<X> x[2][TT][2];  // x of both
  auto load_a = [&](uint32_t b, uint32_t h) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t r = 0; r < NR; ++r)
#pragma unroll
      for (uint32_t j = 0; j < 2u; ++j) wa[r][j] = ab[((uint64_t)b * a.ranks + r) * 256u + (2u * h + j) * 64u];
  };
  auto load_x = [&](uint32_t b, uint32_t h) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t j = 0; j < 2u; ++j)
#pragma unroll
      for (uint32_t t = 0; t < TT; ++t) x[h][t][j] = part_whole(row[t], b * 128u + (2u * h + j) * 32u + c);
  };
  auto products = [&](uint32_t h) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t j = 0; j < 2u; ++j)
#pragma unroll
      for (uint32_t r = 0; r < NR; ++r)
#pragma unroll
        for (uint32_t t = 0; t < TT; ++t)
          acc[t][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wa[r][j]), operand(x[h][t][j]),
                                                              acc[t][r], 0, 0, 0);
  };
  // The wave's blocks: every 8th from b0 on. Each wave begins with another one, so that at any time the workgroups
  // read all places of their rows: all in step they read one place, which is a part of the memory's channels where
  // rows are a power of two apart (67 MB read alone: 18.0 us, so 12.1).
  const uint32_t b0 = split_at * a.split_blocks + wave;
  const uint32_t whole = min(b1, a.k / 128u);  // blocks that end inside the rows
  const uint32_t count = b0 < whole ? (whole - b0 + W - 1u) / W : 0u;
  if (count) {
    uint32_t at = wave % count, b = b0 + at * W;
    load_x(b, 0u);
    for (uint32_t i = 0; i < count; ++i) {
      at = at + 1u == count ? 0u : at + 1u;  // (behind the last one the first again, from the cache)
      const uint32_t b_next = b0 + at * W;
      load_a(b, 0u);
      load_x(b, 1u);
      __builtin_amdgcn_sched_barrier(0);
      products(0u);
      __builtin_amdgcn_sched_barrier(0);
      load_a(b, 1u);
      load_x(b_next, 0u);
      __builtin_amdgcn_sched_barrier(0);
      products(1u);
      __builtin_amdgcn_sched_barrier(0);
      b = b_next;
    }
  }
  const uint32_t b = b0 + count * W;
  if (b < b1) {  // the last block, short
#pragma unroll
    for (uint32_t h = 0; h < 2u; ++h) {
#pragma unroll
      for (uint32_t j = 0; j < 2u; ++j)
#pragma unroll
        for (uint32_t t = 0; t < TT; ++t) x[h][t][j] = part_to(row[t], b * 128u + (2u * h + j) * 32u + c, a.k);
      load_a(b, h);
      products(h);
    }
  }
#pragma unroll
  for (uint32_t t = 0; t < TT; ++t)
#pragma unroll
    for (uint32_t r = 0; r < NR; ++r) part[wave][t * NR + r][lane] = acc[t][r];
  __syncthreads();
}
// Four ranks of a token: place i of 64 TT NR.
template <uint32_t N>
__device__ __forceinline__ v4f joined(const v4f (&part)[8][N][64], uint32_t i) {
  v4f v = part[0][i >> 6][i & 63u];
#pragma unroll
  for (uint32_t w = 1; w < 8u; ++w) v += part[w][i >> 6][i & 63u];
  return v;
}

// u of a tile, of NR of its 16-rank parts (the workgroup's place in z), of one split.
template <typename X, uint32_t TT, uint32_t NR>
__device__ __forceinline__ void shrink(const Adapters& a) {
  __shared__ v4f part[8][TT * NR][64];
  uint4 tile;
  if (!tile_of(a, blockIdx.x, tile) || tile.x >= a.adapters) return;
  const uint32_t split_at = blockIdx.y, r0 = blockIdx.z * NR;
  first_product<X, TT, NR>(a, tile, split_at, r0, part);
  for (uint32_t i = threadIdx.x; i < TT * NR * 64u; i += 512u) {
    const uint32_t l = i & 63u, tr = i >> 6, in = tr / NR * 16u + (l & 15u);
    if (in >= tile.z) continue;
    const v4f v = joined(part, i);
    const uint32_t r = (r0 + tr % NR) * 16u + (l >> 4) * 4u, ranks = 16u * a.ranks;
    if (a.splits > 1u) {
      *reinterpret_cast<v4f*>(static_cast<float*>(a.u) + ((uint64_t)split_at * a.tokens + tile.y + in) * ranks + r) = v;
    } else {
      u32x2 hi, lo;
      split(v, a.scale[tile.x], r, a.rank, hi, lo);
      uint16_t* to = static_cast<uint16_t*>(a.u) + (uint64_t)(tile.y + in) * ranks + r;
      *reinterpret_cast<u32x2*>(to) = hi;
      *reinterpret_cast<u32x2*>(to + (uint64_t)a.tokens * ranks) = lo;
    }
  }
}

// Eight columns past the caches.
typedef uint32_t Once16 __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ Unaligned16 load_once(const uint16_t* from) {
  const Once16 v = __builtin_nontemporal_load(reinterpret_cast<const Once16*>(from));
  return {{v[0], v[1], v[2], v[3]}};
}
__device__ __forceinline__ void store_once(uint16_t* to, const Unaligned16& v) {
  __builtin_nontemporal_store(Once16{v.w[0], v.w[1], v.w[2], v.w[3]}, reinterpret_cast<Once16*>(to));
}

__device__ __forceinline__ void store8(uint16_t* row, uint32_t c, uint32_t n, const Unaligned16& v) {
  if (c + 8u <= n) {
    *reinterpret_cast<Unaligned16*>(row + c) = v;
    return;
  }
#pragma unroll
  for (uint32_t i = 0; i < 8u; ++i)
    if (c + i < n) row[c + i] = (uint16_t)(v.w[i / 2u] >> (16u * (i & 1u)));
}

// out of a tile of TT times 16 tokens. The four waves of a workgroup multiply 64 of 256 columns each and hand the
// sums over through LDS, from where a wave adds and stores whole rows of 256 columns, 512 bytes that lie together:
// as the matrix core leaves them a lane has four columns, and rows of 64 bytes stored so took 60% of a copy's rate.
// `wide` times; the next columns' y and B are under way during a turn.
//
// kOnce: y and out non-temporal, where they are more than the caches keep and would push B out of the L2 (adapter_once).
template <uint32_t TT, uint32_t NR, bool kOnce>
__device__ __forceinline__ void expand(const Adapters& a) {
  constexpr uint32_t kPitch = 260u;  // spreads 16 tokens' rows over the banks
  constexpr uint32_t kRows = 4u * TT, kLoads = kRows / 2u;  // rows of a wave; loads of a lane: two rows at a time
  __shared__ float sums[TT * 16u][kPitch];
  uint4 tile;
  const uint32_t at_tile = blockIdx.x / a.chunks, chunk = blockIdx.x - at_tile * a.chunks;
  if (!tile_of(a, at_tile, tile)) return;
  const bool none = tile.x >= a.adapters;
  if (none && a.in_place) return;
  const uint32_t lane = threadIdx.x & 63u, q = lane >> 4;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t nb = (a.n + 63u) / 64u;
  const uint32_t g0 = chunk * a.wide, g1 = min((a.n + 255u) / 256u, g0 + a.wide);  // groups of 256 columns
  // the wave's rows: lanes 0 .. 31 and 32 .. 63 have one each of every load's two
  const uint16_t* from[kLoads];
  uint16_t* to[kLoads];
  bool there[kLoads];
  const uint32_t c = (lane & 31u) * 8u, half = lane >> 5;
#pragma unroll
  for (uint32_t i = 0; i < kLoads; ++i) {
    const uint32_t row = wave * kRows + 2u * i + half;
    there[i] = row < tile.z;
    const uint32_t token = a.plan[kPlanHead + tile.y + min(row, tile.z - 1u)];
    from[i] = a.y + (uint64_t)token * a.y_stride;
    to[i] = a.out + (uint64_t)token * a.out_stride;
  }
  if (none) {
    for (uint32_t g = g0; g < g1; ++g)
#pragma unroll
      for (uint32_t i = 0; i < kLoads; ++i)
        if (there[i]) store8(to[i], g * 256u + c, a.n, part_to(from[i], g * 256u + c, a.n).w[0]);
    return;
  }
  // u's operands: of a rank up to 16 {rounded, left}, else the rounded ones, then the left ones
  constexpr uint32_t kPairs = NR == 1u ? 1u : NR / 2u, kOperands = NR == 1u ? 1u : NR;
  bf16x8 u[TT][kOperands];
#pragma unroll
  for (uint32_t t = 0; t < TT; ++t) {
    const uint32_t at = tile.y + min(t * 16u + (lane & 15u), tile.z - 1u);
    u32x2 hi[NR], lo[NR];  // of four ranks from rank(i) on
    auto rank = [&](uint32_t i) __attribute__((always_inline)) { return NR == 1u ? q * 4u : i / 2u * 32u + q * 8u + (i & 1u) * 4u; };
    if (a.splits == 1u) {
      const uint16_t* from_u = static_cast<const uint16_t*>(a.u) + (uint64_t)at * (16u * NR);
#pragma unroll
      for (uint32_t i = 0; i < NR; ++i) {
        hi[i] = *reinterpret_cast<const u32x2*>(from_u + rank(i));
        lo[i] = *reinterpret_cast<const u32x2*>(from_u + (uint64_t)a.tokens * (16u * NR) + rank(i));
      }
    } else {
      v4f v[NR];
#pragma unroll
      for (uint32_t i = 0; i < NR; ++i) v[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
      for (uint32_t s = 0; s < a.splits; ++s) {
        const float* from_u = static_cast<const float*>(a.u) + ((uint64_t)s * a.tokens + at) * (16u * NR);
#pragma unroll
        for (uint32_t i = 0; i < NR; ++i) v[i] += *reinterpret_cast<const v4f*>(from_u + rank(i));
      }
      const float scale = a.scale[tile.x];
#pragma unroll
      for (uint32_t i = 0; i < NR; ++i) split(v[i], scale, rank(i), a.rank, hi[i], lo[i]);
    }
    if constexpr (NR == 1u) {
      u[t][0] = __builtin_bit_cast(bf16x8, u32x4{hi[0][0], hi[0][1], lo[0][0], lo[0][1]});
    } else {
#pragma unroll
      for (uint32_t p = 0; p < kPairs; ++p) {
        u[t][p] = __builtin_bit_cast(bf16x8, u32x4{hi[2u * p][0], hi[2u * p][1], hi[2u * p + 1u][0], hi[2u * p + 1u][1]});
        u[t][kPairs + p] = __builtin_bit_cast(bf16x8, u32x4{lo[2u * p][0], lo[2u * p][1], lo[2u * p + 1u][0], lo[2u * p + 1u][1]});
      }
    }
  }
  const u32x4* b_at = reinterpret_cast<const u32x4*>(a.b) + (uint64_t)tile.x * nb * NR * 128u + lane;
  // B of a group in two parts (of a rank up to 32 one): the second is asked for while the first is multiplied, the next
  // group's first and y behind it, so that waiting for B never waits for y (loads are counted in order)
  constexpr uint32_t kParts = NR >= 4u ? 2u : 1u, kPart = 2u * NR / kParts;
  u32x4 b[kParts][kPart];
  Unaligned16 y0[kLoads], y1[kLoads];
  auto whole = [&](uint32_t g) __attribute__((always_inline)) { return (g + 1u) * 256u <= a.n; };
  auto load_b = [&](uint32_t g, uint32_t part) __attribute__((always_inline)) {
    const uint32_t s = min(g * 4u + wave, nb - 1u);
#pragma unroll
    for (uint32_t i = 0; i < kPart; ++i) b[part][i] = b_at[(uint64_t)s * (NR * 128u) + (part * kPart + i) * 64u];
  };
  auto load_y = [&](uint32_t g, Unaligned16 (&y)[kLoads]) __attribute__((always_inline)) {
    if (whole(g)) {
#pragma unroll
      for (uint32_t i = 0; i < kLoads; ++i) {
        const uint16_t* at = from[i] + g * 256u + c;
        y[i] = kOnce ? load_once(at) : *reinterpret_cast<const Unaligned16*>(at);
      }
    } else {
#pragma unroll
      for (uint32_t i = 0; i < kLoads; ++i) y[i] = part_to(from[i], g * 256u + c, a.n).w[0];
    }
  };
  const uint32_t turns = g1 - g0;
  uint32_t g = g0 + at_tile % turns;  // (tiles begin with different columns, as above)
  load_b(g, 0u);
  load_y(g, y0);
  auto group = [&](Unaligned16 (&y)[kLoads], Unaligned16 (&y_next)[kLoads]) __attribute__((always_inline)) {
    const uint32_t at_g = g;
    g = g + 1u == g1 ? g0 : g + 1u;  // (behind the last one the first again, from the cache)
    v4f acc[TT][4];
#pragma unroll
    for (uint32_t t = 0; t < TT; ++t)
#pragma unroll
      for (uint32_t j = 0; j < 4u; ++j) acc[t][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    auto multiply = [&](uint32_t part) __attribute__((always_inline)) {
#pragma unroll
      for (uint32_t p = part * (kPairs / kParts); p < (part + 1u) * (kPairs / kParts); ++p)
#pragma unroll
        for (uint32_t j = 0; j < 4u; ++j) {
          u32x4 w;
          if constexpr (NR == 1u) {
            const uint32_t k = 2u * (j & 1u);
            w = u32x4{b[0][j / 2u][k], b[0][j / 2u][k + 1u], b[0][j / 2u][k], b[0][j / 2u][k + 1u]};
          } else {
            w = b[part][(p * 4u + j) % kPart];
          }
#pragma unroll
          for (uint32_t t = 0; t < TT; ++t)
#pragma unroll
            for (uint32_t o = p; o < kOperands; o += kPairs)
              acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), u[t][o], acc[t][j], 0, 0, 0);
        }
    };
    if constexpr (kParts == 2u) {
      load_b(at_g, 1u);
      __builtin_amdgcn_sched_barrier(0);
    }
    multiply(0u);
    __builtin_amdgcn_sched_barrier(0);
    load_b(g, 0u);
    load_y(g, y_next);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (kParts == 2u) multiply(1u);
#pragma unroll
    for (uint32_t t = 0; t < TT; ++t)
#pragma unroll
      for (uint32_t j = 0; j < 4u; ++j)
        *reinterpret_cast<v4f*>(&sums[t * 16u + (lane & 15u)][wave * 64u + j * 16u + q * 4u]) = acc[t][j];
    nklds::barrier();
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
      const float* d = &sums[wave * kRows + 2u * i + half][c];
      const v4f lo = *reinterpret_cast<const v4f*>(d), hi = *reinterpret_cast<const v4f*>(d + 4);
      const float f[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
      for (uint32_t e = 0; e < 4u; ++e)
        y[i].w[e] = nk::bf16x2_hw(nk::bf16_lo(y[i].w[e]) + f[2u * e], nk::bf16_hi(y[i].w[e]) + f[2u * e + 1u]);
      if (!there[i]) continue;
      if (kOnce && whole(at_g)) store_once(to[i] + at_g * 256u + c, y[i]);
      else store8(to[i], at_g * 256u + c, a.n, y[i]);
    }
    nklds::barrier();
  };
  for (uint32_t turn = 0; turn < turns; turn += 2u) {
    group(y0, y1);
    if (turn + 1u == turns) break;
    group(y1, y0);
  }
}

// Both products of a tile of 16 tokens and 512 columns in one launch: each workgroup works the tile's u out for itself.
template <typename X, uint32_t NR>
__device__ __forceinline__ void fused(const Adapters& a) {
  constexpr uint32_t kPitch = 516u;  // spreads 16 tokens' rows over the banks
  constexpr uint32_t kPairs = NR == 1u ? 1u : NR / 2u, kOperands = NR == 1u ? 1u : NR;
  constexpr uint32_t kSums = 16u * kPitch * 4u, kParts = 8u * NR * 1024u;
  __shared__ __attribute__((aligned(16))) uint8_t memory[kSums > kParts ? kSums : kParts];
  __shared__ u32x2 s_u[2][16][4u * NR + 1u];  // [rounded, left][token][four ranks]
  auto& part = *reinterpret_cast<v4f (*)[8][NR][64]>(memory);
  auto& sums = *reinterpret_cast<float (*)[16][kPitch]>(memory);
  uint4 tile;
  const uint32_t at_tile = blockIdx.x / a.chunks, chunk = blockIdx.x - at_tile * a.chunks;
  if (!tile_of(a, at_tile, tile)) return;
  const bool none = tile.x >= a.adapters;
  if (none && a.in_place) return;
  const uint32_t lane = threadIdx.x & 63u, q = lane >> 4;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t c = chunk * 512u + lane * 8u, nb = (a.n + 63u) / 64u;
  const uint16_t* from[2];
  uint16_t* to[2];
  Unaligned16 y[2];
#pragma unroll
  for (uint32_t i = 0; i < 2u; ++i) {
    const uint32_t token = a.plan[kPlanHead + tile.y + min(wave * 2u + i, tile.z - 1u)];
    from[i] = a.y + (uint64_t)token * a.y_stride;
    to[i] = a.out + (uint64_t)token * a.out_stride;
    y[i] = part_to(from[i], c, a.n).w[0];
  }
  if (!none) {
    const u32x4* b_at = reinterpret_cast<const u32x4*>(a.b) +
                        ((uint64_t)tile.x * nb + min(chunk * 8u + wave, nb - 1u)) * (NR * 128u) + lane;
    u32x4 b[2u * NR];
#pragma unroll
    for (uint32_t i = 0; i < 2u * NR; ++i) b[i] = b_at[i * 64u];
    first_product<X, 1u, NR>(a, tile, 0u, 0u, part);
    if (threadIdx.x < NR * 64u) {
      const uint32_t r = (threadIdx.x >> 6) * 16u + (lane >> 4) * 4u;
      u32x2 hi, lo;
      split(joined(part, threadIdx.x), a.scale[tile.x], r, a.rank, hi, lo);
      s_u[0][lane & 15u][r / 4u] = hi;
      s_u[1][lane & 15u][r / 4u] = lo;
    }
    __syncthreads();
    auto four = [&](uint32_t which, uint32_t r4) __attribute__((always_inline)) { return s_u[which][lane & 15u][r4]; };
    bf16x8 u[kOperands];
    if constexpr (NR == 1u) {
      const u32x2 hi = four(0u, q), lo = four(1u, q);
      u[0] = __builtin_bit_cast(bf16x8, u32x4{hi[0], hi[1], lo[0], lo[1]});
    } else {
#pragma unroll
      for (uint32_t o = 0; o < kOperands; ++o) {
        const u32x2 first = four(o / kPairs, o % kPairs * 8u + q * 2u), second = four(o / kPairs, o % kPairs * 8u + q * 2u + 1u);
        u[o] = __builtin_bit_cast(bf16x8, u32x4{first[0], first[1], second[0], second[1]});
      }
    }
#pragma unroll
    for (uint32_t j = 0; j < 4u; ++j) {
      v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (uint32_t p = 0; p < kPairs; ++p) {
        u32x4 w;
        if constexpr (NR == 1u) {
          const uint32_t k = 2u * (j & 1u);
          w = u32x4{b[j / 2u][k], b[j / 2u][k + 1u], b[j / 2u][k], b[j / 2u][k + 1u]};
        } else {
          w = b[p * 4u + j];
        }
#pragma unroll
        for (uint32_t o = p; o < kOperands; o += kPairs)
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), u[o], acc, 0, 0, 0);
      }
      *reinterpret_cast<v4f*>(&sums[lane & 15u][wave * 64u + j * 16u + q * 4u]) = acc;  // (part has been read: the barrier above)
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 2u; ++i) {
      const float* d = &sums[wave * 2u + i][lane * 8u];
      const v4f lo = *reinterpret_cast<const v4f*>(d), hi = *reinterpret_cast<const v4f*>(d + 4);
      const float f[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
      for (uint32_t e = 0; e < 4u; ++e)
        y[i].w[e] = nk::bf16x2_hw(nk::bf16_lo(y[i].w[e]) + f[2u * e], nk::bf16_hi(y[i].w[e]) + f[2u * e + 1u]);
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < 2u; ++i)
    if (wave * 2u + i < tile.z) store8(to[i], c, a.n, y[i]);
}

}  // namespace nkada

extern "C" __global__ __launch_bounds__(1024) void netra_adapters_plan_gfx950(const int32_t* ids, uint32_t tokens,
                                                                              uint32_t adapters, uint32_t tile,
                                                                              uint32_t* plan) {
  nkada::make_plan(ids, tokens, adapters, tile, plan);
}
#define NETRA_ADAPTERS_PACK(NAME, X)                                                                            \
  extern "C" __global__ __launch_bounds__(256) void netra_adapters_pack_a_##NAME##_gfx950(                      \
      const X* a, uint4* out, uint32_t adapters, uint32_t rank, uint32_t k, uint32_t nr) {                      \
    nkada::pack_a(a, out, adapters, rank, k, nr);                                                               \
  }                                                                                                             \
  extern "C" __global__ __launch_bounds__(256) void netra_adapters_pack_b_##NAME##_gfx950(                      \
      const X* b, uint2* out, uint32_t adapters, uint32_t rank, uint32_t n, uint32_t nr) {                      \
    nkada::pack_b(b, out, adapters, rank, n, nr);                                                               \
  }
NETRA_ADAPTERS_PACK(bf16, uint16_t)
NETRA_ADAPTERS_PACK(f32, float)
// t: 16-token parts of a tile, r: 16-rank parts
#define NETRA_SHRINK(TT, NR)                                                                                    \
  extern "C" __global__ __launch_bounds__(512) void netra_adapters_shrink_bf16_t##TT##r##NR##_gfx950(           \
      nkada::Adapters a) {                                                                                      \
    nkada::shrink<uint16_t, TT, NR>(a);                                                                         \
  }                                                                                                             \
  extern "C" __global__ __launch_bounds__(512) void netra_adapters_shrink_f32_t##TT##r##NR##_gfx950(            \
      nkada::Adapters a) {                                                                                      \
    nkada::shrink<float, TT, NR>(a);                                                                            \
  }
#define NETRA_EXPAND(TT, NR)                                                                                    \
  extern "C" __global__ __launch_bounds__(256) void netra_adapters_expand_t##TT##r##NR##_gfx950(nkada::Adapters a) { \
    nkada::expand<TT, NR, false>(a);                                                                            \
  }                                                                                                             \
  extern "C" __global__ __launch_bounds__(256) void netra_adapters_expand_t##TT##r##NR##_once_gfx950(           \
      nkada::Adapters a) {                                                                                      \
    nkada::expand<TT, NR, true>(a);                                                                             \
  }
#define NETRA_FUSED(NR)                                                                                         \
  extern "C" __global__ __launch_bounds__(512) void netra_adapters_fused_bf16_r##NR##_gfx950(nkada::Adapters a) { \
    nkada::fused<uint16_t, NR>(a);                                                                              \
  }                                                                                                             \
  extern "C" __global__ __launch_bounds__(512) void netra_adapters_fused_f32_r##NR##_gfx950(nkada::Adapters a) { \
    nkada::fused<float, NR>(a);                                                                                 \
  }
NETRA_SHRINK(1, 1)
NETRA_SHRINK(1, 2)
NETRA_SHRINK(1, 4)
NETRA_SHRINK(2, 1)
NETRA_SHRINK(2, 2)
NETRA_SHRINK(2, 4)
NETRA_EXPAND(1, 1)
NETRA_EXPAND(1, 2)
NETRA_EXPAND(1, 4)
NETRA_EXPAND(1, 8)
NETRA_EXPAND(2, 1)
NETRA_EXPAND(2, 2)
NETRA_EXPAND(2, 4)
NETRA_EXPAND(2, 8)
NETRA_FUSED(1)
NETRA_FUSED(2)
NETRA_FUSED(4)
NETRA_FUSED(8)
