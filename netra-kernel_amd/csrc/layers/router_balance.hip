// Per-expert route counts and the router's balance loss with its gradient.
//
// With p_t = softmax(z_t), f_e = E counts_e / sum(counts) and V the tokens that
// count, the loss is c / |V| * sum_t s_t with s_t = sum_e f_e p_te, and its
// gradient c / |V| * p_te (f_e - s_t): both need a token's row once, so one pass
// over the logits gives them together, and neither needs the experts' mean
// probabilities. Nothing here adds floats by atomics: the loss is the sum of the
// workgroups' partial sums in workgroup order, by the last workgroup to finish.
#pragma once
#include "../kernels/moe_numerics.h"

namespace nkbal {

constexpr uint32_t kMaxExperts = 1024;

// Routes of tokens [t0, t1) per expert, and the number of those tokens, into LDS
// words hist[0 .. E) and hist[E] (cleared here). A thread takes whole tokens and
// loads sixteen of a token's ids at a time (past the slots the last one again).
// Bound by latency, loads and then LDS atomics on a few hot experts: 64 tokens of 9 ids
// 3.7 us, a 256th of 50001 tokens in each workgroup 5.5 us.
__device__ __forceinline__ void histogram(const int32_t* __restrict__ ids, uint64_t stride,
                                          const uint8_t* __restrict__ mask, uint32_t t0, uint32_t t1, uint32_t slots,
                                          uint32_t E, uint32_t* hist) {
  for (uint32_t i = threadIdx.x; i <= E; i += blockDim.x) hist[i] = 0u;
  __syncthreads();
  uint32_t mine = 0u;
  for (uint32_t t = t0 + threadIdx.x; t < t1; t += blockDim.x) {
    if (mask && !mask[t]) continue;
    ++mine;
    const int32_t* row = ids + (uint64_t)t * stride;
    for (uint32_t s = 0; s < slots; s += 16u) {
      uint32_t e[16];
#pragma unroll
      for (uint32_t j = 0; j < 16u; ++j) e[j] = (uint32_t)row[min(s + j, slots - 1u)];
#pragma unroll
      for (uint32_t j = 0; j < 16u; ++j)
        if (s + j < slots && e[j] < E) atomicAdd(&hist[e[j]], 1u);
    }
  }
  if (mine) atomicAdd(&hist[E], mine);
  __syncthreads();
}

// exp(x) for x <= 0, about 2 ulp: t = x log2 e rounded, e what the rounding and log2 e's own lost,
// 2^t by the hardware (1 ulp), times 2^e = 1 + e ln 2. Below -200 it is 0 as from where the
// hardware's result is denormal (-87.3); NaN stays NaN.
__device__ __forceinline__ float exp_nonpos(float x) {
  x = x < -200.0f ? -200.0f : x;
  const float t = x * 1.44269502162933349609375f;
  const float e = fmaf(x, 1.92596299112661746887e-8f, fmaf(x, 1.44269502162933349609375f, -t));
  const float p = __builtin_amdgcn_exp2f(t);
  return fmaf(p, e * 0.693147180559945309417f, p);
}

// Sum / maximum over 16 lanes or the wave's 64, in every one of them: DPP exchanges
// inside 16 lanes (neighbour, pair, half row, row), then across the four rows.
template <uint32_t G, bool kMax>
__device__ __forceinline__ float reduce(float v) {
  auto join = [](float a, float b) __attribute__((always_inline)) { return kMax ? fmaxf(a, b) : a + b; };
#define NETRA_DPP(CTRL) __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false))
  v = join(v, NETRA_DPP(0xB1));
  v = join(v, NETRA_DPP(0x4E));
  v = join(v, NETRA_DPP(0x141));
  v = join(v, NETRA_DPP(0x140));
#undef NETRA_DPP
  if constexpr (G == 16u) return v;
  const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = join(__uint_as_float((uint32_t)r16[0]), __uint_as_float((uint32_t)r16[1]));
  const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return join(__uint_as_float((uint32_t)r32[0]), __uint_as_float((uint32_t)r32[1]));
}
__device__ __forceinline__ uint32_t total16(uint32_t v) {
#define NETRA_DPP(CTRL) (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false)
  v += NETRA_DPP(0xB1);
  v += NETRA_DPP(0x4E);
  v += NETRA_DPP(0x141);
  v += NETRA_DPP(0x140);
#undef NETRA_DPP
  return v;
}
template <uint32_t G>
__device__ __forceinline__ uint32_t total(uint32_t v) {
  v = total16(v);
  if constexpr (G == 16u) return v;
  const auto r16 = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = (uint32_t)r16[0] + (uint32_t)r16[1];
  const auto r32 = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return (uint32_t)r32[0] + (uint32_t)r32[1];
}
template <uint32_t G>
__device__ __forceinline__ float sum(float v) {
  return reduce<G, false>(v);
}

// A token's row is held by G lanes (16: a wave takes four tokens at once; 64), NV
// values each: lane l's value j is expert 4 l + 4 G (j / 4) + j % 4.
template <uint32_t G>
__device__ __forceinline__ uint32_t expert(uint32_t lane, uint32_t j) {
  return 4u * (lane % G) + 4u * G * (j / 4u) + j % 4u;
}

// The rows of tokens t .. t + rows - 1 (rows <= 64 / G; the groups of lanes past them
// repeat the last) as they lie in memory, by loads of four values at any element
// address. Rows go through buffer descriptors that end with the last of them: no load
// is under a branch (behind one the compiler drains all loads in flight, the next
// rows' among them). Lanes past a row read the next one's values or zeros, which are not
// used. The range is checked per dword, so bf16 rows' last value has a load of its own.
template <typename X, uint32_t NV>
struct Rows {
  uint32_t w[NV * sizeof(X) / 4u];
  uint32_t last;
};
template <typename X>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* m, uint64_t stride, uint32_t t, uint32_t rows,
                                                            uint32_t E) {
  return nk::buffer_rsrc(static_cast<const X*>(m) + (uint64_t)t * stride,
                         ((rows - 1u) * (uint32_t)stride + E) * (uint32_t)sizeof(X));
}
template <typename X, uint32_t G, uint32_t NV>
__device__ __forceinline__ void load_rows(const void* m, uint64_t stride, uint32_t t, uint32_t rows, uint32_t E,
                                          Rows<X, NV>& v) {
  const uint32_t lane = threadIdx.x & 63u, row = min(lane / G, rows - 1u) * (uint32_t)stride;
  const __amdgpu_buffer_rsrc_t r = rows_rsrc<X>(m, stride, t, rows, E);
#pragma unroll
  for (uint32_t j = 0; j < NV; j += 4u) {
    const int at = (int)((row + expert<G>(lane, j)) * (uint32_t)sizeof(X));
    if constexpr (sizeof(X) == 4) {
      const nk::u32x4 u = __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0);
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) v.w[j + i] = u[i];
    } else {
      const nk::u32x2 u = __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0);
      v.w[j / 2u] = u[0];
      v.w[j / 2u + 1u] = u[1];
    }
  }
  if constexpr (sizeof(X) == 2)
    v.last = (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, (int)((row + E - 1u) * 2u), 0, 0);
}
// Value j, expert e.
template <typename X, uint32_t NV>
__device__ __forceinline__ float at(const Rows<X, NV>& v, uint32_t j, uint32_t e, uint32_t E) {
  if constexpr (sizeof(X) == 4) return __uint_as_float(v.w[j]);
  if (j & 1u) return nk::bf16_hi(v.w[j / 2u]);
  return nk::bf16_lo(e + 1u == E ? v.last : v.w[j / 2u]);  // (an odd place's dword ends with it)
}
// The rows to memory; `rows` as above, rows' ends that are not four values one by one.
template <typename X, uint32_t G, uint32_t NV>
__device__ __forceinline__ void store_rows(void* m, uint64_t stride, uint32_t t, uint32_t rows, uint32_t E,
                                           const float (&v)[NV]) {
  const uint32_t lane = threadIdx.x & 63u, row = lane / G * (uint32_t)stride;
  const __amdgpu_buffer_rsrc_t r = rows_rsrc<X>(m, stride, t, rows, E);
  const bool mine = lane / G < rows;
  constexpr int kNowhere = (int)0x80000000u;
#pragma unroll
  for (uint32_t j = 0; j < NV; j += 4u) {
    const uint32_t e = expert<G>(lane, j);
    const int at = mine && e + 4u <= E ? (int)((row + e) * (uint32_t)sizeof(X)) : kNowhere;
    if constexpr (sizeof(X) == 4) {
      const nk::u32x4 u = {__float_as_uint(v[j]), __float_as_uint(v[j + 1u]), __float_as_uint(v[j + 2u]),
                           __float_as_uint(v[j + 3u])};
      __builtin_amdgcn_raw_buffer_store_b128(u, r, at, 0, 0);
    } else {
      const nk::u32x2 u = {nk::bf16x2_hw(v[j], v[j + 1u]), nk::bf16x2_hw(v[j + 2u], v[j + 3u])};
      __builtin_amdgcn_raw_buffer_store_b64(u, r, at, 0, 0);
    }
  }
  if (E % 4u == 0u) return;
#pragma unroll
  for (uint32_t j = 0; j < NV; j += 4u) {
    const uint32_t e = expert<G>(lane, j);
    const bool tail = mine && e < E && e + 4u > E;
#pragma unroll
    for (uint32_t i = 0; i < 3u; ++i) {
      const int at = tail && e + i < E ? (int)((row + e + i) * (uint32_t)sizeof(X)) : kNowhere;
      if constexpr (sizeof(X) == 4) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v[j + i]), r, at, 0, 0);
      else __builtin_amdgcn_raw_buffer_store_b16((uint16_t)nk::bf16x2_hw(v[j + i], 0.0f), r, at, 0, 0);
    }
  }
}

// One token's softmax by G lanes: v holds z and becomes the gradient, f the experts'
// f_e and bias their biases in the same places. Returns s_t.
template <uint32_t G, uint32_t NV>
__device__ __forceinline__ float token(float (&v)[NV], const float (&f)[NV], const float (&bias)[NV], uint32_t E,
                                       float scale) {
  const uint32_t lane = threadIdx.x & 63u;
  float m = -__builtin_inff();
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) {
    v[j] = expert<G>(lane, j) < E ? v[j] + bias[j] : -__builtin_inff();
    m = fmaxf(m, v[j]);
  }
  m = reduce<G, true>(m);
  if (m == -__builtin_inff()) m = 0.0f;  // all -inf: every p is 0; a NaN stays one
  float total = 0.0f, dot = 0.0f;
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) {
    v[j] = exp_nonpos(v[j] - m);
    total += v[j];
    dot = fmaf(f[j], v[j], dot);
  }
  total = sum<G>(total);
  dot = sum<G>(dot);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const float s = dot * inv, k = inv * scale;
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) v[j] *= (f[j] - s) * k;
  return s;
}

struct Balance {
  const void* z;
  uint64_t z_stride;
  const float* bias;
  const int32_t* ids;         // slots != 0
  uint64_t ids_stride;
  uint32_t slots;
  const uint8_t* mask;
  uint32_t tokens, experts;
  float coefficient;
  int32_t* counts;            // in where slots is 0, else out
  float* loss;
  void* grad;
  uint64_t grad_stride;
  const uint32_t* parts;      // [groups][experts + 1]: partial counts and tokens (null: one workgroup counts itself)
  uint32_t groups;
  float* partial;             // one float per workgroup
  uint32_t* arrived;          // zero before the launch
};

// Counts, then the tokens' rows, 64 / G per wave. With `parts` the counting was
// shared out over the workgroups of the launch before; without, this launch is
// one workgroup. Bound by memory at the largest sizes (32768 x 500 fp32: 131 MB, 25.7 us at best,
// 28.3 in the middle). Else by the vector units and by what every workgroup does once, a chain of
// parts, barriers and the last sum: 32768 x 256 bf16, 34 MB, takes 13.9 us at best and 16.9 in the
// middle, the vector units busy 62% of it by counters (28 instructions a value, and 180 a wave
// besides); 4096 x 256 bf16 7.6 and 9.5 us on 64 CUs, whose vector units are busy 54%; 16 x 16 in
// one workgroup 3.9.
template <typename X, uint32_t G, uint32_t NV>
__device__ __forceinline__ void balance(const Balance& a) {
  __shared__ uint32_t s_count[kMaxExperts + 1u];
  __shared__ float s_wave[16];
  __shared__ uint32_t s_last;
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), waves = blockDim.x >> 6;
  const uint32_t E = a.experts;
  // the wave's first rows are on their way while the counts are made
  constexpr uint32_t kRows = 64u / G;
  const uint32_t step = gridDim.x * waves * kRows, first = (blockIdx.x * waves + wave) * kRows;
  Rows<X, NV> next;
  uint32_t live = 1u;
  // Rows t .. of this wave, and whether a lane's counts (from the last row on: the last again).
  auto load = [&](uint32_t t) __attribute__((always_inline)) {
    t = min(t, a.tokens - 1u);
    const uint32_t rows = min(kRows, a.tokens - t);
    if (a.mask) live = a.mask[t + min(lane / G, rows - 1u)];
    load_rows<X, G, NV>(a.z, a.z_stride, t, rows, E, next);
  };
  if (a.tokens) load(first);
  if (a.parts) {
    for (uint32_t e = threadIdx.x; e <= E; e += blockDim.x) s_count[e] = 0u;
    __syncthreads();
    // an expert's parts by as many threads as have 16 each, their loads in flight together
    const uint32_t threads = (a.groups + 15u) / 16u;
    for (uint32_t i = threadIdx.x; i < threads * (E + 1u); i += blockDim.x) {
      const uint32_t e = i % (E + 1u), k = i / (E + 1u) * 16u;
      uint32_t v[16], c = 0u;
#pragma unroll
      for (uint32_t j = 0; j < 16u; ++j) v[j] = a.parts[(size_t)min(k + j, a.groups - 1u) * (E + 1u) + e];
#pragma unroll
      for (uint32_t j = 0; j < 16u; ++j) c += k + j < a.groups ? v[j] : 0u;
      if (c) atomicAdd(&s_count[e], c);
    }
    __syncthreads();
  } else {
    histogram(a.ids, a.ids_stride, a.mask, 0u, a.tokens, a.slots, E, s_count);
  }
  if (a.slots == 0u) {
    for (uint32_t e = threadIdx.x; e < E; e += blockDim.x) s_count[e] = (uint32_t)a.counts[e];
    __syncthreads();
  } else if (blockIdx.x == 0u) {
    for (uint32_t e = threadIdx.x; e < E; e += blockDim.x) a.counts[e] = (int32_t)s_count[e];
  }
  float f[NV], bias[NV];
  uint32_t routes = 0u;
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) {
    const uint32_t e = expert<G>(lane, j);
    const uint32_t c = e < E ? s_count[e] : 0u;
    routes += c;
    f[j] = (float)c;
    bias[j] = a.bias && e < E ? a.bias[e] : 0.0f;
  }
  routes = total<G>(routes);
  const float per = routes ? (float)E / (float)routes : 0.0f;
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) f[j] *= per;
  const uint32_t valid = s_count[E];
  const float scale = valid ? a.coefficient / (float)valid : 0.0f;
  float mine = 0.0f;
  if (first < a.tokens) {
    for (uint32_t t = first; t < a.tokens; t += step) {
      const uint32_t now = live, rows = min(kRows, a.tokens - t);
      float v[NV];
#pragma unroll
      for (uint32_t j = 0; j < NV; ++j) v[j] = at(next, j, expert<G>(lane, j), E);
      load(t + step);  // on their way during these
      const float s = token<G, NV>(v, f, bias, E, scale);
      if (now && lane % G == 0u && lane / G < rows) mine += s;
      if (a.grad) {
        if (a.mask) {
#pragma unroll
          for (uint32_t j = 0; j < NV; ++j) v[j] = now ? v[j] : 0.0f;
        }
        store_rows<X, G, NV>(a.grad, a.grad_stride, t, rows, E, v);
      }
    }
  }
  mine = sum<64u>(mine);
  if (lane == 0u) s_wave[wave] = mine;
  __syncthreads();
  if (threadIdx.x == 0u) {
    float part = 0.0f;
    for (uint32_t w = 0; w < waves; ++w) part += s_wave[w];
    if (gridDim.x == 1u) {
      *a.loss = part * scale;
      s_last = 0u;
    } else {
      // The partial sum is stored past the caches of this XCD and is there before the
      // arrival is counted; the last to arrive reads the others' the same way. (Release
      // and acquire instead write back and drop an L2 per workgroup: 30 us at 4096 x 256.)
      __hip_atomic_store(&a.partial[blockIdx.x], part, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      s_last = __hip_atomic_fetch_add(a.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1u;
    }
  }
  __syncthreads();
  if (!s_last || wave != 0u) return;
  float all = 0.0f;  // lane l adds workgroups l, l + 64, ..: a fixed order
  for (uint32_t i = lane; i < gridDim.x; i += 64u)
    all += __hip_atomic_load(&a.partial[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  all = sum<64u>(all);
  if (lane == 0u) *a.loss = all * scale;
}

}  // namespace nkbal

// Counts of all tokens by one workgroup.
extern "C" __global__ __launch_bounds__(1024) void netra_router_counts_gfx950(const int32_t* ids, uint64_t stride,
                                                                              const uint8_t* mask, uint32_t tokens,
                                                                              uint32_t slots, uint32_t E,
                                                                              int32_t* counts, uint32_t accumulate) {
  __shared__ uint32_t hist[nkbal::kMaxExperts + 1u];
  nkbal::histogram(ids, stride, mask, 0u, tokens, slots, E, hist);
  for (uint32_t e = threadIdx.x; e < E; e += blockDim.x)
    counts[e] = (int32_t)hist[e] + (accumulate ? counts[e] : 0);
}

// Partial counts: workgroup g those of its `each` tokens, to parts[g][0 .. E]; clears *arrived.
extern "C" __global__ __launch_bounds__(1024) void netra_router_count_parts_gfx950(const int32_t* ids, uint64_t stride,
                                                                                  const uint8_t* mask, uint32_t tokens,
                                                                                  uint32_t slots, uint32_t E,
                                                                                  uint32_t each, uint32_t* parts,
                                                                                  uint32_t* arrived) {
  __shared__ uint32_t hist[nkbal::kMaxExperts + 1u];
  const uint32_t t0 = min(tokens, blockIdx.x * each);
  nkbal::histogram(ids, stride, mask, t0, min(tokens, t0 + each), slots, E, hist);
  for (uint32_t e = threadIdx.x; e <= E; e += blockDim.x) parts[(size_t)blockIdx.x * (E + 1u) + e] = hist[e];
  if (arrived && blockIdx.x == 0u && threadIdx.x == 0u) *arrived = 0u;
}

// counts = (counts +) the sum of the parts; a workgroup takes 16 experts, 16 lanes each.
extern "C" __global__ __launch_bounds__(256) void netra_router_count_sum_gfx950(const uint32_t* parts, uint32_t groups,
                                                                                uint32_t E, int32_t* counts,
                                                                                uint32_t accumulate) {
  __shared__ uint32_t s[16][17];
  const uint32_t k = threadIdx.x >> 4, i = threadIdx.x & 15u, e = blockIdx.x * 16u + i;
  uint32_t c = 0u;
  if (e < E) {
    uint32_t v[16];  // groups <= 256
#pragma unroll
    for (uint32_t j = 0; j < 16u; ++j) v[j] = parts[(size_t)min(k + 16u * j, groups - 1u) * (E + 1u) + e];
#pragma unroll
    for (uint32_t j = 0; j < 16u; ++j) c += k + 16u * j < groups ? v[j] : 0u;
  }
  s[k][i] = c;
  __syncthreads();
  if (k != 0u || e >= E) return;
  for (uint32_t g = 1; g < 16u; ++g) c += s[g][i];
  counts[e] = (int32_t)c + (accumulate ? counts[e] : 0);
}

#define NETRA_BALANCE(NAME, X, G, NV)                                                                       \
  extern "C" __global__ __launch_bounds__(1024) void netra_router_balance_##NAME##_##G##x##NV##_gfx950(     \
      nkbal::Balance a) {                                                                                   \
    nkbal::balance<X, G, NV>(a);                                                                            \
  }
#define NETRA_BALANCES(NAME, X) \
  NETRA_BALANCE(NAME, X, 16, 4) \
  NETRA_BALANCE(NAME, X, 16, 8) \
  NETRA_BALANCE(NAME, X, 16, 16) \
  NETRA_BALANCE(NAME, X, 64, 8) \
  NETRA_BALANCE(NAME, X, 64, 16)
NETRA_BALANCES(bf16, uint16_t)
NETRA_BALANCES(f32, float)
