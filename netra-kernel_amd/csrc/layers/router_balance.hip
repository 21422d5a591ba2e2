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

// exp(x) for x <= 0: n = rint(x log2 e), x - n ln 2 in two parts, 2^(r log2 e) by
// the hardware (|r log2 e| <= 1/2, about 1 ulp), scaled by 2^n. -inf gives 0.
__device__ __forceinline__ float exp_nonpos(float x) {
  const float n = rintf(fmaxf(x, -200.0f) * 1.44269502162933349609375f);
  float r = fmaf(-n, 0.693145751953125f, x);
  r = fmaf(-n, 1.428606765330187045037746429443359375e-06f, r);
  const float p = __builtin_amdgcn_exp2f(r * 1.44269502162933349609375f);
  return x < -126.0f * 0.69314718f ? 0.0f : ldexpf(p, (int)n);
}

// Sum / maximum over the wave's 64 lanes, in every lane: DPP exchanges inside 16
// lanes (neighbour, pair, half row, row), then across the four rows.
template <bool kMax>
__device__ __forceinline__ float wave_reduce(float v) {
  auto join = [](float a, float b) __attribute__((always_inline)) { return kMax ? fmaxf(a, b) : a + b; };
#define NETRA_DPP(CTRL) __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false))
  v = join(v, NETRA_DPP(0xB1));
  v = join(v, NETRA_DPP(0x4E));
  v = join(v, NETRA_DPP(0x141));
  v = join(v, NETRA_DPP(0x140));
#undef NETRA_DPP
  const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = join(__uint_as_float((uint32_t)r16[0]), __uint_as_float((uint32_t)r16[1]));
  const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return join(__uint_as_float((uint32_t)r32[0]), __uint_as_float((uint32_t)r32[1]));
}
__device__ __forceinline__ uint32_t wave_total(uint32_t v) {
#define NETRA_DPP(CTRL) (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false)
  v += NETRA_DPP(0xB1);
  v += NETRA_DPP(0x4E);
  v += NETRA_DPP(0x141);
  v += NETRA_DPP(0x140);
#undef NETRA_DPP
  const auto r16 = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = (uint32_t)r16[0] + (uint32_t)r16[1];
  const auto r32 = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return (uint32_t)r32[0] + (uint32_t)r32[1];
}
__device__ __forceinline__ float wave_sum(float v) { return wave_reduce<false>(v); }
__device__ __forceinline__ float wave_max(float v) { return wave_reduce<true>(v); }

// NV values of a row per lane, in groups of W neighbours (W = 4: 16- or 8-byte
// accesses, for rows aligned to them): lane l's value j is expert
// W l + 64 W (j / W) + j % W.
template <uint32_t W>
__device__ __forceinline__ uint32_t expert(uint32_t lane, uint32_t j) {
  return W * lane + 64u * W * (j / W) + j % W;
}
// Rows go through buffer descriptors that end with the row: no access is under a
// branch (behind one the compiler drains all loads in flight, the next row's
// among them), and lanes past the row read zeros and store nothing.
template <typename X>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(const void* m, uint64_t stride, uint32_t t, uint32_t E) {
  return nk::buffer_rsrc(static_cast<const X*>(m) + (uint64_t)t * stride, E * (uint32_t)sizeof(X));
}
template <typename X, uint32_t NV, uint32_t W>
__device__ __forceinline__ void load_row(__amdgpu_buffer_rsrc_t r, uint32_t E, float (&v)[NV]) {
  const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
  for (uint32_t j = 0; j < NV; j += W) {
    const uint32_t at = expert<W>(lane, j) * (uint32_t)sizeof(X);
    if constexpr (W == 4u && sizeof(X) == 4) {
      const nk::u32x4 u = __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, 0, 0);
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) v[j + i] = __uint_as_float(u[i]);
    } else if constexpr (W == 4u) {
      const nk::u32x2 u = __builtin_amdgcn_raw_buffer_load_b64(r, (int)at, 0, 0);
      v[j] = nk::bf16_lo(u[0]);
      v[j + 1u] = nk::bf16_hi(u[0]);
      v[j + 2u] = nk::bf16_lo(u[1]);
      v[j + 3u] = nk::bf16_hi(u[1]);
    } else if constexpr (sizeof(X) == 4) {
      v[j] = __uint_as_float((uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, (int)at, 0, 0));
    } else {
      v[j] = nk::bf16_f32((uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, (int)at, 0, 0));
    }
  }
}
template <typename X, uint32_t NV, uint32_t W>
__device__ __forceinline__ void store_row(__amdgpu_buffer_rsrc_t r, const float (&v)[NV]) {
  const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
  for (uint32_t j = 0; j < NV; j += W) {
    const uint32_t at = expert<W>(lane, j) * (uint32_t)sizeof(X);
    if constexpr (W == 4u && sizeof(X) == 4) {
      const nk::u32x4 u = {__float_as_uint(v[j]), __float_as_uint(v[j + 1u]), __float_as_uint(v[j + 2u]),
                           __float_as_uint(v[j + 3u])};
      __builtin_amdgcn_raw_buffer_store_b128(u, r, (int)at, 0, 0);
    } else if constexpr (W == 4u) {
      const nk::u32x2 u = {nk::bf16_rne(v[j]) | (uint32_t)nk::bf16_rne(v[j + 1u]) << 16,
                           nk::bf16_rne(v[j + 2u]) | (uint32_t)nk::bf16_rne(v[j + 3u]) << 16};
      __builtin_amdgcn_raw_buffer_store_b64(u, r, (int)at, 0, 0);
    } else if constexpr (sizeof(X) == 4) {
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v[j]), r, (int)at, 0, 0);
    } else {
      __builtin_amdgcn_raw_buffer_store_b16(nk::bf16_rne(v[j]), r, (int)at, 0, 0);
    }
  }
}

// One token's softmax by one wave: v holds z and becomes the gradient, f the
// experts' f_e and bias their biases in the same places. Returns s_t.
template <uint32_t NV, uint32_t W>
__device__ __forceinline__ float token(float (&v)[NV], const float (&f)[NV], const float (&bias)[NV], bool biased,
                                       uint32_t E, float scale) {
  const uint32_t lane = threadIdx.x & 63u;
  float m = -__builtin_inff();
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) {
    if (biased) v[j] += bias[j];
    if (expert<W>(lane, j) >= E) v[j] = -__builtin_inff();
    m = fmaxf(m, v[j]);
  }
  m = wave_max(m);
  if (m == -__builtin_inff()) m = 0.0f;  // all -inf: every p is 0; a NaN stays one
  float sum = 0.0f, dot = 0.0f;
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) {
    const float d = v[j] - m;
    v[j] = d != d ? d : exp_nonpos(d);
    sum += v[j];
    dot = fmaf(f[j], v[j], dot);
  }
  sum = wave_sum(sum);
  dot = wave_sum(dot);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const float s = dot * inv;
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) v[j] = v[j] * inv * (f[j] - s) * scale;
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

// Counts, then the tokens' rows, one per wave. With `parts` the counting was
// shared out over the workgroups of the launch before; without, this launch is
// one workgroup.
template <typename X, uint32_t NV, uint32_t W>
__device__ __forceinline__ void balance(const Balance& a) {
  __shared__ uint32_t s_count[kMaxExperts + 1u];
  __shared__ float s_wave[16];
  __shared__ uint32_t s_last;
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), waves = blockDim.x >> 6;
  const uint32_t E = a.experts;
  // the wave's first row is on its way while the counts are made
  const uint32_t step = gridDim.x * waves, first = blockIdx.x * waves + wave;
  float next[NV];
  uint32_t live = 1u;
  if (a.tokens) {
    const uint32_t t = min(first, a.tokens - 1u);
    if (a.mask) live = a.mask[t];
    load_row<X, NV, W>(row_rsrc<X>(a.z, a.z_stride, t, E), E, next);
  }
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
  uint32_t total = 0u;
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) {
    const uint32_t e = expert<W>(lane, j);
    const uint32_t c = e < E ? s_count[e] : 0u;
    total += c;
    f[j] = (float)c;
    bias[j] = a.bias && e < E ? a.bias[e] : 0.0f;
  }
  total = wave_total(total);
  const float per = total ? (float)E / (float)total : 0.0f;
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) f[j] *= per;
  const uint32_t valid = s_count[E];
  const float scale = valid ? a.coefficient / (float)valid : 0.0f;
  float mine = 0.0f;
  if (first < a.tokens) {
    for (uint32_t t = first; t < a.tokens; t += step) {
      const uint32_t now = live, ahead = min(t + step, a.tokens - 1u);
      float v[NV];
#pragma unroll
      for (uint32_t j = 0; j < NV; ++j) v[j] = next[j];
      // the next row is on its way during this one (behind the last, the last again)
      live = a.mask ? a.mask[ahead] : 1u;
      load_row<X, NV, W>(row_rsrc<X>(a.z, a.z_stride, ahead, E), E, next);
      const float s = token<NV, W>(v, f, bias, a.bias != nullptr, E, scale);
      if (now) mine += s;
      if (a.grad) {
#pragma unroll
        for (uint32_t j = 0; j < NV; ++j) v[j] = now ? v[j] : 0.0f;
        store_row<X, NV, W>(row_rsrc<X>(a.grad, a.grad_stride, t, E), v);
      }
    }
  }
  if (lane == 0u) s_wave[wave] = mine;
  __syncthreads();
  if (threadIdx.x == 0u) {
    float sum = 0.0f;
    for (uint32_t w = 0; w < waves; ++w) sum += s_wave[w];
    if (gridDim.x == 1u) {
      *a.loss = sum * scale;
      s_last = 0u;
    } else {
      // The partial sum is stored past the caches of this XCD and is there before the
      // arrival is counted; the last to arrive reads the others' the same way. (Release
      // and acquire instead write back and drop an L2 per workgroup: 30 us at 4096 x 256.)
      __hip_atomic_store(&a.partial[blockIdx.x], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      s_last = __hip_atomic_fetch_add(a.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1u;
    }
  }
  __syncthreads();
  if (!s_last || wave != 0u) return;
  float sum = 0.0f;  // lane l adds workgroups l, l + 64, ..: a fixed order
  for (uint32_t i = lane; i < gridDim.x; i += 64u)
    sum += __hip_atomic_load(&a.partial[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  sum = wave_sum(sum);
  if (lane == 0u) *a.loss = sum * scale;
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

#define NETRA_BALANCE(NAME, X, NV, W)                                                                            \
  extern "C" __global__ __launch_bounds__(1024) void netra_router_balance_##NAME##_v##NV##x##W##_gfx950(         \
      nkbal::Balance a) {                                                                                        \
    nkbal::balance<X, NV, W>(a);                                                                                 \
  }
#define NETRA_BALANCES(NAME, X)   \
  NETRA_BALANCE(NAME, X, 1, 1)    \
  NETRA_BALANCE(NAME, X, 2, 1)    \
  NETRA_BALANCE(NAME, X, 4, 1)    \
  NETRA_BALANCE(NAME, X, 8, 1)    \
  NETRA_BALANCE(NAME, X, 16, 1)   \
  NETRA_BALANCE(NAME, X, 4, 4)    \
  NETRA_BALANCE(NAME, X, 8, 4)    \
  NETRA_BALANCE(NAME, X, 16, 4)
NETRA_BALANCES(bf16, uint16_t)
NETRA_BALANCES(f32, float)
