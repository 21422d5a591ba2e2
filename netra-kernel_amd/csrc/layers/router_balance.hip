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
constexpr uint32_t kCountThreads = 1024;

__device__ __forceinline__ float value(const uint16_t* p) { return nk::bf16_f32(*p); }
__device__ __forceinline__ float value(const float* p) { return *p; }
__device__ __forceinline__ void put(uint16_t* p, float v) { *p = nk::bf16_rne(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }

// Routes of tokens [t0, t1) and the number of those tokens, into LDS words
// hist[0 .. E) and hist[E] (cleared here).
__device__ __forceinline__ void histogram(const int32_t* __restrict__ ids, uint64_t stride,
                                          const uint8_t* __restrict__ mask, uint32_t t0, uint32_t t1, uint32_t slots,
                                          uint32_t E, uint32_t* hist) {
  for (uint32_t i = threadIdx.x; i <= E; i += blockDim.x) hist[i] = 0u;
  __syncthreads();
  for (uint32_t t = t0 + threadIdx.x; t < t1; t += blockDim.x) {
    if (mask && !mask[t]) continue;
    atomicAdd(&hist[E], 1u);
    const int32_t* row = ids + (uint64_t)t * stride;
    for (uint32_t s = 0; s < slots; ++s) {
      const int32_t e = row[s];
      if ((uint32_t)e < E) atomicAdd(&hist[e], 1u);
    }
  }
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

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (uint32_t o = 1; o < 64u; o <<= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (uint32_t o = 1; o < 64u; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// One token's row by one wave, NV values per lane (expert lane + 64 j). f: the
// experts' f_e in the same places. Returns s_t.
template <typename X, uint32_t NV>
__device__ __forceinline__ float row(const X* __restrict__ z, const float* __restrict__ bias, X* __restrict__ g,
                                     uint32_t E, const float (&f)[NV], float scale) {
  const uint32_t lane = threadIdx.x & 63u;
  float v[NV];
  float m = -__builtin_inff();
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) {
    const uint32_t e = lane + 64u * j;
    v[j] = -__builtin_inff();
    if (e < E) v[j] = value(z + e) + (bias ? bias[e] : 0.0f);
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
  if (g) {
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) {
      const uint32_t e = lane + 64u * j;
      if (e < E) put(g + e, v[j] * inv * (f[j] - s) * scale);
    }
  }
  return s;
}

struct Balance {
  const void* z;
  uint64_t z_stride;
  const float* bias;
  const uint8_t* mask;
  uint32_t tokens, experts;
  float coefficient;
  const int32_t* counts;     // in: the experts' counts
  const uint32_t* valid;     // in: tokens that count (null: all)
  float* loss;
  void* grad;
  uint64_t grad_stride;
  float* partial;            // one float per workgroup
  uint32_t* arrived;         // zero before the launch
};

template <typename X, uint32_t NV>
__device__ __forceinline__ void balance(const Balance& a) {
  __shared__ float s_wave[16];
  __shared__ uint32_t s_last;
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), waves = blockDim.x >> 6;
  const uint32_t E = a.experts;
  float f[NV];
  uint32_t total = 0u;
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) {
    const uint32_t e = lane + 64u * j;
    const uint32_t c = e < E ? (uint32_t)a.counts[e] : 0u;
    total += c;
    f[j] = (float)c;
  }
#pragma unroll
  for (uint32_t o = 1; o < 64u; o <<= 1) total += (uint32_t)__shfl_xor((int)total, o);
  const float per = total ? (float)E / (float)total : 0.0f;
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) f[j] *= per;
  const uint32_t valid = a.valid ? *a.valid : a.tokens;
  const float scale = valid ? a.coefficient / (float)valid : 0.0f;
  float mine = 0.0f;
  for (uint32_t t = blockIdx.x * waves + wave; t < a.tokens; t += gridDim.x * waves) {
    X* g = a.grad ? reinterpret_cast<X*>(a.grad) + (uint64_t)t * a.grad_stride : nullptr;
    if (a.mask && !a.mask[t]) {
      if (g)
        for (uint32_t e = lane; e < E; e += 64u) put(g + e, 0.0f);
      continue;
    }
    mine += row<X, NV>(reinterpret_cast<const X*>(a.z) + (uint64_t)t * a.z_stride, a.bias, g, E, f, scale);
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
      __hip_atomic_store(&a.partial[blockIdx.x], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s_last = __hip_atomic_fetch_add(a.arrived, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1u;
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

// counts (and valid, if not null) of all tokens by one workgroup; clears *arrived if not null.
extern "C" __global__ __launch_bounds__(1024) void netra_router_counts_gfx950(const int32_t* ids, uint64_t stride,
                                                                   const uint8_t* mask, uint32_t tokens,
                                                                   uint32_t slots, uint32_t E, int32_t* counts,
                                                                   uint32_t accumulate, uint32_t* valid,
                                                                   uint32_t* arrived) {
  __shared__ uint32_t hist[nkbal::kMaxExperts + 1u];
  nkbal::histogram(ids, stride, mask, 0u, tokens, slots, E, hist);
  for (uint32_t e = threadIdx.x; e < E; e += blockDim.x)
    counts[e] = (int32_t)hist[e] + (accumulate ? counts[e] : 0);
  if (threadIdx.x == 0u) {
    if (valid) *valid = hist[E];
    if (arrived) *arrived = 0u;
  }
}

#define NETRA_BALANCE(NAME, X, NV)                                                                   \
  extern "C" __global__ __launch_bounds__(256) void netra_router_balance_##NAME##_v##NV##_gfx950(nkbal::Balance a) { \
    nkbal::balance<X, NV>(a);                                                                        \
  }
NETRA_BALANCE(bf16, uint16_t, 1)
NETRA_BALANCE(bf16, uint16_t, 2)
NETRA_BALANCE(bf16, uint16_t, 4)
NETRA_BALANCE(bf16, uint16_t, 8)
NETRA_BALANCE(bf16, uint16_t, 16)
NETRA_BALANCE(f32, float, 1)
NETRA_BALANCE(f32, float, 2)
NETRA_BALANCE(f32, float, 4)
NETRA_BALANCE(f32, float, 8)
NETRA_BALANCE(f32, float, 16)
