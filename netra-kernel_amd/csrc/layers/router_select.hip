// Routing to experts: scores, the choice of the k best (of the best groups), their weights, and
// the weights' gradient.
//
// A token's row is held by G lanes (16: a wave takes four tokens; 64), and lane i of each 16 holds
// the token's i-th choice, so k is at most 16.
//
// What is compared is exact: logits where their own order decides (no bias, groups by their best
// expert), else scores in 64 bits. All of it in 64 bits took 229 us for 32768 tokens of 256 experts.
// So an expert is first a 32-bit key, its score in 22 bits and its index behind it (the
// order of equal ones), which is sorted with one minimum and one maximum an exchange. Only where two neighbours in that
// order that the choice hangs on are nearer than the key's error, and not the same score by the same
// operands, the few experts (or groups) drawn are put in order by their scores in 64 bits; and only where that does not
// settle it, or the scores are a softmax's, the token is done again in 64 bits, by the whole wave: 6 us of one wave's
// time, however few the tokens. Keys of bf16 logits hold all of them and are never done again.
//
// A key's units span the finite biases, so one finite bias far from the others (-1e9 to take an expert out, where -inf has a
// unit of its own) leaves the scores few units or one, and most tokens go to 64 bits: T 32768, 256 experts by sigmoid
// with six such biases 57 us at -1e4 and 63 at -1e9, with groups 96, where -inf takes 13 and 16. So do fp32 logits whose k-th is 32
// and more below the largest: 60 us where near ones take 12.
//
// T 32768, 256 experts by sigmoid, bias and groups: 17 us, bound by its instructions (the vector units are
// busy 91% of the time; the 19 MB alone would take 4). T 64: 3.3 us, a launch.
#pragma once
#include <type_traits>

#include "router_balance.hip"

namespace nksel {

constexpr uint32_t kMost = 16;  // choices of a token, and groups of experts

enum Scoring { kSoftmax, kSigmoid };

// exp(-|z|); NaN stays NaN.
__device__ __forceinline__ float exp_minus(float z) { return nkbal::exp_nonpos(-fabsf(z)); }
// sigmoid(z), to a few ulp at both ends.
__device__ __forceinline__ float sigmoid(float z) {
  const float e = exp_minus(z);
  return (z < 0.0f ? e : 1.0f) / (1.0f + e);
}
// Its derivative; from e, as 1 - sigmoid has few bits left where the sigmoid is near one.
__device__ __forceinline__ float slope(float z) {
  const float e = exp_minus(z), d = 1.0f + e;
  return e / (d * d);
}

struct Select {
  const void* z;
  uint64_t z_stride;
  const float* bias;          // null: none
  const uint8_t* mask;        // null: all tokens
  uint32_t tokens, experts, k, shared;
  uint32_t scoring, groups, each, top_groups, top2, renormalise;
  uint32_t by_logits;         // the choice goes by the logits' order
  float scale;
  int32_t* ids;
  uint64_t ids_stride;
  float* weights;
  uint64_t weights_stride;
};

// Order of logits: the bits of -0 as of 0, of a NaN as of -inf, negative numbers' turned round.
__device__ __forceinline__ uint32_t order(float z) {
  const uint32_t u = __float_as_uint(fmaxf(z + 0.0f, -__builtin_inff()));
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}

template <uint32_t G, bool kMax>
__device__ __forceinline__ uint32_t across(uint32_t v) {
  auto join = [](uint32_t a, uint32_t b) __attribute__((always_inline)) { return kMax ? max(a, b) : min(a, b); };
#define NETRA_DPP(CTRL) (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false)
  v = join(v, NETRA_DPP(0xB1));
  v = join(v, NETRA_DPP(0x4E));
  v = join(v, NETRA_DPP(0x141));
  v = join(v, NETRA_DPP(0x140));
#undef NETRA_DPP
  if constexpr (G == 16u) return v;
  const auto r16 = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = join((uint32_t)r16[0], (uint32_t)r16[1]);
  const auto r32 = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return join((uint32_t)r32[0], (uint32_t)r32[1]);
}

// v of the lane n further on (mod 16) in the row of 16. (Every lane has to be active: never under a
// condition that differs between lanes.)
template <uint32_t N>
__device__ __forceinline__ uint32_t turned(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + (int)(16u - N), 0xF, 0xF, false);
}
template <uint32_t N>
__device__ __forceinline__ float turned(float v) {
  return __uint_as_float(turned<N>(__float_as_uint(v)));
}
template <uint32_t N = 1, typename F>
__device__ __forceinline__ void each_turn(F&& f) {
  if constexpr (N < 16u) {
    f(std::integral_constant<uint32_t, N>{});
    each_turn<N + 1u>(f);
  }
}

// Whether a group (its score is lane g * each_lane's of a row of 16) is among the `top` best by `score`, in an order
// of T; ties to the lower. False in other lanes.
template <typename T, typename Turn>
__device__ __forceinline__ bool kept(T score, uint32_t groups, uint32_t top, uint32_t each_lane, Turn&& turn) {
  const uint32_t g = threadIdx.x & 15u;
  auto leads = [&](uint32_t lane) __attribute__((always_inline)) { return (lane & (each_lane - 1u)) == 0u && lane < groups * each_lane; };
  uint32_t before = 0u;
  each_turn([&](auto n) __attribute__((always_inline)) {
    const uint32_t other = (g + n) & 15u;
    const T s = turn(score, n);
    before += leads(other) && (s > score || (s == score && other < g)) ? 1u : 0u;
  });
  return leads(g) && before < top;
}

// Weights of the choices, lane i of a row of 16 its token's i-th, from its logit z (the row's
// largest logit and the sum of its exponentials where the softmax is over the whole row), and the
// stores.
template <typename X>
__device__ __forceinline__ void finish(const Select& a, uint32_t t, uint32_t id, float top, float total, bool live, bool writes) {
  const uint32_t i = threadIdx.x & 15u;
  const X* row = static_cast<const X*>(a.z) + (uint64_t)t * a.z_stride;
  const bool mine = i < a.k;
  auto value = [&](uint32_t e) __attribute__((always_inline)) {
    if constexpr (sizeof(X) == 4) return row[e];
    else return nk::bf16_f32(row[e]);
  };
  const float z = value(mine ? id : 0u);
  float s;
  if (a.scoring == kSigmoid) {
    s = sigmoid(z);
  } else {
    if (a.renormalise) {
      top = nkbal::reduce<16, true>(mine ? z : -__builtin_inff());
      if (top == -__builtin_inff()) top = 0.0f;
    }
    s = nkbal::exp_nonpos(z - top);
  }
  if (a.renormalise) total = nkbal::sum<16>(mine ? s : 0.0f);
  float w = s;
  if (a.renormalise || a.scoring == kSoftmax) w = total == 0.0f ? 0.0f : s / total;
  w *= a.scale;
  if (!writes || i >= a.k + a.shared) return;
  if (!mine) {
    id = a.experts;
    w = sigmoid(value(a.experts));
  }
  a.ids[(uint64_t)t * a.ids_stride + i] = live ? (int32_t)id : -1;
  a.weights[(uint64_t)t * a.weights_stride + i] = live ? w : 0.0f;
}

__device__ __forceinline__ double sum64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  return v;
}
__device__ __forceinline__ float max64(float v) { return nkbal::reduce<64, true>(v); }

// A 64-bit score's place in the order of scores; a NaN ranks as -inf.
__device__ __forceinline__ uint64_t order(double c) {
  const uint64_t u = (uint64_t)__double_as_longlong((c == c ? c : -__builtin_inf()) + 0.0);
  return u ^ ((uint64_t)((int64_t)u >> 63) | 1ull << 63);
}
template <uint32_t N>
__device__ __forceinline__ uint64_t turned(uint64_t v) {
  return (uint64_t)turned<N>((uint32_t)(v >> 32)) << 32 | turned<N>((uint32_t)v);
}
// An expert's score in 64 bits (of a softmax by its logits).
template <typename X>
__device__ __forceinline__ uint64_t exact_score(const Select& a, const X* row, uint32_t e) {
  float z;
  if constexpr (sizeof(X) == 4) z = row[e];
  else z = nk::bf16_f32(row[e]);
  double c = (double)z;
  if (!a.by_logits) {
    c = 1.0 / (1.0 + exp(-c));
    if (a.bias) c += (double)a.bias[e];
  }
  return order(c);
}
// The score that has this place in the order.
__device__ __forceinline__ double score_of(uint64_t key) {
  const uint64_t u = key >> 63 ? key & ~(1ull << 63) : ~key;
  return __longlong_as_double((long long)u);
}

// One token by a wave, its scores in 64 bits. s: 64 NV values.
template <typename X, uint32_t NV>
__device__ __forceinline__ void select_exact(const Select& a, uint32_t t, double* s) {
  const uint32_t lane = threadIdx.x & 63u, i = lane & 15u, E = a.experts, each = a.each;
  const X* row = static_cast<const X*>(a.z) + (uint64_t)t * a.z_stride;
  float z[NV], top = -__builtin_inff(), total = 0.0f;
  double c[NV];
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) {
    const uint32_t e = lane + 64u * j;
    z[j] = -__builtin_inff();
    if (e < E) {
      if constexpr (sizeof(X) == 4) z[j] = row[e];
      else z[j] = nk::bf16_f32(row[e]);
    }
    top = fmaxf(top, z[j]);
  }
  if (a.scoring == kSoftmax) {
    top = max64(top);
    if (top == -__builtin_inff()) top = 0.0f;
    double all = 0.0;
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) {
      c[j] = exp((double)z[j] - (double)top);
      all += c[j];
    }
    all = sum64(all);
    total = (float)all;
    const double inv = all == 0.0 ? 0.0 : 1.0 / all;
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) c[j] *= inv;
  } else if (!a.by_logits) {
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) c[j] = 1.0 / (1.0 + exp(-(double)z[j]));
  }
  if (a.by_logits) {
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) c[j] = (double)z[j];
  }
  uint32_t taken = 0u;  // of the lane's values: what cannot be chosen
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) {
    const uint32_t e = lane + 64u * j;
    if (e >= E) taken |= 1u << j;
    else if (a.bias) c[j] += (double)a.bias[e];
    if (!(c[j] == c[j])) c[j] = -__builtin_inf();
  }
  if (a.groups > 1u) {
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j)
      if (lane + 64u * j < E) s[lane + 64u * j] = c[j];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    double best = -__builtin_inf(), second = -__builtin_inf();
    if (i < a.groups)
      for (uint32_t m = 0; m < each; m += 8u) {
        double v[8];
#pragma unroll
        for (uint32_t j = 0; j < 8u; ++j) v[j] = s[i * each + min(m + j, each - 1u)];
#pragma unroll
        for (uint32_t j = 0; j < 8u; ++j) {
          if (m + j >= each) v[j] = -__builtin_inf();
          second = fmax(second, fmin(best, v[j]));
          best = fmax(best, v[j]);
        }
      }
    if (a.top2) best += second;
    // (by their places in the order: +inf and -inf together are a NaN, which ranks as -inf and not before all)
    const bool keep = kept(order(best), a.groups, a.top_groups, 1u, [](uint64_t u, auto n) __attribute__((always_inline)) { return turned<decltype(n)::value>(u); });
    const uint32_t bits = (uint32_t)__ballot(keep) & 0xffffu;
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j)
      if (!(bits >> min((lane + 64u * j) / each, 31u) & 1u)) taken |= 1u << j;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  // the bits in the numbers' order; 0 for what cannot be chosen
  uint64_t key[NV];
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) {
    key[j] = taken >> j & 1u ? 0u : order(c[j]);
  }
  uint32_t id = 0u;
  for (uint32_t n = 0; n < a.k; ++n) {
    uint64_t m = key[0];
    uint32_t at = lane;
#pragma unroll
    for (uint32_t j = 1; j < NV; ++j)
      if (key[j] > m) {
        m = key[j];
        at = lane + 64u * j;
      }
    const uint32_t hi = across<64, true>((uint32_t)(m >> 32));
    const bool top_hi = (uint32_t)(m >> 32) == hi;
    const uint32_t lo = across<64, true>(top_hi ? (uint32_t)m : 0u);
    at = across<64, false>(top_hi && (uint32_t)m == lo ? at : ~0u);
    if (i == n) id = at;
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j)
      if (at == lane + 64u * j) key[j] = 0u;
  }
  finish<X>(a, t, id, top, total, true, lane < 16u);
}

// What a key is made of: the whole logit (bf16), the distance to the row's largest logit (fp32), or
// the score and the bias.
enum Kind { kWhole, kDistance, kScore };

// a >= b after.
__device__ __forceinline__ void exchange(uint32_t& a, uint32_t& b) {
  const uint32_t m = min(a, b);
  a = max(a, b);
  b = m;
}
// Falling order, by merging odd and even places of sorted halves (Batcher's network).
template <uint32_t LO, uint32_t N, uint32_t R, uint32_t NV>
__device__ __forceinline__ void merge(uint32_t (&v)[NV]) {
  constexpr uint32_t S = R * 2u;
  if constexpr (S < N) {
    merge<LO, N, S>(v);
    merge<LO + R, N, S>(v);
#pragma unroll
    for (uint32_t i = LO + R; i + R < LO + N; i += S) exchange(v[i], v[i + R]);
  } else {
    exchange(v[LO], v[LO + R]);
  }
}
template <uint32_t LO, uint32_t N, uint32_t NV>
__device__ __forceinline__ void sort(uint32_t (&v)[NV]) {
  if constexpr (N > 1u) {
    sort<LO, N / 2u>(v);
    sort<LO + N / 2u, N / 2u>(v);
    merge<LO, N, 1u>(v);
  }
}

// The n largest of the keys that a token's G lanes have in falling order; lane i gets the i-th. Of a lane's own
// only the first M (n at most) can be among them; with M above 16 all lanes get the next one too (rest; 0: none).
template <uint32_t G, uint32_t M, uint32_t NV>
__device__ __forceinline__ uint32_t draw(const uint32_t (&v)[NV], uint32_t n, uint32_t& rest) {
  constexpr uint32_t L = M < NV ? M : NV;
  const uint32_t i = threadIdx.x & 15u;
  uint32_t key[L], mine = 0u;
#pragma unroll
  for (uint32_t j = 0; j < L; ++j) key[j] = v[j];
  for (uint32_t at = 0; at < n; ++at) {
    const uint32_t m = across<G, true>(key[0]);
    if (i == at) mine = m;
    // by bits: of a choice between two places the compiler makes a place chosen at run time
    const uint32_t gone = key[0] == m ? ~0u : 0u;
#pragma unroll
    for (uint32_t j = 0; j + 1u < L; ++j) key[j] = (key[j] & ~gone) | (key[j + 1u] & gone);
    key[L - 1u] &= ~gone;
  }
  if constexpr (M > kMost) rest = across<G, true>(key[0]);
  return mine;
}

// Each wave takes 64 / G tokens, and no more than those: in a loop over more the compiler works out beforehand
// all that the seldom 64-bit part can use, half as many instructions again.
template <typename X, uint32_t G, uint32_t NV, Kind K>
__device__ __forceinline__ void select(const Select& a) {
  constexpr uint32_t kTokens = 64u / G, kWaves = 4u, kMax = G * NV;
  __shared__ double s_memory[kWaves][kMax > kTokens * kMax / 2u ? kMax : kTokens * kMax / 2u];
  const uint32_t lane = threadIdx.x & 63u, i = lane & 15u;
  const uint32_t E = a.experts;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t b = blockIdx.x * kWaves + wave;
  if (b > (a.tokens - 1u) / kTokens) return;
  // Of a key's upper 22 bits, from 1 on: the units of finite values; of scores 1 is -inf's (and a NaN's), kInf is +inf's, and
  // what finite scores are off by, 3e-6 of the range, does not reach it.
  constexpr float kUnits = 4194237.0f;
  constexpr uint32_t kInf = 4194303u;
  // Scores: lo .. hi over 0 and the finite biases, and a score's 0 .. 1, are the units' range. A sigmoid is
  // off by 5e-7 by the hardware's exponential and reciprocal, a softmax by its sum too, of the largest (mostly far below
  // one: T 32768, 256 experts with a bias 20 us, held against one 26); then the sum with the bias.
  float bias[NV], lo = 0.0f, units = 0.0f;
  float widest = 0.0f;                    // of the biases
  uint32_t near = K == kWhole ? 0u : 4u;  // keys that are apart by no more are not told apart
  // (by scores that are off by `off` of the largest, and their sum with the bias)
  auto apart = [&](float off, float largest) __attribute__((always_inline)) {
    return 3u + (uint32_t)fminf(2.0f * (off * largest + 2.4e-7f * (largest + widest)) * units, 8e6f);
  };
  if constexpr (K == kScore) {
    const __amdgpu_buffer_rsrc_t r = nk::buffer_rsrc(a.bias, a.bias ? E * 4u : 0u);  // (no bias: zeros)
    float hi = 0.0f;
#pragma unroll
    for (uint32_t j = 0; j < NV; j += 4u) {
      const nk::u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, (int)(nkbal::expert<G>(lane, j) * 4u), 0, 0);
#pragma unroll
      for (uint32_t n = 0; n < 4u; ++n) bias[j + n] = __uint_as_float(v[n]);
    }
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) {
      const float f = fabsf(bias[j]) < __builtin_inff() ? bias[j] : 0.0f;
      lo = fminf(lo, f);
      hi = fmaxf(hi, f);
    }
    lo = -nkbal::reduce<G, true>(-lo);
    hi = nkbal::reduce<G, true>(hi);
    units = kUnits / (hi - lo + 1.0f);
    widest = fmaxf(-lo, hi);
    if (a.scoring == kSigmoid) near = apart(6e-7f, 1.0f);
    // lanes' places past the last expert: the least key, behind every expert's that has it too
    if (E < kMax) {
#pragma unroll
      for (uint32_t j = 0; j < NV; ++j) bias[j] = nkbal::expert<G>(lane, j) < E ? bias[j] : -__builtin_inff();
    }
  }
  const uint32_t t0 = b * kTokens, rows = min(kTokens, a.tokens - t0), t = t0 + min(lane / G, rows - 1u);
  nkbal::Rows<X, NV> raw;
  nkbal::load_rows<X, G, NV>(a.z, a.z_stride, t0, rows, E, raw);
  const bool live = !a.mask || a.mask[t];
  const X* row = static_cast<const X*>(a.z) + (uint64_t)t * a.z_stride;
  const bool exact_near = K == kDistance || a.scoring == kSigmoid;  // (a softmax's sum in 64 bits takes the whole row)
  uint32_t key[NV];
  float top = 0.0f, total = 0.0f;
  {
    float z[NV];
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) z[j] = nkbal::at(raw, j, 0u, 0u);
    if (E < kMax || (E & 1u)) {
#pragma unroll
      for (uint32_t j = 0; j < NV; ++j) {
        const uint32_t e = nkbal::expert<G>(lane, j);
        z[j] = e < E ? nkbal::at(raw, j, e, E) : -__builtin_inff();
      }
    }
    if (K == kDistance || a.scoring == kSoftmax) {
      top = z[0];
#pragma unroll
      for (uint32_t j = 1; j < NV; ++j) top = fmaxf(top, z[j]);
      top = nkbal::reduce<G, true>(top);
    }
    if constexpr (K != kScore) {
#pragma unroll
      for (uint32_t j = 0; j < NV; ++j) {
        const uint32_t e = nkbal::expert<G>(lane, j);
        if constexpr (K == kWhole) {
          key[j] = (order(z[j]) & 0xffff0000u) | (0xffffu - e);
        } else {
          // 32 and more below the largest: the least key
          const float x = fmaxf(z[j], -__builtin_inff());
          const float d = x == top ? 0.0f : fminf((top - x) * 0.03125f, 1.0f);
          key[j] = (1u + (uint32_t)(kUnits * (1.0f - d))) << 10 | (1023u - e);
        }
      }
    }
    if (a.scoring == kSoftmax) {
      if (top == -__builtin_inff()) top = 0.0f;
      if (K == kScore || !a.renormalise) {
#pragma unroll
        for (uint32_t j = 0; j < NV; ++j) {
          z[j] = nkbal::exp_nonpos(z[j] - top);
          total += z[j];
        }
        total = nkbal::sum<G>(total);
      }
    }
    if constexpr (K == kScore) {
      if (a.scoring == kSigmoid) {
#pragma unroll
        for (uint32_t j = 0; j < NV; ++j)
          z[j] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z[j] * -1.44269504088896341f));
      } else {
        const float inv = total == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(total);
        near = apart(2.5e-6f, inv);  // the largest is exp(0) / total (a NaN: all are near)
#pragma unroll
        for (uint32_t j = 0; j < NV; ++j) z[j] *= inv;
      }
#pragma unroll
      for (uint32_t j = 0; j < NV; ++j) {
        const uint32_t e = nkbal::expert<G>(lane, j);
        const float c = (z[j] + bias[j] - lo) * units;
        key[j] = (2u + (uint32_t)(int32_t)fminf(fmaxf(c, -1.0f), (float)(kInf - 2u))) << 10 | (1023u - e);
      }
    }
  }
  bool again = false;
  if (a.groups > 1u) {
    uint32_t* s = reinterpret_cast<uint32_t*>(s_memory[wave]) + lane / G * kMax;
#pragma unroll
    for (uint32_t j = 0; j < NV; j += 4u)
      *reinterpret_cast<uint4*>(s + nkbal::expert<G>(lane, j)) = make_uint4(key[j], key[j + 1u], key[j + 2u], key[j + 3u]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    // A group's experts go to as many neighbouring lanes (a power of two) as the groups leave; they join theirs after.
    const uint32_t each_lane = a.groups <= 2u ? 8u : a.groups <= 4u ? 4u : a.groups <= 8u ? 2u : 1u;
    const uint32_t group = i / each_lane, in = i & (each_lane - 1u);
    const uint32_t share = ((a.each + 3u) / 4u + each_lane - 1u) / each_lane * 4u;
    const uint32_t m0 = group < a.groups ? min(in * share, a.each) : 0u, m1 = group < a.groups ? min(m0 + share, a.each) : 0u;
    const uint32_t* from = s + group * a.each;
    auto joined = [&](auto&& take_other) __attribute__((always_inline)) {
      if (each_lane >= 2u) take_other(std::integral_constant<int, 0xB1>{});
      if (each_lane >= 4u) take_other(std::integral_constant<int, 0x4E>{});
      if (each_lane >= 8u) take_other(std::integral_constant<int, 0x141>{});
    };
    uint32_t best = 0u, second = 0u;
    auto take = [&](uint32_t v) __attribute__((always_inline)) {
      second = max(second, min(best, v));
      best = max(best, v);
    };
    if (a.each % 4u == 0u) {
      for (uint32_t m = m0; m < m1; m += 4u) {
        const uint4 v = *reinterpret_cast<const uint4*>(from + m);
        take(v.x);
        take(v.y);
        take(v.z);
        take(v.w);
      }
    } else {
      for (uint32_t m = m0; m < m1; m += 8u) {
        uint32_t v[8];
#pragma unroll
        for (uint32_t n = 0; n < 8u; ++n) v[n] = from[min(m + n, m1 - 1u)];
#pragma unroll
        for (uint32_t n = 0; n < 8u; ++n) take(m + n < m1 ? v[n] : 0u);
      }
    }
    joined([&](auto ctrl) __attribute__((always_inline)) {
      const uint32_t b0 = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)best, decltype(ctrl)::value, 0xF, 0xF, false);
      const uint32_t b1 = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)second, decltype(ctrl)::value, 0xF, 0xF, false);
      take(b0);
      take(b1);
    });
    const bool leads = in == 0u && group < a.groups;  // its score stands for the group
    // (the best expert's key orders the groups itself, as lower groups have lower experts)
    const uint32_t shift = a.top2 ? 4u : 10u;
    // Sums of two: with -inf (as of a NaN, or of both infinities) behind all others, with +inf before all.
    const uint32_t b0 = best >> 10, b1 = second >> 10, sum = b1 == 1u ? 0u : b0 == kInf ? 2u * kInf : b0 + b1;
    const uint32_t score = !leads ? 0u : a.top2 ? sum << 4 | (15u - i) : best;
    uint32_t before = 0u;
    each_turn([&](auto n) __attribute__((always_inline)) {
      before += turned<decltype(n)::value>(score) > score ? 1u : 0u;
    });
    bool keep = before < a.top_groups;
    if constexpr (K != kWhole) {
      const uint32_t least = across<16, false>(keep ? score : ~0u) >> shift;
      const uint32_t most = across<16, true>(keep ? 0u : score) >> shift;
      again = least - most <= (a.top2 ? 2u * near : near);
      // Groups too near: their best experts' scores in 64 bits, if it is certain which experts those are.
      if (exact_near && __ballot(again && live)) {
        uint32_t v[3] = {0u, 0u, 0u};
        auto take3 = [&](uint32_t x) __attribute__((always_inline)) {
          v[2] = max(v[2], min(v[1], x));
          v[1] = max(v[1], min(v[0], x));
          v[0] = max(v[0], x);
        };
        for (uint32_t m = m0; m < m1; ++m) take3(from[m]);
        joined([&](auto ctrl) __attribute__((always_inline)) {
          uint32_t x[3];
#pragma unroll
          for (uint32_t n = 0; n < 3u; ++n) x[n] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v[n], decltype(ctrl)::value, 0xF, 0xF, false);
#pragma unroll
          for (uint32_t n = 0; n < 3u; ++n) take3(x[n]);
        });
        const uint32_t of = a.top2 ? 1u : 0u;
        const bool certain = !leads || v[of + 1u] == 0u || (v[of] >> 10) - (v[of + 1u] >> 10) > near;
        uint64_t exact = 0u;
        if (leads) {
          exact = exact_score(a, row, 1023u - (v[0] & 1023u));
          if (a.top2) exact = order(score_of(exact) + score_of(exact_score(a, row, 1023u - (v[1] & 1023u))));
        }
        keep = kept(exact, a.groups, a.top_groups, each_lane, [](uint64_t u, auto n) __attribute__((always_inline)) { return turned<decltype(n)::value>(u); });
        again = across<16, false>(certain ? 1u : 0u) == 0u;
      }
    }
    // what is not kept leaves by zeros in LDS
    const uint32_t of_row = (uint32_t)(__ballot(keep) >> (lane & 48u)) & 0xffffu;
    if (!(of_row >> (group * each_lane) & 1u)) {
      uint32_t* to = s + group * a.each;
      if (a.each % 4u == 0u) {
        for (uint32_t m = m0; m < m1; m += 4u) *reinterpret_cast<uint4*>(to + m) = make_uint4(0u, 0u, 0u, 0u);
      } else {
        for (uint32_t m = m0; m < m1; ++m) to[m] = 0u;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (uint32_t j = 0; j < NV; j += 4u) {
      const uint4 v = *reinterpret_cast<const uint4*>(s + nkbal::expert<G>(lane, j));
      key[j] = v.x;
      key[j + 1u] = v.y;
      key[j + 2u] = v.z;
      key[j + 3u] = v.w;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  sort<0u, NV>(key);
  // two more than k, to see whether the k-th and the next one are apart
  const uint32_t draws = K == kWhole ? a.k : min(a.k + 2u, kMost);
  uint32_t rest = 0u;
  uint32_t mine = draws <= 10u ? draw<G, 10u>(key, draws, rest) : draw<G, K == kWhole ? 16u : 17u>(key, draws, rest);
  if constexpr (K != kWhole) {
    // Places past the last expert are no choice: where the kept groups have fewer experts than are drawn, such places, whose
    // keys are behind all of theirs, are drawn after them. (Of bf16 logits k are drawn and no more, which the groups have.)
    auto expert_or_none = [&](uint32_t v) __attribute__((always_inline)) { return 1023u - (v & 1023u) < E ? v : 0u; };
    mine = expert_or_none(mine);
    rest = expert_or_none(rest);
  }
  uint32_t id = min(K == kWhole ? 0xffffu - (mine & 0xffffu) : 1023u - (mine & 1023u), E - 1u);
  if constexpr (K != kWhole) {
    // lane i: its choice and the next one. Equal logits and biases are told apart by the index.
    uint32_t zb, bb = 0u;
    if constexpr (sizeof(X) == 4) zb = __float_as_uint(row[id]);
    else zb = row[id];
    if (K == kScore && a.bias) bb = __float_as_uint(a.bias[id]);
    const uint32_t next = turned<1>(mine), nz = turned<1>(zb), nb = turned<1>(bb);
    const bool close = next != 0u && (mine >> 10) - (next >> 10) <= near;
    const bool same = zb == nz && bb == nb;
    const bool next_close = turned<1>(close ? 1u : 0u) != 0u;
    bool bad = i < a.k && close && !same;
    if (i + 1u == a.k) bad = close && (!same || a.k + 2u > kMost || next_close);
    if (a.k == kMost && i + 1u == a.k) bad = rest != 0u && (mine >> 10) - (rest >> 10) <= near;  // no lane holds the next one
    // Choices too near: the order of those drawn by their scores in 64 bits, if what was not drawn is certainly behind
    // the k-th then.
    if (exact_near && __ballot(bad && live)) {
      const bool drawn = i < draws && mine != 0u;
      const uint64_t exact = drawn ? exact_score(a, row, id) : 0u;
      uint32_t before = 0u;
      each_turn([&](auto n) __attribute__((always_inline)) {
        const uint64_t other = turned<decltype(n)::value>(exact);
        const uint32_t other_id = turned<decltype(n)::value>(id);
        before += other > exact || (other == exact && other_id < id) ? 1u : 0u;
      });
      const bool chosen = drawn && before < a.k;
      const uint32_t least = across<16, false>(chosen ? mine >> 10 : ~0u);
      // (up to ten draws have no next one, which would cost every wave 3%; the last one drawn is no less)
      if (draws <= 10u) rest = across<16, false>(i < draws ? mine : ~0u);
      bad = rest != 0u && least - (rest >> 10) <= near;
      const uint32_t place = drawn ? before : ~0u, old = id;
      id = place == i ? old : 0u;
      each_turn([&](auto n) __attribute__((always_inline)) {
        const uint32_t other_place = turned<decltype(n)::value>(place), other_id = turned<decltype(n)::value>(old);
        id = other_place == i ? other_id : id;
      });
    }
    again |= bad;
    uint64_t todo = __ballot(again && live && lane / G < rows);
    const bool done = G == 64u ? todo == 0u : (todo >> (lane & 48u) & 0xffffu) == 0u;
    finish<X>(a, t, id, top, total, live, done && lane / G < rows && (G == 16u || lane < 16u));
    while (todo) {
      const uint32_t at = ((uint32_t)__ffsll((unsigned long long)todo) - 1u) / G;
      select_exact<X, kMax / 64u>(a, t0 + at, s_memory[wave]);
      todo &= G == 64u ? 0ull : ~(0xffffull << (at * 16u));
    }
  } else {
    finish<X>(a, t, id, top, total, live, lane / G < rows && (G == 16u || lane < 16u));
  }
}

struct SelectGradient {
  const float* dw;
  uint64_t dw_stride;
  const void* z;
  uint64_t z_stride;
  const int32_t* ids;
  uint64_t ids_stride;
  const uint8_t* mask;
  uint32_t tokens, experts, k, shared, scoring, renormalise;
  float scale;
  void* grad;                 // of z's type
  uint64_t grad_stride;
  uint32_t accumulate;
};

// The gradient of the logits. Lane i of a row of 16 has the token's i-th choice. Differences of the
// weights' gradients are taken before they are weighted (sum_j s_j (v_i - v_j), not v_i S - sum_j s_j v_j):
// nothing cancels where one expert has almost all. The row goes through LDS. T 32768, 500 experts in fp32,
// every logit with a gradient: 30 us (133 MB, 4.4 TB/s; the vector units are busy 75% of the time); T 4096, 256 experts by
// sigmoid 4.8.
template <typename X, uint32_t G, uint32_t NV>
__device__ __forceinline__ void gradient(const SelectGradient& a) {
  constexpr uint32_t kTokens = 64u / G, kWaves = 4u;
  __shared__ float s_row[kWaves][kTokens][G * NV];
  const uint32_t lane = threadIdx.x & 63u, i = lane & 15u, E = a.experts;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t batches = (a.tokens - 1u) / kTokens + 1u;
  const bool whole = a.scoring == kSoftmax && !a.renormalise;
  float* s = s_row[wave][lane / G];
  // bits of an expert that was not chosen: a NaN that no arithmetic gives
  const float none = __uint_as_float(0xffc0ffeeu);
  auto hit = [&](float v) __attribute__((always_inline)) { return __float_as_uint(v) != 0xffc0ffeeu; };
#pragma unroll
  for (uint32_t j = 0; j < NV; ++j) s[nkbal::expert<G>(lane, j)] = none;
  for (uint32_t b = blockIdx.x * kWaves + wave; b < batches; b += gridDim.x * kWaves) {
    const uint32_t t0 = b * kTokens, rows = min(kTokens, a.tokens - t0), t = t0 + min(lane / G, rows - 1u);
    const bool live = !a.mask || a.mask[t];
    const X* row = static_cast<const X*>(a.z) + (uint64_t)t * a.z_stride;
    auto value = [&](uint32_t e) __attribute__((always_inline)) {
      if constexpr (sizeof(X) == 4) return row[e];
      else return nk::bf16_f32(row[e]);
    };
    nkbal::Rows<X, NV> raw;
    if (whole) nkbal::load_rows<X, G, NV>(a.z, a.z_stride, t0, rows, E, raw);
    const bool slot = i < a.k;
    const uint32_t id = slot ? (uint32_t)a.ids[(uint64_t)t * a.ids_stride + i] : ~0u;
    const bool chosen = id < E && live;
    const float d = i < a.k + a.shared ? a.dw[(uint64_t)t * a.dw_stride + i] : 0.0f;
    const float z = chosen ? value(id) : 0.0f;
    float v = chosen ? d * a.scale : 0.0f, out[NV];
    // The first slot of an expert speaks for all slots that name it: v becomes their sum where the
    // score is one of the whole row.
    bool first = chosen;
    float together = v;
    each_turn([&](auto n) __attribute__((always_inline)) {
      const uint32_t other = (i + n) & 15u;
      const bool again = turned<decltype(n)::value>(id) == id && chosen;
      const float ov = turned<decltype(n)::value>(v);
      if (again) {
        together += ov;
        if (other < i) first = false;
      }
    });
    float mine = 0.0f;  // the choice's gradient
    float inv = 0.0f, q = 0.0f, top = 0.0f;
    if (whole) {
      top = -__builtin_inff();
#pragma unroll
      for (uint32_t j = 0; j < NV; ++j) {
        const uint32_t e = nkbal::expert<G>(lane, j);
        out[j] = e < E ? nkbal::at(raw, j, e, E) : -__builtin_inff();
        top = fmaxf(top, out[j]);
      }
      top = nkbal::reduce<G, true>(top);
      if (top == -__builtin_inff()) top = 0.0f;
      if (first) s[id] = 1.0f;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      float others = 0.0f, total = 0.0f;
#pragma unroll
      for (uint32_t j = 0; j < NV; ++j) {
        out[j] = nkbal::exp_nonpos(out[j] - top);
        total += out[j];
        if (!hit(s[nkbal::expert<G>(lane, j)])) others += out[j];
      }
      total = nkbal::sum<G>(total);
      others = nkbal::sum<G>(others);
      inv = total == 0.0f ? 0.0f : 1.0f / total;
      const float p = first ? nkbal::exp_nonpos(z - top) * inv : 0.0f;
      v = first ? together : 0.0f;
      q = nkbal::sum<16>(p * v);
      float diff = v * (others * inv);
      each_turn([&](auto n) __attribute__((always_inline)) { diff = fmaf(turned<decltype(n)::value>(p), v - turned<decltype(n)::value>(v), diff); });
      mine = p * diff;
    } else {
      float p;
      if (a.scoring == kSigmoid) {
        p = chosen ? sigmoid(z) : 0.0f;
      } else {
        float m = nkbal::reduce<16, true>(chosen ? z : -__builtin_inff());
        if (m == -__builtin_inff()) m = 0.0f;
        p = chosen ? nkbal::exp_nonpos(z - m) : 0.0f;
      }
      float steep = a.scoring == kSigmoid ? slope(z) : p;
      if (a.renormalise) {
        // (each factor by the sum by itself: of small sigmoids 1 / sum^2 is past the range of fp32)
        const float total = nkbal::sum<16>(p);
        const float r = total == 0.0f ? 0.0f : 1.0f / total;
        float diff = 0.0f;
        p *= r;
        steep *= r;
        each_turn([&](auto n) __attribute__((always_inline)) { diff = fmaf(turned<decltype(n)::value>(p), v - turned<decltype(n)::value>(v), diff); });
        v = diff;
      }
      v *= steep;
      if (!chosen) v = 0.0f;
      mine = v;
      if (__ballot(chosen && !first))  // an expert in several slots
        each_turn([&](auto n) __attribute__((always_inline)) {
          const float ov = turned<decltype(n)::value>(v);
          mine += turned<decltype(n)::value>(id) == id && chosen ? ov : 0.0f;
        });
    }
    if (first) s[id] = mine;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (whole) {
#pragma unroll
      for (uint32_t j = 0; j < NV; ++j) out[j] = live ? -(out[j] * inv) * q : 0.0f;
    } else {
#pragma unroll
      for (uint32_t j = 0; j < NV; ++j) out[j] = 0.0f;
    }
#pragma unroll
    for (uint32_t j = 0; j < NV; ++j) {
      const float at = s[nkbal::expert<G>(lane, j)];
      if (hit(at)) out[j] = at;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (first) s[id] = none;
    const bool writes = lane / G < rows;
    X* to = static_cast<X*>(a.grad) + (uint64_t)t * a.grad_stride;
    if (a.accumulate) {
      nkbal::Rows<X, NV> old;
      nkbal::load_rows<X, G, NV>(a.grad, a.grad_stride, t0, rows, E, old);
#pragma unroll
      for (uint32_t j = 0; j < NV; ++j) {
        const uint32_t e = nkbal::expert<G>(lane, j);
        out[j] += e < E ? nkbal::at(old, j, e, E) : 0.0f;
      }
    }
    nkbal::store_rows<X, G, NV>(a.grad, a.grad_stride, t0, rows, E, out);
    if (a.shared && i == a.k && writes && (G == 16u || lane < 16u)) {
      float gate = live ? d * slope(value(E)) : 0.0f;
      if constexpr (sizeof(X) == 4) {
        to[E] = a.accumulate ? to[E] + gate : gate;
      } else {
        if (a.accumulate) gate += nk::bf16_f32(to[E]);
        to[E] = (uint16_t)nk::bf16x2_hw(gate, 0.0f);
      }
    }
  }
}

}  // namespace nksel

#define NETRA_SELECT(NAME, X, KIND, G, NV)                                                                  \
  extern "C" __global__ __launch_bounds__(256) void netra_router_select_##NAME##_##G##x##NV##_gfx950(       \
      nksel::Select a) {                                                                                    \
    nksel::select<X, G, NV, nksel::KIND>(a);                                                                \
  }                                                                                                         \
  extern "C" __global__ __launch_bounds__(256) void netra_router_select_scored_##NAME##_##G##x##NV##_gfx950( \
      nksel::Select a) {                                                                                    \
    nksel::select<X, G, NV, nksel::kScore>(a);                                                              \
  }                                                                                                         \
  extern "C" __global__                                                                                     \
      __launch_bounds__(256) void netra_router_select_gradient_##NAME##_##G##x##NV##_gfx950(nksel::SelectGradient a) { \
    nksel::gradient<X, G, NV>(a);                                                                           \
  }
#define NETRA_SELECTS(NAME, X, KIND)                                                                        \
  NETRA_SELECT(NAME, X, KIND, 16, 4)                                                                        \
  NETRA_SELECT(NAME, X, KIND, 16, 8)                                                                        \
  NETRA_SELECT(NAME, X, KIND, 16, 16)                                                                       \
  NETRA_SELECT(NAME, X, KIND, 16, 32)                                                                       \
  NETRA_SELECT(NAME, X, KIND, 64, 16)
NETRA_SELECTS(bf16, uint16_t, kWhole)
NETRA_SELECTS(f32, float, kDistance)
