// Element types and activations of the row operators (pp_groupnorm.hip, pp_linear.hip): features are [rows, channels] in fp32, bf16
// or fp16, arithmetic is fp32 (sums that run over many rows: fp64, or fp32 chains of a bounded length that are added in fp64), and a result is
// rounded once, when it is stored (the linear layer's dz once more, as the operand of its products: see there).
#pragma once
#include "pp_common.h"

typedef __bf16 pp_bf16;
typedef _Float16 pp_f16;

static inline int pp_dtype_bytes(int dtype) { return dtype == PP_F32 ? 4 : 2; }

template <typename T, int VEC>
struct PPVec {
  typedef T type __attribute__((ext_vector_type(VEC)));
};

// VEC consecutive elements as fp32.  VEC * sizeof(T) is the alignment the caller has checked (16 bytes, or one element)
template <typename T, int VEC>
__device__ __forceinline__ void pp_load(const T* __restrict__ p, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = (float)*p;
  } else {
    const typename PPVec<T, VEC>::type q = *(const typename PPVec<T, VEC>::type*)p;
#pragma unroll
    for (int u = 0; u < VEC; ++u) v[u] = (float)q[u];
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void pp_store(T* __restrict__ p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    *p = (T)v[0];
  } else {
    typename PPVec<T, VEC>::type q;
#pragma unroll
    for (int u = 0; u < VEC; ++u) q[u] = (T)v[u];
    *(typename PPVec<T, VEC>::type*)p = q;
  }
}

// exp(x): the hardware's exp2 on x log2(e); the rounding of that product costs |x| 2^-24 of the result, and a result below 2^-126 is 0
__device__ __forceinline__ float pp_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

// Phi(z) = (1 + erf(z / sqrt 2)) / 2.  With t = min(|z|, 6): Phi(-t) = 2^-q(t), q of degree 9 fitted (least squares, reweighted towards
// the smallest largest error of Phi) to -log2 Phi(-t) on [0, 6].  |error| <= 1.5 2^-24 everywhere, 2.5e-5 of the value down to z = -6
// (where 1 + erf loses all of its bits).  Behind it the exponent goes on as q(6) + d (c1 + c2 d), d = |z| - 6, fitted on [6, 14]: off by
// at most 0.7 % of a Phi below 1e-9, but falling as fast as Phi does, so that z Phi(z) goes to 0 however far z is (a Phi that stayed at
// its value at -6 made gelu(-1e6) -1e-3).  18 instructions, without the two branches of erff that both run in a wave whose values
// differ -- group norm with gelu over 2.5 M rows of 96 channels, bf16: 350 us a pass with erff, see pp_groupnorm.hip
__device__ __forceinline__ float pp_phi(float z) {
  const float t = fminf(fabsf(z), 6.f), d = fabsf(z) - t;
  float q = -1.524596626722996e-07f;
  q = fmaf(q, t, 3.834877588815289e-06f);
  q = fmaf(q, t, -3.800627018790692e-05f);
  q = fmaf(q, t, 0.00015954984701238573f);
  q = fmaf(q, t, 0.00022161900415085256f);
  q = fmaf(q, t, -0.007183804642409086f);
  q = fmaf(q, t, 0.0525796078145504f);
  q = fmaf(q, t, 0.4591817855834961f);
  q = fmaf(q, t, 1.1511082649230957f);
  q = fmaf(q, t, 0.9999999403953552f);
  q = fmaf(d, fmaf(d, 0.7134105526322216f, 8.867419283080718f), q);
  const float e = __builtin_amdgcn_exp2f(-q);
  return z > 0.f ? 1.f - e : e;  // (NaN stays NaN: with it d, q and e are)
}
__device__ __forceinline__ float pp_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + pp_exp(-z)); }

// the same at any element's address: the hardware takes 16-byte accesses that start anywhere
template <typename T, int N>
__device__ __forceinline__ void pp_load_any(const T* __restrict__ p, float (&v)[N]) {
  typename PPVec<T, N>::type q;
  __builtin_memcpy(&q, p, sizeof(q));
#pragma unroll
  for (int u = 0; u < N; ++u) v[u] = (float)q[u];
}
template <typename T, int N>
__device__ __forceinline__ void pp_store_any(T* __restrict__ p, const float (&v)[N]) {
  typename PPVec<T, N>::type q;
#pragma unroll
  for (int u = 0; u < N; ++u) q[u] = (T)v[u];
  __builtin_memcpy(p, &q, sizeof(q));
}

// y = act(z).  `act` is uniform over a launch: the branch costs one scalar compare per vector of elements
__device__ __forceinline__ float pp_act1(float z, int act, float slope) {
  switch (act) {
    case PP_ACT_RELU: return z < 0.f ? 0.f : z;  // (NaN stays NaN)
    case PP_ACT_LEAKY: return z > 0.f ? z : slope * z;
    case PP_ACT_SILU: return z * pp_sigmoid(z);
    case PP_ACT_GELU: return z * pp_phi(z);
    default: return z;
  }
}
// d act(z) / dz; at the kink of relu / leaky the slope of the negative side, as torch has it
__device__ __forceinline__ float pp_dact1(float z, int act, float slope) {
  switch (act) {
    case PP_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case PP_ACT_LEAKY: return z > 0.f ? 1.f : slope;
    case PP_ACT_SILU: {
      const float s = pp_sigmoid(z);
      return s * fmaf(z, 1.f - s, 1.f);
    }
    case PP_ACT_GELU: return fmaf(z * 0.39894228040143268f, pp_exp(-0.5f * z * z), pp_phi(z));
    default: return 1.f;
  }
}

// the same of N values; the branch on `act` stands outside, which also keeps the code short
template <int N>
__device__ __forceinline__ void pp_act(float (&z)[N], int act, float slope) {
#define PP_EACH(ACT) \
  case ACT:          \
    _Pragma("unroll") for (int i = 0; i < N; ++i) z[i] = pp_act1(z[i], ACT, slope); \
    break;
  switch (act) { PP_EACH(PP_ACT_RELU) PP_EACH(PP_ACT_LEAKY) PP_EACH(PP_ACT_SILU) PP_EACH(PP_ACT_GELU) default: break; }
#undef PP_EACH
}
// d[i] *= act'(z[i])
template <int N>
__device__ __forceinline__ void pp_dact(float (&d)[N], const float (&z)[N], int act, float slope) {
#define PP_EACH(ACT) \
  case ACT:          \
    _Pragma("unroll") for (int i = 0; i < N; ++i) d[i] *= pp_dact1(z[i], ACT, slope); \
    break;
  switch (act) { PP_EACH(PP_ACT_RELU) PP_EACH(PP_ACT_LEAKY) PP_EACH(PP_ACT_SILU) PP_EACH(PP_ACT_GELU) default: break; }
#undef PP_EACH
}

static inline bool pp_rows_dtype_ok(int dtype) { return dtype == PP_F32 || dtype == PP_BF16 || dtype == PP_F16; }
static inline bool pp_rows_act_ok(int act) { return act >= PP_ACT_NONE && act <= PP_ACT_GELU; }
