// Element types and activations of the row operators (pp_groupnorm.hip, pp_linear.hip): features are [rows, channels] in fp32, bf16
// or fp16, arithmetic is fp32 (sums that run over many rows: fp64), and a result is rounded once, when it is stored.
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

// y = act(z).  `act` is uniform over a launch: the branch costs one scalar compare per vector of elements
__device__ __forceinline__ float pp_act1(float z, int act, float slope) {
  switch (act) {
    case PP_ACT_RELU: return z < 0.f ? 0.f : z;  // (NaN stays NaN)
    case PP_ACT_LEAKY: return z > 0.f ? z : slope * z;
    case PP_ACT_SILU: return z / (1.f + expf(-z));
    case PP_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    default: return z;
  }
}
// d act(z) / dz; at the kink of relu / leaky the slope of the negative side, as torch has it
__device__ __forceinline__ float pp_dact1(float z, int act, float slope) {
  switch (act) {
    case PP_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case PP_ACT_LEAKY: return z > 0.f ? 1.f : slope;
    case PP_ACT_SILU: {
      const float s = 1.f / (1.f + expf(-z));
      return s * (1.f + z * (1.f - s));
    }
    case PP_ACT_GELU:
      return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * expf(-0.5f * z * z);
    default: return 1.f;
  }
}

static inline bool pp_rows_dtype_ok(int dtype) { return dtype == PP_F32 || dtype == PP_BF16 || dtype == PP_F16; }
static inline bool pp_rows_act_ok(int act) { return act >= PP_ACT_NONE && act <= PP_ACT_GELU; }
