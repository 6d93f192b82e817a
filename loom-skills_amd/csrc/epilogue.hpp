// The epilogue of the products with a bias, an activation and a residual (qmm_linear, qmm_ffn_gate_up), applied by the
// matvec and GEMM kernels to their f32 sums in registers:
//
//   one matrix     y[o] = act(v + bias[c]) + res[o]
//   two matrices   y[o] = act(g + bias[c]) (u + bias2[c]);   swiglu_oai as the experts' (act_fn)
//
// o = row n + c. Everything is f32 until the one rounding of a bf16 output (to nearest even). A kernel takes the
// epilogue as a type parameter: NoEpi is the plain store, whose code is the kernel's own.
#pragma once

#include <type_traits>

#include "common.hpp"

namespace qmm {

struct NoEpi {};
struct Epi {
  const float *bias, *bias2;   // f32 [n] or NULL (bias2: two matrices)
  const void *res;             // [rows, n] f32 or bf16, or NULL; may be y itself (a value is read by the thread that writes it)
  void *y;                     // [rows, n]
  int act;                     // enum qmm_act
  int res_bf16, y_bf16;
};
template <class EP>
inline constexpr bool kEpi = std::is_same_v<EP, Epi>;

// The sigmoid of the whole range: e^-v overflows to infinity for v < -88, whose reciprocal is 0.
__device__ __forceinline__ float sigmoidf_(float v) { return 1.0f / (1.0f + expf(-v)); }
// 2 sqrt(2 / pi) (v + 0.044715 v^3), the argument of GELU's sigmoid form: (1 + tanh(z)) / 2 = 1 / (1 + e^-2z), which
// keeps its relative precision for large negative v where 1 + tanh(z) cancels
__device__ __forceinline__ float gelu_arg(float v) { return 1.5957691216057308f * (v + 0.044715f * v * v * v); }
// Phi(v) = erfc(-v / sqrt 2) / 2, for the same reason as the complement
__device__ __forceinline__ float normal_cdf(float v) { return 0.5f * erfcf(-0.70710678118654752f * v); }

__device__ __forceinline__ float act1(int act, float v) {
  switch (act) {
    case QMM_ACT_SILU: return v / (1.0f + expf(-v));
    case QMM_ACT_RELU: return v > 0.f ? v : (v != v ? v : 0.f);
    case QMM_ACT_GELU: return v / (1.0f + expf(-gelu_arg(v)));
    case QMM_ACT_GELU_ERF: return v * normal_cdf(v);
    case QMM_ACT_SIGMOID: return sigmoidf_(v);
    default: return v;
  }
}
// swiglu_oai's clamps by comparisons, which keep a NaN (fminf and fmaxf return their other argument); other values as act_fn's
__device__ __forceinline__ float oai_gate(float g) { return g > 7.0f ? 7.0f : g; }
__device__ __forceinline__ float oai_up(float u) { return u > 7.0f ? 7.0f : u < -7.0f ? -7.0f : u; }
__device__ __forceinline__ float act2(int act, float g, float u) {
  if (act == QMM_ACT_SWIGLU_OAI) {
    const float xg = oai_gate(g);
    return xg / (1.0f + expf(-1.702f * xg)) * (oai_up(u) + 1.0f);
  }
  return act == QMM_ACT_SILU ? act_fn(act, g, u) : act1(act, g) * u;
}

__device__ __forceinline__ float load_val(const void *p, int bf16, int64_t o) {
  return bf16 ? bf16_to_f32(static_cast<const u16 *>(p)[o]) : static_cast<const float *>(p)[o];
}
__device__ __forceinline__ void store_val(void *p, int bf16, int64_t o, float v) {
  if (bf16) static_cast<u16 *>(p)[o] = __builtin_bit_cast(u16, (__bf16)v);   // to nearest even; a NaN stays one
  else static_cast<float *>(p)[o] = v;
}

// V (4 or 8) neighbouring values at element offset o, a multiple of V of 16-byte aligned rows
template <int V>
__device__ __forceinline__ void load_vals(const void *p, int bf16, int64_t o, float (&v)[V]) {
  if (bf16) {
    u32 d[V / 2];
    __builtin_memcpy(d, __builtin_assume_aligned(static_cast<const u16 *>(p) + o, 2 * V), 2 * V);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) { v[2 * j] = u32_as_f32(d[j] << 16); v[2 * j + 1] = u32_as_f32(d[j] & 0xFFFF0000u); }
  } else {
    __builtin_memcpy(v, __builtin_assume_aligned(static_cast<const float *>(p) + o, 16), 4 * V);
  }
}
template <int V>
__device__ __forceinline__ void store_vals(void *p, int bf16, int64_t o, const float (&v)[V]) {
  if (bf16) {
    __bf16 d[V];
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = (__bf16)v[j];
    __builtin_memcpy(__builtin_assume_aligned(static_cast<u16 *>(p) + o, 2 * V), d, 2 * V);
  } else {
    __builtin_memcpy(__builtin_assume_aligned(static_cast<float *>(p) + o, 16), v, 4 * V);
  }
}

// whether the rows of y and the residual start on 16 bytes
__device__ __forceinline__ bool ep_wide(const Epi &e, int n) {
  return n % 8 == 0 && ((reinterpret_cast<uintptr_t>(e.y) | reinterpret_cast<uintptr_t>(e.res)) & 15) == 0;
}

// output o = row n + c of a one-matrix product
__device__ __forceinline__ void epi_store(const Epi &e, int64_t o, int64_t c, float v) {
  if (e.bias) v += e.bias[c];
  v = act1(e.act, v);
  if (e.res) v += load_val(e.res, e.res_bf16, o);
  store_val(e.y, e.y_bf16, o, v);
}
// and of a two-matrix one
__device__ __forceinline__ void epi_store2(const Epi &e, int64_t o, int64_t c, float g, float u) {
  if (e.bias) g += e.bias[c];
  if (e.bias2) u += e.bias2[c];
  store_val(e.y, e.y_bf16, o, act2(e.act, g, u));
}

// bias values at column c (0 without one), loaded once where a thread finishes many rows of a column
__device__ __forceinline__ float epi_bias(const float *b, int64_t c) { return b ? b[c] : 0.f; }
// v with its bias added, r the residual value
__device__ __forceinline__ void epi_put(const Epi &e, int act, int64_t o, float v, float r) {
  v = act1(act, v);
  store_val(e.y, e.y_bf16, o, e.res ? v + r : v);
}

// The gradients leave as bf16, so their sigmoid is v_exp_f32 and v_rcp_f32 (each about 1 ulp, the argument's product with
// log2 e another |v| half steps of f32): with an IEEE division and a range-reduced expf a value the gradient GEMM's epilogue
// took a fifth of it
__device__ __forceinline__ float sigmoid_fast_(float v) { return __builtin_amdgcn_rcpf(1.0f + __expf(-v)); }

// act(v) and its slope d act / d v (relu: 0 at 0)
__device__ __forceinline__ void act1_slope(int act, float v, float &a, float &da) {
  switch (act) {
    case QMM_ACT_SILU: {
      const float s = sigmoid_fast_(v);
      a = v * s;
      da = s * (1.0f + v * (1.0f - s));
      return;
    }
    case QMM_ACT_RELU:
      a = act1(act, v);
      da = v > 0.f ? 1.f : 0.f;
      return;
    case QMM_ACT_GELU: {   // v s(z): s + v s (1 - s) z'; past the range of v^3 s (1 - s) is 0 and z' infinite
      const float s = sigmoid_fast_(gelu_arg(v)), p = s * (1.0f - s);
      a = v * s;
      da = p > 0.f ? s + v * p * 1.5957691216057308f * (1.0f + 0.134145f * v * v) : s;
      return;
    }
    case QMM_ACT_GELU_ERF: {
      const float c = normal_cdf(v);
      a = v * c;
      da = c + 0.3989422804014327f * v * expf(-0.5f * v * v);
      return;
    }
    case QMM_ACT_SIGMOID: {   // s(v) s(-v) from e = e^-|v|: 1 - s(v) has no bits left for v past 17
      const float e = __expf(-fabsf(v)), r = __builtin_amdgcn_rcpf(1.0f + e);
      a = v < 0.f ? e * r : r;
      da = e * r * r;
      return;
    }
    default:
      a = v;
      da = 1.f;
  }
}
// the gradient of act1(v) at dy
__device__ __forceinline__ float act1_grad(int act, float v, float dy) {
  float a, da;
  act1_slope(act, v, a, da);
  return dy * da;
}
// the gradients of act2(g, u) at dy. swiglu_oai: those of the clamps are 1 up to and at their limits, 0 past them
__device__ __forceinline__ void act2_grad(int act, float g, float u, float dy, float &dg, float &du) {
  if (act == QMM_ACT_SWIGLU_OAI) {
    const float xg = oai_gate(g), yu = oai_up(u), s = sigmoid_fast_(1.702f * xg);
    dg = g > 7.0f ? 0.f : dy * (yu + 1.0f) * s * (1.0f + 1.702f * xg * (1.0f - s));
    du = fabsf(u) > 7.0f ? 0.f : dy * xg * s;
    return;
  }
  float a, da;
  act1_slope(act, g, a, da);
  dg = dy * (u * da);
  du = dy * a;
}

// f(constant) for the activation: one branch for the values that f works on, where a branch a value costs more than the
// activation (relu on Q4_K 12288 x 4096 at 2048 rows 234 us, so 196, without an activation 194)
template <class F>
__device__ __forceinline__ void with_act(int act, F &&f) {
  switch (act) {
    case QMM_ACT_SILU: f(std::integral_constant<int, QMM_ACT_SILU>{}); return;
    case QMM_ACT_SWIGLU_OAI: f(std::integral_constant<int, QMM_ACT_SWIGLU_OAI>{}); return;
    case QMM_ACT_RELU: f(std::integral_constant<int, QMM_ACT_RELU>{}); return;
    case QMM_ACT_GELU: f(std::integral_constant<int, QMM_ACT_GELU>{}); return;
    case QMM_ACT_SIGMOID: f(std::integral_constant<int, QMM_ACT_SIGMOID>{}); return;
    case QMM_ACT_GELU_ERF: f(std::integral_constant<int, QMM_ACT_GELU_ERF>{}); return;
    default: f(std::integral_constant<int, QMM_ACT_NONE>{});
  }
}

// Eight or four values of the lane at t in LDS (t2: those of the second matrix) through the activation. GELU_ERF, some hundred
// instructions, is applied in LDS by a loop over the values; the others are unrolled.
template <int V>
__device__ __forceinline__ void act1_rows(int act, float *t, float (&v)[V]) {
  if (act == QMM_ACT_GELU_ERF) {
#pragma unroll 1
    for (int q = 0; q < V; ++q) t[q] = act1(QMM_ACT_GELU_ERF, t[q]);
    act = QMM_ACT_NONE;
  }
#pragma unroll
  for (int q = 0; q < V; ++q) v[q] = t[q];
  with_act(act, [&](auto a) __attribute__((always_inline)) {
    if constexpr (a.value != QMM_ACT_GELU_ERF && a.value != QMM_ACT_SWIGLU_OAI) {
#pragma unroll
      for (int q = 0; q < V; ++q) v[q] = act1(a.value, v[q]);
    }
  });
}
template <int V>
__device__ __forceinline__ void act2_rows(int act, float *t, const float *t2, float (&v)[V]) {
  if (act == QMM_ACT_GELU_ERF) {
#pragma unroll 1
    for (int q = 0; q < V; ++q) t[q] = act1(QMM_ACT_GELU_ERF, t[q]);
    act = QMM_ACT_NONE;
  }
#pragma unroll
  for (int q = 0; q < V; ++q) v[q] = t[q];
  with_act(act, [&](auto a) __attribute__((always_inline)) {
    if constexpr (a.value != QMM_ACT_GELU_ERF) {
#pragma unroll
      for (int q = 0; q < V; ++q) v[q] = act2(a.value, v[q], t2[q]);
    }
  });
}
// its gradient at dy
template <int V>
__device__ __forceinline__ void act1_grad_rows(int act, float *t, const float (&dy)[V], float (&d)[V]) {
  if (act == QMM_ACT_GELU_ERF) {
#pragma unroll 1
    for (int q = 0; q < V; ++q) t[q] = act1_grad(QMM_ACT_GELU_ERF, t[q], 1.f);
#pragma unroll
    for (int q = 0; q < V; ++q) d[q] = dy[q] * t[q];
    return;
  }
  with_act(act, [&](auto a) __attribute__((always_inline)) {
    if constexpr (a.value != QMM_ACT_GELU_ERF && a.value != QMM_ACT_SWIGLU_OAI) {
#pragma unroll
      for (int q = 0; q < V; ++q) d[q] = act1_grad(a.value, t[q], dy[q]);
    }
  });
}

}  // namespace qmm

// ---- the products that take an epilogue (ep NULL: the plain call); their argument checks hold for a NULL y with ep
int qmm_mv_impl(int fmt, int64_t k, int64_t n, int64_t tokens, int accumulate, const void *x, int x_dtype, const void *w,
                const void *ws, float *y, hipStream_t s, const qmm::Epi *ep);
int qmm_mv_gate_up_impl(int fmt, int64_t k, int64_t n, int64_t tokens, const void *x, int x_dtype, const void *w,
                        const void *ws, const void *w2, const void *ws2, hipStream_t s, const qmm::Epi &ep);
int qmm_mv_q8_impl(int fmt, int64_t k, int64_t n, int64_t tokens, int accumulate, const void *x, int x_dtype,
                   const void *w, float *y, hipStream_t s, const qmm::Epi *ep);
int qmm_mv_gate_up_q8_impl(int fmt, int64_t k, int64_t n, int64_t tokens, const void *x, const void *w, const void *w2,
                           hipStream_t s, const qmm::Epi &ep);
int qmm_mv_mxfp4s_q8_impl(int mode, int64_t k, int64_t n, int64_t tokens, int accumulate, const void *x, int x_dtype,
                          const void *w, const void *ws, const void *w2, const void *ws2, float *y, float *y2,
                          hipStream_t s, const qmm::Epi *ep);
int qmm_gemm_mxfp4_impl(int fmt, int mode, int64_t rows, int64_t k, int64_t n, const void *x, const void *x_scales,
                        const void *w, const void *ws, const void *w2, const void *ws2, void *y, int y_dtype,
                        hipStream_t s, const qmm::Epi *ep);
