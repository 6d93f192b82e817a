// Products on quantized weights with an epilogue: argument checks and the choice of the kernel by the operand's type.
//
//   qmm_linear            y = act(x W^T + bias) + residual
//   qmm_linear_grad       dpre = dy act'(x W^T + bias)
//   qmm_ffn_gate_up       y = act(x Wg^T + bg) (x Wu^T + bu)
//   qmm_ffn_gate_up_grad  dgu[t] = (dy u act'(g), dy act(g)),  g = x Wg^T + bg, u = x Wu^T + bu
//
// A few rows of Q4_0, Q4_K, Q6_K and MXFP4 (qmm_mv_mfma_fits) take mv_mfma.hip, which adds the same exact products in an
// order of its own. The other kernels are the products' own (gemv.hip, gemv_q4k.hip, gemv_q4kt.hip on f32 / bf16 rows;
// gemv_q8.hip, gemv_q4kt.hip, mv_q8_mfma.hip on Q8_1; gemm_tile_kernel.hpp, gemm_dense.hip on row-scaled f16;
// grouped_mxfp4.hip on MXFP8) with the epilogue of epilogue.hpp in place of their plain store: their sums have the bits of
// the call without one.
#include "epilogue.hpp"
#include "gemm_tile.hpp"

using namespace qmm;

int qmm_gemm_epi(int fmt, int kind, int64_t rows, int64_t k, int64_t n, const void *x, const float *scales, const void *w,
                 const void *w2, const void *dy, int dy_bf16, hipStream_t s, const Epi &ep);

bool qmm_mv_mfma_fits(int fmt, int x_dtype, int64_t k, int64_t n, int64_t tokens);
int qmm_mv_mfma(int fmt, int x_dtype, int64_t k, int64_t n, int64_t tokens, const void *x, const void *w, const void *ws,
                const void *w2, const void *ws2, hipStream_t s, const Epi &ep);

namespace {

bool val_dtype(int d) { return d == QMM_F32 || d == QMM_BF16; }
bool val_aligned(const void *p, int d) { return aligned(p, d == QMM_BF16 ? 2 : 4); }

}  // namespace

extern "C" int qmm_linear(int fmt, int act, int64_t tokens, int64_t k, int64_t n, const void *x, int x_dtype,
                          const void *x_scales, const void *w, const void *ws, const float *bias, const void *residual,
                          int res_dtype, void *y, int y_dtype, qmm_stream_t stream) {
  if (act < QMM_ACT_SILU || act > QMM_ACT_SIGMOID || act == QMM_ACT_SWIGLU_OAI) return QMM_ERR_RANGE;
  if (!y) return QMM_ERR_NULL;
  if (!val_dtype(y_dtype) || (residual && !val_dtype(res_dtype))) return QMM_ERR_DTYPE;
  if (!val_aligned(y, y_dtype) || (residual && !val_aligned(residual, res_dtype)) || !aligned(bias, 4)) return QMM_ERR_ALIGN;
  const Epi ep{bias, nullptr, residual, y, act, res_dtype == QMM_BF16, y_dtype == QMM_BF16};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if ((val_dtype(x_dtype) || x_dtype == QMM_Q8) && qmm_mv_mfma_fits(fmt, x_dtype, k, n, tokens))
    return qmm_mv_mfma(fmt, x_dtype, k, n, tokens, x, w, ws, nullptr, nullptr, s, ep);
  switch (x_dtype) {
    case QMM_F32:
    case QMM_BF16: return qmm_mv_impl(fmt, k, n, tokens, 0, x, x_dtype, w, ws, nullptr, s, &ep);
    case QMM_Q8:
      if (fmt == QMM_MXFP4S)
        return qmm_mv_mxfp4s_q8_impl(0, k, n, tokens, 0, x, x_dtype, w, ws, nullptr, nullptr, nullptr, nullptr, s, &ep);
      return qmm_mv_q8_impl(fmt, k, n, tokens, 0, x, x_dtype, w, nullptr, s, &ep);
    case QMM_F16:
      return qmm_gemm_epi(fmt, kTLinear, tokens, k, n, x, static_cast<const float *>(x_scales), w, nullptr, nullptr, 0, s, ep);
    case QMM_MXFP8:
      return qmm_gemm_mxfp4_impl(fmt, QMM_GEMM_STORE, tokens, k, n, x, x_scales, w, ws, nullptr, nullptr, nullptr, QMM_F32,
                                 s, &ep);
    default: return QMM_ERR_DTYPE;
  }
}

extern "C" int qmm_ffn_gate_up(int fmt, int act, int64_t tokens, int64_t k, int64_t n, const void *x, int x_dtype,
                               const void *x_scales, const void *w, const void *ws, const void *w2, const void *ws2,
                               const float *bias, const float *bias2, void *y, int y_dtype, qmm_stream_t stream) {
  if (act < QMM_ACT_SILU || act > QMM_ACT_SIGMOID) return QMM_ERR_RANGE;
  if (!y) return QMM_ERR_NULL;
  if (!val_dtype(y_dtype)) return QMM_ERR_DTYPE;
  if (!val_aligned(y, y_dtype) || !aligned(bias, 4) || !aligned(bias2, 4)) return QMM_ERR_ALIGN;
  const Epi ep{bias, bias2, nullptr, y, act, 0, y_dtype == QMM_BF16};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if ((val_dtype(x_dtype) || x_dtype == QMM_Q8) && qmm_mv_mfma_fits(fmt, x_dtype, k, n, tokens)) {
    if (!w2) return QMM_ERR_NULL;
    return qmm_mv_mfma(fmt, x_dtype, k, n, tokens, x, w, ws, w2, ws2, s, ep);
  }
  switch (x_dtype) {
    case QMM_F32:
    case QMM_BF16: return qmm_mv_gate_up_impl(fmt, k, n, tokens, x, x_dtype, w, ws, w2, ws2, s, ep);
    case QMM_Q8:
      if (fmt == QMM_MXFP4S)
        return qmm_mv_mxfp4s_q8_impl(1, k, n, tokens, 0, x, x_dtype, w, ws, w2, ws2, nullptr, nullptr, s, &ep);
      return qmm_mv_gate_up_q8_impl(fmt, k, n, tokens, x, w, w2, s, ep);
    case QMM_F16:
      return qmm_gemm_epi(fmt, kTGlu, tokens, k, n, x, static_cast<const float *>(x_scales), w, w2, nullptr, 0, s, ep);
    case QMM_MXFP8:
      return qmm_gemm_mxfp4_impl(fmt, QMM_GEMM_SWIGLU, tokens, k, n, x, x_scales, w, ws, w2, ws2, nullptr, QMM_F32, s, &ep);
    default: return QMM_ERR_DTYPE;
  }
}

extern "C" int qmm_ffn_gate_up_grad(int fmt, int act, int64_t tokens, int64_t k, int64_t n, const void *x,
                                    const float *x_scales, const void *w, const void *w2, const float *bias,
                                    const float *bias2, const void *dy, int dy_dtype, void *dgu, qmm_stream_t stream) {
  if (act < QMM_ACT_SILU || act > QMM_ACT_SIGMOID) return QMM_ERR_RANGE;
  if (!dgu) return QMM_ERR_NULL;
  if (!val_dtype(dy_dtype)) return QMM_ERR_DTYPE;
  if (!aligned(dgu, 2) || !val_aligned(dy, dy_dtype) || !aligned(bias, 4) || !aligned(bias2, 4)) return QMM_ERR_ALIGN;
  const Epi ep{bias, bias2, nullptr, dgu, act, 0, 1};
  return qmm_gemm_epi(fmt, kTGluGrad, tokens, k, n, x, x_scales, w, w2, dy, dy_dtype == QMM_BF16,
                      reinterpret_cast<hipStream_t>(stream), ep);
}

extern "C" int qmm_linear_grad(int fmt, int act, int64_t tokens, int64_t k, int64_t n, const void *x, const float *x_scales,
                               const void *w, const float *bias, const void *dy, int dy_dtype, void *dpre,
                               qmm_stream_t stream) {
  if (act < QMM_ACT_SILU || act > QMM_ACT_SIGMOID || act == QMM_ACT_SWIGLU_OAI) return QMM_ERR_RANGE;
  if (!dpre) return QMM_ERR_NULL;
  if (!val_dtype(dy_dtype)) return QMM_ERR_DTYPE;
  if (!aligned(dpre, 2) || !val_aligned(dy, dy_dtype) || !aligned(bias, 4)) return QMM_ERR_ALIGN;
  const Epi ep{bias, nullptr, nullptr, dpre, act, 0, 1};
  return qmm_gemm_epi(fmt, kTLinearGrad, tokens, k, n, x, x_scales, w, nullptr, dy, dy_dtype == QMM_BF16,
                      reinterpret_cast<hipStream_t>(stream), ep);
}
