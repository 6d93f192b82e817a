// Products of 16-bit expert weights W [E, n, k] and rows sorted by expert, with their gradients: argument checks and the choice
// of the kernel. Expert e owns rows offsets[e] .. offsets[e + 1] - 1, as many as it has: no padding between experts.
//
//   qmm_ragged_mm     y[t] = W_e x[t]          few rows an expert on few_rows.hpp, else the tiles of tile_mm.hpp
//   qmm_ragged_mm_t   dx[t] = W_e^T dy[t]
//   qmm_ragged_mm_dw  dW_e = sum_t dy[t] x[t]^T
#include "ragged_mm.hpp"
#include "w4_mm.hpp"

using namespace qmm;

namespace qmm {
int ragged_few(const few::Args &a, bool f16, hipStream_t s) {
  return f16 ? few::launch_tt<few::kWF16, false, 4>(a, s) : few::launch_tt<few::kWBF16, false, 4>(a, s);
}
}  // namespace qmm

namespace {

constexpr int64_t kMaxSide = 1 << 20, kMaxRows = 1 << 24;

int check(int64_t rows, int64_t k, int64_t n, int E, const int32_t *offsets, const void *p, const void *q, int dtype,
          const void *out, int out_dtype) {
  if (dtype != QMM_BF16 && dtype != QMM_F16) return QMM_ERR_DTYPE;
  if (out_dtype != QMM_F32 && out_dtype != dtype) return QMM_ERR_DTYPE;
  if (rows < 0 || rows > kMaxRows || k <= 0 || k > kMaxSide || k % 8 || n <= 0 || n > kMaxSide || n % 8) return QMM_ERR_SHAPE;
  if (E < 1 || E > kMaxRaggedE) return QMM_ERR_RANGE;
  if (!offsets || !out || (rows && (!p || !q))) return QMM_ERR_NULL;
  if (!aligned(p, 16) || !aligned(q, 16) || !aligned(offsets, 4) || !aligned(out, 16)) return QMM_ERR_ALIGN;
  return QMM_OK;
}

bool takes_few_rows(int64_t rows, int64_t k, int64_t n) {
  // Up to 64 rows of 2^17 values in up to 2^30 products. us, few rows against tiles: one matrix 4096 x 4096 16 rows 10 and 12, 32 rows
  // 14 and 13, 64 rows 21 and 15; 1024 x 4096 64 rows 20 and 10; 4096 x 1024 32 rows 5 and 9; 8 experts 1024 x 2048 64 rows 9 and 10,
  // 128 rows 15 and 11; 32 experts 2880 x 2880 32 rows 40 and 44, 128 rows 87 and 82; 128 experts 768 x 2048 64 rows 24 and 25, 512
  // rows 57 and 51. With every row one expert's, whose rows are walked in turn: 64 experts 512 x 512 256 rows 22 and 7.
  return rows <= 64 && rows * k <= 1 << 17 && rows * n * k <= (int64_t)1 << 30;
}

int tiles(int op, tmm::Args &a, const tmm::Plan &p, int64_t outputs, int dtype, int out_dtype, bool rest, void *out,
          void *workspace, int64_t workspace_bytes, qmm_stream_t stream) {
  a.y = out;
  a.y_type = out_dtype;
  if (rest) a.rest = rest_blocks(a.rows, (int64_t)a.N * (out_dtype == QMM_F32 ? 4 : 2));
  if (int st = tmm::in_parts(a, p, outputs, workspace, workspace_bytes)) return st;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return dtype == QMM_F16 ? ragged_tiles_f16(op, a, p.shape, s) : ragged_tiles_bf16(op, a, p.shape, s);
}

bool sizes_ok(int64_t rows, int64_t k, int64_t n, int E) {
  return rows >= 0 && rows <= kMaxRows && k > 0 && k <= kMaxSide && k % 8 == 0 && n > 0 && n <= kMaxSide && n % 8 == 0 && E >= 1 &&
         E <= kMaxRaggedE;
}

}  // namespace

extern "C" int64_t qmm_ragged_mm_workspace_size(int64_t rows, int64_t k, int64_t n, int E) {
  if (!sizes_ok(rows, k, n, E)) return -1;
  return rows && !takes_few_rows(rows, k, n) ? tmm::part_bytes(tmm::plan_rows(tmm::kTiles, rows, E, n, k), rows * n) : 0;
}
extern "C" int64_t qmm_ragged_mm_t_workspace_size(int64_t rows, int64_t k, int64_t n, int E) {
  if (!sizes_ok(rows, k, n, E)) return -1;
  return rows ? tmm::part_bytes(tmm::plan_rows(tmm::kTiles, rows, E, k, n), rows * k) : 0;
}
extern "C" int64_t qmm_ragged_mm_dw_workspace_size(int64_t rows, int64_t k, int64_t n, int E) {
  return sizes_ok(rows, k, n, E) ? tmm::part_bytes(tmm::plan_sum(rows, E, n, k), E * n * k) : -1;
}

extern "C" int64_t qmm_tile_plan(int product, int64_t rows, int64_t k, int64_t n, int E) {
  const bool four_bit = product == QMM_PRODUCT_W4 || product == QMM_PRODUCT_W4_T;
  if (four_bit ? qmm_w4_mm_t_workspace_size(rows, k, n, E) < 0 : !sizes_ok(rows, k, n, E)) return -1;
  if (product == QMM_PRODUCT_RAGGED_DW) {
    const tmm::Plan p = tmm::plan_sum(rows, E, n, k);
    return tmm::plan_word(tmm::kTilesSum[p.shape], p);
  }
  if (product < 0 || product > QMM_PRODUCT_RAGGED_DW) return -1;
  if (rows == 0 || (product == QMM_PRODUCT_RAGGED && takes_few_rows(rows, k, n))) return 0;
  if (product == QMM_PRODUCT_W4) {
    const tmm::Plan p = w4_gemm_plan(rows, E, n, k);
    return tmm::plan_word(w4_gemm_shape(p.shape), p);
  }
  if (product == QMM_PRODUCT_W4_T) {
    const tmm::Plan p = tmm::plan_rows(tmm::kTilesW4, rows, E, k, n);
    return tmm::plan_word(tmm::kTilesW4[p.shape], p);
  }
  const tmm::Plan p = product == QMM_PRODUCT_RAGGED ? tmm::plan_rows(tmm::kTiles, rows, E, n, k) : tmm::plan_rows(tmm::kTiles, rows, E, k, n);
  return tmm::plan_word(tmm::kTiles[p.shape], p);
}

extern "C" int qmm_ragged_mm(int64_t rows, int64_t k, int64_t n, int E, const int32_t *offsets, const void *x, const void *w,
                             int dtype, void *y, int y_dtype, void *workspace, int64_t workspace_bytes,
                             qmm_stream_t stream) {
  const bool rest = zero_rest_asked(y_dtype);
  if (int st = check(rows, k, n, E, offsets, x, w, dtype, rows ? y : w, y_dtype)) return st;
  if (rows == 0) return QMM_OK;
  if (takes_few_rows(rows, k, n)) {
    few::Args a{offsets, E, (int)rows, (int)n, (int)k, static_cast<const u8 *>(x), static_cast<const u8 *>(w),
                      2 * n * k, nullptr, 0, 0, y, y_dtype == QMM_F32 ? 4 : 2};
    a.rest = rest;
    return ragged_few(a, dtype == QMM_F16, reinterpret_cast<hipStream_t>(stream));
  }
  tmm::Args a{};
  a.offsets = offsets, a.E = E, a.rows = (int)rows;
  a.N = (int)n, a.K = (int)k;
  a.a = static_cast<const u8 *>(x), a.a_row = 2 * k;
  a.b = static_cast<const u8 *>(w), a.b_row = 2 * k, a.b_expert = 2 * n * k;
  return tiles(kRaggedY, a, tmm::plan_rows(tmm::kTiles, rows, E, n, k), rows * n, dtype, y_dtype, rest, y, workspace, workspace_bytes, stream);
}

extern "C" int qmm_ragged_mm_t(int64_t rows, int64_t k, int64_t n, int E, const int32_t *offsets, const void *dy, const void *w,
                               int dtype, void *dx, int dx_dtype, void *workspace, int64_t workspace_bytes,
                               qmm_stream_t stream) {
  const bool rest = zero_rest_asked(dx_dtype);
  if (int st = check(rows, k, n, E, offsets, dy, w, dtype, rows ? dx : w, dx_dtype)) return st;
  if (rows == 0) return QMM_OK;
  tmm::Args a{};
  a.offsets = offsets, a.E = E, a.rows = (int)rows;
  a.N = (int)k, a.K = (int)n;
  a.a = static_cast<const u8 *>(dy), a.a_row = 2 * n;
  a.b = static_cast<const u8 *>(w), a.b_row = 2 * k, a.b_expert = 2 * n * k;
  return tiles(kRaggedDX, a, tmm::plan_rows(tmm::kTiles, rows, E, k, n), rows * k, dtype, dx_dtype, rest, dx, workspace, workspace_bytes, stream);
}

extern "C" int qmm_ragged_mm_dw(int64_t rows, int64_t k, int64_t n, int E, const int32_t *offsets, const void *dy,
                                const void *x, int dtype, void *dw, int dw_dtype, void *workspace,
                                int64_t workspace_bytes, qmm_stream_t stream) {
  if (int st = check(rows, k, n, E, offsets, dy, x, dtype, dw, dw_dtype)) return st;
  tmm::Args a{};
  a.offsets = offsets, a.E = E, a.rows = (int)rows;
  a.M = (int)n, a.N = (int)k;
  a.a = static_cast<const u8 *>(dy), a.a_row = 2 * n;
  a.b = static_cast<const u8 *>(x), a.b_row = 2 * k;
  // past the last-level cache's 256 MB dW is written by whole lines that are not kept there: us on one card in turn, 8000 rows of 128
  // experts 768 x 2048 into f32 192 without and 144, 16384 rows of 32 experts 2880 x 2880 into bf16 373 and 355
  const int64_t row = k * (dw_dtype == QMM_F32 ? 4 : 2);
  const tmm::Plan plan = tmm::plan_sum(rows, E, n, k);
  a.stream = plan.splits == 1 && row % 128 == 0 && aligned(dw, 128) && E * n * row > (int64_t)256 << 20;
  return tiles(kRaggedDW, a, plan, E * n * k, dtype, dw_dtype, false, dw, workspace, workspace_bytes, stream);
}
