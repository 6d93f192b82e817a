// The 4-bit products' launchers, a translation unit each (w4_few.hip, w4_gemm.hip, w4_gemm_t.hip). Arguments are checked.
#pragma once
#include "few_rows.hpp"
#include "tile_mm.hpp"

namespace qmm {
int w4_few(const few::Args &a, bool x_f32, int gs, hipStream_t s);
const tmm::Shape &w4_gemm_shape(int shape);
tmm::Plan w4_gemm_plan(int64_t rows, int E, int64_t N, int64_t K);
int w4_gemm(const tmm::Args &a, int shape, int gs, hipStream_t s);
int w4_gemm_t(const tmm::Args &a, int shape, int gs, hipStream_t s);
}  // namespace qmm
