// The ragged products of 16-bit weights: a translation unit a type (ragged_mm_bf16.hip, ragged_mm_f16.hip).
#pragma once
#include "few_rows.hpp"
#include "tile_mm.hpp"

namespace qmm {

enum RaggedOp { kRaggedY = 0, kRaggedDX = 1, kRaggedDW = 2 };
int ragged_tiles_bf16(int op, const tmm::Args &a, int shape, hipStream_t s);
int ragged_tiles_f16(int op, const tmm::Args &a, int shape, hipStream_t s);
int ragged_few(const few::Args &a, bool f16, hipStream_t s);

template <int DT>
int ragged_tiles(int op, const tmm::Args &a, int shape, hipStream_t s) {
  using namespace tmm;
  if (op == kRaggedY) return launch_shape<DT, kRow, kRow, 4>(a, shape, s);
  if (op == kRaggedDX) return launch_shape<DT, kRow, kCol, 4>(a, shape, s);
  if (shape == 0) return launch<DT, kCol, kCol, kSumRagged, 256, 256, 2, 4, 4>(a, s);
  if (shape == 2) return launch<DT, kCol, kCol, kSumRagged, 128, 128, 2, 4, 4, 4>(a, s);
  return launch<DT, kCol, kCol, kSumRagged, 128, 128, 2, 2, 4>(a, s);
}

}  // namespace qmm
