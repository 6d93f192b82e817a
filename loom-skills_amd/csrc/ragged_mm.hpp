// The ragged products of 16-bit weights: a translation unit a type (ragged_mm_bf16.hip, ragged_mm_f16.hip).
#pragma once
#include "few_rows.hpp"
#include "tile_mm.hpp"

namespace qmm {

enum RaggedOp { kRaggedY = 0, kRaggedDX = 1, kRaggedDW = 2 };
int ragged_tiles_bf16(int op, const tmm::Args &a, hipStream_t s);
int ragged_tiles_f16(int op, const tmm::Args &a, hipStream_t s);
int ragged_few(const few::Args &a, bool f16, hipStream_t s);

template <int DT>
int ragged_tiles(int op, const tmm::Args &a, hipStream_t s) {
  using namespace tmm;
  if (op == kRaggedY) return launch_chosen<DT, kRow, kRow, 4>(a, s);
  if (op == kRaggedDX) return launch_chosen<DT, kRow, kCol, 4>(a, s);
  // the weights' gradient writes E n k values, however few rows there are: the larger tile reads less for them (16384 rows of 32
  // experts 2880 x 2880: 380 against 462 us, 8000 of 128 768 x 2048: 190 against 218), unless the matrix does not fill it
  if (std::min(a.M, a.N) > 128) return launch<DT, kCol, kCol, kSumRagged, 256, 256, 2, 4, 4>(a, s);
  return launch<DT, kCol, kCol, kSumRagged, 128, 128, 2, 2, 4>(a, s);
}

}  // namespace qmm
