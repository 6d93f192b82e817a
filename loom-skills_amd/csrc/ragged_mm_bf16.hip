// The ragged products' tiles (tile_mm.hpp) in bf16.
#include "ragged_mm.hpp"

namespace qmm {
int ragged_tiles_bf16(int op, const tmm::Args &a, int shape, hipStream_t s) { return ragged_tiles<QMM_BF16>(op, a, shape, s); }
}  // namespace qmm
