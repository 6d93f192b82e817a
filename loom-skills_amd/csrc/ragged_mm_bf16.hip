// The ragged products' tiles (tile_mm.hpp) in bf16.
#include "ragged_mm.hpp"

namespace qmm {
int ragged_tiles_bf16(int op, const tmm::Args &a, hipStream_t s) { return ragged_tiles<QMM_BF16>(op, a, s); }
}  // namespace qmm
