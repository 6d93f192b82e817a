// The ragged products' tiles (tile_mm.hpp) in f16.
#include "ragged_mm.hpp"

namespace qmm {
int ragged_tiles_f16(int op, const tmm::Args &a, int shape, hipStream_t s) { return ragged_tiles<QMM_F16>(op, a, shape, s); }
}  // namespace qmm
