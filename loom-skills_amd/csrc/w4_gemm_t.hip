// The transposed product of 4-bit weights with group scales, an input gradient, on the tiles of tile_mm.hpp.
#include "w4_mm.hpp"

namespace qmm {
using namespace tmm;

int w4_gemm_t(const Args &a, int shape, int gs, hipStream_t s) {
  if (gs == 1) return launch_shape<QMM_F16, kRow, kW4Col, 1>(a, shape, s);
  return gs == 2 ? launch_shape<QMM_F16, kRow, kW4Col, 2>(a, shape, s) : launch_shape<QMM_F16, kRow, kW4Col, 4>(a, shape, s);
}

}  // namespace qmm
