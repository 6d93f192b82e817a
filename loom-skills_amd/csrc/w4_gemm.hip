// Many rows times 4-bit weights with group scales: the f16 operand's product on the tiles of tile_mm.hpp.
#include "w4_mm.hpp"

namespace qmm {
using namespace tmm;

int w4_gemm(const Args &a, int gs, hipStream_t s) { return gs == 1 ? launch_chosen<QMM_F16, kRow, kW4Row, 1>(a, s) : launch_chosen<QMM_F16, kRow, kW4Row, 2>(a, s); }

}  // namespace qmm
