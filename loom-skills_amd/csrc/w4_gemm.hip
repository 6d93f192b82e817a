// Many rows times 4-bit weights with group scales: the f16 operand's product on the tiles of tile_mm.hpp.
#include "w4_mm.hpp"

namespace qmm {
using namespace tmm;

namespace {
template <int GS>
int pick(const Args &a, hipStream_t s) {
  const int avg = a.offsets ? (a.rows + a.E - 1) / a.E : a.rows;
  if (avg >= 192) return launch<QMM_F16, kRow, kW4Row, kSumFixed, 256, 256, 2, 4, GS>(a, s);
  if (avg > 64) return launch<QMM_F16, kRow, kW4Row, kSumFixed, 128, 128, 2, 2, GS>(a, s);
  return launch<QMM_F16, kRow, kW4Row, kSumFixed, 64, 128, 1, 4, GS>(a, s);
}
}  // namespace

int w4_gemm(const Args &a, int gs, hipStream_t s) { return gs == 1 ? pick<1>(a, s) : pick<2>(a, s); }

}  // namespace qmm
