// Few rows times 4-bit weights with group scales (few_rows.hpp).
#include "w4_mm.hpp"

namespace qmm {

int w4_few(const few::Args &a, bool x_f32, int gs, hipStream_t s) {
  if (gs == 1) return x_f32 ? few::launch_tt<few::kW4, true, 1>(a, s) : few::launch_tt<few::kW4, false, 1>(a, s);
  if (gs == 2) return x_f32 ? few::launch_tt<few::kW4, true, 2>(a, s) : few::launch_tt<few::kW4, false, 2>(a, s);
  return x_f32 ? few::launch_tt<few::kW4, true, 4>(a, s) : few::launch_tt<few::kW4, false, 4>(a, s);
}

}  // namespace qmm
