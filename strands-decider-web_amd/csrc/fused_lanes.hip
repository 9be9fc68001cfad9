// The lanes kernels of every format (fused_lanes.h).
#include "fused_lanes.h"

namespace ha {

hipError_t launch_fused_lanes(const FusedArgs& p, hipStream_t s) {
  switch (2 * p.bits + (p.asym ? 1 : 0)) {
    case 4: return launch_lanes<2, false>(p, s);
    case 5: return launch_lanes<2, true>(p, s);
    case 6: return launch_lanes<3, false>(p, s);
    case 7: return launch_lanes<3, true>(p, s);
    case 8: return launch_lanes<4, false>(p, s);
    case 9: return launch_lanes<4, true>(p, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace ha
