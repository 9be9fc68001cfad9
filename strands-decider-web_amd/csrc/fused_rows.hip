// The rows kernels of every format (fused_rows.h), a file of their own for the compiler's sake.
#include "fused_rows.h"

namespace ha {
namespace {

template <int BITS, bool ASYM>
hipError_t launch(const FusedArgs& p, int mt, int nt, hipStream_t s) {
  switch (8 * mt + nt) {
    case 9: return fused::rows_waves(p.M, p.K, 1, 1) == 16 ? launch_rows_as<BITS, ASYM, 1, 1, 16>(p, s) : launch_rows_as<BITS, ASYM, 1, 1, 8>(p, s);
    case 10: return launch_rows_as<BITS, ASYM, 1, 2, 8>(p, s);
    case 11: return launch_rows_as<BITS, ASYM, 1, 3, 8>(p, s);
    case 12: return launch_rows_as<BITS, ASYM, 1, 4, 8>(p, s);
    case 17: return launch_rows_as<BITS, ASYM, 2, 1, 8>(p, s);
    case 18: return launch_rows_as<BITS, ASYM, 2, 2, 8>(p, s);
    case 19: return launch_rows_as<BITS, ASYM, 2, 3, 8>(p, s);
    case 20: return launch_rows_as<BITS, ASYM, 2, 4, 8>(p, s);
    case 33: return launch_rows_as<BITS, ASYM, 4, 1, 8>(p, s);
    case 34: return launch_rows_as<BITS, ASYM, 4, 2, 8>(p, s);
    case 35: return launch_rows_as<BITS, ASYM, 4, 3, 8>(p, s);
    case 36: return launch_rows_as<BITS, ASYM, 4, 4, 8>(p, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_fused_rows(const FusedArgs& p, int mt, int nt, hipStream_t s) {
  switch (2 * p.bits + (p.asym ? 1 : 0)) {
    case 4: return launch<2, false>(p, mt, nt, s);
    case 5: return launch<2, true>(p, mt, nt, s);
    case 6: return launch<3, false>(p, mt, nt, s);
    case 7: return launch<3, true>(p, mt, nt, s);
    case 8: return launch<4, false>(p, mt, nt, s);
    case 9: return launch<4, true>(p, mt, nt, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace ha
