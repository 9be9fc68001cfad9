// The tile kernels of products of every format (fused_tiles.h), a file of their own for the compiler's sake.
#include "fused_tiles.h"

namespace ha {
namespace {

template <int BITS, bool ASYM>
hipError_t launch(const FusedArgs& p, int rt, int ct, int halves, hipStream_t s) {
  if (halves == 2) return rt == 2 && ct == 1 ? launch_tiles<BITS, ASYM, kEpiAct, 2, 1, 2>(p, s) : hipErrorInvalidValue;
  switch (4 * rt + ct) {
    case 9: return launch_tiles<BITS, ASYM, kEpiAct, 2, 1>(p, s);
    case 10: return launch_tiles<BITS, ASYM, kEpiAct, 2, 2>(p, s);
    case 13: return launch_tiles<BITS, ASYM, kEpiAct, 3, 1>(p, s);
    case 17: return launch_tiles<BITS, ASYM, kEpiAct, 4, 1>(p, s);
  }
  if constexpr (!ASYM) {
    if (rt == 3 && ct == 2) return launch_tiles<BITS, ASYM, kEpiAct, 3, 2>(p, s);
    if (rt == 4 && ct == 2) return launch_tiles<BITS, ASYM, kEpiAct, 4, 2>(p, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_fused_tiles(const FusedArgs& p, int rt, int ct, int halves, hipStream_t s) {
  switch (2 * p.bits + (p.asym ? 1 : 0)) {
    case 4: return launch<2, false>(p, rt, ct, halves, s);
    case 5: return launch<2, true>(p, rt, ct, halves, s);
    case 6: return launch<3, false>(p, rt, ct, halves, s);
    case 7: return launch<3, true>(p, rt, ct, halves, s);
    case 8: return launch<4, false>(p, rt, ct, halves, s);
    case 9: return launch<4, true>(p, rt, ct, halves, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace ha
