// Records of logits (launch_logit_records of fused.hip) of every format: up to 16 rows by the stream kernel
// (fused_stream.h), more by tiles (fused_tiles.h).
#include "fused_plan.h"
#include "fused_stream.h"
#include "fused_tiles.h"

namespace ha {
namespace {

template <int BITS, bool ASYM>
hipError_t launch(const FusedArgs& p, hipStream_t s) {
  if (stream_takes(p)) return launch_stream<BITS, ASYM>(p, s);
  const fused::Plan plan = fused::logit_tiles(p.M, ASYM);
  switch (4 * plan.a + plan.b) {
    case 5: return launch_tiles<BITS, ASYM, kEpiLogits, 1, 1>(p, s);
    case 9: return launch_tiles<BITS, ASYM, kEpiLogits, 2, 1>(p, s);
    case 13: return launch_tiles<BITS, ASYM, kEpiLogits, 3, 1>(p, s);
    case 17: return launch_tiles<BITS, ASYM, kEpiLogits, 4, 1>(p, s);
  }
  if constexpr (!ASYM) return launch_tiles<BITS, ASYM, kEpiLogits, 4, 2>(p, s);
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_logit_tiles(const FusedArgs& p, hipStream_t s) {
  switch (2 * p.bits + (p.asym ? 1 : 0)) {
    case 4: return launch<2, false>(p, s);
    case 5: return launch<2, true>(p, s);
    case 6: return launch<3, false>(p, s);
    case 7: return launch<3, true>(p, s);
    case 8: return launch<4, false>(p, s);
    case 9: return launch<4, true>(p, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace ha
