// Paged decode attention (paged_decode.h) over e2m1 pages.
#include "paged_decode.h"

namespace ugbsa {

hipError_t launch_paged_decode_e2m1(UGBSA_PD_ARGS) {
  UGBSA_PD_KIND(kPagesE2m1, false)
  return hipErrorInvalidValue;
}

}  // namespace ugbsa
