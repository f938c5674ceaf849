// Paged decode attention whose weights are followed: the MASS instances (paged_decode.h).
#include "paged_decode.h"

namespace ugbsa {

hipError_t launch_paged_decode_mass(UGBSA_PD_ARGS) {
  if (c.kind == kPagesE4m3) {
    UGBSA_PD_KIND(kPagesE4m3, true)
  } else if (c.kind == kPagesE2m1) {
    UGBSA_PD_KIND(kPagesE2m1, true)
  } else {
    UGBSA_PD_KIND(kPagesModel, true)
  }
  return hipErrorInvalidValue;
}

// The attention's own, then the rows' statistics and the scores (16-byte aligned).
static int64_t decode_elems(int B, int H, int Hk, int D, int kind, int units) {
  return (paged_decode_ws_elems(B, H, Hk, D, kind, units) + 3) / 4 * 4;
}
int64_t paged_mass_ws_elems(int B, int H, int Hk, int D, int kind, int units) {
  const int64_t rows = static_cast<int64_t>(B) * H;
  return decode_elems(B, H, Hk, D, kind, units) + (2 * rows + 3) / 4 * 4 + rows * units * kBlock;
}

bool paged_mass_fits(int B, int H, int Hk, int D, int kind, int units) {
  return paged_decode_one(D, kind, units) || paged_finish(B, H, Hk, units).grid < 1 << 24;
}

hipError_t launch_paged_mass(const PagedCache& c, const uint16_t* q, int64_t sq_b, int64_t sq_h, int B, int H,
                             const int32_t* lens, const int32_t* table, int64_t st_b, int max_pages,
                             const int32_t* kv_idx, const int32_t* counts, int k_slots, float scale, float* mass,
                             int64_t sm_b, int64_t sm_h, uint16_t* out, int64_t so_b, int64_t so_h, float* ws,
                             hipStream_t stream) {
  const PagedRows rows{lens, table, st_b, max_pages, kv_idx, counts, k_slots};
  const int units = kv_idx != nullptr ? k_slots : max_pages;
  float* ml = ws + decode_elems(B, H, c.Hk, c.D, c.kind, units);
  const PagedScores sc{ml + (2 * static_cast<int64_t>(B) * H + 3) / 4 * 4, ml, units, mass, sm_b, sm_h};
  return launch_paged_decode_mass(c, rows, q, sq_b, sq_h, B, H, scale, out, so_b, so_h, ws, sc, stream);
}

}  // namespace ugbsa
