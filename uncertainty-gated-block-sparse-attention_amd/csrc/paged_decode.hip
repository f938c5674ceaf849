// Paged decode attention (paged_decode.h): the 16-bit and e4m3 instances, and the calls.
#include "paged_decode.h"

namespace ugbsa {

// The pieces, their (m, l), then starts [groups + 2] int32.
int64_t paged_decode_ws_elems(int B, int H, int Hk, int D, int kind, int units) {
  if (paged_decode_one(D, kind, units)) return 0;
  const int64_t pieces = 2 * static_cast<int64_t>(paged_decode_workgroups(B, H, Hk, D, kind, units)) * pd_heads(D);
  return pieces * (D + 2) + static_cast<int64_t>(B) * Hk + 2;
}

hipError_t launch_paged_decode_16(UGBSA_PD_ARGS) {
  if (c.kind == kPagesE4m3) {
    UGBSA_PD_KIND(kPagesE4m3, false)
  } else {
    UGBSA_PD_KIND(kPagesModel, false)
  }
  return hipErrorInvalidValue;
}

hipError_t launch_paged_decode(const PagedCache& c, const uint16_t* q, int64_t sq_b, int64_t sq_h,
                               int B, int H, const int32_t* lens, const int32_t* table, int64_t st_b,
                               int max_pages, const int32_t* kv_idx, const int32_t* counts, int k_slots,
                               float scale, uint16_t* out, int64_t so_b, int64_t so_h, float* ws,
                               hipStream_t stream) {
  const PagedRows rows{lens, table, st_b, max_pages, kv_idx, counts, k_slots};
  const auto launch = c.kind == kPagesE2m1 ? launch_paged_decode_e2m1 : launch_paged_decode_16;
  return launch(c, rows, q, sq_b, sq_h, B, H, scale, out, so_b, so_h, ws, PagedScores{}, stream);
}

}  // namespace ugbsa
