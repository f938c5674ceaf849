// Paged decode attention (paged_decode.h) whose weights are followed: each cached token
// of a KV head gets the sum over its query heads of the weight that the token had,
//
//   mass[b, g, i] += sum over the heads h of g of exp2(x_hi - m_h) / l_h.
//
// A weight is known when its row's maximum and sum are, so the attention launch leaves
// its scaled scores (4 bytes a query head and token) and the rows' statistics, and a third
// launch adds them up, in the heads' order and without atomics: a sequence has its own row.
#include "paged_decode.h"

namespace ugbsa {

// Four tokens (of a page or list entry) per thread, over the heads of a KV head.
__global__ __launch_bounds__(256) void paged_mass_kernel(PagedRows rows, int Hk, int grp, PagedScores sc,
                                                         float* __restrict__ mass, int64_t sm_b, int64_t sm_h) {
  const int g = blockIdx.y, b = blockIdx.z;
  const int i = 4 * (blockIdx.x * 256 + threadIdx.x), unit = i / kBlock;
  const int len = cached_len(rows.lens, b, rows.max_pages);
  int n = rows.max_pages;
  if (rows.kv_idx != nullptr) {
    n = rows.counts == nullptr ? rows.k_slots : rows.counts[b * Hk + g];
    n = min(n, rows.k_slots);
  }
  if (len == 0 || unit >= n) return;
  const int blk =
      rows.kv_idx == nullptr ? unit : rows.kv_idx[(static_cast<int64_t>(b) * Hk + g) * rows.k_slots + unit];
  if (blk < 0 || blk >= rows.max_pages) return;
  const int tok = blk * kBlock + i % kBlock;
  if (tok >= len) return;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  const int64_t row0 = (static_cast<int64_t>(b) * Hk + g) * grp;
#pragma unroll 4
  for (int h = 0; h < grp; ++h) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(sc.x + (row0 + h) * sc.units * kBlock + i);
    const float m = sc.ml[2 * (row0 + h)], l = sc.ml[2 * (row0 + h) + 1];
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      sum[j] += x[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x[j] - m) * inv;   // no key: no weight
  }
  float* to = mass + b * sm_b + g * sm_h + tok;
  f32x4 old = *reinterpret_cast<const f32x4*>(to);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (tok + j < len) old[j] += sum[j];
  *reinterpret_cast<f32x4*>(to) = old;
}

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

hipError_t launch_paged_mass(const PagedCache& c, const uint16_t* q, int64_t sq_b, int64_t sq_h, int B, int H,
                             const int32_t* lens, const int32_t* table, int64_t st_b, int max_pages,
                             const int32_t* kv_idx, const int32_t* counts, int k_slots, float scale, float* mass,
                             int64_t sm_b, int64_t sm_h, uint16_t* out, int64_t so_b, int64_t so_h, float* ws,
                             hipStream_t stream) {
  const PagedRows rows{lens, table, st_b, max_pages, kv_idx, counts, k_slots};
  const int units = kv_idx != nullptr ? k_slots : max_pages;
  float* ml = ws + decode_elems(B, H, c.Hk, c.D, c.kind, units);
  const PagedScores sc{ml + (2 * static_cast<int64_t>(B) * H + 3) / 4 * 4, ml, units};
  const hipError_t e = launch_paged_decode_mass(c, rows, q, sq_b, sq_h, B, H, scale, out, so_b, so_h, ws, sc, stream);
  if (e != hipSuccess) return e;
  paged_mass_kernel<<<dim3((units + 15) / 16, c.Hk, B), 256, 0, stream>>>(rows, c.Hk, H / c.Hk, sc, mass, sm_b, sm_h);
  return hipGetLastError();
}

}  // namespace ugbsa
