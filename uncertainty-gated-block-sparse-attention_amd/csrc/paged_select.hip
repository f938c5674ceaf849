// Page selection for one new token: per (sequence, KV head) the pages its query
// heads attend to, by the Quest score over the pages' K-max / K-min planes.
//
//   s_j   = max over the KV head's query heads h of
//           sum_d (q_hd >= 0 ? q_hd kmax_jd : q_hd kmin_jd)
//   kept  = the first and the last page, and of the others the best by
//           (s desc, page asc) up to k_base pages in all, k_slots where the cut is
//           uncertain: sigma < tau, sigma = clamp((s(k') - s(k' + 1)) /
//           max(s(1) - s(k' + 1), 1e-9), 0, 2) over the others' scores times
//           scaling, s(i) the i-th best, k' = k_base - 2; 2 where nothing is cut.
//
// The list decides whole pages, so near ties matter: scores are summed in fp64,
// where the 16-bit products are exact and sums of them round far below any
// spacing of theirs.
#include "paged.h"

namespace ugbsa {

// Monotone uint64 key of an fp64 score (larger score, larger key; NaN above
// +inf; -0 as +0; never 0 for a competing page).
__device__ __forceinline__ uint64_t double_key(double x) {
  if (x != x) return ~0ull;
  x += 0.0;
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return (u >> 63) ? ~u : (u | (1ull << 63));
}
__device__ __forceinline__ double key_double(uint64_t k) {
  if (k == ~0ull) return __builtin_bit_cast(double, 0x7FF8000000000000ull);
  return __builtin_bit_cast(double, (k >> 63) ? (k ^ (1ull << 63)) : ~k);
}

// keys [B, Hk, max_pages] of the pages between the first and the last of each row:
// one wavefront a page, D / 64 dims a lane.
template <typename E, int D>
__global__ __launch_bounds__(256) void paged_score_kernel(
    PagedCache c, const uint16_t* __restrict__ q, int64_t sq_b, int64_t sq_h, int grp,
    const int32_t* __restrict__ lens, const int32_t* __restrict__ table, int64_t st_b, int max_pages,
    uint64_t* __restrict__ keys) {
  constexpr int L = D / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = blockIdx.y, b = blockIdx.z;
  const int nb = (cached_len(lens, b, max_pages) + kBlock - 1) / kBlock;
  const uint16_t* qb = q + b * sq_b + g * grp * sq_h + L * lane;
  const int64_t row = static_cast<int64_t>(b) * c.Hk + g;
  for (int j = blockIdx.x * 4 + wave; j < nb - 1; j += gridDim.x * 4) {
    if (j == 0) continue;
    const int page = table[b * st_b + j];
    double best = -INFINITY;
    if (page >= 0 && page < c.num_pages) {
      const uint16_t* pl = c.planes + (static_cast<int64_t>(page) * c.Hk + g) * 2 * D + L * lane;
      double hi[L], lo[L];
#pragma unroll
      for (int i = 0; i < L; ++i) hi[i] = E::to_f32(pl[i]), lo[i] = E::to_f32(pl[D + i]);
      for (int h = 0; h < grp; ++h) {
        double acc = 0.0;
#pragma unroll
        for (int i = 0; i < L; ++i) {
          const float x = E::to_f32(qb[h * sq_h + i]);
          acc += static_cast<double>(x) * (x >= 0.f ? hi[i] : lo[i]);
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) acc += __shfl_xor(acc, off, 64);
        best = (acc > best || acc != acc) ? acc : best;
      }
    }
    if (lane == 0) keys[row * max_pages + j] = double_key(best);
  }
}

// Sum over the workgroup (every thread gets it); red: 4 ints.
__device__ __forceinline__ int wg_sum(int x, int* red) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}
__device__ __forceinline__ uint64_t wg_max(uint64_t x, uint64_t* red) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const uint64_t y = __shfl_xor(static_cast<unsigned long long>(x), off, 64);
    x = y > x ? y : x;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  uint64_t a = red[0] > red[1] ? red[0] : red[1], z = red[2] > red[3] ? red[2] : red[3];
  return a > z ? a : z;
}

// One workgroup per row: cut, margin, gate and the ascending list.
__global__ __launch_bounds__(256) void paged_pick_kernel(
    const uint64_t* __restrict__ keys, const int32_t* __restrict__ lens, int Hk, int max_pages,
    float scaling, int k_base, int k_slots, float tau, int32_t* __restrict__ kv_idx,
    int32_t* __restrict__ counts, float* __restrict__ sigma, uint8_t* __restrict__ uncertain) {
  __shared__ int hist[256];
  __shared__ int red[4];
  __shared__ uint64_t red64[4];
  __shared__ uint64_t s_prefix;
  __shared__ int s_left;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int b = static_cast<int>(row / Hk);
  const int nb = (cached_len(lens, b, max_pages) + kBlock - 1) / kBlock;
  const uint64_t* kr = keys + row * max_pages;
  int32_t* list = kv_idx + row * k_slots;

  // the k-th largest key of pages 1 .. nb - 2 (1 <= k <= nb - 2): digit by digit
  auto kth = [&](int k) {
    uint64_t prefix = 0;
    int left = k;
    for (int shift = 56; shift >= 0; shift -= 8) {
      __syncthreads();
      hist[tid] = 0;
      __syncthreads();
      for (int j = 1 + tid; j < nb - 1; j += 256) {
        const uint64_t x = kr[j];
        if (shift == 56 || (x >> (shift + 8)) == (prefix >> (shift + 8)))
          atomicAdd(&hist[(x >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int d = 255;
        while (hist[d] < left) left -= hist[d--];
        s_prefix = prefix | (static_cast<uint64_t>(d) << shift);
        s_left = left;
      }
      __syncthreads();
      prefix = s_prefix;
      left = s_left;
    }
    return prefix;
  };

  float sg = 2.f;
  bool unsure = false;
  uint64_t cut = 0;
  int keep = min(k_base, nb);
  if (nb > k_base) {
    const int k = k_base - 2;
    const uint64_t a = kth(k);
    int not_below = 0;
    uint64_t below = 0, top = 0;
    for (int j = 1 + tid; j < nb - 1; j += 256) {
      const uint64_t x = kr[j];
      if (x >= a) ++not_below;
      else if (x > below) below = x;
      if (x > top) top = x;
    }
    const uint64_t next = wg_sum(not_below, red) > k ? a : 0;
    below = wg_max(below, red64);
    top = wg_max(top, red64);
    const double sc = scaling, c = key_double(next ? next : below) * sc;
    const double reach = key_double(top) * sc - c, ratio = (key_double(a) * sc - c) / (reach > 1e-9 ? reach : 1e-9);
    const double clamped = ratio < 0.0 ? 0.0 : (ratio > 2.0 ? 2.0 : ratio);
    sg = static_cast<float>(clamped);
    unsure = clamped < static_cast<double>(tau);
    cut = a;
    if (unsure) {
      keep = min(k_slots, nb);
      if (nb > keep) cut = kth(keep - 2);
    }
  }
  // pages above the cut, and the lowest of those at it
  int above = 0;
  if (nb > keep) {
    for (int j = 1 + tid; j < nb - 1; j += 256) above += kr[j] > cut;
    above = wg_sum(above, red);
  }
  const int ties = keep - 2 - above;
  int ties_before = 0, out_before = 0;
  for (int j0 = 0; j0 < nb; j0 += 256) {
    const int j = j0 + tid;
    bool in = j < nb, tie = false;
    if (in && nb > keep && j > 0 && j < nb - 1) {
      const uint64_t x = kr[j];
      in = x > cut;
      tie = x == cut;
    }
    // ranks over the workgroup, ties first
    for (int pass = 0; pass < 2; ++pass) {
      const uint64_t bal = __ballot(pass == 0 ? tie : in);
      __syncthreads();
      if ((tid & 63) == 0) red[tid >> 6] = __popcll(bal);
      __syncthreads();
      int rank = lanes_below(bal), all = 0;
      for (int w = 0; w < 4; ++w) {
        if (w < (tid >> 6)) rank += red[w];
        all += red[w];
      }
      if (pass == 0) {
        if (tie) in = ties_before + rank < ties;
        ties_before += all;
      } else {
        if (in) list[out_before + rank] = j;
        out_before += all;
      }
    }
  }
  for (int s = keep + tid; s < k_slots; s += 256) list[s] = max_pages;
  if (tid == 0) {
    counts[row] = keep;
    if (sigma != nullptr) sigma[row] = sg;
    if (uncertain != nullptr) uncertain[row] = unsure ? 1 : 0;
  }
}

template <typename E, int D>
static hipError_t launch_paged_select_t(const PagedCache& c, const uint16_t* q, int64_t sq_b,
                                        int64_t sq_h, int B, int H, const int32_t* lens,
                                        const int32_t* table, int64_t st_b, int max_pages, float scaling,
                                        int k_base, int k_slots, float tau, int32_t* kv_idx,
                                        int32_t* counts, float* sigma, uint8_t* uncertain, uint64_t* keys,
                                        hipStream_t stream) {
  const dim3 grid(min((max_pages + 3) / 4, 256), c.Hk, B);
  paged_score_kernel<E, D><<<grid, 256, 0, stream>>>(c, q, sq_b, sq_h, H / c.Hk, lens, table, st_b,
                                                     max_pages, keys);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  paged_pick_kernel<<<dim3(B * c.Hk), 256, 0, stream>>>(keys, lens, c.Hk, max_pages, scaling, k_base,
                                                        k_slots, tau, kv_idx, counts, sigma, uncertain);
  return hipGetLastError();
}

hipError_t launch_paged_select(const PagedCache& c, const uint16_t* q, int64_t sq_b, int64_t sq_h, int B,
                               int H, const int32_t* lens, const int32_t* table, int64_t st_b,
                               int max_pages, float scaling, int k_base, int k_slots, float tau,
                               int32_t* kv_idx, int32_t* counts, float* sigma, uint8_t* uncertain,
                               uint64_t* keys, hipStream_t stream) {
#define UGBSA_PS(E_, D_)                                                                              \
  return launch_paged_select_t<E_, D_>(c, q, sq_b, sq_h, B, H, lens, table, st_b, max_pages, scaling, \
                                       k_base, k_slots, tau, kv_idx, counts, sigma, uncertain, keys,  \
                                       stream)
  if (c.elem == ElemF16::code) {
    if (c.D == 64) UGBSA_PS(ElemF16, 64);
    if (c.D == 128) UGBSA_PS(ElemF16, 128);
    if (c.D == 256) UGBSA_PS(ElemF16, 256);
  } else {
    if (c.D == 64) UGBSA_PS(ElemBf16, 64);
    if (c.D == 128) UGBSA_PS(ElemBf16, 128);
    if (c.D == 256) UGBSA_PS(ElemBf16, 256);
  }
#undef UGBSA_PS
  return hipErrorInvalidValue;
}

}  // namespace ugbsa
