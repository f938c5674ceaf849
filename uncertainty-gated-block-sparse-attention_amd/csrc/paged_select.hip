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
// where the 16-bit products are exact and a sum rounds at 2^-53 of the terms that the
// score consists of; the bound that a dim does not take has no part in it, however
// large it is.
//
// 64 sequences of up to 128K tokens, 40/8 heads (119 MB of planes): scoring 49 us,
// picking 11.3; one of 32K, 28/4 heads, 4.0 and 6.5.
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

template <int CTRL>
__device__ __forceinline__ double dpp_add(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const int lo = static_cast<int>(u), hi = static_cast<int>(u >> 32);
  const uint32_t l = static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(lo, CTRL, 0xF, 0xF, true));
  const uint32_t h = static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(hi, CTRL, 0xF, 0xF, true));
  return x + __builtin_bit_cast(double, static_cast<uint64_t>(h) << 32 | l);
}
// Sum over groups of LP = 8, 16 or 32 lanes in the VALU (every lane gets it): lanes
// xor 1 and 2, the mirrored half row, the mirrored row, the neighbouring row.
template <int LP>
__device__ __forceinline__ double group_sum(double x) {
  x = dpp_add<0xB1>(x);
  x = dpp_add<0x4E>(x);
  x = dpp_add<0x141>(x);
  if constexpr (LP >= 16) x = dpp_add<0x140>(x);
  if constexpr (LP >= 32) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const auto l = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(u), static_cast<uint32_t>(u), false, false);
    const auto h = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(u >> 32), static_cast<uint32_t>(u >> 32), false, false);
    x = __builtin_bit_cast(double, static_cast<uint64_t>(h[0]) << 32 | l[0]) +
        __builtin_bit_cast(double, static_cast<uint64_t>(h[1]) << 32 | l[1]);
  }
  return x;
}

// fp64 of a 16-bit value: its lower word is 0, so the upper one stands for it.
template <typename E>
__device__ __forceinline__ uint32_t double_top(uint32_t x) {
  return static_cast<uint32_t>(__builtin_bit_cast(uint64_t, static_cast<double>(E::to_f32(x))) >> 32);
}

constexpr int kScoreAhead = 2;          // steps of a wavefront whose loads are in flight

// keys [B, Hk, max_pages] of the pages between the first and the last of each row.
//
// D / 8 lanes take a page, 8 dims each, so a wavefront reads 64 / (D / 8) pages' whole
// planes per step, two 16-byte loads a lane, and converts them to fp64 once for the GC
// heads of a pass, whose q stay in registers as fp64: per dim and head a select by the
// sign of q and an fp64 FMA, which runs at the fp32 rate here.
template <typename E, int D, int GC>
__global__ __launch_bounds__(256) void paged_score_kernel(
    PagedCache c, const uint16_t* __restrict__ q, int64_t sq_b, int64_t sq_h, int grp,
    const int32_t* __restrict__ lens, const int32_t* __restrict__ table, int64_t st_b, int max_pages,
    int per_wave, uint64_t* __restrict__ keys) {
  constexpr int LP = D / 8, NP = 64 / LP;        // lanes a page, pages a step
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = blockIdx.x % c.Hk, b = blockIdx.y;   // a page's heads run side by side
  const int nb = (cached_len(lens, b, max_pages) + kBlock - 1) / kBlock;
  // this wavefront's pages [j0, j1), at most the 64 whose table entries its lanes hold
  const int j0 = (blockIdx.x / c.Hk * 4 + wave) * per_wave, j1 = min(j0 + per_wave, nb);
  if (j0 >= j1) return;
  const int sub = lane / LP, d0 = 8 * (lane % LP);
  const int mine = j0 + lane < j1 ? table[b * st_b + j0 + lane] : -1;
  uint64_t* kr = keys + (static_cast<int64_t>(b) * c.Hk + g) * max_pages;

  u32x4 his[kScoreAhead], los[kScoreAhead];
  int pages[kScoreAhead];
  auto load = [&](int j, u32x4& hi, u32x4& lo, int& page) {
    page = __shfl(mine, j - j0 + sub, 64);
    if (j + sub >= j1 || page < 0 || page >= c.num_pages) page = -1;
    const uint16_t* pl = c.planes + (static_cast<int64_t>(max(page, 0)) * c.Hk + g) * 2 * D + d0;
    hi = *reinterpret_cast<const u32x4*>(pl);
    lo = *reinterpret_cast<const u32x4*>(pl + D);
  };
  for (int h0 = 0; h0 < grp; h0 += GC) {
    double qd[GC][8];
    const uint16_t* qh = q + b * sq_b + (g * grp + h0) * sq_h;
#pragma unroll
    for (int h = 0; h < GC; ++h) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(qh + min(h, grp - 1 - h0) * sq_h + d0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        qd[h][2 * i] = E::to_f32(x[i] & 0xFFFFu);
        qd[h][2 * i + 1] = E::to_f32(x[i] >> 16);
      }
    }
    // the steps in flight: step s of a round of kScoreAhead in registers of its own
#pragma unroll
    for (int s = 0; s < kScoreAhead; ++s)
      if (j0 + s * NP < j1) load(j0 + s * NP, his[s], los[s], pages[s]);
    for (int jr = j0; jr < j1; jr += kScoreAhead * NP) {
      static_for<kScoreAhead>([&](auto sc) {
        constexpr int s = sc;
        const int j = jr + s * NP;
        if (j >= j1) return;
        const u32x4 hi = his[s], lo = los[s];
        const int at = pages[s];
        uint32_t top[8], low[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          top[2 * i] = double_top<E>(hi[i] & 0xFFFFu), low[2 * i] = double_top<E>(lo[i] & 0xFFFFu);
          top[2 * i + 1] = double_top<E>(hi[i] >> 16), low[2 * i + 1] = double_top<E>(lo[i] >> 16);
        }
        const int ahead = j + kScoreAhead * NP;
        if (ahead < j1) load(ahead, his[s], los[s], pages[s]);
        // Past five heads the selects' masks do not fit the SGPRs (and their spills cost 8
        // sequences of up to 64K tokens 3 to 7 % of both launches): a 0 that the compiler does
        // not know keeps the compares with the selects.
        double zero = 0.0;
        if constexpr (GC > 5) asm volatile("s_mov_b64 %0, 0" : "=s"(zero));
        double best = -INFINITY;
#pragma unroll
        for (int h = 0; h < GC; ++h) {
          double acc = 0.0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t w = qd[h][i] >= zero ? top[i] : low[i];
            acc = __builtin_fma(qd[h][i], __builtin_bit_cast(double, static_cast<uint64_t>(w) << 32), acc);
          }
          acc = group_sum<LP>(acc);
          best = acc > best || acc != acc ? acc : best;        // NaN stays
        }
        if (lane % LP != 0 || j + sub >= j1) return;
        if (at < 0) best = -INFINITY;
        uint64_t key = double_key(best);
        if (h0 > 0) {                                // the earlier heads' best, by this lane
          const uint64_t before = kr[j + sub];
          key = before > key ? before : key;
        }
        kr[j + sub] = key;
      });
    }
  }
}

constexpr int kPickKeys = 8;            // keys a thread holds in registers

// One workgroup of NT threads per row: cut, margin, gate and the ascending list.
// REG: rows of up to 8 NT pages, whose keys stay in registers.
//
// The k-th largest key: the keys between the row's extremes go into 4 NT bins of
// equal width, the bin that holds rank k is found by a scan over the bins, and its
// few keys are ranked against each other; a bin of more than NT is binned again.
// Bins relative to the extremes matter: the digits of the keys as they stand share
// their sign and most of the exponent.
template <int NT, bool REG>
__global__ __launch_bounds__(NT) void paged_pick_kernel(
    const uint64_t* __restrict__ keys, const int32_t* __restrict__ lens, int Hk, int max_pages,
    float scaling, int k_base, int k_slots, float tau, int32_t* __restrict__ kv_idx,
    int32_t* __restrict__ counts, float* __restrict__ sigma, uint8_t* __restrict__ uncertain) {
  constexpr int kBits = 31 - __builtin_clz(4 * NT);
  __shared__ int hist[4 * NT];
  __shared__ uint64_t cand[NT];
  __shared__ uint64_t s_max[NT / 64], s_min[NT / 64];
  __shared__ int s_cnt[NT / 64], s_cnt2[NT / 64];
  __shared__ uint64_t s_kth;
  __shared__ int s_bin, s_left, s_in, s_cands;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const int b = static_cast<int>(row / Hk);
  const int nb = (cached_len(lens, b, max_pages) + kBlock - 1) / kBlock;
  const uint64_t* kr = keys + row * max_pages;
  int32_t* list = kv_idx + row * k_slots;
  int keep = min(k_base, nb);
  float sg = 2.f;
  bool unsure = false;

  // thread t has pages [t chunk, (t + 1) chunk); key 0: no competitor
  const int chunk = (nb + NT - 1) / NT, j0 = tid * chunk;
  auto read = [&](int i) -> uint64_t {
    const int j = j0 + i;
    return i < chunk && j > 0 && j < nb - 1 ? kr[j] : 0;
  };
  uint64_t held[kPickKeys];
  if (REG && nb > k_base) {
#pragma unroll
    for (int i = 0; i < kPickKeys; ++i) held[i] = read(i);
  }
  auto each = [&](auto&& f) {
    if constexpr (REG) {
#pragma unroll
      for (int i = 0; i < kPickKeys; ++i)
        if (i < chunk) f(i, held[i]);
    } else {
      for (int i = 0; i < chunk; ++i) f(i, read(i));
    }
  };
  // maximum and (of the nonzero keys) minimum over the workgroup, and a count
  auto reduce = [&](uint64_t mx, uint64_t mn, int n, uint64_t& all_mx, uint64_t& all_mn, int& all_n) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
      const uint64_t a = __shfl_xor(static_cast<unsigned long long>(mx), off, 64);
      const uint64_t z = __shfl_xor(static_cast<unsigned long long>(mn), off, 64);
      mx = a > mx ? a : mx;
      mn = z < mn ? z : mn;
      n += __shfl_xor(n, off, 64);
    }
    __syncthreads();
    if (lane == 0) s_max[wave] = mx, s_min[wave] = mn, s_cnt[wave] = n;
    __syncthreads();
    all_mx = 0, all_mn = ~0ull, all_n = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
      all_mx = s_max[w] > all_mx ? s_max[w] : all_mx;
      all_mn = s_min[w] < all_mn ? s_min[w] : all_mn;
      all_n += s_cnt[w];
    }
  };
  auto kth = [&](int left, uint64_t lo, uint64_t hi) -> uint64_t {
    for (;;) {
      if (lo == hi) return lo;
      const int width = 64 - __builtin_clzll(hi - lo);
      const int shift = width > kBits ? width - kBits : 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) hist[NT * i + tid] = 0;
      if (tid == 0) s_cands = 0;
      __syncthreads();
      each([&](int, uint64_t x) {
        if (x >= lo && x <= hi) atomicAdd(&hist[(x - lo) >> shift], 1);
      });
      __syncthreads();
      // thread t: the four bins below 4 NT - 4 t, an inclusive scan from the top
      const int top = 4 * NT - 1 - 4 * tid;
      int n[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += n[i] = hist[top - i];
      int incl = sum;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int y = __shfl_up(incl, off, 64);
        if (lane >= off) incl += y;
      }
      if (lane == 63) s_cnt[wave] = incl;
      __syncthreads();
      for (int w = 0; w < wave; ++w) incl += s_cnt[w];
      if (incl - sum < left && left <= incl) {       // exactly one thread
        int before = incl - sum, i = 0;
        while (before + n[i] < left) before += n[i++];
        s_bin = top - i;
        s_left = left - before;
        s_in = n[i];
      }
      __syncthreads();
      lo += static_cast<uint64_t>(s_bin) << shift;
      // the topmost bin may reach past hi, and past 2^64 where hi is NaN's or +inf's key
      const uint64_t span = (1ull << shift) - 1;
      hi = hi - lo < span ? hi : lo + span;
      left = s_left;
      if (shift == 0) return lo;
      if (s_in <= NT) break;
    }
    each([&](int, uint64_t x) {
      if (x >= lo && x <= hi) cand[atomicAdd(&s_cands, 1)] = x;
    });
    __syncthreads();
    const int m = s_cands;
    if (tid < m) {
      const uint64_t x = cand[tid];
      int above = 0, same = 0;
      for (int i = 0; i < m; ++i) above += cand[i] > x, same += cand[i] == x;
      if (above < left && left <= above + same) s_kth = x;     // equal keys write the same
    }
    __syncthreads();
    return s_kth;
  };

  uint64_t cut = 0;
  if (nb > k_base) {
    uint64_t mx = 0, mn = ~0ull, top, low, unused;
    int n = 0, all;
    each([&](int, uint64_t x) {
      mx = x > mx ? x : mx;
      if (x != 0 && x < mn) mn = x;
    });
    reduce(mx, mn, 0, top, low, all);
    const int k = k_base - 2;
    const uint64_t a = kth(k, low, top);
    mx = 0;
    each([&](int, uint64_t x) {
      n += x >= a;
      if (x < a && x > mx) mx = x;
    });
    uint64_t below;
    reduce(mx, ~0ull, n, below, unused, all);
    const double sc = scaling, c = key_double(all > k ? a : below) * sc;
    const double reach = key_double(top) * sc - c;         // NaN stays NaN
    const double ratio = (key_double(a) * sc - c) / (reach < 1e-9 ? 1e-9 : reach);
    const double clamped = ratio < 0.0 ? 0.0 : (ratio > 2.0 ? 2.0 : ratio);
    sg = static_cast<float>(clamped);
    unsure = clamped < static_cast<double>(tau);
    cut = a;
    if (unsure) {
      keep = min(k_slots, nb);
      if (nb > keep && keep > k_base) cut = kth(keep - 2, low, top);
    }
  }
  if (nb <= keep) {
    for (int s = tid; s < k_slots; s += NT) list[s] = s < nb ? s : max_pages;
  } else {
    // kept: the first and the last page, those above the cut, and the lowest of
    // those at it; a page's place is what is kept of the pages before it
    int over = 0, ties = 0;
    auto forced = [&](int i) { return j0 + i == 0 || j0 + i == nb - 1; };
    each([&](int i, uint64_t x) {
      if (j0 + i >= nb) return;
      over += forced(i) || x > cut;
      ties += !forced(i) && x == cut;
    });
    int o = over, e = ties;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int y = __shfl_up(o, off, 64), z = __shfl_up(e, off, 64);
      if (lane >= off) o += y, e += z;
    }
    __syncthreads();
    if (lane == 63) s_cnt[wave] = o, s_cnt2[wave] = e;
    __syncthreads();
    int all_over = 0;
    for (int w = 0; w < NT / 64; ++w) {
      if (w < wave) o += s_cnt[w], e += s_cnt2[w];
      all_over += s_cnt[w];
    }
    o -= over, e -= ties;
    const int room = keep - all_over;
    each([&](int i, uint64_t x) {
      if (j0 + i >= nb) return;
      const bool tie = !forced(i) && x == cut;
      const int at = o + min(e, room);
      if ((forced(i) || x > cut || (tie && e < room)) && static_cast<uint32_t>(at) < static_cast<uint32_t>(keep))
        list[at] = j0 + i;
      o += forced(i) || x > cut;
      e += tie;
    });
    for (int s = keep + tid; s < k_slots; s += NT) list[s] = max_pages;
  }
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
  // no row is cut where the budget holds the table's width: nothing to score (one
  // sequence of 64 pages 17.6 -> 13.0 us a call, host included)
  const bool scored = max_pages > k_base;
  // heads a pass: an even share of the group, at most the 8 whose q fit the registers
  const int grp = H / c.Hk, passes = (grp + 7) / 8, gc = (grp + passes - 1) / passes;
  // pages a wavefront: as many as leave the card 4096 wavefronts, from one step to
  // 24 (64 sequences of up to 128K tokens, 40/8 heads, this launch: 16 / 24 / 32 pages
  // 56.2 / 49.4 / 59.9 us at two wavefronts per SIMD)
  constexpr int NP = 512 / D;
  const int64_t pages = static_cast<int64_t>(B) * c.Hk * max_pages;
  int per = static_cast<int>(pages / 4096 < 24 ? pages / 4096 : 24) / NP * NP;
  if (per < NP) per = NP;
  const dim3 grid((max_pages + 4 * per - 1) / (4 * per) * c.Hk, B);
#define UGBSA_SCORE(GC_)                                                                          \
  paged_score_kernel<E, D, GC_><<<grid, 256, 0, stream>>>(c, q, sq_b, sq_h, grp, lens, table, st_b, \
                                                          max_pages, per, keys)
  if (scored) {
    if (gc == 1) UGBSA_SCORE(1);
    else if (gc == 2) UGBSA_SCORE(2);
    else if (gc <= 4) UGBSA_SCORE(4);
    else if (gc == 5) UGBSA_SCORE(5);
    else if (gc <= 7) UGBSA_SCORE(7);
    else UGBSA_SCORE(8);
  }
#undef UGBSA_SCORE
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // few threads for few keys, where barriers cost more than steps (one sequence of 512
  // pages, both launches: 64 / 128 / 256 / 512 threads 12.2 / 11.3 / 11.3 / 12.4 us)
#define UGBSA_PICK(NT_, REG_)                                                                         \
  paged_pick_kernel<NT_, REG_><<<dim3(B * c.Hk), NT_, 0, stream>>>(keys, lens, c.Hk, max_pages, scaling, \
                                                                   k_base, k_slots, tau, kv_idx, counts, \
                                                                   sigma, uncertain)
  if (max_pages <= 128 * kPickKeys) UGBSA_PICK(128, true);
  else if (max_pages <= 256 * kPickKeys) UGBSA_PICK(256, true);
  else if (max_pages <= 512 * kPickKeys) UGBSA_PICK(512, true);
  else UGBSA_PICK(512, false);
#undef UGBSA_PICK
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
