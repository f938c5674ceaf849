// Paged decode attention: one query row per head over the pages of its sequence,
// all of them or those of a list per KV head (paged.h has the cache's layout).
//
// The products are decode.hip's: a wavefront takes 32-key steps (half pages) and
// computes S^T = K . Q^T and O^T += V^T . P^T on 16x16x32 MFMAs with the KV
// head's query heads as the columns, K and V straight from the pages into operand
// registers.  e4m3 pages are widened there, times their tokens' scales, which is
// exact in either 16-bit format.
#include "paged.h"

namespace ugbsa {

constexpr int kPdWaves = 4;       // wavefronts per workgroup
constexpr int kPdStep = 32;       // keys per wavefront step: half a page
// Query heads per workgroup: the 16 MFMA columns; 8 at head_dim 256, where the
// wavefronts' O of 16 heads would take 66 KiB of LDS.
__host__ __device__ constexpr int pd_heads(int D) { return D > 128 ? 8 : 16; }

// The row's pages a list or the block table names.
struct PagedRows {
  const int32_t* lens;
  const int32_t* table;
  int64_t st_b;
  int max_pages;
  const int32_t* kv_idx;    // [B, Hk, k_slots] or null: all pages
  const int32_t* counts;    // [B, Hk] or null: k_slots each
  int k_slots;
};

// Pages (or list entries) of row (b, h).
__device__ __forceinline__ int row_units(const PagedRows& r, int Hk, int b, int h, int len) {
  if (r.kv_idx == nullptr) return (len + kBlock - 1) / kBlock;
  if (len == 0) return 0;
  const int n = r.counts == nullptr ? r.k_slots : r.counts[static_cast<int64_t>(b) * Hk + h];
  return min(max(n, 0), r.k_slots);
}

template <typename E, int D, bool F8>
__global__ __launch_bounds__(64 * kPdWaves) void paged_decode_kernel(
    PagedCache c, PagedRows rows, const uint16_t* __restrict__ q, int64_t sq_b, int64_t sq_h, int grp,
    int chunks, int splits, float scale_log2, uint16_t* __restrict__ out, int64_t so_b, int64_t so_h,
    float* __restrict__ part, float* __restrict__ ml) {
  constexpr int KS = D / 32, DT = D / 16, NH = pd_heads(D);
  constexpr int DPL = D / 16;                    // dims a lane loads per key of V
  // 16-bit rows are read 8 dims a load, or 4 at head_dim 64 (VW = dims a load)
  constexpr int VW = F8 ? DPL : (D == 64 ? 4 : 8), VL = DPL / VW;
  __shared__ float s_o[kPdWaves][NH][D + 4];
  __shared__ float s_ml[kPdWaves][NH][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g4 = lane >> 4, r16 = lane & 15;
  const int split = blockIdx.x, ck = blockIdx.y % chunks, g = blockIdx.y / chunks, b = blockIdx.z;
  const int heads = min(NH, grp - ck * NH);   // live columns
  const int h0 = g * grp + ck * NH;

  const int len = cached_len(rows.lens, b, rows.max_pages);
  const int units = row_units(rows, c.Hk, b, g, len);
  const int per = (units + splits - 1) / splits;
  const int u0 = min(units, split * per), u1 = min(units, u0 + per);
  const int32_t* table = rows.table + b * rows.st_b;
  const int32_t* list = rows.kv_idx == nullptr
                            ? nullptr
                            : rows.kv_idx + (static_cast<int64_t>(b) * c.Hk + g) * rows.k_slots;

  // Q^T columns (heads past the group are zero and never written).  Contraction
  // slot 8 g4 + i of step ks is dim 32 ks + 8 g4 + i; e4m3 rows, 16 codes a load,
  // take dim 64 (ks / 2) + 16 g4 + 8 (ks % 2) + i.
  bf16x8 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int d = F8 ? 64 * (ks / 2) + 16 * g4 + 8 * (ks % 2) : 32 * ks + 8 * g4;
    qf[ks] = r16 < heads ? load_bf16x8(q + b * sq_b + (h0 + r16) * sq_h + d) : zero_bf16x8();
  }
  // MFMA row R of S^T tile mt is key 8 (R >> 2) + 4 mt + (R & 3) of the step:
  // the lane then holds keys 8 g4 + 4 mt + i
  const int krow = 8 * (r16 >> 2) + (r16 & 3);

  // step st of the row: the half page's keys, how many of them exist, its page
  struct Step { int64_t page; int base, left; };
  auto step_at = [&](int st) {
    const int u = st >> 1;
    const int blk = list == nullptr ? u : list[u];
    int page = -1;
    if (blk >= 0 && blk < rows.max_pages && blk * kBlock < len) page = table[blk];
    const bool there = page >= 0 && page < c.num_pages;
    Step s;
    s.page = there ? page : 0;               // an absent page: page 0's keys, none of them live
    s.base = kPdStep * (st & 1);
    s.left = there ? len - blk * kBlock - s.base : 0;
    return s;
  };

  u32x4 kf[2][F8 ? KS / 2 : KS];
  float ksc[2], vsc[8];
  uint32_t vr[8][F8 ? DPL / 4 : DPL / 2];    // V[8 g4 + i][the lane's dims]
  auto load_k = [&](const Step& s) {
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const int slot = s.base + krow + 4 * mt;
      const int64_t at = s.page * c.sk_p + g * c.sk_h + slot * c.sk_n;
      if constexpr (F8) {
        const uint8_t* row = static_cast<const uint8_t*>(c.k) + at + 16 * g4;
#pragma unroll
        for (int j = 0; j < KS / 2; ++j) kf[mt][j] = *reinterpret_cast<const u32x4*>(row + 64 * j);
        ksc[mt] = e8m0(c.k_scale[(s.page * c.Hk + g) * kBlock + slot]);
      } else {
        const uint16_t* row = static_cast<const uint16_t*>(c.k) + at + 8 * g4;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kf[mt][ks] = *reinterpret_cast<const u32x4*>(row + 32 * ks);
      }
    }
  };
  auto load_v = [&](const Step& s) {
    if constexpr (F8) {
      const u32x2 sc = *reinterpret_cast<const u32x2*>(
          c.v_scale + (s.page * c.Hk + g) * kBlock + s.base + 8 * g4);
#pragma unroll
      for (int i = 0; i < 8; ++i) vsc[i] = e8m0((sc[i / 4] >> (8 * (i % 4))) & 0xFFu);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t at = s.page * c.sv_p + g * c.sv_h + (s.base + 8 * g4 + i) * c.sv_n + VW * r16;
      if constexpr (F8) {
        const uint8_t* row = static_cast<const uint8_t*>(c.v) + at;
        if constexpr (DPL == 4) {
          vr[i][0] = *reinterpret_cast<const uint32_t*>(row);
        } else if constexpr (DPL == 8) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(row);
          vr[i][0] = x[0], vr[i][1] = x[1];
        } else {
          const u32x4 x = *reinterpret_cast<const u32x4*>(row);
#pragma unroll
          for (int j = 0; j < 4; ++j) vr[i][j] = x[j];
        }
      } else {
        const uint16_t* row = static_cast<const uint16_t*>(c.v) + at;
#pragma unroll
        for (int l = 0; l < VL; ++l) {
          if constexpr (VW == 8) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(row + 128 * l);
#pragma unroll
            for (int j = 0; j < 4; ++j) vr[i][4 * l + j] = x[j];
          } else {
            const u32x2 x = *reinterpret_cast<const u32x2*>(row);
            vr[i][0] = x[0], vr[i][1] = x[1];
          }
        }
      }
    }
  };

  f32x4 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;    // of head r16; l over this lane's keys

  const int st1 = 2 * u1;
  int st = 2 * u0 + wave;
  Step cur{}, nxt{};
  if (st < st1) {
    cur = step_at(st);
    load_k(cur);
    load_v(cur);
  }
  for (; st < st1; st += kPdWaves) {
    const bool more = st + kPdWaves < st1;
    if (more) nxt = step_at(st + kPdWaves);
    f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        bf16x8 a;
        if constexpr (F8)
          a = e4m3_x8<E>(kf[mt][ks / 2][2 * (ks % 2)], kf[mt][ks / 2][2 * (ks % 2) + 1], ksc[mt]);
        else
          a = __builtin_bit_cast(bf16x8, kf[mt][ks]);
        s[mt] = E::mfma(a, qf[ks], s[mt]);
      }
    if (more) load_k(nxt);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = s[e >> 2][e & 3] * scale_log2;
    if (cur.left < kPdStep) {       // keys past the end, or an absent page
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * g4 + e >= cur.left) {
          x[e] = -INFINITY;
          if constexpr (F8) vsc[e] = 1.f;
#pragma unroll
          for (int j = 0; j < (F8 ? DPL / 4 : DPL / 2); ++j) vr[e][j] = 0u;
        }
    }
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
    const float m_new = fmaxf(m, quad_rows_max(mx));
    const float off = m_new == -INFINITY ? 0.f : m_new;   // no finite score so far: weights 0
    const float alpha = __builtin_amdgcn_exp2f(m - off);
    m = m_new;
    float p[8], sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = __builtin_amdgcn_exp2f(x[e] - off);
      sum += p[e];
    }
    l = l * alpha + sum;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
    // P rounded once to the element format, as the other attention kernels do
    u32x4 pw;
#pragma unroll
    for (int j = 0; j < 4; ++j) pw[j] = E::pack2(p[2 * j], p[2 * j + 1]);
    const bf16x8 pb = __builtin_bit_cast(bf16x8, pw);
    // operand dt: the lane's dim dt of the eight keys
#pragma unroll
    for (int d2 = 0; d2 < DT / 2; ++d2) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (F8) w[i] = e4m3_pair<E>(vr[i][d2 / 2], vsc[i], d2 % 2);
        else w[i] = vr[i][d2];
      }
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        u32x4 a;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          a[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], odd ? 0x07060302u : 0x05040100u);
        o[2 * d2 + odd] = E::mfma(__builtin_bit_cast(bf16x8, a), pb, o[2 * d2 + odd]);
      }
    }
    if (more) load_v(nxt);
    cur = nxt;
  }
  l = quad_rows_sum(l);

  // O^T row R = 4 g4 + i of operand dt is dim VW R + dt % VW of load dt / VW
  // (128 dims a load)
  if (r16 < heads) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s_o[wave][r16][128 * (dt / VW) + VW * (4 * g4 + i) + dt % VW] = o[dt][i];
    if (g4 == 0) {
      s_ml[wave][r16][0] = m;
      s_ml[wave][r16][1] = l;
    }
  }
  __syncthreads();

  const int H = c.Hk * grp;
  for (int i = threadIdx.x; i < heads * D; i += 64 * kPdWaves) {
    const int hh = i / D, d = i % D;
    float mm = s_ml[0][hh][0];
#pragma unroll
    for (int w = 1; w < kPdWaves; ++w) mm = fmaxf(mm, s_ml[w][hh][0]);
    const float off = mm == -INFINITY ? 0.f : mm;
    float acc = 0.f, ll = 0.f;
#pragma unroll
    for (int w = 0; w < kPdWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(s_ml[w][hh][0] - off);
      acc += s_o[w][hh][d] * f;
      ll += s_ml[w][hh][1] * f;
    }
    const int64_t bh = static_cast<int64_t>(b) * H + h0 + hh;
    if (splits == 1) {
      // no key at all: zeros
      out[b * so_b + (h0 + hh) * so_h + d] =
          static_cast<uint16_t>(E::pack2(ll == 0.f ? 0.f : acc / ll, 0.f) & 0xFFFFu);
    } else {
      part[(bh * splits + split) * D + d] = acc;
      if (d == 0) {
        ml[(bh * splits + split) * 2] = mm;
        ml[(bh * splits + split) * 2 + 1] = ll;
      }
    }
  }
}

// out of one (b, head) from its splits.
constexpr int kPdMaxSplits = 512;
template <typename E, int D>
__global__ __launch_bounds__(256) void paged_combine_kernel(const float* __restrict__ part,
                                                            const float* __restrict__ ml, int H,
                                                            int splits, uint16_t* __restrict__ out,
                                                            int64_t so_b, int64_t so_h) {
  __shared__ float s_w[kPdMaxSplits];
  const int64_t bh = blockIdx.x;
  const float* mlb = ml + bh * splits * 2;
  float mx = -INFINITY;
  for (int s = 0; s < splits; ++s) mx = fmaxf(mx, mlb[2 * s]);
  const float off = mx == -INFINITY ? 0.f : mx;
  for (int s = threadIdx.x; s < splits; s += 256) s_w[s] = __builtin_amdgcn_exp2f(mlb[2 * s] - off);
  __syncthreads();
  float total = 0.f;
  for (int s = 0; s < splits; ++s) total += mlb[2 * s + 1] * s_w[s];
  for (int d = threadIdx.x; d < D; d += 256) {
    float acc = 0.f;
    for (int s = 0; s < splits; ++s) acc += part[(bh * splits + s) * D + d] * s_w[s];
    out[(bh / H) * so_b + (bh % H) * so_h + d] =
        static_cast<uint16_t>(E::pack2(total == 0.f ? 0.f : acc / total, 0.f) & 0xFFFFu);
  }
}

// Splits of each row's pages: enough workgroups that every CU holds two, each
// with a page a wavefront pair.
int paged_decode_splits(int B, int H, int Hk, int D, int units) {
  const int64_t rows = static_cast<int64_t>(B) * Hk * ((H / Hk + pd_heads(D) - 1) / pd_heads(D));
  int64_t want = 512 / rows;
  if (want > units / 2) want = units / 2;
  if (want > kPdMaxSplits) want = kPdMaxSplits;
  return want < 1 ? 1 : static_cast<int>(want);
}

template <typename E, int D, bool F8>
static hipError_t launch_paged_decode_t(const PagedCache& c, const PagedRows& rows, const uint16_t* q,
                                        int64_t sq_b, int64_t sq_h, int B, int H, float scale,
                                        uint16_t* out, int64_t so_b, int64_t so_h, float* ws,
                                        hipStream_t stream) {
  const int grp = H / c.Hk, chunks = (grp + pd_heads(D) - 1) / pd_heads(D);
  const int splits = paged_decode_splits(B, H, c.Hk, D, rows.kv_idx ? rows.k_slots : rows.max_pages);
  float* part = ws;
  float* ml = ws + static_cast<int64_t>(B) * H * splits * D;
  paged_decode_kernel<E, D, F8><<<dim3(splits, c.Hk * chunks, B), 64 * kPdWaves, 0, stream>>>(
      c, rows, q, sq_b, sq_h, grp, chunks, splits, scale * kLog2e, out, so_b, so_h, part, ml);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || splits == 1) return e;
  paged_combine_kernel<E, D><<<dim3(B * H), 256, 0, stream>>>(part, ml, H, splits, out, so_b, so_h);
  return hipGetLastError();
}

hipError_t launch_paged_decode(const PagedCache& c, const uint16_t* q, int64_t sq_b, int64_t sq_h,
                               int B, int H, const int32_t* lens, const int32_t* table, int64_t st_b,
                               int max_pages, const int32_t* kv_idx, const int32_t* counts, int k_slots,
                               float scale, uint16_t* out, int64_t so_b, int64_t so_h, float* ws,
                               hipStream_t stream) {
  const PagedRows rows{lens, table, st_b, max_pages, kv_idx, counts, k_slots};
#define UGBSA_PD(E_, D_)                                                                            \
  return c.e4m3 ? launch_paged_decode_t<E_, D_, true>(c, rows, q, sq_b, sq_h, B, H, scale, out, so_b, \
                                                      so_h, ws, stream)                              \
                : launch_paged_decode_t<E_, D_, false>(c, rows, q, sq_b, sq_h, B, H, scale, out,      \
                                                       so_b, so_h, ws, stream)
  if (c.elem == ElemF16::code) {
    if (c.D == 64) UGBSA_PD(ElemF16, 64);
    if (c.D == 128) UGBSA_PD(ElemF16, 128);
    if (c.D == 256) UGBSA_PD(ElemF16, 256);
  } else {
    if (c.D == 64) UGBSA_PD(ElemBf16, 64);
    if (c.D == 128) UGBSA_PD(ElemBf16, 128);
    if (c.D == 256) UGBSA_PD(ElemBf16, 256);
  }
#undef UGBSA_PD
  return hipErrorInvalidValue;
}

}  // namespace ugbsa
