// Paged decode attention: one query row per head over the pages of its sequence,
// all of them or those of a list per KV head (paged.h has the cache's layout).
//
// The products are decode.hip's: a wavefront takes 32-key steps (half pages) and
// computes S^T = K . Q^T and O^T += V^T . P^T on 16x16x32 MFMAs with the KV
// head's query heads as the columns, K and V straight from the pages into operand
// registers.  e4m3 pages are widened there, times their tokens' scales, which is
// exact in either 16-bit format.
//
// Bound by memory: 32 sequences of 64K tokens, 40/8 heads, e4m3 (4.3 GB) 698 us, 6.2
// TB/s; 24 of up to 16K, bf16 (375 MB) 69.5 us, 5.4 TB/s with the joining launch; one of
// 1000 tokens 11 us, two launches of about 4 us.
#include "paged.h"

namespace ugbsa {

constexpr int kPdWaves = 4;       // wavefronts per workgroup
constexpr int kPdStep = 32;       // keys per wavefront step: half a page

// Four dims of a head, over their weights' sum; a row without a key, or whose every
// weight is 0, gives zeros.
template <typename E>
__device__ __forceinline__ void store4(uint16_t* to, f32x4 x, float sum) {
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = sum == 0.f ? 0.f : x[j] / sum;
  reinterpret_cast<uint32_t*>(to)[0] = E::pack2(x[0], x[1]);
  reinterpret_cast<uint32_t*>(to)[1] = E::pack2(x[2], x[3]);
}

// Query heads per workgroup: the 16 MFMA columns; 8 at head_dim 256, where the
// wavefronts' O of 16 heads would take 66 KiB of LDS.
__host__ __device__ constexpr int pd_heads(int D) { return D > 128 ? 8 : 16; }

// The pages that a call's lists or block table name.
struct PagedRows {
  const int32_t* lens;
  const int32_t* table;
  int64_t st_b;
  int max_pages;
  const int32_t* kv_idx;    // [B, Hk, k_slots] or null: all pages
  const int32_t* counts;    // [B, Hk] or null: k_slots each
  int k_slots;
};

// The work of a call is its rows' pages (or list entries), laid end to end: a group
// is a sequence, or with lists a (sequence, KV head), its members the (KV head,)
// head chunks that visit its n pages, one row each.  A row takes n + kPdRowCost
// units of the line, the first kPdRowCost for its start and end.  Workgroup w takes
// units [w per, (w + 1) per), however the batch's lengths are spread, so rows begin
// and end inside workgroups.  A row whose pages one workgroup holds is written by it;
// the pieces of the others meet in paged_combine_kernel: piece 2 w of workgroup w
// continues a row, piece 2 w + 1 begins one.
constexpr int kPdUnits = 2;       // fewest units of a workgroup: a half page a wavefront
constexpr int kPdRowCost = 3;

struct PagedGroups {
  int groups, members, Hk;
};

__device__ __forceinline__ int group_units(const PagedRows& r, int Hk, int i) {
  const int b = r.kv_idx == nullptr ? i : i / Hk;
  const int len = cached_len(r.lens, b, r.max_pages);
  if (r.kv_idx == nullptr) return (len + kBlock - 1) / kBlock;
  const int n = r.counts == nullptr ? r.k_slots : r.counts[i];
  return len == 0 ? 0 : min(max(n, 0), r.k_slots);
}
// Units of a row of n pages on the line.
__device__ __forceinline__ int row_units(int n) { return n > 0 ? n + kPdRowCost : 0; }

// Wavefronts per SIMD that the registers allow, which is also the workgroups per CU
// that a call launches: a line cut into more than are resident leaves a second round
// of them (us, 256 / 512 / 768 / 1024 workgroups: 24 sequences of up to 16K tokens,
// 40/8 heads, bf16 86.1 / 78.4 / 88.1 / 80.1; 32 x 64K in e4m3 1127 / 758 / 727 / 858; 4
// of up to 64K at 16/2 heads, head_dim 256 44.1 / 50.3 / 55.1 / 64.5).
__host__ __device__ constexpr int pd_occupancy(int D, bool F8) {
  return D == 64 ? 4 : (D == 128 ? (F8 ? 3 : 2) : (F8 ? 2 : 1));
}

// ONE: the wavefronts of a workgroup that has a row to itself, 0: workgroups on the line.
template <typename E, int D, bool F8, bool NT, int ONE>
__global__ __launch_bounds__(64 * (ONE ? ONE : kPdWaves), ONE ? 2 : pd_occupancy(D, F8)) void paged_decode_kernel(
    PagedCache c, PagedRows rows, PagedGroups gr, const uint16_t* __restrict__ q, int64_t sq_b,
    int64_t sq_h, int grp, int chunks, float scale_log2, uint16_t* __restrict__ out, int64_t so_b,
    int64_t so_h, int* __restrict__ starts, float* __restrict__ part, float* __restrict__ ml) {
  constexpr int KS = D / 32, DT = D / 16, NH = pd_heads(D);
  constexpr int DPL = D / 16;                    // dims a lane loads per key of V
  // 16-bit rows are read 8 dims a load, or 4 at head_dim 64 (VW = dims a load)
  constexpr int VW = F8 ? DPL : (D == 64 ? 4 : 8), VL = DPL / VW;
  constexpr int SZ = F8 ? 1 : 2, WAVES = ONE ? ONE : kPdWaves;
  __shared__ float s_o[WAVES][NH][D + 4];
  __shared__ float s_ml[WAVES][NH][2];
  __shared__ int s_sum[WAVES], s_start[2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g4 = lane >> 4, r16 = lane & 15;

  int group, member, n, x0, u, u_end;              // n: units of the row, x0 of them before u
  if constexpr (ONE != 0) {
    const bool lists = rows.kv_idx != nullptr;
    group = lists ? blockIdx.y * gr.Hk + blockIdx.x / chunks : blockIdx.y;
    member = lists ? blockIdx.x % chunks : blockIdx.x;
    n = row_units(__builtin_amdgcn_readfirstlane(group_units(rows, gr.Hk, group)));
    x0 = u = 0, u_end = n;
  } else {
    // The line's length, and the row where this workgroup's units begin: up to 64
    // groups lie in a wavefront's lanes, more in the workgroup's threads, some each.
    const bool few = gr.groups <= 64;
    const int each = few ? 1 : (gr.groups + 255) / 256, i0 = (few ? lane : threadIdx.x) * each;
    int mine = 0;
    for (int i = i0; i < min(i0 + each, gr.groups); ++i) mine += row_units(group_units(rows, gr.Hk, i));
    mine *= gr.members;
    int incl = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int y = __shfl_up(incl, off, 64);
      if (lane >= off) incl += y;
    }
    int total = __builtin_amdgcn_readlane(incl, 63);
    if (!few) {
      if (lane == 63) s_sum[wave] = incl;
      __syncthreads();
      total = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        if (w < wave) incl += s_sum[w];
        total += s_sum[w];
      }
    }
    const int per = max(kPdUnits, static_cast<int>((static_cast<uint32_t>(total) + gridDim.x - 1) / gridDim.x));
    if (blockIdx.x == 0 && (!few || wave == 0)) {    // for the joining kernel
      int s = incl - mine;
      for (int i = i0; i < min(i0 + each, gr.groups); ++i) {
        starts[i] = s;
        s += row_units(group_units(rows, gr.Hk, i)) * gr.members;
      }
      if (threadIdx.x == 0) starts[gr.groups] = total, starts[gr.groups + 1] = per;
    }
    if (static_cast<int64_t>(blockIdx.x) * per >= total) return;
    u = blockIdx.x * per;
    u_end = min(u + per, total);
    int off0;                                        // units of the group before u
    if (few) {
      group = __builtin_popcountll(__ballot(incl <= u));
      const int units = __builtin_amdgcn_readlane(mine, group);
      off0 = u - (__builtin_amdgcn_readlane(incl, group) - units);
      n = static_cast<int>(static_cast<uint32_t>(units) / static_cast<uint32_t>(gr.members));
    } else {
      if (incl - mine <= u && u < incl) {            // one thread
        int s = incl - mine;
        for (int i = i0;; ++i) {
          const int k = row_units(group_units(rows, gr.Hk, i)) * gr.members;
          if (u < s + k) {
            s_start[0] = i;
            s_start[1] = u - s;
            break;
          }
          s += k;
        }
      }
      __syncthreads();
      group = __builtin_amdgcn_readfirstlane(s_start[0]);
      off0 = __builtin_amdgcn_readfirstlane(s_start[1]);
      n = __builtin_amdgcn_readfirstlane(row_units(group_units(rows, gr.Hk, group)));
    }
    member = static_cast<int>(static_cast<uint32_t>(off0) / static_cast<uint32_t>(n));
    x0 = off0 - member * n;
  }

  // MFMA row R of S^T tile mt is key 8 (R >> 2) + 4 mt + (R & 3) of the step:
  // the lane then holds keys 8 g4 + 4 mt + i
  const int krow = 8 * (r16 >> 2) + (r16 & 3);
  // byte offsets of the lane's K and V rows within a step (the strides fit, checked on the host)
  const uint32_t k_lane = static_cast<uint32_t>((krow * c.sk_n + (F8 ? 16 : 8) * g4) * SZ);
  const uint32_t v_lane = static_cast<uint32_t>((8 * g4 * c.sv_n + VW * r16) * SZ);
  const uint32_t k_row = static_cast<uint32_t>(c.sk_n * SZ), v_row = static_cast<uint32_t>(c.sv_n * SZ);

  for (;;) {
    // this workgroup's units [x0, x1), and so pages [p0, p1), of row (b, g, ck)
    const int x1 = min(n, x0 + u_end - u);
    const int p0 = max(x0 - kPdRowCost, 0), p1 = max(x1 - kPdRowCost, 0), pages = n - kPdRowCost;
    const int b = rows.kv_idx == nullptr ? group : group / gr.Hk;
    const int g = rows.kv_idx == nullptr ? member / chunks : group % gr.Hk;
    const int ck = rows.kv_idx == nullptr ? member % chunks : member;
    const int heads = min(NH, grp - ck * NH);    // live columns
    const int h0 = g * grp + ck * NH;
    if (ONE && n == 0) {
      for (int i = threadIdx.x; i < heads * (D / 4); i += 64 * WAVES)
        store4<E>(out + b * so_b + (h0 + i / (D / 4)) * so_h + 4 * (i % (D / 4)), f32x4{0.f, 0.f, 0.f, 0.f}, 0.f);
      return;
    }
    const int len = cached_len(rows.lens, b, rows.max_pages);
    const int32_t* table = rows.table + b * rows.st_b;
    const int32_t* list = rows.kv_idx == nullptr
                              ? nullptr
                              : rows.kv_idx + (static_cast<int64_t>(b) * gr.Hk + g) * rows.k_slots;

    // Q^T columns (heads past the group are zero and never written).  Contraction
    // slot 8 g4 + i of step ks is dim 32 ks + 8 g4 + i; e4m3 rows, 16 codes a load,
    // take dim 64 (ks / 2) + 16 g4 + 8 (ks % 2) + i.
    bf16x8 qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = F8 ? 64 * (ks / 2) + 16 * g4 + 8 * (ks % 2) : 32 * ks + 8 * g4;
      qf[ks] = r16 < heads ? load_bf16x8(q + b * sq_b + (h0 + r16) * sq_h + d) : zero_bf16x8();
    }

    gchar* const kg = (gchar*)c.k + g * c.sk_h * SZ;
    gchar* const vg = (gchar*)c.v + g * c.sv_h * SZ;

    // step st of the row: its half page's keys, how many of them exist, its page
    struct Step { int64_t page; int base, left; };
    auto step_at = [&](int st) {
      const int x = st >> 1;
      const int blk = list == nullptr ? x : list[x];
      int page = -1;
      if (blk >= 0 && blk < rows.max_pages && blk * kBlock < len) page = table[blk];
      const bool there = page >= 0 && page < c.num_pages;
      Step s;
      s.page = there ? page : 0;             // an absent page: page 0's keys, none of them live
      s.base = kPdStep * (st & 1);
      s.left = there ? len - blk * kBlock - s.base : 0;
      return s;
    };

    u32x4 kf[2][F8 ? KS / 2 : KS];
    float ksc[2], vsc[8];
    uint32_t vr[8][F8 ? DPL / 4 : DPL / 2];  // V[8 g4 + i][the lane's dims]
    auto load_k = [&](const Step& s) {
      gchar* half = kg + s.page * c.sk_p * SZ + static_cast<uint32_t>(s.base) * k_row;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        gchar* row = half + 4u * mt * k_row;
#pragma unroll
        for (int j = 0; j < (F8 ? KS / 2 : KS); ++j)
          kf[mt][j] = stream_load<NT>(reinterpret_cast<gu32x4*>(row + (k_lane + 64u * j)));
        if constexpr (F8)
          ksc[mt] = e8m0(c.k_scale[(s.page * gr.Hk + g) * kBlock + s.base + krow + 4 * mt]);
      }
    };
    auto load_v = [&](const Step& s) {
      gchar* half = vg + s.page * c.sv_p * SZ + static_cast<uint32_t>(s.base) * v_row;
      if constexpr (F8) {
        const u32x2 sc = *reinterpret_cast<const u32x2*>(
            c.v_scale + (s.page * gr.Hk + g) * kBlock + s.base + 8 * g4);
#pragma unroll
        for (int i = 0; i < 8; ++i) vsc[i] = e8m0((sc[i / 4] >> (8 * (i % 4))) & 0xFFu);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        gchar* row = half + static_cast<uint32_t>(i) * v_row;
        constexpr int LB = VW * SZ;          // bytes of a load
#pragma unroll
        for (int l = 0; l < VL; ++l) {
          gchar* at = row + (v_lane + 256u * l);
          if constexpr (LB == 16) {
            const u32x4 x = stream_load<NT>(reinterpret_cast<gu32x4*>(at));
#pragma unroll
            for (int j = 0; j < 4; ++j) vr[i][4 * l + j] = x[j];
          } else if constexpr (LB == 8) {
            const u32x2 x = stream_load<NT>(reinterpret_cast<gu32x2*>(at));
            vr[i][0] = x[0], vr[i][1] = x[1];
          } else {
            vr[i][0] = stream_load<NT>(reinterpret_cast<gu32*>(at));
          }
        }
      }
    };

    f32x4 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;  // of head r16; l over this lane's keys

    const int st1 = 2 * p1;
    int st = 2 * p0 + wave;
    Step cur{}, nxt{}, far{};
    if (st < st1) {
      cur = step_at(st);
      load_k(cur);
      load_v(cur);
      if (st + WAVES < st1) nxt = step_at(st + WAVES);
    }
    for (; st < st1; st += WAVES) {
      const bool more = st + WAVES < st1;
      // the page after the next one's: its number is on the way during this step
      if (st + 2 * WAVES < st1) far = step_at(st + 2 * WAVES);
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
      if (cur.left < kPdStep) {     // keys past the end, or an absent page
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
      nxt = far;
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

    const bool whole = ONE || (p0 == 0 && p1 == pages);
    const int64_t piece = 2 * static_cast<int64_t>(blockIdx.x) + (p0 == 0 ? 1 : 0);
    for (int i = threadIdx.x; p0 < p1 && i < heads * (D / 4); i += 64 * WAVES) {
      const int hh = i / (D / 4), d = 4 * (i % (D / 4));
      float mm = s_ml[0][hh][0];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) mm = fmaxf(mm, s_ml[w][hh][0]);
      const float off = mm == -INFINITY ? 0.f : mm;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      float ll = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float f = __builtin_amdgcn_exp2f(s_ml[w][hh][0] - off);
        acc += *reinterpret_cast<const f32x4*>(&s_o[w][hh][d]) * f;
        ll += s_ml[w][hh][1] * f;
      }
      if (whole) {
        store4<E>(out + b * so_b + (h0 + hh) * so_h + d, acc, ll);
      } else {
        *reinterpret_cast<f32x4*>(part + (piece * NH + hh) * D + d) = acc;
        if (d == 0) {
          ml[(piece * NH + hh) * 2] = mm;
          ml[(piece * NH + hh) * 2 + 1] = ll;
        }
      }
    }

    u += x1 - x0;
    if (ONE || u >= u_end) return;
    // the next row with pages
    x0 = 0;
    if (++member == gr.members) {
      member = 0;
      for (++group;; group += 64) {
        const int k = group + lane < gr.groups ? row_units(group_units(rows, gr.Hk, group + lane)) : 0;
        const uint64_t some = __ballot(k > 0);
        if (some == 0) continue;                   // u < total: a later group has pages
        const int f = __builtin_ctzll(some);
        n = __builtin_amdgcn_readlane(k, f);
        group += f;
        break;
      }
    }
    __syncthreads();                               // s_o is read by all before it is written again
  }
}

// out of the heads whose rows several workgroups hold, and zeros for rows without
// pages: 256 threads a head, four dims each and the pieces in runs of 1024 / D.
constexpr int kPdMaxWorkgroups = 1024;
constexpr int kPdCombineThreads = 256;
template <typename E, int D>
__global__ __launch_bounds__(kPdCombineThreads) void paged_combine_kernel(
    const int* __restrict__ starts, const float* __restrict__ part, const float* __restrict__ ml,
    PagedGroups gr, int grp, int chunks, bool lists, uint16_t* __restrict__ out, int64_t so_b,
    int64_t so_h) {
  constexpr int RUNS = 4 * kPdCombineThreads / D, NH = pd_heads(D), PT = kPdMaxWorkgroups / kPdCombineThreads;
  __shared__ float s_w[kPdMaxWorkgroups];
  __shared__ float s_red[kPdCombineThreads / 64][2];
  __shared__ f32x4 s_acc[RUNS][D / 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int H = gr.Hk * grp, b = blockIdx.x / H, h = blockIdx.x % H;
  const int g = h / grp, ck = h % grp / NH, hh = h % grp % NH;
  const int group = lists ? b * gr.Hk + g : b, member = lists ? ck : g * chunks + ck;
  const uint32_t s0 = starts[group], s1 = starts[group + 1], per = starts[gr.groups + 1];
  const uint32_t n = (s1 - s0) / static_cast<uint32_t>(gr.members), first = s0 + member * n;
  uint16_t* o = out + b * so_b + h * so_h;
  if (n == 0) {
    if (tid < D) o[tid] = 0;
    return;
  }
  const int wa = static_cast<int>((first + kPdRowCost) / per);
  const int pieces = static_cast<int>((first + n - 1) / per) - wa + 1;
  if (pieces == 1) return;
  auto at = [&](int i) { return (2 * (wa + i) + (i == 0 ? 1 : 0)) * NH + hh; };
  float ms[PT], ls[PT], mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    const int x = kPdCombineThreads * i + tid;
    ms[i] = x < pieces ? ml[2 * at(x)] : -INFINITY;
    ls[i] = x < pieces ? ml[2 * at(x) + 1] : 0.f;
    mx = fmaxf(mx, ms[i]);
  }
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) mx = fmaxf(mx, __shfl_xor(mx, s, 64));
  if (lane == 0) s_red[wave][0] = mx;
  __syncthreads();
  mx = s_red[0][0];
#pragma unroll
  for (int w = 1; w < kPdCombineThreads / 64; ++w) mx = fmaxf(mx, s_red[w][0]);
  const float off = mx == -INFINITY ? 0.f : mx;
  float lt = 0.f;
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    const float w = __builtin_amdgcn_exp2f(ms[i] - off);
    if (kPdCombineThreads * i + tid < pieces) s_w[kPdCombineThreads * i + tid] = w;
    lt += ls[i] * w;
  }
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) lt += __shfl_xor(lt, s, 64);
  if (lane == 0) s_red[wave][1] = lt;
  __syncthreads();
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < kPdCombineThreads / 64; ++w) total += s_red[w][1];

  const int run = tid / (D / 4), d4 = tid % (D / 4);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = run; i < pieces; i += RUNS)
    acc += reinterpret_cast<const f32x4*>(part + static_cast<int64_t>(at(i)) * D)[d4] * s_w[i];
  s_acc[run][d4] = acc;
  __syncthreads();
  if (tid < D / 4) {
#pragma unroll
    for (int r = 1; r < RUNS; ++r) acc += s_acc[r][tid];
    store4<E>(o + 4 * tid, acc, total);
  }
}

// Whether each row gets a workgroup to itself, with no line to find and nothing to
// join: where a row's K and V are at most 256 KB, which one CU streams (about 25 bytes a
// clock) in what the joining launch costs.  us, this form / the line: 512 tokens, 28/4
// heads, head_dim 128, bf16, 1 sequence 9.1 / 10.5, 128 sequences 15.9 / 22.3; 1024
// tokens in e4m3 (256 KB) 10.8 / 11.0 and 19.1 / 23.3, in bf16 (512 KB) 13.3 / 10.8 and
// 23.6 / 26.8: past 256 KB one row is slower this way and many rows are faster.  The rule
// goes by a row's bytes alone and takes the line there.
//
// The bytes are those that the table's width admits; the lengths are on the device.  24
// sequences of 500 tokens, 40/8 heads, in a table of 8 / 256 / 2048 pages: bf16 12.5 / 21.3
// / 21.2 us, e4m3 8.5 / 16.2 / 16.9.
//
// At head_dim 256 in 16 bits this form's instances spill 44 bytes a lane at the two
// wavefronts per SIMD that they are bound to.
static bool paged_decode_one(int D, bool e4m3, int units) {
  return static_cast<int64_t>(units) * (2 * kBlock * D * (e4m3 ? 1 : 2)) <= 256 << 10;
}

// Workgroups of a call: as many as the card holds at once, unless the call's rows
// cannot have kPdUnits for each.
static int paged_decode_workgroups(int B, int H, int Hk, int D, bool e4m3, int units) {
  const int64_t rows = static_cast<int64_t>(B) * Hk * ((H / Hk + pd_heads(D) - 1) / pd_heads(D));
  const int64_t most = (rows * (units + kPdRowCost) + kPdUnits - 1) / kPdUnits;
  const int64_t resident = 256 * pd_occupancy(D, e4m3);
  return static_cast<int>(most < resident ? most : resident);
}

// The pieces, their (m, l), then starts [groups + 2] int32.
int64_t paged_decode_ws_elems(int B, int H, int Hk, int D, bool e4m3, int units) {
  if (paged_decode_one(D, e4m3, units)) return 0;
  const int64_t pieces = 2 * static_cast<int64_t>(paged_decode_workgroups(B, H, Hk, D, e4m3, units)) * pd_heads(D);
  return pieces * (D + 2) + static_cast<int64_t>(B) * Hk + 2;
}

template <typename E, int D, bool F8>
static hipError_t launch_paged_decode_t(const PagedCache& c, const PagedRows& rows, const uint16_t* q,
                                        int64_t sq_b, int64_t sq_h, int B, int H, float scale,
                                        uint16_t* out, int64_t so_b, int64_t so_h, float* ws,
                                        hipStream_t stream) {
  const int grp = H / c.Hk, chunks = (grp + pd_heads(D) - 1) / pd_heads(D);
  const bool lists = rows.kv_idx != nullptr;
  const PagedGroups gr{lists ? B * c.Hk : B, lists ? chunks : c.Hk * chunks, c.Hk};
  if (paged_decode_one(D, F8, lists ? rows.k_slots : rows.max_pages)) {
    // Eight wavefronts a row; four where there are more rows than CUs and a CU's
    // registers hold one workgroup of eight but two or three of four (1024 sequences of
    // up to 1K tokens, e4m3, head_dim 128 106 / 80.5 us, 64 x 8 heads 23.4 / 22.2, but 32 x
    // 4 heads 11.4 / 13.5; head_dim 64 25.4 / 26.3).
    const bool four = D >= 128 && static_cast<int64_t>(B) * c.Hk * chunks > 256;
    const auto kernel = four ? paged_decode_kernel<E, D, F8, false, 4> : paged_decode_kernel<E, D, F8, false, 8>;
    kernel<<<dim3(c.Hk * chunks, B), 64 * (four ? 4 : 8), 0, stream>>>(c, rows, gr, q, sq_b, sq_h, grp, chunks,
                                                                       scale * kLog2e, out, so_b, so_h, nullptr,
                                                                       nullptr, nullptr);
    return hipGetLastError();
  }
  const int wgs = paged_decode_workgroups(B, H, c.Hk, D, F8, lists ? rows.k_slots : rows.max_pages);
  const int64_t pieces = 2 * static_cast<int64_t>(wgs) * pd_heads(D);
  float* part = ws;
  float* ml = part + pieces * D;
  int* starts = reinterpret_cast<int*>(ml + 2 * pieces);
  // Pages are read past the 256 MB memory-side cache where the call can hold three
  // times as much and they would only displace each other there (32 x 16K tokens,
  // 40/8 heads, bf16 362 -> 336 us; 32 x 64K in e4m3 725 -> 698; 24 of up to 16K 77 ->
  // 72); smaller calls may find theirs in it (4 of up to 64K, head_dim 256, 41.1 and
  // 42.2).  The table's width bounds the lengths, which are on the device.
  const int64_t most = static_cast<int64_t>(B) * c.Hk * (lists ? rows.k_slots : rows.max_pages) *
                       (2 * kBlock * D * (F8 ? 1 : 2));
  const auto kernel = most > 768ll << 20 ? paged_decode_kernel<E, D, F8, true, 0>
                                         : paged_decode_kernel<E, D, F8, false, 0>;
  kernel<<<dim3(wgs), 64 * kPdWaves, 0, stream>>>(c, rows, gr, q, sq_b, sq_h, grp, chunks, scale * kLog2e, out,
                                                  so_b, so_h, starts, part, ml);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  paged_combine_kernel<E, D><<<dim3(B * H), kPdCombineThreads, 0, stream>>>(
      starts, part, ml, gr, grp, chunks, lists, out, so_b, so_h);
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
