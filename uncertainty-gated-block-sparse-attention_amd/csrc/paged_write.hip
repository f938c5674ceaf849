// Paged cache: new tokens in, cached tokens out (paged.h has the layout).
//
// Both are copies bound by HBM: a written token costs 4 D bytes read and 2 D
// (e4m3) or 4 D written per head, a read one the reverse.  Six prompts of up to 32K
// tokens, 4 heads, into e4m3 (232 MB): 48 us, 4.8 TB/s; 64K tokens of 8 heads back
// (404 MB): 74.7 us, 5.4 TB/s; a copy of 256 MiB runs at 5.3.
#include "paged.h"

namespace ugbsa {

// Pages that sequence b's new tokens touch.
__device__ __forceinline__ int touched_pages(int len, int n_new) {
  return n_new > 0 ? (len + n_new - 1) / kBlock - len / kBlock + 1 : 0;
}

// One workgroup per (touched page, KV head): it alone writes the page's head, so
// the summary needs no atomics.  A thread takes 8 dims of every (256 / (D / 8))-th
// token; a token's scale is a maximum over its D / 8 neighbouring lanes.
template <typename E, int D, bool F8>
__global__ __launch_bounds__(256) void paged_write_kernel(
    PagedCache c, const uint16_t* __restrict__ k, int64_t sk_t, int64_t sk_h,
    const uint16_t* __restrict__ v, int64_t sv_t, int64_t sv_h, const int32_t* __restrict__ cu_new,
    const int32_t* __restrict__ lens, const int32_t* __restrict__ table, int64_t st_b, int B, int T,
    int max_pages) {
  constexpr int CH = D / 8, RG = 256 / CH;
  __shared__ float red[2][RG][D + 1];
  __shared__ int s_sum[4], s_unit[4];
  const int tid = threadIdx.x, ch = tid % CH, rg = tid / CH;
  const uint32_t h = blockIdx.y, unit = blockIdx.x;
  const int64_t most = static_cast<int64_t>(max_pages) * kBlock;

  // the sequence, its first new token and the page this workgroup is for
  int b = unit, page_at = 0, t0 = unit, t1 = unit + 1;
  if (cu_new != nullptr) {
    int64_t before = 0;                     // touched pages of the sequences already passed
    if (tid == 0) s_unit[0] = -1;
    for (int b0 = 0; b0 < B; b0 += 256) {
      const int i = b0 + tid;
      int n = 0, a0 = 0, a1 = 0;
      if (i < B) {
        a0 = min(max(cu_new[i], 0), T);
        a1 = min(max(cu_new[i + 1], a0), T);
        const int len = max(lens[i], 0);
        const int64_t room = most - len;    // tokens past the table have no page
        if (a1 - a0 > room) a1 = a0 + static_cast<int>(room > 0 ? room : 0);
        n = touched_pages(len, a1 - a0);
      }
      int incl = n;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int y = __shfl_up(incl, off, 64);
        if ((tid & 63) >= off) incl += y;
      }
      if ((tid & 63) == 63) s_sum[tid >> 6] = incl;
      __syncthreads();
      int64_t start = before + incl - n;
      for (int w = 0; w < (tid >> 6); ++w) start += s_sum[w];
      if (unit >= start && unit < start + n) {
        s_unit[0] = i;
        s_unit[1] = static_cast<int>(unit - start);
        s_unit[2] = a0;
        s_unit[3] = a1;
      }
      before += s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
      __syncthreads();
      if (before > unit) break;
    }
    if (s_unit[0] < 0) return;
    b = s_unit[0], page_at = s_unit[1], t0 = s_unit[2], t1 = s_unit[3];
  }
  const int len = max(lens[b], 0);
  const int blk = len / kBlock + page_at;
  if (blk >= max_pages) return;
  const int page = table[b * st_b + blk];
  if (page < 0 || page >= c.num_pages) return;
  // slots [s0, s1) of the page get tokens t, t + 1, ...
  const int s0 = page_at == 0 ? len % kBlock : 0;
  const int t = t0 + (page_at == 0 ? 0 : page_at * kBlock - len % kBlock);
  const int s1 = min(kBlock, s0 + t1 - t);

  float mx[8], mn[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) mx[j] = -INFINITY, mn[j] = INFINITY;
  const int64_t head = static_cast<int64_t>(page) * c.Hk + h;
  for (int s = s0 + rg; s < s1; s += RG) {
    const int64_t tok = t + s - s0;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const uint16_t* src = (kv ? v + tok * sv_t + h * sv_h : k + tok * sk_t + h * sk_h) + 8 * ch;
      const u32x4 raw = stream_load<true>(reinterpret_cast<const u32x4*>(src));
      const int64_t at = page * (kv ? c.sv_p : c.sk_p) + h * (kv ? c.sv_h : c.sk_h) +
                         s * (kv ? c.sv_n : c.sk_n) + 8 * ch;
      float x[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = E::to_f32(raw[j] & 0xFFFFu);
        x[2 * j + 1] = E::to_f32(raw[j] >> 16);
      }
      if (kv == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) mx[j] = fmaxf(mx[j], x[j]), mn[j] = fminf(mn[j], x[j]);
      }
      if constexpr (!F8) {
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(kv ? c.v : c.k) + at) = raw;
      } else {
        // the largest magnitude whose four-bit rounding reads back finite (infinities
        // are held there too; NaN stays NaN and does not count for the scale)
        constexpr float kMost = E::code == ElemF16::code ? 61440.f : 1.875f * 0x1p127f;
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = x[j] > kMost ? kMost : (x[j] < -kMost ? -kMost : x[j]);
          top = fmaxf(top, fabsf(x[j]));
        }
#pragma unroll
        for (int off = CH / 2; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
        // smallest e with top <= 448 2^e = 1.75 2^(e + 8), as a byte e + 127
        const uint32_t bits = __float_as_uint(top);
        const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
        const int byte = bits == 0u ? 127 : max(e, 0);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = ldexpf(x[j], 127 - byte);   // exact
        int lo = 0, hi = 0;
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], lo, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], lo, true);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[4], x[5], hi, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[6], x[7], hi, true);
        *reinterpret_cast<int2*>(static_cast<uint8_t*>(kv ? c.v : c.k) + at) = int2{lo, hi};
        if (ch == 0) (kv ? c.v_scale : c.k_scale)[head * kBlock + s] = static_cast<uint8_t>(byte);
      }
    }
  }
  if (c.planes == nullptr) return;
  if (s1 - s0 == 1) {             // a decode step's token: its threads hold all there is
    if (rg != 0) return;
    uint16_t* out = c.planes + head * 2 * D + 8 * ch;
    u32x4 hi = {0u, 0u, 0u, 0u}, lo = hi;
    if (s0 > 0) {
      hi = *reinterpret_cast<const u32x4*>(out);
      lo = *reinterpret_cast<const u32x4*>(out + D);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (s0 > 0) {
        mx[2 * j] = fmaxf(mx[2 * j], E::to_f32(hi[j] & 0xFFFFu));
        mx[2 * j + 1] = fmaxf(mx[2 * j + 1], E::to_f32(hi[j] >> 16));
        mn[2 * j] = fminf(mn[2 * j], E::to_f32(lo[j] & 0xFFFFu));
        mn[2 * j + 1] = fminf(mn[2 * j + 1], E::to_f32(lo[j] >> 16));
      }
      hi[j] = E::from_f32(mx[2 * j]) | static_cast<uint32_t>(E::from_f32(mx[2 * j + 1])) << 16;
      lo[j] = E::from_f32(mn[2 * j]) | static_cast<uint32_t>(E::from_f32(mn[2 * j + 1])) << 16;
    }
    *reinterpret_cast<u32x4*>(out) = hi;
    *reinterpret_cast<u32x4*>(out + D) = lo;
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    red[0][rg][8 * ch + j] = mx[j];
    red[1][rg][8 * ch + j] = mn[j];
  }
  __syncthreads();
  uint16_t* out = c.planes + head * 2 * D;
  for (int d = tid; d < D; d += 256) {
    float a = -INFINITY, z = INFINITY;
    for (int g = 0; g < RG; ++g) a = fmaxf(a, red[0][g][d]), z = fminf(z, red[1][g][d]);
    if (s0 > 0) {                 // the page's earlier keys; its first token starts it over
      a = fmaxf(a, E::to_f32(out[d]));
      z = fminf(z, E::to_f32(out[D + d]));
    }
    out[d] = E::from_f32(a);      // exact: an input value
    out[D + d] = E::from_f32(z);
  }
}

// One workgroup per (64 output rows, KV head, sequence): rows past the length are
// zeros.  NT: an output that the 256 MB memory-side cache does not hold goes past it,
// as do the pages it comes from.
template <typename E, int D, bool F8, bool NT>
__global__ __launch_bounds__(256) void paged_read_kernel(
    PagedCache c, const int32_t* __restrict__ lens, const int32_t* __restrict__ table, int64_t st_b,
    int max_pages, int N, uint16_t* __restrict__ ko, int64_t sok_b, int64_t sok_h, int64_t sok_n,
    uint16_t* __restrict__ vo, int64_t sov_b, int64_t sov_h, int64_t sov_n) {
  constexpr int CH = D / 8, RG = 256 / CH;
  const int tid = threadIdx.x, ch = tid % CH, rg = tid / CH;
  const int blk = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int len = cached_len(lens, b, max_pages);
  const int page = blk < max_pages && blk * kBlock < len ? table[b * st_b + blk] : -1;
  const int held = page >= 0 && page < c.num_pages ? min(kBlock, len - blk * kBlock) : 0;
  const int rows = min(kBlock, N - blk * kBlock);
  const int64_t head = static_cast<int64_t>(page) * c.Hk + h;
  for (int s = rg; s < rows; s += RG) {
    const int64_t n = static_cast<int64_t>(blk) * kBlock + s;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      u32x4 x = {0u, 0u, 0u, 0u};
      if (s < held) {
        const int64_t at = page * (kv ? c.sv_p : c.sk_p) + h * (kv ? c.sv_h : c.sk_h) +
                           s * (kv ? c.sv_n : c.sk_n) + 8 * ch;
        if constexpr (!F8) {
          x = stream_load<NT>(reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(kv ? c.v : c.k) + at));
        } else {
          const u32x2 code = stream_load<NT>(reinterpret_cast<const u32x2*>(static_cast<const uint8_t*>(kv ? c.v : c.k) + at));
          const float scale = e8m0((kv ? c.v_scale : c.k_scale)[head * kBlock + s]);
          x = __builtin_bit_cast(u32x4, e4m3_x8<E>(code[0], code[1], scale));
        }
      }
      uint16_t* dst = (kv ? vo + b * sov_b + h * sov_h + n * sov_n : ko + b * sok_b + h * sok_h + n * sok_n) + 8 * ch;
      if constexpr (NT) __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(dst));
      else *reinterpret_cast<u32x4*>(dst) = x;
    }
  }
}

#define UGBSA_PAGED_INSTANCES(CALL)                                       \
  do {                                                                    \
    if (c.elem == ElemF16::code) {                                        \
      if (c.e4m3) { UGBSA_PAGED_D(CALL, ElemF16, true); }                 \
      else { UGBSA_PAGED_D(CALL, ElemF16, false); }                       \
    } else {                                                              \
      if (c.e4m3) { UGBSA_PAGED_D(CALL, ElemBf16, true); }                \
      else { UGBSA_PAGED_D(CALL, ElemBf16, false); }                      \
    }                                                                     \
    return hipErrorInvalidValue;                                          \
  } while (0)
#define UGBSA_PAGED_D(CALL, E_, F8_)                                      \
  if (c.D == 64) { CALL(E_, 64, F8_); return hipGetLastError(); }         \
  if (c.D == 128) { CALL(E_, 128, F8_); return hipGetLastError(); }       \
  if (c.D == 256) { CALL(E_, 256, F8_); return hipGetLastError(); }

int64_t paged_write_units(int B, int T, bool ragged) {
  if (!ragged) return B;
  // a sequence's n tokens touch at most n pages and at most (n + 62) / 64 + 1
  const int64_t most = static_cast<int64_t>(T) / kBlock + 2 * static_cast<int64_t>(B);
  return most < T ? most : T;
}

hipError_t launch_paged_write(const PagedCache& c, const uint16_t* k, int64_t sk_t, int64_t sk_h,
                              const uint16_t* v, int64_t sv_t, int64_t sv_h, const int32_t* cu_new,
                              const int32_t* lens, const int32_t* table, int64_t st_b, int B, int T,
                              int max_pages, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(paged_write_units(B, T, cu_new != nullptr)), c.Hk);
#define UGBSA_CALL(E_, D_, F8_)                                                                  \
  paged_write_kernel<E_, D_, F8_><<<grid, 256, 0, stream>>>(c, k, sk_t, sk_h, v, sv_t, sv_h, cu_new, \
                                                            lens, table, st_b, B, T, max_pages)
  UGBSA_PAGED_INSTANCES(UGBSA_CALL);
#undef UGBSA_CALL
}

hipError_t launch_paged_read(const PagedCache& c, const int32_t* lens, const int32_t* table,
                             int64_t st_b, int B, int max_pages, int N, uint16_t* ko, int64_t sok_b,
                             int64_t sok_h, int64_t sok_n, uint16_t* vo, int64_t sov_b, int64_t sov_h,
                             int64_t sov_n, hipStream_t stream) {
  const dim3 grid((N + kBlock - 1) / kBlock, c.Hk, B);
  // 64K tokens of 8 heads from e4m3 (268 MB): 86 -> 81.6 us
  const bool past_cache = 4 * static_cast<int64_t>(B) * c.Hk * N * c.D >= 256 << 20;
#define UGBSA_CALL(E_, D_, F8_)                                                                     \
  (past_cache ? paged_read_kernel<E_, D_, F8_, true> : paged_read_kernel<E_, D_, F8_, false>)       \
      <<<grid, 256, 0, stream>>>(c, lens, table, st_b, max_pages, N, ko, sok_b, sok_h, sok_n, vo, sov_b, \
                                 sov_h, sov_n)
  UGBSA_PAGED_INSTANCES(UGBSA_CALL);
#undef UGBSA_CALL
}

}  // namespace ugbsa
