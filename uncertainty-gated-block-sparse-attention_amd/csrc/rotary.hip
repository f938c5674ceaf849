// Rotary positions of queries and keys in one launch (rotary.h has the mathematics);
// the gradient is the same with sin negated.
//
// Bound by memory: 4 bytes a value, read and written once.
#include <algorithm>

#include "rotary.h"

namespace ugbsa {

// Where the pairs lie: in halves that are whole vectors of eight, or side by side.
constexpr int kHalves = 0, kPairs = 1;

// A load or store that goes past the 256 MB memory-side cache (NT).
template <bool NT>
__device__ __forceinline__ u32x4 load8(const uint16_t* p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  else return *reinterpret_cast<const u32x4*>(p);
}
template <bool NT>
__device__ __forceinline__ void store8(uint16_t* p, u32x4 x) {
  if constexpr (NT) __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(p));
  else *reinterpret_cast<u32x4*>(p) = x;
}

struct RotaryRow {
  const uint16_t* x;
  uint16_t* y;       // null past the heads
};
// Head h of the queries', then the keys', of token (b, m).
__device__ __forceinline__ RotaryRow rotary_row(const RotaryHeads& q, const RotaryHeads& k, int h, uint32_t b,
                                                uint32_t m) {
  if (h < q.heads) return {q.x + b * q.sx_b + h * q.sx_h + m * q.sx_m, q.y + b * q.sy_b + h * q.sy_h + m * q.sy_m};
  h -= q.heads;
  if (h < k.heads) return {k.x + b * k.sx_b + h * k.sx_h + m * k.sx_m, k.y + b * k.sy_b + h * k.sy_h + m * k.sy_m};
  return {nullptr, nullptr};
}

// The pairs of two words of the lower and the upper half.
template <typename E>
__device__ __forceinline__ void turn_words(uint32_t& lo, uint32_t& hi, const float* cs, const float* sn) {
  float a0, a1, b0, b1;
  turn_pair(E::to_f32(lo & 0xFFFFu), E::to_f32(hi & 0xFFFFu), cs[0], sn[0], a0, b0);
  turn_pair(E::to_f32(lo >> 16), E::to_f32(hi >> 16), cs[1], sn[1], a1, b1);
  lo = E::pack2(a0, a1);
  hi = E::pack2(b0, b1);
}

// A thread's two vectors of eight dims of one token: eight pairs, whose cos and sin it works
// out once for its heads (HPT of them, `groups` apart), while their loads are on the way.
// Neighbouring threads hold neighbouring vectors, then neighbouring heads.
template <typename E, int LAYOUT, int HPT, bool NT>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryHeads q, RotaryHeads k, RotaryTable t,
                                                     const int32_t* __restrict__ positions, int64_t sp_b,
                                                     uint32_t M, int D, int chunk_bits, uint32_t groups,
                                                     uint32_t row0, uint32_t units, float sign) {
  const uint32_t unit = blockIdx.x * 256u + threadIdx.x;
  if (unit >= units) return;
  const int chunk = unit & ((1u << chunk_bits) - 1), pairs = t.pairs;
  const uint32_t row = row0 + (unit >> chunk_bits), tok = row / groups, g = row - tok * groups;
  const uint32_t b = tok / M, m = tok - b * M;
  // half layout: dims da .. of the lower half and db .. of the upper, of the dims that turn or of
  // those that pass; else two vectors half a head apart
  const bool turns = LAYOUT == kPairs || 8 * chunk < pairs;
  const int da = LAYOUT == kPairs || turns ? 8 * chunk : 8 * chunk + pairs;
  const int db = LAYOUT == kPairs ? D / 2 + da : (turns ? pairs + da : da + D / 2 - pairs);
  u32x4 va[HPT], vb[HPT];
  uint16_t* to[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const RotaryRow r = rotary_row(q, k, g + i * groups, b, m);
    to[i] = r.y;
    va[i] = vb[i] = u32x4{0u, 0u, 0u, 0u};
    if (to[i] != nullptr) va[i] = load8<NT>(r.x + da), vb[i] = load8<NT>(r.x + db);
  }
  if (turns) {
    const double pos = positions[b * sp_b + m];
    float cs[8], sn[8];
    // all bits of the pairs past the table's, which keep theirs (by branches the compiler made 27 KB
    // of code of this, at one wavefront per SIMD: 8192 tokens 104 us, now 33)
    uint32_t passes[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      passes[i] = LAYOUT == kPairs && (i < 4 ? da : db) / 2 + i % 4 >= pairs ? ~0u : 0u;
      const int j = LAYOUT == kPairs ? min((i < 4 ? da : db) / 2 + i % 4, pairs - 1) : da + i;
      turn_cos_sin(pos, t.turns[j], t.attention, cs[i], sn[i]);
      sn[i] *= sign;
    }
#pragma unroll
    for (int i = 0; i < HPT; ++i) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if constexpr (LAYOUT == kPairs) {
          float a, c;
          turn_pair(E::to_f32(va[i][w] & 0xFFFFu), E::to_f32(va[i][w] >> 16), cs[w], sn[w], a, c);
          va[i][w] = (va[i][w] & passes[w]) | (E::pack2(a, c) & ~passes[w]);
          turn_pair(E::to_f32(vb[i][w] & 0xFFFFu), E::to_f32(vb[i][w] >> 16), cs[4 + w], sn[4 + w], a, c);
          vb[i][w] = (vb[i][w] & passes[4 + w]) | (E::pack2(a, c) & ~passes[4 + w]);
        } else {
          uint32_t lo = va[i][w], hi = vb[i][w];
          turn_words<E>(lo, hi, cs + 2 * w, sn + 2 * w);
          va[i][w] = lo, vb[i][w] = hi;
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < HPT; ++i)
    if (to[i] != nullptr) store8<NT>(to[i] + da, va[i]), store8<NT>(to[i] + db, vb[i]);
}

// Half layout whose halves are no whole vectors: a thread has W neighbouring pairs of a token
// and its heads, or W dims that pass (vectors at addresses of four bytes' alignment, with
// the pairs that are left one by one, took 94 us for 134 MB where this takes 38).
template <typename E, int W, int HPT>
__global__ __launch_bounds__(256) void rotary_odd_kernel(RotaryHeads q, RotaryHeads k, RotaryTable t,
                                                         const int32_t* __restrict__ positions, int64_t sp_b,
                                                         uint32_t M, uint32_t items, uint32_t groups, uint32_t row0,
                                                         uint32_t rows, float sign) {
  using Bits = std::conditional_t<W == 2, uint32_t, uint16_t>;
  const uint32_t unit = blockIdx.x * 256u + threadIdx.x, at = unit / items;
  if (at >= rows) return;
  const int item = static_cast<int>(unit - at * items), pairs = t.pairs;
  const uint32_t row = row0 + at, tok = row / groups, g = row - tok * groups, b = tok / M, m = tok - b * M;
  const bool turns = W * item < pairs;
  const int da = W * item, dc = pairs + da;          // past the pairs: dims from 2 pairs on
  Bits va[HPT], vb[HPT];
  uint16_t* to[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const RotaryRow r = rotary_row(q, k, g + i * groups, b, m);
    to[i] = r.y;
    va[i] = vb[i] = 0;
    if (to[i] != nullptr) {
      if (turns) va[i] = *reinterpret_cast<const Bits*>(r.x + da);
      vb[i] = *reinterpret_cast<const Bits*>(r.x + dc);
    }
  }
  if (turns) {
    const double pos = positions[b * sp_b + m];
    float cs[2], sn[2];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      turn_cos_sin(pos, t.turns[da + i], t.attention, cs[i], sn[i]);
      sn[i] *= sign;
    }
    if constexpr (W == 1) cs[1] = sn[1] = 0.f;
#pragma unroll
    for (int i = 0; i < HPT; ++i) {
      uint32_t lo = va[i], hi = vb[i];
      turn_words<E>(lo, hi, cs, sn);
      va[i] = static_cast<Bits>(lo), vb[i] = static_cast<Bits>(hi);
    }
  }
#pragma unroll
  for (int i = 0; i < HPT; ++i)
    if (to[i] != nullptr) {
      if (turns) *reinterpret_cast<Bits*>(to[i] + da) = va[i];
      *reinterpret_cast<Bits*>(to[i] + dc) = vb[i];
    }
}

// Where it leaves the card some thousand wavefronts a thread takes two heads (512 tokens, 28/4
// heads 5.2 us of one each; 32K tokens, 537 MB, 95 us of two, 98 of four, 103 of one), or four where
// halves are no whole vectors (8192 tokens, 100 of 128 dims, 38 and 68 of one).  Tensors of more
// than 320 MB, in and out, go past the memory-side cache: 2 x 8191 tokens, 40/8 heads,
// head_dim 128 (402 MB a launch) 79 -> 70 us; 67 MB 21 -> 23, 300 MB 70 -> 74.
template <typename E>
static hipError_t launch_rotary_t(const RotaryTable& t, const int32_t* positions, int64_t sp_b,
                                  const RotaryHeads& q, const RotaryHeads& k, int B, int M, int D, bool inverse,
                                  hipStream_t stream) {
  const uint32_t heads = q.heads + k.heads, toks = static_cast<uint32_t>(B) * M;
  const float sign = inverse ? -1.f : 1.f;
  const int bits = D == 64 ? 2 : (D == 128 ? 3 : 4);
  const bool many = (static_cast<uint64_t>(toks) * heads << bits) >= 1u << 21;
  const bool odd = !t.interleaved && t.pairs % 8;
  const uint32_t each = !many ? 1 : (odd ? 4 : 2), groups = (heads + each - 1) / each, rows = toks * groups;
  // A grid holds fewer than 2^32 threads: the rows of the longest calls go in several launches.
  const auto in_pieces = [&](uint32_t threads, auto launch) {        // of a row; launch(first row, rows, grid)
    const uint32_t most = (1u << 31) / threads;
    for (uint32_t row0 = 0; row0 < rows; row0 += most) {
      const uint32_t n = std::min(most, rows - row0);
      launch(row0, n, (n * threads + 255) / 256);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  };
  if (odd) {
    const uint32_t items = (D - t.pairs) / (t.pairs % 2 ? 1 : 2);
    const auto kernel = t.pairs % 2 ? (many ? rotary_odd_kernel<E, 1, 4> : rotary_odd_kernel<E, 1, 1>)
                                    : (many ? rotary_odd_kernel<E, 2, 4> : rotary_odd_kernel<E, 2, 1>);
    return in_pieces(items, [&](uint32_t row0, uint32_t n, uint32_t grid) {
      kernel<<<grid, 256, 0, stream>>>(q, k, t, positions, sp_b, M, items, groups, row0, n, sign);
    });
  }
  const bool past = many && static_cast<uint64_t>(toks) * heads * D * 4 > 320ull << 20;
#define UGBSA_ROT(L_) \
  (past ? rotary_kernel<E, L_, 2, true> : (many ? rotary_kernel<E, L_, 2, false> : rotary_kernel<E, L_, 1, false>))
  const auto kernel = t.interleaved ? UGBSA_ROT(kPairs) : UGBSA_ROT(kHalves);
#undef UGBSA_ROT
  return in_pieces(1u << bits, [&](uint32_t row0, uint32_t n, uint32_t grid) {
    kernel<<<grid, 256, 0, stream>>>(q, k, t, positions, sp_b, M, D, bits, groups, row0, n << bits, sign);
  });
}

hipError_t launch_rotary(const RotaryTable& t, const int32_t* positions, int64_t sp_b, const RotaryHeads& q,
                         const RotaryHeads& k, int B, int M, int D, int elem, bool inverse, hipStream_t stream) {
  return elem == ElemF16::code ? launch_rotary_t<ElemF16>(t, positions, sp_b, q, k, B, M, D, inverse, stream)
                               : launch_rotary_t<ElemBf16>(t, positions, sp_b, q, k, B, M, D, inverse, stream);
}

}  // namespace ugbsa
