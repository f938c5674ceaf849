// Rotary positions of queries and keys in one launch (rotary.h has the mathematics);
// the gradient is the same with sin negated.
//
// Bound by memory: 4 bytes a value, read and written once.
#include "rotary.h"

namespace ugbsa {

// A thread's 16 dims of one token: eight pairs, whose cos and sin it works out once
// for its heads (HPT of them, `groups` apart), while their loads are on the way.
// Neighbouring threads hold neighbouring dims, then neighbouring heads.
template <typename E, bool INTER, int HPT>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryHeads q, RotaryHeads k, RotaryTable t,
                                                     const int32_t* __restrict__ positions, int64_t sp_b,
                                                     uint32_t M, int chunk_bits, uint32_t groups, uint32_t units,
                                                     float sign) {
  const uint32_t unit = blockIdx.x * 256u + threadIdx.x;
  if (unit >= units) return;
  const int chunk = unit & ((1u << chunk_bits) - 1);
  const uint32_t row = unit >> chunk_bits, tok = row / groups, g = row - tok * groups;
  const uint32_t b = tok / M, m = tok - b * M;
  const int pairs = t.pairs, j0 = 8 * chunk;
  // the lower and the upper half of the eight pairs (half layout), or sixteen dims in a row
  const bool split = !INTER && j0 < pairs;
  const int da = split ? j0 : 16 * chunk, db = split ? pairs + j0 : 16 * chunk + 8;
  u32x4 va[HPT], vb[HPT];
  uint16_t* to[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = g + i * groups;
    to[i] = nullptr;
    va[i] = vb[i] = u32x4{0u, 0u, 0u, 0u};
    if (h < q.heads + k.heads) {
      const bool is_q = h < q.heads;
      const int hh = is_q ? h : h - q.heads;
      const uint16_t* x = is_q ? q.x + b * q.sx_b + hh * q.sx_h + m * q.sx_m
                               : k.x + b * k.sx_b + hh * k.sx_h + m * k.sx_m;
      to[i] = is_q ? q.y + b * q.sy_b + hh * q.sy_h + m * q.sy_m
                   : k.y + b * k.sy_b + hh * k.sy_h + m * k.sy_m;
      va[i] = *reinterpret_cast<const u32x4*>(x + da);
      vb[i] = *reinterpret_cast<const u32x4*>(x + db);
    }
  }
  if (j0 < pairs) {
    const double pos = positions[b * sp_b + m];
    float cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = INTER ? min(j0 + i, pairs - 1) : j0 + i;
      turn_cos_sin(pos, t.turns[j], t.attention, cs[i], sn[i]);
      sn[i] *= sign;
    }
#pragma unroll
    for (int i = 0; i < HPT; ++i) {
      if constexpr (INTER) {
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          const uint32_t p = w < 4 ? va[i][w & 3] : vb[i][w & 3];
          float a, c;
          turn_pair(E::to_f32(p & 0xFFFFu), E::to_f32(p >> 16), cs[w], sn[w], a, c);
          const uint32_t y = j0 + w < pairs ? E::pack2(a, c) : p;
          if (w < 4) va[i][w & 3] = y;
          else vb[i][w & 3] = y;
        }
      } else {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          float a0, a1, b0, b1;
          turn_pair(E::to_f32(va[i][w] & 0xFFFFu), E::to_f32(vb[i][w] & 0xFFFFu), cs[2 * w], sn[2 * w], a0, b0);
          turn_pair(E::to_f32(va[i][w] >> 16), E::to_f32(vb[i][w] >> 16), cs[2 * w + 1], sn[2 * w + 1], a1, b1);
          va[i][w] = E::pack2(a0, a1);
          vb[i][w] = E::pack2(b0, b1);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < HPT; ++i)
    if (to[i] != nullptr) {
      *reinterpret_cast<u32x4*>(to[i] + da) = va[i];
      *reinterpret_cast<u32x4*>(to[i] + db) = vb[i];
    }
}

// Half layout whose halves are no whole vectors of eight: a wavefront a token and
// kRotaryOddHeads of its heads, a lane a pair or a dim that passes.
constexpr int kRotaryOddHeads = 4;
template <typename E>
__global__ __launch_bounds__(256) void rotary_odd_kernel(RotaryHeads q, RotaryHeads k, RotaryTable t,
                                                         const int32_t* __restrict__ positions, int64_t sp_b,
                                                         uint32_t M, int D, uint32_t groups, uint32_t rows,
                                                         float sign) {
  const uint32_t row = blockIdx.x * 4u + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= rows) return;
  const uint32_t tok = row / groups, g = row - tok * groups, b = tok / M, m = tok - b * M;
  const double pos = positions[b * sp_b + m];
  const int pairs = t.pairs;
  for (int j = lane; j < D - pairs; j += 64) {
    const bool turn = j < pairs;
    float cs = 1.f, sn = 0.f;
    if (turn) turn_cos_sin(pos, t.turns[j], t.attention, cs, sn);
    sn *= sign;
    for (int i = 0; i < kRotaryOddHeads; ++i) {
      const int h = g + i * groups;
      if (h >= q.heads + k.heads) break;
      const bool is_q = h < q.heads;
      const int hh = is_q ? h : h - q.heads;
      const uint16_t* x = is_q ? q.x + b * q.sx_b + hh * q.sx_h + m * q.sx_m
                               : k.x + b * k.sx_b + hh * k.sx_h + m * k.sx_m;
      uint16_t* y = is_q ? q.y + b * q.sy_b + hh * q.sy_h + m * q.sy_m
                         : k.y + b * k.sy_b + hh * k.sy_h + m * k.sy_m;
      if (turn) {
        float a, c;
        turn_pair(E::to_f32(x[j]), E::to_f32(x[j + pairs]), cs, sn, a, c);
        const uint32_t p = E::pack2(a, c);
        y[j] = static_cast<uint16_t>(p & 0xFFFFu);
        y[j + pairs] = static_cast<uint16_t>(p >> 16);
      } else {
        y[j + pairs] = x[j + pairs];
      }
    }
  }
}

template <typename E>
static hipError_t launch_rotary_t(const RotaryTable& t, const int32_t* positions, int64_t sp_b,
                                  const RotaryHeads& q, const RotaryHeads& k, int B, int M, int D, bool inverse,
                                  hipStream_t stream) {
  const uint32_t heads = q.heads + k.heads, toks = static_cast<uint32_t>(B) * M;
  const float sign = inverse ? -1.f : 1.f;
  if (!t.interleaved && t.pairs % 8) {
    const uint32_t groups = (heads + kRotaryOddHeads - 1) / kRotaryOddHeads, rows = toks * groups;
    rotary_odd_kernel<E><<<(rows + 3) / 4, 256, 0, stream>>>(q, k, t, positions, sp_b, M, D, groups, rows, sign);
    return hipGetLastError();
  }
  const int bits = D == 64 ? 2 : (D == 128 ? 3 : 4);
  const int per = (static_cast<uint64_t>(toks) * heads << bits) >= 1u << 21 ? 4 : 1;
  const uint32_t groups = (heads + per - 1) / per, units = toks * groups << bits;
#define UGBSA_ROT(I_, H_)                                                                                  \
  rotary_kernel<E, I_, H_><<<(units + 255) / 256, 256, 0, stream>>>(q, k, t, positions, sp_b, M, bits, groups, \
                                                                    units, sign)
  if (t.interleaved) {
    if (per == 4) UGBSA_ROT(true, 4); else UGBSA_ROT(true, 1);
  } else {
    if (per == 4) UGBSA_ROT(false, 4); else UGBSA_ROT(false, 1);
  }
#undef UGBSA_ROT
  return hipGetLastError();
}

hipError_t launch_rotary(const RotaryTable& t, const int32_t* positions, int64_t sp_b, const RotaryHeads& q,
                         const RotaryHeads& k, int B, int M, int D, int elem, bool inverse, hipStream_t stream) {
  return elem == ElemF16::code ? launch_rotary_t<ElemF16>(t, positions, sp_b, q, k, B, M, D, inverse, stream)
                               : launch_rotary_t<ElemBf16>(t, positions, sp_b, q, k, B, M, D, inverse, stream);
}

}  // namespace ugbsa
