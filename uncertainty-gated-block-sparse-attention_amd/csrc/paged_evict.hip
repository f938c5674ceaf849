// Eviction from the paged cache by accumulated attention weight: per (sequence, KV head)
// the first tokens, the newest and, of the others, the heaviest, packed in their order
// into other pages.
//
// Picking reads a row's weights a few times over (4 bytes a token, from L2 after the
// first); moving copies the kept tokens' codes, 2 token bytes each way.
#include "paged.h"

namespace ugbsa {

constexpr int kPickThreads = 1024, kPickWaves = kPickThreads / 64;
constexpr int kPickBins = 2048;        // 11, 11 and 10 bits of the key

// Order of a row's tokens, larger first: tokens that stay whatever they weigh, NaN, then
// by weight (zeros of either sign alike); 0: the page is absent, the token is not kept.
struct PickRow {
  const float* mass;
  const int32_t* table;
  int n, first, last, num_pages;       // tokens below first or from last on stay
  __device__ __forceinline__ uint32_t key(int i, float x) const {
    const int page = table[i / kBlock];
    if (i >= n || page < 0 || page >= num_pages) return 0u;
    if (i < first || i >= last) return 0xFFFFFFFFu;
    return x != x ? 0xFFFFFFFEu : float_key(x + 0.f);
  }
  // keys of tokens i .. i + 3 (i a multiple of 4, below n)
  __device__ __forceinline__ void keys4(int i, uint32_t* to) const {
    const f32x4 x = *reinterpret_cast<const f32x4*>(mass + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) to[j] = key(i + j, x[j]);
  }
};

// One workgroup per (KV head, sequence).  The k-th largest key by three digits, then each
// wavefront counts what it keeps of its share of the row and writes it behind the others'.
__global__ __launch_bounds__(kPickThreads) void paged_pick_kernel(
    const float* __restrict__ mass, int64_t sm_b, int64_t sm_h, const int32_t* __restrict__ lens,
    const int32_t* __restrict__ table, int64_t st_b, int max_pages, int num_pages, int keep, int recent, int first,
    int32_t* __restrict__ kept, int32_t* __restrict__ new_lens) {
  __shared__ uint32_t s_hist[kPickBins], s_wave[2][kPickWaves], s_found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = blockIdx.x, b = blockIdx.y;
  const int n = cached_len(lens, b, max_pages);
  const PickRow row{mass + b * sm_b + g * sm_h, table + b * st_b, n, first, max(n - recent, 0), num_pages};
  int32_t* out = kept + (static_cast<int64_t>(b) * gridDim.x + g) * keep;

  uint32_t prefix = 0u, mask = 0u, want = keep;      // want-th largest among the keys of the prefix
  int total = 0;                                      // tokens with a page
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bins = pass == 2 ? 1024 : 2048;
    for (int i = tid; i < kPickBins; i += kPickThreads) s_hist[i] = 0u;
    __syncthreads();
    for (int i = 4 * tid; i < n; i += 4 * kPickThreads) {
      uint32_t k[4];
      row.keys4(i, k);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j < n && (k[j] & mask) == prefix) atomicAdd(&s_hist[(k[j] >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    // bins from the largest: thread t holds bins - 1 - 2 t and the one below it
    const int hi = bins - 1 - 2 * tid;
    const uint32_t c0 = hi >= 0 ? s_hist[hi] : 0u, c1 = hi >= 1 ? s_hist[hi - 1] : 0u;
    const uint32_t ex = wave_excl_scan(c0 + c1, lane);
    if (lane == 63) s_wave[0][wave] = ex + c0 + c1;
    __syncthreads();
    uint32_t before = ex;
    for (int w = 0; w < wave; ++w) before += s_wave[0][w];
    if (pass == 0) {
      uint32_t all = 0u;
      for (int w = 0; w < kPickWaves; ++w) all += s_wave[0][w];
      // the keys of tokens with a page lie above 0x007F0000: the lowest bin holds the absent ones
      total = static_cast<int>(all - s_hist[0]);
      if (total <= keep) break;                       // all of them stay
    }
    if (before < want && want <= before + c0) s_found[0] = hi, s_found[1] = before;
    else if (before + c0 < want && want <= before + c0 + c1) s_found[0] = hi - 1, s_found[1] = before + c0;
    __syncthreads();
    prefix |= s_found[0] << shift;
    mask |= static_cast<uint32_t>(bins - 1) << shift;
    want -= s_found[1];
    __syncthreads();
  }
  // keys above the threshold stay, and the first `ties` equal to it
  const bool all = total <= keep;
  const uint32_t least = all ? 0u : prefix, ties = all ? 0u : want;
  const int count = all ? total : keep;
  if (tid == 0 && g == 0) new_lens[b] = count;
  __syncthreads();

  const int share = ((n + kPickWaves - 1) / kPickWaves + 255) / 256 * 256;
  const int i0 = wave * share, i1 = min(i0 + share, n);
  uint32_t above = 0u, equal = 0u;
  for (int i = i0 + 4 * lane; i < i1; i += 256) {
    uint32_t k[4];
    row.keys4(i, k);
#pragma unroll
    for (int j = 0; j < 4; ++j) above += k[j] > least ? 1u : 0u, equal += k[j] == least && i + j < n ? 1u : 0u;
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) above += shfl_xor_u(above, off), equal += shfl_xor_u(equal, off);
  if (lane == 0) s_wave[0][wave] = above, s_wave[1][wave] = equal;
  __syncthreads();
  uint32_t at = 0u, tied = 0u;                        // kept and tied tokens of the wavefronts before
  for (int w = 0; w < wave; ++w) at += s_wave[0][w], tied += s_wave[1][w];
  at += min(tied, ties);
  for (int base = i0; base < i1; base += 256) {
    const int i = base + 4 * lane;
    uint32_t k[4] = {0u, 0u, 0u, 0u};
    if (i < i1) row.keys4(i, k);
    uint32_t eq = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) eq += i + j < n && k[j] == least ? 1u : 0u;
    const uint32_t eq_before = wave_excl_scan(eq, lane);
    uint32_t t = tied + eq_before, mine = 0u;
    bool stay[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool tie = i + j < n && k[j] == least;
      stay[j] = k[j] > least || (tie && t < ties);
      t += tie ? 1u : 0u;
      mine += stay[j] ? 1u : 0u;
    }
    uint32_t to = at + wave_excl_scan(mine, lane);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (stay[j]) out[to++] = i + j;
    at = __builtin_amdgcn_readlane(to, 63);
    tied += __builtin_amdgcn_readlane(eq_before + eq, 63);
  }
  const int none = max_pages * kBlock;
  for (int i = count + tid; i < keep; i += kPickThreads) out[i] = none;
}

// One workgroup per (new page, KV head, sequence): it alone writes them.  A thread moves 8
// dims of every (256 / (D / 8))-th token; the summary is of the keys as they are stored.
template <typename E, int D, int KIND>
__global__ __launch_bounds__(256) void paged_move_kernel(
    PagedCache c, const float* __restrict__ mass, int64_t sm_b, int64_t sm_h, const int32_t* __restrict__ table,
    int64_t st_b, const int32_t* __restrict__ new_table, int64_t sn_b, const int32_t* __restrict__ kept, int keep,
    const int32_t* __restrict__ new_lens, float* __restrict__ new_mass, int64_t so_b, int64_t so_h) {
  constexpr int CH = D / 8, RG = 256 / CH;
  __shared__ float red[2][RG][D + 1];
  __shared__ int s_token[kBlock];
  const int tid = threadIdx.x, ch = tid % CH, rg = tid / CH;
  const int j = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int count = min(new_lens[b] - j * kBlock, kBlock);        // tokens of this page
  if (tid < kBlock) {
    int token = -1;
    float x = 0.f;
    if (tid < count) {
      token = kept[(static_cast<int64_t>(b) * gridDim.y + h) * keep + j * kBlock + tid];
      x = mass[b * sm_b + h * sm_h + token];
    }
    s_token[tid] = token;
    new_mass[b * so_b + h * so_h + j * kBlock + tid] = x;
  }
  if (count <= 0) return;
  const int page = new_table[b * sn_b + j];
  if (page < 0 || page >= c.num_pages) return;
  __syncthreads();
  float mx[8], mn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) mx[i] = -INFINITY, mn[i] = INFINITY;
  const int64_t head = static_cast<int64_t>(page) * c.Hk + h;
  constexpr int W = KIND == kPagesModel ? 4 : (KIND == kPagesE4m3 ? 2 : 1);     // words of 8 dims
  typedef uint32_t words __attribute__((ext_vector_type(W)));
  constexpr int CB = 4 * W / (KIND == kPagesModel ? 2 : 1);                     // elements of a stride
  using Elem = std::conditional_t<KIND == kPagesModel, uint16_t, uint8_t>;
  for (int s = rg; s < count; s += RG) {
    const int token = s_token[s], from = table[b * st_b + token / kBlock], slot = token % kBlock;
    const int64_t src_head = static_cast<int64_t>(from) * c.Hk + h;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      Elem* pages = static_cast<Elem*>(kv ? c.v : c.k);
      const int64_t sp = kv ? c.sv_p : c.sk_p, sh = h * (kv ? c.sv_h : c.sk_h) + CB * ch, sn = kv ? c.sv_n : c.sk_n;
      const words raw = *reinterpret_cast<const words*>(pages + from * sp + sh + slot * sn);
      *reinterpret_cast<words*>(pages + page * sp + sh + s * sn) = raw;
      uint8_t* scales = kv ? c.v_scale : c.k_scale;
      uint32_t byte = 127u;
      if constexpr (KIND == kPagesE4m3) {
        byte = scales[src_head * kBlock + slot];
        if (ch == 0) scales[head * kBlock + s] = static_cast<uint8_t>(byte);
      }
      if constexpr (KIND == kPagesE2m1) {
        byte = scales[(src_head * (D / 32) + ch / 4) * kBlock + slot];
        if (ch % 4 == 0) scales[(head * (D / 32) + ch / 4) * kBlock + s] = static_cast<uint8_t>(byte);
      }
      if (kv == 0) {
        u32x4 x;
        if constexpr (KIND == kPagesModel) {
          x = u32x4{raw[0], raw[1], raw[2], raw[3]};
        } else if constexpr (KIND == kPagesE4m3) {
          x = __builtin_bit_cast(u32x4, e4m3_x8<E>(raw[0], raw[1], e8m0(byte)));
        } else {
          x = e2m1_x8<E>(raw[0], e8m0(byte));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float lo = E::to_f32(x[i] & 0xFFFFu), hi = E::to_f32(x[i] >> 16);
          mx[2 * i] = fmaxf(mx[2 * i], lo), mn[2 * i] = fminf(mn[2 * i], lo);
          mx[2 * i + 1] = fmaxf(mx[2 * i + 1], hi), mn[2 * i + 1] = fminf(mn[2 * i + 1], hi);
        }
      }
    }
  }
  if (c.planes == nullptr) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) red[0][rg][8 * ch + i] = mx[i], red[1][rg][8 * ch + i] = mn[i];
  __syncthreads();
  uint16_t* out = c.planes + head * 2 * D;
  for (int d = tid; d < D; d += 256) {
    float a = -INFINITY, z = INFINITY;
    for (int r = 0; r < RG; ++r) a = fmaxf(a, red[0][r][d]), z = fminf(z, red[1][r][d]);
    out[d] = E::from_f32(a);
    out[D + d] = E::from_f32(z);
  }
}

hipError_t launch_paged_evict(const PagedCache& c, const float* mass, int64_t sm_b, int64_t sm_h,
                              const int32_t* lens, const int32_t* table, int64_t st_b, int B, int max_pages,
                              const int32_t* new_table, int64_t sn_b, int new_pages, int keep, int recent, int first,
                              int32_t* kept, int32_t* new_lens, float* new_mass, int64_t so_b, int64_t so_h,
                              hipStream_t stream) {
  paged_pick_kernel<<<dim3(c.Hk, B), kPickThreads, 0, stream>>>(mass, sm_b, sm_h, lens, table, st_b, max_pages,
                                                                c.num_pages, keep, recent, first, kept, new_lens);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid(new_pages, c.Hk, B);
#define UGBSA_EV(E_, D_, K_)                                                                                      \
  do {                                                                                                            \
    paged_move_kernel<E_, D_, K_><<<grid, 256, 0, stream>>>(c, mass, sm_b, sm_h, table, st_b, new_table, sn_b, kept, \
                                                            keep, new_lens, new_mass, so_b, so_h);                \
    return hipGetLastError();                                                                                     \
  } while (0)
#define UGBSA_EV_D(E_, K_)              \
  if (c.D == 64) UGBSA_EV(E_, 64, K_);  \
  if (c.D == 128) UGBSA_EV(E_, 128, K_); \
  if (c.D == 256) UGBSA_EV(E_, 256, K_)
#define UGBSA_EV_E(K_)                  \
  if (c.elem == ElemF16::code) {        \
    UGBSA_EV_D(ElemF16, K_);            \
  } else {                              \
    UGBSA_EV_D(ElemBf16, K_);           \
  }
  if (c.kind == kPagesE2m1) {
    UGBSA_EV_E(kPagesE2m1)
  } else if (c.kind == kPagesE4m3) {
    UGBSA_EV_E(kPagesE4m3)
  } else {
    UGBSA_EV_E(kPagesModel)
  }
  return hipErrorInvalidValue;
}

}  // namespace ugbsa
