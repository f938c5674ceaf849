// Eviction from the paged cache by accumulated attention weight: per (sequence, KV head)
// the first tokens, the newest and, of the others, the heaviest, packed in their order
// into other pages.
//
// Picking reads a row's weights a few times over (4 bytes a token, from L2 after the
// first); moving copies the kept tokens' codes, 2 token bytes each way.
#include "paged.h"

namespace ugbsa {

constexpr int kPickBins = 2048;        // 11, 11 and 10 bits of the key

// Order of the tokens that compete, larger first: NaN, then by weight, zeros of either
// sign alike.
constexpr uint32_t kPickNan = 0xFFFFFFFEu, kPickInf = 0xFF800000u;
__device__ __forceinline__ uint32_t pick_key(float x) { return x != x ? kPickNan : float_key(x + 0.f); }

// Top digits of four weights, in the order of their bits (the scan of the bins puts them in
// that of the keys): -0 as 0, NaN as the top bin.
__device__ __forceinline__ void top_digits(f32x4 x, uint32_t* d) {
  const float any = x[0] + x[1] + x[2] + x[3];
  const bool nan = __ballot(any != any) != 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    d[j] = __float_as_uint(x[j] + 0.f) >> 21;
    if (nan && x[j] != x[j]) d[j] = 0x3FFu;
  }
}

// Whether the wavefront's digits are one, as those of tokens that were never looked at.
__device__ __forceinline__ bool one_digit(const uint32_t* d) {
  const uint32_t d0 = __builtin_amdgcn_readfirstlane(d[0]);
  return __ballot(d[0] != d0) == 0 && __ballot(d[1] != d0 || d[2] != d0 || d[3] != d0) == 0;
}

// Weights that nothing was added to are zeros, often most of a row's, and 64 lanes that add to one
// word of LDS do so one behind the other: 128 rows of 32K tokens, 5 in 100 of them not 0, 126 us
// so and 75 with the lanes that agree found first (zeros alone 105 and 69).  Among
// weights over many binades the search would cost 5 in 100 of the call.  Whether enough agree:
__device__ __forceinline__ bool many(uint64_t lanes) { return __builtin_popcountll(lanes) >= 24; }
__device__ __forceinline__ bool alike_digits(const uint32_t* d) {
  return many(__ballot(d[0] == __builtin_amdgcn_readfirstlane(d[0])));
}


// One more in its bin for each lane with `in`; the lane's place there.  The lanes that agree with the
// first of them go with one addition.
__device__ __forceinline__ uint32_t add_to_bin(uint32_t* hist, uint32_t bin, bool in, int lane) {
  const uint64_t have = __ballot(in);
  if (have == 0) return 0u;
  const int lead = __builtin_ctzll(have);
  const uint32_t one = __builtin_amdgcn_readlane(bin, lead);
  const uint64_t same = __ballot(in && bin == one);
  uint32_t at = 0u;
  if (lane == lead) at = atomicAdd(&hist[one], static_cast<uint32_t>(__builtin_popcountll(same)));
  at = __builtin_amdgcn_readlane(at, lead) + lanes_below(same);
  if (in && bin != one) at = atomicAdd(&hist[bin], 1u);
  return at;
}

// A row cut into parts of kPickPart tokens, a workgroup each, and what a part leaves for the
// others: how many of its competing tokens each bin of the top digit holds and where they
// begin, two bins a word; how many tokens stay in any case, and whether a page is absent; and
// the keys, bin by bin.  Of 2048 / 4096 / 8192 tokens, us of a call with the move: 64 rows of 32K
// 52.6 / 43.0 / 41.8 (nearly all alike in their top digit 82 / 60 / 72), 4 of 32K 25.6 / 25.9 / 29.1 (43
// / 44 / 61), 4 of 64K 28.3 / 26.9 / 29.9, 64 of 64K 83 / 60 / 52.
constexpr int kPickPart = 4096, kPickWords = kPickBins / 2;
constexpr int kPickStarts = kPickWords, kPickStay = 2 * kPickWords, kPickKeys = kPickStay + 4;
constexpr int kPickRecord = kPickKeys + kPickPart;
constexpr int kPickMaxParts = 512;

__global__ __launch_bounds__(kPickPart / 8) void paged_digits_kernel(
    const float* __restrict__ mass, int64_t sm_b, int64_t sm_h, const int32_t* __restrict__ lens,
    const int32_t* __restrict__ table, int64_t st_b, int max_pages, int num_pages, int recent, int first,
    int Hk, int rows, int parts, uint32_t* __restrict__ records) {
  constexpr int THREADS = kPickPart / 8, WAVES = THREADS / 64, EACH = kPickBins / THREADS;
  __shared__ uint32_t s_hist[kPickBins], s_keys[kPickPart], s_wave[WAVES], s_stay;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.x % rows, part = blockIdx.x / rows, g = row % Hk, b = row / Hk;
  const int n = cached_len(lens, b, max_pages), t0 = part * kPickPart;
  if (t0 >= n) return;
  const int t1 = min(n - t0, kPickPart) + t0, c0 = min(first, n), c1 = max(n - recent, c0);
  mass += b * sm_b + g * sm_h;
  table += b * st_b;
  f32x4 x[2];
#pragma unroll
  for (int r = 0; r < 2; ++r)
    x[r] = *reinterpret_cast<const f32x4*>(mass + min(t0 + 4 * (tid + THREADS * r), (n - 1) & ~3));
  auto there = [&](int page) { return page >= 0 && page < num_pages; };
  const int page0 = t0 / kBlock + tid;
  const bool gap = page0 < (t1 + kBlock - 1) / kBlock && !there(table[page0]);
#pragma unroll
  for (int j = 0; j < EACH; ++j) s_hist[tid + THREADS * j] = 0u;
  if (tid == 0) s_stay = 0u;
  const bool absent = __builtin_amdgcn_readfirstlane(__syncthreads_or(gap)) != 0;
  // each token's bin and its place in it
  uint32_t stay = 0u, d[2][4], rank[2][4];
  bool in[2][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = t0 + 4 * (tid + THREADS * r), i0 = __builtin_amdgcn_readfirstlane(i);
    top_digits(x[r], d[r]);
    const bool all = i0 >= c0 && i0 + 256 <= c1 && !absent;
    const bool page = all || (i < n && there(table[i / kBlock]));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool mid = i + j >= c0 && i + j < c1;
      in[r][j] = page && mid;
      stay += page && !mid && i + j < n ? 1u : 0u;
    }
    if (all && one_digit(d[r])) {
      uint32_t at = 0u;
      if (lane == 0) at = atomicAdd(&s_hist[d[r][0]], 256u);
      at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
      for (int j = 0; j < 4; ++j) rank[r][j] = at + 4 * lane + j;
    } else if (alike_digits(d[r])) {
#pragma unroll
      for (int j = 0; j < 4; ++j) rank[r][j] = add_to_bin(s_hist, d[r][j], in[r][j], lane);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (in[r][j]) rank[r][j] = atomicAdd(&s_hist[d[r][j]], 1u);
    }
  }
  if (stay != 0u) atomicAdd(&s_stay, stay);
  __syncthreads();
  uint32_t* const rec = records + (static_cast<int64_t>(row) * parts + part) * kPickRecord;
  uint32_t h[EACH], sum = 0u;
#pragma unroll
  for (int j = 0; j < EACH; ++j) sum += h[j] = s_hist[EACH * tid + j];
  const uint32_t ex = wave_excl_scan(sum, lane);
  if (lane == 63) s_wave[wave] = ex + sum;
  __syncthreads();
  uint32_t at = ex, total = 0u;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) at += w < wave ? s_wave[w] : 0u, total += s_wave[w];
#pragma unroll
  for (int j = 0; j < EACH; j += 2) {
    rec[(EACH * tid + j) / 2] = h[j] | h[j + 1] << 16;
    rec[kPickStarts + (EACH * tid + j) / 2] = at | (at + h[j]) << 16;
    s_hist[EACH * tid + j] = at, s_hist[EACH * tid + j + 1] = at + h[j];
    at += h[j] + h[j + 1];
  }
  if (tid == 0) rec[kPickStay] = s_stay, rec[kPickStay + 1] = absent ? 1u : 0u;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (in[r][j]) s_keys[s_hist[d[r][j]] + rank[r][j]] = pick_key(x[r][j]);
  __syncthreads();
  for (uint32_t i = 4 * tid; i < total; i += 4 * THREADS)
    *reinterpret_cast<u32x4*>(rec + kPickKeys + i) = *reinterpret_cast<const u32x4*>(s_keys + i);
}

// One workgroup per (KV head, sequence), or, with PARTS, per part of its tokens.  The first
// tokens and the newest stay; of the others, c0 .. c1 - 1, the `want` largest do: a histogram of
// their keys' top digit, then of the lower ones over the keys of the cut's bin, which are
// listed in LDS where it holds them, fewer digits where the cut falls between two bins.  Then
// each wavefront goes over a run of the row's pages, a token a lane, counts what it keeps and
// writes it behind the others'.
//
// A whole row is one CU's, and its instructions bound it: how many (a pass over 32K tokens at
// 40 of them per 64 tokens took 8.6 us), and that they are fetched (loops unrolled over loads
// in flight are code that runs once).  So rows of up to ROW tokens are copied to LDS and gone
// over by small loops; four tokens a lane and load; membership in a bin, and in what stays, by
// comparing weights with its ends, not keys; what is the same for all lanes in scalar
// registers; and what only some tokens need (ends of the range, absent pages, NaN) behind
// scalar branches.
//
// With PARTS the launch before has counted and sorted each part by the top digit.  Every
// workgroup adds the counts up, and finds the same cut in the row's keys of one bin; it goes
// over its own tokens alone.  A read of what that launch left takes over 1 us, whoever wrote
// it, so 16 parts' counts are on the way at once (four at once: 23 us for 4 rows of 128K
// tokens where this takes 14).
//
// 64 rows of up to 32K tokens (2.6 MB) 9 us and 15, whole 26.7; four of 600 8.5.
template <int ROW, int kPickThreads, bool PARTS = false>
__global__ __launch_bounds__(kPickThreads) void paged_pick_kernel(
    const float* __restrict__ mass, int64_t sm_b, int64_t sm_h, const int32_t* __restrict__ lens,
    const int32_t* __restrict__ table, int64_t st_b, int max_pages, int num_pages, int keep, int recent, int first,
    int32_t* __restrict__ kept, int32_t* __restrict__ new_lens, int Hk, int rows, int max_parts,
    const uint32_t* __restrict__ records) {
  static_assert(!PARTS || (ROW == 0 && kPickMaxParts <= kPickThreads), "parts are read where they are, a thread each");
  constexpr int kPickWaves = kPickThreads / 64, kEach = kPickBins / kPickThreads;
  constexpr int kPickList = PARTS ? 1 : ROW == 0 || ROW > 4096 ? 4096 : ROW;       // keys of the cut's bin that are listed
  __shared__ uint32_t s_hist[kPickBins], s_list[kPickList], s_wave[4][kPickWaves], s_found[3], s_listed, s_stay;
  __shared__ uint8_t s_from[kPickList];
  __shared__ uint32_t s_seg[PARTS ? kPickMaxParts : 1];                // first key and number of the cut's bin, of each part
  __shared__ f32x4 s_row[ROW > 0 ? ROW / 4 : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.x % rows, part = PARTS ? blockIdx.x / rows : 0, g = row % Hk, b = row / Hk;
  const int n = cached_len(lens, b, max_pages), t0 = part * kPickPart;
  if (PARTS && part > 0 && t0 >= n) return;
  const int c0 = min(first, n), c1 = max(n - recent, c0);
  mass += b * sm_b + g * sm_h;
  table += b * st_b;
  int32_t* out = kept + static_cast<int64_t>(row) * keep;

  const int pages = (n + kBlock - 1) / kBlock;
  auto there = [&](int page) { return page >= 0 && page < num_pages; };
  if constexpr (ROW > 0) {
    for (int i = 4 * tid; i < n; i += 16 * kPickThreads) {
      f32x4 x[4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        x[r] = *reinterpret_cast<const f32x4*>(mass + min(i + 4 * kPickThreads * r, (n - 1) & ~3));
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (i + 4 * kPickThreads * r < n) s_row[i / 4 + kPickThreads * r] = x[r];
    }
  }
  bool gap = false;                                   // a page of the row is absent
  const int parts = (n + kPickPart - 1) / kPickPart, hi_bin = kPickBins - 1 - kEach * tid;  // this thread's largest bin
  const bool positive = hi_bin >= kPickBins / 2;
  auto held = [&](int bin) { return bin >= kPickBins / 2 ? bin - kPickBins / 2 : kPickBins - 1 - bin; };   // of pass 0
  uint32_t whole[4] = {}, others[4] = {};     // this thread's bins: of the row, of the parts before
  int stay = 0, base = 0;                             // that stay in any case: of the row, of the parts before
  if constexpr (PARTS) {
    records += static_cast<int64_t>(row) * max_parts * kPickRecord;
    for (int p = lane; p < parts; p += 64) {
      const uint32_t* rec = records + static_cast<int64_t>(p) * kPickRecord + kPickStay;
      const int x = rec[0];
      stay += x;
      base += p < part ? x : 0;
      gap |= rec[1] != 0u;
    }
    // (two words of a record: this thread's four bins, from the lesser raw digit)
    static_assert(!PARTS || kEach == 4, "four bins a thread");
    const uint32_t* mine_at = records + held(positive ? hi_bin - 3 : hi_bin) / 2;
    for (int p0 = 0; p0 < parts; p0 += 16) {
      u32x2 y[16];
#pragma unroll
      for (int r = 0; r < 16; ++r)
        y[r] = *reinterpret_cast<const u32x2*>(mine_at + static_cast<int64_t>(min(p0 + r, parts - 1)) * kPickRecord);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const uint32_t all = p0 + r < parts ? ~0u : 0u, prior = p0 + r < part ? ~0u : 0u;
        const uint32_t z[4] = {y[r][0] & 0xFFFFu, y[r][0] >> 16, y[r][1] & 0xFFFFu, y[r][1] >> 16};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t x = z[j];
          whole[j] += x & all, others[j] += x & prior;
        }
      }
    }
    if (positive) {                                   // their bins fall as the digits rise
      const uint32_t w[4] = {whole[3], whole[2], whole[1], whole[0]}, o[4] = {others[3], others[2], others[1], others[0]};
#pragma unroll
      for (int j = 0; j < 4; ++j) whole[j] = w[j], others[j] = o[j];
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) stay += __shfl_xor(stay, off, 64), base += __shfl_xor(base, off, 64);
    stay = __builtin_amdgcn_readfirstlane(stay), base = __builtin_amdgcn_readfirstlane(base);
  } else {
    for (int p = tid; p < pages; p += kPickThreads) gap |= !there(table[p]);
  }
  for (int i = tid; i < kPickBins; i += kPickThreads) s_hist[i] = 0u;
  if (tid == 0) s_listed = 0u, s_stay = 0u;
  const bool absent = __builtin_amdgcn_readfirstlane(__syncthreads_or(gap)) != 0;

  // four weights from token i on (the row's last four where it ends before)
  constexpr int RUN = ROW > 0 ? 1 : 4;                // loads in flight together
  auto weights = [&](int i) __attribute__((always_inline)) {
    const int at = min(i, (n - 1) & ~3);
    if constexpr (ROW > 0) return s_row[at / 4];
    else return *reinterpret_cast<const f32x4*>(mass + at);
  };
  // f(four weights of the lane, masks of the lanes whose j-th competes, whether all do), 256 tokens a time
  auto visit = [&](auto f) __attribute__((always_inline)) {
#pragma unroll 1
    for (int w0 = (c0 & ~3) + 256 * wave; w0 < c1; w0 += 4 * RUN * kPickThreads) {
      f32x4 x[RUN];
#pragma unroll
      for (int r = 0; r < RUN; ++r) x[r] = weights(w0 + 4 * kPickThreads * r + 4 * lane);
#pragma unroll
      for (int r = 0; r < RUN; ++r) {
        const int i0 = w0 + 4 * kPickThreads * r, i = i0 + 4 * lane;
        if (i0 >= c1) break;
        uint64_t in[4] = {~0ull, ~0ull, ~0ull, ~0ull};
        const bool all = i0 >= c0 && i0 + 256 <= c1 && !absent;
        if (!all) {
          const bool page = i < n && there(table[i / kBlock]);
#pragma unroll
          for (int j = 0; j < 4; ++j) in[j] = __ballot(page && i + j >= c0 && i + j < c1);
        }
        f(x[r], in, all);
      }
    }
  };
  auto mine = [&](uint64_t m) { return (m >> lane & 1) != 0; };
  // this wavefront's runs of 256 tokens: of the row, and of the part, whose tokens it writes
  const int runs = (n + 255) / 256, share = (runs + kPickWaves - 1) / kPickWaves;
  const int q0 = min(wave * share, runs), q1 = min(q0 + share, runs);
  constexpr int PART_RUNS = kPickPart / 256, PART_SHARE = (PART_RUNS + kPickWaves - 1) / kPickWaves;
  const int w0 = PARTS ? min(t0 / 256 + wave * PART_SHARE, runs) : q0, w1 = PARTS ? min(w0 + PART_SHARE, runs) : q1;
  // f(first of 256 tokens, the lane's first, its four weights) over runs r0 .. r1 - 1
  auto run_over = [&](int r0, int r1, auto f) __attribute__((always_inline)) {
#pragma unroll 1
    for (int at = r0; at < r1; at += RUN) {
      f32x4 x[RUN];
#pragma unroll
      for (int r = 0; r < RUN; ++r) x[r] = weights(256 * (at + r) + 4 * lane);
#pragma unroll
      for (int r = 0; r < RUN; ++r) {
        if (at + r >= r1) break;
        f(256 * (at + r), 256 * (at + r) + 4 * lane, x[r]);
      }
    }
  };
  // over the cut's bin of the first `upto` parts: f(key, whether many of the wavefront's agree in these
  // bits), or all(key, how many) where all that it has at once do (4 rows of 128K zeros: a load and a
  // search after the other 229 us, so 63)
  constexpr uint32_t SEG = 8;
  auto segments = [&](int upto, uint32_t bits, auto all, auto f) __attribute__((always_inline)) {
#pragma unroll 1
    for (int p = wave; p < upto; p += kPickWaves) {
      const uint32_t seg = s_seg[p], size = seg >> 16;
      const uint32_t* keys = records + static_cast<int64_t>(p) * kPickRecord + kPickKeys + (seg & 0xFFFFu);
      uint32_t i = 0;
#pragma unroll 1
      for (; i + 64 * SEG <= size; i += 64 * SEG) {             // SEG loads on the way together
        uint32_t k[SEG], other = 0u;
#pragma unroll
        for (uint32_t j = 0; j < SEG; ++j) k[j] = keys[i + 64 * j + lane];
        const uint32_t one = __builtin_amdgcn_readfirstlane(k[0]);
#pragma unroll
        for (uint32_t j = 0; j < SEG; ++j) other |= k[j] ^ one;
        if (__ballot((other & bits) != 0u) == 0) {
          all(one, 64 * SEG);
          continue;
        }
        const bool alike = many(__ballot(((k[0] ^ one) & bits) == 0u));
#pragma unroll
        for (uint32_t j = 0; j < SEG; ++j) f(k[j], alike);
      }
#pragma unroll 1
      for (i += lane; i < size; i += 64) {
        const uint32_t k = keys[i];
        f(k, many(__ballot(((k ^ __builtin_amdgcn_readfirstlane(k)) & bits) == 0u)));
      }
    }
  };
  int more = 0, same = 0;                             // of this lane's: above the cut, and tied

  uint32_t prefix = 0u, mask = 0u, want = 0u;        // want-th largest among the keys of the prefix
  uint32_t least = 0u, ties = 0u;                     // keys above least stay, and the first ties equal to it
  uint32_t top = 0u;                                  // keys of the cut's bin of the top digit
  int total = 0;                                      // tokens with a page
  int sure = kPickBins;                               // tokens of this bin of the top digit and those above stay
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bins = pass == 2 ? 1024 : kPickBins;
    if (pass == 0) {
      if constexpr (!PARTS) {
        if (absent) {                                 // those that stay and are there
          uint32_t have = 0u;
          for (int i = tid; i < n - (c1 - c0); i += kPickThreads) {
            const int t = i < c0 ? i : i + (c1 - c0);
            have += there(table[t / kBlock]) ? 1u : 0u;
          }
          if (have != 0u) atomicAdd(&s_stay, have);
        }
        visit([&](f32x4 x, const uint64_t* in, bool all) __attribute__((always_inline)) {
          uint32_t d[4];
          top_digits(x, d);
          const bool alike = alike_digits(d);
          if (alike && all && one_digit(d)) {
            if (lane == 0) atomicAdd(&s_hist[d[0]], 256u);
            return;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (alike) add_to_bin(s_hist, d[j], mine(in[j]), lane);
            else if (mine(in[j])) atomicAdd(&s_hist[d[j]], 1u);
          }
        });
      }
    } else if (PARTS) {
      segments(parts, mask | static_cast<uint32_t>(bins - 1) << shift, [&](uint32_t k, uint32_t n) {
        if ((k & mask) == prefix && lane == 0) atomicAdd(&s_hist[(k >> shift) & (bins - 1)], n);
      }, [&](uint32_t k, bool alike) __attribute__((always_inline)) {
        const bool one = (k & mask) == prefix;
        if (alike) add_to_bin(s_hist, (k >> shift) & (bins - 1), one, lane);
        else if (one) atomicAdd(&s_hist[(k >> shift) & (bins - 1)], 1u);
      });
    } else if (top <= kPickList) {
      const uint32_t listed = min(s_listed, static_cast<uint32_t>(kPickList));
      for (uint32_t i = tid; i < listed; i += kPickThreads) {
        const uint32_t k = s_list[i];
        add_to_bin(s_hist, (k >> shift) & (bins - 1), (k & mask) == prefix, lane);
      }
    } else {
      visit([&](f32x4 x, const uint64_t* in, bool) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t k = pick_key(x[j]);
          add_to_bin(s_hist, (k >> shift) & (bins - 1), mine(in[j]) && (k & mask) == prefix, lane);
        }
      });
    }
    __syncthreads();
    // bins from the largest: thread t holds kEach from 2047 - kEach t down; the bits of a positive
    // weight's key are its own but for the sign, those of a negative one's turned
    uint32_t h[kEach], sum = 0u;
#pragma unroll
    for (int j = 0; j < kEach; ++j) sum += h[j] = PARTS && pass == 0 ? whole[j & 3] : s_hist[pass > 0 ? hi_bin - j : held(hi_bin - j)];
    const uint32_t ex = wave_excl_scan(sum, lane);
    if (lane == 63) s_wave[0][wave] = ex + sum;
    __syncthreads();
    uint32_t before = ex;
    for (int w = 0; w < wave; ++w) before += s_wave[0][w];
    if (pass == 0) {
      if constexpr (!PARTS) stay = absent ? __builtin_amdgcn_readfirstlane(s_stay) : n - (c1 - c0);
      uint32_t all = 0u;
      for (int w = 0; w < kPickWaves; ++w) all += s_wave[0][w];
      total = stay + __builtin_amdgcn_readfirstlane(all);
      want = keep - stay;
      if (total <= keep) sure = 0;
      if (total <= keep || want == 0u) break;         // all that compete stay, or none
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      if (before < want && want <= before + h[j]) s_found[0] = hi_bin - j, s_found[1] = before, s_found[2] = h[j];
      before += h[j];
    }
    for (int i = tid; i < kPickBins; i += kPickThreads) s_hist[i] = 0u;
    __syncthreads();
    prefix |= static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(s_found[0])) << shift;
    mask |= static_cast<uint32_t>(bins - 1) << shift;
    want -= __builtin_amdgcn_readfirstlane(s_found[1]);
    const uint32_t bin = __builtin_amdgcn_readfirstlane(s_found[2]);
    least = prefix, ties = want;
    if (pass == 0) sure = static_cast<int>(prefix >> 21) + (want == bin ? 0 : 1);
    if (want == bin) {                                // the whole bin stays
      least = prefix - 1u, ties = 0u;
      break;
    }
    if (pass == 0) {
      top = bin;
      // the bin's keys, and what each wavefront holds above the bin
      const bool finite = prefix >= ~kPickInf && prefix < kPickInf, fits = top <= kPickList;
      const float lo = key_float(prefix), end = key_float(prefix + (1u << 21));
      if constexpr (PARTS) {
        if (tid < parts) {
          const uint32_t* rec = records + static_cast<int64_t>(tid) * kPickRecord;
          const int at = held(prefix >> 21), sh = 16 * (at & 1);
          s_seg[tid] = (rec[kPickStarts + at / 2] >> sh & 0xFFFFu) | (rec[at / 2] >> sh & 0xFFFFu) << 16;
        }
      } else run_over(q0, q1, [&](int i0, int i, f32x4 x) __attribute__((always_inline)) {
        bool over[4], in[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          over[j] = !(x[j] < end);                            // finite: or NaN
          in[j] = x[j] >= lo && x[j] < end;
        }
        if (!finite) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t k = pick_key(x[j]);
            over[j] = (k & mask) > prefix, in[j] = (k & mask) == prefix;
          }
        }
        if (absent || i0 < c0 || i0 + 256 > c1) {             // not all of them compete, or are there
          const bool page = i < n && there(table[i / kBlock]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool have = page && i + j < n, mid = i + j >= c0 && i + j < c1;
            over[j] = have && (over[j] || !mid);
            in[j] = in[j] && have && mid;
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) more += over[j] ? 1 : 0;
        if (!fits || __ballot(in[0] || in[1] || in[2] || in[3]) == 0) return;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (in[j]) {
            const uint32_t to = atomicAdd(&s_listed, 1u) % kPickList;
            s_list[to] = pick_key(x[j]);
            s_from[to] = static_cast<uint8_t>(wave);
          }
      });
    }
    __syncthreads();
  }
  const int count = min(total, keep);
  if (tid == 0 && g == 0 && part == 0) new_lens[b] = count;
  if (total > keep && want == 0u && ties == 0u && least == 0u) least = 0xFFFFFFFFu;   // none that compete
  __syncthreads();

  // In weights: keys above least are those not below `low`, or only NaN, or none; equal to it
  // those equal to `tie`, or NaN.
  const bool none = least >= kPickNan, only_nan = !none && least + 1u > kPickInf;
  const float low = total <= keep ? __uint_as_float(0x7FC00000u) : key_float(least + 1u), tie = key_float(least);
  const bool plain = !none && !only_nan && !absent;
  // f(the lane's first token, masks of the lanes whose j-th stays above the cut, and ties)
  auto pass_over = [&](int r0, int r1, auto f) __attribute__((always_inline)) {
    run_over(r0, r1, [&](int i0, int i, f32x4 x) __attribute__((always_inline)) {
      uint64_t gt[4], eq[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        gt[j] = __ballot(!(x[j] < low));
        eq[j] = ties != 0u ? __ballot(x[j] == tie) : 0;
      }
      if (!plain) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint64_t nan = __ballot(x[j] != x[j]);
          gt[j] = none ? 0 : (only_nan ? nan : gt[j]);
          eq[j] = ties != 0u && least == kPickNan ? nan : eq[j];
        }
      }
      if (absent || i0 < c0 || i0 + 256 > c1) {             // not all of them compete, or are there
        const bool page = i < n && there(table[i / kBlock]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint64_t have = __ballot(page && i + j < n), in = __ballot(i + j >= c0 && i + j < c1);
          gt[j] = have & (gt[j] | ~in);
          eq[j] &= have & in;
        }
      }
      f(i, gt, eq);
    });
  };
  auto count_over = [&](int r0, int r1, int& gts, int& eqs) __attribute__((always_inline)) {
    pass_over(r0, r1, [&](int, const uint64_t* gt, const uint64_t* eq) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) gts += mine(gt[j]) ? 1 : 0, eqs += mine(eq[j]) ? 1 : 0;
    });
  };
  const bool listed_all = total > keep && top != 0u && top <= kPickList;
  const uint32_t listed = listed_all ? min(s_listed, static_cast<uint32_t>(kPickList)) : 0u;
  int more0 = 0, same0 = 0;                           // and of the parts before
  if constexpr (PARTS) {
    count_over(w0, w1, more, same);
#pragma unroll
    for (int j = 0; j < kEach; ++j) more0 += hi_bin - j >= sure ? others[j & 3] : 0u;
    if (top != 0u)
      segments(part, ~0u, [&](uint32_t k, uint32_t n) {
        if (lane == 0) more0 += k > least ? n : 0, same0 += k == least ? n : 0;
      }, [&](uint32_t k, bool) __attribute__((always_inline)) {
        more0 += k > least ? 1 : 0, same0 += k == least ? 1 : 0;
      });
  } else if (listed_all) {
    // what the wavefront keeps: from the list where there is one
    for (uint32_t at = 0; at < listed; at += 64) {
      const bool own = at + lane < listed && s_from[min(at + lane, listed - 1u)] == wave;
      const uint32_t k = s_list[min(at + lane, listed - 1u)];
      more += own && k > least ? 1 : 0;
      same += own && k == least ? 1 : 0;
    }
  } else {
    more = 0;
    count_over(q0, q1, more, same);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    more += __shfl_xor(more, off, 64), same += __shfl_xor(same, off, 64);
    if constexpr (PARTS) more0 += __shfl_xor(more0, off, 64), same0 += __shfl_xor(same0, off, 64);
  }
  if (lane == 0) s_wave[0][wave] = more, s_wave[1][wave] = same;
  if (PARTS && lane == 0) s_wave[2][wave] = more0, s_wave[3][wave] = same0;
  __syncthreads();
  int at = base, tied = 0;                            // kept and tied tokens before this wavefront's
  for (int w = 0; w < wave; ++w) at += s_wave[0][w], tied += s_wave[1][w];
  if constexpr (PARTS)
    for (int w = 0; w < kPickWaves; ++w) at += s_wave[2][w], tied += s_wave[3][w];
  at = __builtin_amdgcn_readfirstlane(at + min(tied, static_cast<int>(ties)));
  tied = __builtin_amdgcn_readfirstlane(tied);
  pass_over(w0, w1, [&](int i, const uint64_t* gt, const uint64_t* eq) __attribute__((always_inline)) {
    uint64_t stay[4] = {gt[0], gt[1], gt[2], gt[3]};
    if (ties != 0u && tied < static_cast<int>(ties) && (eq[0] | eq[1] | eq[2] | eq[3]) != 0) {
      // the first `ties` of the row
      int rank = tied;
#pragma unroll
      for (int j = 0; j < 4; ++j) rank += lanes_below(eq[j]), tied += __builtin_popcountll(eq[j]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        stay[j] |= __ballot(mine(eq[j]) && rank < static_cast<int>(ties));
        rank += mine(eq[j]) ? 1 : 0;
      }
    }
    if ((stay[0] | stay[1] | stay[2] | stay[3]) == 0) return;
    int to = at;
#pragma unroll
    for (int j = 0; j < 4; ++j) to += lanes_below(stay[j]), at += __builtin_popcountll(stay[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (mine(stay[j])) {
        if (to < count) out[to] = i + j;
        ++to;
      }
  });
  const int end = max_pages * kBlock;
  if (part > 0) return;
  for (int i = count + tid; i < keep; i += kPickThreads) out[i] = end;
}

// One workgroup per (new page, KV head, sequence): it alone writes them.  A thread moves 8
// dims of every (256 / (D / 8))-th token; the summary is of the keys as they are stored.
// Bound by memory, with the latency of one read behind another (list, table, token): 64 rows of
// up to 4000 tokens, e4m3 (43 MB read, as much written) 19 us.
template <typename E, int D, int KIND>
__global__ __launch_bounds__(256) void paged_move_kernel(
    PagedCache c, const float* __restrict__ mass, int64_t sm_b, int64_t sm_h, const int32_t* __restrict__ table,
    int64_t st_b, int tokens, const int32_t* __restrict__ new_table, int64_t sn_b, const int32_t* __restrict__ kept,
    int keep, const int32_t* __restrict__ new_lens, float* __restrict__ new_mass, int64_t so_b, int64_t so_h) {
  constexpr int CH = D / 8, RG = 256 / CH, IT = kBlock / RG;
  __shared__ float red[2][RG][D + 1];
  __shared__ int s_slot[kBlock], s_page[kBlock];
  const int tid = threadIdx.x, ch = tid % CH, rg = tid / CH;
  const int j = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int count = min(new_lens[b] - j * kBlock, kBlock);        // tokens of this page
  if (tid < kBlock) {
    float x = 0.f;
    if (tid < count) {
      // (in range, and with a page, unless mass changed while the call ran)
      int token = kept[(static_cast<int64_t>(b) * gridDim.y + h) * keep + j * kBlock + tid];
      token = token < 0 || token >= tokens ? 0 : token;
      const int from = table[b * st_b + token / kBlock];
      s_slot[tid] = token % kBlock;
      s_page[tid] = from >= 0 && from < c.num_pages ? from : 0;
      x = mass[b * sm_b + h * sm_h + token];
    }
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
  Elem* const kp = static_cast<Elem*>(c.k) + h * c.sk_h + CB * ch;
  Elem* const vp = static_cast<Elem*>(c.v) + h * c.sv_h + CB * ch;
  // scales: one a token of e4m3, one a token and 32 dims of e2m1
  const int64_t groups = KIND == kPagesE2m1 ? D / 32 : 1;
  const int grp = KIND == kPagesE2m1 ? ch / 4 : 0;
  const bool holds = KIND == kPagesE2m1 ? ch % 4 == 0 : ch == 0;
  // the loads of up to AT tokens a thread, the whole page's up to head_dim 128, then their stores
  // (all eight of head_dim 256 took 456 registers: 16 rows of 16K tokens to 8000 in 16 bits 129 us,
  // now 83)
  constexpr int AT = IT < 4 ? IT : 4;
  words rk[AT], rv[AT];
  uint32_t bk[AT], bv[AT];
#pragma unroll 1
  for (int at = 0; at < IT; at += AT) {
#pragma unroll
    for (int it = 0; it < AT; ++it) {
      const int s = rg + RG * (at + it);
      if (s < count) {
        const int64_t from = s_page[s];
        const int slot = s_slot[s];
        rk[it] = *reinterpret_cast<const words*>(kp + from * c.sk_p + slot * c.sk_n);
        rv[it] = *reinterpret_cast<const words*>(vp + from * c.sv_p + slot * c.sv_n);
        if constexpr (KIND != kPagesModel) {
          const int64_t sc = ((from * c.Hk + h) * groups + grp) * kBlock + slot;
          bk[it] = c.k_scale[sc];
          bv[it] = c.v_scale[sc];
        }
      }
    }
#pragma unroll
    for (int it = 0; it < AT; ++it) {
      const int s = rg + RG * (at + it);
      if (s < count) {
        *reinterpret_cast<words*>(kp + page * c.sk_p + s * c.sk_n) = rk[it];
        *reinterpret_cast<words*>(vp + page * c.sv_p + s * c.sv_n) = rv[it];
        u32x4 x;
        if constexpr (KIND == kPagesModel) {
          x = u32x4{rk[it][0], rk[it][1], rk[it][2], rk[it][3]};
        } else {
          if (holds) {
            const int64_t sc = (head * groups + grp) * kBlock + s;
            c.k_scale[sc] = static_cast<uint8_t>(bk[it]);
            c.v_scale[sc] = static_cast<uint8_t>(bv[it]);
          }
          if constexpr (KIND == kPagesE4m3)
            x = __builtin_bit_cast(u32x4, e4m3_x8<E>(rk[it][0], rk[it][1], e8m0(bk[it])));
          else
            x = e2m1_x8<E>(rk[it][0], e8m0(bk[it]));
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

// Parts of a row, 0 where a workgroup has it whole.  Few long rows leave most CUs idle in that
// form; in this one each part reads the keys of the cut's bin in all parts, which may be most of the
// row.  us with the move, in parts / whole, of weights over many binades, all 0, and all within one
// bin: 4 rows of 64K tokens 27 / 47, 46 / 80, 59 / 73; of 128K 31 / 73, 63 / 134, 91 / 123; of 1M 125 /
// 371, 634 / 916, 1124 / 794; 64 of 32K 43 / 45, 54 / 61, 60 / 57; of 64K 60 / 58, 93 / 89, 120 / 83.  From
// 2048 parts on they lose: 64 rows of 128K 93 / 87, 210 / 148, 311 / 138; 16 of 512K 151 / 213, 555 /
// 474, 981 / 427.  128 rows of 32K take 122 and 110, 4 rows of 16K 30 and 29.
static int paged_evict_parts(int B, int Hk, int max_pages) {
  const int parts = (max_pages + kPickPart / kBlock - 1) / (kPickPart / kBlock);
  const int64_t rows = static_cast<int64_t>(B) * Hk;
  return max_pages > 256 && parts <= kPickMaxParts && rows <= 64 && rows * parts <= 1024 ? parts : 0;
}

int64_t paged_evict_ws_elems(int B, int Hk, int max_pages) {
  return B * static_cast<int64_t>(Hk) * paged_evict_parts(B, Hk, max_pages) * kPickRecord;
}

hipError_t launch_paged_evict(const PagedCache& c, const float* mass, int64_t sm_b, int64_t sm_h,
                              const int32_t* lens, const int32_t* table, int64_t st_b, int B, int max_pages,
                              const int32_t* new_table, int64_t sn_b, int new_pages, int keep, int recent, int first,
                              int32_t* kept, int32_t* new_lens, float* new_mass, int64_t so_b, int64_t so_h,
                              float* workspace, hipStream_t stream) {
  const int rows = B * c.Hk;
  if (const int parts = paged_evict_parts(B, c.Hk, max_pages); parts > 0) {
    uint32_t* const records = reinterpret_cast<uint32_t*>(workspace);
    paged_digits_kernel<<<rows * parts, kPickPart / 8, 0, stream>>>(mass, sm_b, sm_h, lens, table, st_b, max_pages,
                                                                    c.num_pages, recent, first, c.Hk, rows, parts,
                                                                    records);
    paged_pick_kernel<0, 512, true><<<rows * parts, 512, 0, stream>>>(
        mass, sm_b, sm_h, lens, table, st_b, max_pages, c.num_pages, keep, recent, first, kept, new_lens, c.Hk, rows,
        parts, records);
  } else {
    // Rows of up to 2048 tokens have four wavefronts, whose barriers are shorter and several of
    // which share a CU (512 rows of 1000 tokens 10.8 us, 128 of 4096 12.4; with 16 wavefronts the
    // 512 took 18.9); 8192 and 32768 weights fit the LDS of half a CU and of one.
    const int threads = max_pages <= 32 ? 256 : 1024;
    const auto pick = max_pages <= 32    ? paged_pick_kernel<2048, 256>
                      : max_pages <= 128 ? paged_pick_kernel<8192, 1024>
                      : max_pages <= 512 ? paged_pick_kernel<32768, 1024>
                                         : paged_pick_kernel<0, 1024>;
    pick<<<rows, threads, 0, stream>>>(mass, sm_b, sm_h, lens, table, st_b, max_pages, c.num_pages, keep, recent,
                                       first, kept, new_lens, c.Hk, rows, 0, nullptr);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid(new_pages, c.Hk, B);
#define UGBSA_EV(E_, D_, K_)                                                                                      \
  do {                                                                                                            \
    paged_move_kernel<E_, D_, K_><<<grid, 256, 0, stream>>>(c, mass, sm_b, sm_h, table, st_b, max_pages * kBlock,    \
                                                            new_table, sn_b, kept, keep, new_lens, new_mass, so_b, \
                                                            so_h);                                                \
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
