// Writing the paged key / value cache, and giving tokens of it up.
//
// Pages hold `page` tokens (a power of two) of all key heads, (pages, Hk, page, D) 16-bit
// numbers; a sequence's slot s lies in row s % page of page table[b, s / page].
#include "common.h"

#include <algorithm>

namespace qv {

struct PagedCache {
  uint16_t *k, *v;          // pages
  const int32_t* table;     // (B, slots)
  int32_t *lens, *evicted;  // (B)
  float* weights;           // (B, Hk, slots * page); NULL: not kept, nor positions and evicted
  int32_t* positions;
  int B, Hk, slots, pages, page_log2;
  __device__ __forceinline__ long cap() const { return (long)slots << page_log2; }
  // index of slot `at`'s row of head hk, in rows of D; -1 where it has no page
  __device__ __forceinline__ long row(int b, int hk, int at) const {
    const int i = at >> page_log2;
    const int p = i < slots ? table[(long)b * slots + i] : -1;
    if ((uint32_t)p >= (uint32_t)pages) return -1;
    return (((long)p * Hk + hk) << page_log2) + (at & ((1 << page_log2) - 1));
  }
};

// ------------------------------------------------------------------ append
// A thread moves 16 bytes of a key and of a value at a time, in the order of the source.  8 x up to 2900
// packed tokens of 8 heads of 128 into pages of 16: 21 us, 4.5 TB/s; one token for each of 32 sequences
// 3.5 us, launch and three dependent reads.
template <int D>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedCache c, const uint16_t* __restrict__ k,
                                                           const uint16_t* __restrict__ v, const int32_t* start_in,
                                                           const int32_t* counts, const int32_t* cu, int n, long T,
                                                           uint32_t* tickets, int chunk, long k_bs, long k_ts, long k_hs,
                                                           long v_bs, long v_ts, long v_hs) {
  constexpr int U = D / 8;                       // 16-byte units of a row
  const int b = blockIdx.y, tid = threadIdx.x;
  const int cap = (int)c.cap();
  int start = start_in[b];
  start = start < 0 ? 0 : start > cap ? cap : start;
  long tok0 = 0;
  int cnt;
  if (cu) {
    long lo = cu[b], hi = cu[b + 1];
    lo = lo < 0 ? 0 : lo > T ? T : lo;
    hi = hi < lo ? lo : hi > T ? T : hi;
    tok0 = lo, cnt = (int)(hi - lo);
  } else {
    cnt = counts ? counts[b] : n;
    cnt = cnt < 0 ? 0 : cnt > n ? n : cnt;
  }
  if (cnt > cap - start) cnt = cap - start;
  const int per = c.Hk * U;                      // units of a token
  for (long t0 = (long)blockIdx.x * chunk; t0 < cnt; t0 += (long)gridDim.x * chunk) {
    const int toks = (int)(cnt - t0 < chunk ? cnt - t0 : chunk);
    for (long u = tid; u < (long)toks * per; u += 256) {
      const int t = (int)(t0 + u / per), w = (int)(u % per), hk = w / U, d = 8 * (w % U);
      const long to = c.row(b, hk, start + t);
      if (to < 0) continue;
      const long tok = tok0 + t;
      const uint4 x = ld_stream16(k + b * k_bs + tok * k_ts + hk * k_hs + d);
      const uint4 y = ld_stream16(v + b * v_bs + tok * v_ts + hk * v_hs + d);
      *reinterpret_cast<uint4*>(c.k + to * D + d) = x;
      *reinterpret_cast<uint4*>(c.v + to * D + d) = y;
    }
  }
  if (c.weights) {
    // of the new tokens only: what lies in front of them, slots between lens and start among it, is the program's
    const int gone = c.evicted[b];
    for (long t0 = (long)blockIdx.x * chunk; t0 < cnt; t0 += (long)gridDim.x * chunk) {
      const int toks = (int)(cnt - t0 < chunk ? cnt - t0 : chunk);
      for (int i = tid; i < toks * c.Hk; i += 256) {
        const int hk = i / toks, at = start + (int)t0 + i % toks;
        const long to = ((long)b * c.Hk + hk) * cap + at;
        c.weights[to] = 0.f;
        c.positions[to] = at + gone;
      }
    }
  }
  // The length is written when all workgroups of the sequence have read it (as the start or the
  // count): by the last one, found by a ticket that wraps to 0 by itself.
  const bool turn = start_in == c.lens || counts == c.lens;
  if (turn) __syncthreads();
  if (tid == 0) {
    const bool last = !turn ? blockIdx.x == 0
                            : gridDim.x == 1 || atomicInc(tickets + (size_t)b * QV_PAGED_TICKETS, gridDim.x - 1) == gridDim.x - 1;
    if (last) c.lens[b] = start + cnt;
  }
}

// ------------------------------------------------------------------ evict
// Weights as whole numbers in their order: NaN lowest, protected tokens highest (above +inf): all but
// the span from first on.
__device__ __forceinline__ uint32_t evict_key(float w, int pos, uint32_t first, uint32_t span) {
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);       // -0 as 0
  const uint32_t k = u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
  return (uint32_t)pos - first >= span ? 0xFFFFFFFFu : w == w ? k : 0u;
}

constexpr int EVICT_THREADS = 1024, EVICT_WAVES = EVICT_THREADS / 64, EVICT_BINS = 2048;

// Sum over the lanes up to this one.
__device__ __forceinline__ int evict_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);   // inside rows of 16 lanes
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // the last lanes of the rows below
  return x;
}

// Sums over the waves below this one of their numbers, and of all; waves: each call's own words.
template <int N>
__device__ __forceinline__ void evict_below(int (&mine)[N], int (&all)[N], int* waves, int wave, int lane) {
  if (lane == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) waves[n * EVICT_WAVES + wave] = mine[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    mine[n] = all[n] = 0;
#pragma unroll
    for (int w = 0; w < EVICT_WAVES; ++w) {
      const int x = waves[n * EVICT_WAVES + w];
      mine[n] += w < wave ? x : 0;
      all[n] += x;
    }
  }
}

// 2112 tokens of 8 x 8 heads 9.0 us, some 14 barriers and what waits behind each; 32976 tokens of 16 heads
// 24.3 us on 16 CUs: 5 for reading by one CU each, 1 to 3 for each digit, 4 for each of the two walks at the
// end.  Steps that reach past the end, or over keep, have code of their own, others look at nothing but
// the keys (40 % fewer instructions, with the sums of a wave by DPP and one barrier for each sum over the
// waves 27 -> 24.3); flags kept from the first walk for the second gained nothing; 8-bit digits with a counter
// array for each wave, keys from memory each time and two barriers for every 1024 slots ranked: 48.7 and 141 us.
// A workgroup decides for one sequence and head.  The keep-th largest key comes from three
// counts of digits of 11, 11 and 10 bits: the first holds two bits of the mantissa, so that weights
// of a few powers of two spread over enough counters.  Then each wave takes a range of slots in order: which keys
// equal to the keep-th stay (the first ones), then the slots below keep that are given up (holes) and
// the kept ones behind, as ranks: moves[i] = (hole i, kept slot i).  head[.] = (number of moves, tokens).
// KEYS: as many keys are kept in LDS (0: made again from weights and positions each time).
template <int KEYS>
__global__ __launch_bounds__(EVICT_THREADS) void paged_evict_select_kernel(const PagedCache c, int keep, int recent, int first,
                                                                            int2* head, int2* moves, long most) {
  __shared__ __attribute__((aligned(16))) uint32_t keys[KEYS > 0 ? KEYS : 4];
  __shared__ int hist[EVICT_BINS];
  __shared__ __attribute__((aligned(16))) int waves[6 * EVICT_WAVES];       // of three digits, ties, holes and kept ones
  __shared__ int found[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hk = blockIdx.x, b = blockIdx.y;
  const long at = (long)b * c.Hk + hk;
  const int cap = (int)c.cap();
  int len = c.lens[b];
  len = len < 0 ? 0 : len > cap ? cap : len;
  if (len <= keep) {
    if (tid == 0) head[at] = make_int2(0, len);
    return;
  }
  const float* w = c.weights + at * cap;         // 16-byte aligned: cap is a multiple of 16
  const int32_t* pos = c.positions + at * cap;
  const long recent_from = (long)len + c.evicted[b] - recent;
  const uint32_t span = recent_from > first ? (uint32_t)(recent_from - first) : 0;
  // keys of the four slots from i (a multiple of 4) on, 0 behind len (the capacity has them)
  auto make_of = [&](const float4& x, const int4& p) __attribute__((always_inline)) {
    return make_uint4(evict_key(x.x, p.x, first, span), evict_key(x.y, p.y, first, span),
                      evict_key(x.z, p.z, first, span), evict_key(x.w, p.w, first, span));
  };
  auto make = [&](int i) __attribute__((always_inline)) {
    return make_of(*reinterpret_cast<const float4*>(w + i), *reinterpret_cast<const int4*>(pos + i));
  };
  for (int i = tid; i < EVICT_BINS; i += EVICT_THREADS) hist[i] = 0;
  __syncthreads();
  // the first digits are counted on the way; the reads of four steps go out together
  constexpr int STEP = 4 * EVICT_THREADS;
  auto walk = [&](int i0, auto whole) __attribute__((always_inline)) {        // whole: all slots are below len
    constexpr bool WHOLE = decltype(whole)::value;
    float4 x[4];
    int4 p[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = WHOLE || i0 + e * STEP < len ? i0 + e * STEP : 0;
      x[e] = *reinterpret_cast<const float4*>(w + i), p[e] = *reinterpret_cast<const int4*>(pos + i);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + e * STEP;
      if (WHOLE || i < len) {
        const uint4 u = make_of(x[e], p[e]);
        if constexpr (KEYS > 0) *reinterpret_cast<uint4*>(keys + i) = u;
        atomicAdd(&hist[u.x >> 21], 1);
        if (WHOLE || i + 1 < len) atomicAdd(&hist[u.y >> 21], 1);
        if (WHOLE || i + 2 < len) atomicAdd(&hist[u.z >> 21], 1);
        if (WHOLE || i + 3 < len) atomicAdd(&hist[u.w >> 21], 1);
      }
    }
  };
  for (int i0 = 0; i0 < len; i0 += 4 * STEP) {
    if (i0 + 4 * STEP <= len) walk(i0 + 4 * tid, std::true_type{});
    else walk(i0 + 4 * tid, std::false_type{});
  }
  __syncthreads();
  struct Four {
    uint32_t k[4];
    bool in[4];                                  // below len
  };
  auto all_four = [&](int i) __attribute__((always_inline)) {
    uint4 u;
    if constexpr (KEYS > 0) u = *reinterpret_cast<const uint4*>(keys + i);
    else u = make(i);
    return Four{{u.x, u.y, u.z, u.w}, {true, true, true, true}};
  };
  auto four = [&](int i, int end) __attribute__((always_inline)) {
    if (i >= end) return Four{};
    Four f = all_four(i);
#pragma unroll
    for (int e = 1; e < 4; ++e) f.in[e] = i + e < end;
    return f;
  };
  uint32_t prefix = 0, mask = 0;
  int left = keep;                               // kept tokens whose key has the prefix
  int same = 0;                                  // tokens that have it
  if (keep > 0) {
#pragma unroll
    for (int digit = 0; digit < 3; ++digit) {
      const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bins = digit == 2 ? 1024 : 2048;
      if (digit > 0) {
        for (int i = tid; i < EVICT_BINS; i += EVICT_THREADS) hist[i] = 0;
        __syncthreads();
        for (int i0 = 256 * wave; i0 < len; i0 += 4 * EVICT_THREADS) {
          const Four f = i0 + 256 <= len ? all_four(i0 + 4 * lane) : four(i0 + 4 * lane, len);
          bool in[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) in[e] = f.in[e] && (f.k[e] ^ prefix) <= ~mask;
          if (__builtin_amdgcn_ballot_w64(in[0] || in[1] || in[2] || in[3]) == 0) continue;      // few have the prefix
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (in[e]) atomicAdd(&hist[(f.k[e] >> shift) & (bins - 1)], 1);
        }
        __syncthreads();
      }
      // two counters a thread, the highest first: sums from above
      const int hi = EVICT_BINS - 1 - 2 * tid, n0 = hist[hi], n1 = hist[hi - 1];
      const int sum = evict_scan(n0 + n1);
      int lower[1] = {__builtin_amdgcn_readlane(sum, 63)}, total[1];
      evict_below(lower, total, waves + digit * EVICT_WAVES, wave, lane);
      const int above = lower[0] + sum - n0 - n1;
      if (above < left && above + n0 >= left) found[0] = hi, found[1] = left - above, found[2] = n0;
      else if (above + n0 < left && above + n0 + n1 >= left) found[0] = hi - 1, found[1] = left - above - n0, found[2] = n1;
      __syncthreads();
      prefix |= (uint32_t)found[0] << shift, left = found[1], same = found[2];
      mask |= (uint32_t)(bins - 1) << shift;
    }
  }
  // keys above the prefix stay, and the first `left` of those equal to it
  const int per = (len + 256 * EVICT_WAVES - 1) / (256 * EVICT_WAVES) * 256, lo = wave * per, hi = min(len, lo + per);
  // set bits of the four slots' ballots: all, and those of the lanes below
  auto count = [](const uint64_t (&m)[4]) { return __popcll(m[0]) + __popcll(m[1]) + __popcll(m[2]) + __popcll(m[3]); };
  auto before = [](const uint64_t (&m)[4]) {
    int n = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      n = __builtin_amdgcn_mbcnt_hi((uint32_t)(m[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m[e], n));
    return n;
  };
  const bool ties = left < same;                 // else all that are equal to it stay
  int equal = 0;
  if (ties)
    for (int i = lo + 4 * lane; i - 4 * lane < hi; i += 256) {
      const Four f = four(i, hi);
#pragma unroll
      for (int e = 0; e < 4; ++e) equal += __popcll(__builtin_amdgcn_ballot_w64(f.in[e] && f.k[e] == prefix));
    }
  if (ties) {
    int lower[1] = {equal}, total[1];
    evict_below(lower, total, waves + 3 * EVICT_WAVES, wave, lane);
    equal = lower[0];
  }
  // which of the four slots change: holes below keep, kept ones from there on (rank: keys equal to
  // the prefix so far)
  // the 256 slots from i0 on are on one side of keep, and all there
  auto even = [&](int i0) { return i0 + 256 <= hi && (i0 >= keep || i0 + 256 <= keep); };
  auto judge = [&](int i0, int& rank, bool (&on)[4], uint64_t (&ms)[4]) __attribute__((always_inline)) {
    const int i = i0 + 4 * lane;
    if (!ties && keep > 0 && even(i0)) {
      const Four f = all_four(i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        on[e] = (f.k[e] >= prefix) == (i0 >= keep);
        ms[e] = __builtin_amdgcn_ballot_w64(on[e]);
      }
      return;
    }
    const Four f = four(i, hi);
    int free = 4;                                // of the keys equal to the prefix, how many more may stay
    if (ties) {
      uint64_t eq[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) eq[e] = __builtin_amdgcn_ballot_w64(f.in[e] && f.k[e] == prefix);
      free = left - rank - before(eq);
      rank += count(eq);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool same = f.k[e] == prefix;
      const bool stays = keep > 0 && (f.k[e] > prefix || (same && free > 0));
      free -= same;
      on[e] = f.in[e] && stays == (i + e >= keep);
      ms[e] = __builtin_amdgcn_ballot_w64(on[e]);
    }
  };
  int holes = 0, kept = 0, rank = equal;
  bool on[4];
  uint64_t ms[4];
  // of the flags of 256 slots from i0 on: how many are holes
  auto below = [&](int i0, int all) __attribute__((always_inline)) {
    if (i0 + 256 <= keep) return all;
    if (i0 >= keep) return 0;
    int n = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) n += __popcll(__builtin_amdgcn_ballot_w64(on[e] && i0 + 4 * lane + e < keep));
    return n;
  };
  for (int i0 = lo; i0 < hi; i0 += 256) {
    judge(i0, rank, on, ms);
    const int all = count(ms), h = below(i0, all);
    holes += h, kept += all - h;
  }
  int lower[2] = {holes, kept}, total[2];
  evict_below(lower, total, waves + 4 * EVICT_WAVES, wave, lane);
  holes = lower[0], kept = lower[1];
  rank = equal;
  int* const to_of = reinterpret_cast<int*>(moves + at * most);
  const int limit = (int)most;                   // at most half the capacity
  for (int i0 = lo; i0 < hi; i0 += 256) {
    const int i = i0 + 4 * lane;
    judge(i0, rank, on, ms);
    const int all = count(ms);
    if (all == 0) continue;
    const int h = below(i0, all);
    int n = before(ms);                          // the holes come first
    if (even(i0)) {
      n += h ? holes : kept;
      int* const out = to_of + (h ? 0 : 1);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (on[e] && n < limit) out[2 * n] = i + e;
        n += on[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int to = i + e < keep ? holes + n : kept + n - h;
        if (on[e] && to < limit) to_of[2 * to + (i + e < keep ? 0 : 1)] = i + e;
        n += on[e];
      }
    }
    holes += h, kept += all - h;
  }
  if (tid == 0) head[at] = make_int2(total[1], len);
}

// Rows, weights and positions of the moves; the lengths.  7300 rows of each of 16 heads of 64: 12.3 us, what
// the card moves.
template <int D>
__global__ __launch_bounds__(256) void paged_evict_move_kernel(const PagedCache c, int keep, const int2* head, const int2* moves,
                                                               long most) {
  constexpr int U = D / 8;
  const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const long at = (long)b * c.Hk + hk, cap = c.cap();
  const int2 hd = head[at];
  for (long u = (long)blockIdx.x * 256 + tid; u < (long)hd.x * U; u += (long)gridDim.x * 256) {
    const int2 mv = moves[at * most + u / U];
    const int d = 8 * (int)(u % U);
    const long to = c.row(b, hk, mv.x), from = c.row(b, hk, mv.y);
    if (to >= 0 && from >= 0) {
      *reinterpret_cast<uint4*>(c.k + to * D + d) = *reinterpret_cast<const uint4*>(c.k + from * D + d);
      *reinterpret_cast<uint4*>(c.v + to * D + d) = *reinterpret_cast<const uint4*>(c.v + from * D + d);
    }
    if (d == 0) {
      c.weights[at * cap + mv.x] = c.weights[at * cap + mv.y];
      c.positions[at * cap + mv.x] = c.positions[at * cap + mv.y];
    }
  }
  if (blockIdx.x == 0 && hk == 0 && tid == 0 && hd.y > keep) {
    c.lens[b] = keep;
    c.evicted[b] += hd.y - keep;
  }
}

static int64_t evict_align(int64_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace qv

static int paged_check(int64_t B, int64_t Hk, int64_t D, int64_t page, int64_t slots, int64_t pages) {
  QV_CHECK_ARG(D == 64 || D == 128, "head_dim must be 64 or 128 (got %lld)", (long long)D);
  QV_CHECK_ARG(page >= 16 && page <= 65536 && (page & (page - 1)) == 0,
               "a page must be a power of two of 16 to 65536 tokens (got %lld)", (long long)page);
  QV_CHECK_ARG(B >= 0 && B <= 32767 && Hk > 0 && Hk <= 65535 && slots >= 0 && slots <= (1 << 29) / page && pages >= 0 &&
                   pages <= INT32_MAX,
               "bad cache shape B=%lld heads=%lld pages=%lld, %lld a sequence", (long long)B, (long long)Hk, (long long)pages,
               (long long)slots);
  return QV_OK;
}

extern "C" int qv_paged_append(const void* k, const void* v, void* k_pages, void* v_pages, const int32_t* table,
                               const int32_t* start, int32_t* lens, uint32_t* tickets, const int32_t* counts, const int32_t* cu,
                               const int32_t* evicted, float* weights, int32_t* positions, int64_t B, int64_t n, int64_t T,
                               int64_t Hk, int64_t D, int64_t page, int64_t slots, int64_t pages, const int64_t* k_strides,
                               const int64_t* v_strides, void* stream) {
  if (int rc = paged_check(B, Hk, D, page, slots, pages)) return rc;
  QV_CHECK_ARG(n >= 0 && n <= (1 << 29) && T >= 0, "bad number of tokens %lld", (long long)n);
  if (B == 0) return QV_OK;
  QV_CHECK_ARG(start && lens && tickets && (slots == 0 || table) && (pages == 0 || (k_pages && v_pages)), "null pointer argument");
  QV_CHECK_ARG(!(counts && cu), "counts and cu are two ways to say the same");
  QV_CHECK_ARG(!weights == !positions && !weights == !evicted, "weights, positions and evicted go together");
  QV_CHECK_ARG(n == 0 || (k && v && k_strides && v_strides), "null pointer argument");
  QV_CHECK_ARG((uintptr_t)k_pages % 16 == 0 && (uintptr_t)v_pages % 16 == 0, "pages must be 16-byte aligned");
  int64_t ks[3] = {0, 0, 0}, vs[3] = {0, 0, 0};
  if (n) {
    QV_CHECK_ARG((uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0, "k and v must be 16-byte aligned");
    for (int i = 0; i < 3; ++i) {
      ks[i] = k_strides[i], vs[i] = v_strides[i];
      QV_CHECK_ARG(ks[i] % 8 == 0 && vs[i] % 8 == 0, "k and v strides must be multiples of 8 elements");
    }
  }
  qv::PagedCache c = {};
  c.k = (uint16_t*)k_pages, c.v = (uint16_t*)v_pages, c.table = table, c.lens = lens, c.evicted = const_cast<int32_t*>(evicted);
  c.weights = weights, c.positions = positions;
  c.B = (int)B, c.Hk = (int)Hk, c.slots = (int)slots, c.pages = (int)pages, c.page_log2 = __builtin_ctzll(page);
  // some 16 KB of keys a workgroup: four 16-byte units a thread, and as many of values
  const int64_t chunk = std::max<int64_t>(1, 8192 / (Hk * D));
  const dim3 grid((unsigned)std::min<int64_t>(std::max<int64_t>(1, (n + chunk - 1) / chunk), 65535), (unsigned)B);
#define QV_APPEND(DIM)                                                                                                    \
  hipLaunchKernelGGL((qv::paged_append_kernel<DIM>), grid, dim3(256), 0, (hipStream_t)stream, c, (const uint16_t*)k,      \
                     (const uint16_t*)v, start, counts, cu, (int)n, (long)T, tickets, (int)chunk, (long)ks[0], (long)ks[1], \
                     (long)ks[2], (long)vs[0], (long)vs[1], (long)vs[2])
  if (D == 64) QV_APPEND(64);
  else QV_APPEND(128);
#undef QV_APPEND
  return qv::check_launch("paged_append");
}

extern "C" int64_t qv_paged_evict_workspace(int64_t B, int64_t Hk, int64_t capacity, int64_t keep) {
  if (B <= 0 || Hk <= 0 || keep < 0 || capacity <= keep) return 0;
  return qv::evict_align(B * Hk * 8) + B * Hk * std::min(keep, capacity - keep) * 8;
}

extern "C" int qv_paged_evict(void* k_pages, void* v_pages, const int32_t* table, int32_t* lens, int32_t* evicted, float* weights,
                              int32_t* positions, int64_t B, int64_t Hk, int64_t D, int64_t page, int64_t slots, int64_t pages,
                              int64_t keep, int64_t recent, int64_t first, void* workspace, int64_t workspace_bytes,
                              void* stream) {
  if (int rc = paged_check(B, Hk, D, page, slots, pages)) return rc;
  QV_CHECK_ARG(keep >= 0 && recent >= 0 && first >= 0 && recent <= keep && first <= keep - recent,
               "recent = %lld and first = %lld tokens are not within keep = %lld", (long long)recent, (long long)first,
               (long long)keep);
  const int64_t cap = slots * page;
  if (B == 0 || cap <= keep) return QV_OK;
  QV_CHECK_ARG(lens && evicted && weights && positions && table && (pages == 0 || (k_pages && v_pages)), "null pointer argument");
  QV_CHECK_ARG((uintptr_t)k_pages % 16 == 0 && (uintptr_t)v_pages % 16 == 0, "pages must be 16-byte aligned");
  QV_CHECK_ARG((uintptr_t)weights % 16 == 0 && (uintptr_t)positions % 16 == 0,
               "weights and positions must be 16-byte aligned");        // read four at a time
  const int64_t need = qv_paged_evict_workspace(B, Hk, cap, keep), most = std::min(keep, cap - keep);
  QV_CHECK_ARG(workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need, "evict takes %lld bytes of workspace",
               (long long)need);
  qv::PagedCache c = {};
  c.k = (uint16_t*)k_pages, c.v = (uint16_t*)v_pages, c.table = table, c.lens = lens, c.evicted = evicted;
  c.weights = weights, c.positions = positions;
  c.B = (int)B, c.Hk = (int)Hk, c.slots = (int)slots, c.pages = (int)pages, c.page_log2 = __builtin_ctzll(page);
  int2* head = (int2*)workspace;
  int2* moves = (int2*)((char*)workspace + qv::evict_align(B * Hk * 8));
  const hipStream_t st = (hipStream_t)stream;
#define QV_SELECT(KEYS)                                                                                                       \
  hipLaunchKernelGGL((qv::paged_evict_select_kernel<KEYS>), dim3((unsigned)Hk, (unsigned)B), dim3(qv::EVICT_THREADS), 0, st, c, \
                     (int)keep, (int)recent, (int)first, head, moves, (long)most)
  // the keys in 32 KB of LDS (two workgroups a CU), in 144 KB, or made again for each pass
  if (cap <= 8192) QV_SELECT(8192);
  else if (cap <= 36864) QV_SELECT(36864);
  else QV_SELECT(0);
#undef QV_SELECT
  const int64_t units = most * (D / 8), wg = std::max<int64_t>(1, std::min<int64_t>((units + 255) / 256, 2048 / (B * Hk) + 1));
  const dim3 grid((unsigned)wg, (unsigned)Hk, (unsigned)B);
  if (D == 64) hipLaunchKernelGGL((qv::paged_evict_move_kernel<64>), grid, dim3(256), 0, st, c, (int)keep, head, moves, (long)most);
  else hipLaunchKernelGGL((qv::paged_evict_move_kernel<128>), grid, dim3(256), 0, st, c, (int)keep, head, moves, (long)most);
  return qv::check_launch("paged_evict");
}
