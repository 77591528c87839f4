// Attention of sequences of different lengths (kernels: attention_kv.h): packed behind one
// another, each over itself, and over 16-bit keys and values in pages; and what each cached
// token receives of it.
//
// What tokens receive: w_j += sum over the queries and heads of key head hk of p_j,
// p_j = 2^(S_j c - lse), lse = m + log2 l of the row from the attention itself.  The scores are
// computed again, S = Q K^T (not K Q^T: so that a lane holds one key and sums over its registers).
#include "attention_kv.h"

#include <algorithm>

namespace qv {

// ------------------------------------------------------------------ few rows over pages
// Up to 32 rows (queries times heads of a key head).  Bound by the bytes of the keys and values, so
// all CUs have to draw them to the end, whatever the lengths: Hk x shares workgroups, two a CU,
// each takes an equal share of all sequences' 64-slot tiles of a key head, in order: the end of one
// sequence, the next whole, the beginning of a third.  What of a sequence falls into one share is a
// segment; a sequence of several segments is joined by the finishing kernel.  Inside a segment every
// wave has 32-slot tiles of its own, in LDS areas of its own that its copies fill (two stages).  Two
// workgroups of 2 waves (D = 64: 4) a CU rather than one of twice as many: one begins a segment (four
// dependent reads) while the other draws, with 64 KB on their way a CU either way: 12 x 40 heads over up
// to 5000 slots 38.6 us against 43.2, 32 x 32 heads over 2000 41.5 against 49.2.  16 sequences of up to 8001
// slots, 8 heads of 128: 48 us, 5.5 TB/s.
struct KvSteps {
  KvAttn a;               // part, stat: by segment (share + sequence), key head, row
  int shares;             // 0: a workgroup for each sequence and key head
  bool collect;           // tokens are to receive
  int2* info;             // (sequence, key head): first segment, segments
  float* scores;          // (sequence, key head, row, capacity): raw scores; NULL: not kept
};
constexpr int KV_SHARE = 4;   // tiles of a share at least

// Tiles of sequence b; at least one where it has queries, so that their rows are written.
__device__ __forceinline__ int kv_units(const KvAttn& a, int b) {
  if (a.counts && a.counts[b] <= 0) return 0;
  const int n = kv_tiles(kv_len(a, b));
  return n > 0 ? n : 1;
}

template <int D>
struct KvPagedStep {
  static constexpr int WAVES = kv_step_waves(false, D) / 2, THREADS = 64 * WAVES;
  static constexpr int KT = 32, TILE = KT * D * 2;
  static constexpr int LDS = WAVES * 4 * TILE;
};

template <bool BF16, int D>
__global__ __launch_bounds__(KvPagedStep<D>::THREADS)
    __attribute__((amdgpu_waves_per_eu(D == 64 ? 2 : 1, D == 64 ? 2 : 1))) void kv_paged_step_kernel(const KvSteps p) {
  using C = KvPagedStep<D>;
  constexpr int KS = D / 16, NV = D / 32, KT = C::KT, TILE = C::TILE, WAVES = C::WAVES;
  constexpr int DMA = TILE / 1024, RPD = 1024 / (2 * D);
  constexpr uint64_t ALL = 0xFFFFFFFFull;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[C::LDS];
  __shared__ float2 stat[WAVES][32];
  __shared__ int sums[WAVES];
  __shared__ long found[2];
  const KvAttn& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, l32 = lane & 31;
  const int hk = blockIdx.x, nrows = a.Lq * a.G;
  const long cap = (long)a.table_slots << a.page_log2;

  // the share: sequence b from its tile `at` on, `left` tiles; before: tiles of the sequences before b
  int b, at = 0;
  long left, before = 0, per = 1;
  if (p.shares == 0) {
    b = blockIdx.y;
    left = kv_units(a, b);
  } else {
    // tiles of sequence i0 + tid, those of the ones before it, and of all up to the chunk's end
    long base = 0, from = 0;
    int n = 0;
    auto scan = [&](int i0) __attribute__((always_inline)) {
      const int i = i0 + tid;
      n = i < a.B ? kv_units(a, i) : 0;
      int sum = n;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(sum, o);
        sum += lane >= o ? x : 0;
      }
      if (lane == 63) sums[wave] = sum;
      __syncthreads();
      from = base + sum - n;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        from += w < wave ? sums[w] : 0;
        base += sums[w];
      }
    };
    if (tid == 0) found[0] = -1;
    scan(0);                                         // mostly all there is
    for (int i0 = C::THREADS; i0 < a.B; i0 += C::THREADS) {
      __syncthreads();
      scan(i0);
    }
    const long total = base;
    per = (total + p.shares - 1) / p.shares;
    per = per < KV_SHARE ? KV_SHARE : per;
    const long lo = (long)blockIdx.y * per;
    if (lo >= total) return;
    left = total - lo < per ? total - lo : per;
    // the sequence that tile lo falls into
    if (a.B > C::THREADS) {
      base = 0;
      for (int i0 = 0; i0 < a.B; i0 += C::THREADS) {
        __syncthreads();
        scan(i0);
        if (from <= lo && lo < from + n) found[0] = i0 + tid, found[1] = from;
        if (base > lo) break;                        // the same for all threads
      }
    } else if (from <= lo && lo < from + n) {
      found[0] = tid, found[1] = from;
    }
    __syncthreads();
    b = (int)found[0], before = found[1];
    if (b < 0) return;
    at = (int)(lo - before);
  }
  b = __builtin_amdgcn_readfirstlane(b), at = __builtin_amdgcn_readfirstlane(at);

  for (;;) {
    const int units = kv_units(a, b);
    const int mine = left < units - at ? (int)left : units - at;      // tiles of this segment
    if (mine > 0) {
      const bool whole = mine == units;
      const long segment = p.shares == 0 ? b : (long)blockIdx.y + b;
      if (p.info && at == 0 && tid == 0)
        p.info[(long)b * a.Hk + hk] = p.shares == 0 ? make_int2(b, 1)
                                                    : make_int2((int)(before / per) + b,
                                                                (int)((before + units - 1) / per - before / per) + 1);
      const KvRange rg = kv_sequence(a, b);          // the last query sees all tiles
      const int rc = l32 < nrows ? l32 : nrows - 1;
      const int qi = kv_query(a, rc);
      const int upto = a.causal ? rg.len - rg.nq + qi : rg.len - 1;    // the last slot that the row sees
      const int first_upto = a.causal ? rg.len - rg.nq : rg.len - 1;
      KvRows<false, BF16, D> qr;
      qr.fetch(a.q + b * a.q_bs + qi * a.q_ts + (hk * a.G + rc - qi * a.G) * a.q_hs, h);
      qr.finish(a.scale_log2);
      KvState<D> s;
      s.init();
      // tiles of 32 slots; lane 2 i + e holds the page of half e of the wave's tile i, 32 tiles at a time
      // and the next 32 on their way
      const int t1 = min((long)(at + mine) * 2, ((long)rg.len + KT - 1) / KT), first = 2 * at + wave;
      int entries = -1, entries_next = -1;
      uint32_t there = 0;                            // slots of the issued tile that have a page
      auto load_entries = [&](int i) __attribute__((always_inline)) {
        const long slot = ((long)first + (long)WAVES * (i + (lane >> 1))) * KT + 16 * (lane & 1);
        return slot < rg.len ? kv_page(a, b, (int)slot) : -1;
      };
      uint8_t* area = lds + wave * 4 * TILE;
      const uint32_t area0 = lds_addr(area);
      auto issue = [&](int buf, int i) __attribute__((always_inline)) {      // the wave's tile i
        if ((i & 31) == 0 && i > 0) {
          entries = entries_next;
          entries_next = load_entries(i + 32);
        }
        const int key0 = (first + WAVES * i) * KT;
        const int page[2] = {__builtin_amdgcn_readlane(entries, 2 * (i & 31)),
                             __builtin_amdgcn_readlane(entries, 2 * (i & 31) + 1)};
        there = (kv_page_ok(a, page[0]) ? 0xFFFFu : 0u) | (kv_page_ok(a, page[1]) ? 0xFFFF0000u : 0u);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const __amdgpu_buffer_rsrc_t r[2] = {kv_page_rsrc<D>(a, v ? a.v : a.k, page[0], hk, key0),
                                               kv_page_rsrc<D>(a, v ? a.v : a.k, page[1], hk, key0 + 16)};
#pragma unroll
          for (int w = 0; w < DMA; ++w) {
            const int r0 = RPD * w, row = r0 + lane / (D / 8), c = lane % (D / 8);
            const int swizzled = c ^ (v ? kv_fv<D>(row) : kv_fk<D>(row));
            kv_dma16(r[r0 / 16], (uint32_t)(lane / (D / 8)) * (2 * D) + swizzled * 16, (uint32_t)(r0 % 16) * (2 * D),
                     area0 + (2 * buf + v) * TILE + r0 * (2 * D));
          }
        }
      };
      static_assert(2 * DMA == 8 || 2 * DMA == 16, "the wait below counts the copies of one stage");
      bool careful = false;
      for (;;) {
        int tile = first, i = 0, buf = 0;
        entries = load_entries(0), entries_next = load_entries(32);
        if (tile < t1) issue(0, 0);
        for (; tile < t1; tile += WAVES) {
          const int key0 = tile * KT;
          const bool more = tile + WAVES < t1;
          const uint64_t seen = kv_below(rg.len - key0) & there;
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // the other stage's reads are done
          if (more) {
            issue(buf ^ 1, ++i);
            if constexpr (2 * DMA == 8) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");      // this stage's copies have landed
            else asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
          } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
          }
          uint8_t* kt = area + 2 * buf * TILE;
          uint8_t* vt = kt + TILE;
          if (seen != ALL) {                         // value rows that are left out may hold anything
#pragma unroll
            for (int c = lane; c < TILE / 16; c += 64)
              if (!((seen >> (c / (D / 8))) & 1)) reinterpret_cast<uint4*>(vt)[c] = make_uint4(0, 0, 0, 0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          }
          if (careful) {
            kv_take_bad<BF16, D>(vt, KT, seen & kv_below(upto - key0 + 1), h, s);
            for (int c = lane; c < TILE / 16; c += 64) kv_drop_bad<BF16>(reinterpret_cast<uint4*>(vt)[c]);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          }
          f32x16 sc[1];
          uint4 pf[2];
#pragma unroll
          for (int st = 0; st < KS; ++st)
            sc[0] = kv_mfma<BF16>(kv_frag_k<D>(kt, 0, st, h, l32), qr.f[st], st == 0 ? f32x16{} : sc[0]);
          if (seen != ALL || first_upto < key0 + KT - 1) kv_mask<1>(sc, seen & kv_below(upto - key0 + 1), h);
          if (p.scores && l32 < nrows) {
            float* to = p.scores + (((long)b * a.Hk + hk) * nrows + l32) * cap + key0 + 4 * h;
#pragma unroll
            for (int g = 0; g < 4; ++g)              // the capacity is a multiple of 16
              if (g < 2 || key0 + 16 < cap)
                *reinterpret_cast<float4*>(to + 8 * g) =
                    make_float4(sc[0][4 * g], sc[0][4 * g + 1], sc[0][4 * g + 2], sc[0][4 * g + 3]);
          }
          kv_softmax<BF16, D, 1, false, true>(sc, qr.mul, s, pf, [](int) __attribute__((always_inline)) {});
#pragma unroll
          for (int st = 0; st < 2; ++st)
#pragma unroll
            for (int db = 0; db < NV; ++db) s.o[db] = kv_mfma<BF16>(kv_frag_v<D>(vt, db, st, lane), pf[st], s.o[db]);
          buf ^= 1;
        }
        if (careful || !__builtin_amdgcn_ballot_w64(kv_bad<D>(s))) break;
        careful = true;
        s.init();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      // ---- join the waves: every wave's O under the common reference, summed in wave order
      const float l = kv_half_sum(s.l);
      __syncthreads();                               // all tiles read
      if (h == 0) stat[wave][l32] = make_float2(s.m, l);
      __syncthreads();
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) m = fmaxf(m, stat[w][l32].x);
      const float ref = m == -INFINITY ? 0.f : m;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) sum += stat[w][l32].y * __builtin_amdgcn_exp2f(stat[w][l32].x - ref);
      const float by = sum == 0.f ? 0.f : __builtin_amdgcn_exp2f(s.m - ref) / sum;
      float* join = reinterpret_cast<float*>(lds);   // [wave][row][D]
      if (l32 < nrows)
#pragma unroll
        for (int db = 0; db < NV; ++db)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4*>(join + (wave * 32 + l32) * D + 32 * db + 8 * g + 4 * h) =
                make_float4(s.o[db][4 * g] * by, s.o[db][4 * g + 1] * by, s.o[db][4 * g + 2] * by, s.o[db][4 * g + 3] * by);
      __syncthreads();
      const int rows_out = nrows < rg.nq * a.G ? nrows : rg.nq * a.G;
      const long record = (segment * a.Hk + hk) * nrows;
      for (int c = tid; c < rows_out * (D / 4); c += C::THREADS) {
        const int row = c / (D / 4), d = 4 * (c % (D / 4)), query = kv_query(a, row);
        float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(join + (w * 32 + row) * D + d);
          o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
        }
        if (whole) {
          uint16_t* op = a.out + b * a.o_bs + query * a.o_ts + (hk * a.G + row - query * a.G) * a.o_hs + d;
          *reinterpret_cast<uint2*>(op) = make_uint2(pack2<BF16>(o.x, o.y), pack2<BF16>(o.z, o.w));
        } else {
          *reinterpret_cast<float4*>(a.part + (record + row) * D + d) = o;
        }
      }
      if ((!whole || p.collect) && wave == 0 && h == 0 && l32 < rows_out) a.stat[record + l32] = make_float2(m, sum);
    }
    left -= mine, before += units, at = 0;
    if (left <= 0 || ++b >= a.B) return;
    __syncthreads();                                 // the join is read
  }
}

// The rest of it: the first `joins` workgroups of each sequence and key head join the segments of its
// rows, the others add up what its keys receive, from the raw scores: p = 2^(score c - lse).  4.8 us, 7.1
// with 4.8 MB of scores: three dependent reads (segments, their sums, their parts or the scores).
template <bool BF16, int D>
__global__ __launch_bounds__(256) void kv_paged_finish_kernel(const KvSteps p, int joins, float* weights) {
  const KvAttn& a = p.a;
  const int b = blockIdx.z, hk = blockIdx.y, tid = threadIdx.x;
  const int nrows = a.Lq * a.G;
  int nq = a.Lq;
  if (a.counts) nq = a.counts[b] < 0 ? 0 : a.counts[b] < nq ? a.counts[b] : nq;
  const int rows = nq * a.G;
  if (rows == 0) return;                             // no segment, no info
  const int2 in = p.info[(long)b * a.Hk + hk];
  // lengths that another stream changes meanwhile give anything, but no segment outside the workspace
  if (in.x < 0 || in.y < 0 || (long)in.x + in.y > (long)p.shares + a.B) return;
  const long step = (long)a.Hk * nrows, at = in.x * step + (long)hk * nrows;
  if ((int)blockIdx.x < joins) {
    const int i = blockIdx.x * 256 + tid, row = i / (D / 4), d = 4 * (i % (D / 4));
    if (row >= rows) return;
    float m, sum;
    if (in.y <= 1) {                                 // one segment: written already
      const float2 st = a.lse && d == 0 ? a.stat[at + row] : make_float2(0.f, 0.f);
      if (a.lse && d == 0) a.lse[((long)b * a.Hk + hk) * nrows + row] = kv_lse(st.x, st.y);
      return;
    }
    const int qi = kv_query(a, row);
    const float4 o = kv_join<D>(a.stat + at + row, a.part + (at + row) * D + d, step, in.y, m, sum);
    if (a.lse && d == 0) a.lse[((long)b * a.Hk + hk) * nrows + row] = kv_lse(m, sum);
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    uint16_t* op = a.out + b * a.o_bs + qi * a.o_ts + (hk * a.G + row - qi * a.G) * a.o_hs + d;
    *reinterpret_cast<uint2*>(op) = make_uint2(pack2<BF16>(o.x * inv, o.y * inv), pack2<BF16>(o.z * inv, o.w * inv));
    return;
  }
  __shared__ float lse[32];
  const int len = kv_len(a, b), first = ((int)blockIdx.x - joins) * 256;
  if (first >= len) return;
  if (tid < rows) {
    float m = -INFINITY, sum = 0.f;
#pragma unroll 4
    for (int s = 0; s < in.y; ++s) {
      const float2 st = a.stat[at + s * step + tid];
      const float up = fmaxf(m, st.x), r = up == -INFINITY ? 0.f : up;
      sum = sum * __builtin_amdgcn_exp2f(m - r) + st.y * __builtin_amdgcn_exp2f(st.x - r);
      m = up;
    }
    lse[tid] = kv_lse(m, sum);
  }
  __syncthreads();
  const long cap = (long)a.table_slots << a.page_log2, head = (long)b * a.Hk + hk;
  for (int key = first + tid; key < len; key += ((int)gridDim.x - joins) * 256) {
    const float* s = p.scores + head * nrows * cap + key;
    float sum = 0.f;
#pragma unroll 4
    for (int r = 0; r < rows; ++r) {
      const float x = s[r * cap];
      sum += x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(x, a.scale_log2, -lse[r]));
    }
    weights[head * cap + key] += sum;
  }
}

// Many rows: the pieces of split sequences joined.
template <bool BF16, int D>
__global__ __launch_bounds__(256) void kv_paged_join_kernel(const KvAttn a) {
  const int b = blockIdx.z, hk = blockIdx.y;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const int row = (int)(i / (D / 4)), d = 4 * (int)(i % (D / 4));
  const KvRange rg = kv_sequence(a, b);
  const int rows = rg.nq * a.G, row_tiles = (rows + KV_PIECE_ROWS - 1) / KV_PIECE_ROWS;
  if (row >= rows) return;
  const int2 in = a.info[(long)b * a.Hk + hk];
  if (in.y <= 1 || in.x < 0 || (long)in.x + (long)in.y * row_tiles > 2 * a.shares) return;     // written already
  const long step = (long)row_tiles * a.Hk * KV_PIECE_ROWS;
  const long at = ((long)(in.x + row / KV_PIECE_ROWS) * a.Hk + hk) * KV_PIECE_ROWS + row % KV_PIECE_ROWS;
  float m, sum;
  const float4 o = kv_join<D>(a.stat + at, a.part + at * D + d, step, in.y, m, sum);
  if (a.lse && d == 0) a.lse[((long)b * a.Hk + hk) * ((long)a.Lq * a.G) + row] = kv_lse(m, sum);
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  const int qi = kv_query(a, row);
  uint16_t* op = a.out + b * a.o_bs + qi * a.o_ts + (hk * a.G + row - qi * a.G) * a.o_hs + d;
  *reinterpret_cast<uint2*>(op) = make_uint2(pack2<BF16>(o.x * inv, o.y * inv), pack2<BF16>(o.z * inv, o.w * inv));
}

// ------------------------------------------------------------------ what keys receive, many rows
// The scores once more, transposed: a wave keeps 32 keys of one key head in registers (a key to a lane),
// and blocks of 64 rows, shared by the workgroup's waves, come by in LDS, the next one on its way to
// registers meanwhile; no exponential leaves its lane before the end.  The table, the first queries and
// their sums are asked for before the length that decides whether they are needed.  Vector issue
// bounds long ones: 1374 queries of 16 heads of 64 over 31374 slots 162 us, 4.3e12 scores a second, vector
// instructions in 93 % of the cycles, of which 54 % are a score's fused multiply-add, exponential (two
// slots) and addition, the rest the next block's addresses, its way through registers to LDS, and masks.  Short
// ones wait (8 x 300 queries of 8 heads of 128 over up to 2300 slots: 47 %, 17.9 us); 33 of 16 of 128 over
// 9033 8.6, 2 for each block.  Each wave with queries of its own from memory took 377 for the long one and 15 for
// the 33; 64 keys to a wave (fewer reads of LDS, half as many waves) 6 % less, 11.6, and 21.4 for the 8 x 300.
constexpr int KV_RECEIVE = 64;     // rows of a block
template <bool BF16, int D>
__global__ __launch_bounds__(256) void kv_receive_kernel(const KvAttn a, float* weights) {
  constexpr int KS = D / 16, CH = D / 8, U = KV_RECEIVE * CH / 256, KEYS = 128;
  __shared__ __attribute__((aligned(1024))) uint8_t s_q[2][KV_RECEIVE * D * 2];
  __shared__ __attribute__((aligned(16))) float s_lse[2][KV_RECEIVE];
  __shared__ __attribute__((aligned(16))) int s_upto[2][KV_RECEIVE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, l32 = lane & 31;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int all = a.Lq * a.G;                        // rows, those of queries that are not there among them
  const float* lse = a.lse + ((long)b * a.Hk + hk) * all;
  const long cap = (long)a.table_slots << a.page_log2;
  // kv_query without a branch, and no uint4: with either one the block goes through scratch memory
  const uint32_t single = a.g_mul ? 0u : ~0u;
  auto query = [&](int row) __attribute__((always_inline)) { return (int)(__umulhi((uint32_t)row, a.g_mul) + (row & single)); };
  i32x4 next_q[U];
  float next_lse;
  auto fetch = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = tid + 256 * u, row = min(r0 + c / CH, all - 1), qi = query(row);
      next_q[u] = *reinterpret_cast<const i32x4*>(a.q + b * a.q_bs + qi * a.q_ts + (hk * a.G + row - qi * a.G) * a.q_hs + c % CH * 8);
    }
    next_lse = lse[min(r0 + lane, all - 1)];
  };
  auto entry = [&](long key) __attribute__((always_inline)) { return key < cap ? kv_page(a, b, (int)key) : -1; };
  const long start = (long)blockIdx.x * KEYS;
  int page = entry(start + 32 * wave + l32);
  fetch(0);
  __builtin_amdgcn_sched_barrier(0);
  const KvRange rg = kv_sequence(a, b);
  const int rows = rg.nq * a.G, past = rg.len - rg.nq;
  if (rows == 0) return;
  auto upto = [&](int row) __attribute__((always_inline)) { return a.causal ? past + query(row) : rg.len - 1; };
  int fetched = 0, buf = 0;
  for (long k0 = start; k0 < rg.len; k0 += (long)gridDim.x * KEYS) {
    const long first_key = k0 + 32 * wave;           // of the wave
    const int key = (int)(first_key + l32);
    if (k0 != start) page = entry(first_key + l32);
    const bool ok = kv_page_ok(a, page) && first_key + l32 < rg.len;
    // a lane without a key takes some other page's, and its sum goes nowhere
    const uint16_t* kp = a.k + ((((long)(ok ? page : 0) * a.Hk + hk) << a.page_log2) + (key & ((1 << a.page_log2) - 1))) * D;
    uint4 kf[KS];
#pragma unroll
    for (int st = 0; st < KS; ++st) kf[st] = *reinterpret_cast<const uint4*>(kp + 16 * st + 8 * h);
    float* const at = weights + ((long)b * a.Hk + hk) * cap + key;
    const float old = ok && h == 0 ? *at : 0.f;
    float sum = 0.f;
    // from the block of the first row that sees a key of the workgroup's
    const int first = a.causal ? max((int)k0 - past, 0) * a.G & ~(KV_RECEIVE - 1) : 0;
    if (fetched != first) fetch(first);
    for (int r0 = first; r0 < rows; r0 += KV_RECEIVE, buf ^= 1) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = tid + 256 * u, row = c / CH;
        *reinterpret_cast<i32x4*>(s_q[buf] + row * (2 * D) + (c % CH ^ kv_fk<D>(row)) * 16) = next_q[u];
      }
      // rows behind the last see nothing
      if (wave == 0) {
        s_lse[buf][lane] = r0 + lane < rows ? next_lse : INFINITY;
        s_upto[buf][lane] = r0 + lane < rows ? upto(r0 + lane) : -1;
      }
      __syncthreads();                               // and all waves are done with the other stage
      fetched = r0 + KV_RECEIVE < rows ? r0 + KV_RECEIVE : 0;
      fetch(fetched);
      if (first_key >= rg.len) continue;
      auto half = [&](int e) __attribute__((always_inline)) {
        f32x16 sc;
#pragma unroll
        for (int st = 0; st < KS; ++st)
          sc = kv_mfma<BF16>(kv_frag_k<D>(s_q[buf], e, st, h, l32), kf[st], st == 0 ? f32x16{} : sc);
        auto add = [&](auto masked) __attribute__((always_inline)) {
          constexpr bool MASKED = decltype(masked)::value;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int row = 32 * e + 8 * g + 4 * h;
            const float4 l = *reinterpret_cast<const float4*>(&s_lse[buf][row]);
            const float ls[4] = {l.x, l.y, l.z, l.w};
            int4 u = {};
            if constexpr (MASKED) u = *reinterpret_cast<const int4*>(&s_upto[buf][row]);
            const int us[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[4 * g + i], a.scale_log2, -ls[i]));
              sum += !MASKED || key <= us[i] ? p : 0.f;
            }
          }
        };
        // wave-uniform
        if (r0 + 32 * e + 32 > rows || first_key + 31 > upto(r0 + 32 * e)) add(std::true_type{});
        else add(std::false_type{});
      };
      half(0);
      if (r0 + 32 < rows) half(1);
    }
    const float total = kv_half_sum(sum);
    if (ok && h == 0) *at = old + total;
  }
}

static int64_t kv_align(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// What a call over pages keeps in its workspace, in this order, and how it is cut.
struct KvPagedPlan {
  bool few = false;                // up to 32 rows
  int shares = 0;                  // of a key head's work (0: sequences, or their row tiles, are not cut)
  int64_t row_tiles = 0;           // of a sequence, more rows
  bool stored = false;             // scores are kept for what keys receive, else made again
  int64_t info = 0, lse = 0, scores = 0, parts = 0;                  // bytes
  int64_t total() const { return info + lse + scores + parts; }
};
constexpr int64_t KV_SCORES = 1ll << 30;   // most bytes of scores

static KvPagedPlan kv_paged_plan(bool collect, int64_t B, int64_t Lq, int64_t H, int64_t Hk, int64_t D, int64_t keys,
                                 int64_t capacity) {
  const int64_t rows = Lq * (H / Hk);
  KvPagedPlan p;
  const int64_t tiles = (keys + KV_BLOCK - 1) / KV_BLOCK;
  if (rows > 32) {
    p.row_tiles = (rows + KV_PIECE_ROWS - 1) / KV_PIECE_ROWS;
    p.lse = collect ? kv_align(B * Lq * H * 4) : 0;
    // at least the places of the chip, at most what would be cut if all sequences were as long as the
    // longest, and 2048 pieces in all (parts of up to 273 MB)
    // (the join's grid, a thread for 4 dims of each row, has under 2^32 threads)
    if (tiles > 2 * KV_PIECE && Hk <= 512 && rows * (D / 4) <= (1ll << 32) - 256) {
      const int64_t all = B * p.row_tiles * kv_plan(false, B, Lq, H, Hk, D, keys).splits;
      p.shares = (int)std::min<int64_t>(std::max<int64_t>(all, 512 / Hk), 2048 / Hk);
    }
    p.info = kv_align(B * Hk * 8);
    p.parts = 2 * p.shares * Hk * KV_PIECE_ROWS * (D * 4 + 8);
    return p;
  }
  p.few = true;
  // Whole sequences while a wave has at most ten 32-slot tiles of the longest: no join (4 x 16 heads of
  // 64 over 600 slots 12.4 us, shared 16.2; 8 x 16 over 1374 18.3 and 18.9; 2 x 8 of 128 over 3000
  // 67 and 19.4).
  const int waves = D == 64 ? KvPagedStep<64>::WAVES : KvPagedStep<128>::WAVES;
  p.shares = tiles <= 5 * waves || Hk >= 512 ? 0 : (int)(512 / Hk);
  p.info = kv_align(B * Hk * 8);
  p.stored = collect && B * H * Lq * capacity * 4 <= KV_SCORES;
  p.lse = collect && !p.stored ? kv_align(B * Lq * H * 4) : 0;
  p.scores = p.stored ? kv_align(B * Lq * H * capacity * 4) : 0;
  p.parts = p.shares || collect ? (p.shares + B) * Hk * rows * (D * 4 + 8) : 0;
  return p;
}

template <bool BF16, int D>
static void kv_paged_launch(const KvPagedPlan& plan, const KvSteps& p, float* weights, int64_t keys, hipStream_t st) {
  const KvAttn& a = p.a;
  if (!plan.few) {
    const dim3 grid((unsigned)((p.shares + a.B * plan.row_tiles) * a.Hk));
    hipLaunchKernelGGL((kv_attn_pipe_kernel<KV_PAGED, BF16, D>), grid, dim3(256), 0, st, a);
    if (p.shares) {
      const dim3 joins((unsigned)(((int64_t)a.Lq * a.G * (D / 4) + 255) / 256), a.Hk, a.B);
      hipLaunchKernelGGL((kv_paged_join_kernel<BF16, D>), joins, dim3(256), 0, st, a);
    }
  } else {
    hipLaunchKernelGGL((kv_paged_step_kernel<BF16, D>), dim3(a.Hk, p.shares ? p.shares : a.B),
                       dim3(KvPagedStep<D>::THREADS), 0, st, p);
    const int joins = p.shares || a.lse ? (a.Lq * a.G * (D / 4) + 255) / 256 : 0;
    const int receives = plan.stored ? (int)std::min<int64_t>(std::max<int64_t>((keys + 255) / 256, 1), 1024) : 0;
    if (joins + receives > 0)
      hipLaunchKernelGGL((kv_paged_finish_kernel<BF16, D>), dim3(joins + receives, a.Hk, a.B), dim3(256), 0, st, p, joins, weights);
  }
  // a pool without pages: no token receives, and the kernel's lanes without a key would have no page to read
  if (a.lse && a.pages > 0) {
    const dim3 grid((unsigned)std::min<int64_t>(std::max<int64_t>((keys + 127) / 128, 1), 4096), a.Hk, a.B);
    hipLaunchKernelGGL((kv_receive_kernel<BF16, D>), grid, dim3(256), 0, st, a, weights);
  }
}

}  // namespace qv

extern "C" int qv_packed_attention(const void* q, const void* k, const void* v, void* out, int dtype, const int32_t* tiles,
                                   int64_t ntiles, int64_t tile_rows, int64_t frame, int64_t T, int64_t H, int64_t Hk, int64_t D,
                                   const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                   const int64_t* out_strides, float scale, void* stream) {
  qv::KvAttn a = {};
  int64_t qs[3] = {0}, os[3] = {0};
  if (q_strides && out_strides)
    for (int i = 0; i < 2; ++i) qs[i + 1] = q_strides[i], os[i + 1] = out_strides[i];
  if (int rc = qv::kv_common(a, q, out, dtype, 1, T, T, H, Hk, D, q_strides ? qs : nullptr, out_strides ? os : nullptr, scale))
    return rc;
  QV_CHECK_ARG(frame >= 1, "frame must be positive (got %lld)", (long long)frame);
  // a grid has under 2^32 threads
  QV_CHECK_ARG(ntiles >= 0 && ntiles <= ((1 << 24) - 1) / Hk, "bad number of row tiles %lld", (long long)ntiles);
  QV_CHECK_ARG(tile_rows == 128 || (tile_rows == 256 && D == 64), "a tile has 128 rows, or 256 of 64 dims (got %lld)",
               (long long)tile_rows);
  if (T == 0 || ntiles == 0) return QV_OK;
  QV_CHECK_ARG(k && v && k_strides && v_strides && tiles, "null pointer argument");
  QV_CHECK_ARG((uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (uintptr_t)tiles % 16 == 0,
               "k, v and tiles must be 16-byte aligned");
  for (int i = 0; i < 2; ++i)
    QV_CHECK_ARG(k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0, "k and v strides must be multiples of 8 elements");
  for (const int64_t ts : {k_strides[0], v_strides[0]})
    QV_CHECK_ARG(T == 1 || (ts >= D && ts <= (1 << 24)), "k and v token strides must be %lld to 2^24 elements", (long long)D);
  a.k = (const uint16_t*)k, a.v = (const uint16_t*)v;
  a.k_ts = T == 1 ? D : k_strides[0], a.k_hs = k_strides[1];
  a.v_ts = T == 1 ? D : v_strides[0], a.v_hs = v_strides[1];
  a.splits = 1;
  a.tiles = (const int4*)tiles, a.ntiles = (int)ntiles, a.T = T;
  a.frame = frame > INT32_MAX ? INT32_MAX : (int)frame;
  const dim3 grid((unsigned)(ntiles * Hk));
  const hipStream_t st = (hipStream_t)stream;
  if (tile_rows == 256) {
    if (dtype == QV_BF16) hipLaunchKernelGGL((qv::kv_attn_wide_kernel<qv::KV_PACKED, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((qv::kv_attn_wide_kernel<qv::KV_PACKED, false>), grid, dim3(256), 0, st, a);
  } else if (D == 64) {
    if (dtype == QV_BF16) hipLaunchKernelGGL((qv::kv_attn_pipe_kernel<qv::KV_PACKED, true, 64>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((qv::kv_attn_pipe_kernel<qv::KV_PACKED, false, 64>), grid, dim3(256), 0, st, a);
  } else {
    if (dtype == QV_BF16) hipLaunchKernelGGL((qv::kv_attn_pipe_kernel<qv::KV_PACKED, true, 128>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((qv::kv_attn_pipe_kernel<qv::KV_PACKED, false, 128>), grid, dim3(256), 0, st, a);
  }
  return qv::check_launch("packed_attention");
}

extern "C" int64_t qv_paged_attention_workspace(int collect, int64_t B, int64_t Lq, int64_t H, int64_t Hk, int64_t D, int64_t keys,
                                                int64_t capacity) {
  if (B <= 0 || Lq <= 0 || H <= 0 || Hk <= 0 || H % Hk || keys < 0 || capacity < 0 || (D != 64 && D != 128)) return 0;
  const qv::KvPagedPlan p = qv::kv_paged_plan(collect != 0, B, Lq, H, Hk, D, keys, capacity);
  return collect || p.parts ? p.total() : 0;
}

extern "C" int qv_paged_attention(const void* q, void* out, int dtype, const void* k_pages, const void* v_pages,
                                  const int32_t* table, const int32_t* lens, const int32_t* counts, int causal, float* weights,
                                  int64_t B, int64_t Lq, int64_t H, int64_t Hk, int64_t D, int64_t page, int64_t slots,
                                  int64_t pages, int64_t keys, const int64_t* q_strides, const int64_t* out_strides, float scale,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
  qv::KvAttn a = {};
  QV_CHECK_ARG(page >= 16 && page <= 65536 && (page & (page - 1)) == 0,
               "a page must be a power of two of 16 to 65536 tokens (got %lld)", (long long)page);
  QV_CHECK_ARG(slots >= 0 && slots <= (1 << 29) / page && pages >= 0 && pages <= INT32_MAX,
               "bad cache of %lld pages, %lld a sequence", (long long)pages, (long long)slots);
  if (int rc = qv::kv_common(a, q, out, dtype, B, Lq, slots * page, H, Hk, D, q_strides, out_strides, scale)) return rc;
  if (B == 0 || Lq == 0) return QV_OK;
  QV_CHECK_ARG(lens && (slots == 0 || table) && (pages == 0 || (k_pages && v_pages)), "null pointer argument");
  QV_CHECK_ARG((uintptr_t)k_pages % 16 == 0 && (uintptr_t)v_pages % 16 == 0, "pages must be 16-byte aligned");
  a.k = (const uint16_t*)k_pages, a.v = (const uint16_t*)v_pages;
  a.lens = lens, a.counts = counts, a.causal = causal != 0;
  a.table = table, a.table_slots = (int)slots, a.pages = (int)pages, a.page_log2 = __builtin_ctzll(page);
  if (keys < 0 || keys > slots * page) keys = slots * page;
  qv::KvPagedPlan plan = qv::kv_paged_plan(weights != nullptr, B, Lq, H, Hk, D, keys, slots * page);
  char* ws = (char*)workspace;
  if (weights)
    QV_CHECK_ARG(ws && (uintptr_t)ws % 16 == 0 && workspace_bytes >= plan.total(),
                 "adding up what is received takes %lld bytes of workspace", (long long)plan.total());
  qv::KvSteps p = {};
  if (!ws || (uintptr_t)ws % 16 || workspace_bytes < plan.total()) {         // not with weights
    plan.shares = 0;
    ws = nullptr;
  }
  if (ws) {
    char* const parts = ws + plan.info + plan.lse + plan.scores;
    p.info = a.info = (int2*)ws;
    a.part = (float*)parts;
    a.stat = (float2*)(parts + (plan.few ? (plan.shares + B) * H * Lq : 2 * plan.shares * Hk * qv::KV_PIECE_ROWS) * D * 4);
    if (plan.lse) a.lse = (float*)(ws + plan.info);
    if (plan.scores) p.scores = (float*)(ws + plan.info + plan.lse);
  }
  a.shares = plan.shares;
  QV_CHECK_ARG(B <= 65535 && Hk <= 65535 && (plan.shares + B * plan.row_tiles) * Hk <= (1 << 24) - 1, "grid too large");
  p.a = a, p.shares = plan.shares, p.collect = weights != nullptr;
  const hipStream_t st = (hipStream_t)stream;
  if (D == 64) {
    if (dtype == QV_BF16) qv::kv_paged_launch<true, 64>(plan, p, weights, keys, st);
    else qv::kv_paged_launch<false, 64>(plan, p, weights, keys, st);
  } else {
    if (dtype == QV_BF16) qv::kv_paged_launch<true, 128>(plan, p, weights, keys, st);
    else qv::kv_paged_launch<false, 128>(plan, p, weights, keys, st);
  }
  return qv::check_launch("paged_attention");
}
