// Attention of queries over keys of another length, for gfx950: softmax(q k^T scale) v
// with shared key heads (G query heads to a key head), head_dim 64 or 128, over
//  * 16-bit keys and values of the caller (qv_attention_cross), optionally a length
//    and a key mask for each sequence, or
//  * the 8-bit cache of kv_cache.h (qv_kv8_attention), optionally causal.
//
// The G query heads of a key head and the queries form one list of rows, row r =
// (query r / G, head r % G), so that a single query's heads share one pass over the
// keys.  A 64-key tile is S^T = K Q^T, p = 2^(S c - m), O^T += V^T P^T with
// v_mfma_f32_32x32x16; the layouts are those of attention.hip: a lane holds one row's
// scores, which are the second product's operand without a shuffle.  One running
// reference m and sum l per row; m moves only when a score passes it by far.
//
// Forms, by the rows of a key head:
//  * wide: over 128 rows of D = 64; 4 waves of 64 rows, K / V tiles of the workgroup in
//    LDS (16-bit: LDS DMA; 8-bit: codes through registers, converted once by the whole
//    workgroup, stored in fragment order);
//  * pipelined: D = 128, or 33 to 128 rows of D = 64; 4 waves of 32 rows on the same
//    tiles, the next tile's scores and the last one's products beside a softmax;
//  * step: up to 32 rows, every wave its own tiles of the key range (16-bit: LDS
//    areas of its own; 8-bit: fragments straight from memory), joined in LDS.
// In all of them the key range may be split over workgroups, joined by a second kernel.
//
// 8-bit values: scores are products of 16-bit queries with whole numbers, the key
// block's scale goes into c.  bf16 queries become fp16 under a power of two of their
// row, its largest at 2^13 to 2^14: exact down to 2^-30 of that one's power of two, what is
// smaller off by at most 2^-38 of it (half of fp16's last step).  Value codes are multiplied by
// their scale over a power of two 2^ve that all of O carries: exact in fp16, as a
// scale has four significant bits; ve moves (and O with it) only when a block's
// scale leaves 2^(ve - 16) .. 2^(ve + 4).
//
// What a mask leaves out is not used, whatever it holds: scores are replaced, and
// value rows zeroed in LDS (a probability of 0 would not cancel a NaN).  A row that
// sees no key is zero.
#include "kv_cache.h"

namespace qv {

struct KvAttn {
  const uint16_t *q, *k, *v;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  uint16_t* out;
  float* part;            // [split][row][D], each split's own quotient
  float2* stat;           // [split][row]: m (log2 units), l
  const int32_t *lens, *counts;
  const uint8_t* mask;
  long mask_bs;
  int B, Lq, H, Hk, G, Lk, blocks, causal;
  int splits, split_tiles;   // splits of a sequence, key tiles of one: at least split_tiles
  int row_tiles;
  uint32_t g_mul;         // floor(2^32 / G) + 1; 0 for G = 1
  long q_bs, q_ts, q_hs, k_bs, k_ts, k_hs, v_bs, v_ts, v_hs, o_bs, o_ts, o_hs;
  float scale_log2;
};

// The reference m is set 7 below a row's largest score (log2 units), and set anew when
// one passes it by 15: probabilities reach from 2^15, just inside fp16, down to its
// 2^-25, so that what rounds to nothing has under 2^-32 of the weight of a key (with
// the largest at 1 a row of a million even keys beside one large one lost 3 % of its sum).
constexpr float KV_LIFT = 7.0f, KV_TOP = 15.0f, KV_SUM_LIMIT = 32768.0f;
constexpr int KV_VE_UP = 4, KV_VE_DOWN = 16;   // a block's scale against 2^ve
constexpr int KV_VE_RANGE = 60;       // 2^ve stays within 2^-60 of its largest: O * 2^60 is finite

__device__ __forceinline__ float kv_half_max(float x) {
  float a, b;
  pair32(x, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float kv_half_sum(float x) {
  float a, b;
  pair32(x, a, b);
  return a + b;
}

template <bool BF>
__device__ __forceinline__ f32x16 kv_mfma(const uint4& a, const uint4& b, const f32x16& c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two probabilities as packed 16-bit floats, and the sum of such a pair added to t.
template <bool BF>
__device__ __forceinline__ uint32_t kv_pack(float a, float b) {
  if constexpr (BF) {
    const bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    const f16x2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
}
template <bool BF>
__device__ __forceinline__ float kv_add_pair(uint32_t w, float t) {
  if constexpr (BF)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), (bf16x2){(__bf16)1.0f, (__bf16)1.0f}, t, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), (f16x2){(_Float16)1.0f, (_Float16)1.0f}, t, false);
}

// 16 codes to 16 fp16 numbers times f (the scale's part of 2^ve; 1 for keys):
// 0x6400 | (code + 128) is the fp16 number 1152 + code, times f minus 1152 f: one
// packed multiply-add, exact (1152 f has 8 significant bits).
__device__ __forceinline__ void kv_decode(const uint4& u, f16x2 f, uint4& lo, uint4& hi) {
  const f16x2 off = f * (f16x2){(_Float16)-1152.0f, (_Float16)-1152.0f};
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = w[i] ^ 0x80808080u;
    const f16x2 p0 = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u));
    const f16x2 p1 = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u));
    r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(p0, f, off));
    r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(p1, f, off));
  }
  lo = make_uint4(r[0], r[1], r[2], r[3]);
  hi = make_uint4(r[4], r[5], r[6], r[7]);
}

// The scale's part of 2^ve, moving ve where the block needs it (the same in all
// lanes).  top: the largest ve so far.  O moves with it in 32 bits (KvState::follow).
// A row keeps what is above some 2^-60 of the largest scale among the blocks that it
// sees, whatever they weigh (fp16 inputs span 2^40; bf16 ones could pass it).
struct KvUnits {
  int ve = 0, top = -1000;
  bool any = false;
  __device__ __forceinline__ float fit(float s) {
    if (s > 0.f) {
      int e = (int)(__builtin_bit_cast(uint32_t, s) >> 23) - 127;   // s >= 2^-120
      if (!any) {
        ve = top = e, any = true;
      } else if (e > ve + KV_VE_UP || e < ve - KV_VE_DOWN) {
        if (e < top - KV_VE_RANGE) e = top - KV_VE_RANGE;
        ve = e;
        if (e > top) top = e;
      }
    }
    return s > 0.f ? __builtin_ldexpf(s, -ve) : 0.f;
  }
};

// What the scores of a block with key scale ks are multiplied by (1 for the NaN of a marked
// block); kept off 0 so that a masked score (-inf) times it stays -inf: with a scale of 0
// the scores, whole numbers times 16-bit queries, still come to nothing.
__device__ __forceinline__ float kv_factor(float ks, float mul) {
  const float c = (ks >= 0.f ? ks : 1.0f) * mul;
  return c < 1e-37f ? 1e-37f : c;
}

// A block marked by a NaN scale goes into the products as numbers, for a NaN there would
// reach rows that do not see the block (0 * NaN); the sums of those that do become NaN.
__device__ __forceinline__ bool kv_marked(float ks, float vs) { return ks != ks || vs != vs; }

// The fragments of one wave's 32 rows, and what their scores are multiplied by.
template <bool KV8, bool BF16, int D>
struct KvRows {
  static constexpr bool MBF = BF16 && !KV8;   // MFMA type
  uint4 f[D / 16];
  float mul;
  __device__ __forceinline__ void fetch(const uint16_t* p, int h) {
#pragma unroll
    for (int st = 0; st < D / 16; ++st)
      f[st] = *reinterpret_cast<const uint4*>(p + (KV8 ? 32 * (st >> 1) + 16 * h + 8 * (st & 1) : 16 * st + 8 * h));
  }
  __device__ __forceinline__ void finish(float scale_log2) {
    mul = scale_log2;
    if constexpr (KV8 && BF16) {
      u16x2 top = {0, 0};                      // magnitudes order like integers
#pragma unroll
      for (int st = 0; st < D / 16; ++st) {
        const uint32_t w[4] = {f[st].x, f[st].y, f[st].z, f[st].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu));
      }
      float mx = to_f32(top[0] > top[1] ? top[0] : top[1], true);
      mx = mx < INFINITY ? mx : 1.0f;          // such a row comes to nothing anyway
      mx = kv_half_max(mx);
      int e = (int)(__builtin_bit_cast(uint32_t, mx) >> 23) - 127;
      e = e < -100 ? -100 : e;                 // the row's largest comes to 2^13 .. 2^14
      const float up = __builtin_ldexpf(1.0f, 13 - e);
      mul = __builtin_ldexpf(scale_log2, e - 13);
#pragma unroll
      for (int st = 0; st < D / 16; ++st) {
        uint32_t w[4] = {f[st].x, f[st].y, f[st].z, f[st].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = kv_pack<false>(to_f32((uint16_t)w[i], true) * up, to_f32((uint16_t)(w[i] >> 16), true) * up);
        f[st] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
};

// What `upto`, the last key that a row sees (at least -2^28), becomes with the unit of a
// row whose keys are behind it.
constexpr int KV_BEHIND = -(1 << 30);
__device__ __forceinline__ int kv_unit(int upto, int ve) { return upto < KV_BEHIND / 2 ? upto - KV_BEHIND : ve; }

// Running state of 32 rows: O (dims 32 db + 8 (r / 4) + 4 h + r % 4 of the lane's row), m, l.
template <int D>
struct KvState {
  f32x16 o[D / 32];
  float m, l, ref;        // ref: m, 0 while there is none
  __device__ __forceinline__ void init() {
#pragma unroll
    for (int db = 0; db < D / 32; ++db) o[db] = f32x16{};
    m = -INFINITY, l = 0.f, ref = 0.f;
  }
  __device__ __forceinline__ void scale(float by) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] *= by;
  }
  // O from units of 2^from to 2^to, those of the values of the tile at key0.  A row that
  // sees nothing of the tile, nor then of any behind it, stays at 2^from: far larger
  // values, which it does not see, would take its O below what 32 bits hold (the tile's
  // products add zeros to it).  From then on `upto`, its last key, holds that unit.
  __device__ __forceinline__ void follow(int from, int to, int& upto, int key0) {
    const bool sees = upto >= key0;
    scale(__builtin_ldexpf(1.0f, sees ? from - to : 0));
    if (!sees && upto > KV_BEHIND / 2) upto = KV_BEHIND + from;
  }
};

__device__ __forceinline__ uint64_t kv_below(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

// Scores of keys that the lane's row does not see become -inf.  Bit i of seen: key i of the
// tile; the lane holds keys 32 kb + 8 (r / 4) + 4 h + r % 4.  Two bitwise operations a
// score (sign-extended bit, select): compares would want a scalar pair each.
template <int KB>
__device__ __forceinline__ void kv_mask(f32x16 (&sc)[KB], uint64_t seen, int h) {
  const uint64_t mine = seen >> (4 * h);
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    const int w = (int)(uint32_t)(mine >> (32 * kb));
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const uint32_t on = (uint32_t)((w << (31 - (8 * (r >> 2) + (r & 3)))) >> 31);
      const float x = sc[kb][r];
      sc[kb][r] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & on) | (0xFF800000u & ~on));
    }
  }
}

// Probabilities of KB x 32 keys of the lane's row as the second product's operand;
// slot(i) is called before each of the KB * 4 groups of four, kept apart by fences
// if FENCE (left to itself the compiler draws all LDS reads and MFMAs to the front
// and runs out of registers).
template <bool BF, int D, int KB, bool FENCE, class Slot>
__device__ __forceinline__ void kv_softmax(f32x16 (&sc)[KB], float c, KvState<D>& s, uint4 (&pf)[2 * KB], Slot&& slot) {
  constexpr int W = 8 * KB;
  uint32_t pw[W];
  float t = 0.f, t1 = 0.f;          // two chains
  auto word = [&](int w, float ref) __attribute__((always_inline)) {
    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[w >> 3][2 * (w & 7)], c, -ref));
    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[w >> 3][2 * (w & 7) + 1], c, -ref));
    return kv_pack<BF>(p0, p1);
  };
  if constexpr (FENCE) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < W / 2; ++i) {
    slot(i);
    if (i > 0) {
      t = kv_add_pair<BF>(pw[2 * i - 2], t);
      t1 = kv_add_pair<BF>(pw[2 * i - 1], t1);
    }
    pw[2 * i] = word(2 * i, s.ref);
    pw[2 * i + 1] = word(2 * i + 1, s.ref);
    if constexpr (FENCE) __builtin_amdgcn_sched_barrier(0);
  }
  t = kv_add_pair<BF>(pw[W - 2], t);
  t1 = kv_add_pair<BF>(pw[W - 1], t1);
  t += t1;
  // some p may have passed 2^15 only if its lane's sum did (p >= 0)
  if (__builtin_amdgcn_ballot_w64(!(t <= KV_SUM_LIMIT) || s.m == -INFINITY)) {
    float mx = sc[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[kb][r]);
    mx = kv_half_max(mx) * c;
    const bool need = mx > s.m + KV_TOP;
    if (__builtin_amdgcn_ballot_w64(need)) {
      const float m_new = need ? mx - KV_LIFT : s.m;
      const float alpha = need ? __builtin_amdgcn_exp2f(s.m - m_new) : 1.0f;   // 0 where there was none
      s.m = m_new;
      s.ref = m_new == -INFINITY ? 0.f : m_new;
      s.l *= alpha;
      s.scale(alpha);
      t = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) pw[w] = word(w, s.ref);
#pragma unroll
      for (int w = 0; w < W; ++w) t = kv_add_pair<BF>(pw[w], t);
    }
  }
  s.l += t;
#pragma unroll
  for (int st = 0; st < 2 * KB; ++st) pf[st] = make_uint4(pw[4 * st], pw[4 * st + 1], pw[4 * st + 2], pw[4 * st + 3]);
}

// 16-byte chunk c of K / V row r lies at c ^ kv_fk(r) / c ^ kv_fv(r): K fragment
// reads (one row a lane) and transposed V reads (four rows per 16 lanes) then meet
// every bank once.
template <int D>
__device__ __forceinline__ int kv_fk(int r) { return D == 64 ? (r & 7) ^ ((r >> 3) & 1) : r & 15; }
template <int D>
__device__ __forceinline__ int kv_fv(int r) { return D == 64 ? 4 * ((r >> 1) & 1) : 4 * (r & 3); }

typedef short kv_v4i16 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint2 kv_read_tr16(const uint8_t* p) {
  const kv_v4i16 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) kv_v4i16*)(__attribute__((address_space(3))) uint8_t*)p);
  return __builtin_bit_cast(uint2, r);
}

// K fragment (key block kb, k-step st) and V^T fragment (dim block db, k-step st) of a
// 16-bit tile in LDS.
template <int D>
__device__ __forceinline__ uint4 kv_frag_k(const uint8_t* k, int kb, int st, int h, int l32) {
  const int row = 32 * kb + l32;
  return *reinterpret_cast<const uint4*>(k + row * (2 * D) + ((2 * st + h) ^ kv_fk<D>(row)) * 16);
}
template <int D>
__device__ __forceinline__ uint4 kv_frag_v(const uint8_t* v, int db, int st, int lane) {
  const int h = lane >> 5;
  const int dim = 32 * db + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  uint2 r[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int key = 16 * st + 8 * i + 4 * h + ((lane & 15) >> 2);
    r[i] = kv_read_tr16(v + key * (2 * D) + (((dim >> 3) ^ kv_fv<D>(key)) * 16) + ((dim >> 2) & 1) * 8);
  }
  return make_uint4(r[0].x, r[0].y, r[1].x, r[1].y);
}

// lds_dma16 with the wait states that the copy needs behind what the compiler puts
// in front of it: 1 after a write of M0, 5 after a vector instruction that wrote one
// of its scalar registers (a spilled one read back with v_readlane).  The
// compiler does not look into the asm, and without them the wide form's second
// tile went to stale offsets.
__device__ __forceinline__ void kv_dma16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff, uint32_t lds_base) {
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
               :
               : "v"(voff), "s"(r), "s"(soff), "{m0}"(__builtin_amdgcn_readfirstlane(lds_base))
               : "memory");
}

// A 16-bit K or V source, tile by tile (`keys` rows from tile to tile): the address
// of the next tile's first row, 64-bit (a long cache passes the 32 bits of a buffer
// offset), and the bytes of it that may be read: the rest of the sequence, what lies
// behind reads as zero.
struct KvSource {
  const uint8_t* at;
  int64_t step;
  int left, keys;         // keys left of the sequence
  uint32_t row, dims;     // bytes from row to row, of a row
  __device__ __forceinline__ void init(const uint16_t* base, long ts, int D, int len, int64_t key0, int step_keys) {
    at = reinterpret_cast<const uint8_t*>(base) + key0 * ts * 2;
    step = (int64_t)step_keys * ts * 2;
    left = (int)(len - key0);
    keys = step_keys;
    row = (uint32_t)(ts * 2);
    dims = 2 * D;
  }
  // descriptor over the first `most` keys (at most 64, of under 2^25 bytes each: 32 bits hold them)
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(int most) const {
    const int k = left < most ? left : most;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(at), (short)0, k > 0 ? (int)((k - 1) * row + dims) : 0,
                                             0x00020000);
  }
  __device__ __forceinline__ void next() { at += step, left -= keys; }
};

// row / G: exact while row * G < 2^32
__device__ __forceinline__ int kv_query(const KvAttn& a, int row) {
  return a.g_mul ? (int)__umulhi((uint32_t)row, a.g_mul) : row;
}

__device__ __forceinline__ int kv_len(const KvAttn& a, int b) {
  if (!a.lens) return a.Lk;
  const int l = a.lens[b];
  return l < 0 ? 0 : l > a.Lk ? a.Lk : l;
}

__device__ __forceinline__ int kv_tiles(int len) { return (len + KV_BLOCK - 1) / KV_BLOCK; }

// Which part a workgroup of the wide and pipelined forms takes.  In the order (row tile,
// split, key head, sequence) fours of neighbours, which mostly read the same keys, share
// an XCD and its L2, and the fours go round the 8 XCDs.  (Whole sets of row tiles to an
// XCD do not go evenly into its 64 places: sets of 17 over sequences of 6017 and 2053
// tokens left some XCDs with 68 workgroups, a second round, and others with 51.)
constexpr int KV_NEAR = 4;
struct KvPart {
  int b, hk, split, rt;
  bool any;
};
__device__ __forceinline__ KvPart kv_part(const KvAttn& a) {
  const uint32_t x = blockIdx.x & 7, i = blockIdx.x >> 3;
  uint32_t g = i / KV_NEAR * (8 * KV_NEAR) + x * KV_NEAR + i % KV_NEAR;
  KvPart p;
  p.rt = g % a.row_tiles;
  g /= a.row_tiles;
  p.split = g % a.splits;
  g /= a.splits;
  p.hk = g % a.Hk;
  p.b = g / a.Hk;
  p.any = p.b < a.B;
  return p;
}

// The sequence's keys and queries, and the tiles of a split, for rows that see at most
// the keys of query `last_query` (of first_query on): splits lie at the same keys for all
// row tiles, and grow where the sequence is longer than the host knew.
struct KvRange {
  int len, nq, t0, t1;
};
__device__ __forceinline__ KvRange kv_range(const KvAttn& a, int b, int split, int first_query, int last_query) {
  KvRange r;
  r.len = kv_len(a, b);
  r.nq = a.Lq;
  if (a.counts) {
    const int c = a.counts[b];
    r.nq = c < 0 ? 0 : c > a.Lq ? a.Lq : c;
  }
  int last = r.len;                       // keys that the last row sees
  if (a.causal) {
    last = r.len - r.nq + min(last_query, r.nq - 1) + 1;
    last = last < 0 ? 0 : last > r.len ? r.len : last;
  }
  const int nt = first_query < r.nq ? kv_tiles(last) : 0;
  int per = a.split_tiles;
  if ((long)per * a.splits < kv_tiles(r.len)) per = (kv_tiles(r.len) + a.splits - 1) / a.splits;
  r.t0 = min((long)nt, (long)split * per);
  r.t1 = min((long)nt, (long)(split + 1) * per);
  return r;
}

// O's quotient back from units of 2^ve (16-bit values: none): a step of its own, as 2^ve
// over a long sum is no normal number where ve comes near -120, and an exact one unless the
// result is none.
template <bool KV8>
__device__ __forceinline__ float kv_out(float x, float inv, int ve) {
  return KV8 ? __builtin_ldexpf(x * inv, ve) : x * inv;
}

// Store a lane's row: the quotient to out, or to the split's part with m and l.
template <bool KV8, bool BF16, int D>
__device__ __forceinline__ void kv_store(const KvAttn& a, const KvState<D>& s, float l, int ve, const KvPart& p, int row,
                                         int h, bool live) {
  if (!live) return;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const int qi = kv_query(a, row), head = p.hk * a.G + row - qi * a.G;
  if (a.splits == 1) {
    uint16_t* op = a.out + p.b * a.o_bs + qi * a.o_ts + head * a.o_hs;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint2 w;
        w.x = pack2<BF16>(kv_out<KV8>(s.o[db][4 * g], inv, ve), kv_out<KV8>(s.o[db][4 * g + 1], inv, ve));
        w.y = pack2<BF16>(kv_out<KV8>(s.o[db][4 * g + 2], inv, ve), kv_out<KV8>(s.o[db][4 * g + 3], inv, ve));
        *reinterpret_cast<uint2*>(op + 32 * db + 8 * g + 4 * h) = w;
      }
  } else {
    const long at = (((long)p.b * a.splits + p.split) * a.Hk + p.hk) * ((long)a.Lq * a.G) + row;
    float* pp = a.part + at * D;
    if (l != 0.f)                                    // the join reads no part without a sum
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(pp + 32 * db + 8 * g + 4 * h) =
            make_float4(kv_out<KV8>(s.o[db][4 * g], inv, ve), kv_out<KV8>(s.o[db][4 * g + 1], inv, ve),
                        kv_out<KV8>(s.o[db][4 * g + 2], inv, ve), kv_out<KV8>(s.o[db][4 * g + 3], inv, ve));
    if (h == 0) a.stat[at] = make_float2(s.m, l);
  }
}

// ------------------------------------------------------------------ staging
// Tiles of K (V = false) or V in LDS, in order, by the whole workgroup.  16-bit: LDS
// DMA, swizzled rows.  8-bit: codes through registers, decoded once, fragment order.
template <bool KV8, int D, bool V>
struct KvTiles {
  static constexpr int TILE = KV_BLOCK * D * 2;      // bytes
  static constexpr int DMA = TILE / 1024 / 4;        // 1 KB copies of a wave
  static constexpr int RPD = 1024 / (2 * D);         // rows of a copy
  static constexpr int UNITS = KV_BLOCK * D / 16 / 256;   // 16-byte units of a thread
  KvSource src;
  uint32_t row_off, chunk;                           // of the lane in a copy: its row, its swizzled 16 bytes
  const uint4* codes;
  __device__ __forceinline__ void init(const KvAttn& a, int b, int hk, const KvRange& rg, int wave, int lane) {
    if constexpr (KV8) {
      const long block = ((long)b * a.Hk + hk) * a.blocks + rg.t0;
      codes = reinterpret_cast<const uint4*>(V ? a.vc : a.kc) + block * (KV_BLOCK * D / 16) + wave * 64 + lane;
    } else {
      if constexpr (V) src.init(a.v + b * a.v_bs + hk * a.v_hs, a.v_ts, D, rg.len, (int64_t)rg.t0 * KV_BLOCK, KV_BLOCK);
      else src.init(a.k + b * a.k_bs + hk * a.k_hs, a.k_ts, D, rg.len, (int64_t)rg.t0 * KV_BLOCK, KV_BLOCK);
      // copy w of a wave holds rows RPD (DMA wave + w) ..: the swizzle of V depends on the lane
      // only, that of K flips with w
      const int r = lane / (D / 8), c = lane % (D / 8);
      row_off = (uint32_t)r * src.row;
      chunk = (uint32_t)(c ^ (V ? kv_fv<D>(r) : kv_fk<D>(r))) * 16;
    }
  }
  // the next tile on its way to LDS (16-bit) or registers
  __device__ __forceinline__ void start(uint32_t lds, int wave, uint4 (&raw)[UNITS]) {
    if constexpr (KV8) {
#pragma unroll
      for (int u = 0; u < UNITS; ++u) raw[u] = codes[256 * u];
      codes += KV_BLOCK * D / 16;
    } else {
      const auto r = src.rsrc(KV_BLOCK);
#pragma unroll
      for (int w = 0; w < DMA; ++w) {
        const int r0 = RPD * (DMA * wave + w);
        kv_dma16(r, row_off + (V ? chunk : chunk ^ (w * (D == 64 ? 16u : 64u))), (uint32_t)r0 * src.row, lds + r0 * (2 * D));
      }
      src.next();
    }
  }
  static __device__ __forceinline__ void place(uint8_t* lds, _Float16 f, int wave, int lane, const uint4 (&raw)[UNITS]) {
    uint4* t = reinterpret_cast<uint4*>(lds);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      uint4 lo, hi;
      kv_decode(raw[u], (f16x2){f, f}, lo, hi);
      const int at = (4 * u + wave) * 128 + lane;
      t[at] = lo, t[at + 64] = hi;
    }
  }
};

// ------------------------------------------------------------------ pipelined form
// 4 waves of 32 rows.  Beside tile j's softmax run the QK of tile j + 1 and the PV of tile
// j - 1, a few of each in every slot, so that no product stands alone.  K is in LDS two
// tiles ahead, V comes with its own tile, and the workgroup meets once a tile.
// Bound by issue: a wave's tile of D = 128 is 32 MFMAs and 32 exponentials with their
// multiply-adds, conversions and sums, 112 vector instructions beside the MFMAs over 16-bit
// keys and 230 over 8-bit ones.  4096 queries of 16 heads over 10992 keys, two workgroups on
// each CU: 1007 and 918 TF/s (a large fp16 matrix product of the library: 1170), 2.1 and 2.3
// us a tile (one workgroup alone 1.24 and 1.55); there a wave issues in 38 and 41 % of its
// cycles, is ready but held in 40 and 38 %, and the matrix pipe is busy in 47 and 38 %.
// 64 rows a wave would halve the LDS reads, but at D = 128 O and the queries leave no
// registers for it: with O in accumulation registers 1374 queries of 16 heads took 112 us
// instead of 87.  For 33 to 128 rows of D = 64 half of a wide workgroup's rows would be empty.
template <bool KV8, bool BF16, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void kv_attn_pipe_kernel(const KvAttn a) {
  constexpr bool MBF = BF16 && !KV8;
  constexpr int TILE = KV_BLOCK * D * 2;
  constexpr int KS = D / 16, NV = D / 32, NK = 2 * KS, NF = 4 * NV;
  constexpr int ROWS = 128, AHEAD = D == 64 ? 2 : 1;         // slots from a fragment's read to its use
  using TK = KvTiles<KV8, D, false>;
  using TV = KvTiles<KV8, D, true>;
  __shared__ __attribute__((aligned(1024))) uint8_t k_lds[2][TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t v_lds[2][TILE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, l32 = lane & 31;
  const KvPart part = kv_part(a);
  if (!part.any) return;
  const int hk = part.hk, b = part.b;
  const int nrows = a.Lq * a.G;
  const int row0 = part.rt * ROWS;
  const int first_query = kv_query(a, row0);
  const KvRange rg = kv_range(a, b, part.split, first_query, kv_query(a, min(nrows, row0 + ROWS) - 1));
  if (first_query >= rg.nq) return;
  const int wrow = row0 + wave * 32, row = wrow + l32;
  const bool live = wrow < nrows && kv_query(a, wrow) < rg.nq;      // wave-uniform
  const int n = rg.t1 - rg.t0;                               // tiles, counted from 0 below

  KvRows<KV8, BF16, D> qr;
  const int rc = row < nrows ? row : nrows - 1, qi = kv_query(a, rc);
  qr.fetch(a.q + b * a.q_bs + qi * a.q_ts + (hk * a.G + rc - qi * a.G) * a.q_hs, h);    // before the tiles
  __builtin_amdgcn_sched_barrier(0);
  TK kt;
  TV vt;
  kt.init(a, b, hk, rg, wave, lane);
  vt.init(a, b, hk, rg, wave, lane);
  const uint32_t klds0 = lds_addr(k_lds), vlds0 = lds_addr(v_lds);
  // 8-bit: what is on its way to registers.  Block scales come by vector loads: a scalar
  // load in flight would make every wait for an LDS read wait for it, too.
  uint4 kraw[TK::UNITS], vraw[TV::UNITS];
  float ks = 0.f, ks_next = 0.f, vs_next = 0.f;              // ks: of this tile
  const float *ks_at = nullptr, *vs_at = nullptr;
  if constexpr (KV8) {
    long at = ((long)b * a.Hk + hk) * a.blocks + rg.t0;
    asm("" : "+v"(at));
    ks_at = a.ks + at, vs_at = a.vs + at;
  }
  KvUnits units;
  uint8_t mask_byte = 1;
  auto load_mask = [&](int j) __attribute__((always_inline)) {
    const int key = (rg.t0 + j) * KV_BLOCK + lane;
    mask_byte = key < rg.len ? a.mask[b * a.mask_bs + key] : 0;
  };
  // step j: K of j + 2, V of j, the key scale and mask of j + 1
  auto feed = [&](int j) __attribute__((always_inline)) {
    if constexpr (!KV8)
      if (a.mask && j + 1 < n) load_mask(j + 1);
    if (j + 2 < n) kt.start(klds0 + (j & 1) * TILE, wave, kraw);
    vt.start(vlds0 + (j & 1) * TILE, wave, vraw);
    if constexpr (KV8) {
      vs_next = *vs_at++;
      if (j + 1 < n) ks_next = *++ks_at;
    }
  };
  auto settle = [&](int j) __attribute__((always_inline)) {
    if constexpr (KV8) {
      if (j + 2 < n) TK::place(k_lds[j & 1], (_Float16)1.0f, wave, lane, kraw);
      TV::place(v_lds[j & 1], (_Float16)units.fit(vs_next), wave, lane, vraw);
      ks = ks_next;
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    lds_barrier();
  };
  // tiles below edge are seen whole by all rows of the wave
  const int wfirst = kv_query(a, wrow);
  const int edge = !KV8 && a.mask ? 0 : (a.causal ? min(rg.len, rg.len - rg.nq + wfirst + 1) : rg.len) / KV_BLOCK - rg.t0;
  auto visible = [&](int j) __attribute__((always_inline)) {
    uint64_t seen = ~0ull;
    if (j >= edge) {
      seen = kv_below(rg.len - (rg.t0 + j) * KV_BLOCK);
      if constexpr (!KV8)
        if (a.mask) seen = __builtin_amdgcn_ballot_w64(mask_byte != 0);
    }
    return seen;
  };
  // stage j % 2: value rows whose keys are left out may hold anything
  auto clear = [&](int j, uint64_t seen) __attribute__((always_inline)) {
    if constexpr (!KV8) {
      if (seen != ~0ull) {
        uint4* t = reinterpret_cast<uint4*>(v_lds[j & 1]);
#pragma unroll
        for (int i = 0; i < TILE / 16 / 256; ++i) {
          constexpr int ROWS_AT = 256 / (D / 8);     // rows that 256 chunks cover
          const int row = ROWS_AT * i + tid / (D / 8);
          if (!((uint32_t)(seen >> (ROWS_AT * i / 32 * 32)) >> (row & 31) & 1)) t[256 * i + tid] = make_uint4(0, 0, 0, 0);
        }
        lds_barrier();
      }
    }
  };
  KvState<D> s;
  s.init();
  int ve = 0;                                        // of the last tile's values
  int upto = a.causal ? rg.len - rg.nq + qi : rg.len - 1;    // the last key that the row sees
  if (n > 0) {
    // K of tiles 0 and 1; zero in the stage that the first PV reads (its P is zero, too)
    kt.start(klds0, wave, kraw);
    if constexpr (KV8) {
      ks = *ks_at;
      TK::place(k_lds[0], (_Float16)1.0f, wave, lane, kraw);
    }
    if (n > 1) {
      kt.start(klds0 + TILE, wave, kraw);
      if constexpr (KV8) TK::place(k_lds[1], (_Float16)1.0f, wave, lane, kraw);
    }
    if constexpr (!KV8)
      if (a.mask) load_mask(0);
    for (int i = tid; i < TILE / 16; i += 256) reinterpret_cast<uint4*>(v_lds[1])[i] = make_uint4(0, 0, 0, 0);
    if constexpr (!KV8) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    uint64_t before = ~0ull;                         // what the tile before left
    if (!live) {
      // rows past the end: the wave only stages its share
      lds_barrier();
      for (int j = 0; j < n; ++j) {
        clear(j + 1, before);
        before = visible(j);
        feed(j);
        settle(j);
      }
      clear(n - 1, before);
      return;
    }
    qr.finish(a.scale_log2);
    auto frag_k = [&](int stage, int f) __attribute__((always_inline)) {               // f = kb + 2 st
      if constexpr (KV8) return reinterpret_cast<const uint4*>(k_lds[stage])[((f & 1) * KS + (f >> 1)) * 64 + lane];
      else return kv_frag_k<D>(k_lds[stage], f & 1, f >> 1, h, l32);
    };
    auto frag_v = [&](int stage, int f) __attribute__((always_inline)) {               // f = db + NV st
      if constexpr (KV8) return reinterpret_cast<const uint4*>(v_lds[stage])[((f % NV) * 4 + f / NV) * 64 + lane];
      else return kv_frag_v<D>(v_lds[stage], f % NV, f / NV, lane);
    };
    f32x16 sa[2], sb[2];
    uint4 pa[4] = {}, pb[4];
#pragma unroll
    for (int f = 0; f < NK; ++f) sa[f & 1] = kv_mfma<MBF>(frag_k(0, f), qr.f[f >> 1], f < 2 ? f32x16{} : sa[f & 1]);
    lds_barrier();                                   // the first K stage may be written again
    // for the values of tile j
    auto rescale = [&](int j) __attribute__((always_inline)) {
      if constexpr (KV8) {
        if (units.ve != ve) {
          s.follow(ve, units.ve, upto, (rg.t0 + j) * KV_BLOCK);
          ve = units.ve;
        }
      }
    };
    // sc, p: the tile's scores, the probabilities of the tile before; next, pn: the next of each
    auto step = [&](int j, f32x16 (&sc)[2], f32x16 (&next)[2], uint4 (&p)[4], uint4 (&pn)[4]) __attribute__((always_inline)) {
      const int key0 = (rg.t0 + j) * KV_BLOCK;
      const int other = (j + 1) & 1;                 // stage of K of j + 1 and of V of j - 1
      constexpr int PK = NK / 8, PV = NF / 8;        // products of a slot
      uint4 kf[NK], vf[NF];
      clear(j + 1, before);
      auto read = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < PK; ++e) kf[slot * PK + e] = frag_k(other, slot * PK + e);
#pragma unroll
        for (int e = 0; e < PV; ++e) vf[slot * PV + e] = frag_v(other, slot * PV + e);
      };
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) read(i);
      const uint64_t seen = visible(j);
      const float kscale = ks;
      feed(j);
      rescale(j - 1);
      const float c = KV8 ? kv_factor(kscale, qr.mul) : qr.mul;
      if (j >= edge && (KV8 || seen != ~0ull)) kv_mask<2>(sc, seen & kv_below(upto - key0 + 1), h);
      kv_softmax<MBF, D, 2, true>(sc, c, s, pn, [&](int i) __attribute__((always_inline)) {
        if (i + AHEAD < 8) read(i + AHEAD);
#pragma unroll
        for (int e = 0; e < PK; ++e) {
          const int f = i * PK + e;
          next[f & 1] = kv_mfma<MBF>(kf[f], qr.f[f >> 1], f < 2 ? f32x16{} : next[f & 1]);
        }
#pragma unroll
        for (int e = 0; e < PV; ++e) {
          const int f = i * PV + e;
          s.o[f % NV] = kv_mfma<MBF>(vf[f], p[f / NV], s.o[f % NV]);
        }
      });
      before = seen;
      settle(j);
      if constexpr (KV8)
        if (kv_marked(kscale, vs_next) && (seen & kv_below(upto - key0 + 1))) s.l = __builtin_nanf("");
    };
    auto last = [&](uint4 (&p)[4]) __attribute__((always_inline)) {
      clear(n - 1, before);
      rescale(n - 1);
#pragma unroll
      for (int f = 0; f < NF; ++f) s.o[f % NV] = kv_mfma<MBF>(frag_v((n - 1) & 1, f), p[f / NV], s.o[f % NV]);
    };
    int j = 0;
    for (; j + 1 < n; j += 2) {
      step(j, sa, sb, pa, pb);
      step(j + 1, sb, sa, pb, pa);
    }
    if (j < n) {
      step(j, sa, sb, pa, pb);
      last(pb);
    } else {
      last(pa);
    }
  } else if (!live) {
    return;
  }
  kv_store<KV8, BF16, D>(a, s, kv_half_sum(s.l), kv_unit(upto, ve), part, row, h, row < nrows && kv_query(a, row) < rg.nq);
}

// ------------------------------------------------------------------ wide form
// 4 waves of 64 rows (two blocks of 32), D = 64: every fragment that is read from LDS and
// every code that is decoded serves twice the rows.  Inside a tile the second block's QK
// runs beside the first one's softmax, the first one's PV beside the second's.
// Bound by issue: 64 x 64 scores a tile and wave cost 32 MFMAs and 64 exponentials of 8
// cycles with their multiply-adds, conversions and sums, 221 vector instructions beside the
// MFMAs over 16-bit keys and 286 over the cache (attention.hip, whose queries carry the
// scale: 177).  8192 queries of 16 heads over 10992 keys, two workgroups on each CU: 940 and
// 854 TF/s, 2.24 and 2.47 us a tile (one alone 1.36 and 1.54); a wave issues in 47 and 45 %
// of its cycles, is ready but held in 38 and 35 %, the matrix pipe is busy in 43 and 37 %.
// 1374 queries of 16 heads over 10992 keys: 92 us and 7 of join under a trace (86 to 90 in
// all without); over a cache of 43968 tokens 352 and 7 (311 to 323 in all without).
template <bool KV8, bool BF16>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void kv_attn_wide_kernel(const KvAttn a) {
  constexpr int D = 64, QB = 2;
  constexpr bool MBF = BF16 && !KV8;
  constexpr int TILE = KV_BLOCK * D * 2;
  constexpr int ROWS = 4 * 32 * QB;
  using TK = KvTiles<KV8, D, false>;
  using TV = KvTiles<KV8, D, true>;
  __shared__ __attribute__((aligned(1024))) uint8_t k_lds[2][TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t v_lds[2][TILE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, l32 = lane & 31;
  const KvPart part = kv_part(a);
  if (!part.any) return;
  const int hk = part.hk, b = part.b;
  const int nrows = a.Lq * a.G;
  const int row0 = part.rt * ROWS;
  const int first_query = kv_query(a, row0);
  const KvRange rg = kv_range(a, b, part.split, first_query, kv_query(a, min(nrows, row0 + ROWS) - 1));
  if (first_query >= rg.nq) return;
  const int wrow = row0 + wave * 32 * QB;
  const bool live = wrow < nrows && kv_query(a, wrow) < rg.nq;      // wave-uniform
  const int n = rg.t1 - rg.t0;                               // tiles, counted from 0 below

  KvRows<KV8, BF16, D> qr[QB];
  int upto[QB];                                      // the last key that the row sees
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int r = wrow + 32 * qb + l32, rc = r < nrows ? r : nrows - 1, qi = kv_query(a, rc);
    qr[qb].fetch(a.q + b * a.q_bs + qi * a.q_ts + (hk * a.G + rc - qi * a.G) * a.q_hs, h);   // before the tiles
    upto[qb] = a.causal ? rg.len - rg.nq + qi : rg.len - 1;
  }
  __builtin_amdgcn_sched_barrier(0);
  TK kt;
  TV vt;
  kt.init(a, b, hk, rg, wave, lane);
  vt.init(a, b, hk, rg, wave, lane);
  const uint32_t klds0 = lds_addr(k_lds), vlds0 = lds_addr(v_lds);
  uint4 kraw[TK::UNITS], vraw[TV::UNITS];
  const float *ks_at = nullptr, *vs_at = nullptr;            // by vector loads: see the pipelined form
  if constexpr (KV8) {
    long at = ((long)b * a.Hk + hk) * a.blocks + rg.t0;
    asm("" : "+v"(at));
    ks_at = a.ks + at, vs_at = a.vs + at;
  }
  KvUnits units;
  float ks = 0.f, ks_next = 0.f, vs_next = 0.f;
  bool marked = false;
  uint8_t mask_byte = 1;
  // the tile on its way (into stage j % 2), and into place
  auto feed = [&](int j) __attribute__((always_inline)) {
    kt.start(klds0 + (j & 1) * TILE, wave, kraw);
    vt.start(vlds0 + (j & 1) * TILE, wave, vraw);
    if constexpr (KV8) {
      ks_next = *ks_at++, vs_next = *vs_at++;
    } else if (a.mask) {
      const int key = (rg.t0 + j) * KV_BLOCK + lane;
      mask_byte = key < rg.len ? a.mask[b * a.mask_bs + key] : 0;
    }
  };
  auto settle = [&](int j) __attribute__((always_inline)) {
    if constexpr (KV8) {
      TK::place(k_lds[j & 1], (_Float16)1.0f, wave, lane, kraw);
      TV::place(v_lds[j & 1], (_Float16)units.fit(vs_next), wave, lane, vraw);
      ks = ks_next, marked = kv_marked(ks_next, vs_next);
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
  };
  // tiles below edge are seen whole by all rows of the wave
  const int edge =
      !KV8 && a.mask ? 0 : (a.causal ? min(rg.len, rg.len - rg.nq + kv_query(a, wrow) + 1) : rg.len) / KV_BLOCK - rg.t0;
  // the keys of tile j that are there; value rows of the others may hold anything
  auto visible = [&](int j) __attribute__((always_inline)) {
    uint64_t seen = kv_below(rg.len - (rg.t0 + j) * KV_BLOCK);
    if constexpr (!KV8) {
      if (a.mask) seen = __builtin_amdgcn_ballot_w64(mask_byte != 0);
      if (seen != ~0ull) {
        uint4* t = reinterpret_cast<uint4*>(v_lds[j & 1]);
#pragma unroll
        for (int i = 0; i < TILE / 16 / 256; ++i) {
          constexpr int ROWS_AT = 256 / (D / 8);     // rows that 256 chunks cover
          const int row = ROWS_AT * i + tid / (D / 8);
          if (!((uint32_t)(seen >> (ROWS_AT * i / 32 * 32)) >> (row & 31) & 1)) t[256 * i + tid] = make_uint4(0, 0, 0, 0);
        }
        lds_barrier();
      }
    }
    return seen;
  };
  if (n > 0) {
    feed(0);
    settle(0);
  }
  if (!live) {
    // rows past the end: the wave only stages its share
    for (int j = 0; j < n; ++j) {
      lds_barrier();
      visible(j);
      if (j + 1 < n) {
        feed(j + 1);
        settle(j + 1);
      }
    }
    return;
  }
  KvState<D> s[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    qr[qb].finish(a.scale_log2);
    s[qb].init();
  }
  int ve = 0;                                        // of the last tile's values
  for (int j = 0; j < n; ++j) {
    lds_barrier();                                   // tile j is in place, stage j + 1 free
    const int buf = j & 1;
    const uint64_t seen = visible(j);
    float c[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) c[qb] = KV8 ? kv_factor(ks, qr[qb].mul) : qr[qb].mul;
    if constexpr (KV8) {
      if (marked) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
          if (seen & kv_below(upto[qb] - (rg.t0 + j) * KV_BLOCK + 1)) s[qb].l = __builtin_nanf("");
      }
      if (units.ve != ve) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) s[qb].follow(ve, units.ve, upto[qb], (rg.t0 + j) * KV_BLOCK);
        ve = units.ve;
      }
    }
    f32x16 sc[QB][2];
    uint4 pf[QB][4], kf[8], vf[8];
    auto qk = [&](int qb, int f) __attribute__((always_inline)) {    // f = kb + 2 st
      sc[qb][f & 1] = kv_mfma<MBF>(kf[f], qr[qb].f[f >> 1], f < 2 ? f32x16{} : sc[qb][f & 1]);
    };
    auto pv = [&](int qb, int f) __attribute__((always_inline)) {    // f = db + 2 st
      s[qb].o[f & 1] = kv_mfma<MBF>(vf[f], pf[qb][f >> 1], s[qb].o[f & 1]);
    };
    auto mask = [&](int qb) __attribute__((always_inline)) {
      if (j >= edge && (KV8 || seen != ~0ull)) kv_mask<2>(sc[qb], seen & kv_below(upto[qb] - (rg.t0 + j) * KV_BLOCK + 1), h);
    };
#pragma unroll
    for (int f = 0; f < 8; ++f) {
      if constexpr (KV8) kf[f] = reinterpret_cast<const uint4*>(k_lds[buf])[((f & 1) * 4 + (f >> 1)) * 64 + lane];
      else kf[f] = kv_frag_k<D>(k_lds[buf], f & 1, f >> 1, h, l32);
    }
    if (j + 1 < n) feed(j + 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int f = 0; f < 8; ++f) qk(0, f);
    mask(0);
    kv_softmax<MBF, D, 2, true>(sc[0], c[0], s[0], pf[0], [&](int i) __attribute__((always_inline)) {
      qk(1, i);
      if (i >= 4)
#pragma unroll
        for (int f = 2 * (i - 4); f < 2 * (i - 4) + 2; ++f) {
          if constexpr (KV8) vf[f] = reinterpret_cast<const uint4*>(v_lds[buf])[((f & 1) * 4 + (f >> 1)) * 64 + lane];
          else vf[f] = kv_frag_v<D>(v_lds[buf], f & 1, f >> 1, lane);
        }
    });
    mask(1);
    kv_softmax<MBF, D, 2, true>(sc[1], c[1], s[1], pf[1], [&](int i) __attribute__((always_inline)) { pv(0, i); });
    if (j + 1 < n) settle(j + 1);
#pragma unroll
    for (int f = 0; f < 8; ++f) pv(1, f);
  }
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int r = wrow + 32 * qb + l32;
    kv_store<KV8, BF16, D>(a, s[qb], kv_half_sum(s[qb].l), kv_unit(upto[qb], ve), part, r, h, r < nrows && kv_query(a, r) < rg.nq);
  }
}

// ------------------------------------------------------------------ step form
// Bound by the bytes of the keys and values: 16 sequences of 8000 cached tokens, 8 heads of
// 128 dims, 43 us, 6.1 TB/s (a large copy moves 5.2, a read alone more).  16-bit D = 64 takes 8
// waves: 8 x 16 heads over 1374 keys 11.1 us, 4.0 TB/s.  A wave has tiles of its own,
// so that none waits for another before the end; 32 rows fill the MFMA's columns however few
// there are, and cost nothing that the bytes would not.
constexpr int kv_step_waves(bool kv8, int d) { return !kv8 && d == 64 ? 8 : 4; }
template <bool KV8, bool BF16, int D>
struct KvStep {
  static constexpr int WAVES = kv_step_waves(KV8, D);
  static constexpr int KB = KV8 ? 2 : 1;          // 32-key blocks of a tile
  static constexpr int KT = 32 * KB;
  static constexpr int TILE = KT * D * 2;
  static constexpr int LDS = KV8 ? WAVES * 32 * D * 4 : WAVES * 4 * TILE;   // the join's rows / 2 stages of K and V
};
template <bool KV8, bool BF16, int D>
__global__ __launch_bounds__(64 * kv_step_waves(KV8, D))
    __attribute__((amdgpu_waves_per_eu(KV8 || D == 64 ? 2 : 1, KV8 || D == 64 ? 2 : 1))) void
    kv_attn_step_kernel(const KvAttn a) {
  using C = KvStep<KV8, BF16, D>;
  constexpr bool MBF = BF16 && !KV8;
  constexpr int KS = D / 16, NV = D / 32, KB = C::KB, KT = C::KT, TILE = C::TILE;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[C::LDS];
  __shared__ float2 stat[C::WAVES][32];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, l32 = lane & 31;
  // heads first: the first splits of a batch of different lengths are the full ones, and
  // as the fastest index they would all lie on the same XCDs
  const int hk = blockIdx.x, b = blockIdx.z, split = (blockIdx.y + blockIdx.z) % gridDim.y;
  const int nrows = a.Lq * a.G;                      // <= 32
  const KvRange rg = kv_range(a, b, split, 0, a.Lq - 1);
  if (rg.nq == 0) return;
  const long record = (((long)b * a.splits + split) * a.Hk + hk) * nrows;     // of a split's first row
  if (rg.t0 >= rg.t1 && a.splits > 1) {
    if (tid < nrows) a.stat[record + tid] = make_float2(-INFINITY, 0.f);
    return;
  }
  const int rc = l32 < nrows ? l32 : nrows - 1;
  const int qi = kv_query(a, rc);
  const uint16_t* qp = a.q + b * a.q_bs + qi * a.q_ts + (hk * a.G + rc - qi * a.G) * a.q_hs;
  int upto = a.causal ? rg.len - rg.nq + qi : rg.len - 1;    // the last key that the row sees
  const int first_upto = a.causal ? rg.len - rg.nq : rg.len - 1;
  KvRows<KV8, BF16, D> qr;
  KvState<D> s;
  s.init();
  KvUnits units;
  int ve = 0;                                        // of the last tile's values
  if constexpr (KV8) {
    // fragments straight from memory: the next tile's K when this one's are used, its V
    // behind the last product (no spare registers: a spilled one, read back behind these
    // loads, would wait for them)
    const long cache0 = ((long)b * a.Hk + hk) * a.blocks;
    constexpr int U = KV_BLOCK * D / 1024;           // 1 KB pieces of a block's keys or values
    uint4 kraw[U], vraw[U];
    float ks = 0.f, vs = 0.f;
    auto fetch_k = [&](int tile) __attribute__((always_inline)) {
      const uint4* kp = reinterpret_cast<const uint4*>(a.kc) + (cache0 + tile) * (KV_BLOCK * D / 16) + lane;
#pragma unroll
      for (int u = 0; u < U; ++u) kraw[u] = kp[64 * u];
    };
    auto fetch_v = [&](int tile) __attribute__((always_inline)) {
      const uint4* vp = reinterpret_cast<const uint4*>(a.vc) + (cache0 + tile) * (KV_BLOCK * D / 16) + lane;
#pragma unroll
      for (int u = 0; u < U; ++u) vraw[u] = vp[64 * u];
    };
    qr.fetch(qp, h);                                 // before the tiles: loads come back in order
    __builtin_amdgcn_sched_barrier(0);
    int tile = rg.t0 + wave;
    if (tile < rg.t1) {
      fetch_k(tile);
      ks = a.ks[cache0 + tile], vs = a.vs[cache0 + tile];
      fetch_v(tile);
    }
    __builtin_amdgcn_sched_barrier(0);
    qr.finish(a.scale_log2);
    for (; tile < rg.t1; tile += C::WAVES) {
      const int key0 = tile * KV_BLOCK;
      const bool more = tile + C::WAVES < rg.t1;
      const uint64_t seen = kv_below(rg.len - key0);
      f32x16 sc[KB];
      uint4 pf[2 * KB], lo, hi;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int u = 0; u < D / 32; ++u) {
          kv_decode(kraw[kb * (D / 32) + u], (f16x2){(_Float16)1.0f, (_Float16)1.0f}, lo, hi);
          sc[kb] = kv_mfma<MBF>(lo, qr.f[2 * u], u == 0 ? f32x16{} : sc[kb]);
          sc[kb] = kv_mfma<MBF>(hi, qr.f[2 * u + 1], sc[kb]);
        }
      const float c = kv_factor(ks, qr.mul);
      if (kv_marked(ks, vs) && (seen & kv_below(upto - key0 + 1))) s.l = __builtin_nanf("");
      const _Float16 f = (_Float16)units.fit(vs);
      __builtin_amdgcn_sched_barrier(0);
      if (more) {
        fetch_k(tile + C::WAVES);
        ks = a.ks[cache0 + tile + C::WAVES], vs = a.vs[cache0 + tile + C::WAVES];
      }
      if (units.ve != ve) {
        s.follow(ve, units.ve, upto, key0);
        ve = units.ve;
      }
      if (seen != ~0ull || first_upto < key0 + KV_BLOCK - 1) kv_mask<KB>(sc, seen & kv_below(upto - key0 + 1), h);
      kv_softmax<MBF, D, KB, false>(sc, c, s, pf, [](int) __attribute__((always_inline)) {});
#pragma unroll
      for (int db = 0; db < NV; ++db)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          kv_decode(vraw[db * 2 + w], (f16x2){f, f}, lo, hi);
          s.o[db] = kv_mfma<MBF>(lo, pf[2 * w], s.o[db]);
          s.o[db] = kv_mfma<MBF>(hi, pf[2 * w + 1], s.o[db]);
        }
      __builtin_amdgcn_sched_barrier(0);
      if (more) fetch_v(tile + C::WAVES);
    }
  } else {
    // two stages of K and V in LDS for each wave, filled by its own copies
    uint8_t* area = lds + wave * 4 * TILE;
    const uint32_t area0 = lds_addr(area);
    constexpr int DMA = TILE / 1024, RPD = 1024 / (2 * D);
    const int t1 = rg.t1 * (KV_BLOCK / KT);          // in tiles of KT keys
    int tile = rg.t0 * (KV_BLOCK / KT) + wave;
    KvSource sk, sv;
    sk.init(a.k + b * a.k_bs + hk * a.k_hs, a.k_ts, D, rg.len, (int64_t)tile * KT, KT * C::WAVES);
    sv.init(a.v + b * a.v_bs + hk * a.v_hs, a.v_ts, D, rg.len, (int64_t)tile * KT, KT * C::WAVES);
    auto issue = [&](int buf) __attribute__((always_inline)) {      // the wave's next tile
      const auto rk = sk.rsrc(KT), rv = sv.rsrc(KT);
#pragma unroll
      for (int w = 0; w < DMA; ++w) {
        const int r0 = RPD * w, row = r0 + lane / (D / 8), c = lane % (D / 8);
        kv_dma16(rk, (uint32_t)(lane / (D / 8)) * sk.row + ((c ^ kv_fk<D>(row)) * 16), (uint32_t)r0 * sk.row,
                 area0 + 2 * buf * TILE + r0 * (2 * D));
      }
#pragma unroll
      for (int w = 0; w < DMA; ++w) {
        const int r0 = RPD * w, row = r0 + lane / (D / 8), c = lane % (D / 8);
        kv_dma16(rv, (uint32_t)(lane / (D / 8)) * sv.row + ((c ^ kv_fv<D>(row)) * 16), (uint32_t)r0 * sv.row,
                 area0 + (2 * buf + 1) * TILE + r0 * (2 * D));
      }
      sk.next();
      sv.next();
    };
    static_assert(2 * DMA == 8 || 2 * DMA == 16, "the wait below counts the copies of one stage");
    int buf = 0;
    uint8_t mask_byte = 1;
    qr.fetch(qp, h);
    __builtin_amdgcn_sched_barrier(0);
    if (tile < t1) issue(0);
    qr.finish(a.scale_log2);
    for (; tile < t1; tile += C::WAVES) {
      const int key0 = tile * KT;
      const bool more = tile + C::WAVES < t1;
      if (a.mask) {
        const int key = key0 + lane;
        mask_byte = key < rg.len && lane < KT ? a.mask[b * a.mask_bs + key] : 0;
      }
      constexpr uint64_t ALL = KT == 64 ? ~0ull : 0xFFFFFFFFull;
      const uint64_t seen = a.mask ? __builtin_amdgcn_ballot_w64(mask_byte != 0) : kv_below(rg.len - key0) & ALL;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // the other stage's reads are done
      if (more) {
        issue(buf ^ 1);
        if constexpr (2 * DMA == 8) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");      // this stage's copies have landed
        else asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      uint8_t* kt = area + 2 * buf * TILE;
      uint8_t* vt = kt + TILE;
      if (seen != ALL) {                             // value rows that are left out may hold anything
#pragma unroll
        for (int i = lane; i < TILE / 16; i += 64)
          if (!((seen >> (i / (D / 8))) & 1)) reinterpret_cast<uint4*>(vt)[i] = make_uint4(0, 0, 0, 0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      if (seen) {
        f32x16 sc[KB];
        uint4 pf[2 * KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int st = 0; st < KS; ++st)
            sc[kb] = kv_mfma<MBF>(kv_frag_k<D>(kt, kb, st, h, l32), qr.f[st], st == 0 ? f32x16{} : sc[kb]);
        if (seen != ALL) kv_mask<KB>(sc, seen, h);
        kv_softmax<MBF, D, KB, false>(sc, qr.mul, s, pf, [](int) __attribute__((always_inline)) {});
#pragma unroll
        for (int st = 0; st < 2 * KB; ++st)
#pragma unroll
          for (int db = 0; db < NV; ++db) s.o[db] = kv_mfma<MBF>(kv_frag_v<D>(vt, db, st, lane), pf[st], s.o[db]);
      }
      buf ^= 1;
    }
  }
  // ---- join the waves: every wave's O under the common reference, summed in wave order
  const float l = kv_half_sum(s.l);
  __syncthreads();                                   // all tiles read
  if (h == 0) stat[wave][l32] = make_float2(s.m, l);
  __syncthreads();
  float m = -INFINITY;
#pragma unroll
  for (int w = 0; w < C::WAVES; ++w) m = fmaxf(m, stat[w][l32].x);
  const float ref = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < C::WAVES; ++w) sum += stat[w][l32].y * __builtin_amdgcn_exp2f(stat[w][l32].x - ref);
  const float by = sum == 0.f ? 0.f : __builtin_amdgcn_exp2f(s.m - ref) / sum;
  const int unit = kv_unit(upto, ve);
  float* join = reinterpret_cast<float*>(lds);       // [wave][row][D]
  if (l32 < nrows)
#pragma unroll
    for (int db = 0; db < NV; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(join + (wave * 32 + l32) * D + 32 * db + 8 * g + 4 * h) =
            make_float4(kv_out<KV8>(s.o[db][4 * g], by, unit), kv_out<KV8>(s.o[db][4 * g + 1], by, unit),
                        kv_out<KV8>(s.o[db][4 * g + 2], by, unit), kv_out<KV8>(s.o[db][4 * g + 3], by, unit));
  __syncthreads();
  const int rows_out = nrows < rg.nq * a.G ? nrows : rg.nq * a.G;
  for (int i = tid; i < rows_out * (D / 4); i += 64 * C::WAVES) {
    const int row = i / (D / 4), d = 4 * (i % (D / 4)), query = kv_query(a, row);
    float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < C::WAVES; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(join + (w * 32 + row) * D + d);
      o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
    }
    if (a.splits == 1) {
      uint16_t* op = a.out + b * a.o_bs + query * a.o_ts + (hk * a.G + row - query * a.G) * a.o_hs + d;
      *reinterpret_cast<uint2*>(op) = make_uint2(pack2<BF16>(o.x, o.y), pack2<BF16>(o.z, o.w));
    } else {
      *reinterpret_cast<float4*>(a.part + (record + row) * D + d) = o;
    }
  }
  if (a.splits > 1 && wave == 0 && h == 0 && l32 < rows_out) {
    a.stat[record + l32] = make_float2(m, sum);
  }
}

// ------------------------------------------------------------------ join of the splits
// A thread takes 4 dims of one row: sum of the splits' quotients, weighted by l 2^m, with
// a running maximum, so that all loads are on their way at once.  Some 4 us for few rows (the
// launch and two dependent reads), 7 us for 5 splits of 1374 queries of 16 heads of 64 dims.
template <bool BF16, int D>
__global__ __launch_bounds__(256) void kv_attn_join_kernel(const KvAttn a) {
  const int b = blockIdx.z, hk = blockIdx.y;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  const uint32_t row = i / (D / 4), per = (uint32_t)a.Lq * a.G;
  if (row >= per) return;
  const int d = 4 * (int)(i % (D / 4));
  const int qi = kv_query(a, row);
  if (a.counts && qi >= a.counts[b]) return;
  const long rows = (long)a.Hk * per;                // of a split
  const long at = (long)b * a.splits * rows + (long)hk * per + row;
  const float2* stat = a.stat + at;
  const float* part = a.part + at * D + d;
  float m = -INFINITY, sum = 0.f;
  float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float2 st = stat[s * rows];
    const float4 x = *reinterpret_cast<const float4*>(part + s * rows * D);
    const float up = fmaxf(m, st.x), ref = up == -INFINITY ? 0.f : up;
    const float keep = __builtin_amdgcn_exp2f(m - ref), w = st.y * __builtin_amdgcn_exp2f(st.x - ref);
    m = up;
    sum = sum * keep + w;
    // a split that saw nothing (w = 0) has no part; NaN counts
    o.x = o.x * keep + (w != 0.f ? w * x.x : 0.f), o.y = o.y * keep + (w != 0.f ? w * x.y : 0.f);
    o.z = o.z * keep + (w != 0.f ? w * x.z : 0.f), o.w = o.w * keep + (w != 0.f ? w * x.w : 0.f);
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  uint16_t* op = a.out + b * a.o_bs + qi * a.o_ts + (hk * a.G + (int)row - qi * a.G) * a.o_hs + d;
  *reinterpret_cast<uint2*>(op) = make_uint2(pack2<BF16>(o.x * inv, o.y * inv), pack2<BF16>(o.z * inv, o.w * inv));
}

// ------------------------------------------------------------------ launch plan
struct KvPlan {
  bool step;
  int qb, splits, row_tiles;
};

// `keys`: tokens that a sequence may have (a hint: the kernels divide what they find).
static KvPlan kv_plan(bool kv8, int64_t B, int64_t Lq, int64_t H, int64_t Hk, int64_t D, int64_t keys) {
  const int64_t rows = Lq * (H / Hk), heads = B * Hk, tiles = (keys + KV_BLOCK - 1) / KV_BLOCK;
  KvPlan p = {};
  if (rows <= 32) {
    p.step = true, p.qb = 1, p.row_tiles = 1;
    // 8-bit: two workgroups a CU, twice as many splits where sequences may differ (16 of up
    // to 8001 tokens: as fast when all are full, 19 instead of 27 us when all hold 2048).
    // 16-bit: one a CU; from half the CUs on no split, which saves the join, while keys and
    // values fit the 256 MB that the caches behind the L2 hold: 8 x 16 heads of 64 over 1374
    // keys 14.5 us against 18.5 split in two, 6870 keys (225 MB) 37.7 against 40.5; but 10992
    // 93.9 against 72.2 and 43968 365 against 280, as half the CUs do not draw what the HBM
    // gives (heads of 128: 1374 keys 20.9 and 21.0, 13740 187 against 158)
    const bool kept = 4 * heads * keys * D <= (256 << 20);
    const int64_t slots = kv8 ? (B > 1 ? 1024 : 512) : heads >= 128 && kept ? 1 : 256;
    int64_t s = heads < slots ? slots / (heads > 0 ? heads : 1) : 1;
    if (s > tiles / 8) s = tiles / 8;                       // a tile or two for each wave at least
    if (s > 64) s = 64;
    p.splits = (int)(s < 1 ? 1 : s);
    return p;
  }
  p.qb = D == 64 && rows > 128 ? 2 : 1;
  p.row_tiles = (int)((rows + 128 * p.qb - 1) / (128 * p.qb));
  const int64_t wg = heads * p.row_tiles;
  // time of s splits in ns: rounds of 512 workgroups, two a CU (the last cheaper with at
  // most one a CU), each of its tiles and some 3 tiles' worth of prologue and end; the
  // join.  A tile's time lies between those over 16- and 8-bit keys (two a CU: wide 2243 and
  // 2468, D = 128 2092 and 2297; one: 1358 and 1543, 1239 and 1553; few rows of D = 64 1182
  // and 806 over keys that stay in the caches, 1665 and 993 over ones that do not).
  // Several sequences may be of any lengths: the mean of all full, and of half the keys
  // spread over the CUs with one sequence still full.
  const double pair = p.qb == 2 ? 2430 : D == 64 ? 1300 : 2100, one = p.qb == 2 ? 1480 : D == 64 ? 860 : 1240;
  double best = 1e300;
  p.splits = 1;
  for (int64_t s = 1; s <= 64 && s <= (tiles > 1 ? tiles : 1); ++s) {
    const int64_t n = wg * s, rem = n % 512;
    const double per = (double)((tiles + s - 1) / s) + 3;
    double t = (double)(n / 512) * per * pair + (rem == 0 ? 0 : rem <= 256 ? per * one : per * pair);
    if (B > 1) {
      const double half = 0.5 * n * per / 512 * pair;
      t = 0.5 * (t + (half > per * one ? half : per * one));
    }
    if (s > 1) t += 4000 + (double)s * B * H * Lq * D * 8 / 8000;
    if (t < best) best = t, p.splits = (int)s;
  }
  return p;
}

static int64_t kv_split_bytes(int64_t B, int64_t Lq, int64_t H, int64_t D) { return B * Lq * H * (D * 4 + 8); }

template <bool KV8, bool BF16, int D>
static void kv_launch(const KvAttn& a, const KvPlan& p, hipStream_t st) {
  const int64_t n = (int64_t)a.B * a.Hk * p.splits * p.row_tiles, round = 8 * KV_NEAR;
  const unsigned wg = (unsigned)((n + round - 1) / round * round);
  if (p.step) {
    hipLaunchKernelGGL((kv_attn_step_kernel<KV8, BF16, D>), dim3(a.Hk, p.splits, a.B), dim3(64 * kv_step_waves(KV8, D)), 0, st, a);
  } else if (D == 64 && p.qb == 2) {
    hipLaunchKernelGGL((kv_attn_wide_kernel<KV8, BF16>), dim3(wg), dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((kv_attn_pipe_kernel<KV8, BF16, D>), dim3(wg), dim3(256), 0, st, a);
  }
  if (p.splits > 1) {
    const long threads = (long)a.G * a.Lq * (D / 4);
    hipLaunchKernelGGL((kv_attn_join_kernel<BF16, D>), dim3((unsigned)((threads + 255) / 256), a.Hk, a.B), dim3(256), 0, st, a);
  }
}

// Checks and fields that both entries share.
static int kv_common(KvAttn& a, const void* q, void* out, int dtype, int64_t B, int64_t Lq, int64_t Lk,
                     int64_t H, int64_t Hk, int64_t D, const int64_t* qs, const int64_t* os, float scale) {
  QV_CHECK_ARG(dtype == QV_F16 || dtype == QV_BF16, "bad dtype %d", dtype);
  QV_CHECK_ARG(D == 64 || D == 128, "head_dim must be 64 or 128 (got %lld)", (long long)D);
  QV_CHECK_ARG(B >= 0 && Lq >= 0 && Lk >= 0 && H > 0 && Hk > 0 && H % Hk == 0 && B <= (1 << 20) && Lq <= (1 << 28) &&
                   Lk <= (1 << 30) && H <= 65536,
               "bad shape B=%lld Lq=%lld Lk=%lld heads=%lld / %lld", (long long)B, (long long)Lq, (long long)Lk,
               (long long)H, (long long)Hk);
  QV_CHECK_ARG(scale > 0.f && scale < INFINITY, "the scale must be a positive number");
  QV_CHECK_ARG(Lq * (H / Hk) <= INT32_MAX / 2 && Lq * (H / Hk) * (H / Hk) < (1ll << 32) && B * H * Lq <= (1ll << 36),
               "too many rows");
  if (B == 0 || Lq == 0) return QV_OK;
  QV_CHECK_ARG(q && out && qs && os, "null pointer argument");
  QV_CHECK_ARG((uintptr_t)q % 16 == 0 && (uintptr_t)out % 8 == 0, "q must be 16-byte and out 8-byte aligned");
  for (int i = 0; i < 3; ++i)
    QV_CHECK_ARG(qs[i] % 8 == 0 && os[i] % 4 == 0, "q strides must be multiples of 8 elements, out strides of 4");
  a.q = (const uint16_t*)q, a.out = (uint16_t*)out;
  a.B = (int)B, a.Lq = (int)Lq, a.Lk = (int)Lk, a.H = (int)H, a.Hk = (int)Hk, a.G = (int)(H / Hk);
  a.q_bs = qs[0], a.q_ts = qs[1], a.q_hs = qs[2];
  a.o_bs = os[0], a.o_ts = os[1], a.o_hs = os[2];
  a.g_mul = a.G == 1 ? 0 : (uint32_t)((1ull << 32) / a.G + 1);
  a.scale_log2 = scale * 1.4426950408889634f;
  return QV_OK;
}

// Splits that the workspace holds, and where their parts lie.
static int kv_place(KvAttn& a, KvPlan& p, int64_t D, int64_t tiles, void* ws, int64_t ws_bytes) {
  const int64_t per = kv_split_bytes(a.B, a.Lq, a.H, D);
  if (p.splits > 1 && (!ws || (uintptr_t)ws % 16)) p.splits = 1;
  if (p.splits > 1 && p.splits * per > ws_bytes) p.splits = (int)(ws_bytes / per > 1 ? ws_bytes / per : 1);
  a.splits = p.splits, a.row_tiles = p.row_tiles;
  a.split_tiles = (int)((tiles + p.splits - 1) / p.splits);
  QV_CHECK_ARG((int64_t)a.B * a.Hk * p.splits * p.row_tiles <= INT32_MAX - 64 && a.B <= 65535 && a.Hk <= 65535,
               "grid too large");
  a.part = (float*)ws;
  a.stat = (float2*)((char*)ws + (size_t)p.splits * a.B * a.Lq * a.H * D * 4);
  return QV_OK;
}

}  // namespace qv

extern "C" int64_t qv_attention_kv_workspace(int cached, int64_t B, int64_t Lq, int64_t H, int64_t Hk, int64_t D,
                                             int64_t keys) {
  if (B <= 0 || Lq <= 0 || H <= 0 || Hk <= 0 || H % Hk || keys < 0 || (D != 64 && D != 128)) return 0;
  const qv::KvPlan p = qv::kv_plan(cached != 0, B, Lq, H, Hk, D, keys);
  return p.splits > 1 ? p.splits * qv::kv_split_bytes(B, Lq, H, D) : 0;
}

#define QV_KV_LAUNCH(KV8)                                                                          \
  if (D == 64) {                                                                                   \
    if (dtype == QV_BF16) qv::kv_launch<KV8, true, 64>(a, p, (hipStream_t)stream);                 \
    else qv::kv_launch<KV8, false, 64>(a, p, (hipStream_t)stream);                                 \
  } else {                                                                                         \
    if (dtype == QV_BF16) qv::kv_launch<KV8, true, 128>(a, p, (hipStream_t)stream);                \
    else qv::kv_launch<KV8, false, 128>(a, p, (hipStream_t)stream);                                \
  }

extern "C" int qv_attention_cross(const void* q, const void* k, const void* v, void* out, int dtype, const int32_t* lens,
                                  const uint8_t* mask, int64_t mask_stride, int64_t B, int64_t Lq, int64_t Lk, int64_t H,
                                  int64_t Hk, int64_t D, const int64_t* q_strides, const int64_t* k_strides,
                                  const int64_t* v_strides, const int64_t* out_strides, float scale, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  qv::KvAttn a = {};
  if (int rc = qv::kv_common(a, q, out, dtype, B, Lq, Lk, H, Hk, D, q_strides, out_strides, scale))
    return rc;
  if (B == 0 || Lq == 0) return QV_OK;
  if (Lk > 0) {
    QV_CHECK_ARG(k && v && k_strides && v_strides, "null pointer argument");
    QV_CHECK_ARG((uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0, "k and v must be 16-byte aligned");
    for (int i = 0; i < 3; ++i)
      QV_CHECK_ARG(k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0, "k and v strides must be multiples of 8 elements");
    for (const int64_t ts : {k_strides[1], v_strides[1]})
      QV_CHECK_ARG(Lk == 1 || (ts >= D && ts <= (1 << 24)), "k and v token strides must be %lld to 2^24 elements", (long long)D);
    a.k = (const uint16_t*)k, a.v = (const uint16_t*)v;
    a.k_bs = k_strides[0], a.k_ts = Lk == 1 ? D : k_strides[1], a.k_hs = k_strides[2];
    a.v_bs = v_strides[0], a.v_ts = Lk == 1 ? D : v_strides[1], a.v_hs = v_strides[2];
    a.lens = lens, a.mask = mask, a.mask_bs = mask_stride;
  }
  qv::KvPlan p = qv::kv_plan(false, B, Lq, H, Hk, D, Lk);
  if (int rc = qv::kv_place(a, p, D, (Lk + qv::KV_BLOCK - 1) / qv::KV_BLOCK, workspace, workspace_bytes)) return rc;
  QV_KV_LAUNCH(false)
  return qv::check_launch("attention_cross");
}

extern "C" int qv_kv8_attention(const void* q, void* out, int dtype, const void* k_codes, const void* v_codes,
                                const float* k_scales, const float* v_scales, const int32_t* lens, const int32_t* counts,
                                int causal, int64_t B, int64_t Lq, int64_t H, int64_t Hk, int64_t D, int64_t blocks,
                                int64_t keys, const int64_t* q_strides, const int64_t* out_strides, float scale,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  qv::KvAttn a = {};
  QV_CHECK_ARG(blocks > 0 && blocks <= (INT32_MAX >> 8), "bad number of blocks %lld", (long long)blocks);
  if (int rc = qv::kv_common(a, q, out, dtype, B, Lq, blocks * qv::KV_BLOCK, H, Hk, D, q_strides,
                             out_strides, scale))
    return rc;
  if (B == 0 || Lq == 0) return QV_OK;
  QV_CHECK_ARG(k_codes && v_codes && k_scales && v_scales && lens, "null pointer argument");
  QV_CHECK_ARG((uintptr_t)k_codes % 16 == 0 && (uintptr_t)v_codes % 16 == 0, "codes must be 16-byte aligned");
  a.kc = (const uint8_t*)k_codes, a.vc = (const uint8_t*)v_codes, a.ks = k_scales, a.vs = v_scales;
  a.lens = lens, a.counts = counts, a.causal = causal != 0, a.blocks = (int)blocks;
  if (keys < 0 || keys > blocks * qv::KV_BLOCK) keys = blocks * qv::KV_BLOCK;
  qv::KvPlan p = qv::kv_plan(true, B, Lq, H, Hk, D, keys);
  if (int rc = qv::kv_place(a, p, D, (keys + qv::KV_BLOCK - 1) / qv::KV_BLOCK, workspace, workspace_bytes)) return rc;
  QV_KV_LAUNCH(true)
  return qv::check_launch("kv8_attention");
}
