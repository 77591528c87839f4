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
// Forms:
//  * wide: 4 waves, each 32 or 64 rows of its own, K / V tiles of the workgroup in LDS
//    (16-bit: LDS DMA; 8-bit: codes through registers, converted once by the whole
//    workgroup, stored in fragment order);
//  * step: up to 32 rows, every wave its own tiles of the key range (16-bit: LDS
//    areas of its own; 8-bit: fragments straight from memory), joined in LDS.
// In both the key range may be split over workgroups, joined by a second kernel.
//
// 8-bit values: scores are products of 16-bit queries with whole numbers, the key
// block's scale goes into c.  bf16 queries become fp16 under a power of two of their
// row (exact down to 2^-38 of the row's largest).  Value codes are multiplied by
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
  int B, Lq, H, Hk, G, Lk, blocks, causal, splits, row_tiles;
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
// lanes).  top: the largest ve so far.
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
    return __builtin_ldexpf(s, -ve);    // NaN stays NaN
  }
};

// Key-scale factor of the scores; kept off 0 so that a masked score (-inf) times it stays -inf.
__device__ __forceinline__ float kv_factor(float c) { return c < 1e-37f ? 1e-37f : c; }

// The fragments of one wave's 32 rows, and what their scores are multiplied by.
template <bool KV8, bool BF16, int D>
struct KvRows {
  static constexpr bool MBF = BF16 && !KV8;   // MFMA type
  uint4 f[D / 16];
  float mul;
  __device__ __forceinline__ void load(const uint16_t* p, int h, float scale_log2) {
    mul = scale_log2;
#pragma unroll
    for (int st = 0; st < D / 16; ++st)
      f[st] = *reinterpret_cast<const uint4*>(p + (KV8 ? 32 * (st >> 1) + 16 * h + 8 * (st & 1) : 16 * st + 8 * h));
    if constexpr (KV8 && BF16) {
      float mx = 0.f;
#pragma unroll
      for (int st = 0; st < D / 16; ++st) {
        const uint32_t w[4] = {f[st].x, f[st].y, f[st].z, f[st].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mx = fmaxf(mx, fmaxf(__builtin_fabsf(to_f32((uint16_t)w[i], true)), __builtin_fabsf(to_f32((uint16_t)(w[i] >> 16), true))));
      }
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
  float t = 0.f;
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
      t = kv_add_pair<BF>(pw[2 * i - 1], t);
    }
    pw[2 * i] = word(2 * i, s.ref);
    pw[2 * i + 1] = word(2 * i + 1, s.ref);
    if constexpr (FENCE) __builtin_amdgcn_sched_barrier(0);
  }
  t = kv_add_pair<BF>(pw[W - 2], t);
  t = kv_add_pair<BF>(pw[W - 1], t);
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

// A 16-bit K or V source, tile by tile: the address of the next tile's first row and
// the bytes left of the sequence from there (what lies behind them reads as zero).
// 64-bit: a long cache passes the 32 bits of a buffer offset.
struct KvSource {
  const uint8_t* at;
  int64_t left, step;
  uint32_t row;           // bytes from row to row
  __device__ __forceinline__ void init(const uint16_t* base, long ts, int D, int len, int64_t key0, int keys) {
    at = reinterpret_cast<const uint8_t*>(base) + key0 * ts * 2;
    left = ((len - 1 - key0) * ts + D) * 2;
    step = (int64_t)keys * ts * 2;
    row = (uint32_t)(ts * 2);
  }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc() const {
    const int64_t n = left < 0 ? 0 : left > 0xFFFFFFFFll ? 0xFFFFFFFFll : left;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(at), (short)0, (int)(uint32_t)n, 0x00020000);
  }
  __device__ __forceinline__ void next() { at += step, left -= step; }
};

// The sequence's keys, queries and the tiles of a row tile's split.
struct KvRange {
  int len, nq, t0, t1;
};
__device__ __forceinline__ KvRange kv_range(const KvAttn& a, int b, int row0, int rows_tile, int split) {
  KvRange r;
  r.len = a.Lk;
  if (a.lens) {
    const int l = a.lens[b];
    r.len = l < 0 ? 0 : l > a.Lk ? a.Lk : l;
  }
  r.nq = a.Lq;
  if (a.counts) {
    const int c = a.counts[b];
    r.nq = c < 0 ? 0 : c > a.Lq ? a.Lq : c;
  }
  int last = r.len;                       // keys that the tile's last row sees
  if (a.causal) {
    int qi = (row0 + rows_tile - 1) / a.G;
    qi = qi < r.nq ? qi : r.nq - 1;
    last = r.len - r.nq + qi + 1;
    last = last < 0 ? 0 : last > r.len ? r.len : last;
  }
  const int nt = row0 / a.G < r.nq ? (last + KV_BLOCK - 1) / KV_BLOCK : 0;
  r.t0 = (int)((long)nt * split / a.splits);
  r.t1 = (int)((long)nt * (split + 1) / a.splits);
  return r;
}

// Store a lane's row: the quotient to out, or to the split's part with m and l.
template <bool BF16, int D>
__device__ __forceinline__ void kv_store(const KvAttn& a, const KvState<D>& s, float l, int ve, int b, int hk, int row,
                                         int split, int h, bool live) {
  if (!live) return;
  const float inv = l == 0.f ? 0.f : __builtin_ldexpf(1.0f / l, ve);
  const int qi = row / a.G, head = hk * a.G + row % a.G;
  if (a.splits == 1) {
    uint16_t* op = a.out + b * a.o_bs + qi * a.o_ts + head * a.o_hs;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint2 w;
        w.x = pack2<BF16>(s.o[db][4 * g] * inv, s.o[db][4 * g + 1] * inv);
        w.y = pack2<BF16>(s.o[db][4 * g + 2] * inv, s.o[db][4 * g + 3] * inv);
        *reinterpret_cast<uint2*>(op + 32 * db + 8 * g + 4 * h) = w;
      }
  } else {
    const long rows = (long)a.B * a.H * a.Lq;
    const long at = (long)split * rows + ((long)b * a.Hk + hk) * ((long)a.Lq * a.G) + row;
    float* pp = a.part + at * D;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(pp + 32 * db + 8 * g + 4 * h) =
            make_float4(s.o[db][4 * g] * inv, s.o[db][4 * g + 1] * inv, s.o[db][4 * g + 2] * inv, s.o[db][4 * g + 3] * inv);
    if (h == 0) a.stat[at] = make_float2(s.m, l);
  }
}

// ------------------------------------------------------------------ wide form
template <bool KV8, bool BF16, int D, int QB>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(QB == 1 && D == 64 ? 3 : 2, QB == 1 && D == 64 ? 3 : 2))) void kv_attn_wide_kernel(const KvAttn a) {
  constexpr bool MBF = BF16 && !KV8;
  constexpr int TILE = KV_BLOCK * D * 2;             // bytes of a 16-bit K or V tile
  constexpr int KS = D / 16, NV = D / 32;
  constexpr int ROWS = 4 * 32 * QB;
  __shared__ __attribute__((aligned(1024))) uint8_t k_lds[2][TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t v_lds[2][TILE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, l32 = lane & 31;
  // consecutive row tiles of one (sequence, key head, split) share an XCD and its L2
  const int lid = xcd_remap(blockIdx.x, gridDim.x);
  const int rt = lid % a.row_tiles;
  const int split = lid / a.row_tiles % a.splits;
  const int hk = lid / (a.row_tiles * a.splits) % a.Hk;
  const int b = lid / (a.row_tiles * a.splits * a.Hk);
  const int nrows = a.Lq * a.G;
  const int row0 = rt * ROWS;
  const KvRange rg = kv_range(a, b, row0, nrows - row0 < ROWS ? nrows - row0 : ROWS, split);
  if (row0 / a.G >= rg.nq) return;
  const int wrow = row0 + wave * 32 * QB;
  const bool live = wrow < nrows && wrow / a.G < rg.nq;      // wave-uniform

  KvRows<KV8, BF16, D> qr[QB];
  KvState<D> s[QB];
  int row[QB], upto[QB];                             // upto: the last key that the row sees
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    row[qb] = wrow + 32 * qb + l32;
    const int rc = row[qb] < nrows ? row[qb] : nrows - 1;
    const int qi = rc / a.G, head = hk * a.G + rc % a.G;
    qr[qb].load(a.q + b * a.q_bs + qi * a.q_ts + head * a.q_hs, h, a.scale_log2);
    upto[qb] = a.causal ? rg.len - rg.nq + qi : rg.len - 1;
    s[qb].init();
  }
  const int first_upto = a.causal ? rg.len - rg.nq + wrow / a.G : rg.len - 1;    // of the wave's first row

  // ---- tiles of the 16-bit source
  constexpr int DMA = TILE / 1024 / 4;               // 1 KB copies of a wave for K and for V
  constexpr int RPD = 1024 / (2 * D);                // rows of a copy
  const uint32_t klds0 = lds_addr(k_lds), vlds0 = lds_addr(v_lds);
  KvSource sk, sv;
  uint32_t k_voff[DMA], v_voff[DMA];
  if constexpr (!KV8) {
    const int64_t key0 = (int64_t)rg.t0 * KV_BLOCK;
    sk.init(a.k + b * a.k_bs + hk * a.k_hs, a.k_ts, D, rg.len, key0, KV_BLOCK);
    sv.init(a.v + b * a.v_bs + hk * a.v_hs, a.v_ts, D, rg.len, key0, KV_BLOCK);
#pragma unroll
    for (int w = 0; w < DMA; ++w) {
      const int r = RPD * (DMA * wave + w) + lane / (D / 8), c = lane % (D / 8);
      k_voff[w] = (uint32_t)(lane / (D / 8)) * sk.row + ((c ^ kv_fk<D>(r)) * 16);
      v_voff[w] = (uint32_t)(lane / (D / 8)) * sv.row + ((c ^ kv_fv<D>(r)) * 16);
    }
  }
  auto issue16 = [&](int buf) __attribute__((always_inline)) {      // the next tile
    const auto rk = sk.rsrc(), rv = sv.rsrc();
#pragma unroll
    for (int w = 0; w < DMA; ++w) {
      const int r0 = RPD * (DMA * wave + w);
      kv_dma16(rk, k_voff[w], (uint32_t)r0 * sk.row, klds0 + buf * TILE + r0 * (2 * D));
      kv_dma16(rv, v_voff[w], (uint32_t)r0 * sv.row, vlds0 + buf * TILE + r0 * (2 * D));
    }
    sk.next();
    sv.next();
  };
  // ---- tiles of the cache: 16 codes a thread and step, one 16-byte unit
  constexpr int UNITS = KV_BLOCK * D / 16 / 256;     // of a thread for K and for V
  const long cache0 = ((long)b * a.Hk + hk) * a.blocks;
  uint4 kraw[UNITS], vraw[UNITS];
  float ks_next = 0.f, vs_next = 0.f;
  auto fetch8 = [&](int tile) __attribute__((always_inline)) {
    const uint4* kp = reinterpret_cast<const uint4*>(a.kc) + (cache0 + tile) * (KV_BLOCK * D / 16);
    const uint4* vp = reinterpret_cast<const uint4*>(a.vc) + (cache0 + tile) * (KV_BLOCK * D / 16);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      kraw[u] = kp[256 * u + tid];
      vraw[u] = vp[256 * u + tid];
    }
    ks_next = a.ks[cache0 + tile];
    vs_next = a.vs[cache0 + tile];
  };
  KvUnits units;
  auto place8 = [&](int buf) __attribute__((always_inline)) {
    const _Float16 f = (_Float16)units.fit(vs_next);
    uint4* kt = reinterpret_cast<uint4*>(k_lds[buf]);
    uint4* vt = reinterpret_cast<uint4*>(v_lds[buf]);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int unit = 256 * u + tid, at = (unit >> 6) * 128 + (unit & 63);
      uint4 lo, hi;
      kv_decode(kraw[u], (f16x2){(_Float16)1.0f, (_Float16)1.0f}, lo, hi);
      kt[at] = lo, kt[at + 64] = hi;
      kv_decode(vraw[u], (f16x2){f, f}, lo, hi);
      vt[at] = lo, vt[at + 64] = hi;
    }
  };
  auto frag_k = [&](int buf, int kb, int st) __attribute__((always_inline)) {
    if constexpr (KV8) return reinterpret_cast<const uint4*>(k_lds[buf])[(kb * KS + st) * 64 + lane];
    else return kv_frag_k<D>(k_lds[buf], kb, st, h, l32);
  };
  auto frag_v = [&](int buf, int db, int st) __attribute__((always_inline)) {
    if constexpr (KV8) return reinterpret_cast<const uint4*>(v_lds[buf])[(db * 4 + st) * 64 + lane];
    else return kv_frag_v<D>(v_lds[buf], db, st, lane);
  };

  // One tile.  At most 8 K and then 8 V fragments are held at a time (32 registers each).
  // QB = 2: the first block's QK, then the second's beside the first's softmax, the
  // first's PV beside the second's softmax.
  auto compute = [&](int buf, const float (&c)[QB], bool masked, uint64_t seen, int key0) __attribute__((always_inline)) {
    f32x16 sc[QB][2];
    uint4 pf[QB][4];
    constexpr int KG = KS / 4, VG = NV * 4 / 8;      // groups of 8 fragments
    uint4 kf[KG][8], vf[VG][8];
    auto read_k = [&](int g) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) kf[g][i] = frag_k(buf, i & 1, 4 * g + (i >> 1));
    };
    auto read_v = [&](int g, int i) __attribute__((always_inline)) {
      const int f = 8 * g + i;
      vf[g][i] = frag_v(buf, f % NV, f / NV);
    };
    auto qk = [&](int qb, int f) __attribute__((always_inline)) {    // f = 0 .. 2 KS - 1
      const int kb = f & 1, st = f >> 1;
      sc[qb][kb] = kv_mfma<MBF>(kf[f / 8][f % 8], qr[qb].f[st], st == 0 ? f32x16{} : sc[qb][kb]);
    };
    auto pv = [&](int qb, int f) __attribute__((always_inline)) {    // f = 0 .. 4 NV - 1
      s[qb].o[f % NV] = kv_mfma<MBF>(vf[f / 8][f % 8], pf[qb][f / NV], s[qb].o[f % NV]);
    };
    auto mask = [&](int qb) __attribute__((always_inline)) {
      if (masked) kv_mask<2>(sc[qb], seen & kv_below(upto[qb] - key0 + 1), h);
    };
    read_k(0);
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      if (g + 1 < KG) read_k(g + 1);
      if constexpr (KG > 1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 8; ++i) qk(0, 8 * g + i);
    }
    mask(0);
    if constexpr (QB == 2) {
      static_assert(QB == 1 || (KG == 1 && VG == 1), "two row blocks: D = 64");
      kv_softmax<MBF, D, 2, true>(sc[0], c[0], s[0], pf[0], [&](int i) __attribute__((always_inline)) {
        qk(1, i);
        if (i >= 4) {
          read_v(0, 2 * (i - 4));
          read_v(0, 2 * (i - 4) + 1);
        }
      });
      mask(1);
      kv_softmax<MBF, D, 2, true>(sc[1], c[1], s[1], pf[1], [&](int i) __attribute__((always_inline)) { pv(0, i); });
#pragma unroll
      for (int i = 0; i < 8; ++i) pv(1, i);
    } else {
      kv_softmax<MBF, D, 2, (VG > 1)>(sc[0], c[0], s[0], pf[0], [&](int i) __attribute__((always_inline)) {
        if (i >= 4) {
          read_v(0, 2 * (i - 4));
          read_v(0, 2 * (i - 4) + 1);
        }
      });
#pragma unroll
      for (int g = 0; g < VG; ++g) {
        if (g + 1 < VG)
#pragma unroll
          for (int i = 0; i < 8; ++i) read_v(g + 1, i);
        if constexpr (VG > 1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 8; ++i) pv(0, 8 * g + i);
      }
    }
  };

  int ve = 0;                                        // of O
  float ks = 0.f;
  uint8_t mask_byte = 1;
  auto load_mask = [&](int tile) __attribute__((always_inline)) {
    const int key = tile * KV_BLOCK + lane;
    mask_byte = key < rg.len ? a.mask[b * a.mask_bs + key] : 0;
  };
  if (rg.t0 < rg.t1) {
    if constexpr (KV8) {
      fetch8(rg.t0);
      place8(0);
      ks = ks_next;
    } else {
      issue16(0);
      if (a.mask) load_mask(rg.t0);
      __builtin_amdgcn_s_waitcnt(0x0F70);            // vmcnt(0)
    }
    lds_barrier();
  }
  for (int tile = rg.t0; tile < rg.t1; ++tile) {
    const int buf = (tile - rg.t0) & 1, key0 = tile * KV_BLOCK;
    const bool more = tile + 1 < rg.t1;
    uint64_t seen = kv_below(rg.len - key0);
    if constexpr (!KV8) {
      if (a.mask) {
        seen = __builtin_amdgcn_ballot_w64(mask_byte != 0);
        if (more) load_mask(tile + 1);
      }
      if (seen != ~0ull) {                           // value rows that are left out may hold anything
        for (int i = tid; i < TILE / 16; i += 256)
          if (!((seen >> (i / (D / 8))) & 1)) reinterpret_cast<uint4*>(v_lds[buf])[i] = make_uint4(0, 0, 0, 0);
        lds_barrier();
      }
    }
    if (more) {
      if constexpr (KV8) fetch8(tile + 1);
      else issue16(buf ^ 1);
    }
    if (live && seen) {
      float c[QB];
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) c[qb] = KV8 ? kv_factor((ks > 0.f || ks != ks ? ks : 1.0f) * qr[qb].mul) : qr[qb].mul;
      if constexpr (KV8) {
        if (units.ve != ve) {
          const float by = __builtin_ldexpf(1.0f, ve - units.ve);
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) s[qb].scale(by);
        }
      }
      compute(buf, c, seen != ~0ull || first_upto < key0 + KV_BLOCK - 1, seen, key0);
    }
    ve = units.ve;
    if (more) {
      if constexpr (KV8) {
        place8(buf ^ 1);
        ks = ks_next;
      } else {
        __builtin_amdgcn_s_waitcnt(0x0F70);          // vmcnt(0): the next tiles have landed
      }
    }
    lds_barrier();
  }
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
    kv_store<BF16, D>(a, s[qb], kv_half_sum(s[qb].l), ve, b, hk, row[qb], split, h,
                      row[qb] < nrows && row[qb] / a.G < rg.nq);
}

// ------------------------------------------------------------------ step form
template <bool KV8, bool BF16, int D>
struct KvStep {
  static constexpr int WAVES = 4;
  static constexpr int KB = KV8 ? 2 : D == 64 ? 2 : 1;          // 32-key blocks of a tile
  static constexpr int KT = 32 * KB;
  static constexpr int TILE = KT * D * 2;
  static constexpr int LDS = KV8 ? WAVES * 32 * D * 4 : WAVES * 4 * TILE;   // the join's rows / 2 stages of K and V
};
template <bool KV8, bool BF16, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(KV8 ? 2 : 1, KV8 ? 2 : 1))) void kv_attn_step_kernel(const KvAttn a) {
  using C = KvStep<KV8, BF16, D>;
  constexpr bool MBF = BF16 && !KV8;
  constexpr int KS = D / 16, NV = D / 32, KB = C::KB, KT = C::KT, TILE = C::TILE;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[C::LDS];
  __shared__ float2 stat[C::WAVES][32];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, l32 = lane & 31;
  const int split = blockIdx.x % a.splits;
  const int hk = blockIdx.x / a.splits % a.Hk;
  const int b = blockIdx.x / (a.splits * a.Hk);
  const int nrows = a.Lq * a.G;                      // <= 32
  const KvRange rg = kv_range(a, b, 0, nrows, split);
  if (rg.nq == 0) return;
  const int rc = l32 < nrows ? l32 : nrows - 1;
  const int qi = rc / a.G;
  KvRows<KV8, BF16, D> qr;
  qr.load(a.q + b * a.q_bs + qi * a.q_ts + (hk * a.G + rc % a.G) * a.q_hs, h, a.scale_log2);
  const int upto = a.causal ? rg.len - rg.nq + qi : rg.len - 1;
  const int first_upto = a.causal ? rg.len - rg.nq : rg.len - 1;
  KvState<D> s;
  s.init();
  KvUnits units;
  int ve = 0;
  if constexpr (KV8) {
    const long cache0 = ((long)b * a.Hk + hk) * a.blocks;
    constexpr int U = KV_BLOCK * D / 1024;           // 1 KB pieces of a block's keys or values
    uint4 kraw[U], vraw[U];
    float ks = 0.f, vs = 0.f;
    auto fetch = [&](int tile) __attribute__((always_inline)) {
      const uint4* kp = reinterpret_cast<const uint4*>(a.kc) + (cache0 + tile) * (KV_BLOCK * D / 16) + lane;
      const uint4* vp = reinterpret_cast<const uint4*>(a.vc) + (cache0 + tile) * (KV_BLOCK * D / 16) + lane;
#pragma unroll
      for (int u = 0; u < U; ++u) kraw[u] = kp[64 * u];
#pragma unroll
      for (int u = 0; u < U; ++u) vraw[u] = vp[64 * u];
      ks = a.ks[cache0 + tile];
      vs = a.vs[cache0 + tile];
    };
    int tile = rg.t0 + wave;
    if (tile < rg.t1) fetch(tile);
    for (; tile < rg.t1; tile += C::WAVES) {
      const int key0 = tile * KV_BLOCK;
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
      const float c = kv_factor((ks > 0.f || ks != ks ? ks : 1.0f) * qr.mul);
      const _Float16 f = (_Float16)units.fit(vs);
      uint4 vnow[U];
#pragma unroll
      for (int u = 0; u < U; ++u) vnow[u] = vraw[u];
      if (tile + C::WAVES < rg.t1) fetch(tile + C::WAVES);
      if (units.ve != ve) {
        s.scale(__builtin_ldexpf(1.0f, ve - units.ve));
        ve = units.ve;
      }
      if (seen != ~0ull || first_upto < key0 + KV_BLOCK - 1) 
        kv_mask<KB>(sc, seen & kv_below(upto - key0 + 1), h);
      kv_softmax<MBF, D, KB, false>(sc, c, s, pf, [](int) __attribute__((always_inline)) {});
#pragma unroll
      for (int db = 0; db < NV; ++db)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          kv_decode(vnow[db * 2 + w], (f16x2){f, f}, lo, hi);
          s.o[db] = kv_mfma<MBF>(lo, pf[2 * w], s.o[db]);
          s.o[db] = kv_mfma<MBF>(hi, pf[2 * w + 1], s.o[db]);
        }
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
      const auto rk = sk.rsrc(), rv = sv.rsrc();
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
    static_assert(2 * DMA == 16, "the wait below counts the copies of one stage");
    int buf = 0;
    uint8_t mask_byte = 1;
    if (tile < t1) issue(0);
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
        asm volatile("s_waitcnt vmcnt(16)" ::: "memory");      // this stage's copies have landed
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
  const float by = sum == 0.f ? 0.f : __builtin_ldexpf(__builtin_amdgcn_exp2f(s.m - ref) / sum, ve);
  float* join = reinterpret_cast<float*>(lds);       // [wave][row][D]
  if (l32 < nrows)
#pragma unroll
    for (int db = 0; db < NV; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(join + (wave * 32 + l32) * D + 32 * db + 8 * g + 4 * h) =
            make_float4(s.o[db][4 * g] * by, s.o[db][4 * g + 1] * by, s.o[db][4 * g + 2] * by, s.o[db][4 * g + 3] * by);
  __syncthreads();
  const int rows_out = nrows < rg.nq * a.G ? nrows : rg.nq * a.G;
  for (int i = tid; i < rows_out * (D / 4); i += 256) {
    const int row = i / (D / 4), d = 4 * (i % (D / 4));
    float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < C::WAVES; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(join + (w * 32 + row) * D + d);
      o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
    }
    if (a.splits == 1) {
      uint16_t* op = a.out + b * a.o_bs + (row / a.G) * a.o_ts + (hk * a.G + row % a.G) * a.o_hs + d;
      *reinterpret_cast<uint2*>(op) = make_uint2(pack2<BF16>(o.x, o.y), pack2<BF16>(o.z, o.w));
    } else {
      const long rows = (long)a.B * a.H * a.Lq;
      *reinterpret_cast<float4*>(a.part + ((long)split * rows + ((long)b * a.Hk + hk) * nrows + row) * D + d) = o;
    }
  }
  if (a.splits > 1 && wave == 0 && h == 0 && l32 < rows_out) {
    const long rows = (long)a.B * a.H * a.Lq;
    a.stat[(long)split * rows + ((long)b * a.Hk + hk) * nrows + l32] = make_float2(m, sum);
  }
}

// ------------------------------------------------------------------ join of the splits
// A thread takes 4 dims of one row: sum of the splits' quotients, weighted by l 2^m.
template <bool BF16, int D>
__global__ __launch_bounds__(256) void kv_attn_join_kernel(const KvAttn a) {
  const long rows = (long)a.B * a.H * a.Lq;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long at = i / (D / 4);
  if (at >= rows) return;
  const int d = 4 * (int)(i % (D / 4));
  const int per = a.Lq * a.G;
  const int row = (int)(at % per), hk = (int)(at / per % a.Hk), b = (int)(at / per / a.Hk);
  const int qi = row / a.G;
  if (a.counts && qi >= a.counts[b]) return;
  float m = -INFINITY;
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.stat[s * rows + at].x);
  const float ref = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
  float4 o = make_float4(0, 0, 0, 0);
  for (int s = 0; s < a.splits; ++s) {
    const float2 st = a.stat[s * rows + at];
    const float w = st.y * __builtin_amdgcn_exp2f(st.x - ref);
    if (w != 0.f) {                                  // NaN counts
      const float4 x = *reinterpret_cast<const float4*>(a.part + (s * rows + at) * D + d);
      sum += w;
      o.x += w * x.x, o.y += w * x.y, o.z += w * x.z, o.w += w * x.w;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  uint16_t* op = a.out + b * a.o_bs + qi * a.o_ts + (hk * a.G + row % a.G) * a.o_hs + d;
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
  int64_t wg, slots, least;
  if (rows <= 32) {
    p.step = true, p.qb = 1, p.row_tiles = 1;
    wg = heads, slots = kv8 ? 512 : 256, least = 8;         // tiles of a split at least: two a wave
  } else {
    p.qb = D == 64 && rows > 128 ? 2 : 1;
    p.row_tiles = (int)((rows + 128 * p.qb - 1) / (128 * p.qb));
    wg = heads * p.row_tiles, slots = 512, least = 8;
  }
  int64_t s = wg < slots ? slots / (wg > 0 ? wg : 1) : 1;
  if (s > tiles / least) s = tiles / least;
  if (s > 64) s = 64;
  p.splits = (int)(s < 1 ? 1 : s);
  return p;
}

static size_t kv_split_bytes(int64_t B, int64_t Lq, int64_t H, int64_t D) { return (size_t)(B * Lq * H) * (D * 4 + 8); }

template <bool KV8, bool BF16, int D>
static void kv_launch(const KvAttn& a, const KvPlan& p, hipStream_t st) {
  const unsigned wg = (unsigned)(a.B * a.Hk * p.row_tiles * p.splits);
  if (p.step) {
    hipLaunchKernelGGL((kv_attn_step_kernel<KV8, BF16, D>), dim3(wg), dim3(256), 0, st, a);
  } else if constexpr (D == 64) {
    if (p.qb == 2) hipLaunchKernelGGL((kv_attn_wide_kernel<KV8, BF16, D, 2>), dim3(wg), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv_attn_wide_kernel<KV8, BF16, D, 1>), dim3(wg), dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((kv_attn_wide_kernel<KV8, BF16, D, 1>), dim3(wg), dim3(256), 0, st, a);
  }
  if (p.splits > 1) {
    const long threads = (long)a.B * a.H * a.Lq * (D / 4);
    hipLaunchKernelGGL((kv_attn_join_kernel<BF16, D>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, a);
  }
}

// Checks and fields that both entries share.
static int kv_common(KvAttn& a, const char* what, const void* q, void* out, int dtype, int64_t B, int64_t Lq, int64_t Lk,
                     int64_t H, int64_t Hk, int64_t D, const int64_t* qs, const int64_t* os, float scale) {
  QV_CHECK_ARG(dtype == QV_F16 || dtype == QV_BF16, "bad dtype %d", dtype);
  QV_CHECK_ARG(D == 64 || D == 128, "head_dim must be 64 or 128 (got %lld)", (long long)D);
  QV_CHECK_ARG(B >= 0 && Lq >= 0 && Lk >= 0 && H > 0 && Hk > 0 && H % Hk == 0 && B <= (1 << 20) && Lq <= (1 << 28) &&
                   Lk <= (1 << 30) && H <= 65536,
               "bad shape B=%lld Lq=%lld Lk=%lld heads=%lld / %lld", (long long)B, (long long)Lq, (long long)Lk,
               (long long)H, (long long)Hk);
  QV_CHECK_ARG(scale > 0.f && scale < INFINITY, "the scale must be a positive number");
  QV_CHECK_ARG(Lq * (H / Hk) <= INT32_MAX / 2 && B * H * Lq <= (1ll << 36), "too many rows");
  if (B == 0 || Lq == 0) return QV_OK;
  QV_CHECK_ARG(q && out && qs && os, "null pointer argument");
  QV_CHECK_ARG((uintptr_t)q % 16 == 0 && (uintptr_t)out % 8 == 0, "q must be 16-byte and out 8-byte aligned");
  for (int i = 0; i < 3; ++i)
    QV_CHECK_ARG(qs[i] % 8 == 0 && os[i] % 4 == 0, "q strides must be multiples of 8 elements, out strides of 4");
  a.q = (const uint16_t*)q, a.out = (uint16_t*)out;
  a.B = (int)B, a.Lq = (int)Lq, a.Lk = (int)Lk, a.H = (int)H, a.Hk = (int)Hk, a.G = (int)(H / Hk);
  a.q_bs = qs[0], a.q_ts = qs[1], a.q_hs = qs[2];
  a.o_bs = os[0], a.o_ts = os[1], a.o_hs = os[2];
  a.scale_log2 = scale * 1.4426950408889634f;
  return QV_OK;
}

// Splits that the workspace holds, and where their parts lie.
static int kv_place(KvAttn& a, KvPlan& p, int64_t D, void* ws, int64_t ws_bytes) {
  const size_t per = kv_split_bytes(a.B, a.Lq, a.H, D);
  if (p.splits > 1 && (!ws || (uintptr_t)ws % 16 || (size_t)ws_bytes / per < 2)) p.splits = 1;
  if (p.splits > 1 && (size_t)ws_bytes / per < (size_t)p.splits) p.splits = (int)((size_t)ws_bytes / per);
  a.splits = p.splits, a.row_tiles = p.row_tiles;
  QV_CHECK_ARG((int64_t)a.B * a.Hk * p.row_tiles * p.splits <= INT32_MAX &&
                   (int64_t)a.B * a.H * a.Lq * (D / 4) / 256 < INT32_MAX,
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
  return p.splits > 1 ? (int64_t)(p.splits * qv::kv_split_bytes(B, Lq, H, D)) : 0;
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
  if (int rc = qv::kv_common(a, "attention_cross", q, out, dtype, B, Lq, Lk, H, Hk, D, q_strides, out_strides, scale))
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
  if (int rc = qv::kv_place(a, p, D, workspace, workspace_bytes)) return rc;
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
  if (int rc = qv::kv_common(a, "kv8_attention", q, out, dtype, B, Lq, blocks * qv::KV_BLOCK, H, Hk, D, q_strides,
                             out_strides, scale))
    return rc;
  if (B == 0 || Lq == 0) return QV_OK;
  QV_CHECK_ARG(k_codes && v_codes && k_scales && v_scales && lens, "null pointer argument");
  QV_CHECK_ARG((uintptr_t)k_codes % 16 == 0 && (uintptr_t)v_codes % 16 == 0, "codes must be 16-byte aligned");
  a.kc = (const uint8_t*)k_codes, a.vc = (const uint8_t*)v_codes, a.ks = k_scales, a.vs = v_scales;
  a.lens = lens, a.counts = counts, a.causal = causal != 0, a.blocks = (int)blocks;
  if (keys < 0 || keys > blocks * qv::KV_BLOCK) keys = blocks * qv::KV_BLOCK;
  qv::KvPlan p = qv::kv_plan(true, B, Lq, H, Hk, D, keys);
  if (int rc = qv::kv_place(a, p, D, workspace, workspace_bytes)) return rc;
  QV_KV_LAUNCH(true)
  return qv::check_launch("kv8_attention");
}
