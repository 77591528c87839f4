// Rotary positions of several axes (time, height, width, ...) for gfx950.
//
// A head of D dims is cut into pairs (lo, hi); pair j turns by the angle
// pos[axis_j] * theta_j: lo' = lo cos - hi sin, hi' = hi cos + lo sin.  The
// pairs come in chunks of one axis with a fixed distance hi - lo; dims behind
// the rotated ones form a last chunk that is copied.
//
// The angle is a product of an integer position and a frequency that is kept
// in turns (theta / 2 pi) in 64 bits: t = pos * turns, t - rint(t) is exact, and
// only the fraction goes to 32 bits.  A 32-bit product would lose pos * 2^-24 of
// an angle in radians (position 100000: 6e-3); the 64-bit one loses 2^-52 of a
// turn for each unit of t.
//
// A workgroup takes a few tokens with all their heads: its threads load their
// pieces of x (V dims at lo, V at hi; 16 bytes each where sections and strides
// allow it), compute one sine and cosine per (token, pair) into LDS while those
// loads are in flight, and apply them to every head.  Bound by the bytes of x,
// read once and written once.  16 tokens of 24 heads of 128 dims: 3.5 us, the launch and
// two dependent reads; 1374 of 32 heads of 64: 5.3 us, 2.1 TB/s; 43968 of them: 65 us, 5.6 TB/s.
#include "common.h"

namespace qv {

struct RopeAxes {
  int chunks;
  int pair0[6];   // first pair of the chunk (the entry behind the last: D / 2)
  int lo0[5];     // first lo dim
  int gap[5];     // hi - lo
  int axis[5];    // column of the positions; -1: copied
};

constexpr int ROPE_TABLE = 512;   // (token, pair) entries of a workgroup
constexpr int ROPE_UNITS = 4;     // pieces of x that a thread has in flight

template <int DT, int V>
struct RopePiece {
  static constexpr int ES = DT == QV_F32 ? 4 : 2;
  static constexpr int BYTES = V * ES;
  static constexpr int WORDS = BYTES >= 4 ? BYTES / 4 : 1;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (BYTES == 2) {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    } else {
      constexpr int N = BYTES >= 16 ? 4 : BYTES / 4;
      typedef uint32_t vec __attribute__((ext_vector_type(N)));
#pragma unroll
      for (int i = 0; i < WORDS / N; ++i) {
        const vec u = reinterpret_cast<const vec*>(p)[i];
#pragma unroll
        for (int j = 0; j < N; ++j) w[N * i + j] = u[j];
      }
    }
  }
  __device__ __forceinline__ void store(uint8_t* p) const {
    if constexpr (BYTES == 2) {
      *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
    } else {
      constexpr int N = BYTES >= 16 ? 4 : BYTES / 4;
      typedef uint32_t vec __attribute__((ext_vector_type(N)));
#pragma unroll
      for (int i = 0; i < WORDS / N; ++i) {
        vec u;
#pragma unroll
        for (int j = 0; j < N; ++j) u[j] = w[N * i + j];
        reinterpret_cast<vec*>(p)[i] = u;
      }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (DT == QV_F32) return __builtin_bit_cast(float, w[i]);
    else return to_f32((uint16_t)(w[i >> 1] >> (16 * (i & 1))), DT == QV_BF16);
  }
  __device__ __forceinline__ void set(int i, float v) {
    if constexpr (DT == QV_F32) {
      w[i] = __builtin_bit_cast(uint32_t, v);
    } else {
      const uint32_t b = from_f32<DT == QV_BF16>(v);
      if (i & 1) w[i >> 1] |= b << 16;
      else w[i >> 1] = b;
    }
  }
};

// token tile TB: TB * pairs table entries (at most ROPE_TABLE) and TB * H * groups
// pieces of x, taken ROPE_UNITS a thread at a time.  per_tok_mul, groups_mul:
// floor(2^32 / n) + 1 for the pieces of a token and of a head (0 for n = 1: the
// dividend itself), which divide exactly while the dividend times n is below 2^32;
// a workgroup of one token, whose pieces may pass that, does not divide by them.
template <int DT, int V>
__global__ __launch_bounds__(256) void rope_axes_kernel(
    const uint8_t* x, uint8_t* out, const int32_t* __restrict__ pos, int axes, const double* __restrict__ turns, RopeAxes ra,
    long T, int H, int pairs, int TB, uint32_t per_tok_mul, uint32_t groups_mul, long x_ts, long x_hs, long o_ts,
    long o_hs) {   // x and out may be the same
  __shared__ float2 table[ROPE_TABLE];
  const int tid = threadIdx.x;
  const long tok0 = (long)blockIdx.x * TB;
  const int ntok = (int)(T - tok0 < TB ? T - tok0 : TB);
  const int groups = pairs / V, per_tok = H * groups, units = ntok * per_tok;
  constexpr int ES = RopePiece<DT, V>::ES;
  x += tok0 * x_ts * ES;
  out += tok0 * o_ts * ES;

  RopePiece<DT, V> lo[ROPE_UNITS], hi[ROPE_UNITS];
  int entry[ROPE_UNITS];                             // of the table; -1: copied
  int gap[ROPE_UNITS];                               // bytes from lo to hi
  long to[ROPE_UNITS];                               // byte offset in out
  // pieces base .. base + 1023: where they lie (token, head, pairs), and their loads
  auto fetch = [&](int base) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < ROPE_UNITS; ++i) {
      const int u = base + 256 * i + tid;
      if (u < units) {
        const int tok = TB == 1 ? 0 : per_tok_mul ? (int)__umulhi((uint32_t)u, per_tok_mul) : u;
        const int rest = u - tok * per_tok;
        const int head = groups_mul ? (int)__umulhi((uint32_t)rest, groups_mul) : rest;
        const int pair = (rest - head * groups) * V;
        int dim = ra.lo0[0] + pair, ax = ra.axis[0], g = ra.gap[0];
#pragma unroll
        for (int c = 1; c < 5; ++c)
          if (c < ra.chunks && pair >= ra.pair0[c]) dim = ra.lo0[c] + pair - ra.pair0[c], g = ra.gap[c], ax = ra.axis[c];
        entry[i] = ax < 0 ? -1 : tok * pairs + pair;
        gap[i] = g * ES;
        to[i] = (tok * o_ts + head * o_hs + dim) * ES;
        const uint8_t* from = x + (tok * x_ts + head * x_hs + dim) * ES;
        lo[i].load(from);
        hi[i].load(from + gap[i]);
      }
    }
  };
  fetch(0);
  for (int e = tid; e < ntok * pairs; e += 256) {
    const int tok = e / pairs, pair = e - tok * pairs;
    int ax = ra.axis[0];
#pragma unroll
    for (int c = 1; c < 5; ++c)
      if (c < ra.chunks && pair >= ra.pair0[c]) ax = ra.axis[c];
    float s = 0.f, c = 1.f;
    if (ax >= 0) {
      const double t = (double)pos[(tok0 + tok) * axes + ax] * turns[pair];
      sincospif(2.0f * (float)(t - rint(t)), &s, &c);
    }
    table[e] = make_float2(c, s);
  }
  __syncthreads();
  for (int base = 0; base < units; base += 256 * ROPE_UNITS) {
    if (base) fetch(base);
#pragma unroll
    for (int i = 0; i < ROPE_UNITS; ++i) {
      if (base + 256 * i + tid < units) {
        RopePiece<DT, V> a = lo[i], b = hi[i];
        if (entry[i] >= 0) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float2 cs = table[entry[i] + e];
            const float l = lo[i].get(e), h = hi[i].get(e);
            a.set(e, __builtin_fmaf(l, cs.x, -(h * cs.y)));
            b.set(e, __builtin_fmaf(h, cs.x, l * cs.y));
          }
        }
        a.store(out + to[i]);
        b.store(out + to[i] + gap[i]);
      }
    }
  }
}

// The same for large tensors of 8 and more heads of 64 to 512 dims (a power of two) with chunks
// in multiples of 4 (the rule with both sides stands at the entry): a
// lane takes 8 consecutive dims, so that rows are read and written whole, and reads the
// partners of each 4 of them a second time (from the L1).  A row lies within one wave,
// whose loads all come before its stores: x and out may be the same.  43968 tokens of 32
// heads of 64 fp16 dims (16 + 24 + 24 by axis): 65 us, 5.6 TB/s.
template <int DT>
__global__ __launch_bounds__(256) void rope_axes_rows_kernel(
    const uint8_t* x, uint8_t* out, const int32_t* __restrict__ pos, int axes, const double* __restrict__ turns, RopeAxes ra,
    long T, int H, int pairs, int TB, uint32_t h_mul, long x_ts, long x_hs, long o_ts, long o_hs) {
  __shared__ __attribute__((aligned(16))) float2 table[ROPE_TABLE];
  constexpr int ES = RopePiece<DT, 4>::ES;
  const int tid = threadIdx.x;
  const long tok0 = (long)blockIdx.x * TB;
  const int ntok = (int)(T - tok0 < TB ? T - tok0 : TB);
  const int lanes = pairs / 4;                       // of a row
  const int rows = ntok * H, step = 256 / lanes;
  const int dim0 = tid % lanes * 8;
  // this lane's two 4-dim pieces: their first pair (-1: copied), partner and sign
  int entry[2], part[2];
  float sign[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int d = dim0 + 4 * k;
    entry[k] = -1, part[k] = d, sign[k] = 0.f;
#pragma unroll
    for (int c = 0; c < 5; ++c)
      if (c < ra.chunks && ra.axis[c] >= 0) {
        const int len = ra.pair0[c + 1] - ra.pair0[c], lo = d - ra.lo0[c], hi = lo - ra.gap[c];
        if (lo >= 0 && lo < len) entry[k] = ra.pair0[c] + lo, part[k] = d + ra.gap[c], sign[k] = -1.f;
        if (hi >= 0 && hi < len) entry[k] = ra.pair0[c] + hi, part[k] = d - ra.gap[c], sign[k] = 1.f;
      }
  }
  x += tok0 * x_ts * ES;
  out += tok0 * o_ts * ES;
  RopePiece<DT, 8> own[ROPE_UNITS];
  RopePiece<DT, 4> other[ROPE_UNITS][2];
  auto fetch = [&](int base) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < ROPE_UNITS; ++i) {
      const int row = base + step * i + tid / lanes;
      if (row < rows) {
        const int tok = h_mul ? (int)__umulhi((uint32_t)row, h_mul) : row;
        const uint8_t* from = x + (tok * x_ts + (row - tok * H) * x_hs) * ES;
        own[i].load(from + dim0 * ES);
        other[i][0].load(from + part[0] * ES);
        other[i][1].load(from + part[1] * ES);
      }
    }
  };
  fetch(0);
  for (int e = tid; e < ntok * pairs; e += 256) {
    const int tok = e / pairs, pair = e - tok * pairs;
    int ax = ra.axis[0];
#pragma unroll
    for (int c = 1; c < 5; ++c)
      if (c < ra.chunks && pair >= ra.pair0[c]) ax = ra.axis[c];
    float s = 0.f, c = 1.f;
    if (ax >= 0) {
      const double t = (double)pos[(tok0 + tok) * axes + ax] * turns[pair];
      sincospif(2.0f * (float)(t - rint(t)), &s, &c);
    }
    table[e] = make_float2(c, s);
  }
  __syncthreads();
  for (int base = 0; base < rows; base += step * ROPE_UNITS) {
    if (base) fetch(base);
#pragma unroll
    for (int i = 0; i < ROPE_UNITS; ++i) {
      const int row = base + step * i + tid / lanes;
      if (row < rows) {
        const int tok = h_mul ? (int)__umulhi((uint32_t)row, h_mul) : row;
        RopePiece<DT, 8> r = own[i];
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (entry[k] >= 0) {
            const float2* t = table + tok * pairs + entry[k];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 cs = t[e];
              r.set(4 * k + e, __builtin_fmaf(own[i].get(4 * k + e), cs.x, sign[k] * (other[i][k].get(e) * cs.y)));
            }
          }
        r.store(out + (tok * o_ts + (row - tok * H) * o_hs + dim0) * ES);
      }
    }
  }
}

// The same for 16-bit types and sections that leave pieces of 1 or 2 dims: rows are read and
// written whole as above, and turned in LDS in between, a pair to a lane, the pairs of a row
// next to each other (no bank meets twice).  Each wave works on rows of its own, and all
// its loads of a round come before its stores: x and out may be the same.  43968 tokens
// of 32 heads of 64 fp16 dims, 10 + 26 + 28 by axis: 72 us, 5.0 TB/s.
template <int DT>
__global__ __launch_bounds__(256) void rope_axes_staged_kernel(
    const uint8_t* x, uint8_t* out, const int32_t* __restrict__ pos, int axes, const double* __restrict__ turns, RopeAxes ra,
    long T, int H, int pairs, int TB, uint32_t h_mul, long x_ts, long x_hs, long o_ts, long o_hs) {
  typedef RopePiece<DT, 8> Piece;
  constexpr int ES = Piece::ES, K = 4;               // pairs of a lane in each 512 dims of a wave
  __shared__ float2 table[ROPE_TABLE];
  __shared__ __attribute__((aligned(16))) uint8_t stage[4 * ROPE_UNITS * 512 * ES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long tok0 = (long)blockIdx.x * TB;
  const int ntok = (int)(T - tok0 < TB ? T - tok0 : TB);
  const int lanes = pairs / 4, per_wave = 64 / lanes;                // of a row; rows of 512 dims
  const int rows = ntok * H, step = 4 * per_wave;
  const int mine = wave * per_wave, dim0 = lane % lanes * 8;
  uint8_t* own_stage = stage + wave * (ROPE_UNITS * 512 * ES);
  x += tok0 * x_ts * ES;
  out += tok0 * o_ts * ES;
  Piece own[ROPE_UNITS];
  auto fetch = [&](int base) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < ROPE_UNITS; ++i) {
      const int row = base + step * i + mine + lane / lanes;
      if (row < rows) {
        const int tok = h_mul ? (int)__umulhi((uint32_t)row, h_mul) : row;
        own[i].load(x + (tok * x_ts + (row - tok * H) * x_hs + dim0) * ES);
      }
    }
  };
  fetch(0);
  // pair k of the lane: row and pair in the 512 dims, its dims (-1: copied)
  int at[K], pair[K], lo[K], hi[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int q = 64 * k + lane;
    at[k] = q / pairs, pair[k] = q % pairs;
    int dim = ra.lo0[0] + pair[k], g = ra.gap[0], ax = ra.axis[0];
#pragma unroll
    for (int c = 1; c < 5; ++c)
      if (c < ra.chunks && pair[k] >= ra.pair0[c]) dim = ra.lo0[c] + pair[k] - ra.pair0[c], g = ra.gap[c], ax = ra.axis[c];
    lo[k] = ax < 0 ? -1 : (at[k] * 2 * pairs + dim) * ES;
    hi[k] = lo[k] + g * ES;
  }
  for (int e = tid; e < ntok * pairs; e += 256) {
    const int tok = e / pairs, p = e - tok * pairs;
    int ax = ra.axis[0];
#pragma unroll
    for (int c = 1; c < 5; ++c)
      if (c < ra.chunks && p >= ra.pair0[c]) ax = ra.axis[c];
    float s = 0.f, c = 1.f;
    if (ax >= 0) {
      const double t = (double)pos[(tok0 + tok) * axes + ax] * turns[p];
      sincospif(2.0f * (float)(t - rint(t)), &s, &c);
    }
    table[e] = make_float2(c, s);
  }
  __syncthreads();
  for (int base = 0; base < rows; base += step * ROPE_UNITS) {
    if (base) fetch(base);
#pragma unroll
    for (int i = 0; i < ROPE_UNITS; ++i) own[i].store(own_stage + (i * 512 + lane * 8) * ES);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // the wave's other lanes read it
#pragma unroll
    for (int i = 0; i < ROPE_UNITS; ++i) {
      uint8_t* dims = own_stage + i * 512 * ES;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int row = base + step * i + mine + at[k];
        if (row < rows && lo[k] >= 0) {
          const int tok = h_mul ? (int)__umulhi((uint32_t)row, h_mul) : row;
          const float2 cs = table[tok * pairs + pair[k]];
          RopePiece<DT, 1> a, b;
          a.load(dims + lo[k]);
          b.load(dims + hi[k]);
          const float l = a.get(0), h = b.get(0);
          a.set(0, __builtin_fmaf(l, cs.x, -(h * cs.y)));
          b.set(0, __builtin_fmaf(h, cs.x, l * cs.y));
          a.store(dims + lo[k]);
          b.store(dims + hi[k]);
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < ROPE_UNITS; ++i) {
      const int row = base + step * i + mine + lane / lanes;
      if (row < rows) {
        const int tok = h_mul ? (int)__umulhi((uint32_t)row, h_mul) : row;
        own[i].load(own_stage + (i * 512 + lane * 8) * ES);
        own[i].store(out + (tok * o_ts + (row - tok * H) * o_hs + dim0) * ES);
      }
    }
  }
}

template <int DT>
static void rope_axes_launch(int vec, unsigned grid, hipStream_t st, const void* x, void* out, const int32_t* pos, int axes,
                             const double* turns, const RopeAxes& ra, long T, int H, int pairs, int TB,
                             uint32_t per_tok_mul, uint32_t mul, long x_ts, long x_hs, long o_ts, long o_hs) {
#define QV_ROPE(V)                                                                                                   \
  hipLaunchKernelGGL((rope_axes_kernel<DT, V>), dim3(grid), dim3(256), 0, st, (const uint8_t*)x, (uint8_t*)out, pos, \
                     axes, turns, ra, T, H, pairs, TB, per_tok_mul, mul, x_ts, x_hs, o_ts, o_hs)
  if (vec == 0)
    hipLaunchKernelGGL((rope_axes_rows_kernel<DT>), dim3(grid), dim3(256), 0, st, (const uint8_t*)x, (uint8_t*)out, pos, axes,
                       turns, ra, T, H, pairs, TB, mul, x_ts, x_hs, o_ts, o_hs);
  else if (vec == 16) {
    if constexpr (DT != QV_F32)
      hipLaunchKernelGGL((rope_axes_staged_kernel<DT>), dim3(grid), dim3(256), 0, st, (const uint8_t*)x, (uint8_t*)out, pos,
                         axes, turns, ra, T, H, pairs, TB, mul, x_ts, x_hs, o_ts, o_hs);
  }
  else if (vec == 8) QV_ROPE(8);
  else if (vec == 4) QV_ROPE(4);
  else if (vec == 2) QV_ROPE(2);
  else QV_ROPE(1);
#undef QV_ROPE
}

}  // namespace qv

extern "C" int qv_rope_axes(const void* x, void* out, int dtype, const int32_t* positions, const double* turns,
                            const int64_t* sections, int64_t axes, int layout, int64_t T, int64_t H, int64_t D,
                            int64_t x_token_stride, int64_t x_head_stride, int64_t out_token_stride,
                            int64_t out_head_stride, void* stream) {
  QV_CHECK_ARG(dtype == QV_F16 || dtype == QV_BF16 || dtype == QV_F32, "bad dtype %d", dtype);
  QV_CHECK_ARG(axes >= 1 && axes <= 4, "1 to 4 axes are supported (got %lld)", (long long)axes);
  QV_CHECK_ARG(layout == QV_ROPE_BLOCK || layout == QV_ROPE_HALF, "bad layout %d", layout);
  QV_CHECK_ARG(T >= 0 && H > 0 && D > 0 && D % 2 == 0 && D <= 1024 && H <= 4096, "bad shape T=%lld H=%lld D=%lld",
               (long long)T, (long long)H, (long long)D);
  QV_CHECK_ARG(sections, "null sections");
  qv::RopeAxes ra = {};
  int64_t rot = 0;
  for (int a = 0; a < axes; ++a) {
    QV_CHECK_ARG(sections[a] > 0 && sections[a] % 2 == 0 && sections[a] <= D,
                 "section %d must be a positive even number of dims (got %lld)", a, (long long)sections[a]);
    rot += sections[a];
  }
  QV_CHECK_ARG(rot <= D, "sections hold %lld dims of %lld", (long long)rot, (long long)D);
  if (T == 0) return QV_OK;
  QV_CHECK_ARG(x && out && positions && turns, "null pointer argument");
  int64_t at = 0;
  for (int a = 0; a < axes; ++a) {
    ra.pair0[a] = (int)(at / 2);
    ra.lo0[a] = (int)(layout == QV_ROPE_BLOCK ? at : at / 2);
    ra.gap[a] = (int)(layout == QV_ROPE_BLOCK ? sections[a] / 2 : rot / 2);
    ra.axis[a] = a;
    at += sections[a];
  }
  ra.chunks = (int)axes;
  if (rot < D) {
    ra.pair0[axes] = (int)(rot / 2);
    ra.lo0[axes] = (int)rot;
    ra.gap[axes] = (int)(D - rot) / 2;
    ra.axis[axes] = -1;
    ra.chunks = (int)axes + 1;
  }
  ra.pair0[ra.chunks] = (int)(D / 2);
  // the widest piece that starts on its own multiple everywhere: inside the
  // chunks, and at every head and token of x and out
  const int es = dtype == QV_F32 ? 4 : 2;
  int vec = 8;
  auto fits = [&](int64_t v) { return v % vec == 0; };
  for (;; vec /= 2) {
    const int align = vec * es < 16 ? vec * es : 16;
    bool ok = fits(x_token_stride) && fits(x_head_stride) && fits(out_token_stride) && fits(out_head_stride) &&
              fits(D / 2) && (uintptr_t)x % align == 0 && (uintptr_t)out % align == 0;
    for (int c = 0; c < ra.chunks; ++c) ok = ok && fits(ra.pair0[c]) && fits(ra.lo0[c]) && fits(ra.gap[c]);
    if (ok || vec == 1) break;
  }
  QV_CHECK_ARG((uintptr_t)x % es == 0 && (uintptr_t)out % es == 0, "x and out must be aligned to their type");
  const int pairs = (int)(D / 2);
  // whole rows: 8 dims a lane, rows within a wave; from where bytes count, and for 8 heads and
  // more, as fewer leave a workgroup bound by its sines (one head of 64 fp16 dims, 200 MB: pieces
  // of 4 dims 78 us, rows 112; of 1 dim 104, staged 156; 4 heads 37 and 41; 65 and 50).  In us, by
  // bytes read and written:
  //  * 16-bit pieces of 4 dims, 32 heads: 360 MB 71 and 68, 80 MB 16.9 and 16.0, 6 MB 5.5 and 6.4;
  //  * pieces of 8 dims are whole 16 bytes as they are: 360 MB 71.5 and 67.3 (fp32 80 and 74), but
  //    80 MB 13.7 and 15.4 (fp32 15.1 and 16.6); fp32 pieces of 4: 360 MB 71 and 74;
  //  * 16-bit pieces of 1 or 2 dims, staged in LDS: 128 MB 40 and 28 against 26, 60 MB 22 and 16.6
  //    against 16, 16 MB 8.7 and 6.7 against 7.5, 4 MB 4.8 and 4.1 against 5.5 (the 64 MB of the
  //    rows are late for pieces of 1).  32-bit types gain nothing by the stage (360 MB: 146, in
  //    pieces of 1 152, of 2 142).
  const int wide = 8 * es < 16 ? 8 * es : 16;
  const int64_t bytes = 2 * T * H * D * es;
  const bool whole = bytes > (64 << 20) && H >= 8 && D >= 64 && D <= 512 && (D & (D - 1)) == 0 &&
                     x_token_stride % 8 == 0 && x_head_stride % 8 == 0 && out_token_stride % 8 == 0 &&
                     out_head_stride % 8 == 0 && (uintptr_t)x % wide == 0 && (uintptr_t)out % wide == 0;
  const bool rows = whole && (vec == 8 ? bytes > (256 << 20) : vec == 4 && es == 2);
  const bool staged = whole && vec < 4 && es == 2;
  const int64_t per_tok = rows || staged ? H * (D / 8) : H * (pairs / vec);
  // tokens of a workgroup: one round of pieces (1024), at most the table, and
  // enough workgroups to fill the chip
  int64_t tb = 256 * qv::ROPE_UNITS / per_tok;
  if (tb > qv::ROPE_TABLE / pairs) tb = qv::ROPE_TABLE / pairs;
  if (tb > T / 1024) tb = T / 1024;
  if (tb < 1) tb = 1;
  const int64_t grid = (T + tb - 1) / tb;
  const auto mul = [](int64_t n) { return n == 1 ? 0u : (uint32_t)((1ull << 32) / n + 1); };
  const uint32_t per_tok_mul = mul(per_tok), second = rows || staged ? mul(H) : mul(pairs / vec);
  if (rows) vec = 0;
  if (staged) vec = 16;
  QV_CHECK_ARG(grid <= INT32_MAX && per_tok * tb <= INT32_MAX / 2, "too many tokens or heads");
#define QV_ARGS                                                                                                       \
  vec, (unsigned)grid, (hipStream_t)stream, x, out, positions, (int)axes, turns, ra, (long)T, (int)H, pairs, (int)tb, \
      per_tok_mul, second, (long)x_token_stride, (long)x_head_stride, (long)out_token_stride, (long)out_head_stride
  if (dtype == QV_F16) qv::rope_axes_launch<QV_F16>(QV_ARGS);
  else if (dtype == QV_BF16) qv::rope_axes_launch<QV_BF16>(QV_ARGS);
  else qv::rope_axes_launch<QV_F32>(QV_ARGS);
#undef QV_ARGS
  return qv::check_launch("rope_axes");
}
