// Writing and reading back the 8-bit key / value cache (layout: kv_cache.h).
//
// Append.  The scale of a block is the smallest number s of four significant bits
// with 127 s >= amax, amax over the tokens of the call that fall into the block; a
// block that held tokens before keeps the larger of its old scale and s, and where
// that grows, its old codes are rounded again to the new one.  code = rint(x / s),
// ties to even.  Four bits are enough: the step is at most 1/8 coarser than
// amax / 127 (1/16 on average), and code * s has at most 7 + 4 bits, an fp16 number,
// so the matrix products that read the cache see its values without a further
// rounding.  They also make the rounding decision exact in 32 bits: x has at most 11
// bits and the border (n + 1/2) s at most 12.
// A NaN or infinity makes the scale of its (block, head) NaN, and stays until the
// block is begun again: the cache does not hide it.
//
// Both move the new values once and the codes once (append), codes and values once (values).
// A prompt of up to 2900 tokens for each of 8 sequences, half full, 8 heads of 128 fp16 dims:
// append 25.5 us for 72 MB, 2.9 TB/s, as the loads, codes and stores of a block take turns
// behind three barriers; values to float32 30 us for 217 MB, the zeros behind the lengths
// among them.  One token for each of 32 sequences: append 6.3 us, launch and three dependent
// reads; 64 tokens of each as float32: 9.2 us, 21 MB.
#include "kv_cache.h"

namespace qv {

constexpr int KV_TICKET = QV_KV8_TICKETS;   // words from ticket to ticket

// The smallest number of four significant bits that is at least amax / 127, not
// below 2^-120 (so that its reciprocal and every border stay normal numbers); 0
// for 0.  c has the right exponent and its first three fraction bits cut off
// from the quotient; 127 c is exact.
__device__ __forceinline__ float kv_scale(float amax) {
  if (amax == 0.f) return 0.f;
  uint32_t c = __builtin_bit_cast(uint32_t, amax / 127.0f) & 0xFFF00000u;
  if (127.0f * __builtin_bit_cast(float, c) < amax) c += 0x00100000u;
  return c < 0x03800000u ? 0x1p-120f : __builtin_bit_cast(float, c);
}

// rint(x / s), |x| <= 127 s: n = floor of the quotient, at most one off, then the
// exact comparison with the border (n + 1/2) s, which also mends n.
__device__ __forceinline__ int kv_code(float x, float s, float inv) {
  const float a = __builtin_fabsf(x);
  const float n = __builtin_floorf(a * inv);
  const float border = (n + 0.5f) * s;
  int c = (int)n;
  c += a > border || (a == border && (c & 1)) ? 1 : 0;
  return x < 0.f ? -c : c;
}

// Where byte `off` of a block lies while it is put together or taken apart in LDS: 16
// bytes more after every 4 units and after every 32.  Rows of keys (units 32 apart) and
// of values (units 8 apart) would otherwise meet the same banks, 8 to 16 lanes at once.
__host__ __device__ __forceinline__ constexpr int kv_skew(int off) { return off + ((off >> 6) + (off >> 9)) * 16; }

// One workgroup per block that the call touches and key head: D * 2 threads for the
// keys, as many for the values; a thread takes 4 consecutive tokens of 8 dims, one
// dword of a value unit for each dim and 8 bytes of a key unit for each token.
// A whole or a new block, or one whose scale grows, is put together in LDS and
// written in one piece; otherwise only the new tokens' codes are.
template <int D, bool BF16>
__global__ __launch_bounds__(4 * D) void kv8_append_kernel(
    const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, uint8_t* __restrict__ k_codes,
    uint8_t* __restrict__ v_codes, float* __restrict__ k_scales, float* __restrict__ v_scales,
    const int32_t* start_in, int32_t* lens_out, uint32_t* tickets, const int32_t* counts, int n, int Hk,
    int blocks, long k_bs, long k_ts, long k_hs, long v_bs, long v_ts, long v_hs) {
  constexpr int BYTES = KV_BLOCK * D;      // of one block's keys or values
  constexpr int HALF = 2 * D;              // threads for each of the two
  constexpr int STAGE = kv_skew(BYTES);
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * STAGE];
  __shared__ uint32_t wave_max[4 * D / 64];
  const int tid = threadIdx.x;
  const bool val = tid >= HALF;            // wave-uniform
  const int t = val ? tid - HALF : tid;
  const int head = blockIdx.y, b = blockIdx.z;
  const int cap = blocks * KV_BLOCK;
  int start = start_in[b];
  start = start < 0 ? 0 : start > cap ? cap : start;
  int cnt = counts ? counts[b] : n;
  cnt = cnt < 0 ? 0 : cnt > n ? n : cnt;
  if (cnt > cap - start) cnt = cap - start;
  const int block = start / KV_BLOCK + blockIdx.x;
  const int base = block * KV_BLOCK;       // the block's first token
  if (cnt > 0 && base < start + cnt) {
    const int old = base < start ? start - base : 0;   // tokens that stay
    const int end = start + cnt - base < KV_BLOCK ? start + cnt - base : KV_BLOCK;
    const int g = t % (D / 8), tok = 4 * (t / (D / 8));
    uint4 raw[4];
    uint32_t mx = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      raw[r] = make_uint4(0, 0, 0, 0);
      if (tok + r >= old && tok + r < end) {
        const long at = (long)(base + tok + r - start);
        raw[r] = val ? *reinterpret_cast<const uint4*>(v + b * v_bs + at * v_ts + head * v_hs + 8 * g)
                     : *reinterpret_cast<const uint4*>(k + b * k_bs + at * k_ts + head * k_hs + 8 * g);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t w[4] = {raw[r].x, raw[r].y, raw[r].z, raw[r].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {        // magnitudes order like integers, NaN and inf last
        const uint32_t lo = w[i] & 0x7FFFu, hi = (w[i] >> 16) & 0x7FFFu;
        mx = mx > lo ? mx : lo;
        mx = mx > hi ? mx : hi;
      }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
      const uint32_t other = __shfl_xor(mx, o);
      mx = mx > other ? mx : other;
    }
    if (tid % 64 == 0) wave_max[tid / 64] = mx;
    __syncthreads();
    mx = 0;
#pragma unroll
    for (int i = 0; i < HALF / 64; ++i) {
      const uint32_t other = wave_max[(val ? HALF / 64 : 0) + i];
      mx = mx > other ? mx : other;
    }
    const long which = ((long)b * Hk + head) * blocks + block;
    uint8_t* codes = (val ? v_codes : k_codes) + which * BYTES;
    float* scale = (val ? v_scales : k_scales) + which;
    const float was = old ? *scale : 0.f;
    const bool bad = mx >= (BF16 ? 0x7F80u : 0x7C00u);
    float s = bad ? __builtin_nanf("") : kv_scale(to_f32((uint16_t)mx, BF16));
    if (!(s > was) && !bad) s = was;       // the old scale, where it is larger or NaN
    const bool grown = old && s > was;
    const bool whole = !old || grown;      // the same for all threads of a half
    const float inv = s > 0.f ? 1.0f / s : 0.f;
    uint8_t* stage = lds + (val ? STAGE : 0);
    if (whole && (grown || end < KV_BLOCK)) {
      // the old codes, rounded to the new scale, zero behind them
      for (int i = t; i < BYTES / 16; i += HALF) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (grown) {
          u = reinterpret_cast<const uint4*>(codes)[i];
          uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t r = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = (float)(int8_t)(w[j] >> (8 * e)) * was;      // 7 + 4 bits: exact
              r |= (uint32_t)(kv_code(x, s, inv) & 0xFF) << (8 * e);
            }
            w[j] = r;
          }
          u = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *reinterpret_cast<uint4*>(stage + kv_skew(16 * i)) = u;
      }
    }
    __syncthreads();                       // also: every thread has read the old scale
    if (t == 0) *scale = s;
    uint32_t c[4][2];                      // four tokens' codes of 8 dims
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t w[4] = {raw[r].x, raw[r].y, raw[r].z, raw[r].w};
      c[r][0] = c[r][1] = 0;
      if (s > 0.f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = to_f32((uint16_t)(w[e >> 1] >> (16 * (e & 1))), BF16);
          c[r][e >> 2] |= (uint32_t)(kv_code(x, s, inv) & 0xFF) << (8 * (e & 3));
        }
      }
    }
    auto at = [&](int off) __attribute__((always_inline)) { return whole ? stage + kv_skew(off) : codes + off; };
    if (!val) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (tok + r >= old && tok + r < end)
          *reinterpret_cast<uint2*>(at(kv_key_offset<D>(tok + r, 8 * g))) = make_uint2(c[r][0], c[r][1]);
    } else if (tok >= old && tok + 4 <= end) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {        // token 4i is on a dword
        uint32_t w = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) w |= ((c[r][e >> 2] >> (8 * (e & 3))) & 0xFF) << (8 * r);
        *reinterpret_cast<uint32_t*>(at(kv_value_offset<D>(tok, 8 * g + e))) = w;
      }
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (tok + r >= old && tok + r < end)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *at(kv_value_offset<D>(tok + r, 8 * g + e)) = (uint8_t)(c[r][e >> 2] >> (8 * (e & 3)));
    }
    __syncthreads();
    if (whole)
      for (int i = t; i < BYTES / 16; i += HALF)
        reinterpret_cast<uint4*>(codes)[i] = *reinterpret_cast<const uint4*>(stage + kv_skew(16 * i));
  }
  // The length is written when all workgroups of the sequence have read the start and the
  // count, if one of them is the same tensor: by the last one, found by tickets that wrap to
  // 0 by themselves (one for each head and one for the heads, on lines of their own: 376
  // increments of a sequence's one word took longer than the codes).
  const bool turn = start_in == lens_out || counts == lens_out;
  if (turn) __syncthreads();               // a workgroup without tokens has met no barrier so far
  if (tid == 0) {
    bool last = head == 0 && blockIdx.x == 0;
    if (turn) {
      uint32_t* mine = tickets + (size_t)b * (Hk + 1) * KV_TICKET;
      last = gridDim.x == 1 || atomicInc(mine + (head + 1) * KV_TICKET, gridDim.x - 1) == gridDim.x - 1;
      if (last) last = atomicInc(mine, (uint32_t)Hk - 1) == (uint32_t)Hk - 1;
    }
    if (last) lens_out[b] = start + cnt;
  }
}

// values: tokens first[b] .. first[b] + n - 1 (zero where nothing is cached) of the
// keys (z even) or values of one block, head and sequence, in rows of D elements.
template <int D, int DT>
__global__ __launch_bounds__(256) void kv8_values_kernel(
    const uint8_t* __restrict__ k_codes, const uint8_t* __restrict__ v_codes, const float* __restrict__ k_scales,
    const float* __restrict__ v_scales, const int32_t* __restrict__ lens, const int32_t* __restrict__ first_in, int n,
    int Hk, int blocks, uint8_t* __restrict__ k_out, uint8_t* __restrict__ v_out) {
  constexpr int BYTES = KV_BLOCK * D;
  constexpr int ES = DT == QV_F32 ? 4 : 2;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kv_skew(BYTES)];
  const int tid = threadIdx.x, head = blockIdx.y;
  const bool val = blockIdx.z & 1;
  const int b = blockIdx.z >> 1;
  const int cap = blocks * KV_BLOCK;
  int len = lens[b];
  len = len < 0 ? 0 : len > cap ? cap : len;
  int first = first_in ? first_in[b] : 0;
  first = first < 0 ? 0 : first > cap ? cap : first;
  const int block = first / KV_BLOCK + blockIdx.x;
  const int lo = block * KV_BLOCK > first ? block * KV_BLOCK : first;               // tokens lo..hi of this workgroup
  const long stop = (long)first + n;
  const int hi = (long)block * KV_BLOCK + KV_BLOCK < stop ? block * KV_BLOCK + KV_BLOCK : (int)stop;
  if (lo >= hi) return;
  const long which = ((long)b * Hk + head) * blocks + block;
  float s = 0.f;
  if (lo < len) {
    const uint4* from = reinterpret_cast<const uint4*>((val ? v_codes : k_codes) + which * BYTES);
    for (int i = tid; i < BYTES / 16; i += 256) *reinterpret_cast<uint4*>(lds + kv_skew(16 * i)) = from[i];
    s = (val ? v_scales : k_scales)[which];
  }
  __syncthreads();
  uint8_t* out = val ? v_out : k_out;
  // a thread takes 4 dims of 4 consecutive tokens: a dword of codes for each of the tokens
  // (keys) or dims (values)
  for (int i = tid; i < KV_BLOCK / 4 * (D / 4); i += 256) {
    const int tok = 4 * (i / (D / 4)), d = 4 * (i % (D / 4)), p0 = block * KV_BLOCK + tok;
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = *reinterpret_cast<const uint32_t*>(
          lds + kv_skew(val ? kv_value_offset<D>(tok, d + e) : kv_key_offset<D>(tok + e, d)));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int p = p0 + r;
      if (p < lo || p >= hi) continue;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[e] = p < len ? s * (float)(int8_t)(val ? w[e] >> (8 * r) : w[r] >> (8 * e)) : 0.f;
      uint8_t* to = out + ((((long)b * n + (p - first)) * Hk + head) * D + d) * ES;
      if constexpr (DT == QV_F32) {
        *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
      } else {
        *reinterpret_cast<uint2*>(to) = make_uint2(pack2<DT == QV_BF16>(x[0], x[1]), pack2<DT == QV_BF16>(x[2], x[3]));
      }
    }
  }
}

}  // namespace qv

static int kv8_check(int64_t B, int64_t Hk, int64_t D, int64_t blocks) {
  QV_CHECK_ARG(D == 64 || D == 128, "head_dim must be 64 or 128 (got %lld)", (long long)D);
  QV_CHECK_ARG(B >= 0 && B <= 32767 && Hk > 0 && Hk <= 65535 && blocks > 0 && blocks <= (INT32_MAX >> 8),
               "bad cache shape B=%lld heads=%lld blocks=%lld", (long long)B, (long long)Hk, (long long)blocks);
  return QV_OK;
}

extern "C" int qv_kv8_append(const void* k, const void* v, int dtype, void* k_codes, void* v_codes, float* k_scales,
                             float* v_scales, const int32_t* start, int32_t* lens, uint32_t* tickets,
                             const int32_t* counts, int64_t B, int64_t n, int64_t Hk, int64_t D, int64_t blocks,
                             const int64_t* k_strides, const int64_t* v_strides, void* stream) {
  if (int rc = kv8_check(B, Hk, D, blocks)) return rc;
  QV_CHECK_ARG(dtype == QV_F16 || dtype == QV_BF16, "bad dtype %d", dtype);
  QV_CHECK_ARG(n >= 0 && n <= blocks * qv::KV_BLOCK, "%lld new tokens do not fit a cache of %lld", (long long)n,
               (long long)(blocks * qv::KV_BLOCK));
  if (B == 0) return QV_OK;
  QV_CHECK_ARG(k_codes && v_codes && k_scales && v_scales && start && lens && tickets, "null pointer argument");
  QV_CHECK_ARG(n == 0 || (k && v && k_strides && v_strides), "null pointer argument");
  QV_CHECK_ARG((uintptr_t)k_codes % 16 == 0 && (uintptr_t)v_codes % 16 == 0, "codes must be 16-byte aligned");
  int64_t ks[3] = {0, 0, 0}, vs[3] = {0, 0, 0};
  if (n) {
    QV_CHECK_ARG((uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0, "k and v must be 16-byte aligned");
    for (int i = 0; i < 3; ++i) {
      ks[i] = k_strides[i], vs[i] = v_strides[i];
      QV_CHECK_ARG(ks[i] % 8 == 0 && vs[i] % 8 == 0, "k and v strides must be multiples of 8 elements");
    }
  }
  // the blocks that n tokens can touch, wherever the first of them falls
  const dim3 grid((unsigned)(n ? (n + qv::KV_BLOCK - 2) / qv::KV_BLOCK + 1 : 1), (unsigned)Hk, (unsigned)B);
#define QV_APPEND(DIM, BF)                                                                                           \
  hipLaunchKernelGGL((qv::kv8_append_kernel<DIM, BF>), grid, dim3(4 * DIM), 0, (hipStream_t)stream, (const uint16_t*)k, \
                     (const uint16_t*)v, (uint8_t*)k_codes, (uint8_t*)v_codes, k_scales, v_scales, start, lens, tickets, \
                     counts, (int)n, (int)Hk, (int)blocks, (long)ks[0], (long)ks[1], (long)ks[2], (long)vs[0],       \
                     (long)vs[1], (long)vs[2])
  if (D == 64) {
    if (dtype == QV_BF16) QV_APPEND(64, true);
    else QV_APPEND(64, false);
  } else {
    if (dtype == QV_BF16) QV_APPEND(128, true);
    else QV_APPEND(128, false);
  }
#undef QV_APPEND
  return qv::check_launch("kv8_append");
}

extern "C" int qv_kv8_values(const void* k_codes, const void* v_codes, const float* k_scales, const float* v_scales,
                             const int32_t* lens, const int32_t* first, void* k_out, void* v_out, int dtype, int64_t B,
                             int64_t n, int64_t Hk, int64_t D, int64_t blocks, void* stream) {
  if (int rc = kv8_check(B, Hk, D, blocks)) return rc;
  QV_CHECK_ARG(dtype == QV_F16 || dtype == QV_BF16 || dtype == QV_F32, "bad dtype %d", dtype);
  QV_CHECK_ARG(n >= 0 && n <= (INT32_MAX >> 2), "bad number of tokens %lld", (long long)n);
  if (B == 0 || n == 0) return QV_OK;
  QV_CHECK_ARG(k_codes && v_codes && k_scales && v_scales && lens && k_out && v_out, "null pointer argument");
  QV_CHECK_ARG((uintptr_t)k_codes % 16 == 0 && (uintptr_t)v_codes % 16 == 0 && (uintptr_t)k_out % 16 == 0 &&
                   (uintptr_t)v_out % 16 == 0,
               "codes and outputs must be 16-byte aligned");
  const dim3 grid((unsigned)((n + qv::KV_BLOCK - 2) / qv::KV_BLOCK + 1), (unsigned)Hk, (unsigned)(2 * B));
#define QV_VALUES(DIM, DT)                                                                                            \
  hipLaunchKernelGGL((qv::kv8_values_kernel<DIM, DT>), grid, dim3(256), 0, (hipStream_t)stream, (const uint8_t*)k_codes, \
                     (const uint8_t*)v_codes, k_scales, v_scales, lens, first, (int)n, (int)Hk, (int)blocks,          \
                     (uint8_t*)k_out, (uint8_t*)v_out)
  if (D == 64) {
    if (dtype == QV_F32) QV_VALUES(64, QV_F32);
    else if (dtype == QV_BF16) QV_VALUES(64, QV_BF16);
    else QV_VALUES(64, QV_F16);
  } else {
    if (dtype == QV_F32) QV_VALUES(128, QV_F32);
    else if (dtype == QV_BF16) QV_VALUES(128, QV_BF16);
    else QV_VALUES(128, QV_F16);
  }
#undef QV_VALUES
  return qv::check_launch("kv8_values");
}
