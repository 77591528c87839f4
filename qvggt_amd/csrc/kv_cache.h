// The 8-bit key / value cache's blocks, shared by the kernels that write them
// (kv_cache.hip) and the attention that reads them (attention_kv.hip).
//
// A block holds 64 consecutive tokens of one (sequence, key head): 64 * D int8
// codes of the keys, as many of the values, and one fp32 scale for each of the two;
// value = code * scale.  Codes lie in the order in which the attention's MFMA
// fragments want them, in units of 16 bytes, 64 units (one for each lane) in a row,
// so that a wave's load of a fragment is one contiguous KB and nothing has to be
// transposed:
//  * keys: unit (kb, u, lane) = dims 32u + 16 (lane / 32) .. + 15 of token 32 kb + lane % 32;
//  * values: unit (db, w, lane) = the 16 tokens {0..3, 8..11} + 4 (lane / 32) of the
//    16-token groups 2w and 2w + 1, of dim 32 db + lane % 32 (the order in which the
//    scores' MFMA leaves a query's probabilities in that lane's registers).
#pragma once
#include "common.h"

namespace qv {

constexpr int KV_BLOCK = 64;

template <int D>
__host__ __device__ __forceinline__ int kv_key_offset(int tok, int dim) {
  return (((tok >> 5) * (D / 32) + (dim >> 5)) * 64 + ((dim >> 4) & 1) * 32 + (tok & 31)) * 16 + (dim & 15);
}
template <int D>
__host__ __device__ __forceinline__ int kv_value_offset(int tok, int dim) {
  const int group = tok >> 4, in = tok & 15;
  return (((dim >> 5) * 2 + (group >> 1)) * 64 + ((in >> 2) & 1) * 32 + (dim & 31)) * 16 + (group & 1) * 8 +
         ((in >> 3) << 2) + (in & 3);
}

}  // namespace qv
