// Device-side pieces of the paged key/value cache that the set, fetch and
// attention kernels share: where a (page, head) tile and its scales lie, the
// floats that it holds (4 bits: sign, 2 exponent bits, 1 mantissa bit: 0,
// 0.5, 1, 1.5, 2, 3, 4, 6; 8 bits: sign, 4, 3, up to 448; 32 values of a row
// share one power of two), and a request's rows and length.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "wave.h"

namespace shmt {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// A cache as the kernels see it; strides in bytes, between pages.
struct PagedView {
  uint8_t *cache;   // [pages] [kv_heads][2][page][dim / 2 or dim]
  uint8_t *scales;  // [pages] [kv_heads][2][dim / 32][page]
  int64_t cache_stride, scales_stride;
  int64_t pages;
  int kv_heads, log2_page;
};

// The scale byte b stands for 2^(b - 127) and 255 for "not a number". As a float's exponent field it is the
// scale operand of the conversion instructions, which read nothing but that field (0 there is 2^-127).
__device__ __forceinline__ float scale_operand(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// The values that the two codes in byte `B` of `codes` stand for.
template <int B>
__device__ __forceinline__ f32x2 decode2_f32(uint32_t codes, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, B);
}
template <int B>
__device__ __forceinline__ uint32_t decode2_bf16(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B));
}

// The same for the two 8-bit codes in half `H` of `codes`.
template <int H>
__device__ __forceinline__ f32x2 decode2_f32_8(uint32_t codes, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, scale, H != 0);
}
template <int H>
__device__ __forceinline__ uint32_t decode2_bf16_8(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, H != 0));
}

struct Request {
  int64_t first_row;  // of `query`
  int32_t queries;
  int32_t before;  // tokens in front of the first query; negative: the first rows see nothing
};

// Request b's rows and the tokens in front of them, whatever the arrays hold: within the `tokens` rows that there are.
__device__ __forceinline__ Request load_request(const void *starts, const void *kv_lens, int len_bytes, int64_t tokens,
                                                int64_t b) {
  int64_t lo, hi;
  load_int_pair(starts, b, len_bytes, &lo, &hi);
  const int64_t len = load_int(kv_lens, b, len_bytes);
  lo = min(max(lo, int64_t{0}), tokens);
  hi = min(max(hi, lo), tokens);
  Request r;
  r.first_row = lo;
  r.queries = static_cast<int32_t>(hi - lo);
  r.before = static_cast<int32_t>(min(max(len, int64_t{0}), int64_t{0x7fffffff}) - (hi - lo));
  return r;
}

}  // namespace shmt
