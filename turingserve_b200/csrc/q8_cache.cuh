// Keys and values held in 8 bits: e4m3 values in pages [pages, KVH, page, D] with one scale (float32) for each
// (page, kv head): what a row stands for is its value times its page's scale.
//
// A scale is 2^e, e the least integer >= -50 with max |x| <= 448 * 2^e over the rows of the page.  Powers of two cost an
// e4m3 value nothing (it has its own exponent), and a page whose scale has to grow for a new row only moves its rows'
// exponents: what lies below 2^-6 of the new scale is rounded again, each time by at most 2^-10 of that scale, and nothing else
// is.  (Above the least scale a page's largest value is above 224 scales: below 2^-13.8 of that, by 2^-17.8 of it.)  A page with a
// value that is not finite, or above 448 * 2^50, has the scale NaN: all that it holds reads as NaN until its first row is
// written again.  The range of e, 101 steps, is what lets the attention kernels keep one reference for a score and a
// value's scale together (attention_q8_decode.cu).
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace q8 {

constexpr int MIN_EXP = -50, MAX_EXP = 50;
constexpr unsigned NAN_BITS = 0x7fc00000u;

// The scale of a page whose largest magnitude has these bits (of |x| as float32).
__device__ __forceinline__ float scale_for(unsigned amax_bits) {
  if (amax_bits > (((unsigned)(MAX_EXP + 8 + 127) << 23) | 0x600000u)) return __uint_as_float(NAN_BITS);   // 448 = 1.75 * 2^8
  int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < MIN_EXP ? MIN_EXP : e;
  return __uint_as_float((unsigned)(e + 127) << 23);
}

// The larger of a page's scale and what new rows need; NaN stays.
__device__ __forceinline__ float larger_scale(float held, float need) {
  return (held != held || need != need) ? __uint_as_float(NAN_BITS) : fmaxf(held, need);
}

// 1 / s of a power of two s (exact); 0 for NaN, under which rows are stored as zeros.
__device__ __forceinline__ float inverse_scale(float s) { return s != s ? 0.f : __uint_as_float(0x7f000000u - __float_as_uint(s)); }

__device__ __forceinline__ unsigned char to_e4m3(float x) { return (unsigned char)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ float from_e4m3(unsigned char b) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3)));
}
// x times 1 / s on its way to 8 bits; a page that reads as NaN stores zeros (x may be infinite: no product then).
__device__ __forceinline__ unsigned char quantise(float x, float inv) { return inv == 0.f ? 0 : to_e4m3(x * inv); }

// Two e4m3 values as half floats (exact).
__device__ __forceinline__ unsigned half2_of(unsigned short e4m3x2) {
  unsigned r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(e4m3x2));
  return r;
}
__device__ __forceinline__ void halves_of(unsigned w, unsigned& lo, unsigned& hi) {
  lo = half2_of((unsigned short)(w & 0xffffu));
  hi = half2_of((unsigned short)(w >> 16));
}
__device__ __forceinline__ unsigned pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ float ex2_q8(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A query head as half floats: times 2^(7 - e), e the exponent of its largest magnitude, so that a bfloat16 fits whole down to 2^-21
// of that; a score's factor takes it back.  A head that is not finite gets the factor NaN.
__device__ __forceinline__ float query_to_half(float amax, float scale, float& factor) {
  const int e = max((int)(__float_as_uint(amax) >> 23) - 127, -110);
  factor = amax <= 3.4028235e38f ? scale * __uint_as_float((unsigned)(127 - 7 + e) << 23) : __uint_as_float(NAN_BITS);
  return __uint_as_float((unsigned)(127 + 7 - e) << 23);
}
__device__ __forceinline__ float abs_or_inf(float x) { return x != x ? INFINITY : fabsf(x); }

// What the kernels of attention over this cache are called with: see attention_q8.cu, attention_q8_decode.cu, attention_q8_prefill.cu.  One
// record for all three; each reads what it needs.
struct AttendCall {
  void* out;
  const void* q;
  const void *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  const int *block_tables, *q_start, *seq_lens;
  float* scratch;
  long long o_ts, q_ts;
  int B, table_width, max_q_len, max_seq_len, H, KVH, D, page, num_pages, window, dtype;
  int nsplit, cluster, early;
  float scale;
};

}  // namespace q8
