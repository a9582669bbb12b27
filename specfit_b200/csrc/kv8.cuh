// The 8-bit KV cache: layout, checks and device helpers shared by its kernels.
//
// Keys and values of the first `sealed` tokens are e4m3 codes, one byte per
// element, with one fp32 scale per block of `block_tokens` tokens and KV
// head; the rows after them (the tail: the open block and the rows of the
// running pass) are bf16.  A scale is a power of two, 2^e with e the least
// integer (at least -100) for which the block's largest magnitude is at most
// 448 * 2^e, so that
//   * code * scale is exact in bf16 (4 significant bits): reading a block
//     back and sealing it again changes nothing, and
//   * moving a row to a block of another scale is exact too, except for
//     values below 2^-6 of the new scale, which keep 2^-10 of it absolutely.
// e4m3 is a floating-point type, so a scale up to one binade larger than the
// tightest costs no relative precision.  A block that holds a NaN or an
// infinity gets a NaN scale (and zero codes): it reads as NaN.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace sf {

constexpr int kKv8MinExponent = -100;

// Checks shared by every entry point that reads a sf_kv8_rows.
int kv8_check(const sf_kv8_rows* r, bool need_values);

// Kernels that this thread's last attention or weight call launched so far.
int& kv8_launches();

// Whether the requests and heads of something to be written lie apart: each
// is `extent` elements, `b` of them bs apart, `h` hs apart.
inline bool kv8_apart(int64_t b, int64_t bs, int64_t h, int64_t hs, int64_t extent) {
  if (extent <= 0) return true;
  if (b > 1 && bs < extent) return false;
  if (h > 1 && hs < extent) return false;
  if (b <= 1 || h <= 1) return true;
  return bs >= hs ? (bs - extent) / hs >= h - 1 : (hs - extent) / bs >= b - 1;
}

struct Kv8Rows {
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  const __nv_bfloat16* kt;
  const __nv_bfloat16* vt;
  int64_t c_bs, c_hs, s_bs, s_hs, t_bs, t_hs;
  int64_t sealed, tail;
  int hkv, d, block, block_shift;
};

inline Kv8Rows kv8_view(const sf_kv8_rows& r) {
  Kv8Rows o;
  o.k = static_cast<const uint8_t*>(r.k_codes);
  o.v = static_cast<const uint8_t*>(r.v_codes);
  o.ks = r.k_scale;
  o.vs = r.v_scale;
  o.kt = static_cast<const __nv_bfloat16*>(r.k_tail);
  o.vt = static_cast<const __nv_bfloat16*>(r.v_tail);
  o.c_bs = r.code_batch_stride;
  o.c_hs = r.code_head_stride;
  o.s_bs = r.scale_batch_stride;
  o.s_hs = r.scale_head_stride;
  o.t_bs = r.tail_batch_stride;
  o.t_hs = r.tail_head_stride;
  o.sealed = r.sealed;
  o.tail = r.tail;
  o.hkv = r.num_kv_heads;
  o.d = r.head_dim;
  o.block = r.block_tokens;
  o.block_shift = r.block_tokens == 32 ? 5 : (r.block_tokens == 64 ? 6 : 7);
  return o;
}

// 2^e as fp32, e in [-126, 127].
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// log2 of a power of two, rounded down for others.
__device__ __forceinline__ int scale_log2(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }

// The exponent of the power-of-two scale of a block whose largest magnitude
// has the bf16 bits `top` (finite, sign cleared): 448 = 1.75 * 2^8.
__device__ __forceinline__ int kv8_exponent(uint32_t top) {
  const int e = (int)(top >> 7) - 127 - 8 + ((top & 0x7fu) > 96u ? 1 : 0);
  return max(e, kKv8MinExponent);
}

// Two e4m3 codes (the low 16 bits) as exact fp16 values.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
// The high 16 bits.
__device__ __forceinline__ uint32_t e4m3x2_hi_to_f16x2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}

}  // namespace sf
