// Pieces shared by the warp-level (mma.sync) kernels over the 8-bit KV cache.
#pragma once

#include "kv8.cuh"

namespace sf {

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A warp's 8 x 8 matrix of 16-bit values (row g: columns 2c and 2c + 1 of lane 4g + c), transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
template <int Bytes>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool on) {
  const int n = on ? Bytes : 0;  // 0: the destination is filled with zeros
  if constexpr (Bytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// Exponent of the power of two that brings magnitudes up to `top` (bf16
// bits) below 2^14, bounded so that both it and its inverse are normal.
__device__ __forceinline__ int fit_exponent(uint32_t top) {
  return top == 0 ? 0 : max((int)(top >> 7) - 127 - 13, -110);
}


// One query row's part of a thread's A fragments, as fp16 scaled by a power
// of two that is returned: rows r = 0 (row g of the tile) and 1 (row g + 8).
// The dims of k-step s are (s / 4) * 64 + c * 16 + (s % 4) * 4 + {0, 1, 2, 3},
// the order in which a thread's 16-byte pieces of a key hold them.  `row`
// null: zeros.  A row with a NaN or an infinity: zeros, and NaN is returned.  The
// four threads of a quad call this together.
template <int Steps>
__device__ __forceinline__ float q_row_fragments(const __nv_bfloat16* row, int d, int c, uint32_t (&qf)[Steps][4],
                                                 int r) {
  uint2 x[Steps];
  uint32_t top2 = 0;  // two 15-bit magnitudes
#pragma unroll
  for (int s = 0; s < Steps; ++s) {
    const int dim = (s >> 2) * 64 + c * 16 + (s & 3) * 4;
    x[s] = row && dim < d ? *reinterpret_cast<const uint2*>(row + dim) : make_uint2(0, 0);
    top2 = __vmaxu2(__vmaxu2(top2, x[s].x & 0x7fff7fffu), x[s].y & 0x7fff7fffu);
  }
  uint32_t top = max(top2 & 0xffffu, top2 >> 16);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const bool bad = top >= 0x7f80u;
  const int e = bad ? 0 : fit_exponent(top);
  const float inv = pow2f(-e);
#pragma unroll
  for (int s = 0; s < Steps; ++s) {
    if (bad) x[s] = make_uint2(0, 0);
    qf[s][r] = pack_f16x2(bf_lo(x[s].x) * inv, bf_hi(x[s].x) * inv);
    qf[s][r + 2] = pack_f16x2(bf_lo(x[s].y) * inv, bf_hi(x[s].y) * inv);
  }
  return bad ? __int_as_float(0x7fc00000) : pow2f(e);
}

}  // namespace sf
