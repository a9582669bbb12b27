// Attention over the 8-bit KV cache on tcgen05, for passes with many query
// rows (a 65-row verification tree has 520 packed rows per KV head, a prompt
// chunk thousands), head_dim 128.  Same results as kv8_attn.cu.
//
// With M packed rows a key costs 512 M operations for 256 bytes, so from M of
// about 70 on the tensor cores, not the codes' bytes, are the floor; next to
// them the exponentials (128 x 128 a tile and block at 16 a clock: 1,024
// clocks, as long as the two MMAs take) and the decoding of the codes.  Hence:
//   * A CTA owns one KV head, a key range walked in blocks of 128, and two
//     "lanes" of 128 rows whose chains S = Q K^T -> softmax -> O += P V
//     alternate on the tensor core: one lane's MMAs run under the other's
//     softmax.  With more than 128 packed rows the lanes are two row tiles
//     that share every decoded block; with fewer they are the same rows over
//     the even and the odd blocks (two partial results).
//   * K is never decoded.  A bf16 query is the sum of two e4m3 numbers (its
//     upper and its lower 4 significant bits) once its row is scaled by a
//     power of two, exactly but for bits below 2^-10 of the scaled row (2^-17
//     of its largest value), so S = Q_hi K^T + Q_lo K^T on the fp8 tensor rate,
//     twice bf16's: the same time as one bf16 product.  A key's scale
//     multiplies the fp32 scores.  Tail keys (bf16) are split the same way,
//     with a power of two per key: four products instead of two.
//   * A first kernel (kv8_prep_kernel) lays out what is not codes, once per call:
//     the query tiles and the blocks that hold tail rows, as images of the
//     shared-memory tiles, which a CTA copies whole.  Done by every CTA this
//     took 18,000 clocks of set-up and 17,000 a tail block, and its code made
//     the main loop's slower.
//   * V is decoded to fp16 by four warps, one conversion per two codes, exactly;
//     a tail value's row has a power of two of its own.  These scales enter the
//     exponent: P = 2^(s + log2 scale - reference), the reference a row's own
//     maximum of s + log2 scale over the keys that it sees, and the sum of the
//     probabilities is that of P times the inverse, a factor for 32 keys of one
//     scale.  (A unit for the whole head, applied to V, made every block 0 that
//     was 2^25 below the largest, a key that no row sees included.)
//   * Codes come by TMA: K straight into the operand layout, V raw.  (Loaded
//     into registers a block ahead they are waited for at the next proxy fence,
//     which waits for every load of its warp: 2,200 clocks a block.)
//   * P stays in TMEM: two softmax threads a row (sixteen warps: with eight a
//     scheduler had too little to issue) read 64 scores each, write fp16
//     probabilities over scores that they have read, and the P V MMA takes A
//     from there.  The two meet once a block, at a barrier that also says
//     whether either half wants a larger reference.
//   * O stays in TMEM.  A row's reference moves only when the sum of 64 P,
//     kept times 2^7, passes 2^15 (so none is too large for fp16), and O is
//     read, scaled and written back in the first blocks and hardly ever after.
//     The maximum is not looked for otherwise.
//   * Each lane has its own MMA warp: one that served both spent as long on
//     waits, commits and descriptors as the tensor core on the products.  A lock
//     keeps a lane's P V and next S together: interleaved, both lanes get their
//     scores late and at once, and then fight for the exponentials; one after
//     the other, a lane's softmax runs under the other's products.
//   * Waiting warps sleep in the barrier (up to 20 us a try): as they polled they
//     took issue slots from the softmax warps.
//   * What a softmax thread spills matters: shared memory leaves 28 KB of L1, and the
//     512 threads' stacks stop fitting at 56 bytes each (48 now; forms of this code
//     with 64, 72 and 96 bytes took 410, 519 and 657 us in the case below).  Hence one path of little code for
//     whole blocks of codes, and a rolled one, key by key, for what is masked, tail
//     or far apart in scale; half a block that no row of a warp sees is passed over.
// What it measured: 1,000 rows of 32 heads over 17,391 tokens 396 us, 700
// TFLOP/s; 8 requests of 65 rows over 4,161 tokens 85 us.  A block of two lanes
// takes about 5,400 clocks, the MMAs 2,050 and the exponentials 2,050 of them;
// what bounds it is the chain of one lane (scores, 64 exponentials a thread,
// probabilities to TMEM, two products), of which two fit beside each other.
// P is rounded to fp16 (half a step, 2^-11 relative; the bf16 output's is 2^-8, and 32
// bits would be four times the tensor time); sums are fp32 of the unrounded values.
// TMEM: S / P of lane t in columns [128 t, 128 t + 128), O in [256 + 128 t, ...).
//
// Every wait is bounded (sm100_ptx.cuh); one that gives up records its site
// and the CTA drains its MMAs and returns.
#include <algorithm>

#include "kv8_attn.h"
#include "sm100_ptx.cuh"
#include "swiglu.h"

namespace sf {
namespace {

__device__ int g_kv8_tc_status;

constexpr int kD = 128;
constexpr int kBM = 128;
constexpr int kKB = 128;
constexpr int kHalf = 128 * 128;        // a 128-row tile of e4m3 (bytes); hi, then lo
constexpr int kRegion = 128 * 128;      // one 64-element column region of a 128-row bf16 tile (bytes)
constexpr int kTileBytes = 2 * kRegion;
constexpr int kStages = 2;
constexpr int kSoftmaxWarps = 16, kDecodeWarps = 4;
constexpr int kMmaWarp = kSoftmaxWarps + kDecodeWarps;  // and the next: one per lane
constexpr int kLoadWarp = kMmaWarp + 2;
constexpr int kThreads = (kLoadWarp + 1) * 32;
constexpr int kMaxRanges = 64;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kOCol = 256;
constexpr float kMaxSum = 0x1p15f; // of a row's 64 probabilities of a block, before the reference moves
constexpr float kPShift = 7.f;  // probabilities are kept times 2^7
// Where neither |v| nor what a row's reference lies above its largest score
// passes these, P 2^-v stands for the probability: the largest one's P is at least
// 2^-80, so fp32 holds what is down to 2^-46 of it.
constexpr float kMaxV = 40.f, kMaxAbove = 40.f;

struct __align__(16) Tail {
  float red[2][2][kBM], sum[2][2][kBM];  // per lane, half and row: maxima and final sums, for the other half
  int pair_ok[kSoftmaxWarps];
  // Per block (ring of 4) and key: scale * log2(e) * K scale (NaN for a key that
  // holds one), v = log2 of the V scale times 2^7 (kMinValueScale if less), 2^min(v, 0),
  // 2^-max(v, 0); per 32 keys, of the first: the first two, and 2^-v.
  float4 key[4][kKB], group[4][kKB / 32];
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t raw_full, raw_empty;
  uint64_t s_full[2], p_full[2];
  uint64_t q_ready, mma_done;
  uint32_t tmem_base;
  int abort_flag;
  int tensor_lock;  // held by the lane that is issuing its products
};

constexpr size_t kSmemBytes = 1024 + 2 * kTileBytes + 2 * kStages * kTileBytes + kHalf + sizeof(Tail);

// Byte offset of 16-byte chunk c of row r of a bf16 tile (c < 16: two
// 64-element regions) or an e4m3 one (c < 8): 128-byte rows, 128-byte swizzle.
__device__ __forceinline__ uint32_t sw128(int r, int c) {
  return (uint32_t)((c >> 3) * kRegion + (r >> 3) * 1024 + (r & 7) * 128 + (((c & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN counts as the least
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Eight codes as fp16.
__device__ __forceinline__ uint4 decode8(const uint2& c) {
  return make_uint4(e4m3x2_to_f16x2(c.x), e4m3x2_hi_to_f16x2(c.x), e4m3x2_to_f16x2(c.y), e4m3x2_hi_to_f16x2(c.y));
}
// Eight bf16 values as fp16, times a power of two.
__device__ __forceinline__ uint32_t tail2(uint32_t w, float inv) {
  return pack_f16x2(__uint_as_float(w << 16) * inv, __uint_as_float(w & 0xffff0000u) * inv);
}
__device__ __forceinline__ uint4 tail8(const uint4& x, float inv) {
  return make_uint4(tail2(x.x, inv), tail2(x.y, inv), tail2(x.z, inv), tail2(x.w, inv));
}
// Two bf16 values times `inv` (a power of two that brings them within 448) as
// e4m3 pairs hi + lo, by way of fp16, which holds them exactly down to 2^-17.
__device__ __forceinline__ void split2(uint32_t w, float inv, uint32_t& hi, uint32_t& lo) {
  const uint32_t x = pack_f16x2(__uint_as_float(w << 16) * inv, __uint_as_float(w & 0xffff0000u) * inv);
  uint16_t h, l;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(h) : "r"(x));
  const uint32_t back = e4m3x2_to_f16x2(h);
  const __half2 rest = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&back));
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(l) : "r"(*reinterpret_cast<const uint32_t*>(&rest)));
  hi = h;
  lo = l;
}
// The largest magnitude (bf16 bits) of a row that eight threads hold, 16 values each.
__device__ __forceinline__ uint32_t row_top(const uint32_t (&in)[8]) {
  uint32_t top2 = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top2 = __vmaxu2(top2, in[j] & 0x7fff7fffu);
  uint32_t top = max(top2 & 0xffffu, top2 >> 16);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  return max(top, __shfl_xor_sync(0xffffffffu, top, 4));
}
__device__ __forceinline__ void split_store(const uint32_t (&in)[8], float inv, uint8_t* hi_at, uint8_t* lo_at) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t h0, h1, l0, l1;
    split2(in[2 * j], inv, h0, l0);
    split2(in[2 * j + 1], inv, h1, l1);
    h[j] = __byte_perm(h0, h1, 0x5410);
    l[j] = __byte_perm(l0, l1, 0x5410);
  }
  *reinterpret_cast<uint4*>(hi_at) = make_uint4(h[0], h[1], h[2], h[3]);
  *reinterpret_cast<uint4*>(lo_at) = make_uint4(l[0], l[1], l[2], l[3]);
}
// The largest of 16 scores, scaled.
__device__ __forceinline__ float scaled_max(const float (&x)[16], float f) {
  float a = fmaxf(x[0], x[1]), d = fmaxf(x[2], x[3]);
#pragma unroll
  for (int j = 4; j < 16; j += 4) {
    a = max3(a, x[j], x[j + 1]);
    d = max3(d, x[j + 2], x[j + 3]);
  }
  a = fmaxf(a, d);
  return a == -INFINITY ? a : a * f;
}
// 16 scores to 2^(f x - base), as fp16 pairs, and their sums.
__device__ __forceinline__ void probabilities(const float (&x)[16], float f, float base, uint64_t (&ls)[2],
                                              uint32_t* pk) {
  const uint64_t f2 = ptx::pack2(f, f), b2 = ptx::pack2(-base, -base);
#pragma unroll
  for (int j = 0; j < 16; j += 2) {
    float y0, y1;
    ptx::unpack2(ptx::fma2(ptx::pack2(x[j], x[j + 1]), f2, b2), y0, y1);
    const float p0 = ex2(y0), p1 = ex2(y1);
    ls[(j >> 1) & 1] = ptx::add2(ls[(j >> 1) & 1], ptx::pack2(p0, p1));
    pk[j / 2] = pack_f16x2(p0, p1);
  }
}
// A key's constants, loaded where they are used: sixteen at once cost 64 registers.
__device__ __forceinline__ float4 load_key(const float4* key) {
  float4 k;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(k.x), "=f"(k.y), "=f"(k.z), "=f"(k.w)
               : "r"(ptx::smem_u32(key)));
  return k;
}
// The same key by key, 0 where the row does not see the key; `ls` sums the
// probabilities, `ps` P.  One exponential for both, of the larger of the two, so
// that it is not lost where the other is far below.
__device__ __forceinline__ void weighed(const float (&x)[16], const float4* key, float qf, uint32_t vis, float base,
                                        float& ls, float& ps, uint32_t* pk) {
#pragma unroll
  for (int j = 0; j < 16; j += 2) {
    float p[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 k = load_key(key + j + i);
      const float y = (vis >> (j + i)) & 1u ? ex2(x[j + i] * (k.x * qf) - (base - fmaxf(k.y, 0.f))) : 0.f;
      ls = fmaf(y, k.w, ls);
      p[i] = y * k.z;
      ps += p[i];
    }
    pk[j / 2] = pack_f16x2(p[0], p[1]);
  }
}
// The largest of 16 scores (mx) and of their sums with v (mv), of the keys that
// the row sees (NaN counts as the least).
__device__ __forceinline__ void masked_max(const float (&x)[16], const float4* key, float qf, uint32_t vis, float& mx,
                                           float& mv) {
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float4 k = load_key(key + j);
    const float y = (vis >> j) & 1u ? x[j] * (k.x * qf) : -INFINITY;
    mx = fmaxf(mx, y);
    mv = fmaxf(mv, y + k.y);
  }
}

// Whether any of the 64 threads that meet at barrier `id` says so.
__device__ __forceinline__ bool pair_any(int id, bool mine) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)mine), "r"(id)
      : "memory");
  return r != 0;
}

// A warp's wait and arrival, by one lane: 32 lanes at one barrier are served
// one after another.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int site) {
  int ok = 0;
  if ((threadIdx.x & 31) == 0) ok = ptx::mbar_wait(bar, parity, abort_flag, &g_kv8_tc_status, site) ? 1 : 0;
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();  // what the other lanes wrote and fenced is before the arrival
  if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(bar);
}

// The query head (within its group) of packed row n: n / q_len.
__device__ __forceinline__ int row_head(const Kv8Attn& p, int n) { return (int)(((uint64_t)n * p.q_magic) >> 40); }

// grid: (blocks that are not codes alone, which take longest, then query tiles;
// batch * hkv).
__global__ void __launch_bounds__(256, 2)
kv8_prep_kernel(Kv8Attn p, Kv8Prep w) {
  pdl_wait();
  pdl_trigger();
  const int bh = blockIdx.y, kvh = bh % p.c.hkv, req = bh / p.c.hkv;
  const int row = threadIdx.x >> 3, part = threadIdx.x & 7;  // row of 32 in a pass, 16 dims of it
  const uint32_t at0 = sw128(row, part);                     // 32 rows on: 4,096 bytes
  const int others = (int)gridDim.x - w.tiles;
  if ((int)blockIdx.x >= others) {
    const int tile = blockIdx.x - others, packed = p.group * p.q_len;
    uint8_t* img = w.q + ((int64_t)bh * w.tiles + tile) * kTileBytes + at0;
    uint4 x[4][2];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = tile * kBM + u * 32 + row;
      const bool on = at < packed;
      const int h = on ? row_head(p, at) : 0, t = on ? at - h * p.q_len : 0;
      const __nv_bfloat16* src = p.q + req * p.q_bs + (int64_t)(kvh * p.group + h) * p.q_hs + (int64_t)t * p.q_rs +
                                 part * 16;
      x[u][0] = on ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
      x[u][1] = on ? *reinterpret_cast<const uint4*>(src + 8) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t in[8] = {x[u][0].x, x[u][0].y, x[u][0].z, x[u][0].w, x[u][1].x, x[u][1].y, x[u][1].z, x[u][1].w};
      const uint32_t top = row_top(in);
      const bool nan = top >= 0x7f80u;  // the row answers NaN
      const int e = nan ? 0 : kv8_exponent(top);
      split_store(in, pow2f(-e), img + u * 4096, img + u * 4096 + kHalf);
      if (part == 0) {
        const int64_t at = ((int64_t)bh * w.tiles + tile) * kBM + u * 32 + row;
        const float f = nan ? __int_as_float(0x7fc00000) : pow2f(e);
        if (w.qf) w.qf[at] = f;
        if (w.rowc) {
          const int pr = tile * kBM + u * 32 + row;
          float lse = -INFINITY;
          if (pr < packed) {
            const int h = row_head(p, pr);
            lse = p.lse[((int64_t)req * p.heads + kvh * p.group + h) * p.q_len + (pr - h * p.q_len)];
          }
          // Rows that see nothing, and those past the last, add 2^-infinity.
          float* c = w.rowc + 2 * (at - u * 32 - row) + u * 32 + row;
          c[0] = f * p.scale_log2;
          c[kBM] = lse == -INFINITY ? lse : -lse * 1.4426950408889634f;
        }
      }
    }
    return;
  }
  const bool values = w.v != nullptr;
  const int sealed = (int)p.c.sealed;
  const float* vsc = p.c.vs + req * p.c.s_bs + kvh * p.c.s_hs;
  const float* ksc = p.c.ks + req * p.c.s_bs + kvh * p.c.s_hs;
  const __nv_bfloat16* kt = p.c.kt + req * p.c.t_bs + kvh * p.c.t_hs;
  const __nv_bfloat16* vt = p.c.vt + req * p.c.t_bs + kvh * p.c.t_hs;
  const int blk = blockIdx.x;
  const uint8_t* kc = p.c.k + req * p.c.c_bs + kvh * p.c.c_hs + part * 16;
  const uint8_t* vc = p.c.v + req * p.c.c_bs + kvh * p.c.c_hs + part * 8;  // dims 8 part .. and 64 + 8 part ..
  uint8_t* kimg = w.k + ((int64_t)bh * w.blocks + blk) * kTileBytes + at0;
  uint8_t* vimg = w.v + ((int64_t)bh * w.blocks + blk) * kTileBytes + at0;
  float* kf = w.kf + ((int64_t)bh * w.blocks + blk) * kKB;
  float* vf = w.vf + ((int64_t)bh * w.blocks + blk) * kKB;
  const int key0 = w.first + blk * kKB;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int key = key0 + u * 32 + row;
    uint4 a = make_uint4(0, 0, 0, 0), c = a, x = a, y = a;
    float f = 1.f, fv = 1.f;
    if (key0 + u * 32 < sealed) {  // the 32 rows of a pass are all codes or all tail
      a = *reinterpret_cast<const uint4*>(kc + (int64_t)key * kD);
      f = ksc[key >> p.c.block_shift];
      if (values) {
        fv = vsc[key >> p.c.block_shift];
        if (fv != fv) {  // rows that see the key answer NaN; its codes are zeros
          f = fv;
          fv = 1.f;
        }
        x = decode8(*reinterpret_cast<const uint2*>(vc + (int64_t)key * kD));
        y = decode8(*reinterpret_cast<const uint2*>(vc + (int64_t)key * kD + 64));
      }
      *reinterpret_cast<uint4*>(kimg + u * 4096) = a;
      *reinterpret_cast<uint4*>(kimg + u * 4096 + kHalf) = c;  // codes have no lower part
    } else {
      if (key < p.kv_len) {
        const int64_t at = (int64_t)(key - sealed) * kD;
        a = *reinterpret_cast<const uint4*>(kt + at + part * 16);
        c = *reinterpret_cast<const uint4*>(kt + at + part * 16 + 8);
        if (values) {
          x = *reinterpret_cast<const uint4*>(vt + at + part * 8);
          y = *reinterpret_cast<const uint4*>(vt + at + part * 8 + 64);
        }
      }
      uint32_t in[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
      const uint32_t vals[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
      const uint32_t ktop = row_top(in), vtop = row_top(vals);
      const bool nan = max(ktop, vtop) >= 0x7f80u;  // rows that see the key answer NaN
      if (nan) {
#pragma unroll
        for (int j = 0; j < 8; ++j) in[j] = 0;
        x = y = make_uint4(0, 0, 0, 0);
      }
      const int e = nan ? 0 : kv8_exponent(ktop);
      split_store(in, pow2f(-e), kimg + u * 4096, kimg + u * 4096 + kHalf);
      f = nan ? __int_as_float(0x7fc00000) : pow2f(e);
      const int ev = nan ? 0 : kv8_exponent(vtop);
      fv = pow2f(ev);
      x = tail8(x, pow2f(-ev));
      y = tail8(y, pow2f(-ev));
    }
    if (values) {
      *reinterpret_cast<uint4*>(vimg + u * 4096) = x;
      *reinterpret_cast<uint4*>(vimg + u * 4096 + kRegion) = y;
    }
    if (part == 0) {
      kf[u * 32 + row] = f;
      if (values) vf[u * 32 + row] = fv;
    }
  }
}

// One lane's turn at the tensor core.  False: the wait gave up.
__device__ __forceinline__ bool take_turn(int* lock, volatile int* abort_flag, int site) {
  uint64_t t0 = 0;
  for (uint32_t i = 0;; ++i) {
    if (atomicCAS_block(lock, 0, 1) == 0) return true;
    if ((i & 15u) == 15u) {
      if (*abort_flag) return false;
      const uint64_t now = ptx::globaltimer_ns();
      if (t0 == 0) {
        t0 = now;
      } else if (now - t0 > ptx::kWaitLimitNs) {
        *abort_flag = 1;
        atomicCAS(&g_kv8_tc_status, 0, site);
        return false;
      }
    }
  }
}

__global__ void __launch_bounds__(kThreads, 1)
kv8_attn_tc_kernel(const __grid_constant__ CUtensorMap tm_k, Kv8Attn p, Kv8Prep w, int dual, int ranges) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = smem;
  uint8_t* k_s = q_s + 2 * kTileBytes;
  uint8_t* v_s = k_s + kStages * kTileBytes;
  uint8_t* raw_s = v_s + kStages * kTileBytes;  // one block's V codes
  Tail* tail = reinterpret_cast<Tail*>(raw_s + kHalf);
  volatile int* abort_flag = &tail->abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.x;
  const int req = blockIdx.z / ranges, range = blockIdx.z % ranges;
  const int packed = p.group * p.q_len;
  const int tile0 = dual ? blockIdx.y * 2 : 0;
  const int key_lo = range * p.keys_per_split;
  const int key_hi = min(p.kv_len, key_lo + p.keys_per_split);
  const int nblocks = key_hi > key_lo ? (key_hi - key_lo + kKB - 1) / kKB : 0;
  // Lanes in use, and the blocks of lane t: all of them, or every other one.
  const int nlanes = dual ? ((tile0 + 1) * kBM < packed ? 2 : 1) : min(2, nblocks);
  // Blocks of codes alone come first; the others are laid out already.
  const int coded = max(0, min(nblocks, ((int)p.c.sealed - key_lo) / kKB));
  auto lane_blocks = [&](int t) { return dual ? nblocks : (nblocks - t + 1) / 2; };
  auto block_of = [&](int t, int i) { return dual ? i : 2 * i + t; };

  if (threadIdx.x == 0) {
    const int users = dual ? nlanes : 1;  // lanes that read one block
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(&tail->k_full[s], kDecodeWarps + 1);  // scales or tail rows, and the copy
      ptx::mbar_init(&tail->k_empty[s], users);
      ptx::mbar_init(&tail->v_full[s], kDecodeWarps);
      ptx::mbar_init(&tail->v_empty[s], users);
    }
    ptx::mbar_init(&tail->raw_full, 1);
    ptx::mbar_init(&tail->raw_empty, kDecodeWarps);
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(&tail->s_full[t], 1);
      ptx::mbar_init(&tail->p_full[t], kSoftmaxWarps / 2);
    }
    ptx::mbar_init(&tail->q_ready, 1);
    ptx::mbar_init(&tail->mma_done, 2);
    tail->abort_flag = 0;
    tail->tensor_lock = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(&tail->tmem_base, kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = tail->tmem_base;

  if (warp == kLoadWarp) {
    // ---------------- TMA producer ----------------
    if (lane == 0 && nblocks > 0) {
      const int bh = req * p.c.hkv + kvh;
      const uint32_t qbytes = (dual ? nlanes : 1) * kTileBytes;
      ptx::mbar_arrive_expect_tx(&tail->q_ready, qbytes);
      ptx::bulk_load(q_s, w.q + ((int64_t)bh * w.tiles + tile0) * kTileBytes, qbytes, &tail->q_ready);
      const uint8_t* vc = p.c.v + req * p.c.c_bs + kvh * p.c.c_hs;
      int b = 0;
      bool ok = true;
      for (; ok && b < nblocks; ++b) {
        const int s = b % kStages, key0 = key_lo + b * kKB;
        ok = ptx::mbar_wait(&tail->k_empty[s], ((b / kStages) & 1) ^ 1, abort_flag, &g_kv8_tc_status, 51);
        if (!ok) break;
        if (b >= coded) {
          ptx::mbar_arrive_expect_tx(&tail->k_full[s], kTileBytes);
          ptx::bulk_load(k_s + s * kTileBytes, w.k + ((int64_t)bh * w.blocks + (key0 - w.first) / kKB) * kTileBytes,
                         kTileBytes, &tail->k_full[s]);
          continue;  // V of such a block: the decoders ask for it
        }
        ptx::mbar_arrive_expect_tx(&tail->k_full[s], kHalf);
        ptx::tma_load_4d(k_s + s * kTileBytes, &tm_k, &tail->k_full[s], 0, key0, kvh, req);
        ok = ptx::mbar_wait(&tail->raw_empty, (b & 1) ^ 1, abort_flag, &g_kv8_tc_status, 52);
        if (!ok) break;
        ptx::mbar_arrive_expect_tx(&tail->raw_full, kHalf);
        ptx::bulk_load(raw_s, vc + (int64_t)key0 * kD, kHalf, &tail->raw_full);
      }
      if (!ok) {  // another role gave up: let the copies in flight land before the CTA ends
        volatile int never = 0;
        ptx::mbar_wait(&tail->q_ready, 0, &never, &g_kv8_tc_status, 53);
        for (int i = max(0, b - 1); i <= b && i < nblocks; ++i)
          ptx::mbar_wait(&tail->k_full[i % kStages], (i / kStages) & 1, &never, &g_kv8_tc_status, 53);
        if (b > 0 && coded > 0)
          ptx::mbar_wait(&tail->raw_full, (min(b, coded) - 1) & 1, &never, &g_kv8_tc_status, 54);
      }
    }
  } else if (warp >= kMmaWarp) {
    // ---------------- MMA issuer of one lane ----------------
    if (lane == 0) {
      const int t = warp - kMmaWarp, blocks = t < nlanes ? lane_blocks(t) : 0;
      const uint32_t idesc_s = ptx::idesc_e4m3_f32(kBM, kKB);
      const uint32_t idesc_o = ptx::idesc_f16_f32(kBM, kD) | ptx::kIdescBMajorMN;
      constexpr uint64_t kLo = kHalf >> 4, kStep = 32 >> 4;
      const uint64_t qdesc = ptx::smem_desc_k_sw128(ptx::smem_u32(q_s + (dual ? t : 0) * kTileBytes));
      const uint32_t scol = tmem + t * kBM, ocol = tmem + kOCol + t * kD;
      bool ok = blocks == 0 || ptx::mbar_wait(&tail->q_ready, 0, abort_flag, &g_kv8_tc_status, 41);
      // O += P V of block i - 1, then S of block i over that block's P, which
      // the MMAs just issued read first.
#pragma unroll 1
      for (int i = 0; ok && i <= blocks && blocks > 0; ++i) {
        const int bo = block_of(t, i - 1), so = bo & 1, bs = block_of(t, i), ss = bs & 1;
        if (i < blocks && !ptx::mbar_wait(&tail->k_full[ss], (bs / kStages) & 1, abort_flag, &g_kv8_tc_status, 42)) break;
        if (i > 0 &&
            (!ptx::mbar_wait(&tail->v_full[so], (bo / kStages) & 1, abort_flag, &g_kv8_tc_status, 43) ||
             !ptx::mbar_wait(&tail->p_full[t], (i - 1) & 1, abort_flag, &g_kv8_tc_status, 44)))
          break;
        if (!take_turn(&tail->tensor_lock, abort_flag, 56)) break;
        ptx::tc_fence_after();
        if (i > 0) {
          const uint64_t vdesc = ptx::smem_desc_mn_sw128(ptx::smem_u32(v_s + so * kTileBytes), kRegion);
#pragma unroll
          for (int k = 0; k < kKB / 16; ++k)
            ptx::umma_f16_ta(ocol, scol + (k >> 2) * 64 + (k & 3) * 8, vdesc + (uint64_t)((k * 16 * 128) >> 4), idesc_o,
                             i > 1 || k != 0);
          ptx::umma_commit(&tail->v_empty[so]);
        }
        if (i < blocks) {
          const uint64_t kdesc = ptx::smem_desc_k_sw128(ptx::smem_u32(k_s + ss * kTileBytes));
          // hi and lo of Q with K; a block with tail keys has a lower part of K too.
          const int parts = bs >= coded ? 4 : 2;
#pragma unroll 1
          for (int x = 0; x < parts; ++x) {
            const uint64_t qd = qdesc + (x & 1) * kLo, kd = kdesc + (x >> 1) * kLo;
#pragma unroll
            for (int k = 0; k < kD / 32; ++k)
              ptx::umma_f8(scol, qd + k * kStep, kd + k * kStep, idesc_s, x != 0 || k != 0);
          }
          ptx::umma_commit(&tail->s_full[t]);
          ptx::umma_commit(&tail->k_empty[ss]);
        }
        atomicExch_block(&tail->tensor_lock, 0);
      }
      ptx::umma_commit(&tail->mma_done);
      volatile int never = 0;
      ptx::mbar_wait(&tail->mma_done, 0, &never, &g_kv8_tc_status, 45);
    }
  } else if (warp >= kSoftmaxWarps) {
    // ---------------- decoders ----------------
    const int ct = threadIdx.x - kSoftmaxWarps * 32, bh = req * p.c.hkv + kvh;
    const int row = ct >> 3, part = ct & 7;  // row of 16 in a pass, 8 + 8 dims of it
    const float* ksc = p.c.ks + req * p.c.s_bs + kvh * p.c.s_hs;
    const float* vsc = p.c.vs + req * p.c.s_bs + kvh * p.c.s_hs;
    float ks = 0.f, vs = 1.f;  // scales of key ct of the next block
    auto load_ks = [&](int b) {
      const int key = key_lo + b * kKB + ct;
      if (b < coded) {
        vs = vsc[key >> p.c.block_shift];
        ks = ksc[key >> p.c.block_shift];
        if (vs != vs) {  // a block with a NaN among its values: NaN scores, zero codes
          ks = vs;
          vs = 1.f;
        }
      } else {
        ks = w.kf[(int64_t)bh * w.blocks * kKB + (key - w.first)];
        vs = w.vf[(int64_t)bh * w.blocks * kKB + (key - w.first)];
      }
    };
    if (nblocks > 0) load_ks(0);
    // K of block b is on its way; here its scales.  False: a wait gave up.
    auto store_k = [&](int b) -> bool {
      const int s = b % kStages;
      if (!warp_wait(&tail->k_empty[s], ((b / kStages) & 1) ^ 1, abort_flag, 46)) return false;
      // Ring of four: block b - 4's softmax is over.  (The scores that freed this
      // stage, block b - 2's, were issued after P V of the lane's block before.)
      const float kf = ks * p.scale_log2;
      float v = (float)(scale_log2(vs) + (int)kPShift), s128 = vs * 0x1p7f, inv;
      if (const uint32_t mantissa = __float_as_uint(vs) & 0x7fffffu) {
        v += log2f(__uint_as_float(mantissa | 0x3f800000u));
        inv = 1.f / s128;
      } else {
        inv = pow2f(-(int)v);
      }
      tail->key[b & 3][ct] =
          make_float4(kf, fmaxf(v, (float)kMinValueScale), v < 0.f ? s128 : 1.f, v > 0.f ? inv : 1.f);
      if (lane == 0) tail->group[b & 3][ct >> 5] = make_float4(kf, v, inv, 0.f);
      warp_arrive(&tail->k_full[s]);
      return true;
    };
    auto store_v = [&](int b) -> bool {
      const int s = b % kStages;
      if (b < coded && !warp_wait(&tail->raw_full, b & 1, abort_flag, 55)) return false;
      if (!warp_wait(&tail->v_empty[s], ((b / kStages) & 1) ^ 1, abort_flag, 47)) return false;
      if (b >= coded) {  // laid out already
        if (ct == 0) {
          ptx::mbar_arrive_expect_tx(&tail->v_full[s], kTileBytes);
          ptx::bulk_load(v_s + s * kTileBytes,
                         w.v + ((int64_t)bh * w.blocks + (key_lo + b * kKB - w.first) / kKB) * kTileBytes, kTileBytes,
                         &tail->v_full[s]);
        } else if (lane == 0) {
          ptx::mbar_arrive(&tail->v_full[s]);
        }
        return true;
      }
      // The two halves of a row, odd rows the upper one first: four rows of a
      // warp then cover all banks.
      const uint8_t* raw = raw_s + row * kD + part * 8;
      const int h0 = (row & 1) * 64, h1 = 64 - h0;
      uint8_t* vst = v_s + s * kTileBytes + sw128(row, part);  // 16 rows on: 2,048 bytes
      uint8_t *to0 = vst + h0 * (kRegion / 64), *to1 = vst + h1 * (kRegion / 64);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const uint2 a = *reinterpret_cast<const uint2*>(raw + u * 16 * kD + h0);
        const uint2 c = *reinterpret_cast<const uint2*>(raw + u * 16 * kD + h1);
        *reinterpret_cast<uint4*>(to0 + u * 2048) = decode8(a);
        *reinterpret_cast<uint4*>(to1 + u * 2048) = decode8(c);
      }
      warp_arrive(&tail->raw_empty);
      ptx::fence_proxy_async_smem();
      warp_arrive(&tail->v_full[s]);
      return true;
    };
    // K runs a block ahead of V.  (With one row tile each lane has one stage, and
    // a V that waited for its lane's last P V in front of the other lane's K
    // would wait for good.)
    bool ok = nblocks > 0 && store_k(0);
    if (ok && nblocks > 1) load_ks(1);
    int b = 0;
    for (; ok && b < nblocks; ++b) {
      if (b + 1 < nblocks) {
        ok = store_k(b + 1);
        if (!ok) break;
        if (b + 2 < nblocks) load_ks(b + 2);
      }
      ok = store_v(b);
    }
    if (!ok && ct == 0) {  // copies of V that this thread asked for land before the CTA ends
      volatile int never = 0;
      for (int i = max(coded, b - 2); i < b; ++i)
        ptx::mbar_wait(&tail->v_full[i % kStages], (i / kStages) & 1, &never, &g_kv8_tc_status, 57);
    }
  } else {
    // ---------------- softmax / epilogue: two threads per row ----------------
    const int t = warp >> 3, half = (warp >> 2) & 1, quad = warp & 3;
    const int pair_bar = 3 + t * 4 + quad;  // the two warps of a lane's quadrant
    const int r = quad * 32 + lane;
    const int pr = (tile0 + (dual ? t : 0)) * kBM + r;
    const bool rok = pr < packed;
    const bool warp_ok = t < nlanes && pr - lane < packed;  // uniform over the pair of warps

    const float qf = rok ? w.qf[((int64_t)req * p.c.hkv + kvh) * w.tiles * kBM + pr] : 0.f;

    const uint32_t scol = tmem + ((uint32_t)(quad * 32) << 16) + t * kBM + half * 64;  // this half's scores
    const uint32_t ocol = scol + kOCol;
    const int row0 = rok ? pr - row_head(p, pr) * p.q_len : 0;
    const uint32_t* rbits = p.bits ? p.bits + req * p.bits_bs + (int64_t)row0 * p.words : nullptr;
    const int n = t < nlanes ? lane_blocks(t) : 0;
    float m = -INFINITY, l = 0.f;  // the reference (base 2) of O and of the sum of the probabilities
    bool ok = true, close = true;  // close: the reference is not far above the row's scores (uniform over the warp)
    for (int i = 0; i < n; ++i) {
      const int b = block_of(t, i), key0 = key_lo + b * kKB + half * 64;
      const bool full = key0 + 64 <= p.prefix;  // no mask to read
      uint64_t win = ~0ull;
      if (!full) win = rok ? kv8_window(p, rbits, key0) : 0ull;
      ok = warp_wait(&tail->s_full[t], i & 1, abort_flag, 48);
      if (warp_ok) {
        // Every key visible and one scale per 32 of them: the rule in a long context.
        const bool plain = full && key0 + 64 <= (int)p.c.sealed;
        const float4 *key = tail->key[b & 3] + half * 64, *group = tail->group[b & 3] + half * 2;
        uint32_t pk[32];  // 64 probabilities
        // Once under the reference as it is.  If the sum of a row's 64 P (in
        // either half) passes 2^15, one of them may be too large for fp16: then
        // (and for the first block) the maximum is found, and they are taken
        // under it.  (A maximum in every pass was 36 of 230 instructions.)  The
        // scores stay in TMEM until the probabilities are settled.
        if (ok) ptx::tc_fence_after();
#pragma unroll 1
        for (int pass = i == 0 ? 1 : 0;; ++pass) {
          if (pass) {
            float mx = -INFINITY, mv = -INFINITY;
            if (ok) {
#pragma unroll 1
              for (int c = 0; c < 4; ++c) {
                float sc[16];
                ptx::tmem_ld_16(scol + c * 16, sc);
                if (plain) {
                  const float y = scaled_max(sc, group[c >> 1].x * qf);
                  mx = fmaxf(mx, y);
                  mv = fmaxf(mv, y + fmaxf(group[c >> 1].y, (float)kMinValueScale));
                } else {
                  masked_max(sc, key + c * 16, qf, (uint32_t)(win >> (c * 16)), mx, mv);
                }
              }
            }
            close = close && !__any_sync(0xffffffffu, mv > m && mv - mx > kMaxAbove);
            // The other half's maximum, and whether its wait succeeded: both warps
            // of the pair go on or stop together.
            tail->red[t][half][r] = mv;
            if (lane == 0) tail->pair_ok[warp] = (ok ? 1 : 0) | (close ? 2 : 0);
            ptx::named_bar_sync(pair_bar, 64);
            const int both = tail->pair_ok[warp] & tail->pair_ok[warp ^ 4];
            if (!(both & 1)) {
              ok = false;
              break;
            }
            close = both & 2;
            const float mnew = fmaxf(m, fmaxf(mv, tail->red[t][half ^ 1][r]) - kPShift);
            // Nothing summed yet: O and l are 0.  In two steps: l may be far from 1, and one
            // factor below what fp32 holds.
            const float step = m == -INFINITY ? 1.f : ex2(0.5f * (m - mnew)), alpha = step * step;
            m = mnew;
            l = l * step * step;
            if (i > 0) {  // P V of the block before is complete, as its successor's scores are
#pragma unroll 1
              for (int c = 0; c < 4; ++c) {
                float ov[16];
                ptx::tmem_ld_16(ocol + c * 16, ov);
                uint32_t w[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(ov[j] * alpha);
                ptx::tmem_st_16(ocol + c * 16, w);
              }
            }
          }
          const float base = m == -INFINITY ? 0.f : m;
          float sum = 0.f, psum = 0.f;  // of the probabilities, and of P
          if (ok) {
            if (plain && close && fmaxf(fabsf(group[0].y), fabsf(group[1].y)) <= kMaxV) {
#pragma unroll
              for (int g = 0; g < 2; ++g) {
                const float4 gr = group[g];
                uint64_t ls[2] = {0, 0};
#pragma unroll
                for (int c = 2 * g; c < 2 * g + 2; ++c) {  // 16 at a time: nothing is spilled
                  float sc[16];
                  ptx::tmem_ld_16(scol + c * 16, sc);
                  probabilities(sc, gr.x * qf, base - gr.y, ls, pk + c * 8);
                }
                float s0, s1;
                ptx::unpack2(ptx::add2(ls[0], ls[1]), s0, s1);
                psum += s0 + s1;
                sum = fmaf(s0 + s1, gr.z, sum);
              }
            } else {
              // Key by key: masked blocks, tail rows, scales far apart.  Not unrolled
              // (the registers move down instead): four copies of this body made the path
              // above it a quarter slower, by what was spilled.
#pragma unroll
              for (int j = 0; j < 32; ++j) pk[j] = 0;
              const int chunks = __any_sync(0xffffffffu, win != 0) ? 4 : 0;  // 0: no row of the warp sees any of them
#pragma unroll 1
              for (int c = 0; c < chunks; ++c) {
                float sc[16];
                ptx::tmem_ld_16(scol + c * 16, sc);
#pragma unroll
                for (int j = 0; j < 24; ++j) pk[j] = pk[j + 8];
                weighed(sc, key + c * 16, qf, (uint32_t)(win >> (c * 16)), base, sum, psum, pk + 24);
              }
            }
          }
          if (pass || !pair_any(pair_bar, !ok || !(psum <= kMaxSum) || (m == -INFINITY && rok))) {
            l += sum;
            break;
          }
        }
        if (ok) {
          ptx::tmem_st_32(scol, pk);  // over scores that have been read
          ptx::tmem_wait_st();
        }
      }
      if (!ok) break;
      ptx::tc_fence_before();
      warp_arrive(&tail->p_full[t]);
    }
    if (ok && warp_ok) {  // the pair agrees on this: the row's sum is both halves'
      tail->sum[t][half][r] = l;
      ptx::named_bar_sync(pair_bar, 64);
      l = tail->sum[t][0][r] + tail->sum[t][1][r];
    }
    // The output rows of this lane.
    const bool mine = dual ? t < nlanes : true;  // one row tile: both lanes write a partial result
    if (ok && mine && nblocks > 0)  // also before shared memory is used again
      ok = warp_wait(&tail->mma_done, 0, abort_flag, 49);
    if (ok && mine && pr - lane < packed) {
      const int qhead = rok ? row_head(p, pr) : 0, row = rok ? pr - qhead * p.q_len : 0;
      const int head = kvh * p.group + qhead;
      ptx::tc_fence_after();
      const bool direct = p.splits == 1;
      const int part = dual ? range : 2 * range + t;
      const int64_t idx = (((int64_t)req * p.splits + part) * p.heads + head) * p.q_len + row;
      // P carries 2^7.  Partial results are in units in which the row's sum is about
      // 1, wherever the scale of its values put the reference.
      const int lx = !direct && l > 0.f && l < INFINITY ? max(-100, min(100, scale_log2(l))) : 0;
      const float f = direct ? (l == 0.f ? 0.f : 0x1p-7f / l) : pow2f(-7 - lx);
      // Rows leave in whole lines: 32 rows x 32 columns at a time through this
      // warp's part of the K and V stages, which no MMA reads any more.
      const int64_t off = rok ? (direct ? (int64_t)req * p.out_bs + ((int64_t)row * p.heads + head) * kD : idx * kD) : -1;
      uint8_t* turn = k_s + warp * 32 * 144;
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        uint32_t ov[32];
        if (n > 0) {
          ptx::tmem_ld_32(ocol + c * 32, ov);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) ov[j] = 0;
        }
        __syncwarp();
        const int col0 = half * 64 + c * 32;
        if (direct) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = pack_bf16x2(__uint_as_float(ov[8 * j + 2 * k]) * f, __uint_as_float(ov[8 * j + 2 * k + 1]) * f);
            *reinterpret_cast<uint4*>(turn + lane * 80 + j * 16) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
#pragma unroll 1
          for (int k = 0; k < 4; ++k) {
            const int rr = k * 8 + (lane >> 2), col = lane & 3;
            const int64_t o = __shfl_sync(0xffffffffu, off, rr);
            const uint4 w = *reinterpret_cast<const uint4*>(turn + rr * 80 + col * 16);
            if (o >= 0) *reinterpret_cast<uint4*>(p.out + o + col0 + col * 8) = w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<float4*>(turn + lane * 144 + j * 16) =
                make_float4(__uint_as_float(ov[4 * j]) * f, __uint_as_float(ov[4 * j + 1]) * f,
                            __uint_as_float(ov[4 * j + 2]) * f, __uint_as_float(ov[4 * j + 3]) * f);
          __syncwarp();
#pragma unroll 2
          for (int k = 0; k < 8; ++k) {
            const int rr = k * 4 + (lane >> 3), col = lane & 7;
            const int64_t o = __shfl_sync(0xffffffffu, off, rr);
            const float4 w = *reinterpret_cast<const float4*>(turn + rr * 144 + col * 16);
            if (o >= 0) *reinterpret_cast<float4*>(p.part_o + o + col0 + col * 4) = w;
          }
        }
      }
      if (rok && half == 0) {
        if (direct) {
          if (p.lse)
            p.lse[((int64_t)req * p.heads + head) * p.q_len + row] =
                l == 0.f ? -INFINITY : (m == -INFINITY ? l : (m + log2f(l)) * 0.69314718055994531f);
        } else {
          p.part_ml[idx * 2] = m + (float)lx;
          p.part_ml[idx * 2 + 1] = l * pow2f(-lx);
        }
      }
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, kTmemCols);
  }
}

struct Shape {
  bool dual;
  int64_t tiles, pairs;  // row tiles, CTAs over them
};
Shape shape_of(int64_t packed) {
  const int64_t tiles = (packed + kBM - 1) / kBM;
  return {tiles > 1, tiles, tiles > 1 ? (tiles + 1) / 2 : 1};
}

}  // namespace

// Microseconds a call, this kernel's against the warp-level one's, four KV heads
// (4,159 tokens; 32,831; eight requests of 4,159):
//   48 packed rows: 22 / 30 / 31 against 18 / 27 / 28
//   64:             22 / 31 / 32 against 15 / 33 / 36
//   80:             22 / 31 / 33 against 18 / 37 / 46
//   128:            23 / 32 / 36 against 21 / 53 / 75
bool kv8_use_tc(int head_dim, int64_t packed, int64_t kv_len) { return head_dim == kD && packed > 64 && kv_len > 0; }

// Heads and requests of their own rows: what a tensor map can describe.
bool kv8_tc_layout(const Kv8Rows& c, int batch) {
  return (c.hkv == 1 || c.c_hs >= c.sealed * kD) && (batch == 1 || c.c_bs >= c.sealed * kD);
}

// The number of key ranges that minimises (waves of CTAs) x (blocks of a CTA
// + its fixed cost, about three blocks: set-up, Q, the pipeline's fill and
// drain, the partial result) plus the merge's reading of the partials.
Kv8Split kv8_split_tc(int batch, int hkv, int64_t packed, int64_t kv_len) {
  const Shape sh = shape_of(packed);
  const int64_t units = (int64_t)batch * hkv * sh.pairs;
  const int64_t blocks = (kv_len + kKB - 1) / kKB;
  const int64_t sms = num_sms();
  int64_t best = 1, best_per = blocks;
  double best_cost = 1e30;
  for (int64_t s = 1; s <= std::min<int64_t>(blocks, kMaxRanges); ++s) {
    const int64_t per = (blocks + s - 1) / s, used = (blocks + per - 1) / per;
    const double cost = (double)((units * used + sms - 1) / sms) * ((double)per + 3.0) + 0.05 * (double)used;
    if (cost < best_cost - 1e-9) {
      best_cost = cost;
      best = used;
      best_per = per;
    }
  }
  return {(int)(sh.dual ? best : 2 * best), (int)(best_per * kKB)};
}

// Blocks that are not codes alone: from the one that holds the first tail row
// to the end.  (The boundary is a multiple of 32: without a tail that can be a
// last block that the codes do not fill.)
static int64_t tail_blocks(int64_t sealed, int64_t kv_len) { return (kv_len + kKB - 1) / kKB - sealed / kKB; }

size_t kv8_prep_layout(Kv8Prep* w, void* base, bool for_mass, int64_t heads, int64_t packed, int64_t sealed,
                       int64_t kv_len) {
  const int64_t tiles = shape_of(packed).tiles, blocks = tail_blocks(sealed, kv_len);
  uint8_t* at = static_cast<uint8_t*>(base);
  size_t used = 0;
  auto take = [&](size_t bytes) {
    uint8_t* p = at + used;
    used += (bytes + 127) / 128 * 128;
    return p;
  };
  Kv8Prep r = {};
  r.tiles = (int)tiles;
  r.blocks = (int)blocks;
  r.first = (int)(sealed / kKB * kKB);
  r.q = take((size_t)heads * tiles * kTileBytes);
  r.k = take((size_t)heads * blocks * kTileBytes);
  r.kf = reinterpret_cast<float*>(take((size_t)heads * blocks * kKB * sizeof(float)));
  if (for_mass) {
    r.rowc = reinterpret_cast<float*>(take((size_t)heads * tiles * 2 * kBM * sizeof(float)));
  } else {
    r.v = take((size_t)heads * blocks * kTileBytes);  // not null even so: values are laid out
    r.qf = reinterpret_cast<float*>(take((size_t)heads * tiles * kBM * sizeof(float)));
    r.vf = reinterpret_cast<float*>(take((size_t)heads * blocks * kKB * sizeof(float)));
  }
  if (w) *w = r;
  return used;
}

int kv8_prep(const Kv8Attn& p, const Kv8Prep& w, cudaStream_t stream) {
  const dim3 grid((unsigned)(w.tiles + w.blocks), (unsigned)(p.batch * p.c.hkv));
  SF_CHECK_CUDA(launch_pdl(kv8_prep_kernel, grid, dim3(256), 0, stream, p, w));
  SF_CHECK_LAUNCH();
  ++kv8_launches();
  return SF_OK;
}

int kv8_key_map(CUtensorMap* map, const Kv8Rows& c, int batch) {
  // K's codes, 16 bits at a time (bytes are bytes): [batch][heads][tokens][64].
  *map = {};
  if (c.sealed < kKB) return SF_OK;  // no block of codes alone, no load by this map
  const cuuint64_t dims[4] = {64, (cuuint64_t)c.sealed, (cuuint64_t)c.hkv, (cuuint64_t)batch};
  const int64_t hs = c.hkv > 1 ? c.c_hs : c.sealed * kD, bs = batch > 1 ? c.c_bs : c.hkv * hs;
  const cuuint64_t strides[3] = {kD, (cuuint64_t)hs, (cuuint64_t)bs};
  const cuuint32_t box[4] = {64, kKB, 1, 1};
  return tma_encode_bf16(map, c.k, 4, dims, strides, box);
}

int kv8_attention_tc(const Kv8Attn& p, void* prep, cudaStream_t stream) {
  static std::atomic<unsigned long long> configured{0};
  if (int rc = once_per_device(configured, [] {
        SF_CHECK_CUDA(cudaFuncSetAttribute(kv8_attn_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)kSmemBytes));
        return SF_OK;
      }))
    return rc;
  const Shape sh = shape_of((int64_t)p.group * p.q_len);
  const int ranges = sh.dual ? p.splits : p.splits / 2;
  const int64_t heads = (int64_t)p.batch * p.c.hkv;
  SF_CHECK_ARG(sh.pairs < 65536 && (int64_t)ranges * p.batch < 65536, "too many query rows or requests");
  Kv8Prep w;
  kv8_prep_layout(&w, prep, false, heads, (int64_t)p.group * p.q_len, p.c.sealed, p.kv_len);
  if (int rc = kv8_prep(p, w, stream)) return rc;
  CUtensorMap tm_k;
  if (int rc = kv8_key_map(&tm_k, p.c, p.batch)) return rc;
  const dim3 grid((unsigned)p.c.hkv, (unsigned)sh.pairs, (unsigned)(ranges * p.batch));
  SF_CHECK_CUDA(launch_pdl(kv8_attn_tc_kernel, grid, dim3(kThreads), kSmemBytes, stream, tm_k, p, w, sh.dual ? 1 : 0,
                           ranges));
  SF_CHECK_LAUNCH();
  ++kv8_launches();
  return SF_OK;
}

int kv8_tc_status(int* status, int reset) {
  SF_CHECK_CUDA(cudaMemcpyFromSymbol(status, g_kv8_tc_status, sizeof(int)));
  if (reset) {
    const int zero = 0;
    SF_CHECK_CUDA(cudaMemcpyToSymbol(g_kv8_tc_status, &zero, sizeof(int)));
  }
  return SF_OK;
}

}  // namespace sf
