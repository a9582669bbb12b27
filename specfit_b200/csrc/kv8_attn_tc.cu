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
//   * Four warps decode: codes are loaded a block ahead into registers,
//     turned into bf16 and stored in the swizzled operand layout.  An e4m3
//     code shifted into a bf16's bits is the value times 2^-120; one multiply
//     by a power of two (times the block's V scale, exact) puts it right, 2.25
//     instructions an element.  It takes the codes of a 4-byte word as
//     (0, 2), (1, 3), so the dims of K, V, Q and the output are in that order;
//     K's scale multiplies the fp32 scores, 32 keys at a time.
//   * P stays in TMEM: a softmax thread (one per row) reads its scores,
//     writes bf16 probabilities over them, and the P V MMA takes A from there.
//   * O stays in TMEM.  A row's reference maximum moves only when a score
//     exceeds it by more than 8 (base 2), so O is read, scaled and written
//     back in the first blocks and hardly ever after (bf16 and fp32 have room
//     for 2^8).  It is safe then: a lane's scores of block j are issued, hence
//     complete, after its P V of block j - 1.
// P is rounded to bf16 (2^-9 relative); sums are fp32 of the unrounded values.
// TMEM: S / P of lane t in columns [128 t, 128 t + 128), O in [256 + 128 t, ...).
//
// Every wait is bounded (sm100_ptx.cuh); one that gives up records its site
// and the CTA drains its MMAs and returns.
#include <algorithm>

#include "kv8_attn.h"
#include "sm100_ptx.cuh"

namespace sf {
namespace {

__device__ int g_kv8_tc_status;

constexpr int kD = 128;
constexpr int kBM = 128;
constexpr int kKB = 128;
constexpr int kRegion = 128 * 128;      // one 64-element column region of a 128-row bf16 tile (bytes)
constexpr int kTileBytes = 2 * kRegion;
constexpr int kStages = 2;
constexpr int kSoftmaxWarps = 8, kDecodeWarps = 4;
constexpr int kThreads = (kSoftmaxWarps + kDecodeWarps + 1) * 32;
constexpr int kMmaWarp = kSoftmaxWarps + kDecodeWarps;
constexpr int kMaxRanges = 64;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kOCol = 256;
constexpr float kSlack = 8.f;

struct __align__(16) Tail {
  float kf[4][4];  // per block (ring of 4) and 32 keys: scale * log2(e) * K scale; NaN for a block that holds one
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[2], p_full[2];
  uint64_t q_ready, mma_done;
  uint32_t tmem_base;
  int abort_flag;
};

constexpr size_t kSmemBytes = 1024 + 2 * kTileBytes + 2 * kStages * kTileBytes + sizeof(Tail);

// Byte offset of 16-byte chunk c (0..15) of row r: two 64-element regions of
// 128-byte rows, 128-byte swizzle.
__device__ __forceinline__ uint32_t sw128(int r, int c) {
  return (uint32_t)((c >> 3) * kRegion + (r >> 3) * 1024 + (r & 7) * 128 + (((c & 7) ^ (r & 7)) << 4));
}
__device__ __forceinline__ uint64_t kstep_offset(int k) {
  return (uint64_t)(((k >> 2) * kRegion + (k & 3) * 32) >> 4);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Four codes as bf16 pairs (0, 2) and (1, 3), times `mul` (2^120 and more).
__device__ __forceinline__ void decode4(uint32_t w, uint32_t mul, uint32_t& p02, uint32_t& p13) {
  const uint32_t x = w << 8;
  p02 = mul_bf16x2((x & 0x80008000u) | ((x >> 4) & 0x07f007f0u), mul);
  p13 = mul_bf16x2((w & 0x80008000u) | ((w >> 4) & 0x07f007f0u), mul);
}
// bf16 values d0 .. d3 of two words in the same order.
__device__ __forceinline__ void permute4(uint32_t d01, uint32_t d23, uint32_t& p02, uint32_t& p13) {
  p02 = __byte_perm(d01, d23, 0x5410);
  p13 = __byte_perm(d01, d23, 0x7632);
}
__device__ __forceinline__ bool nonfinite2(uint32_t w) {
  return (w & 0x7fffu) >= 0x7f80u || (w & 0x7fff0000u) >= 0x7f800000u;
}
__device__ __forceinline__ uint32_t finite2(uint32_t w) {  // non-finite halves become 0
  if ((w & 0x7fffu) >= 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7fff0000u) >= 0x7f800000u) w &= 0xffffu;
  return w;
}

__global__ void __launch_bounds__(kThreads, 1)
kv8_attn_tc_kernel(Kv8Attn p, int dual, int ranges) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = smem;
  uint8_t* k_s = q_s + 2 * kTileBytes;
  uint8_t* v_s = k_s + kStages * kTileBytes;
  Tail* tail = reinterpret_cast<Tail*>(v_s + kStages * kTileBytes);
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
  auto lane_blocks = [&](int t) { return dual ? nblocks : (nblocks - t + 1) / 2; };
  auto block_of = [&](int t, int i) { return dual ? i : 2 * i + t; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(&tail->k_full[s], kDecodeWarps * 32);
      ptx::mbar_init(&tail->k_empty[s], 1);
      ptx::mbar_init(&tail->v_full[s], kDecodeWarps * 32);
      ptx::mbar_init(&tail->v_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(&tail->s_full[t], 1);
      ptx::mbar_init(&tail->p_full[t], 128);
    }
    ptx::mbar_init(&tail->q_ready, 256);
    ptx::mbar_init(&tail->mma_done, 1);
    tail->abort_flag = 0;
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

  if (warp == kMmaWarp) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      const uint32_t idesc_s = ptx::idesc_bf16_f32(kBM, kKB);
      const uint32_t idesc_o = ptx::idesc_bf16_f32(kBM, kD) | ptx::kIdescBMajorMN;
      bool ok = nblocks == 0 || ptx::mbar_wait(&tail->q_ready, 0, abort_flag, &g_kv8_tc_status, 41);
      auto issue_s = [&](int t, int i) -> bool {
        const int b = block_of(t, i), s = b % kStages;
        if (!ptx::mbar_wait(&tail->k_full[s], (b / kStages) & 1, abort_flag, &g_kv8_tc_status, 42)) return false;
        ptx::tc_fence_after();
        const uint64_t qdesc = ptx::smem_desc_k_sw128(ptx::smem_u32(q_s + (dual ? t : 0) * kTileBytes));
        const uint64_t kdesc = ptx::smem_desc_k_sw128(ptx::smem_u32(k_s + s * kTileBytes));
#pragma unroll
        for (int k = 0; k < kD / 16; ++k)
          ptx::umma_f16(tmem + t * kBM, qdesc + kstep_offset(k), kdesc + kstep_offset(k), idesc_s, k != 0);
        ptx::umma_commit(&tail->s_full[t]);
        if (!dual || t == nlanes - 1) ptx::umma_commit(&tail->k_empty[s]);
        return true;
      };
      auto issue_o = [&](int t, int i) -> bool {
        const int b = block_of(t, i), s = b % kStages;
        if (!ptx::mbar_wait(&tail->v_full[s], (b / kStages) & 1, abort_flag, &g_kv8_tc_status, 43)) return false;
        if (!ptx::mbar_wait(&tail->p_full[t], i & 1, abort_flag, &g_kv8_tc_status, 44)) return false;
        ptx::tc_fence_after();
        const uint64_t vdesc = ptx::smem_desc_mn_sw128(ptx::smem_u32(v_s + s * kTileBytes), kRegion);
#pragma unroll
        for (int k = 0; k < kKB / 16; ++k)
          ptx::umma_f16_ta(tmem + kOCol + t * kD, tmem + t * kBM + k * 8, vdesc + (uint64_t)((k * 16 * 128) >> 4),
                           idesc_o, i != 0 || k != 0);
        if (!dual || t == nlanes - 1) ptx::umma_commit(&tail->v_empty[s]);
        return true;
      };
      for (int t = 0; ok && t < nlanes; ++t) ok = lane_blocks(t) == 0 || issue_s(t, 0);
      for (int i = 0; ok && i < lane_blocks(0); ++i)
        for (int t = 0; ok && t < nlanes; ++t) {
          if (i >= lane_blocks(t)) continue;
          ok = issue_o(t, i);
          // Over P of block i, which the MMAs just issued read first.
          if (ok && i + 1 < lane_blocks(t)) ok = issue_s(t, i + 1);
        }
      ptx::umma_commit(&tail->mma_done);
      volatile int never = 0;
      ptx::mbar_wait(&tail->mma_done, 0, &never, &g_kv8_tc_status, 45);
    }
  } else if (warp >= kSoftmaxWarps) {
    // ---------------- decoders ----------------
    const int ct = threadIdx.x - kSoftmaxWarps * 32;
    const int row = ct >> 3, part = ct & 7;  // row of 16 in a pass, 16 dims of it
    const int sealed = (int)p.c.sealed;
    const uint8_t* kc = p.c.k + req * p.c.c_bs + kvh * p.c.c_hs + part * 16;
    const uint8_t* vc = p.c.v + req * p.c.c_bs + kvh * p.c.c_hs + part * 16;
    const float* ksc = p.c.ks + req * p.c.s_bs + kvh * p.c.s_hs;
    const float* vsc = p.c.vs + req * p.c.s_bs + kvh * p.c.s_hs;
    const __nv_bfloat16* kt = p.c.kt + req * p.c.t_bs + kvh * p.c.t_hs + part * 16;
    const __nv_bfloat16* vt = p.c.vt + req * p.c.t_bs + kvh * p.c.t_hs + part * 16;
    uint4 kr[8], vr[8];
    float vs[4], ks = 0.f;
    auto load = [&](int b) {
      const int key0 = key_lo + b * kKB;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int key = key0 + u * 16 + row;
        if (key < sealed) kr[u] = __ldg(reinterpret_cast<const uint4*>(kc + (int64_t)key * kD));
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int key = key0 + u * 16 + row;
        if (key < sealed) vr[u] = __ldg(reinterpret_cast<const uint4*>(vc + (int64_t)key * kD));
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) vs[g] = key0 + g * 32 < sealed ? __ldg(vsc + ((key0 + g * 32) >> p.c.block_shift)) : 1.f;
      if (ct < 4) ks = key0 + ct * 32 < sealed ? __ldg(ksc + ((key0 + ct * 32) >> p.c.block_shift)) : 1.f;
    };
    // 16 dims of a row into chunks 2 part and 2 part + 1, the higher dims first
    // for the upper parts: eight lanes then hit different banks.
    const int swap = part >> 2;
    auto store = [&](uint8_t* base, int r, const uint32_t (&w)[8]) {
      const uint4 lo = make_uint4(w[0], w[1], w[2], w[3]), hi = make_uint4(w[4], w[5], w[6], w[7]);
      *reinterpret_cast<uint4*>(base + sw128(r, 2 * part + swap)) = swap ? hi : lo;
      *reinterpret_cast<uint4*>(base + sw128(r, 2 * part + 1 - swap)) = swap ? lo : hi;
    };
    if (nblocks > 0) load(0);
    for (int b = 0; b < nblocks; ++b) {
      const int s = b % kStages, key0 = key_lo + b * kKB;
      const uint32_t ph = (b / kStages) & 1;
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(&tail->k_empty[s], ph ^ 1, abort_flag, &g_kv8_tc_status, 46))) break;
      if (ct < 4) {
        // Ring of four: block b - 4's softmax is over (its K stage was freed twice since).
        const float v = ct == 0 ? vs[0] : (ct == 1 ? vs[1] : (ct == 2 ? vs[2] : vs[3]));
        tail->kf[b & 3][ct] = v != v ? v : ks * p.scale_log2;
      }
      uint8_t* kst = k_s + s * kTileBytes;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int r = u * 16 + row;
        uint32_t w[8];
        if (key0 + u * 16 < sealed) {  // the 16 rows of a pass are all codes or all tail
          const uint32_t in[4] = {kr[u].x, kr[u].y, kr[u].z, kr[u].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) decode4(in[j], 0x7b807b80u, w[2 * j], w[2 * j + 1]);
        } else {
          uint4 a = make_uint4(0, 0, 0, 0), c = a, x = a, y = a;
          if (key0 + r < key_hi) {
            const int64_t at = (int64_t)(key0 + r - sealed) * kD;
            a = *reinterpret_cast<const uint4*>(kt + at);
            c = *reinterpret_cast<const uint4*>(kt + at + 8);
            x = *reinterpret_cast<const uint4*>(vt + at);
            y = *reinterpret_cast<const uint4*>(vt + at + 8);
          }
          int bad = nonfinite2(x.x) | nonfinite2(x.y) | nonfinite2(x.z) | nonfinite2(x.w) | nonfinite2(y.x) |
                    nonfinite2(y.y) | nonfinite2(y.z) | nonfinite2(y.w);
          bad |= __shfl_xor_sync(0xffffffffu, bad, 1);
          bad |= __shfl_xor_sync(0xffffffffu, bad, 2);
          bad |= __shfl_xor_sync(0xffffffffu, bad, 4);
          permute4(a.x, a.y, w[0], w[1]);
          permute4(a.z, a.w, w[2], w[3]);
          permute4(c.x, c.y, w[4], w[5]);
          permute4(c.z, c.w, w[6], w[7]);
          if (bad) w[0] = 0x7fc07fc0u;  // a NaN key: rows that see it answer NaN
        }
        store(kst, r, w);
      }
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(&tail->k_full[s]);
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(&tail->v_empty[s], ph ^ 1, abort_flag, &g_kv8_tc_status, 47))) break;
      uint8_t* vst = v_s + s * kTileBytes;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int r = u * 16 + row;
        uint32_t w[8];
        if (key0 + u * 16 < sealed) {
          const uint32_t in[4] = {vr[u].x, vr[u].y, vr[u].z, vr[u].w};
          const float f = vs[u >> 1];
          const uint32_t e = f != f ? 0u : (__float_as_uint(f) >> 23) + 120u;  // 2^120 * f, biased
          // A NaN scale: its codes are zeros and count as zeros here.
          const uint32_t mul = min(e, 254u) * 0x00800080u;
#pragma unroll
          for (int j = 0; j < 4; ++j) decode4(in[j], mul, w[2 * j], w[2 * j + 1]);
          if (e > 254u) {  // values above 2^16: the rest of the scale in a second product
            const uint32_t more = (127u + e - 254u) * 0x00800080u;
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = mul_bf16x2(w[j], more);
          }
        } else {
          uint4 x = make_uint4(0, 0, 0, 0), y = x;
          if (key0 + r < key_hi) {
            const int64_t at = (int64_t)(key0 + r - sealed) * kD;
            x = *reinterpret_cast<const uint4*>(vt + at);
            y = *reinterpret_cast<const uint4*>(vt + at + 8);
          }
          permute4(finite2(x.x), finite2(x.y), w[0], w[1]);
          permute4(finite2(x.z), finite2(x.w), w[2], w[3]);
          permute4(finite2(y.x), finite2(y.y), w[4], w[5]);
          permute4(finite2(y.z), finite2(y.w), w[6], w[7]);
        }
        store(vst, r, w);
      }
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(&tail->v_full[s]);
      if (b + 1 < nblocks) load(b + 1);
    }
  } else {
    // ---------------- softmax / epilogue: one thread per row ----------------
    const int t = warp >> 2, quad = warp & 3;
    const int r = quad * 32 + lane;
    const int pr = (tile0 + (dual ? t : 0)) * kBM + r;
    const bool rok = pr < packed;
    const bool warp_ok = t < nlanes && pr - lane < packed;  // uniform over the warp
    const int row = rok ? pr % p.q_len : 0;
    const int head = kvh * p.group + (rok ? pr / p.q_len : 0);

    if (dual ? t < nlanes : t == 0) {  // Q row -> shared memory
      const __nv_bfloat16* qrow = p.q + req * p.q_bs + head * p.q_hs + row * p.q_rs;
      uint8_t* qt = q_s + t * kTileBytes;
#pragma unroll 4
      for (int c = 0; c < kD / 8; ++c) {
        const uint4 x = rok ? *reinterpret_cast<const uint4*>(qrow + c * 8) : make_uint4(0, 0, 0, 0);
        uint4 y;
        permute4(x.x, x.y, y.x, y.y);
        permute4(x.z, x.w, y.z, y.w);
        *reinterpret_cast<uint4*>(qt + sw128(r, c)) = y;
      }
      ptx::fence_proxy_async_smem();
    }
    ptx::mbar_arrive(&tail->q_ready);

    const uint32_t scol = tmem + ((uint32_t)(quad * 32) << 16) + t * kBM;
    const uint32_t ocol = tmem + ((uint32_t)(quad * 32) << 16) + kOCol + t * kD;
    const uint32_t* rbits = p.bits ? p.bits + req * p.bits_bs + (int64_t)row * p.words : nullptr;
    const int n = t < nlanes ? lane_blocks(t) : 0;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int b = block_of(t, i), key0 = key_lo + b * kKB;
      const bool full = key0 + kKB <= p.prefix;
      uint64_t win[2] = {~0ull, ~0ull};
      if (!full) {
        win[0] = rok ? kv8_window(p, rbits, key0) : 0ull;
        win[1] = rok ? kv8_window(p, rbits, key0 + 64) : 0ull;
      }
      ok = __all_sync(0xffffffffu, ptx::mbar_wait(&tail->s_full[t], i & 1, abort_flag, &g_kv8_tc_status, 48));
      if (!ok) break;
      ptx::tc_fence_after();
      if (warp_ok) {
        const float4 f4 = *reinterpret_cast<const float4*>(tail->kf[b & 3]);
        const float f[4] = {f4.x, f4.y, f4.z, f4.w};
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t sv[32];
          ptx::tmem_ld_32(scol + c * 32, sv);
          float a = -INFINITY, d = -INFINITY;
          if (full) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              a = fmaxf(a, __uint_as_float(sv[j]));
              d = fmaxf(d, __uint_as_float(sv[j + 1]));
            }
          } else {
            const uint32_t w = (uint32_t)(win[c >> 1] >> ((c & 1) * 32));
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if ((w >> j) & 1u) a = fmaxf(a, __uint_as_float(sv[j]));
          }
          a = fmaxf(a, d);
          mx = fmaxf(mx, a == -INFINITY ? a : a * f[c]);
        }
        if (__any_sync(0xffffffffu, mx > m + kSlack || (m == -INFINITY && mx > -INFINITY))) {
          const float mnew = fmaxf(m, mx);
          const float alpha = m == -INFINITY ? 1.f : ex2(m - mnew);  // nothing summed yet: O and l are 0
          m = mnew;
          l *= alpha;
          if (i > 0) {
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t ov[32];
              ptx::tmem_ld_32(ocol + c * 32, ov);
#pragma unroll
              for (int j = 0; j < 32; ++j) ov[j] = __float_as_uint(__uint_as_float(ov[j]) * alpha);
              ptx::tmem_st_32(ocol + c * 32, ov);
            }
          }
        }
        const float base = m == -INFINITY ? 0.f : m;
        float l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t sv[32], pk[16];
          ptx::tmem_ld_32(scol + c * 32, sv);
          if (full) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float p0 = ex2(fmaf(__uint_as_float(sv[j]), f[c], -base));
              const float p1 = ex2(fmaf(__uint_as_float(sv[j + 1]), f[c], -base));
              l0 += p0;
              l1 += p1;
              pk[j / 2] = pack_bf16x2(p0, p1);
            }
          } else {
            const uint32_t w = (uint32_t)(win[c >> 1] >> ((c & 1) * 32));
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float p0 = (w >> j) & 1u ? ex2(fmaf(__uint_as_float(sv[j]), f[c], -base)) : 0.f;
              const float p1 = (w >> (j + 1)) & 1u ? ex2(fmaf(__uint_as_float(sv[j + 1]), f[c], -base)) : 0.f;
              l0 += p0;
              l1 += p1;
              pk[j / 2] = pack_bf16x2(p0, p1);
            }
          }
          ptx::tmem_st_16(scol + c * 16, pk);  // columns whose scores have been read
        }
        l += l0 + l1;
        ptx::tmem_wait_st();
      }
      ptx::tc_fence_before();
      ptx::mbar_arrive(&tail->p_full[t]);
    }
    // The output rows of this lane.
    const bool mine = dual ? t < nlanes : true;  // one row tile: both lanes write a partial result
    if (ok && mine && n > 0)
      ok = __all_sync(0xffffffffu, ptx::mbar_wait(&tail->mma_done, 0, abort_flag, &g_kv8_tc_status, 49));
    if (ok && mine && pr - lane < packed) {
      ptx::tc_fence_after();
      const bool direct = p.splits == 1;
      const int part = dual ? range : 2 * range + t;
      const int64_t idx = (((int64_t)req * p.splits + part) * p.heads + head) * p.q_len + row;
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t ov[32];
        if (n > 0) {
          ptx::tmem_ld_32(ocol + c * 32, ov);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) ov[j] = 0;
        }
        if (!rok) continue;
        if (direct) {
          __nv_bfloat16* dst = p.out + req * p.out_bs + ((int64_t)row * p.heads + head) * kD + c * 32;
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint4 w;
            w.x = pack_bf16x2(__uint_as_float(ov[j]) * inv, __uint_as_float(ov[j + 2]) * inv);
            w.y = pack_bf16x2(__uint_as_float(ov[j + 1]) * inv, __uint_as_float(ov[j + 3]) * inv);
            w.z = pack_bf16x2(__uint_as_float(ov[j + 4]) * inv, __uint_as_float(ov[j + 6]) * inv);
            w.w = pack_bf16x2(__uint_as_float(ov[j + 5]) * inv, __uint_as_float(ov[j + 7]) * inv);
            *reinterpret_cast<uint4*>(dst + j) = w;
          }
        } else {
          float* dst = p.part_o + idx * kD + c * 32;
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<uint4*>(dst + j) = make_uint4(ov[j], ov[j + 2], ov[j + 1], ov[j + 3]);
        }
      }
      if (rok) {
        if (direct) {
          if (p.lse)
            p.lse[((int64_t)req * p.heads + head) * p.q_len + row] =
                l == 0.f ? -INFINITY : (m == -INFINITY ? l : (m + log2f(l)) * 0.69314718055994531f);
        } else {
          p.part_ml[idx * 2] = m;
          p.part_ml[idx * 2 + 1] = l;
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
  int64_t pairs;  // CTAs over the rows
};
Shape shape_of(int64_t packed) {
  const int64_t tiles = (packed + kBM - 1) / kBM;
  return {tiles > 1, tiles > 1 ? (tiles + 1) / 2 : 1};
}

}  // namespace

bool kv8_use_tc(int head_dim, int64_t packed, int64_t kv_len) { return head_dim == kD && packed >= 48 && kv_len > 0; }

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

int kv8_attention_tc(const Kv8Attn& p, cudaStream_t stream) {
  static std::atomic<unsigned long long> configured{0};
  if (int rc = once_per_device(configured, [] {
        SF_CHECK_CUDA(cudaFuncSetAttribute(kv8_attn_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)kSmemBytes));
        return SF_OK;
      }))
    return rc;
  const Shape sh = shape_of((int64_t)p.group * p.q_len);
  const int ranges = sh.dual ? p.splits : p.splits / 2;
  SF_CHECK_ARG(sh.pairs < 65536 && (int64_t)ranges * p.batch < 65536, "too many query rows or requests");
  const dim3 grid((unsigned)p.c.hkv, (unsigned)sh.pairs, (unsigned)(ranges * p.batch));
  SF_CHECK_CUDA(launch_pdl(kv8_attn_tc_kernel, grid, dim3(kThreads), kSmemBytes, stream, p, sh.dual ? 1 : 0, ranges));
  SF_CHECK_LAUNCH();
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
