// The attention weight that each cached token received (kv8_mass.cu), on
// tcgen05, for passes with many query rows; head_dim 128.
//
//   mass[j] += sum_r 2^(kf_j * qf_r * (k_j . q_r) - lse_r)
//
// The floor is the exponentials, one per (row, key), 16 a clock and SM; the
// products take half of that (both on the fp8 rate: a query is the sum of two
// e4m3 numbers, kv8_attn_tc.cu has why).  With the keys as the MMA's rows a
// thread owns one key: the sum over the query rows stays in its registers.
//   * A CTA walks blocks of 128 keys, all blocks of all heads dealt out in
//     order; for each it takes the head's query tiles (images laid out by
//     kv8_prep_kernel) one after the other.  Up to five tiles stay in shared
//     memory while the head stays the same (a 65-row tree has five).
//   * D[128 keys x 128 rows] goes to one of four TMEM buffers; two lanes of
//     eight warps take them in turn, two threads a key, 64 rows each.
//   * A cache too short for all SMs: the query tiles are dealt out in parts, whose
//     sums a second kernel adds to the mass, again in one order.
//   * At a block's end one warp adds the four partial sums of a key, in one
//     order, so the same inputs give the same bits.
// What it measured: 8 requests of 65 rows, 32 heads, over 4,161 tokens 46 us (the
// warp-level kernel 265), 2.3 times the exponentials' 20; a CTA's last block, the
// one with a mask, takes twice a full one's time.
// Every wait is bounded; a warp whose wait gave up skips the work but still
// meets the others at the barriers.
#include <cuda.h>
#include <math.h>

#include <algorithm>

#include "kv8_attn.h"
#include "sm100_ptx.cuh"

namespace sf {
namespace {

__device__ int g_kv8_mass_status;

constexpr int kD = 128;
constexpr int kKB = 128;              // keys of a block (MMA M)
constexpr int kBM = 128;              // query rows of a tile (MMA N)
constexpr int kHalf = 128 * 128;      // one e4m3 tile (bytes)
constexpr int kTileBytes = 2 * kHalf; // hi and lo
constexpr int kQStages = 5;
constexpr int kKStages = 2;
constexpr int kBufs = 4;              // of D
constexpr int kSumWarps = 16;
constexpr int kThreads = (kSumWarps + 3) * 32;
constexpr int kMmaWarp = kSumWarps, kLoadWarp = kSumWarps + 1, kAddWarp = kSumWarps + 2;

struct __align__(16) Tail {
  float rowc[kQStages][2][kBM];
  float part[2][4][kKB];  // by block parity: a key's sums, by lane and half of a tile's rows
  uint64_t q_full[kQStages], q_empty[kQStages];
  uint64_t k_full[kKStages], k_empty[kKStages], lo_full, lo_empty;
  uint64_t d_full[kBufs], d_empty[kBufs];
  uint64_t part_full[2], part_empty[2];
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort_flag;
};

constexpr size_t kSmemBytes = 1024 + kQStages * kTileBytes + (kKStages + 1) * kHalf + sizeof(Tail);

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__global__ void __launch_bounds__(kThreads, 1)
kv8_mass_tc_kernel(const __grid_constant__ CUtensorMap tm_k, Kv8Attn p, Kv8Prep w, float* __restrict__ mass,
                   int64_t m_bs, int64_t m_hs, int nblocks, int per_cta, int tiles_part, float* __restrict__ parts) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = smem;
  uint8_t* k_s = q_s + kQStages * kTileBytes;
  uint8_t* lo_s = k_s + kKStages * kHalf;  // the lower part of a block with tail keys
  Tail* tail = reinterpret_cast<Tail*>(lo_s + kHalf);
  volatile int* abort_flag = &tail->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = p.batch * p.c.hkv * nblocks;  // (head, block), the head first
  const int u0 = min(units, (int)blockIdx.x * per_cta), u1 = min(units, u0 + per_cta);
  // This CTA's query tiles: all of them, or one part (then its sums go to `parts`).
  const int t0 = blockIdx.y * tiles_part, tiles = min(tiles_part, w.tiles - t0);
  const bool resident = tiles <= kQStages;
  const int sealed = (int)p.c.sealed;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kQStages; ++s) {
      ptx::mbar_init(&tail->q_full[s], 1);
      ptx::mbar_init(&tail->q_empty[s], 1 + kSumWarps);  // the products, and the readers of the row constants
    }
    for (int s = 0; s < kKStages; ++s) {
      ptx::mbar_init(&tail->k_full[s], 1);
      ptx::mbar_init(&tail->k_empty[s], 1);
    }
    ptx::mbar_init(&tail->lo_full, 1);
    ptx::mbar_init(&tail->lo_empty, 1);
    for (int s = 0; s < kBufs; ++s) {
      ptx::mbar_init(&tail->d_full[s], 1);
      ptx::mbar_init(&tail->d_empty[s], kSumWarps / 2);
    }
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(&tail->part_full[s], kSumWarps);
      ptx::mbar_init(&tail->part_empty[s], 1);
    }
    ptx::mbar_init(&tail->mma_done, 1);
    tail->abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(&tail->tmem_base, 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = tail->tmem_base;

  // The query tiles are loaded per head where they all fit, else per block: the
  // n-th load of the CTA goes to stage n % kQStages.  A stage is free again once
  // its last product and its last reader are done.
  if (warp == kLoadWarp) {
    if (lane == 0) {
      bool ok = true;
      int n = 0, nk = 0, nlo = 0;
      for (int u = u0; ok && u < u1; ++u) {
        const int bh = u / nblocks, blk = u - bh * nblocks, key0 = blk * kKB;
        const int kvh = bh % p.c.hkv, req = bh / p.c.hkv;
        const int ks = nk % kKStages;
        ok = ptx::mbar_wait(&tail->k_empty[ks], ((nk / kKStages) & 1) ^ 1, abort_flag, &g_kv8_mass_status, 61);
        if (!ok) break;
        ptx::mbar_arrive_expect_tx(&tail->k_full[ks], kHalf);
        ++nk;
        if (key0 + kKB <= sealed) {
          ptx::tma_load_4d(k_s + ks * kHalf, &tm_k, &tail->k_full[ks], 0, key0, kvh, req);
        } else {
          const uint8_t* img = w.k + ((int64_t)bh * w.blocks + (key0 - w.first) / kKB) * kTileBytes;
          ptx::bulk_load(k_s + ks * kHalf, img, kHalf, &tail->k_full[ks]);
          ok = ptx::mbar_wait(&tail->lo_empty, (nlo & 1) ^ 1, abort_flag, &g_kv8_mass_status, 62);
          if (!ok) break;
          ptx::mbar_arrive_expect_tx(&tail->lo_full, kHalf);
          ptx::bulk_load(lo_s, img + kHalf, kHalf, &tail->lo_full);
          ++nlo;
        }
        if (resident && u != u0 && blk != 0) continue;  // the head's tiles are here
        for (int i = 0; ok && i < tiles; ++i, ++n) {
          const int s = n % kQStages;
          const int64_t at = (int64_t)bh * w.tiles + t0 + i;
          ok = ptx::mbar_wait(&tail->q_empty[s], ((n / kQStages) & 1) ^ 1, abort_flag, &g_kv8_mass_status, 63);
          if (!ok) break;
          ptx::mbar_arrive_expect_tx(&tail->q_full[s], kTileBytes + (uint32_t)sizeof(tail->rowc[0]));
          ptx::bulk_load(q_s + s * kTileBytes, w.q + at * kTileBytes, kTileBytes,
                         &tail->q_full[s]);
          ptx::bulk_load(tail->rowc[s], w.rowc + at * 2 * kBM, sizeof(tail->rowc[0]),
                         &tail->q_full[s]);
        }
      }
      if (!ok) {  // let the copies in flight land before the CTA ends
        volatile int never = 0;
        for (int i = max(0, n - kQStages); i < n; ++i)
          ptx::mbar_wait(&tail->q_full[i % kQStages], (i / kQStages) & 1, &never, &g_kv8_mass_status, 64);
        for (int i = max(0, nk - kKStages); i < nk; ++i)
          ptx::mbar_wait(&tail->k_full[i % kKStages], (i / kKStages) & 1, &never, &g_kv8_mass_status, 64);
        if (nlo > 0) ptx::mbar_wait(&tail->lo_full, (nlo - 1) & 1, &never, &g_kv8_mass_status, 64);
      }
    }
  } else if (warp == kMmaWarp) {
    if (lane == 0) {
      const uint32_t idesc = ptx::idesc_e4m3_f32(kKB, kBM);
      constexpr uint64_t kLo = kHalf >> 4, kStep = 32 >> 4;
      bool ok = true;
      int n0 = 0, nk = 0, nlo = 0, m = 0;  // n0: the load number of this block's first tile
      for (int u = u0; ok && u < u1; ++u, ++nk) {
        const int blk = u % nblocks, key0 = blk * kKB;
        if (u != u0 && (blk == 0 || !resident)) n0 += tiles;
        const bool last = !resident || u + 1 == u1 || blk + 1 == nblocks;  // of these tiles
        const bool mixed = key0 + kKB > sealed;
        const int ks = nk % kKStages;
        ok = ptx::mbar_wait(&tail->k_full[ks], (nk / kKStages) & 1, abort_flag, &g_kv8_mass_status, 65) &&
             (!mixed || ptx::mbar_wait(&tail->lo_full, nlo & 1, abort_flag, &g_kv8_mass_status, 66));
        if (!ok) break;
        const uint64_t khi = ptx::smem_desc_k_sw128(ptx::smem_u32(k_s + ks * kHalf));
        const uint64_t klo = ptx::smem_desc_k_sw128(ptx::smem_u32(lo_s));
        for (int i = 0; ok && i < tiles; ++i, ++m) {
          const int n = n0 + i, s = n % kQStages, buf = m % kBufs;
          ok = ptx::mbar_wait(&tail->q_full[s], (n / kQStages) & 1, abort_flag, &g_kv8_mass_status, 67) &&
               ptx::mbar_wait(&tail->d_empty[buf], ((m / kBufs) & 1) ^ 1, abort_flag, &g_kv8_mass_status, 68);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint64_t q = ptx::smem_desc_k_sw128(ptx::smem_u32(q_s + s * kTileBytes));
#pragma unroll 1
          for (int x = 0; x < (mixed ? 4 : 2); ++x) {  // hi and lo of Q with K, then with K's lower part
            const uint64_t kd = x >> 1 ? klo : khi, qd = q + (x & 1) * kLo;
#pragma unroll
            for (int k = 0; k < kD / 32; ++k)
              ptx::umma_f8(tmem + buf * kBM, kd + k * kStep, qd + k * kStep, idesc, x != 0 || k != 0);
          }
          ptx::umma_commit(&tail->d_full[buf]);
          if (last) ptx::umma_commit(&tail->q_empty[s]);
        }
        if (!ok) break;
        ptx::umma_commit(&tail->k_empty[ks]);
        if (mixed) {
          ptx::umma_commit(&tail->lo_empty);
          ++nlo;
        }
      }
      ptx::umma_commit(&tail->mma_done);
      volatile int never = 0;
      ptx::mbar_wait(&tail->mma_done, 0, &never, &g_kv8_mass_status, 69);
    }
  } else if (warp == kAddWarp) {
    // ---------------- adds a block's sums to the mass, four keys a lane ----------------
    bool ok = true;
    for (int u = u0; u < u1; ++u) {
      const int bh = u / nblocks, key = (u - bh * nblocks) * kKB + lane, nu = u - u0;
      const int kvh = bh % p.c.hkv, req = bh / p.c.hkv;
      float* const to = parts ? parts + ((int64_t)blockIdx.y * p.batch * p.c.hkv + bh) * p.kv_len + key
                              : mass + req * m_bs + kvh * m_hs + key;
      float before[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) before[j] = !parts && key + j * 32 < p.kv_len ? to[j * 32] : 0.f;
      ok = ok && ptx::mbar_wait(&tail->part_full[nu & 1], (nu >> 1) & 1, abort_flag, &g_kv8_mass_status, 73);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const float(*x)[kKB] = tail->part[nu & 1];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = lane + j * 32;
        if (key + j * 32 < p.kv_len) to[j * 32] = before[j] + ((x[0][at] + x[1][at]) + (x[2][at] + x[3][at]));
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&tail->part_empty[nu & 1]);
    }
  } else {
    // ---------------- sums: lane t takes every other tile, two threads a key, 64 rows each ----------------
    const int t = warp >> 3, half = (warp >> 2) & 1, quad = warp & 3;
    const int key_in = quad * 32 + lane;
    const uint32_t col = tmem + ((uint32_t)(quad * 32) << 16) + half * 64;
    const int packed = p.group * p.q_len;
    bool ok = true;
    int m = 0, s0 = 0, qphase = 0;  // stage and phase of this block's first tile
    // The key's scale is loaded a block ahead.
    auto key_scale = [&](int u) {
      const int bh = u / nblocks, key = (u - bh * nblocks) * kKB + key_in;
      const int kvh = bh % p.c.hkv, req = bh / p.c.hkv;
      return (key - key_in) + kKB <= sealed ? p.c.ks[req * p.c.s_bs + kvh * p.c.s_hs + (key >> p.c.block_shift)]
                                            : w.kf[(int64_t)bh * w.blocks * kKB + (key - w.first)];
    };
    float next_kf = u0 < u1 ? key_scale(u0) : 0.f;
    for (int u = u0; u < u1; ++u) {
      const int bh = u / nblocks, blk = u - bh * nblocks, key0 = blk * kKB;
      const bool fresh = u == u0 || blk == 0 || !resident;  // tiles not seen yet
      const bool last = !resident || u + 1 == u1 || blk + 1 == nblocks;
      const bool full = key0 + kKB <= p.prefix;  // no mask to read
      const float kf = next_kf;
      if (u + 1 < u1) next_kf = key_scale(u + 1);
      const uint64_t kf2 = ptx::pack2(kf, kf);
      uint64_t acc[2] = {0, 0};
      int s = s0, phase = qphase;
      for (int i = 0; i < tiles; ++i, ++m) {
        if ((m & 1) == t) {
          const int buf = m % kBufs, row0 = (t0 + i) * kBM + half * 64;
          uint32_t seen[2] = {0, 0};  // rows row0 + lane and 32 on: which of the warp's keys they see
          if (!full) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int pr = row0 + x * 32 + lane;
              const int h = (int)(((uint64_t)pr * p.q_magic) >> 40), row = pr - h * p.q_len, req = bh / p.c.hkv;
              if (pr < packed)
                seen[x] = (uint32_t)kv8_window(
                    p, p.bits ? p.bits + req * p.bits_bs + (int64_t)row * p.words : nullptr, key0 + quad * 32);
            }
          }
          if (fresh) ok = ok && ptx::mbar_wait(&tail->q_full[s], phase, abort_flag, &g_kv8_mass_status, 70);
          ok = ok && ptx::mbar_wait(&tail->d_full[buf], (m / kBufs) & 1, abort_flag, &g_kv8_mass_status, 71);
          ok = __all_sync(0xffffffffu, ok);
          if (ok) {
            ptx::tc_fence_after();
            uint32_t d[2][16];
            const int rows = packed - row0;  // the last tile's are fewer
            ptx::tmem_ld_16_async(col + buf * kBM, d[0]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t(&dc)[16] = d[c & 1];
              ptx::tmem_wait_ld_16(dc);
              if (c * 16 >= rows) break;
              if (c < 3) ptx::tmem_ld_16_async(col + buf * kBM + (c + 1) * 16, d[(c + 1) & 1]);
              const float* f = tail->rowc[s][0] + half * 64 + c * 16;
              const float* l = tail->rowc[s][1] + half * 64 + c * 16;
              if (full) {
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                  const ulonglong2 ff = *reinterpret_cast<const ulonglong2*>(f + j);
                  const ulonglong2 ll = *reinterpret_cast<const ulonglong2*>(l + j);
                  const uint64_t y[2] = {ptx::fma2(ptx::pack2(__uint_as_float(dc[j]), __uint_as_float(dc[j + 1])),
                                                   ptx::mul2(ff.x, kf2), ll.x),
                                         ptx::fma2(ptx::pack2(__uint_as_float(dc[j + 2]), __uint_as_float(dc[j + 3])),
                                                   ptx::mul2(ff.y, kf2), ll.y)};
#pragma unroll
                  for (int x = 0; x < 2; ++x) {
                    float y0, y1;
                    ptx::unpack2(y[x], y0, y1);
                    acc[x] = ptx::add2(acc[x], ptx::pack2(ex2(y0), ex2(y1)));
                  }
                }
              } else {
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                  const float2 ff = *reinterpret_cast<const float2*>(f + j);
                  const float2 ll = *reinterpret_cast<const float2*>(l + j);
                  const uint32_t w0 = __shfl_sync(0xffffffffu, seen[c >> 1], (c & 1) * 16 + j);
                  const uint32_t w1 = __shfl_sync(0xffffffffu, seen[c >> 1], (c & 1) * 16 + j + 1);
                  const float y0 = fmaf(__uint_as_float(dc[j]), ff.x * kf, ll.x);
                  const float y1 = fmaf(__uint_as_float(dc[j + 1]), ff.y * kf, ll.y);
                  acc[(j >> 1) & 1] = ptx::add2(acc[(j >> 1) & 1], ptx::pack2((w0 >> lane) & 1u ? ex2(y0) : 0.f,
                                                                             (w1 >> lane) & 1u ? ex2(y1) : 0.f));
                }
              }
            }
            ptx::tc_fence_before();
            __syncwarp();
          }
          if (lane == 0) ptx::mbar_arrive(&tail->d_empty[buf]);
        }
        // Both lanes have then read this tile's row constants for the last time.
        if (last && lane == 0) ptx::mbar_arrive(&tail->q_empty[s]);
        if (++s == kQStages) s = 0, phase ^= 1;
      }
      if (last) s0 = s, qphase = phase;
      float a[4];
      ptx::unpack2(acc[0], a[0], a[1]);
      ptx::unpack2(acc[1], a[2], a[3]);
      const int nu = u - u0;
      ok = ok && ptx::mbar_wait(&tail->part_empty[nu & 1], ((nu >> 1) & 1) ^ 1, abort_flag, &g_kv8_mass_status, 72);
      tail->part[nu & 1][t * 2 + half][key_in] = (a[0] + a[1]) + (a[2] + a[3]);
      __syncwarp();
      ok = __all_sync(0xffffffffu, ok);
      if (lane == 0) ptx::mbar_arrive(&tail->part_full[nu & 1]);
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// mass += the parts' sums, in order.  grid: (keys, batch * hkv).
__global__ void __launch_bounds__(256)
kv8_mass_add_kernel(const float* __restrict__ parts, int count, float* __restrict__ mass, int64_t m_bs, int64_t m_hs,
                    int hkv, int kv_len) {
  pdl_wait();
  pdl_trigger();
  const int bh = blockIdx.y, key = blockIdx.x * 256 + threadIdx.x;
  if (key >= kv_len) return;
  float sum = 0.f;
#pragma unroll 8
  for (int i = 0; i < count; ++i) sum += parts[((int64_t)i * gridDim.y + bh) * kv_len + key];
  mass[(bh / hkv) * m_bs + (bh % hkv) * m_hs + key] += sum;
}

// A short cache has few blocks: its query tiles are then dealt out too, in
// parts of at least two, so that no SM is idle (four heads, 641 tokens, 321 rows:
// 19 us instead of 44; one part where the blocks fill the SMs).
struct Parts {
  int tiles, count;  // of a part; parts
};
Parts parts_of(int64_t units, int64_t tiles) {
  const int64_t want = std::min<int64_t>(std::max<int64_t>(1, num_sms() / units), std::max<int64_t>(1, tiles / 2));
  const int64_t per = (tiles + want - 1) / want;
  return {(int)per, (int)((tiles + per - 1) / per)};
}
int64_t blocks_of(int64_t kv_len) { return (kv_len + kKB - 1) / kKB; }

}  // namespace

// Microseconds a call, this kernel's against the warp-level one's, four KV heads
// (4,159 tokens; 32,831; eight requests of 4,159):
//   48 packed rows: 10 / 18 / 20 against 9 / 18 / 22
//   64:             11 / 19 / 20 against 10 / 20 / 25
//   96:             11 / 19 / 21 against 14 / 46 / 55
bool kv8_mass_use_tc(int head_dim, int64_t packed) { return head_dim == kD && packed >= 64; }

size_t kv8_mass_tc_bytes(int64_t heads, int64_t packed, int64_t sealed, int64_t kv_len) {
  Kv8Prep w;
  const size_t prep = kv8_prep_layout(&w, nullptr, true, heads, packed, sealed, kv_len);
  const Parts parts = parts_of(heads * blocks_of(kv_len), w.tiles);
  return prep + (parts.count > 1 ? (size_t)parts.count * heads * kv_len * sizeof(float) : 0);
}

int kv8_mass_tc(const Kv8Attn& p, float* mass, int64_t m_bs, int64_t m_hs, void* prep, cudaStream_t stream) {
  static std::atomic<unsigned long long> configured{0};
  if (int rc = once_per_device(configured, [] {
        SF_CHECK_CUDA(cudaFuncSetAttribute(kv8_mass_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)kSmemBytes));
        return SF_OK;
      }))
    return rc;
  const int64_t heads = (int64_t)p.batch * p.c.hkv, nblocks = blocks_of(p.kv_len);
  SF_CHECK_ARG(heads * nblocks < (1 << 30), "too many keys for one call");
  Kv8Prep w;
  const size_t used = kv8_prep_layout(&w, prep, true, heads, (int64_t)p.group * p.q_len, p.c.sealed, p.kv_len);
  const Parts parts = parts_of(heads * nblocks, w.tiles);
  float* sums = parts.count > 1 ? reinterpret_cast<float*>(static_cast<uint8_t*>(prep) + used) : nullptr;
  if (int rc = kv8_prep(p, w, stream)) return rc;
  CUtensorMap tm_k;
  if (int rc = kv8_key_map(&tm_k, p.c, p.batch)) return rc;
  const int64_t units = heads * nblocks, per = (units + num_sms() - 1) / num_sms();
  SF_CHECK_CUDA(launch_pdl(kv8_mass_tc_kernel, dim3((unsigned)((units + per - 1) / per), (unsigned)parts.count),
                           dim3(kThreads), kSmemBytes, stream, tm_k, p, w, mass, m_bs, m_hs, (int)nblocks, (int)per,
                           parts.tiles, sums));
  SF_CHECK_LAUNCH();
  ++kv8_launches();
  if (sums) {
    SF_CHECK_CUDA(launch_pdl(kv8_mass_add_kernel, dim3((unsigned)((p.kv_len + 255) / 256), (unsigned)heads), dim3(256),
                             0, stream, static_cast<const float*>(sums), parts.count, mass, m_bs, m_hs, p.c.hkv,
                             p.kv_len));
    SF_CHECK_LAUNCH();
    ++kv8_launches();
  }
  return SF_OK;
}

int kv8_mass_tc_status(int* status, int reset) {
  SF_CHECK_CUDA(cudaMemcpyFromSymbol(status, g_kv8_mass_status, sizeof(int)));
  if (reset) {
    const int zero = 0;
    SF_CHECK_CUDA(cudaMemcpyToSymbol(g_kv8_mass_status, &zero, sizeof(int)));
  }
  return SF_OK;
}

}  // namespace sf
