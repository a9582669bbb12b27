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
//   * At a block's end the four partial sums of a key are added in one order,
//     so the same inputs give the same bits.
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
constexpr int kThreads = (kSumWarps + 2) * 32;
constexpr int kMmaWarp = kSumWarps, kLoadWarp = kSumWarps + 1;

struct __align__(16) Tail {
  float2 rowc[kQStages][kBM];
  float part[2][4][kKB];  // by block parity: lane and half's sums of a key
  uint64_t q_full[kQStages], q_empty[kQStages];
  uint64_t k_full[kKStages], k_empty[kKStages], lo_full, lo_empty;
  uint64_t d_full[kBufs], d_empty[kBufs];
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
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int site) {
  int ok = 0;
  if ((threadIdx.x & 31) == 0) ok = ptx::mbar_wait(bar, parity, abort_flag, &g_kv8_mass_status, site) ? 1 : 0;
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

__global__ void __launch_bounds__(kThreads, 1)
kv8_mass_tc_kernel(const __grid_constant__ CUtensorMap tm_k, Kv8Attn p, Kv8Prep w, float* __restrict__ mass,
                   int64_t m_bs, int64_t m_hs, int nblocks, int per_cta) {
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
  const bool resident = w.tiles <= kQStages;
  const int sealed = (int)p.c.sealed;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kQStages; ++s) {
      ptx::mbar_init(&tail->q_full[s], 1);
      ptx::mbar_init(&tail->q_empty[s], 1 + kSumWarps / 2);  // the products, and the readers of the row constants
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
        for (int i = 0; ok && i < w.tiles; ++i, ++n) {
          const int s = n % kQStages;
          ok = ptx::mbar_wait(&tail->q_empty[s], ((n / kQStages) & 1) ^ 1, abort_flag, &g_kv8_mass_status, 63);
          if (!ok) break;
          ptx::mbar_arrive_expect_tx(&tail->q_full[s], kTileBytes + (uint32_t)sizeof(tail->rowc[0]));
          ptx::bulk_load(q_s + s * kTileBytes, w.q + ((int64_t)bh * w.tiles + i) * kTileBytes, kTileBytes,
                         &tail->q_full[s]);
          ptx::bulk_load(tail->rowc[s], w.rowc + ((int64_t)bh * w.tiles + i) * kBM, sizeof(tail->rowc[0]),
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
        if (u != u0 && (blk == 0 || !resident)) n0 += w.tiles;
        const bool last = !resident || u + 1 == u1 || blk + 1 == nblocks;  // of these tiles
        const bool mixed = key0 + kKB > sealed;
        const int ks = nk % kKStages;
        ok = ptx::mbar_wait(&tail->k_full[ks], (nk / kKStages) & 1, abort_flag, &g_kv8_mass_status, 65) &&
             (!mixed || ptx::mbar_wait(&tail->lo_full, nlo & 1, abort_flag, &g_kv8_mass_status, 66));
        if (!ok) break;
        const uint64_t khi = ptx::smem_desc_k_sw128(ptx::smem_u32(k_s + ks * kHalf));
        const uint64_t klo = ptx::smem_desc_k_sw128(ptx::smem_u32(lo_s));
        for (int i = 0; ok && i < w.tiles; ++i, ++m) {
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
  } else {
    // ---------------- sums: a key's two threads of lane t ----------------
    const int t = warp >> 3, half = (warp >> 2) & 1, quad = warp & 3;
    const int key_in = quad * 32 + lane;
    const uint32_t col = tmem + ((uint32_t)(quad * 32) << 16) + half * 64;
    const int packed = p.group * p.q_len;
    bool ok = true;
    int n0 = 0, m = 0, parity = 0;
    for (int u = u0; u < u1; ++u, parity ^= 1) {
      const int bh = u / nblocks, blk = u - bh * nblocks, key0 = blk * kKB, key = key0 + key_in;
      const int kvh = bh % p.c.hkv, req = bh / p.c.hkv;
      if (u != u0 && (blk == 0 || !resident)) n0 += w.tiles;
      const bool last = !resident || u + 1 == u1 || blk + 1 == nblocks;
      const bool full = key0 + kKB <= p.prefix;  // no mask to read
      const float kf = key0 + kKB <= sealed
                           ? p.c.ks[req * p.c.s_bs + kvh * p.c.s_hs + (key >> p.c.block_shift)]
                           : w.kf[(int64_t)bh * w.blocks * kKB + (key - w.first)];
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int i = 0; i < w.tiles; ++i, ++m) {
        if ((m & 1) != t) continue;
        const int n = n0 + i, s = n % kQStages, buf = m % kBufs;
        ok = ok && warp_wait(&tail->q_full[s], (n / kQStages) & 1, abort_flag, 70);
        ok = ok && warp_wait(&tail->d_full[buf], (m / kBufs) & 1, abort_flag, 71);
        if (ok) {
          ptx::tc_fence_after();
          const float4* rc = reinterpret_cast<const float4*>(tail->rowc[s] + half * 64);  // two rows each
          const int row0 = i * kBM + half * 64;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float d[16];
            ptx::tmem_ld_16(col + buf * kBM + c * 16, d);
            if (full) {
#pragma unroll
              for (int j = 0; j < 16; j += 2) {
                const float4 r = rc[c * 8 + j / 2];
                acc[j & 2] += ex2(fmaf(d[j], r.x * kf, -r.y));
                acc[(j & 2) + 1] += ex2(fmaf(d[j + 1], r.z * kf, -r.w));
              }
            } else {
              // Visibility of this key for 16 rows, their words loaded together.
              uint32_t word[16];
              const int at = key - p.prefix;
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const int pr = row0 + c * 16 + j;
                const int h = (int)(((uint64_t)pr * p.q_magic) >> 40), row = pr - h * p.q_len;
                word[j] = 0;
                if (pr < packed && key < p.kv_len)
                  word[j] = at < 0 ? ~0u : (p.bits ? p.bits[req * p.bits_bs + (int64_t)row * p.words + (at >> 5)] : 0u);
              }
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float2 r = tail->rowc[s][half * 64 + c * 16 + j];
                if ((word[j] >> (at & 31)) & 1u) acc[j & 3] += ex2(fmaf(d[j], r.x * kf, -r.y));
              }
            }
          }
          ptx::tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(&tail->d_empty[buf]);
          // The lane that summed a tile's last block is the last reader of its constants.
          if (last) ptx::mbar_arrive(&tail->q_empty[s]);
        }
      }
      tail->part[parity][t * 2 + half][key_in] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
      ptx::named_bar_sync(1, kSumWarps * 32);
      if (warp < 4 && ok && key < p.kv_len) {  // t = 0, half = 0: this thread's key
        const float* x = tail->part[parity][0];
        mass[req * m_bs + kvh * m_hs + key] += (x[key_in] + x[kKB + key_in]) + (x[2 * kKB + key_in] + x[3 * kKB + key_in]);
      }
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

}  // namespace

bool kv8_mass_use_tc(int head_dim, int64_t packed) { return head_dim == kD && packed >= 96; }

int kv8_mass_tc(const Kv8Attn& p, float* mass, int64_t m_bs, int64_t m_hs, void* prep, cudaStream_t stream) {
  static std::atomic<unsigned long long> configured{0};
  if (int rc = once_per_device(configured, [] {
        SF_CHECK_CUDA(cudaFuncSetAttribute(kv8_mass_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)kSmemBytes));
        return SF_OK;
      }))
    return rc;
  const int64_t heads = (int64_t)p.batch * p.c.hkv, nblocks = ((int64_t)p.kv_len + kKB - 1) / kKB;
  SF_CHECK_ARG(heads * nblocks < (1 << 30), "too many keys for one call");
  Kv8Prep w;
  kv8_prep_layout(&w, prep, true, heads, (int64_t)p.group * p.q_len, p.c.sealed, p.kv_len);
  if (int rc = kv8_prep(p, w, stream)) return rc;
  CUtensorMap tm_k;
  if (int rc = kv8_key_map(&tm_k, p.c, p.batch)) return rc;
  const int64_t units = heads * nblocks, per = (units + num_sms() - 1) / num_sms();
  SF_CHECK_CUDA(launch_pdl(kv8_mass_tc_kernel, dim3((unsigned)((units + per - 1) / per)), dim3(kThreads), kSmemBytes,
                           stream, tm_k, p, w, mass, m_bs, m_hs, (int)nblocks, (int)per));
  SF_CHECK_LAUNCH();
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
