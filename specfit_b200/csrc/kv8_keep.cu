// Which cached tokens stay: per request and KV head the first `sinks`, the
// last `recent`, and of those between the `budget - sinks - recent` that
// received the most attention weight, as ascending indices.  Among equal
// weights the earlier token stays; a NaN counts as the least weight.
//
// A radix selection, not a sort: the weights are mapped to integers of the
// same order, three 11-bit histogram passes find the smallest kept key and how
// many of its equals are kept, and one ordered pass writes the indices.  The
// floor is one read of the weights (4 bytes a token), which for the sizes in
// use (512 KB a head at 131,072 tokens) is below launch latency: what bounds
// the kernel is the chain of passes, so a cluster of up to eight CTAs shares
// a head, each with its own slice (in registers up to 8,192 tokens, so that
// up to 65,536 tokens of a head are read once) and adds its peers' histograms
// through distributed shared memory.  Tokens that no row looked at are many,
// and their zeros would all hit one counter: a warp adds them at once.
// Integer counts only, so the result does not depend on the order of the
// atomics.  (Four 8-bit passes over memory, with every digit matched across
// the warp, took 40 us for 16 heads of 65,557 tokens; this takes 29 us, 32 with one
// histogram and a second barrier of the cluster in each pass.)
#include <cooperative_groups.h>

#include "kv8.cuh"

namespace sf {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kPer = 4;  // consecutive weights of one thread in a tile
constexpr int kTile = kThreads * kPer;
constexpr int kHeld = 4;  // tiles that a CTA holds in registers
constexpr int kBits = 11, kBins = 1 << kBits, kPasses = 3;  // 11 + 11 + 10 bits
constexpr int kBinsPer = kBins / kThreads;

struct KeepParams {
  const float* mass;
  int64_t m_bs, m_hs;
  int hkv;
  int length, budget, sinks, recent;
  int slice;  // middle tokens of one CTA, a multiple of kTile
  int32_t* keep;
};

// Larger float, larger key; -0 equals +0; NaN below everything.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ int warp_sum_i(int v) { return (int)__reduce_add_sync(0xffffffffu, (unsigned)v); }

// Held: the CTA's slice is at most kHeld tiles and stays in registers.
// Two CTAs fit an SM, so that sixteen clusters of eight run at once: one at a
// time, a GPC of fewer than 16 SMs holds only one, and the rest wait for it.
template <bool Held>
__global__ void __launch_bounds__(kThreads, 2)
kv_keep_kernel(KeepParams p) {
  pdl_wait();
  pdl_trigger();
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  __shared__ __align__(16) uint32_t hists[2][kBins];  // by pass parity: one is cleared while peers read the other
  __shared__ uint32_t warp_sums[kWarps];
  __shared__ uint32_t prefix_s, want_s;
  __shared__ int counts[2];                 // this CTA's kept-above and equal counts
  __shared__ uint32_t scan[kHeld][kWarps];  // kept-above | equal << 16 of a tile's warps, then of what is before them
  const int head = blockIdx.y;  // b * hkv + h
  const int b = head / p.hkv, h = head % p.hkv;
  const int mid = p.length - p.sinks - p.recent;
  const int want0 = p.budget - p.sinks - p.recent;
  const float* m = p.mass + b * p.m_bs + h * p.m_hs + p.sinks;
  int32_t* out = p.keep + (int64_t)head * p.budget;
  const int lo = min(mid, rank * p.slice), hi = min(mid, lo + p.slice);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  // The always-kept ends.
  for (int i = rank * kThreads + tid; i < p.sinks; i += ranks * kThreads) out[i] = i;
  for (int i = rank * kThreads + tid; i < p.recent; i += ranks * kThreads)
    out[p.budget - p.recent + i] = p.length - p.recent + i;
  if (want0 == 0) return;  // the whole cluster

  // This thread's keys of tile t: tokens base + tid * kPer + {0 .. kPer - 1}.
  const int tiles = (hi - lo + kTile - 1) / kTile;
  uint32_t held[kHeld][kPer];
  auto load = [&](int t, uint32_t (&key)[kPer]) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = lo + t * kTile + tid * kPer + j;
      key[j] = i < hi ? order_key(m[i]) : 0u;
    }
  };
  if constexpr (Held) {
#pragma unroll
    for (int t = 0; t < kHeld; ++t) load(t, held[t]);
  }
  // f(tile, keys) over the tiles in order; past the slice's end keys are no token's.
  auto each_tile = [&](auto&& f) {
    if constexpr (Held) {
#pragma unroll
      for (int t = 0; t < kHeld; ++t)
        if (t < tiles) f(t, held[t]);
    } else {
      for (int t = 0; t < tiles; ++t) {
        uint32_t key[kPer];
        load(t, key);
        f(t, key);
      }
    }
  };
  constexpr uint32_t kZero = 0x80000000u;  // the key of +0

  // The most significant digit first: `prefix` is the digits found so far,
  // `want` how many keys that match it are still to be kept.
  uint32_t prefix = 0, want = (uint32_t)want0;
  static_assert(kBinsPer == 4, "four bins a thread");
  *reinterpret_cast<uint4*>(&hists[0][tid * kBinsPer]) = make_uint4(0, 0, 0, 0);
  __syncthreads();
#pragma unroll 1
  for (int pass = 0; pass < kPasses; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const uint32_t bins_mask = pass == 2 ? 1023u : 2047u;
    const uint32_t mask = pass == 0 ? 0u : (pass == 1 ? 0xffe00000u : 0xfffffc00u);
    uint32_t* const hist = hists[pass & 1];
    each_tile([&](int t, uint32_t (&key)[kPer]) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const bool in = lo + t * kTile + tid * kPer + j < hi && (key[j] & mask) == prefix;
        const uint32_t zeros = __ballot_sync(0xffffffffu, in && key[j] == kZero);
        if (in && key[j] != kZero) atomicAdd(&hist[(key[j] >> shift) & bins_mask], 1u);
        if (lane == 0 && zeros) atomicAdd(&hist[(kZero >> shift) & bins_mask], (uint32_t)__popc(zeros));
      }
    });
    cluster.sync();  // also: the pass before has been read by every peer
    *reinterpret_cast<uint4*>(&hists[(pass & 1) ^ 1][tid * kBinsPer]) = make_uint4(0, 0, 0, 0);
    // Thread t: the four bins whose rank from the top is 4 t .. 4 t + 3.
    const int bin0 = kBins - kBinsPer * (tid + 1);
    uint4 total = make_uint4(0, 0, 0, 0);
    uint4 part[kMaxCluster];
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r)  // all of them in flight together
      part[r] = r < ranks ? *reinterpret_cast<const uint4*>(cluster.map_shared_rank(hist, r) + bin0)
                          : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      const uint4 x = part[r];
      total.x += x.x;
      total.y += x.y;
      total.z += x.z;
      total.w += x.w;
    }
    const uint32_t mine[4] = {total.w, total.z, total.y, total.x};  // from the top
    uint32_t sum = mine[0] + mine[1] + mine[2] + mine[3], before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += up;
    }
    if (lane == 31) warp_sums[warp] = before;
    __syncthreads();
    before -= sum;
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      if (w < warp) before += warp_sums[w];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (before < want && want <= before + mine[j]) {  // one thread of the CTA
        prefix_s = prefix | ((uint32_t)(bin0 + 3 - j) << shift);
        want_s = want - before;
      }
      before += mine[j];
    }
    __syncthreads();  // the digit may be read, the other histogram is clear
    prefix = prefix_s;
    want = want_s;
  }

  // Now `prefix` is the smallest kept key and the first `want` of its equals stay.
  int gt = 0, eq = 0;
  each_tile([&](int t, uint32_t (&key)[kPer]) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const bool in = lo + t * kTile + tid * kPer + j < hi;
      gt += in && key[j] > prefix;
      eq += in && key[j] == prefix;
    }
  });
  gt = warp_sum_i(gt);
  eq = warp_sum_i(eq);
  if (tid < 2) counts[tid] = 0;
  __syncthreads();
  if (lane == 0) {
    atomicAdd(&counts[0], gt);
    atomicAdd(&counts[1], eq);
  }
  cluster.sync();
  int gt0 = 0, eq0 = 0;  // kept-above and equal tokens in the slices before this one
  for (int r = 0; r < rank; ++r) {
    const int* c = cluster.map_shared_rank(counts, r);
    gt0 += c[0];
    eq0 += c[1];
  }
  // Ordered: where a thread's tokens of a tile go depends on how many kept-above
  // and equal ones are before them; both counts of a tile fit 16 bits.
  const int limit = (int)want;
  auto count = [&](int t, const uint32_t (&key)[kPer]) {
    uint32_t c = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const bool in = lo + t * kTile + tid * kPer + j < hi;
      c += (in && key[j] > prefix ? 1u : 0u) + (in && key[j] == prefix ? 0x10000u : 0u);
    }
    return c;
  };
  auto warp_scan = [&](uint32_t c) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, c, o);
      if (lane >= o) c += up;
    }
    return c;
  };
  auto write = [&](int t, const uint32_t (&key)[kPer], int gb, int eb) {
    const int base = lo + t * kTile + tid * kPer;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (base + j >= hi) break;
      if (key[j] > prefix) {
        out[p.sinks + gb + min(eb, limit)] = p.sinks + base + j;
        ++gb;
      } else if (key[j] == prefix) {
        if (eb < limit) out[p.sinks + gb + eb] = p.sinks + base + j;
        ++eb;
      }
    }
  };
  if constexpr (Held) {
    uint32_t before[kHeld];
#pragma unroll
    for (int t = 0; t < kHeld; ++t) {
      const uint32_t c = count(t, held[t]), incl = warp_scan(c);
      before[t] = incl - c;
      if (lane == 31) scan[t][warp] = incl;
    }
    __syncthreads();
    static_assert(kHeld * kWarps == 64, "two entries a lane below");
    if (warp == 0) {  // the warps' counts in tile order; a slice's sums fit 16 bits too (8,192)
      uint32_t* flat = &scan[0][0];
      const uint32_t a = flat[2 * lane], c = flat[2 * lane + 1], incl = warp_scan(a + c);
      flat[2 * lane] = incl - a - c;
      flat[2 * lane + 1] = incl - c;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < kHeld; ++t) {
      const uint32_t at = scan[t][warp] + before[t];
      write(t, held[t], gt0 + (int)(at & 0xffffu), eq0 + (int)(at >> 16));
    }
  } else {
    for (int t = 0; t < tiles; ++t) {
      uint32_t key[kPer];
      load(t, key);
      const uint32_t c = count(t, key), incl = warp_scan(c);
      if (lane == 31) scan[0][warp] = incl;
      __syncthreads();
      uint32_t at = incl - c, all = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const uint32_t x = scan[0][w];
        if (w < warp) at += x;
        all += x;
      }
      write(t, key, gt0 + (int)(at & 0xffffu), eq0 + (int)(at >> 16));
      gt0 += (int)(all & 0xffffu);
      eq0 += (int)(all >> 16);
      __syncthreads();
    }
  }
  cluster.sync();  // no CTA leaves while its counts may be read
}

}  // namespace
}  // namespace sf

extern "C" int sf_kv_keep_heaviest(const float* mass, int64_t mass_batch_stride, int64_t mass_head_stride, int batch,
                                   int num_kv_heads, int64_t length, int64_t budget, int64_t sinks, int64_t recent,
                                   int32_t* keep, void* stream) {
  using namespace sf;
  SF_CHECK_ARG(batch > 0 && num_kv_heads > 0 && (int64_t)batch * num_kv_heads <= 65535,
               "batch and num_kv_heads must be positive, their product at most 65535");
  SF_CHECK_ARG(length >= 0 && length < (1 << 30), "length must be in [0, 2^30)");
  SF_CHECK_ARG(sinks >= 0 && recent >= 0 && sinks <= budget && recent <= budget - sinks && budget <= length,
               "sinks + recent <= budget <= length is needed");
  if (budget == 0) return SF_OK;
  SF_CHECK_ARG(mass && keep, "null pointer argument");
  KeepParams p;
  p.mass = mass;
  p.m_bs = mass_batch_stride;
  p.m_hs = mass_head_stride;
  p.hkv = num_kv_heads;
  p.length = (int)length;
  p.budget = (int)budget;
  p.sinks = (int)sinks;
  p.recent = (int)recent;
  p.keep = keep;
  const int64_t mid = length - sinks - recent;
  // One CTA per tile of 2,048 tokens, up to the cluster's eight.
  unsigned ranks = 1;
  while (ranks < kMaxCluster && (int64_t)ranks * kTile < mid) ranks *= 2;
  p.slice = (int)(((mid + ranks - 1) / ranks + kTile - 1) / kTile * kTile);
  const dim3 grid(ranks, (unsigned)(batch * num_kv_heads));
  if (p.slice <= kHeld * kTile)
    SF_CHECK_CUDA(launch_pdl_cluster(kv_keep_kernel<true>, grid, dim3(kThreads), 0, as_stream(stream), ranks, 1u, p));
  else
    SF_CHECK_CUDA(launch_pdl_cluster(kv_keep_kernel<false>, grid, dim3(kThreads), 0, as_stream(stream), ranks, 1u, p));
  SF_CHECK_LAUNCH();
  return SF_OK;
}
