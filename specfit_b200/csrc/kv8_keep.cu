// Which cached tokens stay: per request and KV head the first `sinks`, the
// last `recent`, and of those between the `budget - sinks - recent` that
// received the most attention weight, as ascending indices.  Among equal
// weights the earlier token stays; a NaN counts as the least weight.
//
// A radix selection, not a sort: the weights are mapped to integers of the
// same order, four 8-bit histogram passes find the smallest kept key and how
// many of its equals are kept, and one ordered pass writes the indices.  The
// floor is one read of the weights (4 bytes a token), which for the sizes in
// use (512 KB a head at 131,072 tokens) is below launch latency: what bounds
// the kernel is the chain of passes, so a cluster of up to eight CTAs shares
// a head, each with its own slice (in L1 / L2 after the first pass), and
// adds its peers' histograms through distributed shared memory.  Integer
// counts only, so the result does not depend on the order of the atomics.
#include <cooperative_groups.h>

#include "kv8.cuh"

namespace sf {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kPer = 4;  // consecutive weights of one thread in the ordered pass
constexpr int kTile = kThreads * kPer;

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

__global__ void __launch_bounds__(kThreads)
kv_keep_kernel(KeepParams p) {
  pdl_wait();
  pdl_trigger();
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  __shared__ uint32_t hist[256];
  __shared__ uint32_t total[256];
  __shared__ uint32_t prefix_s, want_s;
  __shared__ int counts[2];                 // this CTA's kept-above and equal counts
  __shared__ int scan_gt[kWarps], scan_eq[kWarps];
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

  // Four passes, the most significant digit first: `prefix` is the digits
  // found so far, `want` how many keys that match it are still to be kept.
  uint32_t prefix = 0, want = (uint32_t)want0;
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    const uint32_t mask = pass == 0 ? 0u : 0xffffffffu << (shift + 8);
    for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
    __syncthreads();
    for (int base = lo; base < hi; base += kThreads) {
      const int i = base + tid;
      bool in = false;
      uint32_t digit = 0;
      if (i < hi) {
        const uint32_t key = order_key(m[i]);
        in = (key & mask) == prefix;
        digit = (key >> shift) & 255u;
      }
      // Equal digits (a head's many zeros, a narrow range) are counted once per warp.
      const uint32_t tag = in ? digit : 256u;
      const uint32_t peers = __match_any_sync(0xffffffffu, tag);
      if (in && lane == __ffs(peers) - 1) atomicAdd(&hist[digit], (uint32_t)__popc(peers));
    }
    cluster.sync();
    if (tid < 256) {
      uint32_t sum = 0;
      for (int r = 0; r < ranks; ++r) sum += cluster.map_shared_rank(hist, r)[tid];
      total[tid] = sum;
    }
    __syncthreads();
    if (warp == 0) {  // the digit at which the count from the top reaches `want`
      uint32_t mine[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        mine[j] = total[255 - (lane * 8 + j)];
        sum += mine[j];
      }
      uint32_t before = sum;  // inclusive scan over the lanes, then made exclusive
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
      }
      before -= sum;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (before < want && want <= before + mine[j]) {
          prefix_s = prefix | ((uint32_t)(255 - (lane * 8 + j)) << shift);
          want_s = want - before;
        }
        before += mine[j];
      }
      if (lane == 0 && want == 0) {  // nothing of the middle is kept
        prefix_s = 0xffffffffu;
        want_s = 0;
      }
    }
    cluster.sync();  // the histograms may be cleared
    prefix = prefix_s;
    want = want_s;
    if (want == 0) break;  // uniform over the cluster: only when want0 is 0
  }
  if (want0 == 0) return;  // every CTA of the cluster has passed the sync above

  // Now `prefix` is the smallest kept key and the first `want` of its equals stay.
  int gt = 0, eq = 0;
  for (int i = lo + tid; i < hi; i += kThreads) {
    const uint32_t key = order_key(m[i]);
    gt += key > prefix;
    eq += key == prefix;
  }
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
  const int limit = (int)want;
  for (int base = lo; base < hi; base += kTile) {
    uint32_t key[kPer];
    int g = 0, e = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = base + tid * kPer + j;
      key[j] = i < hi ? order_key(m[i]) : 0u;
      g += i < hi && key[j] > prefix;
      e += i < hi && key[j] == prefix;
    }
    int gi = g, ei = e;  // inclusive scans
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, gi, o), c = __shfl_up_sync(0xffffffffu, ei, o);
      if (lane >= o) {
        gi += a;
        ei += c;
      }
    }
    if (lane == 31) {
      scan_gt[warp] = gi;
      scan_eq[warp] = ei;
    }
    __syncthreads();
    int gb = gt0, eb = eq0, gall = 0, eall = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) {
        gb += scan_gt[w];
        eb += scan_eq[w];
      }
      gall += scan_gt[w];
      eall += scan_eq[w];
    }
    gb += gi - g;
    eb += ei - e;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = base + tid * kPer + j;
      if (i >= hi) break;
      if (key[j] > prefix) {
        out[p.sinks + gb + min(eb, limit)] = p.sinks + i;
        ++gb;
      } else if (key[j] == prefix) {
        if (eb < limit) out[p.sinks + gb + eb] = p.sinks + i;
        ++eb;
      }
    }
    gt0 += gall;
    eq0 += eall;
    __syncthreads();
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
  SF_CHECK_ARG(sinks >= 0 && recent >= 0 && sinks + recent <= budget && budget <= length,
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
  SF_CHECK_CUDA(launch_pdl_cluster(kv_keep_kernel, grid, dim3(kThreads), 0, as_stream(stream), ranks, 1u, p));
  SF_CHECK_LAUNCH();
  return SF_OK;
}
