// How much attention each cached token received: for one pass,
//   mass[b, kvh, j] += sum over the query heads of kvh and the query rows r
//                      that see j of exp(scale * q_r . k_j - lse_r)
// with the log-sum-exp that the attention of the same pass returned.
//
// The floor is one read of K's codes (128 bytes a token and KV head at D =
// 128) and of the mass.  The keys stay: a warp decodes 16 of them into
// registers once and walks all query rows over them, 16 at a time, so the
// codes are read and decoded once whatever the number of rows, and a key's
// sum never leaves its warp (no atomics: the same inputs give the same bits).
// The tile after the present one is on its way to registers, with the mass so
// far: one token over 65,569 tokens, 32 heads, takes 14 us (25 without), 2.5
// TB/s; four to five of them are the launch, Q and the first tile.
// Query rows are staged in shared memory in MMA fragment order, 64 at a time,
// as fp16 with a power of two taken out of each (kv8_attn.cu has the reasons).
#include <math.h>

#include <algorithm>

#include "kv8_attn.h"
#include "kv8_mma.cuh"

namespace sf {
namespace {

constexpr int kWarps = 4;
constexpr int kKeys = 16;               // of a warp
constexpr int kTileKeys = kWarps * kKeys;
constexpr int kChunkRows = kWarps * 16; // query rows staged at a time

struct MassParams {
  Kv8Attn a;  // lse is read here
  float* mass;
  int64_t m_bs, m_hs;
  int tiles;  // key tiles of 64
};

// grid: (CTAs over the key tiles, batch * hkv).
template <int DT>
__global__ void __launch_bounds__(kWarps * 32, 4)
kv8_mass_kernel(MassParams mp) {
  pdl_wait();
  pdl_trigger();
  const Kv8Attn& p = mp.a;
  constexpr int kSteps = DT / 16, kChunks = DT / 64;
  __shared__ __align__(16) uint4 qs_frag[kWarps][kSteps][32];
  __shared__ float row_f[kChunkRows], row_lse[kChunkRows], tail_k[kWarps][kKeys];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int kvh = blockIdx.y % p.c.hkv, req = blockIdx.y / p.c.hkv;
  const int packed = p.group * p.q_len;
  const int sealed = (int)p.c.sealed, d = p.c.d;
  const int chunks = (packed + kChunkRows - 1) / kChunkRows;
  const uint8_t* kc = p.c.k + req * p.c.c_bs + kvh * p.c.c_hs;
  const float* ksc = p.c.ks + req * p.c.s_bs + kvh * p.c.s_hs;
  const __nv_bfloat16* kt = p.c.kt + req * p.c.t_bs + kvh * p.c.t_hs;
  float* mass = mp.mass + req * mp.m_bs + kvh * mp.m_hs;
  int staged = -1;

  // What a tile reads, a tile ahead: the codes, their scale and the mass so far.
  uint4 next[2][kChunks];
  float next_scale = 1.f, next_mass[4];
  auto load = [&](int tile) {
    const int key0 = tile * kTileKeys + warp * kKeys;
    if (key0 < sealed) {
      next_scale = ksc[key0 >> p.c.block_shift];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
          const int byte = j * 64 + c * 16;
          next[t][j] = make_uint4(0, 0, 0, 0);
          if (byte < d) next[t][j] = *reinterpret_cast<const uint4*>(kc + (int64_t)(key0 + t * 8 + g) * d + byte);
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int key = key0 + 2 * c + (k & 1) + (k >> 1) * 8;
      next_mass[k] = g == 0 && key < p.kv_len ? mass[key] : 0.f;
    }
  };
  if ((int)blockIdx.x < mp.tiles) load(blockIdx.x);
  for (int tile = blockIdx.x; tile < mp.tiles; tile += gridDim.x) {
    const int key0 = tile * kTileKeys + warp * kKeys;
    // This warp's keys as fp16 B fragments.
    uint32_t kf[2][kSteps][2];
    const bool coded = key0 < sealed;
    float kscale = 1.f;  // of the codes; tail keys have theirs in shared memory
    if (coded) {
      kscale = next_scale;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
          const uint4 w = next[t][j];
          const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            kf[t][j * 4 + i][0] = e4m3x2_to_f16x2(ww[i]);
            kf[t][j * 4 + i][1] = e4m3x2_hi_to_f16x2(ww[i]);
          }
        }
    } else {
      // Tail rows: a power of two of its own for each, so that one which no row sees
      // leaves the others what they are; NaN for one with a NaN or an infinity.
      __syncwarp();  // the tile before has been read
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int key = key0 + t * 8 + g;
        const __nv_bfloat16* row = kt + (int64_t)(key - sealed) * d;
        uint2 x[kSteps];
        uint32_t top2 = 0;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const int dim = (s >> 2) * 64 + c * 16 + (s & 3) * 4;
          x[s] = key < p.kv_len && dim < d ? *reinterpret_cast<const uint2*>(row + dim) : make_uint2(0, 0);
          top2 = __vmaxu2(__vmaxu2(top2, x[s].x & 0x7fff7fffu), x[s].y & 0x7fff7fffu);
        }
        top2 = __vmaxu2(top2, __shfl_xor_sync(0xffffffffu, top2, 1));
        top2 = __vmaxu2(top2, __shfl_xor_sync(0xffffffffu, top2, 2));
        const uint32_t top = max(top2 & 0xffffu, top2 >> 16);
        const bool bad = top >= 0x7f80u;
        const int e = bad ? 0 : fit_exponent(top);
        const float inv = pow2f(-e);
        if (c == 0) tail_k[warp][t * 8 + g] = bad ? __int_as_float(0x7fc00000) : pow2f(e);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          if (bad) x[s] = make_uint2(0, 0);
          kf[t][s][0] = pack_f16x2(bf_lo(x[s].x) * inv, bf_hi(x[s].x) * inv);
          kf[t][s][1] = pack_f16x2(bf_lo(x[s].y) * inv, bf_hi(x[s].y) * inv);
        }
      }
      __syncwarp();
    }

    float before[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) before[k] = next_mass[k];
    if (tile + (int)gridDim.x < mp.tiles) load(tile + gridDim.x);

    float acc[4] = {0.f, 0.f, 0.f, 0.f};  // keys 2c, 2c + 1, 8 + 2c, 9 + 2c
    for (int chunk = 0; chunk < chunks; ++chunk) {
      if (chunk != staged) {  // one chunk in all: staged once per CTA
        __syncthreads();
        const int row0 = chunk * kChunkRows + warp * 16;
        uint32_t qf[kSteps][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int pr = row0 + g + 8 * r;
          const bool ok = pr < packed;
          const int t = ok ? pr % p.q_len : 0;
          const int head = kvh * p.group + (ok ? pr / p.q_len : 0);
          const __nv_bfloat16* qrow = p.q + req * p.q_bs + head * p.q_hs + t * p.q_rs;
          const float f = q_row_fragments<kSteps>(ok ? qrow : nullptr, d, c, qf, r);
          if (c == 0) {
            const float lse = ok ? p.lse[((int64_t)req * p.heads + head) * p.q_len + t] : -INFINITY;
            row_f[warp * 16 + g + 8 * r] = f * p.scale_log2;
            row_lse[warp * 16 + g + 8 * r] = lse == -INFINITY ? INFINITY : lse * 1.4426950408889634f;
          }
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) qs_frag[warp][s][lane] = make_uint4(qf[s][0], qf[s][1], qf[s][2], qf[s][3]);
        __syncthreads();
        staged = chunk;
      }
      const int tiles = min(kWarps, (packed - chunk * kChunkRows + 15) / 16);
      for (int i = 0; i < tiles; ++i) {
        float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          const uint4 w = qs_frag[i][st][lane];
          const uint32_t a[4] = {w.x, w.y, w.z, w.w};
          mma_f16(s[0], a, kf[0][st][0], kf[0][st][1]);
          mma_f16(s[1], a, kf[1][st][0], kf[1][st][1]);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (chunk * kChunkRows + i * 16 + 8 * r >= packed) break;  // a lone token's group of 8 heads or fewer
          const int at = i * 16 + g + 8 * r, pr = chunk * kChunkRows + at;
          uint32_t vis = 15u;
          if (key0 + kKeys > p.prefix) {
            const int t = pr % p.q_len;
            const uint32_t* rbits = p.bits ? p.bits + req * p.bits_bs + (int64_t)t * p.words : nullptr;
            const uint32_t w = pr < packed ? (uint32_t)kv8_window(p, rbits, key0) : 0u;
            vis = ((w >> (2 * c)) & 3u) | (((w >> (8 + 2 * c)) & 3u) << 2);
          }
          const float rf = row_f[at], lse = row_lse[at];  // rows past the last: lse +infinity
          if (coded) {
            const float f = rf * kscale;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if ((vis >> k) & 1u) acc[k] += ex2(s[k >> 1][2 * r + (k & 1)] * f - lse);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if ((vis >> k) & 1u) acc[k] += ex2(s[k >> 1][2 * r + (k & 1)] * (rf * tail_k[warp][(k >> 1) * 8 + 2 * c + (k & 1)]) - lse);
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) acc[k] += __shfl_xor_sync(0xffffffffu, acc[k], off);
    if (g == 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int key = key0 + 2 * c + (k & 1) + (k >> 1) * 8;
        if (key < p.kv_len) mass[key] = before[k] + acc[k];
      }
    }
  }
}

template <int DT>
int launch_mass(const MassParams& p, cudaStream_t stream) {
  const int64_t heads = (int64_t)p.a.batch * p.a.c.hkv;
  // About four CTAs per SM in all, each with its share of the key tiles.
  const int64_t want = std::max<int64_t>(1, (4 * (int64_t)num_sms() + heads - 1) / heads);
  const dim3 grid((unsigned)std::min<int64_t>(want, p.tiles), (unsigned)heads);
  SF_CHECK_CUDA(launch_pdl(kv8_mass_kernel<DT>, grid, dim3(kWarps * 32), 0, stream, p));
  SF_CHECK_LAUNCH();
  ++kv8_launches();
  return SF_OK;
}

}  // namespace
}  // namespace sf

extern "C" size_t sf_kv8_mass_workspace_bytes(int batch, int num_heads, int num_kv_heads, int head_dim, int64_t q_len,
                                             int64_t sealed, int64_t tail) {
  using namespace sf;
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || head_dim <= 0 ||
      head_dim > 128 || q_len <= 0 || sealed < 0 || tail < 0 || sealed + tail <= 0 || q_len >= (1 << 30) ||
      sealed >= (1 << 30) || tail >= (1 << 30))
    return 0;
  const int64_t packed = (int64_t)(num_heads / num_kv_heads) * q_len;
  if (!kv8_mass_use_tc(head_dim, packed)) return 0;
  return kv8_mass_tc_bytes((int64_t)batch * num_kv_heads, packed, sealed, sealed + tail);
}

extern "C" int sf_kv8_attention_mass(const void* q, int64_t q_batch_stride, int64_t q_head_stride,
                                     int64_t q_row_stride, int num_heads, int64_t q_len, const float* lse,
                                     const sf_kv8_rows* rows, const uint32_t* tree_bits, int bit_words,
                                     int64_t bits_batch_stride, int64_t prefix_len, float scale, float* mass,
                                     int64_t mass_batch_stride, int64_t mass_head_stride, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  using namespace sf;
  kv8_launches() = 0;
  if (int rc = kv8_check(rows, false)) return rc;
  const int64_t kv_len = rows->sealed + rows->tail;
  SF_CHECK_ARG(num_heads > 0 && num_heads % rows->num_kv_heads == 0,
               "num_heads must be a positive multiple of num_kv_heads");
  SF_CHECK_ARG(q_len >= 0 && prefix_len >= 0 && prefix_len <= kv_len && kv_len < (1 << 30), "invalid lengths");
  const int group = num_heads / rows->num_kv_heads;
  SF_CHECK_ARG((int64_t)group * q_len < (1 << 20), "too many query rows");
  if (q_len == 0 || kv_len == 0) return SF_OK;
  SF_CHECK_ARG(scale > 0.f && scale < INFINITY, "scale must be positive and finite");
  SF_CHECK_ARG(q && lse && mass, "null pointer argument");
  SF_CHECK_ARG(kv_len == prefix_len || (tree_bits && (int64_t)bit_words * 32 >= kv_len - prefix_len),
               "tree_bits must cover the keys from prefix_len on");
  SF_CHECK_ARG(aligned16(q) && q_batch_stride % 8 == 0 && q_head_stride % 8 == 0 && q_row_stride % 8 == 0,
               "q rows must be 16-byte aligned");
  SF_CHECK_ARG(kv8_apart(rows->batch, mass_batch_stride, rows->num_kv_heads, mass_head_stride, kv_len),
               "requests and heads of mass must not overlap");
  const size_t need = sf_kv8_mass_workspace_bytes(rows->batch, num_heads, rows->num_kv_heads, rows->head_dim, q_len,
                                                  rows->sealed, rows->tail);
  if (workspace_bytes < need || (need && !workspace))
    return set_error(SF_ERR_WORKSPACE, "8-bit cache mass workspace needs %zu bytes", need);
  SF_CHECK_ARG(need == 0 || aligned16(workspace), "workspace must be 16-byte aligned");
  MassParams m = {};
  m.a.c = kv8_view(*rows);
  m.a.q = static_cast<const __nv_bfloat16*>(q);
  m.a.q_bs = q_batch_stride;
  m.a.q_hs = q_head_stride;
  m.a.q_rs = q_row_stride;
  m.a.bits = kv_len == prefix_len ? nullptr : tree_bits;
  m.a.words = bit_words;
  m.a.bits_bs = bits_batch_stride;
  m.a.batch = rows->batch;
  m.a.heads = num_heads;
  m.a.group = group;
  m.a.q_len = (int)q_len;
  m.a.q_magic = ((1ull << 40) + (uint64_t)q_len - 1) / (uint64_t)q_len;
  m.a.kv_len = (int)kv_len;
  m.a.prefix = (int)prefix_len;
  m.a.scale_log2 = scale * 1.4426950408889634f;
  m.a.lse = const_cast<float*>(lse);
  m.mass = mass;
  m.m_bs = mass_batch_stride;
  m.m_hs = mass_head_stride;
  m.tiles = (int)((kv_len + kTileKeys - 1) / kTileKeys);
  if (need && kv8_tc_layout(m.a.c, rows->batch))
    return kv8_mass_tc(m.a, mass, mass_batch_stride, mass_head_stride, workspace, as_stream(stream));
  return rows->head_dim <= 64 ? launch_mass<64>(m, as_stream(stream)) : launch_mass<128>(m, as_stream(stream));
}
