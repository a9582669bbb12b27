// Tree-masked GQA attention over the 8-bit KV cache: the warp-level kernel,
// the merge of the key ranges, and the entry points.
//
//   s_rj = scale * q_r . k_j,  o_r = sum_j exp(s_rj - lse_r) v_j,  lse_r = ln sum_j exp(s_rj)
//
// over the keys j that row r sees (all before prefix_len, and those whose bit
// is set).  A row that sees nothing answers zeros and lse = -infinity.
//
// The floor is one read of the codes (256 bytes a token and KV head at
// D = 128).  With the query heads of one KV head packed into one 16-row MMA
// tile (row = head_in_group * Tq + t) a few query rows need 2 MMAs per 8 keys
// and 16 dims, far below the tensor rate, so what has to be kept small is the
// work per element: loading, decoding, and the softmax.
//   * Every warp walks its own 32-key units of the CTA's range with its own
//     online softmax; the four warps and the splits are joined at the end.
//     Nothing in the loop waits for another warp.
//   * Dims of a key are a sum, keys of a value too, so both may be taken in
//     any order: a thread's 16 consecutive code bytes ARE its MMA fragments
//     (K: four k-steps of one key; V: one column of 16 output tiles), so the
//     loop needs no transpose.  A warp copies its units into its own ring
//     (cp.async), 512 consecutive bytes an instruction: with each thread copying
//     the bytes that it uses itself, eight rows of 64 bytes an instruction, 131,072
//     tokens took 33 us instead of 30.
//   * At most eight query rows (a token of a group of eight heads): keys, then
//     dims, are the MMA's 16 rows and the query rows its 8 columns, half the MMAs
//     and exponentials of the other way round (38 to 33 us).  Probabilities turn
//     from key rows to query-row columns by 8 x 8 transposes in registers.
//   * Codes become fp16 (exact) by one conversion per two; Q as fp16 is exact
//     too once each row is scaled by a power of two (fp16's 11 bits hold
//     bf16's 8 over 30 binades below the row's largest; what is smaller is
//     below 2^-30 of it).  K's scale multiplies the fp32 scores.
//   * V's scale enters the exponent: P = 2^(s + log2 scale - m), so m, a row's own
//     reference, is the largest of s + log2 scale among the keys that it sees,
//     and only what is below 2^-26 of the row's largest probability times scale
//     is rounded more than fp16's 11 bits (P is kept times 2^12).  One exponential
//     gives P and the probability, the larger of the two, and the other by a
//     power of two.  (A unit for a warp's accumulators, the largest scale that it
//     had met, lost a row's small values beside large ones that the row did not see.)
//   * m moves only when a score exceeds it by more than 3 (base 2), so
//     accumulators are rarely rescaled.
//   * What bounds it is a warp's chain of instructions (three warps a scheduler
//     issue in one clock of four): of the 20 or so that 16 codes take, 6 are
//     conversions (ALU, half rate) and 2 MMAs.  Hence 32 keys a step (645
//     instructions for 16 keys were 43 us at 131,072 tokens), Q's fragments from
//     shared memory (one 16-byte load for four MMAs), tail units converted there
//     too, and addresses that are constants where D is the tile's width.
// What it measured: one token, 32 heads over 131,113 tokens, 27 us, 5.0 TB/s, of
// which about five are the launch, Q, the join and the partial results, and 7
// more the merge; over 529 tokens 8.8.  (30 us while a tail unit's loads came a key
// after the other: the last range's CTA ended late.)  Four CTAs an SM, with a ring of 12 KB a warp, took 37: each
// has that cost, and a shorter range.
// Tail units (bf16 rows: few): a power of two per key is taken out of its row of K,
// another out of its row of V, and they enter the same fragments.  A key with a NaN
// or an infinity in either row (a sealed block that holds one) has a NaN score, so
// that rows which do not see it stay what they are.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "kv8_attn.h"
#include "kv8_mma.cuh"

namespace sf {
namespace {

constexpr int kWarps = 4;
constexpr int kRows = 16;      // packed query rows of a CTA
constexpr int kUnit = 32;      // keys of one step of a warp: within one block of codes
constexpr int kHalves = kUnit / 16;
constexpr int kStages = 2;     // units of a warp's ring
constexpr int kStep = kWarps * kUnit;
constexpr int kMaxSplits = 128;
constexpr int kMaxCluster = 8; // key ranges that a cluster joins itself
// Up to so many steps of a CTA the ranges are at most a cluster's: a token
// over 545 / 1,569 tokens 8.8 / 9.5 us against 10.0 / 10.0 with a range a step and
// the merge kernel (8 rows: 11.0 / 12.6 against 11.9 / 14.1), and one launch less;
// at 2,593 tokens they are equal (11.5 / 10.8; 15.5 / 17.2), at 4,129 the merge is
// faster (11.5 / 11.0; 16.6 / 14.7).
constexpr int kClusterSteps = 24;
constexpr float kPShift = 12.f;  // probabilities are kept times 2^12
constexpr float kSlack = 3.f;    // a row's reference maximum may lag by this (base 2)

template <int DT>
struct Layout {
  static constexpr int kKChunks = DT / 64;             // 16-byte chunks of a key per thread
  static constexpr int kVBytes = DT / 8;               // bytes of a value row per thread
  static constexpr int kSteps = DT / 16;               // MMA k-steps of Q K^T
  static constexpr int kTiles = DT / 8;                // output tiles of P V
  static constexpr int kKBytes = 2 * kHalves * kKChunks * 16;  // per thread and unit
  static constexpr int kVKeys = 4 * kHalves;           // keys of a thread in P V
  static constexpr int kUnitBytes = 32 * (kKBytes + kVKeys * kVBytes);  // K and V codes
  static constexpr int kRing = kWarps * kStages * kUnitBytes;
  // A tail unit as fp16 takes twice its codes' bytes, in the ring, where no copy is in flight by then.
  static_assert(kStages >= 2, "a tail unit needs two stages");
  static constexpr int kJoin = kWarps * kRows * DT * 4;
  // The CTA's own rows, where its cluster reads them: behind the warps'.
  static constexpr int kRows0 = kJoin, kNeed = kJoin + kRows * DT * 4;
  static constexpr int kSmem = kRing > kNeed ? kRing : kNeed;
};

// A unit of tail rows as fp16 fragments in this thread's slots of `out`
// ([K: key tiles x steps][V: halves x output tiles] of 32 lanes), each row scaled
// by a power of two of its own; zeros for keys from key_hi on.  First the rows as
// they are, all on their way at once, then their magnitudes, then each slot in
// place.  For key i of the unit: kscale[i], the scale of its K row, NaN if that
// holds a NaN or an infinity; vlog[i], log2 of its V row's, NaN likewise.
template <int DT>
__device__ __forceinline__ void tail_unit(const __nv_bfloat16* kt, const __nv_bfloat16* vt, int key0, int sealed,
                                          int key_hi, int d, int g, int c, int lane, uint2* out, float* kscale,
                                          float* vlog) {
  using L = Layout<DT>;
  constexpr int kKSlots = 2 * kHalves * L::kSteps;
  const uint32_t slots = smem_addr(out) + (uint32_t)lane * 8;
#pragma unroll 1
  for (int t = 0; t < 2 * kHalves; ++t) {
    const int key = key0 + t * 8 + g;
    const __nv_bfloat16* row = kt + (int64_t)(key < key_hi ? key - sealed : 0) * d;
#pragma unroll
    for (int st = 0; st < L::kSteps; ++st) {
      const int dim = (st >> 2) * 64 + c * 16 + (st & 3) * 4;
      const bool on = key < key_hi && dim < d;
      cp_async<8>(slots + (uint32_t)((t * L::kSteps + st) * 256), on ? row + dim : kt, on);
    }
  }
#pragma unroll 1
  for (int k = 0; k < L::kVKeys; ++k) {  // half k / 4; keys 2c, 2c + 1, 8 + 2c, 9 + 2c of it
    const int key = key0 + (k >> 2) * 16 + 2 * c + (k & 1) + ((k >> 1) & 1) * 8;
    const bool on = key < key_hi && g * L::kVBytes < d;
    const __nv_bfloat16* row = on ? vt + (int64_t)(key - sealed) * d + g * L::kVBytes : vt;
#pragma unroll
    for (int w = 0; w < L::kVBytes / 4; ++w)
      cp_async<8>(slots + (uint32_t)((kKSlots + (k >> 2) * L::kTiles + 4 * w + (k & 3)) * 256), row + (on ? w * 4 : 0),
                  on);
  }
  cp_commit();
  cp_wait<0>();
  // Largest magnitudes (15-bit integers, two rows a register): of K rows t * 8 + g,
  // whose dims a quad holds, and of V rows 2c, 2c + 1, 8 + 2c, 9 + 2c of a half,
  // whose dims the eight lanes of a column hold.
  uint32_t ktop[kHalves], vtop[2 * kHalves];
  auto top_of = [](uint32_t t2) { return max(t2 & 0xffffu, t2 >> 16); };
#pragma unroll
  for (int t = 0; t < kHalves; ++t) {
    uint32_t a = 0, b = 0;
#pragma unroll
    for (int st = 0; st < L::kSteps; ++st) {
      const uint2 x = out[((2 * t) * L::kSteps + st) * 32 + lane], y = out[((2 * t + 1) * L::kSteps + st) * 32 + lane];
      a = __vmaxu2(__vmaxu2(a, x.x & 0x7fff7fffu), x.y & 0x7fff7fffu);
      b = __vmaxu2(__vmaxu2(b, y.x & 0x7fff7fffu), y.y & 0x7fff7fffu);
    }
    ktop[t] = top_of(a) | top_of(b) << 16;
  }
#pragma unroll
  for (int k = 0; k < 2 * kHalves; ++k) {
    uint32_t a = 0, b = 0;
#pragma unroll
    for (int w = 0; w < L::kTiles / 4; ++w) {
      const uint2* at = out + (kKSlots + (k >> 1) * L::kTiles + 4 * w + (k & 1) * 2) * 32 + lane;
      const uint2 x = at[0], y = at[32];
      a = __vmaxu2(__vmaxu2(a, x.x & 0x7fff7fffu), x.y & 0x7fff7fffu);
      b = __vmaxu2(__vmaxu2(b, y.x & 0x7fff7fffu), y.y & 0x7fff7fffu);
    }
    vtop[k] = top_of(a) | top_of(b) << 16;
  }
#pragma unroll
  for (int off = 1; off < 4; off <<= 1)
#pragma unroll
    for (int t = 0; t < kHalves; ++t) ktop[t] = __vmaxu2(ktop[t], __shfl_xor_sync(0xffffffffu, ktop[t], off));
#pragma unroll
  for (int off = 4; off < 32; off <<= 1)
#pragma unroll
    for (int k = 0; k < 2 * kHalves; ++k) vtop[k] = __vmaxu2(vtop[k], __shfl_xor_sync(0xffffffffu, vtop[k], off));
#pragma unroll
  for (int t = 0; t < 2 * kHalves; ++t) {
    const uint32_t top = (ktop[t >> 1] >> (16 * (t & 1))) & 0xffffu;
    const bool bad = top >= 0x7f80u;
    const int e = bad ? 0 : fit_exponent(top);
    const float inv = pow2f(-e);
    if (c == 0) kscale[t * 8 + g] = bad ? __int_as_float(0x7fc00000) : pow2f(e);
#pragma unroll 4
    for (int st = 0; st < L::kSteps; ++st) {
      uint2* at = out + (t * L::kSteps + st) * 32 + lane;
      const uint2 w = bad ? make_uint2(0, 0) : *at;
      *at = make_uint2(pack_f16x2(bf_lo(w.x) * inv, bf_hi(w.x) * inv), pack_f16x2(bf_lo(w.y) * inv, bf_hi(w.y) * inv));
    }
  }
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    float inv[4];
    bool bad[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t top = (vtop[2 * h + (k >> 1)] >> (16 * (k & 1))) & 0xffffu;
      bad[k] = top >= 0x7f80u;
      // Magnitudes below 2^9, like codes; a row of zeros counts as the smallest.
      const int e = top == 0 ? -105 : fit_exponent(bad[k] ? 0 : top) + 5;
      inv[k] = pow2f(-e);
      if (g == 0) vlog[h * 16 + 2 * c + (k & 1) + (k >> 1) * 8] = bad[k] ? __int_as_float(0x7fc00000) : (float)e;
    }
#pragma unroll 2
    for (int w = 0; w < L::kTiles / 4; ++w) {
      uint2* at = out + (kKSlots + h * L::kTiles + 4 * w) * 32 + lane;
      float f[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint2 u = bad[k] ? make_uint2(0, 0) : at[k * 32];
        f[k][0] = bf_lo(u.x) * inv[k];
        f[k][1] = bf_hi(u.x) * inv[k];
        f[k][2] = bf_lo(u.y) * inv[k];
        f[k][3] = bf_hi(u.y) * inv[k];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) at[i * 32] = make_uint2(pack_f16x2(f[0][i], f[1][i]), pack_f16x2(f[2][i], f[3][i]));
    }
  }
  __syncwarp();  // the scales, for the other lanes
}

// grid: (hkv, row tiles, splits * batch).  Full: D is DT.  Narrow: at most
// eight query rows.
template <int DT, bool Full, bool Narrow>
__global__ void __launch_bounds__(kWarps * 32, 3)
kv8_attn_kernel(Kv8Attn p) {
  using L = Layout<DT>;
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float join_m[kWarps][kRows], join_l[kWarps][kRows];
  __shared__ float2 row_ml[kRows];  // of the CTA, for its cluster
  __shared__ __align__(16) uint4 q_frag[L::kSteps][32];
  __shared__ float tail_k[kWarps][kUnit], tail_v[kWarps][kUnit];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int kvh = blockIdx.x;
  const int req = blockIdx.z / p.splits, split = blockIdx.z % p.splits;
  const int key_lo = split * p.keys_per_split;
  const int key_hi = min(p.kv_len, key_lo + p.keys_per_split);
  const int packed = p.group * p.q_len;
  const int sealed = (int)p.c.sealed;
  const int d = Full ? DT : p.c.d;

  const uint8_t* kc = p.c.k + req * p.c.c_bs + kvh * p.c.c_hs;
  const uint8_t* vc = p.c.v + req * p.c.c_bs + kvh * p.c.c_hs;
  const float* ksc = p.c.ks + req * p.c.s_bs + kvh * p.c.s_hs;
  const float* vsc = p.c.vs + req * p.c.s_bs + kvh * p.c.s_hs;
  const __nv_bfloat16* kt = p.c.kt + req * p.c.t_bs + kvh * p.c.t_hs;
  const __nv_bfloat16* vt = p.c.vt + req * p.c.t_bs + kvh * p.c.t_hs;

  // A warp's ring: [stage][K: 32 keys x DT bytes][V]; a row's 16-byte chunks in
  // an order of its own (k_chunk, v_chunk) that spreads what 8 lanes read at once
  // over the banks.
  const uint32_t ring = smem_addr(smem) + (uint32_t)warp * kStages * L::kUnitBytes;
  auto k_chunk = [](int row, int chunk) { return DT == 128 ? chunk ^ ((row & 1) << 2) : chunk; };
  auto v_chunk = [](int row, int chunk) {
    return DT == 128 ? chunk ^ (((row >> 1) & 3) << 1) : chunk ^ (((row >> 1) & 1) << 1);
  };
  auto load_unit = [&](int key0, int stage) {
    if (key0 < key_hi && key0 < sealed) {
      constexpr int kChunksRow = DT / 16, kRowsAt = 32 / kChunksRow;  // a copy's rows: consecutive bytes
      const int row = lane / kChunksRow, chunk = lane % kChunksRow;
      const bool on = Full || chunk * 16 < d;
      const uint32_t at = ring + (uint32_t)stage * L::kUnitBytes;
      const int64_t from = (int64_t)(key0 + row) * d + (on ? chunk * 16 : 0);
#pragma unroll
      for (int i = 0; i < kUnit / kRowsAt; ++i) {
        const int r = i * kRowsAt + row;
        cp_async<16>(at + (uint32_t)(r * DT + k_chunk(r, chunk) * 16), kc + from + i * kRowsAt * d, on);
      }
#pragma unroll
      for (int i = 0; i < kUnit / kRowsAt; ++i) {
        const int r = i * kRowsAt + row;
        cp_async<16>(at + (uint32_t)(kUnit * DT + r * DT + v_chunk(r, chunk) * 16), vc + from + i * kRowsAt * d, on);
      }
    }
    cp_commit();
  };

  uint2* tail_s = reinterpret_cast<uint2*>(smem + (size_t)warp * kStages * L::kUnitBytes);
  const int first = key_lo + warp * kUnit;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) load_unit(first + s * kStep, s);

  // Q fragments of rows g and g + 8: the dims of k-step (j, w) of this
  // thread are j * 64 + c * 16 + w * 4 + {0, 1, 2, 3}.  Every warp needs the same
  // ones: each writes a quarter of them.
  // The rows whose scores this thread gets: g and g + 8, or 2c and 2c + 1.
  auto row_of = [&](int r) { return Narrow ? 2 * c + r : g + 8 * r; };
  float qs[2];                 // scale * log2(e) * (power of two taken out of the row)
  const uint32_t* rbits[2];
  bool rok[2];
  {
    uint32_t qf[L::kSteps][4];
#pragma unroll
    for (int r = 0; r < (Narrow ? 1 : 2); ++r) {
      const int pr = blockIdx.y * kRows + g + r * 8;
      const bool on = pr < packed;
      const int qh = on ? (int)(((uint64_t)pr * p.q_magic) >> 40) : 0, t = on ? pr - qh * p.q_len : 0;
      const __nv_bfloat16* qrow = p.q + req * p.q_bs + (int64_t)(kvh * p.group + qh) * p.q_hs + t * p.q_rs;
      qs[r] = p.scale_log2 * q_row_fragments<L::kSteps>(on ? qrow : nullptr, d, c, qf, r);
    }
    if constexpr (Narrow) {
      const float f = qs[0];
#pragma unroll
      for (int r = 0; r < 2; ++r) qs[r] = __shfl_sync(0xffffffffu, f, (2 * c + r) * 4);
#pragma unroll
      for (int st = 0; st < L::kSteps; ++st) qf[st][1] = qf[st][3] = 0;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int pr = blockIdx.y * kRows + row_of(r);
      rok[r] = pr < packed;
      const int qh = rok[r] ? (int)(((uint64_t)pr * p.q_magic) >> 40) : 0, t = rok[r] ? pr - qh * p.q_len : 0;
      rbits[r] = p.bits ? p.bits + req * p.bits_bs + (int64_t)t * p.words : nullptr;
    }
#pragma unroll
    for (int st = 0; st < L::kSteps; ++st)
      if ((st & (kWarps - 1)) == warp) q_frag[st][lane] = make_uint4(qf[st][0], qf[st][2], qf[st][1], qf[st][3]);
    __syncthreads();
  }

  constexpr int kOTiles = Narrow ? L::kTiles / 2 : L::kTiles;
  float o[kOTiles][4];
#pragma unroll
  for (int t = 0; t < kOTiles; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[t][i] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  int stage = 0;
  for (int key0 = first; key0 < key_hi; key0 += kStep) {
    {
      int ahead = stage + kStages - 1;
      if (ahead >= kStages) ahead -= kStages;
      __syncwarp();  // every lane has read the unit before
      load_unit(key0 + (kStages - 1) * kStep, ahead);
    }
    cp_wait<kStages - 1>();  // this lane's pieces of this unit have landed,
    __syncwarp();            // and the other lanes'
    const uint8_t* at = smem + (size_t)warp * kStages * L::kUnitBytes + (size_t)stage * L::kUnitBytes;
    if (++stage == kStages) stage = 0;

    constexpr int kX = (Narrow ? 2 : 4) * kHalves;  // this thread's keys of a row
    constexpr int kSTiles = (Narrow ? 1 : 2) * kHalves;
    float s[kSTiles][4];
#pragma unroll
    for (int t = 0; t < kSTiles; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[t][i] = 0.f;
    float kscale;
    int v = 0;  // log2 of the V scale, rounded down, and what it lacks (1 for a power of two)
    float vrest = 1.f;
    const bool coded = key0 < sealed;
    if (coded) {
      kscale = ksc[key0 >> p.c.block_shift];
      const float vscale = vsc[key0 >> p.c.block_shift];
      if (vscale != vscale)  // a block with a NaN among its values: its keys' scores are NaN
        kscale = vscale;
      else
        v = scale_log2(vscale), vrest = vscale * pow2f(-v);
#pragma unroll
      for (int j = 0; j < L::kKChunks; ++j) {
        uint32_t w[2 * kHalves][4];
#pragma unroll
        for (int t = 0; t < 2 * kHalves; ++t) {
          const uint4 x = *reinterpret_cast<const uint4*>(at + (t * 8 + g) * DT + k_chunk(g, j * 4 + c) * 16);
          w[t][0] = x.x;
          w[t][1] = x.y;
          w[t][2] = x.z;
          w[t][3] = x.w;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (Narrow) {
            const uint2 qv = *reinterpret_cast<const uint2*>(&q_frag[j * 4 + i][lane]);
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
              const uint32_t ka[4] = {e4m3x2_to_f16x2(w[2 * h][i]), e4m3x2_to_f16x2(w[2 * h + 1][i]),
                                      e4m3x2_hi_to_f16x2(w[2 * h][i]), e4m3x2_hi_to_f16x2(w[2 * h + 1][i])};
              mma_f16(s[h], ka, qv.x, qv.y);
            }
          } else {
            const uint4 qv = q_frag[j * 4 + i][lane];
            const uint32_t qa[4] = {qv.x, qv.z, qv.y, qv.w};
#pragma unroll
            for (int t = 0; t < 2 * kHalves; ++t)
              mma_f16(s[t], qa, e4m3x2_to_f16x2(w[t][i]), e4m3x2_hi_to_f16x2(w[t][i]));
          }
        }
      }
    } else {
      tail_unit<DT>(kt, vt, key0, sealed, key_hi, d, g, c, lane, tail_s, tail_k[warp], tail_v[warp]);
#pragma unroll
      for (int st = 0; st < L::kSteps; ++st) {
        const uint4 qv = q_frag[st][lane];
        uint2 b[2 * kHalves];
#pragma unroll
        for (int t = 0; t < 2 * kHalves; ++t) b[t] = tail_s[(t * L::kSteps + st) * 32 + lane];
        if constexpr (Narrow) {
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            const uint32_t ka[4] = {b[2 * h].x, b[2 * h + 1].x, b[2 * h].y, b[2 * h + 1].y};
            mma_f16(s[h], ka, qv.x, qv.y);
          }
        } else {
          const uint32_t qa[4] = {qv.x, qv.z, qv.y, qv.w};
#pragma unroll
          for (int t = 0; t < 2 * kHalves; ++t) mma_f16(s[t], qa, b[t].x, b[t].y);
        }
      }
    }

    // Scores in base 2, those not seen -infinity: keys 2c, 2c + 1 (narrow: g) of each key tile.
    auto key_of = [&](int i) { return Narrow ? i * 8 + g : (i >> 1) * 8 + 2 * c + (i & 1); };
    auto score = [&](int r, int i) { return s[i >> 1][Narrow ? 2 * (i & 1) + r : 2 * r + (i & 1)]; };
    float x[2][kX], mx[2];  // mx: the largest, with log2 of its value's scale
    const bool open = key0 + kUnit <= p.prefix;  // no mask to read (prefix_len <= kv_len)
    bool grow = false;
    if (coded) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float f = qs[r] * kscale;
#pragma unroll
        for (int i = 0; i < kX; ++i) x[r][i] = score(r, i) * f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kX; ++i) {
        const float vl = tail_v[warp][key_of(i)];
        const float kf = vl == vl ? tail_k[warp][key_of(i)] : vl;
#pragma unroll
        for (int r = 0; r < 2; ++r) x[r][i] = score(r, i) * (qs[r] * kf);
      }
    }
    if (!open) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t w = rok[r] ? (uint32_t)kv8_window(p, rbits[r], key0) : 0u;
#pragma unroll
        for (int i = 0; i < kX; ++i)
          if (!((w >> key_of(i)) & 1u)) x[r][i] = -INFINITY;
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (coded) {
        mx[r] = x[r][0];
#pragma unroll
        for (int i = 1; i < kX; ++i) mx[r] = fmaxf(mx[r], x[r][i]);  // NaN is passed over
        mx[r] += (float)max(v + (vrest > 1.f ? 1 : 0), kMinValueScale);
      } else {
        mx[r] = -INFINITY;
#pragma unroll
        for (int i = 0; i < kX; ++i)
          mx[r] = fmaxf(mx[r], x[r][i] + fmaxf(tail_v[warp][key_of(i)], (float)kMinValueScale));
      }
      grow |= mx[r] > m[r] + kSlack;  // m -infinity: any score
    }
    float corr[2] = {1.f, 1.f};
    bool rescale = false;
    if (__any_sync(0xffffffffu, grow)) {
      rescale = true;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float y = fmaxf(m[r], mx[r]);
#pragma unroll
        for (int off = Narrow ? 4 : 1; off < (Narrow ? 32 : 4); off <<= 1)  // the threads of a row
          y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, off));
        // In two steps: l may be far from 1, and one factor below what fp32 holds.
        const float half = m[r] == -INFINITY ? 0.f : ex2(0.5f * (m[r] - y));
        m[r] = y;
        l[r] = l[r] * half * half;
        corr[r] = half * half;
      }
    }
    if (rescale) {
#pragma unroll
      for (int t = 0; t < kOTiles; ++t) {
        o[t][0] *= corr[0];
        o[t][1] *= corr[Narrow ? 1 : 0];
        o[t][2] *= corr[Narrow ? 0 : 1];
        o[t][3] *= corr[1];
      }
    }
    uint32_t pa[kHalves][4];
    const float base0 = (m[0] == -INFINITY ? 0.f : m[0]) - kPShift, base1 = (m[1] == -INFINITY ? 0.f : m[1]) - kPShift;
    if (coded) {
      const float vh = (float)max(v, 0), pm = pow2f(min(v, 0)) * vrest, em = pow2f(-max(v, 0));
      float sum[2] = {0.f, 0.f};
      if constexpr (Narrow) {
#pragma unroll
        for (int i = 0; i < kX; ++i) {
          const float e0 = ex2(x[0][i] - (base0 - vh)), e1 = ex2(x[1][i] - (base1 - vh));
          sum[0] += e0;
          sum[1] += e1;
          // Key g, rows 2c and 2c + 1; turned: keys 2c and 2c + 1, row g.
          pa[i >> 1][i & 1] = transpose_8x8(pack_f16x2(e0 * pm, e1 * pm));
        }
      } else {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float base = (r ? base1 : base0) - vh;
#pragma unroll
          for (int i = 0; i < kX; i += 2) {
            const float e0 = ex2(x[r][i] - base), e1 = ex2(x[r][i + 1] - base);
            sum[r] += e0 + e1;
            pa[i >> 2][r + (i & 2)] = pack_f16x2(e0 * pm, e1 * pm);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) l[r] = fmaf(sum[r], em, l[r]);
    } else {
      auto weigh = [&](int i, float (&pr)[2]) {
        const float vl = tail_v[warp][key_of(i)];
        const int vi = vl == vl ? (int)vl : 0;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float y = ex2(x[r][i] - ((r ? base1 : base0) - (float)max(vi, 0)));
          l[r] = fmaf(y, pow2f(-max(vi, 0)), l[r]);
          pr[r] = y * pow2f(min(vi, 0));
        }
      };
      if constexpr (Narrow) {
#pragma unroll
        for (int i = 0; i < kX; ++i) {
          float pr[2];
          weigh(i, pr);
          pa[i >> 1][i & 1] = transpose_8x8(pack_f16x2(pr[0], pr[1]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < kX; i += 2) {
          float pr[2], pq[2];
          weigh(i, pr);
          weigh(i + 1, pq);
#pragma unroll
          for (int r = 0; r < 2; ++r) pa[i >> 2][r + (i & 2)] = pack_f16x2(pr[r], pq[r]);
        }
      }
    }

    // Output tile t, column g: dim g * kVBytes + t.
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      if (coded) {
        uint32_t vf[4][L::kVBytes / 4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = h * 16 + 2 * c + (k & 1) + (k >> 1) * 8, byte = g * L::kVBytes;
          const uint8_t* a = at + kUnit * DT + row * DT + v_chunk(row, byte >> 4) * 16 + (byte & 15);
          if constexpr (L::kVBytes == 16) {
            const uint4 w = *reinterpret_cast<const uint4*>(a);
            vf[k][0] = w.x;
            vf[k][1] = w.y;
            vf[k][2] = w.z;
            vf[k][3] = w.w;
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(a);
            vf[k][0] = w.x;
            vf[k][1] = w.y;
          }
        }
#pragma unroll
        for (int w = 0; w < L::kVBytes / 4; ++w) {
          const uint32_t a01 = __byte_perm(vf[0][w], vf[1][w], 0x5140), a23 = __byte_perm(vf[0][w], vf[1][w], 0x7362);
          const uint32_t b01 = __byte_perm(vf[2][w], vf[3][w], 0x5140), b23 = __byte_perm(vf[2][w], vf[3][w], 0x7362);
          if constexpr (Narrow) {  // two output tiles are the 16 rows of an MMA
            const uint32_t v0[4] = {e4m3x2_to_f16x2(a01), e4m3x2_hi_to_f16x2(a01), e4m3x2_to_f16x2(b01),
                                    e4m3x2_hi_to_f16x2(b01)};
            const uint32_t v1[4] = {e4m3x2_to_f16x2(a23), e4m3x2_hi_to_f16x2(a23), e4m3x2_to_f16x2(b23),
                                    e4m3x2_hi_to_f16x2(b23)};
            mma_f16(o[2 * w + 0], v0, pa[h][0], pa[h][1]);
            mma_f16(o[2 * w + 1], v1, pa[h][0], pa[h][1]);
          } else {
            mma_f16(o[4 * w + 0], pa[h], e4m3x2_to_f16x2(a01), e4m3x2_to_f16x2(b01));
            mma_f16(o[4 * w + 1], pa[h], e4m3x2_hi_to_f16x2(a01), e4m3x2_hi_to_f16x2(b01));
            mma_f16(o[4 * w + 2], pa[h], e4m3x2_to_f16x2(a23), e4m3x2_to_f16x2(b23));
            mma_f16(o[4 * w + 3], pa[h], e4m3x2_hi_to_f16x2(a23), e4m3x2_hi_to_f16x2(b23));
          }
        }
      } else {
#pragma unroll
        for (int t = 0; t < L::kTiles; t += 2) {
          const uint2* at_t = tail_s + (2 * kHalves * L::kSteps + h * L::kTiles + t) * 32 + lane;
          const uint2 b = at_t[0], e = at_t[32];
          if constexpr (Narrow) {
            const uint32_t v[4] = {b.x, e.x, b.y, e.y};
            mma_f16(o[t / 2], v, pa[h][0], pa[h][1]);
          } else {
            mma_f16(o[t], pa[h], b.x, b.y);
            mma_f16(o[t + 1], pa[h], e.x, e.y);
          }
        }
      }
    }
  }
  cp_wait<0>();

  // Join the four warps: rows' sums over the four threads of a quad, then
  // partial outputs through shared memory (the ring's space).
  float unit[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
#pragma unroll
    for (int off = Narrow ? 4 : 1; off < (Narrow ? 32 : 4); off <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], off);
    // From here on in units in which a row's sum is about 1, wherever the scale of
    // its values put the reference; P's 2^12 goes too.
    const int lx = l[r] > 0.f && l[r] < INFINITY ? max(-100, min(100, scale_log2(l[r]) - (int)kPShift)) : 0;
    unit[r] = pow2f(-(int)kPShift - lx);
    if (Narrow ? g == 0 : c == 0) {
      join_m[warp][row_of(r)] = m[r] + (float)lx;
      join_l[warp][row_of(r)] = l[r] * unit[r];
    }
  }
  __syncthreads();  // every warp is done with the ring
  float* po = reinterpret_cast<float*>(smem) + (size_t)warp * kRows * DT;
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int t = 0; t < kOTiles; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // Column 2c + i of tile t: dim (2c + i) * kVBytes + t.  Narrow: row g + 8i of
        // tile t: dim g * kVBytes + 2t + i.
        const float y = o[t][Narrow ? 2 * i + r : 2 * r + i];
        po[row_of(r) * DT + (Narrow ? g * L::kVBytes + 2 * t + i : (2 * c + i) * L::kVBytes + t)] =
            y * unit[r];
      }
  __syncthreads();
  constexpr int kPerRow = DT / 4, kJoinRows = Narrow ? 8 : kRows;
  auto store_row = [&](int pr, int col, const float(&acc)[4], float sum, float gm) {
    const int qh = (int)(((uint64_t)pr * p.q_magic) >> 40);
    const int head = kvh * p.group + qh, t = pr - qh * p.q_len;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    __nv_bfloat162 lo = __floats2bfloat162_rn(acc[0] * inv, acc[1] * inv);
    __nv_bfloat162 hi = __floats2bfloat162_rn(acc[2] * inv, acc[3] * inv);
    uint2 w;
    w.x = *reinterpret_cast<uint32_t*>(&lo);
    w.y = *reinterpret_cast<uint32_t*>(&hi);
    *reinterpret_cast<uint2*>(p.out + req * p.out_bs + ((int64_t)t * p.heads + head) * d + col) = w;
    if (p.lse && col == 0)
      p.lse[((int64_t)req * p.heads + head) * p.q_len + t] =
          sum == 0.f ? -INFINITY : (gm == -INFINITY ? sum : (gm + log2f(sum)) * 0.69314718055994531f);
  };
  for (int i = threadIdx.x; i < kJoinRows * kPerRow; i += kWarps * 32) {
    const int row = i / kPerRow, col = (i % kPerRow) * 4;
    const int pr = blockIdx.y * kRows + row;
    if (pr >= packed || col >= d) continue;
    float gm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) gm = fmaxf(gm, join_m[w][row]);
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = join_m[w][row];
      const float f = mw == -INFINITY ? 0.f : exp2f(mw - gm);
      const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem) +
                                                        ((size_t)w * kRows + row) * DT + col);
      sum += f * join_l[w][row];  // a NaN passes even where f is 0
      acc[0] += f * y.x;
      acc[1] += f * y.y;
      acc[2] += f * y.z;
      acc[3] += f * y.w;
    }
    const int qh = (int)(((uint64_t)pr * p.q_magic) >> 40);
    const int head = kvh * p.group + qh, t = pr - qh * p.q_len;
    if (p.splits == 1) {
      store_row(pr, col, acc, sum, gm);
    } else if (p.splits <= kMaxCluster) {
      *reinterpret_cast<float4*>(smem + L::kRows0 + (row * DT + col) * 4) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (col == 0) row_ml[row] = make_float2(gm, sum);
    } else {
      const int64_t idx = (((int64_t)req * p.splits + split) * p.heads + head) * p.q_len + t;
      *reinterpret_cast<float4*>(p.part_o + idx * d + col) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (col == 0) {
        p.part_ml[idx * 2] = gm;
        p.part_ml[idx * 2 + 1] = sum;
      }
    }
  }
  if (p.splits > 1 && p.splits <= kMaxCluster) {
    // The cluster is the row tile's key ranges: each CTA joins a part of the
    // rows from all of them, in range order.
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int i = (int)cluster.block_rank() * kWarps * 32 + threadIdx.x; i < kJoinRows * kPerRow;
         i += p.splits * kWarps * 32) {
      const int row = i / kPerRow, col = (i % kPerRow) * 4;
      const int pr = blockIdx.y * kRows + row;
      if (pr >= packed || col >= d) continue;
      float2 ml[kMaxCluster];
      float4 y[kMaxCluster];
      float gm = -INFINITY;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {
        if (r >= p.splits) break;
        ml[r] = *cluster.map_shared_rank(row_ml + row, r);
        y[r] = *cluster.map_shared_rank(reinterpret_cast<const float4*>(smem + L::kRows0 + (row * DT + col) * 4), r);
        gm = fmaxf(gm, ml[r].x);
      }
      float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {
        if (r >= p.splits) break;
        const float f = ml[r].x == -INFINITY ? 0.f : exp2f(ml[r].x - gm);
        sum += f * ml[r].y;  // a NaN passes even where f is 0
        acc[0] += f * y[r].x;
        acc[1] += f * y[r].y;
        acc[2] += f * y[r].z;
        acc[3] += f * y[r].w;
      }
      store_row(pr, col, acc, sum, gm);
    }
    cluster.sync();  // no CTA leaves while its rows may be read
  }
}

// A joined row's output, four dims a lane, and its log-sum-exp.
__device__ __forceinline__ void store_joined(const Kv8Attn& p, int64_t pair, int64_t req, int64_t at, int lane,
                                             const float (&acc)[4], float sum, float gm) {
  const int head = (int)(at / p.q_len), t = (int)(at % p.q_len), d = p.c.d;
  if (p.lse && lane == 0)
    p.lse[pair] = sum == 0.f ? -INFINITY : (gm == -INFINITY ? sum : (gm + log2f(sum)) * 0.69314718055994531f);
  if (lane * 4 >= d) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  __nv_bfloat162 lo = __floats2bfloat162_rn(acc[0] * inv, acc[1] * inv);
  __nv_bfloat162 hi = __floats2bfloat162_rn(acc[2] * inv, acc[3] * inv);
  uint2 w;
  w.x = *reinterpret_cast<uint32_t*>(&lo);
  w.y = *reinterpret_cast<uint32_t*>(&hi);
  *reinterpret_cast<uint2*>(p.out + req * p.out_bs + ((int64_t)t * p.heads + head) * d + lane * 4) = w;
}

// Joins up to N key ranges, a warp per (request, head, row): everything is
// loaded at once.
template <int N>
__global__ void __launch_bounds__(256)
kv8_merge_few_kernel(Kv8Attn p) {
  pdl_wait();
  pdl_trigger();
  const int64_t per_req = (int64_t)p.heads * p.q_len;
  const int lane = threadIdx.x & 31, d = p.c.d;
  const int64_t pair = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (pair >= per_req * p.batch) return;
  const int64_t req = pair / per_req, at = pair - req * per_req;
  const int64_t base = req * p.splits * per_req + at;
  float2 ml[N];
  float4 y[N];
#pragma unroll
  for (int s = 0; s < N; ++s) {
    ml[s] = s < p.splits ? *reinterpret_cast<const float2*>(p.part_ml + (base + s * per_req) * 2)
                         : make_float2(-INFINITY, 0.f);
    y[s] = s < p.splits && lane * 4 < d
               ? *reinterpret_cast<const float4*>(p.part_o + (base + s * per_req) * d + lane * 4)
               : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float gm = -INFINITY;
#pragma unroll
  for (int s = 0; s < N; ++s) gm = fmaxf(gm, ml[s].x);
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll
  for (int s = 0; s < N; ++s) {
    const float f = ml[s].x == -INFINITY ? 0.f : exp2f(ml[s].x - gm);
    sum += f * ml[s].y;  // a NaN passes even where f is 0
    acc[0] += f * y[s].x;
    acc[1] += f * y[s].y;
    acc[2] += f * y[s].z;
    acc[3] += f * y[s].w;
  }
  store_joined(p, pair, req, at, lane, acc, sum, gm);
}

// Joins the key ranges: W warps per (request, head, row), four dims a lane.
// Each warp adds every W-th range, eight loads in flight (one warp that walked
// 74 ranges of a 131,072-token context took 16 us); the warps' sums are added
// in warp order, so the same ranges give the same bits.
template <int W>
__global__ void __launch_bounds__(256)
kv8_merge_kernel(Kv8Attn p) {
  pdl_wait();
  pdl_trigger();
  __shared__ float4 part[8][32];
  const int64_t per_req = (int64_t)p.heads * p.q_len;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = warp % W;
  const int64_t pair = (int64_t)blockIdx.x * (8 / W) + warp / W;
  const bool on = pair < per_req * p.batch;
  const int64_t req = on ? pair / per_req : 0, at = on ? pair % per_req : 0;
  const int64_t base = req * p.splits * per_req + at;
  const int d = p.c.d, splits = on ? p.splits : 0;
  constexpr int kPer = kMaxSplits / 32;  // ranges of a lane
  float2 ml[kPer];
  float gm = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int s = i * 32 + lane;
    ml[i] = s < splits ? *reinterpret_cast<const float2*>(p.part_ml + (base + s * per_req) * 2)
                       : make_float2(-INFINITY, 0.f);
    gm = fmaxf(gm, ml[i].x);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const float w = ml[i].x == -INFINITY ? 0.f : exp2f(ml[i].x - gm);
    sum += w * ml[i].y;  // a NaN passes even where w is 0
    const int n = min(32, splits - i * 32);
#pragma unroll 8
    for (int j = mine; j < n; j += W) {
      const float f = __shfl_sync(0xffffffffu, w, j);
      if (lane * 4 < d) {
        const float4 y =
            *reinterpret_cast<const float4*>(p.part_o + (base + (int64_t)(i * 32 + j) * per_req) * d + lane * 4);
        acc[0] += f * y.x;
        acc[1] += f * y.y;
        acc[2] += f * y.z;
        acc[3] += f * y.w;
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  part[warp][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  if (mine != 0) return;
#pragma unroll
  for (int i = 1; i < W; ++i) {
    const float4 y = part[warp + i][lane];
    acc[0] += y.x;
    acc[1] += y.y;
    acc[2] += y.z;
    acc[3] += y.w;
  }
  if (on) store_joined(p, pair, req, at, lane, acc, sum, gm);
}

template <int N>
int launch_merge_few(const Kv8Attn& p, cudaStream_t stream) {
  const int64_t pairs = (int64_t)p.batch * p.heads * p.q_len;
  SF_CHECK_CUDA(launch_pdl(kv8_merge_few_kernel<N>, dim3((unsigned)((pairs + 7) / 8)), dim3(256), 0, stream, p));
  SF_CHECK_LAUNCH();
  ++kv8_launches();
  return SF_OK;
}

template <int W>
int launch_merge(const Kv8Attn& p, cudaStream_t stream) {
  const int64_t pairs = (int64_t)p.batch * p.heads * p.q_len;
  SF_CHECK_CUDA(launch_pdl(kv8_merge_kernel<W>, dim3((unsigned)((pairs * W + 7) / 8)), dim3(256), 0, stream, p));
  SF_CHECK_LAUNCH();
  ++kv8_launches();
  return SF_OK;
}

template <int DT, bool Full, bool Narrow>
int launch_mma(const Kv8Attn& p, cudaStream_t stream) {
  static std::atomic<unsigned long long> configured{0};
  if (int rc = once_per_device(configured, [] {
        SF_CHECK_CUDA(cudaFuncSetAttribute(kv8_attn_kernel<DT, Full, Narrow>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           Layout<DT>::kSmem));
        return SF_OK;
      }))
    return rc;
  const int64_t tiles = ((int64_t)p.group * p.q_len + kRows - 1) / kRows;
  SF_CHECK_ARG(tiles < 65536 && (int64_t)p.splits * p.batch < 65536, "too many query rows or requests");
  const dim3 grid((unsigned)p.c.hkv, (unsigned)tiles, (unsigned)(p.splits * p.batch));
  if (p.splits > 1 && p.splits <= kMaxCluster)
    SF_CHECK_CUDA(launch_pdl_cluster3(kv8_attn_kernel<DT, Full, Narrow>, grid, dim3(kWarps * 32), Layout<DT>::kSmem,
                                      stream, dim3(1, 1, (unsigned)p.splits), p));
  else
    SF_CHECK_CUDA(launch_pdl(kv8_attn_kernel<DT, Full, Narrow>, grid, dim3(kWarps * 32), Layout<DT>::kSmem, stream, p));
  SF_CHECK_LAUNCH();
  ++kv8_launches();
  return SF_OK;
}

template <int DT, bool Full>
int launch_rows(const Kv8Attn& p, cudaStream_t stream) {
  return (int64_t)p.group * p.q_len <= 8 ? launch_mma<DT, Full, true>(p, stream)
                                         : launch_mma<DT, Full, false>(p, stream);
}

size_t partial_bytes(const Kv8Split& s, int batch, int heads, int head_dim, int64_t q_len) {
  return s.splits == 1 ? 0 : (size_t)batch * s.splits * heads * q_len * (head_dim + 2) * sizeof(float);
}

}  // namespace

// Three resident CTAs per SM, in short contexts one cluster a row tile; a range is at least one step of the four warps.
Kv8Split kv8_split_mma(int batch, int hkv, int64_t packed, int64_t kv_len) {
  const int64_t units = (int64_t)batch * hkv * ((packed + kRows - 1) / kRows);
  const int64_t steps = (kv_len + kStep - 1) / kStep;
  int64_t want = std::max<int64_t>(1, 3 * (int64_t)num_sms() / units);
  if (steps <= kClusterSteps) want = std::min<int64_t>(want, kMaxCluster);
  want = std::min<int64_t>(want, std::min<int64_t>(kMaxSplits, std::max<int64_t>(1, steps)));
  const int64_t per = std::max<int64_t>(1, (steps + want - 1) / want);
  return {(int)std::max<int64_t>(1, (steps + per - 1) / per), (int)(per * kStep)};
}

}  // namespace sf

extern "C" size_t sf_kv8_attention_workspace_bytes(int batch, int num_heads, int num_kv_heads, int head_dim,
                                                  int64_t q_len, int64_t sealed, int64_t tail) {
  using namespace sf;
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || head_dim <= 0 ||
      head_dim > 128 || q_len <= 0 || sealed < 0 || tail < 0 || sealed + tail <= 0 || q_len >= (1 << 30) ||
      sealed >= (1 << 30) || tail >= (1 << 30))
    return 0;
  const int64_t kv_len = sealed + tail;
  // Enough for either kernel: which one runs depends on the cache's strides too.
  const int64_t packed = (int64_t)(num_heads / num_kv_heads) * q_len;
  const Kv8Split mma = kv8_split_mma(batch, num_kv_heads, packed, kv_len);
  size_t need = mma.splits <= kMaxCluster ? 0 : partial_bytes(mma, batch, num_heads, head_dim, q_len);
  if (kv8_use_tc(head_dim, packed, kv_len))
    need = std::max(need, partial_bytes(kv8_split_tc(batch, num_kv_heads, packed, kv_len), batch, num_heads, head_dim,
                                        q_len) +
                              15 + kv8_prep_layout(nullptr, nullptr, false, (int64_t)batch * num_kv_heads, packed, sealed, kv_len));
  return need;
}

extern "C" int sf_kv8_tree_attention(const void* q, int64_t q_batch_stride, int64_t q_head_stride,
                                     int64_t q_row_stride, int num_heads, int64_t q_len, const sf_kv8_rows* rows,
                                     const uint32_t* tree_bits, int bit_words, int64_t bits_batch_stride,
                                     int64_t prefix_len, float scale, void* out, int64_t out_batch_stride, float* lse,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  using namespace sf;
  kv8_launches() = 0;
  if (int rc = kv8_check(rows, true)) return rc;
  const int64_t kv_len = rows->sealed + rows->tail;
  SF_CHECK_ARG(num_heads > 0 && num_heads % rows->num_kv_heads == 0,
               "num_heads must be a positive multiple of num_kv_heads");
  SF_CHECK_ARG(q_len >= 0 && prefix_len >= 0 && prefix_len <= kv_len && kv_len < (1 << 30), "invalid lengths");
  const int group = num_heads / rows->num_kv_heads;
  SF_CHECK_ARG((int64_t)group * q_len < (1 << 20), "too many query rows");
  if (q_len == 0) return SF_OK;
  SF_CHECK_ARG(scale > 0.f && scale < INFINITY, "scale must be positive and finite");
  SF_CHECK_ARG(q && out, "null pointer argument");
  SF_CHECK_ARG(kv_len == prefix_len || (tree_bits && (int64_t)bit_words * 32 >= kv_len - prefix_len),
               "tree_bits must cover the keys from prefix_len on");
  SF_CHECK_ARG(aligned16(q) && q_batch_stride % 8 == 0 && q_head_stride % 8 == 0 && q_row_stride % 8 == 0,
               "q rows must be 16-byte aligned");
  SF_CHECK_ARG(aligned16(out) && out_batch_stride % 8 == 0, "out must be 16-byte aligned");
  SF_CHECK_ARG(kv8_apart(rows->batch, out_batch_stride, 1, 0, q_len * num_heads * rows->head_dim),
               "requests of out must not overlap");
  const size_t need = sf_kv8_attention_workspace_bytes(rows->batch, num_heads, rows->num_kv_heads, rows->head_dim,
                                                       q_len, rows->sealed, rows->tail);
  if (workspace_bytes < need || (need && !workspace))
    return set_error(SF_ERR_WORKSPACE, "8-bit cache attention workspace needs %zu bytes", need);
  SF_CHECK_ARG(need == 0 || aligned16(workspace), "workspace must be 16-byte aligned");
  Kv8Attn p;
  p.c = kv8_view(*rows);
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_bs = q_batch_stride;
  p.q_hs = q_head_stride;
  p.q_rs = q_row_stride;
  p.bits = kv_len == prefix_len ? nullptr : tree_bits;
  p.words = bit_words;
  p.bits_bs = bits_batch_stride;
  p.batch = rows->batch;
  p.heads = num_heads;
  p.group = group;
  p.q_len = (int)q_len;
  p.q_magic = ((1ull << 40) + (uint64_t)q_len - 1) / (uint64_t)q_len;
  p.kv_len = (int)kv_len;
  p.prefix = (int)prefix_len;
  p.scale = scale;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_bs = out_batch_stride;
  p.lse = lse;
  const int64_t packed = (int64_t)group * q_len;
  const bool tc = kv8_use_tc(rows->head_dim, packed, kv_len) && kv8_tc_layout(p.c, rows->batch);
  const Kv8Split s = tc ? kv8_split_tc(rows->batch, rows->num_kv_heads, packed, kv_len)
                        : kv8_split_mma(rows->batch, rows->num_kv_heads, packed, kv_len);
  p.splits = s.splits;
  p.keys_per_split = s.keys_per_split;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + (size_t)rows->batch * s.splits * num_heads * q_len * rows->head_dim;
  cudaStream_t st = as_stream(stream);
  int rc;
  if (tc)
    rc = kv8_attention_tc(p, static_cast<uint8_t*>(workspace) +
                                 (partial_bytes(s, rows->batch, num_heads, rows->head_dim, q_len) + 15) / 16 * 16,
                          st);
  else
    rc = rows->head_dim == 128  ? launch_rows<128, true>(p, st)
         : rows->head_dim > 64  ? launch_rows<128, false>(p, st)
         : rows->head_dim == 64 ? launch_rows<64, true>(p, st)
                                : launch_rows<64, false>(p, st);
  if (rc || s.splits == 1 || (!tc && s.splits <= kMaxCluster)) return rc;
  if (s.splits <= 4) return launch_merge_few<4>(p, st);
  if (s.splits <= 16) return launch_merge_few<16>(p, st);
  return s.splits <= 32 ? launch_merge<4>(p, st) : launch_merge<8>(p, st);
}
