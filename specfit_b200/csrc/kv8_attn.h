// Parameters shared by the kernels that attend to the 8-bit KV cache and the
// merge of their partial results.
#pragma once

#include <cuda.h>

#include "kv8.cuh"
#include "tree_attn.h"

namespace sf {

struct Kv8Attn {
  Kv8Rows c;
  const __nv_bfloat16* q;
  int64_t q_bs, q_hs, q_rs;
  const uint32_t* bits;  // [batch, q_len, words] over the keys from prefix_len on; nullable
  int words;
  int64_t bits_bs;
  int batch, heads, group, q_len;
  // ceil(2^40 / q_len): n / q_len = (n * q_magic) >> 40 for n, q_len < 2^20.
  // (q_magic * q_len exceeds 2^40 by less than q_len, so the quotient by less
  // than n / 2^40 < 1 / q_len.)
  uint64_t q_magic;
  int kv_len, prefix;
  float scale, scale_log2;  // the softmax scale, and times log2(e)
  int splits, keys_per_split;
  float* part_o;   // [batch, splits, heads, q_len, D] unnormalised
  float* part_ml;  // [batch, splits, heads, q_len, 2]: (reference max, sum), base 2
  __nv_bfloat16* out;  // [batch, q_len, heads, D]
  int64_t out_bs;
  float* lse;      // [batch, heads, q_len]; nullable
};

// Visibility of keys key0 + i, i in [0, 64), for one query row, as bit i.
__device__ __forceinline__ uint64_t kv8_window(const Kv8Attn& p, const uint32_t* rbits, int key0) {
  uint64_t w;
  if (rbits) {
    w = tree_mask_window(rbits, p.words, key0 - p.prefix);
  } else {
    const int n = p.prefix - key0;
    w = n >= 64 ? ~0ull : (n <= 0 ? 0ull : (1ull << n) - 1);
  }
  const int valid = p.kv_len - key0;
  if (valid < 64) w &= valid <= 0 ? 0ull : (1ull << valid) - 1;
  return w;
}

// A row's reference is the largest of a score plus log2 of its value's scale, or
// this where that is less: sums of probabilities, in units of the reference,
// then stay below 2^(75 + log2 of the keys), and only values below 2^-75 or so, where
// a row sees no larger ones, lose digits.
constexpr int kMinValueScale = -60;

// Key ranges per (request, KV head, row tile) for `units` such units of work.
struct Kv8Split {
  int splits, keys_per_split;
};

// The warp-level kernel (kv8_attn.cu).
Kv8Split kv8_split_mma(int batch, int hkv, int64_t packed_rows, int64_t kv_len);

// The tcgen05 kernel (kv8_attn_tc.cu), for many query rows.  `splits` counts
// partial results: with one row tile a CTA writes two.
bool kv8_use_tc(int head_dim, int64_t packed_rows, int64_t kv_len);
bool kv8_tc_layout(const Kv8Rows& c, int batch);
Kv8Split kv8_split_tc(int batch, int hkv, int64_t packed_rows, int64_t kv_len);
int kv8_attention_tc(const Kv8Attn& p, void* prep, cudaStream_t stream);

// What a first kernel lays out for the tcgen05 kernels, for each (request, KV
// head) bh: the query tiles and the blocks of 128 keys that hold tail rows, as
// images of the kernels' shared-memory tiles.
struct Kv8Prep {
  uint8_t* q;    // [bh][tiles][hi, lo: 128 rows x 128, e4m3, swizzled]
  uint8_t* k;    // [bh][blocks][hi, lo], the blocks from key `first` on
  float* kf;     // [bh][blocks * 128]: a key's scale; NaN for a key that holds one
  // For attention (null otherwise):
  uint8_t* v;    // [bh][blocks][128 keys x 128, fp16 in units of `vf`, swizzled]
  float* vf;     // [bh][blocks * 128]: a value row's scale
  float* qf;     // [bh][tiles * 128]: the power of two taken out of a query row; NaN for a row that holds one
  // For the mass (null otherwise):
  float* rowc;   // [bh][tiles][2][128]: that power times scale * log2(e); -lse * log2(e)
  int tiles, blocks, first;
};
// Fills `w` (nullable) with places from `base` (16-byte aligned) on; returns the bytes.
size_t kv8_prep_layout(Kv8Prep* w, void* base, bool for_mass, int64_t heads, int64_t packed_rows, int64_t sealed,
                       int64_t kv_len);
int kv8_prep(const Kv8Attn& p, const Kv8Prep& w, cudaStream_t stream);
// Tensor map of K's codes: boxes of 128 keys.
int kv8_key_map(CUtensorMap* map, const Kv8Rows& c, int batch);

// The mass on tcgen05 (kv8_mass_tc.cu).
bool kv8_mass_use_tc(int head_dim, int64_t packed_rows);
size_t kv8_mass_tc_bytes(int64_t heads, int64_t packed_rows, int64_t sealed, int64_t kv_len);
int kv8_mass_tc(const Kv8Attn& p, float* mass, int64_t m_bs, int64_t m_hs, void* prep, cudaStream_t stream);
int kv8_mass_tc_status(int* status, int reset);
int kv8_tc_status(int* status, int reset);

}  // namespace sf
