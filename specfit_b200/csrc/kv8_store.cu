// Writing the 8-bit KV cache: sealing bf16 rows, reading rows back as bf16,
// and moving the kept rows of an eviction into a new cache.
//
// All three are streams over rows, bound by memory: sealing reads 2 bytes and
// writes 1 per element, compaction reads a kept row's 1 byte and writes 1.
// One CTA owns one block of tokens of one head of K or of V: it holds the
// whole block (at most 128 x 128 values) in registers as bf16 pairs, finds
// the block's largest magnitude, and writes codes and scale, so each input
// byte is read once.  The magnitudes are compared as 15-bit integers (bf16
// orders like its bits), two per instruction, which also finds NaN and
// infinity (the largest integers).
//
// Sealing 32,768 tokens of four heads: 15 us, 6.7 TB/s of bytes read and written.
// Reading them back: 31 us, 3.2 TB/s.  Compaction of 16 heads to 8,192 tokens each:
// 25 us, 2.7 TB/s; there the chain of a CTA is what bounds it (indices, rows, the
// block's maximum, codes), of which six fit on an SM, so its threads hold few
// registers and load all at once.
#include <algorithm>
#include <memory>
#include <new>

#include "kv8.cuh"

namespace sf {

int& kv8_launches() {
  static thread_local int n = 0;
  return n;
}

int kv8_check(const sf_kv8_rows* r, bool need_values) {
  SF_CHECK_ARG(r != nullptr, "null pointer argument");
  SF_CHECK_ARG(r->batch > 0 && r->num_kv_heads > 0 && (int64_t)r->batch * r->num_kv_heads <= 65535,
               "batch and num_kv_heads must be positive, their product at most 65535");
  SF_CHECK_ARG(r->head_dim > 0 && r->head_dim <= 128 && r->head_dim % 16 == 0,
               "head_dim must be a multiple of 16 in [16, 128]");
  SF_CHECK_ARG(r->block_tokens == 32 || r->block_tokens == 64 || r->block_tokens == 128,
               "block_tokens must be 32, 64 or 128");
  SF_CHECK_ARG(r->sealed >= 0 && r->tail >= 0 && r->sealed % r->block_tokens == 0 &&
                   r->sealed < (1 << 30) && r->tail < (1 << 30),
               "sealed must be a whole number of blocks, lengths below 2^30");
  if (r->sealed > 0) {
    SF_CHECK_ARG(r->k_codes && r->k_scale && (!need_values || (r->v_codes && r->v_scale)), "null pointer argument");
    SF_CHECK_ARG(aligned16(r->k_codes) && (!need_values || aligned16(r->v_codes)) &&
                     r->code_batch_stride % 16 == 0 && r->code_head_stride % 16 == 0,
                 "codes must be 16-byte aligned");
  }
  if (r->tail > 0) {
    SF_CHECK_ARG(r->k_tail && (!need_values || r->v_tail), "null pointer argument");
    SF_CHECK_ARG(aligned16(r->k_tail) && (!need_values || aligned16(r->v_tail)) &&
                     r->tail_batch_stride % 8 == 0 && r->tail_head_stride % 8 == 0,
                 "tail rows must be 16-byte aligned");
  }
  return SF_OK;
}

namespace {

constexpr int kThreads = 256;

// Row and 8-element chunk of element chunk i of a block: rows of `per_row` chunks.
__device__ __forceinline__ void row_chunk(int i, int per_row, int& row, int& ch) {
  if (per_row == 16) {
    row = i >> 4;
    ch = i & 15;
  } else if (per_row == 8) {
    row = i >> 3;
    ch = i & 7;
  } else {
    row = i / per_row;
    ch = i - row * per_row;
  }
}

// Where the rows of a block come from: bf16 rows in order (sealing) ...
struct SourceRows {
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  int64_t bs, hs, rs;
};
// ... or kept rows of a cache, by index (compaction).
struct SourceKept {
  Kv8Rows c;
  const int32_t* keep;  // [batch * hkv, n]
  int64_t n;
  const float* mass;    // nullable
  float* mass_out;
  int64_t m_bs, m_hs, mo_bs, mo_hs;
};

struct Target {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  __nv_bfloat16* kt;
  __nv_bfloat16* vt;
  int64_t c_bs, c_hs, s_bs, s_hs, t_bs, t_hs;
  int64_t first_block;  // the block that grid x = 0 writes
  int64_t full_blocks;  // blocks of this launch; the CTA after them writes the tail
  int hkv, d, block;
};

// 8 codes of one scale as 8 bf16 values (exact; NaN for a NaN scale).
__device__ __forceinline__ uint4 codes_to_bf16(uint2 c, float scale) {
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t w = i ? c.y : c.x;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t h = j ? e4m3x2_hi_to_f16x2(w) : e4m3x2_to_f16x2(w);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * scale, f.y * scale);
      o[i * 2 + j] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Eight elements (chunk ch of cache row `row`) of a cache as bf16.
__device__ __forceinline__ uint4 cache_chunk(const Kv8Rows& c, int b, int h, bool is_v, int64_t row, int ch) {
  if (row < c.sealed) {
    const uint8_t* codes = (is_v ? c.v : c.k) + b * c.c_bs + h * c.c_hs + row * c.d + ch * 8;
    const float* sc = (is_v ? c.vs : c.ks) + b * c.s_bs + h * c.s_hs + (row >> c.block_shift);
    return codes_to_bf16(*reinterpret_cast<const uint2*>(codes), *sc);
  }
  const __nv_bfloat16* t = (is_v ? c.vt : c.kt) + b * c.t_bs + h * c.t_hs + (row - c.sealed) * c.d + ch * 8;
  return *reinterpret_cast<const uint4*>(t);
}

// This thread's chunks of the rows from row0 on, zeros past the last.
template <int kChunks>
__device__ __forceinline__ void load_rows(const SourceRows& s, int b, int h, bool is_v, int64_t row0, int chunks,
                                          int per_row, uint4 (&x)[kChunks]) {
  const __nv_bfloat16* from = (is_v ? s.v : s.k) + b * s.bs + h * s.hs;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int i = threadIdx.x + j * kThreads;
    int r, ch;
    row_chunk(i, per_row, r, ch);
    x[j] = i < chunks ? *reinterpret_cast<const uint4*>(from + (row0 + r) * s.rs + ch * 8) : make_uint4(0, 0, 0, 0);
  }
}
// Indices, then codes and scales, each for all chunks at once: a chunk after
// the other this was eight latencies instead of two.
template <int kChunks>
__device__ __forceinline__ void load_rows(const SourceKept& s, int b, int h, bool is_v, int64_t row0, int chunks,
                                          int per_row, uint4 (&x)[kChunks]) {
  const int32_t* keep = s.keep + ((int64_t)b * s.c.hkv + h) * s.n + row0;
  const uint8_t* codes = (is_v ? s.c.v : s.c.k) + b * s.c.c_bs + h * s.c.c_hs;
  const float* scales = (is_v ? s.c.vs : s.c.ks) + b * s.c.s_bs + h * s.c.s_hs;
  const __nv_bfloat16* tail = (is_v ? s.c.vt : s.c.kt) + b * s.c.t_bs + h * s.c.t_hs;
  int32_t at[kChunks];
  int r[kChunks], ch[kChunks];
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int i = threadIdx.x + j * kThreads;
    row_chunk(i, per_row, r[j], ch[j]);
    at[j] = i < chunks ? keep[r[j]] : -1;
    if (at[j] >= s.c.sealed + s.c.tail) at[j] = -1;  // not a row of the cache
  }
  uint2 c[kChunks];
  float scale[kChunks];
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const bool coded = at[j] >= 0 && at[j] < s.c.sealed;
    c[j] = coded ? *reinterpret_cast<const uint2*>(codes + (int64_t)at[j] * s.c.d + ch[j] * 8) : make_uint2(0, 0);
    scale[j] = coded ? scales[at[j] >> s.c.block_shift] : 1.f;
  }
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    x[j] = codes_to_bf16(c[j], scale[j]);  // zeros where there is no row
    if (at[j] >= s.c.sealed)
      x[j] = *reinterpret_cast<const uint4*>(tail + (at[j] - s.c.sealed) * s.c.d + ch[j] * 8);
  }
}

__device__ __forceinline__ int64_t source_rows(const SourceRows&, int64_t full) { return full; }
__device__ __forceinline__ int64_t source_rows(const SourceKept& s, int64_t) { return s.n; }

__device__ __forceinline__ void move_mass(const SourceRows&, int, int, int64_t, int) {}
__device__ __forceinline__ void move_mass(const SourceKept& s, int b, int h, int64_t row0, int rows) {
  if (!s.mass) return;
  for (int i = threadIdx.x; i < rows; i += kThreads) {
    const int32_t at = s.keep[((int64_t)b * s.c.hkv + h) * s.n + row0 + i];
    const bool ok = at >= 0 && at < s.c.sealed + s.c.tail;
    s.mass_out[b * s.mo_bs + h * s.mo_hs + row0 + i] = ok ? s.mass[b * s.m_bs + h * s.m_hs + at] : 0.f;
  }
}

// grid: (blocks [+ 1 for the tail], batch * hkv, 2: K and V).  kChunks: 16-byte
// bf16 chunks that a thread holds, block * D / 8 / kThreads rounded up; few of
// them leave registers for more CTAs on an SM.
template <typename Source, int kChunks>
__global__ void __launch_bounds__(kThreads, kChunks <= 4 ? 6 : 4)
kv8_write_kernel(Source src, Target t) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t tops[kThreads / 32];
  const int h = blockIdx.y % t.hkv, b = blockIdx.y / t.hkv;
  const bool is_v = blockIdx.z != 0;
  const int64_t row0 = (int64_t)blockIdx.x * t.block;
  const int per_row = t.d >> 3;  // 8-element chunks of a row
  const int64_t n = source_rows(src, t.full_blocks * t.block);
  const int rows = (int)min((int64_t)t.block, n - row0);
  const int chunks = rows * per_row;
  uint4 x[kChunks];
  load_rows(src, b, h, is_v, row0, chunks, per_row, x);
  if (!is_v) move_mass(src, b, h, row0, rows);
  if ((int64_t)blockIdx.x >= t.full_blocks) {  // rows that do not fill a block stay bf16
    __nv_bfloat16* dst = (is_v ? t.vt : t.kt) + b * t.t_bs + h * t.t_hs;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      const int i = threadIdx.x + j * kThreads;
      if (i < chunks) *reinterpret_cast<uint4*>(dst + (int64_t)i * 8) = x[j];
    }
    return;
  }
  uint32_t top2 = 0;  // two 15-bit magnitudes
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    top2 = __vmaxu2(top2, x[j].x & 0x7fff7fffu);
    top2 = __vmaxu2(top2, x[j].y & 0x7fff7fffu);
    top2 = __vmaxu2(top2, x[j].z & 0x7fff7fffu);
    top2 = __vmaxu2(top2, x[j].w & 0x7fff7fffu);
  }
  uint32_t top = max(top2 & 0xffffu, top2 >> 16);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) top = max(top, tops[w]);
  const bool bad = top >= 0x7f80u;  // a NaN or an infinity
  const int e = bad ? 0 : kv8_exponent(top);
  const float inv = pow2f(-e);
  const int64_t blk = t.first_block + blockIdx.x;
  if (threadIdx.x == 0)
    (is_v ? t.vs : t.ks)[b * t.s_bs + h * t.s_hs + blk] = bad ? __int_as_float(0x7fc00000) : pow2f(e);
  uint8_t* dst = (is_v ? t.v : t.k) + b * t.c_bs + h * t.c_hs + blk * t.block * t.d;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int i = threadIdx.x + j * kThreads;
    if (i >= chunks) continue;
    const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
    uint32_t o[2] = {0, 0};
    if (!bad) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        // Exact products (a power of two), one rounding to nearest-even.
        const float2 f = make_float2(__uint_as_float(w[p] << 16) * inv, __uint_as_float(w[p] & 0xffff0000u) * inv);
        o[p >> 1] |= (uint32_t)__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3) << (16 * (p & 1));
      }
    }
    *reinterpret_cast<uint2*>(dst + (int64_t)i * 8) = make_uint2(o[0], o[1]);
  }
}

// Rows [first, first + count) of a cache as bf16; grid (chunk blocks, batch * hkv, 2).
__global__ void __launch_bounds__(kThreads)
kv8_read_kernel(Kv8Rows c, int64_t first, int64_t count, __nv_bfloat16* __restrict__ k_out,
                __nv_bfloat16* __restrict__ v_out, int64_t o_bs, int64_t o_hs) {
  pdl_wait();
  pdl_trigger();
  const int h = blockIdx.y % c.hkv, b = blockIdx.y / c.hkv;
  const bool is_v = blockIdx.z != 0;
  const int per_row = c.d >> 3;
  __nv_bfloat16* dst = (is_v ? v_out : k_out) + b * o_bs + h * o_hs;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < count * per_row;
       i += (int64_t)gridDim.x * kThreads)
    *reinterpret_cast<uint4*>(dst + i * 8) = cache_chunk(c, b, h, is_v, first + i / per_row, (int)(i % per_row));
}

template <typename Source>
int launch_write(const Source& src, const Target& t, dim3 grid, cudaStream_t stream) {
  const int chunks = (t.block * t.d / 8 + kThreads - 1) / kThreads;
  if (chunks <= 2)
    SF_CHECK_CUDA(launch_pdl(kv8_write_kernel<Source, 2>, grid, dim3(kThreads), 0, stream, src, t));
  else if (chunks <= 4)
    SF_CHECK_CUDA(launch_pdl(kv8_write_kernel<Source, 4>, grid, dim3(kThreads), 0, stream, src, t));
  else
    SF_CHECK_CUDA(launch_pdl(kv8_write_kernel<Source, 8>, grid, dim3(kThreads), 0, stream, src, t));
  SF_CHECK_LAUNCH();
  return SF_OK;
}

Target make_target(const sf_kv8_rows& r, int64_t first_block, int64_t full_blocks) {
  Target t;
  t.k = static_cast<uint8_t*>(r.k_codes);
  t.v = static_cast<uint8_t*>(r.v_codes);
  t.ks = r.k_scale;
  t.vs = r.v_scale;
  t.kt = static_cast<__nv_bfloat16*>(r.k_tail);
  t.vt = static_cast<__nv_bfloat16*>(r.v_tail);
  t.c_bs = r.code_batch_stride;
  t.c_hs = r.code_head_stride;
  t.s_bs = r.scale_batch_stride;
  t.s_hs = r.scale_head_stride;
  t.t_bs = r.tail_batch_stride;
  t.t_hs = r.tail_head_stride;
  t.first_block = first_block;
  t.full_blocks = full_blocks;
  t.hkv = r.num_kv_heads;
  t.d = r.head_dim;
  t.block = r.block_tokens;
  return t;
}

// Memory of one buffer: `extent` bytes for each of count[0] * count[1] * count[2]
// pieces (requests, heads, rows that do not follow each other), stride bytes apart.
struct Region {
  const void* at = nullptr;
  int64_t extent = 0, count[3] = {1, 1, 1}, stride[3] = {0, 0, 0};
  int64_t pieces() const { return at == nullptr || extent <= 0 ? 0 : count[0] * count[1] * count[2]; }
  uintptr_t start(int64_t n) const {
    const int64_t k = n % count[2], j = n / count[2] % count[1], i = n / count[2] / count[1];
    return reinterpret_cast<uintptr_t>(at) + (uintptr_t)(i * stride[0] + j * stride[1] + k * stride[2]);
  }
  // From the first byte to behind the last.
  void span(uintptr_t& lo, uintptr_t& hi) const {
    lo = hi = reinterpret_cast<uintptr_t>(at);
    for (int i = 0; i < 3; ++i) (stride[i] < 0 ? lo : hi) += (uintptr_t)((count[i] - 1) * stride[i]);
    hi += (uintptr_t)extent;
  }
};

// Whether two buffers share memory.  Views of one buffer may lie between each
// other, so where their spans meet the pieces are compared (and taken to share
// memory if there is none to compare them in: no exception leaves a C entry).
bool meet(const Region& x, const Region& y) {
  const int64_t nx = x.pieces(), ny = y.pieces();
  if (nx == 0 || ny == 0) return false;
  uintptr_t xlo, xhi, ylo, yhi;
  x.span(xlo, xhi);
  y.span(ylo, yhi);
  if (xhi <= ylo || yhi <= xlo) return false;
  const std::unique_ptr<uintptr_t[]> at(new (std::nothrow) uintptr_t[nx]);
  if (!at) return true;
  for (int64_t i = 0; i < nx; ++i) at[i] = x.start(i);
  std::sort(at.get(), at.get() + nx);
  for (int64_t i = 0; i < ny; ++i) {
    const uintptr_t lo = y.start(i), hi = lo + (uintptr_t)y.extent;
    // The first piece of x that ends behind lo: they are all as long.
    const uintptr_t* p = std::upper_bound(at.get(), at.get() + nx, lo, [&](uintptr_t l, uintptr_t a) {
      return a + (uintptr_t)x.extent > l;
    });
    if (p != at.get() + nx && *p < hi) return true;
  }
  return false;
}

// Up to eight buffers.
struct Regions {
  Region r[8];
  int n = 0;
  void add(const void* at, int64_t extent, int64_t b, int64_t bs, int64_t h, int64_t hs, int64_t rows = 1,
           int64_t rs = 0) {
    r[n++] = Region{at, extent, {b, h, rows}, {bs, hs, rs}};
  }
  // The buffers of a cache: codes and scales of `tokens` tokens from token `first` on, and
  // `tail` rows.  `one`: keys and values are the same data, so their buffers may be
  // the same too (written twice with one content).
  void add_cache(const sf_kv8_rows& c, int64_t first, int64_t tokens, int64_t tail, bool one = false) {
    const int64_t b = c.batch, h = c.num_kv_heads, d = c.head_dim, blocks = tokens / c.block_tokens;
    for (int v = 0; v < 2; ++v) {
      const char* codes = static_cast<const char*>(v ? c.v_codes : c.k_codes);
      const float* scale = v ? c.v_scale : c.k_scale;
      const void* rows = v ? c.v_tail : c.k_tail;
      const bool again = one && v;
      if (codes && !(again && codes == c.k_codes))
        add(codes + first * d, tokens * d, b, c.code_batch_stride, h, c.code_head_stride);
      if (scale && !(again && scale == c.k_scale))
        add(scale + first / c.block_tokens, blocks * 4, b, c.scale_batch_stride * 4, h, c.scale_head_stride * 4);
      if (!(again && rows == c.k_tail)) add(rows, tail * d * 2, b, c.tail_batch_stride * 2, h, c.tail_head_stride * 2);
    }
  }
};

// Whether anything written shares memory with anything else written or read.
bool overlap(const Regions& written, const Regions& read) {
  for (int i = 0; i < written.n; ++i) {
    for (int j = i + 1; j < written.n; ++j)
      if (meet(written.r[i], written.r[j])) return true;
    for (int j = 0; j < read.n; ++j)
      if (meet(written.r[i], read.r[j])) return true;
  }
  return false;
}

bool target_apart(const sf_kv8_rows& r) {
  auto apart = [&](int64_t bs, int64_t hs, int64_t extent) {
    return kv8_apart(r.batch, bs, r.num_kv_heads, hs, extent);
  };
  return apart(r.code_batch_stride, r.code_head_stride, r.sealed * r.head_dim) &&
         apart(r.scale_batch_stride, r.scale_head_stride, r.sealed / r.block_tokens) &&
         apart(r.tail_batch_stride, r.tail_head_stride, r.tail * r.head_dim);
}

}  // namespace
}  // namespace sf

extern "C" int sf_kv8_launches(void) { return sf::kv8_launches(); }

extern "C" int sf_kv8_seal(const void* k, const void* v, int64_t batch_stride, int64_t head_stride,
                           int64_t row_stride, const sf_kv8_rows* rows, int64_t first_block, int64_t blocks,
                           void* stream) {
  using namespace sf;
  if (int rc = kv8_check(rows, true)) return rc;
  SF_CHECK_ARG(blocks >= 0 && first_block >= 0 && blocks < (1 << 24) &&
                   first_block <= rows->sealed / rows->block_tokens - blocks,
               "blocks to seal must lie within the cache's sealed rows");
  if (blocks == 0) return SF_OK;
  SF_CHECK_ARG(k && v, "null pointer argument");
  SF_CHECK_ARG(target_apart(*rows), "requests and heads of the target must not overlap");
  SF_CHECK_ARG(aligned16(k) && aligned16(v) && batch_stride % 8 == 0 && head_stride % 8 == 0 && row_stride % 8 == 0,
               "k/v rows must be 16-byte aligned");
  Regions to, from;
  to.add_cache(*rows, first_block * rows->block_tokens, blocks * rows->block_tokens, 0, k == v);
  for (const void* p : {k, v})
    from.add(p, rows->head_dim * 2, rows->batch, batch_stride * 2, rows->num_kv_heads, head_stride * 2,
             blocks * rows->block_tokens, row_stride * 2);
  SF_CHECK_ARG(!overlap(to, from), "the blocks to seal and their rows must not overlap");
  const SourceRows src{static_cast<const __nv_bfloat16*>(k), static_cast<const __nv_bfloat16*>(v), batch_stride,
                       head_stride, row_stride};
  const dim3 grid((unsigned)blocks, (unsigned)(rows->batch * rows->num_kv_heads), 2);
  return launch_write(src, make_target(*rows, first_block, blocks), grid, as_stream(stream));
}

extern "C" int sf_kv8_read(const sf_kv8_rows* rows, int64_t first, int64_t count, void* k_out, void* v_out,
                           int64_t out_batch_stride, int64_t out_head_stride, void* stream) {
  using namespace sf;
  if (int rc = kv8_check(rows, true)) return rc;
  SF_CHECK_ARG(first >= 0 && count >= 0 && count <= rows->sealed + rows->tail &&
                   first <= rows->sealed + rows->tail - count,
               "rows to read must lie within the cache");
  if (count == 0) return SF_OK;
  SF_CHECK_ARG(k_out && v_out, "null pointer argument");
  SF_CHECK_ARG(aligned16(k_out) && aligned16(v_out) && out_batch_stride % 8 == 0 && out_head_stride % 8 == 0,
               "output rows must be 16-byte aligned");
  const int64_t want = (count * (rows->head_dim / 8) + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)(want < 4096 ? want : 4096), (unsigned)(rows->batch * rows->num_kv_heads), 2);
  SF_CHECK_CUDA(launch_pdl(kv8_read_kernel, grid, dim3(kThreads), 0, as_stream(stream), kv8_view(*rows), first,
                           count, static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out),
                           out_batch_stride, out_head_stride));
  SF_CHECK_LAUNCH();
  return SF_OK;
}

extern "C" int sf_kv8_compact(const sf_kv8_rows* rows, const int32_t* keep, int64_t n, const sf_kv8_rows* out,
                              const float* mass, int64_t mass_batch_stride, int64_t mass_head_stride,
                              float* mass_out, int64_t mass_out_batch_stride, int64_t mass_out_head_stride,
                              void* stream) {
  using namespace sf;
  if (int rc = kv8_check(rows, true)) return rc;
  if (int rc = kv8_check(out, true)) return rc;
  SF_CHECK_ARG(out->batch == rows->batch && out->num_kv_heads == rows->num_kv_heads &&
                   out->head_dim == rows->head_dim && out->block_tokens == rows->block_tokens,
               "both caches must share batch, heads, head_dim and block_tokens");
  SF_CHECK_ARG(n >= 0 && n <= rows->sealed + rows->tail, "more rows kept than the cache holds");
  SF_CHECK_ARG(out->sealed == n / out->block_tokens * out->block_tokens && out->tail == n - out->sealed,
               "the new cache must hold the kept rows: whole blocks sealed, the rest as its tail");
  SF_CHECK_ARG((mass == nullptr) == (mass_out == nullptr), "pass both mass and mass_out or neither");
  if (n == 0) return SF_OK;
  SF_CHECK_ARG(keep, "null pointer argument");
  SF_CHECK_ARG(target_apart(*out) && (mass == nullptr || kv8_apart(out->batch, mass_out_batch_stride, out->num_kv_heads,
                                                                   mass_out_head_stride, n)),
               "requests and heads of the target must not overlap");
  Regions to, from;
  to.add_cache(*out, 0, out->sealed, out->tail,
               (rows->sealed == 0 || (rows->k_codes == rows->v_codes && rows->k_scale == rows->v_scale)) &&
                   (rows->tail == 0 || rows->k_tail == rows->v_tail));
  to.add(mass_out, n * 4, out->batch, mass_out_batch_stride * 4, out->num_kv_heads, mass_out_head_stride * 4);
  from.add_cache(*rows, 0, rows->sealed, rows->tail);
  from.add(mass, (rows->sealed + rows->tail) * 4, out->batch, mass_batch_stride * 4, out->num_kv_heads,
           mass_head_stride * 4);
  from.add(keep, (int64_t)out->batch * out->num_kv_heads * n * 4, 1, 0, 1, 0);
  SF_CHECK_ARG(!overlap(to, from), "compaction writes to buffers of its own: they must not overlap others");
  SourceKept src{kv8_view(*rows), keep, n, mass, mass_out, mass_batch_stride, mass_head_stride,
                 mass_out_batch_stride, mass_out_head_stride};
  const int64_t full = out->sealed / out->block_tokens;
  const dim3 grid((unsigned)(full + (out->tail > 0 ? 1 : 0)), (unsigned)(rows->batch * rows->num_kv_heads), 2);
  return launch_write(src, make_target(*out, 0, full), grid, as_stream(stream));
}
