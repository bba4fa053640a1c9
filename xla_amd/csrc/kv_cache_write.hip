// Quantises new key and value rows into the pages of an 8-bit cache, one scale for each block of tokens and
// head.  For every block that a call touches, and each head:
//
//   s = max|x| / qmax over the block's new rows; where the block held rows of the sequence before,
//   s = max(s, old scale) and the held codes become rn(clamp(c * (old / s)));  code = rn(clamp(x / s)).
//
// qmax is 127 (s8) or 448 (f8e4m3fn).  Every operation is f32 and rounded once (IEEE quotients), so codes and
// scales are reproducible bit for bit; the codes are the only rounding to fewer bits and are what is asked for.
//
// Bound: HBM; 2 bytes read and 1 written per value.  16 prompts, 8 heads of 128 to f8: 13.3 us, 4.3 TB/s; 128 single rows
// to s8: 5.2 us, which is latency (lengths and offsets, table, rows, codes).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_cache.h"

namespace xla_amd {

namespace {

int Log2Exact(int64_t x) {
  for (int i = 0; i < 31; ++i)
    if (x == (int64_t)1 << i) return i;
  return -1;
}

}  // namespace

int MakeKvCacheView(const XlaAmdKvCache& p, const char* what, KvCacheView* c) {
  const int kBad = XLA_FFI_Error_Code_INVALID_ARGUMENT;
  const int page_log2 = Log2Exact(p.page_size), block_log2 = Log2Exact(p.block);
  if (p.cache_dtype != XLA_FFI_DataType_S8 && p.cache_dtype != XLA_FFI_DataType_F8E4M3FN)
    return Fail(kBad, "%s: the cache must be S8 or F8E4M3FN", what);
  if (page_log2 < 4 || page_log2 > 10) return Fail(kBad, "%s: the page size must be a power of two from 16 to 1024", what);
  if (block_log2 < 0 || block_log2 > page_log2)
    return Fail(kBad, "%s: the block of a scale must be a power of two that divides the page", what);
  if (p.head_size < 16 || p.head_size > 256 || p.head_size % 16 != 0)
    return Fail(kBad, "%s: the head size must be a multiple of 16 from 16 to 256", what);
  if (p.pages < 0 || p.batch < 0 || p.table_width < 0 || p.rows < 0) return Fail(kBad, "%s: negative size", what);
  if (p.kv_heads < 1 || p.kv_heads > 1024) return Fail(kBad, "%s: kv_heads must be 1 to 1024", what);
  if (p.pages > INT32_MAX || p.rows >= (1 << 24) || p.batch > (1 << 20) ||
      p.table_width > (int64_t)(INT32_MAX - 1024) / p.page_size)
    return Fail(kBad, "%s: at most 2^31 - 1 pages, fewer than 2^24 rows, 2^20 sequences and 2^31 positions", what);
  if (p.batch > 0 && p.rows > 0) {
    if (!p.kv_lens || !p.q_offsets || (p.table_width > 0 && !p.page_table))
      return Fail(kBad, "%s: null page_table, kv_lens or q_offsets", what);
    if (p.pages > 0 && (!p.k_cache || !p.v_cache || !p.k_scales || !p.v_scales))
      return Fail(kBad, "%s: null cache or scales", what);
  }
  if ((((uintptr_t)p.k_cache | (uintptr_t)p.v_cache) & 15) != 0 ||
      (((uintptr_t)p.k_scales | (uintptr_t)p.v_scales | (uintptr_t)p.page_table | (uintptr_t)p.kv_lens |
        (uintptr_t)p.q_offsets) & 3) != 0)
    return Fail(kBad, "%s: the caches must be aligned to 16 bytes, scales and integers to 4", what);
  c->codes[0] = (uint8_t*)p.k_cache;
  c->codes[1] = (uint8_t*)p.v_cache;
  c->scales[0] = p.k_scales;
  c->scales[1] = p.v_scales;
  c->table = p.page_table;
  c->lens = p.kv_lens;
  c->offsets = p.q_offsets;
  c->pages = (int)p.pages;
  c->heads = (int)p.kv_heads;
  c->head = (int)p.head_size;
  c->page_log2 = page_log2;
  c->block_log2 = block_log2;
  c->batch = (int)p.batch;
  c->width = p.pages > 0 ? (int)p.table_width : 0;  // without pages no position exists
  c->rows = (int)p.rows;
  return 0;
}

namespace {

// Four f32 in the code range (or NaN: code 0) -> four codes.
template <bool F8>
__device__ __forceinline__ uint32_t to_codes(const float* x) {
  constexpr float kMax = F8 ? 448.0f : 127.0f;
  float t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float q = x[i] == x[i] ? x[i] : 0.0f;
    t[i] = __builtin_amdgcn_fmed3f(q, -kMax, kMax);
  }
  if constexpr (F8) return pack_f8x4(t[0], t[1], t[2], t[3]);
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) r |= ((uint32_t)(int)__builtin_rintf(t[i]) & 0xffu) << (8 * i);
  return r;
}

template <bool F8>
__device__ __forceinline__ float from_code(uint32_t w, int i) {
  const uint32_t c = (w >> (8 * i)) & 0xffu;
  if constexpr (F8) return f8e4m3fn_to_f32(c);
  return (float)(int8_t)c;
}

// Blocks that a sequence's new rows touch.
__device__ __forceinline__ int touched_blocks(const KvCacheView& c, int b) {
  const KvSequence s = kv_sequence(c, b);
  if (s.n == 0 || s.len == 0) return 0;
  return ((s.len - 1) >> c.block_log2) - (max(s.len - s.n, 0) >> c.block_log2) + 1;
}

typedef uint16_t ushortx2 __attribute__((ext_vector_type(2)));

// The larger magnitudes of two pairs of bf16, as bits: every NaN is above every number.
__device__ __forceinline__ uint32_t larger_pair(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushortx2, a), __builtin_bit_cast(ushortx2, b & 0x7fff7fffu)));
}

__device__ __forceinline__ uint32_t larger_pairs(uint32_t top, uintx4 w) {
  return larger_pair(larger_pair(larger_pair(larger_pair(top, w[0]), w[1]), w[2]), w[3]);
}

// Re-scales the codes that a block held before (its first `units` groups of eight) where its scale grows;
// returns the block's scale.
template <bool F8>
__device__ __forceinline__ float settle_scale(uint32_t top, int units, int lane, float* scale_at, uint8_t* codes) {
  const float amax = bits_to_f32(top > 0x7f800000u ? 0x7fc00000u : top);
  float scale = amax / (F8 ? 448.0f : 127.0f);
  if (units > 0) {
    const float old = *scale_at;
    if (old > scale || old != old) scale = old;
    if (scale != old) {
      const float ratio = old / scale;
      for (int u = lane; u < units; u += 64) {
        uintx2* at = reinterpret_cast<uintx2*>(codes) + u;
        const uintx2 w = *at;
        uintx2 o;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float t[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) t[i] = from_code<F8>(w[h], i) * ratio;
          o[h] = to_codes<F8>(t);
        }
        *at = o;
      }
    }
  }
  return scale;
}

// Eight values over an ordinary scale that is at least their maximum / qmax: the quotients are numbers and none
// rounds beyond qmax, so nothing is selected or clamped.  A zero quotient has lost its sign in div_by_ordinary's
// correction; the codes take the values' signs (s8 has no negative zero).  s8: 1.5 * 2^23 + q holds the nearest
// even integer in its low byte.
template <bool F8>
__device__ __forceinline__ uintx2 quantise8_ordinary(uintx4 w, float scale, float inverse) {
  float t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = i & 1 ? bf16hi_to_f32(w[i >> 1]) : bf16lo_to_f32(w[i >> 1]);
    const float q = x * inverse;
    t[i] = __builtin_fmaf(__builtin_fmaf(-q, scale, x), inverse, q);
    if (!F8) t[i] += 12582912.0f;
  }
  uintx2 o;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (F8) {
      const uint32_t signs = __builtin_amdgcn_perm(w[2 * h + 1], w[2 * h], 0x07050301u);  // high bytes of the four values
      const uint32_t codes = pack_f8x4(t[4 * h], t[4 * h + 1], t[4 * h + 2], t[4 * h + 3]);
      o[h] = (codes & 0x7f7f7f7fu) | (signs & 0x80808080u);
    } else {
      const uint32_t lo = __builtin_amdgcn_perm(f32_to_bits(t[4 * h + 1]), f32_to_bits(t[4 * h]), 0x0c0c0400u);
      const uint32_t hi = __builtin_amdgcn_perm(f32_to_bits(t[4 * h + 3]), f32_to_bits(t[4 * h + 2]), 0x04000c0cu);
      o[h] = lo | hi;
    }
  }
  return o;
}

// The same for any scale; a zero or NaN one gives code 0, as does a quotient that is no number.
template <bool F8>
__device__ __forceinline__ uintx2 quantise8(uintx4 w, float scale) {
  float t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = i & 1 ? bf16hi_to_f32(w[i >> 1]) : bf16lo_to_f32(w[i >> 1]);
    t[i] = scale > 0.0f ? x / scale : 0.0f;
  }
  return uintx2{to_codes<F8>(t), to_codes<F8>(t + 4)};
}

// One wave for a block and head, keys and values together: finding the block and its page costs a wave more than
// its arithmetic does.  A lane holds kHeld groups of eight values of each while the maximum is found (16 rows of 128
// values, or one row of a decode step); a block with more new values reads them again, from L2.  128 single rows took
// 7.4 us with a wave for keys and one for values.
constexpr int kHeld = 4;

template <bool F8>
__global__ __launch_bounds__(256) void kv_cache_write_kernel(KvCacheView c, const uint16_t* __restrict__ k,
                                                             const uint16_t* __restrict__ v) {
  const int lane = threadIdx.x & 63;
  const int head = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (head >= c.heads) return;
  int64_t index;
  const int b = kv_find_item(c.batch, blockIdx.x, lane, &index, [&](int s) { return touched_blocks(c, s); });
  if (b < 0) return;
  const KvSequence s = kv_sequence(c, b);
  const int start = max(s.len - s.n, 0);
  const int first = ((start >> c.block_log2) + (int)index) << c.block_log2;  // the block's first position
  const int from = max(first, start), to = min(first + (1 << c.block_log2), s.len);
  const int page = kv_page(c, b, first);
  if (page < 0) return;
  const int in_page = first & ((1 << c.page_log2) - 1);
  const int chunks = c.head >> 3;  // groups of eight values in a row
  const int held = from - first;   // rows of the sequence that the block held before
  const int units = (to - from) * chunks;
  const int64_t x = ((int64_t)(s.row0 + s.n - (s.len - from)) * c.heads + head) * c.head;
  const int64_t row_stride = (int64_t)c.heads * c.head;
  const int64_t code = kv_row(c, page, head, in_page), scale_at = kv_scale(c, page, head, in_page);
  auto read = [&](const uint16_t* src, int u) {
    const int r = u / chunks;
    return *reinterpret_cast<const uintx4*>(src + x + r * row_stride + (u - r * chunks) * 8);
  };
  uintx4 held_values[2][kHeld];
  uint32_t top[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int u = lane + 64 * i;
#pragma unroll
    for (int w = 0; w < 2; ++w) held_values[w][i] = u < units ? read(w ? v : k, u) : uintx4{0u, 0u, 0u, 0u};
  }
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
#pragma unroll
    for (int w = 0; w < 2; ++w) top[w] = larger_pairs(top[w], held_values[w][i]);
  for (int u = lane + 64 * kHeld; u < units; u += 64)
#pragma unroll
    for (int w = 0; w < 2; ++w) top[w] = larger_pairs(top[w], read(w ? v : k, u));
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
#pragma unroll
    for (int w = 0; w < 2; ++w) top[w] = larger_pair(top[w], (uint32_t)__shfl_xor((int)top[w], off));
#pragma unroll
  for (int w = 0; w < 2; ++w) top[w] = max(top[w] << 16, top[w] & 0xffff0000u);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    uint8_t* codes = c.codes[w] + code;
    const float scale = settle_scale<F8>(top[w], held * chunks, lane, c.scales[w] + scale_at, codes);
    uintx2* out = reinterpret_cast<uintx2*>(codes + (int64_t)held * c.head);
    if (ordinary_divisor(scale)) {
      const float inverse = 1.0f / scale;
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (lane + 64 * i < units) out[lane + 64 * i] = quantise8_ordinary<F8>(held_values[w][i], scale, inverse);
      for (int u = lane + 64 * kHeld; u < units; u += 64) out[u] = quantise8_ordinary<F8>(read(w ? v : k, u), scale, inverse);
    } else {
      for (int u = lane; u < units; u += 64) out[u] = quantise8<F8>(read(w ? v : k, u), scale);
    }
    if (lane == 0) c.scales[w][scale_at] = scale;
  }
}

}  // namespace

int LaunchKvCacheWrite(const XlaAmdKvCacheWrite& p, hipStream_t stream) {
  KvCacheView c;
  if (int rc = MakeKvCacheView(p.cache, "kv_cache_write", &c)) return rc;
  if (c.rows > 0 && (!p.k || !p.v)) return Fail(XLA_FFI_Error_Code_INVALID_ARGUMENT, "kv_cache_write: null k or v");
  if ((((uintptr_t)p.k | (uintptr_t)p.v) & 15) != 0)
    return Fail(XLA_FFI_Error_Code_INVALID_ARGUMENT, "kv_cache_write: k and v must be aligned to 16 bytes");
  if (c.rows == 0 || c.batch == 0 || c.pages == 0 || c.width == 0) return 0;
  if (c.codes[0] == c.codes[1] || c.scales[0] == c.scales[1])
    return Fail(XLA_FFI_Error_Code_INVALID_ARGUMENT, "kv_cache_write: keys and values need buffers of their own");
  // n rows touch at most n blocks and at most (n - 2) / block + 2
  int64_t items = ((int64_t)c.rows >> c.block_log2) + 2 * (int64_t)c.batch;
  if (items > c.rows) items = c.rows;
  const dim3 grid((unsigned)items, (unsigned)((c.heads + 3) / 4));
  if (p.cache.cache_dtype == XLA_FFI_DataType_F8E4M3FN) {
    SetLastKernel("kv_cache_write_f8");
    kv_cache_write_kernel<true><<<grid, 256, 0, stream>>>(c, (const uint16_t*)p.k, (const uint16_t*)p.v);
  } else {
    SetLastKernel("kv_cache_write_s8");
    kv_cache_write_kernel<false><<<grid, 256, 0, stream>>>(c, (const uint16_t*)p.k, (const uint16_t*)p.v);
  }
  return CheckLaunch("kv_cache_write");
}

}  // namespace xla_amd
