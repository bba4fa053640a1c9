// What the kernels over an 8-bit paged key/value cache share: the cache as a kernel sees it, where a
// sequence's rows and positions lie, and how a workgroup finds its piece of a ragged call.
#ifndef XLA_AMD_CSRC_KV_CACHE_H_
#define XLA_AMD_CSRC_KV_CACHE_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_numerics.h"
#include "launch.h"

namespace xla_amd {

// Integers that no kernel writes while another reads them: a read whose index is the same in all lanes goes through
// the scalar cache, also behind stores and loads to LDS.
typedef const __attribute__((address_space(4))) int* const_ints_t;
static __device__ __forceinline__ int const_int(const int* p, int64_t i) { return ((const_ints_t)(uintptr_t)p)[i]; }

struct KvCacheView {
  uint8_t* codes[2];  // k, v: [pages, heads, page, head]
  float* scales[2];   // [pages, heads, page / block]
  const int* table;   // [batch, width]
  const int* lens;    // [batch]
  const int* offsets; // [batch + 1]
  int pages, heads, head;
  int page_log2, block_log2;
  int batch, width, rows;
};

// Rows [row0, row0 + n) of the call belong to the sequence and stand at its positions [len - n, len); where
// the length is smaller than n the first rows have no position.  Offsets and lengths are clamped so
// that no value of theirs leads outside the operands.
struct KvSequence {
  int row0, n, len;
};

static __device__ __forceinline__ KvSequence kv_sequence(const KvCacheView& c, int b) {
  KvSequence s;
  s.row0 = min(max(const_int(c.offsets, b), 0), c.rows);
  s.n = min(max(const_int(c.offsets, b + 1), s.row0), c.rows) - s.row0;
  s.len = min(max(const_int(c.lens, b), 0), c.width << c.page_log2);
  return s;
}

// The page that holds position `pos` of sequence b, or -1 where the table names none.
static __device__ __forceinline__ int kv_page(const KvCacheView& c, int b, int pos) {
  const int page = const_int(c.table, (int64_t)b * c.width + (pos >> c.page_log2));
  return (unsigned)page < (unsigned)c.pages ? page : -1;
}

// Index of the first byte of row `row` of a page and head; cache sizes pass 32 bits.
static __device__ __forceinline__ int64_t kv_row(const KvCacheView& c, int page, int head, int row) {
  return ((((int64_t)page * c.heads + head) << c.page_log2) + row) * c.head;
}
static __device__ __forceinline__ int64_t kv_scale(const KvCacheView& c, int page, int head, int row) {
  return (((int64_t)page * c.heads + head) << (c.page_log2 - c.block_log2)) + (row >> c.block_log2);
}

__device__ __forceinline__ int64_t uniform64(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)(uint64_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)x >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// Descriptor of `bytes` bytes from base (the same in all lanes) on: loads past them, all of them where bytes is 0,
// return 0.
static __device__ __forceinline__ __amdgpu_buffer_rsrc_t kv_rsrc(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(uniform64((int64_t)(uintptr_t)base)), 0,
                                           __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

// Finds item `item` of a ragged call by itself: sequence b has cost(b) items, in order.  64 sequences at a
// time, lane l reads what sequence b0 + l has, a scan over the lanes gives the items before each.
// All 64 lanes must be active.  Returns the sequence, or -1 past the last item; *index: which of its items.
template <class Cost>
static __device__ __forceinline__ int kv_find_item(int batch, int64_t item, int lane, int64_t* index, Cost cost) {
  int64_t seen = 0;
  for (int b0 = 0; b0 < batch; b0 += 64) {
    const int b = b0 + lane;
    const int n = b < batch ? cost(b) : 0;
    int incl = n;  // (a sequence has at most as many items as the call has rows, 2^24, so this stays below 2^31)
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int t = __shfl_up(incl, off);
      if (lane >= off) incl += t;
    }
    const int64_t before = seen + incl - n;
    const unsigned long long hit = __ballot(item >= before && item < before + n);
    if (hit != 0ull) {
      const int src = __builtin_ctzll(hit);
      *index = item - (seen + __shfl(incl - n, src));
      return __builtin_amdgcn_readfirstlane(b0 + src);
    }
    seen += __shfl(incl, 63);
  }
  *index = 0;
  return -1;
}

// Checks what a launcher can see of a cache and fills the kernels' view of it; 0 or the error.
int MakeKvCacheView(const XlaAmdKvCache& p, const char* what, KvCacheView* c);

}  // namespace xla_amd
#endif  // XLA_AMD_CSRC_KV_CACHE_H_
