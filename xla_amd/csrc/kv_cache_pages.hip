// Book-keeping of a page pool on the device, and copying of whole pages.
//
// RESERVE, FORK and FREE take two launches.  Workgroup 0 of the first decides the requests (for the first two it
// collects as many free pages, lowest first, as they ask for) while the others copy the reference counts.  The
// second has one workgroup for each sequence, which writes its row of the new table and adjusts the counts
// of its pages with integer atomics, whose order changes nothing.  COMPACT takes three: count, rank, rewrite.
//
// Bound: the latency of the launches; the state is a few hundred kilobytes.  RESERVE for 256 sequences in 16384 pages 8.0
// us, COMPACT of 131072 pages under 512 sequences 11.3 (28.6 with every workgroup counting all pages before its own).
// In 131072 pages, 512 sequences: RESERVE 9 us, FORK 10, FREE 6 where the pages in use lie anywhere.  RESERVE and FORK look
// for free pages from page 0 on, 1024 after 1024: where the pages in use lie in front, as COMPACT leaves them, they take
// 59 and 60 us with half of the pool in use, 100 and 101 with nine tenths.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_cache.h"

namespace xla_amd {
namespace {

struct PagesView {
  const int* table;
  const int* lens;
  const int* refs;
  const int* request;
  int* table_out;
  int* lens_out;
  int* refs_out;
  int* moves;
  int* status;
  // scratch
  int* slot;   // [pages] the free pages that are given away, in order
  int* rank;   // [pages] COMPACT: a page's place among the free pages below U, or among those that move
  int* mover;  // [pages] COMPACT: the pages that move, the last one first
  int* used;   // [pages / kRankPages] COMPACT: pages in use of each group
  int* plan;   // [batch] RESERVE: where the sequence's slots begin, or -1; FORK: its pair + 1; FREE: 1 if freed
  int* pair;   // [requests] FORK: the pair's slot, -1: granted without one, -2: refused
  int* total;  // [2] COMPACT: pages in use, pages that move
  int batch, width, pages, page, requests;
};

constexpr int kThreads = 1024;

// Pages that hold `len` tokens, at most a row of the table.
__device__ __forceinline__ int held_pages(const PagesView& v, int len) {
  return len <= 0 ? 0 : (int)min(((int64_t)len + v.page - 1) / v.page, (int64_t)v.width);
}

// Exclusive prefix sum over the workgroup, and the sum of all.
template <class T>
__device__ __forceinline__ T block_prefix(T x, T* total) {
  __shared__ T part[kThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T incl = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T t = __shfl_up(incl, off);
    if (lane >= off) incl += t;
  }
  __syncthreads();
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    const T t = part[w];
    before += w < wave ? t : 0;
    all += t;
  }
  *total = all;
  return before + incl - x;
}

// Writes the first `wanted` free pages to v.slot and returns how many there are (workgroup 0).
__device__ int collect_free(const PagesView& v, int wanted) {
  int found = 0;
  for (int p0 = 0; p0 < v.pages && found < wanted; p0 += kThreads) {
    const int p = p0 + threadIdx.x;
    const int is_free = p < v.pages && v.refs[p] == 0 ? 1 : 0;
    int all;
    const int at = found + block_prefix(is_free, &all);
    if (is_free && at < wanted) v.slot[at] = p;
    found += all;
  }
  return min(found, wanted);
}

// What sequence b asks for: pages, or -1 where the request is refused.
__device__ __forceinline__ int reserve_need(const PagesView& v, int b) {
  const int len = v.lens[b], want = v.request[b];
  if (want < len || (int64_t)want > (int64_t)v.width * v.page) return -1;
  return held_pages(v, want) - held_pages(v, len);
}

__device__ void plan_reserve(const PagesView& v) {
  int64_t total = 0, all;  // 2^20 sequences may ask for 2^31 pages each
  for (int b0 = 0; b0 < v.batch; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    block_prefix<int64_t>(b < v.batch ? max(reserve_need(v, b), 0) : 0, &all);
    total += all;
  }
  const int have = collect_free(v, (int)min(total, (int64_t)v.pages));
  int64_t before = 0;
  for (int b0 = 0; b0 < v.batch; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    const int need = b < v.batch ? reserve_need(v, b) : -1;
    const int64_t at = before + block_prefix<int64_t>(max(need, 0), &all);
    before += all;
    if (b < v.batch) {
      const bool granted = need == 0 || (need > 0 && at + need <= have);
      v.plan[b] = granted ? (int)min(at, (int64_t)v.pages) : -1;
      v.status[b] = granted ? 1 : 0;
      v.lens_out[b] = granted ? v.request[b] : v.lens[b];
    }
  }
}

// 1 where the pair needs a page, 0 where it does not, -1 where it is refused (all but the free pages).
__device__ __forceinline__ int fork_need(const PagesView& v, int i) {
  const int src = v.request[2 * i], dst = v.request[2 * i + 1];
  if ((unsigned)src >= (unsigned)v.batch || (unsigned)dst >= (unsigned)v.batch || src == dst) return -1;
  if (v.lens[dst] > 0 || v.plan[dst] != i + 1) return -1;  // an earlier pair names dst
  const int len = v.lens[src];
  // a full page is shared; so is what a length beyond the table claims
  return len > 0 && (int64_t)len <= (int64_t)v.width * v.page && len % v.page != 0 ? 1 : 0;
}

__device__ void plan_fork(const PagesView& v) {
  for (int b = threadIdx.x; b < v.batch; b += kThreads) v.plan[b] = 0x7fffffff;
  __syncthreads();
  for (int i = threadIdx.x; i < v.requests; i += kThreads) {
    const int dst = v.request[2 * i + 1];
    if ((unsigned)dst < (unsigned)v.batch) atomicMin(&v.plan[dst], i + 1);  // the first pair has it
  }
  __syncthreads();
  int total = 0, all;
  for (int i0 = 0; i0 < v.requests; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    block_prefix(i < v.requests ? max(fork_need(v, i), 0) : 0, &all);
    total += all;
  }
  const int have = collect_free(v, total);
  __syncthreads();  // the slots are read below
  int before = 0, granted_all = 0;
  for (int i0 = 0; i0 < v.requests; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    const int need = i < v.requests ? fork_need(v, i) : -1;
    const int at = before + block_prefix(max(need, 0), &all);
    before += all;
    if (i < v.requests) {
      const bool granted = need == 0 || (need > 0 && at < have);
      v.pair[i] = !granted ? -2 : need > 0 ? at : -1;
      v.status[i] = granted ? 1 : 0;
      if (need > 0 && granted) {
        const int src = v.request[2 * i];
        v.moves[2 * at] = v.table[(int64_t)src * v.width + held_pages(v, v.lens[src]) - 1];
        v.moves[2 * at + 1] = v.slot[at];
      }
    }
  }
  granted_all = min(before, have);
  for (int i = granted_all + threadIdx.x; i < v.requests; i += kThreads) v.moves[2 * i] = v.moves[2 * i + 1] = -1;
}

__device__ void plan_free(const PagesView& v) {
  for (int b = threadIdx.x; b < v.batch; b += kThreads) v.plan[b] = 0x7fffffff;
  __syncthreads();
  for (int i = threadIdx.x; i < v.requests; i += kThreads) {
    const int b = v.request[i];
    if ((unsigned)b < (unsigned)v.batch) atomicMin(&v.plan[b], i + 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < v.requests; i += kThreads) {
    const int b = v.request[i];
    v.status[i] = (unsigned)b < (unsigned)v.batch && v.plan[b] == i + 1 ? 1 : 0;
  }
}

// RESERVE, FORK, FREE: the decisions (workgroup 0) and a copy of the counts (the others).
template <int OP>
__global__ __launch_bounds__(kThreads) void kv_pages_plan_kernel(PagesView v) {
  if (blockIdx.x == 0) {
    if (OP == XLA_AMD_KV_PAGES_RESERVE) plan_reserve(v);
    if (OP == XLA_AMD_KV_PAGES_FORK) plan_fork(v);
    if (OP == XLA_AMD_KV_PAGES_FREE) plan_free(v);
    return;
  }
  for (int64_t p = (int64_t)(blockIdx.x - 1) * kThreads + threadIdx.x; p < v.pages; p += (int64_t)(gridDim.x - 1) * kThreads)
    v.refs_out[p] = v.refs[p];
}

// The new row of every sequence, one workgroup each.
template <int OP>
__global__ __launch_bounds__(256) void kv_pages_rows_kernel(PagesView v) {
  const int b = blockIdx.x;
  const int len = v.lens[b];
  const int plan = v.plan[b];
  int from = b, have = held_pages(v, len), new_len = len;
  int slot = -1;  // FORK: where the copy of the last page lies
  bool forked = false;
  if (OP == XLA_AMD_KV_PAGES_FORK && plan != 0x7fffffff && v.pair[plan - 1] != -2) {
    forked = true;
    from = v.request[2 * (plan - 1)];
    new_len = v.lens[from];
    have = held_pages(v, new_len);
    slot = v.pair[plan - 1];
  }
  const bool freed = OP == XLA_AMD_KV_PAGES_FREE && plan != 0x7fffffff;
  const int want = OP == XLA_AMD_KV_PAGES_RESERVE && plan >= 0 ? held_pages(v, v.request[b]) : have;
  for (int j = threadIdx.x; j < v.width; j += blockDim.x) {
    int page = j < have ? v.table[(int64_t)from * v.width + j] : -1;
    const bool valid = (unsigned)page < (unsigned)v.pages;
    if (OP == XLA_AMD_KV_PAGES_RESERVE && j >= have && j < want) {
      page = v.slot[plan + j - have];
      v.refs_out[page] = 1;
    }
    if (forked && j < have) {
      if (slot >= 0 && j == have - 1) {
        page = v.slot[slot];
        v.refs_out[page] = 1;
      } else if (valid) {
        atomicAdd(&v.refs_out[page], 1);
      }
    }
    if (freed && j < have) {
      if (valid) atomicSub(&v.refs_out[page], 1);
      page = -1;
    }
    v.table_out[(int64_t)b * v.width + j] = page;
  }
  if (OP != XLA_AMD_KV_PAGES_RESERVE && threadIdx.x == 0) v.lens_out[b] = freed ? 0 : new_len;
}

constexpr int kRankPages = 4 * kThreads;  // pages of a ranking workgroup, four neighbours a thread

__device__ __forceinline__ int4 four_counts(const PagesView& v, int64_t p) {
  int4 r = {0, 0, 0, 0};
  if (p + 3 < v.pages && ((uintptr_t)v.refs & 15) == 0) return *reinterpret_cast<const int4*>(v.refs + p);
  if (p < v.pages) r.x = v.refs[p];
  if (p + 1 < v.pages) r.y = v.refs[p + 1];
  if (p + 2 < v.pages) r.z = v.refs[p + 2];
  if (p + 3 < v.pages) r.w = v.refs[p + 3];
  return r;
}

// COMPACT, first launch: pages in use among each kRankPages.
__global__ __launch_bounds__(kThreads) void kv_pages_count_kernel(PagesView v) {
  const int4 r = four_counts(v, (int64_t)blockIdx.x * kRankPages + 4 * threadIdx.x);
  int all;
  block_prefix((r.x != 0) + (r.y != 0) + (r.z != 0) + (r.w != 0), &all);
  if (threadIdx.x == 0) v.used[blockIdx.x] = all;
}

// COMPACT, second launch: with U pages in use, the free pages below U and the pages in use from U on get their
// ranks; the latter count from the end, so that no rank needs the number of them.
__global__ __launch_bounds__(kThreads) void kv_pages_rank_kernel(PagesView v) {
  int before = 0, used = 0, mine;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += kThreads) {
    const int u = v.used[i];
    used += u;
    before += i < (int)blockIdx.x ? u : 0;
  }
  int all_used, all_before;
  block_prefix(used, &all_used);
  block_prefix(before, &all_before);
  const int64_t p0 = (int64_t)blockIdx.x * kRankPages + 4 * threadIdx.x;
  const int4 r = four_counts(v, p0);
  const int counts[4] = {r.x, r.y, r.z, r.w};
  int at = all_before + block_prefix((r.x != 0) + (r.y != 0) + (r.z != 0) + (r.w != 0), &mine);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = (int)(p0 + i);
    if (p >= v.pages) break;
    if (p == all_used) v.total[1] = all_used - at;  // pages that move: those in use, less those below U
    if (counts[i] != 0) {
      if (p >= all_used) {
        v.rank[p] = all_used - 1 - at;
        v.mover[all_used - 1 - at] = p;
      }
      ++at;
    } else if (p < all_used) {
      v.rank[p] = p - at;
      v.slot[p - at] = p;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    v.total[0] = all_used;
    if (all_used == v.pages) v.total[1] = 0;
  }
}

// COMPACT, third launch: the first `batch` workgroups rewrite the table, the others the counts and moves.
__global__ __launch_bounds__(256) void kv_pages_compact_kernel(PagesView v) {
  const int used = v.total[0], moving = v.total[1];
  if ((int)blockIdx.x < v.batch) {
    const int b = blockIdx.x;
    const int len = v.lens[b], have = held_pages(v, len);
    for (int j = threadIdx.x; j < v.width; j += blockDim.x) {
      int page = j < have ? v.table[(int64_t)b * v.width + j] : -1;
      if ((unsigned)page < (unsigned)v.pages && page >= used && v.refs[page] != 0) page = v.slot[moving - 1 - v.rank[page]];
      v.table_out[(int64_t)b * v.width + j] = page;
    }
    if (threadIdx.x == 0) v.lens_out[b] = len;
    return;
  }
  const int64_t p = (int64_t)(blockIdx.x - v.batch) * blockDim.x + threadIdx.x;
  if (p >= v.pages) return;
  int count = 0;
  if (p < used) {
    count = v.refs[p];
    if (count == 0) count = v.refs[v.mover[moving - 1 - v.rank[p]]];  // as many free pages below U as pages move
  }
  v.refs_out[p] = count;
  if (p < v.pages / 2) {
    v.moves[2 * p] = p < moving ? v.mover[moving - 1 - p] : -1;
    v.moves[2 * p + 1] = p < moving ? v.slot[p] : -1;
  }
}

size_t Align16(size_t x) { return (x + 15) & ~(size_t)15; }

struct CopyView {
  const int* moves;
  int pages, buffers, parts;  // parts: of the large buffers together
  int64_t items;
  uint8_t* base[XLA_AMD_KV_CACHE_MAX_BUFFERS];
  int64_t bytes[XLA_AMD_KV_CACHE_MAX_BUFFERS];
};

// A workgroup copies kCopyPart bytes of one page of a large buffer, each thread four loads and then four stores, or the
// pages of all small buffers.  4096 pages of 2 x 64 KB: 219 us, 4.9 TB/s (222 with one load a thread); a list in
// the pages' order takes 185: what bounds it is the order of the pages.
constexpr int kCopyPart = 16384, kCopySmall = 4096;
constexpr int64_t kCopyGrid = 1 << 22;  // workgroups; a longer list of moves goes round again

template <class T, int N>
__device__ __forceinline__ void copy_part(uint8_t* dst, const uint8_t* src, int64_t bytes, int first, int step) {
  T* d = reinterpret_cast<T*>(dst);
  const T* s = reinterpret_cast<const T*>(src);
  const int64_t n = bytes / (int64_t)sizeof(T);
  for (int64_t i = first; i < n; i += (int64_t)N * step) {
    T x[N];
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (i + k * step < n) x[k] = __builtin_nontemporal_load(&s[i + k * step]);
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (i + k * step < n) __builtin_nontemporal_store(x[k], &d[i + k * step]);
  }
}

__device__ __forceinline__ void copy_bytes(uint8_t* dst, const uint8_t* src, int64_t bytes, uint64_t low, int first, int step) {
  if ((low & 15) == 0) copy_part<uintx4, 4>(dst, src, bytes, first, step);
  else if ((low & 3) == 0) copy_part<uint32_t, 4>(dst, src, bytes, first, step);
  else copy_part<uint8_t, 4>(dst, src, bytes, first, step);
}

__device__ __forceinline__ void copy_item(const CopyView& v, int64_t move, int part) {
  const int64_t src = const_int(v.moves, 2 * move), dst = const_int(v.moves, 2 * move + 1);
  if ((uint64_t)src >= (uint64_t)v.pages || (uint64_t)dst >= (uint64_t)v.pages || src == dst) return;
  if (part == v.parts) {
    // the small buffers, a wave each
    for (int i = threadIdx.x >> 6; i < v.buffers; i += 4)
      if (v.bytes[i] <= kCopySmall)
        copy_bytes(v.base[i] + dst * v.bytes[i], v.base[i] + src * v.bytes[i], v.bytes[i],
                   (uint64_t)(uintptr_t)v.base[i] | (uint64_t)v.bytes[i], threadIdx.x & 63, 64);
    return;
  }
  int buffer = 0, at = part;
  for (; buffer < v.buffers; ++buffer) {
    const int n = v.bytes[buffer] <= kCopySmall ? 0 : (int)((v.bytes[buffer] + kCopyPart - 1) / kCopyPart);
    if (at < n) break;
    at -= n;
  }
  const int64_t bytes = v.bytes[buffer], from = (int64_t)at * kCopyPart;
  copy_bytes(v.base[buffer] + dst * bytes + from, v.base[buffer] + src * bytes + from, min(bytes - from, (int64_t)kCopyPart),
             (uint64_t)(uintptr_t)v.base[buffer] | (uint64_t)bytes, threadIdx.x, 256);
}

__global__ __launch_bounds__(256) void kv_cache_copy_pages_kernel(CopyView v) {
  const unsigned per = (unsigned)v.parts + 1;
  copy_item(v, blockIdx.x / per, (int)(blockIdx.x % per));
  for (int64_t i = (int64_t)blockIdx.x + gridDim.x; i < v.items; i += gridDim.x) copy_item(v, i / per, (int)(i % per));
}

}  // namespace

size_t KvCachePagesWorkspaceBytes(int64_t batch, int64_t pages, int64_t requests) {
  if (batch < 0 || pages < 0 || requests < 0) return 0;
  return 3 * Align16((size_t)pages * 4) + Align16((size_t)batch * 4) + Align16((size_t)requests * 4) +
         Align16(((size_t)pages / kRankPages + 1) * 4) + 16;
}

int LaunchKvCachePages(const XlaAmdKvCachePages& p, hipStream_t stream) {
  const int kBad = XLA_FFI_Error_Code_INVALID_ARGUMENT;
  const bool asks = p.op == XLA_AMD_KV_PAGES_FORK || p.op == XLA_AMD_KV_PAGES_FREE;
  if (p.op < 0 || p.op > XLA_AMD_KV_PAGES_COMPACT) return Fail(kBad, "kv_cache_pages: unknown op %d", p.op);
  if (p.page_size < 1 || p.page_size > (1 << 20)) return Fail(kBad, "kv_cache_pages: page_size must be 1 to 2^20");
  if (p.batch < 0 || p.table_width < 0 || p.pages < 0 || p.requests < 0)
    return Fail(kBad, "kv_cache_pages: negative size");
  if (p.batch > (1 << 20) || p.pages > (1 << 28) || p.requests > (1 << 20) || p.table_width > INT32_MAX / p.page_size)
    return Fail(kBad, "kv_cache_pages: at most 2^20 sequences and requests, 2^28 pages and 2^31 positions");
  if ((p.batch > 0 && (!p.kv_lens || !p.kv_lens_out || (p.table_width > 0 && (!p.page_table || !p.page_table_out)))) ||
      (p.pages > 0 && (!p.ref_counts || !p.ref_counts_out)))
    return Fail(kBad, "kv_cache_pages: null state");
  if ((asks && p.requests > 0 && (!p.request || !p.status)) ||
      (p.op == XLA_AMD_KV_PAGES_RESERVE && p.batch > 0 && (!p.request || !p.status)))
    return Fail(kBad, "kv_cache_pages: null request or status");
  if ((p.op == XLA_AMD_KV_PAGES_FORK && p.requests > 0 && !p.moves) ||
      (p.op == XLA_AMD_KV_PAGES_COMPACT && p.pages > 1 && !p.moves))
    return Fail(kBad, "kv_cache_pages: null moves");
  const void* in[4] = {p.page_table, p.kv_lens, p.ref_counts, p.request};
  const void* out[6] = {p.page_table_out, p.kv_lens_out, p.ref_counts_out, p.moves, p.status, p.workspace};
  for (const void* i : in)
    for (const void* o : out)
      if (i && i == o) return Fail(kBad, "kv_cache_pages: the new state takes buffers other than the old one's");
  if (!p.workspace || p.workspace_bytes < KvCachePagesWorkspaceBytes(p.batch, p.pages, p.requests))
    return Fail(kBad, "kv_cache_pages: scratch must hold xla_amd_kv_cache_pages_workspace_bytes = %zu bytes, got %zu",
                KvCachePagesWorkspaceBytes(p.batch, p.pages, p.requests), p.workspace ? p.workspace_bytes : (size_t)0);
  uintptr_t low = (uintptr_t)p.workspace & 15;
  for (const void* i : in) low |= (uintptr_t)i & 3;
  for (const void* o : out) low |= (uintptr_t)o & 3;
  if (low) return Fail(kBad, "kv_cache_pages: scratch must be aligned to 16 bytes, the other buffers to 4");

  PagesView v{};
  v.table = p.page_table;
  v.lens = p.kv_lens;
  v.refs = p.ref_counts;
  v.request = p.request;
  v.table_out = p.page_table_out;
  v.lens_out = p.kv_lens_out;
  v.refs_out = p.ref_counts_out;
  v.moves = p.moves;
  v.status = p.status;
  uint8_t* w = (uint8_t*)p.workspace;
  const size_t page_ints = Align16((size_t)p.pages * 4);
  v.slot = (int*)w;
  v.rank = (int*)(w + page_ints);
  v.mover = (int*)(w + 2 * page_ints);
  v.plan = (int*)(w + 3 * page_ints);
  v.pair = (int*)(w + 3 * page_ints + Align16((size_t)p.batch * 4));
  v.used = (int*)((char*)v.pair + Align16((size_t)p.requests * 4));
  v.total = (int*)((char*)v.used + Align16(((size_t)p.pages / kRankPages + 1) * 4));
  v.batch = (int)p.batch;
  v.width = (int)p.table_width;
  v.pages = (int)p.pages;
  v.page = (int)p.page_size;
  v.requests = asks ? (int)p.requests : 0;
  const int copiers = (int)((p.pages + 8 * kThreads - 1) / (8 * kThreads));
  const dim3 plan_grid(1 + (copiers > 256 ? 256 : copiers));
  switch (p.op) {
    case XLA_AMD_KV_PAGES_RESERVE:
      SetLastKernel("kv_cache_pages_reserve");
      kv_pages_plan_kernel<XLA_AMD_KV_PAGES_RESERVE><<<plan_grid, kThreads, 0, stream>>>(v);
      if (v.batch > 0) kv_pages_rows_kernel<XLA_AMD_KV_PAGES_RESERVE><<<v.batch, 256, 0, stream>>>(v);
      break;
    case XLA_AMD_KV_PAGES_FORK:
      SetLastKernel("kv_cache_pages_fork");
      kv_pages_plan_kernel<XLA_AMD_KV_PAGES_FORK><<<plan_grid, kThreads, 0, stream>>>(v);
      if (v.batch > 0) kv_pages_rows_kernel<XLA_AMD_KV_PAGES_FORK><<<v.batch, 256, 0, stream>>>(v);
      break;
    case XLA_AMD_KV_PAGES_FREE:
      SetLastKernel("kv_cache_pages_free");
      kv_pages_plan_kernel<XLA_AMD_KV_PAGES_FREE><<<plan_grid, kThreads, 0, stream>>>(v);
      if (v.batch > 0) kv_pages_rows_kernel<XLA_AMD_KV_PAGES_FREE><<<v.batch, 256, 0, stream>>>(v);
      break;
    default: {
      SetLastKernel("kv_cache_pages_compact");
      const int ranks = (int)(p.pages / kRankPages) + 1;
      kv_pages_count_kernel<<<ranks, kThreads, 0, stream>>>(v);
      kv_pages_rank_kernel<<<ranks, kThreads, 0, stream>>>(v);
      const int64_t grid = p.batch + (p.pages + 255) / 256;
      if (grid > 0) kv_pages_compact_kernel<<<(unsigned)grid, 256, 0, stream>>>(v);
    }
  }
  return CheckLaunch("kv_cache_pages");
}

int LaunchKvCacheCopyPages(const XlaAmdKvCacheCopyPages& p, hipStream_t stream) {
  const int kBad = XLA_FFI_Error_Code_INVALID_ARGUMENT;
  if (p.num_buffers < 1 || p.num_buffers > XLA_AMD_KV_CACHE_MAX_BUFFERS || !p.buffers || !p.page_bytes)
    return Fail(kBad, "kv_cache_copy_pages: 1 to %d buffers", XLA_AMD_KV_CACHE_MAX_BUFFERS);
  if (p.num_moves < 0 || p.pages < 0 || p.pages > INT32_MAX || p.num_moves > INT32_MAX)
    return Fail(kBad, "kv_cache_copy_pages: at most 2^31 - 1 pages and moves");
  if (p.num_moves > 0 && (!p.moves || ((uintptr_t)p.moves & 3))) return Fail(kBad, "kv_cache_copy_pages: null or unaligned moves");
  CopyView v{};
  v.moves = p.moves;
  v.pages = (int)p.pages;
  v.buffers = (int)p.num_buffers;
  int64_t most = 0, parts = 0;
  for (int i = 0; i < v.buffers; ++i) {
    if (p.page_bytes[i] < 0 || p.page_bytes[i] > INT32_MAX)
      return Fail(kBad, "kv_cache_copy_pages: a page of a buffer holds at most 2^31 - 1 bytes");
    if (!p.buffers[i] && p.pages > 0 && p.page_bytes[i] > 0) return Fail(kBad, "kv_cache_copy_pages: null buffer");
    v.base[i] = (uint8_t*)p.buffers[i];
    v.bytes[i] = p.page_bytes[i];
    if (v.bytes[i] > most) most = v.bytes[i];
    if (v.bytes[i] > kCopySmall) parts += (v.bytes[i] + kCopyPart - 1) / kCopyPart;
  }
  if (p.num_moves == 0 || p.pages == 0 || most == 0) return 0;
  v.parts = (int)parts;  // at most 64 buffers of 2^17 each
  v.items = (parts + 1) * p.num_moves;  // below 2^23 * 2^31
  SetLastKernel("kv_cache_copy_pages");
  kv_cache_copy_pages_kernel<<<(unsigned)(v.items < kCopyGrid ? v.items : kCopyGrid), 256, 0, stream>>>(v);
  return CheckLaunch("kv_cache_copy_pages");
}

}  // namespace xla_amd
