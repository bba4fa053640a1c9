// Softmax attention over an 8-bit paged key/value cache.
//
//   x_j = softmax_scale * ks_j * sum_d q_d kc_jd, with softcap: softcap * tanh(x_j / softcap)
//   out_d = sum_j exp(x_j - m) vs_j vc_jd / sum_j exp(x_j - m),  lse = m + log sum_j exp(x_j - m)
//
// over the positions j that the row sees, with the running maximum m and sum of a softmax.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "kv_cache.h"

namespace xla_amd {
namespace {

struct AttentionView {
  KvCacheView c;
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  int q_heads, group;  // group: heads of q for each head of the cache
  float scale;
  float cap, per_cap;  // softcap in units of log 2, as the scores are (0: none), and its reciprocal
  int causal, window;
};

// The first position that the row at position p sees.  A row in front of its sequence (p < 0) sees none; its p less a
// window of nearly 2^31 would leave 32 bits.
static __device__ __forceinline__ int window_start(const AttentionView& v, int p) {
  return v.window > 0 ? max(0, max(p, 0) - v.window + 1) : 0;
}

// A tile of packed rows whose positions several workgroups share.
struct __attribute__((aligned(16))) CutTile {
  int row0;    // the sequence's first row
  int first;   // packed row of the sequence where the tile begins
  int rows;    // 0: no tile
  int pieces;
};

// ---- few rows for each sequence: the cache is streamed once ------------------------------------------
//
// A workgroup of four waves takes the packed rows (row, head of the group) of one sequence and cache head, 16
// or 32 at a time, along a range of 128-position units, 32 positions a wave; each wave has its own running
// maximum, sum and result, which meet in LDS at the end of the range.  Per wave and 32 positions, with c = lane & 15 and
// g = lane >> 4:
//   S^T = K Q^T   a lane reads 16-byte pieces of key rows c from its ring, widened to bf16 (exact for
//                 both code types); the result has column (row of q) c and keys 4 g + i of either 16.
//   O^T = V^T P^T the scores of a lane are, without moving, the operand's keys 4 g + i of both 16s; a lane holds
//                 values d = 16 i + c of those eight keys, read transposed from LDS and widened to f16.
// The sums over d and over keys run in whatever order the operands share, so nothing is shuffled but maxima.
// Scales stay out of the operands: the key's on the f32 score, the value's on the weight, which is rounded to
// f16 there.
//
// Where the keys are split: all sequences' units (times their tiles of rows) stand in one line, which is cut
// into as many equal pieces as there are workers for a head, so a batch of mixed lengths fills the device
// evenly.  A range that covers a tile whole writes the result; any other writes f32 sums to the
// scratch, at most two for each worker, and a second launch joins them in order.  The worker in whose range a cut
// tile begins notes where its pieces are, so the second launch looks for nothing.
//
// Bound: HBM, 2 (head + 4 / block) bytes for each position and cache head.  64 sequences of up to 8192 positions, 32 heads
// on 8 of 128, s8: 110 us, 4.9 TB/s, where a linear read reaches 7.05; four sequences of 131072, 64 heads on 8, f8: 185 us,
// 5.4 TB/s.  With tables that name 64 pages again and again, which stay in the caches, they take 80 and 123 us.
constexpr int kUnit = 128;

struct DecodeView {
  AttentionView a;
  float* partial;   // [heads][2 * workers][tile rows][head + 2], or null: ranges are whole tiles
  CutTile* cuts;    // [workers], of the tile that a worker begins and others go on with
  int workers;      // for each head
  int rows_from, rows_to;  // sequences with rows_from < n * group <= rows_to are this kernel's
};

// Tiles of packed rows of a sequence and the units of positions that any of its rows sees.
struct DecodeSpan {
  KvSequence s;
  int lo, hi;  // positions [lo, hi)
  int tiles, units, first;  // first: the first unit
};

template <int RT>
__device__ __forceinline__ DecodeSpan decode_span(const DecodeView& v, int b) {
  DecodeSpan r;
  r.s = kv_sequence(v.a.c, b);
  const int rows = r.s.n * v.a.group;
  r.lo = window_start(v.a, r.s.len - r.s.n);
  r.hi = r.s.len;
  const bool mine = rows > v.rows_from && rows <= v.rows_to;
  r.tiles = mine ? (rows + RT - 1) / RT : 0;
  r.first = r.lo / kUnit;
  r.units = max((r.hi + kUnit - 1) / kUnit - r.first, 1);  // a sequence that sees nothing has its zeros written
  return r;
}

__device__ __forceinline__ int64_t shfl64(int64_t x, int src) {
  const int lo = __shfl((int)(uint32_t)(uint64_t)x, src), hi = __shfl((int)(uint32_t)((uint64_t)x >> 32), src);
  return (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
}

// Where an entry of a line lies in which sequence b has entries(b) of them.
struct LineSpot {
  int b;           // the sequence, -1 past the end
  int64_t before;  // entries before the sequence's
  int64_t total;
};

// 64 sequences at a time: lane l holds sequence b0 + l, scans over the lanes give what lies before each.  Entry
// at(total) is looked for.
template <class Entries, class At>
__device__ __forceinline__ LineSpot line_find(int batch, int lane, Entries entries, At at) {
  LineSpot r{-1, 0, 0};
  auto cost = [&](int b) -> int64_t { return b < batch ? entries(b) : 0; };
  int64_t units = cost(lane);
  if (batch > 64) {
    int64_t sum = units;
    for (int b = lane + 64; b < batch; b += 64) sum += cost(b);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += shfl64(sum, lane ^ off);
    r.total = uniform64(sum);
  }
  int64_t seen = 0, want = batch > 64 ? at(r.total) : 0;
  for (int b0 = 0; b0 < batch; b0 += 64) {
    if (b0 > 0) units = cost(b0 + lane);
    int64_t upto = units;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int64_t t = shfl64(upto, lane - off);
      if (lane >= off) upto += t;
    }
    if (batch <= 64) {
      r.total = uniform64(shfl64(upto, 63));
      want = at(r.total);
    }
    const unsigned long long hit = __ballot(want < seen + upto && want >= seen + upto - units);
    if (hit != 0ull) {
      const int src = __builtin_ctzll(hit);
      r.b = __builtin_amdgcn_readfirstlane(b0 + src);
      r.before = seen + uniform64(shfl64(upto - units, src));
      return r;
    }
    seen += uniform64(shfl64(upto, 63));
  }
  return r;
}

// Units that a worker takes of the line: worker w has [w * piece, (w + 1) * piece).
__device__ __forceinline__ int64_t worker_piece(int64_t total, int workers) {
  return (uint64_t)total < (1ull << 31) ? (int64_t)(((uint32_t)total + (uint32_t)workers - 1) / (uint32_t)workers)
                                        : (total + workers - 1) / workers;
}

__device__ __forceinline__ int divide(int64_t x, int64_t by) {
  return (uint64_t)(x | by) < (1ull << 31) ? (int)((uint32_t)x / (uint32_t)by) : (int)(x / by);
}

// Two codes at byte places i, i + 1 -> two bf16 in a dword, exact.
template <bool F8, int I>
__device__ __forceinline__ uint32_t widen2(uint32_t w) {
  if constexpr (F8) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, I != 0));
  } else {
    const float a = (float)(int8_t)(w >> (8 * I)), b = (float)(int8_t)(w >> (8 * I + 8));
    return __builtin_amdgcn_perm(f32_to_bits(b), f32_to_bits(a), 0x07060302u);
  }
}

// Eight codes -> eight bf16.
template <bool F8>
__device__ __forceinline__ bf16x8 widen8(uint32_t lo, uint32_t hi) {
  return __builtin_bit_cast(bf16x8, uintx4{widen2<F8, 0>(lo), widen2<F8, 2>(lo), widen2<F8, 0>(hi), widen2<F8, 2>(hi)});
}

typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));

// Two codes at bytes 0 and 2 (S8; the other bytes 0) -> two f16, exact: 1024 + 128 + c, less 1152.
__device__ __forceinline__ uint32_t s8_to_f16(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(halfx2, w ^ 0x64806480u) - halfx2{(_Float16)1152.0f, (_Float16)1152.0f});
}

// Four codes -> four f16, exact.
template <bool F8>
__device__ __forceinline__ uintx2 widen4_f16(uint32_t w) {
  if constexpr (F8) {
    return uintx2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))};
  } else {
    return uintx2{s8_to_f16(__builtin_amdgcn_perm(0u, w, 0x0c010c00u)), s8_to_f16(__builtin_amdgcn_perm(0u, w, 0x0c030c02u))};
  }
}

template <bool F8>
__device__ __forceinline__ halfx8 widen8_f16(uint32_t lo, uint32_t hi) {
  const uintx2 a = widen4_f16<F8>(lo), b = widen4_f16<F8>(hi);
  return __builtin_bit_cast(halfx8, uintx4{a[0], a[1], b[0], b[1]});
}

// Bytes T and T + 1 (T even; word T / 4) of eight keys -> eight f16 each.
template <bool F8, int T, int N>
__device__ __forceinline__ void columns(const uint32_t (&k)[8][N], uintx4& first, uintx4& second) {
  constexpr int W = T >> 2;
  constexpr uint32_t I = T & 3;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const uint32_t a = k[2 * p][W], b = k[2 * p + 1][W];
    if constexpr (F8) {
      // byte I of both keys, then byte I + 1 of both, as the conversion reads them
      const uintx2 both = widen4_f16<true>(__builtin_amdgcn_perm(b, a, 0x05010400u + 0x01010101u * I));
      first[p] = both[0];
      second[p] = both[1];
    } else {
      first[p] = s8_to_f16(__builtin_amdgcn_perm(b, a, 0x0c040c00u + 0x00010001u * I));
      second[p] = s8_to_f16(__builtin_amdgcn_perm(b, a, 0x0c050c01u + 0x00010001u * I));
    }
  }
}

// A row's maximum before any score: below every other number, and finite, so that a difference to it is no NaN.
constexpr float kNoScore = -0x1.fffffep127f;

// A weight times its value's scale goes into the matrix instruction as f16, which rounds it by 2^-11 at most; bf16 would
// by 2^-8, as much as the result's own rounding, and the result would be 1.4 times as far from the exact one.  f16's range
// is narrow, so a row's weights and sums carry a factor, a power of two, that keeps every scale times the factor in
// [kLeast, kMost].  Weights are 2^5 at most (the maximum in use may lag behind by that much), so none passes 2^15, and
// the row's sum times the factor stays at 1/2 or above, so the smallest keep an absolute error of 2^-24 of the sum.  Where a
// scale leaves that range, the weights themselves and their sum so far (`weighed`, with the factor) choose the next
// factor, in a branch.  A prompt of 4096 rows, 32 heads on 8 of 128, whose value scales deviate by a factor of two takes 191
// us, one with equal scales 205, by a factor of four 256.
constexpr float kMost = 1024.0f, kLeast = 1.0f, kLag = 5.0f;

// of scales times the factor
template <int N>
__device__ __forceinline__ bool factor_fits(const float (&x)[N]) {
  float most = __builtin_fabsf(x[0]), least = most;
#pragma unroll
  for (int i = 1; i < N; ++i) {
    most = __builtin_fmaxf(most, __builtin_fabsf(x[i]));
    least = __builtin_fminf(least, __builtin_fabsf(x[i]));
  }
  return least >= kLeast && most <= kMost;
}

// A factor is 2^-123 to 2^99, the step from one to the next at most 2^100 up.
__device__ __forceinline__ float reciprocal(float factor) { return bits_to_f32((254u << 23) - f32_to_bits(factor)); }

// The factor of a row after a step whose largest weight times scale is `weight`; `weighed` is the sum of those before,
// with the factor.  It stays unless the weight would pass kMost or all so far is below 1/2; the larger is then 16
// to 32, with room for later scales on both sides.
__device__ __forceinline__ float new_factor(float weight, float weighed, float factor) {
  const float most = __builtin_fmaxf(weight, weighed * reciprocal(factor));
  const bool high = weight * factor > kMost;
  if (!(high || most * factor < 0.5f) || most == 0.0f) return factor;
  const uint32_t e = min(max(f32_to_bits(high ? weight : most) >> 23, 32u), 254u);
  return __builtin_fminf(bits_to_f32((258u - e) << 23), factor * 0x1p100f);
}

// A scale times a new factor; finite, so that a weight of 0 cancels it.
__device__ __forceinline__ float finite_product(float scale, float factor) {
  constexpr float kMax = 3.4028234663852886e38f;
  return __builtin_amdgcn_fmed3f(scale * factor, -kMax, kMax);
}

__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{a, b}, halfx2));
}

// Keeps what follows in its branch: work that few steps need is not done by all of them and thrown away.
#define KV_CACHE_INLINE __attribute__((always_inline))  // of a lambda: its captures stay in registers
#define KV_CACHE_RARE() asm volatile("")
// Steps of products and what is to run meanwhile stay side by side.
#define KV_CACHE_FENCE() __builtin_amdgcn_sched_barrier(0)

// Scores x, in units of log 2, become cap tanh(t) with t = x / cap.  Below |t| = 1/2 that is x plus x times a polynomial in
// t^2 (tanh(t) / t - 1 over t^2, at Chebyshev's four points of [0, 1/4]: off by 2^-24 of the result), so that a cap far
// above the scores leaves them as exact as they were; from there on cap (1 - 2 / (1 + e^(2 t))), whose rounding is 2^-21.5
// of the result at 1/2 and less above.  Small t are the usual case, and a wave that has no others takes no exponential:
// 2048 rows of 32 heads on 8 of 128, causal, take 111 us under a cap of 50 and 142 under a cap of 1, which most scores pass.
__device__ __forceinline__ float capped_near(float x, float per_cap) {
  const float t = x * per_cap, u = t * t;
  float p = __builtin_fmaf(u, 0.01798875f, -0.05338711f);
  p = __builtin_fmaf(p, u, 0.13330476f);
  p = __builtin_fmaf(p, u, -0.3333331f);
  return __builtin_fmaf(x * u, p, x);
}

__device__ __forceinline__ float capped(float x, float cap, float per_cap) {
  const float t = x * per_cap;
  const float z = __builtin_amdgcn_exp2f(t * 2.88539008177792681f);
  const float far = cap * __builtin_fmaf(__builtin_amdgcn_rcpf(1.0f + z), -2.0f, 1.0f);
  return __builtin_fabsf(t) >= 0.5f ? far : capped_near(x, per_cap);
}

template <int N>
__device__ __forceinline__ void cap_scores(float (&x)[N], float cap, float per_cap) {
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) most = __builtin_fmaxf(most, __builtin_fabsf(x[i]));
  if (__any(most * per_cap >= 0.5f)) {
    KV_CACHE_RARE();
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = capped(x[i], cap, per_cap);
  } else {
    KV_CACHE_RARE();
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = capped_near(x[i], per_cap);
  }
}

// Rows first to first + 63, where they belong to no sequence: 0, lse -infinity.
__device__ void clear_rows_of_nobody(const AttentionView& v, int first) {
  const KvCacheView& c = v.c;
  __shared__ int owned[64];
  if (threadIdx.x < 64) owned[threadIdx.x] = 0;
  __syncthreads();
  for (int b = threadIdx.x; b < c.batch; b += blockDim.x) {
    const KvSequence s = kv_sequence(c, b);
    const int from = max(s.row0, first), to = min(s.row0 + s.n, first + 64);
    for (int r = from; r < to; ++r) owned[r - first] = 1;
  }
  __syncthreads();
  for (int r = 0; r < 64 && first + r < c.rows; ++r) {
    if (owned[r]) continue;
    const int64_t at = (int64_t)(first + r) * v.q_heads;
    uintx4* o = reinterpret_cast<uintx4*>(v.out + at * c.head);
    for (int i = threadIdx.x; i < v.q_heads * c.head / 8; i += blockDim.x) o[i] = uintx4{0u, 0u, 0u, 0u};
    if (v.lse)
      for (int i = threadIdx.x; i < v.q_heads; i += blockDim.x) v.lse[at + i] = -INFINITY;
  }
}

// A scale that is NaN or infinite makes the score NaN, which reaches the rows that see the position and no others: an
// infinite key scale would leave some of them a weight of zero or a capped score, and a weight of zero would not cancel a
// value scale that is no number.  0 times either is NaN where it is no number, and else 0.
__device__ __forceinline__ void keep_to_its_rows(float& key_scale, float& value_scale) {
  key_scale = __builtin_fmaf(key_scale, 0.0f, key_scale);
  key_scale = __builtin_fmaf(value_scale, 0.0f, key_scale);
  value_scale = __builtin_fabsf(value_scale) < INFINITY ? value_scale : 0.0f;
}

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef int intx2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) intx2* lds_tr_ptr_t;

// (functions of their own: inside a lambda these builtins cost the kernel its launch stub)
// 64 lanes x 16 bytes into 1 KiB of LDS from `to` on, in the order of the lanes; past the buffer's end zeros.
__device__ __forceinline__ void load16_to_lds(__amdgpu_buffer_rsrc_t r, uint8_t* to, uint32_t from) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)to, 16, from, 0, 0, 0);
}
// 64 lanes x 4 bytes, each lane from an address of its own.
__device__ __forceinline__ void load4_to_lds(const char* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (lds_ptr_t)to, 4, 0, 0);
}
// In every 16 lanes: lane i points at 8 bytes of row i / 2, the even lanes at one octet, the odd ones at the next;
// lane j receives byte j of the eight rows.
__device__ __forceinline__ intx2 read_columns(const uint8_t* from) {
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_tr_ptr_t)from);
}

// A wave's ring in LDS: each slot holds 32 positions as they lie in the pages, keys and values, and 64 scales.
constexpr int decode_depth(int dp) { return dp == 64 ? 3 : 2; }
constexpr int decode_slot(int dp) { return 64 * dp + 256; }
constexpr int decode_residents(int dp) { return dp == 256 ? 1 : 2; }  // workgroups that share a CU

template <bool F8, int DP, int QT, bool SMALL>
__global__ __launch_bounds__(256, decode_residents(DP)) void kv_cache_attention_decode_kernel(DecodeView v) {
  constexpr int RT = 16 * QT;        // packed rows of a tile
  constexpr int NI = DP / 64;        // 1024-byte loads for 16 positions; 16-byte pieces of a key row in a lane
  constexpr int VT = DP / 16;        // matrix tiles along the head
  constexpr int NC = DP / 16;        // 16-byte pieces of a row in LDS
  constexpr int KX = NC < 8 ? NC - 1 : 7;
  constexpr int NF = DP + 4;         // row stride of the sums in LDS
  constexpr int S = SMALL ? 4 : 1;   // scales of four neighbouring positions
  constexpr int DEPTH = decode_depth(DP), SLOT = decode_slot(DP), PER = 4 * NI + 1;
  static_assert(4 * 16 * NF * 4 <= 4 * DEPTH * SLOT, "the sums take the ring's place");
  __shared__ __attribute__((aligned(1024))) uint8_t ring[4 * DEPTH * SLOT];
  __shared__ float tops[4][RT], totals[4][RT];
  const KvCacheView& c = v.a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int head = blockIdx.y;
  if ((int)blockIdx.x >= v.workers) {
    if (head == 0) clear_rows_of_nobody(v.a, 64 * (blockIdx.x - v.workers));
    return;
  }
  int64_t piece = 1;
  const LineSpot spot = line_find(
      c.batch, lane,
      [&](int b) {
        const DecodeSpan s = decode_span<RT>(v, b);
        return (int64_t)s.tiles * s.units;
      },
      [&](int64_t total) {
        piece = worker_piece(total, v.workers);
        return piece * blockIdx.x;
      });
  int64_t pos = piece * blockIdx.x, before = spot.before;
  const int64_t stop = min(pos + piece, spot.total);
  int b = spot.b;
  CutTile cut = {0, 0, 0, 0};

  // Where a lane's 16 bytes of a load come from: LDS is filled in order, so the pieces of a row are exchanged at the
  // source.  Keys: piece ^ (row & 7), met again when 16 rows are read a piece at a time; values: piece ^ (row & 3, and
  // 4 for the second 16 rows), when eight rows are read transposed.  A head shorter than DP repeats its end, which q's
  // zeros cancel on one side and the results beyond it are dropped on the other.
  const int stride = c.head;
  uint32_t kfrom[NI], vfrom[2][NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = (64 * i + lane) / NC, q = (64 * i + lane) % NC;
    kfrom[i] = (uint32_t)(r * stride + min(16 * (q ^ (r & KX)), stride - 16));
#pragma unroll
    for (int h = 0; h < 2; ++h) vfrom[h][i] = (uint32_t)(r * stride + min(16 * (q ^ (((r & 3) + 4 * h) & KX)), stride - 16));
  }
  uint8_t* const mine = ring + wave * DEPTH * SLOT;
  const int kread = col * DP + ((NI * grp) << 4), kswap = (col & KX) << 4;
  // transposing read: lane i of 16 points at row i / 2 of eight, 8 bytes of a piece, and receives column i of the piece
  const int vrow = (lane & 15) >> 1;
  const int vread = 32 * DP + (16 * (vrow >> 2) + 4 * grp + (vrow & 3)) * DP + ((vrow & KX) << 4) + 8 * (lane & 1);
  const float factor = v.a.scale * 1.44269504088896341f;  // scores in units of log 2, which exp2 takes as they are
  const int in_page = (1 << c.page_log2) - 1;

  while (b >= 0 && b < c.batch && pos < stop) {
    const DecodeSpan sp = decode_span<RT>(v, b);
    if (sp.tiles == 0) {
      ++b;
      continue;
    }
    const int64_t at = pos - before;  // inside the sequence
    const int tile = divide(at, sp.units);
    if (tile >= sp.tiles) {
      before += (int64_t)sp.tiles * sp.units;
      ++b;
      continue;
    }
    const int u0 = (int)(at - (int64_t)tile * sp.units);
    int u1 = (int)min((int64_t)sp.units, (int64_t)u0 + (stop - pos));
    if (!v.partial) {
      // whole tiles: the worker in whose range a tile begins has all of it
      if (u0 != 0) {
        pos += sp.units - u0;
        continue;
      }
      u1 = sp.units;
    }
    pos += u1 - u0;

    // page numbers are read a step before the loads that need them
    const int* table = c.table + (int64_t)b * c.width;
    const int last = max(sp.hi - 1, 0);
    auto name = [&](int j0, int (&page)[2]) KV_CACHE_INLINE {
#pragma unroll
      for (int h = 0; h < 2; ++h) page[h] = const_int(table, min(j0 + 16 * h, last) >> c.page_log2);
    };
    // 16 positions that no row sees, or that have no page, become zeros (an empty buffer); returns what is there
    auto load = [&](int j0, const int (&pages)[2], int slot) KV_CACHE_INLINE {
      uint8_t* const to = mine + slot * SLOT;
      int there = 0;
      int64_t scale_at[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = j0 + 16 * h, named = __builtin_amdgcn_readfirstlane(pages[h]);
        const bool has = (unsigned)named < (unsigned)c.pages && j < sp.hi && j + 16 > sp.lo;
        const int page = has ? named : 0, row = j & in_page;
        there |= has ? 1 << h : 0;
        const int64_t at = kv_row(c, page, head, row);
        scale_at[h] = kv_scale(c, page, head, 0) * 4;
        const __amdgpu_buffer_rsrc_t kr = kv_rsrc(c.codes[0] + at, has ? 16 * stride : 0);
        const __amdgpu_buffer_rsrc_t vr = kv_rsrc(c.codes[1] + at, has ? 16 * stride : 0);
#pragma unroll
        for (int i = 0; i < NI; ++i)
          load16_to_lds(kr, to + 16 * DP * h + 1024 * i, kfrom[i]);
#pragma unroll
        for (int i = 0; i < NI; ++i)
          load16_to_lds(vr, to + 32 * DP + 16 * DP * h + 1024 * i, vfrom[h][i]);
      }
      // lanes 0 to 31: key scales of the 32 positions, 32 to 63: value scales
      const int row = ((j0 & in_page) + (lane & 31)) & in_page;  // (the second 16 may begin a page)
      const char* from = reinterpret_cast<const char*>(lane & 32 ? c.scales[1] : c.scales[0]) + (lane & 16 ? scale_at[1] : scale_at[0]);
      load4_to_lds(from + (row >> c.block_log2) * 4, to + 64 * DP);
      return there;
    };
    const int j_end = (sp.first + u1) * kUnit;
    int j = (sp.first + u0) * kUnit + 32 * wave;
    int there[DEPTH], pages[2];
    const bool any = sp.hi > 0;
    if (any) name(j, pages);

    // the tile's rows: packed row r is row r / group and head r % group
    const int r0 = tile * RT, rows = min(sp.s.n * v.a.group - r0, RT);
    bf16x8 q[QT][DP / 32];
    int sees_lo[QT], sees_hi[QT];  // positions that this lane's row sees
    int all_lo = sp.lo, all_hi = sp.hi;  // ... and that every row of the tile sees
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const int r = r0 + min(16 * t + col, rows - 1);
      const int i = r / v.a.group, h = r - i * v.a.group;
      const uint16_t* qr = v.a.q + ((int64_t)(sp.s.row0 + i) * v.a.q_heads + head * v.a.group + h) * c.head;
#pragma unroll
      for (int s = 0; s < DP / 32; ++s) {
        const int d = grp * (DP / 4) + 8 * s;
        q[t][s] = d < c.head ? *reinterpret_cast<const bf16x8*>(qr + d) : bf16x8{};
      }
      const int p = sp.s.len - sp.s.n + i;
      sees_hi[t] = v.a.causal ? min(sp.hi, p + 1) : sp.hi;
      sees_lo[t] = window_start(v.a, p);
    }
    if (v.a.causal) all_hi = min(all_hi, sp.s.len - sp.s.n + r0 / v.a.group + 1);
    if (v.a.window > 0) all_lo = window_start(v.a, sp.s.len - sp.s.n + (r0 + rows - 1) / v.a.group);

    // q is here before the loop's loads are counted
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int s = 0; s < DP / 32; ++s) asm volatile("" ::"v"(q[t][s]));
    if (any) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        there[d] = 0;
        if (j + d * kUnit < j_end) {
          there[d] = load(j + d * kUnit, pages, d);
          name(j + (d + 1) * kUnit, pages);
        }
      }
    }

    floatx4 acc[QT][VT];
    float top[QT], sum[QT], factor_v[QT], weighed[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      top[t] = kNoScore;
      factor_v[t] = 1.0f;
      weighed[t] = 0.0f;
      sum[t] = 0.0f;
#pragma unroll
      for (int i = 0; i < VT; ++i) acc[t][i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    auto step = [&](int slot) KV_CACHE_INLINE {
      // this slot's loads are the oldest under way
      if (j + (DEPTH - 1) * kUnit < j_end) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((DEPTH - 1) * PER) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      const uint8_t* const from = mine + slot * SLOT;
      uintx4 k[2][NI];
      intx2 raw[VT];
      float ks[2 * S], vs[2 * S];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < NI; ++i) k[h][i] = *reinterpret_cast<const uintx4*>(from + 16 * DP * h + ((kread + 16 * i) ^ kswap));
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < S; ++i) {
          ks[h * S + i] = *reinterpret_cast<const float*>(from + 64 * DP + 4 * (16 * h + 4 * grp + i));
          vs[h * S + i] = *reinterpret_cast<const float*>(from + 64 * DP + 4 * (32 + 16 * h + 4 * grp + i));
        }
#pragma unroll
      for (int t = 0; t < VT; ++t) raw[t] = read_columns(from + (vread ^ (t << 4)));
      const int here = there[slot], j0 = j;
      // the slot is empty again
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (j + DEPTH * kUnit < j_end) {
        there[slot] = load(j + DEPTH * kUnit, pages, slot);
        name(j + (DEPTH + 1) * kUnit, pages);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (here == 0) return;
      const bool edge = j0 < all_lo || j0 + 32 > all_hi || here != 3;
      if (F8 && (j0 < sp.lo || j0 + 32 > sp.hi)) {
        KV_CACHE_RARE();
        // positions that nobody sees may hold NaN codes, which a weight of zero does not cancel
        uint32_t keep[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int at = j0 + 16 * (e >> 2) + 4 * grp + (e & 3);
          keep[e >> 2] |= at >= sp.lo && at < sp.hi ? 0xffu << (8 * (e & 3)) : 0u;
        }
#pragma unroll
        for (int t = 0; t < VT; ++t) raw[t] = intx2{(int)(raw[t][0] & keep[0]), (int)(raw[t][1] & keep[1])};
      }
#pragma unroll
      for (int i = 0; i < 2 * S; ++i) keep_to_its_rows(ks[i], vs[i]);
      floatx4 s[QT][2];
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) s[t][h] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int m = 0; m < DP / 32; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bf16x8 kk = widen8<F8>(k[h][m >> 1][2 * (m & 1)], k[h][m >> 1][2 * (m & 1) + 1]);
#pragma unroll
          for (int t = 0; t < QT; ++t) s[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kk, q[t][m], s[t][h], 0, 0, 0);
          // one piece widened while the one before is multiplied, and no more of them in registers
          __builtin_amdgcn_sched_barrier(0);
        }
      halfx8 p[QT];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = s[t][e >> 2][e & 3] * (ks[(e >> 2) * S + (e & (S - 1))] * factor);
        if (v.a.cap > 0.0f) {
          KV_CACHE_RARE();
          cap_scores(y, v.a.cap, v.a.per_cap);
        }
        if (edge) {
          KV_CACHE_RARE();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int at = j0 + 16 * (e >> 2) + 4 * grp + (e & 3);
            y[e] = ((here >> (e >> 2)) & 1) && at >= sees_lo[t] && at < sees_hi[t] ? y[e] : -INFINITY;
          }
        }
        float most = y[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) most = __builtin_fmaxf(most, y[e]);
        if (__any(most > top[t] + kLag)) {
          most = __builtin_fmaxf(most, __shfl_xor(most, 16));
          most = __builtin_fmaxf(most, __shfl_xor(most, 32));
          const float now = __builtin_fmaxf(top[t], most);
          const float scale = __builtin_amdgcn_exp2f(top[t] - now);
          top[t] = now;
          sum[t] *= scale;
          weighed[t] *= scale;
#pragma unroll
          for (int i = 0; i < VT; ++i) acc[t][i] *= scale;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = __builtin_amdgcn_exp2f(y[e] - top[t]);
        float x[2 * S];
#pragma unroll
        for (int i = 0; i < 2 * S; ++i) x[i] = vs[i] * factor_v[t];
        if (__any(!factor_fits(x))) {
          KV_CACHE_RARE();
          float weight = 0.0f, before = weighed[t];
#pragma unroll
          for (int e = 0; e < 8; ++e) weight = __builtin_fmaxf(weight, __builtin_fabsf(y[e] * vs[(e >> 2) * S + (e & (S - 1))]));
#pragma unroll
          for (int off = 16; off < 64; off *= 2) {
            weight = __builtin_fmaxf(weight, __shfl_xor(weight, off));
            before = __builtin_fmaxf(before, __shfl_xor(before, off));
          }
          const float now = new_factor(weight, before, factor_v[t]);
          const float step = now * reciprocal(factor_v[t]);
          factor_v[t] = now;
          weighed[t] *= step;
#pragma unroll
          for (int i = 0; i < VT; ++i) acc[t][i] *= step;
#pragma unroll
          for (int i = 0; i < 2 * S; ++i) x[i] = finite_product(vs[i], now);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float four = (y[4 * h] + y[4 * h + 1]) + (y[4 * h + 2] + y[4 * h + 3]);
          sum[t] += four;
          if constexpr (SMALL) {
#pragma unroll
            for (int e = 0; e < 4; ++e) weighed[t] = __builtin_fmaf(y[4 * h + e], __builtin_fabsf(x[4 * h + e]), weighed[t]);
          } else {
            weighed[t] = __builtin_fmaf(four, __builtin_fabsf(x[h]), weighed[t]);
          }
        }
        uintx4 w;
#pragma unroll
        for (int e = 0; e < 8; e += 2)
          w[e >> 1] = pack_f16x2(y[e] * x[(e >> 2) * S + (e & (S - 1))], y[e + 1] * x[(e >> 2) * S + ((e + 1) & (S - 1))]);
        p[t] = __builtin_bit_cast(halfx8, w);
      }
#pragma unroll
      for (int i = 0; i < VT; ++i) {
        const halfx8 vv = widen8_f16<F8>(raw[i][0], raw[i][1]);
#pragma unroll
        for (int t = 0; t < QT; ++t) acc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, p[t], acc[t][i], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (any) {
      while (j < j_end) {
        static_for<0, DEPTH>([&](auto d) KV_CACHE_INLINE {
          if (j < j_end) {
            step(decltype(d)::value);
            j += kUnit;
          }
        });
      }
    }

    // the four waves' sums, 16 rows at a time, where the ring was (each wave has taken all it asked for)
    float* const sums = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      sum[t] += __shfl_xor(sum[t], 16);
      sum[t] += __shfl_xor(sum[t], 32);
      if (grp == 0) {
        tops[wave][16 * t + col] = top[t];
        totals[wave][16 * t + col] = sum[t];
      }
    }
    const bool whole = u0 == 0 && u1 == sp.units;
    if (u0 == 0 && !whole)
      cut = CutTile{sp.s.row0, r0, rows, divide(before + (int64_t)(tile + 1) * sp.units - 1, piece) - (int)blockIdx.x + 1};
    // a range that begins inside a tile is its worker's first, one that ends inside its last
    float* part = v.partial + ((int64_t)head * 2 * v.workers + 2 * blockIdx.x + (u0 == 0 ? 1 : 0)) * RT * (c.head + 2);
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      __syncthreads();
      {
        const int r = 16 * t + col;
        const float m = __builtin_fmaxf(__builtin_fmaxf(tops[0][r], tops[1][r]), __builtin_fmaxf(tops[2][r], tops[3][r]));
        const float scale = __builtin_amdgcn_exp2f(top[t] - m);
        const float less = reciprocal(factor_v[t]);
#pragma unroll
        for (int i = 0; i < VT; ++i)
          *reinterpret_cast<floatx4*>(&sums[(wave * 16 + col) * NF + 16 * i + 4 * grp]) = acc[t][i] * scale * less;
      }
      __syncthreads();
      const int r = 16 * t + (tid >> 4);
      if (r < rows) {
        const float m = __builtin_fmaxf(__builtin_fmaxf(tops[0][r], tops[1][r]), __builtin_fmaxf(tops[2][r], tops[3][r]));
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) l += totals[w][r] * __builtin_amdgcn_exp2f(tops[w][r] - m);
        const int i = (r0 + r) / v.a.group, h = r0 + r - i * v.a.group;
        const int64_t at_row = (int64_t)(sp.s.row0 + i) * v.a.q_heads + head * v.a.group + h;
        const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
        for (int d = (tid & 15) * 4; d < c.head; d += 64) {
          floatx4 o = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int w = 0; w < 4; ++w) o += *reinterpret_cast<const floatx4*>(&sums[(w * 16 + (tid >> 4)) * NF + d]);
          if (whole) {
            const uintx2 packed = {pack_bf16x2(o[0] * inverse, o[1] * inverse), pack_bf16x2(o[2] * inverse, o[3] * inverse)};
            *reinterpret_cast<uintx2*>(v.a.out + at_row * c.head + d) = packed;
          } else {
            *reinterpret_cast<floatx4*>(part + r * c.head + d) = o;
          }
        }
        if ((tid & 15) == 0) {
          if (!whole) {
            part[RT * c.head + r] = m;
            part[RT * c.head + RT + r] = l;
          } else if (v.a.lse) {
            v.a.lse[at_row] = l == 0.0f ? -INFINITY : (m + __builtin_log2f(l)) * 0.693147180559945309f;
          }
        }
      }
    }
    __syncthreads();  // tops, sums and the ring are the next range's
  }
  if (v.partial && head == 0 && tid == 0) v.cuts[blockIdx.x] = cut;
}

// ---- many rows for each sequence ---------------------------------------------------------------------
//
// A workgroup of four waves takes 128 packed rows of a sequence and cache head, 32 a wave, and goes
// over the positions 64 at a time.  The four waves widen a stage's codes (exact) once for all: keys to bf16
// as [position][d], values to f16, transposed, as [d][position], both in LDS, two stages taking turns with one barrier
// each; the next stage's codes are on their way in registers.  Per wave and stage, with n = lane & 31 and h = lane >> 5:
//   S^T = K Q^T   column n of the result is a row of q, a lane holds positions 8 j + 4 h + i
//   O^T = V^T P^T where the values lie in LDS in that same order of positions, so the weights go from one
//                 product into the next without leaving their lane.
// Scales and roundings are as above.
//
// A stage goes in halves of 32 positions, so that vector instructions stand in the shadow of matrix instructions: the
// second half's scores run among the first half's exponentials, the first half's results among the second half's
// exponentials, the second half's results among the widening of the next stage.
//
// 16-byte pieces of a key row are stored at piece ^ (position & 15), those of a value row at
// piece ^ ((d ^ d >> 2) & 7): eight lanes that read or write together then meet eight different places.
//
// Bound: two waves share a SIMD, and each needs 1400 cycles of vector instructions (a quarter of them exponentials) and
// 1024 of matrix instructions for a stage of a head of 128, the matrix pipes being busy for 38% of the time.  8192 rows of
// 32 heads on 8192 positions, causal: 630 to 670 us from run to run, 820 to 870 TFLOP/s, where a large product of matrices
// reaches 1357.
constexpr int kStage = 64;
constexpr int kPromptRows = 128;
// Where a call has few tiles, their positions are cut: into pieces that give kPieces workgroups at most (six chunks of
// prompts, 312 tiles and heads: 127 us with 512, which cuts none, 76 with 768 and two pieces a tile, 70 with 1024, 84 with
// 1536), kLeastSplits to kMostSplits for a tile, of kLeastStages stages or more.  512 workgroups run at a time, so tiles
// that fill them once stay whole: 4 chunks of 512 rows on 4096 positions (512 tiles and heads) take 179 us whole and 199
// cut in two, two prompts of 1024 65 and 73; from 342 tiles and heads on, where three pieces each would be too many, part
// of the device has nothing to do.  How many tiles there are is device data, so each workgroup counts them.
constexpr int kPieces = 1024;
constexpr int kLeastSplits = 3;
constexpr int kMostSplits = 16;
constexpr int kLeastStages = 4;

struct PromptView {
  AttentionView a;
  float* partial;   // [pieces][heads][tile rows][head + 2], or null: no tile is cut
  CutTile* cuts;    // [pieces], of the tile whose first piece it is
  int slots;        // pieces of tiles, at most
  int pieces;       // wanted, if tiles can be cut
  int rows_from;    // sequences with more packed rows than this are this kernel's
};

__device__ __forceinline__ int prompt_tiles(const AttentionView& v, int rows_from, int b) {
  const int rows = kv_sequence(v.c, b).n * v.group;
  return rows > rows_from ? (rows + kPromptRows - 1) / kPromptRows : 0;
}

template <bool F8, int DP, bool SMALL>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void kv_cache_attention_prompt_kernel(PromptView v) {
  constexpr int RT = kPromptRows;
  constexpr int KC = DP / 8;             // 16-byte pieces of a key row
  constexpr int KX = KC < 16 ? KC - 1 : 15;
  constexpr int KN = DP / 64;            // pieces of 16 codes that a lane stages of the keys
  constexpr int VN = DP < 128 ? 1 : DP / 128;  // groups of 8 positions x 4 values that a lane stages
  constexpr int S = SMALL ? 4 : 1;       // scales of four neighbouring positions
  constexpr int QK = DP / 16;            // steps of 32 positions' scores, and of their results
  constexpr int PIECES = 2 * KN + 2 * VN;  // of a lane's staging
  __shared__ uintx4 keys[2][kStage * KC];
  __shared__ uintx4 vals[2][DP * 8];
  __shared__ float kscale[2][kStage], vscale[2][kStage];
  __shared__ int there[2][4];
  const KvCacheView& c = v.a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, h = lane >> 5;
  const int head = blockIdx.x % c.heads, slot = v.slots - 1 - blockIdx.x / c.heads;  // the last tiles of a prompt see the most
  int splits = 1;
  const LineSpot spot = line_find(
      c.batch, lane, [&](int b) { return (int64_t)prompt_tiles(v.a, v.rows_from, b); },
      [&](int64_t total) {
        if (v.partial && kLeastSplits * total <= v.pieces) splits = (int)min((uint32_t)v.pieces / max((uint32_t)total, 1u), (uint32_t)kMostSplits);
        return (int64_t)((uint32_t)slot / (uint32_t)splits);
      });
  const int tile = slot / splits, split = slot - tile * splits;
  const bool notes = v.partial && head == 0 && tid == 0 && slot < v.pieces;
  if (spot.b < 0) {
    if (notes) v.cuts[slot] = CutTile{0, 0, 0, 0};
    return;
  }
  const int b = spot.b;
  const KvSequence s = kv_sequence(c, b);
  const int r0 = __builtin_amdgcn_readfirstlane((int)(tile - spot.before)) * RT, rows = min(s.n * v.a.group - r0, RT);
  const int p_first = s.len - s.n + r0 / v.a.group, p_last = s.len - s.n + (r0 + rows - 1) / v.a.group;
  // positions that some row of the tile sees, and that all of them see
  const int lo = window_start(v.a, p_first);
  const int hi = v.a.causal ? min(s.len, p_last + 1) : s.len;
  const int all_lo = window_start(v.a, p_last);
  const int all_hi = v.a.causal ? min(s.len, p_first + 1) : s.len;
  const int u_first = lo / kStage, u_count = max((hi + kStage - 1) / kStage - u_first, 0);
  splits = min(splits, max(u_count / kLeastStages, 1));
  if (notes) v.cuts[slot] = CutTile{s.row0, r0, split == 0 && splits > 1 ? rows : 0, splits};
  if (split >= splits) return;
  const int u0 = u_first + (int)((int64_t)u_count * split / splits);
  const int u1 = u_first + (int)((int64_t)u_count * (split + 1) / splits);

  bf16x8 q[DP / 16];
  int sees_lo, sees_hi;
  {
    const int r = r0 + min(wave * 32 + n, rows - 1);
    const int i = r / v.a.group, g = r - i * v.a.group;
    const uint16_t* qr = v.a.q + ((int64_t)(s.row0 + i) * v.a.q_heads + head * v.a.group + g) * c.head;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) q[k] = 16 * k < c.head ? *reinterpret_cast<const bf16x8*>(qr + 16 * k + 8 * h) : bf16x8{};
    const int p = s.len - s.n + i;
    sees_hi = v.a.causal ? min(s.len, p + 1) : s.len;
    sees_lo = window_start(v.a, p);
  }
  floatx16 acc[DP / 32];
  float top = kNoScore, sum = 0.0f, factor_v = 1.0f, weighed = 0.0f;
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = 0.0f;
  const float factor = v.a.scale * 1.44269504088896341f;  // scores in units of log 2, which exp2 takes as they are
  const int* table = c.table + (int64_t)b * c.width;
  const int in_page = (1 << c.page_log2) - 1, in_block = (1 << c.block_log2) - 1;

  // Stage: wave w brings positions 16 w to 16 w + 15.  Keys: 16 codes a piece, lane -> (position, piece); values: lane ->
  // (eight positions as S^T orders them, four values).
  uintx4 kraw[KN];
  uint32_t vraw[VN][8];
  float ks_raw, vs_raw;
  bool present;
  const int kpos = lane / (DP / 16), kpiece = lane % (DP / 16);  // 64 / (DP / 16) positions at once
  const int vquad = lane % (DP < 128 ? DP / 4 : 32), vhalf = DP < 128 ? (lane / (DP / 4)) & 1 : h;
  auto page_of = [&](int u) KV_CACHE_INLINE {
    return const_int(table, min(u * kStage + 16 * wave, hi - 1) >> c.page_log2);
  };
  auto fetch = [&](int u, int page) KV_CACHE_INLINE {
    const int j = u * kStage + 16 * wave;
    present = (unsigned)page < (unsigned)c.pages && u < u1 && j < hi && j + 16 > lo;
    page = present ? page : 0;  // read, and masked
    const int row = (u * kStage + 16 * wave) & in_page;
    const int64_t at = kv_row(c, page, head, row);
    const uint8_t* kp = c.codes[0] + at;
    const uint8_t* vp = c.codes[1] + at;
#pragma unroll
    for (int i = 0; i < KN; ++i)
      kraw[i] = *reinterpret_cast<const uintx4*>(kp + (uint32_t)((i * (1024 / DP) + kpos) * c.head + min(16 * kpiece, c.head - 16)));
#pragma unroll
    for (int i = 0; i < VN; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        vraw[i][e] = *reinterpret_cast<const uint32_t*>(
            vp + (uint32_t)((8 * (e >> 2) + 4 * vhalf + (e & 3)) * c.head + min(128 * i + 4 * vquad, c.head - 4)));
    const int64_t sc = kv_scale(c, page, head, row);
    const float* ksp = c.scales[0] + sc;
    const float* vsp = c.scales[1] + sc;
    const uint32_t place = (uint32_t)((row & in_block) + (lane & 15)) >> c.block_log2;
    ks_raw = ksp[place];
    vs_raw = vsp[place];
  };
  auto stage_scales = [&](int u, int buf) KV_CACHE_INLINE {
    const int j0 = u * kStage + 16 * wave;
    if (F8 && (!present || j0 < lo || j0 + 16 > hi)) {
      KV_CACHE_RARE();
      // positions that nobody sees may hold NaN codes, which a weight of zero does not cancel
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = j0 + 8 * (e >> 2) + 4 * vhalf + (e & 3);
#pragma unroll
        for (int i = 0; i < VN; ++i) vraw[i][e] = present && j >= lo && j < hi ? vraw[i][e] : 0u;
      }
    }
    float ks = ks_raw, vs = vs_raw;
    keep_to_its_rows(ks, vs);
    if (lane < 16) {
      kscale[buf][16 * wave + lane] = ks * factor;
      vscale[buf][16 * wave + lane] = vs;
    }
    if (lane == 0) there[buf][wave] = present ? 1 : 0;
  };
  auto stage_piece = [&](auto at, int buf) KV_CACHE_INLINE {
    constexpr int P = decltype(at)::value;
    if constexpr (P < 2 * KN) {
      constexpr int I = P / 2, H = P % 2;
      const int pos = 16 * wave + I * (1024 / DP) + kpos;
      keys[buf][pos * KC + ((2 * kpiece + H) ^ (pos & KX))] = __builtin_bit_cast(uintx4, widen8<F8>(kraw[I][2 * H], kraw[I][2 * H + 1]));
    } else {
      constexpr int I = (P - 2 * KN) / 2, T = 2 * ((P - 2 * KN) % 2);
      const int d = 128 * I + 4 * vquad + T;
      uint32_t one[8][1];
#pragma unroll
      for (int e = 0; e < 8; ++e) one[e][0] = vraw[I][e];
      uintx4 va, vb;
      columns<F8, T>(one, va, vb);
      vals[buf][d * 8 + ((2 * wave + vhalf) ^ ((d ^ (d >> 2)) & 7))] = va;
      vals[buf][d * 8 + 8 + ((2 * wave + vhalf) ^ (((d + 1) ^ (d >> 2)) & 7))] = vb;
    }
  };

  floatx16 sc[2];
  halfx8 p[2][2];
  float kq[4 * S], vq[4 * S], more, more_weighed;  // vq: with the factor
  auto key_piece = [&](int buf, int kt, int k) KV_CACHE_INLINE {
    const int pos = 32 * kt + n;
    return __builtin_bit_cast(bf16x8, keys[buf][pos * KC + ((2 * k + h) ^ (pos & KX))]);
  };
  auto value_piece = [&](int buf, int kt, int at) KV_CACHE_INLINE {  // at: which 16 positions, then which 32 values
    const int g = 2 * kt + at / (DP / 32), d = 32 * (at % (DP / 32)) + n;
    return __builtin_bit_cast(halfx8, vals[buf][d * 8 + ((2 * g + h) ^ ((d ^ (d >> 2)) & 7))]);
  };
  auto score = [&](auto kt_, bf16x8 a, auto k_) KV_CACHE_INLINE {
    constexpr int KT = decltype(kt_)::value, K = decltype(k_)::value;
    floatx16 from = sc[KT];
    if constexpr (K == 0) {
#pragma unroll
      for (int e = 0; e < 16; ++e) from[e] = 0.0f;
    }
    sc[KT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, q[K], from, 0, 0, 0);
  };
  auto result = [&](auto kt_, halfx8 a, auto at_) KV_CACHE_INLINE {
    constexpr int KT = decltype(kt_)::value, G = decltype(at_)::value / (DP / 32), I = decltype(at_)::value % (DP / 32);
    acc[I] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, p[KT][G], acc[I], 0, 0, 0);
  };
  // The scales of a half; where scores are capped or some position is not seen, the scores themselves are made final.
  auto prepare = [&](bool edge, int buf, int j0, auto kt_) KV_CACHE_INLINE {
    constexpr int KT = decltype(kt_)::value;
#pragma unroll
    for (int i = 0; i < 4 * S; ++i) {
      const int pos = 32 * KT + 8 * (i / S) + 4 * h + i % S;
      kq[i] = kscale[buf][pos];
      vq[i] = vscale[buf][pos] * factor_v;
    }
    if (v.a.cap > 0.0f) {
      KV_CACHE_RARE();
      float x[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = sc[KT][r] * kq[(r >> 2) * S + (r & (S - 1))];
      cap_scores(x, v.a.cap, v.a.per_cap);
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[KT][r] = x[r];
#pragma unroll
      for (int i = 0; i < 4 * S; ++i) kq[i] = 1.0f;
    }
    if (edge) {
      KV_CACHE_RARE();
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int pos = j0 + 32 * KT + 8 * (r >> 2) + 4 * h + (r & 3);
        const bool seen = there[buf][2 * KT + (r >> 3)] != 0 && pos >= sees_lo && pos < sees_hi;
        sc[KT][r] = seen ? sc[KT][r] * kq[(r >> 2) * S + (r & (S - 1))] : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 4 * S; ++i) kq[i] = 1.0f;
    }
  };
  // the weights of positions 8 I + 4 h to + 3 of a half
  auto weigh = [&](auto kt_, auto unit) KV_CACHE_INLINE {
    constexpr int KT = decltype(kt_)::value, I = decltype(unit)::value;
    float w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[KT][4 * I + e], kq[I * S + (e & (S - 1))], -top));
    const float four = (w[0] + w[1]) + (w[2] + w[3]);
    more = I == 0 ? four : more + four;
    if constexpr (I == 0) more_weighed = 0.0f;
    if constexpr (!SMALL) more_weighed = __builtin_fmaf(four, __builtin_fabsf(vq[I]), more_weighed);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] *= vq[I * S + (e & (S - 1))];
      if constexpr (SMALL) more_weighed += __builtin_fabsf(w[e]);
    }
    uintx4 packed = I & 1 ? __builtin_bit_cast(uintx4, p[KT][I >> 1]) : uintx4{0u, 0u, 0u, 0u};
    packed[2 * (I & 1)] = pack_f16x2(w[0], w[1]);
    packed[2 * (I & 1) + 1] = pack_f16x2(w[2], w[3]);
    p[KT][I >> 1] = __builtin_bit_cast(halfx8, packed);
  };
  // Where the weights' sum shows that the maximum in use lags too far behind, or a scale leaves the factor's range, the
  // half is weighed again, on scores that are products rounded as the maximum is: the unrounded ones that it was weighed on
  // first may lie beside it by 2^-24 of themselves, which from scores of 2^27 on is more than a weight bears.
  auto catch_up = [&](int buf, auto kt_) KV_CACHE_INLINE {
    constexpr int KT = decltype(kt_)::value;
    if (__any(more > 32.0f || !factor_fits(vq))) {
      KV_CACHE_RARE();
      float most = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        sc[KT][r] *= kq[(r >> 2) * S + (r & (S - 1))];
        most = __builtin_fmaxf(most, sc[KT][r]);
      }
#pragma unroll
      for (int i = 0; i < 4 * S; ++i) kq[i] = 1.0f;
      most = __builtin_fmaxf(most, __shfl_xor(most, 32));
      const float now = __builtin_fmaxf(top, most);
      const float scale = __builtin_amdgcn_exp2f(top - now);
      top = now;
      sum *= scale;
      float weight = 0.0f;
#pragma unroll
      for (int i = 0; i < 4 * S; ++i) vq[i] = vscale[buf][32 * KT + 8 * (i / S) + 4 * h + i % S];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int i = (r >> 2) * S + (r & (S - 1));
        weight = __builtin_fmaxf(weight, __builtin_fabsf(__builtin_amdgcn_exp2f(sc[KT][r] - top) * vq[i]));
      }
      weight = __builtin_fmaxf(weight, __shfl_xor(weight, 32));
      const float next = new_factor(weight, __builtin_fmaxf(weighed, __shfl_xor(weighed, 32)) * scale, factor_v);
      const float step = scale * (next * reciprocal(factor_v));
      factor_v = next;
      weighed *= step;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) acc[i] *= step;
#pragma unroll
      for (int i = 0; i < 4 * S; ++i) vq[i] = finite_product(vq[i], next);
      static_for<0, 4>([&](auto unit) KV_CACHE_INLINE { weigh(kt_, unit); });
    }
    sum += more;
    weighed += more_weighed;
  };
  constexpr std::integral_constant<int, 0> kFirst{};
  constexpr std::integral_constant<int, 1> kSecond{};

  if (u0 < u1) {
    fetch(u0, page_of(u0));
    stage_scales(u0, 0);
    static_for<0, PIECES>([&](auto at) KV_CACHE_INLINE { stage_piece(at, 0); });
    int next = page_of(u0 + 2);
    fetch(u0 + 1, page_of(u0 + 1));
    __syncthreads();
    for (int u = u0; u < u1; ++u) {
      const int buf = (u - u0) & 1, j0 = u * kStage;
      {
        bf16x8 a = key_piece(buf, 0, 0);
        static_for<0, QK>([&](auto k) KV_CACHE_INLINE {
          constexpr int K = decltype(k)::value;
          const bf16x8 now = a;
          if constexpr (K + 1 < QK) a = key_piece(buf, 0, K + 1);
          score(kFirst, now, k);
        });
      }
      const bool gap = (there[buf][0] & there[buf][1] & there[buf][2] & there[buf][3]) == 0;
      const bool edge = __builtin_amdgcn_readfirstlane((int)(gap || j0 < all_lo || j0 + kStage > all_hi)) != 0;
      prepare(edge, buf, j0, kFirst);
      {
        bf16x8 a = key_piece(buf, 1, 0);
        static_for<0, QK>([&](auto k) KV_CACHE_INLINE {
          constexpr int K = decltype(k)::value;
          const bf16x8 now = a;
          if constexpr (K + 1 < QK) a = key_piece(buf, 1, K + 1);
          score(kSecond, now, k);
          static_for<K * 4 / QK, (K + 1) * 4 / QK>([&](auto unit) KV_CACHE_INLINE { weigh(kFirst, unit); });
          KV_CACHE_FENCE();
        });
      }
      catch_up(buf, kFirst);
      prepare(edge, buf, j0, kSecond);
      {
        halfx8 a = value_piece(buf, 0, 0);
        static_for<0, QK>([&](auto k) KV_CACHE_INLINE {
          constexpr int K = decltype(k)::value;
          const halfx8 now = a;
          if constexpr (K + 1 < QK) a = value_piece(buf, 0, K + 1);
          result(kFirst, now, k);
          static_for<K * 4 / QK, (K + 1) * 4 / QK>([&](auto unit) KV_CACHE_INLINE { weigh(kSecond, unit); });
          KV_CACHE_FENCE();
        });
      }
      catch_up(buf, kSecond);
      // past the last stage, of whatever is there
      stage_scales(u + 1, buf ^ 1);
      {
        halfx8 a = value_piece(buf, 1, 0);
        static_for<0, QK>([&](auto k) KV_CACHE_INLINE {
          constexpr int K = decltype(k)::value;
          const halfx8 now = a;
          if constexpr (K + 1 < QK) a = value_piece(buf, 1, K + 1);
          result(kSecond, now, k);
          static_for<K * PIECES / QK, (K + 1) * PIECES / QK>([&](auto at) KV_CACHE_INLINE { stage_piece(at, buf ^ 1); });
          KV_CACHE_FENCE();
        });
      }
      fetch(u + 2, next);
      next = page_of(u + 3);
      __syncthreads();
    }
  }

  const float l = sum + __shfl_xor(sum, 32);
  const int r = wave * 32 + n;
  if (r >= rows) return;
  const int i = (r0 + r) / v.a.group, g = r0 + r - i * v.a.group;
  const int64_t at_row = (int64_t)(s.row0 + i) * v.a.q_heads + head * v.a.group + g;
  const bool joined = splits > 1;
  float* part = joined ? v.partial + ((int64_t)slot * c.heads + head) * RT * (c.head + 2) : nullptr;
  const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
  const float less = reciprocal(factor_v);
#pragma unroll
  for (int i2 = 0; i2 < DP / 32; ++i2)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 32 * i2 + 8 * e + 4 * h;
      if (d >= c.head) continue;
      floatx4 o;
#pragma unroll
      for (int f = 0; f < 4; ++f) o[f] = acc[i2][4 * e + f] * less;
      if (joined) *reinterpret_cast<floatx4*>(part + (int64_t)r * c.head + d) = o;
      else *reinterpret_cast<uintx2*>(v.a.out + at_row * c.head + d) =
          uintx2{pack_bf16x2(o[0] * inverse, o[1] * inverse), pack_bf16x2(o[2] * inverse, o[3] * inverse)};
    }
  if (h == 0 && joined) {
    part[(int64_t)RT * c.head + r] = top;
    part[(int64_t)RT * c.head + RT + r] = l;
  } else if (h == 0 && v.a.lse) {
    v.a.lse[at_row] = l == 0.0f ? -INFINITY : (top + __builtin_log2f(l)) * 0.693147180559945309f;
  }
}

// ---- the pieces of cut tiles joined --------------------------------------------------------------------

struct JoinPart {
  const CutTile* cuts;
  const float* partial;
  int64_t head_step, cut_step, piece_step;  // floats from head to head, tile to tile, piece to piece
  int64_t back;     // less for the pieces after the first
  int tile_rows;
};

struct JoinView {
  AttentionView a;
  JoinPart parts[2];
  unsigned blocks;  // the first part's
};

// L lanes for a row, four values each; the pieces in their order.  The maxima and sums of up to L pieces are a lane's
// each, and the results are under way four pieces at a time.
// Bound: three dependent reads (the tile's note, the maxima, the results): 4.2 us for one sequence, 5.0 for 64.
template <int L>
__global__ __launch_bounds__(256) void kv_cache_attention_join_kernel(JoinView v) {
  const JoinPart& p = blockIdx.x < v.blocks ? v.parts[0] : v.parts[1];
  const int at = (int)(blockIdx.x - (blockIdx.x < v.blocks ? 0u : v.blocks)) * (256 / L);
  const int size = v.a.c.head, head = blockIdx.y, lane = threadIdx.x & (L - 1);
  const int item = at / p.tile_rows;
  const CutTile cut = p.cuts[item];
  const int r = at % p.tile_rows + (int)threadIdx.x / L;
  if (r >= cut.rows) return;
  const float* first = p.partial + head * p.head_step + item * p.cut_step;
  auto piece = [&](int w) { return first + (w * p.piece_step - (w > 0 ? p.back : 0)); };
  const int64_t tops = (int64_t)p.tile_rows * size + r;
  const int d = min(4 * lane, size - 4);
  float m = kNoScore, l = 0.0f;
  floatx4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int w0 = 0; w0 < cut.pieces; w0 += L) {
    const int here = min(cut.pieces - w0, L);
    const float* q = piece(w0 + min(lane, here - 1)) + tops;
    const float top = q[0], sum = q[p.tile_rows];
    float now = __builtin_fmaxf(m, top);
#pragma unroll
    for (int off = L / 2; off > 0; off >>= 1) now = __builtin_fmaxf(now, __shfl_xor(now, off, L));
    const float old = __builtin_amdgcn_exp2f(m - now);
    const float scale = lane < here ? __builtin_amdgcn_exp2f(top - now) : 0.0f;
    m = now;
    l = l * old + sum * scale;
    o *= old;
    for (int w = 0; w < here; w += 4) {
      floatx4 x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = *reinterpret_cast<const floatx4*>(piece(w0 + min(w + e, here - 1)) + (int64_t)r * size + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) o += x[e] * (w + e < here ? __shfl(scale, w + e, L) : 0.0f);
    }
  }
#pragma unroll
  for (int off = L / 2; off > 0; off >>= 1) l += __shfl_xor(l, off, L);
  const int i = (cut.first + r) / v.a.group, g = cut.first + r - i * v.a.group;
  const int64_t at_row = (int64_t)(cut.row0 + i) * v.a.q_heads + head * v.a.group + g;
  const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
  if (4 * lane < size)
    *reinterpret_cast<uintx2*>(v.a.out + at_row * size + d) =
        uintx2{pack_bf16x2(o[0] * inverse, o[1] * inverse), pack_bf16x2(o[2] * inverse, o[3] * inverse)};
  if (lane == 0 && v.a.lse) v.a.lse[at_row] = l == 0.0f ? -INFINITY : (m + __builtin_log2f(l)) * 0.693147180559945309f;
}

// Packed rows of a sequence up to which the streaming kernel takes it in calls that both kernels serve, two of its
// tiles: 64 sequences on 4096 positions take 201 us there and 202 in the other with 36 packed rows each, 214 and 182 with
// 48, 217 and 179 with 64, and with 68, a third tile, 310 and 188; with 64 on 1024 positions 64 in either.
constexpr int kFewRows = 64;
// Packed rows beyond one row for each sequence up to which the streaming kernel takes a whole call, since two
// kernels one after the other each have an end at which little runs.  32 heads on 8 of 128, streaming alone and both:
// 63 single rows and one chunk of 512 on 4096 positions (2044 to spare) 140 and 172 us, a prompt of 512 22 and 36;
// 64 x 17 rows on 4096 (4096 to spare) 304 and 188, a prompt of 2048 (8188) 192 and 90.  Shapes alone are known here: a
// sequence without rows counts as one with a row, so a table of more slots than the call uses leaves a prompt of up to
// that many rows more with the streaming kernel, and rows of nobody count as rows to spare.
constexpr int kSpareRows = 2048;

// How a call runs, from its shapes alone (lengths are device data).
struct DecodePlan {
  int dp, qt;       // padded head; tiles of 16 rows
  int64_t tiles;    // at most
  int workers;      // for each cache head
  bool split;       // whether a tile can be cut at all
  size_t bytes;     // of scratch for the cut tiles' sums
};

DecodePlan PlanDecode(int64_t rows, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head, int64_t positions, bool few) {
  DecodePlan d;
  const int64_t group = q_heads / kv_heads;
  d.dp = head <= 64 ? 64 : head <= 128 ? 128 : 256;
  const int64_t mean = batch > 0 ? (rows + batch - 1) / batch * group : 0;
  d.qt = mean <= 16 ? 1 : 2;
  d.tiles = rows * group / (16 * d.qt) + batch;
  const int64_t most = batch * (kFewRows / (16 * d.qt));
  if (few && d.tiles > most) d.tiles = most;
  const int64_t units = d.tiles * ((positions + kUnit - 1) / kUnit);
  const int64_t slots = 256 * decode_residents(d.dp);
  int64_t w = slots / kv_heads;  // no more than run at a time: each has an equal piece
  if (w > units) w = units;
  d.workers = w < 1 ? 1 : (int)w;
  // A second launch costs more than four units one after the other (two of a head above 128).  Eight heads of 128, cut and
  // whole: one sequence of 500 positions 10.6 and 9.8 us, of 760 11.3 and 11.5; eight 12.4 and 10.1, 13.0 and 14.3;
  // 64 of 500 19.3 and 17.2.  A head of 256: one of 250 13.2 and 10.8, of 500 13.0 and 13.7.
  d.split = positions > (d.dp == 256 ? 2 : 4) * kUnit && batch > 0;
  d.bytes = d.split ? (size_t)(d.workers * (sizeof(CutTile) + kv_heads * 2 * 16 * d.qt * (head + 2) * 4)) : 0;
  return d;
}

struct PromptPlan {
  bool used;
  int pieces;       // 0: no tile is cut
  int64_t slots;    // pieces of tiles, at most
  size_t bytes;
};

PromptPlan PlanPrompt(int64_t rows, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head, int64_t positions) {
  PromptPlan d{};
  const int64_t group = q_heads / kv_heads;
  d.used = batch > 0 && (rows - batch) * group > kSpareRows;
  if (!d.used) return d;
  d.slots = rows * group / kPromptRows + min(batch, rows * group / kFewRows);
  const int64_t pieces = kPieces / kv_heads;
  if (rows * group / kPromptRows < pieces && positions >= 2 * kLeastStages * kStage) {
    d.pieces = (int)pieces;
    if (d.slots < pieces) d.slots = d.slots * kMostSplits < pieces ? d.slots * kMostSplits : pieces;
    d.bytes = (size_t)pieces * (sizeof(CutTile) + kv_heads * kPromptRows * (head + 2) * 4);
  }
  return d;
}

template <bool F8, int DP>
void LaunchPrompt(const PromptView& v, hipStream_t stream) {
  const unsigned grid = (unsigned)(v.slots * v.a.c.heads);
  if (v.a.c.block_log2 < 2) kv_cache_attention_prompt_kernel<F8, DP, true><<<grid, 256, 0, stream>>>(v);
  else kv_cache_attention_prompt_kernel<F8, DP, false><<<grid, 256, 0, stream>>>(v);
}

template <bool F8>
void LaunchPrompt(int dp, const PromptView& v, hipStream_t stream) {
  if (dp == 64) LaunchPrompt<F8, 64>(v, stream);
  else if (dp == 128) LaunchPrompt<F8, 128>(v, stream);
  else LaunchPrompt<F8, 256>(v, stream);
}

template <bool F8, int DP, int QT>
void LaunchDecode(const DecodeView& v, dim3 grid, hipStream_t stream) {
  if (v.a.c.block_log2 < 2) kv_cache_attention_decode_kernel<F8, DP, QT, true><<<grid, 256, 0, stream>>>(v);
  else kv_cache_attention_decode_kernel<F8, DP, QT, false><<<grid, 256, 0, stream>>>(v);
}

template <bool F8>
void LaunchDecode(const DecodePlan& d, const DecodeView& v, dim3 grid, hipStream_t stream) {
  if (d.dp == 64) d.qt == 1 ? LaunchDecode<F8, 64, 1>(v, grid, stream) : LaunchDecode<F8, 64, 2>(v, grid, stream);
  else if (d.dp == 128) d.qt == 1 ? LaunchDecode<F8, 128, 1>(v, grid, stream) : LaunchDecode<F8, 128, 2>(v, grid, stream);
  else d.qt == 1 ? LaunchDecode<F8, 256, 1>(v, grid, stream) : LaunchDecode<F8, 256, 2>(v, grid, stream);
}

}  // namespace

size_t KvCacheAttentionWorkspaceBytes(int64_t rows, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_size,
                                      int64_t max_positions) {
  if (rows <= 0 || batch <= 0 || kv_heads <= 0 || q_heads < kv_heads || head_size <= 0 || max_positions <= 0) return 0;
  // the two kernels of a call run one after the other: their sums lie behind each other
  const PromptPlan p = PlanPrompt(rows, batch, q_heads, kv_heads, head_size, max_positions);
  return PlanDecode(rows, batch, q_heads, kv_heads, head_size, max_positions, p.used).bytes + p.bytes;
}

int LaunchKvCacheAttention(const XlaAmdKvCacheAttention& p, hipStream_t stream) {
  const int kBad = XLA_FFI_Error_Code_INVALID_ARGUMENT;
  AttentionView v{};
  if (int rc = MakeKvCacheView(p.cache, "kv_cache_attention", &v.c)) return rc;
  if (p.q_heads < 1 || p.q_heads > 65535 || p.q_heads % p.cache.kv_heads != 0)
    return Fail(kBad, "kv_cache_attention: q_heads must be a multiple of kv_heads, at most 65535");
  if (p.window < 0) return Fail(kBad, "kv_cache_attention: window must not be negative");
  if (p.window > 0 && !p.causal) return Fail(kBad, "kv_cache_attention: a window needs causal");
  if (!(p.softcap >= 0.0f) || !(p.softcap < INFINITY)) return Fail(kBad, "kv_cache_attention: softcap must be a number that is not negative");
  if (!(p.softmax_scale > -INFINITY && p.softmax_scale < INFINITY))
    return Fail(kBad, "kv_cache_attention: softmax_scale must be a number");
  // (a grid holds fewer than 2^32 threads: 256 for every 128 packed rows, and for every sequence of 64 and more)
  if (p.cache.rows * p.q_heads > 1 << 29) return Fail(kBad, "kv_cache_attention: at most 2^29 rows times heads");
  if (v.c.rows > 0 && (!p.q || !p.out)) return Fail(kBad, "kv_cache_attention: null q or out");
  if ((((uintptr_t)p.q | (uintptr_t)p.out | (uintptr_t)p.workspace) & 15) != 0 || ((uintptr_t)p.lse & 3) != 0)
    return Fail(kBad, "kv_cache_attention: q, out and scratch must be aligned to 16 bytes, lse to 4");
  if (v.c.rows == 0) return 0;
  v.q = (const uint16_t*)p.q;
  v.out = (uint16_t*)p.out;
  v.lse = p.lse;
  v.q_heads = (int)p.q_heads;
  v.group = (int)(p.q_heads / p.cache.kv_heads);
  v.scale = p.softmax_scale;
  if (p.softcap > 0.0f) {
    // between the smallest and the largest normal number, so that both are numbers: a cap below 2^-126 leaves no score that
    // differs from 0 in f32's weights
    v.cap = (float)(p.softcap * 1.44269504088896341);
    v.cap = v.cap < 0x1p-126f ? 0x1p-126f : v.cap < 0x1.fffffep127f ? v.cap : 0x1.fffffep127f;
    v.per_cap = 1.0f / v.cap;
  }
  v.causal = p.causal;
  const int64_t positions = p.cache.table_width * p.cache.page_size;
  v.window = p.window >= positions ? 0 : (int)p.window;  // every position that a causal row sees is nearer
  const PromptPlan pr = PlanPrompt(v.c.rows, v.c.batch, p.q_heads, p.cache.kv_heads, p.cache.head_size, positions);
  const int64_t reach = v.window > 0 ? min(positions, (int64_t)v.window + kUnit) : positions;  // of a row, in whole units
  const DecodePlan d = PlanDecode(v.c.rows, v.c.batch, p.q_heads, p.cache.kv_heads, p.cache.head_size, reach, pr.used);
  DecodeView dv{};
  dv.a = v;
  dv.workers = d.workers;
  dv.rows_to = pr.used ? kFewRows : INT32_MAX;
  const bool scratch = p.workspace && p.workspace_bytes >= d.bytes + pr.bytes;
  if (d.split && scratch) {
    dv.cuts = (CutTile*)p.workspace;
    dv.partial = (float*)(dv.cuts + d.workers);
  }
  const dim3 grid((unsigned)(d.workers + (v.c.rows + 63) / 64), (unsigned)v.c.heads);
  char name[64];
  const bool f8 = p.cache.cache_dtype == XLA_FFI_DataType_F8E4M3FN;
  snprintf(name, sizeof(name), "kv_cache_attention_decode_%s_d%d_m%d%s", f8 ? "f8" : "s8", d.dp, 16 * d.qt, dv.partial ? "_split" : "");
  SetLastKernel(name);
  if (f8) LaunchDecode<true>(d, dv, grid, stream);
  else LaunchDecode<false>(d, dv, grid, stream);
  JoinView jv{};
  jv.a = v;
  const int lanes = d.dp / 4, join_rows = 256 / lanes;
  unsigned joins = 0;
  if (dv.partial) {
    const int64_t size = (int64_t)16 * d.qt * (v.c.head + 2);
    // a worker's second piece is the one that begins its tile, the next workers go on in their first
    jv.parts[0] = JoinPart{dv.cuts, dv.partial + size, 2 * d.workers * size, 2 * size, 2 * size, size, 16 * d.qt};
    joins = jv.blocks = (unsigned)(d.workers * (16 * d.qt) / join_rows);
  }
  if (pr.used) {
    PromptView pv{};
    pv.a = v;
    pv.slots = (int)pr.slots;
    pv.pieces = pr.pieces;
    pv.rows_from = kFewRows;
    if (pr.pieces > 0 && scratch) {
      pv.cuts = (CutTile*)((char*)p.workspace + d.bytes);
      pv.partial = (float*)(pv.cuts + pr.pieces);
      const int64_t size = (int64_t)kPromptRows * (v.c.head + 2);
      jv.parts[1] = JoinPart{pv.cuts, pv.partial, size, v.c.heads * size, v.c.heads * size, 0, kPromptRows};
      joins += (unsigned)(min(pr.slots, (int64_t)pr.pieces) * kPromptRows / join_rows);
    }
    snprintf(name, sizeof(name), "kv_cache_attention_prompt_%s_d%d_m%d%s", f8 ? "f8" : "s8", d.dp, kPromptRows,
             pv.partial ? "_split" : "");
    SetLastKernel(name);
    if (f8) LaunchPrompt<true>(d.dp, pv, stream);
    else LaunchPrompt<false>(d.dp, pv, stream);
  }
  if (joins > 0) {
    const dim3 grid((unsigned)joins, (unsigned)v.c.heads);
    if (d.dp == 64) kv_cache_attention_join_kernel<16><<<grid, 256, 0, stream>>>(jv);
    else if (d.dp == 128) kv_cache_attention_join_kernel<32><<<grid, 256, 0, stream>>>(jv);
    else kv_cache_attention_join_kernel<64><<<grid, 256, 0, stream>>>(jv);
  }
  return CheckLaunch("kv_cache_attention");
}

}  // namespace xla_amd
