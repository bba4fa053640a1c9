// Softmax attention over an 8-bit paged key/value cache.
//
//   x_j = softmax_scale * ks_j * sum_d q_d kc_jd, with softcap: softcap * tanh(x_j / softcap)
//   out_d = sum_j exp(x_j - m) vs_j vc_jd / sum_j exp(x_j - m),  lse = m + log sum_j exp(x_j - m)
//
// over the positions j that the row sees, with the running maximum m and sum of a softmax.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_cache.h"

namespace xla_amd {
namespace {

struct AttentionView {
  KvCacheView c;
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  int q_heads, group;  // group: heads of q for each head of the cache
  float scale, softcap;
  int causal, window;
};

template <bool F8>
__device__ __forceinline__ float code_value(uint32_t c) {
  if constexpr (F8) return f8e4m3fn_to_f32(c);
  return (float)(int8_t)c;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = __builtin_fmaxf(v, __shfl_xor(v, off));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// One wave for a row and head: 64 positions at a time, a lane each for the scores, then the lanes go along
// the head for the values.
template <bool F8>
__global__ __launch_bounds__(64) void kv_cache_attention_row_kernel(AttentionView v) {
  const KvCacheView& c = v.c;
  const int lane = threadIdx.x, row = blockIdx.x, qh = blockIdx.y, head = qh / v.group;
  __shared__ float q[256], weight[64];
  __shared__ int page_of[64];
  const int64_t at = ((int64_t)row * v.q_heads + qh) * c.head;
  for (int d = lane; d < c.head; d += 64) q[d] = bf16_to_f32(v.q[at + d]);
  int b = -1;
  for (int b0 = 0; b0 < c.batch && b < 0; b0 += 64) {
    bool mine = false;
    if (b0 + lane < c.batch) {
      const KvSequence s = kv_sequence(c, b0 + lane);
      mine = row >= s.row0 && row < s.row0 + s.n;
    }
    const unsigned long long hit = __ballot(mine);
    if (hit != 0ull) b = b0 + __builtin_ctzll(hit);
  }
  float m = -INFINITY, sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (b >= 0) {
    const KvSequence s = kv_sequence(c, b);
    const int pos = s.len - s.n + (row - s.row0);
    const int end = v.causal ? min(s.len, pos + 1) : s.len;
    const int begin = v.window > 0 ? max(0, pos - v.window + 1) : 0;
    const int in_page = (1 << c.page_log2) - 1;
    for (int j0 = begin; j0 < end; j0 += 64) {
      const int j = j0 + lane;
      const int page = j < end ? kv_page(c, b, j) : -1;
      float x = -INFINITY, vs = 0.0f;
      if (page >= 0) {
        const uint8_t* k = c.codes[0] + kv_row(c, page, head, j & in_page);
        float dot = 0.0f;
        for (int d = 0; d < c.head; ++d) dot = __builtin_fmaf(q[d], code_value<F8>(k[d]), dot);
        x = dot * (c.scales[0][kv_scale(c, page, head, j & in_page)] * v.scale);
        if (v.softcap > 0.0f) x = v.softcap * tanhf(x / v.softcap);
        vs = c.scales[1][kv_scale(c, page, head, j & in_page)];
      }
      const float top = __builtin_fmaxf(m, wave_max(x));
      const float rescale = m == -INFINITY ? 0.0f : expf(m - top);
      const float p = page >= 0 ? expf(x - top) : 0.0f;
      sum = sum * rescale + wave_sum(p);
      m = top;
      __syncthreads();
      weight[lane] = page >= 0 ? p * vs : 0.0f;
      page_of[lane] = page;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] *= rescale;
      for (int t = 0; t < min(64, end - j0); ++t) {
        if (page_of[t] < 0) continue;
        const uint8_t* w = c.codes[1] + kv_row(c, page_of[t], head, (j0 + t) & in_page);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (lane + 64 * i < c.head) acc[i] = __builtin_fmaf(weight[t], code_value<F8>(w[lane + 64 * i]), acc[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < c.head) v.out[at + lane + 64 * i] = f32_to_bf16(sum == 0.0f ? 0.0f : acc[i] / sum);
  if (v.lse && lane == 0) v.lse[(int64_t)row * v.q_heads + qh] = sum == 0.0f ? -INFINITY : m + logf(sum);
}

}  // namespace

size_t KvCacheAttentionWorkspaceBytes(int64_t rows, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_size,
                                      int64_t max_positions) {
  return 0;
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
  v.softcap = p.softcap;
  v.causal = p.causal;
  v.window = p.window > INT32_MAX ? 0 : (int)p.window;  // no position lies further back
  const dim3 grid((unsigned)v.c.rows, (unsigned)v.q_heads);
  SetLastKernel("kv_cache_attention_row");
  if (p.cache.cache_dtype == XLA_FFI_DataType_F8E4M3FN) kv_cache_attention_row_kernel<true><<<grid, 64, 0, stream>>>(v);
  else kv_cache_attention_row_kernel<false><<<grid, 64, 0, stream>>>(v);
  return CheckLaunch("kv_cache_attention");
}

}  // namespace xla_amd
