// Attention over a serving cache: softmax(scale q K^T) V of one entry's rows (drafted tokens x heads
// of a group) against the positions that its view shows (cache_ops.h).
//
// With s_t = scale q . k_t over the visible positions t, one pass keeps m = max s_t,
// l = sum exp(s_t - m) and o = sum exp(s_t - m) v_t in float32; a later maximum M rescales l and o
// by exp(m - M), and parts of the cache join the same way. out = o / l; a row that sees nothing has
// l = 0 and an output of zero. Positions that a row does not see never enter a sum, whatever they
// hold.
#include <hip/hip_fp16.h>

#include "cache_ops.h"
#include "device_utils.h"
#include "runtime.h"

namespace ct2x {

namespace {

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float(float x) { return x; }
template <>
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float(uint16_t x) { return __uint_as_float(static_cast<uint32_t>(x) << 16); }

constexpr int kThreads = 256;

// One workgroup per (entry, row): the waves walk tiles of 64 positions, lane = position for the
// scores, lane = channel for the outputs, and join in LDS.
template <typename T>
__global__ __launch_bounds__(kThreads) void cache_attention_kernel(CacheAttnParams p) {
  __shared__ float q_s[256];
  __shared__ float m_s[4], l_s[4], o_s[4][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;  // ((b * tokens) + i) * heads + h
  const int64_t h = row % p.heads, i = row / p.heads % p.tokens, b = row / p.heads / p.tokens;
  const int64_t hkv = h / (p.heads / p.heads_kv);
  const int dhead = static_cast<int>(p.dhead);
  const int64_t room = p.t_max - (p.view == CacheView::kTree ? p.tokens : 0);
  int64_t len = p.lengths ? p.lengths[b] : p.length;
  len = len < 0 ? 0 : (len > room ? room : len);
  int64_t end = p.view == CacheView::kTree ? len + p.tokens : len;
  if (p.view == CacheView::kBlocks) end = p.top * p.block;
  for (int d = threadIdx.x; d < dhead; d += kThreads) q_s[d] = p.q[row * dhead + d];
  __syncthreads();
  const int64_t words = (p.tokens + 63) / 64;
  const uint64_t* mask = p.mask ? p.mask + (b * p.tokens + i) * words : nullptr;
  const int32_t* selected = p.selected ? p.selected + (b * p.heads_kv + hkv) * p.top : nullptr;
  const T* k = static_cast<const T*>(p.k) + (b * p.heads_kv + hkv) * p.t_max * dhead;
  const T* v = static_cast<const T*>(p.v) + (b * p.heads_kv + hkv) * p.t_max * dhead;
  float* raw = p.weights ? static_cast<float*>(p.scratch) + (b * p.heads + h) * p.t_max : nullptr;

  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int64_t t0 = wave * 64; t0 < end; t0 += kThreads) {
    int64_t t = t0 + lane;
    bool visible = t < end;
    if (p.view == CacheView::kBlocks) {
      const int32_t j = visible ? selected[t / p.block] : -1;
      t = j * p.block + t % p.block;
      visible = j >= 0 && t < len;
    } else if (p.view == CacheView::kTree && visible && t >= len) {
      const int64_t j = t - len;
      visible = mask ? (mask[j >> 6] >> (j & 63)) & 1 : j <= i;
    }
    float s = -INFINITY;
    if (visible) {
      float dot = 0.f;
      for (int d = 0; d < dhead; ++d) dot = fmaf(q_s[d], to_float(k[t * dhead + d]), dot);
      s = dot * p.scale;
      if (raw) raw[t] = s;
    }
    const float top = fmaxf(m, wave_max(s));
    const float base = top == -INFINITY ? 0.f : top;
    const float e = visible ? expf(s - base) : 0.f, keep = m == -INFINITY ? 0.f : expf(m - base);
    l = l * keep + wave_sum(e);
    for (int c = 0; c < 4; ++c) o[c] *= keep;
    m = top;
    for (int j = 0; j < 64; ++j) {
      if (!__shfl(visible, j)) continue;
      const float e_j = __shfl(e, j);
      const int64_t t_j = __shfl(t, j);
      for (int c = 0; c < 4; ++c)
        if (c * 64 + lane < dhead) o[c] = fmaf(e_j, to_float(v[t_j * dhead + c * 64 + lane]), o[c]);
    }
  }
  if (lane == 0) {
    m_s[wave] = m;
    l_s[wave] = l;
  }
  for (int c = 0; c < 4; ++c) o_s[wave][c * 64 + lane] = o[c];
  __syncthreads();
  float top = -INFINITY, total = 0.f;
  for (int w = 0; w < 4; ++w) top = fmaxf(top, m_s[w]);
  const float base = top == -INFINITY ? 0.f : top;
  float keep[4];
  for (int w = 0; w < 4; ++w) {
    keep[w] = m_s[w] == -INFINITY ? 0.f : expf(m_s[w] - base);
    total += l_s[w] * keep[w];
  }
  const float inverse = total == 0.f ? 0.f : 1.f / total;
  for (int d = threadIdx.x; d < dhead; d += kThreads) {
    float sum = 0.f;
    for (int w = 0; w < 4; ++w) sum += o_s[w][d] * keep[w];
    p.out[row * dhead + d] = total == 0.f ? 0.f : sum * inverse;
  }
  if (raw) {  // the row's statistics wait behind the scores of all rows
    float* stats = static_cast<float*>(p.scratch) + p.batch * p.heads * p.t_max + (b * p.heads + h) * 2;
    if (threadIdx.x == 0) {
      stats[0] = base;
      stats[1] = inverse;
    }
  }
}

// weights[b, hkv, t] += sum over the group's heads of exp(s_t - m) / l
__global__ __launch_bounds__(kThreads) void cache_weights_kernel(CacheAttnParams p) {
  const int64_t tiles = (p.t_max + kThreads - 1) / kThreads, unit = blockIdx.x / tiles;
  const int64_t b = unit / p.heads_kv, hkv = unit % p.heads_kv;
  const int64_t group = p.heads / p.heads_kv;
  int64_t len = p.lengths ? p.lengths[b] : p.length;
  len = len < 0 ? 0 : (len > p.t_max ? p.t_max : len);
  const int64_t t = blockIdx.x % tiles * kThreads + threadIdx.x;
  if (t >= len) return;
  const float* raw = static_cast<const float*>(p.scratch);
  const float* stats = raw + p.batch * p.heads * p.t_max;
  float sum = 0.f;
  for (int64_t h = b * p.heads + hkv * group; h < b * p.heads + (hkv + 1) * group; ++h)
    sum += expf(raw[h * p.t_max + t] - stats[2 * h]) * stats[2 * h + 1];
  p.weights[(b * p.heads_kv + hkv) * p.t_max + t] += sum;
}

template <typename T>
void launch_typed(const CacheAttnParams& p, hipStream_t stream) {
  hipLaunchKernelGGL((cache_attention_kernel<T>), dim3(static_cast<unsigned>(p.batch * p.tokens * p.heads)),
                     dim3(kThreads), 0, stream, p);
}

}  // namespace

int64_t cache_attention_scratch_bytes(const CacheAttnParams& p) {
  return p.view == CacheView::kDense ? p.batch * p.heads * (p.t_max + 2) * 4 : 0;
}

void launch_cache_attention(const CacheAttnParams& p, hipStream_t stream) {
  if (p.kv_dtype == 0) launch_typed<float>(p, stream);
  else if (p.kv_dtype == 4) launch_typed<__half>(p, stream);
  else launch_typed<uint16_t>(p, stream);
  if (p.weights)
    hipLaunchKernelGGL(cache_weights_kernel,
                       dim3(static_cast<unsigned>((p.t_max + kThreads - 1) / kThreads * p.batch * p.heads_kv)),
                       dim3(kThreads), 0, stream, p);
}

}  // namespace ct2x
