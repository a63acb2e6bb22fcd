// Upkeep of a serving cache (cache_ops.h): which positions an eviction keeps and their move, the
// bounds of blocks of keys, and the blocks that a query selects by them.
//
// Choices are whole numbers, so their order is exact: scores are compared as the unsigned integers
// that sort like them (NaN above every number, -0 equal to +0), the lower position wins a tie. The
// threshold of the best n is found by radix selection from the top byte down - a histogram of 256
// counts per byte -, then one ordered pass takes everything above it and the first of those equal to it.
#include <hip/hip_fp16.h>

#include "cache_ops.h"
#include "device_utils.h"
#include "runtime.h"

namespace ct2x {

namespace {

constexpr int kThreads = 256;
constexpr int kSelectThreads = 1024;

__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xfffffffeu;
  if (x == 0.f) x = 0.f;  // -0
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint64_t order_key(double x) {
  if (x != x) return 0xfffffffffffffffeull;
  if (x == 0.) x = 0.;
  const uint64_t u = __double_as_longlong(x);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

__device__ __forceinline__ int64_t clamped_length(const int32_t* lengths, int64_t length, int64_t b, int64_t t_max) {
  const int64_t n = lengths ? lengths[b] : length;
  return n < 0 ? 0 : (n > t_max ? t_max : n);
}

// The `want` (>= 1, <= n) best of key(0 .. n): *threshold = the smallest key taken, returns how many
// of the keys equal to it are taken. All threads of the workgroup call.
template <typename K, typename F>
__device__ int64_t select_threshold(F key, int64_t n, int64_t want, K* threshold) {
  __shared__ uint32_t histogram[256];
  __shared__ uint32_t digit_s;
  __shared__ uint32_t above_s;
  K prefix = 0, known = 0;
  for (int shift = sizeof(K) * 8 - 8; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += blockDim.x) histogram[i] = 0;
    __syncthreads();
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
      const K x = key(i);
      if ((x & known) == prefix) atomicAdd(&histogram[(x >> shift) & 255], 1u);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int64_t above = 0;
      int digit = 255;
      while (above + histogram[digit] < want) above += histogram[digit--];
      digit_s = digit;
      above_s = static_cast<uint32_t>(above);
    }
    __syncthreads();
    want -= above_s;
    prefix |= static_cast<K>(digit_s) << shift;
    known |= static_cast<K>(255) << shift;
  }
  *threshold = prefix;
  return want;
}

// emit(slot, i) for the i of 0 .. n with key(i) > threshold or among the first `ties` equal to it,
// slots 0, 1, .. in order of i. Returns how many. All threads of the workgroup call.
template <typename K, typename F, typename G>
__device__ int64_t emit_selected(F key, int64_t n, K threshold, int64_t ties, G emit) {
  __shared__ uint32_t taken_s[kSelectThreads / 64], equal_s[kSelectThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  int64_t slot = 0, equal = 0;
  for (int64_t i0 = 0; i0 < n; i0 += blockDim.x) {
    const int64_t i = i0 + threadIdx.x;
    const K x = i < n ? key(i) : 0;
    const bool same = i < n && x == threshold;
    const uint64_t same_bits = __ballot(same), below = (1ull << lane) - 1;
    if (lane == 0) equal_s[wave] = __popcll(same_bits);
    __syncthreads();
    int64_t rank = equal, all = equal;
    for (int w = 0; w < waves; ++w) {
      if (w < wave) rank += equal_s[w];
      all += equal_s[w];
    }
    rank += __popcll(same_bits & below);
    const bool take = i < n && (x > threshold || (same && rank < ties));
    const uint64_t take_bits = __ballot(take);
    if (lane == 0) taken_s[wave] = __popcll(take_bits);
    __syncthreads();
    int64_t at = slot, next = slot;
    for (int w = 0; w < waves; ++w) {
      if (w < wave) at += taken_s[w];
      next += taken_s[w];
    }
    if (take) emit(at + __popcll(take_bits & below), i);
    slot = next;
    equal = all;
    __syncthreads();
  }
  return slot;
}

// positions[b, hkv, :]: what stays, ascending, -1 behind the last
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(CacheEvictParams p) {
  const int64_t row = blockIdx.x, b = row / p.heads_kv;
  const int64_t n = clamped_length(p.lengths, p.length, b, p.t_max);
  const float* w = p.weights + row * p.t_max;
  int32_t* positions = p.positions + row * p.budget;
  const int64_t kept = n < p.budget ? n : p.budget;
  int64_t slot = 0, old = 0;
  if (n > p.budget && p.budget > p.recent) {
    old = n - p.recent;
    auto key = [&](int64_t i) { return order_key(w[i]); };
    uint32_t threshold;
    const int64_t ties = select_threshold<uint32_t>(key, old, p.budget - p.recent, &threshold);
    slot = emit_selected<uint32_t>(key, old, threshold, ties,
                                   [&](int64_t at, int64_t i) { positions[at] = static_cast<int32_t>(i); });
  }
  for (int64_t i = slot + threadIdx.x; i < p.budget; i += blockDim.x)
    positions[i] = i < kept ? static_cast<int32_t>(n - kept + i) : -1;
}

// One workgroup moves 256 bytes of every kept row of a (entry, head)'s keys or values, in steps
// that are read before they are written: a row moves to the front only, so that a step never
// overwrites what a later one reads and the output may be the input.
__global__ __launch_bounds__(kThreads) void evict_move_kernel(CacheEvictParams p, int row_bytes, int slices) {
  constexpr int kRows = kThreads / 16;
  const int64_t row = blockIdx.x / (2 * slices);
  const int slice = blockIdx.x % slices, value = blockIdx.x / slices % 2;
  const int64_t b = row / p.heads_kv;
  const int32_t* positions = p.positions + row * p.budget;
  const char* from = static_cast<const char*>(value ? p.v : p.k) + row * p.t_max * row_bytes;
  char* to = static_cast<char*>(value ? p.v_out : p.k_out) + row * p.t_max_out * row_bytes;
  const float* w = p.weights + row * p.t_max;
  float* w_out = p.weights_out + row * p.t_max_out;
  const int at = slice * 256 + (threadIdx.x & 15) * 16;
  for (int64_t j0 = 0; j0 < p.budget; j0 += kRows) {
    const int64_t j = j0 + threadIdx.x / 16;
    const int32_t t = j < p.budget ? positions[j] : -1;
    const bool moves = t >= 0 && at < row_bytes;
    const bool first = t >= 0 && (threadIdx.x & 15) == 0 && blockIdx.x % (2 * slices) == 0;
    int4 data = {0, 0, 0, 0};
    float weight = 0.f;
    if (moves) data = *reinterpret_cast<const int4*>(from + t * static_cast<int64_t>(row_bytes) + at);
    if (first) weight = w[t];
    __syncthreads();
    if (moves) *reinterpret_cast<int4*>(to + j * row_bytes + at) = data;
    if (first) w_out[j] = weight;
  }
  if (blockIdx.x % (2 * slices * p.heads_kv) == 0 && threadIdx.x == 0) {
    const int64_t n = clamped_length(p.lengths, p.length, b, p.t_max);
    p.lengths_out[b] = static_cast<int32_t>(n < p.budget ? n : p.budget);
  }
}

template <typename T>
__device__ __forceinline__ float load_float(T x);
template <>
__device__ __forceinline__ float load_float(float x) { return x; }
template <>
__device__ __forceinline__ float load_float(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float load_float(uint16_t x) { return __uint_as_float(static_cast<uint32_t>(x) << 16); }

// One thread per channel of a (entry, head, block). NaN keys make NaN bounds.
template <typename T>
__global__ __launch_bounds__(kThreads) void block_bounds_kernel(CacheBoundsParams p, int64_t blocks) {
  const int64_t j = blockIdx.x % blocks, row = blockIdx.x / blocks, b = row / p.heads_kv;
  const int64_t n = clamped_length(p.lengths, p.length, b, p.t_max);
  int64_t first = p.first ? p.first[b] : 0;
  first = first < 0 ? 0 : first;
  if (j < first / p.block || j * p.block >= n) return;
  const int64_t end = (j + 1) * p.block < n ? (j + 1) * p.block : n;
  const T* k = static_cast<const T*>(p.k) + row * p.t_max * p.dhead;
  T* out = static_cast<T*>(p.bounds) + (row * blocks + j) * 2 * p.dhead;
  for (int64_t d = threadIdx.x; d < p.dhead; d += kThreads) {
    T low = k[j * p.block * p.dhead + d], high = low;
    for (int64_t t = j * p.block + 1; t < end; ++t) {
      const T x = k[t * p.dhead + d];
      const float f = load_float(x);
      if (!(f >= load_float(low)) && load_float(low) == load_float(low)) low = x;
      if (!(f <= load_float(high)) && load_float(high) == load_float(high)) high = x;
    }
    out[d] = low;
    out[p.dhead + d] = high;
  }
}

// scores[b, hkv, j] = max over the group's heads of sum_d max(q_d min_d, q_d max_d), float64: a
// choice between blocks must not depend on how the sum was ordered.
template <typename T>
__global__ __launch_bounds__(kThreads) void block_scores_kernel(CacheSelectParams p, int64_t blocks) {
  const int64_t tiles = (blocks + kThreads - 1) / kThreads, row = blockIdx.x / tiles;
  const int64_t b = row / p.heads_kv, hkv = row % p.heads_kv, group = p.heads / p.heads_kv;
  const int64_t n = clamped_length(p.lengths, p.length, b, p.t_max);
  const int64_t j = blockIdx.x % tiles * static_cast<int64_t>(kThreads) + threadIdx.x;
  if (j * p.block >= n) return;
  const T* low = static_cast<const T*>(p.bounds) + (row * blocks + j) * 2 * p.dhead;
  double best = 0.;
  for (int64_t g = 0; g < group; ++g) {
    const float* q = p.q + (b * p.heads + hkv * group + g) * p.dhead;
    double sum = 0.;
    for (int64_t d = 0; d < p.dhead; ++d) {
      const double x = q[d], a = x * load_float(low[d]), c = x * load_float(low[p.dhead + d]);
      sum += a != a || a > c ? a : c;
    }
    if (g == 0 || sum > best || sum != sum) best = sum;
    if (best != best) break;
  }
  p.scores[row * blocks + j] = best;
}

__global__ __launch_bounds__(kSelectThreads) void block_select_kernel(CacheSelectParams p, int64_t blocks) {
  const int64_t row = blockIdx.x, b = row / p.heads_kv;
  const int64_t n = clamped_length(p.lengths, p.length, b, p.t_max);
  const int64_t count = (n + p.block - 1) / p.block;
  const double* scores = p.scores + row * blocks;
  int32_t* selected = p.selected + row * p.top;
  int64_t taken = count;
  if (count > p.top) {
    auto key = [&](int64_t j) {
      return j < p.sink || j >= count - p.local ? ~0ull : order_key(scores[j]);
    };
    uint64_t threshold;
    const int64_t ties = select_threshold<uint64_t>(key, count, p.top, &threshold);
    emit_selected<uint64_t>(key, count, threshold, ties,
                            [&](int64_t at, int64_t j) { selected[at] = static_cast<int32_t>(j); });
    taken = p.top;
  } else {
    for (int64_t j = threadIdx.x; j < count; j += blockDim.x) selected[j] = static_cast<int32_t>(j);
  }
  for (int64_t j = taken + threadIdx.x; j < p.top; j += blockDim.x) selected[j] = -1;
}

template <typename T>
void bounds_typed(const CacheBoundsParams& p, int64_t blocks, hipStream_t stream) {
  hipLaunchKernelGGL((block_bounds_kernel<T>), dim3(static_cast<unsigned>(p.batch * p.heads_kv * blocks)),
                     dim3(kThreads), 0, stream, p, blocks);
}

template <typename T>
void scores_typed(const CacheSelectParams& p, int64_t blocks, hipStream_t stream) {
  hipLaunchKernelGGL((block_scores_kernel<T>),
                     dim3(static_cast<unsigned>((blocks + kThreads - 1) / kThreads * p.batch * p.heads_kv)),
                     dim3(kThreads), 0, stream, p, blocks);
}

}  // namespace

void launch_cache_evict(const CacheEvictParams& p, hipStream_t stream) {
  const int row_bytes = static_cast<int>(p.dhead) * (p.kv_dtype == 0 ? 4 : 2);
  const int slices = (row_bytes + 255) / 256;
  const unsigned rows = static_cast<unsigned>(p.batch * p.heads_kv);
  hipLaunchKernelGGL(evict_select_kernel, dim3(rows), dim3(kSelectThreads), 0, stream, p);
  hipLaunchKernelGGL(evict_move_kernel, dim3(rows * 2 * slices), dim3(kThreads), 0, stream, p, row_bytes, slices);
}

void launch_cache_block_bounds(const CacheBoundsParams& p, hipStream_t stream) {
  const int64_t blocks = (p.t_max + p.block - 1) / p.block;
  if (p.kv_dtype == 0) bounds_typed<float>(p, blocks, stream);
  else if (p.kv_dtype == 4) bounds_typed<__half>(p, blocks, stream);
  else bounds_typed<uint16_t>(p, blocks, stream);
}

void launch_cache_select(const CacheSelectParams& p, hipStream_t stream) {
  const int64_t blocks = (p.t_max + p.block - 1) / p.block;
  if (p.kv_dtype == 0) scores_typed<float>(p, blocks, stream);
  else if (p.kv_dtype == 4) scores_typed<__half>(p, blocks, stream);
  else scores_typed<uint16_t>(p, blocks, stream);
  hipLaunchKernelGGL(block_select_kernel, dim3(static_cast<unsigned>(p.batch * p.heads_kv)), dim3(kSelectThreads),
                     0, stream, p, blocks);
}

}  // namespace ct2x
