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
// A launch has less than 2^32 threads: more rows - (entry, head of the cache) pairs - take several launches.
constexpr int64_t kMostGroups = int64_t{1} << 21;

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

__device__ __forceinline__ uint32_t wave_and(uint32_t x) {
  auto meet = [&](auto ctrl, auto rows) {
    x &= static_cast<uint32_t>(__builtin_amdgcn_update_dpp(-1, static_cast<int>(x), decltype(ctrl)::value,
                                                           decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  meet(integral_constant<int, 0x111>(), integral_constant<int, 0xf>());
  meet(integral_constant<int, 0x112>(), integral_constant<int, 0xf>());
  meet(integral_constant<int, 0x114>(), integral_constant<int, 0xf>());
  meet(integral_constant<int, 0x118>(), integral_constant<int, 0xf>());
  meet(integral_constant<int, 0x142>(), integral_constant<int, 0xa>());
  meet(integral_constant<int, 0x143>(), integral_constant<int, 0xc>());
  return __builtin_amdgcn_readlane(x, 63);
}
__device__ __forceinline__ uint64_t wave_and(uint64_t x) {
  return static_cast<uint64_t>(wave_and(static_cast<uint32_t>(x >> 32))) << 32 | wave_and(static_cast<uint32_t>(x));
}

// Keys 0 .. n - 1 spread over a workgroup: every wave has a stretch of them, its lanes the positions
// in turn. The first kKeep of a lane stay in registers, what a longer row has beyond is read again by
// every pass.
template <typename K, typename F>
struct Keys {
  static constexpr int kKeep = 16;
  F key;
  int lane, from, to;
  K kept[kKeep];
  __device__ __forceinline__ Keys(F key, int n) : key(key) {
    const int wave = threadIdx.x >> 6, waves = kSelectThreads / 64;
    const int stretch = ((n + waves - 1) / waves + 63) / 64 * 64;
    lane = threadIdx.x & 63;
    from = wave * stretch;
    to = from + stretch < n ? from + stretch : n;
    // all at once for a long stretch (requests without a branch between them), what there is of a short one
    const bool few = stretch <= 4 * 64;
#pragma unroll
    for (int u = 0; u < kKeep; ++u) kept[u] = 0;
    if (few) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (from + u * 64 < to) kept[u] = key(from + u * 64 + lane < to ? from + u * 64 + lane : 0);
    } else {
#pragma unroll
      for (int u = 0; u < kKeep; ++u) kept[u] = key(from + u * 64 + lane < to ? from + u * 64 + lane : 0);
    }
  }
  // visit(i, key(i), whether there is an i), whole waves at a time
  template <typename G>
  __device__ __forceinline__ void each(G visit) const {
#pragma unroll
    for (int u = 0; u < kKeep; ++u) {
      if (from + u * 64 >= to) return;
      const int i = from + u * 64 + lane;
      visit(i, kept[u], i < to);
    }
    for (int i0 = from + kKeep * 64; i0 < to; i0 += 64 * 4) {
      K x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * 64 + lane;
        x[u] = key(i < to ? i : 0);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * 64 + lane;
        visit(i, x[u], i < to);
      }
    }
  }
};

// The `want` (1 .. n) best: *threshold = the smallest key taken, returns how many of the keys equal to
// it are taken. All threads of the workgroup call. Bits that all keys share are skipped (a first pass
// finds them: scores of one layer have their exponent in common, and every key would meet in one bin),
// and the search ends with the byte whose bin is taken whole.
template <typename K, typename F>
__device__ int select_threshold(const Keys<K, F>& keys, int want, K* threshold) {
  constexpr int kWaves = kSelectThreads / 64, kBytes = sizeof(K);
  __shared__ uint32_t histograms[kBytes][256];  // of every byte that a search may come to
  __shared__ K both_s[kWaves], none_s[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < kBytes * 256; i += kSelectThreads) histograms[i / 256][i % 256] = 0;
  K both = ~static_cast<K>(0), none = both;
  keys.each([&](int, K x, bool there) {
    both &= there ? x : ~static_cast<K>(0);
    none &= there ? ~x : ~static_cast<K>(0);
  });
  both = wave_and(both);
  none = wave_and(none);
  if (lane == 0) {
    both_s[wave] = both;
    none_s[wave] = none;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    both &= both_s[w];
    none &= none_s[w];
  }
  const K differ = ~(both | none);
  if (differ == 0) {
    *threshold = both;
    return want;
  }
  int upto = 64 - __clzll(static_cast<unsigned long long>(differ));  // bits below `upto` are searched
  K known = upto >= static_cast<int>(sizeof(K)) * 8 ? 0 : ~static_cast<K>(0) << upto;
  K prefix = both & known;
  for (int pass = 0; upto > 0; ++pass) {
    const int bits = upto < 8 ? upto : 8, shift = upto - bits;
    uint32_t* histogram = histograms[pass];
    keys.each([&](int, K x, bool there) {
      if (there && (x & known) == prefix)
        atomicAdd(&histogram[static_cast<uint32_t>(x >> shift) & ((1u << bits) - 1)], 1u);
    });
    __syncthreads();
    // every wave finds the bin by itself, lane 0 with the four highest
    uint32_t bin[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += bin[i] = histogram[255 - 4 * lane - i];
    const uint32_t upto_lane = wave_scan(sum);
    uint32_t above = upto_lane - sum, taken = bin[0];
    int digit = 255 - 4 * lane;
#pragma unroll
    for (int i = 1; i < 4; ++i)
      if (above + taken < static_cast<uint32_t>(want)) {
        above += taken;
        taken = bin[i];
        digit = 255 - 4 * lane - i;
      }
    const int at = __builtin_ctzll(__ballot(upto_lane >= static_cast<uint32_t>(want)));
    want -= __builtin_amdgcn_readlane(above, at);
    prefix |= static_cast<K>(__builtin_amdgcn_readlane(digit, at)) << shift;
    known |= static_cast<K>((1u << bits) - 1) << shift;
    upto = shift;
    // Everything with this prefix is taken: nothing below it is, whatever its lower bits. (As a
    // threshold the prefix itself: it may be no key, then none is equal to it and all are above.)
    if (__builtin_amdgcn_readlane(taken, at) == want) break;
  }
  *threshold = prefix;
  return want;
}

// emit(slot, i) for the i with key(i) > threshold or among the first `ties` equal to it, slots 0, 1, ..
// in order of i. Returns how many. All threads of the workgroup call: the waves count, add up, emit.
template <typename K, typename F, typename G>
__device__ int emit_selected(const Keys<K, F>& keys, K threshold, int ties, G emit) {
  constexpr int kWaves = kSelectThreads / 64;
  __shared__ int above_w[kWaves], equal_w[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int above = 0, equal = 0;
  keys.each([&](int, K x, bool there) {
    above += __popcll(__ballot(there && x > threshold));
    equal += __popcll(__ballot(there && x == threshold));
  });
  if (lane == 0) {
    above_w[wave] = above;
    equal_w[wave] = equal;
  }
  __syncthreads();
  int slot = 0, rank = 0, all = 0, all_equal = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) {
      slot += above_w[w];
      rank += equal_w[w];
    }
    all += above_w[w];
    all_equal += equal_w[w];
  }
  slot += rank < ties ? rank : ties;
  const uint64_t below = (1ull << lane) - 1;
  keys.each([&](int i, K x, bool there) {
    const bool same = there && x == threshold;
    const uint64_t same_bits = __ballot(same);
    const bool take = there && (x > threshold || (same && rank + __popcll(same_bits & below) < ties));
    const uint64_t bits = __ballot(take);
    if (take) emit(slot + __popcll(bits & below), i);
    slot += __popcll(bits);
    rank += __popcll(same_bits);
  });
  return all + (all_equal < ties ? all_equal : ties);
}

// positions[b, hkv, :]: what stays, ascending, -1 behind the last. One workgroup per row: bound by the
// latency of its passes (64 rows of 16 k weights: 16 us; histograms split by lane took the same).
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(CacheEvictParams p, int64_t row0) {
  const int64_t row = row0 + blockIdx.x, b = row / p.heads_kv;
  const int n = static_cast<int>(clamped_length(p.lengths, p.length, b, p.t_max));
  const int budget = static_cast<int>(p.budget), recent = static_cast<int>(p.recent);
  const float* w = p.weights + row * p.t_max;
  int32_t* positions = p.positions + row * p.budget;
  const int kept = n < budget ? n : budget;
  int slot = 0;
  if (n > budget && budget > recent) {
    const int old = n - recent;
    auto key = [&](int i) { return order_key(w[i]); };
    const Keys<uint32_t, decltype(key)> keys(key, old);
    uint32_t threshold;
    const int ties = select_threshold(keys, budget - recent, &threshold);
    slot = emit_selected(keys, threshold, ties, [&](int at, int i) { positions[at] = i; });
  }
  for (int i = slot + threadIdx.x; i < budget; i += blockDim.x) positions[i] = i < kept ? n - kept + i : -1;
}

// A workgroup moves one cache line (128 bytes) of the kept rows of a (entry, head)'s keys or values,
// kMoveSteps rows per thread between two barriers. Rows only ever move to the front, so that the rows
// of a step are read before any later step's place is written: one workgroup that takes all steps in
// turn may write where it reads. Apart, `chunks` workgroups take the steps. Bound by the copy: 64 rows of
// 4096 kept positions of 128 bfloat16 apart 56 us, 4.8 TB/s.
constexpr int kMoveThreads = 512, kMoveSteps = 4;
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(CacheEvictParams p, int64_t row0, int row_bytes,
                                                                  int slices, int chunks) {
  constexpr int kRows = kMoveThreads / 8;
  const int chunk = blockIdx.x % chunks, part = blockIdx.x / chunks % (2 * slices);
  const int64_t row = row0 + blockIdx.x / chunks / (2 * slices), b = row / p.heads_kv;
  const int slice = part >> 1, value = part & 1;
  const int32_t* positions = p.positions + row * p.budget;
  const char* from = static_cast<const char*>(value ? p.v : p.k) + row * p.t_max * row_bytes;
  char* to = static_cast<char*>(value ? p.v_out : p.k_out) + row * p.t_max_out * row_bytes;
  const float* w = p.weights + row * p.t_max;
  float* w_out = p.weights_out + row * p.t_max_out;
  const int at = slice * 128 + (threadIdx.x & 7) * 16, budget = static_cast<int>(p.budget);
  const bool weighs = part == 0 && (threadIdx.x & 7) == 0;
  for (int j0 = chunk * kRows * kMoveSteps; j0 < budget; j0 += chunks * kRows * kMoveSteps) {
    int4 data[kMoveSteps];
    float weight[kMoveSteps];
    int t[kMoveSteps];
#pragma unroll
    for (int i = 0; i < kMoveSteps; ++i) {
      const int j = j0 + i * kRows + (threadIdx.x >> 3);
      t[i] = j < budget ? positions[j] : -1;
    }
#pragma unroll
    for (int i = 0; i < kMoveSteps; ++i) {
      data[i] = int4{0, 0, 0, 0};
      weight[i] = 0.f;
      if (t[i] >= 0 && at < row_bytes)
        data[i] = *reinterpret_cast<const int4*>(from + t[i] * static_cast<int64_t>(row_bytes) + at);
      if (t[i] >= 0 && weighs) weight[i] = w[t[i]];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMoveSteps; ++i) {
      const int64_t j = j0 + i * kRows + (threadIdx.x >> 3);
      if (t[i] >= 0 && at < row_bytes) *reinterpret_cast<int4*>(to + j * row_bytes + at) = data[i];
      if (t[i] >= 0 && weighs) w_out[j] = weight[i];
    }
  }
  if (chunk == 0 && part == 0 && row == b * p.heads_kv && threadIdx.x == 0) {
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

// the way back of a value that came from T
template <typename T>
__device__ __forceinline__ T store_float(float x);
template <>
__device__ __forceinline__ float store_float(float x) { return x; }
template <>
__device__ __forceinline__ __half store_float(float x) { return __float2half(x); }
template <>
__device__ __forceinline__ uint16_t store_float(float x) { return static_cast<uint16_t>(__float_as_uint(x) >> 16); }

// 16 bytes of a row as floats
template <typename T>
__device__ __forceinline__ void unpack(const int4& x, float (&y)[16 / sizeof(T)]) {
  const T* t = reinterpret_cast<const T*>(&x);
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) y[i] = load_float(t[i]);
}

// A wave per (entry, head, block): 16 bytes of a row per lane, lanes of the same channels joined by
// lane exchanges. Rows behind the end repeat the last one, which changes no minimum. minimum /
// maximum hand on a NaN, and every bound is a key's value, so the way back to 16 bits is exact. Bound by
// the reads: 4 entries of up to 32 k positions, 8 heads of 128 float16: 39.6 us, 5.0 TB/s.
template <typename T>
__global__ __launch_bounds__(kThreads) void block_bounds_kernel(CacheBoundsParams p, int64_t blocks, int walkers,
                                                                int lanes) {
  constexpr int V = 16 / sizeof(T);
  const int64_t row = blockIdx.x / walkers, b = row / p.heads_kv;
  const int n = static_cast<int>(clamped_length(p.lengths, p.length, b, p.t_max));
  const int block = static_cast<int>(p.block);
  int first = p.first ? p.first[b] : 0;
  first = first < 0 ? 0 : first / block;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int channel = (lane & (lanes - 1)) * V, at = lane / lanes, step = 64 / lanes;
  const bool there = channel < p.dhead;
  const T* k = static_cast<const T*>(p.k) + row * p.t_max * p.dhead + (there ? channel : 0);
  for (int64_t j = first + blockIdx.x % walkers * (kThreads / 64) + wave; j * block < n; j += walkers * (kThreads / 64)) {
    const int start = static_cast<int>(j) * block, last = (start + block < n ? start + block : n) - 1;
    float low[V], high[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      low[i] = INFINITY;
      high[i] = -INFINITY;
    }
    for (int t = start + at; t <= last + at; t += 8 * step) {
      int4 x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int64_t from = t + u * step < last ? t + u * step : last;
        x[u] = *reinterpret_cast<const int4*>(k + from * p.dhead);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        float y[V];
        unpack<T>(x[u], y);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          low[i] = __builtin_elementwise_minimum(low[i], y[i]);
          high[i] = __builtin_elementwise_maximum(high[i], y[i]);
        }
      }
    }
    for (int o = lanes; o < 64; o <<= 1)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        low[i] = __builtin_elementwise_minimum(low[i], __shfl_xor(low[i], o, 64));
        high[i] = __builtin_elementwise_maximum(high[i], __shfl_xor(high[i], o, 64));
      }
    if (lane < lanes && there) {
      T out[2][V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        out[0][i] = store_float<T>(low[i]);
        out[1][i] = store_float<T>(high[i]);
      }
      T* to = static_cast<T*>(p.bounds) + (row * blocks + j) * 2 * p.dhead + channel;
      *reinterpret_cast<int4*>(to) = *reinterpret_cast<const int4*>(out[0]);
      *reinterpret_cast<int4*>(to + p.dhead) = *reinterpret_cast<const int4*>(out[1]);
    }
  }
}

template <int kControl>
__device__ __forceinline__ double dpp_double(double x) {
  const int64_t bits = __double_as_longlong(x);
  const int low = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits), kControl, 0xf, 0xf, false);
  const int high = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits >> 32), kControl, 0xf, 0xf, false);
  return __longlong_as_double(static_cast<int64_t>(high) << 32 | static_cast<uint32_t>(low));
}

// scores[b, hkv, j] = max over the group's heads of sum_d (q_d >= 0 ? q_d max_d : q_d min_d), NaN where
// a bound is; float64, since a choice between blocks must not depend on how the sum was ordered. Eight
// lanes per block, each with every eighth 16 bytes of its channels, kPair blocks at a time; the heads'
// queries wait in LDS as float64, split into max(q, 0) and min(q, 0): two products by converted bounds
// instead of a choice per head. A bound that is not finite leaves no sum finite (0 x inf is NaN): such
// blocks are summed again by the choice. Bound by the float64 products and the latency of two dependent
// reads more than by the bounds' bytes: 8 entries of 1024 blocks, 32 / 8 heads of 128 bfloat16 11 us, the
// choice after it 7.4. (Both in one workgroup per row, for few blocks: no faster, 22.4 us for the whole call
// at 129 blocks either way, and 3 % slower from 128 channels on.)
template <typename T>
__global__ __launch_bounds__(kThreads) void block_scores_kernel(CacheSelectParams p, int64_t blocks, int walkers) {
  constexpr int V = 16 / sizeof(T), kHeads = 4, kPair = 2, kBlocks = kThreads / 8;  // heads, blocks at a time
  __shared__ double2 q_s[kHeads][256];
  const int64_t row = blockIdx.x / walkers;
  const int64_t b = row / p.heads_kv, hkv = row % p.heads_kv;
  const int group = static_cast<int>(p.heads / p.heads_kv), dhead = static_cast<int>(p.dhead);
  const int n = static_cast<int>(clamped_length(p.lengths, p.length, b, p.t_max));
  const int block = static_cast<int>(p.block), count = (n + block - 1) / block;
  if (count <= p.top) return;  // (all blocks are taken: no scores are looked at)
  const int part = threadIdx.x & 7;
  // the eight lanes' channels side by side: they are read together, from all banks
  auto slot_of = [](int d) { return d / (8 * V) * (8 * V) + d % V * 8 + d / V % 8; };
  const T* bounds = static_cast<const T*>(p.bounds) + row * blocks * 2 * dhead;
  for (int h0 = 0; h0 < group; h0 += kHeads) {
    const int heads = group - h0 < kHeads ? group - h0 : kHeads;
    for (int j0 = static_cast<int>(blockIdx.x % walkers) * kPair * kBlocks, first = j0; j0 < count;
         j0 += walkers * kPair * kBlocks) {
      const T* low[kPair];
      double sum[kPair][kHeads] = {};
#pragma unroll
      for (int u = 0; u < kPair; ++u) {
        const int j = j0 + u * kBlocks + (threadIdx.x >> 3);
        low[u] = bounds + static_cast<int64_t>(j < count ? j : count - 1) * 2 * dhead;
      }
      int4 next[kPair][2];
      auto request = [&](int d) {
#pragma unroll
        for (int u = 0; u < kPair; ++u)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            next[u][i] = *reinterpret_cast<const int4*>(low[u] + (d < dhead ? d : 0) + i * dhead);
      };
      request(part * V);
      if (j0 == first) {  // (the first bounds are on their way while the queries are laid out)
        if (h0) __syncthreads();
        for (int i = threadIdx.x; i < kHeads * dhead; i += kThreads) {
          const int h = i / dhead;
          const double q = h < heads ? p.q[(b * p.heads + hkv * group + h0) * dhead + i] : 0.;
          q_s[h][slot_of(i - h * dhead)] = q >= 0. ? double2{q, 0.} : q < 0. ? double2{0., q} : double2{q, q};
        }
        __syncthreads();
      }
      for (int d = part * V; d < dhead; d += 8 * V) {
        float x[kPair][V], y[kPair][V];
#pragma unroll
        for (int u = 0; u < kPair; ++u) {
          unpack<T>(next[u][0], x[u]);
          unpack<T>(next[u][1], y[u]);
        }
        request(d + 8 * V);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          double a[kPair], c[kPair];  // (converted once for all heads)
#pragma unroll
          for (int u = 0; u < kPair; ++u) {
            a[u] = x[u][i];
            c[u] = y[u][i];
          }
#pragma unroll
          for (int h = 0; h < kHeads; ++h) {
            const double2 q = q_s[h][slot_of(d + i)];
#pragma unroll
            for (int u = 0; u < kPair; ++u) sum[u][h] = fma(q.y, a[u], fma(q.x, c[u], sum[u][h]));
          }
        }
      }
      // The eight lanes add up and share out at once: a block's four sums to the lane across (7 - i) or
      // kept, two of them two lanes on, one to the neighbour. A lane ends with head (bits 1, 0) of block
      // (bit 2).
      const bool upper = part & 4, second = part & 2, odd = part & 1;
      auto share = [&] {
        double s4[kHeads], s2[2];
#pragma unroll
        for (int h = 0; h < kHeads; ++h)
          s4[h] = (upper ? sum[1][h] : sum[0][h]) + dpp_double<0x141>(upper ? sum[0][h] : sum[1][h]);
#pragma unroll
        for (int h = 0; h < 2; ++h)
          s2[h] = (second ? s4[2 + h] : s4[h]) + dpp_double<0x4e>(second ? s4[h] : s4[2 + h]);
        return (odd ? s2[1] : s2[0]) + dpp_double<0xb1>(odd ? s2[0] : s2[1]);
      };
      double mine = share();
      int nan = 0;  // bit u: block u has a NaN bound
      if (!__all(fabs(mine) < INFINITY)) {
#pragma unroll
        for (int u = 0; u < kPair; ++u) {
#pragma unroll
          for (int h = 0; h < kHeads; ++h) sum[u][h] = 0.;
          for (int d0 = part * V; d0 < dhead; d0 += 8 * V)
            for (int d = d0; d < d0 + V; ++d) {
              const float x = load_float(low[u][d]), y = load_float(low[u][dhead + d]);
              nan |= __builtin_isunordered(x, y) ? 1 << u : 0;
#pragma unroll
              for (int h = 0; h < kHeads; ++h) {
                const double2 q = q_s[h][slot_of(d)];
                sum[u][h] = fma(q.x + q.y, static_cast<double>(q.y < 0. ? x : y), sum[u][h]);
              }
            }
        }
        mine = share();
        nan |= __builtin_amdgcn_update_dpp(0, nan, 0x141, 0xf, 0xf, false);
        nan |= __builtin_amdgcn_update_dpp(0, nan, 0x4e, 0xf, 0xf, false);
        nan |= __builtin_amdgcn_update_dpp(0, nan, 0xb1, 0xf, 0xf, false);
      }
      // the larger of two, NaN above all
      auto larger = [](double a, double c) { return c > a || c != c ? c : a; };
      double best = (part & 3) < heads ? mine : -INFINITY;
      best = larger(best, dpp_double<0xb1>(best));
      best = larger(best, dpp_double<0x4e>(best));
      const int j = j0 + (part >> 2) * kBlocks + (threadIdx.x >> 3);
      if ((part & 3) == 0 && j < count) {
        if (h0) best = larger(best, p.scores[row * blocks + j]);
        p.scores[row * blocks + j] = nan >> (part >> 2) & 1 ? __builtin_nan("") : best;
      }
    }
  }
}

__global__ __launch_bounds__(kSelectThreads) void block_select_kernel(CacheSelectParams p, int64_t row0, int64_t blocks) {
  const int64_t row = row0 + blockIdx.x, b = row / p.heads_kv;
  const int64_t n = clamped_length(p.lengths, p.length, b, p.t_max);
  const int count = static_cast<int>((n + p.block - 1) / p.block), top = static_cast<int>(p.top);
  const double* scores = p.scores + row * blocks;
  int32_t* selected = p.selected + row * p.top;
  if (count > top) {
    auto key = [&](int j) { return j < p.sink || j >= count - p.local ? ~0ull : order_key(scores[j]); };
    const Keys<uint64_t, decltype(key)> keys(key, count);
    uint64_t threshold;
    const int ties = select_threshold(keys, top, &threshold);
    emit_selected(keys, threshold, ties, [&](int at, int j) { selected[at] = j; });
  } else {
    for (int j = threadIdx.x; j < top; j += blockDim.x) selected[j] = j < count ? j : -1;
  }
}

// Workgroups per (entry, head): enough for eight on every CU, at most one for `pieces` each.
int walkers_for(int64_t rows, int64_t pieces) {
  const int64_t fill = (2048 + rows - 1) / rows;
  return static_cast<int>(fill < pieces ? fill : pieces);
}

// launch(first row, workgroups) for stretches of rows with `per_row` workgroups each
template <typename F>
void for_rows(int64_t rows, int64_t per_row, F launch) {
  const int64_t most = kMostGroups / per_row;
  for (int64_t row0 = 0; row0 < rows; row0 += most)
    launch(row0, static_cast<unsigned>((rows - row0 < most ? rows - row0 : most) * per_row));
}

template <typename T>
void bounds_typed(const CacheBoundsParams& p, int64_t blocks, hipStream_t stream) {
  const int64_t rows = p.batch * p.heads_kv;
  const int walkers = walkers_for(rows, (blocks + kThreads / 64 - 1) / (kThreads / 64));
  int lanes = 1;
  while (lanes * 16 < static_cast<int>(p.dhead * sizeof(T))) lanes *= 2;
  hipLaunchKernelGGL((block_bounds_kernel<T>), dim3(static_cast<unsigned>(rows * walkers)), dim3(kThreads), 0, stream,
                     p, blocks, walkers, lanes);
}

template <typename T>
void scores_typed(const CacheSelectParams& p, int64_t blocks, hipStream_t stream) {
  const int64_t rows = p.batch * p.heads_kv;
  const int walkers = walkers_for(rows, (blocks + kThreads / 4 - 1) / (kThreads / 4));
  hipLaunchKernelGGL((block_scores_kernel<T>), dim3(static_cast<unsigned>(rows * walkers)), dim3(kThreads), 0, stream,
                     p, blocks, walkers);
}

}  // namespace

void launch_cache_evict(const CacheEvictParams& p, hipStream_t stream) {
  const int row_bytes = static_cast<int>(p.dhead) * (p.kv_dtype == 0 ? 4 : 2);
  const int slices = (row_bytes + 127) / 128;
  const int64_t rows = p.batch * p.heads_kv;
  const int64_t steps = (p.budget + kMoveThreads / 8 * kMoveSteps - 1) / (kMoveThreads / 8 * kMoveSteps);
  // in place the steps have an order
  const int chunks = p.k == p.k_out || p.v == p.v_out || p.weights == p.weights_out ? 1 : walkers_for(rows * 2 * slices, steps);
  for_rows(rows, 1, [&](int64_t row0, unsigned groups) {
    hipLaunchKernelGGL(evict_select_kernel, dim3(groups), dim3(kSelectThreads), 0, stream, p, row0);
  });
  for_rows(rows, 2 * slices * chunks, [&](int64_t row0, unsigned groups) {
    hipLaunchKernelGGL(evict_move_kernel, dim3(groups), dim3(kMoveThreads), 0, stream, p, row0, row_bytes, slices,
                       chunks);
  });
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
  for_rows(p.batch * p.heads_kv, 1, [&](int64_t row0, unsigned groups) {
    hipLaunchKernelGGL(block_select_kernel, dim3(groups), dim3(kSelectThreads), 0, stream, p, row0, blocks);
  });
}

}  // namespace ct2x
