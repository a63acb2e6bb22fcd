// Attention over a serving cache and the upkeep of that cache (attention_cache.hip, cache_ops.hip):
// a tree of drafted tokens, one token that leaves its probabilities behind, eviction, block bounds,
// attention over selected blocks. Key / value caches [batch, heads_kv, t_max, dhead] in float32 /
// float16 / bfloat16, queries and outputs float32.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace ct2x {

// sums over the lanes up to each
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  auto moved = [&](auto ctrl, auto rows) {
    return static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  x += moved(integral_constant<int, 0x111>(), integral_constant<int, 0xf>());  // 1, 2, 4, 8 to the right in a row
  x += moved(integral_constant<int, 0x112>(), integral_constant<int, 0xf>());
  x += moved(integral_constant<int, 0x114>(), integral_constant<int, 0xf>());
  x += moved(integral_constant<int, 0x118>(), integral_constant<int, 0xf>());
  x += moved(integral_constant<int, 0x142>(), integral_constant<int, 0xa>());  // the rows before, summed
  x += moved(integral_constant<int, 0x143>(), integral_constant<int, 0xc>());
  return x;
}

// What an attention over the cache reads besides the committed positions of an entry.
enum class CacheView {
  kTree,    // + the drafted tokens behind them, by the tree's mask
  kDense,   // nothing more
  kBlocks,  // only the positions of selected blocks
};

struct CacheAttnParams {
  const float* q = nullptr;  // [batch, tokens, heads, dhead]
  const void* k = nullptr;   // [batch, heads_kv, t_max, dhead]
  const void* v = nullptr;
  int kv_dtype = 0;
  const int32_t* lengths = nullptr;  // [batch] committed positions (nullptr = `length`)
  int64_t length = 0;
  int64_t batch = 0, tokens = 1, heads = 0, heads_kv = 0, dhead = 0, t_max = 0;
  float scale = 1.f;
  float* out = nullptr;  // [batch, tokens, heads, dhead]
  CacheView view = CacheView::kDense;
  // kTree: bit j of words [b, i, :] = drafted token i sees drafted token j (nullptr: j <= i)
  const uint64_t* mask = nullptr;
  // kDense: weights [batch, heads_kv, t_max] += probabilities (nullptr = none)
  float* weights = nullptr;
  // kBlocks: selected [batch, heads_kv, top] block numbers, ascending, -1 behind the last
  const int32_t* selected = nullptr;
  int64_t block = 0, top = 0;
  void* scratch = nullptr;  // cache_attention_scratch_bytes(...)
};

int64_t cache_attention_scratch_bytes(const CacheAttnParams& p);
void launch_cache_attention(const CacheAttnParams& p, hipStream_t stream);

struct CacheEvictParams {
  const void* k = nullptr;
  const void* v = nullptr;
  int kv_dtype = 0;
  const float* weights = nullptr;  // [batch, heads_kv, t_max]
  const int32_t* lengths = nullptr;
  int64_t length = 0;
  int64_t batch = 0, heads_kv = 0, dhead = 0, t_max = 0, budget = 0, recent = 0, t_max_out = 0;
  void* k_out = nullptr;  // [batch, heads_kv, t_max_out, dhead]; == k: in place
  void* v_out = nullptr;
  float* weights_out = nullptr;      // [batch, heads_kv, t_max_out]
  int32_t* positions = nullptr;      // [batch, heads_kv, budget]
  int32_t* lengths_out = nullptr;    // [batch]
};
void launch_cache_evict(const CacheEvictParams& p, hipStream_t stream);

struct CacheBoundsParams {
  const void* k = nullptr;
  int kv_dtype = 0;
  const int32_t* first = nullptr;  // [batch] first new position (nullptr = 0)
  const int32_t* lengths = nullptr;
  int64_t length = 0;
  int64_t batch = 0, heads_kv = 0, dhead = 0, t_max = 0, block = 0;
  void* bounds = nullptr;  // [batch, heads_kv, ceil(t_max / block), 2, dhead]
};
void launch_cache_block_bounds(const CacheBoundsParams& p, hipStream_t stream);

// selected [batch, heads_kv, top]: the blocks of an entry's q rows (group heads each) by the bounds
struct CacheSelectParams {
  const float* q = nullptr;  // [batch, heads, dhead]
  const void* bounds = nullptr;
  int kv_dtype = 0;
  const int32_t* lengths = nullptr;
  int64_t length = 0;
  int64_t batch = 0, heads = 0, heads_kv = 0, dhead = 0, t_max = 0, block = 0, top = 0, sink = 0, local = 0;
  double* scores = nullptr;  // [batch, heads_kv, ceil(t_max / block)]
  int32_t* selected = nullptr;
};
void launch_cache_select(const CacheSelectParams& p, hipStream_t stream);

}  // namespace ct2x
