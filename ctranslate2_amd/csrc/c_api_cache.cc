// extern "C" surface of the attention over a serving cache and of the cache's upkeep
// (include/ct2_mi355.h, "attention over a serving cache"). Argument checking + launch + error
// translation only; no arithmetic happens on the host.

#include "../../include/ct2_mi355.h"

#include <string>

#include "cache_ops.h"
#include "runtime.h"

using namespace ct2x;

#define API_TRY try {
#define API_CATCH                                     \
  }                                                   \
  catch (const std::exception& e) {                   \
    set_last_error(e.what());                         \
    return 1;                                         \
  }                                                   \
  return 0;
#define API_SIZE_CATCH                                \
  }                                                   \
  catch (const std::exception& e) {                   \
    set_last_error(e.what());                         \
    return -1;                                        \
  }

namespace {

#define CACHE_CHECK(cond, msg) CT2X_CHECK(cond, std::string(name) + ": " msg)

int64_t element_bytes(int dtype) { return dtype == CT2X_F32 ? 4 : 2; }

int64_t aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// What every entry point of the family asks of the cache's sizes.
void check_cache(const char* name, int64_t batch, int64_t heads_kv, int64_t dhead, int64_t t_max) {
  CACHE_CHECK(batch >= 0 && heads_kv >= 1, "batch must be >= 0 and heads_kv >= 1");
  CACHE_CHECK(dhead >= 8 && dhead <= 256 && dhead % 8 == 0, "dhead must be a multiple of 8 in [8, 256]");
  CACHE_CHECK(t_max >= 1 && t_max <= ((int64_t{1} << 31) - (int64_t{1} << 20)) / (dhead * 4),
              "t_max must be >= 1 and t_max * dhead * 4 at most 2^31 - 2^20 (one head of one entry)");
  CACHE_CHECK(batch <= (int64_t{1} << 22) / heads_kv, "batch * heads_kv above 2^22");
}

void check_heads(const char* name, int64_t batch, int64_t tokens, int64_t heads, int64_t heads_kv) {
  CACHE_CHECK(heads >= heads_kv && heads % heads_kv == 0, "heads must be a multiple of heads_kv");
  CACHE_CHECK(heads / heads_kv <= 1024, "heads / heads_kv above 1024");
  CACHE_CHECK(batch * tokens <= (int64_t{1} << 26) / heads, "batch * tokens * heads above 2^26");
}

void check_type(const char* name, int dtype) {
  CACHE_CHECK(dtype == CT2X_F32 || dtype == CT2X_F16 || dtype == CT2X_BF16,
              "the cache type must be CT2X_F32, CT2X_F16 or CT2X_BF16");
}

void check_length(const char* name, const int32_t* d_lengths, int64_t length, int64_t room) {
  CACHE_CHECK(d_lengths != nullptr || (length >= 0 && length <= room),
              "length does not fit the cache (it is read when d_lengths is NULL)");
}

template <typename... P>
void check_pointers(const char* name, const P*... pointers) {
  for (const void* p : {static_cast<const void*>(pointers)...})
    CACHE_CHECK(p != nullptr, "a required pointer is NULL");
}

template <typename... P>
void check_alignment(const char* name, const P*... pointers) {
  for (const void* p : {static_cast<const void*>(pointers)...})
    CACHE_CHECK(reinterpret_cast<uintptr_t>(p) % 16 == 0, "tensors must be aligned to 16 bytes");
}

// The bytes that an argument covers.
struct Span {
  const void* at;
  int64_t bytes;
  bool apart(const Span& other) const {
    const uintptr_t x = reinterpret_cast<uintptr_t>(at), y = reinterpret_cast<uintptr_t>(other.at);
    return bytes == 0 || other.bytes == 0 || x + bytes <= y || y + other.bytes <= x;
  }
};

void check_scratch(const char* name, const void* d_scratch, int64_t bytes, int64_t need) {
  CACHE_CHECK(need == 0 || (d_scratch != nullptr && bytes >= need),
              "scratch missing or smaller than the _scratch_bytes() function says");
}

CacheAttnParams attention_sizes(CacheView view, int64_t batch, int64_t tokens, int64_t heads, int64_t heads_kv,
                                int64_t dhead, int64_t t_max) {
  CacheAttnParams p;
  p.view = view;
  p.batch = batch;
  p.tokens = tokens;
  p.heads = heads;
  p.heads_kv = heads_kv;
  p.dhead = dhead;
  p.t_max = t_max;
  return p;
}

void check_tree(const char* name, int64_t batch, int64_t tokens, int64_t heads, int64_t heads_kv, int64_t dhead,
                int64_t t_max) {
  check_cache(name, batch, heads_kv, dhead, t_max);
  CACHE_CHECK(tokens >= 0 && tokens <= 1024 && tokens <= t_max, "tokens must be in [0, 1024] and fit t_max");
  check_heads(name, batch, tokens, heads, heads_kv);
}

void check_dense(const char* name, int64_t batch, int64_t heads, int64_t heads_kv, int64_t dhead, int64_t t_max) {
  check_cache(name, batch, heads_kv, dhead, t_max);
  check_heads(name, batch, 1, heads, heads_kv);
}

void check_block(const char* name, int64_t block) {
  CACHE_CHECK(block >= 16 && block <= 256 && block % 16 == 0, "block must be a multiple of 16 in [16, 256]");
}

CacheAttnParams blocks_sizes(const char* name, int64_t batch, int64_t heads, int64_t heads_kv, int64_t dhead,
                             int64_t t_max, int64_t block, int64_t top) {
  check_dense(name, batch, heads, heads_kv, dhead, t_max);
  check_block(name, block);
  CACHE_CHECK(top >= 1 && top <= (int64_t{1} << 20), "top must be in [1, 2^20]");
  CacheAttnParams p = attention_sizes(CacheView::kBlocks, batch, 1, heads, heads_kv, dhead, t_max);
  p.block = block;
  p.top = top;
  return p;
}

// scores | selected | the attention's own
struct BlocksScratch {
  int64_t selected, attention, total;
  explicit BlocksScratch(const CacheAttnParams& p) {
    const int64_t blocks = (p.t_max + p.block - 1) / p.block;
    selected = aligned(p.batch * p.heads_kv * blocks * 8);
    attention = selected + aligned(p.batch * p.heads_kv * p.top * 4);
    total = attention + cache_attention_scratch_bytes(p);
  }
};

}  // namespace

extern "C" {

int64_t ct2x_attention_tree_scratch_bytes(int64_t batch, int64_t tokens, int64_t heads, int64_t heads_kv,
                                          int64_t dhead, int64_t t_max) {
  API_TRY
  check_tree("ct2x_attention_tree_scratch_bytes", batch, tokens, heads, heads_kv, dhead, t_max);
  return cache_attention_scratch_bytes(
      attention_sizes(CacheView::kTree, batch, tokens, heads, heads_kv, dhead, t_max));
  API_SIZE_CATCH
}

int ct2x_attention_tree(const float* d_q, const void* d_k_cache, const void* d_v_cache, int kv_dtype,
                        const int32_t* d_lengths, int64_t length, const uint64_t* d_tree_mask, int64_t batch,
                        int64_t tokens, int64_t heads, int64_t heads_kv, int64_t dhead, int64_t t_max, float scale,
                        float* d_out, void* d_scratch, int64_t scratch_bytes, void* stream) {
  API_TRY
  const char* name = "ct2x_attention_tree";
  check_tree(name, batch, tokens, heads, heads_kv, dhead, t_max);
  check_type(name, kv_dtype);
  check_length(name, d_lengths, length, t_max - tokens);
  if (batch == 0 || tokens == 0) return 0;
  check_pointers(name, d_q, d_k_cache, d_v_cache, d_out);
  check_alignment(name, d_q, d_k_cache, d_v_cache, d_out, d_scratch);
  CacheAttnParams p = attention_sizes(CacheView::kTree, batch, tokens, heads, heads_kv, dhead, t_max);
  check_scratch(name, d_scratch, scratch_bytes, cache_attention_scratch_bytes(p));
  p.q = d_q;
  p.k = d_k_cache;
  p.v = d_v_cache;
  p.kv_dtype = kv_dtype;
  p.lengths = d_lengths;
  p.length = length;
  p.mask = d_tree_mask;
  p.scale = scale;
  p.out = d_out;
  p.scratch = d_scratch;
  launch_cache_attention(p, resolve_stream(stream));
  check_last_launch("attention_tree");
  API_CATCH
}

int64_t ct2x_attention_accumulate_scratch_bytes(int64_t batch, int64_t heads, int64_t heads_kv, int64_t dhead,
                                                int64_t t_max) {
  API_TRY
  check_dense("ct2x_attention_accumulate_scratch_bytes", batch, heads, heads_kv, dhead, t_max);
  return cache_attention_scratch_bytes(attention_sizes(CacheView::kDense, batch, 1, heads, heads_kv, dhead, t_max));
  API_SIZE_CATCH
}

int ct2x_attention_accumulate(const float* d_q, const void* d_k_cache, const void* d_v_cache, int kv_dtype,
                              const int32_t* d_lengths, int64_t length, int64_t batch, int64_t heads,
                              int64_t heads_kv, int64_t dhead, int64_t t_max, float scale, float* d_weights,
                              float* d_out, void* d_scratch, int64_t scratch_bytes, void* stream) {
  API_TRY
  const char* name = "ct2x_attention_accumulate";
  check_dense(name, batch, heads, heads_kv, dhead, t_max);
  check_type(name, kv_dtype);
  check_length(name, d_lengths, length, t_max);
  if (batch == 0) return 0;
  check_pointers(name, d_q, d_k_cache, d_v_cache, d_weights, d_out);
  check_alignment(name, d_q, d_k_cache, d_v_cache, d_out, d_scratch);
  CacheAttnParams p = attention_sizes(CacheView::kDense, batch, 1, heads, heads_kv, dhead, t_max);
  check_scratch(name, d_scratch, scratch_bytes, cache_attention_scratch_bytes(p));
  p.q = d_q;
  p.k = d_k_cache;
  p.v = d_v_cache;
  p.kv_dtype = kv_dtype;
  p.lengths = d_lengths;
  p.length = length;
  p.scale = scale;
  p.weights = d_weights;
  p.out = d_out;
  p.scratch = d_scratch;
  launch_cache_attention(p, resolve_stream(stream));
  check_last_launch("attention_accumulate");
  API_CATCH
}

int ct2x_cache_evict(const void* d_k_cache, const void* d_v_cache, int kv_dtype, const float* d_weights,
                     const int32_t* d_lengths, int64_t length, int64_t batch, int64_t heads_kv, int64_t dhead,
                     int64_t t_max, int64_t budget, int64_t recent, int64_t t_max_out, void* d_k_out, void* d_v_out,
                     float* d_weights_out, int32_t* d_positions, int32_t* d_lengths_out, void* stream) {
  API_TRY
  const char* name = "ct2x_cache_evict";
  check_cache(name, batch, heads_kv, dhead, t_max);
  check_type(name, kv_dtype);
  check_length(name, d_lengths, length, t_max);
  CACHE_CHECK(budget >= 1 && recent >= 0 && recent <= budget, "budget must be >= 1 and recent in [0, budget]");
  check_cache(name, batch, heads_kv, dhead, t_max_out);
  CACHE_CHECK(t_max_out >= budget, "t_max_out is smaller than the budget");
  if (batch == 0) return 0;
  check_pointers(name, d_k_cache, d_v_cache, d_weights, d_k_out, d_v_out, d_weights_out, d_positions, d_lengths_out);
  check_alignment(name, d_k_cache, d_v_cache, d_k_out, d_v_out);
  // in place, or nowhere near: what one workgroup writes, another may still have to read
  const int64_t row = dhead * element_bytes(kv_dtype), in = batch * heads_kv * t_max, out = batch * heads_kv * t_max_out;
  const Span inputs[] = {{d_k_cache, in * row}, {d_v_cache, in * row}, {d_weights, in * 4},
                         {d_lengths, d_lengths ? batch * 4 : 0}};
  const Span outputs[] = {{d_k_out, out * row}, {d_v_out, out * row}, {d_weights_out, out * 4},
                          {d_lengths_out, batch * 4}, {d_positions, batch * heads_kv * budget * 4}};
  for (int o = 0; o < 5; ++o) {
    for (int i = 0; i < 4; ++i) {
      // an output's own input: the first three with the same room, the lengths always
      const bool in_place = o == i && outputs[o].at == inputs[i].at && (o == 3 || t_max == t_max_out);
      CACHE_CHECK(in_place || outputs[o].apart(inputs[i]),
                  "outputs and inputs overlap (an output may be its own input, with the same t_max)");
    }
    for (int i = 0; i < o; ++i) CACHE_CHECK(outputs[o].apart(outputs[i]), "two outputs overlap");
  }
  CacheEvictParams p;
  p.k = d_k_cache;
  p.v = d_v_cache;
  p.kv_dtype = kv_dtype;
  p.weights = d_weights;
  p.lengths = d_lengths;
  p.length = length;
  p.batch = batch;
  p.heads_kv = heads_kv;
  p.dhead = dhead;
  p.t_max = t_max;
  p.budget = budget;
  p.recent = recent;
  p.t_max_out = t_max_out;
  p.k_out = d_k_out;
  p.v_out = d_v_out;
  p.weights_out = d_weights_out;
  p.positions = d_positions;
  p.lengths_out = d_lengths_out;
  launch_cache_evict(p, resolve_stream(stream));
  check_last_launch("cache_evict");
  API_CATCH
}

int ct2x_cache_block_bounds(const void* d_k_cache, int kv_dtype, const int32_t* d_first, const int32_t* d_lengths,
                            int64_t length, int64_t batch, int64_t heads_kv, int64_t dhead, int64_t t_max,
                            int64_t block, void* d_bounds, void* stream) {
  API_TRY
  const char* name = "ct2x_cache_block_bounds";
  check_cache(name, batch, heads_kv, dhead, t_max);
  check_type(name, kv_dtype);
  check_length(name, d_lengths, length, t_max);
  check_block(name, block);
  if (batch == 0) return 0;
  check_pointers(name, d_k_cache, d_bounds);
  check_alignment(name, d_k_cache, d_bounds);
  CacheBoundsParams p;
  p.k = d_k_cache;
  p.kv_dtype = kv_dtype;
  p.first = d_first;
  p.lengths = d_lengths;
  p.length = length;
  p.batch = batch;
  p.heads_kv = heads_kv;
  p.dhead = dhead;
  p.t_max = t_max;
  p.block = block;
  p.bounds = d_bounds;
  launch_cache_block_bounds(p, resolve_stream(stream));
  check_last_launch("cache_block_bounds");
  API_CATCH
}

int64_t ct2x_attention_blocks_scratch_bytes(int64_t batch, int64_t heads, int64_t heads_kv, int64_t dhead,
                                            int64_t t_max, int64_t block, int64_t top) {
  API_TRY
  return BlocksScratch(blocks_sizes("ct2x_attention_blocks_scratch_bytes", batch, heads, heads_kv, dhead, t_max,
                                    block, top)).total;
  API_SIZE_CATCH
}

int ct2x_attention_blocks(const float* d_q, const void* d_k_cache, const void* d_v_cache, int kv_dtype,
                          const void* d_bounds, const int32_t* d_lengths, int64_t length, int64_t batch,
                          int64_t heads, int64_t heads_kv, int64_t dhead, int64_t t_max, int64_t block, int64_t top,
                          int64_t sink, int64_t local, float scale, float* d_out, int32_t* d_selected,
                          void* d_scratch, int64_t scratch_bytes, void* stream) {
  API_TRY
  const char* name = "ct2x_attention_blocks";
  CacheAttnParams p = blocks_sizes(name, batch, heads, heads_kv, dhead, t_max, block, top);
  check_type(name, kv_dtype);
  check_length(name, d_lengths, length, t_max);
  CACHE_CHECK(sink >= 0 && local >= 0 && sink <= top && local <= top - sink, "sink + local must be in [0, top]");
  CACHE_CHECK(scale > 0.f, "scale must be positive (the bounds are of q . k)");
  if (batch == 0) return 0;
  check_pointers(name, d_q, d_k_cache, d_v_cache, d_bounds, d_out);
  check_alignment(name, d_q, d_k_cache, d_v_cache, d_bounds, d_out, d_scratch);
  const BlocksScratch scratch(p);
  check_scratch(name, d_scratch, scratch_bytes, scratch.total);
  char* base = static_cast<char*>(d_scratch);
  CacheSelectParams s;
  s.q = d_q;
  s.bounds = d_bounds;
  s.kv_dtype = kv_dtype;
  s.lengths = d_lengths;
  s.length = length;
  s.batch = batch;
  s.heads = heads;
  s.heads_kv = heads_kv;
  s.dhead = dhead;
  s.t_max = t_max;
  s.block = block;
  s.top = top;
  s.sink = sink;
  s.local = local;
  s.scores = reinterpret_cast<double*>(base);
  s.selected = d_selected ? d_selected : reinterpret_cast<int32_t*>(base + scratch.selected);
  p.q = d_q;
  p.k = d_k_cache;
  p.v = d_v_cache;
  p.kv_dtype = kv_dtype;
  p.lengths = d_lengths;
  p.length = length;
  p.scale = scale;
  p.out = d_out;
  p.selected = s.selected;
  p.scratch = base + scratch.attention;
  hipStream_t hip_stream = resolve_stream(stream);
  launch_cache_select(s, hip_stream);
  check_last_launch("attention_blocks (selection)");
  launch_cache_attention(p, hip_stream);
  check_last_launch("attention_blocks");
  API_CATCH
}

}  // extern "C"
