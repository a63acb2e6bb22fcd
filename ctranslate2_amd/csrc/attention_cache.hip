// Attention over a serving cache: softmax(scale q K^T) V of one entry's rows (drafted tokens x heads
// of a group) against the positions that its view shows (cache_ops.h).
//
// With s_t = scale q . k_t over the visible positions t, one pass keeps m = max s_t,
// l = sum exp(s_t - m) and o = sum exp(s_t - m) v_t in float32; a later maximum M rescales l and o
// by exp(m - M), and parts of the cache join the same way. out = o / l; a row that sees nothing has
// l = 0 and an output of zero. Positions that a row does not see never enter a sum, whatever they
// hold.
//
// Matrix cores. A wave takes kStep positions and NT tiles of 16 rows:
//   S^T = K Q^T   the key rows as they lie in memory are the A operand, rows of q the columns of B;
//                 a lane then holds kLane consecutive positions of one row (its column), so that
//                 the row's maximum and rescaling are the lane's own but for two lane swaps;
//   O^T = V^T P^T P^T is that same register file: the position that a lane's element stands for is a
//                 free choice of which key row went into which row of the A operand, and it is made so
//                 that B's layout comes out. V^T's rows are channels: a lane loads W consecutive
//                 channels of a position (256 bytes per 16 lanes) and MFMA number e takes the e-th of
//                 each, so output row r of MFMA e is channel W r + e and nothing is transposed; the
//                 16-bit types pair positions with one v_perm per register.
// Up to 32 rows (a decode step, a small tree) every wave loads its own positions straight into the
// operands' registers, the next step's requested as they come free: bound by the reads. From 33 rows on,
// heads of up to 128 channels: tiles of 16 KB of keys and of values in LDS, filled by loads that bypass the
// registers, one tile ahead, shared by four or eight waves of 16 rows each, of 32 in long calls (make_plan):
// bound by the matrix cores (and, on short caches, by a workgroup's way in and out: queries split, parts
// written and joined).
// Measured, with finish_kernel: 32 entries of 5.2 k positions on average, 8 heads of 128 bfloat16, one
// token of 32 heads: 157 us, 4.4 TB/s (a copy: 5.06); 4 entries of 23 k, 64 tokens: 298 to 305 us, 0.95 to 0.98
// PFLOP/s of 16-bit products, three for each of the formula's (a library product of 8192^3: 1.12); 16 entries of
// 1.3 k, 26 tokens: 55 us. Tried with two terms of bfloat16 on the second, where they and 32 rows a wave took 200 us:
// four row tiles per wave without LDS 452 us (outputs and queries need all 512 registers and spill), values by
// the transposing LDS read instead of v_perm 220 against 207.
//
// 16-bit caches: a query (scaled by a power of two to [1, 2) first) and a probability enter as a sum of
// 16-bit terms - the output is float32, and one term would cost 2^-8 (bfloat16) or 2^-11 (float16).
// A term's rest is at most half its step, and its sign one bit more: three of bfloat16 leave 2^-26 (two 2^-17),
// two of float16 2^-23. float16's steps end at 2^-24, so that a second term of something small holds
// only its first bits. A query's is therefore what the first left times 2^11, with sums of its own that
// join the others' times 2^-11: 2^-23 of an element is left, or 2^-36 of the row's largest (unscaled: 2^-25 of the
// row's largest; 300 positions, one query channel of 16384 beside others of 2: outputs off by 4e-4). A
// probability's range ends below 2^16 and begins at 2^13 (kLift): 2^-23 of it is left, or 2^-38 of the row's
// largest. (Sums of their own for it as well: 5 to 15 % of a tree's time, 340 for 290 us on 16 x 64 tokens and
// 8 k positions.)
// float32 caches use the float32 MFMA, nothing is rounded.
//
// Work is cut evenly whatever the lengths: the rounds (kStep positions per wave that shares a row
// group) of all (entry, head, row group) units form one line, workgroup w of G takes the w-th G-th of
// it. A unit that lies within one workgroup is finished there; the others leave (m, l, o) per part
// and finish_kernel adds them. A workgroup leaves at most two such parts (its first and its last
// unit); the one that begins a unit writes down where its parts are.
#include <hip/hip_fp16.h>

#include <algorithm>
#include <atomic>

#include "cache_line.h"
#include "cache_ops.h"
#include "device_utils.h"
#include "runtime.h"

namespace ct2x {

namespace {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;  // of a workgroup whose waves load for themselves; shared tiles: 512
constexpr int waves_of(bool shared) { return shared ? 8 : 4; }
constexpr float kLog2e = 1.44269504088896340736f;
// Buffer offsets that are out of range of every head's region (at most 2^31 - 2^20 bytes), the load
// returns zeros: of a row that is not there, and of channels behind dhead; their sum does not wrap.
constexpr uint32_t kNoRow = 0x80000000u, kNoChannel = 0x7ff00000u;

constexpr int kF32 = 0, kF16 = 4, kBF16 = 5;

// How a launch cuts its work; the same on the host and in every kernel of a call.
struct CachePlan {
  bool shared;      // positions shared through LDS
  int tiles;        // tiles of 16 rows of a wave
  int row_waves;    // waves of a workgroup that take different rows; the others share rows and take
                    // different positions
  int unit_rows;    // rows of a unit
  int row_groups;   // units per (entry, head of the cache)
  int round_shift;  // log2 of the positions of a round
  int group, rows;  // heads of a head of the cache, rows of an entry and head
  uint32_t block_magic;  // ceil(2^32 / (block / 16)), 0 for blocks of 16
  int grid;         // workgroups at most
  int min_rounds;   // per workgroup
  bool whole;       // one workgroup per unit
  int64_t score_pitch;  // accumulate: floats between the score rows
  // scratch, in floats
  int64_t records, parts_ml, parts_o, stats, scores, total;
  int join_groups;  // workgroups of finish_kernel that join parts
  int weight_tiles; // and those per (entry, head) that add up the weights
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return static_cast<int64_t>(static_cast<uint32_t>(uniform(static_cast<int>(x)))) |
         static_cast<int64_t>(uniform(static_cast<int>(x >> 32))) << 32;
}

__device__ __forceinline__ int committed(const CacheAttnParams& p, int64_t b) {
  const int64_t room = p.t_max - (p.view == CacheView::kTree ? p.tokens : 0);
  // (by the scalar cache where b is the wave's)
  const auto* lengths = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(
      reinterpret_cast<uintptr_t>(p.lengths));
  const int64_t n = p.lengths ? lengths[b] : p.length;
  return static_cast<int>(n < 0 ? 0 : (n > room ? room : n));
}

// positions that entry b's rows walk (selected blocks: counted block by block)
__device__ __forceinline__ int walked(const CacheAttnParams& p, int64_t b) {
  const int n = committed(p, b);
  if (p.view == CacheView::kTree) return n + static_cast<int>(p.tokens);
  if (p.view == CacheView::kDense) return n;
  const int block = static_cast<int>(p.block), blocks = (n + block - 1) / block, top = static_cast<int>(p.top);
  return (blocks < top ? blocks : top) * block;
}

// at least one: an entry without positions still has outputs to write
__device__ __forceinline__ int rounds_of(const CacheAttnParams& p, const CachePlan& plan, int64_t b) {
  const int n = (walked(p, b) + (1 << plan.round_shift) - 1) >> plan.round_shift;
  return n < 1 ? 1 : n;
}

// ---- the types -------------------------------------------------------------------------------

template <int kType>
struct Mfma {  // 16-bit
  static __device__ __forceinline__ v4f mul(v4u a, v4u b, v4f c) {
    if constexpr (kType == kF16)
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0,
                                                     0);
  }
  // the pair x0, x1 as a sum of kTerms pairs of 16-bit values, up to half a step of the last, each after the
  // first times 1 / back
  template <int kTerms>
  static __device__ __forceinline__ void split(float x0, float x1, uint32_t (&terms)[kTerms], float back = 1.f) {
    v2f x = {x0, x1};
#pragma unroll
    for (int t = 0; t < kTerms; ++t) {
      if constexpr (kType == kF16) {
        const v2h y = __builtin_convertvector(x, v2h);
        terms[t] = __builtin_bit_cast(uint32_t, y);
        x = (x - __builtin_convertvector(y, v2f)) * (1.f / back);
      } else {
        const v2bf y = __builtin_convertvector(x, v2bf);
        terms[t] = __builtin_bit_cast(uint32_t, y);
        x -= __builtin_convertvector(y, v2f);
      }
    }
  }
};

// Keeps what is computed from x where it is written: not moved out of a loop or a branch that is
// seldom taken, where it would hold registers all along.
__device__ __forceinline__ void rare(int& x) { asm volatile("" : "+v"(x)); }

// the larger / the sum over the four lanes of a row (lanes c, c + 16, c + 32, c + 48)
__device__ __forceinline__ float rows_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
  x = fmaxf(__int_as_float(a[0]), __int_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  return fmaxf(__int_as_float(b[0]), __int_as_float(b[1]));
}
__device__ __forceinline__ float rows_sum(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
  x = __int_as_float(a[0]) + __int_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  return __int_as_float(b[0]) + __int_as_float(b[1]);
}

// exp2(m - base) of a running maximum that may still be -inf
__device__ __forceinline__ float shift_of(float m, float base) { return __builtin_amdgcn_exp2f(m - base); }
__device__ __forceinline__ float finite_base(float m) { return m == -INFINITY ? 0.f : m; }

template <int kType, int DP, int NT>
struct Tile {
  static constexpr bool kHalf = kType != kF32;
  static constexpr int kStep = kHalf ? 32 : 16;   // positions of a wave's step
  static constexpr int kLane = kStep / 4;         // positions of a row that a lane holds
  static constexpr int kBytes = kHalf ? 2 : 4;
  static constexpr int kChunks = kHalf ? DP / 32 : DP / 16;  // K: loads of 16 bytes per key row and lane
  static constexpr int kKeyTiles = kStep / 16;
  static constexpr int W = kHalf ? (DP == 64 ? 4 : 8) : 4;  // V: channels of a load
  static constexpr int H = DP / (16 * W);                    // V: loads per position and lane
  static constexpr int E = H * W;                            // output tiles of 16 channels
  static constexpr int kWords = W * kBytes / 4;              // registers of a V load
  // shared tiles of keys / of values in LDS
  static constexpr int kTileBytes = 16384;
  static constexpr int kTileKeys = kTileBytes / (DP * kBytes);
  static constexpr int kRowChunks = DP * kBytes / 16;
};

typedef __attribute__((address_space(3))) void lds_void;

// ---- the kernel ------------------------------------------------------------------------------

// kShared: the four waves take different rows of the same positions; keys and values come from tiles in
// LDS that the workgroup fills, one ahead of the one in use.
template <int kType, int DP, int NT, CacheView kView, bool kShared>
struct Worker {
  using T = Tile<kType, DP, NT>;
  const CacheAttnParams& p;
  const CachePlan& plan;
  char* lds;  // join_waves: 2 x NT x (E x 4 + 2) x 64 floats; kShared: 2 x (keys, values) tiles
  static constexpr int kWaves = waves_of(kShared);
  int lane, g, c, chunk, wave_r, wave_k, key_waves;
  int group, rows, row_bytes;
  // byte offsets of the lane's channels in a row (kShared: of LDS)
  uint32_t k_channel[T::kChunks], v_channel[T::H];

  // the unit
  int64_t b;
  int hkv, row0;   // row0: first row of the wave
  int len, end;    // committed positions, positions walked
  const char *k_base, *v_base;
  __amdgpu_buffer_rsrc_t k_rsrc, v_rsrc;
  const int32_t* selected;

  // 16-bit terms of a query and of a probability: three of bfloat16 and two of float16 carry float32. Two of
  // bfloat16 (2^-17) and 32 rows a wave took 200 us where 16 rows and three take 305 (4 entries of 23 k, 64
  // tokens), with an error twice that of float32 arithmetic (4.6e-6 against 2.1e-6; three: 9.8e-7): not taken.
  static constexpr int kTerms = !T::kHalf ? 1 : kType == kBF16 ? 3 : 2;
  static constexpr bool kApart = kType == kF16;  // the products of the queries' second terms have sums of their own
  static constexpr float kBack = kApart ? 1.f / 2048 : 1.f;  // and this factor
  uint32_t queries[kTerms][NT][T::kChunks][4];
  // Probabilities are 2^(s + kLift - reference): the reference is a maximum that later ones exceed by up to
  // kSlack, so that outputs are rescaled seldom. float16 ends below 2^16, its steps at 2^-24: 2^15 at most.
  static constexpr float kSlack = kType == kF16 ? 2.f : 8.f, kLift = kType == kF16 ? 13.f : 0.f;
  float factor[NT];  // > 0: scores are factor times what the matrix cores give, to the base 2
  float m[NT], l[NT];  // m: without the factor until the walk ends
  v4f o[NT][T::E];
  v4u k[T::kKeyTiles][T::kChunks];
  uint32_t v[T::kLane][T::H][T::kWords];

  __device__ __forceinline__ Worker(const CacheAttnParams& p, const CachePlan& plan, char* lds)
      : p(p), plan(plan), lds(lds) {
    lane = threadIdx.x & 63;
    g = lane >> 4;
    c = lane & 15;
    // Row r of V^T's tiles is channel chunk(r): r with its two base-4 digits exchanged, so that an output
    // row's four lanes hold neighbouring chunks and store whole lines together.
    chunk = (c & 3) * 4 + (c >> 2);
    const int wave = uniform(threadIdx.x >> 6);
    wave_r = wave % plan.row_waves;
    wave_k = wave / plan.row_waves;
    key_waves = kWaves / plan.row_waves;
    group = plan.group;
    rows = plan.rows;
    row_bytes = static_cast<int>(p.dhead) * T::kBytes;
#pragma unroll
    for (int s = 0; s < T::kChunks; ++s) {
      const int byte = s * 64 + g * 16;
      if constexpr (kShared) k_channel[s] = ((s * 4 + g) ^ c) % T::kRowChunks * 16;
      else k_channel[s] = byte < row_bytes ? byte : kNoChannel;
    }
#pragma unroll
    for (int h = 0; h < T::H; ++h) {
      const int byte = (h * 16 + chunk) * T::W * T::kBytes;
      v_channel[h] = kShared || byte < row_bytes ? byte : kNoChannel;
    }
  }

  // first element of a row's query and output
  __device__ __forceinline__ int64_t row_at(int row) const {
    const int i = row / group, h = row - i * group;
    return ((b * p.tokens + i) * p.heads + hkv * group + h) * p.dhead;
  }

  // the unit's rounds r0 .. r1 - 1: their first keys and values are requested before the queries
  __device__ __forceinline__ void begin(int64_t entry, int unit, int r0, int r1) {
    b = entry;
    hkv = unit / plan.row_groups;
    row0 = (unit % plan.row_groups * plan.row_waves + wave_r) * NT * 16;
    len = uniform(committed(p, b));
    end = uniform(walked(p, b));
    const int64_t head = b * p.heads_kv + hkv;
    const int64_t offset = uniform64(head * p.t_max * row_bytes);
    k_base = static_cast<const char*>(p.k) + offset;
    v_base = static_cast<const char*>(p.v) + offset;
    // the region that loads may reach: the entry's positions, nothing behind them
    const int reach = (kView == CacheView::kTree ? end : len) * row_bytes;
    k_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(k_base), 0, reach, 0x00027000);
    v_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(v_base), 0, reach, 0x00027000);
    if constexpr (kView == CacheView::kBlocks) selected = p.selected + uniform64(head * p.top);
    if constexpr (kShared) {
      __syncthreads();  // nobody reads the tiles of the unit before
      stage((r0 * key_waves + wave_k) * T::kTileKeys, 0);
    } else {
      const int step = step_of(r0, r1);
      load_keys(step);
      load_values(step);
    }
    load_queries();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = -INFINITY;
      l[n] = 0.f;
#pragma unroll
      for (int e = 0; e < T::E; ++e) o[n][e] = v4f{0.f, 0.f, 0.f, 0.f};
    }
  }

  // Rows that are not there repeat row 0, channels behind dhead the first ones (their keys are zeros):
  // nothing of them is stored, and all loads go out together.
  __device__ __forceinline__ void load_queries() {
    const float sign = p.scale < 0.f ? -1.f : 1.f, size = fabsf(p.scale) * kLog2e;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = row0 + n * 16 + c;
      const float* q = p.q + row_at(row < rows ? row : 0);
      constexpr int kFloats = T::kHalf ? 8 : 4;
      float x[T::kChunks][kFloats];
#pragma unroll
      for (int s = 0; s < T::kChunks; ++s) {
        const int d = (s * 4 + g) * kFloats;
#pragma unroll
        for (int i = 0; i < kFloats; i += 4) {
          const v4f y = *reinterpret_cast<const v4f*>(q + (d < p.dhead ? d : 0) + i);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[s][i + j] = y[j];
        }
      }
      float f = size;
      if constexpr (T::kHalf) {
        float most = 1.17549435e-38f;
#pragma unroll
        for (int s = 0; s < T::kChunks; ++s)
#pragma unroll
          for (int j = 0; j < kFloats; ++j) most = fmaxf(most, fabsf(x[s][j]));
        // to [1, 2) by a power of two, which the factor takes back: float16 has no room for less or more
        const uint32_t exponent = __float_as_uint(rows_max(most)) >> 23;  // 1 .. 255
        const uint32_t e = exponent < 253 ? exponent : 253;
        f *= __uint_as_float(e << 23);
        const float down = sign * __uint_as_float((254 - e) << 23);
#pragma unroll
        for (int s = 0; s < T::kChunks; ++s)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t terms[kTerms];
            Mfma<kType>::split(x[s][2 * j] * down, x[s][2 * j + 1] * down, terms, kBack);
#pragma unroll
            for (int t = 0; t < kTerms; ++t) queries[t][n][s][j] = terms[t];
          }
      } else {
#pragma unroll
        for (int s = 0; s < T::kChunks; ++s)
#pragma unroll
          for (int j = 0; j < 4; ++j) queries[0][n][s][j] = __float_as_uint(x[s][j] * sign);
      }
      factor[n] = f < 1.17549435e-38f ? 1.17549435e-38f : f;  // (above zero: -inf times it stays -inf)
    }
  }

  // cache position of walked position t (a multiple of 4); negative: none
  __device__ __forceinline__ int position(int t) const {
    if constexpr (kView != CacheView::kBlocks) return t;
    if (t >= end) return -1;
    // t / block, exact below 2^28 (blocks of 16: 2^32 / 1 does not fit the multiplier)
    const uint32_t u = static_cast<uint32_t>(t) >> 4;
    const int j = static_cast<int>(plan.block_magic == 0u ? u : __umulhi(u, plan.block_magic));
    const int at = selected[j], block = static_cast<int>(p.block);
    return at < 0 ? -1 : at * block + t - j * block;
  }

  __device__ __forceinline__ uint32_t byte_of(int at) const {
    return at < 0 ? kNoRow : static_cast<uint32_t>(at) * static_cast<uint32_t>(row_bytes);
  }

  // step: first walked position; negative: nothing to load (zeros)
  __device__ __forceinline__ void load_keys(int step) {
#pragma unroll
    for (int i = 0; i < T::kKeyTiles; ++i) {
      // row c of tile i is the position that the lanes' elements i * 4 .. i * 4 + 3 stand for
      const int key = T::kHalf ? (c >> 2) * 8 + i * 4 : (c >> 2) * 4;
      const int at = step < 0 ? -1 : position(step + key);
      const uint32_t row = at < 0 ? kNoRow : byte_of(at + (c & 3));
#pragma unroll
      for (int s = 0; s < T::kChunks; ++s)
        k[i][s] = __builtin_amdgcn_raw_buffer_load_b128(k_rsrc, row + k_channel[s], 0, 0);
    }
  }

  __device__ __forceinline__ void load_values(int step) {
    const int at = step < 0 ? -1 : position(step + g * T::kLane);
    const uint32_t row = byte_of(at);
#pragma unroll
    for (int j = 0; j < T::kLane; ++j)
#pragma unroll
      for (int h = 0; h < T::H; ++h) {
        const uint32_t from = row + v_channel[h] + j * row_bytes;
        if constexpr (T::kWords == 4) {
          const v4u x = __builtin_amdgcn_raw_buffer_load_b128(v_rsrc, from, 0, 0);
#pragma unroll
          for (int w = 0; w < 4; ++w) v[j][h][w] = x[w];
        } else {
          const v2u x = __builtin_amdgcn_raw_buffer_load_b64(v_rsrc, from, 0, 0);
          v[j][h][0] = x[0];
          v[j][h][1] = x[1];
        }
      }
  }

  // Tiles of positions t .. t + kTileKeys - 1 on their way into LDS, 16 bytes per lane and request.
  // Loads fill LDS in lane order, so the keys' swizzle - a row's 16-byte units are permuted by the
  // number of the lane that will read it as its A row, which puts the 16 rows that lanes read
  // together on all banks - is made by what a lane asks for.
  __device__ __forceinline__ void stage(int t, int buffer) {
    char* to = lds + (wave_k * 2 + buffer) * 2 * T::kTileBytes;
    int at = lane;
    rare(at);  // (the offsets are made again per tile: kept, they would cost the registers of a row tile)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int piece = wave_r + i * plan.row_waves;  // of 1 KB
      if (piece >= T::kTileBytes / 1024) break;
      const int row = (piece * 64 + at) / T::kRowChunks, unit = at % T::kRowChunks;
      const int reader = T::kHalf ? (row & 3) | (row >> 3 & 3) << 2 : row & 15;
      const int k_byte = (unit ^ (reader % T::kRowChunks)) * 16, v_byte = unit * 16;
      const uint32_t from = static_cast<uint32_t>(t + row) * static_cast<uint32_t>(row_bytes);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(k_rsrc, (lds_void*)(to + piece * 1024), 16,
                                               from + (k_byte < row_bytes ? k_byte : kNoChannel), 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(v_rsrc, (lds_void*)(to + T::kTileBytes + piece * 1024), 16,
                                               from + (v_byte < row_bytes ? v_byte : kNoChannel), 0, 0, 0);
    }
  }

  // the step's keys / values from the tile; `first`: its first row there
  __device__ __forceinline__ void read_keys(const char* tile, int first) {
#pragma unroll
    for (int i = 0; i < T::kKeyTiles; ++i) {
      const int row = first + (T::kHalf ? (c >> 2) * 8 + i * 4 + (c & 3) : c);
#pragma unroll
      for (int s = 0; s < T::kChunks; ++s)
        k[i][s] = *reinterpret_cast<const v4u*>(tile + row * DP * T::kBytes + k_channel[s]);
    }
  }
  __device__ __forceinline__ void read_values(const char* tile, int first) {
#pragma unroll
    for (int j = 0; j < T::kLane; ++j)
#pragma unroll
      for (int h = 0; h < T::H; ++h) {
        const char* from = tile + (first + g * T::kLane + j) * DP * T::kBytes + v_channel[h];
        if constexpr (T::kWords == 4) {
          const v4u x = *reinterpret_cast<const v4u*>(from);
#pragma unroll
          for (int w = 0; w < 4; ++w) v[j][h][w] = x[w];
        } else {
          const v2u x = *reinterpret_cast<const v2u*>(from);
          v[j][h][0] = x[0];
          v[j][h][1] = x[1];
        }
      }
  }

  // bit j: row `row` does not see cache position at + j (at < 0: there is none)
  __device__ __forceinline__ uint32_t hidden_from(int row, int at) const {
    constexpr uint32_t kAll = (1u << T::kLane) - 1;
    if (at < 0) return kAll;
    const uint32_t old = at + T::kLane <= len ? kAll : at < len ? (1u << (len - at)) - 1 : 0u;
    if (kView != CacheView::kTree || row >= rows) return kAll & ~old;
    const int first = at - len, i = row / group, tokens = static_cast<int>(p.tokens);  // drafted token of bit 0
    uint32_t seen = 0u;
    if (!p.mask) {  // tokens up to i
      const int upto = i + 1 - first;
      seen = upto >= T::kLane ? kAll : upto > 0 ? (1u << upto) - 1 : 0u;
    } else {
      const int words = (tokens + 63) / 64, from = first < 0 ? 0 : first, word = from >> 6;
      const uint64_t* mask = p.mask + (b * tokens + i) * words;
      const uint64_t low = mask[word < words ? word : 0], high = mask[word + 1 < words ? word + 1 : 0];
      const int shift = from & 63;
      const uint64_t bits = low >> shift | (shift ? high << (64 - shift) : 0ull);
      seen = first > -T::kLane ? static_cast<uint32_t>(bits << (from - first)) & kAll : 0u;
    }
    const int there = end - at;  // (positions behind the last drafted token)
    if (there < T::kLane) seen &= there > 0 ? (1u << there) - 1 : 0u;
    return kAll & ~(old | seen);
  }

  // x with zeros in the place of what is not finite
  __device__ __forceinline__ static uint32_t finite_part(uint32_t x) {
    if constexpr (kType == kF32) return (x & 0x7f800000u) != 0x7f800000u ? x : 0u;
    constexpr uint32_t e = kType == kF16 ? 0x7c00u : 0x7f80u;
    return ((x & e) != e ? x & 0xffffu : 0u) | ((x >> 16 & e) != e ? x & 0xffff0000u : 0u);
  }

  // first of the W neighbouring channels o[n][h W ..][i] that a lane has of a row
  __device__ __forceinline__ int channel_of(int h, int i) const { return (h * 16 + i * 4 + g) * T::W; }

  // one step over positions step .. step + kStep - 1, whose keys and values are in registers or on
  // their way; `next` is loaded as their registers come free (kShared: they are in `tile`, the
  // keys in registers; `more`: the tile holds another step)
  __device__ __forceinline__ void advance(int step, int next, bool& not_finite, const char* tile = nullptr, int first = 0,
                                          bool more = false) {
    // (a wave in its products goes first, the SIMD's other one fills the gaps: 1 % of a long tree)
    if constexpr (kShared) __builtin_amdgcn_s_setprio(1);
    float s[NT][T::kLane];
    {
      v4f acc[NT][T::kKeyTiles], acc_low[NT][T::kKeyTiles];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < T::kKeyTiles; ++i) acc[n][i] = acc_low[n][i] = v4f{0.f, 0.f, 0.f, 0.f};
      // (independent products follow each other: a product waits for the one that it adds to)
#pragma unroll
      for (int x = 0; x < T::kChunks; ++x)
        if constexpr (T::kHalf) {
#pragma unroll
          for (int t = 0; t < kTerms; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < T::kKeyTiles; ++i) {
                const v4u q = {queries[t][n][x][0], queries[t][n][x][1], queries[t][n][x][2], queries[t][n][x][3]};
                v4f& to = kApart && t == 1 ? acc_low[n][i] : acc[n][i];
                to = Mfma<kType>::mul(k[i][x], q, to);
              }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n)
              acc[n][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[0][x][j]),
                                                               __uint_as_float(queries[0][n][x][j]), acc[n][0], 0, 0, 0);
        }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < T::kLane; ++j) {
          s[n][j] = acc[n][j / 4][j % 4];
          if constexpr (kApart) s[n][j] = fmaf(acc_low[n][j / 4][j % 4], kBack, s[n][j]);
        }
    }
    if constexpr (kShared) {
      __builtin_amdgcn_s_setprio(0);
      read_values(tile + T::kTileBytes, first);
      if (more) read_keys(tile, first + T::kStep);
    } else {
      load_keys(next);
    }

    const int at = position(step + g * T::kLane);
    if (kView == CacheView::kBlocks ? !__all(at >= 0 && at + T::kLane <= len) : step + T::kStep > len) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        int row = row0 + n * 16 + c;
        rare(row);
        const uint32_t hidden = hidden_from(row, at);
#pragma unroll
        for (int j = 0; j < T::kLane; ++j)
          if (hidden >> j & 1) s[n][j] = -INFINITY;
      }
      if constexpr (kView == CacheView::kTree) {
        // a drafted position's NaN and infinite values would reach rows that do not see it as 0 x inf:
        // they wait for add_not_finite(), and with them those of the step's committed positions
#pragma unroll
        for (int j = 0; j < T::kLane; ++j)
#pragma unroll
          for (int h = 0; h < T::H; ++h)
#pragma unroll
            for (int w = 0; w < T::kWords; ++w) {
              const uint32_t x = finite_part(v[j][h][w]);
              not_finite |= x != v[j][h][w];
              v[j][h][w] = x;
            }
      }
    }
    if (kView == CacheView::kDense && p.weights) {
      // the scores (times log2 e) wait for the row's statistics; the rows' pitch is a multiple of a step
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int row = row0 + n * 16 + c;
        if (row < rows) {
          float* to = static_cast<float*>(p.scratch) + plan.scores +
                      ((b * p.heads_kv + hkv) * rows + row) * plan.score_pitch + step + g * T::kLane;
#pragma unroll
          for (int j = 0; j < T::kLane; j += 4)
            *reinterpret_cast<v4f*>(to + j) =
                v4f{s[n][j], s[n][j + 1], s[n][j + 2], s[n][j + 3]} * factor[n];
        }
      }
    }

    // a maximum that grew by less than kSlack stays the reference
    float most[NT];
    bool grown = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      most[n] = s[n][0];
#pragma unroll
      for (int j = 1; j < T::kLane; ++j) most[n] = fmaxf(most[n], s[n][j]);
      most[n] = fmaxf(m[n], rows_max(most[n]));
      grown |= (most[n] - m[n]) * factor[n] > kSlack;
    }
    if (__any(grown)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float keep = __builtin_amdgcn_exp2f((m[n] - finite_base(most[n])) * factor[n]);
        l[n] *= keep;
#pragma unroll
        for (int e = 0; e < T::E; ++e) o[n][e] *= keep;
        m[n] = most[n];
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float base = finite_base(m[n]) * factor[n] - kLift;
#pragma unroll
      for (int j = 0; j < T::kLane; ++j) {
        s[n][j] = __builtin_amdgcn_exp2f(fmaf(s[n][j], factor[n], -base));
        l[n] += s[n][j];
      }
    }

    if constexpr (kShared) __builtin_amdgcn_s_setprio(1);
    add_values(s);
    if constexpr (kShared) __builtin_amdgcn_s_setprio(0);
    if constexpr (!kShared) load_values(next);
  }

  __device__ __forceinline__ void add_values(const float (&s)[NT][T::kLane]) {
    if constexpr (T::kHalf) {
      v4u probability[kTerms][NT];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t terms[kTerms];
          Mfma<kType>::split(s[n][2 * j], s[n][2 * j + 1], terms);
#pragma unroll
          for (int t = 0; t < kTerms; ++t) probability[t][n][j] = terms[t];
        }
#pragma unroll
      for (int h = 0; h < T::H; ++h)
#pragma unroll
        for (int e = 0; e < T::W; ++e) {
          v4u a;
#pragma unroll
          for (int w = 0; w < 4; ++w)
            a[w] = __builtin_amdgcn_perm(v[2 * w + 1][h][e >> 1], v[2 * w][h][e >> 1],
                                         e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int t = 0; t < kTerms; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n)
              o[n][h * T::W + e] = Mfma<kType>::mul(a, probability[t][n], o[n][h * T::W + e]);
        }
    } else {
#pragma unroll
      for (int h = 0; h < T::H; ++h)
#pragma unroll
        for (int e = 0; e < T::W; ++e)
#pragma unroll
          for (int j = 0; j < T::kLane; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n)
              o[n][h * T::W + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[j][h][e]), s[n][j],
                                                                        o[n][h * T::W + e], 0, 0, 0);
    }
  }

  // The NaN and infinite values that the walk took out, to the rows that see them: of the drafted positions and
  // of the committed ones in the step that those begin in. (A probability is above zero, so its product with
  // them is what they are.)
  __device__ void add_not_finite(int r0, int r1) {
    constexpr int kStretch = kShared ? T::kTileKeys : T::kStep;  // of a wave in a round
    const int first = len / T::kStep * T::kStep;
#pragma unroll 1
    for (int r = r0; r < r1; ++r) {
      const int t = (r << plan.round_shift) + wave_k * kStretch, to = t + kStretch < end ? t + kStretch : end;
#pragma unroll 1
      for (int at = t < first ? first : t; at < to; ++at) {
        bool seen[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) seen[n] = !(hidden_from(row0 + n * 16 + c, at) & 1);
#pragma unroll
        for (int h = 0; h < T::H; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // channels behind dhead read as zeros or as other channels: they are not stored
            const uint32_t byte = byte_of(at) + channel_of(h, i) * T::kBytes;
            v2u y[T::kWords / 2];
#pragma unroll
            for (int w = 0; w < T::kWords / 2; ++w)
              y[w] = __builtin_amdgcn_raw_buffer_load_b64(v_rsrc, byte + 8 * w, 0, 0);
#pragma unroll
            for (int e = 0; e < T::W; ++e) {
              float value;
              if constexpr (kType == kF32) {
                value = __uint_as_float(y[e >> 1][e & 1]);
              } else {
                const uint32_t bits = e & 1 ? y[e >> 2][e >> 1 & 1] >> 16 : y[e >> 2][e >> 1 & 1] & 0xffffu;
                if constexpr (kType == kF16) value = __builtin_bit_cast(v2h, bits)[0];
                else value = __uint_as_float(bits << 16);
              }
              const bool bad = !(fabsf(value) < INFINITY);
#pragma unroll
              for (int n = 0; n < NT; ++n)
                if (bad && seen[n]) o[n][h * T::W + e][i] += value;
            }
          }
      }
    }
  }

  // first position of the wave's step in round r, -1 if it has none
  __device__ __forceinline__ int step_of(int r, int r1) const {
    const int t = (r << plan.round_shift) + wave_k * T::kStep;
    return r < r1 && t < end ? t : -1;
  }

  __device__ __forceinline__ void walk(int r0, int r1) {
    bool not_finite = false;
    if constexpr (kShared) {
#pragma unroll 1
      for (int r = r0; r < r1; ++r) {
        // this tile has arrived and the other one is read: no later request may still be under way here
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\ns_barrier" ::: "memory");
        const int t = (r * key_waves + wave_k) * T::kTileKeys, buffer = (r - r0) & 1;
        const char* tile = lds + (wave_k * 2 + buffer) * 2 * T::kTileBytes;
        read_keys(tile, 0);
        if (r + 1 < r1) stage(t + key_waves * T::kTileKeys, buffer ^ 1);
#pragma unroll 1
        for (int i = 0; i < T::kTileKeys && t + i < end; i += T::kStep)
          advance(t + i, 0, not_finite, tile, i, i + T::kStep < T::kTileKeys);
      }
    } else {
      int step = step_of(r0, r1);
#pragma unroll 1
      for (int r = r0; step >= 0; ++r) {
        const int next = step_of(r + 1, r1);
        advance(step, next, not_finite);
        step = next;
      }
    }
    if (kView == CacheView::kTree && __any(not_finite)) add_not_finite(r0, r1);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      l[n] = rows_sum(l[n]);
      if (m[n] != -INFINITY) m[n] = m[n] * factor[n] - kLift;
    }
  }

  // waves that took other positions of the same rows hand theirs to the first
  __device__ __forceinline__ void join_waves() {
    constexpr int kFloats = NT * (T::E * 4 + 2) * 64;
    for (int half = key_waves / 2; half >= 1; half /= 2) {
      float* mine = reinterpret_cast<float*>(lds) + (wave_r * half + wave_k % half) * kFloats;
      __syncthreads();
      if (wave_k >= half && wave_k < 2 * half) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float* to = mine + n * (T::E * 4 + 2) * 64;
#pragma unroll
          for (int e = 0; e < T::E; ++e) *reinterpret_cast<v4f*>(to + (e * 64 + lane) * 4) = o[n][e];
          to[T::E * 256 + lane] = m[n];
          to[T::E * 256 + 64 + lane] = l[n];
        }
      }
      __syncthreads();
      if (wave_k < half) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float* from = mine + n * (T::E * 4 + 2) * 64;
          const float m1 = from[T::E * 256 + lane], l1 = from[T::E * 256 + 64 + lane];
          const float most = fmaxf(m[n], m1), base = finite_base(most);
          const float a = shift_of(m[n], base), d = shift_of(m1, base);
          l[n] = l[n] * a + l1 * d;
          m[n] = most;
#pragma unroll
          for (int e = 0; e < T::E; ++e) {
            const v4f x = *reinterpret_cast<const v4f*>(from + (e * 64 + lane) * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][e][i] = o[n][e][i] * a + x[i] * d;
          }
        }
      }
    }
  }

  // the unit's outputs, or a part's (m, l, o)
  __device__ __forceinline__ void finish(bool complete, int64_t part) {
    if (key_waves > 1) join_waves();
    if (wave_k != 0) return;
    float* scratch = static_cast<float*>(p.scratch);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = row0 + n * 16 + c;
      if (row >= rows) continue;
      float* to;
      float by = 1.f;
      if (complete) {
        to = p.out + row_at(row);
        by = l[n] == 0.f ? 0.f : 1.f / l[n];
        if (kView == CacheView::kDense && p.weights && g == 0)
          *reinterpret_cast<v2f*>(scratch + plan.stats + ((b * p.heads_kv + hkv) * rows + row) * 2) =
              v2f{finite_base(m[n]), by};
      } else {
        const int64_t slot = part * plan.unit_rows + row - row0 + wave_r * NT * 16;
        to = scratch + plan.parts_o + slot * p.dhead;
        if (g == 0) *reinterpret_cast<v2f*>(scratch + plan.parts_ml + slot * 2) = v2f{m[n], l[n]};
      }
#pragma unroll
      for (int h = 0; h < T::H; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int w = 0; w < T::W; w += 4) {
            const int d = (h * 16 + i * 4 + g) * T::W + w;
            v4f x;
#pragma unroll
            for (int y = 0; y < 4; ++y) x[y] = l[n] == 0.f ? 0.f : o[n][h * T::W + w + y][i] * by;
            if (d < p.dhead) *reinterpret_cast<v4f*>(to + d) = x;
          }
    }
  }
};

constexpr int waves_per_simd(int dp) { return dp == 256 ? 1 : 2; }

template <int kType, int DP, int NT, CacheView kView, bool kShared>
__global__ __launch_bounds__(64 * waves_of(kShared), waves_per_simd(DP))
void cache_attention_kernel(CacheAttnParams p, CachePlan plan) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  Worker<kType, DP, NT, kView, kShared> worker(p, plan, lds);
  const uint32_t units = static_cast<uint32_t>(p.heads_kv) * plan.row_groups;
  Line line{0, 0, 1, 0};
  int64_t b = 0;
  Stretch stretch{0, 0, 0, 0};
  if (plan.whole) {
    b = blockIdx.x / units;
    stretch = Stretch::whole(blockIdx.x % units, uniform(rounds_of(p, plan, b)));
  } else {
    const int lane = threadIdx.x & 63;
    auto rounds = [&](int64_t entry) {
      return entry < p.batch ? static_cast<uint32_t>(rounds_of(p, plan, entry)) * units : 0u;
    };
    uint32_t upto = 0, mine = 0;
    for (int64_t b0 = 0; b0 < p.batch; b0 += 64) {
      mine = rounds(b0 + lane);
      upto = wave_scan(mine);
      line.total += __builtin_amdgcn_readlane(upto, 63);
    }
    const uint32_t groups = line.total / plan.min_rounds;
    line.groups = groups < 1 ? 1 : (groups > static_cast<uint32_t>(plan.grid) ? plan.grid : groups);
    line.each = line.total / line.groups;
    line.longer = line.total - line.each * line.groups;
    if (blockIdx.x >= line.groups) return;
    stretch.x = line.start(blockIdx.x);
    stretch.x1 = line.start(blockIdx.x + 1);
    // the entry that the stretch begins in
    uint32_t before = 0;
    for (;; b += 64) {
      if (p.batch > 64) {
        mine = rounds(b + lane);
        upto = wave_scan(mine);
      }
      const uint64_t behind = __ballot(before + upto > stretch.x);
      if (behind) {
        const int at = __builtin_ctzll(behind);
        before += __builtin_amdgcn_readlane(upto - mine, at);
        b += at;
        break;
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
    stretch.before = before;
  }
  const uint32_t x0 = stretch.x;
#pragma unroll 1
  while (stretch.x < stretch.x1) {
    const uint32_t n = uniform(rounds_of(p, plan, b));
    const Stretch::Part part = stretch.part(n);
    worker.begin(b, part.unit, part.r0, part.r1);
    worker.walk(part.r0, part.r1);
    // a part that begins the workgroup's stretch is its first, any other its last
    const int slot = blockIdx.x * 2 + (stretch.x == x0 ? 0 : 1);
    if (!plan.whole && part.r0 == 0 && threadIdx.x == 0) {
      const int count = static_cast<int>(line.holder(stretch.x + n - 1) - blockIdx.x) + 1;
      reinterpret_cast<int2*>(static_cast<float*>(p.scratch) + plan.records)[b * units + part.unit] = int2{slot, count};
    }
    worker.finish(part.r0 == 0 && part.r1 == n, slot);
    if (stretch.pass(part, n, units)) ++b;
  }
}

// Where the parts of a unit are: the first in its slot, the others in the first slots of the
// workgroups that follow.
struct Parts {
  int first, count;
  __device__ __forceinline__ Parts(const CacheAttnParams& p, const CachePlan& plan, int64_t unit) {
    const int2 record =
        reinterpret_cast<const int2*>(static_cast<const float*>(p.scratch) + plan.records)[unit];
    first = record.x;
    count = record.y;
  }
  __device__ __forceinline__ int64_t row(const CachePlan& plan, int i, int local) const {
    return static_cast<int64_t>(i == 0 ? first : ((first >> 1) + i) * 2) * plan.unit_rows + local;
  }
};

// out = sum exp(m_i - M) o_i / sum exp(m_i - M) l_i of the rows of units with several parts: 32 lanes per
// row (64 for heads beyond 128 channels) with four channels each. One pass over the parts, eight requested
// together, their maximum kept as it grows: bound by the latency of two dependent reads (the record, the
// parts), so that what counts is how many rows are on the chip at once.
__device__ void join_rows(const CacheAttnParams& p, const CachePlan& plan) {
  constexpr int kAhead = 8;
  const int lanes = p.dhead > 128 ? 64 : 32, lane = threadIdx.x & (lanes - 1);
  const int group = plan.group, rows = plan.rows, dhead = static_cast<int>(p.dhead);
  const int64_t at = blockIdx.x * static_cast<int64_t>(kThreads / lanes) + threadIdx.x / lanes;
  const int64_t unit = at / plan.unit_rows, head = unit / plan.row_groups;
  if (head >= p.batch * p.heads_kv) return;
  const int local = static_cast<int>(at - unit * plan.unit_rows);
  const int row = static_cast<int>(unit - head * plan.row_groups) * plan.unit_rows + local;
  if (row >= rows) return;
  const Parts parts(p, plan, unit);
  if (parts.count == 1) return;
  const float* scratch = static_cast<const float*>(p.scratch);
  const v2f* ml = reinterpret_cast<const v2f*>(scratch + plan.parts_ml);
  const int channel = lane * 4 < dhead ? lane * 4 : 0;
  float most = -INFINITY, total = 0.f;
  v4f o = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < parts.count; i0 += kAhead) {
    v2f part[kAhead];
    v4f x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t from = parts.row(plan, i0 + u < parts.count ? i0 + u : i0, local);
      part[u] = ml[from];
      x[u] = *reinterpret_cast<const v4f*>(scratch + plan.parts_o + from * dhead + channel);
    }
    float higher = most;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) higher = fmaxf(higher, part[u][0]);
    const float base = finite_base(higher), keep = shift_of(most, base);
    total *= keep;
    o *= keep;
    most = higher;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i0 + u >= parts.count) break;
      const float weight = shift_of(part[u][0], base);
      total += weight * part[u][1];
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] += weight * x[u][c];
    }
  }
  const float by = total == 0.f ? 0.f : 1.f / total;
  const int64_t b = head / p.heads_kv, hkv = head - b * p.heads_kv;
  const int i = row / group;
  float* to = p.out + ((b * p.tokens + i) * p.heads + hkv * group + row - i * group) * dhead;
  if (lane * 4 < dhead) *reinterpret_cast<v4f*>(to + lane * 4) = total == 0.f ? v4f{0.f, 0.f, 0.f, 0.f} : o * by;
}

// weights[b, hkv, t] += sum over the group's heads of exp(s_t - m) / l
constexpr int kWeightSteps = 4;  // positions of a thread
__device__ void add_weights(const CacheAttnParams& p, const CachePlan& plan, int64_t index) {
  __shared__ v2f stats_s[1024];
  const int64_t head = index / plan.weight_tiles;
  const int t0 = static_cast<int>(index - head * plan.weight_tiles) * kThreads * kWeightSteps + threadIdx.x;
  const int group = plan.group;
  const int len = committed(p, head / p.heads_kv);
  if (t0 - static_cast<int>(threadIdx.x) >= len) return;
  const float* scratch = static_cast<const float*>(p.scratch);
  const float* scores = scratch + plan.scores + head * group * plan.score_pitch;
  float* weights = p.weights + head * p.t_max;
  // the first heads' scores and the old weights are requested before the statistics are looked for
  constexpr int kAhead = 4;
  int t[kWeightSteps];
  float sum[kWeightSteps], old[kWeightSteps], ahead[kAhead][kWeightSteps];
#pragma unroll
  for (int u = 0; u < kWeightSteps; ++u) {
    t[u] = t0 + u * kThreads < len ? t0 + u * kThreads : 0;
    sum[u] = 0.f;
    old[u] = weights[t[u]];
#pragma unroll
    for (int r = 0; r < kAhead; ++r) ahead[r][u] = scores[(r < group ? r : 0) * plan.score_pitch + t[u]];
  }
  for (int r = threadIdx.x; r < group; r += kThreads) {
    v2f stats = reinterpret_cast<const v2f*>(scratch + plan.stats)[head * group + r];
    if (!plan.whole) {
      const Parts parts(p, plan, head * plan.row_groups + r / plan.unit_rows);
      if (parts.count > 1) {
        const int local = r % plan.unit_rows;
        const v2f* ml = reinterpret_cast<const v2f*>(scratch + plan.parts_ml);
        float most = -INFINITY, total = 0.f;
#pragma unroll 4
        for (int i = 0; i < parts.count; ++i) most = fmaxf(most, ml[parts.row(plan, i, local)][0]);
        const float base = finite_base(most);
#pragma unroll 4
        for (int i = 0; i < parts.count; ++i) {
          const v2f part = ml[parts.row(plan, i, local)];
          total += part[1] * shift_of(part[0], base);
        }
        stats = v2f{base, total == 0.f ? 0.f : 1.f / total};
      }
    }
    stats_s[r] = stats;
  }
  __syncthreads();
  auto add = [&](int r, const float (&score)[kWeightSteps]) {
    const v2f stats = stats_s[r];
#pragma unroll
    for (int u = 0; u < kWeightSteps; ++u) sum[u] += __builtin_amdgcn_exp2f(score[u] - stats[0]) * stats[1];
  };
#pragma unroll
  for (int r = 0; r < kAhead; ++r)
    if (r < group) add(r, ahead[r]);
#pragma unroll 2
  for (int r = kAhead; r < group; ++r) {
    float score[kWeightSteps];
#pragma unroll
    for (int u = 0; u < kWeightSteps; ++u) score[u] = scores[r * plan.score_pitch + t[u]];
    add(r, score);
  }
#pragma unroll
  for (int u = 0; u < kWeightSteps; ++u)
    if (t0 + u * kThreads < len) weights[t[u]] = old[u] + sum[u];
}

__global__ __launch_bounds__(kThreads) void finish_kernel(CacheAttnParams p, CachePlan plan) {
  if (blockIdx.x < static_cast<unsigned>(plan.join_groups)) join_rows(p, plan);
  else add_weights(p, plan, blockIdx.x - plan.join_groups);
}

// ---- the host's side -------------------------------------------------------------------------

int padded_head(int64_t dhead) { return dhead <= 64 ? 64 : (dhead <= 128 ? 128 : 256); }

CachePlan make_plan(const CacheAttnParams& p) {
  CachePlan plan;
  const int64_t rows = p.tokens * (p.heads / p.heads_kv);
  const int dp = padded_head(p.dhead), element = p.kv_dtype == kF32 ? 4 : 2;
  // Few rows: every wave loads for itself. From 33 on, heads of up to 128: tiles in LDS, which four or
  // eight waves with rows of their own share. bfloat16, heads of 128, 16 entries of 1.1 k on average, four rows a
  // token: 8 tokens 33.4 us apart, 38.3 shared; 16 tokens 48.8 and 40.3.
  plan.shared = p.view == CacheView::kTree && rows > 32 && dp <= 128;
  const int waves = waves_of(plan.shared);
  // 32 rows a wave read the tiles half as often, 16 have a shorter way in and out: the former where there are
  // rows for eight such waves and enough positions times rows. float16, heads of 128, 64 tokens, us by 16 / 32:
  // 4 entries of 500 32 / 46, 4 of 2000 50 / 64, 4 of 8000 103 / 107, 16 of 8000 340 / 298; float32 51 / 69,
  // 104 / 113, 301 / 296, 1135 / 1045. Three bfloat16 terms of 32 rows of 128 channels are more than the
  // registers: 16 of 8000 take 414 us by 16, 518 by 32.
  const bool long_tree = rows > 128 && rows * p.t_max * p.heads_kv * p.batch >= 60000000;
  plan.tiles = plan.shared && long_tree && (p.kv_dtype != kBF16 || dp <= 64) ? 2 : 1;
  plan.row_waves = plan.shared ? 4 : 1;
  while (plan.row_waves < waves && plan.row_waves * 16 * plan.tiles < rows) plan.row_waves *= 2;
  plan.unit_rows = 16 * plan.tiles * plan.row_waves;
  plan.row_groups = static_cast<int>((rows + plan.unit_rows - 1) / plan.unit_rows);
  const int round_keys =
      (plan.shared ? 16384 / (dp * element) : element == 4 ? 16 : 32) * (waves / plan.row_waves);
  plan.round_shift = __builtin_ctz(round_keys);
  plan.group = static_cast<int>(p.heads / p.heads_kv);
  plan.rows = static_cast<int>(rows);
  plan.block_magic =
      p.view == CacheView::kBlocks ? static_cast<uint32_t>(((1ull << 32) + p.block / 16 - 1) / (p.block / 16)) : 0u;
  plan.grid = plan.shared ? 256 : 512;
  // 128 positions at least where a part is many rows
  plan.min_rounds = plan.shared ? std::max(1, 128 / round_keys) : 1;
  const int64_t walked = p.view == CacheView::kBlocks ? p.top * p.block : p.t_max;
  const int64_t units = p.batch * p.heads_kv * plan.row_groups;
  // A workgroup alone with its unit writes no parts, and a tree's call is then one launch; the line keeps the
  // workgroups even where units are few or long. Rounds up to which the former was the faster, for less than
  // 192 units, less than 512 and more; heads of 128, us, line / alone, units and positions (bfloat16):
  // tree 4 tokens, 64 x 512: 14.1 / 13.4, 192 x 1020: 30.0 / 22.0, 512 x 2044: 70.8 / 63.4; 24 tokens,
  // 64 x 1020: 31 / 48, 512 x 1532: 146 / 120; blocks 64 x 1024: 29 / 41, 512 x 1024: 76 / 74;
  // accumulate 192 x 250: 15.2 / 13.3, 512 x 1000: 39 / 36. (Entries without a figure of their own lie between
  // those of their row.) Lengths are not known here, t_max is: a cache with much more room than its entries fill
  // gets the line.
  static constexpr int kAlone[3][3] = {{2, 8, 16}, {2, 4, 32}, {8, 16, 32}};
  const int many = units >= 512 ? 2 : units >= 192 ? 1 : 0;
  const int view = p.view == CacheView::kDense ? 0 : p.view == CacheView::kBlocks ? 1 : 2;
  plan.whole = walked <= round_keys * kAlone[view][many] || units >= 2048 ||
               line_is_too_long(units, (walked + round_keys - 1) / round_keys);
  // scratch
  auto up = [](int64_t floats) { return (floats + 63) / 64 * 64; };
  const int64_t parts = plan.whole ? 0 : 2ll * plan.grid * plan.unit_rows;
  plan.records = 0;
  plan.parts_ml = plan.whole ? 0 : up(units * 2);
  plan.parts_o = plan.parts_ml + up(parts * 2);
  plan.stats = plan.parts_o + up(parts * p.dhead);
  plan.scores = plan.stats;
  plan.total = plan.stats;
  plan.score_pitch = 0;
  if (p.view == CacheView::kDense) {
    plan.score_pitch = up(p.t_max);
    plan.scores = plan.stats + up(p.batch * p.heads * 2);
    plan.total = plan.scores + p.batch * p.heads * plan.score_pitch;
  }
  const int join_rows = kThreads / (p.dhead > 128 ? 64 : 32);
  plan.join_groups = plan.whole ? 0 : static_cast<int>((units * plan.unit_rows + join_rows - 1) / join_rows);
  plan.weight_tiles =
      p.weights ? static_cast<int>((p.t_max + kThreads * kWeightSteps - 1) / (kThreads * kWeightSteps)) : 0;
  return plan;
}

template <int kType, int DP, int NT, CacheView kView, bool kShared = false>
void launch_tiles(const CacheAttnParams& p, const CachePlan& plan, hipStream_t stream) {
  using T = Tile<kType, DP, NT>;
  constexpr int waves = waves_of(kShared);
  const int64_t units = p.batch * p.heads_kv * plan.row_groups;
  const int key_waves = waves / plan.row_waves;
  const size_t join = key_waves > 1 ? sizeof(float) * (waves / 2) * NT * (T::E * 4 + 2) * 64 : 0;
  const size_t lds = kShared ? std::max<size_t>(join, 4 * T::kTileBytes * key_waves) : join;
  const auto kernel = cache_attention_kernel<kType, DP, NT, kView, kShared>;
  if constexpr (kShared) {  // more than 64 KiB of dynamic LDS has to be opted into once per device
    static std::atomic<bool> configured[64];
    int device = 0;
    CT2X_HIP_CHECK(hipGetDevice(&device));
    if (!configured[device & 63].load(std::memory_order_acquire)) {
      CT2X_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                         hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
      configured[device & 63].store(true, std::memory_order_release);
    }
  }
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(plan.whole ? units : plan.grid)), dim3(64 * waves), lds, stream,
                     p, plan);
}

template <int kType, int DP>
void launch_head(const CacheAttnParams& p, const CachePlan& plan, hipStream_t stream) {
  if (p.view == CacheView::kDense) return launch_tiles<kType, DP, 1, CacheView::kDense>(p, plan, stream);
  if (p.view == CacheView::kBlocks) return launch_tiles<kType, DP, 1, CacheView::kBlocks>(p, plan, stream);
  if constexpr (DP < 256) {
    if constexpr (kType != kBF16 || DP <= 64)
      if (plan.tiles == 2) return launch_tiles<kType, DP, 2, CacheView::kTree, true>(p, plan, stream);
    if (plan.shared) return launch_tiles<kType, DP, 1, CacheView::kTree, true>(p, plan, stream);
  }
  launch_tiles<kType, DP, 1, CacheView::kTree>(p, plan, stream);
}

template <int kType>
void launch_typed(const CacheAttnParams& p, const CachePlan& plan, hipStream_t stream) {
  const int dp = padded_head(p.dhead);
  if (dp == 64) launch_head<kType, 64>(p, plan, stream);
  else if (dp == 128) launch_head<kType, 128>(p, plan, stream);
  else launch_head<kType, 256>(p, plan, stream);
}

}  // namespace

int64_t cache_attention_scratch_bytes(const CacheAttnParams& p) {
  // the types differ in their rounds and tiles: as much as the largest takes
  int64_t most = 0;
  CacheAttnParams other = p;
  for (int type : {kF32, kF16, kBF16}) {
    other.kv_dtype = type;
    most = std::max(most, make_plan(other).total);
  }
  return most * 4;
}

void launch_cache_attention(const CacheAttnParams& p, hipStream_t stream) {
  const CachePlan plan = make_plan(p);
  if (p.kv_dtype == kF32) launch_typed<kF32>(p, plan, stream);
  else if (p.kv_dtype == kF16) launch_typed<kF16>(p, plan, stream);
  else launch_typed<kBF16>(p, plan, stream);
  const int64_t finish = plan.join_groups + plan.weight_tiles * p.batch * p.heads_kv;
  if (finish)
    hipLaunchKernelGGL(finish_kernel, dim3(static_cast<unsigned>(finish)), dim3(kThreads), 0, stream, p, plan);
}

}  // namespace ct2x
