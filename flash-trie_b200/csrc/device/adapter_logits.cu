// The vocabulary projection of many requests at once, each request with a
// low-rank adapter of its own beside the shared weight:
//
//   u[t, r] = s_a sum_d h[t, d] A_a[r, d]
//   y[t, v] = sum_d h[t, d] W[v, d] + sum_r u[t, r] B_a[v, r]
//
// The logits are made on the tensor cores with the vocabulary as the row side
// of the product: a tile is 128 vocabulary entries by up to 256 tokens, so few
// tokens cost a narrow product, not padded rows, and a thread of the epilogue
// holds one vocabulary entry for the tokens of its tile, whose stores run
// along the vocabulary.  u is made before, in 32 bits.
//
// The low-rank part has two forms.  "Sorted": the tokens are put in order of
// their adapters, each adapter's at a multiple of 16 columns, and every group
// adds its u B^T to its own columns with further tensor products; u goes in as
// 16-bit parts: a bf16 part leaves at most 2^-8 of its power of two, a value of
// the power 2^-9 or below for the next, so that two parts lose 2^-17 and the
// three for f32 logits 2^-26; two f16 parts lose 2^-23, or 2^-25 absolute.  A
// token whose largest value is beyond the type's range, or so small that 2^-25
// would show, takes no part in these products: its values stay in 32 bits and
// the epilogue adds its low-rank part, slowly but the same as "direct" does.  No
// column is shared, so an adapter with infinities reaches no other one's
// requests.  "Direct": the tokens stay as they are, a kernel of its own makes
// the low-rank part in 32 bits and the epilogue adds it, for batches whose
// groups are so small that padding them would cost more.
#include <algorithm>
#include <string>

#include "../engine.hpp"
#include "cuda_util.hpp"
#include "head_ops.hpp"
#include "row_stream.cuh"
#include "sm100.cuh"
#include "tbs_kernel.cuh"

namespace ftb {
namespace {

constexpr uint32_t kMaxRank = 256;
constexpr uint32_t kMaxAdapters = 65536;

constexpr int kTileV = 128;   // vocabulary entries of one product's rows; a tile has one or two such halves
constexpr int kTileD = 64;    // inner dimension of a stage: 128-byte rows
constexpr int kMaxTileT = 256;
constexpr int kMaxStages = 12;
constexpr uint32_t kMaxParts = 3;
constexpr int kEpilogue = 512;            // threads of warps 0-15; with half of them the stores take half as long again
constexpr int kThreads = kEpilogue + 64;  // warp 16: loads, warp 17: products
constexpr uint32_t kLoadWarp = kEpilogue / 32, kProductWarp = kLoadWarp + 1;
constexpr uint32_t kMaxSortRequests = 8192;
static_assert(kEpilogue >= kMaxTileT, "a thread of the epilogue looks up each column");

template <typename T>
__device__ __forceinline__ void unpack8(uint4 q, float (&v)[8]) {
  unpack(q, v, (const T *)nullptr);
}

// A group has at least 16 columns, so that a tile has 16 groups at most.
constexpr uint32_t kTileGroups = kMaxTileT / 16 + 1;

__device__ __forceinline__ uint32_t pack_pair(float x, float y, const __nv_bfloat16 *) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_pair(float x, float y, const __half *) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_pair(float, float, const float *) { return 0; }  // not reached

// Stores under a predicate: as branches, one after the other, they take twice as
// long (690 and 340 cycles for 16 columns).
__device__ __forceinline__ void store_if(bool yes, uint32_t *to, uint32_t x) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %0, 0;\n\t@q st.global.b32 [%1], %2;\n\t}" ::"r"((uint32_t)yes), "l"(to),
               "r"(x));
}
__device__ __forceinline__ void store_if(bool yes, float *to, float x) {
  store_if(yes, reinterpret_cast<uint32_t *>(to), __float_as_uint(x));
}
template <typename T>
__device__ __forceinline__ void store_if(bool yes, T *to, float x) {
  T h;
  from_f32(x, h);
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %0, 0;\n\t@q st.global.b16 [%1], %2;\n\t}" ::"r"((uint32_t)yes), "l"(to),
               "h"(*reinterpret_cast<const uint16_t *>(&h)));
}

struct Group {
  int32_t adapter;  // -1: none
  uint32_t col0, col1, pad;
};

// Where the sorted form keeps its order (all in the workspace).
struct Sorted {
  uint32_t *head;        // [0] groups, [1] columns
  Group *groups;
  uint32_t *tile_first;  // first group of each tile of tokens
  Group *tile_groups;    // [tiles][kTileGroups]: the groups with columns in a tile, then one that begins nowhere
  uint32_t *req_col;     // first column of each request
  // Token of a column, with kWide if its low-rank values are in `wide` alone;
  // -1 padding; -2 - token: of a request whose adapter does not exist.
  int32_t *col_token;
  float *wide;           // [tokens][rank], written for tokens with kWide
  void *hidden;          // [columns][dim]
  uint8_t *u;            // [rank / width][columns / 8][parts][8 columns][width], swizzled as in shared memory
  uint32_t columns;      // upper bound, a multiple of 16
  uint32_t parts;
  uint32_t width;        // low-rank rows that a product's operands hold side by side: 16, 32 or 64
  // One request: its tokens are in order as they are. There are no tables and
  // no moved tokens; only u and, where the request has an adapter, its tokens'
  // entries of col_token are written.
  bool single;
};

constexpr int32_t kWide = 1 << 24;  // above any token's number
constexpr uint64_t kMaxTokens = 0x3FFFFF;
static_assert(kMaxTokens < kWide, "a token's number and the flag share a word");

// Whether the 16-bit parts hold the low-rank values of a token, by the largest
// magnitude among them.  f16 ends at 65504, and below 2^-8 the 2^-25 that its
// two parts leave is more than 2^-17 of the largest.  bf16 has f32's range;
// there the parts' own range ends.
__device__ __forceinline__ bool parts_hold(float most, const __half *) {
  return most == 0.0f || (most >= 0x1p-8f && most <= 65504.0f);
}
__device__ __forceinline__ bool parts_hold(float most, const __nv_bfloat16 *) {
  return most == 0.0f || (most >= 0x1p-100f && most <= 0x1p+127f);
}

// Sum over the items of the threads before this one, and over all.
__device__ uint32_t block_exclusive(uint32_t x, uint32_t *total, uint32_t *sm /* [32] */) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t s = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(~0u, s, d);
    if (lane >= (uint32_t)d) s += o;
  }
  __syncthreads();
  if (lane == 31) sm[warp] = s;
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (uint32_t w = 0; w < (blockDim.x >> 5); ++w) {
    if (w < warp) before += sm[w];
    all += sm[w];
  }
  *total = all;
  return before + s - x;
}

// One CTA of 1024 threads: the requests in order of (adapter, request), their
// groups and columns.  The sort key is unique, so the order is always the same.
// Latency: 6.7 us for 8 requests, 9 for 64 of 20 tokens.
__global__ void __launch_bounds__(1024) order_kernel(const int32_t *ids, uint32_t n, uint32_t L, uint32_t num_adapters,
                                                     uint32_t slots, uint32_t tile_t, Sorted o) {
  extern __shared__ unsigned long long key[];  // [slots], then u32 [slots] group of a position, u32 [slots] its start
  uint32_t *group_pos = reinterpret_cast<uint32_t *>(key + slots);
  uint32_t *group_col = group_pos + slots;
  __shared__ uint32_t sm[32];
  for (uint32_t i = threadIdx.x; i < slots; i += 1024) {
    unsigned long long k = ~0ull;
    if (i < n) {
      const int32_t id = ids[i];
      k = (unsigned long long)((uint32_t)id < num_adapters ? (uint32_t)id + 1 : 0) << 32 | i;
    }
    key[i] = k;
  }
  for (uint32_t size = 2; size <= slots; size <<= 1)
    for (uint32_t step = size >> 1; step; step >>= 1) {
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < slots / 2; i += 1024) {
        const uint32_t a = 2 * i - (i & (step - 1)), b = a + step;
        const bool up = (a & size) == 0;
        const unsigned long long x = key[a], y = key[b];
        if ((x > y) == up) key[a] = y, key[b] = x;
      }
    }
  __syncthreads();
  // Each thread owns `per` neighbouring positions.
  const uint32_t per = (slots + 1023) / 1024, p0 = threadIdx.x * per;
  auto head = [&](uint32_t i) { return i < n && (i == 0 || (key[i] >> 32) != (key[i - 1] >> 32)); };
  uint32_t mine = 0, groups;
  for (uint32_t i = p0; i < p0 + per && i < slots; ++i) mine += head(i);
  uint32_t g = block_exclusive(mine, &groups, sm);
  const uint32_t g_before = g;
  for (uint32_t i = p0; i < p0 + per && i < slots; ++i)
    if (head(i)) group_pos[g++] = i;
  __syncthreads();
  auto width = [&](uint32_t q) {
    const uint32_t end = q + 1 < groups ? group_pos[q + 1] : n;
    return ((end - group_pos[q]) * L + 15) / 16 * 16;
  };
  uint32_t wide = 0, columns;
  for (uint32_t q = p0; q < p0 + per && q < groups; ++q) wide += width(q);
  uint32_t col = block_exclusive(wide, &columns, sm);
  for (uint32_t q = p0; q < p0 + per && q < groups; ++q) {
    const uint32_t w = width(q), end = q + 1 < groups ? group_pos[q + 1] : n;
    const uint32_t used = (end - group_pos[q]) * L;
    group_col[q] = col;
    o.groups[q] = Group{(int32_t)(uint32_t)(key[group_pos[q]] >> 32) - 1, col, col + w, 0};
    for (uint32_t c = used; c < w; ++c) o.col_token[col + c] = -1;
    for (uint32_t t = (col + tile_t - 1) / tile_t; t * tile_t < col + w; ++t) o.tile_first[t] = q;
    col += w;
  }
  if (threadIdx.x == 0) o.head[0] = groups, o.head[1] = columns;
  __syncthreads();
  for (uint32_t q = p0; q < p0 + per && q < groups; ++q) {
    const Group mine = o.groups[q];
    for (uint32_t t = mine.col0 / tile_t; t * tile_t < mine.col1; ++t) {
      const uint32_t at = t * kTileGroups + q - o.tile_first[t];
      o.tile_groups[at] = mine;
      if (mine.col1 >= (t + 1) * tile_t || q + 1 == groups) o.tile_groups[at + 1] = Group{-1, ~0u, ~0u, 0};
    }
  }
  g = g_before;  // groups that begin before this thread's positions
  for (uint32_t i = p0; i < p0 + per && i < n; ++i) {
    if (head(i)) ++g;
    o.req_col[(uint32_t)key[i]] = group_col[g - 1] + (i - group_pos[g - 1]) * L;
  }
}

constexpr int kShrinkTokens = 4, kShrinkRows = 4;

// u of up to four tokens of a request: a warp takes four low-rank rows, its
// lanes the inner dimension. The sorted form also moves the tokens to their
// columns and splits u into 16-bit parts, laid out as the products read them,
// the parts of eight columns next to one another; the values meet in shared
// memory before, where each token's largest decides whether parts hold them.
// Tokens four to a CTA, so that
// a few of them spread over many SMs: latency, 3.6 us for 8 tokens of D = 512
// and 6.5 for 128 of 768; 23 us for 1280 tokens of 2048 and rank 64, each CTA
// reading its adapter's rows from L2.
template <typename T, bool kSorted>
__global__ void __launch_bounds__(256) shrink_kernel(ft_adapter_args a, float *u, Sorted o) {
  const uint32_t per = (a.num_outpos + kShrinkTokens - 1) / kShrinkTokens;
  const uint32_t req = blockIdx.x / per, l0 = blockIdx.x % per * kShrinkTokens;
  const uint32_t count = min((uint32_t)kShrinkTokens, a.num_outpos - l0);
  const uint64_t tok = (uint64_t)req * a.num_outpos + l0;
  const int32_t id = a.adapter_ids[req];
  const bool has = (uint32_t)id < a.num_adapters;
  const T *h = static_cast<const T *>(a.hidden) + tok * a.dim;
  const uint32_t lane = threadIdx.x & 31;
  uint32_t col = 0;
  __shared__ float low[kSorted ? kShrinkTokens : 1][kSorted ? kMaxRank : 1];
  __shared__ bool wide[kShrinkTokens];
  sm100::launch_next();
  if (kSorted && o.single) {
    col = l0;
    if (!has) return;
  } else if (kSorted) {
    col = o.req_col[req] + l0;
    uint4 *to = reinterpret_cast<uint4 *>(static_cast<T *>(o.hidden) + (uint64_t)col * a.dim);
    const uint4 *from = reinterpret_cast<const uint4 *>(h);
    for (uint32_t i = threadIdx.x; i < count * (a.dim / 8); i += 256) to[i] = from[i];
    if (!has) {  // its columns take no part in any group's products
      const int32_t t = (int32_t)(tok + threadIdx.x);
      if (threadIdx.x < count) o.col_token[col + threadIdx.x] = id == -1 ? t : -2 - t;
      return;
    }
  }
  const float scale = has && a.scale ? a.scale[id] : 1.0f;
  // Rows up to the next multiple of 16 exist as zeros in the sorted form.
  const uint32_t rows = kSorted ? (a.rank + 15) / 16 * 16 : a.rank;
  for (uint32_t r = (threadIdx.x >> 5) * kShrinkRows; r < rows; r += 8 * kShrinkRows) {
    float s[kShrinkRows][kShrinkTokens] = {};
    if (has && r < a.rank) {
      const T *w = static_cast<const T *>(a.lora_a) + ((uint64_t)id * a.rank + r) * a.dim;
      for (uint32_t d = lane * 8; d < a.dim; d += 256) {
        uint4 wq[kShrinkRows], xq[kShrinkTokens];
#pragma unroll
        for (int i = 0; i < kShrinkRows; ++i) wq[i] = __ldg(reinterpret_cast<const uint4 *>(w + (uint64_t)i * a.dim + d));
#pragma unroll
        for (int q = 0; q < kShrinkTokens; ++q)
          xq[q] = __ldg(reinterpret_cast<const uint4 *>(h + (uint64_t)min(q, (int)count - 1) * a.dim + d));
#pragma unroll
        for (int q = 0; q < kShrinkTokens; ++q) {
          float x[8];
          unpack8<T>(xq[q], x);
#pragma unroll
          for (int i = 0; i < kShrinkRows; ++i) {
            float y[8];
            unpack8<T>(wq[i], y);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[i][q] = fmaf(x[e], y[e], s[i][q]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kShrinkRows; ++i)
#pragma unroll
        for (int q = 0; q < kShrinkTokens; ++q) {
#pragma unroll
          for (int d = 16; d; d >>= 1) s[i][q] += __shfl_xor_sync(~0u, s[i][q], d);
          s[i][q] *= scale;
        }
    }
    if (lane < count * kShrinkRows) {  // lane: token lane / 4, row r + lane % 4
      const uint32_t q = lane / kShrinkRows, i = lane % kShrinkRows;
      float v = 0.0f;
#pragma unroll
      for (int x = 0; x < kShrinkRows; ++x)
#pragma unroll
        for (int y = 0; y < kShrinkTokens; ++y)
          if (i == x && q == y) v = s[x][y];
      if (kSorted)
        low[q][r + i] = v;
      else
        u[(tok + q) * a.rank + r + i] = v;
    }
  }
  if (!kSorted) return;
  __syncthreads();
  if (const uint32_t q = threadIdx.x >> 5; q < count) {
    float most = 0.0f;
    for (uint32_t r = lane; r < a.rank; r += 32) most = fmaxf(most, fabsf(low[q][r]));
#pragma unroll
    for (int d = 16; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
    if (lane == 0) {
      wide[q] = !parts_hold(most, (const T *)nullptr);
      o.col_token[col + q] = (int32_t)(tok + q) | (wide[q] ? kWide : 0);
    }
  }
  __syncthreads();
  const uint32_t row = o.width * 2;
  for (uint32_t i = threadIdx.x; i < count * rows; i += 256) {
    const uint32_t q = i / rows, r = i % rows, c = col + q;
    float v = low[q][r];
    if (wide[q]) {
      if (r < a.rank) o.wide[(tok + q) * a.rank + r] = v;
      v = 0.0f;
    }
    uint8_t *at = o.u + ((uint64_t)(r / o.width) * (o.columns / 8) + c / 8) * o.parts * 8 * row +
                  sm100::swizzled(c % 8 * row + r % o.width * 2, row);
    for (uint32_t part = 0; part < o.parts; ++part) {
      T x;
      from_f32(v, x);
      *reinterpret_cast<T *>(at + part * 8 * row) = x;
      v -= to_f32(x);  // what is left for the next part
    }
  }
}

constexpr int kExpandThreads = 256, kExpandRows = 4, kExpandTokens = 4;

// The direct form's low-rank part: four vocabulary entries per thread, 256
// apart, for the tokens of one request. What costs here is getting to the rows
// of B, so that four are on their way at once; rows staged through shared
// memory in whole lines came out three times slower. 7.7 us for 37 single
// tokens with 40 adapters by 32000 of rank 16 (38 MB of rows, 4.9 TB/s).
template <typename T>
__global__ void __launch_bounds__(kExpandThreads) expand_kernel(ft_adapter_args a, const float *u, float *delta) {
  sm100::launch_next();
  const uint32_t blocks = (a.vocab + kExpandThreads * kExpandRows - 1) / (kExpandThreads * kExpandRows);
  const uint32_t req = blockIdx.x / blocks, v0 = blockIdx.x % blocks * (kExpandThreads * kExpandRows) + threadIdx.x;
  const int32_t id = a.adapter_ids[req];
  sm100::wait_for_previous();  // u
  if ((uint32_t)id >= a.num_adapters) return;
  const T *b = static_cast<const T *>(a.lora_b) + ((uint64_t)id * a.vocab + v0) * a.rank;
  const uint64_t apart = (uint64_t)kExpandThreads * a.rank;
  const uint32_t vocab = a.vocab, rank = a.rank;
  for (uint32_t l0 = 0; l0 < a.num_outpos; l0 += kExpandTokens) {
    const uint64_t t0 = (uint64_t)req * a.num_outpos + l0;
    const uint32_t count = min((uint32_t)kExpandTokens, a.num_outpos - l0);
    float acc[kExpandRows][kExpandTokens] = {};
    for (uint32_t r = 0; r < rank; r += 8) {
      uint4 q[kExpandRows];
#pragma unroll
      for (int i = 0; i < kExpandRows; ++i)
        q[i] = v0 + i * kExpandThreads < vocab ? __ldg(reinterpret_cast<const uint4 *>(b + i * apart + r)) : uint4{};
#pragma unroll
      for (int x = 0; x < kExpandTokens; ++x) {
        if (x >= (int)count) break;
        const float4 *p = reinterpret_cast<const float4 *>(u + (t0 + x) * rank + r);
        const float4 x0 = __ldcg(p), x1 = __ldcg(p + 1);
#pragma unroll
        for (int i = 0; i < kExpandRows; ++i) {
          float w[8];
          unpack8<T>(q[i], w);
          float s = acc[i][x];
          s = fmaf(x0.x, w[0], s), s = fmaf(x0.y, w[1], s), s = fmaf(x0.z, w[2], s), s = fmaf(x0.w, w[3], s);
          s = fmaf(x1.x, w[4], s), s = fmaf(x1.y, w[5], s), s = fmaf(x1.z, w[6], s), s = fmaf(x1.w, w[7], s);
          acc[i][x] = s;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kExpandRows; ++i)
#pragma unroll
      for (int x = 0; x < kExpandTokens; ++x)
        if (x < (int)count && v0 + i * kExpandThreads < vocab) delta[(t0 + x) * vocab + v0 + i * kExpandThreads] = acc[i][x];
  }
}

struct LogitsPlan {
  uint32_t columns;    // tokens, or the sorted form's upper bound
  uint32_t tile_t;     // columns of a tile, a multiple of 16
  uint32_t tiles_t;
  uint32_t halves;     // 128 vocabulary entries each
  uint32_t tiles_v;
  uint32_t stage;      // bytes
  uint32_t stages;
  uint32_t acc;        // tensor memory columns of an accumulator
  uint32_t split;      // accumulators of a half: the inner dimension's chunks take turns
  uint32_t buffers;    // sets of accumulators: with two, a tile's products run while the last one is stored
  // Bytes that a group of columns takes in a stage: for its adapter's rows, and
  // for its low-rank values per column; and how many columns fit.
  uint32_t group_rows, group_column, group_most;
};

struct alignas(16) LogitsShared {
  uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2], drained;
  // By turns for every other tile: where a column's logits begin in the output
  // (in bytes; negative: it has none), and which columns' logits are NaN.
  int64_t begin[2][kMaxTileT];
  uint32_t wrong[2][kMaxTileT / 32];
  uint32_t more[2][kMaxTileT / 32];  // which columns' low-rank part the epilogue adds
  uint32_t tmem, gave_up;
};

LogitsPlan plan_logits(const ft_adapter_args &a, uint32_t columns, uint32_t parts, uint32_t width) {
  LogitsPlan p;
  p.columns = columns;
  p.tiles_t = (columns + kMaxTileT - 1) / kMaxTileT;
  p.tile_t = ((columns + p.tiles_t - 1) / p.tiles_t + 15) / 16 * 16;
  p.acc = 32;
  while (p.acc < p.tile_t) p.acc *= 2;
  // Two halves share the tokens' part of a stage, where there are tiles enough
  // for all SMs: an SM takes in 64 bytes a cycle, and one half by 256 columns
  // needs 96 to keep the tensor cores busy, two need 64.
  // The tensor cores cut each partial sum instead of rounding it, so that a sum
  // of D products comes out D 5e-10 too small on average (1.6e-6 off, relative,
  // at D = 2048): two sums of half the length are half as far off. 16-bit
  // logits do not show it.
  p.split = a.out_dtype == FT_DTYPE_F32 && a.dim > 1024 ? 2 : 1;
  p.halves = a.vocab >= 148 * 4 * kTileV && (p.split == 1 || p.acc <= 64) ? 2 : 1;
  p.buffers = std::min<uint32_t>(2, 512 / (p.halves * p.split * p.acc));
  p.tiles_v = (a.vocab + p.halves * kTileV - 1) / (p.halves * kTileV);
  p.stage = (p.halves * kTileV + std::max(p.tile_t, 16 * parts)) * kTileD * 2;
  p.stages = std::min<uint32_t>(kMaxStages, (220 * 1024) / p.stage);
  p.group_rows = p.halves * kTileV * width * 2;
  p.group_column = parts * width * 2;
  p.group_most = parts ? (p.stage - p.group_rows) / p.group_column / 16 * 16 : 0;
  return p;
}
size_t logits_smem(const LogitsPlan &p) { return 1024 + (size_t)p.stages * p.stage; }

// sum_r u[r] b[r] of a token whose low-rank values are in 32 bits alone. Rows of B
// come one by one: with such tokens alone, 0.64 ms instead of 0.17 for 20 tokens
// by 500k x 1024 of rank 16, 8 instead of 0.55 for 1280 by 100k x 2048 of rank 64.
template <typename T>
__device__ __noinline__ float wide_part(const T *b, const float *u, uint32_t rank) {
  float s = 0.0f;
  for (uint32_t r = 0; r < rank; r += 8) {
    float w[8];
    unpack8<T>(__ldg(reinterpret_cast<const uint4 *>(b + r)), w);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(__ldcg(u + r + e), w[e], s);
  }
  return s;
}

// What a walk reads again and again, in registers.
struct Walk {
  uint32_t tile_t, stage, group_rows, group_column, group_most, width, slices, chunks;
};

// The stages of a tile in the order that loads and products both take them:
// the shared projection's, then those of each group that has columns in it.
// f(chunk) for the first, a stage each. The others share stages as far as they
// fit: g(adapter, first column, width, low-rank slice, offset in the stage),
// with open() before the first of a stage and close() after the last. A
// callback that returns false ends the walk.
// `mine`: the tile's groups, one a lane. The whole warp takes part.
template <typename F, typename Open, typename G, typename Close>
__device__ __forceinline__ bool walk_tile(const Walk &k, bool sorted, const Group &mine, uint32_t c0, F &&f, Open &&open,
                                          G &&g, Close &&close) {
  for (uint32_t c = 0; c < k.chunks; ++c)
    if (!f(c)) return false;
  if (!sorted) return true;
  const uint32_t c1 = c0 + k.tile_t;
  uint32_t used = 0;
  for (uint32_t i = 0;; ++i) {
    // A reduction rather than a shuffle: its result is uniform.
    const bool from = (threadIdx.x & 31) == i;
    const uint32_t col0 = __reduce_or_sync(~0u, from ? mine.col0 : 0), col1 = __reduce_or_sync(~0u, from ? mine.col1 : 0);
    const int32_t adapter = (int32_t)__reduce_or_sync(~0u, from ? (uint32_t)mine.adapter : 0);
    if (col0 >= c1) break;  // the list ends with such a one
    if (adapter < 0) continue;
    const uint32_t end = min(col1, c1);
    for (uint32_t w0 = max(col0, c0); w0 < end; w0 += k.group_most)
      for (uint32_t j = 0; j < k.slices; ++j) {
        const uint32_t w = min(k.group_most, end - w0), need = k.group_rows + w * k.group_column;
        if (used && used + need > k.stage) {
          close();
          used = 0;
        }
        if (!used && !open()) return false;
        g(adapter, w0, w, j, used);
        used += need;
      }
  }
  if (used) close();
  return true;
}

// Persistent, one CTA per SM.  Tiles that share a stretch of the weight are
// neighbours in the order, so that it comes from DRAM once.
//
// Few tokens: bound by the weight's bytes, 688 us for 20 tokens by 2.2M x 1024
// bf16 (4.6 GB, 6.7 TB/s), 156 us for 128 by 500k x 768 with f32 logits (1.02
// GB, 6.6 TB/s) and 182 with eight adapters.  Full batches: bound by what an SM
// takes in and by the power limit.  1280 tokens by 500k x 2048 with 16 adapters
// of rank 64 take 2.39 to 2.5 ms (1080 to 1130 TFLOP/s of useful products).  By
// 100k, the shared product alone takes 382 us (1373 TFLOP/s) and with adapters 485 to 500: the
// padded columns make a sixth tile of tokens, which loads the weight once more
// (a seventh of the time), the rest are the adapters' rows and values.
template <typename T, typename O, bool kSorted>
__global__ void __launch_bounds__(kThreads, 1)
    logits_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_h,
                  const __grid_constant__ CUtensorMap map_b, const __grid_constant__ ft_adapter_args a,
                  const __grid_constant__ LogitsPlan p, const float *delta, const __grid_constant__ Sorted o,
                  uint32_t *status) {
  using namespace sm100;
  extern __shared__ uint8_t raw[];
  uint8_t *buf = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  __shared__ LogitsShared sh;
  const uint32_t warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t bytes_w = p.halves * kTileV * kTileD * 2, bytes = p.stage;
  volatile uint32_t *gave_up = &sh.gave_up;
  if (threadIdx.x == 0) {
    sh.gave_up = 0;
    for (uint32_t s = 0; s < p.stages; ++s) mbar_init(&sh.full[s], 1), mbar_init(&sh.empty[s], 1);
    for (int b = 0; b < 2; ++b) mbar_init(&sh.acc_full[b], 1), mbar_init(&sh.acc_empty[b], kEpilogue);
    mbar_init(&sh.drained, 1);
    mbar_init_fence();
    prefetch_map(&map_w);
    prefetch_map(&map_h);
  }
  if (warp == kProductWarp) tmem_alloc(&sh.tmem, p.buffers * p.halves * p.split * p.acc);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  // What the kernel before this one left: the tables here, u where the loads
  // come to it, the direct form's sums in the epilogue.
  const bool tables = kSorted && !o.single;
  if (tables) wait_for_previous();
  const uint32_t columns = tables ? o.head[1] : p.columns;
  const uint32_t tiles_t = (columns + p.tile_t - 1) / p.tile_t;
  const uint32_t tiles = tiles_t * p.tiles_v;
  const Walk walk{p.tile_t, p.stage, p.group_rows, p.group_column, p.group_most, o.width,
                  kSorted ? (a.rank + o.width - 1) / o.width : 0, (a.dim + kTileD - 1) / kTileD};
  const int32_t only = kSorted && o.single ? a.adapter_ids[0] : -1;
  const bool single_low = kSorted && o.single && (uint32_t)only < a.num_adapters;

  // A tile's groups, one a lane, are fetched while the tile before is under
  // way: a look into global memory takes microseconds when the memory is busy,
  // and neither loads nor products may pause for it.
  auto fetch = [&](uint32_t tile) {
    if (kSorted && o.single)
      return lane ? Group{-1, ~0u, ~0u, 0} : Group{(uint32_t)only < a.num_adapters ? only : -1, 0, columns, 0};
    return kSorted && lane < kTileGroups && tile < tiles ? o.tile_groups[tile % tiles_t * kTileGroups + lane]
                                                         : Group{-1, ~0u, ~0u, 0};
  };

  const bool lead = elect_one();
  uint32_t sent = 0;  // stages filled so far (the loads' warp)
  if (warp == kLoadWarp) {
    uint32_t at = 0;  // stage
    bool ok = true;
    const uint8_t *low = o.u;
    const uint32_t slice = o.columns;
    auto open = [&] {  // the next stage, once it is free
      if (sent >= p.stages) ok = mbar_wait(&sh.empty[at], (sent / p.stages - 1) & 1, gave_up);
      ok = __all_sync(~0u, ok);
      return ok;
    };
    auto next = [&] {
      ++sent;
      at = at + 1 == p.stages ? 0 : at + 1;
    };
    Group ahead = fetch(blockIdx.x);
    for (uint32_t tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
      const Group mine = ahead;
      ahead = fetch(tile + gridDim.x);
      const int32_t v0 = (int32_t)(tile / tiles_t * p.halves * kTileV), t0 = (int32_t)(tile % tiles_t * p.tile_t);
      walk_tile(
          walk, kSorted, mine, (uint32_t)t0,
          [&](uint32_t c) {
            if (!open()) return false;
            uint8_t *st = buf + (size_t)at * bytes;
            mbar_expect(&sh.full[at], bytes_w + p.tile_t * kTileD * 2, lead);
            tma_load_2d(st, &map_w, &sh.full[at], (int32_t)(c * kTileD), v0, lead);
            tma_load_2d(st + bytes_w, &map_h, &sh.full[at], (int32_t)(c * kTileD), t0, lead);
            next();
            return true;
          },
          [&] {
            if (o.single) wait_for_previous();
            return open();
          },
          [&](int32_t adapter, uint32_t w0, uint32_t w, uint32_t j, uint32_t offset) {
            uint8_t *st = buf + (size_t)at * bytes + offset;
            mbar_expect_more(&sh.full[at], walk.group_rows + w * walk.group_column, lead);
            tma_load_3d(st, &map_b, &sh.full[at], (int32_t)(j * walk.width), v0, adapter, lead);
            bulk_load(st + walk.group_rows, low + ((uint64_t)j * slice + w0) * walk.group_column, w * walk.group_column,
                      &sh.full[at], lead);
          },
          [&] {
            mbar_arrive(&sh.full[at], lead);
            next();
          });
    }
  } else if (warp == kProductWarp) {
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    uint32_t at = 0, phase = 0, n = 0;
    bool ok = true;
    const uint64_t first_w = operand(buf), first_h = operand(buf + bytes_w);
    const uint32_t parts = o.parts, rank = a.rank, halves = p.halves, acc = p.acc, split = p.split;
    const uint32_t next_half = split * acc;
    auto open = [&] {
      ok = mbar_wait(&sh.full[at], phase, gave_up);
      ok = __all_sync(~0u, ok);
      fence_after();
      return ok;
    };
    auto done = [&] {  // the stage is free when the products so far have ended
      if (++at == p.stages) at = 0, phase ^= 1;
    };
    Group ahead = fetch(blockIdx.x);
    for (uint32_t tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, ++n) {
      const Group mine = ahead;
      ahead = fetch(tile + gridDim.x);
      const uint32_t b = n % p.buffers, d = tmem + b * halves * next_half, c0 = tile % tiles_t * p.tile_t;
      const uint32_t shape = mma_shape(kBf16, kTileV, min(p.tile_t, (columns - c0 + 15) / 16 * 16));
      if (n >= p.buffers) ok = __all_sync(~0u, mbar_wait(&sh.acc_empty[b], (n / p.buffers - 1) & 1, gave_up));
      if (!ok) break;
      fence_after();
      walk_tile(
          walk, kSorted, mine, c0,
          [&](uint32_t c) {
            if (!open()) return false;
            const uint64_t w = first_w + (at * bytes >> 4), h = first_h + (at * bytes >> 4);
            const uint32_t turn = c & (split - 1), into = d + turn * acc;
            const bool begun = c >= split;
#pragma unroll
            for (int k = 0; k < kTileD / 16; ++k) mma_f16(into, w + 2 * k, h + 2 * k, shape, begun || k > 0, lead);
            if (halves == 2) {
#pragma unroll
              for (int k = 0; k < kTileD / 16; ++k)
                mma_f16(into + next_half, w + (kTileV * kTileD * 2 >> 4) + 2 * k, h + 2 * k, shape, begun || k > 0, lead);
            }
            mma_commit(&sh.empty[at], lead);
            done();
            return true;
          },
          open,
          [&](int32_t, uint32_t w0, uint32_t w, uint32_t j, uint32_t offset) {
            // Loops over counts that are known here: with bounds looked up on the
            // way every product took 160 cycles.
            const uint32_t row = walk.width * 2;
            const uint8_t *st = buf + (size_t)at * bytes + offset;
            const uint64_t bw = operand(st, row, 8 * row), uw = operand(st + walk.group_rows, row, parts * 8 * row);
            const uint32_t steps = (min(rank - j * walk.width, walk.width) + 15) / 16;
            const uint32_t narrow = mma_shape(kBf16, kTileV, w), to = d + (w0 - c0);
#pragma unroll
            for (uint32_t k = 0; k < kTileD / 16; ++k)
              if (k < steps) {
#pragma unroll
                for (uint32_t x = 0; x < kMaxParts; ++x)
                  if (x < parts) {
                    mma_f16(to, bw + 2 * k, uw + (x * 8 * row >> 4) + 2 * k, narrow, true, lead);
                    if (halves == 2)
                      mma_f16(to + next_half, bw + (kTileV * row >> 4) + 2 * k, uw + (x * 8 * row >> 4) + 2 * k, narrow, true,
                              lead);
                  }
              }
          },
          [&] {
            mma_commit(&sh.empty[at], lead);
            done();
          });
      if (ok) mma_commit(&sh.acc_full[b], lead);
    }
  } else {
    // Warps with the same w % 4 read the same quarter of tensor memory (its
    // lanes 32 (w % 4) on); they share the halves and the blocks of 16 columns.
    uint32_t n = 0;
    bool ok = true;
    const uint32_t halves = p.halves, buffers = p.buffers, tile_t = p.tile_t, vocab = a.vocab;
    const uint32_t half = halves == 2 ? warp >> 3 : 0, row = half * kTileV + (warp & 3) * 32 + lane;
    const uint32_t first = (halves == 2 ? warp >> 2 & 1 : warp >> 2) * 16, stride = halves == 2 ? 32 : 64;
    const uint32_t odd = lane & 1;
    const int64_t pitch = (int64_t)vocab * sizeof(O);
    const bool pairs = sizeof(O) == 2 && vocab % 2 == 0;
    const uint32_t split = p.split, apart = p.acc, set = halves * split * apart;
    const uint32_t mine = tmem + half * split * apart + ((warp & 3) << 21);
    uint8_t *const logits = static_cast<uint8_t *>(a.out);
    if (single_low) wait_for_previous();  // col_token
    for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++n) {
      const uint32_t b = n % buffers, t0 = tile % tiles_t * tile_t;
      const uint32_t v = tile / tiles_t * halves * kTileV + row;
      const bool live = v < vocab;
      const uint32_t count = min(tile_t, columns - t0);
      if (threadIdx.x < kMaxTileT) {  // thread c looks up what column c is
        const uint32_t c = threadIdx.x;
        int32_t token = -1;
        bool bad = false, more = false;
        if (c < count) {
          token = (int32_t)(t0 + c);
          if (kSorted && o.single) {
            bad = !single_low && only != -1;
            if (t0 + c >= a.num_outpos)
              token = -1;
            else if (single_low)
              token = __ldcg(&o.col_token[t0 + c]);
          } else if (kSorted) {
            token = __ldcg(&o.col_token[t0 + c]);
            bad = token < -1;
            if (bad) token = -2 - token;
          } else if (delta) {
            const int32_t id = a.adapter_ids[token / a.num_outpos];
            more = (uint32_t)id < a.num_adapters;
            bad = !more && id != -1;
          }
          if (kSorted && token >= kWide) {
            token -= kWide;
            more = true;
          }
        }
        sh.begin[n & 1][c] = token < 0 ? -1 : (int64_t)token * pitch;
        const uint32_t bads = __ballot_sync(~0u, bad), mores = __ballot_sync(~0u, more);
        if (lane == 0) sh.wrong[n & 1][warp] = bads, sh.more[n & 1][warp] = mores;
      }
      // One warp looks for the products' end and the others wait at the block's
      // barrier: sixteen warps that look would take the issue slots from the
      // warps that load and multiply (160 instead of 70 cycles a product).
      const int64_t *begin = sh.begin[n & 1];
      if (!kSorted && delta && n == 0) wait_for_previous();
      if (warp == 0 && ok) mbar_wait(&sh.acc_full[b], (n / buffers) & 1, gave_up);
      asm volatile("bar.sync 1, %0;" ::"n"(kEpilogue) : "memory");
      ok = __all_sync(~0u, ok && !*gave_up);
      if (ok) fence_after();
      for (uint32_t c0 = first; c0 < count; c0 += stride) {
        uint32_t acc[16];
        if (ok) {
          tmem_load16(mine + b * set + c0, acc);
          if (split == 2) {
            uint32_t rest[16];
            tmem_load16(mine + b * set + apart + c0, rest);
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[e] = __float_as_uint(__uint_as_float(acc[e]) + __uint_as_float(rest[e]));
          }
        } else {
          // A wait ran out: no result is better than a wrong one.
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[e] = 0x7FC00000;
        }
        const uint32_t wrong = sh.wrong[n & 1][c0 / 32] >> (c0 % 32) & 0xFFFF;
        if (!kSorted && delta) {
          const uint32_t any = sh.more[n & 1][c0 / 32] >> (c0 % 32) & 0xFFFF;
          // Not through the read-only path: this kernel may begin while the
          // one before it still writes these.
          float add[16];
#pragma unroll
          for (int e = 0; e < 16; ++e)
            add[e] = live && (any >> e & 1) ? __ldcg(&delta[(uint64_t)(t0 + c0 + e) * vocab + v]) : 0.0f;
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[e] = __float_as_uint(__uint_as_float(acc[e]) + add[e]);
        }
        if (kSorted) {
          const uint32_t any = sh.more[n & 1][c0 / 32] >> (c0 % 32) & 0xFFFF;
          if (any && live) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (any >> e & 1) {
                const uint32_t token = (uint32_t)(begin[c0 + e] / pitch);
                const int32_t id = o.single ? only : a.adapter_ids[token / a.num_outpos];
                acc[e] = __float_as_uint(__uint_as_float(acc[e]) +
                                         wide_part(static_cast<const T *>(a.lora_b) + ((uint64_t)id * vocab + v) * a.rank,
                                                   o.wide + (uint64_t)token * a.rank, a.rank));
              }
          }
        }
        if (wrong) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (wrong >> e & 1) acc[e] = 0x7FC00000;
        }
        uint8_t *out = logits + (uint64_t)v * sizeof(O);
        if (pairs) {
          // Neighbouring lanes trade, so that each has two entries of one token
          // and stores them together.
          out -= odd * 2;
          int64_t at[8];
          uint32_t two[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) at[e] = begin[c0 + 2 * e + odd];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t got = __shfl_xor_sync(~0u, odd ? acc[2 * e] : acc[2 * e + 1], 1);
            two[e] = pack_pair(__uint_as_float(odd ? got : acc[2 * e]), __uint_as_float(odd ? acc[2 * e + 1] : got),
                               static_cast<O *>(nullptr));
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) store_if(live && at[e] >= 0, reinterpret_cast<uint32_t *>(out + at[e]), two[e]);
        } else {
          int64_t at[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) at[e] = begin[c0 + e];
#pragma unroll
          for (int e = 0; e < 16; ++e)
            store_if(live && at[e] >= 0, reinterpret_cast<O *>(out + at[e]), __uint_as_float(acc[e]));
        }
      }
      if (ok) {
        fence_before();
        mbar_arrive(&sh.acc_empty[b]);
      }
    }
  }
  __syncwarp();
  __syncthreads();
  if (sh.gave_up) {
    // Whichever warp gave up, neither copies nor products may be under way when
    // the block ends: wait for the last fill of each stage, and for the products
    // issued so far (if nothing failed the epilogue has seen all of them).
    if (warp == kLoadWarp)
      for (uint32_t s = 0; s < p.stages && s < sent; ++s) mbar_settle(&sh.full[s], (sent - 1 - s) / p.stages & 1);
    if (warp == kProductWarp) {
      mma_commit(&sh.drained, lead);
      mbar_settle(&sh.drained, 0);
    }
    if (threadIdx.x == 0 && status) atomicOr(status, kStatusLogits);
  }
  fence_before();
  __syncthreads();
  fence_after();
  wait_for_previous();  // so that this kernel's end stands for that one's
  if (warp == kProductWarp) tmem_free(tmem, p.buffers * p.halves * p.split * p.acc);
}

// A launch that, with `early`, may begin before the kernel launched before it has
// ended; it waits for that one itself. Only behind a kernel of the same call:
// the call's inputs may come from whatever ran before that.
template <typename... Params, typename... Args>
void launch(bool early, unsigned grid, unsigned threads, size_t smem, cudaStream_t stream, void (*kernel)(Params...),
            Args... args) {
  cudaLaunchAttribute overlap;
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &overlap;
  cfg.numAttrs = early ? 1 : 0;
  CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
}

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                              const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult found;
    CUDA_TRY(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found));
    if (!p || found != cudaDriverEntryPointSuccess) throw CudaError("CUDA error: the driver has no cuTensorMapEncodeTiled");
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// `layers` arrays of rows of `inner` 16-bit values, loaded as boxes of `width`
// (16, 32 or 64) values by `box` rows, swizzled over that width; what lies
// outside reads as 0.
CUtensorMap make_map(const void *base, bool bf16, uint64_t inner, uint64_t rows, uint64_t layers, uint32_t width,
                     uint32_t box, const char *what) {
  CUtensorMap m;
  const cuuint64_t dims[3] = {inner, rows, layers}, strides[2] = {inner * 2, inner * rows * 2};
  const cuuint32_t tile[3] = {width, box, 1}, step[3] = {1, 1, 1};
  const CUtensorMapSwizzle swizzle = width == 64   ? CU_TENSOR_MAP_SWIZZLE_128B
                                     : width == 32 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                   : CU_TENSOR_MAP_SWIZZLE_32B;
  const CUresult rc =
      encode_fn()(&m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, layers ? 3 : 2,
                  const_cast<void *>(base), dims, strides, tile, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS)
    throw CudaError(std::string("CUDA error: cuTensorMapEncodeTiled refused ") + what + " (" + std::to_string((int)rc) + ")");
  return m;
}

int sm_count() {
  int dev = 0, n = 0;
  CUDA_TRY(cudaGetDevice(&dev));
  CUDA_TRY(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
  return n;
}

void check_adapter(const ft_adapter_args &a) {
  if (a.dtype != FT_DTYPE_BF16 && a.dtype != FT_DTYPE_F16)
    throw InvalidArgument("adapter_logits: hidden and weight must be bf16 or f16");
  if (a.out_dtype != a.dtype && a.out_dtype != FT_DTYPE_F32)
    throw InvalidArgument("adapter_logits: the logits are of the inputs' type or f32");
  if (a.num_outpos == 0 || a.vocab == 0 || a.dim == 0) throw InvalidArgument("adapter_logits: num_outpos, vocab and dim must be positive");
  if (a.dim % 8) throw InvalidArgument("adapter_logits: dim must be a multiple of 8");
  if (a.num_adapters && (a.rank == 0 || a.rank % 8 || a.rank > kMaxRank))
    throw InvalidArgument("adapter_logits: rank must be a multiple of 8 in [8, 256]");
  if (a.num_adapters > kMaxAdapters) throw InvalidArgument("adapter_logits: at most 65536 adapters");
  // Token and vocabulary coordinates of a tile are 32-bit.
  if ((uint64_t)a.n * a.num_outpos > kMaxTokens || a.vocab > 0x3FFFFF00u || a.dim > 0xFFFFFF ||
      (uint64_t)(a.vocab / kTileV + 1) * ((uint64_t)a.n * a.num_outpos / 16 + 1) > 0x7FFFFFFF ||
      (uint64_t)(a.vocab / kExpandThreads + 1) * a.n > 0x7FFFFFFF)
    throw InvalidArgument("adapter_logits: too many tokens or too large a vocabulary");
}

uint64_t align256(uint64_t x) { return (x + 255) & ~(uint64_t)255; }

// Which form a call takes and where its workspace's parts lie.
struct Layout {
  bool sorted = false, single = false;
  uint32_t tokens = 0, columns = 0, parts = 0, width = 0;
  uint64_t delta = 0, head = 0, groups = 0, tile_first = 0, tile_groups = 0, req_col = 0, col_token = 0, hidden = 0, u = 0, wide = 0,
           end = 0;
};

Layout layout_of(const ft_adapter_args &a) {
  Layout l;
  l.tokens = l.columns = a.n * a.num_outpos;
  if (!a.num_adapters || l.tokens == 0) return l;
  // Padding a group to a multiple of 16 columns adds at most 16 - gcd(L, 16).
  const uint64_t groups = std::min<uint64_t>(a.n, (uint64_t)a.num_adapters + 1);
  uint32_t step = 1;
  while (step < 16 && a.num_outpos % (2 * step) == 0) step *= 2;
  l.single = a.n == 1;
  const uint64_t most = ((uint64_t)l.tokens + (l.single ? 0 : groups * (16 - step)) + 15) / 16 * 16;
  // Padding costs products of the shared projection, the direct form products on
  // the CUDA cores, r for each logit. 256 tokens by 100k x 1024, us sorted and
  // direct: 64 groups of rank 64 (4.8 times the columns) 340 and 909, of rank 16
  // 280 and 245; 64 of 4 tokens, rank 32 (4 times) 171 and 207; 100 of 2 tokens,
  // rank 16 (8 times) 266 and 176.
  l.sorted = l.single || (a.n <= kMaxSortRequests && 16 * most <= (uint64_t)l.tokens * (32 + a.rank));
  if (!l.sorted) {
    l.delta = align256((uint64_t)l.tokens * a.rank * 4);
    l.end = l.delta + align256((uint64_t)l.tokens * a.vocab * 4);
    return l;
  }
  l.columns = (uint32_t)most;
  l.width = a.rank <= 16 ? 16 : a.rank <= 32 ? 32 : 64;
  l.parts = a.dtype == FT_DTYPE_BF16 && a.out_dtype == FT_DTYPE_F32 ? 3 : 2;
  uint64_t at = 256;
  auto place = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += align256(bytes);
    return here;
  };
  l.u = place((uint64_t)((a.rank + l.width - 1) / l.width) * most * l.parts * l.width * 2);
  l.col_token = place(4 * most);
  l.wide = place(4ull * l.tokens * a.rank);
  if (l.single) {
    l.end = at;
    return l;
  }
  l.groups = place(sizeof(Group) * groups);
  l.tile_first = place(4 * (most / 16 + 1));
  l.tile_groups = place(sizeof(Group) * kTileGroups * (most / plan_logits(a, l.columns, l.parts, l.width).tile_t + 1));
  l.req_col = place(4ull * a.n);
  l.hidden = place(most * a.dim * 2);
  l.end = at;
  return l;
}

}  // namespace

uint64_t adapter_logits_workspace(const ft_adapter_args &a) {
  check_adapter(a);
  return layout_of(a).end;
}

void adapter_logits_device(const ft_adapter_args &a, uint32_t *status, void *ws, uint64_t ws_bytes,
                           cudaStream_t stream) {
  check_adapter(a);
  if (a.n == 0) return;
  if (reinterpret_cast<uintptr_t>(status) & 3)
    throw InvalidArgument("adapter_logits: the status word is not aligned to its 4 bytes");
  const void *need[] = {a.hidden, a.weight, a.out};
  for (const void *p : need)
    if (!p) fail(ErrorKind::kNull, "MARISA_NULL_ERROR: adapter_logits: hidden, weight or out is NULL");
  if (a.num_adapters && (!a.adapter_ids || !a.lora_a || !a.lora_b))
    fail(ErrorKind::kNull, "MARISA_NULL_ERROR: adapter_logits: adapter_ids, lora_a or lora_b is NULL");
  const void *sixteen[] = {a.hidden, a.weight, a.out, a.num_adapters ? a.lora_a : nullptr,
                           a.num_adapters ? a.lora_b : nullptr};
  for (const void *p : sixteen)
    if (reinterpret_cast<uintptr_t>(p) & 15)
      throw InvalidArgument("adapter_logits: hidden, weight, lora_a, lora_b and out must start on 16-byte boundaries");
  const Layout l = layout_of(a);
  if (ws_bytes < l.end || (l.end && (!ws || (reinterpret_cast<uintptr_t>(ws) & 255))))
    throw InvalidArgument("adapter_logits: needs a 256-byte aligned workspace of " + std::to_string(l.end) + " bytes");
  const LogitsPlan p = plan_logits(a, l.columns, l.parts, l.width);
  uint8_t *w = static_cast<uint8_t *>(ws);
  float *u = a.num_adapters && !l.sorted ? reinterpret_cast<float *>(w) : nullptr;
  float *delta = u ? reinterpret_cast<float *>(w + l.delta) : nullptr;
  Sorted o{};
  if (l.sorted)
    o = Sorted{reinterpret_cast<uint32_t *>(w + l.head),    reinterpret_cast<Group *>(w + l.groups),
               reinterpret_cast<uint32_t *>(w + l.tile_first),
               reinterpret_cast<Group *>(w + l.tile_groups), reinterpret_cast<uint32_t *>(w + l.req_col),
               reinterpret_cast<int32_t *>(w + l.col_token), reinterpret_cast<float *>(w + l.wide), w + l.hidden,
               w + l.u, l.columns, l.parts, l.width, l.single};
  const bool bf16 = a.dtype == FT_DTYPE_BF16;
  const CUtensorMap map_w = make_map(a.weight, bf16, a.dim, a.vocab, 0, kTileD, p.halves * kTileV, "weight");
  const CUtensorMap map_h = make_map(l.sorted && !l.single ? o.hidden : a.hidden, bf16, a.dim,
                                     l.sorted && !l.single ? l.columns : l.tokens, 0, kTileD, p.tile_t, "hidden");
  CUtensorMap map_b = map_w;
  if (l.sorted) map_b = make_map(a.lora_b, bf16, a.rank, a.vocab, a.num_adapters, l.width, p.halves * kTileV, "lora_b");
  const size_t smem = logits_smem(p);
  const unsigned grid = std::min<unsigned>(p.tiles_t * p.tiles_v, (unsigned)sm_count());
  const unsigned shrink = a.n * ((a.num_outpos + kShrinkTokens - 1) / kShrinkTokens);
  if (l.sorted && !l.single) {
    uint32_t slots = 2;
    while (slots < a.n) slots <<= 1;
    const size_t room = 16ull * slots;
    allow_shared(order_kernel, 16 * (int)kMaxSortRequests);
    order_kernel<<<1, 1024, room, stream>>>(a.adapter_ids, a.n, a.num_outpos, a.num_adapters, slots, p.tile_t, o);
    CUDA_TRY(cudaGetLastError());
  }
  auto logits = [&](auto *kernel) {
    allow_shared(kernel, 221 * 1024);
    launch(a.num_adapters != 0, grid, kThreads, smem, stream, kernel, map_w, map_h, map_b, a, p, (const float *)delta, o,
           status);
  };
  auto run = [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (l.sorted)
      shrink_kernel<T, true><<<shrink, 256, 0, stream>>>(a, u, o);
    else if (u)
      shrink_kernel<T, false><<<shrink, 256, 0, stream>>>(a, u, o);
    CUDA_TRY(cudaGetLastError());
    if (u) {
      const uint32_t rows = kExpandThreads * kExpandRows;
      launch(true, a.n * ((a.vocab + rows - 1) / rows), kExpandThreads, 0, stream, expand_kernel<T>, a, (const float *)u,
             delta);
    }
    if (l.sorted)
      a.out_dtype == FT_DTYPE_F32 ? logits(logits_kernel<T, float, true>) : logits(logits_kernel<T, T, true>);
    else
      a.out_dtype == FT_DTYPE_F32 ? logits(logits_kernel<T, float, false>) : logits(logits_kernel<T, T, false>);
  };
  if (bf16)
    run((__nv_bfloat16 *)nullptr);
  else
    run((__half *)nullptr);
}

}  // namespace ftb
