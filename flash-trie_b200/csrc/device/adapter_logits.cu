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
// two or three 16-bit parts, so that no more than 2^-18 of it is lost (2^-27
// for f32 logits).  No column is shared, so an adapter with infinities reaches
// no other one's requests.  "Direct": the tokens stay as they are and the
// epilogue adds the products in 32 bits, for batches whose groups are so small
// that padding them would cost more.
#include <algorithm>
#include <string>

#include "../engine.hpp"
#include "cuda_util.hpp"
#include "head_ops.hpp"
#include "row_stream.cuh"
#include "sm100.cuh"

namespace ftb {
namespace {

constexpr uint32_t kMaxRank = 256;
constexpr uint32_t kMaxAdapters = 65536;

constexpr int kTileV = 128;   // vocabulary entries of a tile (rows of the product)
constexpr int kTileD = 64;    // inner dimension of a stage: 128-byte rows
constexpr int kMaxTileT = 256;
constexpr int kMaxStages = 12;
constexpr int kEpilogue = 256;            // threads of warps 0-7
constexpr int kThreads = kEpilogue + 64;  // warp 8: loads, warp 9: products
constexpr uint32_t kMaxSortRequests = 8192;

template <typename T>
__device__ __forceinline__ void unpack8(uint4 q, float (&v)[8]) {
  unpack(q, v, (const T *)nullptr);
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
  uint32_t *req_col;     // first column of each request
  int32_t *col_token;    // token of a column; -1 padding; -2 - token: of a request whose adapter does not exist
  void *hidden;          // [columns][dim]
  void *u;               // [parts][columns][rank]
  uint32_t columns;      // upper bound, a multiple of 16
  uint32_t parts;
};

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
  g = g_before;  // groups that begin before this thread's positions
  for (uint32_t i = p0; i < p0 + per && i < n; ++i) {
    if (head(i)) ++g;
    o.req_col[(uint32_t)key[i]] = group_col[g - 1] + (i - group_pos[g - 1]) * L;
  }
}

constexpr int kShrinkTokens = 4;

// u of up to four tokens of a request: a warp per low-rank row, its lanes over
// the inner dimension.  The sorted form also moves the tokens to their columns
// and splits u into 16-bit parts.
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
  if (kSorted) {
    col = o.req_col[req] + l0;
    uint4 *to = reinterpret_cast<uint4 *>(static_cast<T *>(o.hidden) + (uint64_t)col * a.dim);
    const uint4 *from = reinterpret_cast<const uint4 *>(h);
    for (uint32_t i = threadIdx.x; i < count * (a.dim / 8); i += 256) to[i] = from[i];
    if (threadIdx.x < count) {
      const int32_t t = (int32_t)(tok + threadIdx.x);
      o.col_token[col + threadIdx.x] = has || id == -1 ? t : -2 - t;
    }
    if (!has) return;  // its columns take no part in any group's products
  }
  for (uint32_t r = threadIdx.x >> 5; r < a.rank; r += 8) {
    float s[kShrinkTokens] = {};
    if (has) {
      const T *w = static_cast<const T *>(a.lora_a) + ((uint64_t)id * a.rank + r) * a.dim;
      for (uint32_t d = lane * 8; d < a.dim; d += 256) {
        float y[8];
        unpack8<T>(__ldg(reinterpret_cast<const uint4 *>(w + d)), y);
#pragma unroll
        for (int q = 0; q < kShrinkTokens; ++q) {
          if (q >= (int)count) break;
          float x[8];
          unpack8<T>(__ldg(reinterpret_cast<const uint4 *>(h + (uint64_t)q * a.dim + d)), x);
#pragma unroll
          for (int e = 0; e < 8; ++e) s[q] = fmaf(x[e], y[e], s[q]);
        }
      }
#pragma unroll
      for (int q = 0; q < kShrinkTokens; ++q) {
#pragma unroll
        for (int d = 16; d; d >>= 1) s[q] += __shfl_xor_sync(~0u, s[q], d);
        s[q] *= a.scale ? a.scale[id] : 1.0f;
      }
    }
    if (lane < count) {
      float v = s[0];
#pragma unroll
      for (int q = 1; q < kShrinkTokens; ++q) v = lane == q ? s[q] : v;
      if (!kSorted) {
        u[(tok + lane) * a.rank + r] = v;
      } else {
        for (uint32_t part = 0; part < o.parts; ++part) {
          T x;
          from_f32(v, x);
          static_cast<T *>(o.u)[((uint64_t)part * o.columns + col + lane) * a.rank + r] = x;
          // What is left for the next part; nothing behind an infinity.
          const float back = to_f32(x);
          v = fabsf(back) < -kNegInf ? v - back : 0.0f;
        }
      }
    }
  }
}

struct LogitsPlan {
  uint32_t columns;    // tokens, or the sorted form's upper bound
  uint32_t tile_t;     // columns of a tile, a multiple of 16
  uint32_t tiles_t;
  uint32_t tiles_v;
  uint32_t stages;
  uint32_t tmem_half;  // columns of one of the two accumulators
};

struct alignas(8) LogitsShared {
  uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
  uint32_t tmem, gave_up;
};

LogitsPlan plan_logits(const ft_adapter_args &a, uint32_t columns) {
  LogitsPlan p;
  p.columns = columns;
  p.tiles_t = (columns + kMaxTileT - 1) / kMaxTileT;
  p.tile_t = ((columns + p.tiles_t - 1) / p.tiles_t + 15) / 16 * 16;
  p.tiles_v = (a.vocab + kTileV - 1) / kTileV;
  const uint32_t stage = (kTileV + p.tile_t) * kTileD * 2;
  p.stages = std::min<uint32_t>(kMaxStages, (225 * 1024) / stage);
  p.tmem_half = 32;
  while (p.tmem_half < p.tile_t) p.tmem_half *= 2;
  return p;
}
size_t logits_smem(const LogitsPlan &p) { return 1024 + (size_t)p.stages * (kTileV + p.tile_t) * kTileD * 2; }

// The stages of a tile in the order that loads and products both take them:
// the shared projection's, then those of each group that has columns in it.
// f(chunk) for the first; g(group, first column, width, rank offset, first
// part, parts) for the others.  A callback that returns false ends the walk.
template <typename F, typename G>
__device__ __forceinline__ bool walk_tile(const ft_adapter_args &a, const Sorted &o, bool sorted, uint32_t tile_t,
                                          uint32_t groups, uint32_t tt, uint32_t chunks, F &&f, G &&g) {
  for (uint32_t c = 0; c < chunks; ++c)
    if (!f(c)) return false;
  if (!sorted) return true;
  const uint32_t c0 = tt * tile_t, c1 = c0 + tile_t;
  for (uint32_t i = o.tile_first[tt]; i < groups; ++i) {
    const Group q = o.groups[i];
    if (q.col0 >= c1) break;
    if (q.adapter < 0) continue;
    const uint32_t w0 = max(q.col0, c0), w = min(q.col1, c1) - w0;
    const uint32_t at_once = min(o.parts, tile_t / w);
    for (uint32_t r = 0; r < a.rank; r += kTileD)
      for (uint32_t part = 0; part < o.parts; part += at_once)
        if (!g(q.adapter, w0, w, r, part, min(at_once, o.parts - part))) return false;
  }
  return true;
}

// Persistent, one CTA per SM.  Tiles that share a stretch of the weight are
// neighbours in the order, so that it comes from DRAM once.
template <typename T, typename O, bool kSorted>
__global__ void __launch_bounds__(kThreads, 1)
    logits_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_h,
                  const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_u,
                  ft_adapter_args a, LogitsPlan p, const float *u, Sorted o) {
  using namespace sm100;
  extern __shared__ uint8_t raw[];
  uint8_t *buf = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  __shared__ LogitsShared sh;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bytes_w = kTileV * kTileD * 2, bytes = bytes_w + p.tile_t * kTileD * 2;
  const uint32_t groups = kSorted ? o.head[0] : 0, columns = kSorted ? o.head[1] : p.columns;
  const uint32_t tiles_t = (columns + p.tile_t - 1) / p.tile_t;
  const uint32_t tiles = tiles_t * p.tiles_v, chunks = (a.dim + kTileD - 1) / kTileD;
  volatile uint32_t *gave_up = &sh.gave_up;
  if (threadIdx.x == 0) {
    sh.gave_up = 0;
    for (uint32_t s = 0; s < p.stages; ++s) mbar_init(&sh.full[s], 1), mbar_init(&sh.empty[s], 1);
    for (int b = 0; b < 2; ++b) mbar_init(&sh.acc_full[b], 1), mbar_init(&sh.acc_empty[b], kEpilogue);
    mbar_init_fence();
    prefetch_map(&map_w);
    prefetch_map(&map_h);
  }
  if (warp == 9) tmem_alloc(&sh.tmem, 2 * p.tmem_half);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;

  if (warp == 8) {
    if (elect_one()) {
      uint32_t at = 0, sent = 0;  // stage, and number of stages filled so far
      bool ok = true;
      auto take = [&](uint32_t expect) -> uint8_t * {  // the next stage, once it is free
        if (sent >= p.stages) ok = mbar_wait(&sh.empty[at], (sent / p.stages - 1) & 1, gave_up);
        if (!ok) return nullptr;
        mbar_expect(&sh.full[at], expect);
        return buf + (size_t)at * bytes;
      };
      auto next = [&] {
        ++sent;
        at = at + 1 == p.stages ? 0 : at + 1;
      };
      for (uint32_t tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
        const int32_t v0 = (int32_t)(tile / tiles_t * kTileV);
        const uint32_t tt = tile % tiles_t;
        walk_tile(
            a, o, kSorted, p.tile_t, groups, tt, chunks,
            [&](uint32_t c) {
              uint8_t *st = take(bytes);
              if (!st) return false;
              tma_load_2d(st, &map_w, &sh.full[at], (int32_t)(c * kTileD), v0);
              tma_load_2d(st + bytes_w, &map_h, &sh.full[at], (int32_t)(c * kTileD), (int32_t)(tt * p.tile_t));
              next();
              return true;
            },
            [&](int32_t adapter, uint32_t w0, uint32_t w, uint32_t r, uint32_t part, uint32_t parts) {
              uint8_t *st = take(bytes_w + parts * w * kTileD * 2);
              if (!st) return false;
              tma_load_3d(st, &map_b, &sh.full[at], (int32_t)r, v0, adapter);
              for (uint32_t x = 0; x < parts; ++x)
                for (uint32_t i = 0; i < w; i += 16)
                  tma_load_2d(st + bytes_w + (x * w + i) * kTileD * 2, &map_u, &sh.full[at], (int32_t)r,
                              (int32_t)((part + x) * o.columns + w0 + i));
              next();
              return true;
            });
      }
      // Copies must not land in a block that has ended: wait for the last fill
      // of each stage (the products saw all of them full if nothing failed).
      if (!ok)
        for (uint32_t s = 0; s < p.stages && s < sent; ++s) {
          const uint32_t fill = (sent - 1 - s) / p.stages;
          for (uint32_t i = 0; i < kWaitTries && !mbar_try(&sh.full[s], fill & 1); ++i) {
          }
        }
    }
  } else if (warp == 9) {
    if (elect_one()) {
      constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
      uint32_t at = 0, phase = 0, n = 0;
      bool ok = true;
      auto done = [&] {  // the stage is free when the products so far have ended
        mma_commit(&sh.empty[at]);
        if (++at == p.stages) at = 0, phase ^= 1;
      };
      for (uint32_t tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, ++n) {
        const uint32_t b = n & 1, d = tmem + b * p.tmem_half, tt = tile % tiles_t, c0 = tt * p.tile_t;
        const uint32_t shape = mma_shape(kBf16, kTileV, min(p.tile_t, (columns - c0 + 15) / 16 * 16));
        if (n >= 2) ok = mbar_wait(&sh.acc_empty[b], (n / 2 - 1) & 1, gave_up);
        if (!ok) break;
        fence_after();
        ok = walk_tile(
            a, o, kSorted, p.tile_t, groups, tt, chunks,
            [&](uint32_t c) {
              if (!mbar_wait(&sh.full[at], phase, gave_up)) return false;
              fence_after();
              const uint64_t w = operand(buf + (size_t)at * bytes), h = operand(buf + (size_t)at * bytes + bytes_w);
#pragma unroll
              for (int k = 0; k < kTileD / 16; ++k) mma_f16(d, w + 2 * k, h + 2 * k, shape, c > 0 || k > 0);
              done();
              return true;
            },
            [&](int32_t, uint32_t w0, uint32_t w, uint32_t r, uint32_t, uint32_t parts) {
              if (!mbar_wait(&sh.full[at], phase, gave_up)) return false;
              fence_after();
              const uint8_t *st = buf + (size_t)at * bytes;
              const uint64_t bw = operand(st);
              const uint32_t steps = (min(a.rank - r, (uint32_t)kTileD) + 15) / 16, narrow = mma_shape(kBf16, kTileV, w);
              for (uint32_t x = 0; x < parts; ++x) {
                const uint64_t uw = operand(st + bytes_w + x * w * kTileD * 2);
                for (uint32_t k = 0; k < steps; ++k) mma_f16(d + (w0 - c0), bw + 2 * k, uw + 2 * k, narrow, true);
              }
              done();
              return true;
            });
        if (ok) mma_commit(&sh.acc_full[b]);
      }
    }
  } else {
    // Warps w and w + 4 read the same quarter of tensor memory (its lanes
    // 32 (w % 4) on); they take alternate blocks of 16 columns.
    uint32_t n = 0;
    bool ok = true;
    const uint32_t row = (warp & 3) * 32 + lane;
    for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++n) {
      const uint32_t b = n & 1, t0 = tile % tiles_t * p.tile_t;
      const uint32_t v = tile / tiles_t * kTileV + row;
      const bool live = v < a.vocab;
      const uint32_t count = min(p.tile_t, columns - t0);
      if (ok) ok = mbar_wait(&sh.acc_full[b], (n / 2) & 1, gave_up);
      ok = __all_sync(~0u, ok);
      if (ok) fence_after();
      for (uint32_t c0 = (warp >> 2) * 16; c0 < count; c0 += 32) {
        // Lane e (and e + 16) looks up what column c0 + e is.
        const uint32_t mine = t0 + c0 + (lane & 15);
        int32_t token = -1, id = -1;
        if (c0 + (lane & 15) < count) {
          token = kSorted ? o.col_token[mine] : (int32_t)mine;
          if (!kSorted && u) id = a.adapter_ids[mine / a.num_outpos];
        }
        uint32_t acc[16];
        if (ok) {
          tmem_load16(tmem + b * p.tmem_half + c0 + ((warp & 3) << 21), acc);
        } else {
          // A wait ran out: no result is better than a wrong one.
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[e] = 0x7FC00000;
        }
        if (!kSorted && u) {
          // The low-rank part in 32 bits; all 16 rows of B on their way before
          // the first is used.
          const uint32_t any = __ballot_sync(~0u, (uint32_t)id < a.num_adapters) & 0xFFFF;
          const uint32_t wrong = __ballot_sync(~0u, (uint32_t)id >= a.num_adapters && id != -1) & 0xFFFF;
          const T *base = static_cast<const T *>(a.lora_b) + (uint64_t)(live ? v : 0) * a.rank;
          for (uint32_t r = 0; any && r < a.rank; r += 8) {
            uint4 w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int32_t at = __shfl_sync(~0u, id, e);
              const int32_t before = e ? __shfl_sync(~0u, id, e ? e - 1 : 0) : -1;
              if (any >> e & 1) {
                if (e && at == before)
                  w[e] = w[e ? e - 1 : 0];
                else
                  w[e] = __ldg(reinterpret_cast<const uint4 *>(base + (uint64_t)at * a.vocab * a.rank + r));
              } else {
                w[e] = make_uint4(0, 0, 0, 0);
              }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              if (any >> e & 1) {
                float y[8];
                unpack8<T>(w[e], y);
                const float4 *x = reinterpret_cast<const float4 *>(u + (uint64_t)(t0 + c0 + e) * a.rank + r);
                const float4 x0 = __ldg(x), x1 = __ldg(x + 1);
                float s = __uint_as_float(acc[e]);
                s = fmaf(x0.x, y[0], s), s = fmaf(x0.y, y[1], s), s = fmaf(x0.z, y[2], s), s = fmaf(x0.w, y[3], s);
                s = fmaf(x1.x, y[4], s), s = fmaf(x1.y, y[5], s), s = fmaf(x1.z, y[6], s), s = fmaf(x1.w, y[7], s);
                acc[e] = __float_as_uint(s);
              }
            }
          }
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (wrong >> e & 1) acc[e] = 0x7FC00000;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          int32_t to = __shfl_sync(~0u, token, e);
          float y = __uint_as_float(acc[e]);
          if (kSorted && to < -1) {
            to = -2 - to;
            y = __int_as_float(0x7FC00000);
          }
          if (live && to >= 0) from_f32(y, static_cast<O *>(a.out)[(uint64_t)to * a.vocab + v]);
        }
      }
      if (ok) {
        fence_before();
        mbar_arrive(&sh.acc_empty[b]);
      }
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 9) tmem_free(tmem, 2 * p.tmem_half);
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

// `layers` arrays of rows of `inner` 16-bit values, loaded as boxes of 64
// values by `box` rows with the 128-byte swizzle; what lies outside reads as 0.
CUtensorMap make_map(const void *base, bool bf16, uint64_t inner, uint64_t rows, uint64_t layers, uint32_t box,
                     const char *what) {
  CUtensorMap m;
  const cuuint64_t dims[3] = {inner, rows, layers}, strides[2] = {inner * 2, inner * rows * 2};
  const cuuint32_t tile[3] = {(cuuint32_t)kTileD, box, 1}, step[3] = {1, 1, 1};
  const CUresult rc =
      encode_fn()(&m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, layers ? 3 : 2,
                  const_cast<void *>(base), dims, strides, tile, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
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
  if ((uint64_t)a.n * a.num_outpos > 0x3FFFFF || a.vocab > 0x7FFFFF00u || a.dim > 0xFFFFFF ||
      (uint64_t)(a.vocab / kTileV + 1) * ((uint64_t)a.n * a.num_outpos / 16 + 1) > 0x7FFFFFFF)
    throw InvalidArgument("adapter_logits: too many tokens or too large a vocabulary");
}

uint64_t align256(uint64_t x) { return (x + 255) & ~(uint64_t)255; }

// Which form a call takes and where its workspace's parts lie.
struct Layout {
  bool sorted = false;
  uint32_t tokens = 0, columns = 0, parts = 0;
  uint64_t head = 0, groups = 0, tile_first = 0, req_col = 0, col_token = 0, hidden = 0, u = 0, end = 0;
};

Layout layout_of(const ft_adapter_args &a) {
  Layout l;
  l.tokens = l.columns = a.n * a.num_outpos;
  if (!a.num_adapters) return l;
  // Padding a group to a multiple of 16 columns adds at most 16 - gcd(L, 16).
  const uint64_t groups = std::min<uint64_t>(a.n, (uint64_t)a.num_adapters + 1);
  uint32_t step = 1;
  while (step < 16 && a.num_outpos % (2 * step) == 0) step *= 2;
  const uint64_t most = ((uint64_t)l.tokens + groups * (16 - step) + 15) / 16 * 16;
  l.sorted = a.n <= kMaxSortRequests && most <= 2 * (uint64_t)l.tokens;
  if (!l.sorted) {
    l.end = align256((uint64_t)l.tokens * a.rank * 4);
    return l;
  }
  l.columns = (uint32_t)most;
  l.parts = a.dtype == FT_DTYPE_BF16 && a.out_dtype == FT_DTYPE_F32 ? 3 : 2;
  uint64_t at = 256;
  auto place = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += align256(bytes);
    return here;
  };
  l.groups = place(sizeof(Group) * groups);
  l.tile_first = place(4 * (most / 16 + 1));
  l.req_col = place(4ull * a.n);
  l.col_token = place(4 * most);
  l.hidden = place(most * a.dim * 2);
  l.u = place(l.parts * most * a.rank * 2);
  l.end = at;
  return l;
}

}  // namespace

uint64_t adapter_logits_workspace(const ft_adapter_args &a) {
  check_adapter(a);
  return layout_of(a).end;
}

void adapter_logits_device(const ft_adapter_args &a, void *ws, uint64_t ws_bytes, cudaStream_t stream) {
  check_adapter(a);
  if (a.n == 0) return;
  const void *need[] = {a.hidden, a.weight, a.out};
  for (const void *p : need)
    if (!p) fail(ErrorKind::kNull, "MARISA_NULL_ERROR: adapter_logits: hidden, weight or out is NULL");
  if (a.num_adapters && (!a.adapter_ids || !a.lora_a || !a.lora_b))
    fail(ErrorKind::kNull, "MARISA_NULL_ERROR: adapter_logits: adapter_ids, lora_a or lora_b is NULL");
  const void *sixteen[] = {a.hidden, a.weight, a.num_adapters ? a.lora_a : nullptr, a.num_adapters ? a.lora_b : nullptr};
  for (const void *p : sixteen)
    if (reinterpret_cast<uintptr_t>(p) & 15)
      throw InvalidArgument("adapter_logits: hidden, weight, lora_a and lora_b must start on 16-byte boundaries");
  const Layout l = layout_of(a);
  if (ws_bytes < l.end || (l.end && (!ws || (reinterpret_cast<uintptr_t>(ws) & 255))))
    throw InvalidArgument("adapter_logits: needs a 256-byte aligned workspace of " + std::to_string(l.end) + " bytes");
  const LogitsPlan p = plan_logits(a, l.columns);
  uint8_t *w = static_cast<uint8_t *>(ws);
  float *u = a.num_adapters && !l.sorted ? reinterpret_cast<float *>(w) : nullptr;
  Sorted o{};
  if (l.sorted)
    o = Sorted{reinterpret_cast<uint32_t *>(w + l.head),    reinterpret_cast<Group *>(w + l.groups),
               reinterpret_cast<uint32_t *>(w + l.tile_first), reinterpret_cast<uint32_t *>(w + l.req_col),
               reinterpret_cast<int32_t *>(w + l.col_token), w + l.hidden,
               w + l.u,                                      l.columns,
               l.parts};
  const bool bf16 = a.dtype == FT_DTYPE_BF16;
  const CUtensorMap map_w = make_map(a.weight, bf16, a.dim, a.vocab, 0, kTileV, "weight");
  const CUtensorMap map_h = make_map(l.sorted ? o.hidden : a.hidden, bf16, a.dim, l.columns, 0, p.tile_t, "hidden");
  CUtensorMap map_b = map_w, map_u = map_w;
  if (l.sorted) {
    map_b = make_map(a.lora_b, bf16, a.rank, a.vocab, a.num_adapters, kTileV, "lora_b");
    map_u = make_map(o.u, bf16, a.rank, (uint64_t)l.parts * l.columns, 0, 16, "the low-rank values");
  }
  const size_t smem = logits_smem(p);
  const unsigned grid = std::min<unsigned>(p.tiles_t * p.tiles_v, (unsigned)sm_count());
  const unsigned shrink = a.n * ((a.num_outpos + kShrinkTokens - 1) / kShrinkTokens);
  if (l.sorted) {
    uint32_t slots = 2;
    while (slots < a.n) slots <<= 1;
    const size_t room = 16ull * slots;
    if (room > 32 * 1024)
      CUDA_TRY(cudaFuncSetAttribute(order_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)room));
    order_kernel<<<1, 1024, room, stream>>>(a.adapter_ids, a.n, a.num_outpos, a.num_adapters, slots, p.tile_t, o);
    CUDA_TRY(cudaGetLastError());
  }
  auto launch = [&](auto *kernel) {
    CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kernel<<<grid, kThreads, smem, stream>>>(map_w, map_h, map_b, map_u, a, p, u, o);
    CUDA_TRY(cudaGetLastError());
  };
  auto run = [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (l.sorted)
      shrink_kernel<T, true><<<shrink, 256, 0, stream>>>(a, u, o);
    else if (u)
      shrink_kernel<T, false><<<shrink, 256, 0, stream>>>(a, u, o);
    CUDA_TRY(cudaGetLastError());
    if (l.sorted)
      a.out_dtype == FT_DTYPE_F32 ? launch(logits_kernel<T, float, true>) : launch(logits_kernel<T, T, true>);
    else
      a.out_dtype == FT_DTYPE_F32 ? launch(logits_kernel<T, float, false>) : launch(logits_kernel<T, T, false>);
  };
  if (bf16)
    run((__nv_bfloat16 *)nullptr);
  else
    run((__half *)nullptr);
}

}  // namespace ftb
