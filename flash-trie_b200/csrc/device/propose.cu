// The search's proposals from a model's logits: per row the log-softmax over
// the vocabulary and its k largest entries, exact, equal logits in order of
// the token id.
//
//   logp[v] = x[v] - m - log(sum_u exp(x[u] - m)),  m = max_u x[u]
//
// The entries are ordered by the 64-bit key (logit as an ordered integer,
// complement of the id), which no two share, so the k-th largest key separates
// the proposals from the rest.
//
// The logits are read once.  A row is cut into stretches, a CTA each.  A
// sample spread over the row gives a bound that a little more than k entries
// should pass; the CTA streams its stretch, adds to the softmax sum and notes
// the vectors in which something passes the bound (a few instructions; taking
// the entries out at once would cost a fifth of the stream's time); then it
// fetches those again and keeps what passes.  The CTA that ends last in its row
// joins the sums, selects the k largest of what all have kept, and sorts them.
// The bound is a guess only: a stretch that keeps more than fits is read again
// with a bound that rises (`careful`), and a row that kept fewer than k is read
// again by its last CTA without one.
//
// Large batches are bound by the logits' bytes: 93 us for 256 rows of 500009 f32
// (512 MB, 5.5 TB/s), k 256, a CTA per row.  One request is bound by latency
// around its stream: 47.3 us for 20 rows of 2.2M bf16 (88 MB, 13.5 us at the
// copy rate), k 1000; 14.7 us for 8 rows of 32000 f32, k 64.
#include <algorithm>
#include <string>

#include "../engine.hpp"
#include "cuda_util.hpp"
#include "head_ops.hpp"
#include "row_stream.cuh"

namespace ftb {
namespace {

constexpr int kThreads = 512;
constexpr uint32_t kBins = 2048;
constexpr float kFltMax = 3.402823466e+38f;

typedef unsigned long long Key;

// Order-preserving integer of a float; -0 and 0 are the same.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(__fadd_rn(x, 0.0f));
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ Key key_of(float x, int64_t id) { return (Key)ordered(x) << 32 | (uint32_t)~(uint32_t)id; }

struct ProposePlan {
  uint32_t chunks;      // CTAs per row
  uint32_t cap;         // entries that a CTA can keep
  uint32_t hits;        // vectors that it can note
  uint32_t emit;        // entries that a CTA hands on
  uint32_t slots;       // power of two >= k and 64
  uint64_t vecs_chunk;  // 16-byte vectors per stretch
};

constexpr uint32_t kFew = 256;  // entries of a bin that are ranked by counting

struct Shared {
  uint32_t hist[kBins];
  Key few[kFew];
  Key least;
  uint32_t scan[kThreads / 32];
  Key low[kThreads / 32], high[kThreads / 32];
  SoftSum sums[kThreads / 32];
  SoftSum sum;
  uint32_t count, hits, bin, above, low32, high32;
  bool last;
};

// The bin, from the top, in which the need-th entry lies, and the number of
// entries above it; bin kBins if there are fewer.
__device__ void find_bin(Shared &sh, uint32_t need, uint32_t &bin, uint32_t &above) {
  constexpr int kPer = kBins / kThreads;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  uint32_t mine[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) sum += mine[i] = sh.hist[kBins - 1 - (threadIdx.x * kPer + i)];
  uint32_t s = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(~0u, s, d);
    if (lane >= (uint32_t)d) s += o;
  }
  if (lane == 31) sh.scan[warp] = s;
  if (threadIdx.x == 0) sh.bin = kBins, sh.above = 0;
  __syncthreads();
  uint32_t before = s - sum;
  for (uint32_t w = 0; w < warp; ++w) before += sh.scan[w];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (before < need && before + mine[i] >= need) sh.bin = kBins - 1 - (threadIdx.x * kPer + i), sh.above = before;
    before += mine[i];
  }
  __syncthreads();
  bin = sh.bin;
  above = sh.above;
}

__device__ void clear_bins(Shared &sh) {
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < kBins; b += kThreads) sh.hist[b] = 0;
  __syncthreads();
}

__device__ void block_range(Shared &sh, Key &low, Key &high) {
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    low = min(low, (Key)__shfl_xor_sync(~0u, low, d));
    high = max(high, (Key)__shfl_xor_sync(~0u, high, d));
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.low[threadIdx.x >> 5] = low, sh.high[threadIdx.x >> 5] = high;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) low = min(low, sh.low[w]), high = max(high, sh.high[w]);
}

// Keeps the entries of list[0, count) that are not below the returned key: at
// least the k largest, and at most k + slack.  Radix selection, 11 bits a
// pass, from the highest bit in which the entries differ.  count >= k.  With
// low <= high at least k entries are known to lie in [low, high] and none above.
__device__ Key keep_largest(Shared &sh, Key *list, uint32_t count, uint32_t k, uint32_t slack, Key low = ~0ull,
                            Key high = 0) {
  if (low > high) {
    for (uint32_t i = threadIdx.x; i < count; i += kThreads) low = min(low, list[i]), high = max(high, list[i]);
    block_range(sh, low, high);
  }
  uint32_t need = k, sure = 0;
  for (;;) {
    const Key span = high - low;
    const int bits = span ? 64 - __clzll((long long)span) : 0, shift = bits > 11 ? bits - 11 : 0;
    clear_bins(sh);
    for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
      const Key x = list[i];
      if (x >= low && x <= high) atomicAdd(&sh.hist[(uint32_t)((x - low) >> shift)], 1u);
    }
    uint32_t bin, above;
    find_bin(sh, need, bin, above);
    const uint32_t in_bin = sh.hist[bin];
    low += (Key)bin << shift;
    if (shift == 0 || sure + above + in_bin <= k + slack) break;
    high = min(high, low + (((Key)1 << shift) - 1));
    need -= above;
    sure += above;
    if (in_bin <= kFew) {
      // Each entry of the bin counts those above it: the need-th is the one.
      if (threadIdx.x == 0) sh.count = 0;
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
        const Key x = list[i];
        if (x >= low && x <= high) sh.few[atomicAdd(&sh.count, 1u)] = x;
      }
      __syncthreads();
      if (threadIdx.x < in_bin) {
        const Key x = sh.few[threadIdx.x];
        uint32_t rank = 0;
        for (uint32_t i = 0; i < in_bin; ++i) rank += sh.few[i] > x;
        if (rank == need - 1) sh.least = x;
      }
      __syncthreads();
      low = sh.least;
      break;
    }
  }
  // In place: a round's entries are read before any is written, and no write
  // goes beyond the entries read so far. A warp asks for its places at once.
  constexpr int kRound = 4;
  __syncthreads();
  if (threadIdx.x == 0) sh.count = 0;
  for (uint32_t i0 = 0; i0 < count; i0 += kRound * kThreads) {
    Key x[kRound];
    uint32_t votes[kRound], all = 0;
#pragma unroll
    for (int q = 0; q < kRound; ++q) {
      const uint32_t i = i0 + q * kThreads + threadIdx.x;
      x[q] = i < count ? list[i] : 0;
      votes[q] = __ballot_sync(~0u, i < count && x[q] >= low);
      all += __popc(votes[q]);
    }
    __syncthreads();
    const uint32_t lane = threadIdx.x & 31;
    uint32_t at = 0;
    if (lane == 0 && all) at = atomicAdd(&sh.count, all);
    at = __shfl_sync(~0u, at, 0);
#pragma unroll
    for (int q = 0; q < kRound; ++q) {
      if (votes[q] >> lane & 1) list[at + __popc(votes[q] & ((1u << lane) - 1))] = x[q];
      at += __popc(votes[q]);
    }
    if (i0 + kRound * kThreads < count) __syncthreads();
  }
  __syncthreads();
  return low;
}

__device__ __forceinline__ void exchange(Key &x, Key other, bool smaller) {
  if ((other < x) == smaller) x = other;
}

// Ascending bitonic sort of list[0, slots), a power of two of at least 64.
// Steps within 64 entries run in the registers of a warp, two entries a lane.
__device__ void sort_ascending(Key *list, uint32_t slots) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto in_warps = [&](uint32_t size, uint32_t last) {  // the steps below 64 of stages size..last
    for (uint32_t base = warp * 64; base < slots; base += kThreads * 2) {
      Key x = list[base + lane], y = list[base + lane + 32];
      for (uint32_t z = size; z <= last; z <<= 1) {
        if (z >= 64) {
          const bool up = (base & z) == 0;
          if ((x > y) == up) {
            const Key t = x;
            x = y, y = t;
          }
        }
        for (uint32_t step = min(z, 32u * 2) / 2 == 32 ? 16 : z / 2; step; step >>= 1) {
          const bool first = (lane & step) == 0;
          exchange(x, __shfl_xor_sync(~0u, x, step), first == (((base + lane) & z) == 0));
          exchange(y, __shfl_xor_sync(~0u, y, step), first == (((base + lane + 32) & z) == 0));
        }
      }
      list[base + lane] = x, list[base + lane + 32] = y;
    }
    __syncthreads();
  };
  __syncthreads();
  in_warps(2, 64);
  for (uint32_t size = 128; size <= slots; size <<= 1) {
    for (uint32_t step = size >> 1; step >= 64; step >>= 1) {
      for (uint32_t i = threadIdx.x; i < slots / 2; i += kThreads) {
        const uint32_t a = 2 * i - (i & (step - 1)), b = a + step;
        const bool up = (a & size) == 0;
        const Key x = list[a], y = list[b];
        if ((x > y) == up) list[a] = y, list[b] = x;
      }
      __syncthreads();
    }
    in_warps(size, size);
  }
}

// One stretch with a bound that rises: whenever the next step might not fit,
// all but the k largest (and a little more) go.  The ids rise, so what equals
// the bound's logit later on comes after k others.
template <typename T>
__device__ void careful(Shared &sh, Key *list, const RowVecs<T> &r, int64_t v0, int64_t v1, uint32_t k, uint32_t cap) {
  constexpr int N = RowVecs<T>::N;
  float bound = kNegInf;
  __syncthreads();
  if (threadIdx.x == 0) sh.count = 0;
  for (int64_t i0 = v0; i0 < v1; i0 += kThreads) {
    __syncthreads();
    const uint32_t count = sh.count;
    if (count + kThreads * N > cap) bound = unordered((uint32_t)(keep_largest(sh, list, count, k, 256) >> 32));
    __syncthreads();
    const int64_t i = i0 + threadIdx.x;
    if (i < v1) {
      float v[N];
      if (r.whole(i))
        unpack(r.load_whole(i), v, (const T *)nullptr);
      else
        r.load_edge(i, v);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (v[e] > bound) list[atomicAdd(&sh.count, 1u)] = key_of(v[e], r.first(i) + e);
    }
  }
  __syncthreads();
}

// A bound below the row's k-th largest logit, from a sample of it: groups of
// eight vectors in the middle of equal parts of the row. Small parts matter: a
// vocabulary in order of frequency has its best logits at one end, and with
// long stretches the sample would see too many of them or none; single vectors
// cost three times as much to fetch.
template <typename T>
__device__ float sample_bound(Shared &sh, const RowVecs<T> &r, uint32_t k) {
  constexpr int N = RowVecs<T>::N, kLoads = 4;
  const int64_t vecs = r.count();
  const int loads = (int)max((int64_t)1, min((int64_t)kLoads, vecs / (2 * kThreads))), parts = loads * kThreads / 8;
  const int64_t each = vecs / parts;
  uint4 q[kLoads];
  int64_t at[kLoads];
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const int part = (u * kThreads + (int)threadIdx.x) / 8;
    at[u] = u < loads ? part * each + each / 2 + threadIdx.x % 8 : vecs;  // vecs: nothing
    if (r.whole(at[u])) q[u] = r.load_whole(at[u]);
  }
  for (uint32_t b = threadIdx.x; b < kBins; b += kThreads) sh.hist[b] = 0;
  if (threadIdx.x == 0) sh.low32 = 0xFFFFFFFFu, sh.high32 = 0;
  __syncthreads();
  // The k-th logit is expected at rank k (sample size) / V of the sample, give or
  // take its square root; four of them and 4 more are left for safety (a row
  // for which that is too few is read again).
  const float rank = (float)k * (float)(loads * kThreads * N) / (float)r.len;
  const uint32_t need = (uint32_t)(rank + 4.0f * sqrtf(rank)) + 4;
  // The best `need` of the sample are hardly ever two in one vector while they
  // are few: each vector's best then stands for it (an eighth of the work), and
  // where two meet the bound is a little low.
  const bool few = need <= kThreads / 8;
  uint32_t key[kLoads][N];
  uint32_t low = 0xFFFFFFFFu, high = 0;
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    float v[N];
    if (r.whole(at[u]))
      unpack(q[u], v, (const T *)nullptr);
    else
      r.load_edge(at[u], v);
    if (few) {
#pragma unroll
      for (int e = 1; e < N; ++e) v[0] = fmaxf(v[0], v[e]), v[e] = kNegInf;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (few && e) break;
      key[u][e] = v[e] > kNegInf ? ordered(v[e]) : 0;
      if (key[u][e]) low = min(low, key[u][e]), high = max(high, key[u][e]);
    }
  }
  low = __reduce_min_sync(~0u, low), high = __reduce_max_sync(~0u, high);
  if ((threadIdx.x & 31) == 0) atomicMin(&sh.low32, low), atomicMax(&sh.high32, high);
  __syncthreads();
  low = sh.low32, high = sh.high32;
  if (high == 0) return kNegInf;
  const uint32_t span = high - low;
  const int bits = 32 - __clz((int)span), shift = bits > 11 ? bits - 11 : 0;
#pragma unroll
  for (int u = 0; u < kLoads; ++u)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (few && e) break;
      if (key[u][e]) atomicAdd(&sh.hist[(key[u][e] - low) >> shift], 1u);
    }
  uint32_t bin, above;
  find_bin(sh, need, bin, above);
  if (bin == kBins) return kNegInf;
  // The bin's least logit still passes. Below 0 comes the largest negative
  // number, not -0, which 0 would not pass.
  const uint32_t least = low + (bin << shift) - 1;
  return unordered(least - (least == 0x7FFFFFFFu));
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
    propose_kernel(const T *logits, uint32_t vocab, uint32_t k, int order, ProposePlan p, SoftSum *part, uint32_t *counts,
                   uint32_t *tickets, Key *kept, uint32_t *out_id, float *out_lp) {
  extern __shared__ Key list[];  // [cap], then u32 [hits]
  uint32_t *hit = reinterpret_cast<uint32_t *>(list + p.cap);
  __shared__ Shared sh;
  constexpr int N = RowVecs<T>::N;
  const uint64_t row = blockIdx.x / p.chunks;
  const uint32_t chunk = blockIdx.x % p.chunks;
  const RowVecs<T> r(logits + row * vocab, vocab);
  const int64_t v0 = (int64_t)(chunk * p.vecs_chunk), v1 = min(v0 + (int64_t)p.vecs_chunk, r.count());
  if (threadIdx.x == 0) sh.count = sh.hits = 0;
  const bool sampled = vocab > p.cap;
  const float bound = sampled ? sample_bound(sh, r, k) : kNegInf;
  __syncthreads();
  auto note = [&](int64_t i, float top) {
    if (top > bound) {
      const uint32_t at = atomicAdd(&sh.hits, 1u);
      if (at < p.hits) hit[at] = (uint32_t)(i - v0);
    }
  };
  // Four vectors of each thread on their way while four are added up; three
  // are 3% slower, five no faster on bf16, and eight that are added up as soon
  // as they are all there 7%: the CTAs of a row that fits on the GPU at once
  // start together, and between the steps nothing would be on its way.
  SoftSum s = soft_stream<T, kThreads, 4>(r, v0, v1, bound, note);
  s = soft_join_block<kThreads>(s, sh.sums);  // a barrier: all hits are noted
  const uint32_t hits = sh.hits;
  if (hits <= p.hits)
    for (uint32_t h = threadIdx.x; h < hits; h += kThreads) {
      const int64_t i = v0 + hit[h];
      float v[N];
      if (r.whole(i))
        unpack(r.load_whole(i), v, (const T *)nullptr);
      else
        r.load_edge(i, v);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (v[e] > bound) {
          const uint32_t at = atomicAdd(&sh.count, 1u);
          if (at < p.cap) list[at] = key_of(v[e], r.first(i) + e);
        }
    }
  __syncthreads();
  uint32_t count = sh.count;
  if (hits > p.hits || count > p.cap) {
    careful(sh, list, r, v0, v1, k, p.cap);
    count = sh.count;
  }
  if (p.chunks > 1) {
    // Hand the stretch's sum and entries on; the row's last CTA goes on alone.
    if (count > p.emit) {
      keep_largest(sh, list, count, k, 256);
      count = sh.count;
    }
    Key *to = kept + (uint64_t)blockIdx.x * p.emit;
    for (uint32_t i = threadIdx.x; i < count; i += kThreads) to[i] = list[i];
    __syncthreads();
    if (threadIdx.x == 0) {
      part[blockIdx.x] = s;
      counts[blockIdx.x] = count;
      __threadfence();
      sh.last = atomicAdd(&tickets[row], 1u) == p.chunks - 1;
    }
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    // Every thread looks up the same counts (64 at most) and sums.
    uint32_t total = 0;
    s = SoftSum::none();
    const uint64_t first = row * p.chunks;
    if (threadIdx.x < p.chunks) sh.hist[threadIdx.x] = __ldcg(&counts[first + threadIdx.x]);
    if (threadIdx.x == 0) sh.count = 0;
    if (threadIdx.x < 32) {
      for (uint32_t c = threadIdx.x; c < p.chunks; c += 32)
        s = soft_join(s, SoftSum{__ldcg(&part[first + c].m), __ldcg(&part[first + c].z)});
      s = soft_join_warp(s);
    }
    __syncthreads();
    uint32_t *before = sh.hist + 64;  // entries of the stretches before each
    for (uint32_t c = 0; c < p.chunks; ++c) {
      if (threadIdx.x == c) before[c] = total;
      total += sh.hist[c];
    }
    __syncthreads();
    if (total <= p.cap) {
      // Each entry to its place: most come from few stretches, so that the threads
      // share all entries and look up where each one is.
#pragma unroll 4
      for (uint32_t i = threadIdx.x; i < total; i += kThreads) {
        uint32_t c = 0;
        for (uint32_t step = 32; step; step >>= 1)
          if (c + step < p.chunks && before[c + step] <= i) c += step;
        list[i] = __ldcg(&kept[(first + c) * p.emit + (i - before[c])]);
      }
      count = total;
    } else {
      Key least = 0;
      for (uint32_t c = 0; c < p.chunks; ++c) {
        const uint32_t have = __ldcg(&counts[first + c]);
        __syncthreads();
        count = sh.count;
        if (count + have > p.cap) least = keep_largest(sh, list, count, k, 0);  // k + emit fit, no more
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < have; i += kThreads) {
          const Key x = __ldcg(&kept[(first + c) * p.emit + i]);
          if (x >= least) list[atomicAdd(&sh.count, 1u)] = x;
        }
      }
      __syncthreads();
      count = sh.count;
    }
    __syncthreads();
  }
  bool bounded = sampled && bound > kNegInf;  // k entries above the bound are in the list
  if (bounded && count < k) {
    careful(sh, list, r, 0, r.count(), k, p.cap);
    count = sh.count;
    bounded = false;
  }
  if (threadIdx.x == 0) sh.sum = s;
  __syncthreads();
  s = sh.sum;
  if (!s.valid()) count = 0;
  if (count > k) {
    if (bounded)
      keep_largest(sh, list, count, k, 0, (Key)ordered(bound) << 32, (Key)ordered(s.m) << 32 | 0xFFFFFFFFu);
    else
      keep_largest(sh, list, count, k, 0);
    count = sh.count;
  }
  // Ascending by (id) or by (falling logit, id).
  for (uint32_t i = threadIdx.x; i < p.slots; i += kThreads) {
    Key x = ~0ull;
    if (i < count) {
      const uint32_t id = ~(uint32_t)list[i], v = (uint32_t)(list[i] >> 32);
      x = order == 0 ? (Key)id << 32 | v : (Key)~v << 32 | id;
    }
    list[i] = x;
  }
  sort_ascending(list, p.slots);
  const float logz = logf(s.z);
  for (uint32_t i = threadIdx.x; i < k; i += kThreads) {
    uint32_t id = 0xFFFFFFFFu;
    float lp = -kFltMax;
    if (i < count) {
      const Key e = list[i];
      id = order == 0 ? (uint32_t)(e >> 32) : (uint32_t)e;
      const uint32_t v = order == 0 ? (uint32_t)e : ~(uint32_t)(e >> 32);
      lp = (unordered(v) - s.m) - logz;
    }
    out_id[row * k + i] = id;
    out_lp[row * k + i] = lp;
  }
}

void check_propose(const ft_propose_args &a) {
  if (a.dtype != FT_DTYPE_F32 && a.dtype != FT_DTYPE_BF16 && a.dtype != FT_DTYPE_F16)
    throw InvalidArgument("propose: unknown dtype");
  if (a.vocab == 0 || a.vocab == 0xFFFFFFFFu) throw InvalidArgument("propose: vocab must be positive and below 2^32 - 1");
  if (a.topk == 0 || a.topk > kMaxTopk)
    throw InvalidArgument("propose: topk must be in [1, " + std::to_string(kMaxTopk) + "]");
  if (a.order != 0 && a.order != 1) throw InvalidArgument("propose: order must be 0 (by id) or 1 (by log-probability)");
  if (a.rows > 0x7FFFFFFF) throw InvalidArgument("propose: too many rows");
}

uint64_t align256(uint64_t x) { return (x + 255) & ~(uint64_t)255; }

struct Layout {
  ProposePlan p;
  uint64_t part, counts, tickets, kept, end;
};

Layout layout_of(const ft_propose_args &a) {
  Layout l;
  ProposePlan &p = l.p;
  p.slots = 64;
  while (p.slots < a.topk) p.slots <<= 1;
  // Room for what passes the sampled bound: a few thousand entries for small
  // k, up to 1.9 k for large; 96 KB at k = 1000, so that two CTAs fit on an SM.
  // `careful` needs room for topk + 256 and a step of all threads.
  p.cap = std::max(a.topk + 512 + kThreads * 8, 2 * a.topk + 4096);
  p.hits = std::min(4096 + a.topk / 2 * 3, (uint32_t)(225 * 1024 - sizeof(Shared) - 8 * p.cap) / 4);
  p.emit = a.topk + 4096;  // cap - emit >= topk: a list that lacks room for another has topk entries
  const uint64_t vecs = ((uint64_t)a.vocab * (a.dtype == FT_DTYPE_F32 ? 4 : 2) + 15) / 16 + 1;
  const uint64_t slots = 148 * 2;
  uint64_t chunks = a.rows ? (a.rows >= slots ? 1 : slots / a.rows) : 1;
  chunks = std::max<uint64_t>(1, std::min<uint64_t>({chunks, (vecs + 2047) / 2048, 64}));
  p.vecs_chunk = (vecs + chunks - 1) / chunks;
  p.chunks = (uint32_t)((vecs + p.vecs_chunk - 1) / p.vecs_chunk);
  const uint64_t ctas = p.chunks > 1 ? a.rows * p.chunks : 0;
  l.part = 0;
  l.counts = align256(sizeof(SoftSum) * ctas);
  l.tickets = l.counts + align256(4 * ctas);
  l.kept = l.tickets + align256(p.chunks > 1 ? 4 * a.rows : 0);
  l.end = l.kept + align256(8 * ctas * p.emit);
  return l;
}

}  // namespace

uint64_t propose_workspace(const ft_propose_args &a) {
  check_propose(a);
  return layout_of(a).end;
}

void propose_device(const ft_propose_args &a, void *ws, uint64_t ws_bytes, cudaStream_t stream) {
  check_propose(a);
  if (a.rows == 0) return;
  if (!a.logits || !a.topk_id || !a.topk_logp)
    fail(ErrorKind::kNull, "MARISA_NULL_ERROR: propose: logits, topk_id or topk_logp is NULL");
  if (reinterpret_cast<uintptr_t>(a.logits) % (a.dtype == FT_DTYPE_F32 ? 4 : 2))
    throw InvalidArgument("propose: logits is not aligned to its elements");
  const Layout l = layout_of(a);
  if (ws_bytes < l.end || (l.end && (!ws || (reinterpret_cast<uintptr_t>(ws) & 255))))
    throw InvalidArgument("propose: needs a 256-byte aligned workspace of " + std::to_string(l.end) + " bytes");
  uint8_t *w = static_cast<uint8_t *>(ws);
  if (l.p.chunks > 1) CUDA_TRY(cudaMemsetAsync(w + l.tickets, 0, 4 * a.rows, stream));
  const size_t smem = 8ull * l.p.cap + 4ull * l.p.hits;
  auto run = [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    allow_shared(propose_kernel<T>, 225 * 1024 - (int)sizeof(Shared));
    propose_kernel<T><<<(unsigned)(a.rows * l.p.chunks), kThreads, smem, stream>>>(
        static_cast<const T *>(a.logits), a.vocab, a.topk, a.order, l.p, reinterpret_cast<SoftSum *>(w + l.part),
        reinterpret_cast<uint32_t *>(w + l.counts), reinterpret_cast<uint32_t *>(w + l.tickets),
        reinterpret_cast<Key *>(w + l.kept), a.topk_id, a.topk_logp);
    CUDA_TRY(cudaGetLastError());
  };
  if (a.dtype == FT_DTYPE_F32)
    run((float *)nullptr);
  else if (a.dtype == FT_DTYPE_BF16)
    run((__nv_bfloat16 *)nullptr);
  else
    run((__half *)nullptr);
}

}  // namespace ftb
