// Scores of candidate sequences under a model's logits, the preference loss
// on pairs of them, and the gradient of the logits.
//
//   logp_j = sum_{l < len_j} (x[l, tok_jl] - lse_l)
//   d/dx[l, v] = sum_j w_j [l < len_j] ([tok_jl = v] - exp(x[l, v] - lse_l))
//
// All candidates of a request share its logits, so one pass over a row gives
// its (maximum, sum) for every candidate, and in the gradient the candidates'
// softmax parts add up to one number per row, W_l = sum of w_j over the live
// ones: a row's gradient is -W_l p[v], put right at the at most C distinct
// tokens.  Both passes are bound by the bytes of the logits.
#include <algorithm>
#include <cmath>
#include <string>

#include "../engine.hpp"
#include "cuda_util.hpp"
#include "head_ops.hpp"
#include "row_stream.cuh"

namespace ftb {
namespace {

constexpr int kStatThreads = 512;
constexpr int kMaxChunks = 64;
constexpr int kMaxCandidates = 8192;
constexpr int kScoreThreads = 256;
constexpr int kScoreLanes = 8;   // lanes that share a candidate's positions
constexpr int kScoreTile = 64;   // positions whose statistics are staged at a time
constexpr int kPairThreads = 1024;
constexpr int kPlanThreads = 1024;

uint64_t align256(uint64_t x) { return (x + 255) & ~(uint64_t)255; }
int dtype_size(int dtype) { return dtype == FT_DTYPE_F32 ? 4 : 2; }

struct RowPlan {
  uint64_t rows;
  uint32_t chunks;      // CTAs per row
  uint64_t vecs_chunk;  // 16-byte vectors per chunk
};

RowPlan plan_rows(uint64_t rows, uint32_t vocab, int dtype) {
  RowPlan p;
  p.rows = rows;
  const uint64_t vecs = ((uint64_t)vocab * dtype_size(dtype) + 15) / 16 + 1;
  // A chunk is at least one pass of a CTA with four vectors per thread
  // (32 KB); a row is split so far that two full waves of CTAs (four fit on an
  // SM) share the work.
  const uint64_t least = kStatThreads * 4;
  uint64_t want = rows ? 148 * 8 / rows : 1;
  want = std::max<uint64_t>(1, std::min<uint64_t>({want, (vecs + least - 1) / least, (uint64_t)kMaxChunks}));
  p.vecs_chunk = (vecs + want - 1) / want;
  p.chunks = (uint32_t)((vecs + p.vecs_chunk - 1) / p.vecs_chunk);
  return p;
}

// Partial (maximum, sum) of chunk blockIdx.y of row blockIdx.x. Bound by the
// logits' bytes: 35 us for 48 rows of 2.2M bf16 (211 MB, 6.0 TB/s) behind
// kernels that left nothing to write back, 47 us behind a gradient of that size;
// 24 us for 64 rows of 500009 f32 (128 MB). Four CTAs on an SM with two vectors
// of each thread on their way: with half as many CTAs and twice the vectors a
// row of 32000 takes 7.0 us instead of 5.6.
template <typename T>
__global__ void __launch_bounds__(kStatThreads, 4)
    row_stats_kernel(const T *logits, uint32_t vocab, uint64_t vecs_chunk, SoftSum *part) {
  __shared__ SoftSum sm[kStatThreads / 32];
  const RowVecs<T> r(logits + (uint64_t)blockIdx.x * vocab, vocab);
  const int64_t v0 = (int64_t)(blockIdx.y * vecs_chunk);
  const int64_t v1 = min(v0 + (int64_t)vecs_chunk, r.count());
  SoftSum s = soft_stream<T, kStatThreads, 2>(r, v0, v1, -kNegInf, [](int64_t, float) {});
  s = soft_join_block<kStatThreads>(s, sm);
  if (threadIdx.x == 0) part[(uint64_t)blockIdx.x * gridDim.y + blockIdx.y] = s;
}

// Scores of 32 candidates of one request: eight lanes each, which take every
// eighth position and add in 64 bits (a preference's margin is a small
// difference of such sums). Latency of one look at the statistics and one at
// each logit: 3 us for 10 candidates of 8 positions, 6.9 us for 1000 of 24.
template <typename T>
__global__ void __launch_bounds__(kScoreThreads)
    score_kernel(const T *logits, const uint32_t *tokens, const int32_t *lengths, uint32_t vocab, uint32_t L, uint32_t C,
                 uint32_t chunks, const SoftSum *part, SoftSum *stats, float *logp, double *logp64, uint32_t *ticket) {
  __shared__ double sm_base[kScoreTile];  // lse; +inf where the row has nothing but -inf
  const uint32_t per = kScoreThreads / kScoreLanes, blocks = (C + per - 1) / per;
  const uint64_t req = blockIdx.x / blocks;
  const uint32_t blk = blockIdx.x % blocks;
  const uint32_t j = blk * per + threadIdx.x / kScoreLanes, sub = threadIdx.x % kScoreLanes;
  if (ticket && blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
  const int32_t len = j < C ? lengths[req * C + j] : 0;
  const bool bad = len < 0 || (uint32_t)len > L;
  const uint32_t n = bad ? 0 : (uint32_t)len;
  const uint32_t *tok = tokens + (req * C + (j < C ? j : 0)) * L;
  double sum = 0.0;
  for (uint32_t l0 = 0; l0 < L; l0 += kScoreTile) {
    __syncthreads();
    {  // four threads join a position's partial sums
      const uint32_t at = threadIdx.x / 4, l = l0 + at;
      const SoftSum *p = part + (req * L + l) * chunks;
      const uint32_t have = l < L ? chunks : 0;
      SoftSum s = SoftSum::none();
      for (uint32_t c = threadIdx.x % 4; c < have; c += 4) s.m = fmaxf(s.m, p[c].m);
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) s.m = fmaxf(s.m, __shfl_xor_sync(~0u, s.m, d));
      for (uint32_t c = threadIdx.x % 4; c < have; c += 4) s.z += p[c].z * factor_from(p[c].m, s.m);
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) s.z += __shfl_xor_sync(~0u, s.z, d);
      if (threadIdx.x % 4 == 0 && l < L) {
        sm_base[at] = s.z == 0.0f ? (double)-kNegInf : (double)s.m + log((double)s.z);
        if (blk == 0) stats[req * L + l] = s;
      }
    }
    __syncthreads();
    const uint32_t end = min(n, l0 + kScoreTile);
#pragma unroll 4
    for (uint32_t l = l0 + sub; l < end; l += kScoreLanes) {
      const uint32_t t = tok[l];
      const double x = t < vocab ? (double)to_f32(logits[(req * L + l) * vocab + t]) : (double)kNegInf;
      sum += x - sm_base[l - l0];
    }
  }
#pragma unroll
  for (int d = 1; d < kScoreLanes; d <<= 1) sum += __shfl_xor_sync(~0u, sum, d);
  if (bad) sum = __longlong_as_double(0x7FF8000000000000ll);
  if (j < C && sub == 0) {
    if (logp) logp[req * C + j] = (float)sum;
    if (logp64) logp64[req * C + j] = sum;
  }
}

__device__ double2 block_sum(double2 v, double2 *sm /* [kPairThreads / 32] */) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v.x += __shfl_xor_sync(~0u, v.x, d), v.y += __shfl_xor_sync(~0u, v.y, d);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  double2 s = make_double2(0.0, 0.0);
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) s.x += sm[w].x, s.y += sm[w].y;
  return s;
}

// Sums that do not depend on the order of the additions: integers in units of a
// power of two that leaves room for `terms` of them of magnitude below
// 2^exponent.  For a thousand terms a unit is 2^-51 of that magnitude.
struct FixedSum {
  double up, down;
  __device__ FixedSum(int exponent, uint32_t terms) {
    const int bits = 62 - (32 - __clz((int)terms)) - exponent;
    up = scalbn(1.0, bits);
    down = scalbn(1.0, -bits);
  }
  __device__ unsigned long long of(double x) const { return (unsigned long long)__double2ll_rn(x * up); }
  __device__ double value(unsigned long long s) const { return (double)(long long)s * down; }
};

// The power of two above a weight's magnitude, as an integer that compares as
// the magnitudes do: |w| < 2^(power_above(w) - 1022).  Weights below 2^-300
// count as that; no f32 holds them.
__device__ __forceinline__ uint32_t power_above(double w) {
  return max((uint32_t)__double2hiint(w) >> 20 & 0x7FFu, 1022u - 300u);
}

// Adds to a 64-bit sum in shared memory. There, the hardware adds 32 bits at
// once but 64 only in a loop that tries again whenever another thread was
// faster: a thousand pairs with one chosen candidate took 44 us instead of 9,
// a thousand candidates with one token 30 instead of 6.5.
__device__ __forceinline__ void add_shared(unsigned long long *sum, unsigned long long x) {
  uint32_t *low = reinterpret_cast<uint32_t *>(sum);
  const uint32_t add = (uint32_t)x, was = atomicAdd(low, add);
  const uint32_t rest = (uint32_t)(x >> 32) + (was + add < was);
  if (rest) atomicAdd(low + 1, rest);
}

// The pairs of one request per CTA: margins, this request's loss and pair
// count, and each candidate's gradient, added up in shared memory as integers
// so that it is the same in any order.  Weights fall with e^-margin, so that
// each candidate's sum has a unit of its own, by its largest weight: the first
// pass finds that and the second adds (a thread keeps its first pair's weight,
// those of further pairs are worked out again).  The CTA that ends last adds up
// the requests.  Latency of looks one after the other: 10.1 us for 1000 pairs,
// 8.0 for 8.
__global__ void __launch_bounds__(kPairThreads)
    pair_kernel(ft_preference_args p, uint32_t n, uint32_t C, const double *logp64, double2 *part, uint32_t *ticket) {
  // [C] sums, u32 [C] the power above each one's largest weight (0: no pair),
  // then C bits: the candidate is in a pair without a margin.
  extern __shared__ unsigned long long acc[];
  uint32_t *top = reinterpret_cast<uint32_t *>(acc + C), *broken = top + C;
  __shared__ double2 sm[kPairThreads / 32];
  __shared__ bool last;
  const uint64_t req = blockIdx.x;
  const double *lp = logp64 + req * C;
  const float *ref = p.ref_logp + req * C;
  const int32_t *chosen = p.chosen + req * p.pairs, *rejected = p.rejected + req * p.pairs;
  const double beta = p.beta, e = p.label_smoothing;
  auto margin_of = [&](int32_t c, int32_t r) { return beta * ((lp[c] - (double)ref[c]) - (lp[r] - (double)ref[r])); };
  auto weight_of = [&](double z, double t /* exp(-|z|) */) {
    const double big = 1.0 / (1.0 + t), small = t / (1.0 + t);  // sigmoids of |z| and -|z|
    return beta * (e * (z >= 0 ? big : small) - (1.0 - e) * (z >= 0 ? small : big));
  };
  auto there = [&](int32_t c, int32_t r) { return c >= 0 && r >= 0 && (uint32_t)c < C && (uint32_t)r < C; };
  for (uint32_t j = threadIdx.x; j < C; j += kPairThreads) acc[j] = 0, top[j] = 0;
  for (uint32_t j = threadIdx.x; j < (C + 31) / 32; j += kPairThreads) broken[j] = 0;
  __syncthreads();
  double loss = 0.0, count = 0.0, kept = 0.0;
  for (uint32_t q = threadIdx.x; q < p.pairs; q += kPairThreads) {
    const int32_t c = chosen[q], r = rejected[q];
    float margin = 0.0f;
    if (c >= 0 && r >= 0) {
      count += 1.0;
      if (there(c, r)) {
        const double z = margin_of(c, r);
        const double t = exp(-fabs(z)), soft = log1p(t);
        const double pos = soft + (z < 0 ? -z : 0.0), neg = soft + (z > 0 ? z : 0.0);
        // A weight of zero takes its side away whatever that side's value.
        loss += (e < 1.0 ? (1.0 - e) * pos : 0.0) + (e > 0.0 ? e * neg : 0.0) + (z != z ? z : 0.0);
        margin = (float)z;
        if (z == z) {
          const double w = weight_of(z, t);
          const uint32_t power = power_above(w);
          atomicMax(&top[c], power);
          atomicMax(&top[r], power);
          if (q == threadIdx.x) kept = w;
        } else {
          atomicOr(&broken[(uint32_t)c / 32], 1u << (c % 32));
          atomicOr(&broken[(uint32_t)r / 32], 1u << (r % 32));
        }
      } else {
        margin = __int_as_float(0x7FC00000);
        loss += (double)margin;
      }
    }
    p.margin[req * p.pairs + q] = margin;
  }
  const double2 sums = block_sum(make_double2(loss, count), sm);  // its barriers make top and broken complete
  const uint32_t terms = 2 * (uint32_t)sums.y;
  for (uint32_t q = threadIdx.x; q < p.pairs; q += kPairThreads) {
    const int32_t c = chosen[q], r = rejected[q];
    if (!there(c, r)) continue;
    double w = kept;
    if (q != threadIdx.x) {
      const double z = margin_of(c, r);
      if (z != z) continue;
      w = weight_of(z, exp(-fabs(z)));
    }
    if (w == 0.0) continue;
    add_shared(&acc[c], FixedSum((int)top[c] - 1022, terms).of(w));
    add_shared(&acc[r], FixedSum((int)top[r] - 1022, terms).of(-w));
  }
  __syncthreads();
  for (uint32_t j = threadIdx.x; j < C; j += kPairThreads) {
    const float g = top[j] ? (float)FixedSum((int)top[j] - 1022, terms).value(acc[j]) : 0.0f;
    p.grad[req * C + j] = broken[j / 32] >> (j % 32) & 1 ? __int_as_float(0x7FC00000) : g;
  }
  if (threadIdx.x == 0) {
    part[req] = sums;
    __threadfence();
    last = atomicAdd(ticket, 1u) == n - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double2 all = make_double2(0.0, 0.0);
  for (uint32_t i = threadIdx.x; i < n; i += kPairThreads) {
    const double2 v = __ldcg(&part[i]);
    all.x += v.x;
    all.y += v.y;
  }
  all = block_sum(all, sm);
  if (threadIdx.x == 0) {
    const double by = p.mean ? 1.0 / (all.y > 1.0 ? all.y : 1.0) : 1.0;
    *p.loss = (float)(all.x * by);
    *p.factor = (float)by;
  }
}

// One CTA per row: W, and the summed weight of each distinct token of the live
// candidates.  The tokens meet in a hash table in shared memory (at most half
// full) whose sums are integers, so that they are the same in any order; the
// list's order is not, and nothing depends on it.  Each token's sum has a unit
// of its own, by the exponent of its largest weight, which the first pass finds.
// A weight that is not finite makes W NaN, and with it the row's gradient.
// Latency: 6.2 us for 48 rows of 1000 candidates, 4.1 for 128 of 10.
__global__ void __launch_bounds__(kPlanThreads)
    scatter_plan_kernel(const uint32_t *tokens, const int32_t *lengths, const SoftSum *stats, const float *grad,
                        const float *factor, const float *upstream, uint32_t vocab, uint32_t L, uint32_t C,
                        uint32_t slots, uint32_t *out_tok, float *out_w, uint32_t *out_n, float *out_total) {
  // [slots] sums, which begin as the exponent; u32 [slots] tokens; u8 [slots] exponents.
  extern __shared__ unsigned long long acc[];
  uint32_t *key = reinterpret_cast<uint32_t *>(acc + slots);
  uint8_t *power = reinterpret_cast<uint8_t *>(key + slots);
  __shared__ double2 sm[32];
  __shared__ uint32_t found, largest;
  const uint64_t row = blockIdx.x, req = row / L;
  const uint32_t l = (uint32_t)(row % L), lane = threadIdx.x & 31;
  const bool dead = stats[row].z == 0.0f;
  // Up to eight candidates a thread: everything about them is fetched at once.
  constexpr int kMost = kMaxCandidates / kPlanThreads;
  float weight[kMost];
  uint32_t token[kMost];
  double total = 0.0;
  uint32_t top = 0;  // of the magnitudes' bits, which compare as the magnitudes do
#pragma unroll
  for (int q = 0; q < kMost; ++q) {
    const uint32_t j = threadIdx.x + q * blockDim.x;
    weight[q] = 0.0f, token[q] = 0xFFFFFFFFu;
    if (j < C) {
      const int32_t len = lengths[req * C + j];
      const float w = grad[req * C + j];
      const uint32_t t = tokens[(req * C + j) * L + l];
      if (!dead && len >= 0 && (uint32_t)len <= L && l < (uint32_t)len) weight[q] = w, token[q] = t;
      total += weight[q];
      top = max(top, __float_as_uint(weight[q]) & 0x7FFFFFFFu);
    }
  }
  for (uint32_t i = threadIdx.x; i < slots; i += blockDim.x) acc[i] = 0, key[i] = 0xFFFFFFFFu;
  if (threadIdx.x == 0) found = largest = 0;
  __syncthreads();
  top = __reduce_max_sync(~0u, top);
  if (lane == 0) atomicMax(&largest, top);
  total = block_sum(make_double2(total, 0.0), sm).x;  // its barriers make `largest` complete
  top = largest;
  const double scale = (factor ? (double)*factor : 1.0) * (upstream ? (double)*upstream : 1.0);
  if (top >= 0x7F800000u) total = __longlong_as_double(0x7FF8000000000000ll);
  if (top == 0 || top >= 0x7F800000u) {  // zeros alone, or NaN everywhere
    if (threadIdx.x == 0) out_n[row] = 0, out_total[row] = (float)(total * scale);
    return;
  }
  // A weight of exponent field e is below 2^(e - 126).  token[q] becomes its slot.
  auto fixed = [&](uint32_t e) { return FixedSum((int)e - 126, C); };
#pragma unroll
  for (int q = 0; q < kMost; ++q) {
    const uint32_t t = token[q];
    token[q] = 0xFFFFFFFFu;
    if (t >= vocab) continue;
    uint32_t at = (t * 2654435761u) >> (32 - __popc(slots - 1));
    for (uint32_t i = 0; i < slots; ++i, at = (at + 1) & (slots - 1)) {
      const uint32_t was = atomicCAS(&key[at], 0xFFFFFFFFu, t);
      if (was == 0xFFFFFFFFu || was == t) break;
    }
    token[q] = at;
    atomicMax(reinterpret_cast<uint32_t *>(&acc[at]), __float_as_uint(weight[q]) >> 23 & 0xFFu);
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kMost; ++q)
    if (token[q] < slots) power[token[q]] = (uint8_t)acc[token[q]];  // one value, whoever writes it
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kMost; ++q)
    if (token[q] < slots) add_shared(&acc[token[q]], fixed(power[token[q]]).of(weight[q]));
  __syncthreads();
  for (uint32_t i0 = 0; i0 < slots; i0 += blockDim.x) {  // a warp asks for its places at once
    const uint32_t i = i0 + threadIdx.x;
    const bool has = i < slots && key[i] != 0xFFFFFFFFu;
    const uint32_t votes = __ballot_sync(~0u, has);
    uint32_t at = 0;
    if (lane == 0 && votes) at = atomicAdd(&found, __popc(votes));
    at = __shfl_sync(~0u, at, 0) + __popc(votes & ((1u << lane) - 1));
    if (has) {
      out_tok[row * C + at] = key[i];
      out_w[row * C + at] = (float)(fixed(power[i]).value(acc[i] - power[i]) * scale);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) out_n[row] = found, out_total[row] = (float)(total * scale);
}

__device__ __forceinline__ uint4 pack(const float (&v)[4], const float *) {
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ uint4 pack(const float (&v)[8], const __nv_bfloat16 *) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack(const float (&v)[8], const __half *) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The gradient of a chunk of row blockIdx.x: the softmax part first, then, after
// the CTA's barrier, its tokens' entries over it. The chunks come in the
// opposite order of the statistics', so that what those read last is still in
// L2, and the gradient leaves it first: 73 -> 68 us for 48 rows of 2.2M bf16
// (422 MB in and out, 6.2 TB/s).
template <typename T>
__global__ void __launch_bounds__(kStatThreads)
    row_grad_kernel(const T *logits, T *grad, uint32_t vocab, uint32_t C, uint64_t vecs_chunk, const SoftSum *stats,
                    const uint32_t *tok, const float *tok_w, const uint32_t *tok_n, const float *total) {
  constexpr int N = RowVecs<T>::N;
  const uint64_t row = blockIdx.x;
  const RowVecs<T> in(logits + row * vocab, vocab), out(grad + row * vocab, vocab);
  const int64_t v0 = (int64_t)((gridDim.y - 1 - blockIdx.y) * vecs_chunk);
  const int64_t v1 = min(v0 + (int64_t)vecs_chunk, out.count());
  T *g = grad + row * vocab;
  const SoftSum s = stats[row];
  const float w = total[row], k = -w / s.z, base = s.m;
  const bool zero = w == 0.0f;
  const bool same = in.head == out.head;
  const float2 minus = make_float2(-base, -base), k2 = make_float2(k, k);
  auto whole = [&](int64_t i, uint4 q) {
    float v[N];
    unpack(q, v, (const T *)nullptr);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 y = mul2(k2, exp_below2(add2(make_float2(v[e], v[e + 1]), minus)));
      v[e] = y.x, v[e + 1] = y.y;
    }
    __stcs(reinterpret_cast<uint4 *>(g + out.first(i)), pack(v, (const T *)nullptr));
  };
  auto one_by_one = [&](int64_t i) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int64_t at = out.first(i) + e;
      if (at >= 0 && at < (int64_t)vocab) from_f32(zero ? 0.0f : k * exp_below(to_f32(in.row[at]) - base), g[at]);
    }
  };
  constexpr int U = 4;
  int64_t i = v0 + threadIdx.x;
  for (; i + (U - 1) * kStatThreads < v1; i += U * kStatThreads) {
    if (out.whole(i) && out.whole(i + (U - 1) * kStatThreads) && (same || zero)) {
      uint4 q[U];
      if (zero) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          __stcs(reinterpret_cast<uint4 *>(g + out.first(i + u * kStatThreads)), make_uint4(0, 0, 0, 0));
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = in.load_whole(i + u * kStatThreads);
#pragma unroll
        for (int u = 0; u < U; ++u) whole(i + u * kStatThreads, q[u]);
      }
    } else {
#pragma unroll 1
      for (int u = 0; u < U; ++u) one_by_one(i + u * kStatThreads);
    }
  }
  for (; i < v1; i += kStatThreads) {
    if (out.whole(i) && same && !zero)
      whole(i, in.load_whole(i));
    else
      one_by_one(i);
  }
  const uint32_t n = tok_n[row];
  if (n == 0) return;
  __syncthreads();
  const uint32_t *t = tok + row * C;
  const int64_t e0 = max((int64_t)0, out.first(v0)), e1 = min((int64_t)vocab, out.first(v1));
  if (e0 >= e1) return;
  for (uint32_t i = threadIdx.x; i < n; i += kStatThreads) {
    const uint32_t at = t[i];
    if (at < e0 || at >= e1) continue;
    const float p = zero ? 0.0f : k * exp_below(to_f32(in.row[at]) - base);
    from_f32(tok_w[row * C + i] + p, g[at]);
  }
}

void check_sequence(const ft_sequence_args &a, const char *what) {
  const std::string w = what;
  if (a.dtype != FT_DTYPE_F32 && a.dtype != FT_DTYPE_BF16 && a.dtype != FT_DTYPE_F16)
    throw InvalidArgument(w + ": unknown dtype");
  if (a.num_outpos == 0 || a.vocab == 0 || a.candidates == 0)
    throw InvalidArgument(w + ": num_outpos, vocab and candidates must be positive");
  if (a.candidates > (uint32_t)kMaxCandidates) throw InvalidArgument(w + ": at most 8192 candidates per request");
  // Grids: one CTA per row, and per 32 candidates of a request.
  const uint64_t most = 0x7FFFFFFF;
  if ((uint64_t)a.n * a.num_outpos > most || (uint64_t)a.n * ((a.candidates + 31) / 32) > most)
    throw InvalidArgument(w + ": n * num_outpos or n * candidates is too large");
}

void check_room(const void *ws, uint64_t have, uint64_t need, const char *what) {
  if (need && !ws) fail(ErrorKind::kNull, std::string("MARISA_NULL_ERROR: ") + what + ": workspace is NULL");
  if (have < need)
    throw InvalidArgument(std::string(what) + ": workspace of " + std::to_string(have) + " bytes, needs " +
                          std::to_string(need));
  if (reinterpret_cast<uintptr_t>(ws) & 255)
    throw InvalidArgument(std::string(what) + ": the workspace must be 256-byte aligned");
}

void check_aligned(const void *p, uintptr_t to, const char *what) {
  if (reinterpret_cast<uintptr_t>(p) % to) throw InvalidArgument(std::string(what) + " is not aligned to its elements");
}

void need_ptr(const void *p, const char *what) {
  if (!p) fail(ErrorKind::kNull, std::string("MARISA_NULL_ERROR: ") + what + " is NULL");
}

struct GradLayout {
  uint64_t tok, w, n, total, end;
};

GradLayout grad_layout(const ft_sequence_args &a) {
  const uint64_t rows = (uint64_t)a.n * a.num_outpos;
  GradLayout g;
  g.tok = 0;
  g.w = align256(4 * rows * a.candidates);
  g.n = g.w + align256(4 * rows * a.candidates);
  g.total = g.n + align256(4 * rows);
  g.end = g.total + align256(4 * rows);
  return g;
}

uint64_t part_bytes(const ft_sequence_args &a) {
  const RowPlan p = plan_rows((uint64_t)a.n * a.num_outpos, a.vocab, a.dtype);
  return align256(sizeof(SoftSum) * p.rows * p.chunks);
}

struct PairLayout {
  uint64_t lp, part, ticket, end;
};

PairLayout pair_layout(const ft_sequence_args &a) {
  PairLayout l;
  l.lp = part_bytes(a);
  l.part = l.lp + align256(8ull * a.n * a.candidates);
  l.ticket = l.part + align256(16ull * a.n);
  l.end = l.ticket + 256;
  return l;
}

template <typename F>
void by_dtype(int dtype, F &&f) {
  if (dtype == FT_DTYPE_F32)
    f((float *)nullptr);
  else if (dtype == FT_DTYPE_BF16)
    f((__nv_bfloat16 *)nullptr);
  else
    f((__half *)nullptr);
}

void scores(const ft_sequence_args &a, char *ws, double *logp64, uint32_t *ticket, cudaStream_t stream) {
  const RowPlan p = plan_rows((uint64_t)a.n * a.num_outpos, a.vocab, a.dtype);
  SoftSum *part = reinterpret_cast<SoftSum *>(ws);
  const uint32_t per = kScoreThreads / kScoreLanes, blocks = (a.candidates + per - 1) / per;
  by_dtype(a.dtype, [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const T *x = static_cast<const T *>(a.logits);
    row_stats_kernel<T><<<dim3((unsigned)p.rows, p.chunks), kStatThreads, 0, stream>>>(x, a.vocab, p.vecs_chunk, part);
    CUDA_TRY(cudaGetLastError());
    score_kernel<T><<<a.n * blocks, kScoreThreads, 0, stream>>>(x, a.tokens, a.lengths, a.vocab, a.num_outpos,
                                                               a.candidates, p.chunks, part,
                                                               reinterpret_cast<SoftSum *>(a.stats), a.logp, logp64,
                                                               ticket);
    CUDA_TRY(cudaGetLastError());
  });
}

void need_inputs(const ft_sequence_args &a) {
  need_ptr(a.logits, "logits");
  need_ptr(a.tokens, "tokens");
  need_ptr(a.lengths, "lengths");
  need_ptr(a.stats, "stats");
  check_aligned(a.logits, (uintptr_t)dtype_size(a.dtype), "logits");
}

}  // namespace

uint64_t sequence_logp_workspace(const ft_sequence_args &a) {
  check_sequence(a, "sequence_logp");
  return std::max(part_bytes(a), grad_layout(a).end);
}

void sequence_logp_device(const ft_sequence_args &a, void *ws, uint64_t ws_bytes, cudaStream_t stream) {
  check_sequence(a, "sequence_logp");
  if (a.n == 0) return;
  need_inputs(a);
  need_ptr(a.logp, "logp");
  check_room(ws, ws_bytes, part_bytes(a), "sequence_logp");
  scores(a, static_cast<char *>(ws), nullptr, nullptr, stream);
}

void sequence_grad_device(const ft_sequence_args &a, const float *grad, const float *factor, const float *upstream,
                          void *ws, uint64_t ws_bytes, cudaStream_t stream) {
  check_sequence(a, "sequence_grad");
  if (a.n == 0) return;
  need_inputs(a);
  need_ptr(a.grad_logits, "grad_logits");
  need_ptr(grad, "grad");
  check_aligned(a.grad_logits, (uintptr_t)dtype_size(a.dtype), "grad_logits");
  const GradLayout g = grad_layout(a);
  check_room(ws, ws_bytes, g.end, "sequence_grad");
  const RowPlan p = plan_rows((uint64_t)a.n * a.num_outpos, a.vocab, a.dtype);
  char *w = static_cast<char *>(ws);
  uint32_t *tok = reinterpret_cast<uint32_t *>(w + g.tok), *cnt = reinterpret_cast<uint32_t *>(w + g.n);
  float *tok_w = reinterpret_cast<float *>(w + g.w), *total = reinterpret_cast<float *>(w + g.total);
  const SoftSum *stats = reinterpret_cast<const SoftSum *>(a.stats);
  uint32_t slots = 32;
  while (slots < 2 * a.candidates) slots <<= 1;
  const uint32_t threads = std::min<uint32_t>(kPlanThreads, (a.candidates + 31) / 32 * 32);
  const size_t smem = 13ull * slots;
  allow_shared(scatter_plan_kernel, 13 * 2 * kMaxCandidates);
  scatter_plan_kernel<<<(unsigned)p.rows, threads, smem, stream>>>(a.tokens, a.lengths, stats, grad, factor, upstream,
                                                                   a.vocab, a.num_outpos, a.candidates, slots, tok,
                                                                   tok_w, cnt, total);
  CUDA_TRY(cudaGetLastError());
  by_dtype(a.dtype, [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    row_grad_kernel<T><<<dim3((unsigned)p.rows, p.chunks), kStatThreads, 0, stream>>>(
        static_cast<const T *>(a.logits), static_cast<T *>(a.grad_logits), a.vocab, a.candidates, p.vecs_chunk, stats,
        tok, tok_w, cnt, total);
    CUDA_TRY(cudaGetLastError());
  });
}

uint64_t preference_workspace(const ft_sequence_args &a) {
  check_sequence(a, "preference_loss");
  return pair_layout(a).end;
}

void preference_loss_device(const ft_sequence_args &a, const ft_preference_args &p, void *ws, uint64_t ws_bytes,
                            cudaStream_t stream) {
  check_sequence(a, "preference_loss");
  if (!(p.label_smoothing >= 0.0f && p.label_smoothing <= 1.0f))
    throw InvalidArgument("preference_loss: label_smoothing must be in [0, 1]");
  if (!std::isfinite(p.beta)) throw InvalidArgument("preference_loss: beta must be finite");
  if (p.pairs >= 1u << 30) throw InvalidArgument("preference_loss: too many pairs per request");
  need_ptr(p.loss, "loss");
  need_ptr(p.factor, "factor");
  if (a.n == 0) {
    CUDA_TRY(cudaMemsetAsync(p.loss, 0, 4, stream));
    CUDA_TRY(cudaMemsetAsync(p.factor, 0, 4, stream));
    return;
  }
  need_inputs(a);
  need_ptr(p.ref_logp, "ref_logp");
  need_ptr(p.grad, "grad");
  if (p.pairs) {
    need_ptr(p.chosen, "chosen");
    need_ptr(p.rejected, "rejected");
    need_ptr(p.margin, "margin");
  }
  const PairLayout l = pair_layout(a);
  check_room(ws, ws_bytes, l.end, "preference_loss");
  char *w = static_cast<char *>(ws);
  double *lp = reinterpret_cast<double *>(w + l.lp);
  uint32_t *ticket = reinterpret_cast<uint32_t *>(w + l.ticket);
  scores(a, w, lp, ticket, stream);
  const size_t smem = 12ull * a.candidates + 4 * ((a.candidates + 31) / 32);
  allow_shared(pair_kernel, 12 * kMaxCandidates + kMaxCandidates / 8);
  pair_kernel<<<a.n, kPairThreads, smem, stream>>>(p, a.n, a.candidates, lp, reinterpret_cast<double2 *>(w + l.part),
                                                   ticket);
  CUDA_TRY(cudaGetLastError());
}

}  // namespace ftb
