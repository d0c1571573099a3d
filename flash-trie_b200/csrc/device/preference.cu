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
  // (32 KB); a row is split so far that eight waves of CTAs share the work.
  const uint64_t least = kStatThreads * 4;
  uint64_t want = rows ? (148 * 8 + rows - 1) / rows : 1;
  want = std::max<uint64_t>(1, std::min<uint64_t>({want, (vecs + least - 1) / least, (uint64_t)kMaxChunks}));
  p.vecs_chunk = (vecs + want - 1) / want;
  p.chunks = (uint32_t)((vecs + p.vecs_chunk - 1) / p.vecs_chunk);
  return p;
}

// Partial (maximum, sum) of chunk blockIdx.y of row blockIdx.x.
template <typename T>
__global__ void __launch_bounds__(kStatThreads)
    row_stats_kernel(const T *logits, uint32_t vocab, uint64_t vecs_chunk, SoftSum *part) {
  __shared__ SoftSum sm[kStatThreads / 32];
  const RowVecs<T> r(logits + (uint64_t)blockIdx.x * vocab, vocab);
  const int64_t v0 = (int64_t)(blockIdx.y * vecs_chunk);
  const int64_t v1 = min(v0 + (int64_t)vecs_chunk, r.count());
  SoftSum s = SoftSum::none();
  soft_stream<T, kStatThreads, 4>(r, v0, v1, s);
  s = soft_join_block<kStatThreads>(s, sm);
  if (threadIdx.x == 0) part[(uint64_t)blockIdx.x * gridDim.y + blockIdx.y] = s;
}

// Scores of 32 candidates of one request: eight lanes each, which take every
// eighth position and add in 64 bits (a preference's margin is a small
// difference of such sums).
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
      SoftSum s = SoftSum::none();
      if (l < L)
        for (uint32_t c = threadIdx.x % 4; c < chunks; c += 4) s = soft_join(s, part[(req * L + l) * chunks + c]);
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        const SoftSum o{__shfl_xor_sync(~0u, s.m, d), __shfl_xor_sync(~0u, s.z, d)};
        s = soft_join(s, o);
      }
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

__device__ double block_sum(double v, double *sm /* [kPairThreads / 32] */) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) s += sm[w];
  return s;
}

// The pairs of one request per CTA: margins, this request's loss and pair
// count, and each candidate's gradient, summed over the pairs in a fixed
// order (a warp per candidate, its lanes over the pairs).  The CTA that ends
// last adds up the requests.
__global__ void __launch_bounds__(kPairThreads)
    pair_kernel(ft_preference_args p, uint32_t n, uint32_t C, const double *logp64, float *coef, double2 *part,
                uint32_t *ticket) {
  __shared__ double sm[kPairThreads / 32];
  __shared__ bool last;
  const uint64_t req = blockIdx.x;
  const double *lp = logp64 + req * C;
  const float *ref = p.ref_logp + req * C;
  double loss = 0.0, count = 0.0;
  for (uint32_t q = threadIdx.x; q < p.pairs; q += kPairThreads) {
    const int32_t c = p.chosen[req * p.pairs + q], r = p.rejected[req * p.pairs + q];
    float margin = 0.0f, w = 0.0f;
    if (c >= 0 && r >= 0) {
      count += 1.0;
      if ((uint32_t)c < C && (uint32_t)r < C) {
        const double z = (double)p.beta * ((lp[c] - (double)ref[c]) - (lp[r] - (double)ref[r]));
        const double e = p.label_smoothing, soft = log1p(exp(-fabs(z)));
        const double pos = soft + (z < 0 ? -z : 0.0), neg = soft + (z > 0 ? z : 0.0);
        const double sig = 1.0 / (1.0 + exp(-z)), gis = 1.0 / (1.0 + exp(z));
        // A weight of zero takes its side away whatever that side's value.
        loss += (e < 1.0 ? (1.0 - e) * pos : 0.0) + (e > 0.0 ? e * neg : 0.0) + (z != z ? z : 0.0);
        margin = (float)z;
        w = (float)((double)p.beta * (e * sig - (1.0 - e) * gis));
      } else {
        margin = __int_as_float(0x7FC00000);
        loss += (double)margin;
      }
    }
    p.margin[req * p.pairs + q] = margin;
    coef[req * p.pairs + q] = w;
  }
  loss = block_sum(loss, sm);
  count = block_sum(count, sm);
  __syncthreads();  // the block's coef values are visible to all of it
  const uint32_t lane = threadIdx.x & 31;
  for (uint32_t j = threadIdx.x >> 5; j < C; j += kPairThreads / 32) {
    double g = 0.0;
    for (uint32_t q = lane; q < p.pairs; q += 32) {
      const int32_t c = p.chosen[req * p.pairs + q], r = p.rejected[req * p.pairs + q];
      const float w = coef[req * p.pairs + q];
      if ((uint32_t)c == j) g += w;
      if ((uint32_t)r == j) g -= w;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) g += __shfl_xor_sync(~0u, g, d);
    if (lane == 0) p.grad[req * C + j] = (float)g;
  }
  if (threadIdx.x == 0) {
    part[req] = make_double2(loss, count);
    __threadfence();
    last = atomicAdd(ticket, 1u) == n - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  loss = count = 0.0;
  for (uint32_t i = threadIdx.x; i < n; i += kPairThreads) {
    const double2 v = __ldcg(&part[i]);
    loss += v.x;
    count += v.y;
  }
  loss = block_sum(loss, sm);
  count = block_sum(count, sm);
  if (threadIdx.x == 0) {
    const double by = p.mean ? 1.0 / (count > 1.0 ? count : 1.0) : 1.0;
    *p.loss = (float)(loss * by);
    *p.factor = (float)by;
  }
}

// One CTA per row: W, and the row's live (token, candidate) pairs sorted, with
// the summed weight of each distinct token at its first entry.  Adding in the
// candidates' order keeps the result the same from run to run.
__global__ void scatter_plan_kernel(const uint32_t *tokens, const int32_t *lengths, const SoftSum *stats, const float *grad,
                                    const float *factor, const float *upstream, uint32_t vocab, uint32_t L, uint32_t C,
                                    uint32_t slots, uint32_t *out_tok, float *out_w, uint32_t *out_n, float *out_total) {
  extern __shared__ unsigned long long key[];
  __shared__ double sm[32];
  __shared__ uint32_t live;
  const uint64_t row = blockIdx.x, req = row / L;
  const uint32_t l = (uint32_t)(row % L);
  const double scale = (factor ? (double)*factor : 1.0) * (upstream ? (double)*upstream : 1.0);
  const bool dead = stats[row].z == 0.0f;
  double total = 0.0;
  if (threadIdx.x == 0) live = 0;
  __syncthreads();
  for (uint32_t j = threadIdx.x; j < slots; j += blockDim.x) {
    unsigned long long k = ~0ull;
    if (j < C && !dead) {
      const int32_t len = lengths[req * C + j];
      if (len >= 0 && (uint32_t)len <= L && l < (uint32_t)len) {
        const uint32_t t = tokens[(req * C + j) * L + l];
        total += grad[req * C + j];
        if (t < vocab) k = ((unsigned long long)t << 32) | j;
      }
    }
    key[j] = k;
  }
  total = block_sum(total, sm) * scale;
  for (uint32_t size = 2; size <= slots; size <<= 1)
    for (uint32_t step = size >> 1; step; step >>= 1) {
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < slots / 2; i += blockDim.x) {
        const uint32_t a = 2 * i - (i & (step - 1)), b = a + step;
        const bool up = (a & size) == 0;
        const unsigned long long x = key[a], y = key[b];
        if ((x > y) == up) key[a] = y, key[b] = x;
      }
    }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < C; i += blockDim.x) {
    const unsigned long long k = key[i];
    if (k == ~0ull) continue;
    const uint32_t t = (uint32_t)(k >> 32);
    if (i + 1 == slots || key[i + 1] == ~0ull) live = i + 1;  // one thread: the last live entry
    double w = 0.0;
    if (i == 0 || (uint32_t)(key[i - 1] >> 32) != t)
      for (uint32_t q = i; q < slots && (uint32_t)(key[q] >> 32) == t && key[q] != ~0ull; ++q)
        w += grad[req * C + (uint32_t)key[q]];
    out_tok[row * C + i] = t;
    out_w[row * C + i] = (float)(w * scale);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    out_n[row] = live;
    out_total[row] = (float)total;
  }
}

__device__ uint32_t lower_bound(const uint32_t *a, uint32_t n, uint32_t x) {
  uint32_t lo = 0;
  while (n) {
    const uint32_t h = n / 2;
    if (a[lo + h] < x)
      lo += h + 1, n -= h + 1;
    else
      n = h;
  }
  return lo;
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

// The gradient of chunk blockIdx.y of row blockIdx.x: the softmax part first,
// then, after the CTA's barrier, its tokens' entries over it.
template <typename T>
__global__ void __launch_bounds__(kStatThreads)
    row_grad_kernel(const T *logits, T *grad, uint32_t vocab, uint32_t C, uint64_t vecs_chunk, const SoftSum *stats,
                    const uint32_t *tok, const float *tok_w, const uint32_t *tok_n, const float *total) {
  constexpr int N = RowVecs<T>::N;
  const uint64_t row = blockIdx.x;
  const RowVecs<T> in(logits + row * vocab, vocab), out(grad + row * vocab, vocab);
  const int64_t v0 = (int64_t)(blockIdx.y * vecs_chunk);
  const int64_t v1 = min(v0 + (int64_t)vecs_chunk, out.count());
  T *g = grad + row * vocab;
  const SoftSum s = stats[row];
  const float w = total[row], k = -w / s.z, base = s.m;
  const bool zero = w == 0.0f;
  const bool same = in.head == out.head;
  for (int64_t i = v0 + threadIdx.x; i < v1; i += kStatThreads) {
    float v[N];
    if (zero) {
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = 0.0f;
    } else {
      if (same && out.whole(i)) {
        unpack(in.load_whole(i), v, (const T *)nullptr);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int64_t at = out.first(i) + e;
          v[e] = (at >= 0 && at < (int64_t)vocab) ? to_f32(in.row[at]) : kNegInf;
        }
      }
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = k * exp_below(v[e] - base);
    }
    if (out.whole(i)) {
      *reinterpret_cast<uint4 *>(g + out.first(i)) = pack(v, (const T *)nullptr);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int64_t at = out.first(i) + e;
        if (at >= 0 && at < (int64_t)vocab) from_f32(v[e], g[at]);
      }
    }
  }
  const uint32_t n = tok_n[row];
  if (n == 0) return;
  __syncthreads();
  const uint32_t *t = tok + row * C;
  const int64_t e0 = max((int64_t)0, out.first(v0)), e1 = min((int64_t)vocab, out.first(v1));
  if (e0 >= e1) return;
  const uint32_t a = lower_bound(t, n, (uint32_t)e0);
  for (uint32_t i = a + threadIdx.x; i < n && t[i] < e1; i += kStatThreads) {
    if (i > 0 && t[i - 1] == t[i]) continue;
    const float p = zero ? 0.0f : k * exp_below(to_f32(in.row[t[i]]) - base);
    from_f32(tok_w[row * C + i] + p, g[t[i]]);
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
  uint64_t lp, coef, part, ticket, end;
};

PairLayout pair_layout(const ft_sequence_args &a, uint32_t pairs) {
  PairLayout l;
  l.lp = part_bytes(a);
  l.coef = l.lp + align256(8ull * a.n * a.candidates);
  l.part = l.coef + align256(4ull * a.n * pairs);
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
  uint32_t slots = 2;
  while (slots < a.candidates) slots <<= 1;
  const uint32_t threads = std::min<uint32_t>(1024, std::max<uint32_t>(32, slots / 2));
  const size_t smem = 8ull * slots;
  if (smem > 48 * 1024)
    CUDA_TRY(cudaFuncSetAttribute(scatter_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
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

uint64_t preference_workspace(const ft_sequence_args &a, uint32_t pairs) {
  check_sequence(a, "preference_loss");
  return pair_layout(a, pairs).end;
}

void preference_loss_device(const ft_sequence_args &a, const ft_preference_args &p, void *ws, uint64_t ws_bytes,
                            cudaStream_t stream) {
  check_sequence(a, "preference_loss");
  if (!(p.label_smoothing >= 0.0f && p.label_smoothing <= 1.0f))
    throw InvalidArgument("preference_loss: label_smoothing must be in [0, 1]");
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
  const PairLayout l = pair_layout(a, p.pairs);
  check_room(ws, ws_bytes, l.end, "preference_loss");
  char *w = static_cast<char *>(ws);
  double *lp = reinterpret_cast<double *>(w + l.lp);
  uint32_t *ticket = reinterpret_cast<uint32_t *>(w + l.ticket);
  scores(a, w, lp, ticket, stream);
  pair_kernel<<<a.n, kPairThreads, 0, stream>>>(p, a.n, a.candidates, lp, reinterpret_cast<float *>(w + l.coef),
                                                reinterpret_cast<double2 *>(w + l.part), ticket);
  CUDA_TRY(cudaGetLastError());
}

}  // namespace ftb
