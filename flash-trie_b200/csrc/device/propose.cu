// The search's proposals from a model's logits: per row the log-softmax over
// the vocabulary and its k largest entries, exact, equal logits in order of
// the token id.
//
//   logp[v] = x[v] - m - log(sum_u exp(x[u] - m)),  m = max_u x[u]
//
// One CTA per row.  The entries are ordered by the 64-bit key (logit as an
// ordered integer, complement of the id), which no two share, so the k-th
// largest key separates the proposals from the rest.  It is found by radix
// selection, 11 bits a pass.
#include <algorithm>
#include <string>

#include "../engine.hpp"
#include "cuda_util.hpp"
#include "head_ops.hpp"
#include "row_stream.cuh"

namespace ftb {
namespace {

constexpr int kThreads = 1024;
constexpr uint32_t kBins = 2048;
constexpr float kFltMax = 3.402823466e+38f;

// Order-preserving integer of a float; -0 and 0 are the same.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(__fadd_rn(x, 0.0f));
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

template <typename T, typename F>
__device__ __forceinline__ void for_each(const RowVecs<T> &r, F &&f) {
  constexpr int N = RowVecs<T>::N;
  const int64_t n = r.count();
  for (int64_t i = threadIdx.x; i < n; i += kThreads) {
    float v[N];
    if (r.whole(i))
      unpack(r.load_whole(i), v, (const T *)nullptr);
    else
      r.load_edge(i, v);
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (v[e] > kNegInf) f(((uint64_t)ordered(v[e]) << 32) | (uint32_t)~(uint32_t)(r.first(i) + e), v[e]);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    propose_kernel(const T *logits, uint32_t vocab, uint32_t k, int order, uint32_t slots, uint32_t *out_id, float *out_lp) {
  extern __shared__ unsigned long long list[];
  __shared__ SoftSum sm[kThreads / 32];
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t got, sm_digit, sm_above;
  __shared__ SoftSum sm_sum;
  const uint64_t row = blockIdx.x;
  const RowVecs<T> r(logits + row * vocab, vocab);
  SoftSum s = SoftSum::none();
  soft_stream<T, kThreads, 4>(r, 0, r.count(), s);
  s = soft_join_block<kThreads>(s, sm);
  if (threadIdx.x == 0) sm_sum = s, got = 0;
  __syncthreads();
  s = sm_sum;
  if (s.valid()) {
    // prefix: the bits of the k-th largest key known so far; need: its rank
    // among the keys that share them.
    uint64_t prefix = 0;
    uint32_t need = k;
    bool all = false;
    for (int shift = 53; shift > -11 && !all; shift -= 11) {
      const int sh = shift < 0 ? 0 : shift, bits = shift < 0 ? 11 + shift : 11;
      const uint64_t above = sh + bits >= 64 ? 0 : ~0ull << (sh + bits);
      for (uint32_t b = threadIdx.x; b < kBins; b += kThreads) hist[b] = 0;
      __syncthreads();
      for_each(r, [&](uint64_t key, float) {
        if ((key & above) == prefix) atomicAdd(&hist[(uint32_t)(key >> sh) & ((1u << bits) - 1)], 1u);
      });
      __syncthreads();
      if (threadIdx.x == 0) {
        uint32_t sum = 0;
        int d = (1 << bits) - 1;
        for (; d >= 0; --d) {
          if (sum + hist[d] >= need) break;
          sum += hist[d];
        }
        sm_digit = (uint32_t)d;
        sm_above = sum;
      }
      __syncthreads();
      if ((int)sm_digit < 0) {
        all = true;  // fewer than k entries: all of them
      } else {
        prefix |= (uint64_t)sm_digit << sh;
        need -= sm_above;
      }
      __syncthreads();
    }
    const uint64_t least = all ? 0 : prefix;
    for_each(r, [&](uint64_t key, float) {
      if (key >= least) {
        const uint32_t at = atomicAdd(&got, 1u);
        const uint32_t id = ~(uint32_t)key, v = (uint32_t)(key >> 32);
        list[at] = order == 0 ? ((uint64_t)id << 32) | v : ((uint64_t)~v << 32) | id;
      }
    });
    __syncthreads();
  }
  const uint32_t n = got;
  for (uint32_t i = n + threadIdx.x; i < slots; i += kThreads) list[i] = ~0ull;
  for (uint32_t size = 2; size <= slots; size <<= 1)
    for (uint32_t step = size >> 1; step; step >>= 1) {
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < slots / 2; i += kThreads) {
        const uint32_t a = 2 * i - (i & (step - 1)), b = a + step;
        const bool up = (a & size) == 0;
        const unsigned long long x = list[a], y = list[b];
        if ((x > y) == up) list[a] = y, list[b] = x;
      }
    }
  __syncthreads();
  const float logz = logf(s.z);
  for (uint32_t i = threadIdx.x; i < k; i += kThreads) {
    uint32_t id = 0xFFFFFFFFu;
    float lp = -kFltMax;
    if (i < n) {
      const unsigned long long e = list[i];
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

}  // namespace

uint64_t propose_workspace(const ft_propose_args &a) {
  check_propose(a);
  return 0;
}

void propose_device(const ft_propose_args &a, void *ws, uint64_t ws_bytes, cudaStream_t stream) {
  check_propose(a);
  if (a.rows == 0) return;
  if (!a.logits || !a.topk_id || !a.topk_logp)
    fail(ErrorKind::kNull, "MARISA_NULL_ERROR: propose: logits, topk_id or topk_logp is NULL");
  if (reinterpret_cast<uintptr_t>(a.logits) % (a.dtype == FT_DTYPE_F32 ? 4 : 2))
    throw InvalidArgument("propose: logits is not aligned to its elements");
  uint32_t slots = 2;
  while (slots < a.topk) slots <<= 1;
  const size_t smem = 8ull * slots;
  auto run = [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (smem > 32 * 1024)
      CUDA_TRY(cudaFuncSetAttribute(propose_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    propose_kernel<T><<<(unsigned)a.rows, kThreads, smem, stream>>>(static_cast<const T *>(a.logits), a.vocab, a.topk,
                                                                    a.order, slots, a.topk_id, a.topk_logp);
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
