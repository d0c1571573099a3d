// Streaming over rows of logits (f32, bf16 or f16, any alignment) and the
// running maximum and sum of a softmax.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace ftb {

constexpr float kNegInf = -__builtin_huge_valf();
// log2(e) as the sum of two floats: one alone is 1.3e-8 off, which would
// shift every log-sum by that times its mean distance from the maximum.
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLog2eRest = (float)(1.4426950408889634074 - (double)1.4426950408889634f);

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
// One rounding to nearest.
__device__ __forceinline__ void from_f32(float v, float &o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16 &o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half &o) { o = __float2half_rn(v); }

// e^d; d is a difference to a maximum or to a base a little below it.
__device__ __forceinline__ float exp_below(float d) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaf(d, kLog2eRest, d * kLog2e)));
  return y;
}

// e^d for d <= 0 (a rounding above at most), for the few factors that whole sums
// are multiplied by: the base-2 instruction's results are 5e-8 low on average,
// which would add up from join to join.  Cody and Waite's reduction by multiples
// of ln 2 in two parts, and Taylor's polynomial on [-ln 2 / 2, ln 2 / 2], whose
// remainder is 5e-9 of the result; a step off at most in all.  0 below e^-86.
__device__ __forceinline__ float exp_factor(float d) {
  constexpr double kLn2 = 0.69314718055994530942;
  constexpr float kHigh = (float)kLn2, kRest = (float)(kLn2 - (double)kHigh);
  if (!(d > -86.0f)) return d != d ? d : 0.0f;
  const float n = rintf(d * kLog2e), g = fmaf(-n, kRest, fmaf(-n, kHigh, d));
  float p = 1.0f / 5040.0f;
  p = fmaf(p, g, 1.0f / 720.0f);
  p = fmaf(p, g, 1.0f / 120.0f);
  p = fmaf(p, g, 1.0f / 24.0f);
  p = fmaf(p, g, 1.0f / 6.0f);
  p = fmaf(p, g, 0.5f);
  p = fmaf(p, g, 1.0f);
  p = fmaf(p, g, 1.0f);
  return p * __int_as_float(((int)n + 127) << 23);
}

// A row's elements lie in 16-byte vectors counted from the aligned address at
// or below its first element; vector i holds elements [i*N - head, i*N - head + N).
template <typename T>
struct RowVecs {
  static constexpr int N = 16 / (int)sizeof(T);
  const T *row;
  int64_t len;
  int head;
  __device__ RowVecs(const T *r, int64_t n) : row(r), len(n), head((int)((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T))) {}
  __device__ int64_t count() const { return (head + len + N - 1) / N; }
  // First element of vector i (may lie before the row for i = 0).
  __device__ int64_t first(int64_t i) const { return i * N - head; }
  __device__ bool whole(int64_t i) const { return first(i) >= 0 && first(i) + N <= len; }
  __device__ uint4 load_whole(int64_t i) const { return __ldg(reinterpret_cast<const uint4 *>(row + first(i))); }
  // The vector's values; elements outside the row read as -inf, and none of
  // them is touched in memory.
  __device__ void load_edge(int64_t i, float (&v)[N]) const {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int64_t at = first(i) + e;
      v[e] = (at >= 0 && at < len) ? to_f32(row[at]) : kNegInf;
    }
  }
};

__device__ __forceinline__ void unpack(uint4 q, float (&v)[4], const float *) {
  v[0] = __uint_as_float(q.x), v[1] = __uint_as_float(q.y), v[2] = __uint_as_float(q.z), v[3] = __uint_as_float(q.w);
}
__device__ __forceinline__ void unpack(uint4 q, float (&v)[8], const __nv_bfloat16 *) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void unpack(uint4 q, float (&v)[8], const __half *) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// Two f32 values per register pair: sm_100a adds and multiplies such pairs in
// one instruction, which halves what the streaming loops have to issue.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long &>(r))
      : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long &>(r))
      : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long &>(r))
      : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)),
        "l"(reinterpret_cast<unsigned long long &>(c)));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// exp_below of both.
__device__ __forceinline__ float2 exp_below2(float2 d) {
  const float2 t = fma2(d, make_float2(kLog2eRest, kLog2eRest), mul2(d, make_float2(kLog2e, kLog2e)));
  return make_float2(ex2(t.x), ex2(t.y));
}

// Largest of a vector's values (NaN ones aside).
__device__ __forceinline__ float top_of(uint4 q, const float *) {
  return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
}
template <typename H2>
__device__ __forceinline__ H2 top_pairs(uint4 q) {
  const H2 *h = reinterpret_cast<const H2 *>(&q);
  return __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
}
__device__ __forceinline__ float top_of(uint4 q, const __nv_bfloat16 *) {
  const float2 f = __bfloat1622float2(top_pairs<__nv_bfloat162>(q));
  return fmaxf(f.x, f.y);
}
__device__ __forceinline__ float top_of(uint4 q, const __half *) {
  const float2 f = __half22float2(top_pairs<__half2>(q));
  return fmaxf(f.x, f.y);
}

// (maximum, sum of exp(x - maximum)).  A NaN or +inf among the values leaves the
// sum NaN; nothing but -inf leaves (-inf, 0).  Exponentials are off by 2^-22 at
// most, that of a difference of 0 is exact.
struct SoftSum {
  float m, z;
  __device__ static SoftSum none() { return {kNegInf, 0.0f}; }
  __device__ bool valid() const { return z > 0.0f && z < -kNegInf; }  // false for NaN too
};

// What a sum with maximum x is multiplied by under the maximum m >= x.
__device__ __forceinline__ float factor_from(float x, float m) {
  return exp_factor(x - (m == kNegInf ? 0.0f : m));
}

// A thread's sum under way, relative to a base that stays while the values pass
// it by no more than kSlack (e^8 of room, of e^88): a base that followed every
// new maximum would have the sum multiplied, and rounded, in most steps.
struct SoftRun {
  static constexpr float kSlack = 8.0f;
  float m, base, z;  // largest value so far, base <= m, sum of exp(x - base)
  __device__ static SoftRun none() { return {kNegInf, kNegInf, 0.0f}; }
  __device__ __forceinline__ void raise(float top) {  // before values up to `top` are added
    m = fmaxf(m, top);
    if (top - base > kSlack) {  // hardly ever more than once after the first values
      z *= exp_below(base - top);
      base = top;
    }
  }
  __device__ __forceinline__ float from() const { return base == kNegInf ? 0.0f : base; }
  __device__ SoftSum sum() const { return {m, z * factor_from(base, m)}; }
};

// Returns the largest of the values (NaN ones aside).
template <int N>
__device__ __forceinline__ float soft_add(SoftRun &s, const float (&v)[N]) {
  float top = v[0];
#pragma unroll
  for (int e = 1; e < N; ++e) top = fmaxf(top, v[e]);
  s.raise(top);
  const float base = s.from();
  float a = 0.0f;
#pragma unroll
  for (int e = 0; e < N; ++e) a += exp_below(v[e] - base);
  s.z += a;
  return top;
}

// The same for U whole vectors (and each one's largest value): one look at the
// maximum for all of them.
template <typename T, int U>
__device__ __forceinline__ float soft_add(SoftRun &s, const uint4 (&q)[U], float (&tops)[U]) {
  constexpr int N = RowVecs<T>::N;
#pragma unroll
  for (int u = 0; u < U; ++u) tops[u] = top_of(q[u], (const T *)nullptr);
  float top = tops[0];
#pragma unroll
  for (int u = 1; u < U; ++u) top = fmaxf(top, tops[u]);
  s.raise(top);
  const float base = s.from();
  const float2 minus = make_float2(-base, -base);
  float2 a = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float v[N];
    unpack(q[u], v, (const T *)nullptr);
#pragma unroll
    for (int e = 0; e < N; e += 2) a = add2(a, exp_below2(add2(make_float2(v[e], v[e + 1]), minus)));
  }
  s.z += a.x + a.y;
  return top;
}

__device__ __forceinline__ SoftSum soft_join(SoftSum a, SoftSum b) {
  SoftSum r;
  r.m = fmaxf(a.m, b.m);
  r.z = a.z * factor_from(a.m, r.m) + b.z * factor_from(b.m, r.m);
  return r;
}

// Joins the sums of a warp in a fixed order: all lanes have the result.  The
// maximum comes first, so that each sum is multiplied once.
__device__ __forceinline__ SoftSum soft_join_warp(SoftSum s) {
  float m = s.m;
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
  s.z *= factor_from(s.m, m);
  s.m = m;
#pragma unroll
  for (int d = 16; d; d >>= 1) s.z += __shfl_xor_sync(~0u, s.z, d);
  return s;
}

// Joins the block's partial sums in a fixed order; thread 0 has the result.
template <int THREADS>
__device__ SoftSum soft_join_block(SoftSum s, SoftSum *smem /* [THREADS / 32] */) {
  constexpr int kWarps = THREADS / 32;
  static_assert(kWarps <= 32, "a warp joins the warps' sums");
  s = soft_join_warp(s);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) s = soft_join_warp(threadIdx.x < kWarps ? smem[threadIdx.x] : SoftSum::none());
  return s;
}

// This thread's share of the sum of a row's vectors [v0, v1), U of them added while
// U more are on their way; calls note(vector, its largest value) for those that
// may hold something above `bound`.
template <typename T, int THREADS, int U, typename Note>
__device__ __forceinline__ SoftSum soft_stream(const RowVecs<T> &r, int64_t v0, int64_t v1, float bound, Note &&note) {
  constexpr int N = RowVecs<T>::N;
  SoftRun s = SoftRun::none();
  constexpr int64_t kStep = U * THREADS;
  // The vectors that the row's ends cut, one by one; [w0, w1) are whole.
  const int64_t w0 = r.whole(v0) ? v0 : v0 + 1, w1 = v1 > w0 && !r.whole(v1 - 1) ? v1 - 1 : v1;
  auto edge = [&](int64_t i) {
    float v[N];
    r.load_edge(i, v);
    note(i, soft_add(s, v));
  };
  if (threadIdx.x == 0 && w0 > v0) edge(v0);
  if (threadIdx.x == 32 && w1 < v1) edge(v1 - 1);
  int64_t i = w0 + threadIdx.x;
  auto full = [&](int64_t at) { return at + (U - 1) * THREADS < w1; };
  auto fetch = [&](uint4 (&q)[U], int64_t at) {
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = r.load_whole(at + u * THREADS);
  };
  auto take = [&](const uint4 (&q)[U], int64_t at) {
    float tops[U];
    if (soft_add<T, U>(s, q, tops) > bound) {
#pragma unroll
      for (int u = 0; u < U; ++u) note(at + u * THREADS, tops[u]);
    }
  };
  if (full(i)) {
    uint4 q[U], ahead[U];
    fetch(q, i);
    for (;;) {
      if (!full(i + kStep)) {
        take(q, i);
        i += kStep;
        break;
      }
      fetch(ahead, i + kStep);
      take(q, i);
      i += kStep;
      if (!full(i + kStep)) {
        take(ahead, i);
        i += kStep;
        break;
      }
      fetch(q, i + kStep);
      take(ahead, i);
      i += kStep;
    }
  }
  for (; i < w1; i += THREADS) {
    float v[N];
    unpack(r.load_whole(i), v, (const T *)nullptr);
    note(i, soft_add(s, v));
  }
  return s.sum();
}

}  // namespace ftb
