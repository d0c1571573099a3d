// The vocabulary projection of many requests at once, each request with a
// low-rank adapter of its own beside the shared weight:
//
//   u[t, r] = s_a sum_d h[t, d] A_a[r, d]
//   y[t, v] = sum_d h[t, d] W[v, d] + sum_r u[t, r] B_a[v, r]
//
// Two kernels: the first makes u in 32 bits (D r products per token), the
// second the logits, a tile of 64 vocabulary entries by 16 tokens per CTA.
#include <algorithm>
#include <string>

#include "../engine.hpp"
#include "cuda_util.hpp"
#include "head_ops.hpp"
#include "row_stream.cuh"

namespace ftb {
namespace {

constexpr uint32_t kMaxRank = 256;
constexpr uint32_t kMaxAdapters = 65536;

template <typename T>
__global__ void shrink_kernel(ft_adapter_args a, float *u) {
  const uint64_t tok = blockIdx.x, req = tok / a.num_outpos;
  const int32_t id = a.adapter_ids[req];
  const T *h = static_cast<const T *>(a.hidden) + tok * a.dim;
  const uint32_t lane = threadIdx.x & 31;
  for (uint32_t r = threadIdx.x >> 5; r < a.rank; r += blockDim.x >> 5) {
    float s = 0.0f;
    if (id >= 0 && (uint32_t)id < a.num_adapters) {
      const T *w = static_cast<const T *>(a.lora_a) + ((uint64_t)id * a.rank + r) * a.dim;
      for (uint32_t d = lane; d < a.dim; d += 32) s = fmaf(to_f32(h[d]), to_f32(w[d]), s);
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
      s *= a.scale ? a.scale[id] : 1.0f;
    } else if (id != -1) {
      s = __int_as_float(0x7FC00000);
    }
    if (lane == 0) u[tok * a.rank + r] = s;
  }
}

constexpr int kTileV = 64, kTileT = 16, kTileD = 32;

template <typename T, typename O>
__global__ void __launch_bounds__(256) logits_kernel(ft_adapter_args a, const float *u, uint64_t tokens) {
  __shared__ float w[kTileD][kTileV + 1], h[kTileD][kTileT + 1];
  const uint64_t t0 = (uint64_t)blockIdx.y * kTileT;
  const uint32_t v0 = blockIdx.x * kTileV;
  const uint32_t tv = threadIdx.x % kTileV, tt = threadIdx.x / kTileV;  // each thread: one v, 4 tokens
  float acc[4] = {};
  for (uint32_t d0 = 0; d0 < a.dim; d0 += kTileD) {
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kTileV * kTileD; i += 256) {
      const uint32_t v = v0 + i / kTileD, d = d0 + i % kTileD;
      w[i % kTileD][i / kTileD] =
          v < a.vocab && d < a.dim ? to_f32(static_cast<const T *>(a.weight)[(uint64_t)v * a.dim + d]) : 0.0f;
    }
    for (uint32_t i = threadIdx.x; i < kTileT * kTileD; i += 256) {
      const uint64_t t = t0 + i / kTileD;
      const uint32_t d = d0 + i % kTileD;
      h[i % kTileD][i / kTileD] = t < tokens && d < a.dim ? to_f32(static_cast<const T *>(a.hidden)[t * a.dim + d]) : 0.0f;
    }
    __syncthreads();
    for (int d = 0; d < kTileD; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[q] = fmaf(w[d][tv], h[d][tt * 4 + q], acc[q]);
  }
  const uint32_t v = v0 + tv;
  if (v >= a.vocab) return;
  for (int q = 0; q < 4; ++q) {
    const uint64_t t = t0 + tt * 4 + q;
    if (t >= tokens) continue;
    if (u) {
      const int32_t id = a.adapter_ids[t / a.num_outpos];
      if (id >= 0 && (uint32_t)id < a.num_adapters) {
        const T *b = static_cast<const T *>(a.lora_b) + ((uint64_t)id * a.vocab + v) * a.rank;
        for (uint32_t r = 0; r < a.rank; ++r) acc[q] = fmaf(u[t * a.rank + r], to_f32(b[r]), acc[q]);
      } else if (id != -1) {
        acc[q] = __int_as_float(0x7FC00000);
      }
    }
    from_f32(acc[q], static_cast<O *>(a.out)[t * a.vocab + v]);
  }
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
  if ((uint64_t)a.n * a.num_outpos > 0x3FFFFF || a.vocab > 0x7FFFFF00u || a.dim > 0x7FFFFF00u)
    throw InvalidArgument("adapter_logits: too many tokens or too large a vocabulary");
}

uint64_t align256(uint64_t x) { return (x + 255) & ~(uint64_t)255; }

}  // namespace

uint64_t adapter_logits_workspace(const ft_adapter_args &a) {
  check_adapter(a);
  return a.num_adapters ? align256((uint64_t)a.n * a.num_outpos * a.rank * 4) : 0;
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
  const uint64_t bytes = adapter_logits_workspace(a);
  if (ws_bytes < bytes || (bytes && (!ws || (reinterpret_cast<uintptr_t>(ws) & 255))))
    throw InvalidArgument("adapter_logits: needs a 256-byte aligned workspace of " + std::to_string(bytes) + " bytes");
  const uint64_t tokens = (uint64_t)a.n * a.num_outpos;
  float *u = a.num_adapters ? static_cast<float *>(ws) : nullptr;
  const dim3 grid((a.vocab + kTileV - 1) / kTileV, (unsigned)((tokens + kTileT - 1) / kTileT));
  auto run = [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (u) {
      shrink_kernel<T><<<(unsigned)tokens, 256, 0, stream>>>(a, u);
      CUDA_TRY(cudaGetLastError());
    }
    if (a.out_dtype == FT_DTYPE_F32)
      logits_kernel<T, float><<<grid, 256, 0, stream>>>(a, u, tokens);
    else
      logits_kernel<T, T><<<grid, 256, 0, stream>>>(a, u, tokens);
    CUDA_TRY(cudaGetLastError());
  };
  if (a.dtype == FT_DTYPE_BF16)
    run((__nv_bfloat16 *)nullptr);
  else
    run((__half *)nullptr);
}

}  // namespace ftb
