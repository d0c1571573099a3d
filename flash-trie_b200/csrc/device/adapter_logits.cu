// The vocabulary projection of many requests at once, each request with a
// low-rank adapter of its own beside the shared weight:
//
//   u[t, r] = s_a sum_d h[t, d] A_a[r, d]
//   y[t, v] = sum_d h[t, d] W[v, d] + sum_r u[t, r] B_a[v, r]
//
// Two kernels.  The first makes u in 32 bits (D r products per token).  The
// second makes the logits on the tensor cores with the vocabulary as the row
// side of the product: a tile is 128 vocabulary entries by up to 256 tokens,
// so few tokens cost a narrow product, not padded rows, and a thread of the
// epilogue holds one vocabulary entry for all tokens of its tile, whose stores
// run along the vocabulary.
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
constexpr int kThreads = 192;  // warps 0-3: epilogue, 4: loads, 5: products

template <typename T>
__device__ __forceinline__ void unpack8(uint4 q, float (&v)[8]) {
  unpack(q, v, (const T *)nullptr);
}

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
      for (uint32_t d = lane * 8; d < a.dim; d += 256) {
        float x[8], y[8];
        unpack8<T>(__ldg(reinterpret_cast<const uint4 *>(h + d)), x);
        unpack8<T>(__ldg(reinterpret_cast<const uint4 *>(w + d)), y);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(x[e], y[e], s);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
      s *= a.scale ? a.scale[id] : 1.0f;
    }
    if (lane == 0) u[tok * a.rank + r] = s;
  }
}

struct LogitsPlan {
  uint32_t tokens;       // n * num_outpos
  uint32_t tile_t;       // tokens of a tile, a multiple of 16
  uint32_t tiles_t;
  uint32_t tiles_v;
  uint32_t stages;
  uint32_t tmem_half;    // columns of one of the two accumulators
};

struct alignas(8) LogitsShared {
  uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
  uint32_t tmem, gave_up;
};

LogitsPlan plan_logits(const ft_adapter_args &a) {
  LogitsPlan p;
  p.tokens = a.n * a.num_outpos;
  p.tiles_t = (p.tokens + kMaxTileT - 1) / kMaxTileT;
  const uint32_t each = (p.tokens + p.tiles_t - 1) / p.tiles_t;
  p.tile_t = (each + 15) / 16 * 16;
  p.tiles_v = (a.vocab + kTileV - 1) / kTileV;
  const uint32_t stage = (kTileV + p.tile_t) * kTileD * 2;
  p.stages = std::min<uint32_t>(kMaxStages, (225 * 1024) / stage);
  p.tmem_half = 32;
  while (p.tmem_half < p.tile_t) p.tmem_half *= 2;
  return p;
}
size_t logits_smem(const LogitsPlan &p) { return 1024 + (size_t)p.stages * (kTileV + p.tile_t) * kTileD * 2; }

// Persistent, one CTA per SM.  Tiles that share a stretch of the weight are
// neighbours in the order, so that it comes from DRAM once.
template <typename T, typename O>
__global__ void __launch_bounds__(kThreads, 1)
    logits_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_h, ft_adapter_args a,
                  LogitsPlan p, const float *u) {
  using namespace sm100;
  extern __shared__ uint8_t raw[];
  uint8_t *buf = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  __shared__ LogitsShared sh;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bytes_w = kTileV * kTileD * 2, bytes_h = p.tile_t * kTileD * 2, bytes = bytes_w + bytes_h;
  const uint32_t tiles = p.tiles_t * p.tiles_v, chunks = (a.dim + kTileD - 1) / kTileD;
  volatile uint32_t *gave_up = &sh.gave_up;
  if (threadIdx.x == 0) {
    sh.gave_up = 0;
    for (uint32_t s = 0; s < p.stages; ++s) mbar_init(&sh.full[s], 1), mbar_init(&sh.empty[s], 1);
    for (int b = 0; b < 2; ++b) mbar_init(&sh.acc_full[b], 1), mbar_init(&sh.acc_empty[b], 128);
    mbar_init_fence();
    prefetch_map(&map_w);
    prefetch_map(&map_h);
  }
  if (warp == 5) tmem_alloc(&sh.tmem, 2 * p.tmem_half);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;

  if (warp == 4) {
    if (elect_one()) {
      uint32_t at = 0, sent = 0;  // stage and number of stages filled so far
      bool ok = true;
      for (uint32_t tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
        const int32_t v0 = (int32_t)(tile / p.tiles_t * kTileV), t0 = (int32_t)(tile % p.tiles_t * p.tile_t);
        for (uint32_t c = 0; c < chunks; ++c) {
          if (sent >= p.stages) ok = mbar_wait(&sh.empty[at], (sent / p.stages - 1) & 1, gave_up);
          if (!ok) break;
          uint8_t *st = buf + (size_t)at * bytes;
          mbar_expect(&sh.full[at], bytes);
          tma_load_2d(st, &map_w, &sh.full[at], (int32_t)(c * kTileD), v0);
          tma_load_2d(st + bytes_w, &map_h, &sh.full[at], (int32_t)(c * kTileD), t0);
          ++sent;
          at = at + 1 == p.stages ? 0 : at + 1;
        }
      }
      // Copies must not land in a block that has ended: wait for the stages
      // still in flight (those before were seen full by the products).
      if (!ok)
        for (uint32_t s = 0; s < p.stages && s < sent; ++s) {
          const uint32_t fills = (sent - 1 - s) / p.stages;  // number of the last fill of stage s
          for (uint32_t i = 0; i < kWaitTries && !mbar_try(&sh.full[s], fills & 1); ++i) {
          }
        }
    }
  } else if (warp == 5) {
    if (elect_one()) {
      const uint32_t shape = mma_shape(sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value, kTileV, p.tile_t);
      uint32_t at = 0, phase = 0, n = 0;
      bool ok = true;
      for (uint32_t tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, ++n) {
        const uint32_t b = n & 1, d = tmem + b * p.tmem_half;
        if (n >= 2) ok = mbar_wait(&sh.acc_empty[b], (n / 2 - 1) & 1, gave_up);
        if (!ok) break;
        fence_after();
        for (uint32_t c = 0; c < chunks; ++c) {
          ok = mbar_wait(&sh.full[at], phase, gave_up);
          if (!ok) break;
          fence_after();
          const uint64_t w = operand(buf + (size_t)at * bytes), h = operand(buf + (size_t)at * bytes + bytes_w);
#pragma unroll
          for (int k = 0; k < kTileD / 16; ++k) mma_f16(d, w + 2 * k, h + 2 * k, shape, c > 0 || k > 0);
          mma_commit(&sh.empty[at]);
          if (++at == p.stages) at = 0, phase ^= 1;
        }
        if (ok) mma_commit(&sh.acc_full[b]);
      }
    }
  } else {
    uint32_t n = 0;
    bool ok = true;
    for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++n) {
      const uint32_t b = n & 1;
      const uint32_t v = tile / p.tiles_t * kTileV + threadIdx.x, t0 = tile % p.tiles_t * p.tile_t;
      const bool live = v < a.vocab;
      if (ok) ok = mbar_wait(&sh.acc_full[b], (n / 2) & 1, gave_up);
      ok = __all_sync(~0u, ok);
      if (ok) fence_after();
      O *out = static_cast<O *>(a.out) + (uint64_t)t0 * a.vocab + v;
      const uint32_t count = min(p.tile_t, p.tokens - t0);
      for (uint32_t c0 = 0; c0 < count; c0 += 16) {
        uint32_t acc[16];
        if (ok) {
          tmem_load16(tmem + b * p.tmem_half + c0 + (warp << 21), acc);
        } else {
          // A wait ran out: no result is better than a wrong one.
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[e] = 0x7FC00000;
        }
        if (u && live) {
          // The low-rank part in 32 bits: the entry's row of the adapter's B,
          // read once for all neighbouring tokens of the same request.
          for (uint32_t c = c0; c < min(c0 + 16, count);) {
            const uint32_t req = (t0 + c) / a.num_outpos;
            const uint32_t end = min(min(c0 + 16, count), (req + 1) * a.num_outpos - t0);
            const int32_t id = a.adapter_ids[req];
            if ((uint32_t)id < a.num_adapters) {
              const T *row = static_cast<const T *>(a.lora_b) + ((uint64_t)id * a.vocab + v) * a.rank;
              for (uint32_t r = 0; r < a.rank; r += 8) {
                float w[8];
                unpack8<T>(__ldg(reinterpret_cast<const uint4 *>(row + r)), w);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  if (c0 + e >= c && c0 + e < end) {
                    const float4 *x = reinterpret_cast<const float4 *>(u + (uint64_t)(t0 + c0 + e) * a.rank + r);
                    const float4 x0 = __ldg(x), x1 = __ldg(x + 1);
                    float s = __uint_as_float(acc[e]);
                    s = fmaf(x0.x, w[0], s), s = fmaf(x0.y, w[1], s), s = fmaf(x0.z, w[2], s), s = fmaf(x0.w, w[3], s);
                    s = fmaf(x1.x, w[4], s), s = fmaf(x1.y, w[5], s), s = fmaf(x1.z, w[6], s), s = fmaf(x1.w, w[7], s);
                    acc[e] = __float_as_uint(s);
                  }
                }
              }
            } else if (id != -1) {
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (c0 + e >= c && c0 + e < end) acc[e] = 0x7FC00000;
            }
            c = end;
          }
        }
        if (live) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (c0 + e < count) from_f32(__uint_as_float(acc[e]), out[(uint64_t)(c0 + e) * a.vocab]);
        }
        __syncwarp();
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
  if (warp == 5) tmem_free(tmem, 2 * p.tmem_half);
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

// Rows of `inner` 16-bit values, loaded as boxes of 64 values by `box` rows
// with the 128-byte swizzle; what lies outside reads as 0.
CUtensorMap make_map(const void *base, bool bf16, uint64_t inner, uint64_t rows, uint32_t box, const char *what) {
  CUtensorMap m;
  const cuuint64_t dims[2] = {inner, rows}, strides[1] = {inner * 2};
  const cuuint32_t tile[2] = {(cuuint32_t)kTileD, box}, step[2] = {1, 1};
  const CUresult rc =
      encode_fn()(&m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
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
  const LogitsPlan p = plan_logits(a);
  float *u = a.num_adapters ? static_cast<float *>(ws) : nullptr;
  const bool bf16 = a.dtype == FT_DTYPE_BF16;
  const CUtensorMap map_w = make_map(a.weight, bf16, a.dim, a.vocab, kTileV, "weight");
  const CUtensorMap map_h = make_map(a.hidden, bf16, a.dim, p.tokens, p.tile_t, "hidden");
  const size_t smem = logits_smem(p);
  const unsigned grid = std::min<unsigned>(p.tiles_t * p.tiles_v, (unsigned)sm_count());
  auto run = [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (u) {
      shrink_kernel<T><<<p.tokens, 256, 0, stream>>>(a, u);
      CUDA_TRY(cudaGetLastError());
    }
    auto *kernel = a.out_dtype == FT_DTYPE_F32 ? logits_kernel<T, float> : logits_kernel<T, T>;
    CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kernel<<<grid, kThreads, smem, stream>>>(map_w, map_h, a, p, u);
    CUDA_TRY(cudaGetLastError());
  };
  if (a.dtype == FT_DTYPE_BF16)
    run((__nv_bfloat16 *)nullptr);
  else
    run((__half *)nullptr);
}

}  // namespace ftb
