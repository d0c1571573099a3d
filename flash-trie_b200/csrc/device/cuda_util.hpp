#pragma once

#include <cuda_runtime.h>

#include <stdexcept>
#include <string>

namespace ftb {

class CudaError : public std::runtime_error {
 public:
  explicit CudaError(const std::string &m) : std::runtime_error(m) {}
};

[[noreturn]] inline void throw_cuda(cudaError_t e, const char *what, const char *file, int line) {
  throw CudaError(std::string("CUDA error: ") + cudaGetErrorString(e) + " (" + what + " at " + file + ":" +
                  std::to_string(line) + ")");
}

// Lets a kernel have up to `most` bytes of dynamic shared memory. Every caller
// of a kernel gives the same `most`: a smaller one would take effect for a call
// that another thread is about to make.
template <typename K>
inline void allow_shared(K *kernel, int most) {
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e != cudaSuccess) throw_cuda(e, "cudaFuncSetAttribute", __FILE__, __LINE__);
}

}  // namespace ftb

#define CUDA_TRY(expr)                                                   \
  do {                                                                   \
    cudaError_t ft_e_ = (expr);                                          \
    if (ft_e_ != cudaSuccess) ::ftb::throw_cuda(ft_e_, #expr, __FILE__, __LINE__); \
  } while (0)
