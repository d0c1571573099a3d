// Launchers of the model-side operators (declared in include/flashtrie_b200.h):
// the vocabulary projection with per-request adapters, the proposals, the
// sequence scores and the preference loss.  They run on the current device,
// enqueue on `stream` and keep no state between calls.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "../../../include/flashtrie_b200.h"

namespace ftb {

uint64_t propose_workspace(const ft_propose_args &a);
void propose_device(const ft_propose_args &a, void *ws, uint64_t ws_bytes, cudaStream_t stream);

uint64_t sequence_logp_workspace(const ft_sequence_args &a);
void sequence_logp_device(const ft_sequence_args &a, void *ws, uint64_t ws_bytes, cudaStream_t stream);
void sequence_grad_device(const ft_sequence_args &a, const float *grad, const float *factor, const float *upstream,
                          void *ws, uint64_t ws_bytes, cudaStream_t stream);

uint64_t preference_workspace(const ft_sequence_args &a);
void preference_loss_device(const ft_sequence_args &a, const ft_preference_args &p, void *ws, uint64_t ws_bytes,
                            cudaStream_t stream);

uint64_t adapter_logits_workspace(const ft_adapter_args &a);
void adapter_logits_device(const ft_adapter_args &a, uint32_t *status, void *ws, uint64_t ws_bytes,
                           cudaStream_t stream);

}  // namespace ftb
