// Sequence operators: what the C entries (nkb_sequence_abi.cpp) and the kernels share.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>
#include "../../include/nuka_b200.h"

namespace nkb {

void SetLastError(const char* text);           // the text of nuka_last_error_message()

// Each launch_* enqueues its kernels and returns the runtime's answer; arguments are checked by the caller.
cudaError_t launch_episodes_from_offsets(const nuka_b200_episodes_t& p, const int32_t* offsets, cudaStream_t stream);
cudaError_t launch_episodes_from_done(const nuka_b200_episodes_t& p, const uint8_t* done, cudaStream_t stream);

uint64_t recurrence_workspace(const nuka_b200_episodes_t& plan, int64_t channels);
cudaError_t launch_recurrence(const nuka_b200_recurrence_t& d, bool backward, cudaStream_t stream);
cudaError_t launch_recurrence_step(uint32_t dtype, int64_t n, int64_t channels, const void* x, int64_t x_stride, const void* gate, int64_t gate_stride,
                                   const uint8_t* fresh, float* state, void* h, cudaStream_t stream);

uint64_t heads_workspace(int64_t tokens, int64_t dim);
cudaError_t launch_heads(const nuka_b200_heads_t& d, bool backward, cudaStream_t stream);

int64_t attention_pitch(int64_t tokens);
cudaError_t launch_attention(const nuka_b200_attention_t& d, bool backward, cudaStream_t stream);

uint64_t history_workspace(const nuka_b200_history_t& d);
cudaError_t launch_history(const nuka_b200_history_t& d, cudaStream_t stream);
cudaError_t launch_history_advance(int32_t* position, const uint8_t* fresh, int64_t envs, cudaStream_t stream);

}  // namespace nkb
