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

uint64_t convolution_workspace(const nuka_b200_episodes_t& plan, int64_t channels, int64_t width);
cudaError_t launch_convolution(const nuka_b200_convolution_t& d, bool backward, cudaStream_t stream);
cudaError_t launch_convolution_step(const nuka_b200_convolution_step_t& d, cudaStream_t stream);

uint64_t scan_kept(const nuka_b200_episodes_t& plan, int64_t channels, int64_t states);
uint64_t scan_workspace(const nuka_b200_episodes_t& plan, int64_t channels, int64_t states, bool backward);
int64_t scan_blocks(const nuka_b200_episodes_t& plan, int64_t channels, int64_t states);
cudaError_t launch_scan(const nuka_b200_scan_t& d, bool backward, cudaStream_t stream);
cudaError_t launch_scan_step(const nuka_b200_scan_step_t& d, cudaStream_t stream);

uint64_t heads_workspace(int64_t tokens, int64_t dim);
cudaError_t launch_heads(const nuka_b200_heads_t& d, bool backward, cudaStream_t stream);

int64_t attention_pitch(int64_t tokens);
uint64_t attention_workspace(const nuka_b200_attention_t& d, int64_t sinks);
cudaError_t launch_attention(const nuka_b200_attention_t& d, int64_t sinks, void* workspace, bool backward, cudaStream_t stream);

uint64_t history_workspace(const nuka_b200_history_t& d);
cudaError_t launch_history(const nuka_b200_history_t& d, int64_t sinks, cudaStream_t stream);
cudaError_t launch_history_advance(int32_t* position, const uint8_t* fresh, int64_t envs, cudaStream_t stream);

}  // namespace nkb
