// The C entries of the sequence operators: arguments are checked here, kernels are enqueued by the launch_* functions.
// Nothing here allocates or throws.
#include <cstdio>
#include "nkb_sequence.h"

namespace {

nuka_result_t Refuse(nuka_result_t code, const char* text) { nkb::SetLastError(text); return code; }
nuka_result_t Invalid(const char* text) { return Refuse(NUKA_RESULT_INVALID_ARG, text); }

nuka_result_t Ran(cudaError_t e) {
    if (e == cudaSuccess) return NUKA_RESULT_OK;
    nkb::SetLastError(cudaGetErrorString(e));
    cudaGetLastError();
    return NUKA_RESULT_CUDA_ERROR;
}

cudaStream_t StreamOf(void* s) { return static_cast<cudaStream_t>(s); }
bool Aligned(const void* p, uint64_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0u; }
uint64_t SizeOf(uint32_t dtype) { return dtype == NUKA_B200_F32 ? 4u : 2u; }
constexpr int64_t kMostTokens = (1ll << 31) - 1025;     // token indices, and a tile past them, fit 32 bits

const char* PlanFault(const nuka_b200_episodes_t* p) {
    if (p == nullptr) return "the plan is null";
    if (p->tokens < 0 || p->rows < 0 || p->tokens > kMostTokens || p->rows > kMostTokens) return "tokens or rows of the plan are negative or too many";
    if (p->tokens != 0 && p->rows == 0) return "tokens without a row";
    if (p->length < 0 || (p->length != 0 && p->length * p->rows != p->tokens)) return "rows of one length do not give the plan's tokens";
    if (p->tokens != 0 && (p->first == nullptr || p->end == nullptr || p->link == nullptr || p->tail == nullptr)) return "an array of the plan is null";
    for (const int32_t* a : {p->first, p->end, p->link, p->tail})
        if (!Aligned(a, 4)) return "an array of the plan does not lie on 4 bytes";
    return nullptr;
}

}  // namespace

extern "C" {

nuka_result_t nuka_b200_episodes_from_offsets(const nuka_b200_episodes_t* plan, const int32_t* offsets, void* stream) {
    if (const char* fault = PlanFault(plan)) return Invalid(fault);
    if (plan->tokens != 0 && (offsets == nullptr || !Aligned(offsets, 4))) return Invalid("offsets are null or not on 4 bytes");
    return Ran(nkb::launch_episodes_from_offsets(*plan, offsets, StreamOf(stream)));
}

nuka_result_t nuka_b200_episodes_from_done(const nuka_b200_episodes_t* plan, const uint8_t* done, void* stream) {
    if (const char* fault = PlanFault(plan)) return Invalid(fault);
    if (plan->tokens != 0 && plan->length == 0) return Invalid("the rows' length is 0");
    if (plan->tokens != 0 && done == nullptr) return Invalid("done is null");
    return Ran(nkb::launch_episodes_from_done(*plan, done, StreamOf(stream)));
}

uint64_t nuka_b200_recurrence_workspace(const nuka_b200_episodes_t* plan, int64_t channels) {
    return PlanFault(plan) != nullptr || plan->tokens == 0 || channels <= 0 ? 0u : nkb::recurrence_workspace(*plan, channels);
}

static nuka_result_t Recurrence(const nuka_b200_recurrence_t* desc, bool backward, void* stream) {
    if (desc == nullptr) return Invalid("recurrence desc is null");
    const nuka_b200_recurrence_t& d = *desc;
    if (const char* fault = PlanFault(d.plan)) return Invalid(fault);
    if (d.dtype > NUKA_B200_BF16) return Refuse(NUKA_RESULT_NOT_SUPPORTED, "dtype must be F32, F16 or BF16");
    if (d.channels < 0 || d.channels > (1 << 24)) return Invalid("channels must be 0 to 2^24");
    if (d.x_stride < 0 || d.gate_stride < 0) return Invalid("a stride is negative");
    if (d.plan->tokens == 0 || d.channels == 0) return NUKA_RESULT_OK;
    const uint64_t size = SizeOf(d.dtype);
    if (d.x == nullptr || d.gate == nullptr || d.h == nullptr) return Invalid("x, gate or h is null");
    if (!backward && d.state == nullptr) return Invalid("state is null");
    if (backward && (d.dh == nullptr || d.dx == nullptr || d.dgate == nullptr)) return Invalid("dh, dx or dgate is null");
    for (const void* p : {d.x, d.gate, static_cast<const void*>(d.h), d.dh, static_cast<const void*>(d.dx), static_cast<const void*>(d.dgate)})
        if (!Aligned(p, size)) return Invalid("a tensor does not lie on a multiple of its type's size");
    for (const float* p : {d.initial, static_cast<const float*>(d.state), d.dstate, static_cast<const float*>(d.dinitial)})
        if (!Aligned(p, 4)) return Invalid("a state does not lie on a multiple of 4 bytes");
    if (d.plan->tokens / 32 * (d.channels / 32 + 1) > (1ll << 31)) return Refuse(NUKA_RESULT_NOT_SUPPORTED, "too many tokens times channels");
    const uint64_t need = nkb::recurrence_workspace(*d.plan, d.channels);
    if (need != 0u && (d.workspace == nullptr || d.workspace_bytes < need || !Aligned(d.workspace, 8))) return Invalid("the workspace is null, too small or not on 8 bytes");
    return Ran(nkb::launch_recurrence(d, backward, StreamOf(stream)));
}

nuka_result_t nuka_b200_recurrence(const nuka_b200_recurrence_t* desc, void* stream) { return Recurrence(desc, false, stream); }
nuka_result_t nuka_b200_recurrence_backward(const nuka_b200_recurrence_t* desc, void* stream) { return Recurrence(desc, true, stream); }

nuka_result_t nuka_b200_recurrence_step(uint32_t dtype, int64_t n, int64_t channels, const void* x, int64_t x_stride, const void* gate, int64_t gate_stride,
                                        const uint8_t* fresh, float* state, void* h, void* stream) {
    if (dtype > NUKA_B200_BF16) return Refuse(NUKA_RESULT_NOT_SUPPORTED, "dtype must be F32, F16 or BF16");
    if (n < 0 || channels < 0 || channels > (1 << 24) || n > kMostTokens || x_stride < 0 || gate_stride < 0) return Invalid("a size or stride is negative or too large");
    if (n == 0 || channels == 0) return NUKA_RESULT_OK;
    if (x == nullptr || gate == nullptr || state == nullptr || h == nullptr) return Invalid("x, gate, state or h is null");
    if (!Aligned(x, SizeOf(dtype)) || !Aligned(gate, SizeOf(dtype)) || !Aligned(h, SizeOf(dtype)) || !Aligned(state, 4)) return Invalid("a tensor does not lie on a multiple of its type's size");
    if (n * ((channels + 3) / 4) / 32 > (1ll << 31)) return Refuse(NUKA_RESULT_NOT_SUPPORTED, "too many envs times channels");
    return Ran(nkb::launch_recurrence_step(dtype, n, channels, x, x_stride, gate, gate_stride, fresh, state, h, StreamOf(stream)));
}

static const char* ConvolutionFault(uint32_t dtype, int64_t channels, int64_t width) {
    if (dtype > NUKA_B200_BF16) return "dtype must be F32, F16 or BF16";
    if (width < 2 || width > 4) return "width must be 2, 3 or 4";
    if (channels < 0 || channels > (1 << 24)) return "channels must be 0 to 2^24";
    return nullptr;
}

uint64_t nuka_b200_convolution_workspace(const nuka_b200_episodes_t* plan, int64_t channels, int64_t width) {
    return PlanFault(plan) != nullptr || plan->tokens == 0 || channels <= 0 || ConvolutionFault(0, channels, width) != nullptr ? 0u : nkb::convolution_workspace(*plan, channels, width);
}

static nuka_result_t Convolution(const nuka_b200_convolution_t* desc, bool backward, void* stream) {
    if (desc == nullptr) return Invalid("convolution desc is null");
    const nuka_b200_convolution_t& d = *desc;
    if (const char* fault = PlanFault(d.plan)) return Invalid(fault);
    if (const char* fault = ConvolutionFault(d.dtype, d.channels, d.width)) return Refuse(NUKA_RESULT_NOT_SUPPORTED, fault);
    if (d.x_stride < 0) return Invalid("a stride is negative");
    if (!Aligned(d.weight, 4) || !Aligned(d.bias, 4) || (backward && (!Aligned(d.dweight, 4) || !Aligned(d.dbias, 4)))) return Invalid("a weight or its gradient does not lie on 4 bytes");
    if (d.channels == 0) return NUKA_RESULT_OK;
    const uint64_t size = SizeOf(d.dtype);
    if (d.plan->tokens != 0) {
        if (d.x == nullptr || d.weight == nullptr) return Invalid("x or weight is null");
        if (!backward && (d.y == nullptr || d.state == nullptr)) return Invalid("y or state is null");
        if (backward && (d.dy == nullptr || d.dx == nullptr)) return Invalid("dy or dx is null");
    }
    for (const void* p : {d.x, d.initial, static_cast<const void*>(d.y), static_cast<const void*>(d.state)})
        if (!Aligned(p, size)) return Invalid("a tensor does not lie on a multiple of its type's size");
    if (backward)
        for (const void* p : {d.dy, d.dstate, static_cast<const void*>(d.dx), static_cast<const void*>(d.dinitial)})
            if (!Aligned(p, size)) return Invalid("a gradient does not lie on a multiple of its type's size");
    if ((d.plan->tokens / 128 + 1) * (d.channels / 32 + 1) > (1ll << 30)) return Refuse(NUKA_RESULT_NOT_SUPPORTED, "too many tokens times channels");
    if (backward && d.plan->tokens != 0 && (d.dweight != nullptr || d.dbias != nullptr) &&
        (d.workspace == nullptr || !Aligned(d.workspace, 4) || d.workspace_bytes < nkb::convolution_workspace(*d.plan, d.channels, d.width))) return Invalid("the workspace is null, too small or not on 4 bytes");
    return Ran(nkb::launch_convolution(d, backward, StreamOf(stream)));
}

nuka_result_t nuka_b200_convolution(const nuka_b200_convolution_t* desc, void* stream) { return Convolution(desc, false, stream); }
nuka_result_t nuka_b200_convolution_backward(const nuka_b200_convolution_t* desc, void* stream) { return Convolution(desc, true, stream); }

nuka_result_t nuka_b200_convolution_step(const nuka_b200_convolution_step_t* desc, void* stream) {
    if (desc == nullptr) return Invalid("convolution step desc is null");
    const nuka_b200_convolution_step_t& d = *desc;
    if (const char* fault = ConvolutionFault(d.dtype, d.channels, d.width)) return Refuse(NUKA_RESULT_NOT_SUPPORTED, fault);
    if (d.envs < 0 || d.envs > kMostTokens || d.x_stride < 0) return Invalid("a size or stride is negative or too large");
    if (d.envs == 0 || d.channels == 0) return NUKA_RESULT_OK;
    if (d.x == nullptr || d.weight == nullptr || d.state == nullptr || d.y == nullptr) return Invalid("x, weight, state or y is null");
    for (const void* p : {d.x, static_cast<const void*>(d.state), static_cast<const void*>(d.y)})
        if (!Aligned(p, SizeOf(d.dtype))) return Invalid("a tensor does not lie on a multiple of its type's size");
    if (!Aligned(d.weight, 4) || !Aligned(d.bias, 4)) return Invalid("a weight does not lie on 4 bytes");
    if (d.envs * d.channels / 128 >= (1ll << 31) - 1) return Refuse(NUKA_RESULT_NOT_SUPPORTED, "too many envs times channels");
    return Ran(nkb::launch_convolution_step(d, StreamOf(stream)));
}

static const char* ScanFault(uint32_t dtype, int64_t channels, int64_t states) {
    if (dtype > NUKA_B200_BF16) return "dtype must be F32, F16 or BF16";
    if (states < 1 || states > 64) return "states must be 1 to 64";
    if (channels < 0 || channels > (1 << 24)) return "channels must be 0 to 2^24";
    return nullptr;
}

uint64_t nuka_b200_scan_kept(const nuka_b200_episodes_t* plan, int64_t channels, int64_t states) {
    return PlanFault(plan) != nullptr || plan->tokens == 0 || channels <= 0 || ScanFault(0, channels, states) != nullptr ? 0u : nkb::scan_kept(*plan, channels, states);
}
uint64_t nuka_b200_scan_workspace(const nuka_b200_episodes_t* plan, int64_t channels, int64_t states, uint32_t backward) {
    return PlanFault(plan) != nullptr || plan->tokens == 0 || channels <= 0 || ScanFault(0, channels, states) != nullptr ? 0u : nkb::scan_workspace(*plan, channels, states, backward != 0u);
}

static nuka_result_t Scan(const nuka_b200_scan_t* desc, bool backward, void* stream) {
    if (desc == nullptr) return Invalid("scan desc is null");
    const nuka_b200_scan_t& d = *desc;
    if (const char* fault = PlanFault(d.plan)) return Invalid(fault);
    if (const char* fault = ScanFault(d.dtype, d.channels, d.states)) return Refuse(NUKA_RESULT_NOT_SUPPORTED, fault);
    if (d.x_stride < 0 || d.delta_stride < 0 || d.gate_stride < 0 || d.b_stride < 0 || d.c_stride < 0) return Invalid("a stride is negative");
    for (const float* p : {d.decay, d.skip, d.delta_bias, d.initial, static_cast<const float*>(d.state)})
        if (!Aligned(p, 4)) return Invalid("a weight or state does not lie on 4 bytes");
    if (backward)
        for (const float* p : {d.dstate, static_cast<const float*>(d.ddecay), static_cast<const float*>(d.dskip), static_cast<const float*>(d.ddelta_bias), static_cast<const float*>(d.dinitial)})
            if (!Aligned(p, 4)) return Invalid("a weight's or state's gradient does not lie on 4 bytes");
    const uint64_t size = SizeOf(d.dtype);
    if (d.channels == 0 && backward && d.plan->tokens != 0)                // of what a call without channels is asked for, B's and C's gradients alone are not empty
        for (const void* p : {static_cast<const void*>(d.db), static_cast<const void*>(d.dc)})
            if (p == nullptr || !Aligned(p, size)) return Invalid("a gradient is null or does not lie on a multiple of its type's size");
    if (d.channels == 0 || d.plan->tokens == 0) return Ran(nkb::launch_scan(d, backward, StreamOf(stream)));
    for (const void* p : {d.x, d.delta, d.b, d.c, static_cast<const void*>(d.decay)})
        if (p == nullptr) return Invalid("x, delta, b, c or decay is null");
    if (!backward && (d.y == nullptr || d.state == nullptr)) return Invalid("y or state is null");
    for (const void* p : {d.x, d.delta, d.gate, d.b, d.c, static_cast<const void*>(d.y)})
        if (!Aligned(p, size)) return Invalid("a tensor does not lie on a multiple of its type's size");
    if (backward) {
        for (const void* p : {d.dy, static_cast<const void*>(d.dx), static_cast<const void*>(d.ddelta), static_cast<const void*>(d.db), static_cast<const void*>(d.dc)})
            if (p == nullptr || !Aligned(p, size)) return Invalid("a gradient is null or does not lie on a multiple of its type's size");
        if ((d.gate != nullptr && d.dgate == nullptr) || !Aligned(d.dgate, size)) return Invalid("dgate is null or does not lie on a multiple of its type's size");
    }
    if (nkb::scan_blocks(*d.plan, d.channels, d.states) > (1ll << 30)) return Refuse(NUKA_RESULT_NOT_SUPPORTED, "too many tokens times channels");
    if ((backward || d.kept != nullptr) && (d.kept == nullptr || !Aligned(d.kept, 16) || d.kept_bytes < nkb::scan_kept(*d.plan, d.channels, d.states)))
        return Invalid("what is kept for the gradient is null, too small or not on 16 bytes");
    const uint64_t need = nkb::scan_workspace(*d.plan, d.channels, d.states, backward);
    if (need != 0u && (d.workspace == nullptr || d.workspace_bytes < need || !Aligned(d.workspace, 16))) return Invalid("the workspace is null, too small or not on 16 bytes");
    return Ran(nkb::launch_scan(d, backward, StreamOf(stream)));
}

nuka_result_t nuka_b200_scan(const nuka_b200_scan_t* desc, void* stream) { return Scan(desc, false, stream); }
nuka_result_t nuka_b200_scan_backward(const nuka_b200_scan_t* desc, void* stream) { return Scan(desc, true, stream); }

nuka_result_t nuka_b200_scan_step(const nuka_b200_scan_step_t* desc, void* stream) {
    if (desc == nullptr) return Invalid("scan step desc is null");
    const nuka_b200_scan_step_t& d = *desc;
    if (const char* fault = ScanFault(d.dtype, d.channels, d.states)) return Refuse(NUKA_RESULT_NOT_SUPPORTED, fault);
    if (d.envs < 0 || d.envs > kMostTokens) return Invalid("envs are negative or too many");
    if (d.x_stride < 0 || d.delta_stride < 0 || d.gate_stride < 0 || d.b_stride < 0 || d.c_stride < 0) return Invalid("a stride is negative");
    if (d.envs == 0 || d.channels == 0) return NUKA_RESULT_OK;
    for (const void* p : {d.x, d.delta, d.b, d.c, static_cast<const void*>(d.decay), static_cast<const void*>(d.state), static_cast<const void*>(d.y)})
        if (p == nullptr) return Invalid("x, delta, b, c, decay, state or y is null");
    for (const void* p : {d.x, d.delta, d.gate, d.b, d.c, static_cast<const void*>(d.y)})
        if (!Aligned(p, SizeOf(d.dtype))) return Invalid("a tensor does not lie on a multiple of its type's size");
    for (const float* p : {d.decay, d.skip, d.delta_bias, static_cast<const float*>(d.state)})
        if (!Aligned(p, 4)) return Invalid("a weight or state does not lie on 4 bytes");
    if (d.envs * d.channels / 8 >= (1ll << 31) - 1) return Refuse(NUKA_RESULT_NOT_SUPPORTED, "too many envs times channels");
    return Ran(nkb::launch_scan_step(d, StreamOf(stream)));
}

uint64_t nuka_b200_heads_workspace(int64_t tokens, int64_t dim) { return tokens <= 0 || dim <= 0 ? 0u : nkb::heads_workspace(tokens, dim); }

static nuka_result_t Heads(const nuka_b200_heads_t* desc, bool backward, void* stream) {
    if (desc == nullptr) return Invalid("heads desc is null");
    const nuka_b200_heads_t& d = *desc;
    if (d.dtype > NUKA_B200_BF16) return Refuse(NUKA_RESULT_NOT_SUPPORTED, "dtype must be F32, F16 or BF16");
    if (d.tokens < 0 || d.tokens > kMostTokens || d.heads_q < 0 || d.heads_k < 0 || d.heads_q > 65536 || d.heads_k > 65536) return Invalid("tokens or heads are negative or too many");
    if (d.dim < 8 || d.dim > 256 || d.dim % 8 != 0 || d.turned < 0 || d.turned > d.dim || d.turned % 8 != 0)
        return Refuse(NUKA_RESULT_NOT_SUPPORTED, "dim and turned must be multiples of 8, dim 8 to 256, turned at most dim");
    if (!(d.eps >= 0.f)) return Invalid("eps must not be negative");
    if (!Aligned(d.first, 4) || !Aligned(d.positions, 4)) return Invalid("the plan's first or positions do not lie on 4 bytes");
    if (!Aligned(d.q_weight, 4) || !Aligned(d.k_weight, 4) || (backward && (!Aligned(d.dq_weight, 4) || !Aligned(d.dk_weight, 4)))) return Invalid("a weight or its gradient does not lie on 4 bytes");
    if (d.tokens == 0) return Ran(nkb::launch_heads(d, backward, StreamOf(stream)));
    if (d.turned != 0 && (d.frequencies == nullptr || !Aligned(d.frequencies, 8))) return Invalid("frequencies are null or not on 8 bytes");
    if (d.turned != 0 && d.first == nullptr && d.positions == nullptr) return Invalid("neither the plan's first nor positions are given");
    const uint64_t four = 4 * SizeOf(d.dtype);
    const void* need[] = {d.heads_q ? d.q : nullptr, d.heads_k ? d.k : nullptr};
    const void* out[] = {backward ? d.dq : d.q_out, backward ? d.dk : d.k_out};
    const void* grad[] = {d.dq_out, d.dk_out};
    const int64_t heads[] = {d.heads_q, d.heads_k}, strides[] = {d.q_stride, d.k_stride}, head_strides[] = {d.q_head_stride, d.k_head_stride};
    for (int i = 0; i < 2; ++i) {
        if (heads[i] == 0) continue;
        if (need[i] == nullptr || out[i] == nullptr || (backward && grad[i] == nullptr)) return Invalid("a tensor of queries or keys is null");
        if (!Aligned(need[i], four) || !Aligned(out[i], four) || (backward && !Aligned(grad[i], four))) return Invalid("queries and keys must lie on multiples of four values");
        if (strides[i] < 0 || head_strides[i] < 0 || strides[i] % 4 != 0 || head_strides[i] % 4 != 0) return Invalid("strides must be multiples of four values, not negative");
    }
    if (backward && (d.dq_weight != nullptr || d.dk_weight != nullptr) &&
        (d.workspace == nullptr || !Aligned(d.workspace, 4) || d.workspace_bytes < nkb::heads_workspace(d.tokens, d.dim))) return Invalid("the workspace is null, too small or not on 4 bytes");
    return Ran(nkb::launch_heads(d, backward, StreamOf(stream)));
}

nuka_result_t nuka_b200_heads(const nuka_b200_heads_t* desc, void* stream) { return Heads(desc, false, stream); }
nuka_result_t nuka_b200_heads_backward(const nuka_b200_heads_t* desc, void* stream) { return Heads(desc, true, stream); }

int64_t nuka_b200_attention_pitch(int64_t tokens) { return tokens <= 0 ? 0 : nkb::attention_pitch(tokens); }

static nuka_result_t Attention(const nuka_b200_attention_t* desc, int64_t sinks, void* workspace, uint64_t workspace_bytes, bool backward, void* stream) {
    if (desc == nullptr) return Invalid("attention desc is null");
    const nuka_b200_attention_t& d = *desc;
    if (const char* fault = PlanFault(d.plan)) return Invalid(fault);
    if (d.dtype != NUKA_B200_F16 && d.dtype != NUKA_B200_BF16) return Refuse(NUKA_RESULT_NOT_SUPPORTED, "dtype must be F16 or BF16");
    if (d.heads_k < 1 || d.heads_q < 1 || d.heads_q > 65536 || d.heads_q % d.heads_k != 0) return Invalid("heads_q must be a positive multiple of heads_k, at most 65536");
    if (d.dim < 8 || d.dim > 128 || d.dim % 8 != 0) return Refuse(NUKA_RESULT_NOT_SUPPORTED, "dim must be a multiple of 8, 8 to 128");
    if (d.window < 0 || sinks < 0) return Invalid("window and sinks must not be negative");
    if (!(d.scale > 0.f) || d.scale > 3.0e38f) return Invalid("scale must be greater than 0 and finite");
    if (d.plan->tokens == 0) return NUKA_RESULT_OK;
    if ((d.plan->tokens / 64 + 1) * d.heads_q > (1ll << 30)) return Refuse(NUKA_RESULT_NOT_SUPPORTED, "too many tokens times heads");
    for (const void* p : {d.q, d.k, d.v, static_cast<const void*>(d.out)}) {
        if (p == nullptr) return Invalid("q, k, v or out is null");
        if (!Aligned(p, 16)) return Invalid("a tensor does not lie on 16 bytes");
    }
    if (!Aligned(d.lse, 16) || (backward && (d.lse == nullptr || d.delta == nullptr || !Aligned(d.delta, 16)))) return Invalid("lse or delta is null or not on 16 bytes");
    if (backward)
        for (const void* p : {d.dout, static_cast<const void*>(d.dq), static_cast<const void*>(d.dk), static_cast<const void*>(d.dv)})
            if (p == nullptr || !Aligned(p, 16)) return Invalid("a gradient is null or not on 16 bytes");
    // a size of 1 has no stride
    const struct { int64_t size, stride; } strides[] = {{d.plan->tokens, d.q_stride}, {d.heads_q, d.q_head_stride}, {d.plan->tokens, d.k_stride}, {d.heads_k, d.k_head_stride},
                                                        {d.plan->tokens, d.v_stride}, {d.heads_k, d.v_head_stride}};
    for (const auto& s : strides)
        if (s.size > 1 && (s.stride < d.dim || s.stride % 8 != 0 || s.stride >= (1ll << 38))) return Invalid("strides must be multiples of 8 values, at least dim");
    const uint64_t need = backward ? nkb::attention_workspace(d, sinks) : 0u;
    if (need != 0u && (workspace == nullptr || workspace_bytes < need || !Aligned(workspace, 16))) return Invalid("the workspace is null, too small or not on 16 bytes");
    return Ran(nkb::launch_attention(d, sinks, workspace, backward, StreamOf(stream)));
}

nuka_result_t nuka_b200_attention(const nuka_b200_attention_t* desc, void* stream) { return Attention(desc, 0, nullptr, 0, false, stream); }
nuka_result_t nuka_b200_attention_backward(const nuka_b200_attention_t* desc, void* stream) { return Attention(desc, 0, nullptr, 0, true, stream); }
nuka_result_t nuka_b200_attention_sinks(const nuka_b200_attention_t* desc, int64_t sinks, void* stream) { return Attention(desc, sinks, nullptr, 0, false, stream); }
uint64_t nuka_b200_attention_sinks_workspace(const nuka_b200_attention_t* desc, int64_t sinks) {
    return desc == nullptr || PlanFault(desc->plan) != nullptr || desc->heads_k < 1 || desc->heads_k > 65536 || desc->dim < 8 || desc->dim > 128 ? 0u : nkb::attention_workspace(*desc, sinks);
}
nuka_result_t nuka_b200_attention_sinks_backward(const nuka_b200_attention_t* desc, int64_t sinks, void* workspace, uint64_t workspace_bytes, void* stream) {
    return Attention(desc, sinks, workspace, workspace_bytes, true, stream);
}

static const char* HistoryFault(const nuka_b200_history_t& d) {
    if (d.envs < 0 || d.envs > kMostTokens || d.capacity < 1 || d.capacity > (1 << 30)) return "envs must not be negative, capacity 1 to 2^30";
    if (d.heads_k < 1 || d.heads_q < 1 || d.heads_q > 65536 || d.heads_q % d.heads_k != 0) return "heads_q must be a positive multiple of heads_k, at most 65536";
    return nullptr;
}

uint64_t nuka_b200_history_workspace(const nuka_b200_history_t* desc) {
    return desc == nullptr || HistoryFault(*desc) != nullptr || desc->envs == 0 ? 0u : nkb::history_workspace(*desc);
}

static nuka_result_t History(const nuka_b200_history_t* desc, int64_t sinks, void* stream) {
    if (desc == nullptr) return Invalid("history desc is null");
    const nuka_b200_history_t& d = *desc;
    if (d.dtype != NUKA_B200_F16 && d.dtype != NUKA_B200_BF16) return Refuse(NUKA_RESULT_NOT_SUPPORTED, "dtype must be F16 or BF16");
    if (const char* fault = HistoryFault(d)) return Invalid(fault);
    if (d.dim < 8 || d.dim > 128 || d.dim % 8 != 0) return Refuse(NUKA_RESULT_NOT_SUPPORTED, "dim must be a multiple of 8, 8 to 128");
    if (!(d.scale > 0.f) || d.scale > 3.0e38f) return Invalid("scale must be greater than 0 and finite");
    if (sinks < 0 || sinks >= d.capacity) return Invalid("sinks must not be negative, and fewer than the capacity");
    if (d.envs == 0) return NUKA_RESULT_OK;
    if (d.envs * d.heads_q > (1ll << 31) - 1024) return Refuse(NUKA_RESULT_NOT_SUPPORTED, "too many envs times heads");
    for (const void* p : {d.q, d.k, d.v, static_cast<const void*>(d.keys), static_cast<const void*>(d.values), static_cast<const void*>(d.out)}) {
        if (p == nullptr) return Invalid("q, k, v, keys, values or out is null");
        if (!Aligned(p, 16)) return Invalid("a tensor does not lie on 16 bytes");
    }
    if (d.position == nullptr || !Aligned(d.position, 4)) return Invalid("position is null or not on 4 bytes");
    for (int64_t s : {d.q_stride, d.q_head_stride, d.k_stride, d.k_head_stride, d.v_stride, d.v_head_stride})
        if (s < 0 || s % 8 != 0) return Invalid("strides must be multiples of 8 values, not negative");
    const uint64_t need = nkb::history_workspace(d);
    if (need != 0u && (d.workspace == nullptr || d.workspace_bytes < need || !Aligned(d.workspace, 16))) return Invalid("the workspace is null, too small or not on 16 bytes");
    return Ran(nkb::launch_history(d, sinks, StreamOf(stream)));
}

nuka_result_t nuka_b200_history(const nuka_b200_history_t* desc, void* stream) { return History(desc, 0, stream); }
nuka_result_t nuka_b200_history_sinks(const nuka_b200_history_t* desc, int64_t sinks, void* stream) { return History(desc, sinks, stream); }

nuka_result_t nuka_b200_history_advance(int32_t* position, const uint8_t* fresh, int64_t envs, void* stream) {
    if (envs < 0 || envs > kMostTokens) return Invalid("envs are negative or too many");
    if (envs != 0 && (position == nullptr || !Aligned(position, 4))) return Invalid("position is null or not on 4 bytes");
    return Ran(nkb::launch_history_advance(position, fresh, envs, StreamOf(stream)));
}

}  // extern "C"
