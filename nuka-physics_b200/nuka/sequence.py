"""Sequence operators of a policy with memory: what a policy over the episodes of a rollout needs next to ``nuka.vec_env``.

A token is one control step of one env.  Tokens lie one behind the other in rows (an env's part of a rollout, or a whole episode);
``Episodes`` says where each token's episode begins and ends, and all operators over rollouts read it.  Each has a form for one token of
every env, for acting:

    over a rollout (training)                      one token of every env (acting)
    gated_recurrence(x, gate, episodes, initial)   gated_recurrence_step(x, gate, state, fresh)
    short_convolution(x, weight, bias, episodes)   short_convolution_step(x, weight, bias, state, fresh)
    selective_scan(x, delta, ..., episodes)        selective_scan_step(x, delta, ..., state, fresh)
    rotate_heads(q, k, ..., episodes, ...)         rotate_heads(q, k, ..., positions, ...)
    episode_attention(q, k, v, episodes)           history_attention(q, k, v, cache)

Tensors live on one GPU; the work is enqueued on torch's current stream of that GPU and nothing waits for it.  Operators over
rollouts take part in automatic differentiation (once).  Needs torch with CUDA.
"""
import ctypes

import torch
from torch.autograd import forward_ad

from . import _abi, _check

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


# Acting is one small call after the other: what is checked on every call is written to cost little, messages are put together only when they are raised.
def _expect(ok, text):
    if not ok:
        raise ValueError(text)


def _on_gpu(first, *others):
    """The GPU that all of the tensors are on (None is left out)."""
    index = first.get_device()
    if not first.is_cuda:
        raise ValueError("tensors must be on the GPU")
    for tensor in others:
        if tensor is not None and tensor.get_device() != index:
            raise ValueError("tensors must be on one GPU")
    return first.device


def _dtype(tensor, allowed, what):
    if tensor.dtype not in allowed:
        names = ", ".join(str(d).replace("torch.", "") for d in allowed)
        raise ValueError(f"{what} must be one of {names}, not {str(tensor.dtype).replace('torch.', '')}")
    return _DTYPES[tensor.dtype]


# what torch.cuda.current_stream(index).cuda_stream and torch.cuda.current_device() give, without the objects on the way
_raw_stream, _current_device = getattr(torch._C, "_cuda_getCurrentRawStream", None), getattr(torch._C, "_cuda_getDevice", None)
if _raw_stream is None or _current_device is None:
    _raw_stream, _current_device = (lambda index: torch.cuda.current_stream(index).cuda_stream), torch.cuda.current_device


def _call(device, function, *args):
    """One call of the library on torch's current stream of `device`, which it returns."""
    index = device.index
    stream = _raw_stream(index)
    if _current_device() != index:
        with torch.cuda.device(device):
            code = function(*args, stream)
    else:
        code = function(*args, stream)
    if code:
        _check(code)
    return stream


# A kernel has written the tensor: told to autograd, which refuses a gradient that would read what it was.
_written = torch.autograd.graph.increment_version


def _ptr(tensor):
    return None if tensor is None else tensor.data_ptr()


def _flags(tensor, shape, device, what):
    if not (tensor.dtype in (torch.bool, torch.uint8) and tensor.shape == shape and tensor.device == device):
        raise ValueError(f"{what} must be {tuple(shape)} bool or uint8 on {device}")
    return tensor.contiguous()


def _empty(like):
    return torch.empty_like(like, memory_format=torch.contiguous_format)


def _stride(tensor, dim):
    return tensor.stride(dim) if tensor.shape[dim] > 1 else 0


def _channels_last(tensor, multiple=1, size=1, least=0):
    """The tensor as it is where its last dimension is contiguous, its other strides are multiples of `multiple` values and at least `least`, and it lies on
    `size` bytes, else a copy."""
    strides, shape = tensor.stride(), tensor.shape
    if (strides[-1] == 1 or shape[-1] == 1) and (size == 1 or tensor.data_ptr() % size == 0):
        for s, n in zip(strides[:-1], shape):
            if n > 1 and (s % multiple or s < least):
                break
        else:
            return tensor
    return tensor.clone(memory_format=torch.contiguous_format)


def _rows(tensor):
    """The tensor as it is where its last dimension is contiguous, else a copy."""
    return tensor if tensor.stride(-1) == 1 else _channels_last(tensor)


def _point(desc, names, tensors, strides=None, size=1):
    """Sets the descriptor's addresses to those that the tensors have. What a backward pass finds saved may lie elsewhere than in the forward call, and otherwise (offloaded, worked
    out again): False where a stride is not what it was or an address is not on `size` bytes."""
    fits = True
    for i, (name, x) in enumerate(zip(names, tensors)):
        at = x.data_ptr()
        setattr(desc, name, at)
        if strides is not None and (x.stride() != strides[i] or at % size):
            fits = False
    return fits


class Episodes:
    """How a rollout's tokens are cut into rows and episodes, on the GPU.  Made once per rollout, for all layers and passes over it."""

    def __init__(self, tokens, rows, length, device):
        self.tokens, self.rows, self.device = int(tokens), int(rows), torch.device(device)
        self._rows_may_be_empty, self._stream = length == 0, None
        self._plan = torch.empty((4, self.tokens), dtype=torch.int32, device=device)
        base, step = self._plan.data_ptr(), 4 * self.tokens
        self._desc = _abi.EpisodesDesc(base, base + step, base + 2 * step, base + 3 * step, self.tokens, self.rows, length)
        self._ref = ctypes.pointer(self._desc)

    @classmethod
    def from_offsets(cls, offsets, tokens):
        """Rows are whole episodes: row r holds the tokens offsets[r] to offsets[r + 1].  `offsets`: int32 on the GPU, rows + 1 of them, ascending from 0
        to `tokens` (they are not read back to be checked)."""
        _expect(offsets.dim() == 1 and offsets.numel() >= 1 and offsets.dtype == torch.int32, "offsets must be a vector of int32")
        _expect(tokens >= 0, "tokens must not be negative")
        device = _on_gpu(offsets)
        offsets = offsets.contiguous()
        plan = cls(tokens, offsets.numel() - 1, 0, device)
        plan._stream = _call(device, _abi.lib().nuka_b200_episodes_from_offsets, plan._ref, offsets.data_ptr())
        return plan

    @classmethod
    def from_done(cls, done):
        """A rollout of N envs over T control steps, its tokens env after env: `done` (N x T, bool or uint8, on the GPU) is set where an
        episode ended with that token, as ``NukaVecEnv.step`` reports it."""
        _expect(done.dim() == 2, "done must be envs x steps")
        device = _on_gpu(done)
        done = _flags(done, done.shape, device, "done")
        plan = cls(done.numel(), done.shape[0], done.shape[1], device)
        plan._stream = _call(device, _abi.lib().nuka_b200_episodes_from_done, plan._ref, done.data_ptr())
        return plan

    def _read_on(self, stream):
        """A call on `stream` reads the plan: its memory is kept from other use until that call has ended, wherever the plan was made."""
        if stream != self._stream:
            self._plan.record_stream(torch.cuda.current_stream(self.device))

    @property
    def first(self):
        """Index of the first token of each token's episode."""
        return self._plan[0]

    @property
    def end(self):
        """Index behind the last token of each token's episode."""
        return self._plan[1]

    @property
    def positions(self):
        """Each token's number in its episode, from 0."""
        return torch.arange(self.tokens, dtype=torch.int32, device=self.device) - self._plan[0]


def _tokens_of(tensor, episodes, dims, what):
    if tensor.dim() != dims or tensor.shape[0] != episodes.tokens:
        raise ValueError(f"{what} must have {dims} dimensions, the first of {episodes.tokens} tokens")


# ---- the gated linear recurrence -----------------------------------------------------------------------------------
def _recur(x, gate, initial, episodes):
    device, dtype, channels = x.device, _DTYPES[x.dtype], x.shape[1]
    h = torch.empty(x.shape, dtype=x.dtype, device=device)
    if not episodes._rows_may_be_empty:
        state = torch.empty((episodes.rows, channels), dtype=torch.float32, device=device)
    elif initial is None:
        state = torch.zeros((episodes.rows, channels), dtype=torch.float32, device=device)
    else:
        state = initial.clone()
    lib = _abi.lib()
    need = lib.nuka_b200_recurrence_workspace(episodes._ref, channels)
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    desc = _abi.RecurrenceDesc(episodes._ref, dtype, channels, x.data_ptr(), gate.data_ptr(), _stride(x, 0), _stride(gate, 0), _ptr(initial), h.data_ptr(), state.data_ptr(),
                               None, None, None, None, None, _ptr(workspace), need)
    episodes._read_on(_call(device, lib.nuka_b200_recurrence, ctypes.byref(desc)))
    return h, state


def _differentiated(*tensors):
    """Whether the call goes through its autograd function: where a gradient may be asked for, and in forward mode, which that function refuses (a tangent would be lost otherwise)."""
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for x in tensors:
            if x is not None and x.requires_grad:
                return True
    return False


def _once(backward):
    """Gradients that cannot be differentiated again, at no cost where nobody asks for it."""
    guarded = torch.autograd.function.once_differentiable(backward)
    return staticmethod(lambda ctx, *grads: (guarded if torch.is_grad_enabled() else backward)(ctx, *grads))


class _Recurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, initial, episodes):
        h, state = _recur(x, gate, initial, episodes)
        ctx.episodes, ctx.has_initial = episodes, initial is not None
        ctx.save_for_backward(x, gate, h, *([initial] if initial is not None else []))
        ctx.set_materialize_grads(False)
        return h, state

    @_once
    def backward(ctx, dh, dstate):
        x, gate, h, *initial = ctx.saved_tensors
        # what is saved may come back elsewhere and with other strides (offloaded, worked out again)
        x, gate, h, initial, episodes = _channels_last(x), _channels_last(gate), h.contiguous(), initial[0].contiguous() if initial else None, ctx.episodes
        device, dtype, channels = x.device, _DTYPES[x.dtype], x.shape[1]
        dh = torch.zeros_like(h) if dh is None else dh.contiguous()
        dstate = None if dstate is None else dstate.contiguous()
        dx, dgate = _empty(x), _empty(x)
        dinitial = None
        if ctx.has_initial and ctx.needs_input_grad[2]:
            if not episodes._rows_may_be_empty:
                dinitial = torch.empty_like(initial)
            else:                                   # an empty row ends with the state that it began with
                dinitial = torch.zeros_like(initial) if dstate is None else dstate.clone()
        lib = _abi.lib()
        need = lib.nuka_b200_recurrence_workspace(episodes._ref, channels)
        workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        desc = _abi.RecurrenceDesc(episodes._ref, dtype, channels, x.data_ptr(), gate.data_ptr(), _stride(x, 0), _stride(gate, 0), _ptr(initial), h.data_ptr(), None,
                                   dh.data_ptr(), _ptr(dstate), dx.data_ptr(), dgate.data_ptr(), _ptr(dinitial), _ptr(workspace), need)
        episodes._read_on(_call(device, lib.nuka_b200_recurrence_backward, ctypes.byref(desc)))
        return dx, dgate, dinitial, None


def gated_recurrence(x, gate, episodes, initial=None):
    """h_t = a_t h_{t-1} + (1 - a_t) x_t with a_t = sigmoid(gate_t), channel by channel over each episode.

    x, gate: tokens x channels, f32, f16 or bf16.  initial: rows x channels f32, the state that each row begins with (the one its env had
    when the rollout began), None for 0; an episode that begins inside a row begins with 0.  Returns (h, state): h like x, state (rows x channels f32) the
    state that each row ends with, not rounded.  States and sums are in 32 bits; the gate's gradient is formed from the returned h, so where a 16-bit h is close to x it is off by
    half a unit of h times its factor."""
    device = _on_gpu(x, gate, initial, episodes._plan)
    _dtype(x, _DTYPES, "x")
    _tokens_of(x, episodes, 2, "x")
    _expect(gate.shape == x.shape and gate.dtype == x.dtype, "gate must be like x")
    if initial is not None:
        if initial.shape != (episodes.rows, x.shape[1]) or initial.dtype != torch.float32:
            raise ValueError(f"initial must be {episodes.rows} x {x.shape[1]} float32 on {device}")
        initial = initial.contiguous()
    train = _differentiated(x, gate, initial)
    x, gate = _channels_last(x), _channels_last(gate)
    return _Recurrence.apply(x, gate, initial, episodes) if train else _recur(x, gate, initial, episodes)


def gated_recurrence_step(x, gate, state, fresh=None):
    """The recurrence for one token of each env.  x, gate: envs x channels; state: envs x channels f32, contiguous, updated in place; fresh: envs, bool or
    uint8, set where the token begins an episode (the state before it counts as 0).  Returns h, the new state in x's type.  No gradient."""
    device = _on_gpu(x, gate, state, fresh)
    dtype = _dtype(x, _DTYPES, "x")
    _expect(x.dim() == 2 and gate.shape == x.shape and gate.dtype == x.dtype, "x and gate must be envs x channels, of one type")
    _expect(state.shape == x.shape and state.dtype == torch.float32 and state.is_contiguous(), "state must be contiguous float32, envs x channels")
    x, gate = _channels_last(x), _channels_last(gate)
    if fresh is not None:
        fresh = _flags(fresh, x.shape[:1], device, "fresh")
    h = torch.empty(x.shape, dtype=x.dtype, device=device)
    _call(device, _abi.lib().nuka_b200_recurrence_step, dtype, x.shape[0], x.shape[1], x.data_ptr(), _stride(x, 0), gate.data_ptr(), _stride(gate, 0), _ptr(fresh), state.data_ptr(), h.data_ptr())
    _written(state)
    return h


# ---- the short causal convolution -----------------------------------------------------------------------------------
def _final_state(episodes, initial, shape, dtype, device):
    """Where the state that each row ends with goes: an empty row ends with what it began with."""
    if not episodes._rows_may_be_empty:
        return torch.empty(shape, dtype=dtype, device=device)
    return torch.zeros(shape, dtype=dtype, device=device) if initial is None else initial.clone(memory_format=torch.contiguous_format)


def _workspace(need, device):
    return torch.empty(need, dtype=torch.uint8, device=device) if need else None


def _convolve(x, weight, bias, initial, episodes, silu):
    device, channels = x.device, x.shape[1]
    y, state = torch.empty(x.shape, dtype=x.dtype, device=device), _final_state(episodes, initial, (episodes.rows, weight.shape[1] - 1, channels), x.dtype, device)
    desc = _abi.ConvolutionDesc(episodes._ref, _DTYPES[x.dtype], silu, channels, weight.shape[1], x.data_ptr(), _stride(x, 0), weight.data_ptr(), _ptr(bias), _ptr(initial), y.data_ptr(), state.data_ptr())
    episodes._read_on(_call(device, _abi.lib().nuka_b200_convolution, ctypes.byref(desc)))
    return y, state


class _Convolution(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, initial, episodes, silu):
        ctx.episodes, ctx.silu, ctx.given = episodes, silu, (bias is not None, initial is not None)
        ctx.save_for_backward(x, weight, *(v for v in (bias, initial) if v is not None))
        ctx.set_materialize_grads(False)
        return _convolve(x, weight, bias, initial, episodes, silu)

    @_once
    def backward(ctx, dy, dstate):
        x, weight, *rest = ctx.saved_tensors
        # what is saved may come back elsewhere and with other strides (offloaded, worked out again)
        x, weight, rest = _channels_last(x), weight.contiguous(), [v.contiguous() for v in rest]
        bias, initial = rest[0] if ctx.given[0] else None, rest[-1] if ctx.given[1] else None
        episodes, device, channels, width = ctx.episodes, x.device, x.shape[1], weight.shape[1]
        dy = torch.zeros(x.shape, dtype=x.dtype, device=device) if dy is None else dy.contiguous()
        dstate = None if dstate is None else dstate.contiguous()
        dx, dinitial = _empty(x), None
        if initial is not None and ctx.needs_input_grad[3]:
            dinitial = _final_state(episodes, dstate, initial.shape, x.dtype, device)
        dweight = _empty(weight) if ctx.needs_input_grad[1] else None
        dbias = _empty(bias) if bias is not None and ctx.needs_input_grad[2] else None
        lib = _abi.lib()
        need = lib.nuka_b200_convolution_workspace(episodes._ref, channels, width) if dweight is not None or dbias is not None else 0
        workspace = _workspace(need, device)
        desc = _abi.ConvolutionDesc(episodes._ref, _DTYPES[x.dtype], ctx.silu, channels, width, x.data_ptr(), _stride(x, 0), weight.data_ptr(), _ptr(bias), _ptr(initial), None, None,
                                    dy.data_ptr(), _ptr(dstate), dx.data_ptr(), _ptr(dinitial), _ptr(dweight), _ptr(dbias), _ptr(workspace), need)
        episodes._read_on(_call(device, lib.nuka_b200_convolution_backward, ctypes.byref(desc)))
        return dx, dweight, dbias, dinitial, None, None


def _convolution_weights(weight, bias, channels):
    if weight.dim() != 2 or weight.dtype is not torch.float32 or weight.shape[0] != channels or not 2 <= weight.shape[1] <= 4:
        raise ValueError(f"weight must be float32, {channels} channels x 2, 3 or 4 taps")
    if bias is not None and (bias.shape != (channels,) or bias.dtype != torch.float32):
        raise ValueError(f"bias must be float32, {channels} channels")
    return weight.contiguous(), None if bias is None else bias.contiguous()


def short_convolution(x, weight, bias, episodes, initial=None, silu=False):
    """y_t = bias + sum over j of weight[:, j] x_{t - width + 1 + j}, channel by channel over each episode, with `silu` times its own logistic function.

    x: tokens x channels, f32, f16 or bf16.  weight: channels x width float32, width 2 to 4, the present token's last.  bias: channels float32, or None.  Inputs before an episode are 0.
    initial: rows x (width - 1) x channels in x's type, what came before each row (the state of its env when the rollout began), None for 0.  Returns (y, state): y like x,
    state like initial, the last inputs of each row's last episode. Sums are in 32 bits."""
    device = _on_gpu(x, weight, bias, initial, episodes._plan)
    _dtype(x, _DTYPES, "x")
    _tokens_of(x, episodes, 2, "x")
    weight, bias = _convolution_weights(weight, bias, x.shape[1])
    if initial is not None:
        shape = (episodes.rows, weight.shape[1] - 1, x.shape[1])
        if initial.shape != shape or initial.dtype != x.dtype:
            raise ValueError(f"initial must be {' x '.join(map(str, shape))} of x's type on {device}")
        initial = initial.contiguous()
    train = _differentiated(x, weight, bias, initial)
    x = _channels_last(x)
    return _Convolution.apply(x, weight, bias, initial, episodes, bool(silu)) if train else _convolve(x, weight, bias, initial, episodes, bool(silu))


def short_convolution_step(x, weight, bias, state, fresh=None, silu=False):
    """The convolution for one token of each env.  x: envs x channels; state: envs x (width - 1) x channels of x's type, contiguous, updated in place; fresh: envs, bool or
    uint8, set where the token begins an episode (the inputs before it count as 0).  Returns y like x.  No gradient."""
    device = _on_gpu(x, weight, bias, state, fresh)
    dtype = _dtype(x, _DTYPES, "x")
    _expect(x.dim() == 2, "x must be envs x channels")
    envs, channels = x.shape
    weight, bias = _convolution_weights(weight, bias, channels)
    width = weight.shape[1]
    if state.shape != (envs, width - 1, channels) or state.dtype != x.dtype or not state.is_contiguous():
        raise ValueError(f"state must be contiguous, {envs} x {width - 1} x {channels} of x's type")
    x = _rows(x)
    if fresh is not None:
        fresh = _flags(fresh, x.shape[:1], device, "fresh")
    y = torch.empty((envs, channels), dtype=x.dtype, device=device)
    desc = _abi.ConvolutionStepDesc(dtype, bool(silu), envs, channels, width, x.data_ptr(), x.stride(0) if envs > 1 else 0, weight.data_ptr(), _ptr(bias), _ptr(fresh), state.data_ptr(), y.data_ptr())
    _call(device, _abi.lib().nuka_b200_convolution_step, ctypes.byref(desc))
    _written(state)
    return y


# ---- the selective scan ----------------------------------------------------------------------------------------------
_SCANNED = ("x", "delta", "gate", "b", "c")              # what has a stride of its own


def _scan(tensors, episodes, train):
    """`tensors`: by the descriptor's names, None where not given.  (y, state, what a backward pass needs beside the inputs)."""
    x, decay, initial = tensors["x"], tensors["decay"], tensors["initial"]
    device, (channels, states) = x.device, decay.shape
    y, state = torch.empty(x.shape, dtype=x.dtype, device=device), _final_state(episodes, initial, (episodes.rows, channels, states), torch.float32, device)
    lib = _abi.lib()
    kept = torch.empty(lib.nuka_b200_scan_kept(episodes._ref, channels, states), dtype=torch.uint8, device=device) if train else None
    need = lib.nuka_b200_scan_workspace(episodes._ref, channels, states, 0)
    workspace = _workspace(need, device)
    desc = _scan_desc(tensors, episodes)
    desc.y, desc.state, desc.workspace, desc.workspace_bytes = y.data_ptr(), state.data_ptr(), _ptr(workspace), need
    if train:
        desc.kept, desc.kept_bytes = _ptr(kept), kept.numel()
    episodes._read_on(_call(device, lib.nuka_b200_scan, ctypes.byref(desc)))
    return y, state, kept


def _scan_desc(t, episodes):
    channels, states = t["decay"].shape
    return _abi.ScanDesc(episodes._ref, _DTYPES[t["x"].dtype], channels, states, *(_ptr(t[name]) for name in _SCANNED), *(0 if t[name] is None else _stride(t[name], 0) for name in _SCANNED),
                         t["decay"].data_ptr(), _ptr(t["skip"]), _ptr(t["delta_bias"]), _ptr(t["initial"]))


_SCAN_INPUTS = ("x", "delta", "decay", "b", "c", "initial", "skip", "gate", "delta_bias")


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, episodes, *inputs):
        y, state, kept = _scan(dict(zip(_SCAN_INPUTS, inputs)), episodes, True)
        ctx.episodes, ctx.names = episodes, [name for name, x in zip(_SCAN_INPUTS, inputs) if x is not None]
        ctx.save_for_backward(*(x for x in inputs if x is not None), kept)
        ctx.set_materialize_grads(False)
        return y, state

    @_once
    def backward(ctx, dy, dstate):
        *saved, kept = ctx.saved_tensors
        # what is saved may come back elsewhere and with other strides (offloaded, worked out again)
        t = {name: _channels_last(x) if name in _SCANNED else x.contiguous() for name, x in zip(ctx.names, saved)}
        t = {name: t.get(name) for name in _SCAN_INPUTS}
        kept = _channels_last(kept.contiguous(), 1, 16)
        x, episodes = t["x"], ctx.episodes
        device, (channels, states) = x.device, t["decay"].shape
        dy = torch.zeros(x.shape, dtype=x.dtype, device=device) if dy is None else dy.contiguous()
        dstate = None if dstate is None else dstate.contiguous()
        wanted = dict(zip(_SCAN_INPUTS, ctx.needs_input_grad[1:]))
        grads = {name: _empty(v) for name, v in t.items() if v is not None and (name in _SCANNED or wanted[name])}
        if "initial" in grads:
            grads["initial"] = _final_state(episodes, dstate, t["initial"].shape, torch.float32, device)
        lib = _abi.lib()
        need = lib.nuka_b200_scan_workspace(episodes._ref, channels, states, 1)
        workspace = _workspace(need, device)
        desc = _scan_desc(t, episodes)
        desc.kept, desc.kept_bytes, desc.dy, desc.dstate, desc.workspace, desc.workspace_bytes = _ptr(kept), kept.numel(), dy.data_ptr(), _ptr(dstate), _ptr(workspace), need
        for name, v in grads.items():
            setattr(desc, "d" + name, v.data_ptr())
        episodes._read_on(_call(device, lib.nuka_b200_scan_backward, ctypes.byref(desc)))
        return (None, *(grads.get(name) for name in _SCAN_INPUTS))


def _scan_inputs(x, delta, decay, b, c, skip, gate, delta_bias, strides=None):
    """Checks what the scan and its step have in common; the inputs as the kernels take them. `strides`: those of x, delta, b and c where the caller has them, made those of what is returned."""
    dtype, shape = x.dtype, x.shape
    if dtype not in _DTYPES:
        _dtype(x, _DTYPES, "x")
    if len(shape) != 2 or decay.dim() != 2 or decay.dtype != torch.float32:
        raise ValueError("x must have 2 dimensions, the second of channels, and decay must be float32, channels x 1 to 64 states")
    (count, channels), (rows, states) = shape, decay.shape
    if rows != channels or not 1 <= states <= 64:
        raise ValueError("x must have 2 dimensions, the second of channels, and decay must be float32, channels x 1 to 64 states")
    narrow = (count, states)
    if not (delta.shape == shape and delta.dtype is dtype and b.shape == narrow and b.dtype is dtype and c.shape == narrow and c.dtype is dtype and (gate is None or (gate.shape == shape and gate.dtype is dtype))):
        raise ValueError(f"delta and gate must be like x, b and c {count} x {states}, of x's type")
    for v in (skip, delta_bias):
        if v is not None and (v.dtype is not torch.float32 or v.shape != (channels,)):
            raise ValueError("skip and delta_bias must be float32, one per channel")
    # kept as they are where their last dimension is contiguous
    if strides is None or not strides[0][-1] == strides[1][-1] == strides[2][-1] == strides[3][-1] == 1:
        x, delta, b, c = _rows(x), _rows(delta), _rows(b), _rows(c)
        if strides is not None:
            strides[:] = x.stride(), delta.stride(), b.stride(), c.stride()
    return (x, delta, decay.contiguous(), b, c, None if skip is None else skip.contiguous(), None if gate is None else _rows(gate), None if delta_bias is None else delta_bias.contiguous())


def selective_scan(x, delta, decay, b, c, episodes, initial=None, skip=None, gate=None, delta_bias=None):
    """h_t = exp(dt decay) h_{t-1} + dt x_t b_t with dt = softplus(delta_t + delta_bias), a state of channels x states; y_t = h_t c_t + skip x_t, with `gate` times gate_t / (1 + exp(-gate_t)).

    x, delta, gate: tokens x channels, f32, f16 or bf16.  b, c: tokens x states, of x's type; all at any stride (views of projections).  decay: channels x states float32, 1 to 64 states, below 0 where
    a state fades.  skip, delta_bias: channels float32, or None.  initial: rows x channels x states float32, the state that each row begins with, None for 0; an episode that begins inside a row
    begins with 0.  Returns (y, state): y like x, state like initial, what each row ends with.  Rates, states and sums are in 32 bits; exp(dt decay) is off by up to 2^-22 (1 + |dt decay|) of itself, as its argument is rounded
    to 32 bits, and 0 below 2^-126. Where a gradient may
    be asked for, the states before each fourth or eighth token are kept (at 16 states 8 bytes for each value of x, up to twice that where rows are short)."""
    device = _on_gpu(x, delta, decay, b, c, initial, skip, gate, delta_bias, episodes._plan)
    _tokens_of(x, episodes, 2, "x")
    x, delta, decay, b, c, skip, gate, delta_bias = _scan_inputs(x, delta, decay, b, c, skip, gate, delta_bias)
    if initial is not None:
        if initial.shape != (episodes.rows, *decay.shape) or initial.dtype != torch.float32:
            raise ValueError(f"initial must be {episodes.rows} x {decay.shape[0]} x {decay.shape[1]} float32 on {device}")
        initial = initial.contiguous()
    inputs = (x, delta, decay, b, c, initial, skip, gate, delta_bias)
    return _Scan.apply(episodes, *inputs) if _differentiated(*inputs) else _scan(dict(zip(_SCAN_INPUTS, inputs)), episodes, False)[:2]


def selective_scan_step(x, delta, decay, b, c, state, fresh=None, skip=None, gate=None, delta_bias=None):
    """The scan for one token of each env.  x, delta, gate: envs x channels; b, c: envs x states; state: envs x channels x states float32, contiguous, updated in place; fresh: envs, bool or
    uint8, set where the token begins an episode (the state before it counts as 0).  Returns y like x.  No gradient."""
    device = _on_gpu(x, delta, decay, b, c, state, fresh, skip, gate, delta_bias)
    strides = [x.stride(), delta.stride(), b.stride(), c.stride()]
    x, delta, decay, b, c, skip, gate, delta_bias = _scan_inputs(x, delta, decay, b, c, skip, gate, delta_bias, strides)
    (envs, channels), states = x.shape, decay.shape[1]
    if state.shape != (envs, channels, states) or state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError(f"state must be contiguous float32, {envs} x {channels} x {states}")
    if fresh is not None:
        fresh = _flags(fresh, x.shape[:1], device, "fresh")
    y = torch.empty((envs, channels), dtype=x.dtype, device=device)
    by = (strides[0][0], strides[1][0], 0 if gate is None else gate.stride(0), strides[2][0], strides[3][0]) if envs > 1 else (0, 0, 0, 0, 0)
    desc = _abi.ScanStepDesc(_DTYPES[x.dtype], envs, channels, states, x.data_ptr(), delta.data_ptr(), None if gate is None else gate.data_ptr(), b.data_ptr(), c.data_ptr(), *by, decay.data_ptr(),
                             None if skip is None else skip.data_ptr(), None if delta_bias is None else delta_bias.data_ptr(), None if fresh is None else fresh.data_ptr(), state.data_ptr(), y.data_ptr())
    _call(device, _abi.lib().nuka_b200_scan_step, ctypes.byref(desc))
    _written(state)
    return y


# ---- norms of queries and keys, and their rotation -----------------------------------------------------------------
def rotary_frequencies(turned, base=10000.0, trained=0, context=0, low=1.0, high=32.0):
    """Angle per position of each of the turned / 2 pairs (float64, on the CPU): base^(-2 i / turned).  With `trained` and a longer `context`, pairs that
    turn fewer than `low` times within the trained context are slowed down by context / trained, pairs that turn more than `high` times stay, those between are mixed
    (the frequency part of the YaRN paper, Peng et al. 2023)."""
    _expect(turned >= 0 and turned % 2 == 0, "turned must be even")
    f = float(base) ** (-torch.arange(0, turned, 2, dtype=torch.float64) / max(turned, 1))
    if trained and context > trained:
        keep = ((trained * f / (2 * torch.pi) - low) / (high - low)).clamp(0.0, 1.0)
        f = f * (keep + (1 - keep) * (trained / context))
    return f


def _turn(q, k, q_weight, k_weight, first, positions, frequencies, eps, pairs, episodes):
    device = q.device
    tokens, heads_q, dim = q.shape
    q_out, k_out = _empty(q), _empty(k)
    desc = _abi.HeadsDesc(_ptr(first), _ptr(positions), _ptr(frequencies), _DTYPES[q.dtype], pairs, tokens, heads_q, k.shape[1], dim,
                          0 if frequencies is None else 2 * frequencies.numel(), q.data_ptr(), k.data_ptr(), _stride(q, 0), _stride(q, 1), _stride(k, 0), _stride(k, 1),
                          _ptr(q_weight), _ptr(k_weight), eps, q_out.data_ptr(), k_out.data_ptr())
    stream = _call(device, _abi.lib().nuka_b200_heads, ctypes.byref(desc))
    if episodes is not None:
        episodes._read_on(stream)
    return q_out, k_out, desc


class _Heads(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, first, positions, frequencies, eps, pairs, episodes):
        q_out, k_out, desc = _turn(q, k, q_weight, k_weight, first, positions, frequencies, eps, pairs, episodes)
        tensors = {"q": q, "k": k, "q_weight": q_weight, "k_weight": k_weight, "first": first, "positions": positions, "frequencies": frequencies}
        ctx.names = [name for name, x in tensors.items() if x is not None]
        tensors = [tensors[name] for name in ctx.names]
        ctx.save_for_backward(*tensors)
        ctx.desc, ctx.strides, ctx.episodes = desc, [x.stride() for x in tensors], episodes
        ctx.set_materialize_grads(False)
        return q_out, k_out

    @_once
    def backward(ctx, dq_out, dk_out):
        tensors, desc = ctx.saved_tensors, _abi.HeadsDesc.from_buffer_copy(ctx.desc)
        size = 4 * tensors[0].element_size()
        if not _point(desc, ctx.names, tensors, ctx.strides, size):
            tensors = [_channels_last(x, 4, size) if i < 2 else _channels_last(x.contiguous(), 1, size) for i, x in enumerate(tensors)]
            _point(desc, ctx.names, tensors)
            desc.q_stride, desc.q_head_stride, desc.k_stride, desc.k_head_stride = (_stride(x, i) for x in tensors[:2] for i in (0, 1))
        q, k = tensors[:2]
        device = q.device
        dq_out, dk_out = (torch.zeros(x.shape, dtype=x.dtype, device=device) if d is None else _channels_last(d.contiguous(), 1, size) for x, d in ((q, dq_out), (k, dk_out)))
        dq, dk = _empty(q), _empty(k)
        dw = [_empty(tensors[ctx.names.index(name)]) if name in ctx.names and ctx.needs_input_grad[2 + i] else None for i, name in enumerate(("q_weight", "k_weight"))]
        lib = _abi.lib()
        need = lib.nuka_b200_heads_workspace(q.shape[0], q.shape[2]) if dw[0] is not None or dw[1] is not None else 0
        workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        desc.dq_out, desc.dk_out, desc.dq, desc.dk = dq_out.data_ptr(), dk_out.data_ptr(), dq.data_ptr(), dk.data_ptr()
        desc.dq_weight, desc.dk_weight, desc.workspace, desc.workspace_bytes = _ptr(dw[0]), _ptr(dw[1]), _ptr(workspace), need
        stream = _call(device, lib.nuka_b200_heads_backward, ctypes.byref(desc))
        if ctx.episodes is not None:
            ctx.episodes._read_on(stream)
        return dq, dk, dw[0], dw[1], None, None, None, None, None, None


def rotate_heads(q, k, q_weight, k_weight, positions, frequencies, eps=1e-6, interleaved=False, exact_angles=False):
    """Each head's queries and keys divided by their root mean square, times a weight per column, then turned by their position.

    q: tokens x heads x dim, k: tokens x key heads x dim, f32, f16 or bf16, heads and tokens at any stride (views of one projection).  q_weight, k_weight: dim f32, or None.
    positions: an ``Episodes`` (each token's number in its episode) or int32 per token.  frequencies: float64 on the GPU, one per turned pair, no gradient
    (``rotary_frequencies``; twice as many columns are turned, the others only normed), or None; the angle is their product in 32 bits, as programs
    have it that train in 32 bits, and off by up to about position x 2^-24 radians; with `exact_angles` it is taken in 64 bits.  Pairs are (i, i + turned / 2), or with `interleaved` (2 i, 2 i + 1).
    dim and the number of turned columns are multiples of 8, dim at most 256.  Returns (q, k), contiguous."""
    episodes = positions if isinstance(positions, Episodes) else None
    _on_gpu(q, k, q_weight, k_weight, frequencies, episodes._plan if episodes is not None else positions)
    _dtype(q, _DTYPES, "q")
    _expect(q.dim() == 3 and k.dim() == 3 and k.dtype == q.dtype and k.shape[0] == q.shape[0] and k.shape[2] == q.shape[2], "q and k must be tokens x heads x dim, of one type")
    for w in (q_weight, k_weight):
        _expect(w is None or (w.shape == q.shape[2:] and w.dtype == torch.float32), "weights must be float32, one per column of a head")
    _expect(frequencies is None or (frequencies.dim() == 1 and frequencies.dtype == torch.float64), "frequencies must be a vector of float64")
    if episodes is not None:
        _tokens_of(q, episodes, 3, "q")
        first, positions = episodes.first, None
    else:
        _expect(positions.dtype == torch.int32 and positions.shape == q.shape[:1], "positions must be an Episodes or int32, one per token")
        first, positions = None, positions.contiguous()
    q_weight, k_weight, frequencies = (None if x is None else x.contiguous() for x in (q_weight, k_weight, frequencies))
    size, pairs = 4 * q.element_size(), bool(interleaved) | (_abi.EXACT_ANGLES if exact_angles else 0)
    q, k = _channels_last(q, 4, size), _channels_last(k, 4, size)
    if not _differentiated(q, k, q_weight, k_weight):
        return _turn(q, k, q_weight, k_weight, first, positions, frequencies, float(eps), pairs, episodes)[:2]
    return _Heads.apply(q, k, q_weight, k_weight, first, positions, frequencies, float(eps), pairs, episodes)


# ---- attention over packed episodes --------------------------------------------------------------------------------
def _attend(q, k, v, episodes, scale, window, sinks, train):
    """(out, the statistics that a backward pass needs beside it, the call's descriptor)."""
    device = q.device
    out = torch.empty(q.shape, dtype=q.dtype, device=device)
    lib = _abi.lib()
    lse = torch.empty((q.shape[1], lib.nuka_b200_attention_pitch(episodes.tokens)), dtype=torch.float32, device=device) if train else None
    desc = _abi.AttentionDesc(episodes._ref, _DTYPES[q.dtype], q.shape[1], k.shape[1], q.shape[2], window, scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), _stride(q, 0), _stride(q, 1),
                              _stride(k, 0), _stride(k, 1), _stride(v, 0), _stride(v, 1), out.data_ptr(), _ptr(lse))
    if sinks:
        stream = _call(device, lib.nuka_b200_attention_sinks, ctypes.byref(desc), sinks)
    else:
        stream = _call(device, lib.nuka_b200_attention, ctypes.byref(desc))
    episodes._read_on(stream)
    return out, lse, desc


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, episodes, scale, window, sinks):
        out, lse, desc = _attend(q, k, v, episodes, scale, window, sinks, True)
        tensors = (q, k, v, out, lse)
        ctx.save_for_backward(*tensors)
        ctx.desc, ctx.strides, ctx.episodes, ctx.sinks = desc, [x.stride() for x in tensors], episodes, sinks
        return out

    @_once
    def backward(ctx, dout):
        tensors, desc, names = ctx.saved_tensors, _abi.AttentionDesc.from_buffer_copy(ctx.desc), ("q", "k", "v", "out", "lse")
        if not _point(desc, names, tensors, ctx.strides, 16):
            tensors = [_channels_last(x, 8, 16, x.shape[2]) if i < 3 else _channels_last(x.contiguous(), 1, 16) for i, x in enumerate(tensors)]
            _point(desc, names, tensors)
            desc.q_stride, desc.q_head_stride, desc.k_stride, desc.k_head_stride, desc.v_stride, desc.v_head_stride = (_stride(x, i) for x in tensors[:3] for i in (0, 1))
        lse = tensors[4]
        device = lse.device
        dout = _channels_last(dout.contiguous(), 1, 16)
        dq, dk, dv = _empty(tensors[0]), _empty(tensors[1]), _empty(tensors[2])
        delta = _empty(lse)
        desc.dout, desc.delta, desc.dq, desc.dk, desc.dv = dout.data_ptr(), delta.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        if ctx.sinks:
            lib = _abi.lib()
            need = lib.nuka_b200_attention_sinks_workspace(ctypes.byref(desc), ctx.sinks)
            workspace = _workspace(need, device)
            stream = _call(device, lib.nuka_b200_attention_sinks_backward, ctypes.byref(desc), ctx.sinks, _ptr(workspace), need)
        else:
            stream = _call(device, _abi.lib().nuka_b200_attention_backward, ctypes.byref(desc))
        ctx.episodes._read_on(stream)
        return dq, dk, dv, None, None, None, None


def episode_attention(q, k, v, episodes, scale=None, window=None, sinks=0):
    """Causal attention over each episode: a token sees itself and the tokens of its episode before it, with `window` at most the last `window` of these, and beside them the
    episode's first `sinks` ones (which without a window are seen anyway).

    q: tokens x heads x dim, k and v: tokens x key heads x dim, f16 or bf16, tokens and heads at any stride (views of one projection); the heads are a multiple
    of the key heads, and as many heads share one key head.  dim: a multiple of 8, at most 128 (64 and 128 waste nothing).  scale: dim^-0.5 unless given.
    Returns tokens x heads x dim.  Sums and statistics are in 32 bits; probabilities and, backwards, their gradients are rounded to the inputs' type, so train in f16 with a
    loss scale. Gradients of a row whose probabilities' gradients leave f16's range are worked out in 32 bits, slowly."""
    _on_gpu(q, k, v, episodes._plan)
    _dtype(q, (torch.float16, torch.bfloat16), "q")
    for x, what in ((q, "q"), (k, "k"), (v, "v")):
        _tokens_of(x, episodes, 3, what)
    _expect(k.dtype == q.dtype and v.dtype == q.dtype and k.shape == v.shape and k.shape[2] == q.shape[2], "q, k and v must be of one type and dim, k and v of one shape")
    _expect(k.shape[1] > 0 and q.shape[1] % k.shape[1] == 0 and q.shape[1] > 0, "the heads must be a multiple of the key heads")
    _expect(q.shape[2] > 0, "heads must have columns")
    _expect(window is None or window >= 1, "window must be at least 1")
    _expect(sinks >= 0, "sinks must not be negative")
    scale, window, sinks = q.shape[2] ** -0.5 if scale is None else float(scale), 0 if window is None else int(window), 0 if window is None else int(sinks)
    train = _differentiated(q, k, v)
    q, k, v = (_channels_last(x, 8, 16, x.shape[2]) for x in (q, k, v))
    return _Attention.apply(q, k, v, episodes, scale, window, sinks) if train else _attend(q, k, v, episodes, scale, window, sinks, False)[0]


# ---- attention of one token over a cached history ------------------------------------------------------------------
class HistoryCache:
    """Keys and values of the last `capacity` tokens of each env, for one layer: a ring of envs x capacity x key heads x dim. With `sinks`, fewer than the capacity, its first
    places keep the first tokens of the env's episode, and the last `capacity` - `sinks` of the others are a ring behind them.

    ``position`` (envs, int32) is the number of each env's present token in its episode; ``advance(fresh)`` moves on to the next token of every env.  Layers of one
    policy share it: give one cache's ``position`` to the others and advance once per control step.  `buffers`: (keys, values, position) to use in place of new ones."""

    def __init__(self, envs, capacity, kv_heads, head_dim, dtype=torch.bfloat16, device="cuda", position=None, buffers=None, sinks=0):
        _expect(dtype in (torch.float16, torch.bfloat16), "dtype must be float16 or bfloat16")
        _expect(envs >= 0 and capacity >= 1 and kv_heads >= 1 and head_dim >= 8, "envs must not be negative, capacity and kv_heads at least 1, head_dim at least 8")
        _expect(0 <= sinks < capacity, "sinks must not be negative, and fewer than the capacity")
        self.sinks = int(sinks)
        shape = (int(envs), int(capacity), int(kv_heads), int(head_dim))
        if buffers is None:
            buffers = (torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                       torch.full(shape[:1], -1, dtype=torch.int32, device=device) if position is None else position)
        self.keys, self.values, self.position = buffers
        self.device = _on_gpu(*buffers)
        for x in buffers[:2]:
            _expect(tuple(x.shape) == shape and x.dtype == dtype and x.is_contiguous(), f"keys and values must be contiguous, {shape} {dtype}")
        _expect(tuple(self.position.shape) == shape[:1] and self.position.dtype == torch.int32 and self.position.is_contiguous(), "position must be contiguous int32, one per env")
        self._workspaces = {}                   # per number of heads

    def advance(self, fresh=None):
        """The next token of every env; envs with `fresh` set (envs, bool or uint8) begin an episode and forget what they held."""
        if fresh is not None:
            fresh = _flags(fresh, self.position.shape, self.device, "fresh")
        _call(self.device, _abi.lib().nuka_b200_history_advance, self.position.data_ptr(), _ptr(fresh), self.position.numel())

    def _workspace(self, heads):
        """[address, bytes, the tensor, its stream] of what a call with this many heads needs beside the cache, zeroed once.  One that is made while a graph is captured is that call's alone: its memory is the
        graph's, and each replay zeroes it."""
        found = self._workspaces.get(heads)
        if found is None:
            envs, capacity, heads_k, dim = self.keys.shape
            need = _abi.lib().nuka_b200_history_workspace(ctypes.byref(_abi.HistoryDesc(_DTYPES[self.keys.dtype], envs, capacity, heads, heads_k, dim)))
            kept = torch.zeros(need, dtype=torch.uint8, device=self.device)
            found = [kept.data_ptr() or None, need, kept, None]             # the stream: the first call's, which comes next
            if not torch.cuda.is_current_stream_capturing():
                self._workspaces[heads] = found
        return found


def history_attention(q, k, v, cache, scale=None):
    """Attention of one token of each env over what `cache` holds of its episode, the token itself among it: what ``episode_attention`` gives for the
    episode's last token, with the cache's capacity as the window (less its sinks, where it has some, and with them as sinks).  q: envs x heads x dim, k and v: envs x key heads x dim, in the cache's type, at any stride; k and v are
    written into the cache.  scale: dim^-0.5 unless given.  Returns envs x heads x dim.  Probabilities are rounded to the cache's type, sums are in 32 bits.  No gradient."""
    device = _on_gpu(q, k, v, cache.keys)
    envs, capacity, heads_k, dim = cache.keys.shape
    dtype = cache.keys.dtype
    if q.dim() != 3 or q.shape[0] != envs or q.shape[2] != dim or q.shape[1] == 0 or q.shape[1] % heads_k:
        raise ValueError(f"q must be {envs} x a multiple of {heads_k} x {dim}")
    if k.shape != (envs, heads_k, dim) or v.shape != k.shape:
        raise ValueError(f"k and v must be {envs} x {heads_k} x {dim}")
    if q.dtype != dtype or k.dtype != dtype or v.dtype != dtype:
        raise ValueError(f"q, k and v must be {dtype}, as the cache is")
    q, k, v = _channels_last(q, 8, 16), _channels_last(k, 8, 16), _channels_last(v, 8, 16)
    out = torch.empty(q.shape, dtype=dtype, device=device)
    workspace = cache._workspace(q.shape[1])
    desc = _abi.HistoryDesc(_DTYPES[dtype], envs, capacity, q.shape[1], heads_k, dim, dim ** -0.5 if scale is None else float(scale), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                            _stride(q, 0), _stride(q, 1), _stride(k, 0), _stride(k, 1), _stride(v, 0), _stride(v, 1), cache.keys.data_ptr(), cache.values.data_ptr(),
                            cache.position.data_ptr(), out.data_ptr(), *workspace[:2])
    if cache.sinks:
        stream = _call(device, _abi.lib().nuka_b200_history_sinks, ctypes.byref(desc), cache.sinks)
    else:
        stream = _call(device, _abi.lib().nuka_b200_history, ctypes.byref(desc))
    if workspace[3] is None:
        workspace[3] = stream
    elif workspace[1] and stream != workspace[3]:
        workspace[2].record_stream(torch.cuda.current_stream(device))
    return out
