"""Which memory the selective operators and attention with first tokens that stay touch, for plans that say what offsets ought to say and for plans made from offsets that lie: everything that a call is handed lies inside a
larger buffer.  What it writes leaves the buffers' margins as they were, bit for bit; what it reads around its inputs, and in workspaces before it has written them, is NaN, so results are finite only where nothing of that is read."""
import ctypes
import itertools

import pytest

torch = pytest.importorskip("torch")
import nuka  # noqa: E402,F401
from nuka import _abi  # noqa: E402

pytestmark = pytest.mark.gpu

PAD = 4096
NAME = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
TRUE = [[0, 13, 13, 40], [0, 40], list(range(41)), [0, 300, 301, 700], [0, 700]]
LIES = [[0, 50, 20, 10], [-5, 3, 1000, 7], [90, 95, 99, 2 ** 31 - 1], [0, 0, 0, 0], [-(2 ** 31), -1, -7, 12], [5, 4, 3, 2, 1], [650, 20, 2 ** 31 - 1, 3, 500]]


class Buffers:
    def __init__(self, seed):
        self.gen, self.all = torch.Generator(device="cuda").manual_seed(seed), []

    def _inside(self, shape, dtype, margin):
        size = 1
        for n in shape:
            size *= n
        buffer = torch.full((2 * PAD + size,), margin, dtype=dtype, device="cuda")
        return buffer, buffer[PAD:PAD + size].view(shape)

    def given(self, *shape, dtype=torch.float32, apart=0, make=None):
        """Values, `apart` NaNs between rows."""
        buffer, inside = self._inside((*shape[:-1], shape[-1] + apart), dtype, float("nan"))
        values = torch.empty(shape, device="cuda").normal_(generator=self.gen)
        inside[..., :shape[-1]] = (values if make is None else make(values)).to(dtype)
        self.all.append((buffer, buffer.clone(), None, None))
        return inside[..., :shape[-1]]

    def wanted(self, *shape, dtype=torch.float32, fill=0.0):
        buffer, inside = self._inside(shape, dtype, 3.0)
        inside.fill_(fill)
        self.all.append((buffer, buffer.clone(), inside, fill))
        return inside

    def bytes(self, count):
        """Memory to work in: NaN, whatever type it is read as."""
        buffer, inside = self._inside((int(count),), torch.uint8, 0xff)
        self.all.append((buffer, buffer.clone(), inside, None))
        return inside

    def check(self):
        torch.cuda.synchronize()
        for buffer, before, inside, fill in self.all:
            bits = lambda x: x.contiguous().view(torch.uint8)
            if inside is None:
                assert torch.equal(bits(buffer), bits(before))
                continue
            ends = [slice(None, PAD), slice(PAD + inside.numel(), None)]
            assert all(torch.equal(bits(buffer[e]), bits(before[e])) for e in ends)
            if fill is not None:
                assert torch.isfinite(inside).all()


def _at(tensor):
    return None if tensor is None else tensor.data_ptr()


def _plan(buffers, offsets, tokens):
    at = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    first, end, link, tail = (buffers.wanted(tokens, dtype=torch.int32, fill=-9) for _ in range(4))
    desc = _abi.EpisodesDesc(_at(first), _at(end), _at(link), _at(tail), tokens, len(offsets) - 1, 0)
    assert _abi.lib().nuka_b200_episodes_from_offsets(ctypes.byref(desc), at.data_ptr(), None) == 0
    t = torch.arange(tokens, device="cuda")
    assert ((first >= 0) & (first <= t) & (end > t) & (end <= tokens)).all()
    for rows in (link, tail):
        assert ((rows >= -1) & (rows < len(offsets) - 1)).all()
    return desc


def _cases():
    return [(offsets, tokens) for offsets, tokens in [*((o, o[-1]) for o in TRUE), *itertools.product(LIES, (40, 700))]]


@pytest.mark.parametrize("dtype", list(NAME))
@pytest.mark.parametrize("channels,states", [(8, 4), (70, 16), (37, 33)])
def test_the_scan(dtype, channels, states):
    lib = _abi.lib()
    for n, (offsets, tokens) in enumerate(_cases()):
        m = Buffers(n)
        plan, rows, apart = _plan(m, offsets, tokens), len(offsets) - 1, n % 2 * 3
        x, delta, gate = (m.given(tokens, channels, dtype=dtype, apart=apart) for _ in range(3))
        b, c = (m.given(tokens, states, dtype=dtype, apart=apart) for _ in range(2))
        decay, skip, bias = m.given(channels, states, make=lambda v: -v.abs()), m.given(channels), m.given(channels)
        first, dy, dstate = m.given(rows, channels, states), m.given(tokens, channels, dtype=dtype), m.given(rows, channels, states)
        kept = m.bytes(lib.nuka_b200_scan_kept(ctypes.byref(plan), channels, states))
        work = [m.bytes(lib.nuka_b200_scan_workspace(ctypes.byref(plan), channels, states, back)) for back in (0, 1)]
        y, state = m.wanted(tokens, channels, dtype=dtype), m.wanted(rows, channels, states)
        desc = _abi.ScanDesc(plan=ctypes.pointer(plan), dtype=NAME[dtype], channels=channels, states=states, x=_at(x), delta=_at(delta), gate=_at(gate), b=_at(b), c=_at(c), x_stride=x.stride(0), delta_stride=delta.stride(0),
                             gate_stride=gate.stride(0), b_stride=b.stride(0), c_stride=c.stride(0), decay=_at(decay), skip=_at(skip), delta_bias=_at(bias), initial=_at(first), y=_at(y), state=_at(state), kept=_at(kept),
                             kept_bytes=kept.numel(), workspace=_at(work[0]), workspace_bytes=work[0].numel())
        assert lib.nuka_b200_scan(ctypes.byref(desc), None) == 0
        m.check()
        grads = {name: m.wanted(tokens, channels, dtype=dtype) for name in ("dx", "ddelta", "dgate")}
        grads.update(db=m.wanted(tokens, states, dtype=dtype), dc=m.wanted(tokens, states, dtype=dtype), ddecay=m.wanted(channels, states), dskip=m.wanted(channels), ddelta_bias=m.wanted(channels),
                     dinitial=m.wanted(rows, channels, states))
        for name, v in {**grads, "dy": dy, "dstate": dstate, "workspace": work[1]}.items():
            setattr(desc, name, _at(v))
        desc.workspace_bytes = work[1].numel()
        assert lib.nuka_b200_scan_backward(ctypes.byref(desc), None) == 0
        m.check()
    envs = 37
    m = Buffers(99)
    x, delta, gate = (m.given(envs, channels, dtype=dtype, apart=5) for _ in range(3))
    b, c = (m.given(envs, states, dtype=dtype, apart=1) for _ in range(2))
    decay, skip, bias = m.given(channels, states, make=lambda v: -v.abs()), m.given(channels), m.given(channels)
    state, y = m.wanted(envs, channels, states, fill=1.0), m.wanted(envs, channels, dtype=dtype)
    step = _abi.ScanStepDesc(dtype=NAME[dtype], envs=envs, channels=channels, states=states, x=_at(x), delta=_at(delta), gate=_at(gate), b=_at(b), c=_at(c), x_stride=x.stride(0), delta_stride=delta.stride(0),
                             gate_stride=gate.stride(0), b_stride=b.stride(0), c_stride=c.stride(0), decay=_at(decay), skip=_at(skip), delta_bias=_at(bias), state=_at(state), y=_at(y))
    assert lib.nuka_b200_scan_step(ctypes.byref(step), None) == 0
    m.check()


@pytest.mark.parametrize("dtype", list(NAME))
@pytest.mark.parametrize("channels,width", [(8, 4), (70, 3), (300, 2), (37, 4)])
def test_the_convolution(dtype, channels, width):
    lib = _abi.lib()
    for n, (offsets, tokens) in enumerate(_cases()):
        m = Buffers(n)
        plan, rows = _plan(m, offsets, tokens), len(offsets) - 1
        x, first = m.given(tokens, channels, dtype=dtype, apart=n % 2 * 3), m.given(rows, width - 1, channels, dtype=dtype)
        weight, bias = m.given(channels, width), m.given(channels)
        y, state = m.wanted(tokens, channels, dtype=dtype), m.wanted(rows, width - 1, channels, dtype=dtype)
        desc = _abi.ConvolutionDesc(plan=ctypes.pointer(plan), dtype=NAME[dtype], silu=n % 3 != 0, channels=channels, width=width, x=_at(x), x_stride=x.stride(0), weight=_at(weight), bias=_at(bias), initial=_at(first),
                                    y=_at(y), state=_at(state))
        assert lib.nuka_b200_convolution(ctypes.byref(desc), None) == 0
        m.check()
        work = m.bytes(lib.nuka_b200_convolution_workspace(ctypes.byref(plan), channels, width))
        given = dict(dy=m.given(tokens, channels, dtype=dtype), dstate=m.given(rows, width - 1, channels, dtype=dtype), dx=m.wanted(tokens, channels, dtype=dtype), dinitial=m.wanted(rows, width - 1, channels, dtype=dtype),
                     dweight=m.wanted(channels, width), dbias=m.wanted(channels), workspace=work)
        for name, v in given.items():
            setattr(desc, name, _at(v))
        desc.workspace_bytes = work.numel()
        assert lib.nuka_b200_convolution_backward(ctypes.byref(desc), None) == 0
        m.check()
    m, envs = Buffers(98), 37
    x, weight, bias = m.given(envs, channels, dtype=dtype, apart=5), m.given(channels, width), m.given(channels)
    state, y = m.wanted(envs, width - 1, channels, dtype=dtype, fill=1.0), m.wanted(envs, channels, dtype=dtype)
    step = _abi.ConvolutionStepDesc(dtype=NAME[dtype], silu=1, envs=envs, channels=channels, width=width, x=_at(x), x_stride=x.stride(0), weight=_at(weight), bias=_at(bias), state=_at(state), y=_at(y))
    assert lib.nuka_b200_convolution_step(ctypes.byref(step), None) == 0
    m.check()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads_q,heads_k,dim,window,sinks", [(2, 1, 64, 7, 3), (3, 3, 40, 100, 20), (4, 2, 128, 30, 70)])
def test_attention_with_first_tokens_that_stay(dtype, heads_q, heads_k, dim, window, sinks):
    lib = _abi.lib()
    for n, (offsets, tokens) in enumerate(_cases()):
        m = Buffers(n)
        plan, apart = _plan(m, offsets, tokens), n % 2 * 8
        q = m.given(tokens, heads_q * dim, dtype=dtype, apart=apart)
        k, v = (m.given(tokens, heads_k * dim, dtype=dtype, apart=apart) for _ in range(2))
        pitch = lib.nuka_b200_attention_pitch(tokens)
        out, lse = m.wanted(tokens, heads_q, dim, dtype=dtype), m.bytes(4 * heads_q * pitch)
        desc = _abi.AttentionDesc(plan=ctypes.pointer(plan), dtype=NAME[dtype], heads_q=heads_q, heads_k=heads_k, dim=dim, window=window, scale=dim ** -0.5, q=_at(q), k=_at(k), v=_at(v), q_stride=q.stride(0), q_head_stride=dim,
                                  k_stride=k.stride(0), k_head_stride=dim, v_stride=v.stride(0), v_head_stride=dim, out=_at(out), lse=_at(lse))
        assert lib.nuka_b200_attention_sinks(ctypes.byref(desc), sinks, None) == 0
        m.check()
        work = m.bytes(lib.nuka_b200_attention_sinks_workspace(ctypes.byref(desc), sinks))
        given = dict(dout=m.given(tokens, heads_q * dim, dtype=dtype), delta=m.bytes(4 * heads_q * pitch), dq=m.wanted(tokens, heads_q, dim, dtype=dtype), dk=m.wanted(tokens, heads_k, dim, dtype=dtype),
                     dv=m.wanted(tokens, heads_k, dim, dtype=dtype))
        for name, t in given.items():
            setattr(desc, name, _at(t))
        assert lib.nuka_b200_attention_sinks_backward(ctypes.byref(desc), sinks, _at(work) if work.numel() else None, work.numel(), None) == 0
        m.check()
