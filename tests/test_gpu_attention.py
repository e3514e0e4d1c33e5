"""Attention over packed episodes against its definition in 64 bits.

Bounds, value by value.  An output is rounded once (half a unit u of itself), and so is each probability before it meets its value row: u sum p |v|.
Backwards dv has the same from do; dq and dk have u sum |ds| |k| from ds's rounding, and sum p |k| times u |do| . |o| because D = do . o reads the
rounded output.  What is worked out in 32 bits (scores of up to a few dozen, their exponentials, sums) is off by 2^-15 of the sum of the terms' sizes at most.
In f16 a probability or its gradient below 2^-14 is rounded to a multiple of 2^-24."""
import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import nuka  # noqa: E402
from nuka import _abi, sequence as S  # noqa: E402

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
STEP = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
SUMS = 2.0 ** -15


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, dtype=torch.bfloat16, scale=1.0):
    return torch.empty(shape, device="cuda").normal_(0.0, scale, generator=gen).to(dtype)


def _plan_of(lengths):
    return S.Episodes.from_offsets(torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda"), int(sum(lengths)))


def _seen(plan, window):
    at = torch.arange(plan.tokens, device="cuda")
    low = plan.first.long()
    if window:
        low = torch.maximum(low, at - window + 1)
    return (at[None, :] <= at[:, None]) & (at[None, :] >= low[:, None])


def _reference(q, k, v, plan, scale, window, do=None):
    """Outputs and, with `do`, gradients in 64 bits, and the sums of the sizes that the bounds are made of; head by head."""
    q, k, v = (x.detach().double() for x in (q, k, v))
    group, unseen = q.shape[1] // k.shape[1], ~_seen(plan, window)
    got = {n: torch.zeros_like(x) for n, x in (("o", q), ("o_p", q), ("dq", q), ("dq_s", q), ("dq_n", q), ("dk", k), ("dk_s", k), ("dk_n", k), ("dv", v), ("dv_p", v), ("dv_n", v), ("o_n", q))}
    for h in range(q.shape[1]):
        g = h // group
        p = torch.softmax((q[:, h] @ k[:, g].t() * scale).masked_fill(unseen, -math.inf), -1)
        o = p @ v[:, g]
        got["o"][:, h], got["o_p"][:, h], got["o_n"][:, h] = o, p @ v[:, g].abs(), (~unseen).double() @ v[:, g].abs()
        if do is None:
            continue
        d = do[:, h].double()
        dp, delta, slack = d @ v[:, g].t(), (d * o).sum(-1, keepdim=True), (d.abs() * o.abs()).sum(-1, keepdim=True)
        ds, size = p * (dp - delta) * scale, p * (d.abs() @ v[:, g].abs().t() * SUMS + (dp.abs() + delta.abs()) * SUMS + slack * 2.0 ** -7 * UNIT_OF[0]) * scale + (p * (dp - delta)).abs() * scale * UNIT_OF[1]
        got["dv"][:, g] += p.t() @ d
        got["dv_p"][:, g] += p.t() @ d.abs()
        got["dv_n"][:, g] += (~unseen).double().t() @ d.abs()
        got["dq"][:, h], got["dq_s"][:, h], got["dq_n"][:, h] = ds @ k[:, g], size @ k[:, g].abs(), scale * (~unseen).double() @ k[:, g].abs()
        got["dk"][:, g] += ds.t() @ q[:, h]
        got["dk_s"][:, g] += size.t() @ q[:, h].abs()
        got["dk_n"][:, g] += scale * (~unseen).double().t() @ q[:, h].abs()
    return got


UNIT_OF = [1.0, 2.0 ** -8]           # of the type that is tested: the output's unit in units of bf16's over 2, and the type's own


def _close(got, want, bound, what):
    assert torch.isfinite(got).all(), what
    off = (got.double() - want).abs()
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert worst <= 0, f"{what}: {worst:.3e} beyond its bound, off by up to {off.max().item():.3e}"


def _bounds(w, unit, step):
    """(value, bound) of the outputs and gradients of _reference."""
    return {"o": (w["o"], unit * (w["o"].abs() + w["o_p"]) + SUMS * w["o_p"] + step * w["o_n"] + step), "dq": (w["dq"], unit * w["dq"].abs() + w["dq_s"] + step * w["dq_n"] + step),
            "dk": (w["dk"], unit * w["dk"].abs() + w["dk_s"] + step * w["dk_n"] + step), "dv": (w["dv"], unit * (w["dv"].abs() + w["dv_p"]) + SUMS * w["dv_p"] + step * w["dv_n"] + step)}


def _check(q, k, v, plan, do, window=None, scale=None):
    unit, step = UNIT[q.dtype], STEP[q.dtype]
    UNIT_OF[:] = [unit * 2.0 ** 7, unit]
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    o = S.episode_attention(q, k, v, plan, scale=scale, window=window)
    grads = torch.autograd.grad(o, [q, k, v], do)
    w = _reference(q, k, v, plan, q.shape[2] ** -0.5 if scale is None else scale, window, do)
    for (name, (want, bound)), got in zip(_bounds(w, unit, step).items(), [o.detach(), *grads]):
        _close(got, want, bound, name)


def _inputs(gen, n, heads_q, heads_k, dim, dtype, scale=1.2):
    both = _normal(gen, n, (heads_q + 2 * heads_k) * dim, dtype=dtype, scale=scale)           # views of one projection
    cut = lambda low, heads: both[:, low * dim:(low + heads) * dim].unflatten(1, (heads, dim))
    return cut(0, heads_q), cut(heads_q, heads_k), cut(heads_q + heads_k, heads_k), _normal(gen, n, heads_q, dim, dtype=dtype)


LENGTHS = {"one": [1], "two": [2], "a tile": [128], "a tile and one": [129], "short": [24] * 20, "odd": [5, 0, 300, 1, 1, 77, 0, 130], "long": [1000], "ones": [1] * 140, "late": [100, 400]}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_and_its_gradient(dtype, lengths, dim):
    plan = _plan_of(LENGTHS[lengths])
    q, k, v, do = _inputs(_gen(dim + len(lengths)), plan.tokens, 4, 2, dim, dtype)
    _check(q, k, v, plan, do)


@pytest.mark.parametrize("heads_q,heads_k", [(1, 1), (3, 3), (6, 2), (8, 1)])
@pytest.mark.parametrize("dim", [8, 32, 40, 96, 120])
def test_head_layouts_and_sizes(heads_q, heads_k, dim):
    plan = _plan_of([150, 3, 90])
    q, k, v, do = _inputs(_gen(dim + heads_q), plan.tokens, heads_q, heads_k, dim, torch.bfloat16)
    _check(q, k, v, plan, do)


@pytest.mark.parametrize("window", [1, 2, 64, 127, 128, 129, 1000])
@pytest.mark.parametrize("dim", [64, 128])
def test_windows(window, dim):
    plan = _plan_of([500, 90, 1, 60])
    q, k, v, do = _inputs(_gen(window), plan.tokens, 2, 1, dim, torch.bfloat16)
    _check(q, k, v, plan, do, window=window)


def test_rollouts_with_episodes_that_end_inside():
    plan = S.Episodes.from_done(torch.rand((13, 61), generator=_gen(1), device="cuda") < 0.05)
    q, k, v, do = _inputs(_gen(2), plan.tokens, 4, 2, 64, torch.bfloat16)
    _check(q, k, v, plan, do)


@pytest.mark.parametrize("rows,length", [(300, 1), (90, 3), (50, 24), (11, 37), (5, 100), (3, 128), (2, 129)])
@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (128, torch.float16)])
def test_rows_of_one_length(rows, length, dim, dtype):
    """Rows that share a tile whole, with and without a remainder of the tile, and rows that are too long for it."""
    plan = S.Episodes.from_done(torch.rand((rows, length), generator=_gen(rows), device="cuda") < 0.03)
    q, k, v, do = _inputs(_gen(length), plan.tokens, 4, 2, dim, dtype)
    _check(q, k, v, plan, do, window=None if length != 37 else 9)


def test_more_jobs_than_blocks():
    """Blocks that take several tiles and heads in turn, of very different lengths."""
    plan = _plan_of([900, 3, 0, 1, 1300, 40, 700, 129])
    q, k, v, do = _inputs(_gen(20), plan.tokens, 32, 4, 64, torch.bfloat16)
    _check(q, k, v, plan, do)
    q, k, v, do = _inputs(_gen(21), plan.tokens, 24, 24, 72, torch.bfloat16)
    _check(q, k, v, plan, do, window=300)


@pytest.mark.parametrize("heads_q,heads_k", [(6, 1), (12, 1), (16, 2)])
@pytest.mark.parametrize("lengths", [[300, 20], [1100]])
@pytest.mark.parametrize("dim", [64, 128])
def test_heads_shared_by_blocks(heads_q, heads_k, lengths, dim):
    """Few jobs: several blocks have some heads of a key head's group each, and add up."""
    plan = _plan_of(lengths)
    q, k, v, do = _inputs(_gen(dim + heads_q), plan.tokens, heads_q, heads_k, dim, torch.bfloat16)
    _check(q, k, v, plan, do)


@pytest.mark.parametrize("size,scale", [(8.0, None), (1.0, 1.0), (1.0, 1e-3)])
@pytest.mark.parametrize("dim", [64, 128])
def test_sharp_and_flat_softmax(size, scale, dim):
    """Scores of hundreds, where the running maximum jumps from tile to tile and most probabilities are 0; scores that hardly differ."""
    plan = _plan_of([700, 20])
    q, k, v, do = _inputs(_gen(3), plan.tokens, 2, 2, dim, torch.bfloat16)
    o = S.episode_attention(q * size, k * size, v, plan, scale=scale)
    w = _reference(q * size, k * size, v, plan, dim ** -0.5 if scale is None else scale, None)
    # scores of up to some 1000: their 32-bit rounding is 2^-24 of it, in the exponent
    _close(o, w["o"], UNIT[q.dtype] * (w["o"].abs() + w["o_p"]) + 2.0 ** -12 * w["o_p"], "o")


def test_scores_that_only_fall_and_only_rise():
    """Tiles whose maximum is far below, and far above, the one before."""
    plan = _plan_of([640])
    ramp = torch.linspace(-40, 40, 640, device="cuda")
    for r in (ramp, -ramp):
        q = torch.ones(640, 1, 64, device="cuda", dtype=torch.bfloat16)
        k = (r[:, None, None] / 8 * torch.ones(1, 1, 64, device="cuda")).bfloat16()
        v, do = _normal(_gen(4), 640, 1, 64), _normal(_gen(5), 640, 1, 64)
        _check(q, k, v, plan, do)


def test_keys_that_are_not_finite_stay_in_their_episode():
    plan = _plan_of([40, 50, 200])
    q, k, v, do = _inputs(_gen(6), plan.tokens, 2, 1, 64, torch.bfloat16)
    want = S.episode_attention(q, k, v, plan)
    k = k.clone()
    k[60], k[70] = math.nan, math.inf
    got = S.episode_attention(q, k, v, plan)
    other = torch.ones(plan.tokens, dtype=torch.bool, device="cuda")
    other[60:90] = False
    assert torch.equal(got[other], want[other]) and torch.isnan(got[60:90]).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("what", ["q", "k", "v", "do"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_what_is_not_finite_stays_in_its_episode(dim, what, value):
    """One token of one episode: outputs and gradients of the others are what they are without it, within the bounds of all values (they share tiles, and are worked out row by row)."""
    plan = _plan_of([30, 40, 200, 24, 90])
    names = ("q", "k", "v", "do")
    clean = dict(zip(names, (x.clone() for x in _inputs(_gen(30), plan.tokens, 4, 2, dim, torch.bfloat16))))
    spoilt = {n: x.clone() for n, x in clean.items()}
    spoilt[what][100, 0, 5] = value                        # in the third episode
    UNIT_OF[:] = [UNIT[torch.bfloat16] * 2.0 ** 7, UNIT[torch.bfloat16]]
    w = _reference(*(clean[n] for n in names[:3]), plan, dim ** -0.5, None, clean["do"])
    q, k, v = (spoilt[n].requires_grad_() for n in names[:3])
    o = S.episode_attention(q, k, v, plan)
    outs = [o.detach(), *torch.autograd.grad(o, [q, k, v], spoilt["do"])]
    other = torch.ones(plan.tokens, dtype=torch.bool, device="cuda")
    other[70:270] = False
    for (name, (want, bound)), got in zip(_bounds(w, UNIT[torch.bfloat16], 0.0).items(), outs):
        _close(got[other], want[other], bound[other], name)
    spoils = {"q": [0], "k": [0], "v": [0], "do": [1, 2, 3]}[what]
    assert all(not torch.isfinite(outs[n][70:270]).all() for n in spoils)
    # rows of the same episode from before the token do not see it
    assert torch.isfinite(outs[0][70:100]).all()


def test_same_bits_every_time_strides_and_streams():
    plan = _plan_of([3000, 17, 900])
    q, k, v, do = _inputs(_gen(7), plan.tokens, 4, 2, 64, torch.bfloat16)
    outs = []
    side = torch.cuda.Stream()
    for way in range(3):
        a, b, c = (x.detach().clone().requires_grad_() if way == 1 else x.detach().requires_grad_() for x in (q, k, v))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side if way == 2 else torch.cuda.current_stream()):
            o = S.episode_attention(a, b, c, plan)
            outs.append([o.detach(), *torch.autograd.grad(o, [a, b, c], do)])
        torch.cuda.synchronize()
    for other in outs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(outs[0], other))
    # one key row for all tokens, keys that all heads share by broadcast, odd addresses: the same as of copies
    wide = _normal(_gen(8), plan.tokens, 2, 65)
    for a in (wide[:, :, 1:], wide[:, :1, :64].expand(-1, 2, -1), wide[:1, :, :64].expand(plan.tokens, -1, -1), wide.transpose(0, 1).contiguous().transpose(0, 1)[:, :, :64]):
        assert torch.equal(S.episode_attention(q, a, a, plan), S.episode_attention(q, a.contiguous(), a.contiguous(), plan))


def test_gradient_against_differences():
    plan = _plan_of([90, 60])
    gen = _gen(9)
    q, k, v, do = (x.float() for x in _inputs(gen, 150, 2, 1, 32, torch.float16, 0.5))
    loss = lambda *x: (S.episode_attention(*(y.half() for y in x), plan).double() * do.double()).sum()
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    for n, grad in enumerate(grads):
        # along the gradient itself, a step long enough that the roundings of f16 (2^-11 of each of 9600 terms, random signs) stay below a hundredth of the change
        d = grad / grad.norm()
        step = 0.5
        ends = [loss(*(x + s * step * d if n == j else x for j, x in enumerate((q, k, v)))).item() for s in (1, -1)]
        assert abs((ends[0] - ends[1]) / (2 * step) / grad.double().norm().item() - 1) <= 0.03


def test_no_tokens():
    plan = _plan_of([0, 0])
    q = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    o = S.episode_attention(q, q, q, plan)
    assert o.shape == (0, 2, 64) and torch.autograd.grad(o.sum(), q)[0].shape == q.shape


def test_wrong_arguments_are_refused():
    plan = _plan_of([10])
    q = torch.zeros(10, 4, 64, dtype=torch.bfloat16, device="cuda")
    for bad in (lambda: S.episode_attention(q.float(), q.float(), q.float(), plan), lambda: S.episode_attention(q, q[:, :3], q[:, :3], plan), lambda: S.episode_attention(q, q[:, :2], q, plan),
                lambda: S.episode_attention(q[:9], q[:9], q[:9], plan), lambda: S.episode_attention(q, q.half(), q.half(), plan), lambda: S.episode_attention(q, q, q, plan, window=0),
                lambda: S.episode_attention(q, q[:, :0], q[:, :0], plan), lambda: S.episode_attention(q.cpu(), q.cpu(), q.cpu(), plan)):
        with pytest.raises(ValueError):
            bad()
    wide = torch.zeros(10, 1, 136, dtype=torch.bfloat16, device="cuda")
    for bad in (lambda: S.episode_attention(wide, wide, wide, plan), lambda: S.episode_attention(q[:, :, :12], q[:, :, :12], q[:, :, :12], plan),
                lambda: S.episode_attention(q, q, q, plan, scale=0.0), lambda: S.episode_attention(q, q, q, plan, scale=math.nan), lambda: S.episode_attention(q, q, q, plan, scale=math.inf)):
        with pytest.raises(nuka.NukaError):
            bad()
    lib = _abi.lib()
    ok = dict(plan=plan._ref, dtype=2, heads_q=4, heads_k=4, dim=64, window=0, scale=0.125, q=q.data_ptr(), k=q.data_ptr(), v=q.data_ptr(), q_stride=256, q_head_stride=64, k_stride=256,
              k_head_stride=64, v_stride=256, v_head_stride=64, out=q.data_ptr())
    call = lambda back=False, **change: (lib.nuka_b200_attention_backward if back else lib.nuka_b200_attention)(ctypes.byref(_abi.AttentionDesc(**{**ok, **change})), None)
    for change in (dict(q=None), dict(q=q.data_ptr() + 8), dict(q_stride=255), dict(k_head_stride=0), dict(heads_k=3), dict(window=-1), dict(lse=q.data_ptr() + 4), dict(plan=None), dict(back=True)):
        assert call(**change) == _abi.INVALID_ARG, change
        assert lib.nuka_last_error_message() != b""
    assert call(dtype=0) == 7 and lib.nuka_b200_attention(None, None) == _abi.INVALID_ARG
