"""Sequence operators against their definitions in 64 bits: plan, gated recurrence, norms and rotation of heads.

Bounds.  A value rounded once to a type is off by at most half a unit in its last place, 2^-8 (bf16), 2^-11 (f16) of itself.  What is worked
out in 32 bits before is off by its roundings: about 2^-22 a step for a sigmoid and a product, over the few hundred steps that a
state remembers, with random signs: 2^-17 of the largest value.  The gradient of a gate reads h in its rounded type, which adds half a unit of
h times its factor."""
import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import nuka  # noqa: E402
from nuka import _abi, sequence as S  # noqa: E402

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
STEPS = 2.0 ** -17


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return torch.empty(shape, device="cuda").normal_(shift, scale, generator=gen).to(dtype)


def _close(got, want, bound, what):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert worst <= 0, f"{what}: {worst:.3e} beyond its bound, off by up to {off.max().item():.3e}"


def _plan_of(lengths):
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda")
    return S.Episodes.from_offsets(offsets, int(sum(lengths))), offsets


# ---- plan ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lengths", [[1], [0, 1, 0], [5, 0, 3, 1, 700, 0], [64] * 33, [0, 0], []])
def test_plan_from_offsets(lengths):
    plan, _ = _plan_of(lengths)
    at = np.concatenate([[0], np.cumsum(lengths)]).astype(int)
    first, end, link, tail = plan._plan.cpu().numpy()
    want = np.array([(at[r], at[r + 1], r if t == at[r] else -1, r if t + 1 == at[r + 1] else -1) for r in range(len(lengths)) for t in range(at[r], at[r + 1])]).reshape(-1, 4)
    assert np.array_equal(np.stack([first, end, link, tail], 1), want)
    assert np.array_equal(plan.positions.cpu().numpy(), np.arange(len(want)) - want[:, 0])


@pytest.mark.parametrize("shape,often", [((1, 1), 0.5), ((7, 24), 0.1), ((3, 2500), 0.01), ((2, 1025), 0.0), ((5, 40), 1.0), ((4, 0), 0.0)])
def test_plan_from_done(shape, often):
    done = torch.rand(shape, generator=_gen(1), device="cuda") < often
    plan = S.Episodes.from_done(done)
    n, length = shape
    d = done.cpu().numpy()
    want = []
    for r in range(n):
        begins = [0] + [t + 1 for t in range(length - 1) if d[r, t]]
        for t in range(length):
            first = max(b for b in begins if b <= t)
            end = min([b for b in begins if b > t] + [length])
            want.append((r * length + first, r * length + end, r if t == 0 else -2 if t == first else -1, r if t == length - 1 else -1))
    assert np.array_equal(plan._plan.cpu().numpy().T, np.array(want).reshape(-1, 4))


def test_offsets_that_lie_stay_inside_the_tokens():
    """Offsets are read on the device only: descending, negative and too large ones give a plan whose every index is a token."""
    for offsets in ([0, 50, 20, 10], [-5, 3, 1000, 7], [10, 10, 10, 10], [90, 95, 99, 2 ** 31 - 1]):
        plan = S.Episodes.from_offsets(torch.tensor(offsets, dtype=torch.int32, device="cuda"), 40)
        first, end, link, tail = plan._plan.cpu().numpy()
        t = np.arange(40)
        assert (first >= 0).all() and (first <= t).all() and (end > t).all() and (end <= 40).all()
        assert ((link >= -2) & (link < 3)).all() and ((tail >= -1) & (tail < 3)).all() and link[0] != -1


# ---- recurrence ------------------------------------------------------------------------------------------------------
def _recurrence_64(x, gate, plan, initial):
    """h, final states, and the h before each token, one token after the other."""
    first, end, link, tail = (v.tolist() for v in plan._plan.cpu())
    a = 1 / (1 + torch.exp(-gate))
    h, before = torch.zeros_like(x), torch.zeros_like(x)
    state = initial.clone()
    for t in range(x.shape[0]):
        if link[t] >= 0:
            before[t] = initial[link[t]]
        elif link[t] == -1:
            before[t] = h[t - 1]
        h[t] = a[t] * before[t] + (1 - a[t]) * x[t]
        if tail[t] >= 0:
            state[tail[t]] = h[t]
    return h, state, before


def _recurrence_grad_64(x, gate, plan, before, dh, dstate):
    first, end, link, tail = (v.tolist() for v in plan._plan.cpu())
    a = 1 / (1 + torch.exp(-gate))
    lam = torch.zeros_like(x)
    dinitial = dstate.clone()
    carry = torch.zeros_like(x[0]) if len(x) else None
    for t in range(x.shape[0] - 1, -1, -1):
        lam[t] = dh[t] + (carry if end[t] != t + 1 else 0) + (dstate[tail[t]] if tail[t] >= 0 else 0)
        carry = a[t] * lam[t]
        if link[t] >= 0:
            dinitial[link[t]] = carry
    return (1 - a) * lam, lam * (before - x) * a * (1 - a), dinitial, lam * a * (1 - a)


ROWS = {"one token": [1], "one row": [300], "odd rows": [5, 0, 3, 1, 700, 129, 0], "a long row": [9000], "short rows": [24] * 50, "chunk": [128, 64, 128], "empty": [0, 0]}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", list(ROWS))
@pytest.mark.parametrize("channels", [1, 6, 70, 128])
def test_recurrence_and_its_gradient(dtype, rows, channels):
    if rows == "a long row" and channels not in (1, 70):
        pytest.skip("the long row is walked once for each layout")
    gen, lengths = _gen(len(rows) + channels), ROWS[rows]
    plan, _ = _plan_of(lengths)
    n = sum(lengths)
    x, gate = _normal(gen, n, channels, dtype=dtype).requires_grad_(), _normal(gen, n, channels, dtype=dtype, scale=2.0, shift=2.0).requires_grad_()
    initial = _normal(gen, len(lengths), channels).requires_grad_()
    dh, dstate = _normal(gen, n, channels, dtype=dtype), _normal(gen, len(lengths), channels)
    h, state = S.gated_recurrence(x, gate, plan, initial)
    grads = torch.autograd.grad([h, state], [x, gate, initial], [dh, dstate])
    x64, g64, i64 = (v.detach().cpu().double() for v in (x, gate, initial))
    want_h, want_state, before = _recurrence_64(x64, g64, plan, i64)
    wants = _recurrence_grad_64(x64, g64, plan, before, dh.cpu().double(), dstate.cpu().double())
    unit, size = UNIT[dtype], lambda v: v.abs().max() if v.numel() else 0.0
    _close(h.detach().cpu(), want_h, unit * want_h.abs() + STEPS * size(want_h), "h")
    _close(state.detach().cpu(), want_state, STEPS * size(want_state), "state")
    _close(grads[0].cpu(), wants[0], unit * wants[0].abs() + STEPS * size(wants[0]), "dx")
    _close(grads[1].cpu(), wants[1], unit * (wants[1].abs() + (wants[3] * before).abs()) + STEPS * size(wants[1]), "dgate")
    _close(grads[2].cpu(), wants[2], STEPS * size(wants[2]), "dinitial")


@pytest.mark.parametrize("shape,often", [((9, 24), 0.1), ((2, 1500), 0.005), ((3, 64), 1.0)])
def test_recurrence_over_a_rollout_with_episodes_that_end_inside(shape, often):
    gen = _gen(3)
    done = torch.rand(shape, generator=gen, device="cuda") < often
    plan = S.Episodes.from_done(done)
    n, c = done.numel(), 40
    x, gate = (_normal(gen, n, c, dtype=torch.bfloat16).requires_grad_() for _ in range(2))
    dh = _normal(gen, n, c, dtype=torch.bfloat16)
    h, state = S.gated_recurrence(x, gate, plan)                    # no initial state: rows begin with 0
    dx, dgate = torch.autograd.grad(h, [x, gate], dh)
    zero = torch.zeros(shape[0], c, dtype=torch.float64)
    x64, g64 = x.detach().cpu().double(), gate.detach().cpu().double()
    want_h, want_state, before = _recurrence_64(x64, g64, plan, zero)
    want = _recurrence_grad_64(x64, g64, plan, before, dh.cpu().double(), zero)
    u = UNIT[torch.bfloat16]
    _close(h.detach().cpu(), want_h, u * want_h.abs() + STEPS * want_h.abs().max(), "h")
    _close(state.detach().cpu(), want_state, STEPS * want_state.abs().max(), "state")
    _close(dx.cpu(), want[0], u * want[0].abs() + STEPS * want[0].abs().max(), "dx")
    _close(dgate.cpu(), want[1], u * (want[1].abs() + (want[3] * before).abs()) + STEPS * want[1].abs().max(), "dgate")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("channels,length", [(20, 1), (64, 7), (37, 24), (72, 16), (256, 9)])
def test_many_rows_of_one_length(dtype, channels, length):
    """Rows enough for a warp each: the same values as of the rows one by one in other plans, gradients among them."""
    gen, n = _gen(channels + length), 2400
    done = torch.rand((n, length), generator=gen, device="cuda") < 0.1
    plan = S.Episodes.from_done(done)
    x, gate = (_normal(gen, n * length, channels, dtype=dtype).requires_grad_() for _ in range(2))
    initial = _normal(gen, n, channels).requires_grad_()
    dh, dstate = _normal(gen, n * length, channels, dtype=dtype), _normal(gen, n, channels)
    h, state = S.gated_recurrence(x, gate, plan, initial)
    grads = torch.autograd.grad([h, state], [x, gate, initial], [dh, dstate])
    x64, g64, i64 = (v.detach().cpu().double() for v in (x, gate, initial))
    some = torch.cat([torch.arange(r * length, (r + 1) * length) for r in (0, 1, 5, 1203, n - 1)])
    rows = [0, 1, 5, 1203, n - 1]
    small = S.Episodes.from_done(done[rows])
    want_h, want_state, before = _recurrence_64(x64[some], g64[some], small, i64[rows])
    want = _recurrence_grad_64(x64[some], g64[some], small, before, dh.cpu().double()[some], dstate.cpu().double()[rows])
    u = UNIT[dtype]
    _close(h.detach().cpu()[some], want_h, u * want_h.abs() + STEPS * want_h.abs().max(), "h")
    _close(state.detach().cpu()[rows], want_state, STEPS * want_state.abs().max(), "state")
    _close(grads[0].cpu()[some], want[0], u * want[0].abs() + STEPS * want[0].abs().max(), "dx")
    _close(grads[1].cpu()[some], want[1], u * (want[1].abs() + (want[3] * before).abs()) + STEPS * want[1].abs().max(), "dgate")
    _close(grads[2].cpu()[rows], want[2], STEPS * want[2].abs().max(), "dinitial")
    # and every row against the chunks' kernel, by offsets in place of one length, where no episode ends inside
    plain = S.Episodes.from_done(torch.zeros_like(done))
    offsets = S.Episodes.from_offsets(torch.arange(n + 1, dtype=torch.int32, device="cuda") * length, n * length)
    for got, other in zip(S.gated_recurrence(x, gate, plain, initial), S.gated_recurrence(x, gate, offsets, initial)):
        assert (got.double() - other.double()).abs().max().item() <= 2 * max(UNIT[got.dtype], STEPS) * other.abs().max().item()


def test_what_is_not_finite_stays_in_its_episode():
    lengths = [100, 90, 300, 40]
    plan, offsets = _plan_of(lengths)
    gen = _gen(4)
    clean_x, clean_g = _normal(gen, 530, 8), _normal(gen, 530, 8)
    dh = _normal(gen, 530, 8)
    outs = []
    for spoil in (False, True):
        x, g = clean_x.clone(), clean_g.clone()
        if spoil:
            x[150, 3], x[160, 4], g[170, 5], dh[120, 6] = math.nan, math.inf, math.nan, -math.inf       # all in the second row
        x.requires_grad_(); g.requires_grad_()
        initial = torch.zeros(4, 8, device="cuda")
        if spoil:
            initial[1, 7] = math.nan
        h, state = S.gated_recurrence(x, g, plan, initial)
        outs.append([h.detach(), *torch.autograd.grad(h, [x, g], dh)])
    other = torch.ones(530, dtype=torch.bool, device="cuda")
    other[100:190] = False
    for clean, spoiled in zip(*outs):
        assert torch.equal(clean[other], spoiled[other])
    assert torch.isnan(outs[1][0][150:190, 3]).all() and torch.isnan(outs[1][0][100:190, 7]).all()


def test_saturated_gates():
    """Gates so large that a is 0 or 1 in 32 bits: the state is kept or replaced exactly, gradients vanish without a NaN."""
    plan, _ = _plan_of([64])
    x = _normal(_gen(5), 64, 4).requires_grad_()
    g = torch.zeros(64, 4, device="cuda")
    g[:, 0], g[:, 1], g[:, 2], g[:, 3] = 200.0, -200.0, math.inf, -math.inf
    g.requires_grad_()
    initial = torch.full((1, 4), 3.0, device="cuda")
    h, _ = S.gated_recurrence(x, g, plan, initial)
    dx, dg = torch.autograd.grad(h.sum(), [x, g])
    assert (h[:, 0] == 3).all() and (h[:, 2] == 3).all() and torch.equal(h[:, 1], x[:, 1]) and torch.equal(h[:, 3], x[:, 3])
    assert torch.isfinite(dx).all() and (dg == 0).all()


def test_recurrence_gives_the_same_bits_every_time_and_takes_strided_inputs():
    plan, _ = _plan_of([20000, 3, 11000])
    both = _normal(_gen(6), 31003, 2 * 66, dtype=torch.bfloat16)
    x, gate = both[:, :66], both[:, 66:]                                       # two views of one projection
    outs = []
    for a, b in ((x, gate), (x.contiguous(), gate.contiguous()), (x, gate)):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        h, state = S.gated_recurrence(a, b, plan)
        outs.append([h.detach(), state.detach(), *torch.autograd.grad(h, [a, b], x.contiguous())])
    for other in outs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(outs[0], other))
    # broadcast over channels and over tokens, odd addresses: the same as of a copy
    for odd in (both[:, 1:67], both[:, :1].expand(-1, 66), both[:1, :66].expand(31003, -1), both.t()[:66].t()[:, ::2]):
        h = S.gated_recurrence(odd, odd, plan)[0]
        assert torch.equal(h, S.gated_recurrence(odd.contiguous(), odd.contiguous(), plan)[0])


def test_recurrence_gradient_against_differences():
    plan = S.Episodes.from_done(torch.rand((3, 50), generator=_gen(7), device="cuda") < 0.1)
    gen = _gen(8)
    x, g, i = _normal(gen, 150, 10).requires_grad_(), _normal(gen, 150, 10).requires_grad_(), _normal(gen, 3, 10).requires_grad_()
    w, ws = _normal(gen, 150, 10), _normal(gen, 3, 10)
    loss = lambda *a: sum((u.double() * v.double()).sum() for u, v in zip(S.gated_recurrence(a[0], a[1], plan, a[2]), (w, ws)))
    grads = torch.autograd.grad(loss(x, g, i), [x, g, i])
    for k, (v, grad) in enumerate(zip((x, g, i), grads)):
        d = _normal(gen, *v.shape)
        step = 1e-2
        ends = [loss(*(u.detach() + s * step * d if j == k else u.detach() for j, u in enumerate((x, g, i)))).item() for s in (1, -1)]
        # the differences' own error: step^2 / 6 of a third derivative (about the slope itself), 1e-4, and 32-bit roundings over the step, 1e-4 too
        slope = (grad.double() * d.double()).sum().item()
        assert abs((ends[0] - ends[1]) / (2 * step) - slope) <= 2e-3 * (abs(slope) + math.sqrt((grad.double() * d.double()).square().sum().item()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,channels", [(1, 256), (1, 1), (37, 30), (1000, 64), (0, 8)])
def test_steps_follow_the_scan(dtype, n, channels):
    """Acting token by token gives the states that the scan over the rollout gives: both in 32 bits, in another order of rounding."""
    gen, steps = _gen(9), 12
    done = torch.rand((n, steps), generator=gen, device="cuda") < 0.2
    x, gate = (_normal(gen, n, steps, channels, dtype=dtype) for _ in range(2))
    state = _normal(gen, n, channels)
    plan = S.Episodes.from_done(done)
    want_h, want = S.gated_recurrence(x.reshape(-1, channels), gate.reshape(-1, channels), plan, state.clone())
    for t in range(steps):
        h = S.gated_recurrence_step(x[:, t], gate[:, t], state, done[:, t - 1] if t else None)
        _close(h, want_h.view(n, steps, channels)[:, t].double(), 2 * UNIT[dtype] * h.double().abs() + STEPS * 4, f"h of step {t}")
    _close(state, want.double(), STEPS * 4, "state")


def test_recurrence_on_another_stream():
    plan, _ = _plan_of([5000, 100])
    x = _normal(_gen(10), 5100, 64)
    want = S.gated_recurrence(x, x, plan)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = S.gated_recurrence(x, x, plan)[0]
        assert torch.equal(got, want)
    torch.cuda.current_stream().wait_stream(side)


# ---- heads -----------------------------------------------------------------------------------------------------------
def _heads_64(x, w, position, frequencies, eps, interleaved):
    n = 2 * frequencies.numel()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w
    angle = (position.float()[:, None, None] * frequencies.float()).double()         # the definition: a product in 32 bits
    u, v = (y[..., 0:n:2], y[..., 1:n:2]) if interleaved else (y[..., :n // 2], y[..., n // 2:n])
    a, b = u * angle.cos() - v * angle.sin(), u * angle.sin() + v * angle.cos()
    return torch.cat([torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1), y[..., n:]], -1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,turned,interleaved", [(64, 64, False), (64, 32, True), (128, 128, True), (32, 8, False), (96, 48, False), (8, 8, True), (256, 256, False), (200, 0, False), (40, 24, True)])
@pytest.mark.parametrize("lengths,heads_q,heads_k", [([1], 1, 1), ([30, 0, 3, 41], 8, 2), ([17], 3, 3)])
def test_heads_and_their_gradient(dtype, dim, turned, interleaved, lengths, heads_q, heads_k):
    """Norm, weight and turn: a product each, so a few units in the last place of 32 bits before the one rounding; sums over dim values and, for the weights,
    over tokens times heads add the square root of their number."""
    gen = _gen(dim + turned)
    plan, _ = _plan_of(lengths)
    n = sum(lengths)
    both = _normal(gen, n, (heads_q + 2 * heads_k) * dim, dtype=dtype, scale=1.3)
    q = both[:, :heads_q * dim].unflatten(1, (heads_q, dim)).detach().requires_grad_()
    k = both[:, heads_q * dim:(heads_q + heads_k) * dim].unflatten(1, (heads_k, dim)).detach().requires_grad_()
    wq, wk = (_normal(gen, dim, scale=0.3, shift=1.0).requires_grad_() for _ in range(2))
    f = S.rotary_frequencies(turned).cuda()
    out = S.rotate_heads(q, k, wq, wk, plan, f, 1e-5, interleaved)
    cot = [_normal(gen, *o.shape, dtype=dtype) for o in out]
    grads = torch.autograd.grad(out, [q, k, wq, wk], cot)
    for name, x, w, got, dy, dx, dw in (("q", q, wq, out[0], cot[0], grads[0], grads[2]), ("k", k, wk, out[1], cot[1], grads[1], grads[3])):
        x64, w64 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
        want = _heads_64(x64, w64, plan.positions, f, 1e-5, interleaved)
        want_dx, want_dw = torch.autograd.grad(want, [x64, w64], dy.double())
        unit, ulps = UNIT[dtype], 16 * 2.0 ** -23
        _close(got.detach(), want.detach(), unit * want.detach().abs() + ulps * want.detach().abs().max(), name)
        _close(dx, want_dx, unit * want_dx.abs() + ulps * want_dx.abs().max(), "d" + name)
        _close(dw, want_dw, ulps * math.sqrt(n * x.shape[1]) * (dy.double().abs().max() * 4), "dw" + name)


def test_heads_at_far_positions():
    """Sines and cosines of angles of millions are as exact as those of small ones: whole turns are taken off in 64 bits."""
    f = S.rotary_frequencies(64).cuda()
    q = _normal(_gen(11), 5, 2, 64)
    positions = torch.tensor([0, 1, 131071, 1000003, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    got = S.rotate_heads(q, q, None, None, positions, f)[0]
    want = _heads_64(q.double(), None, positions, f, 1e-6, False)
    _close(got, want, 16 * 2.0 ** -23 * want.abs().max(), "q")


def test_heads_rows_of_zeros_and_views():
    f = S.rotary_frequencies(16).cuda()
    positions = torch.arange(6, dtype=torch.int32, device="cuda")
    q = torch.zeros(6, 2, 32, device="cuda", requires_grad=True)
    out = S.rotate_heads(q, q, None, None, positions, f)
    grad, = torch.autograd.grad(out[0].sum(), [q])
    assert (out[0] == 0).all() and torch.isfinite(grad).all()
    base = _normal(_gen(12), 6, 3, 33)
    for view in (base[:, :, :32], base[:, :, 1:], base[:, :1, 1:].expand(-1, 3, -1), base[:1, :, 1:].expand(6, -1, -1), base.transpose(0, 1)[:, :, :32].transpose(0, 1)):
        a, b = S.rotate_heads(view, view, None, None, positions, f), S.rotate_heads(view.contiguous(), view.contiguous(), None, None, positions, f)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_heads_gradient_against_differences_and_without_weights():
    gen = _gen(13)
    f = S.rotary_frequencies(24).cuda()
    positions = torch.arange(20, dtype=torch.int32, device="cuda")
    q, k, w = _normal(gen, 20, 3, 40).requires_grad_(), _normal(gen, 20, 1, 40).requires_grad_(), _normal(gen, 40, shift=1.0).requires_grad_()
    cq, ck = _normal(gen, 20, 3, 40), _normal(gen, 20, 1, 40)
    loss = lambda a, b, c: sum((u.double() * v.double()).sum() for u, v in zip(S.rotate_heads(a, b, None, c, positions, f, interleaved=True), (cq, ck)))
    grads = torch.autograd.grad(loss(q, k, w), [q, k, w])
    for i, (v, grad) in enumerate(zip((q, k, w), grads)):
        d, step = _normal(gen, *v.shape), 1e-2
        ends = [loss(*(u.detach() + s * step * d if j == i else u.detach() for j, u in enumerate((q, k, w)))).item() for s in (1, -1)]
        slope = (grad.double() * d.double()).sum().item()
        assert abs((ends[0] - ends[1]) / (2 * step) - slope) <= 2e-3 * (abs(slope) + math.sqrt((grad.double() * d.double()).square().sum().item()))


def test_frequencies_for_long_contexts():
    """Pairs that turn often within the trained context stay, those that hardly turn are slowed down by the whole factor."""
    f, g = S.rotary_frequencies(64), S.rotary_frequencies(64, trained=1024, context=4096)
    turns = 1024 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.allclose(g[turns <= 1], f[turns <= 1] / 4, rtol=1e-12, atol=0)
    mixed = (turns > 1) & (turns < 32)
    assert mixed.any() and (g[mixed] < f[mixed]).all() and (g[mixed] > f[mixed] / 4).all()


# ---- refusals --------------------------------------------------------------------------------------------------------
def test_wrong_arguments_are_refused():
    plan, offsets = _plan_of([4, 5])
    x = torch.zeros(9, 8, device="cuda")
    q = torch.zeros(9, 2, 16, device="cuda")
    f = torch.ones(4, dtype=torch.float64, device="cuda")
    with pytest.raises(ValueError, match="on the GPU"):
        S.gated_recurrence(x.cpu(), x.cpu(), plan)
    for bad in (lambda: S.gated_recurrence(x[:8], x[:8], plan), lambda: S.gated_recurrence(x, x.half(), plan), lambda: S.gated_recurrence(x.double(), x.double(), plan),
                lambda: S.gated_recurrence(x, x, plan, torch.zeros(3, 8, device="cuda")), lambda: S.gated_recurrence(x, x, plan, torch.zeros(2, 8, device="cuda").half()),
                lambda: S.gated_recurrence_step(x, x, x[:, :4]), lambda: S.gated_recurrence_step(x, x, x.half()), lambda: S.gated_recurrence_step(x, x, x.clone(), torch.zeros(8, dtype=torch.bool, device="cuda")),
                lambda: S.rotate_heads(q, q[:, :, :8], None, None, plan, f), lambda: S.rotate_heads(q, q, None, None, plan, f.float()),
                lambda: S.rotate_heads(q, q, torch.ones(8, device="cuda"), None, plan, f), lambda: S.rotate_heads(q, q, None, None, torch.zeros(9, device="cuda"), f),
                lambda: S.Episodes.from_offsets(offsets.long(), 9), lambda: S.Episodes.from_done(x[0]), lambda: S.Episodes.from_offsets(offsets, -1)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: S.rotate_heads(q[:, :, :12], q[:, :, :12], None, None, plan, f), lambda: S.rotate_heads(q, q, None, None, plan, torch.ones(9, dtype=torch.float64, device="cuda")),
                lambda: S.rotate_heads(q, q, None, None, plan, f[:3]), lambda: S.rotate_heads(q, q, None, None, plan, f, eps=-1.0),
                lambda: S.Episodes.from_offsets(offsets[:1], 9)):
        with pytest.raises(nuka.NukaError):
            bad()


def test_the_c_entries_refuse_what_they_cannot_take():
    lib = _abi.lib()
    plan, _ = _plan_of([200, 100])
    x = torch.zeros(300, 8, device="cuda")
    ok = dict(plan=plan._ref, dtype=0, channels=8, x=x.data_ptr(), gate=x.data_ptr(), x_stride=8, gate_stride=8, h=x.data_ptr(), state=x.data_ptr())
    call = lambda **change: lib.nuka_b200_recurrence(ctypes.byref(_abi.RecurrenceDesc(**{**ok, **change})), None)
    assert lib.nuka_b200_recurrence(None, None) == _abi.INVALID_ARG
    small, _ = _plan_of([10])
    assert lib.nuka_b200_recurrence_workspace(plan._ref, 8) > 0 and lib.nuka_b200_recurrence_workspace(small._ref, 8) == 0
    for change in (dict(x=None), dict(h=None), dict(state=None), dict(x=x.data_ptr() + 2), dict(x_stride=-8), dict(channels=-1), dict(), dict(workspace=x.data_ptr(), workspace_bytes=64)):
        assert call(**change) == _abi.INVALID_ARG, change                       # the last two: no workspace, too small a one
        assert lib.nuka_last_error_message() != b""
    assert call(dtype=3) == 7
    plan_of = lambda **change: ctypes.byref(_abi.EpisodesDesc(**{**dict(first=x.data_ptr(), end=x.data_ptr(), link=x.data_ptr(), tail=x.data_ptr(), tokens=9, rows=2, length=0), **change}))
    for length in (0, 4, -1):                                                   # 2 rows of 4 are not 9 tokens
        assert lib.nuka_b200_episodes_from_done(plan_of(length=length), x.data_ptr(), None) == _abi.INVALID_ARG
    for change in (dict(tokens=-1), dict(tokens=2 ** 31), dict(rows=0), dict(link=None)):
        assert lib.nuka_b200_episodes_from_offsets(plan_of(**change), x.data_ptr(), None) == _abi.INVALID_ARG
    assert lib.nuka_b200_heads(None, None) == _abi.INVALID_ARG and lib.nuka_b200_recurrence_step(0, 1, 8, None, 8, None, 8, None, None, None, None) == _abi.INVALID_ARG
    assert lib.nuka_b200_recurrence_step(9, 1, 8, x.data_ptr(), 8, x.data_ptr(), 8, None, x.data_ptr(), x.data_ptr(), None) == 7
