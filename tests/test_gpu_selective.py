"""The short causal convolution and the selective scan against their definitions in 64 bits, worked out token after token.

Bounds.  A value rounded once to a type is off by at most half a unit in its last place, `unit` of itself (and half a step of 2^-24 where f16 ends).  What is worked out in 32 bits is off by its
roundings: an exponential by 2^-22 of itself, its argument by 2^-23 of that, a product or sum by 2^-24; SLIP = 2^-20 of the sum of the terms' sizes covers the few of them in each formula.
What a state has gathered is followed by the same recurrence as the state: E_t = a (E_{t-1} + SLIP (1 + dt |A|) H_{t-1}) + SLIP |dt x B| with H the sum of the sizes; backwards alike.
An exponential below 2^-126, the least normal value of 32 bits, is 0: off by TINY = 2^-126 at most, times what it multiplies; what products of that size round to, 64 of them in a sum, is below 2^-120.
Sums over tokens are made in chains of at most a few hundred terms: 2^-15 of the sum of the sizes."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import nuka  # noqa: E402
from nuka import sequence as S  # noqa: E402

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
STEP = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
SLIP, CHAIN, TINY = 2.0 ** -20, 2.0 ** -15, 2.0 ** -126


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return torch.empty(shape, device="cuda").normal_(shift, scale, generator=gen).to(dtype)


def _plan_of(lengths):
    return S.Episodes.from_offsets(torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda"), int(sum(lengths)))


def _done_plan(rows, length, often, seed=3):
    done = torch.rand((rows, length), generator=_gen(seed), device="cuda") < often
    return S.Episodes.from_done(done)


def _walk(plan):
    """(token, the row that it begins or None, whether it begins an episode, the row that it ends or None), in order."""
    _, _, link, tail = plan._plan.tolist()
    return [(t, link[t] if link[t] >= 0 else None, link[t] != -1, tail[t] if tail[t] >= 0 else None) for t in range(plan.tokens)]


def _close(got, want, bound, what, unit=0.0, step=0.0):
    if want is None:
        assert got is None, what
        return
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    off, bound = (got.double() - want).abs(), bound + unit * want.abs() + step + 64 * TINY
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert worst <= 0, f"{what}: {worst:.3e} beyond its bound, off by up to {off.max().item():.3e}"


def _silu(x):
    r = torch.special.expit(x)
    return x * r, r * (1 + x * (1 - r))


# ---- convolution -----------------------------------------------------------------------------------------------------
def _reference_convolution(x, weight, bias, initial, plan, silu, dy, dstate):
    """{name: (value, bound)} by walking the tokens with the last inputs, then back."""
    x, weight, dy = x.detach().double(), weight.detach().double(), dy.double()
    channels, width = weight.shape
    bias = torch.zeros(channels, dtype=torch.float64, device="cuda") if bias is None else bias.detach().double()
    start = torch.zeros(plan.rows, width - 1, channels, dtype=torch.float64, device="cuda") if initial is None else initial.detach().double()
    windows, size, state = [], [], start.clone()
    ds, slip = [], []
    y, y_slip = torch.zeros_like(x), torch.zeros_like(x)
    window = None
    for t, row, begins, ends in _walk(plan):
        if begins:
            window = start[row] if row is not None else torch.zeros_like(start[0])
        window = torch.cat([window, x[t][None]])
        s = bias + (window * weight.t()).sum(0)
        sizes = bias.abs() + (window * weight.t()).abs().sum(0)
        act, slope = _silu(s) if silu else (s, torch.ones_like(s))
        y[t], y_slip[t] = act, SLIP * sizes * (1 + s.abs())
        windows.append(window)
        ds.append(dy[t] * slope)
        slip.append(dy[t].abs() * SLIP * (2 + sizes))
        window = window[1:]
        if ends is not None:
            state[ends] = window
    dx, dx_slip, dw, dw_size, dinitial, dinitial_slip = (torch.zeros_like(v) for v in (x, x, weight, weight, start, start))
    dinitial_slip += 0.0
    reach = torch.zeros(width - 1, channels, dtype=torch.float64, device="cuda")
    reach_slip = torch.zeros_like(reach)
    for t, row, begins, ends in reversed(_walk(plan)):
        if ends is not None:                        # nothing comes back from another row
            reach = dstate[ends].double() if dstate is not None else torch.zeros_like(reach)
            reach_slip = reach.abs() * SLIP
        grad = torch.cat([torch.zeros_like(reach[:1]), reach]) + weight.t() * ds[t]
        grad_slip = torch.cat([torch.zeros_like(reach[:1]), reach_slip]) + weight.t().abs() * slip[t]
        dx[t], dx_slip[t] = grad[-1], grad_slip[-1]
        dw += (windows[t] * ds[t]).t()
        dw_size += (windows[t].abs() * (slip[t] + CHAIN * ds[t].abs())).t()
        reach, reach_slip = grad[:-1], grad_slip[:-1]
        if begins:
            if row is not None:
                dinitial[row], dinitial_slip[row] = reach, reach_slip
            reach, reach_slip = torch.zeros_like(reach), torch.zeros_like(reach)
    for row in range(plan.rows):                    # an empty row ends with what it began with
        if dstate is not None and row not in {r for _, r, _, _ in _walk(plan)}:
            dinitial[row] = dstate[row].double()
    nothing = torch.zeros(channels, dtype=torch.float64, device="cuda")
    db = sum(ds) if ds else nothing
    db_size = sum(a + CHAIN * b.abs() for a, b in zip(slip, ds)) if ds else nothing
    return {"y": (y, y_slip), "state": (state, torch.zeros_like(state)), "x": (dx, dx_slip), "weight": (dw, dw_size), "bias": (db, db_size), "initial": (dinitial, dinitial_slip)}


def _check_convolution(plan, channels, width, dtype, seed=0, silu=True, bias=True, initial=True, dstate=True, strided=True):
    gen = _gen(seed)
    x = _normal(gen, plan.tokens, 2 * channels, dtype=dtype)[:, :channels] if strided else _normal(gen, plan.tokens, channels, dtype=dtype)
    weight, b = _normal(gen, channels, width), _normal(gen, channels) if bias else None
    first = _normal(gen, plan.rows, width - 1, channels, dtype=dtype) if initial else None
    leaves = {name: v.detach().requires_grad_() for name, v in (("x", x), ("weight", weight), ("bias", b), ("initial", first)) if v is not None}
    y, state = S.short_convolution(leaves["x"], leaves["weight"], leaves.get("bias"), plan, leaves.get("initial"), silu=silu)
    dy, ds = _normal(gen, *y.shape, dtype=dtype), _normal(gen, *state.shape, dtype=dtype) if dstate else None
    grads = torch.autograd.grad([y, state] if dstate else [y], list(leaves.values()), [dy, ds] if dstate else [dy])
    want = _reference_convolution(x, weight, b, first, plan, silu, dy, ds)
    for name, got in [("y", y.detach()), ("state", state.detach()), *zip(leaves, grads)]:
        floating = name in ("weight", "bias")
        _close(got, *want[name], name, UNIT[torch.float32 if floating else dtype], 0.0 if floating else STEP[dtype])
    plain = S.short_convolution(x, weight, b, plan, first, silu=silu)                 # without gradients, the same
    assert torch.equal(plain[0], y) and torch.equal(plain[1], state)


PLANS = {"one": lambda: _plan_of([1]), "rows of one": lambda: _done_plan(37, 1, 0.5), "short": lambda: _done_plan(70, 24, 0.1), "odd": lambda: _plan_of([5, 0, 300, 1, 1, 77, 0, 130, 2, 3]), "long": lambda: _plan_of([1000, 33]),
         "many ends": lambda: _done_plan(3, 250, 0.4), "all ends": lambda: _done_plan(2, 100, 1.1), "edges": lambda: _plan_of([32, 31, 33, 64, 2]), "no tokens": lambda: _plan_of([0, 0])}


@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("plan", list(PLANS))
def test_convolution_and_its_gradients(dtype, plan):
    _check_convolution(PLANS[plan](), 40, 4, dtype)


@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("channels", [1, 7, 8, 257, 264])
def test_convolution_sizes(width, channels):
    for dtype in UNIT:
        _check_convolution(_done_plan(9, 40, 0.1), channels, width, dtype, seed=channels, strided=channels % 2 == 0)


@pytest.mark.parametrize("change", [dict(silu=False), dict(bias=False), dict(initial=False), dict(dstate=False), dict(initial=False, dstate=False, bias=False, silu=False)])
def test_convolution_options(change):
    _check_convolution(_plan_of([2, 0, 70, 1]), 24, 4, torch.bfloat16, **change)


@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("width,channels", [(2, 5), (3, 32), (4, 260)])
def test_convolution_steps_are_the_convolution(dtype, width, channels):
    """Token after token of every env, with episodes that begin on the way: the bits of the training form, whose order of operations they have."""
    envs, steps = 11, 9
    gen = _gen(width)
    done = torch.rand((envs, steps), generator=gen, device="cuda") < 0.3
    x, weight, bias = _normal(gen, envs, steps, channels, dtype=dtype), _normal(gen, channels, width), _normal(gen, channels)
    state = _normal(gen, envs, width - 1, channels, dtype=dtype)
    y, last = S.short_convolution(x.flatten(0, 1), weight, bias, S.Episodes.from_done(done), state, silu=True)
    fresh = None
    for t in range(steps):
        got = S.short_convolution_step(x[:, t], weight, bias, state, fresh, silu=True)
        assert torch.equal(got, y.view(envs, steps, channels)[:, t]), t
        fresh = done[:, t]
    assert torch.equal(state, last)


# ---- scan --------------------------------------------------------------------------------------------------------------
def _softplus(u):
    return torch.logaddexp(u, torch.zeros_like(u))


def _reference_scan(v, plan, dy, dstate):
    """{name: (value, bound)}: the states and the sizes of what they gathered, token by token, then back."""
    v = {name: None if x is None else x.detach().double() for name, x in v.items()}
    x, b, c, decay = v["x"], v["b"], v["c"], v["decay"]
    channels, states = decay.shape
    zero = lambda *shape: torch.zeros(shape, dtype=torch.float64, device="cuda")
    skip = zero(channels) if v["skip"] is None else v["skip"]
    u = v["delta"] + (0.0 if v["delta_bias"] is None else v["delta_bias"])
    start = zero(plan.rows, channels, states) if v["initial"] is None else v["initial"]
    dt, slope = _softplus(u), torch.special.expit(u)
    act, act_slope = (torch.ones_like(x), torch.zeros_like(x)) if v["gate"] is None else _silu(v["gate"])
    a = torch.exp(dt[:, :, None] * decay)
    loss = SLIP * (1 + (dt[:, :, None] * decay).abs())              # of an exponential and what it multiplies
    into = (dt * x)[:, :, None] * b[:, None]
    hs, before, H_before, E_before, H, E = [], [], [], [], [], []
    state, state_slip, h, size, slip = start.clone(), torch.zeros_like(start), None, None, None
    for t, row, begins, ends in _walk(plan):
        if begins:
            h = start[row] if row is not None else zero(channels, states)
            size, slip = h.abs(), torch.zeros_like(h)
        before.append(h), H_before.append(size), E_before.append(slip)
        h = a[t] * h + into[t]
        slip = a[t] * (slip + loss[t] * size) + TINY * size + SLIP * into[t].abs()
        size = a[t] * size + into[t].abs()
        hs.append(h), H.append(size), E.append(slip)
        if ends is not None:
            state[ends], state_slip[ends] = h, slip
    stack = lambda xs: torch.stack(xs) if xs else zero(0, channels, states)
    hs, before, H_before, E_before, H, E = map(stack, (hs, before, H_before, E_before, H, E))
    raw = (hs * c[:, None]).sum(-1) + skip * x
    raw_slip = ((E + SLIP * H) * c.abs()[:, None]).sum(-1) + SLIP * (skip * x).abs()
    out = {"y": (raw * act, act.abs() * raw_slip + SLIP * (raw * act).abs()), "state": (state, state_slip)}
    if dy is None:
        return out
    dy = dy.double()
    d = dy * act
    m, M, EM = (torch.zeros_like(hs) for _ in range(3))
    dinitial, dinitial_slip = torch.zeros_like(start), torch.zeros_like(start)
    back = back_size = back_slip = None
    begun = set()
    for t, row, begins, ends in reversed(_walk(plan)):
        if ends is not None:
            back = zero(channels, states) if dstate is None else dstate[ends].double()
            back_size, back_slip = back.abs(), torch.zeros_like(back)
        own = d[t][:, None] * c[t]
        m[t], M[t], EM[t] = back + own, back_size + own.abs(), back_slip + SLIP * (own.abs() + back_size)
        back, back_size, back_slip = a[t] * m[t], a[t] * M[t], a[t] * (EM[t] + loss[t] * M[t]) + TINY * M[t]
        if begins:
            if row is not None:
                dinitial[row], dinitial_slip[row] = back, back_slip
                begun.add(row)
            back, back_size, back_slip = (torch.zeros_like(back) for _ in range(3))
    for row in set(range(plan.rows)) - begun:
        if dstate is not None:
            dinitial[row] = dstate[row].double()
    through = m * a * before
    through_slip = a * (EM * H_before + M * E_before + loss * M * H_before) + TINY * M * H_before
    through_size = a * M * H_before
    by_b, by_b_slip = (m * b[:, None]).sum(-1), ((EM + SLIP * M) * b.abs()[:, None]).sum(-1)
    ddt = (through * decay).sum(-1) + by_b * x
    ddt_slip = ((through_slip + SLIP * through_size) * decay.abs()).sum(-1) + by_b_slip * x.abs() + SLIP * (by_b * x).abs()
    ddelta, ddelta_slip = ddt * slope, ddt_slip * slope + SLIP * (ddt * slope).abs() + SLIP * (through_size * decay.abs()).sum(-1) * slope
    out.update(
        x=(by_b * dt + skip * d, by_b_slip * dt + SLIP * ((by_b * dt).abs() + (skip * d).abs())), delta=(ddelta, ddelta_slip),
        decay=((through * dt[:, :, None]).sum(0), ((through_slip + CHAIN * through_size) * dt[:, :, None]).sum(0)),
        b=((m * (dt * x)[:, :, None]).sum(1), ((EM + SLIP * M) * (dt * x).abs()[:, :, None]).sum(1)), c=((d[:, :, None] * hs).sum(1), (d.abs()[:, :, None] * (E + SLIP * H)).sum(1)),
        initial=(dinitial, dinitial_slip), skip=((d * x).sum(0), CHAIN * (d * x).abs().sum(0)),
        gate=(dy * raw * act_slope, (dy.abs() * (act_slope.abs() + SLIP) * raw_slip + 4 * SLIP * (dy * raw).abs())),
        delta_bias=(ddelta.sum(0), (ddelta_slip + CHAIN * (ddelta.abs())).sum(0)))
    return out


FLOATS = ("decay", "initial", "skip", "delta_bias", "state")


def _scan_inputs(gen, plan, channels, states, dtype, gate=True, skip=True, delta_bias=True, initial=True, rows=None, shift=-1.0):
    n, rows = (plan.tokens, plan.rows) if plan is not None else (rows, None)
    both, narrow = _normal(gen, n, 2 * channels + 1, dtype=dtype), _normal(gen, n, 2 * states + 3, dtype=dtype)          # views of projections, at odd strides
    v = {"x": both[:, :channels], "delta": _normal(gen, n, channels, dtype=dtype), "decay": -torch.rand((channels, states), generator=gen, device="cuda") * 4, "b": narrow[:, 3:3 + states],
         "c": narrow[:, 3 + states:], "initial": _normal(gen, rows, channels, states) if initial and plan is not None else None, "skip": _normal(gen, channels) if skip else None,
         "gate": both[:, channels + 1:] if gate else None, "delta_bias": _normal(gen, channels, shift=shift) if delta_bias else None}
    return v


def _check_scan(plan, channels, states, dtype, seed=0, dstate=True, **options):
    gen = _gen(seed)
    v = _scan_inputs(gen, plan, channels, states, dtype, **options)
    leaves = {name: None if x is None else x.detach().requires_grad_() for name, x in v.items()}
    y, state = S.selective_scan(episodes=plan, **leaves)
    dy, ds = _normal(gen, *y.shape, dtype=dtype), _normal(gen, *state.shape) if dstate else None
    given = {name: x for name, x in leaves.items() if x is not None}
    grads = torch.autograd.grad([y, state] if dstate else [y], list(given.values()), [dy, ds] if dstate else [dy])
    want = _reference_scan(v, plan, dy, ds)
    for name, got in [("y", y.detach()), ("state", state.detach()), *zip(given, grads)]:
        kind = torch.float32 if name in FLOATS else dtype
        _close(got, *want[name], name, UNIT[kind], STEP[kind])
    plain = S.selective_scan(episodes=plan, **v)                    # without gradients, the same
    assert torch.equal(plain[0], y) and torch.equal(plain[1], state)


@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("plan", list(PLANS))
def test_scan_and_its_gradients(dtype, plan):
    _check_scan(PLANS[plan](), 40, 16, dtype)


@pytest.mark.parametrize("states", [1, 4, 5, 8, 12, 16, 20, 32, 33, 64])
@pytest.mark.parametrize("channels", [1, 7, 32, 129])
def test_scan_sizes(states, channels):
    for dtype in (torch.float32, torch.bfloat16):
        _check_scan(_done_plan(6, 30, 0.1), channels, states, dtype, seed=channels + states)


@pytest.mark.parametrize("states", [6, 16, 24, 48])
def test_scan_of_long_rows(states):
    """Rows that are cut into segments, walked twice; episodes that begin at segments' edges and rows that end inside."""
    _check_scan(_plan_of([700, 64, 0, 320, 1]), 9, states, torch.float32, seed=states)
    _check_scan(_done_plan(2, 500, 0.004), 33, states, torch.bfloat16, seed=states)


@pytest.mark.parametrize("change", [dict(gate=False), dict(skip=False), dict(delta_bias=False), dict(initial=False), dict(dstate=False), dict(gate=False, skip=False, delta_bias=False, initial=False, dstate=False),
                                    dict(shift=-6.0), dict(shift=30.0)])
def test_scan_options(change):
    _check_scan(_plan_of([2, 0, 70, 1]), 24, 16, torch.bfloat16, **change)
    _check_scan(_plan_of([200]), 24, 8, torch.float32, **change)


@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("channels,states", [(5, 3), (32, 16), (70, 20), (9, 64)])
def test_scan_steps_are_the_scan(dtype, channels, states):
    """Token after token of every env, with episodes that begin on the way, within both forms' bounds."""
    envs, steps = 11, 9
    gen = _gen(states)
    done = torch.rand((envs, steps), generator=gen, device="cuda") < 0.3
    plan = S.Episodes.from_done(done)
    v = _scan_inputs(gen, plan, channels, states, dtype)
    want = _reference_scan(v, plan, None, None)
    state, fresh = v["initial"].clone(), None
    for t in range(steps):
        at = torch.arange(envs, device="cuda") * steps + t
        token = {name: x[at] if name in ("x", "delta", "b", "c", "gate") else x for name, x in v.items() if name != "initial"}
        y = S.selective_scan_step(state=state, fresh=fresh, **token)
        _close(y, want["y"][0][at], want["y"][1][at], f"y {t}", UNIT[dtype], STEP[dtype])
        fresh = done[:, t]
    _close(state, *want["state"], "state", UNIT[torch.float32])


def test_gradients_against_differences():
    """Along a direction of all inputs at once: what the gradients give, and the difference of the definition's two values in 64 bits (off by 1e-8 of itself at this step)."""
    plan, gen = _plan_of([37, 3, 0, 90]), _gen(5)
    v = {name: x.detach() for name, x in _scan_inputs(gen, plan, 10, 7, torch.float32).items()}
    leaves = {name: x.requires_grad_() for name, x in v.items()}
    y, state = S.selective_scan(episodes=plan, **leaves)
    dy, ds = _normal(gen, *y.shape), _normal(gen, *state.shape)
    grads = dict(zip(leaves, torch.autograd.grad([y, state], list(leaves.values()), [dy, ds])))
    way = {name: _normal(gen, *x.shape).double() * 0.1 for name, x in v.items()}
    value = lambda by: sum((f.double() * w[0]).sum() for f, w in zip((dy, ds), (lambda o: (o["y"], o["state"]))(_reference_scan({n: x.detach().double() + by * way[n] for n, x in v.items()}, plan, None, None))))
    step = 1e-4
    want = ((value(step) - value(-step)) / (2 * step)).item()
    got = sum((grads[n].double() * way[n]).sum() for n in grads).item()
    bounds = _reference_scan(v, plan, dy, ds)
    slack = sum(((bounds[n][1] + UNIT[torch.float32] * bounds[n][0].abs()) * way[n].abs()).sum() for n in grads).item()
    assert abs(got - want) <= slack + 1e-6 * (1 + abs(want))
    x, weight, bias, first = _normal(gen, plan.tokens, 6), _normal(gen, 6, 4), _normal(gen, 6), _normal(gen, plan.rows, 3, 6)
    leaves = [t.requires_grad_() for t in (x, weight, bias, first)]
    y, state = S.short_convolution(leaves[0], leaves[1], leaves[2], plan, leaves[3], silu=True)
    dy, ds = _normal(gen, *y.shape), _normal(gen, *state.shape)
    grads = torch.autograd.grad([y, state], leaves, [dy, ds])
    way = [_normal(gen, *t.shape).double() * 0.1 for t in leaves]
    value = lambda by: (lambda o: (o["y"][0] * dy).sum() + (o["state"][0] * ds).sum())(_reference_convolution(*(t.detach().double() + by * w for t, w in zip(leaves, way)), plan, True, dy, None))
    want = ((value(step) - value(-step)) / (2 * step)).item()
    got = sum((g.double() * w).sum() for g, w in zip(grads, way)).item()
    bounds = _reference_convolution(x, weight, bias, first, plan, True, dy, ds)
    slack = sum(((bounds[n][1] + UNIT[torch.float32] * bounds[n][0].abs()) * w.abs()).sum() for n, w in zip(("x", "weight", "bias", "initial"), way)).item()
    assert abs(got - want) <= slack + 1e-6 * (1 + abs(want))


# ---- what programs do around a call ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(UNIT))
def test_sums_and_gates_of_any_size(dtype):
    """s / (1 + exp(-s)) and its slope where the exponential ends at infinity or 0: the slope's and the value's own size is then that of TINY or of s, 1 or 0, times products of at most one such factor."""
    top = float(torch.finfo(dtype).max)
    s = torch.tensor([-top, -top / 4, -top / 64, -1000.0, -200.0, -100.0, -20.0, 0.0, 20.0, 100.0, 1000.0, top / 64, top / 4], device="cuda").to(dtype)[:, None].expand(-1, 8).contiguous().requires_grad_()
    plan, tokens = _plan_of([s.shape[0]]), s.shape[0]
    dy = _normal(_gen(1), tokens, 8, dtype=dtype)
    value, slope = _silu(s.detach().double())
    unit = UNIT[dtype] + SLIP
    weight = torch.tensor([0.0, 1.0], device="cuda").expand(8, 2).contiguous()
    y, _ = S.short_convolution(s, weight, None, plan, silu=True)
    dx, = torch.autograd.grad(y, s, dy)
    _close(y.detach(), value, 64 * TINY, "y", unit, STEP[dtype])
    _close(dx, dy.double() * slope, 64 * TINY + SLIP * dy.double().abs(), "dx", unit, STEP[dtype])
    # states of nothing, so that y = x / 2 silu(gate)
    x, none = torch.ones(tokens, 8, device="cuda", dtype=dtype, requires_grad=True), torch.zeros(tokens, 4, device="cuda", dtype=dtype)
    y, _ = S.selective_scan(x, torch.zeros_like(x), -torch.ones(8, 4, device="cuda"), none, none, plan, skip=torch.full((8,), 0.5, device="cuda"), gate=s)
    _close(y.detach(), value / 2, 64 * TINY, "scan's y", unit, STEP[dtype])
    small = s.detach().double() <= 1000
    dx, dgate = torch.autograd.grad(y, (x, s), dy * small.to(dtype))            # of x's gradient only what fits the type
    _close(dx, dy.double() * small * value / 2, 64 * TINY, "scan's dx", unit, STEP[dtype])
    _close(dgate, dy.double() * small * slope / 2, 64 * TINY + SLIP * dy.double().abs(), "dgate", unit, STEP[dtype])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_not_finite_stays_in_its_episode(bad):
    """A value of one episode's input: outputs, states and gradients of the other episodes keep their bits."""
    plan = _plan_of([150, 40, 300, 9])
    other = torch.ones(plan.tokens, dtype=torch.bool, device="cuda")
    other[150:190] = False
    rows = torch.tensor([0, 2, 3], device="cuda")

    def run(v, name, spoil, call):
        v = {n: x.clone() for n, x in v.items()}
        if spoil:
            v[name][170] = bad
        leaves = {n: x.requires_grad_() for n, x in v.items()}
        y, state = call(leaves)
        dy = torch.ones_like(y)
        per_token = [n for n in leaves if leaves[n].shape[0] == plan.tokens]
        grads = torch.autograd.grad(y, [leaves[n] for n in per_token], dy)
        return [y[other], state[rows], *(g[other] for g in grads)]

    v = _scan_inputs(_gen(6), plan, 20, 16, torch.float32)
    for name in ("x", "delta", "b", "c", "gate"):
        for a, b in zip(run(v, name, False, lambda l: S.selective_scan(episodes=plan, **l)), run(v, name, True, lambda l: S.selective_scan(episodes=plan, **l))):
            assert torch.equal(a, b), name
    weight, bias = _normal(_gen(7), 20, 4), _normal(_gen(8), 20)
    call = lambda l: S.short_convolution(l["x"], weight, bias, plan, l["initial"], silu=True)
    v = {"x": _normal(_gen(9), plan.tokens, 20), "initial": _normal(_gen(10), 4, 3, 20)}
    for a, b in zip(run(v, "x", False, call), run(v, "x", True, call)):
        assert torch.equal(a, b)


def _layer(v, weight, plan, first):
    y, tail = S.short_convolution(v["x"], weight, None, plan, first, silu=True)
    return S.selective_scan(y, *(v[n] for n in ("delta", "decay", "b", "c")), plan, v["initial"], v["skip"], v["gate"], v["delta_bias"]), tail


def test_the_same_call_gives_the_same_bits_in_graphs_and_on_other_streams():
    plan, gen = _plan_of([600, 0, 100, 3]), _gen(11)
    v = {n: x.detach().requires_grad_() for n, x in _scan_inputs(gen, plan, 48, 16, torch.bfloat16).items()}
    weight, first = _normal(gen, 48, 4).requires_grad_(), _normal(gen, 4, 3, 48, dtype=torch.bfloat16).requires_grad_()
    leaves = [*v.values(), weight, first]

    def run():
        (y, state), tail = _layer(v, weight, plan, first)
        return [y, state, tail, *torch.autograd.grad([y, state], leaves, [torch.ones_like(y), torch.ones_like(state)])]

    want = [x.detach().clone() for x in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(2):
        for x in out:
            x.detach().fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_checkpointing_and_unused_outputs():
    from torch.utils.checkpoint import checkpoint
    plan, gen = _plan_of([130, 60]), _gen(12)
    v = {n: x.detach().requires_grad_() for n, x in _scan_inputs(gen, plan, 33, 9, torch.float32).items()}
    call = lambda *xs: S.selective_scan(episodes=plan, **dict(zip(v, xs)))
    y, state = call(*v.values())
    want = torch.autograd.grad(y.sum() + state.sum(), list(v.values()))
    y, state = checkpoint(call, *v.values(), use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y.sum() + state.sum(), list(v.values())), want))
    _, state = call(*v.values())                                    # only the state is asked for
    got = dict(zip(v, torch.autograd.grad(state.sum(), [v[n] for n in v])))
    bounds = _reference_scan(v, plan, torch.zeros_like(y), torch.ones_like(state))
    for name, g in got.items():
        _close(g, *bounds[name], name, UNIT[torch.float32])
    few = S.selective_scan(v["x"].detach(), v["delta"], v["decay"].detach(), v["b"].detach(), v["c"].detach(), plan)[0]       # one leaf only
    assert torch.isfinite(torch.autograd.grad(few.sum(), v["delta"])[0]).all()


def test_refusals():
    plan = _plan_of([5, 3])
    v = _scan_inputs(_gen(13), plan, 8, 4, torch.bfloat16)
    good = lambda **change: S.selective_scan(episodes=plan, **{**v, **change})
    good()
    for change in (dict(x=v["x"][:4]), dict(x=v["x"].double()), dict(delta=v["delta"].float()), dict(delta=v["delta"][:, :4]), dict(b=v["b"][:, :3]), dict(c=v["c"].float()), dict(decay=v["decay"].bfloat16()),
                   dict(decay=v["decay"][:4]), dict(decay=torch.zeros(8, 65, device="cuda")), dict(decay=torch.zeros(8, 0, device="cuda")), dict(skip=v["skip"][:3]), dict(skip=v["skip"].half()),
                   dict(gate=v["gate"].float()), dict(delta_bias=v["delta_bias"].double()), dict(initial=v["initial"][:1]), dict(initial=v["initial"].half()), dict(x=v["x"].cpu())):
        with pytest.raises(ValueError):
            good(**change)
    x, weight = v["x"], _normal(_gen(14), 8, 4)
    for args in ((x, weight[:, :1], None, plan), (x, torch.zeros(8, 5, device="cuda"), None, plan), (x, weight[:4], None, plan), (x, weight.half(), None, plan), (x, weight, torch.zeros(7, device="cuda"), plan),
                 (x, weight, None, plan, torch.zeros(2, 3, 8, device="cuda")), (x, weight, None, plan, torch.zeros(2, 2, 8, dtype=torch.bfloat16, device="cuda")), (x[:3], weight, None, plan)):
        with pytest.raises(ValueError):
            S.short_convolution(*args)
    state = torch.zeros(8, 8, 3, dtype=torch.bfloat16, device="cuda")
    for args in ((x, weight, None, state.transpose(1, 2)), (x, weight, None, torch.zeros(8, 3, 8, device="cuda")), (x, weight, None, torch.zeros(7, 3, 8, dtype=torch.bfloat16, device="cuda"))):
        with pytest.raises(ValueError):
            S.short_convolution_step(*args)
    with pytest.raises(ValueError):
        S.selective_scan_step(v["x"], v["delta"], v["decay"], v["b"], v["c"], torch.zeros(8, 4, 8, device="cuda").transpose(1, 2))
    with pytest.raises(ValueError):
        S.selective_scan_step(v["x"], v["delta"], v["decay"], v["b"], v["c"], torch.zeros(8, 8, 4, device="cuda"), fresh=torch.zeros(8, device="cuda"))
    y, _ = S.selective_scan(episodes=plan, **{**v, "x": v["x"].clone().requires_grad_()})
    with pytest.raises(RuntimeError):                               # gradients of gradients
        torch.autograd.grad(torch.autograd.grad(y.float().sum(), _leaf(y), create_graph=True)[0].sum(), _leaf(y))


def _leaf(y):
    node = y.grad_fn
    while True:
        for after, _ in node.next_functions:
            if after is not None and hasattr(after, "variable"):
                return after.variable
        node = next(after for after, _ in node.next_functions if after is not None)


def test_offsets_that_lie_stay_inside_the_tensors():
    """The plan is clamped on the device, so are the operators' reads: values of a wrong plan, and memory around the tensors as it was."""
    for offsets in ([0, 50, 20, 10], [-5, 3, 1000, 7], [90, 95, 99, 2 ** 31 - 1]):
        plan = S.Episodes.from_offsets(torch.tensor(offsets, dtype=torch.int32, device="cuda"), 40)
        v = _scan_inputs(_gen(15), plan, 8, 4, torch.float32)
        leaves = {n: x.detach().requires_grad_() for n, x in v.items()}
        y, state = S.selective_scan(episodes=plan, **leaves)
        torch.autograd.grad(y.sum(), list(leaves.values()))
        x = v["x"].detach().clone().requires_grad_()
        y, state = S.short_convolution(x, _normal(_gen(16), 8, 4), None, plan, _normal(_gen(17), 3, 3, 8), silu=True)
        torch.autograd.grad(y.sum(), x)
    torch.cuda.synchronize()


def test_more_values_than_32_bits_count():
    """Tensors of more than 2^31 values: the last rows of a batch, and their gradients, are what they are in a batch of their own, bit for bit (rows of one short length are worked out alike)."""
    rows, length, channels, states, few = 34000, 32, 2048, 4, 3
    assert rows * length * channels > 2 ** 31
    gen, dtype = _gen(20), torch.bfloat16
    cut = slice((rows - few) * length, None)

    def make(n):
        return torch.empty(rows * length, n, dtype=dtype, device="cuda")

    x, delta = make(channels), make(channels)
    b, c = (_normal(gen, rows * length, states, dtype=dtype) for _ in range(2))
    decay, taps = -torch.rand((channels, states), generator=gen, device="cuda"), _normal(gen, channels, 4)
    x.zero_(), delta.zero_()
    x[cut], delta[cut] = _normal(gen, few * length, channels, dtype=dtype), _normal(gen, few * length, channels, dtype=dtype)
    done = torch.rand((rows, length), generator=gen, device="cuda") < 0.05
    whole, part = S.Episodes.from_done(done), S.Episodes.from_done(done[-few:].contiguous())

    def run(plan, x, delta, b, c, at):
        x, delta, b, c = (v.detach().requires_grad_() for v in (x, delta, b, c))
        y, state = S.selective_scan(x, delta, decay, b, c, plan)
        dy = torch.zeros_like(y)
        dy[at] = 1.0
        out = [y[at], state[-few:], *(g[at] for g in torch.autograd.grad(y, [x, delta, b, c], dy))]
        out = [v.detach().clone() for v in out]
        del y, dy
        y, state = S.short_convolution(x, taps, None, plan, silu=True)
        dy = torch.zeros_like(y)
        dy[at] = 1.0
        return out + [y[at].detach().clone(), state[-few:].detach(), torch.autograd.grad(y, x, dy)[0][at].clone()]

    want = run(part, x[cut].clone(), delta[cut].clone(), b[cut].clone(), c[cut].clone(), slice(None))
    got = run(whole, x, delta, b, c, cut)
    del x, delta
    torch.cuda.empty_cache()
    for n, (a, w) in enumerate(zip(got, want)):
        assert torch.isfinite(a).all() and a.abs().sum() > 0 and torch.equal(a, w), n
