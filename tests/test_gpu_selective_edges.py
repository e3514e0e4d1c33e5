"""Calls of the selective operators at the ends of what they take: no channels, sums over many tokens, and a policy whose layers are worked out in 16 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import nuka  # noqa: E402,F401
from nuka import memory_policy as M, sequence as S  # noqa: E402
from test_gpu_selective import _check_scan, _done_plan  # noqa: E402

pytestmark = pytest.mark.gpu

SLIP = 2.0 ** -20                       # of what the few roundings of a formula in 32 bits come to, an exponential's (and its argument's) among them


def _rows_of(*lengths):
    ends = torch.tensor([0, *lengths]).cumsum(0)
    return S.Episodes.from_offsets(ends.to(torch.int32).cuda(), int(ends[-1]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths", [(37, 0, 5), (700,), (0, 0)])
def test_a_scan_without_channels(dtype, lengths):
    """Gradients of B and C are sums over no channel, whatever the memory held that they come in."""
    plan, states = _rows_of(*lengths), 9
    leaf = lambda *shape, dtype=dtype: torch.ones(shape, dtype=dtype, device="cuda", requires_grad=True)
    tokens = plan.tokens
    x, delta, gate, b, c = leaf(tokens, 0), leaf(tokens, 0), leaf(tokens, 0), leaf(tokens, states), leaf(tokens, states)
    decay, skip, bias, first = leaf(0, states, dtype=torch.float32), *(leaf(0, dtype=torch.float32) for _ in range(2)), leaf(plan.rows, 0, states, dtype=torch.float32)
    y, state = S.selective_scan(x, delta, decay, b, c, plan, first, skip, gate, bias)
    assert y.shape == (tokens, 0) and state.shape == (plan.rows, 0, states)
    dirty = [torch.full((tokens, states), 7.25, dtype=dtype, device="cuda") for _ in range(64)]
    torch.cuda.synchronize()
    del dirty
    leaves = [x, delta, decay, b, c, first, skip, gate, bias]
    for leaf, grad in zip(leaves, torch.autograd.grad([y, state], leaves, [torch.ones_like(y), torch.ones_like(state)])):
        assert grad.shape == leaf.shape and not grad.any()


def _sums_of_equal_tokens(rows, length, states, dt, slope, decay, gate):
    """{name: (value, bound)} of a channel's sums over all tokens, where x, b, c and dy are 1 in all of them: the terms' own error by the recurrences that the states follow."""
    a, loss = np.exp(dt * decay), SLIP * (1 + dt * np.abs(decay))
    h, E = np.zeros(states), np.zeros(states)
    before, slips = np.zeros((length, states)), np.zeros((length, states))
    for t in range(length):
        before[t], slips[t] = h, E
        h, E = a * h + dt, a * (E + loss * h) + SLIP * dt
    back, EB = np.zeros(states), np.zeros(states)
    ddecay, ddecay_slip, dbias, dbias_slip = np.zeros(states), np.zeros(states), 0.0, 0.0
    for t in range(length - 1, -1, -1):
        m, EM = back + gate, EB + SLIP * (back + gate)
        through, slip = m * a * before[t], a * (EM * before[t] + m * slips[t] + loss * m * before[t])
        ddecay += through * dt
        ddecay_slip += slip * dt + SLIP * through * dt
        dbias += (np.sum(through * decay) + np.sum(m)) * slope
        dbias_slip += (np.sum((slip + SLIP * through) * np.abs(decay)) + np.sum(EM + SLIP * m) + SLIP * abs(np.sum(through * decay) + np.sum(m))) * slope
        back, EB = a * m, a * (EM + loss * m)
    return {"decay": (rows * ddecay, rows * ddecay_slip), "delta_bias": (rows * dbias, rows * dbias_slip), "skip": (rows * length * gate, SLIP * rows * length * gate)}


@pytest.mark.parametrize("dtype,rows,length,channels,states", [(torch.bfloat16, 1, 16381, 4744, 64), (torch.bfloat16, 4, 4100, 4744, 64), (torch.float16, 1, 4200, 18960, 32), (torch.bfloat16, 1, 4200, 37920, 16),
                                                               (torch.float32, 3, 1400, 37920, 12), (torch.bfloat16, 1, 4200, 75904, 8)])
def test_weights_gradients_of_many_tokens(dtype, rows, length, channels, states):
    """So many channels that one warp has all tokens of its own.  Sums of n terms of one sign, one by one, are off by up to n 2^-24 of themselves: n is the 1024 terms of a warp's registers, as many parts as these make of
    all tokens, and the 32 of the last sum, and not all the tokens (of 16381, the gradients of decays were off by 2^-12.1)."""
    tokens = rows * length
    plan = S.Episodes.from_done(torch.zeros(rows, length, dtype=torch.bool, device="cuda")) if rows > 1 else _rows_of(length)
    full = lambda value, *shape: torch.full(shape, value, dtype=dtype, device="cuda")
    decay = torch.linspace(-0.3, -1.7, states, device="cuda").expand(channels, states).contiguous().requires_grad_()
    skip, bias = (torch.zeros(channels, device="cuda", requires_grad=True) for _ in range(2))
    x, delta, gate = full(1.0, tokens, channels), full(0.5, tokens, channels), full(0.7, tokens, channels)
    y, _ = S.selective_scan(x, delta, decay, full(1.0, tokens, states), full(1.0, tokens, states), plan, skip=skip, gate=gate, delta_bias=bias)
    got = dict(zip(("decay", "skip", "delta_bias"), torch.autograd.grad(y, [decay, skip, bias], torch.ones_like(y))))
    z, u = gate[0, 0].item(), 0.5
    want = _sums_of_equal_tokens(rows, length, states, np.log1p(np.exp(u)), 1 / (1 + np.exp(-u)), decay[0].detach().double().cpu().numpy(), z / (1 + np.exp(-z)))
    chain = (1024 + -(-tokens // 1024) + 32) * 2.0 ** -24
    for name, grad in got.items():
        value, bound = (torch.as_tensor(v, dtype=torch.float64, device="cuda") for v in want[name])
        off = (grad.double() - value).abs() - bound - chain * value.abs()       # of every channel
        assert off.max().item() <= 0, f"{name}: off by {((grad.double() - value).abs() / value.abs()).max().item():.3e} of itself"


def test_the_convolutions_weights_gradients_of_many_tokens():
    """So many channels that four warps have all tokens.  n terms of one sign, one by one: 1024 tokens of a warp and a walk of 128 at most more, the block's four warps, the blocks."""
    tokens, channels, width = 65536, 28420, 4
    plan = _rows_of(tokens)
    x, weight, bias = torch.ones(tokens, channels, dtype=torch.bfloat16, device="cuda"), torch.zeros(channels, width, device="cuda", requires_grad=True), torch.linspace(-2.0, 2.0, channels, device="cuda", requires_grad=True)
    y, _ = S.short_convolution(x, weight, bias, plan, silu=True)
    dw, db = torch.autograd.grad(y, [weight, bias], torch.ones_like(y))
    s = bias.detach().double()
    r = torch.special.expit(s)
    ds = r * (1 + s * (1 - r))
    loss = SLIP * r * (1 + s.abs() * (1 + s.abs())) + (1024 + 128 + 4 + 64) * 2.0 ** -24 * ds.abs()
    for got, count in [(db, tokens), *((dw[:, j], tokens - width + 1 + j) for j in range(width))]:          # inputs before the episode are 0
        off = (got.double() - ds * count).abs() - loss * count
        assert off.max().item() <= 0, f"off by {((got.double() - ds * count).abs() / (ds * count).abs()).max().item():.3e}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("states", [0, 16])
def test_a_policy_under_autocast(dtype, states):
    """Both kinds of layer, over two rollouts: acting and training are one policy, and it has gradients.  A layer has eight results that are rounded to 16 bits (inputs, taps, rates, scan, products, scores, attention,
    its product) and there are two: where both forms' values of about 1 fall on different sides each time, actions are 16 x 2^-8 apart."""
    torch.manual_seed(states)
    envs, steps = 5, 11
    policy = M.MemoryPolicy(12, 3, width=128, heads=4, kv_heads=2, history=16, states=states, sinks=2).cuda()
    memory, fresh = M.Memory(policy, envs, "cuda"), None
    with torch.autocast("cuda", dtype=dtype):
        for _ in range(2):
            obs, done = torch.randn(envs, steps, 12, device="cuda"), torch.rand(envs, steps, device="cuda") < 0.2
            first = [s if fresh is None else s.masked_fill(fresh.view(-1, *[1] * (s.dim() - 1)), 0.0) for s in memory.begin_rollout()]
            acted = []
            for t in range(steps):
                acted.append(policy.act(obs[:, t], memory, fresh)[0].float())
                fresh = done[:, t]
            mean, value = policy(obs, done, first)
            assert mean.dtype == dtype and all(s.dtype == torch.float32 for s in memory.states)
            assert (torch.stack(acted, 1) - mean.float()).abs().max().item() <= 16 * 2.0 ** -8 * max(1.0, mean.abs().max().item())
    (mean.float().square().sum() + value.float().sum()).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in policy.parameters() if p is not policy.log_std)


def test_histories_begin_anew_with_a_rollout():
    """First control steps that stay are those of the rollout's part of an episode: of a rollout before only the states go on."""
    torch.manual_seed(1)
    policy = M.MemoryPolicy(12, 3, width=64, heads=2, kv_heads=1, history=8, states=4, sinks=3).cuda()
    obs, outs = torch.randn(4, 20, 12, device="cuda"), []
    for before in (0, 5, 13):
        memory = M.Memory(policy, 4, "cuda")
        for t in range(before):
            policy.act(-obs[:, t], memory)
        memory.begin_rollout()
        for state in memory.states:
            state.zero_()
        outs.append(torch.stack([policy.act(obs[:, t], memory)[0] for t in range(20)]))
    assert torch.equal(outs[1], outs[0]) and torch.equal(outs[2], outs[0])


@pytest.mark.parametrize("size", [2.0, 16.0, 60.0, 80.0])
@pytest.mark.parametrize("states", [8, 16, 64])
def test_exponentials_of_large_arguments(size, states):
    """What a state of 1 fades to, forwards, as a gradient and in a step.  The argument is a product of three factors, dt, decay and log2(e), the last off by 2^-26 of itself, two products rounded by 2^-24 each: 2.3 x 2^-24 of it
    in all, and dt itself, above 20, by half a unit; the exponential is off by as much as its argument, and by the instruction's own 2^-22: below 2^-22 (1 + |dt decay|)."""
    channels, dt = 512, 24.0
    decay = -torch.linspace(size / 16, size, channels * states, device="cuda").view(channels, states) / dt
    plan, none, narrow = _rows_of(1), torch.zeros(1, channels, device="cuda"), torch.zeros(1, states, device="cuda")
    first = torch.ones(1, channels, states, device="cuda", requires_grad=True)
    _, state = S.selective_scan(none, none + dt, decay, narrow, narrow, plan, first)
    back, = torch.autograd.grad(state, first, torch.ones_like(state))
    stepped = torch.ones(1, channels, states, device="cuda")
    S.selective_scan_step(none, none + dt, decay, narrow, narrow, stepped)
    argument = decay.double() * np.logaddexp(dt, 0.0)
    want = argument.exp()
    for what, got in (("state", state.detach()), ("gradient", back), ("step", stepped)):
        off = (got[0].double() - want).abs() / want - 2.0 ** -22 * (1 + argument.abs())
        assert off.max().item() <= 0, what


@pytest.mark.parametrize("length", [1, 2, 3, 5, 7])
@pytest.mark.parametrize("states", [5, 16, 33])
def test_rows_of_less_than_a_chunk(length, states):
    """Several rows to a walk: each begins with its own initial state, and leaves its own."""
    for rows, dtype in ((41, torch.bfloat16), (1, torch.float32), (23, torch.float16)):
        _check_scan(_done_plan(rows, length, 0.2, seed=length), 37, states, dtype, seed=length)
