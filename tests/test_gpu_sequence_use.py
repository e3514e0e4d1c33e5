"""Sequence operators as programs use them around the plain call: checkpointing, saved-tensor hooks, graphs, streams, inputs at the edge of what is finite."""
import pytest

torch = pytest.importorskip("torch")
import nuka  # noqa: E402,F401
from nuka import sequence as S  # noqa: E402

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return torch.empty(shape, device="cuda").normal_(shift, scale, generator=gen).to(dtype)


def _plan_of(lengths):
    offsets = torch.tensor([0, *lengths], dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)
    return S.Episodes.from_offsets(offsets, sum(lengths))


# ---- what is saved for the backward pass -------------------------------------------------------------------------------
def _operators():
    gen, plan = _gen(1), _plan_of([300, 1, 77, 122])
    f, w = S.rotary_frequencies(64).cuda(), _normal(gen, 64, shift=1.0, scale=0.2)
    both = _normal(gen, 500, 8 * 64, dtype=torch.bfloat16)
    cut = lambda x, low, n: x[:, low * 64:(low + n) * 64].unflatten(1, (n, 64))
    x, g, i = _normal(gen, 500, 96), _normal(gen, 500, 96), _normal(gen, 4, 96)
    return {"recurrence": (lambda x, g, i: S.gated_recurrence(x * 1.5, g * 1.5, plan, i * 1.5), [x, g, i]),
            "heads": (lambda y, w: S.rotate_heads(cut(y * 1.5, 0, 4), cut(y * 1.5, 4, 2), w * 1.5, w * 0.5, plan, f), [both, w]),
            "attention": (lambda y: [S.episode_attention(cut(y * 1.5, 0, 4), cut(y * 1.5, 4, 2), cut(y * 1.5, 6, 2), plan)], [both])}


def _grads(run, leaves):
    leaves = [x.detach().clone().requires_grad_() for x in leaves]
    out = run(*leaves)
    # what was freed since the forward pass is written over, as a program's other layers would
    junk = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(8)] + [torch.full((500, n), float("nan"), dtype=torch.bfloat16, device="cuda") for n in (512, 256, 128) * 4]
    cot = [torch.cos(torch.arange(o.numel(), device="cuda")).view(o.shape).to(o.dtype) for o in out]
    grads = torch.autograd.grad(out, leaves, cot)
    del junk
    return grads


@pytest.mark.parametrize("operator", ["recurrence", "heads", "attention"])
@pytest.mark.parametrize("way", ["checkpoint", "on the CPU", "copies"])
def test_gradients_under_checkpointing_and_hooks(operator, way):
    """Bit for bit what they are without: the backward pass reads what saved tensors return, wherever they are by then."""
    run, leaves = _operators()[operator]
    want = _grads(run, leaves)
    if way == "checkpoint":
        from torch.utils.checkpoint import checkpoint
        got = _grads(lambda *a: checkpoint(run, *a, use_reentrant=False), leaves)
    else:
        with torch.autograd.graph.save_on_cpu() if way == "on the CPU" else torch.autograd.graph.saved_tensors_hooks(lambda x: x.clone(), lambda x: x.clone()):
            got = _grads(run, leaves)
    assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(want, got))


# ---- norms of heads with little or nothing added to the mean square -----------------------------------------------------
def _normed_64(x, w, eps):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,dim", [(1, 64), (17, 64), (33, 64), (5, 200), (7, 40)])
def test_heads_without_eps(dtype, tokens, dim):
    """Tokens that do not fill a block's last pass: lanes without a token add nothing to the weights' gradients.  Bounds: a few units in the last place of 32 bits before the one rounding,
    for the weights times the square root of the number of terms."""
    gen = _gen(tokens)
    positions = torch.zeros(tokens, dtype=torch.int32, device="cuda")
    q, k = (_normal(gen, tokens, n, dim, dtype=dtype).requires_grad_() for n in (3, 1))
    w = _normal(gen, dim, shift=1.0, scale=0.2).requires_grad_()
    out = S.rotate_heads(q, k, w, w, positions, None, eps=0.0)
    cot = [_normal(gen, *o.shape, dtype=dtype) for o in out]
    dq, dk, dw = torch.autograd.grad(out, [q, k, w], cot)
    leaves = [x.detach().double().requires_grad_() for x in (q, k, w)]
    want = torch.autograd.grad([_normed_64(leaves[0], leaves[2], 0.0), _normed_64(leaves[1], leaves[2], 0.0)], leaves, [c.double() for c in cot])
    unit, ulps = (2.0 ** -8 if dtype is torch.bfloat16 else 2.0 ** -23), 16 * 2.0 ** -23
    for got, x in ((dq, want[0]), (dk, want[1])):
        assert ((got.double() - x).abs() <= unit * x.abs() + ulps * x.abs().max()).all()
    assert ((dw.double() - want[2]).abs() <= ulps * (4 * tokens) ** 0.5 * max(c.double().abs().max().item() for c in cot) * 4).all()


def test_heads_of_tiny_values_and_tiny_eps():
    """A row of zeros and rows whose squares are far below 1: the cube of one over the root is beyond 32 bits, the gradient is not."""
    positions = torch.zeros(3, dtype=torch.int32, device="cuda")
    gen = _gen(2)
    q = _normal(gen, 3, 2, 64) * torch.tensor([0.0, 1e-15, 1e-14], device="cuda")[:, None, None]
    q.requires_grad_()
    out = S.rotate_heads(q, q, None, None, positions, None, eps=1e-30)
    cot = _normal(gen, 3, 2, 64)
    dq, = torch.autograd.grad(out[0], q, cot)
    x = q.detach().double().requires_grad_()
    want, = torch.autograd.grad(_normed_64(x, 1.0, 1e-30), x, cot.double())
    # row by row, whose gradients are of very different sizes; the eps itself is 2^-24 off in 32 bits
    off, size = (dq.double() - want).abs().amax(-1), want.abs().amax(-1)
    assert torch.isfinite(dq).all() and (off <= 16 * 2.0 ** -23 * size).all()


# ---- attention next to what is not finite --------------------------------------------------------------------------------
import math  # noqa: E402

import test_gpu_attention as A  # noqa: E402


@pytest.mark.parametrize("dim,heads_q,heads_k", [(64, 2, 1), (128, 2, 2), (64, 8, 1), (128, 8, 1), (40, 4, 4)])
@pytest.mark.parametrize("what", ["q", "k", "v", "do"])
@pytest.mark.parametrize("value", [math.nan, -math.inf])
def test_neighbours_of_a_spoilt_episode(dim, heads_q, heads_k, what, value):
    """A whole episode spoilt, in every head and in one column: the others of its tiles are what they are without it, with heads of a group in one block and dealt out over a cluster's."""
    plan = A._plan_of([30, 40, 200, 24, 90])
    names = ("q", "k", "v", "do")
    clean = dict(zip(names, (x.clone() for x in A._inputs(_gen(dim + heads_q), plan.tokens, heads_q, heads_k, dim, torch.bfloat16))))
    spoilt = {n: x.clone() for n, x in clean.items()}
    spoilt[what][70:270, :, 3] = value
    A.UNIT_OF[:] = [A.UNIT[torch.bfloat16] * 2.0 ** 7, A.UNIT[torch.bfloat16]]
    w = A._reference(*(clean[n] for n in names[:3]), plan, dim ** -0.5, None, clean["do"])
    q, k, v = (spoilt[n].requires_grad_() for n in names[:3])
    o = S.episode_attention(q, k, v, plan)
    outs = [o.detach(), *torch.autograd.grad(o, [q, k, v], spoilt["do"])]
    other = torch.ones(plan.tokens, dtype=torch.bool, device="cuda")
    other[70:270] = False
    for (name, (want, bound)), got in zip(A._bounds(w, A.UNIT[torch.bfloat16], 0.0).items(), outs):
        A._close(got[other], want[other], bound[other], name)
    # of the spoilt episode what does not meet the spoilt column is what its definition gives, too
    if what == "v" and dim == 64:
        columns = [c for c in range(dim) if c != 3]
        want, bound = A._bounds(w, A.UNIT[torch.bfloat16], 0.0)["o"]
        A._close(outs[0][..., columns], want[..., columns], bound[..., columns], "o")
        assert not torch.isfinite(outs[0][70:270, :, 3]).any()
    if what == "do" and dim == 64:
        columns = [c for c in range(dim) if c != 3]
        want, bound = A._bounds(w, A.UNIT[torch.bfloat16], 0.0)["dv"]
        A._close(outs[3][..., columns], want[..., columns], bound[..., columns], "dv")
        assert not torch.isfinite(outs[1][70:270]).any() and not torch.isfinite(outs[2][70:270]).any()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("what", ["k", "v", "do"])
def test_long_episodes_beside_a_long_spoilt_one(dim, what):
    """30000 finite tokens share tiles with 20000 spoilt ones, which 700 finite ones follow.  The last rows of the first, whose tiles are mixed, against 64 bits, all others bit for bit
    against the call without what is spoilt; no block gives up meanwhile.  Keys' gradients take D from the outputs of the mixed rows, which have other roundings where values are
    spoilt: twice the outputs' bound, in D and in dS's rounding, and one rounding more."""
    lengths, hq, hk = [30000, 20000, 700], 4, 2
    plan = A._plan_of(lengths)
    q, k, v, do = (x.clone() for x in A._inputs(_gen(dim), plan.tokens, hq, hk, dim, torch.bfloat16))

    def run(q, k, v, do):
        a, b, c = (x.detach().requires_grad_() for x in (q, k, v))
        o = S.episode_attention(a, b, c, plan)
        return [o.detach(), *torch.autograd.grad(o, [a, b, c], do)]

    clean = run(q, k, v, do)
    spoilt = {"q": q.clone(), "k": k.clone(), "v": v.clone(), "do": do.clone()}
    spoilt[what][30000:50000:7] = math.inf                  # as a loss scale that is too large leaves them
    got = run(**spoilt)
    near = 256                                              # a tile of 128 rows, wherever it begins
    for n, (x, y) in enumerate(zip(got, clean)):
        assert torch.isfinite(x[:30000]).all() and torch.isfinite(x[50000:]).all()
        if what != "v" or n != 2:
            assert torch.equal(x[:30000 - near], y[:30000 - near]) and torch.equal(x[50000 + near:], y[50000 + near:])
    u, sums = A.UNIT[torch.bfloat16], A.SUMS
    rows = torch.arange(30000 - near, 30000, device="cuda")
    seen = torch.arange(30000, device="cuda")[None, :] <= rows[:, None]
    for h in range(hq):
        g = h // (hq // hk)
        kk, vv, qq, dd = k[:30000, g].double(), v[:30000, g].double(), q[rows, h].double(), do[rows, h].double()
        p = torch.softmax((qq @ kk.t() * dim ** -0.5).masked_fill(~seen, -math.inf), -1)
        o, size = p @ vv, p @ vv.abs()
        assert ((got[0][rows, h].double() - o).abs() <= u * (o.abs() + size) + sums * size).all()
        dp, delta = dd @ vv.t(), (dd * o).sum(-1, keepdim=True)
        ds = p * (dp - delta) * dim ** -0.5
        # as the module's bounds: rounding of dS and of the output that D is made of, 32-bit sums
        each = ds.abs() * u + p * (dd.abs() @ vv.abs().t() + dp.abs() + delta.abs()) * sums * dim ** -0.5 + p * (dd.abs() * o.abs()).sum(-1, keepdim=True) * u * dim ** -0.5
        dq = ds @ kk
        assert ((got[1][rows, h].double() - dq).abs() <= u * dq.abs() + each @ kk.abs()).all()
    for g in range(hk):                                     # the last keys are seen by the last queries only
        dk, dv, bk, bv = (torch.zeros(near, dim, dtype=torch.float64, device="cuda") for _ in range(4))
        far = torch.zeros(30000, dim, dtype=torch.float64, device="cuda")
        for h in range(g * hq // hk, (g + 1) * hq // hk):
            kk, vv, qq, dd = k[:30000, g].double(), v[:30000, g].double(), q[rows, h].double(), do[rows, h].double()
            p = torch.softmax((qq @ kk.t() * dim ** -0.5).masked_fill(~seen, -math.inf), -1)
            o, size = p @ vv, p @ vv.abs()
            dp, delta = dd @ vv.t(), (dd * o).sum(-1, keepdim=True)
            ds = p * (dp - delta) * dim ** -0.5
            each = ds.abs() * u + p * (dd.abs() @ vv.abs().t() + dp.abs() + delta.abs()) * sums * dim ** -0.5 + p * (dd.abs() * o.abs()).sum(-1, keepdim=True) * u * dim ** -0.5
            last = slice(30000 - near, 30000)
            far += (2 * u * ds.abs() + p * 2 * (dd.abs() * (u * (o.abs() + size) + sums * size)).sum(-1, keepdim=True) * dim ** -0.5).t() @ qq.abs()
            dk += ds[:, last].t() @ qq
            dv += p[:, last].t() @ dd
            bk += each[:, last].t() @ qq.abs()
            bv += p[:, last].t() @ dd.abs()
        assert ((got[2][rows, g].double() - dk).abs() <= u * dk.abs() + bk).all()
        assert ((got[2][:30000 - near, g].double() - clean[2][:30000 - near, g].double()).abs() <= 2 * u * clean[2][:30000 - near, g].double().abs() + far[:30000 - near]).all()
        assert ((got[3][rows, g].double() - dv).abs() <= u * (dv.abs() + bv) + sums * bv).all()


@pytest.mark.parametrize("dim,heads_q,heads_k", [(64, 4, 2), (128, 4, 2), (64, 8, 1)])
def test_f16_gradients_beyond_the_range_of_its_probabilities(dim, heads_q, heads_k):
    """dS above 65504 is an infinity in f16; the gradients that it goes into are not, and come out as exact as ever."""
    plan = A._plan_of([3, 200, 40, 1, 600])
    q, k, v, do = A._inputs(_gen(5), plan.tokens, heads_q, heads_k, dim, torch.float16)
    q, k, v, do = q * 0.25, k * 0.05, v * 4, do * 4096
    s = (q.double().transpose(0, 1) @ k.double().repeat_interleave(heads_q // heads_k, 1).permute(1, 2, 0)) * dim ** -0.5
    p = torch.softmax(s.masked_fill(~A._seen(plan, None), -math.inf), -1)
    dp = do.double().transpose(0, 1) @ v.double().repeat_interleave(heads_q // heads_k, 1).permute(1, 2, 0)
    assert (p * (dp - (p * dp).sum(-1, keepdim=True))).abs().max() > 65504
    A._check(q, k, v, plan, do)


# ---- graphs ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("envs,capacity", [(1, 4096), (3, 1000), (2000, 40)])
def test_an_acting_step_in_a_graph(envs, capacity):
    """Captured before any call of these sizes: replays give what calls give, bit for bit, and so does a call outside between the capture and the first replay."""
    gen = _gen(3)
    f = S.rotary_frequencies(64).cuda()
    state, fresh = _normal(gen, envs, 96), torch.zeros(envs, dtype=torch.bool, device="cuda")
    x, both = _normal(gen, envs, 96), _normal(gen, envs, 12, 64, dtype=torch.bfloat16)

    def made():
        cache = S.HistoryCache(envs, capacity, 2, 64)
        cache.keys.normal_(generator=_gen(4))
        cache.values.normal_(generator=_gen(5))
        cache.position.copy_(torch.arange(envs, device="cuda") * 2 + capacity // 2)
        return cache, state.clone()

    def step(cache, state):
        cache.advance(fresh)
        h = S.gated_recurrence_step(x, x, state, fresh)
        q, k = S.rotate_heads(both[:, :8], both[:, 8:10], None, None, cache.position, f)
        return h, S.history_attention(q, k, both[:, 10:], cache)

    def inputs(t):
        x.copy_(torch.sin(torch.arange(x.numel(), device="cuda") + t).view_as(x))
        both.copy_(torch.cos(torch.arange(both.numel(), device="cuda") * 0.7 + t).view_as(both))
        fresh.copy_(torch.arange(envs, device="cuda") % 5 == t)

    captured, called = made(), made()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(*made())                                       # the library is loaded, and nothing of the captured cache is used
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step(*captured)
    inputs(9)
    q = _normal(gen, envs, 8, 64, dtype=torch.bfloat16)
    k = _normal(gen, envs, 2, 64, dtype=torch.bfloat16)
    here = (captured[0].keys.clone(), captured[0].values.clone(), captured[0].position.clone())
    first, second = S.history_attention(q, k, k, captured[0]), S.history_attention(q, k, k, S.HistoryCache(envs, capacity, 2, 64, buffers=here))
    assert torch.equal(first, second) and torch.isfinite(first).all()
    captured[0].keys.copy_(called[0].keys)
    captured[0].values.copy_(called[0].values)
    for t in range(4):
        inputs(t)
        graph.replay()
        want = step(*called)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert torch.equal(captured[1], called[1]) and torch.equal(captured[0].keys, called[0].keys) and torch.equal(captured[0].position, called[0].position)
    del graph


# ---- angles ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("turned", [64, 24])
def test_exact_angles(interleaved, turned):
    """Products of position and frequency in 64 bits, forwards and backwards, at positions that 32 bits do not tell apart; without them the angle is the 32-bit product's, as documented.
    Norm, sine and turn in 32 bits: sixteen units in the last place."""
    gen = _gen(6)
    f = S.rotary_frequencies(turned, base=500.0).cuda()
    positions = torch.tensor([0, 1, 700, 50000, 131071, 2 ** 24 + 1, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    q = _normal(gen, 7, 3, 64).requires_grad_()
    cot = _normal(gen, 7, 3, 64)
    x = q.detach().double().requires_grad_()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    worst = []
    for exact in (True, False):
        angle = positions.double()[:, None, None] * f if exact else (positions.float()[:, None, None] * f.float()).double()
        u, v = (y[..., 0:turned:2], y[..., 1:turned:2]) if interleaved else (y[..., :turned // 2], y[..., turned // 2:turned])
        a, b = u * angle.cos() - v * angle.sin(), u * angle.sin() + v * angle.cos()
        want = torch.cat([torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1), y[..., turned:]], -1)
        got = S.rotate_heads(q, q, None, None, positions, f, interleaved=interleaved, exact_angles=exact)[1]
        grad, = torch.autograd.grad(got, q, cot)
        want_grad, = torch.autograd.grad(want, x, cot.double(), retain_graph=True)
        for g, w in ((got, want), (grad, want_grad)):
            assert ((g.double() - w).abs() <= 16 * 2.0 ** -23 * w.abs().max()).all()
        worst.append(got.detach())
    assert (worst[0] - worst[1])[:3].abs().max() < 1e-3 and (worst[0] - worst[1])[3:].abs().max() > 1e-3


# ---- streams ---------------------------------------------------------------------------------------------------------------
def test_plans_and_workspaces_outlive_calls_on_other_streams():
    """Memory that belongs to a plan or a cache alone is not handed out again while a call on a stream other than its own may still read it."""
    q = _normal(_gen(7), 4000, 2, 64, dtype=torch.bfloat16)
    f = S.rotary_frequencies(64).cuda()
    x = _normal(_gen(8), 4000, 40)
    calls = {"attention": lambda plan: S.episode_attention(q, q, q, plan), "recurrence": lambda plan: S.gated_recurrence(x, x, plan), "heads": lambda plan: S.rotate_heads(q, q, None, None, plan, f)}
    side = torch.cuda.Stream()
    for name, call in calls.items():
        want = call(_plan_of([1500, 2500]))
        plan = _plan_of([1500, 2500])
        at, size = plan._plan.data_ptr(), plan._plan.numel()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)                   # about 10 ms
            got = call(plan)
        del plan
        taken = [torch.empty(size, dtype=torch.int32, device="cuda") for _ in range(8)]
        assert not side.query() and all(t.data_ptr() != at for t in taken), name
        torch.cuda.synchronize()
        for a, b in zip(got, want) if isinstance(got, tuple) else ((got, want),):
            assert torch.equal(a, b)
    cache = S.HistoryCache(1, 4096, 2, 64)
    first = S.history_attention(q[:1], q[:1], q[:1], cache)
    (_, size, kept, _), = cache._workspaces.values()
    at = kept.data_ptr()
    del kept
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        again = S.history_attention(q[:1], q[:1], q[:1], cache)
    cache._workspaces.clear()
    taken = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(8)]
    assert not side.query() and all(t.data_ptr() != at for t in taken)
    torch.cuda.synchronize()
    assert torch.equal(first, again)


def test_two_threads_differentiate_one_graph():
    """A retained graph, differentiated by two threads at once, each on its stream with gradients of its own: what each gets alone."""
    import threading
    plan = _plan_of([700, 1300])
    f = S.rotary_frequencies(64).cuda()
    q, k, v = (_normal(_gen(9 + n), 2000, 2, 64, dtype=torch.bfloat16).requires_grad_() for n in range(3))
    out = S.episode_attention(*S.rotate_heads(q, k, None, None, plan, f), v, plan)
    cots = [_normal(_gen(20 + n), 2000, 2, 64, dtype=torch.bfloat16) for n in range(2)]
    want = [torch.autograd.grad(out, [q, k, v], c, retain_graph=True) for c in cots]
    torch.cuda.synchronize()
    got = [[], []]

    def work(n):
        for _ in range(20):
            got[n].append(torch.autograd.grad(out, [q, k, v], cots[n], retain_graph=True))

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for n in range(2):
        assert len(got[n]) == 20 and all(torch.equal(a, b) for g in got[n] for a, b in zip(g, want[n]))


@pytest.mark.parametrize("rows,length", [(1, 131071), (3, 40000)])
def test_plans_of_very_long_rows(rows, length):
    done = torch.rand((rows, length), generator=_gen(11), device="cuda") < 2e-4
    plan = S.Episodes.from_done(done)
    d = done.cpu()
    at = torch.arange(rows * length, dtype=torch.int32).view(rows, length)
    begins = torch.cat([torch.ones(rows, 1, dtype=torch.bool), d[:, :-1]], 1)
    first = torch.where(begins, at, 0).cummax(1).values
    ends = torch.cat([d[:, :-1], torch.ones(rows, 1, dtype=torch.bool)], 1)
    end = torch.where(ends, at + 1, 2 ** 31 - 1).flip(1).cummin(1).values.flip(1)
    assert torch.equal(plan.first.cpu(), first.flatten()) and torch.equal(plan.end.cpu(), end.flatten())
