"""Attention over the last tokens of an episode and its first ones, in the training form and over a cache that keeps them, against the definition in 64 bits.
Bounds as for attention without first tokens that stay."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")
import nuka  # noqa: E402
from nuka import _abi, sequence as S  # noqa: E402
import test_gpu_attention as A  # noqa: E402
import test_gpu_history as H  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture
def check(monkeypatch):
    def run(lengths, window, sinks, heads_q=2, heads_k=1, dim=64, dtype=torch.bfloat16, seed=0, plan=None, scale=None):
        plan = A._plan_of(lengths) if plan is None else plan
        q, k, v, do = A._inputs(A._gen(seed + window + sinks), plan.tokens, heads_q, heads_k, dim, dtype)
        unit, step = A.UNIT[dtype], A.STEP[dtype]
        A.UNIT_OF[:] = [unit * 2.0 ** 7, unit]
        windowed = type(A._seen)(A._seen.__code__, A._seen.__globals__)
        at = torch.arange(plan.tokens, device="cuda")
        first = plan.first.long()[:, None]
        monkeypatch.setattr(A, "_seen", lambda plan, window: windowed(plan, window) | ((at[None, :] <= at[:, None]) & (at[None, :] >= first) & (at[None, :] < first + sinks)))
        q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
        o = S.episode_attention(q, k, v, plan, scale=scale, window=window, sinks=sinks)
        grads = torch.autograd.grad(o, [q, k, v], do)
        w = A._reference(q, k, v, plan, dim ** -0.5 if scale is None else scale, window, do)
        monkeypatch.undo()
        for (name, (want, bound)), got in zip(A._bounds(w, unit, step).items(), [o.detach(), *grads]):
            A._close(got, want, bound, name)
        assert torch.equal(S.episode_attention(q.detach(), k.detach(), v.detach(), plan, scale=scale, window=window, sinks=sinks), o)
    return run


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths", list(A.LENGTHS))
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_and_its_gradient(check, dtype, lengths, dim):
    check(A.LENGTHS[lengths], 40, 4, 4, 2, dim, dtype, seed=dim)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 127, 128, 129, 700])
@pytest.mark.parametrize("sinks", [1, 4, 64, 65, 130, 1000])
def test_windows_and_sinks(check, window, sinks):
    """Sinks that end inside a tile and at its edge, that reach the window and pass it, of an episode that begins in, at the end of, and before a tile; more of them than tokens."""
    check([500, 127, 90, 1, 60, 300], window, sinks, dim=64 if window % 2 else 128)


@pytest.mark.parametrize("rows,length", [(300, 1), (50, 24), (5, 100), (3, 128), (2, 129), (3, 400)])
def test_rows_of_one_length(check, rows, length):
    plan = S.Episodes.from_done(torch.rand((rows, length), generator=A._gen(rows), device="cuda") < 0.03)
    check(None, 7, 3, 4, 2, 64, plan=plan)
    check(None, 30, 10, 4, 2, 128, torch.float16, plan=plan)


@pytest.mark.parametrize("heads_q,heads_k,dim", [(1, 1, 8), (3, 3, 40), (6, 2, 96), (8, 1, 120), (16, 2, 64), (12, 1, 128)])
def test_head_layouts_and_jobs_shared_by_blocks(check, heads_q, heads_k, dim):
    check([700, 3, 90], 50, 5, heads_q, heads_k, dim)


def test_more_jobs_than_blocks(check):
    check([900, 3, 0, 1, 1300, 40, 700, 129], 100, 8, 32, 4, 64)
    check([900, 3, 0, 1, 1300, 40, 700, 129], 33, 70, 24, 24, 72)


@pytest.mark.parametrize("dim", [64, 128])
def test_sharp_softmax(check, dim):
    check([700, 20], 60, 6, dim=dim, scale=1.0)


def test_without_a_window_or_with_a_long_one_all_are_seen():
    plan = A._plan_of([300, 41])
    q, k, v, _ = A._inputs(A._gen(1), plan.tokens, 2, 1, 64, torch.bfloat16)
    want = S.episode_attention(q, k, v, plan)
    assert torch.equal(S.episode_attention(q, k, v, plan, sinks=5), want) and torch.equal(S.episode_attention(q, k, v, plan, window=300, sinks=0), S.episode_attention(q, k, v, plan, window=300))
    off = (S.episode_attention(q, k, v, plan, window=300, sinks=5).float() - want.float()).abs().max().item()
    assert off <= 2 * A.UNIT[torch.bfloat16] * 2 * v.float().abs().max().item()          # the same rows, in steps that begin elsewhere


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("what", ["q", "k", "v", "do"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("token", [71, 250])
def test_what_is_not_finite_stays_in_its_episode(dim, what, value, token):
    """A value of a first token that stays, and of a late one: the other episodes' outputs and gradients are what they are without it, within the bounds of all values."""
    plan = A._plan_of([30, 40, 200, 24, 90])
    names = ("q", "k", "v", "do")
    clean = dict(zip(names, (x.clone() for x in A._inputs(A._gen(30), plan.tokens, 4, 2, dim, torch.bfloat16))))
    spoilt = {n: x.clone() for n, x in clean.items()}
    spoilt[what][token, 0, 5] = value
    outs = []
    for x in (clean, spoilt):
        q, k, v = (x[n].requires_grad_() for n in names[:3])
        o = S.episode_attention(q, k, v, plan, window=20, sinks=3)
        outs.append([o.detach(), *torch.autograd.grad(o, [q, k, v], x["do"])])
    other = torch.ones(plan.tokens, dtype=torch.bool, device="cuda")
    other[70:270] = False
    for n, (a, b) in enumerate(zip(*outs)):                # clean ones are within their bounds by the tests above; worked out row by row they differ by the roundings of probabilities
        a, b = a[other].float(), b[other].float()
        assert torch.isfinite(b).all() and (a - b).abs().max().item() <= 2.0 ** -5 * (1 + a.abs().max().item()), n
    # rows of the same episode that do not see the token are finite
    if what in ("k", "v"):
        unseen = torch.arange(70, 270, device="cuda")
        unseen = unseen[(unseen < token) | ((unseen >= token + 20) & (token >= 73))]
        assert torch.isfinite(outs[1][0][unseen]).all()
        # an infinite key against a query below 0 in that column is a score of -infinity, which weighs 0: such a row is finite by its definition
        assert (what == "k" and value == math.inf) or not torch.isfinite(outs[1][0][token:token + 1]).all()


def test_same_bits_streams_and_a_graph():
    plan = A._plan_of([3000, 17, 900])
    q, k, v, do = A._inputs(A._gen(7), plan.tokens, 4, 2, 64, torch.bfloat16)
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))

    def run():
        o = S.episode_attention(q, k, v, plan, window=64, sinks=4)
        return [o, *torch.autograd.grad(o, [q, k, v], do)]

    want = [x.detach().clone() for x in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.synchronize()
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


def test_gradients_under_checkpointing():
    from torch.utils.checkpoint import checkpoint
    plan = A._plan_of([300, 20])
    q, k, v, do = A._inputs(A._gen(8), plan.tokens, 2, 1, 64, torch.float16)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    call = lambda *x: S.episode_attention(*x, plan, window=30, sinks=2)
    want = torch.autograd.grad(call(*leaves), leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(checkpoint(call, *leaves, use_reentrant=False), leaves, do), want))


# ---- the cache ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,d", [(8, 2, 64), (1, 1, 128), (3, 3, 32), (12, 1, 64), (4, 4, 120)])
@pytest.mark.parametrize("cap,sinks", [(50, 3), (50, 49), (17, 16), (2, 1), (700, 64)])
def test_places_before_at_and_after_the_ring_comes_round(dtype, hq, hk, d, cap, sinks):
    gen, positions = H._gen(hq + d), [-1, 0, 1, sinks - 1, sinks, cap - 1, cap, cap + 1, 2 * cap - sinks, 1000003, 2 ** 31 - 1]
    envs = len(positions)
    keys, values = H._normal(gen, envs, cap, hk, d, dtype=dtype), H._normal(gen, envs, cap, hk, d, dtype=dtype)
    position = torch.tensor(positions, dtype=torch.int32, device="cuda")
    for e, n in enumerate(positions):                      # what an earlier episode left there may be anything
        keys[e, max(n, 0):], values[e, max(n, 0):] = math.nan, math.inf
    cache = S.HistoryCache(envs, cap, hk, d, dtype, buffers=(keys, values, position), sinks=sinks)
    q, k, v = H._normal(gen, envs, hq, d, dtype=dtype, scale=1.5), H._normal(gen, envs, hk, d, dtype=dtype), H._normal(gen, envs, hk, d, dtype=dtype)
    want_keys, want_values = keys.clone(), values.clone()
    for e, n in enumerate(positions):
        n = max(n, 0)
        place = n if n < sinks else sinks + (n - sinks) % (cap - sinks)
        want_keys[e, place], want_values[e, place] = k[e], v[e]
    for _ in range(2):                                     # the second time finds its own token in the cache, and workspaces as they were
        o = S.history_attention(q, k, v, cache)
        bits = lambda x: x.view(torch.int16)
        assert torch.equal(bits(cache.keys), bits(want_keys)) and torch.equal(bits(cache.values), bits(want_values))
        want, size = H._reference(q, want_keys, want_values, (position.long().clamp(min=0) + 1).clamp(max=cap), d ** -0.5)
        assert torch.isfinite(o).all()
        off = (o.double() - want).abs() - (H.UNIT[dtype] * (want.abs() + size) + 2.0 ** -15 * size + (2.0 ** -24 if dtype is torch.float16 else 0))
        assert off.max().item() <= 0, off.max().item()


@pytest.mark.parametrize("cap,sinks", [(16, 4), (9, 1), (40, 39)])
def test_acting_follows_attention_over_the_rollout(cap, sinks):
    """Token by token with a cache gives what attention over the whole rollout gives with as many first tokens and the rest of the cache as its window."""
    gen, envs, steps = H._gen(3), 6, 70
    done = torch.rand((envs, steps), generator=gen, device="cuda") < 0.04
    q, k, v = H._normal(gen, envs, steps, 4, 64), H._normal(gen, envs, steps, 2, 64), H._normal(gen, envs, steps, 2, 64)
    want = S.episode_attention(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), S.Episodes.from_done(done), window=cap - sinks, sinks=sinks).view(envs, steps, 4, 64)
    cache = S.HistoryCache(envs, cap, 2, 64, sinks=sinks)
    for t in range(steps):
        cache.advance(done[:, t - 1] if t else None)
        o = S.history_attention(q[:, t], k[:, t], v[:, t], cache)
        # two kernels' roundings of outputs and probabilities: 4 units of values up to 4 in all
        assert (o.float() - want[:, t].float()).abs().max().item() <= 4 * H.UNIT[torch.bfloat16] * 4


def test_wrong_arguments_are_refused():
    plan = A._plan_of([10])
    q = torch.zeros(10, 4, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        S.episode_attention(q, q, q, plan, window=4, sinks=-1)
    for sinks in (-1, 8, 9):
        with pytest.raises(ValueError):
            S.HistoryCache(2, 8, 1, 64, sinks=sinks)
    lib = _abi.lib()
    ok = dict(plan=plan._ref, dtype=2, heads_q=4, heads_k=4, dim=64, window=4, scale=0.125, q=q.data_ptr(), k=q.data_ptr(), v=q.data_ptr(), q_stride=256, q_head_stride=64, k_stride=256,
              k_head_stride=64, v_stride=256, v_head_stride=64, out=q.data_ptr())
    assert lib.nuka_b200_attention_sinks(ctypes.byref(_abi.AttentionDesc(**ok)), -1, None) == _abi.INVALID_ARG
    assert lib.nuka_b200_attention_sinks_backward(ctypes.byref(_abi.AttentionDesc(**ok)), 2, None, 0, None) == _abi.INVALID_ARG
    ring = dict(dtype=2, envs=1, capacity=8, heads_q=1, heads_k=1, dim=64, scale=1.0, q=q.data_ptr(), k=q.data_ptr(), v=q.data_ptr(), keys=q.data_ptr(), values=q.data_ptr(), position=q.data_ptr(), out=q.data_ptr())
    for sinks in (-1, 8):
        assert lib.nuka_b200_history_sinks(ctypes.byref(_abi.HistoryDesc(**ring)), sinks, None) == _abi.INVALID_ARG
