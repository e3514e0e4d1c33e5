"""What the selective operators and attention with first tokens that stay hand to the library, and what the library's entries refuse, without a GPU: the package's calls go to a recorder, the
entries' refusals come before anything is read or launched."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
from nuka import _abi, sequence as S  # noqa: E402


@pytest.fixture
def calls(monkeypatch):
    """Tensors of the CPU are taken, and (entry's name, its arguments) of each call is kept; nothing is worked out."""
    seen = []
    monkeypatch.setattr(S, "_on_gpu", lambda first, *others: first.device)
    monkeypatch.setattr(S, "_call", lambda device, function, *args: seen.append((function.__name__, [getattr(a, "_obj", a) for a in args])))
    return seen


def _plan(rows=2, length=5):
    return S.Episodes.from_offsets(torch.arange(rows + 1, dtype=torch.int32) * length, rows * length)


def _scan(leaves):
    return S.selective_scan(*leaves[:5], _plan(), *leaves[5:])[0]


OPERATORS = {
    "convolution": (lambda leaves: S.short_convolution(*leaves[:3], _plan(), leaves[3], silu=True)[0], lambda: [torch.randn(10, 8), torch.randn(8, 4), torch.randn(8), torch.randn(2, 3, 8)],
                    ("x", "weight", "bias", "initial")),
    "scan": (_scan, lambda: [torch.randn(10, 8), torch.randn(10, 8), -torch.rand(8, 4), torch.randn(10, 4), torch.randn(10, 4), torch.randn(2, 8, 4), torch.randn(8), torch.randn(10, 8), torch.randn(8)],
             ("x", "delta", "decay", "b", "c", "initial", "skip", "gate", "delta_bias", "kept")),
    "attention": (lambda leaves: S.episode_attention(*leaves, _plan(), window=3, sinks=2), lambda: [torch.randn(10, 2, 16).bfloat16() for _ in range(3)], ("q", "k", "v", "out", "lse")),
}


@pytest.mark.parametrize("operator", list(OPERATORS))
@pytest.mark.parametrize("turned", [False, True])
def test_gradients_read_what_saved_tensors_return(calls, operator, turned):
    """Hooks (offloading, checkpointing) give back other tensors than were saved, of other strides perhaps: the backward call has their addresses, or those of copies of
    them, and strides that go with them."""
    run, make, fields = OPERATORS[operator]
    leaves = [x.requires_grad_() for x in make()]
    kept, back = [], []

    def unpack(x):
        y = x.clone()
        if turned and y.dim() >= 2:                        # the same values, dimensions the other way round
            y = y.transpose(0, 1).contiguous().transpose(0, 1)
        back.append(y)
        return y

    with torch.autograd.graph.saved_tensors_hooks(lambda x: kept.append(x.clone()) or kept[-1], unpack):
        out = run(leaves)
    for _ in range(2):
        back.clear()
        grads = torch.autograd.grad(out, leaves, torch.ones_like(out), retain_graph=True)
        name, (desc, *_) = calls[-1]
        assert name.endswith("_backward")
        at = {x.data_ptr(): x for x in back}
        for field in fields:
            assert getattr(desc, field)
            if not turned:
                assert getattr(desc, field) in at, field
        for leaf, grad in zip(leaves, grads):
            assert grad.shape == leaf.shape and grad.dtype == leaf.dtype and grad.is_contiguous()
        for field in [f for f in fields if hasattr(desc, f + "_stride")]:
            assert getattr(desc, f"{field}_stride") >= leaves[fields.index(field)][0].numel() or turned
    assert calls[-1][1][0] is not calls[-2][1][0]


@pytest.mark.parametrize("operator", list(OPERATORS))
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused_and_not_dropped(calls, operator, grad):
    import torch.autograd.forward_ad as fwd
    run, make, _ = OPERATORS[operator]
    leaves = make()
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        run(leaves)
        for n in range(len(leaves)):
            duals = [fwd.make_dual(x, torch.ones_like(x)) if n == i else x for i, x in enumerate(leaves)]
            with pytest.raises(NotImplementedError):
                run(duals)


def test_which_entry_is_called(calls, monkeypatch):
    """First tokens that stay have entries of their own; calls without any are what they were."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    q = torch.randn(10, 2, 16).bfloat16()
    for window, sinks, name in ((None, 0, "nuka_b200_attention"), (None, 4, "nuka_b200_attention"), (3, 0, "nuka_b200_attention"), (3, 4, "nuka_b200_attention_sinks")):
        S.episode_attention(q, q, q, _plan(), window=window, sinks=sinks)
        assert calls[-1][0] == name and calls[-1][1][1:] == ([4] if name.endswith("sinks") else [])
    one = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    for sinks in (0, 3):
        S.history_attention(one, one, one, S.HistoryCache(1, 8, 2, 64, device="cpu", sinks=sinks))
        assert calls[-1][0] == ("nuka_b200_history_sinks" if sinks else "nuka_b200_history") and calls[-1][1][1:] == ([sinks] if sinks else [])


def test_rows_that_may_be_empty_end_with_what_they_began_with(calls):
    x, weight, first = torch.randn(10, 8), torch.randn(8, 4), torch.randn(2, 3, 8)
    state = S.short_convolution(x, weight, None, _plan(), first)[1]
    assert torch.equal(state, first) and state.data_ptr() != first.data_ptr()
    assert not S.short_convolution(x, weight, None, _plan())[1].any()
    b, start = torch.randn(10, 4), torch.randn(2, 8, 4)
    state = S.selective_scan(x, x, -torch.rand(8, 4), b, b, _plan(), start)[1]
    assert torch.equal(state, start) and state.data_ptr() != start.data_ptr()


def test_wrong_arguments_are_refused(calls):
    run, make, _ = OPERATORS["scan"]
    good = make()
    run(good)
    before = len(calls)
    bad = [good[0][:9], good[1][:, :7], good[2].double(), good[3][:, :3], good[4].half(), good[5][:1], good[6][:3], good[7].half(), good[8].double()]
    for n, x in enumerate(bad):
        with pytest.raises(ValueError):
            run([x if n == i else y for i, y in enumerate(good)])
    with pytest.raises(ValueError):
        S.selective_scan_step(good[0], *good[1:5], torch.zeros(10, 8, 3))
    with pytest.raises(ValueError):
        S.selective_scan_step(good[0], *good[1:5], torch.zeros(10, 8, 4), fresh=torch.zeros(9, dtype=torch.bool))
    for weight in (torch.randn(8, 1), torch.randn(8, 5), torch.randn(7, 4), torch.randn(8, 4).half()):
        with pytest.raises(ValueError):
            S.short_convolution(good[0], weight, None, _plan())
    assert {name for name, _ in calls[before:]} <= {"nuka_b200_episodes_from_offsets"}


AT = 1 << 20


def _plan_desc(**change):
    return ctypes.pointer(_abi.EpisodesDesc(**{**dict(first=AT, end=AT, link=AT, tail=AT, tokens=8, rows=2, length=4), **change}))


def _code(function, kind, ok, extra=(), **change):
    return function(ctypes.byref(kind(**{**ok, **change})), *extra, None)


def test_the_convolutions_entries_refuse():
    lib, invalid, unsupported = _abi.lib(), _abi.INVALID_ARG, 7
    ok = dict(plan=_plan_desc(), dtype=2, channels=8, width=4, x=AT, x_stride=8, weight=AT, y=AT, state=AT, dy=AT, dx=AT, dweight=AT, dbias=AT, workspace=AT, workspace_bytes=1 << 30)
    for change in (dict(plan=None), dict(plan=_plan_desc(rows=-1)), dict(plan=_plan_desc(link=AT + 1)), dict(x=None), dict(weight=None), dict(y=None), dict(state=None), dict(x=AT + 1), dict(y=AT + 1), dict(initial=AT + 1),
                   dict(weight=AT + 2), dict(bias=AT + 1), dict(x_stride=-1)):
        assert _code(lib.nuka_b200_convolution, _abi.ConvolutionDesc, ok, **change) == invalid, change
    for change in (dict(dy=None), dict(dx=None), dict(dy=AT + 1), dict(dinitial=AT + 1), dict(dstate=AT + 1), dict(dweight=AT + 2), dict(workspace=None), dict(workspace_bytes=8), dict(workspace=AT + 2)):
        assert _code(lib.nuka_b200_convolution_backward, _abi.ConvolutionDesc, ok, **change) == invalid, change
    for change in (dict(dtype=3), dict(width=1), dict(width=5), dict(channels=-1), dict(channels=1 << 25)):
        assert _code(lib.nuka_b200_convolution, _abi.ConvolutionDesc, ok, **change) == unsupported, change
    huge = _plan_desc(tokens=1 << 30, rows=1, length=0)
    assert _code(lib.nuka_b200_convolution, _abi.ConvolutionDesc, ok, plan=huge, channels=1 << 20) == unsupported
    step = dict(dtype=2, envs=4, channels=8, width=4, x=AT, x_stride=8, weight=AT, state=AT, y=AT)
    for change in (dict(envs=-1), dict(x=None), dict(weight=None), dict(state=None), dict(y=None), dict(x=AT + 1), dict(state=AT + 1), dict(weight=AT + 2), dict(x_stride=-8)):
        assert _code(lib.nuka_b200_convolution_step, _abi.ConvolutionStepDesc, step, **change) == invalid, change
    assert _code(lib.nuka_b200_convolution_step, _abi.ConvolutionStepDesc, step, width=6) == unsupported
    assert _code(lib.nuka_b200_convolution_step, _abi.ConvolutionStepDesc, step, envs=0) == 0 and _code(lib.nuka_b200_convolution, _abi.ConvolutionDesc, ok, channels=0) == 0
    for function in (lib.nuka_b200_convolution, lib.nuka_b200_convolution_backward, lib.nuka_b200_convolution_step):
        assert function(None, None) == invalid and lib.nuka_last_error_message()
    assert lib.nuka_b200_convolution_workspace(_plan_desc(), 8, 4) > 0 and lib.nuka_b200_convolution_workspace(_plan_desc(), 8, 5) == 0 and lib.nuka_b200_convolution_workspace(None, 8, 4) == 0


def test_the_scans_entries_refuse():
    lib, invalid, unsupported = _abi.lib(), _abi.INVALID_ARG, 7
    ok = dict(plan=_plan_desc(), dtype=2, channels=8, states=16, x=AT, delta=AT, b=AT, c=AT, x_stride=8, delta_stride=8, b_stride=16, c_stride=16, decay=AT, y=AT, state=AT, kept=AT, kept_bytes=1 << 40, dy=AT, dx=AT,
              ddelta=AT, db=AT, dc=AT, workspace=AT, workspace_bytes=1 << 40)
    for change in (dict(plan=None), dict(x=None), dict(delta=None), dict(b=None), dict(c=None), dict(decay=None), dict(y=None), dict(state=None), dict(x=AT + 1), dict(gate=AT + 1), dict(decay=AT + 2), dict(initial=AT + 2),
                   dict(skip=AT + 1), dict(delta_bias=AT + 2), dict(x_stride=-1), dict(b_stride=-1), dict(kept=AT + 8), dict(kept_bytes=16)):
        assert _code(lib.nuka_b200_scan, _abi.ScanDesc, ok, **change) == invalid, change
    for change in (dict(kept=None), dict(dy=None), dict(dx=None), dict(ddelta=None), dict(db=None), dict(dc=None), dict(dc=AT + 1), dict(gate=AT), dict(ddecay=AT + 2), dict(dinitial=AT + 1), dict(dstate=AT + 2), dict(workspace=None),
                   dict(workspace=AT + 4), dict(workspace_bytes=64)):
        assert _code(lib.nuka_b200_scan_backward, _abi.ScanDesc, ok, **change) == invalid, change
    for change in (dict(dtype=3), dict(states=0), dict(states=65), dict(channels=-1), dict(channels=1 << 25)):
        assert _code(lib.nuka_b200_scan, _abi.ScanDesc, ok, **change) == unsupported, change
    assert _code(lib.nuka_b200_scan, _abi.ScanDesc, ok, plan=_plan_desc(tokens=1 << 30, rows=1 << 30, length=1), channels=1 << 12) == unsupported
    long = _plan_desc(tokens=4096, rows=1, length=0)
    assert lib.nuka_b200_scan_workspace(long, 8, 16, 0) > 0 and _code(lib.nuka_b200_scan, _abi.ScanDesc, ok, plan=long, workspace=None) == invalid
    step = dict(dtype=2, envs=4, channels=8, states=16, x=AT, delta=AT, b=AT, c=AT, x_stride=8, delta_stride=8, b_stride=16, c_stride=16, decay=AT, state=AT, y=AT)
    for change in (dict(envs=-1), dict(x=None), dict(delta=None), dict(b=None), dict(c=None), dict(decay=None), dict(state=None), dict(y=None), dict(gate=AT + 1), dict(state=AT + 2), dict(c_stride=-1)):
        assert _code(lib.nuka_b200_scan_step, _abi.ScanStepDesc, step, **change) == invalid, change
    assert _code(lib.nuka_b200_scan_step, _abi.ScanStepDesc, step, states=0) == unsupported and _code(lib.nuka_b200_scan_step, _abi.ScanStepDesc, step, envs=0) == 0
    for function in (lib.nuka_b200_scan, lib.nuka_b200_scan_backward, lib.nuka_b200_scan_step):
        assert function(None, None) == invalid and lib.nuka_last_error_message()
    assert lib.nuka_b200_scan_kept(_plan_desc(), 8, 65) == 0 and lib.nuka_b200_scan_workspace(None, 8, 16, 1) == 0


def test_the_sinks_entries_refuse():
    lib, invalid = _abi.lib(), _abi.INVALID_ARG
    plan = _plan_desc(tokens=4096, rows=2, length=0)
    ok = dict(plan=plan, dtype=2, heads_q=4, heads_k=4, dim=64, window=64, scale=0.125, q=AT, k=AT, v=AT, q_stride=256, q_head_stride=64, k_stride=256, k_head_stride=64, v_stride=256, v_head_stride=64, out=AT, lse=AT,
              dout=AT, delta=AT, dq=AT, dk=AT, dv=AT)
    need = lib.nuka_b200_attention_sinks_workspace(ctypes.byref(_abi.AttentionDesc(**ok)), 4)
    assert need > 0
    for sinks, change, workspace, size in ((-1, {}, AT, need), (4, dict(window=-1), AT, need), (4, {}, None, need), (4, {}, AT, need - 1), (4, {}, AT + 8, need), (4, dict(q=None), AT, need), (4, dict(lse=None), AT, need)):
        assert _code(lib.nuka_b200_attention_sinks_backward, _abi.AttentionDesc, ok, (sinks, workspace, size), **change) == invalid, (sinks, change)
    assert _code(lib.nuka_b200_attention_sinks, _abi.AttentionDesc, ok, (-1,)) == invalid
    for sinks, change in ((0, {}), (4, dict(window=0)), (100, {}), (4, dict(plan=_plan_desc(tokens=4096, rows=128, length=32))), (4, dict(plan=_plan_desc(tokens=0, rows=0, length=0))), (4, dict(plan=None))):
        assert lib.nuka_b200_attention_sinks_workspace(ctypes.byref(_abi.AttentionDesc(**{**ok, **change})), sinks) == 0, (sinks, change)
    ring = dict(dtype=2, envs=1, capacity=8, heads_q=1, heads_k=1, dim=64, scale=1.0, q=AT, k=AT, v=AT, keys=AT, values=AT, position=AT, out=AT)
    for sinks in (-1, 8, 9):
        assert _code(lib.nuka_b200_history_sinks, _abi.HistoryDesc, ring, (sinks,)) == invalid
    assert _code(lib.nuka_b200_history_sinks, _abi.HistoryDesc, ring, (3,), envs=0) == 0


def test_a_policys_states_are_forgotten_where_an_episode_ended():
    """States of any number of dimensions."""
    from types import SimpleNamespace
    from nuka import memory_policy as M
    policy = M.MemoryPolicy(12, 3, width=32, heads=1, kv_heads=1, layers=2, history=8, states=5, sinks=2)
    shapes = [(3, *shape) for layer in policy.layers for shape in layer.kept()]
    assert shapes == [(3, 3, 64), (3, 64, 5)] * 2
    states = [torch.full(shape, float("nan")) for shape in shapes]
    memory = SimpleNamespace(begin_rollout=lambda: [s.clone() for s in states])
    act = SimpleNamespace(act=lambda obs, memory, fresh: (torch.zeros(3, 2), torch.zeros(3)), log_std=torch.zeros(2))
    env = SimpleNamespace(step=lambda action: (torch.zeros(3, 4), torch.zeros(3), None, None, {"done": torch.zeros(3, dtype=torch.bool)}))
    rollout = M.Rollout(env, act, memory, torch.zeros(3, 4), torch.tensor([True, False, True]), 2)
    for kept in rollout.states:
        assert not kept[[0, 2]].any() and kept[1].isnan().all()
    for bad in (dict(sinks=8), dict(sinks=-1), dict(states=65)):
        with pytest.raises(ValueError):
            M.MemoryPolicy(12, 3, width=32, heads=1, kv_heads=1, history=8, **bad)
