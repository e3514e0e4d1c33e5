"""What nuka.sequence hands to the library and to torch, without a GPU: its calls go to a recorder in the library's place."""
import ctypes
import math
import os
import re

import pytest

torch = pytest.importorskip("torch")
from nuka import _abi, sequence as S  # noqa: E402


@pytest.fixture
def calls(monkeypatch):
    """Tensors of the CPU are taken, and (entry's name, descriptor) of each call is kept; nothing is worked out."""
    seen = []
    monkeypatch.setattr(S, "_on_gpu", lambda first, *others: first.device)
    monkeypatch.setattr(S, "_call", lambda device, function, *args: seen.append((function.__name__, getattr(args[0], "_obj", None))))
    return seen


def _plan(rows=2, length=5):
    return S.Episodes.from_offsets(torch.arange(rows + 1, dtype=torch.int32) * length, rows * length)


def _recurrence(leaves):
    return S.gated_recurrence(leaves[0], leaves[1], _plan(), leaves[2])[0]


def _heads(leaves):
    return sum(S.rotate_heads(*leaves, _plan(), torch.ones(4, dtype=torch.float64)))


def _attention(leaves):
    return S.episode_attention(*leaves, _plan())


# the operator, its leaves, and the fields of its backward call that come from the forward pass
OPERATORS = {
    "recurrence": (_recurrence, lambda: [torch.randn(10, 8), torch.randn(10, 8), torch.randn(2, 8)], ("x", "gate", "initial", "h")),
    "heads": (_heads, lambda: [torch.randn(10, 2, 16), torch.randn(10, 2, 16), torch.ones(16), torch.ones(16)], ("q", "k", "q_weight", "k_weight", "first", "frequencies")),
    "attention": (_attention, lambda: [torch.randn(10, 2, 16).bfloat16() for _ in range(3)], ("q", "k", "v", "out", "lse")),
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
        if turned and y.dim() == 3:                        # the same values, heads before tokens
            y = y.transpose(0, 1).contiguous().transpose(0, 1)
        back.append(y)
        return y

    with torch.autograd.graph.saved_tensors_hooks(lambda x: kept.append(x.clone()) or kept[-1], unpack):
        out = run(leaves)
    for _ in range(2):                                     # a graph that is kept: each pass has a descriptor of its own
        back.clear()
        torch.autograd.grad(out, leaves, torch.ones_like(out), retain_graph=True)
        name, desc = calls[-1]
        assert name.endswith("_backward")
        at = {x.data_ptr(): x for x in back}
        for field in fields:
            if not (turned and field == "out"):            # contiguous, so a copy of what was turned
                assert getattr(desc, field) in at, field
        for field in ("q", "k", "v") if operator != "recurrence" else ():
            if hasattr(desc, field):
                x = at[getattr(desc, field)]
                assert (getattr(desc, field + "_stride"), getattr(desc, field + "_head_stride")) == x.stride()[:2]
    assert calls[-1][1] is not calls[-2][1]


def test_the_rows_of_an_attention_kernel_meet_at_one_barrier():
    """A wait of a kernel that gives up does so warp by warp.  Warps that go on and warps that gave up meet at the same named barriers in the same order only because there is one of
    them: with two, the first could wait at one and the second at the other, and such a wait has no limit."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nuka-physics_b200", "csrc", "nkb_attention.cu")
    with open(path) as f:
        kernels = f.read().split("__global__")[1:]
    met = [set(re.findall(r"\bmeet\(([^,]*),", body)) for body in kernels]
    assert len(kernels) == 3 and all(len(m) <= 1 for m in met) and any(met), met


def test_a_workspace_made_while_a_graph_is_captured_is_not_kept(calls, monkeypatch):
    """Its zeroing is a node of that graph: a call outside the graph, before the first replay, would count on what nothing zeroed."""
    q, k = torch.zeros(1, 8, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    cache = S.HistoryCache(1, 4096, 2, 64, device="cpu")
    zeros, capturing = torch.zeros, [True]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(torch, "zeros", lambda *a, **b: zeros(*a, **b).fill_(7) if capturing[0] else zeros(*a, **b))         # zeroed by a replay, not now
    S.history_attention(q, k, k, cache)
    assert calls[-1][1].workspace_bytes > 0 and calls[-1][1].workspace
    capturing[0] = False
    S.history_attention(q, k, k, cache)
    outside = calls[-1][1]
    assert ctypes.string_at(outside.workspace, outside.workspace_bytes) == bytes(outside.workspace_bytes)
    for capturing[0] in (False, True):                     # kept from then on, by captures too
        S.history_attention(q, k, k, cache)
        assert calls[-1][1].workspace == outside.workspace


@pytest.mark.parametrize("operator", list(OPERATORS))
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused_and_not_dropped(calls, operator, grad):
    """A tangent that an operator cannot carry on is an error, with or without gradients recorded; without a tangent the call is as ever."""
    import torch.autograd.forward_ad as fwd
    run, make, _ = OPERATORS[operator]
    leaves = make()
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        run(leaves)
        for n in range(len(leaves)):
            duals = [fwd.make_dual(x, torch.ones_like(x)) if n == i else x for i, x in enumerate(leaves)]
            with pytest.raises(NotImplementedError):
                run(duals)
    run(leaves)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: run([x, *leaves[1:]]), (leaves[0],), (leaves[0],))


def test_the_c_entries_refuse_addresses_that_their_loads_cannot_take():
    """Nothing is launched, so this needs no GPU; the addresses are never read."""
    lib, at = _abi.lib(), 1 << 20
    plan = lambda **change: _abi.EpisodesDesc(**{**dict(first=at, end=at, link=at, tail=at, tokens=8, rows=2, length=4), **change})
    refused = lambda code: code == _abi.INVALID_ARG and b"byte" in lib.nuka_last_error_message()
    for name in ("first", "end", "link", "tail"):
        odd = ctypes.byref(plan(**{name: at + 2}))
        assert refused(lib.nuka_b200_episodes_from_offsets(odd, at, None)) and refused(lib.nuka_b200_episodes_from_done(odd, at, None))
    assert refused(lib.nuka_b200_episodes_from_offsets(ctypes.byref(plan()), at + 2, None))
    ok = dict(first=at, dtype=0, tokens=8, heads_q=2, heads_k=1, dim=64, turned=0, q=at, k=at, q_stride=128, q_head_stride=64, k_stride=64, k_head_stride=64, eps=1e-6, q_out=at, k_out=at,
              dq_out=at, dk_out=at, dq=at, dk=at, workspace=at, workspace_bytes=1 << 20)
    heads = lambda back, **change: (lib.nuka_b200_heads_backward if back else lib.nuka_b200_heads)(ctypes.byref(_abi.HeadsDesc(**{**ok, **change})), None)
    for change in (dict(first=at + 1), dict(first=None, positions=at + 2), dict(q_weight=at + 2)):
        assert refused(heads(False, frequencies=at, turned=64, **change)), change
    for change in (dict(dq_weight=at + 2), dict(dk_weight=at + 1)):
        assert refused(heads(True, **change)), change
        assert refused(heads(True, tokens=0, **change)), change             # zeroed in their place


def test_a_rollout_forgets_states_that_are_not_finite():
    """What ended with the last rollout does not go on into this one, whatever it was: acting forgets it, and so does the state that the training form begins with."""
    from types import SimpleNamespace
    from nuka import memory_policy as M
    state = torch.tensor([[1.0, math.nan], [math.inf, 2.0], [3.0, 4.0]])
    fresh = torch.tensor([True, True, False])
    memory = SimpleNamespace(begin_rollout=lambda: [state.clone(), state.clone()])
    policy = SimpleNamespace(act=lambda obs, memory, fresh: (torch.zeros(3, 2), torch.zeros(3)), log_std=torch.zeros(2))
    env = SimpleNamespace(step=lambda action: (torch.zeros(3, 4), torch.zeros(3), None, None, {"done": torch.zeros(3, dtype=torch.bool)}))
    rollout = M.Rollout(env, policy, memory, torch.zeros(3, 4), fresh, 2)
    for kept in rollout.states:
        assert torch.equal(kept, torch.tensor([[0.0, 0.0], [0.0, 0.0], [3.0, 4.0]]))


def test_heads_without_columns_are_refused(calls):
    q = torch.zeros(10, 2, 0, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        S.episode_attention(q, q, q, _plan())
