"""What the selective operators' entries refuse at the ends of what they take, and what autograd is told, without a GPU."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
from nuka import _abi, sequence as S  # noqa: E402

AT = 1 << 20


def _plan(**change):
    return ctypes.pointer(_abi.EpisodesDesc(**{**dict(first=AT, end=AT, link=AT, tail=AT, tokens=8, rows=2, length=4), **change}))


def test_a_scan_without_channels_has_gradients_of_b_and_c():
    lib = _abi.lib()
    ok = dict(plan=_plan(), dtype=2, channels=0, states=16, b=AT, c=AT, b_stride=16, c_stride=16, db=AT, dc=AT)
    for change in (dict(db=None), dict(dc=None), dict(db=AT + 1), dict(dc=AT + 1)):
        assert lib.nuka_b200_scan_backward(ctypes.byref(_abi.ScanDesc(**{**ok, **change})), None) == _abi.INVALID_ARG, change
    assert lib.nuka_b200_scan(ctypes.byref(_abi.ScanDesc(**ok)), None) == 0
    assert lib.nuka_b200_scan_backward(ctypes.byref(_abi.ScanDesc(**{**ok, "plan": _plan(tokens=0, rows=2, length=0)})), None) == 0


@pytest.mark.parametrize("kind", ["recurrence", "convolution", "scan"])
def test_a_state_that_was_stepped_on_has_no_gradients_of_what_it_was(kind, monkeypatch):
    """A step writes the state in place. Autograd, which keeps what a row began with for the backward pass, refuses the gradient then, as for torch's own operators in place."""
    monkeypatch.setattr(S, "_on_gpu", lambda first, *others: first.device)
    monkeypatch.setattr(S, "_call", lambda device, function, *args: None)
    plan, x = S.Episodes.from_offsets(torch.arange(3, dtype=torch.int32) * 5, 10), torch.randn(10, 8, requires_grad=True)
    b, decay, taps, one = torch.randn(10, 4), -torch.rand(8, 4), torch.randn(8, 4), torch.randn(2, 8)
    state = torch.zeros({"recurrence": (2, 8), "convolution": (2, 3, 8), "scan": (2, 8, 4)}[kind])
    over = {"recurrence": lambda: S.gated_recurrence(x, x, plan, state), "convolution": lambda: S.short_convolution(x, taps, None, plan, state), "scan": lambda: S.selective_scan(x, x, decay, b, b, plan, state)}[kind]
    step = {"recurrence": lambda: S.gated_recurrence_step(one, one, state), "convolution": lambda: S.short_convolution_step(one, taps, None, state),
            "scan": lambda: S.selective_scan_step(one, one, decay, b[:2], b[:2], state)}[kind]
    y, _ = over()
    torch.autograd.grad(y.sum(), x)
    y, _ = over()
    step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)
    with torch.inference_mode():                            # where nothing is counted
        state = torch.zeros_like(state)
        step()


def test_far_queries_of_one_long_row_among_short_ones():
    """Sinks of long rows have their far queries worked out apart, however short the rows beside them are on average; those of short rows only where there are few sinks."""
    lib = _abi.lib()
    ok = dict(dtype=2, heads_q=8, heads_k=2, dim=64, window=256, scale=0.125)
    need = lambda sinks, **plan: lib.nuka_b200_attention_sinks_workspace(ctypes.byref(_abi.AttentionDesc(**{**ok, "plan": _plan(**plan)})), sinks)
    for sinks in (4, 16, 17, 64):
        assert need(sinks, tokens=17384, rows=21, length=0) > 0, sinks
        assert need(sinks, tokens=20000, rows=5, length=4000) > 0 and need(sinks, tokens=16384, rows=1, length=0) > 0
        assert (need(sinks, tokens=20000, rows=40, length=500) > 0) == (sinks <= 16)
    assert need(65, tokens=16384, rows=1, length=0) == 0
    ok["window"] = 2 ** 63 - 1                              # without end
    assert need(4, tokens=16384, rows=1, length=0) == 0


@pytest.mark.parametrize("length", [1, 2, 3, 5, 7, 8, 15, 24, 64])
@pytest.mark.parametrize("states", [8, 16, 64])
def test_what_is_kept_for_short_rows(length, states):
    """States before each fourth (up to 8 states) or eighth token, in 32 bits; chunks of tokens begin anew with rows of eight tokens and more, and with every sixteen or so of shorter ones."""
    rows, channels, chunk = 840, 512, 4 if states == 8 else 8
    kept = _abi.lib().nuka_b200_scan_kept(_plan(tokens=rows * length, rows=rows, length=length), channels, states)
    together = length if length >= 8 else -(-16 // length) * length
    assert kept == -(-rows * length // together) * -(-together // chunk) * channels * states * 4
    assert kept <= 2 * rows * length * channels * states * 4 // chunk
