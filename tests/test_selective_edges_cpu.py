"""What the selective operators' entries refuse at the ends of what they take, without a GPU."""
import ctypes

import pytest

pytest.importorskip("torch")
from nuka import _abi  # noqa: E402

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
