"""Gradients of first tokens that stay where some rows' far queries are worked out apart and others' by the keys' kernel: long rows beside short ones, as many sinks as there may be, against the definition in 64 bits."""
import pytest

torch = pytest.importorskip("torch")
import nuka  # noqa: E402,F401
from test_gpu_sinks import check  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sinks", [16, 17, 40, 64, 65])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_rows_among_short_ones(check, sinks, dim):  # noqa: F811
    """Of 1500, 30 and 1131 tokens behind the window, and of 1023, 1024 and 1025 behind the tile that the sinks lie in or begin in."""
    check([50, 3, 1532, 62, 1, 1163, 0, 90], 32, sinks, 4, 2, dim)
    check([1023 + 128 + 31, 1024 + 128 + 31, 1025 + 128 + 31], 32, sinks, 2, 2, dim, torch.float16)


def test_more_rows_than_places(check):  # noqa: F811
    check([1200] * 2 + [70] * 30 + [1200], 20, 33, 16, 1, 64)
