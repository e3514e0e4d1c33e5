"""Calls of the selective operators at the ends of what they take: no channels."""
import pytest

torch = pytest.importorskip("torch")
import nuka  # noqa: E402,F401
from nuka import sequence as S  # noqa: E402

pytestmark = pytest.mark.gpu


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
