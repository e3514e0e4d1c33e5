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
