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
