"""Attention of one token of each env over its cached history, against the definition in 64 bits and against attention over whole episodes.

Bounds: as for attention over episodes: one rounding of the output, one of each probability (half a unit u each: u |o| + u sum p |v|), 32-bit work 2^-15 of sum p |v|."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")
import nuka  # noqa: E402
from nuka import _abi, sequence as S  # noqa: E402

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, dtype=torch.bfloat16, scale=1.0):
    return torch.empty(shape, device="cuda").normal_(0.0, scale, generator=gen).to(dtype)


def _reference(q, keys, values, held, scale):
    """Over keys as they lie in the cache after the token was written: the order does not matter."""
    envs, cap, hk, d = keys.shape
    group = q.shape[1] // hk
    out, size = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for e in range(envs):
        n = int(held[e])
        for h in range(q.shape[1]):
            v = values[e, :n, h // group].double()
            p = torch.softmax(keys[e, :n, h // group].double() @ q[e, h].double() * scale, 0)
            out[e, h], size[e, h] = p @ v, p @ v.abs()
    return out, size


def _check(gen, envs, cap, hq, hk, d, dtype, positions, scale=None):
    keys, values = _normal(gen, envs, cap, hk, d, dtype=dtype), _normal(gen, envs, cap, hk, d, dtype=dtype)
    position = torch.tensor(positions, dtype=torch.int32, device="cuda")
    for e, n in enumerate(positions):                      # what an earlier episode left there may be anything
        keys[e, max(n, 0):], values[e, max(n, 0):] = math.nan, math.inf
    cache = S.HistoryCache(envs, cap, hk, d, dtype, buffers=(keys, values, position))
    q, k, v = _normal(gen, envs, hq, d, dtype=dtype, scale=1.5), _normal(gen, envs, hk, d, dtype=dtype), _normal(gen, envs, hk, d, dtype=dtype)
    want_keys, want_values = keys.clone(), values.clone()
    at = position.clamp(min=0).long()
    want_keys[torch.arange(envs), at % cap], want_values[torch.arange(envs), at % cap] = k, v
    for _ in range(2):                                     # the second time finds its own token in the cache, and workspaces as they were
        o = S.history_attention(q, k, v, cache, scale)
        bits = lambda x: x.view(torch.int16)
        assert torch.equal(bits(cache.keys), bits(want_keys)) and torch.equal(bits(cache.values), bits(want_values))
        want, size = _reference(q, want_keys, want_values, (at + 1).clamp(max=cap), d ** -0.5 if scale is None else scale)
        assert torch.isfinite(o).all()
        off = (o.double() - want).abs() - (UNIT[dtype] * (want.abs() + size) + 2.0 ** -15 * size + (2.0 ** -24 if dtype is torch.float16 else 0))
        assert off.max().item() <= 0, off.max().item()
    return o


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,d", [(8, 2, 64), (1, 1, 128), (3, 3, 32), (12, 1, 64), (40, 2, 64), (6, 2, 96), (2, 1, 8), (4, 4, 120)])
def test_rings_before_at_and_after_they_come_round(dtype, hq, hk, d):
    cap = 50
    _check(_gen(hq + d), 9, cap, hq, hk, d, dtype, [-1, 0, 1, 15, 16, 49, 50, 99, 1000003])


@pytest.mark.parametrize("cap", [1, 16, 64, 200, 5000])
@pytest.mark.parametrize("envs", [1, 3])
def test_long_and_short_histories_of_few_envs(cap, envs):
    for n in (0, 1, cap // 2, cap - 1, cap, 2 * cap + 3):
        _check(_gen(cap + n), envs, cap, 4, 2, 64, torch.bfloat16, [max(0, n - e) for e in range(envs)])


def test_sharp_and_flat_softmax():
    _check(_gen(1), 2, 700, 2, 1, 64, torch.bfloat16, [699, 300], scale=3.0)
    _check(_gen(2), 2, 700, 2, 1, 128, torch.float16, [699, 300], scale=1e-4)


def test_acting_follows_attention_over_the_rollout():
    """Token by token with a cache gives what attention over the whole rollout with the cache's capacity as its window gives, through ends of episodes."""
    gen, envs, steps, cap = _gen(3), 6, 70, 16
    done = torch.rand((envs, steps), generator=gen, device="cuda") < 0.06
    q, k, v = _normal(gen, envs, steps, 4, 64), _normal(gen, envs, steps, 2, 64), _normal(gen, envs, steps, 2, 64)
    want = S.episode_attention(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), S.Episodes.from_done(done), window=cap).view(envs, steps, 4, 64)
    cache = S.HistoryCache(envs, cap, 2, 64)
    plan = S.Episodes.from_done(done)
    for t in range(steps):
        cache.advance(done[:, t - 1] if t else None)
        assert torch.equal(cache.position, plan.positions.view(envs, steps)[:, t])
        o = S.history_attention(q[:, t], k[:, t], v[:, t], cache)
        # two kernels' roundings of outputs and probabilities: 4 units of values up to 4 in all
        assert (o.float() - want[:, t].float()).abs().max().item() <= 4 * UNIT[torch.bfloat16] * 4


def test_same_bits_and_streams_and_strides():
    gen = _gen(4)
    keys, values, position = _normal(gen, 2, 3000, 2, 64), _normal(gen, 2, 3000, 2, 64), torch.tensor([2500, 77], dtype=torch.int32, device="cuda")
    both = _normal(gen, 2, 9, 64)
    q, k, v = both[:, :4], both[:, 4:6], both[:, 6:8]
    cache = S.HistoryCache(2, 3000, 2, 64, buffers=(keys, values, position))
    first = S.history_attention(q, k, v, cache)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(S.history_attention(q.contiguous(), k.contiguous(), v.contiguous(), cache), first)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(S.history_attention(q[:, :1].expand(-1, 4, -1), k, v, cache)[:, 0], first[:, 0])


def test_a_cache_beyond_32_bit_offsets():
    """Places of a cache whose offset passes 2^32 bytes and 2^31 values."""
    envs, cap, hk, d = 3, 8 << 20, 1, 128
    free, _ = torch.cuda.mem_get_info()
    if free < 20 << 30:
        pytest.skip("needs 13 GB")
    keys, values = (torch.empty(envs, cap, hk, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    position = torch.tensor([5, 100, cap - 1], dtype=torch.int32, device="cuda")
    gen = _gen(5)
    for e, n in enumerate((5, 100, cap - 1)):
        if e < 2:
            keys[e, :n], values[e, :n] = _normal(gen, n, hk, d), _normal(gen, n, hk, d)
        else:
            keys[e].zero_()
            values[e].zero_()
    keys[2, cap - 300:cap - 1], values[2, cap - 300:cap - 1] = _normal(gen, 299, hk, d, scale=4.0), _normal(gen, 299, hk, d)
    q, k, v = _normal(gen, envs, 2, d, scale=4.0), _normal(gen, envs, hk, d, scale=4.0), _normal(gen, envs, hk, d)
    o = S.history_attention(q, k, v, S.HistoryCache(envs, cap, hk, d, buffers=(keys, values, position)), scale=1.0)
    assert torch.equal(keys[2, cap - 1], k[2]) and torch.equal(values[2, cap - 1], v[2])
    # the far env: its 8 M zero keys score 0, the last 300 up to hundreds
    kk, vv = keys[2, cap - 300:, 0].double(), values[2, cap - 300:, 0].double()
    for h in range(2):
        s = kk @ q[2, h].double()
        top = max(s.max().item(), 0.0)
        w = torch.exp(s - top)
        total = w.sum() + (cap - 300) * math.exp(-top)
        want, size = w @ vv / total, w @ vv.abs() / total
        # scores of hundreds: 2^-24 of them in the exponent
        assert ((o[2, h].double() - want).abs() <= UNIT[torch.bfloat16] * (want.abs() + size) + 2.0 ** -12 * size).all()


def test_wrong_arguments_are_refused():
    cache = S.HistoryCache(2, 8, 2, 64)
    q, k = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    for bad in (lambda: S.history_attention(q[:1], k, k, cache), lambda: S.history_attention(q[:, :3], k, k, cache), lambda: S.history_attention(q, k[:, :1], k[:, :1], cache),
                lambda: S.history_attention(q.half(), k.half(), k.half(), cache), lambda: S.history_attention(q, q, q, cache), lambda: S.HistoryCache(2, 0, 2, 64), lambda: S.HistoryCache(2, 8, 2, 64, torch.float32),
                lambda: S.HistoryCache(2, 8, 2, 64, buffers=(cache.keys, cache.values[:, :4], cache.position)), lambda: cache.advance(torch.zeros(3, dtype=torch.bool, device="cuda")),
                lambda: S.HistoryCache(2, 8, 2, 64, position=cache.position.long())):
        with pytest.raises(ValueError):
            bad()
    odd = S.HistoryCache(2, 8, 2, 60)
    with pytest.raises(nuka.NukaError):
        S.history_attention(q[:, :, :60], k[:, :, :60], k[:, :, :60], odd)
    with pytest.raises(nuka.NukaError):
        S.history_attention(q, k, k, cache, scale=-1.0)
    lib = _abi.lib()
    x = torch.zeros(1 << 16, dtype=torch.bfloat16, device="cuda")
    at = x.data_ptr()
    ok = dict(dtype=2, envs=2, capacity=256, heads_q=4, heads_k=2, dim=64, scale=1.0, q=at, k=at, v=at, q_stride=256, q_head_stride=64, k_stride=128, k_head_stride=64, v_stride=128, v_head_stride=64,
              keys=at, values=at, position=at, out=at)
    call = lambda **change: lib.nuka_b200_history(ctypes.byref(_abi.HistoryDesc(**{**ok, **change})), None)
    for change in (dict(q=None), dict(keys=at + 8), dict(position=None), dict(heads_k=3), dict(capacity=0), dict(q_stride=4), dict(k_stride=-8), dict(), dict(workspace=at, workspace_bytes=16)):
        assert call(**change) == _abi.INVALID_ARG, change                       # the last two: no workspace, too small a one
    assert call(dtype=0) == 7 and call(dim=136) == 7 and lib.nuka_b200_history(None, None) == _abi.INVALID_ARG
    assert lib.nuka_b200_history_advance(None, None, 2, None) == _abi.INVALID_ARG and lib.nuka_b200_history_advance(None, None, -1, None) == _abi.INVALID_ARG
