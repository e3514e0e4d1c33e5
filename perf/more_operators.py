"""Further sequence operators of a policy with memory (``nuka.sequence``): a selective state space layer, and attention whose window keeps an episode's first tokens.

A token is one control step of one env.  Tokens lie in rows, one behind the other: a row is an env's part of a rollout (with episodes
that end inside it) or a whole episode.  Kinds of case:

    convolution        the short causal convolution over each episode, channel by channel, forwards, or forwards and backwards
    convolution_step   its form for one token of every env, on the policy's state
    scan               the selective scan over each episode, forwards, or forwards and backwards
    scan_step          its form for one token of every env
    attention          causal attention over the last tokens of the episode and its first ones, forwards, or forwards and backwards
    history            attention of one token of every env over a cache that keeps the episode's first tokens beside the last ones

The plain form is the formulas in elementary tensor operations in 32 bits, attention on rows padded to the longest.
"""
import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.getcwd(), "nuka-physics_b200"))

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "f32": 4}


def listed():
    def rows(kind, name, rows, tokens, episode, dtype, train, **more):
        return {"name": name, "kind": kind, "rows": rows, "tokens": tokens, "episode": episode, "dtype": dtype, "train": train, **more}

    return [
        # one robot under a trained policy: all latency
        {"name": "convolution-step-1", "kind": "convolution_step", "envs": 1, "channels": 512, "width": 4, "dtype": "f32"},
        # the training batch of a policy 256 wide, its layers twice as wide inside: 4096 envs, 24 control steps each, episodes of up to 1000 steps end inside
        rows("convolution", "convolution-train-4096x24", 4096, 4096 * 24, 1000, "bf16", True, channels=512, width=4),
        # a few very long recordings of different lengths
        rows("convolution", "convolution-train-long", 3, 131071, 0, "fp16", True, channels=1024, width=4),
        # one robot: latency again, with the layer's states
        {"name": "scan-step-1", "kind": "scan_step", "envs": 1, "channels": 512, "states": 16, "dtype": "f32"},
        # one token for each env of a standard batch while the policy acts
        {"name": "scan-step-4096", "kind": "scan_step", "envs": 4096, "channels": 512, "states": 16, "dtype": "bf16"},
        # the training batch
        rows("scan", "scan-train-4096x24", 4096, 4096 * 24, 1000, "bf16", True, channels=512, states=16),
        # long recordings of different lengths, learnt from end to end
        rows("scan", "scan-train-long", 3, 32749, 0, "bf16", True, channels=1024, states=16),
        # values of a recorded batch of an odd size, no gradient, few states
        rows("scan", "scan-forward-1000x37", 1000, 37000, 200, "f32", False, channels=200, states=8),
        # whole episodes of different lengths, up to the 1000 control steps of a full one; the first steps of each stay visible
        rows("attention", "attention-train-episodes", 40, 20011, 0, "bf16", True, heads_q=8, heads_k=2, dim=64, window=64, sinks=4),
        # two long recordings with a wide window
        rows("attention", "attention-train-long", 2, 16384, 0, "bf16", True, heads_q=8, heads_k=2, dim=128, window=1024, sinks=16),
        # one robot with a long history: latency, few heads
        {"name": "history-1x8192", "kind": "history", "envs": 1, "capacity": 8192, "sinks": 16, "heads_q": 8, "heads_k": 2, "dim": 64, "dtype": "bf16"},
        # a standard batch acting with 256 control steps of history, rings that have come round among them
        {"name": "history-4096x256", "kind": "history", "envs": 4096, "capacity": 256, "sinks": 4, "heads_q": 8, "heads_k": 2, "dim": 64, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["convolution", "convolution", "convolution_step", "scan", "scan", "scan", "scan_step", "attention", "attention", "attention", "history"])
    sixteen = rng.choice(["bf16", "bf16", "fp16"])
    dtype = rng.choice(["f32", sixteen, sixteen])
    if kind == "convolution_step":
        return {"kind": kind, "envs": _log(rng, 1, 8192), "channels": 8 * _log(rng, 4, 128), "width": rng.choice([2, 3, 4, 4]), "dtype": dtype}
    if kind == "scan_step":
        envs, channels = _log(rng, 1, 8192), 8 * _log(rng, 4, 128)
        return {"kind": kind, "envs": min(envs, (1 << 21) // channels), "channels": channels, "states": rng.choice([8, 16, 16, 32, 5]), "dtype": dtype}
    if kind == "history":
        capacity = _log(rng, 32, 16384)
        return {"kind": kind, "envs": _log(rng, 1, max(1, min(4096, (1 << 20) // capacity))), "capacity": capacity, "sinks": min(capacity - 1, _log(rng, 1, 64)), "heads_k": rng.choice([1, 2]),
                "heads_q": 2 * rng.choice([1, 2, 4]), "dim": rng.choice([32, 64, 64, 128]), "dtype": sixteen}
    train, rows = rng.random() < 0.7, _log(rng, 1, 4096)
    case = {"kind": kind, "rows": rows, "tokens": max(rows, _log(rng, 64, 98304)), "train": train, "episode": 0, "dtype": dtype}
    if kind in ("convolution", "scan"):
        # rows of one length with episodes that end inside, or whole episodes
        case["episode"] = rng.choice([0, _log(rng, 16, 1000)])
        channels = 8 * _log(rng, 4, 128)
        if kind == "convolution":
            case.update(channels=channels, width=rng.choice([2, 3, 4, 4]))
        else:
            states = rng.choice([8, 16, 16, 32, 5])
            case.update(channels=channels, states=states)
            # no more values of the state over all tokens than the listed ones have, and no longer a chain
            case["tokens"] = max(64, min(case["tokens"], 4096 * 24 * 512 * 16 // (channels * max(states, 16)), 32768 if rows < 8 else 98304))
            case["rows"] = rows = min(rows, case["tokens"])
        if case["episode"]:
            case["tokens"] = rows * max(1, case["tokens"] // rows)
        return case
    group, heads_k = rng.choice([1, 2, 4]), rng.choice([1, 2, 4])
    # the plain form holds rows x longest^2 scores of every head: keep to what the listed ones have
    while heads_k * group * max(_lengths(case["rows"], case["tokens"], 0)) ** 2 * case["rows"] > 1 << 30:
        case["rows"], case["tokens"] = max(1, case["rows"] // 2), max(1, case["tokens"] // 2)
    return {**case, "heads_q": heads_k * group, "heads_k": heads_k, "dim": rng.choice([32, 64, 64, 128]), "window": _log(rng, 16, 1024), "sinks": _log(rng, 1, 64), "dtype": sixteen}


def _lengths(rows, tokens, episode):
    """Lengths of the rows, longest first: all alike where episodes end inside them, else spread over a factor of about ten, one empty."""
    if episode:
        return [tokens // rows] * rows
    if tokens % rows == 0 and tokens // rows < 2 or rows == 1:
        return [tokens // rows] * rows
    rng = random.Random(rows * 1000003 + tokens)
    share = [0.1 + rng.random() for _ in range(rows - 1)] + [0.0]
    total = sum(share)
    lengths = [int(tokens * s / total) for s in share]
    lengths[0] += tokens - sum(lengths)
    return sorted(lengths, reverse=True)


def _rows(case, seed):
    """The rows in an order of this seed: their offsets, at which of their tokens an episode begins (the first always), and the flags of episodes' ends."""
    rng = random.Random(seed)
    lengths = _lengths(case["rows"], case["tokens"], case["episode"])
    rng.shuffle(lengths)
    offsets = [0]
    for n in lengths:
        offsets.append(offsets[-1] + n)
    offsets = torch.tensor(offsets, dtype=torch.int32)
    start = torch.zeros(case["tokens"], dtype=torch.bool)
    start[offsets[:-1].long().clamp(max=case["tokens"] - 1)[offsets[1:] > offsets[:-1]]] = True
    done = None
    if case["episode"]:
        rows, length, episode = case["rows"], case["tokens"] // case["rows"], case["episode"]
        phase = torch.tensor(rng.sample(range(rows), rows)) * episode // rows           # how far into its episode each env is
        done = (torch.arange(length)[None, :] + phase[:, None]) % episode == episode - 1
        start.view(rows, length)[:, 1:] |= done[:, :-1]
    return offsets, start, done


def _place(position, capacity, sinks):
    """Where the cache keeps the token number `position` of an episode."""
    return torch.where(position < sinks, position, sinks + (position - sinks) % (capacity - sinks))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=dtype):
        return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(shift, scale, generator=gen).to(dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    kind, s = case["kind"], {"case": case}
    if kind == "history":
        n, cap, sinks, hq, hk, d = (case[k] for k in ("envs", "capacity", "sinks", "heads_q", "heads_k", "dim"))
        # histories between empty and twice the ring's length, in an order of this seed
        position = (torch.arange(n, device="cuda") * 2 + 1) * cap // n
        position = position[torch.randperm(n, generator=gen, device="cuda")].int()
        s.update(q=normal(n, hq, d, scale=1.5), k=normal(n, hk, d), v=normal(n, hk, d), position=position)
        held = (torch.arange(cap, device="cuda")[None, :] < position[:, None])[:, :, None, None]
        s["keys"], s["values"] = (torch.where(held, normal(n, cap, hk, d), torch.zeros((), dtype=dtype, device="cuda")) for _ in range(2))
        if own:
            from nuka import sequence
            s["cache"] = sequence.HistoryCache(n, cap, hk, d, dtype, buffers=(s["keys"], s["values"], position), sinks=sinks)
        return s
    if kind in ("convolution", "convolution_step"):
        c, width = case["channels"], case["width"]
        s.update(weight=normal(c, width, scale=width ** -0.5, dtype=torch.float32), bias=normal(c, scale=0.2, dtype=torch.float32))
    if kind in ("scan", "scan_step"):
        c, n = case["channels"], case["states"]
        # rates as such layers begin with: time constants of 1 to 1000 control steps, states that fade 1 to N times as fast
        rate = torch.exp(uniform(c) * math.log(100.0) + math.log(0.001))
        s.update(decay=-torch.arange(1, n + 1, device="cuda") * (0.8 + 0.4 * uniform(c, n)), skip=normal(c, scale=0.3, shift=1.0, dtype=torch.float32), delta_bias=torch.log(torch.expm1(rate)))
    if kind in ("convolution_step", "scan_step"):
        n = case["envs"]
        s.update(x=normal(n, c), fresh=uniform(n) < 0.01)
        if kind == "convolution_step":
            s["state"] = normal(n, width - 1, c)
        else:
            s.update(delta=normal(n, c), gate=normal(n, c), b=normal(n, case["states"]), c=normal(n, case["states"]), state=normal(n, c, case["states"], dtype=torch.float32, scale=0.1))
        return s
    offsets, start, done = _rows(case, seed)
    s["offsets"], s["start"] = offsets.cuda(), start.cuda()
    if own:
        from nuka import sequence
        s["plan"] = sequence.Episodes.from_done(done.cuda()) if done is not None else sequence.Episodes.from_offsets(s["offsets"], case["tokens"])
    t = case["tokens"]
    if kind == "convolution":
        both = normal(t, 2 * c)                                     # one projection gives the convolution's input and the layer's gate
        s.update(x=both[:, :c], initial=normal(case["rows"], width - 1, c))
        if case["train"]:
            s["dy"] = normal(t, c)
    elif kind == "scan":
        n = case["states"]
        both = normal(t, 2 * c)
        narrow = normal(t, 2 * n + 16)                              # one projection gives what the rates are made of, B and C
        s.update(x=normal(t, c), gate=both[:, c:], delta=normal(t, c), b=narrow[:, 16:16 + n], c=narrow[:, 16 + n:], initial=normal(case["rows"], c, n, dtype=torch.float32, scale=0.1))
        if case["train"]:
            s["dy"] = normal(t, c)
    else:
        hq, hk, d = case["heads_q"], case["heads_k"], case["dim"]
        both = normal(t, (hq + 2 * hk) * d, scale=1.2)              # one projection gives queries, keys and values
        for name, low, n in (("q", 0, hq), ("k", hq, hk), ("v", hq + hk, hk)):
            s[name] = both[:, low * d:(low + n) * d].unflatten(1, (n, d))
        if case["train"]:
            s["do"] = normal(t, hq, d)
    if case["train"]:
        for name in NAMES[kind]:
            s[name] = s[name].detach().requires_grad_()
    return s


# what has a gradient
NAMES = {"convolution": ("x", "weight", "bias", "initial"), "scan": ("x", "delta", "decay", "b", "c", "skip", "gate", "delta_bias", "initial"), "attention": ("q", "k", "v")}


# ---- the plain form ----------------------------------------------------------------------------------------------
def _silu(x):
    sigmoid = torch.sigmoid(x)
    return x * sigmoid, sigmoid * (1 + x * (1 - sigmoid))           # and its derivative


def _first(s):
    """The index of each token's episode's first token."""
    at = torch.arange(s["start"].numel(), device="cuda")
    return torch.cummax(torch.where(s["start"], at, 0), 0).values


def _begins(s):
    """The rows that hold tokens, the first token of each and the last."""
    offsets = s["offsets"].long()
    rows = (offsets[1:] > offsets[:-1]).nonzero()[:, 0]
    return rows, offsets[rows], offsets[rows + 1] - 1


def _plain_convolution(s):
    case = s["case"]
    width, t, dtype = case["width"], case["tokens"], s["x"].dtype
    x, weight, initial = s["x"].float(), s["weight"], s["initial"].float()
    rows, begins, ends = _begins(s)
    # all tokens behind the rows' initial ones; `at[k]`: which of them each token's k-th last input is, number 0 a row of zeros
    inputs = torch.cat([torch.zeros_like(x[:1]), initial.flatten(0, 1), x])
    token, first, base = torch.arange(t, device="cuda"), _first(s), 1 + case["rows"] * (width - 1)
    row = torch.zeros(t, dtype=torch.long, device="cuda")
    row[begins] = rows
    row = torch.cummax(row, 0).values
    whole = torch.zeros(t, dtype=torch.bool, device="cuda")         # the episode began the row
    whole[begins] = True
    whole = whole[first]

    def index(k):
        before = token - k - first
        from_initial = 1 + row * (width - 1) + width - 1 + before
        return torch.where(before >= 0, base + token - k, torch.where(whole & (before >= 1 - width), from_initial, 0))

    at = [index(k) for k in range(width)]
    total = s["bias"] + sum(weight[:, width - 1 - k] * inputs[at[k]] for k in range(width))
    y, slope = _silu(total)
    state = initial.clone()
    state[rows] = torch.stack([inputs[index(k)[ends]] for k in range(width - 2, -1, -1)], 1)
    out = {"y": y.to(dtype), "state": state.to(dtype)}
    if case["train"]:
        ds = s["dy"].float() * slope
        dinputs, dweight = torch.zeros_like(inputs), torch.zeros_like(weight)
        for k in range(width):
            dweight[:, width - 1 - k] = (ds * inputs[at[k]]).sum(0)
            real = at[k] > 0
            dinputs[at[k][real]] += weight[:, width - 1 - k] * ds[real]         # no token is the k-th last input of two
        out.update(dx=dinputs[base:].to(dtype), dweight=dweight, dbias=ds.sum(0), dinitial=dinputs[1:base].view_as(initial).to(dtype))
    return out


def _plain_convolution_step(s):
    state = torch.where(s["fresh"][:, None, None], 0.0, s["state"].float())
    window = torch.cat([state, s["x"].float()[:, None]], 1)
    y, _ = _silu(s["bias"] + (window * s["weight"].t()).sum(1))
    s["state"].copy_(window[:, 1:])
    return {"y": y.to(s["x"].dtype), "state": s["state"]}


def _scan(a, b, longest):
    """h with h_t = a_t h_{t-1} + b_t down the first dimension, by doubling; no chain is longer than `longest`."""
    step = 1
    a, b = a.clone(), b.clone()
    while step < min(longest, a.shape[0]):
        b[step:] += a[step:] * b[:-step]                            # the right side is worked out whole before the left changes
        a[step:] = a[step:] * a[:-step]
        step *= 2
    return b


def _plain_scan(s):
    case, dtype = s["case"], s["x"].dtype
    x, delta, b, c, z = (s[name].float() for name in ("x", "delta", "b", "c", "gate"))
    longest = max(_lengths(case["rows"], case["tokens"], case["episode"]))
    rows, begins, ends = _begins(s)
    u = delta + s["delta_bias"]
    dt = torch.clamp(u, min=0.0) + torch.log1p(torch.exp(-u.abs()))
    a = torch.exp(dt[:, :, None] * s["decay"])
    into = (dt * x)[:, :, None] * b[:, None]
    into[begins] += a[begins] * s["initial"][rows]
    lead = torch.where(s["start"][:, None, None], 0.0, a)
    h = _scan(lead, into, longest)
    del into
    y = (h * c[:, None]).sum(-1) + s["skip"] * x
    silu, slope = _silu(z)
    state = s["initial"].clone()
    state[rows] = h[ends]
    out = {"y": (y * silu).to(dtype), "state": state}
    if case["train"]:
        do = s["dy"].float()
        dy = do * silu
        lead = torch.cat([lead[1:], torch.zeros_like(lead[:1])])    # a_{t+1}, nothing across an episode's end
        grad = _scan(lead.flip(0), (dy[:, :, None] * c[:, None]).flip(0), longest).flip(0)
        del lead
        dc = (dy[:, :, None] * h).sum(1)
        before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
        before = torch.where(s["start"][:, None, None], 0.0, before)
        before[begins] = s["initial"][rows]
        dinitial = torch.zeros_like(s["initial"])
        dinitial[rows] = (a * grad)[begins]
        part = before.mul_(a).mul_(grad)                            # the gradient of dt times the decay
        dinto = (grad * b[:, None]).sum(-1)
        ddelta = ((part * s["decay"]).sum(-1) + dinto * x) * torch.sigmoid(u)
        out.update(dx=(dinto * dt + s["skip"] * dy).to(dtype), ddelta=ddelta.to(dtype), ddecay=(part * dt[:, :, None]).sum(0), db=(grad * (dt * x)[:, :, None]).sum(1).to(dtype), dc=dc.to(dtype),
                   dskip=(dy * x).sum(0), dgate=(do * y * slope).to(dtype), ddelta_bias=ddelta.sum(0), dinitial=dinitial)
    return out


def _plain_scan_step(s):
    x, b, c, z = (s[name].float() for name in ("x", "b", "c", "gate"))
    u = s["delta"].float() + s["delta_bias"]
    dt = torch.clamp(u, min=0.0) + torch.log1p(torch.exp(-u.abs()))
    before = torch.where(s["fresh"][:, None, None], 0.0, s["state"])
    s["state"].copy_(torch.exp(dt[:, :, None] * s["decay"]) * before + (dt * x)[:, :, None] * b[:, None])
    y = (s["state"] * c[:, None]).sum(-1) + s["skip"] * x
    return {"y": (y * _silu(z)[0]).to(s["x"].dtype), "state": s["state"]}


def _plain_attention(s):
    case, offsets = s["case"], s["offsets"].long()
    hq, hk, d, dtype = case["heads_q"], case["heads_k"], case["dim"], s["q"].dtype
    at = offsets[:-1, None] + torch.arange(max(_lengths(case["rows"], case["tokens"], case["episode"])), device="cuda")
    held = at < offsets[1:, None]
    at = at.clamp(max=case["tokens"] - 1)
    n, length = at.shape
    first, group, scale = _first(s)[at], hq // hk, d ** -0.5

    def rows(x):                                                    # tokens x heads x dim -> row, key head, (head of the group, token), dim
        x = torch.where(held[:, :, None, None], x.float()[at], 0.0)
        return x.view(n, length, hk, -1, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)

    def tokens(x):
        return x.view(n, hk, -1, length, d).permute(0, 3, 1, 2, 4).reshape(n, length, -1, d)[held].to(dtype)

    seen = (at[:, None, :] <= at[:, :, None]) & (at[:, None, :] >= first[:, :, None]) & held[:, None, :]
    seen &= (at[:, None, :] > at[:, :, None] - case["window"]) | (at[:, None, :] < first[:, :, None] + case["sinks"])
    q, k, v = rows(s["q"]), rows(s["k"]), rows(s["v"])
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).view(n, hk, group, length, length)
    p.masked_fill_(~seen[:, None, None], -1e30)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    p = p.view(n, hk, group * length, length)
    o = torch.matmul(p, v)
    out = {"o": tokens(o)}
    if case["train"]:
        do = rows(s["do"])
        out["dv"] = tokens(torch.matmul(p.transpose(-1, -2), do))
        ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out["dq"] = tokens(torch.matmul(ds, k))
        out["dk"] = tokens(torch.matmul(ds.transpose(-1, -2), q))
    return out


def _plain_history(s):
    case = s["case"]
    n, cap, hk, d = case["envs"], case["capacity"], case["heads_k"], case["dim"]
    env, position = torch.arange(n, device="cuda"), s["position"].long()
    place = _place(position, cap, case["sinks"])
    s["keys"][env, place] = s["k"]
    s["values"][env, place] = s["v"]
    held = torch.arange(cap, device="cuda") <= position[:, None]
    q = s["q"].float().view(n, hk, -1, d)
    p = torch.matmul(q, s["keys"].float().permute(0, 2, 3, 1)) * d ** -0.5
    p = torch.where(held[:, None, None], p, -1e30)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p, s["values"].float().transpose(1, 2))
    return {"o": o.reshape(n, -1, d).to(s["q"].dtype), "keys": s["keys"], "values": s["values"]}


def _own(s):
    from nuka import sequence
    case, kind = s["case"], s["case"]["kind"]
    if kind == "convolution_step":
        return {"y": sequence.short_convolution_step(s["x"], s["weight"], s["bias"], s["state"], s["fresh"], silu=True), "state": s["state"]}
    if kind == "scan_step":
        y = sequence.selective_scan_step(s["x"], s["delta"], s["decay"], s["b"], s["c"], s["state"], s["fresh"], skip=s["skip"], gate=s["gate"], delta_bias=s["delta_bias"])
        return {"y": y, "state": s["state"]}
    if kind == "history":
        return {"o": sequence.history_attention(s["q"], s["k"], s["v"], s["cache"]), "keys": s["keys"], "values": s["values"]}
    if kind == "convolution":
        y, state = sequence.short_convolution(s["x"], s["weight"], s["bias"], s["plan"], s["initial"], silu=True)
        out, by = {"y": y.detach(), "state": state.detach()}, "dy"
    elif kind == "scan":
        y, state = sequence.selective_scan(s["x"], s["delta"], s["decay"], s["b"], s["c"], s["plan"], s["initial"], skip=s["skip"], gate=s["gate"], delta_bias=s["delta_bias"])
        out, by = {"y": y.detach(), "state": state.detach()}, "dy"
    else:
        y = sequence.episode_attention(s["q"], s["k"], s["v"], s["plan"], window=case["window"], sinks=case["sinks"])
        out, by = {"o": y.detach()}, "do"
    if case["train"]:
        grads = torch.autograd.grad(y, [s[name] for name in NAMES[kind]], s[by])
        out.update(zip(["d" + name for name in NAMES[kind]], grads))
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return globals()["_plain_" + state["case"]["kind"]](state)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------
def _exact_convolution(s):
    """Token after token, the rows side by side; gradients by automatic differentiation of one channel block's sums at a time."""
    case, offsets = s["case"], s["offsets"].tolist()
    width, starts = case["width"], s["start"].cpu()
    x, weight, bias, initial = (s[name].detach().double() for name in ("x", "weight", "bias", "initial"))
    # each row behind its initial tokens, each episode inside it behind zeros: then nothing has to be looked up
    where, source, row_of = [], [], []
    place = 0
    lasts = {}
    for row, (low, high) in enumerate(zip(offsets, offsets[1:])):
        begins = [low] + (low + 1 + starts[low + 1:high].nonzero()[:, 0]).tolist() if high > low else []
        for k, begin in enumerate(begins):
            end = begins[k + 1] if k + 1 < len(begins) else high
            row_of.append((place, row if k == 0 else -1))
            place += width - 1
            where.append(torch.arange(place, place + end - begin))
            source.append(torch.arange(begin, end))
            place += end - begin
        if high > low:
            lasts[row] = place
    where, source = torch.cat(where).cuda(), torch.cat(source).cuda()
    heads = torch.tensor([p for p, r in row_of if r >= 0]).cuda()
    of_row = torch.tensor([r for _, r in row_of if r >= 0]).cuda()
    steps = torch.arange(width - 1, device="cuda")
    out = {name: torch.zeros_like(v) for name, v in (("y", x), ("state", initial), ("dx", x), ("dweight", weight), ("dbias", bias), ("dinitial", initial))}
    out["state"].copy_(initial)
    block = max(1, (1 << 27) // max(1, place))
    for low in range(0, case["channels"], block):
        cut = slice(low, low + block)
        leaves = [v.clone().requires_grad_(case["train"]) for v in (x[:, cut], weight[cut], bias[cut], initial[:, :, cut])]
        line = torch.zeros(place, leaves[0].shape[1], dtype=torch.float64, device="cuda")
        line = line.index_put((heads[:, None] + steps,), leaves[3][of_row]).index_put((where,), leaves[0][source])
        total = leaves[2] + sum(leaves[1][:, j] * line[where - (width - 1) + j] for j in range(width))
        y = total / (1 + torch.exp(-total))
        out["y"][source, cut] = y.detach()
        some = torch.tensor(list(lasts), device="cuda")
        out["state"][some, :, cut] = line.detach()[torch.tensor(list(lasts.values()), device="cuda")[:, None] - (width - 1) + steps]
        if case["train"]:
            dx, dw, db, di = torch.autograd.grad(y, leaves, s["dy"].double()[source, cut])
            out["dx"][:, cut], out["dweight"][cut], out["dbias"][cut], out["dinitial"][:, :, cut] = dx, dw, db, di
    return out if case["train"] else {"y": out["y"], "state": out["state"]}


def _exact_convolution_step(s):
    state = s["state"].double() * (~s["fresh"])[:, None, None]
    total = s["bias"].double() + s["x"].double() * s["weight"][:, -1].double()
    for j in range(state.shape[1]):
        total = total + state[:, j] * s["weight"][:, j].double()
    return {"y": total * torch.special.expit(total), "state": torch.stack([*state.unbind(1)[1:], s["x"].double()], 1)}


def _softplus(u):
    return torch.logaddexp(u, torch.zeros_like(u))


def _exact_scan(s):
    """Rows side by side, one token after the other; gradients by walking back, as many channels at a time as fit."""
    case, offsets = s["case"], s["offsets"].long()
    lengths = offsets[1:] - offsets[:-1]
    starts = s["start"].clone()
    starts[offsets[:-1][lengths > 0]] = False                       # a row's first token goes on from the initial state
    order = torch.argsort(lengths, descending=True)                 # the rows still running are the first ones
    running = [int(v) for v in (lengths[None, :] > torch.arange(int(lengths.max()), device="cuda")[:, None]).sum(1).cpu()]
    base = offsets[order]
    names = ("y", "state") + (tuple("d" + name for name in NAMES["scan"]) if case["train"] else ())
    of = {"y": "x", "state": "initial", **{"d" + name: name for name in NAMES["scan"]}}
    out = {name: torch.zeros(s[of[name]].shape, dtype=torch.float64, device="cuda") for name in names}
    b, c = s["b"].detach().double(), s["c"].detach().double()
    block = max(1, (1 << 30) // (case["tokens"] * case["states"]))
    for low in range(0, case["channels"], block):
        cut = slice(low, low + block)
        x, delta, z = (s[name].detach()[:, cut].double() for name in ("x", "delta", "gate"))
        decay, skip, bias = (s[name].detach()[cut].double() for name in ("decay", "skip", "delta_bias"))
        state = s["initial"].detach()[:, cut].double()
        u = delta + bias
        dt = _softplus(u)
        hs = torch.empty(case["tokens"], x.shape[1], case["states"], dtype=torch.float64, device="cuda")
        state = state[order]
        begun = state.clone()
        keep = (~starts).double()
        for t, n in enumerate(running):
            at = base[:n] + t
            state[:n] = torch.exp(dt[at][:, :, None] * decay) * (state[:n] * keep[at][:, None, None]) + (dt[at] * x[at])[:, :, None] * b[at][:, None]
            hs[at] = state[:n]
        out["state"][order, cut] = state
        y = torch.einsum("tcn,tn->tc", hs, c) + skip * x
        sigmoid = torch.special.expit(z)
        out["y"][:, cut] = y * z * sigmoid
        if not case["train"]:
            continue
        do = s["dy"][:, cut].double()
        dy = do * z * sigmoid
        out["dgate"][:, cut] = do * y * (sigmoid + z * sigmoid * (1 - sigmoid))
        out["dskip"][cut] = (dy * x).sum(0)
        out["dc"] += torch.einsum("tc,tcn->tn", dy, hs)
        back = torch.zeros_like(state)
        ddt, dinto = torch.zeros_like(x), torch.zeros_like(x)
        for t in range(len(running) - 1, -1, -1):
            n = running[t]
            at = base[:n] + t
            grad = back[:n] + dy[at][:, :, None] * c[at][:, None]
            into = dt[at] * x[at]
            prior = begun[:n] if t == 0 else hs[at - 1] * keep[at][:, None, None]
            a = torch.exp(dt[at][:, :, None] * decay)
            through = grad * a * prior
            out["ddecay"][cut] += (through * dt[at][:, :, None]).sum(0)
            ddt[at] = (through * decay).sum(-1)
            dinto[at] = (grad * b[at][:, None]).sum(-1)
            out["db"][at] += (grad * into[:, :, None]).sum(1)
            back[:n] = a * grad * keep[at][:, None, None]
        first = lengths[order] > 0
        out["dinitial"][order[first], cut] = back[first]
        du = (ddt + dinto * x) * torch.special.expit(u)
        out["ddelta"][:, cut], out["ddelta_bias"][cut] = du, du.sum(0)
        out["dx"][:, cut] = dinto * dt + skip * dy
    return out


def _exact_scan_step(s):
    x, delta, z, b, c, state = (s[name].double() for name in ("x", "delta", "gate", "b", "c", "state"))
    dt = _softplus(delta + s["delta_bias"].double())
    state = torch.exp(torch.einsum("ec,cn->ecn", dt, s["decay"].double())) * state * (~s["fresh"])[:, None, None] + torch.einsum("ec,en->ecn", dt * x, b)
    y = torch.einsum("ecn,en->ec", state, c) + s["skip"].double() * x
    return {"y": y * z * torch.special.expit(z), "state": state}


def _exact_attention(s):
    """Rows of one length at a time, few enough that the scores fit, one head at a time; gradients by automatic differentiation."""
    case, offsets = s["case"], s["offsets"].tolist()
    hq, hk, d = case["heads_q"], case["heads_k"], case["dim"]
    q, k, v = (s[name].detach().double() for name in ("q", "k", "v"))
    episode = s["start"].long().cumsum(0)
    token = torch.arange(case["tokens"], device="cuda")
    number = token - token[s["start"]][episode - 1]                 # of each token in its episode
    o = torch.zeros_like(q)
    grads = [torch.zeros_like(x) for x in (q, k, v)]
    by_length = {}
    for low, high in zip(offsets, offsets[1:]):
        by_length.setdefault(high - low, []).append(low)
    for length, lows in by_length.items():
        many = max(1, (1 << 28) // max(1, length * length))
        for i in range(0, len(lows) if length else 0, many):
            at = torch.tensor(lows[i:i + many], device="cuda")[:, None] + torch.arange(length, device="cuda")
            far = at[:, :, None] - at[:, None, :]
            seen = (far >= 0) & (episode[at][:, :, None] == episode[at][:, None, :]) & ((far < case["window"]) | (number[at] < case["sinks"])[:, None, :])
            for head in range(hq):
                x = [y[at, h].requires_grad_(case["train"]) for y, h in ((q, head), (k, head // (hq // hk)), (v, head // (hq // hk)))]
                p = torch.softmax((x[0] @ x[1].transpose(1, 2) / math.sqrt(d)).masked_fill(~seen, -math.inf), -1)
                y = p @ x[2]
                o[at, head] = y.detach()
                if case["train"]:
                    for grad, part, h in zip(grads, torch.autograd.grad(y, x, s["do"][at, head].double()), (head, head // (hq // hk), head // (hq // hk))):
                        grad[at, h] += part
                del p, y
    return {"o": o, **(dict(zip(("dq", "dk", "dv"), grads)) if case["train"] else {})}


def _exact_history(s):
    case = s["case"]
    n, cap, sinks, group = case["envs"], case["capacity"], case["sinks"], case["heads_q"] // case["heads_k"]
    position = s["position"].long()
    slot = torch.tensor([p if p < sinks else sinks + (p - sinks) % (cap - sinks) for p in position.tolist()], device="cuda")
    last = position.clamp(max=cap - 1)
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    now = torch.arange(cap, device="cuda")[None, :] == slot[:, None]
    keys, values = (torch.where(now[:, :, None, None], s[new][:, None], s[old]) for new, old in (("k", "keys"), ("v", "values")))
    for head in range(case["heads_q"]):
        score = (keys[:, :, head // group].double() * s["q"][:, None, head].double()).sum(-1) / math.sqrt(case["dim"])
        p = torch.softmax(score.masked_fill(torch.arange(cap, device="cuda") > last[:, None], -math.inf), -1)
        o[:, head] = (p[:, :, None] * values[:, :, head // group].double()).sum(1)
    return {"o": o, "keys": keys.double(), "values": values.double()}


def exact(case, seed):
    return globals()["_exact_" + case["kind"]](prepare(case, seed))


def _pairs(case):
    """Query-key pairs that attention has to look at, for one query head."""
    def within(n):
        w, f = case["window"], case["sinks"]
        if n <= w:
            return n * (n + 1) // 2
        far = n - w                                                 # tokens of number w and on see the first ones too: one of those below `f` for each token behind the window's length, f at most
        return w * (w + 1) // 2 + far * w + (far * f - f * (f - 1) // 2 if far >= f else far * (far + 1) // 2)

    return sum(within(n) for n in _lengths(case["rows"], case["tokens"], 0))


def work(case):
    size, kind = BYTES[case["dtype"]], case["kind"]
    if kind == "history":
        n, cap, hq, hk, d = (case[k] for k in ("envs", "capacity", "heads_q", "heads_k", "dim"))
        held = sum(min(cap, (2 * i + 1) * cap // n + 1) for i in range(n))
        return {"bytes": 2 * held * hk * d * size + n * (2 * hq + 2 * hk) * d * size, "flops": 4 * held * hq * d}
    if kind == "convolution_step":
        n, width = case["envs"] * case["channels"], case["width"]
        return {"bytes": n * size * 2 * width + case["channels"] * 4 * (width + 1), "flops": n * (2 * width + 8)}
    if kind == "scan_step":
        n, states = case["envs"] * case["channels"], case["states"]
        return {"bytes": n * (4 * size + 8 * states) + case["envs"] * 2 * states * size + case["channels"] * 4 * (states + 2), "flops": n * (7 * states + 20)}
    t, train = case["tokens"], case["train"]
    if kind == "convolution":
        n, width = t * case["channels"], case["width"]
        state = case["rows"] * (width - 1) * case["channels"]
        return {"bytes": n * size * (4 if train else 2) + state * size * (3 if train else 2) + case["channels"] * 4 * (width + 1) * (2 if train else 1), "flops": n * (2 * width + 8) * (4 if train else 1)}
    if kind == "scan":
        n, states = t * case["channels"], case["states"]
        state, narrow = case["rows"] * case["channels"] * states, t * 2 * states
        return {"bytes": n * size * (8 if train else 4) + state * (12 if train else 8) + narrow * size * (2 if train else 1) + case["channels"] * 4 * (states + 2) * (2 if train else 1),
                "flops": n * (7 * states + 20) * (4 if train else 1)}
    hq, hk, d = case["heads_q"], case["heads_k"], case["dim"]
    return {"bytes": t * d * size * (hq + hk) * (4 if train else 2), "flops": (14 if train else 4) * d * hq * _pairs(case)}
