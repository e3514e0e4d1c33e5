"""Sequence operators of a policy with memory (``nuka.sequence``), as a policy that acts in ``nuka.vec_env.NukaVecEnv`` and trains on
its rollouts calls them.

A token is one control step of one env.  Tokens lie in rows, one behind the other: a row is an env's part of a rollout (with episodes
that end inside it) or a whole episode.  Kinds of case:

    recurrence        the gated linear recurrence over rows, forwards, or forwards and backwards
    recurrence_step   its form for one token of every env, on the policy's state
    heads             norms of queries and keys with the rotation of positions, forwards, or forwards and backwards
    attention         causal attention over the rows' episodes, forwards, or forwards and backwards
    history           attention of one token of every env over the env's cached history, the token's own key and value written to it

The plain form is the formulas in elementary tensor operations in 32 bits, on rows padded to the longest.
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
EPS = 1e-6


def listed():
    def recurrence(name, rows, tokens, episode, channels, dtype, train):
        return {"name": name, "kind": "recurrence", "rows": rows, "tokens": tokens, "episode": episode, "channels": channels, "dtype": dtype, "train": train}

    def heads(name, rows, tokens, episode, heads_q, heads_k, dim, turned, interleaved, context, dtype, train, acting=False):
        return {"name": name, "kind": "heads", "acting": acting, "rows": rows, "tokens": tokens, "episode": episode, "heads_q": heads_q, "heads_k": heads_k, "dim": dim,
                "turned": turned, "interleaved": interleaved, "context": context, "dtype": dtype, "train": train}

    def attention(name, rows, tokens, episode, heads_q, heads_k, dim, window, dtype, train):
        return {"name": name, "kind": "attention", "rows": rows, "tokens": tokens, "episode": episode, "heads_q": heads_q, "heads_k": heads_k, "dim": dim,
                "window": window, "dtype": dtype, "train": train}

    return [
        # one robot under a trained recurrent policy: all latency
        {"name": "recurrence-step-1", "kind": "recurrence_step", "envs": 1, "channels": 256, "dtype": "f32"},
        # a training batch of the recurrent policy: 4096 envs, 24 control steps each, episodes of up to 1000 steps end inside
        recurrence("recurrence-train-4096x24", 4096, 4096 * 24, 1000, 256, "bf16", True),
        # a few very long recordings of different lengths, learnt from end to end
        recurrence("recurrence-train-long", 3, 131071, 0, 1024, "bf16", True),
        # values of a recorded batch of an odd size, no gradient
        recurrence("recurrence-forward-1000x37", 1000, 37000, 200, 200, "f32", False),
        # one token for each env of a standard batch while the policy acts, half of each head turned
        heads("heads-forward-4096x1", 4096, 4096, 0, 8, 2, 64, 32, False, 0, "bf16", False, acting=True),
        # the training batch, queries, keys and values from one projection
        heads("heads-train-4096x24", 4096, 4096 * 24, 1000, 8, 2, 64, 64, False, 0, "bf16", True),
        # long recordings, pairs side by side, frequencies stretched for a context four times the one trained at
        heads("heads-train-long", 5, 49999, 0, 16, 4, 128, 128, True, 32768, "fp16", True),
        # the training batch of an attention policy: short rows, most of them within one episode
        attention("attention-train-4096x24", 4096, 4096 * 24, 1000, 8, 2, 64, 0, "bf16", True),
        # whole episodes of different lengths, up to the 1000 control steps of a full one
        attention("attention-train-episodes", 40, 20011, 0, 8, 2, 64, 0, "bf16", True),
        # a long recording read as one prompt
        attention("attention-forward-16384", 1, 16384, 0, 8, 2, 128, 0, "bf16", False),
        # one robot with a long history under an attention policy: latency, few heads
        {"name": "history-1x8192", "kind": "history", "envs": 1, "capacity": 8192, "heads_q": 8, "heads_k": 2, "dim": 64, "dtype": "bf16"},
        # a standard batch acting with 256 control steps of history, rings that have come round among them
        {"name": "history-4096x256", "kind": "history", "envs": 4096, "capacity": 256, "heads_q": 8, "heads_k": 2, "dim": 64, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["recurrence", "recurrence_step", "heads", "attention", "history"])
    sixteen = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "recurrence_step":
        return {"kind": kind, "envs": _log(rng, 1, 16384), "channels": 8 * _log(rng, 4, 128), "dtype": rng.choice(["f32", sixteen])}
    if kind == "history":
        capacity = _log(rng, 32, 16384)
        return {"kind": kind, "envs": _log(rng, 1, max(1, min(4096, (1 << 20) // capacity))), "capacity": capacity, "heads_k": rng.choice([1, 2]),
                "heads_q": 2 * rng.choice([1, 2, 4]), "dim": rng.choice([32, 64, 64, 128]), "dtype": sixteen}
    train, rows = rng.random() < 0.7, _log(rng, 1, 4096)
    tokens = max(rows, _log(rng, 64, 98304))
    case = {"kind": kind, "rows": rows, "tokens": tokens, "train": train}
    if kind == "recurrence":
        # rows of one length with episodes that end inside, or whole episodes
        case["episode"] = rng.choice([0, _log(rng, 16, 1000)])
        if case["episode"]:
            case["tokens"] = rows * max(1, tokens // rows)
        return {**case, "channels": 8 * _log(rng, 4, 128), "dtype": rng.choice(["f32", sixteen])}
    group, heads_k = rng.choice([1, 2, 4]), rng.choice([1, 2, 4])
    dim = rng.choice([32, 64, 64, 128])
    if kind == "heads":
        acting = not train and rng.random() < 0.5
        case["tokens"] = rows if acting else tokens
        return {**case, "acting": acting, "episode": 0, "heads_q": heads_k * group, "heads_k": heads_k, "dim": dim, "turned": rng.choice([dim, dim // 2]), "interleaved": rng.random() < 0.5,
                "context": rng.choice([0, 32768]), "dtype": rng.choice(["f32", sixteen])}
    # the plain form holds rows x longest^2 scores of every head: keep to what the listed ones have
    while heads_k * group * sum(_lengths(case["rows"], case["tokens"], 0)[:1]) ** 2 * case["rows"] > 1 << 29:
        case["rows"], case["tokens"] = max(1, case["rows"] // 2), max(1, case["tokens"] // 2)
    return {**case, "episode": 0, "heads_q": heads_k * group, "heads_k": heads_k, "dim": dim, "window": rng.choice([0, 0, _log(rng, 16, 512)]), "dtype": sixteen}


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
    """The rows in an order of this seed: their lengths, and at which of their tokens an episode begins (the first always)."""
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


def _pairs(case):
    """Query-key pairs that attention has to look at, for one query head."""
    def within(n):
        w = case["window"] or n
        return n * (n + 1) // 2 if n <= w else w * (w + 1) // 2 + (n - w) * w

    if not case["episode"]:
        return sum(within(n) for n in _lengths(case["rows"], case["tokens"], 0))
    rows, length, episode = case["rows"], case["tokens"] // case["rows"], case["episode"]
    total = 0
    for row in range(rows):
        at, left = row * episode // rows, length
        while left > 0:
            part = min(left, episode - at)
            total, left, at = total + within(part), left - part, 0
    return total


def frequencies(case):
    """Angles per token of a pair, in 64 bits: base 10000, slowed down fourfold where a turn is longer than the stretched context's quarter."""
    f = 10000.0 ** (-torch.arange(0, case["turned"], 2, dtype=torch.float64) / case["turned"])
    if case["context"]:
        f = torch.where(2 * math.pi / f > case["context"] / 4, f / 4, f)
    return f


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=dtype):
        return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(shift, scale, generator=gen).to(dtype)

    kind, s = case["kind"], {"case": case}
    if kind == "recurrence_step":
        n, c = case["envs"], case["channels"]
        s.update(x=normal(n, c), gate=normal(n, c, scale=1.5, shift=2.0), state=normal(n, c, dtype=torch.float32),
                 fresh=torch.rand(n, generator=gen, device="cuda") < 0.01)
        return s
    if kind == "history":
        n, cap, hq, hk, d = (case[k] for k in ("envs", "capacity", "heads_q", "heads_k", "dim"))
        # histories between empty and twice the ring's length, in an order of this seed
        position = (torch.arange(n, device="cuda") * 2 + 1) * cap // n
        position = position[torch.randperm(n, generator=gen, device="cuda")].int()
        s.update(q=normal(n, hq, d, scale=1.5), k=normal(n, hk, d), v=normal(n, hk, d), position=position)
        held = (torch.arange(cap, device="cuda")[None, :] < position[:, None])[:, :, None, None]
        s["keys"], s["values"] = (torch.where(held, normal(n, cap, hk, d), torch.zeros((), dtype=dtype, device="cuda")) for _ in range(2))
        if own:
            from nuka import sequence
            s["cache"] = sequence.HistoryCache(n, cap, hk, d, dtype, buffers=(s["keys"], s["values"], position))
        return s
    offsets, start, done = _rows(case, seed)
    s["offsets"], s["start"] = offsets.cuda(), start.cuda()
    if own:
        from nuka import sequence
        s["plan"] = sequence.Episodes.from_done(done.cuda()) if done is not None else sequence.Episodes.from_offsets(s["offsets"], case["tokens"])
    t = case["tokens"]
    if kind == "recurrence":
        c = case["channels"]
        s.update(x=normal(t, c), gate=normal(t, c, scale=1.5, shift=2.0), initial=normal(case["rows"], c, dtype=torch.float32))
        if case["train"]:
            s["dh"] = normal(t, c)
        names = ("x", "gate", "initial")
    else:
        hq, hk, d = case["heads_q"], case["heads_k"], case["dim"]
        both = normal(t, (hq + 2 * hk) * d, scale=1.2)              # one projection gives queries, keys and values
        for name, low, n in (("q", 0, hq), ("k", hq, hk), ("v", hq + hk, hk)):
            s[name] = both[:, low * d:(low + n) * d].unflatten(1, (n, d))
        names = ("q", "k", "v")
        if kind == "heads":
            del s["v"]
            names = ("q", "k", "wq", "wk")
            if case["acting"]:                                      # one token of every env, each somewhere in its episode
                s["plan"] = s["positions"] = torch.randint(0, 1000, (t,), generator=gen, device="cuda", dtype=torch.int32)
            s.update(wq=normal(d, scale=0.2, shift=1.0, dtype=torch.float32), wk=normal(d, scale=0.2, shift=1.0, dtype=torch.float32), frequencies=frequencies(case).cuda())
            if case["train"]:
                s.update(dq=normal(t, hq, d), dk=normal(t, hk, d))
        elif case["train"]:
            s["do"] = normal(t, hq, d)
    if case["train"]:
        for name in names:
            s[name] = s[name].detach().requires_grad_()
    return s


# ---- the plain form ----------------------------------------------------------------------------------------------
def _first(s):
    """The index of each token's episode's first token."""
    at = torch.arange(s["start"].numel(), device="cuda")
    return torch.cummax(torch.where(s["start"], at, 0), 0).values


def _scan(a, b):
    """h with h_t = a_t h_{t-1} + b_t down the first dimension, by doubling."""
    step = 1
    while step < a.shape[0]:
        b = torch.cat([b[:step], b[step:] + a[step:] * b[:-step]])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _plain_recurrence(s):
    x, gate, initial, offsets = s["x"].float(), s["gate"].float(), s["initial"], s["offsets"].long()
    a = torch.sigmoid(gate)
    lead = torch.where(s["start"][:, None], 0.0, a)                 # a token that begins an episode or a row takes nothing from the token before it
    rows = (offsets[1:] > offsets[:-1]).nonzero()[:, 0]
    begins, ends = offsets[rows], offsets[rows + 1] - 1
    before = torch.zeros_like(x)
    before[begins] = initial[rows]
    h = _scan(lead, (1 - a) * x + a * before)
    state = initial.clone()
    state[rows] = h[ends]
    out = {"h": h.to(s["x"].dtype), "state": state}
    if s["case"]["train"]:
        dh = s["dh"].float()
        lead = torch.cat([lead[1:], torch.zeros_like(lead[:1])])    # a_{t+1}, nothing across an episode's end
        grad = _scan(lead.flip(0), dh.flip(0)).flip(0)
        before[1:] += torch.where(s["start"][1:, None], 0.0, h[:-1])
        dinitial = torch.zeros_like(initial)
        dinitial[rows] = (a * grad)[begins]
        out.update(dx=((1 - a) * grad).to(s["x"].dtype), dgate=(grad * (before - x) * a * (1 - a)).to(s["x"].dtype), dinitial=dinitial)
    return out


def _plain_recurrence_step(s):
    a = torch.sigmoid(s["gate"].float())
    before = torch.where(s["fresh"][:, None], 0.0, s["state"])
    s["state"].copy_(a * before + (1 - a) * s["x"].float())
    return {"h": s["state"].to(s["x"].dtype), "state": s["state"]}


def _turn(case, x, cos, sin):
    n = case["turned"]
    if case["interleaved"]:
        u, v = x[..., 0:n:2], x[..., 1:n:2]
        turned = torch.stack([u * cos - v * sin, u * sin + v * cos], -1).flatten(-2)
    else:
        u, v = x[..., :n // 2], x[..., n // 2:n]
        turned = torch.cat([u * cos - v * sin, u * sin + v * cos], -1)
    return torch.cat([turned, x[..., n:]], -1)


def _plain_heads(s):
    case = s["case"]
    at = s["positions"] if case["acting"] else torch.arange(case["tokens"], device="cuda") - _first(s)
    angle = at.float()[:, None, None] * s["frequencies"].float()
    cos, sin = torch.cos(angle), torch.sin(angle)
    out = {}
    for name in ("q", "k"):
        x, w = s[name].float(), s["w" + name]
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        out[name] = _turn(case, x * r * w, cos, sin).to(s[name].dtype)
        if case["train"]:
            dy = _turn(case, s["d" + name].float(), cos, -sin)
            e = dy * w
            out["d" + name] = (r * e - x * (r ** 3 * (x * e).mean(-1, keepdim=True))).to(s[name].dtype)
            out["dw" + name] = (dy * x * r).sum((0, 1))
    return out


def _padded(s):
    """Token of every place of the rows padded to the longest, and which places hold one."""
    offsets = s["offsets"].long()
    at = offsets[:-1, None] + torch.arange(max(_lengths(s["case"]["rows"], s["case"]["tokens"], s["case"]["episode"])), device="cuda")
    return at.clamp(max=s["case"]["tokens"] - 1), at < offsets[1:, None]


def _plain_attention(s):
    case = s["case"]
    hq, hk, d, dtype = case["heads_q"], case["heads_k"], case["dim"], s["q"].dtype
    at, held = _padded(s)
    n, length = at.shape
    first, group, scale = _first(s)[at], hq // hk, d ** -0.5

    def rows(x):                                                    # tokens x heads x dim -> row, key head, (head of the group, token), dim
        x = torch.where(held[:, :, None, None], x.float()[at], 0.0)
        return x.view(n, length, hk, -1, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)

    def tokens(x):
        return x.view(n, hk, -1, length, d).permute(0, 3, 1, 2, 4).reshape(n, length, -1, d)[held].to(dtype)

    seen = (at[:, None, :] <= at[:, :, None]) & (at[:, None, :] >= first[:, :, None]) & held[:, None, :]
    if case["window"]:
        seen &= at[:, None, :] > at[:, :, None] - case["window"]
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
    s["keys"][env, position % cap] = s["k"]
    s["values"][env, position % cap] = s["v"]
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
    if kind == "recurrence_step":
        return {"h": sequence.gated_recurrence_step(s["x"], s["gate"], s["state"], s["fresh"]), "state": s["state"]}
    if kind == "history":
        return {"o": sequence.history_attention(s["q"], s["k"], s["v"], s["cache"]), "keys": s["keys"], "values": s["values"]}
    if kind == "recurrence":
        h, state = sequence.gated_recurrence(s["x"], s["gate"], s["plan"], s["initial"])
        out, names, of, by = {"h": h.detach(), "state": state.detach()}, ("x", "gate", "initial"), [h], "dh"
    elif kind == "heads":
        q, k = sequence.rotate_heads(s["q"], s["k"], s["wq"], s["wk"], s["plan"], s["frequencies"], eps=EPS, interleaved=case["interleaved"])
        out, names, of, by = {"q": q.detach(), "k": k.detach()}, ("q", "k", "wq", "wk"), [q, k], ("dq", "dk")
    else:
        o = sequence.episode_attention(s["q"], s["k"], s["v"], s["plan"], window=case["window"] or None)
        out, names, of, by = {"o": o.detach()}, ("q", "k", "v"), [o], "do"
    if case["train"]:
        by = [s[by]] if isinstance(by, str) else [s[name] for name in by]
        grads = torch.autograd.grad(of, [s[name] for name in names], by)
        out.update(zip(["d" + name for name in names], grads))
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return globals()["_plain_" + state["case"]["kind"]](state)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------
def _exact_recurrence(s):
    """Rows side by side, one token after the other; gradients by differentiating the steps backwards."""
    case, offsets = s["case"], s["offsets"].long()
    lengths = offsets[1:] - offsets[:-1]
    x, g, initial = (s[name].detach().double() for name in ("x", "gate", "initial"))
    z, keep = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
    starts = s["start"].clone()
    starts[offsets[:-1][lengths > 0]] = False                       # a row's first token goes on from the initial state
    h, before, state = torch.zeros_like(x), torch.zeros_like(x), initial.clone()
    order = torch.argsort(lengths, descending=True)                 # the rows still running are the first ones
    running = [int(v) for v in (lengths[None, :] > torch.arange(int(lengths.max()), device="cuda")[:, None]).sum(1).cpu()]
    for t, n in enumerate(running):
        rows = order[:n]
        at = offsets[rows] + t
        prior = state[rows] * (~starts[at])[:, None]
        before[at] = prior
        now = z[at] * prior + keep[at] * x[at]
        h[at] = now
        state[rows] = now
    out = {"h": h, "state": state}
    if case["train"]:
        dh, back = s["dh"].double(), torch.zeros_like(initial)
        grad = torch.zeros_like(x)
        for t in range(len(running) - 1, -1, -1):
            rows = order[:running[t]]
            at = offsets[rows] + t
            lam = dh[at] + back[rows]
            grad[at] = lam
            back[rows] = z[at] * lam * (~starts[at])[:, None]
        dinitial = torch.zeros_like(initial)
        some = lengths > 0
        dinitial[some] = (z * grad)[offsets[:-1][some]]
        out.update(dx=keep * grad, dgate=grad * (before - x) * z * keep, dinitial=dinitial)
    return out


def _exact_recurrence_step(s):
    z = 1 / (1 + torch.exp(-s["gate"].double()))
    h = z * s["state"].double() * (~s["fresh"])[:, None] + (1 - z) * s["x"].double()
    return {"h": h, "state": h}


def _exact_heads(s):
    case, n = s["case"], s["case"]["turned"]
    at = torch.arange(case["tokens"], device="cuda")
    begins = at[s["start"]]
    at = s["positions"] if case["acting"] else at - begins[torch.searchsorted(begins, at, right=True) - 1]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), at.double()[:, None] * s["frequencies"])[:, None]
    out = {}
    for name in ("q", "k"):
        x, w = s[name].detach().double().requires_grad_(), s["w" + name].detach().double().requires_grad_()
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + EPS) * w
        first = list(range(0, n, 2)) if case["interleaved"] else list(range(n // 2))
        second = list(range(1, n, 2)) if case["interleaved"] else list(range(n // 2, n))
        z = torch.complex(y[..., first], y[..., second]) * turn
        order = torch.tensor(first + second + list(range(n, case["dim"]))).argsort().cuda()
        y = torch.cat([z.real, z.imag, y[..., n:]], -1)[..., order]
        out[name] = y.detach()
        if case["train"]:
            out["d" + name], out["dw" + name] = torch.autograd.grad(y, [x, w], s["d" + name].double())
    return out


def _exact_attention(s):
    """Rows of one length at a time, few enough that the scores fit, one head at a time; gradients by automatic differentiation."""
    case, offsets = s["case"], s["offsets"].tolist()
    t, hq, hk, d = case["tokens"], case["heads_q"], case["heads_k"], case["dim"]
    q, k, v = (s[name].detach().double() for name in ("q", "k", "v"))
    episode = s["start"].long().cumsum(0)
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
            seen = (far >= 0) & (episode[at][:, :, None] == episode[at][:, None, :]) & (far < (case["window"] or length))
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
    n, cap, group = case["envs"], case["capacity"], case["heads_q"] // case["heads_k"]
    slot, last = s["position"].long() % cap, s["position"].long().clamp(max=cap - 1)
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


def work(case):
    size, kind = BYTES[case["dtype"]], case["kind"]
    if kind == "recurrence_step":
        n = case["envs"] * case["channels"]
        return {"bytes": n * (3 * size + 8), "flops": 8 * n}
    if kind == "history":
        n, cap, hq, hk, d = (case[k] for k in ("envs", "capacity", "heads_q", "heads_k", "dim"))
        held = sum(min(cap, (2 * i + 1) * cap // n + 1) for i in range(n))
        return {"bytes": 2 * held * hk * d * size + n * (2 * hq + 2 * hk) * d * size, "flops": 4 * held * hq * d}
    t, train = case["tokens"], case["train"]
    if kind == "recurrence":
        n, rows = t * case["channels"], case["rows"] * case["channels"]
        return {"bytes": n * size * (6 if train else 3) + rows * (12 if train else 8), "flops": n * (24 if train else 8)}
    hq, hk, d = case["heads_q"], case["heads_k"], case["dim"]
    if kind == "heads":
        n = t * (hq + hk) * d
        return {"bytes": n * size * (4 if train else 2), "flops": n * (24 if train else 8)}
    pairs = _pairs(case)
    return {"bytes": t * d * size * (hq + hk) * (4 if train else 2), "flops": (14 if train else 4) * d * hq * pairs}
