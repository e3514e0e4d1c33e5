"""A policy with memory over ``nuka.vec_env.NukaVecEnv``: what ``nuka.sequence`` is for, in one small model.

A layer is a gated linear recurrence, which remembers for as long as it likes in a state of fixed size, and attention over the last ``history`` control
steps, which remembers those exactly. With ``sinks`` some of the ``history`` are the first control steps that it has of an episode, beside the last ones: histories begin anew with every rollout, in which a policy
trains, so those are the episode's own first steps where it began in the rollout, else the rollout's first ones, and a rollout of no more than ``history`` - ``sinks`` steps is all seen anyway. With ``states`` a selective
scan behind a short convolution takes the recurrence's place: as many values of state a channel, and rates, inputs and outputs that depend on the token. The policy acts token by token (``act``, on a ``Memory``) and trains on whole rollouts (calling it), with the
same result; episodes end at any control step of any env.

    python -m nuka.memory_policy [--envs 1024] [--steps 24] [--rollouts 20] [--states 0] [--sinks 0]

runs a plain policy gradient on the quadruped: rollouts of --steps control steps by acting, then one update from the training form.
"""
import torch
from torch import nn

from . import sequence


class Memory:
    """What a policy remembers of each env: the recurrences' states (or the convolutions' and scans') and the histories of keys and values of each layer."""

    def __init__(self, policy, envs, device):
        heads, dim = policy.kv_heads, policy.width // policy.heads
        self.states = [torch.zeros(envs, *shape, device=device) for layer in policy.layers for shape in layer.kept()]
        cache = lambda position: sequence.HistoryCache(envs, policy.history, heads, dim, torch.bfloat16, device, position=position, sinks=policy.sinks)
        first = cache(None)
        self.caches = [first] + [cache(first.position) for _ in policy.layers[1:]]

    def begin_rollout(self):
        """A new rollout: the states go on, the histories begin anew, as the training form sees them.  Returns the states for the training form."""
        self.caches[0].position.fill_(-1)
        return [state.clone() for state in self.states]


class Layer(nn.Module):
    def __init__(self, width, heads, kv_heads):
        super().__init__()
        dim = width // heads
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.recurrence_norm, self.attention_norm = nn.LayerNorm(width), nn.LayerNorm(width)
        self.recurrence_in, self.recurrence_out = nn.Linear(width, 2 * width), nn.Linear(width, width)
        self.qkv, self.attention_out = nn.Linear(width, (heads + 2 * kv_heads) * dim, bias=False), nn.Linear(width, width)
        self.q_weight, self.k_weight = nn.Parameter(torch.ones(dim)), nn.Parameter(torch.ones(dim))
        with torch.no_grad():
            self.recurrence_in.bias[width:].uniform_(1.0, 5.0)             # gates that remember for 3 to 150 control steps at first

    def inputs(self, x):
        """x and gate of the recurrence."""
        return self.recurrence_in(self.recurrence_norm(x)).chunk(2, -1)

    def kept(self):
        """The shapes of an env's states."""
        return [(self.recurrence_out.in_features,)]

    def remember(self, x, episodes, states):
        h, _ = sequence.gated_recurrence(*self.inputs(x), episodes, *states)
        return self.recurrence_out(h)

    def remember_step(self, x, states, fresh):
        return self.recurrence_out(sequence.gated_recurrence_step(*self.inputs(x), *states, fresh))

    def projections(self, x):
        both = self.qkv(self.attention_norm(x)).to(torch.bfloat16).unflatten(-1, (self.heads + 2 * self.kv_heads, self.dim))
        return both.split((self.heads, self.kv_heads, self.kv_heads), -2)


class SelectiveLayer(Layer):
    """A layer whose recurrence is a selective scan of `states` values a channel, behind a convolution over `TAPS` tokens, twice as wide as the policy."""
    TAPS = 4

    def __init__(self, width, heads, kv_heads, states):
        super().__init__(width, heads, kv_heads)
        inner, self.states, self.rank = 2 * width, states, max(1, width // 16)
        self.recurrence_in, self.recurrence_out = nn.Linear(width, 2 * inner, bias=False), nn.Linear(inner, width)
        self.taps, self.taps_bias = nn.Parameter(torch.empty(inner, self.TAPS).uniform_(-1.0, 1.0) * self.TAPS ** -0.5), nn.Parameter(torch.zeros(inner))
        self.selection, self.rates = nn.Linear(inner, self.rank + 2 * states, bias=False), nn.Linear(self.rank, inner, bias=False)
        self.log_decay = nn.Parameter(torch.arange(1, states + 1, dtype=torch.float32).log().repeat(inner, 1))
        # states that remember for 10 to 1000 control steps at first, the faster ones of a channel a fraction of that
        self.rates_bias = nn.Parameter(torch.empty(inner).uniform_(0.001, 0.1).expm1().log())
        self.skip = nn.Parameter(torch.ones(inner))

    def kept(self):
        inner = self.recurrence_out.in_features
        return [(self.TAPS - 1, inner), (inner, self.states)]

    def _selected(self, x):
        rate, b, c = self.selection(x).split((self.rank, self.states, self.states), -1)
        return self.rates(rate), -self.log_decay.exp(), b, c

    def remember(self, x, episodes, states):
        x, gate = self.inputs(x)
        first = None if states[0] is None else states[0].to(x.dtype)        # the convolution's state has its inputs' type, which autocast may have made 16 bits
        x, _ = sequence.short_convolution(x, self.taps, self.taps_bias, episodes, first, silu=True)
        y, _ = sequence.selective_scan(x, *self._selected(x), episodes, states[1], self.skip, gate, self.rates_bias)
        return self.recurrence_out(y)

    def remember_step(self, x, states, fresh):
        x, gate = self.inputs(x)
        kept = states[0].to(x.dtype)
        x = sequence.short_convolution_step(x, self.taps, self.taps_bias, kept, fresh, silu=True)
        if kept is not states[0]:
            states[0].copy_(kept)
        return self.recurrence_out(sequence.selective_scan_step(x, *self._selected(x), states[1], fresh, self.skip, gate, self.rates_bias))


class MemoryPolicy(nn.Module):
    def __init__(self, obs_width, actions, width=256, heads=4, kv_heads=2, layers=2, history=64, states=0, sinks=0):
        super().__init__()
        if width % heads or heads % kv_heads or width // heads % 8 or width // heads > 128:
            raise ValueError("heads must divide width into at most 128 columns each, a multiple of 8, and kv_heads must divide heads")
        if not 0 <= sinks < history or not 0 <= states <= 64:
            raise ValueError("sinks must be fewer than the history, and states at most 64")
        self.width, self.heads, self.kv_heads, self.history, self.sinks = width, heads, kv_heads, history, sinks
        self.embed = nn.Linear(obs_width, width)
        self.layers = nn.ModuleList(SelectiveLayer(width, heads, kv_heads, states) if states else Layer(width, heads, kv_heads) for _ in range(layers))
        self.norm, self.action, self.value = nn.LayerNorm(width), nn.Linear(width, actions), nn.Linear(width, 1)
        self.log_std = nn.Parameter(torch.full((actions,), -1.0))
        self.register_buffer("frequencies", sequence.rotary_frequencies(width // heads), persistent=False)

    def _each(self, states):
        """The layers, each with its own of `states`."""
        at = 0
        for layer in self.layers:
            count = len(layer.kept())
            yield layer, [None] * count if states is None else states[at:at + count]
            at += count

    def forward(self, obs, done, states=None):
        """The training form. obs: envs x steps x width of the record; done: envs x steps, set where an episode ended with that step; states: of the
        layers, as ``Memory.begin_rollout`` gave them. Returns (mean actions, values), envs x steps x ..."""
        envs, steps = done.shape
        episodes = sequence.Episodes.from_done(done)
        x = self.embed(obs.reshape(envs * steps, -1))
        for layer, kept in self._each(states):
            x = x + layer.remember(x, episodes, kept)
            q, key, v = layer.projections(x)
            q, key = sequence.rotate_heads(q, key, layer.q_weight, layer.k_weight, episodes, self.frequencies)
            o = sequence.episode_attention(q, key, v, episodes, window=self.history - self.sinks, sinks=self.sinks)
            x = x + layer.attention_out(o.flatten(1).float())
        x = self.norm(x)
        return self.action(x).view(envs, steps, -1), self.value(x).view(envs, steps)

    @torch.no_grad()
    def act(self, obs, memory, fresh=None):
        """One control step of every env: (mean actions, values).  fresh: envs, set where this step begins an episode (the env was done with the step before)."""
        memory.caches[0].advance(fresh)
        x = self.embed(obs)
        for (layer, kept), cache in zip(self._each(memory.states), memory.caches):
            x = x + layer.remember_step(x, kept, fresh)
            q, key, v = layer.projections(x)
            q, key = sequence.rotate_heads(q, key, layer.q_weight, layer.k_weight, cache.position, self.frequencies)
            x = x + layer.attention_out(sequence.history_attention(q, key, v, cache).flatten(1).float())
        x = self.norm(x)
        return self.action(x), self.value(x)[:, 0]


class Rollout:
    """`steps` control steps of every env under the policy, envs first: obs, actions, rewards, done, and the states that it began with."""

    def __init__(self, env, policy, memory, obs, fresh, steps):
        self.states = memory.begin_rollout()
        if fresh is not None:                       # what ended with the last rollout does not go on into this one
            self.states = [state.masked_fill(fresh.view(-1, *[1] * (state.dim() - 1)), 0.0) for state in self.states]
        kept = []
        for _ in range(steps):
            mean, _ = policy.act(obs, memory, fresh)
            action = mean + policy.log_std.detach().exp() * torch.randn_like(mean)
            after, reward, _, _, info = env.step(action)
            kept.append((obs, mean, action, reward, info["done"]))
            obs, fresh = after, info["done"]
        self.obs, self.means, self.actions, self.rewards, self.done = (torch.stack(x, 1) for x in zip(*kept))
        self.next_obs, self.fresh = obs, fresh


def update(policy, optimizer, rollout, discount=0.97):
    """One policy-gradient step on a rollout, advantages against the value head."""
    with torch.no_grad():
        returns, running = torch.zeros_like(rollout.rewards), torch.zeros_like(rollout.rewards[:, 0])
        for t in range(rollout.rewards.shape[1] - 1, -1, -1):
            running = rollout.rewards[:, t] + discount * running * ~rollout.done[:, t]
            returns[:, t] = running
    mean, value = policy(rollout.obs, rollout.done, rollout.states)
    advantage = returns - value.detach()
    advantage = (advantage - advantage.mean()) / (advantage.std() + 1e-6)
    log_prob = torch.distributions.Normal(mean, policy.log_std.exp()).log_prob(rollout.actions).sum(-1)
    loss = -(log_prob * advantage).mean() + 0.5 * (returns - value).square().mean()
    optimizer.zero_grad(set_to_none=True)
    loss.backward()
    nn.utils.clip_grad_norm_(policy.parameters(), 1.0)
    optimizer.step()
    return float(rollout.rewards.mean()), float(loss.detach())


def main(argv=None):
    import argparse
    import nuka
    from nuka import templates
    from nuka.vec_env import NukaVecEnv
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    for name, value in (("envs", 1024), ("steps", 24), ("rollouts", 20), ("states", 0), ("sinks", 0)):
        parser.add_argument("--" + name, type=int, default=value)
    a = parser.parse_args(argv)
    torch.manual_seed(0)
    device = nuka.Device.create(0)
    env = NukaVecEnv(device, templates.quadruped(0).blob(), a.envs)
    policy = MemoryPolicy(env.obs_width, env.num_joints, states=a.states, sinks=a.sinks).cuda()
    optimizer = torch.optim.Adam(policy.parameters(), 3e-4)
    memory, obs, fresh = Memory(policy, a.envs, "cuda"), env.reset(), None
    for k in range(a.rollouts):
        rollout = Rollout(env, policy, memory, obs, fresh, a.steps)
        obs, fresh = rollout.next_obs, rollout.fresh
        reward, loss = update(policy, optimizer, rollout)
        print(f"rollout {k}: {a.envs * a.steps} control steps, mean reward {reward:.4f}, loss {loss:.4f}", flush=True)
    env.close()
    device.destroy()


if __name__ == "__main__":
    main()
