"""A policy with memory over ``nuka.vec_env.NukaVecEnv``: what ``nuka.sequence`` is for, in one small model.

A layer is a gated linear recurrence, which remembers for as long as it likes in a state of fixed size, and attention over the last ``history`` control
steps, which remembers those exactly. The policy acts token by token (``act``, on a ``Memory``) and trains on whole rollouts (calling it), with the
same result; episodes end at any control step of any env.

    python -m nuka.memory_policy [--envs 1024] [--steps 24] [--rollouts 20]

runs a plain policy gradient on the quadruped: rollouts of --steps control steps by acting, then one update from the training form.
"""
import torch
from torch import nn

from . import sequence


class Memory:
    """What a policy remembers of each env: the recurrences' states and the histories of keys and values of each layer."""

    def __init__(self, policy, envs, device):
        heads, dim = policy.kv_heads, policy.width // policy.heads
        self.states = [torch.zeros(envs, policy.width, device=device) for _ in policy.layers]
        first = sequence.HistoryCache(envs, policy.history, heads, dim, torch.bfloat16, device)
        self.caches = [first] + [sequence.HistoryCache(envs, policy.history, heads, dim, torch.bfloat16, device, position=first.position) for _ in policy.layers[1:]]

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

    def projections(self, x):
        both = self.qkv(self.attention_norm(x)).to(torch.bfloat16).unflatten(-1, (self.heads + 2 * self.kv_heads, self.dim))
        return both.split((self.heads, self.kv_heads, self.kv_heads), -2)


class MemoryPolicy(nn.Module):
    def __init__(self, obs_width, actions, width=256, heads=4, kv_heads=2, layers=2, history=64):
        super().__init__()
        if width % heads or heads % kv_heads or width // heads % 8 or width // heads > 128:
            raise ValueError("heads must divide width into at most 128 columns each, a multiple of 8, and kv_heads must divide heads")
        self.width, self.heads, self.kv_heads, self.history = width, heads, kv_heads, history
        self.embed = nn.Linear(obs_width, width)
        self.layers = nn.ModuleList(Layer(width, heads, kv_heads) for _ in range(layers))
        self.norm, self.action, self.value = nn.LayerNorm(width), nn.Linear(width, actions), nn.Linear(width, 1)
        self.log_std = nn.Parameter(torch.full((actions,), -1.0))
        self.register_buffer("frequencies", sequence.rotary_frequencies(width // heads), persistent=False)

    def forward(self, obs, done, states=None):
        """The training form. obs: envs x steps x width of the record; done: envs x steps, set where an episode ended with that step; states: of each
        layer, as ``Memory.begin_rollout`` gave them. Returns (mean actions, values), envs x steps x ..."""
        envs, steps = done.shape
        episodes = sequence.Episodes.from_done(done)
        x = self.embed(obs.reshape(envs * steps, -1))
        for k, layer in enumerate(self.layers):
            h, _ = sequence.gated_recurrence(*layer.inputs(x), episodes, None if states is None else states[k])
            x = x + layer.recurrence_out(h)
            q, key, v = layer.projections(x)
            q, key = sequence.rotate_heads(q, key, layer.q_weight, layer.k_weight, episodes, self.frequencies)
            o = sequence.episode_attention(q, key, v, episodes, window=self.history)
            x = x + layer.attention_out(o.flatten(1).float())
        x = self.norm(x)
        return self.action(x).view(envs, steps, -1), self.value(x).view(envs, steps)

    @torch.no_grad()
    def act(self, obs, memory, fresh=None):
        """One control step of every env: (mean actions, values).  fresh: envs, set where this step begins an episode (the env was done with the step before)."""
        memory.caches[0].advance(fresh)
        x = self.embed(obs)
        for layer, state, cache in zip(self.layers, memory.states, memory.caches):
            x = x + layer.recurrence_out(sequence.gated_recurrence_step(*layer.inputs(x), state, fresh))
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
            self.states = [state.masked_fill(fresh[:, None], 0.0) for state in self.states]
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
    for name, value in (("envs", 1024), ("steps", 24), ("rollouts", 20)):
        parser.add_argument("--" + name, type=int, default=value)
    a = parser.parse_args(argv)
    torch.manual_seed(0)
    device = nuka.Device.create(0)
    env = NukaVecEnv(device, templates.quadruped(0).blob(), a.envs)
    policy = MemoryPolicy(env.obs_width, env.num_joints).cuda()
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
