"""A policy with memory over the vectorised env: its acting and its training form are one policy, and it learns."""
import pytest

torch = pytest.importorskip("torch")
import nuka  # noqa: E402,F401
from nuka import memory_policy as M, templates as T  # noqa: E402
from nuka.vec_env import NukaVecEnv  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("envs,steps,history", [(16, 40, 16), (1, 24, 64), (37, 9, 4)])
def test_acting_and_training_forms_agree(device, envs, steps, history):
    """Two rollouts through ends of episodes. The forms differ by roundings of bf16 keys, values, probabilities and outputs (2^-8 of values of about 1, in
    two layers), so by a few hundredths of the actions' spread of about 1 at most."""
    torch.manual_seed(envs)
    env = NukaVecEnv(device, T.quadruped(0).blob(), envs, episode_length_s=0.3)                # 15 control steps an episode
    policy = M.MemoryPolicy(env.obs_width, env.num_joints, width=128, heads=4, kv_heads=2, history=history).cuda()
    with torch.no_grad():
        policy.action.weight.mul_(3.0)
    memory, obs, fresh = M.Memory(policy, envs, "cuda"), env.reset(), None
    for _ in range(2):
        rollout = M.Rollout(env, policy, memory, obs, fresh, steps)
        mean, _ = policy(rollout.obs, rollout.done, rollout.states)
        assert bool(rollout.done.any()) or steps < 15
        assert (mean - rollout.means).abs().max().item() <= 0.05 * max(1.0, mean.abs().max().item())
        # memory is at work: without it (every step an episode of its own) the actions are others
        alone, _ = policy(rollout.obs, torch.ones_like(rollout.done))
        assert (alone - rollout.means).abs().max().item() > 0.1
        obs, fresh = rollout.next_obs, rollout.fresh
    env.close()


def test_it_learns(device):
    """Clones a policy that looks two control steps back: only memory can tell the two apart, and the loss falls."""
    torch.manual_seed(0)
    envs, steps = 64, 24
    env = NukaVecEnv(device, T.quadruped(0).blob(), envs)
    policy = M.MemoryPolicy(env.obs_width, env.num_joints, width=64, heads=2, kv_heads=1, layers=1, history=8).cuda()
    optimizer = torch.optim.Adam(policy.parameters(), 3e-3)
    memory = M.Memory(policy, envs, "cuda")
    rollout = M.Rollout(env, policy, memory, env.reset(), None, steps)
    reward, loss = M.update(policy, optimizer, rollout)
    assert reward == reward and loss == loss and all(torch.isfinite(p).all() and p.grad is not None for p in policy.parameters())
    target = torch.cat([torch.zeros_like(rollout.actions[:, :2]), rollout.obs[:, :-2, 24:36]], 1).clamp(-1, 1)
    losses = []
    for _ in range(60):
        mean, _ = policy(rollout.obs, rollout.done, rollout.states)
        loss = (mean - target).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    assert losses[-1] < 0.5 * losses[0]
    env.close()
