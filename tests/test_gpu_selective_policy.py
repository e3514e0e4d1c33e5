"""The policy with memory with selective layers and first tokens that stay: its acting and its training form are one policy, and it takes a training step."""
import pytest

torch = pytest.importorskip("torch")
import nuka  # noqa: E402,F401
from nuka import memory_policy as M, templates as T  # noqa: E402
from nuka.vec_env import NukaVecEnv  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("envs,steps,history,states,sinks", [(16, 40, 16, 16, 3), (1, 24, 64, 8, 0), (37, 9, 4, 0, 2), (5, 70, 12, 20, 4)])
def test_acting_and_training_forms_agree(device, envs, steps, history, states, sinks):
    """Two rollouts through ends of episodes. The forms differ by roundings of bf16 keys, values, probabilities and outputs (2^-8 of values of about 1, in
    two layers), so by a few hundredths of the actions' spread of about 1 at most."""
    torch.manual_seed(envs)
    env = NukaVecEnv(device, T.quadruped(0).blob(), envs, episode_length_s=0.3)                # 15 control steps an episode
    policy = M.MemoryPolicy(env.obs_width, env.num_joints, width=128, heads=4, kv_heads=2, history=history, states=states, sinks=sinks).cuda()
    with torch.no_grad():
        policy.action.weight.mul_(3.0)
    memory, obs, fresh = M.Memory(policy, envs, "cuda"), env.reset(), None
    for _ in range(2):
        rollout = M.Rollout(env, policy, memory, obs, fresh, steps)
        mean, _ = policy(rollout.obs, rollout.done, rollout.states)
        assert (mean - rollout.means).abs().max().item() <= 0.05 * max(1.0, mean.abs().max().item())
        obs, fresh = rollout.next_obs, rollout.fresh
    optimizer = torch.optim.SGD(policy.parameters(), 1e-3)
    reward, loss = M.update(policy, optimizer, rollout)
    assert reward == reward and loss == loss and all(p.grad is not None and torch.isfinite(p.grad).all() for p in policy.parameters())
    env.close()


def test_gradients_against_differences():
    """A policy of one selective layer in 32 bits, its attention's part left out by weights of 0: the gradient along itself, against differences of the loss.
    At this step the third derivative's share is below a hundredth. Actions are worked out in 32 bits, through five products of up to 64 terms each, off by about 2^-22 of themselves: the loss, a sum of
    their squared differences, by up to 2^-22 of itself, which for weights of small influence (those of the rates) is the larger part."""
    torch.manual_seed(3)
    policy = M.MemoryPolicy(12, 3, width=32, heads=1, kv_heads=1, layers=1, history=8, states=6).cuda()
    with torch.no_grad():
        for w in (policy.layers[0].attention_out.weight, policy.layers[0].attention_out.bias):
            w.zero_()
    obs, done = torch.randn(9, 20, 12, device="cuda"), torch.rand(9, 20, device="cuda") < 0.1
    target = torch.randn(9, 20, 3, device="cuda")
    loss = lambda: ((policy(obs, done)[0] - target).double() ** 2).sum() / 27
    layer = policy.layers[0]
    names = [layer.taps, layer.taps_bias, layer.rates.weight, layer.rates_bias, layer.log_decay, layer.skip, layer.selection.weight, layer.recurrence_in.weight]
    grads = torch.autograd.grad(loss(), names)
    for w, g in zip(names, grads):
        with torch.no_grad():
            step = 1e-2 * w.norm().clamp(min=1.0) / g.norm()            # the convolution's bias begins at 0
            kept = w.clone()
            ends = []
            for s in (1, -1):
                w.copy_(kept + s * step * g)
                ends.append(loss().item())
            w.copy_(kept)
            change = 2 * step.item() * g.double().square().sum().item()
            assert abs(ends[0] - ends[1] - change) <= 0.02 * change + 2.0 ** -22 * ends[0]
