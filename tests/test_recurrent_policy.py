"""RecurrentPolicy (the sequence operators as a policy uses them) and MetaWorldTorchVectorEnv.policy_rollout."""
import pytest
import torch


from metaworld_amd.recurrent_policy import RecurrentPolicy
from metaworld_amd.torch_env import MetaWorldTorchVectorEnv

gpu = pytest.mark.gpu


class Spring:
    """a policy of plain torch operations with a memory: the actions depend on how long the episode has been going on"""
    def __init__(self, device):
        self.device, self.seen = device, []

    def initial_state(self, batch):
        return torch.full((batch,), float("nan"), device=self.device)

    def act(self, obs, state, reset):
        state.copy_(torch.where(reset, torch.zeros_like(state), state + 1))
        self.seen.append((obs.clone(), reset.clone()))
        return torch.sin(state[:, None] * torch.tensor([0.3, 0.5, 0.7, 1.1], device=self.device) + obs[:, :4])


def _rollout_is_the_loop(lib, device):
    kw = dict(num_envs=24, seed=5, use_one_hot=True, precision="fp32", lib=lib, max_episode_steps=9, device=device)
    env, twin = MetaWorldTorchVectorEnv("MT10", **kw), MetaWorldTorchVectorEnv("MT10", **kw)
    policy = Spring(device)
    r = env.policy_rollout(policy, 31, record=True)
    assert r["episodes"].tolist() == [3] * 24 and (r["successes"] <= r["episodes"]).all()
    want = torch.zeros(31, dtype=torch.bool)
    want[::9] = True
    assert torch.equal(r["reset"].cpu(), want.expand(24, 31))
    obs, _ = twin.reset()
    for t in range(31):
        assert torch.equal(r["obs"][:, t], obs) and torch.equal(policy.seen[t][0], obs) and torch.equal(policy.seen[t][1], r["reset"][:, t])
        obs, reward, *_ = twin.step(r["actions"][:, t])
        assert torch.equal(r["rewards"][:, t], reward)
    again = env.policy_rollout(Spring(device), 10)
    assert set(again) == {"episodes", "successes"} and again["episodes"].tolist() == [1] * 24
    env.close(), twin.close()


def test_rollout_on_host_harness(hostsim):
    _rollout_is_the_loop(hostsim, "cpu")


@gpu
def test_rollout_on_gpu(gpulib):
    _rollout_is_the_loop(gpulib, "cuda:0")


def test_policy_has_no_cpu_fallback_and_keeps_its_configuration(tmp_path):
    policy = RecurrentPolicy(49, width=32, layers=2, states=8, taps=3, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no CPU fallback"):
        policy(torch.zeros(2, 3, 49))
    with pytest.raises(ValueError, match="no CPU fallback"):
        policy.act(torch.zeros(2, 49), policy.initial_state(2))
    policy.save(tmp_path / "p.pt")
    other = RecurrentPolicy.load(tmp_path / "p.pt", device="cpu")
    assert other.config == policy.config and all(torch.equal(a, b) for a, b in zip(policy.state_dict().values(), other.state_dict().values()))
    conv, scan = other.initial_state(5)[1]
    assert conv.shape == (5, 2, 64) and conv.dtype == torch.bfloat16 and scan.shape == (5, 64, 8) and scan.dtype == torch.float32


def plain_policy(p, obs, reset):
    """RecurrentPolicy.forward in 64 bits, token by token, from its weights"""
    w = {k: v for k, v in p.items()}
    norm = lambda x, a, b: torch.nn.functional.layer_norm(x, x.shape[-1:], a, b)
    x = obs @ w["embed.weight"].T + w["embed.bias"]
    batch, time, width = x.shape
    for k in range(sum(n.endswith("log_A") for n in w)):
        g = {n.split(".", 2)[2]: v for n, v in w.items() if n.startswith(f"layers.{k}.")}
        v, z = (norm(x, g["norm_weight"], g["norm_bias"]) @ g["into.weight"].T).chunk(2, -1)
        inner, taps = g["conv_weight"].shape
        states = g["log_A"].shape[1]
        rank = g["step.weight"].shape[1]
        line, h, out = torch.zeros(batch, taps - 1, inner, dtype=x.dtype), torch.zeros(batch, inner, states, dtype=x.dtype), []
        for t in range(time):
            keep = (~reset[:, t])[:, None, None].to(x.dtype)
            line, h = line * keep, h * keep
            window = torch.cat([line, v[:, t, None]], 1)
            line = window[:, 1:]
            s = torch.nn.functional.silu((window * g["conv_weight"].T).sum(1) + g["conv_bias"])
            d, B, C = (s @ g["select.weight"].T).split([rank, states, states], -1)
            d = torch.nn.functional.softplus(d @ g["step.weight"].T + g["dt_bias"], threshold=40)
            h = torch.exp(d[..., None] * -torch.exp(g["log_A"])) * h + (d * s)[..., None] * B[:, None]
            out.append(((h * C[:, None]).sum(-1) + g["D"] * s) * torch.nn.functional.silu(z[:, t]))
        x = x + torch.stack(out, 1) @ g["out.weight"].T
    return torch.tanh(norm(x, w["norm_weight"], w["norm_bias"]) @ w["head.weight"].T + w["head.bias"])


@gpu
def test_values_and_gradients_against_the_plain_policy():
    torch.manual_seed(3)
    policy = RecurrentPolicy(49, width=48, layers=2).cuda()
    obs, target = torch.randn(6, 37, 49), torch.randn(6, 37, 4)
    reset = torch.rand(6, 37) < 0.1
    reset[:, 0] = True
    actions, _ = policy(obs.cuda(), reset.cuda())
    (actions - target.cuda()).square().sum().backward()
    weights = {k: v.detach().double().cpu().requires_grad_() for k, v in policy.named_parameters()}
    want = plain_policy(weights, obs.double(), reset)
    (want - target.double()).square().sum().backward()
    # float32 through two layers of a few hundred additions each: 2^-24 x some thousand operations
    assert (actions.detach().double().cpu() - want.detach()).abs().max() < 2e-4
    for k, v in policy.named_parameters():
        g, r = v.grad.double().cpu(), weights[k].grad
        assert (g - r).norm() <= 2e-4 * r.norm() + 1e-9, (k, float((g - r).norm() / r.norm()))


@gpu
@pytest.mark.parametrize("dtype,most", [(torch.float32, 1e-4), (torch.bfloat16, 0.1)])
def test_acting_is_the_forward_pass_token_by_token(dtype, most):
    """most: float32 as above; bfloat16 rounds the activations a few dozen times by 2^-9 of values of order one, in another place in the two forms"""
    torch.manual_seed(4)
    policy = RecurrentPolicy(39, width=64, layers=3, dtype=dtype).cuda()
    obs = torch.randn(50, 21, 39, device="cuda", dtype=torch.float64)
    reset = torch.rand(50, 21, device="cuda") < 0.1
    reset[:, 0] = True
    state = policy.initial_state(50)
    for conv, scan in state:
        conv.fill_(float("nan")), scan.fill_(float("nan"))           # of an episode before: not seen
    acted = torch.stack([policy.act(obs[:, t], state, reset[:, t]) for t in range(21)], 1)
    with torch.no_grad():
        whole, after = policy(obs, reset)
        halves = [policy(obs[:, :10], reset[:, :10])]
        halves.append(policy(obs[:, 10:], reset[:, 10:], state=halves[0][1]))
    assert acted.dtype == dtype and torch.isfinite(acted).all()
    assert (acted.float() - whole.float()).abs().max() < most and (torch.cat([h[0] for h in halves], 1).float() - whole.float()).abs().max() < most
    for (a, b), (c, d) in zip(state, after):
        assert (a.float() - c.float()).abs().max() < 10 * most and (b - d).abs().max() < 10 * most


@gpu
def test_policy_in_the_environments(gpulib):
    """acts in 50 environments, whose episodes end; a training pass over what was recorded sees the same actions and has gradients everywhere"""
    env = MetaWorldTorchVectorEnv("ML10-train", num_envs=50, seed=1, precision="fp32", lib=gpulib, max_episode_steps=12)
    torch.manual_seed(0)
    policy = RecurrentPolicy(env.ctx.D, width=32).cuda()
    r = env.policy_rollout(policy, 30, record=True)
    assert r["episodes"].tolist() == [2] * 50 and r["actions"].abs().max() <= 1
    actions, _ = policy(r["obs"], r["reset"])
    assert (actions.detach() - r["actions"]).abs().max() < 1e-3          # observations of order one, float32
    (actions * r["rewards"][..., None].float()).sum().backward()
    for k, v in policy.named_parameters():
        assert torch.isfinite(v.grad).all() and v.grad.abs().max() > 0, k
    env.close()
