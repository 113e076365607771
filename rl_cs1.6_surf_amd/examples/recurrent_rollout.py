"""A policy with a memory on the rendered views: one rollout and one update, end to end.

Every decision renders all envs (``GpuLidar.render``), takes the views, coarsened, through a small encoder and a memory block
(``recurrent.causal_conv_step``, ``selective_scan_step``), and draws an action of each env from its logits with the
env's own uniform number (``draw_actions``). Episodes end anywhere; the next decision resets that env's memory. The
update runs the same block over whole rollouts (``causal_conv``, ``selective_scan`` with ``resets``), where one call
does what the rollout did in as many steps as there were decisions, takes a policy gradient through it and clips it
over all parameters (``clip_grad_norm``).

    python rl_cs1.6_surf_amd/examples/recurrent_rollout.py [--envs 2048] [--decisions 128] [--updates 3]

The envs are no simulation: a scene of ramps, poses that drift, and the mean depth seen as the reward (the way ahead
being free), so that the whole loop runs on the synthetic scenes of this package.
"""
from __future__ import annotations

import argparse
import math
import sys
import time
from pathlib import Path

_PKG = str(Path(__file__).resolve().parents[1])
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

import torch  # noqa: E402
from torch import nn  # noqa: E402

from surfgym import recurrent, synth, vision  # noqa: E402


class Memory(nn.Module):
    """A selective state space block: projection, short causal convolution, scan, projection. ``forward`` takes whole
    rollouts (batch, length, features), ``step`` one decision (batch, features) with the two states it moves on."""

    def __init__(self, features: int, channels: int, states: int = 16, width: int = 4, rank: int = 16):
        super().__init__()
        self.channels, self.states, self.width, self.rank = channels, states, width, rank
        self.inward = nn.Linear(features, 2 * channels, bias=False)
        self.weight = nn.Parameter(torch.randn(channels, width) / math.sqrt(width))
        self.bias = nn.Parameter(torch.zeros(channels))
        self.select = nn.Linear(channels, rank + 2 * states, bias=False)
        self.rate = nn.Linear(rank, channels, bias=False)
        # steps between a thousandth and a tenth, decay rates 1 .. states
        step = torch.exp(torch.rand(channels) * math.log(100.0) + math.log(1e-3))
        self.dt_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self.log_rates = nn.Parameter(torch.log(torch.arange(1, states + 1).float()).repeat(channels, 1))
        self.skip = nn.Parameter(torch.ones(channels))
        self.outward = nn.Linear(channels, features, bias=False)

    def initial(self, batch: int, dtype, device):
        return (torch.zeros(batch, self.width - 1, self.channels, dtype=dtype, device=device),
                torch.zeros(batch, self.channels, self.states, device=device))

    def _selected(self, x):
        d, b, c = self.select(x).split([self.rank, self.states, self.states], dim=-1)
        return self.rate(d), b, c

    def forward(self, f, resets):
        x, z = self.inward(f).chunk(2, dim=-1)              # halves of one tensor, read where they lie
        x = recurrent.causal_conv(x, self.weight, self.bias, resets=resets)
        dt, b, c = self._selected(x)
        y = recurrent.selective_scan(x, dt, -torch.exp(self.log_rates), b, c, D=self.skip, z=z, dt_bias=self.dt_bias,
                                     resets=resets)
        return f + self.outward(y)

    def step(self, f, resets, window, state):
        x, z = self.inward(f).chunk(2, dim=-1)
        x = recurrent.causal_conv_step(x, window, self.weight, self.bias, resets=resets)
        dt, b, c = self._selected(x)
        y = recurrent.selective_scan_step(x, dt, -torch.exp(self.log_rates), b, c, state, D=self.skip, z=z,
                                          dt_bias=self.dt_bias, resets=resets)
        return f + self.outward(y)


class Policy(nn.Module):
    def __init__(self, height: int, width: int, actions: int, features: int = 128, channels: int = 256):
        super().__init__()
        self.encoder = nn.Sequential(nn.Linear(height // 4 * (width // 4), 2 * features), nn.SiLU(),
                                     nn.Linear(2 * features, features))
        self.memory = Memory(features, channels)
        self.head = nn.Linear(features, actions)
        self.size = (height, width)

    def see(self, views):
        h, w = self.size
        coarse = views.unflatten(-1, (h // 4, 4, w // 4, 4)).mean(dim=(-3, -1))
        return self.encoder(coarse.flatten(-2))


class Envs:
    """Poses that drift through a scene of ramps; episodes that end with a chance of one in a hundred a decision."""

    def __init__(self, envs: int, device, seed: int = 0):
        w = synth.WORKLOADS["small_ramps"]
        self.scene = w.scene()
        self.lidar = vision.GpuLidar.from_grid(self.scene.sdf, self.scene.mins, self.scene.cell,
                                               range_units=w.range_units, near_range=w.near_range,
                                               max_steps=w.max_steps, hit_eps=w.hit_eps, device=device)
        p = w.poses(self.scene, envs)
        self.start = tuple(torch.as_tensor(v, device=device).float() for v in (p.origin, p.yaw, p.pitch, p.ducked))
        self.origin, self.yaw = self.start[0].clone(), self.start[1].clone()
        self.rng = torch.Generator(device=device).manual_seed(seed)
        self.ended = torch.ones(envs, dtype=torch.bool, device=device)     # an episode begins

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.rng, device=self.origin.device)

    def render(self, out):
        self.lidar.render(self.origin, self.yaw, self.start[2], self.start[3], out=out)

    def act(self, action, actions: int):
        """Turns by the action and moves on; which envs' episodes ended."""
        self.yaw = self.yaw + (action.float() / (actions - 1) - 0.5) * 20.0
        r = torch.deg2rad(self.yaw)
        self.origin = self.origin + 4.0 * torch.stack([r.cos(), r.sin(), torch.zeros_like(r)], dim=1)
        self.ended = self.uniform(self.yaw.shape[0]) < 0.01
        self.origin = torch.where(self.ended[:, None], self.start[0], self.origin)
        self.yaw = torch.where(self.ended, self.start[1], self.yaw)


@torch.no_grad()
def rollout(policy, envs, decisions: int, actions: int, temperature: float = 1.0):
    """One rollout of every env: a dict of (envs, decisions, ...) tensors."""
    n, dev = envs.yaw.shape[0], envs.yaw.device
    dtype = policy.head.weight.dtype
    h, w = policy.size
    r = {"views": torch.empty(n, decisions, h * w, dtype=dtype, device=dev),
         "resets": torch.empty(n, decisions, dtype=torch.bool, device=dev),
         "actions": torch.empty(n, decisions, dtype=torch.int64, device=dev),
         "logp": torch.empty(n, decisions, device=dev), "logits": torch.empty(n, decisions, actions, device=dev)}
    frame = torch.empty(n, h, w, device=dev)
    window, state = policy.memory.initial(n, dtype, dev)
    envs.ended.fill_(True)
    for t in range(decisions):
        r["resets"][:, t] = envs.ended
        envs.render(frame)
        r["views"][:, t] = frame.flatten(1)
        f = policy.memory.step(policy.see(r["views"][:, t]), envs.ended, window, state)
        logits = policy.head(f)
        action, logp = recurrent.draw_actions(logits, envs.uniform(n), temperature=temperature)
        r["actions"][:, t], r["logp"][:, t], r["logits"][:, t] = action, logp, logits
        envs.act(action, actions)
    r["reward"] = r["views"].float().mean(-1)
    return r


def returns_of(reward, resets, discount: float):
    """Discounted sums of what follows within an episode."""
    out = torch.zeros_like(reward)
    ahead = torch.zeros_like(reward[:, 0])
    for t in range(reward.shape[1] - 1, -1, -1):
        ahead = out[:, t] = reward[:, t] + discount * ahead
        ahead = torch.where(resets[:, t], torch.zeros_like(ahead), ahead)
    return out


def update(policy, optimiser, r, max_norm: float = 0.5):
    """One policy gradient over whole rollouts: (loss, gradient norm, how far the logits are from the rollout's)."""
    logits = policy.head(policy.memory(policy.see(r["views"]), r["resets"])).float()
    far = float((logits.detach() - r["logits"]).abs().max())
    logp = logits.log_softmax(-1).gather(-1, r["actions"][..., None])[..., 0]
    gain = returns_of(r["reward"], r["resets"], 0.97)
    gain = (gain - gain.mean()) / (gain.std() + 1e-6)
    # the draws' own log-probabilities weigh them, as they would weigh those of an older policy
    ratio = torch.exp(logp - r["logp"])
    loss = -torch.minimum(ratio * gain, ratio.clamp(0.8, 1.2) * gain).mean()
    optimiser.zero_grad()
    loss.backward()
    norm = recurrent.clip_grad_norm([p.grad for p in policy.parameters()], max_norm)
    optimiser.step()
    return float(loss.detach()), float(norm), far


def main(argv=None):
    a = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    a.add_argument("--envs", type=int, default=2048)
    a.add_argument("--decisions", type=int, default=128)
    a.add_argument("--updates", type=int, default=3)
    a.add_argument("--actions", type=int, default=27)
    a.add_argument("--minibatch", type=int, default=256, help="envs an update takes at once")
    a = a.parse_args(argv)
    torch.manual_seed(0)
    dev = torch.device("cuda", torch.cuda.current_device())
    envs = Envs(a.envs, dev)
    policy = Policy(envs.lidar.H, envs.lidar.W, a.actions).to(dev)
    optimiser = torch.optim.Adam(policy.parameters(), lr=3e-4)
    for k in range(a.updates):
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        r = rollout(policy, envs, a.decisions, a.actions)
        torch.cuda.synchronize()
        t1 = time.perf_counter()
        for at in range(0, a.envs, a.minibatch):
            loss, norm, far = update(policy, optimiser, {k: v[at:at + a.minibatch] for k, v in r.items()})
            first = far if at == 0 else first
        torch.cuda.synchronize()
        t2 = time.perf_counter()
        print(f"update {k}: rollout {1e3 * (t1 - t0):.0f} ms, update {1e3 * (t2 - t1):.0f} ms, reward "
              f"{float(r['reward'].mean()):.4f}, loss {loss:.4f}, gradient norm {norm:.3f}, prompt against steps "
              f"{first:.1e}", flush=True)


if __name__ == "__main__":
    main()
