"""The example that runs the operators together, small: rollout by steps, update over whole rollouts."""
from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "rl_cs1.6_surf_amd" / "examples"))

pytestmark = pytest.mark.gpu


def test_a_rollout_and_an_update(dev):
    import recurrent_rollout as ex
    torch.manual_seed(0)
    envs = ex.Envs(24, dev)
    policy = ex.Policy(envs.lidar.H, envs.lidar.W, 9, features=32, channels=48).to(dev)
    optimiser = torch.optim.Adam(policy.parameters(), lr=1e-3)
    for _ in range(2):
        r = ex.rollout(policy, envs, 40, 9)
        assert bool(r["resets"][:, 0].all()) and bool(r["resets"][:, 1:].any())     # episodes end inside, too
        assert int(r["actions"].min()) >= 0 and int(r["actions"].max()) < 9
        # the draw's log-probability is the softmax's at the index: two fp32 softmaxes of numbers up to 10
        want = r["logits"].double().log_softmax(-1).gather(-1, r["actions"][..., None])[..., 0]
        assert float((r["logp"] - want).abs().max()) < 1e-5
        before = [p.detach().clone() for p in policy.parameters()]
        loss, norm, far = ex.update(policy, optimiser, r)
        # fp32 all through; the encoder's and projections' sums over up to 2000 terms come in another order
        assert far < 1e-3
        assert norm > 0.0 and loss == loss
        assert all(not torch.equal(a, b) for a, b in zip(before, policy.parameters()))
        grads = torch.cat([p.grad.flatten() for p in policy.parameters()])
        assert float(grads.double().norm()) <= 0.5 * (1 + 1e-5)


def test_the_drop_in_serves_the_operators(tmp_path):
    """Under the trainer's own package name, next to the renderer."""
    import subprocess
    (tmp_path / "surfgym").mkdir()
    (tmp_path / "surfgym" / "__init__.py").write_text("STAND_IN = True\n")
    pkg = Path(__file__).resolve().parents[1] / "rl_cs1.6_surf_amd"
    code = (f"import sys; sys.path.insert(0, {str(pkg)!r}); import surfgym_mi355x; surfgym_mi355x.install(); "
            f"sys.path.insert(0, {str(tmp_path)!r}); import torch; from surfgym import recurrent, STAND_IN; "
            "t, _ = recurrent.draw_actions(torch.zeros(3, 4, device='cuda'), torch.full((3,), 0.6, device='cuda')); "
            "assert t.tolist() == [2, 2, 2]; print('served')")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and "served" in out.stdout, out.stderr
