"""oracle.recurrent's gradients against central differences of its forward formulas, in 64 bits.

A difference quotient with step e of a smooth function is off by O(e^2) and by 1e-16 |f| / e: with e = 1e-5 and
values around 1 to 10 that is about 1e-9, hence 1e-7.
"""
from __future__ import annotations

import pytest
import torch

from oracle import recurrent as ref


def _differences(f, inputs, grads, n=6):
    g = torch.Generator().manual_seed(0)
    for name, want in grads.items():
        t = inputs[name]
        for _ in range(n):
            v = torch.randn(t.shape, generator=g, dtype=torch.float64)
            e = 1e-5
            got = (f({**inputs, name: t + e * v}) - f({**inputs, name: t - e * v})) / (2 * e)
            assert abs(float(got) - float((want * v).sum())) < 1e-7 * max(1.0, abs(float(got))), name


def _rand(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


@pytest.mark.parametrize("width", [1, 2, 4])
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("n", [1, 2, 7])
def test_convolution_gradients(width, silu, n):
    b, d = 2, 3
    t = {"x": _rand(b, n, d, seed=1), "weight": _rand(d, width, seed=2), "bias": _rand(d, seed=3),
         "state": _rand(b, width - 1, d, seed=4)}
    dy, ds = _rand(b, n, d, seed=5), _rand(b, width - 1, d, seed=6)
    resets = torch.zeros(b, n, dtype=torch.bool)
    resets[1, n // 2] = True

    def f(v):
        y, s = ref.conv(v["x"], v["weight"], v["bias"], silu=silu, resets=resets, state=v["state"])
        return (y * dy).sum() + (s * ds).sum()

    _, _, grads = ref.conv_grad(t["x"], t["weight"], t["bias"], silu=silu, resets=resets, state=t["state"], dy=dy,
                                dstate_out=ds)
    _differences(f, t, grads)


@pytest.mark.parametrize("softplus", [False, True])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("n", [1, 2, 7])
def test_scan_gradients(softplus, gated, n):
    b, d, m = 2, 3, 4
    t = {"x": _rand(b, n, d, seed=1), "dt": _rand(b, n, d, seed=2), "A": -_rand(d, m, seed=3).abs(),
         "B": _rand(b, n, m, seed=4), "C": _rand(b, n, m, seed=5), "D": _rand(d, seed=6),
         "dt_bias": _rand(d, seed=7), "state": _rand(b, d, m, seed=8)}
    if gated:
        t["z"] = _rand(b, n, d, seed=9)
    dy, ds = _rand(b, n, d, seed=10), _rand(b, d, m, seed=11)
    resets = torch.zeros(b, n, dtype=torch.bool)
    resets[1, n // 2] = True

    def run(v, **kw):
        return ref.scan_grad(v["x"], v["dt"], v["A"], v["B"], v["C"], D=v["D"], z=v.get("z"), dt_bias=v["dt_bias"],
                             softplus=softplus, resets=resets, state=v["state"], **kw)

    def f(v):
        y, s, _ = run(v)
        return (y * dy).sum() + (s * ds).sum()

    _differences(f, t, run(t, dy=dy, dstate_out=ds)[2])


def test_a_call_cut_in_two_goes_on_where_it_stopped():
    b, n, d, m = 2, 9, 3, 4
    x, dt, z = (_rand(b, n, d, seed=i) for i in (1, 2, 3))
    A, B, C = -_rand(d, m, seed=4).abs(), _rand(b, n, m, seed=5), _rand(b, n, m, seed=6)
    w = _rand(d, 4, seed=7)
    resets = torch.zeros(b, n, dtype=torch.bool)
    resets[0, 5] = resets[1, 0] = True
    for cut in (1, 2, 4, 6, 8):
        lo, hi = slice(0, cut), slice(cut, n)
        y, s = ref.scan(x, dt, A, B, C, z=z, resets=resets)
        y1, s1 = ref.scan(x[:, lo], dt[:, lo], A, B[:, lo], C[:, lo], z=z[:, lo], resets=resets[:, lo])
        y2, s2 = ref.scan(x[:, hi], dt[:, hi], A, B[:, hi], C[:, hi], z=z[:, hi], resets=resets[:, hi], state=s1)
        assert torch.allclose(torch.cat([y1, y2], 1), y, atol=1e-14) and torch.allclose(s2, s, atol=1e-14)
        y, s = ref.conv(x, w, resets=resets)
        y1, s1 = ref.conv(x[:, lo], w, resets=resets[:, lo])
        y2, s2 = ref.conv(x[:, hi], w, resets=resets[:, hi], state=s1)
        assert torch.allclose(torch.cat([y1, y2], 1), y, atol=1e-14) and torch.equal(s2, s)


def test_kept_probabilities_by_hand():
    x = torch.log(torch.tensor([0.1, 0.4, 0.4, 0.05, 0.05], dtype=torch.float64))
    assert torch.allclose(ref.kept_probabilities(x), torch.exp(x))
    assert ref.kept_probabilities(x, top_k=1).tolist() == [0, 1, 0, 0, 0]      # a tie goes to the lowest index
    assert torch.allclose(ref.kept_probabilities(x, top_p=0.5), torch.tensor([0, 0.5, 0.5, 0, 0], dtype=torch.float64))
    assert ref.kept_probabilities(x, top_p=0.0).tolist() == [0, 1, 0, 0, 0]
    assert (ref.kept_probabilities(x, min_p=0.2) > 0).tolist() == [True, True, True, False, False]
    assert (ref.kept_probabilities(x, top_k=4) > 0).tolist() == [True, True, True, True, False]
    assert ref.kept_probabilities(x, temperature=0.0).tolist() == [0, 1, 0, 0, 0]
    assert ref.kept_probabilities(x, mask=torch.zeros(5, dtype=torch.bool)) is None
