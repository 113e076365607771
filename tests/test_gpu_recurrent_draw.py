"""surfgym.recurrent's draw and clipping against oracle.recurrent (64 bits).

The draw inverts a cumulative distribution, so its answer is known wherever the uniform number is not at a step of
it: the kernel's weights are off by at most 2^-22 (exp) and 2^-40, its uniform number by 2^-24, all relative to the
sum, so a number at least 2^-20 from every step of the oracle's has one answer. Log-probabilities: three fp32
roundings of numbers up to 40, 1e-5.
"""
from __future__ import annotations

import math

import pytest
import torch

from oracle import recurrent as ref
from surfgym import recurrent as ops

pytestmark = pytest.mark.gpu

FAR = 2.0 ** -20
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _settle(settings, i):
    """Row i's settings as the operator takes them: fp32 numbers, top_p in whole 2^-24."""
    out = {}
    for k, v in settings.items():
        v = v[i] if torch.is_tensor(v) else v
        out[k] = v if k == "mask" else int(v) if k == "top_k" else torch.tensor(float(v)).item()
    if "top_p" in out:
        out["top_p"] = math.floor(out["top_p"] * 2 ** 24) / 2 ** 24
    return out


def _check(dev, logits, settings, seed=0, uniform=None):
    """Draws a row each at a number that has one answer, and compares."""
    rows = logits.shape[0]
    u, want, logp = torch.zeros(rows), [], []
    g = _gen(seed)
    for i in range(rows):
        p = ref.kept_probabilities(logits[i], **_settle(settings, i))
        if p is None:
            want.append(-1)
            logp.append(0.0)
            continue
        c = p.cumsum(0)
        for _ in range(200):
            v = torch.rand((), generator=g) if uniform is None else uniform[i]
            if uniform is not None or float((c - v).abs().min()) > FAR:
                break
        u[i] = v
        j = int((c <= float(v)).sum())
        j = min(j, int(p.nonzero()[-1]))
        want.append(j)
        logp.append(math.log(float(p[j])))
    on = {k: v.to(dev) if torch.is_tensor(v) else v for k, v in settings.items()}
    token, lp = ops.draw_actions(logits.to(dev), u.to(dev), **on)
    assert token.dtype == torch.int64 and lp.dtype == torch.float32
    assert token.tolist() == want
    assert float((lp.cpu() - torch.tensor(logp)).abs().max()) < 1e-5
    return token


SETTINGS = [dict(), dict(temperature=0.7, top_k=5), dict(top_p=0.8), dict(min_p=0.1, temperature=2.0),
            dict(temperature=0.8, top_k=40, top_p=0.9, min_p=0.01), dict(temperature=0.0), dict(top_k=1),
            dict(top_p=0.0), dict(top_k=1000, top_p=0.99)]


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 255, 256, 1000, 1024, 1025, 4099, 8192, 8193, 20011])
@pytest.mark.parametrize("dtype", TYPES)
def test_draws(dev, vocab, dtype):
    for n, s in enumerate(SETTINGS):
        logits = (torch.randn(7, vocab, generator=_gen(n + vocab)) * 3).to(dtype)
        print("case draw", vocab, dtype, s, flush=True)
        _check(dev, logits, s, seed=n)


@pytest.mark.parametrize("vocab", [100, 3000, 100003])
@pytest.mark.parametrize("dtype", TYPES)
def test_ties(dev, vocab, dtype):
    """Few distinct values: whole ranges of equal logits at the thresholds, of which the first are taken."""
    g = _gen(vocab)
    logits = torch.randint(0, 4, (6, vocab), generator=g).to(dtype)
    logits[1] = 2.5
    logits[2] = -logits[2] * 0.0                      # zeros of both signs are equal
    for s in (dict(top_k=vocab // 3), dict(top_p=0.37), dict(top_k=vocab // 2, top_p=0.5), dict(top_k=1),
              dict(temperature=0.0), dict(top_k=7, min_p=0.9), dict(top_p=0.9, min_p=0.2)):
        print("case ties", vocab, dtype, s, flush=True)
        _check(dev, logits, s, seed=1)


@pytest.mark.parametrize("vocab", [10, 2000, 30000])
def test_masks_infinities_and_nan(dev, vocab):
    g = _gen(vocab)
    logits = torch.randn(8, vocab, generator=g) * 2
    mask = torch.rand(8, vocab, generator=g) < 0.5
    mask[0], mask[1] = False, False
    mask[1, vocab - 1] = True
    logits[2][~mask[2]] = float("nan")                # what is masked may be anything
    logits[3][~mask[3]] = float("inf")
    logits[4] = float("-inf")                         # nothing left, without a mask's help
    logits[5] = torch.finfo(torch.float32).min        # the lowest value is a value
    logits[6, 1:3] = float("inf")
    mask[6, 1:3] = True
    for s in (dict(), dict(top_k=3, top_p=0.9), dict(min_p=0.5, temperature=0.5)):
        for stride in (0, 3):
            m = mask if not stride else torch.cat([mask, mask[:, :3]], 1)[:, :vocab]
            _check(dev, logits, s | {"mask": m}, seed=2)
    token, logp = ops.draw_actions(logits.to(dev), torch.full((8,), 0.5, device=dev))
    assert token[2] == -1 and logp[2].isnan()         # and one that is not masked is told
    assert token[4] == -1 and logp[4] == 0.0
    extreme = torch.full((3, vocab), -1e30)
    extreme[:, vocab // 2] = 1e30
    assert ops.draw_actions(extreme.to(dev), torch.tensor([0.0, 0.5, 0.999], device=dev))[0].tolist() == [vocab // 2] * 3


def test_settings_of_each_row(dev):
    rows, vocab = 24, 5000
    g = _gen(3)
    logits = (torch.randn(rows, vocab, generator=g) * 3).to(torch.bfloat16)
    s = {"temperature": torch.rand(rows, generator=g) + 0.1, "top_p": torch.rand(rows, generator=g) * 0.9 + 0.05,
         "top_k": torch.randint(0, 300, (rows,), generator=g, dtype=torch.int32),
         "min_p": torch.rand(rows, generator=g) * 0.1}
    s["temperature"][5], s["top_p"][6], s["top_k"][7], s["top_k"][8] = 0.0, 1.0, 6000, -1
    _check(dev, logits, s, seed=4)
    # a row's answer is its own: alone, in another order, in a wider tensor
    u = torch.rand(rows, generator=g).to(dev)
    on = {k: v.to(dev) for k, v in s.items()}
    token, logp = ops.draw_actions(logits.to(dev), u, **on)
    turn = torch.randperm(rows, generator=g).to(dev)
    t2, l2 = ops.draw_actions(logits.to(dev)[turn], u[turn], **{k: v[turn] for k, v in on.items()})
    assert torch.equal(t2, token[turn]) and torch.equal(l2, logp[turn])
    wide = torch.zeros(rows, vocab + 5, dtype=torch.bfloat16, device=dev)[:, 3:vocab + 3]
    wide.copy_(logits)
    t3, l3 = ops.draw_actions(wide, u, **on)
    assert torch.equal(t3, token) and torch.equal(l3, logp)
    for i in (0, 9, 23):
        t4, l4 = ops.draw_actions(logits.to(dev)[i:i + 1], u[i:i + 1], **{k: v[i:i + 1] for k, v in on.items()})
        assert t4 == token[i] and l4 == logp[i]


@pytest.mark.parametrize("vocab", [6, 1500])
def test_frequencies(dev, vocab):
    """Evenly spaced numbers hit each index as often as its probability says, to within one."""
    n = 4096
    x = torch.randn(vocab, generator=_gen(8)) * 2
    p = ref.kept_probabilities(x, temperature=0.9, top_p=0.95)
    u = (torch.arange(n) + 0.5) / n
    token, _ = ops.draw_actions(x.to(dev).expand(n, vocab), u.to(dev), temperature=0.9, top_p=0.95)
    count = torch.bincount(token.cpu(), minlength=vocab).double()
    assert float((count - n * p).abs().max()) <= 1.0 + n * FAR


def test_ends_of_the_uniform_number(dev):
    x = torch.zeros(6, 10)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, float("nan")])
    token, _ = ops.draw_actions(x.to(dev), u.to(dev))
    assert token.tolist() == [0, 9, 9, 9, 0, 0]


def test_draw_of_far_rows_and_on_streams(dev):
    vocab = 4000
    far = torch.empty((1 << 31) + vocab, dtype=torch.bfloat16, device=dev).as_strided((2, vocab), (1 << 31, 1))
    x = torch.randn(2, vocab, generator=_gen(1)).to(torch.bfloat16)
    far.copy_(x)
    u = torch.tensor([0.3, 0.6], device=dev)
    want = ops.draw_actions(x.to(dev), u, top_k=30)
    assert torch.equal(ops.draw_actions(far, u, top_k=30)[0], want[0])
    side = torch.cuda.Stream(dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = ops.draw_actions(x.to(dev), u, top_k=30)
    side.synchronize()
    assert torch.equal(got[0], want[0])
    logits, uu = x.to(dev), u.clone()
    grads = [torch.randn(1000, device=dev) for _ in range(3)]
    held = [g.clone() for g in grads]
    out = [torch.empty_like(g) for g in grads]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    print("case draw and clip captured", flush=True)
    with torch.cuda.graph(graph):
        token, logp = ops.draw_actions(logits, uu, top_k=30, top_p=0.9)
        norm = ops.clip_grad_norm(grads, 1.0, out=out)
    for k in range(3):
        logits.copy_(torch.randn(2, vocab, generator=_gen(k)).to(torch.bfloat16))
        for g, h in zip(grads, held):
            g.copy_(h * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        t2, l2 = ops.draw_actions(logits, uu, top_k=30, top_p=0.9)
        out2 = [torch.empty_like(g) for g in grads]
        n2 = ops.clip_grad_norm(grads, 1.0, out=out2)
        assert torch.equal(token, t2) and torch.equal(logp, l2)
        assert torch.equal(norm, n2) and all(torch.equal(a, b) for a, b in zip(out, out2))


def test_draw_refusals(dev):
    x, u = torch.zeros(2, 5, device=dev), torch.zeros(2, device=dev)
    for f in (lambda: ops.draw_actions(x.cpu(), u), lambda: ops.draw_actions(x, u[:1]),
              lambda: ops.draw_actions(x, u.double()), lambda: ops.draw_actions(x.double(), u),
              lambda: ops.draw_actions(x, u, mask=torch.ones(2, 4, dtype=torch.bool, device=dev)),
              lambda: ops.draw_actions(x, u, mask=torch.ones(2, 5, device=dev)),
              lambda: ops.draw_actions(x, u, top_k=torch.ones(2, device=dev)),
              lambda: ops.draw_actions(x, u, temperature=torch.ones(3, device=dev))):
        with pytest.raises(ValueError):
            f()
    from surfgym import _sdfr
    with pytest.raises(_sdfr.SdfrError, match="vocabulary"):
        ops.draw_actions(torch.zeros(1, (1 << 18) + 1, device=dev), u[:1])
    token, logp = ops.draw_actions(torch.zeros(0, 5, device=dev), u[:0])
    assert token.shape == logp.shape == (0,)


# ------------------------------------------------------------------ clipping --
def _grads(dev, sizes, dtypes, scale, seed=0):
    g = _gen(seed)
    return [(torch.randn(n, generator=g) * scale).to(dtypes[i % len(dtypes)]).to(dev) for i, n in enumerate(sizes)]


@pytest.mark.parametrize("sizes", [[1], [7, 0, 4096, 4097], [100000, 3, 8191], [5] * 97, [1000 + i for i in range(300)],
                                   [9_000_001, 65536]])
@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float16, torch.float32, torch.bfloat16]])
def test_clipping(dev, sizes, dtypes):
    """The sum of squares is exact to 2^-50 or so: the norm is the 64-bit one rounded, and a clipped value the
    product in fp32 with a factor one rounding off, then rounded to its type."""
    for scale, clipped in ((3.0, True), (1e-6, False)):
        grads = _grads(dev, sizes, dtypes, scale)
        grads[0][0] = scale
        held = [g.clone() for g in grads]
        norm, factor = ref.clip([g.cpu() for g in grads], 1.0)
        assert (factor < 1.0) == clipped
        out = [torch.full_like(g, 7.0) for g in grads]
        got = ops.clip_grad_norm(grads, 1.0, out=out)
        assert abs(float(got) - norm) <= 2.0 ** -23 * norm
        assert all(torch.equal(a, b) for a, b in zip(grads, held))
        again = ops.clip_grad_norm(grads, 1.0)
        assert torch.equal(again, got) and all(torch.equal(a, b) for a, b in zip(grads, out))
        for g, h in zip(grads, held):
            unit = {torch.float32: 2.0 ** -22, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}[g.dtype]
            want = h.double() * factor
            assert bool(((g.double() - want).abs() <= unit * want.abs() + 6e-8 * (g.dtype == torch.float16)).all())
            if not clipped:
                assert torch.equal(g, h)


def test_clipping_of_views_at_any_address(dev):
    flat = torch.randn(10007, generator=_gen(1)).to(torch.bfloat16).to(dev)
    views = [flat[1:4000], flat[4001:4002], flat[4003:10000]]
    held = flat.clone()
    norm, factor = ref.clip([v.cpu() for v in views], 0.5)
    got = ops.clip_grad_norm(views, 0.5)
    assert abs(float(got) - norm) <= 2.0 ** -23 * norm
    for i in (0, 4000, 4002, *range(10000, 10007)):
        assert flat[i] == held[i]
    assert bool(((flat[1:4000].double() - held[1:4000].double() * factor).abs()
                 <= 2.0 ** -7 * held[1:4000].double().abs()).all())
    turned = torch.randn(33, 65, generator=_gen(2)).to(dev).t()          # dense, another order
    want = turned / (turned.double().norm() + 1e-6).float()
    ops.clip_grad_norm([turned], 1.0)
    assert torch.allclose(turned, want, rtol=1e-6, atol=0)


def test_clipping_of_what_is_not_finite(dev):
    big = torch.full((5000,), 1e30, device=dev)                          # squares past fp32
    norm = ops.clip_grad_norm([big], 1.0)
    assert abs(float(norm) / (1e30 * math.sqrt(5000)) - 1) < 1e-6
    assert abs(float(big.double().norm()) - 1) < 1e-6
    for bad in (float("nan"), float("inf")):
        g = [torch.ones(10, device=dev), torch.ones(5000, device=dev, dtype=torch.bfloat16)]
        g[1][77] = bad
        norm = ops.clip_grad_norm(g, 1.0)
        assert math.isnan(norm) if math.isnan(bad) else math.isinf(norm)
        assert g[1][77].isnan()
        assert bool(g[0].isnan().all()) if math.isnan(bad) else not g[0].any()


def test_clip_refusals(dev):
    g = torch.ones(4, 6, device=dev)
    for f in (lambda: ops.clip_grad_norm([], 1.0), lambda: ops.clip_grad_norm([g.cpu()], 1.0),
              lambda: ops.clip_grad_norm([g.double()], 1.0), lambda: ops.clip_grad_norm([g[:, ::2]], 1.0),
              lambda: ops.clip_grad_norm([g], 1.0, out=[]), lambda: ops.clip_grad_norm([g], 1.0, out=[g.half()]),
              lambda: ops.clip_grad_norm([g], 1.0, out=[g.t()])):
        with pytest.raises(ValueError):
            f()
    from surfgym import _sdfr
    with pytest.raises(_sdfr.SdfrError, match="negative"):
        ops.clip_grad_norm([g], -1.0)


@pytest.mark.parametrize("vocab", [9000, 20011, 65536, 70001])
def test_many_rows_draw_as_few_do(dev, vocab):
    """More rows than compute units may take another kernel; the answers are the same bits."""
    x = (torch.randn(300, vocab, generator=_gen(vocab)) * 3).to(torch.bfloat16).to(dev)
    u = torch.rand(300, generator=_gen(1)).to(dev)
    for s in (dict(), dict(top_k=50), dict(top_p=0.9), dict(top_k=700, top_p=0.95, min_p=0.01), dict(min_p=0.02)):
        token, logp = ops.draw_actions(x, u, **s)
        for at in (0, 100, 200):
            t, p = ops.draw_actions(x[at:at + 100], u[at:at + 100], **s)
            assert torch.equal(t, token[at:at + 100]) and torch.equal(p, logp[at:at + 100])


@pytest.mark.parametrize("vocab", [3000, 20000, 100000])
@pytest.mark.parametrize("equal", [100, 250, 300, 1000])
def test_some_of_many_equal_candidates(dev, vocab, equal):
    """Thresholds that fall among equal logits, few enough to rank and more."""
    g = _gen(vocab + equal)
    x = torch.randn(4, vocab, generator=g)
    for i in range(4):
        x[i, torch.randperm(vocab, generator=g)[:equal]] = 6.0
        x[i, torch.randperm(vocab, generator=g)[:5]] = 7.0
    for s in (dict(top_k=equal // 2), dict(top_k=equal // 2, top_p=0.6), dict(top_p=0.3), dict(top_k=5 + equal, top_p=0.9)):
        print("case equal", vocab, equal, s, flush=True)
        _check(dev, x, s, seed=3)


@pytest.mark.parametrize("vocab", [700, 3000, 20011])
def test_far_apart_and_far_from_zero(dev, vocab):
    """One logit so far above that the others weigh nothing; logits whose spacing is a sixteenth; tiny and huge
    temperatures."""
    g = _gen(vocab)
    x = torch.randn(4, vocab, generator=g)
    x[0, vocab // 3] = 100.0
    x[1, vocab // 3], x[1, vocab // 2] = 100.0, 100.0
    x[2] = x[2] * 3 + 1e6
    x[3] = x[3] * 3 - 1e6
    for s in (dict(top_k=50), dict(top_k=50, top_p=0.9), dict(top_p=0.9), dict(min_p=0.1), dict(temperature=1e-3, top_p=0.9),
              dict(temperature=1e4, top_p=0.5), dict(temperature=1e4, top_k=20, min_p=0.5)):
        print("case far", vocab, s, flush=True)
        _check(dev, x, s, seed=5)
