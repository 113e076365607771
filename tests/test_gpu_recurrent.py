"""surfgym.recurrent's memory operators against oracle.recurrent (64 bits) on the same inputs.

Tolerances, as the 2-norm of the difference over that of the result. The kernels compute in fp32 from inputs that
the oracle takes as they are. A step commits about six roundings of 2^-24, which are independent and add up as
their square root over at most 700 steps: 6 x 2^-24 x 26 = 1e-5, doubled; gradients go through the recurrence twice:
4e-5. Outputs of 16 bits are rounded once: at most half a unit, 2^-9 (bf16) and 2^-12 (fp16, 2^-11 relative) each,
doubled.
"""
from __future__ import annotations

import pytest
import torch

from oracle import recurrent as ref
from surfgym import recurrent as ops

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
OUT = {F32: 2e-5, F16: 2.0 ** -10, BF16: 2.0 ** -8}
GRAD = {F32: 4e-5, F16: 2.0 ** -10, BF16: 2.0 ** -8}


def _near(got, want, tol, what):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    err, size = float((got - want).norm()), float(want.norm())
    assert err <= tol * max(size, 1e-6), f"{what}: {err / max(size, 1e-30):.2e} over {tol:.0e}"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _scan_inputs(b, n, d, m, dtype, *, gate, skip, bias, resets, state, seed=0):
    g = _gen(seed + 1000 * n + d)
    t = {"x": torch.randn(b, n, d, generator=g).to(dtype), "dt": (torch.randn(b, n, d, generator=g) * 0.5 - 2).to(dtype),
         "A": -torch.rand(d, m, generator=g) * m - 0.5, "B": torch.randn(b, n, m, generator=g).to(dtype),
         "C": torch.randn(b, n, m, generator=g).to(dtype)}
    if gate:
        t["z"] = torch.randn(b, n, d, generator=g).to(dtype)
    if skip:
        t["D"] = torch.randn(d, generator=g)
    if bias:
        t["dt_bias"] = torch.randn(d, generator=g) * 0.5
    if state:
        t["state"] = torch.randn(b, d, m, generator=g)
    r = torch.rand(b, n, generator=g) < resets if resets else None
    dy, ds = torch.randn(b, n, d, generator=g).to(dtype), torch.randn(b, d, m, generator=g)
    return t, r, dy, ds


def _scan(t, r, softplus=True):
    kw = {k: t[k] for k in ("D", "z", "dt_bias", "state") if k in t}
    return ops.selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], softplus=softplus, resets=r,
                              return_state=True, **kw)


def _scan_ref(t, r, softplus=True, **kw):
    kw |= {k: t[k] for k in ("D", "z", "dt_bias", "state") if k in t}
    return ref.scan_grad(t["x"], t["dt"], t["A"], t["B"], t["C"], softplus=softplus, resets=r, **kw)


def _check_scan(dev, b, n, d, m, dtype, softplus=True, **opts):
    t, r, dy, ds = _scan_inputs(b, n, d, m, dtype, **opts)
    y, s, grads = _scan_ref(t, r, softplus, dy=dy, dstate_out=ds)
    gt = {k: v.to(dev).requires_grad_() for k, v in t.items()}
    gr = r.to(dev) if r is not None else None
    what = f"b {b} n {n} d {d} m {m} {dtype} {opts}"
    print("case scan", what, flush=True)
    with torch.no_grad():
        plain_y, plain_s = _scan(gt, gr, softplus)
    got_y, got_s = _scan(gt, gr, softplus)
    assert torch.equal(plain_y, got_y) and torch.equal(plain_s, got_s), what
    _near(got_y, y, OUT[dtype], what + " y")
    _near(got_s, s, OUT[F32], what + " state")
    got = torch.autograd.grad((got_y, got_s), list(gt.values()), (dy.to(dev), ds.to(dev)))
    for k, v in zip(gt, got):
        _near(v, grads[k], GRAD[v.dtype], what + " d" + k)


SIZES = [(1, 1, 1, 1), (2, 2, 3, 2), (2, 7, 5, 3), (3, 8, 64, 16), (2, 9, 65, 16), (1, 64, 130, 8), (2, 65, 63, 9),
         (1, 130, 70, 32), (2, 33, 20, 17), (1, 700, 33, 16), (40, 17, 129, 4)]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_scan_and_gradients(dev, size, dtype):
    _check_scan(dev, *size, dtype, gate=True, skip=True, bias=True, resets=0.05, state=True)


@pytest.mark.parametrize("opts", [dict(gate=False, skip=False, bias=False, resets=0.0, state=False),
                                  dict(gate=True, skip=False, bias=False, resets=0.0, state=True),
                                  dict(gate=False, skip=True, bias=True, resets=0.5, state=False),
                                  dict(gate=True, skip=True, bias=False, resets=1.0, state=True)])
@pytest.mark.parametrize("n", [5, 200])
def test_scan_options(dev, opts, n):
    _check_scan(dev, 2, n, 37, 16, F32, **opts)


def test_scan_without_softplus(dev):
    b, n, d, m = 2, 70, 37, 16
    t, r, dy, ds = _scan_inputs(b, n, d, m, F32, gate=True, skip=True, bias=False, resets=0.05, state=True)
    t["dt"] = t["dt"].abs() * 0.1
    y, s, grads = _scan_ref(t, r, False, dy=dy, dstate_out=ds)
    gt = {k: v.to(dev).requires_grad_() for k, v in t.items()}
    got_y, got_s = _scan(gt, r.to(dev), False)
    _near(got_y, y, OUT[F32], "y")
    for (k, _), v in zip(gt.items(), torch.autograd.grad((got_y, got_s), list(gt.values()), (dy.to(dev), ds.to(dev)))):
        _near(v, grads[k], GRAD[F32], "d" + k)


def test_scan_gradient_against_differences(dev):
    """The kernels' gradients against difference quotients of the 64-bit forward formula along a direction."""
    t, r, dy, ds = _scan_inputs(2, 40, 19, 5, F32, gate=True, skip=True, bias=True, resets=0.1, state=True)
    gt = {k: v.to(dev).requires_grad_() for k, v in t.items()}
    y, s = _scan(gt, r.to(dev))
    got = dict(zip(gt, torch.autograd.grad((y, s), list(gt.values()), (dy.to(dev), ds.to(dev)))))
    for k, v in t.items():
        u = torch.randn(v.shape, generator=_gen(3), dtype=torch.float64)

        def f(e):
            yy, ss, _ = _scan_ref({**t, k: v.double() + e * u}, r)
            return float((yy * dy).sum() + (ss * ds).sum())

        want = (f(1e-5) - f(-1e-5)) / 2e-5
        have = float((got[k].cpu().double() * u).sum())
        assert abs(have - want) <= 4e-5 * float(got[k].norm()) * float(u.norm()), k


@pytest.mark.parametrize("n", [40, 500])
def test_scan_reads_strided_inputs_where_they_lie(dev, n):
    """Halves of one projection, time-major rollouts, B and C shared by all sequences, odd offsets."""
    b, d, m = 3, 45, 16
    t, r, dy, ds = _scan_inputs(b, n, d, m, BF16, gate=True, skip=True, bias=True, resets=0.02, state=True)
    joint = torch.zeros(n, b, 2 * d + 1, dtype=BF16)
    joint[..., 1:d + 1], joint[..., d + 1:] = t["x"].transpose(0, 1), t["z"].transpose(0, 1)
    joint = joint.to(dev)
    proj = torch.zeros(b, n, d + 2 * m, dtype=BF16)
    t["B"], t["C"] = t["B"][:1].expand(b, n, m).contiguous(), t["C"]
    proj[..., :d], proj[..., d:d + m], proj[..., d + m:] = t["dt"], t["B"], t["C"]
    proj = proj.to(dev)
    resets = r.t().contiguous().to(dev).t()
    one = t["B"][:1].to(dev).requires_grad_()
    gt = {k: v.to(dev) for k, v in t.items()} | {
        "x": joint.transpose(0, 1)[..., 1:d + 1], "z": joint.transpose(0, 1)[..., d + 1:], "dt": proj[..., :d],
        "C": proj[..., d + m:], "B": one.expand(b, n, m)}
    y, s, grads = _scan_ref(t, r, dy=dy, dstate_out=ds)
    leaf = gt["x"].detach().requires_grad_()
    assert not leaf.is_contiguous()
    got_y, got_s = _scan({**gt, "x": leaf}, resets)
    _near(got_y, y, OUT[BF16], "y")
    turned = dy.transpose(0, 1).contiguous().to(dev).transpose(0, 1)
    dx, dB = torch.autograd.grad((got_y, got_s), (leaf, one), (turned, ds.to(dev)))
    _near(dx, grads["x"], GRAD[BF16], "dx")
    # b gradients of 16 bits are added up, in 16 bits
    _near(dB, grads["B"].sum(0, keepdim=True), 3 * GRAD[BF16], "dB")


def test_scan_past_offsets_of_32_bits(dev):
    b, n, d, m = 2, 20, 8, 16
    t, r, dy, ds = _scan_inputs(b, n, d, m, BF16, gate=False, skip=True, bias=True, resets=0.0, state=True)
    far = torch.empty((1 << 31) + 4096, dtype=BF16, device=dev)
    x = far.as_strided((b, n, d), (1 << 31, d, 1))
    x.copy_(t["x"])
    y, s, _ = _scan_ref(t, r)
    got_y, got_s = _scan({**{k: v.to(dev) for k, v in t.items()}, "x": x}, None)
    _near(got_y, y, OUT[BF16], "y")
    _near(got_s, s, OUT[F32], "state")


def test_nothing_comes_over_a_reset(dev):
    """What a sequence left behind is not multiplied by zero: infinities and NaN before a reset stay there."""
    b, n, d, m = 2, 300, 20, 16
    t, _, _, _ = _scan_inputs(b, n, d, m, F32, gate=True, skip=True, bias=True, resets=0.0, state=True)
    r = torch.zeros(b, n, dtype=torch.bool)
    r[0, 0], r[0, 150], r[1, 131] = True, True, True
    clean_y, clean_s, _ = _scan_ref(t, r)
    t["state"][0] = float("inf")
    t["x"][0, 100:150] = float("nan")
    t["x"][1, 7] = float("inf")
    y, s = _scan({k: v.to(dev) for k, v in t.items()}, r.to(dev))
    y, s = y.cpu().double(), s.cpu().double()
    for got, want in ((y[0, :100], clean_y[0, :100]), (y[0, 150:], clean_y[0, 150:]), (y[1, 131:], clean_y[1, 131:]),
                      (s, clean_s)):
        _near(got, want, OUT[F32], "after a reset")
    w, x = torch.randn(d, 4, generator=_gen(5)), t["x"]
    want, ws = ref.conv(torch.nan_to_num(x, nan=0.0, posinf=0.0), w, resets=r)
    got, gs = ops.causal_conv(x.to(dev), w.to(dev), resets=r.to(dev), return_state=True)
    _near(got[0, 150:], want[0, 150:], OUT[F32], "convolution after a reset")
    _near(got[1, 131:], want[1, 131:], OUT[F32], "convolution after a reset")


@pytest.mark.parametrize("m", [1, 4, 6, 8, 13, 16, 32])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_scan_steps_follow_the_scan(dev, m, dtype):
    b, n, d = 5, 6, 67
    t, r, _, _ = _scan_inputs(b, n, d, m, dtype, gate=True, skip=True, bias=True, resets=0.2, state=True)
    y, s, _ = _scan_ref(t, r)
    gt = {k: v.to(dev) for k, v in t.items()}
    gr = r.to(dev)
    state = gt["state"].clone()
    out = torch.empty(b, n, d, dtype=dtype, device=dev)
    for i in range(n):
        args = (gt["x"][:, i], gt["dt"][:, i], gt["A"], gt["B"][:, i], gt["C"][:, i], state)
        kw = dict(D=gt["D"], z=gt["z"][:, i], dt_bias=gt["dt_bias"], resets=gr[:, i])
        other = torch.full_like(state, float("nan"))
        before = state.clone()
        first = ops.selective_scan_step(*args, state_out=other, **kw)
        assert torch.equal(state, before)
        got = ops.selective_scan_step(*args, out=out[:, i], **kw)
        assert got.data_ptr() == out[:, i].data_ptr()
        assert torch.equal(first, got) and torch.equal(other, state)
    _near(out, y, OUT[dtype], "y")
    _near(state, s, OUT[F32], "state")


# ------------------------------------------------------------- convolution --
def _conv_inputs(b, n, d, width, dtype, resets, seed=0):
    g = _gen(seed + n + 100 * d)
    t = {"x": torch.randn(b, n, d, generator=g).to(dtype), "weight": torch.randn(d, width, generator=g),
         "bias": torch.randn(d, generator=g), "state": torch.randn(b, width - 1, d, generator=g).to(dtype)}
    r = torch.rand(b, n, generator=g) < resets if resets else None
    return t, r, torch.randn(b, n, d, generator=g).to(dtype), torch.randn(b, width - 1, d, generator=g).to(dtype)


@pytest.mark.parametrize("size", [(1, 1, 1, 1), (2, 1, 9, 4), (2, 2, 9, 4), (1, 3, 8, 8), (3, 15, 17, 2), (2, 16, 64, 4),
                                  (2, 17, 33, 3), (2, 18, 40, 5), (1, 131, 24, 4), (5, 40, 515, 4), (2, 50, 7, 8),
                                  (700, 33, 12, 4)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("silu", [False, True])
def test_convolution_and_gradients(dev, size, dtype, silu):
    b, n, d, width = size
    for resets, whole in ((0.1, True), (0.0, False)):
        t, r, dy, ds = _conv_inputs(b, n, d, width, dtype, resets)
        print("case conv", size, dtype, silu, resets, flush=True)
        keys = ["x", "weight", "bias", "state"] if whole else ["x", "weight"]
        kw = {k: t[k] for k in keys[2:]}
        y, s, grads = ref.conv_grad(t["x"], t["weight"], silu=silu, resets=r, dy=dy, dstate_out=ds, **kw)
        gt = {k: t[k].to(dev).requires_grad_() for k in keys}
        got_y, got_s = ops.causal_conv(gt["x"], gt["weight"], silu=silu, resets=r.to(dev) if r is not None else None,
                                       return_state=True, **{k: gt[k] for k in keys[2:]})
        _near(got_y, y, OUT[dtype], "y")
        assert torch.equal(got_s.cpu().double(), s)       # inputs, moved
        got = torch.autograd.grad((got_y, got_s), [gt[k] for k in keys], (dy.to(dev), ds.to(dev)))
        for k, v in zip(keys, got):
            if v.numel():
                _near(v, grads[k], GRAD[v.dtype], "d" + k)


def test_convolution_reads_strided_inputs_where_they_lie(dev):
    b, n, d = 3, 37, 21
    t, r, dy, _ = _conv_inputs(b, n, d, 4, BF16, 0.1)
    wide = torch.zeros(n, b, d + 3, dtype=BF16)
    wide[..., 2:d + 2] = t["x"].transpose(0, 1)
    x = wide.to(dev).transpose(0, 1)[..., 2:d + 2].requires_grad_()
    y, _, grads = ref.conv_grad(t["x"], t["weight"], resets=r, dy=dy)
    got = ops.causal_conv(x, t["weight"].to(dev), resets=r.to(dev).to(torch.uint8))
    _near(got, y, OUT[BF16], "y")
    dx, = torch.autograd.grad(got, x, dy.transpose(0, 1).contiguous().to(dev).transpose(0, 1))
    _near(dx, grads["x"], GRAD[BF16], "dx")
    far = torch.empty((1 << 31) + 4096, dtype=BF16, device=dev).as_strided((2, n, d), (1 << 31, d, 1))
    far.copy_(t["x"][:2])
    _near(ops.causal_conv(far, t["weight"].to(dev)), ref.conv(t["x"][:2], t["weight"])[0], OUT[BF16], "far")


@pytest.mark.parametrize("width", [1, 2, 4, 7])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_convolution_steps_follow_the_convolution(dev, width, dtype):
    b, n, d = 5, 9, 43
    t, r, _, _ = _conv_inputs(b, n, d, width, dtype, 0.2)
    y, s = ref.conv(t["x"], t["weight"], t["bias"], resets=r, state=t["state"])
    gt = {k: v.to(dev) for k, v in t.items()}
    state, out = gt["state"].clone(), torch.empty(b, n, d, dtype=dtype, device=dev)
    for i in range(n):
        args = (gt["x"][:, i], state, gt["weight"], gt["bias"])
        other = torch.full_like(state, float("nan"))
        first = ops.causal_conv_step(*args, resets=r[:, i].to(dev), state_out=other)
        got = ops.causal_conv_step(*args, resets=r[:, i].to(dev), out=out[:, i])
        assert torch.equal(first, got) and torch.equal(other, state)
    _near(out, y, OUT[dtype], "y")
    assert torch.equal(state.cpu().double(), s)


# ------------------------------------------------------------------- manner --
def test_calls_are_cut_anywhere(dev):
    b, n, d, m = 2, 300, 40, 16
    t, r, _, _ = _scan_inputs(b, n, d, m, F32, gate=True, skip=True, bias=True, resets=0.02, state=True)
    gt = {k: v.to(dev) for k, v in t.items()}
    r = r.to(dev)
    w = torch.randn(d, 4, generator=_gen(1)).to(dev)
    y, s = _scan(gt, r)
    cy, cs = ops.causal_conv(gt["x"], w, resets=r, return_state=True)
    for cut in (1, 2, 15, 64, 299):
        parts, state, cparts, cstate = [], gt["state"], [], None
        for at in (slice(0, cut), slice(cut, n)):
            part = {k: v[:, at] if k in ("x", "dt", "z", "B", "C") else v for k, v in gt.items()}
            yy, state = _scan({**part, "state": state}, r[:, at])
            parts.append(yy)
            yy, cstate = ops.causal_conv(gt["x"][:, at], w, resets=r[:, at], state=cstate, return_state=True)
            cparts.append(yy)
        _near(torch.cat(parts, 1), y.cpu(), OUT[F32], "y")
        _near(state, s.cpu(), OUT[F32], "state")
        assert torch.equal(torch.cat(cparts, 1), cy) and torch.equal(cstate, cs)


def test_empty_batches(dev):
    for b, n, d in ((0, 4, 8), (2, 0, 8), (2, 4, 0)):
        x = torch.randn(b, n, d, device=dev)
        A, B = -torch.ones(d, 16, device=dev), torch.randn(b, n, 16, device=dev)
        y, s = ops.selective_scan(x, x, A, B, B, return_state=True)
        assert y.shape == x.shape and s.shape == (b, d, 16) and not s.any()
        y, s = ops.causal_conv(x, torch.ones(d, 4, device=dev), return_state=True)
        assert y.shape == x.shape and s.shape == (b, 3, d)
        assert ops.causal_conv_step(x.new_zeros(b, d), s, torch.ones(d, 4, device=dev)).shape == (b, d)


def test_runs_on_the_current_stream_and_in_a_graph(dev):
    """Behind the work that makes its inputs on a side stream, and captured: replayed on new inputs with eager calls
    in between, each replay the same bits as the eager call."""
    b, n, d, m = 3, 400, 70, 16
    sets = []
    for seed in range(3):
        t, r, dy, _ = _scan_inputs(b, n, d, m, F32, gate=True, skip=True, bias=True, resets=0.02, state=True, seed=seed)
        sets.append(({k: v.to(dev) for k, v in t.items()}, r.to(dev), dy.to(dev)))
    w = torch.randn(d, 4, generator=_gen(1)).to(dev)

    def work(t, r, dy):
        t = {k: v.detach().requires_grad_() for k, v in t.items()}
        y, s = _scan(t, r)
        c = ops.causal_conv(t["x"], w, resets=r)
        grads = torch.autograd.grad((y, s, c), list(t.values()), (dy, torch.ones_like(s), dy))
        return [v.detach() for v in (y, s, c)] + list(grads)

    want = [work(*s) for s in sets]
    again = work(*sets[0])
    assert all(torch.equal(a, b) for a, b in zip(again, want[0]))
    torch.cuda.synchronize()
    side = torch.cuda.Stream(dev)
    print("case side stream", flush=True)
    with torch.cuda.stream(side):
        big = torch.randn(2048, 2048, device=dev)
        for _ in range(10):
            big = big @ big * 1e-3
        late = {k: v + (big[0, 0] * 0.0).nan_to_num() for k, v in sets[0][0].items()}
        got = work(late, *sets[0][1:])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    t, r, dy = {k: v.clone() for k, v in sets[0][0].items()}, sets[0][1].clone(), sets[0][2].clone()
    state, y = torch.zeros_like(t["state"]), torch.empty(b, d, device=dev)
    graph = torch.cuda.CUDAGraph()
    print("case captured", flush=True)
    with torch.cuda.graph(graph):
        out, _ = ops.selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], D=t["D"], z=t["z"], dt_bias=t["dt_bias"],
                                    resets=r, state=t["state"], return_state=True)
        c = ops.causal_conv(t["x"], w, resets=r)
        ops.selective_scan_step(t["x"][:, 0], t["dt"][:, 0], t["A"], t["B"][:, 0], t["C"][:, 0], t["state"], out=y,
                                state_out=state)
    for (nt, nr, ndy), wanted in zip(sets, want):
        for k in t:
            t[k].copy_(nt[k])
        r.copy_(nr)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, wanted[0]) and torch.equal(c, wanted[2])
        s2 = nt["state"].clone()
        y2 = ops.selective_scan_step(nt["x"][:, 0], nt["dt"][:, 0], nt["A"], nt["B"][:, 0], nt["C"][:, 0], s2)
        assert torch.equal(y, y2) and torch.equal(state, s2)


def test_refusals(dev):
    x = torch.randn(2, 5, 8, device=dev)
    A, B = -torch.ones(8, 16, device=dev), torch.randn(2, 5, 16, device=dev)
    w = torch.ones(8, 4, device=dev)
    bad = [lambda: ops.selective_scan(x.cpu(), x, A, B, B), lambda: ops.selective_scan(x, x.half(), A, B, B),
           lambda: ops.selective_scan(x, x[:, :4], A, B, B), lambda: ops.selective_scan(x, x, A[:4], B, B),
           lambda: ops.selective_scan(x, x, A.half(), B, B), lambda: ops.selective_scan(x, x, A, B[..., :8], B),
           lambda: ops.selective_scan(x, x, -torch.ones(8, 33, device=dev), B, B),
           lambda: ops.selective_scan(x.double(), x.double(), A, B, B),
           lambda: ops.selective_scan(x, x, A, B, B, resets=torch.zeros(2, 4, dtype=torch.bool, device=dev)),
           lambda: ops.selective_scan(x, x, A, B, B, resets=torch.zeros(2, 5, device=dev)),
           lambda: ops.selective_scan(x, x, A, B, B, state=torch.zeros(2, 8, 15, device=dev)),
           lambda: ops.selective_scan(x[0], x[0], A, B, B),
           lambda: ops.selective_scan_step(x[:, 0], x[:, 0], A, B[:, 0], B[:, 0],
                                           torch.zeros(2, 16, 8, device=dev).transpose(1, 2)),
           lambda: ops.selective_scan_step(x[:, 0], x[:, 0], A, B[:, 0], B[:, 0], torch.zeros(2, 8, 16, device=dev),
                                           out=torch.zeros(2, 8, device=dev, dtype=BF16)),
           lambda: ops.causal_conv(x, torch.ones(8, 9, device=dev)), lambda: ops.causal_conv(x, w[:4]),
           lambda: ops.causal_conv(x, w.half()), lambda: ops.causal_conv(x, w, torch.ones(7, device=dev)),
           lambda: ops.causal_conv(x, w, state=torch.zeros(2, 2, 8, device=dev)),
           lambda: ops.causal_conv(x, w, state=torch.zeros(2, 3, 8, device=dev, dtype=BF16)),
           lambda: ops.causal_conv_step(x[:, 0], torch.zeros(2, 4, 8, device=dev), w)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
