"""What the operators of a recurrent policy are measured on (surfgym.recurrent).

A case is a dict of plain values; ``kind`` names the operator it goes through:

* ``conv`` / ``conv_train`` / ``conv_step``: the short causal convolution over a rollout or a
  prompt, with its gradients, and for one decision of every env;
* ``scan`` / ``scan_train`` / ``scan_step``: the selective state space scan, likewise;
* ``draw``: one action or token a row from logits and a given random number a row;
* ``clip``: the global gradient norm over many tensors, and clipping to it.

Rollouts are the renderer's: up to 2048 envs, 128 decisions, episodes that begin anywhere
(``resets``). Prompts are one or a few long sequences.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_ROOT = Path(__file__).resolve().parents[1]
for _p in (str(_ROOT), str(_ROOT / "rl_cs1.6_surf_amd")):
    if _p not in sys.path:
        sys.path.insert(0, _p)

_DEV = "cuda"
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _ops():
    from surfgym import recurrent
    return recurrent


# ------------------------------------------------------------------- cases --
def _conv(kind, batch, length, channels, width=4, dtype="bf16", silu=True, resets=0.0):
    return {"kind": kind, "batch": batch, "length": length, "channels": channels, "width": width,
            "dtype": dtype, "silu": silu, "resets": resets}


def _scan(kind, batch, length, channels, states=16, dtype="bf16", gate=True, resets=0.0):
    return {"kind": kind, "batch": batch, "length": length, "channels": channels, "states": states,
            "dtype": dtype, "gate": gate, "resets": resets}


def _draw(rows, vocab, dtype="f32", legal=1.0, top_k=0, top_p=1.0, min_p=0.0, each=False, spread=3.0):
    return {"kind": "draw", "rows": rows, "vocab": vocab, "dtype": dtype, "legal": legal, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "each": each, "spread": spread}


def _clip(tensors, elements, dtype="f32", scale=1.0):
    return {"kind": "clip", "tensors": tensors, "elements": elements, "dtype": dtype, "scale": scale}


def listed():
    return [
        # the update's minibatch: 256 envs' rollouts of 128 decisions, episodes beginning inside them
        {"name": "conv_rollout_train", **_conv("conv_train", 256, 128, 512, resets=0.005)},
        # one decision of every env: the window moves on by one
        {"name": "conv_decision_2048", **_conv("conv_step", 2048, 1, 512)},
        # the smallest call: a few envs that are evaluated, latency counts
        {"name": "scan_decision_64", **_scan("scan_step", 64, 1, 256, dtype="f32")},
        # one decision of every env of a rollout
        {"name": "scan_decision_2048", **_scan("scan_step", 2048, 1, 1024)},
        # one long prompt: few rows, a long axis
        {"name": "scan_prompt_8192", **_scan("scan", 1, 8192, 1024)},
        # the update's minibatch through the memory, episodes beginning inside it
        {"name": "scan_rollout_train", **_scan("scan_train", 256, 128, 512, resets=0.005)},
        # packed sequences of odd sizes in full precision
        {"name": "scan_packed_train", **_scan("scan_train", 2, 3001, 751, dtype="f32", resets=0.002)},
        # a rollout's actions: a small head, some actions illegal in some states
        {"name": "draw_actions_2048", **_draw(2048, 243, legal=0.8)},
        # one token of one sequence
        {"name": "draw_one_token", **_draw(1, 50001, top_k=50, top_p=0.95)},
        # a served batch, every row with settings of its own
        {"name": "draw_batch_256", **_draw(256, 131072, dtype="bf16", each=True)},
        # the gradients of a policy of 2 M parameters
        {"name": "clip_policy", **_clip(26, 1_957_500, scale=3.0)},
        # a large model's: many tensors of half precision, the norms' and biases' in full
        {"name": "clip_many", **_clip(290, 400_000_000, dtype="bf16")},
    ]


def _between(rng, lo, hi):
    """A whole number, spread over the logarithm of its range."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["conv", "conv_train", "conv_step", "scan", "scan_train", "scan_step", "draw", "draw", "clip"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "draw":
        vocab = _between(rng, 2, 200_000)
        rows = _between(rng, 1, max(1, min(4096, 30_000_000 // vocab)))
        return _draw(rows, vocab, dtype, rng.choice([1.0, 1.0, 0.7]), rng.choice([0, 0, 1, 40, 1000]),
                     rng.choice([1.0, 0.9, 0.99]), rng.choice([0.0, 0.0, 0.05]), rng.random() < 0.4,
                     rng.uniform(0.5, 5.0))
    if kind == "clip":
        n = _between(rng, 1, 400)
        return _clip(n, _between(rng, 64 * n, 300_000_000), dtype, rng.choice([1.0, 1e-4]))
    resets = rng.choice([0.0, 0.0, 0.004, 0.05])
    channels = _between(rng, 16, 2500)
    if kind.endswith("step"):
        batch = _between(rng, 1, max(1, min(4096, 2_000_000 // channels)))
        length = 1
    else:
        most = 14_000_000 // channels
        length = _between(rng, 1, min(8192, most))
        batch = _between(rng, 1, max(1, min(2048, most // length)))
    if kind.startswith("conv"):
        return _conv(kind, batch, length, channels, rng.choice([2, 3, 4, 4]), dtype, rng.random() < 0.7, resets)
    return _scan(kind, batch, length, channels, rng.choice([4, 8, 13, 16, 16]), dtype, rng.random() < 0.7, resets)


# ------------------------------------------------------------------ inputs --
def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(int(seed))


def _clip_sizes(case):
    """Sizes that add up to about ``elements``: three quarters of the tensors are small (biases,
    norms), the rest share what is left evenly, each a little odd."""
    n, total = case["tensors"], case["elements"]
    small = [min(1 + (i * 389) % 4097, max(1, total // (8 * n))) for i in range(3 * n // 4)]
    large = n - len(small)
    left = (total - sum(small)) // large
    return [max(1, left + 3 * (2 * i - large)) for i in range(large)] + small


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    dt = _TYPES[case["dtype"]]
    f32 = {"device": _DEV, "dtype": torch.float32}

    def rand(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, **f32) * scale).to(dtype)

    def chance(p, *shape):
        return torch.rand(*shape, generator=g, **f32) < p

    s = dict(case)
    if kind == "draw":
        n, v = case["rows"], case["vocab"]
        s["logits"] = rand(n, v, scale=case["spread"])
        s["uniform"] = torch.rand(n, generator=g, **f32)
        s["mask"] = None
        if case["legal"] < 1.0:
            s["mask"] = chance(case["legal"], n, v)
            s["mask"][:, 0] = True                   # there is always something to do
        s["temperature"], s["k"], s["p"], s["m"] = 0.8, case["top_k"], case["top_p"], case["min_p"]
        if case["each"]:
            pick = torch.tensor([0, 20, 50, 200, 1000], device=_DEV, dtype=torch.int32)
            s["temperature"] = torch.rand(n, generator=g, **f32) * 0.6 + 0.6
            s["k"] = pick[torch.randint(0, 5, (n,), generator=g, device=_DEV)]
            s["p"] = torch.rand(n, generator=g, **f32) * 0.2 + 0.8
            s["m"] = torch.rand(n, generator=g, **f32) * 0.04 * chance(0.5, n)
        return s
    if kind == "clip":
        sizes = _clip_sizes(case)
        s["grads"] = [rand(k, scale=case["scale"] * 1e-3, dtype=dt if k > 4097 else torch.float32) for k in sizes]
        # the clipped ones go into flat buffers, one a type, each at a multiple of 64 elements
        flats, s["out"] = {}, []
        for kind_, only in (("f32", torch.float32), (case["dtype"], dt)):
            total = sum((x.numel() + 63) // 64 * 64 for x in s["grads"] if x.dtype == only)
            flats[kind_] = torch.zeros(total, device=_DEV, dtype=only)
        at = dict.fromkeys(flats, 0)
        for x in s["grads"]:
            kind_ = "f32" if x.dtype == torch.float32 else case["dtype"]
            s["out"].append(flats[kind_][at[kind_]:at[kind_] + x.numel()])
            at[kind_] += (x.numel() + 63) // 64 * 64
        s["flats"] = flats
        return s
    b, n, d = case["batch"], case["length"], case["channels"]
    s["resets"] = chance(case["resets"], b, n) if case["resets"] > 0.0 else None
    if kind.startswith("conv"):
        w = case["width"]
        s["x"] = rand(b, n, d)
        s["weight"] = rand(d, w, scale=w ** -0.5, dtype=torch.float32)
        s["bias"] = rand(d, scale=0.1, dtype=torch.float32)
        s["state"] = rand(b, w - 1, d)
        s["dy"] = rand(b, n, d)
        s["state_out"], s["out"] = torch.empty_like(s["state"]), torch.empty_like(s["x"])
    else:
        m = case["states"]
        s["x"] = torch.nn.functional.silu(rand(b, n, d, dtype=torch.float32)).to(dt)
        s["dt"] = rand(b, n, d, scale=0.5)
        # steps between a thousandth and a tenth, rates 1 ... states: what such a memory starts with
        step = torch.exp(torch.rand(d, generator=g, **f32) * math.log(100.0) + math.log(1e-3))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
        s["A"] = -torch.arange(1, m + 1, **f32) * (1.0 + 0.2 * torch.rand(d, m, generator=g, **f32))
        s["B"], s["C"] = rand(b, n, m), rand(b, n, m)
        s["D"] = 1.0 + rand(d, scale=0.1, dtype=torch.float32)
        s["z"] = rand(b, n, d) if case["gate"] else None
        s["state"] = rand(b, d, m, dtype=torch.float32, scale=0.3)
        s["dy"] = rand(b, n, d)
        s["state_out"], s["out"] = torch.empty_like(s["state"]), torch.empty_like(s["x"])
    return s


# -------------------------------------------------------------- plain forms --
def _ages(resets, b, n):
    """Steps since the last reset at or before each step; counts on from before the start."""
    t = torch.arange(n, device=_DEV).expand(b, n)
    if resets is None:
        return t + (1 << 20)
    since = torch.where(resets, t, t.new_full((), -(1 << 20)))
    return t - since.cummax(dim=1).values


def _plain_conv(s, grads):
    x, w, bias = s["x"].float(), s["weight"], s["bias"]
    b, n, d = x.shape
    width = w.shape[1]
    lag = torch.arange(width - 1, -1, -1, device=_DEV)                 # of column k of the weights
    full = torch.cat([s["state"].float(), x], dim=1)                   # row t + width - 1 is step t
    seen = _ages(s["resets"], b, n)[:, :, None] >= lag                 # (b, n, width)
    win = full.unfold(1, width, 1) * seen[:, :, None, :]               # (b, n, d, width)
    pre = (win * w).sum(-1) + bias
    gate = torch.sigmoid(pre) if s["silu"] else torch.ones_like(pre)
    y = pre * gate if s["silu"] else pre
    # what the next call's window starts with: the last rows, cleared before the last reset
    rows = full[:, n:] * (_ages(s["resets"], b, n)[:, -1:, None] >= lag[1:, None])
    out = {"y": y.to(s["x"].dtype), "state": rows.to(s["x"].dtype)}
    if not grads:
        return out
    dpre = s["dy"].float()
    dpre = dpre * gate * (1.0 + pre * (1.0 - gate)) if s["silu"] else dpre
    taps = dpre[..., None] * seen[:, :, None, :]                       # (b, n, d, width)
    out["dweight"] = (taps * full.unfold(1, width, 1)).sum((0, 1))
    out["dbias"] = dpre.sum((0, 1))
    taps = torch.nn.functional.pad(taps * w, (0, 0, 0, 0, width - 1, width - 1))
    # row r of `full` is column k's input at step r - k
    dfull = sum(taps[:, width - 1 - k: width - 1 - k + n + width - 1, :, k] for k in range(width))
    out["dx"] = dfull[:, width - 1:].to(s["x"].dtype)
    out["dstate"] = dfull[:, :width - 1].to(s["x"].dtype)
    return out


def _linear_recurrence(a, b):
    """h[:, t] = a[:, t] h[:, t - 1] + b[:, t] by doubling: after each turn a step has taken in twice as
    many before it."""
    back = 1
    while back < a.shape[1]:
        b = torch.cat([b[:, :back], torch.addcmul(b[:, back:], a[:, back:], b[:, :-back])], dim=1)
        a = torch.cat([a[:, :back], a[:, back:] * a[:, :-back]], dim=1)
        back *= 2
    return b


def _plain_scan(s, grads):
    x, raw, A = s["x"].float(), s["dt"].float() + s["dt_bias"], s["A"]
    B, C, D = s["B"].float(), s["C"].float(), s["D"]
    step = raw.clamp(min=0.0) + torch.log1p(torch.exp(-raw.abs()))
    a = torch.exp(step[..., None] * A)
    if s["resets"] is not None:
        a = a * ~s["resets"][:, :, None, None]
    ins = (step * x)[..., None] * B[:, :, None, :]
    first = ins.clone()
    first[:, 0] += a[:, 0] * s["state"]
    h = _linear_recurrence(a, first)
    y = (h * C[:, :, None, :]).sum(-1) + D * x
    z = s["z"].float() if s["z"] is not None else None
    gate = z * torch.sigmoid(z) if z is not None else 1.0
    out = {"y": (y * gate).to(s["x"].dtype), "state": h[:, -1].clone()}
    if not grads:
        return out
    dt = s["x"].dtype
    dout = s["dy"].float()
    dy = dout * gate
    if z is not None:
        sig = torch.sigmoid(z)
        out["dz"] = (dout * y * sig * (1.0 + z * (1.0 - sig))).to(dt)
    out["dC"] = (dy[..., None] * h).sum(2).to(dt)
    carried = torch.cat([s["state"][:, None], h[:, :-1]], dim=1) * a   # what each step keeps
    del h, first
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], dim=1)
    g = _linear_recurrence(after.flip(1), (dy[..., None] * C[:, :, None, :]).flip(1)).flip(1)
    del after
    out["dB"] = (g * (step * x)[..., None]).sum(2).to(dt)
    gb = (g * B[:, :, None, :]).sum(-1)
    kept = g * carried
    out["dx"] = (step * gb + D * dy).to(dt)
    dstep = x * gb + (kept * A).sum(-1)
    draw_ = dstep * torch.sigmoid(raw)
    out["ddt"] = draw_.to(dt)
    out["ddt_bias"] = draw_.sum((0, 1))
    out["dA"] = (kept * step[..., None]).sum((0, 1))
    out["dD"] = (dy * x).sum((0, 1))
    out["dstate"] = g[:, 0] * a[:, 0]
    return out


def _column(v, n, dtype):
    return v[:, None] if torch.is_tensor(v) else torch.full((n, 1), v, device=_DEV, dtype=dtype)


def _share(part, total):
    """floor(part * total / 2^24) for whole numbers part <= 2^24, total < 2^58, and whether a rest is left."""
    low = part * (total & 0xFFFFFFFF)
    return part * (total >> 32) * 256 + (low >> 24), (low & 0xFFFFFF) != 0


def _plain_draw(s):
    """Weights are whole multiples of 2^-40 of the likeliest's, so that their sums are exact and an answer does
    not go by the order in which they are added up."""
    x = s["logits"].float()
    n, v = x.shape
    if s["mask"] is not None:
        x = x.masked_fill(~s["mask"], -math.inf)
    t = _column(s["temperature"], n, torch.float32)
    k = _column(s["k"], n, torch.int32).long()
    p = _column(s["p"], n, torch.float32)
    least = _column(s["m"], n, torch.float32)
    top = x.max(dim=1, keepdim=True).values
    z = torch.where(x == top, torch.zeros_like(x), (x - top) * (1.0 / t))
    e = torch.exp(z)
    w = (e * 2.0 ** 40).long()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    k = torch.where((k <= 0) | (k > v), v, k)
    ws = ws * (torch.arange(v, device=_DEV) < k)
    mass = ws.cumsum(1)
    whole, rest = _share((p.clamp(0.0, 1.0) * 2.0 ** 24).long(), mass[:, -1:])
    bound = (whole + rest).clamp(min=1)
    ws = ws * ((mass - ws < bound) | (p >= 1.0))
    ws = ws * (e.gather(1, order) >= least.clamp(max=1.0))
    kept = torch.zeros_like(w).scatter_(1, order, ws)
    mass = kept.cumsum(1)
    total = mass[:, -1:]
    r = (s["uniform"][:, None].clamp(0.0, 1.0) * 2.0 ** 24).long().clamp(max=(1 << 24) - 1)
    token = (mass > _share(r, total)[0]).to(torch.uint8).argmax(dim=1)
    logp = z.gather(1, token[:, None]) - torch.log(total.float() * 2.0 ** -40)
    return {"token": token, "logp": logp[:, 0]}


def _plain_clip(s, max_norm=1.0):
    parts = torch.stack([(x.float() * x.float()).sum() for x in s["grads"]])
    norm = parts.sum().sqrt()
    scale = (max_norm / (norm + 1e-6)).clamp(max=1.0)
    for x, o in zip(s["grads"], s["out"]):
        o.copy_(x.float() * scale)
    return {"norm": norm, **s["flats"]}


# --------------------------------------------------------------------- runs --
def _run_own(s):
    ops = _ops()
    kind = s["kind"]
    if kind == "draw":
        token, logp = ops.draw_actions(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["k"],
                                       top_p=s["p"], min_p=s["m"], mask=s["mask"])
        return {"token": token, "logp": logp}
    if kind == "clip":
        return {"norm": ops.clip_grad_norm(s["grads"], 1.0, out=s["out"]), **s["flats"]}
    first = s["resets"][:, 0] if s["resets"] is not None else None
    if kind == "conv_step":
        ops.causal_conv_step(s["x"][:, 0], s["state"], s["weight"], s["bias"], silu=s["silu"], resets=first,
                             out=s["out"][:, 0], state_out=s["state_out"])
        return {"y": s["out"], "state": s["state_out"]}
    if kind == "scan_step":
        ops.selective_scan_step(s["x"][:, 0], s["dt"][:, 0], s["A"], s["B"][:, 0], s["C"][:, 0], s["state"],
                                D=s["D"], z=s["z"][:, 0] if s["z"] is not None else None, dt_bias=s["dt_bias"],
                                resets=first, out=s["out"][:, 0], state_out=s["state_out"])
        return {"y": s["out"], "state": s["state_out"]}
    if kind == "conv":
        y, state = ops.causal_conv(s["x"], s["weight"], s["bias"], silu=s["silu"], resets=s["resets"],
                                   state=s["state"], return_state=True)
        return {"y": y, "state": state}
    if kind == "scan":
        y, state = ops.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                                      dt_bias=s["dt_bias"], resets=s["resets"], state=s["state"], return_state=True)
        return {"y": y, "state": state}
    if kind == "conv_train":
        x, w, bias, st = (s[k].detach().requires_grad_() for k in ("x", "weight", "bias", "state"))
        y, state = ops.causal_conv(x, w, bias, silu=s["silu"], resets=s["resets"], state=st, return_state=True)
        dx, dw, db, ds = torch.autograd.grad(y, (x, w, bias, st), s["dy"])
        return {"y": y.detach(), "state": state.detach(), "dweight": dw, "dbias": db, "dx": dx, "dstate": ds}
    names = ["x", "dt", "A", "B", "C", "D", "dt_bias", "state"] + (["z"] if s["z"] is not None else [])
    t = {k: s[k].detach().requires_grad_() for k in names}
    y, state = ops.selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], D=t["D"], z=t.get("z"),
                                  dt_bias=t["dt_bias"], resets=s["resets"], state=t["state"], return_state=True)
    d = dict(zip(names, torch.autograd.grad(y, [t[k] for k in names], s["dy"])))
    out = {"y": y.detach(), "state": state.detach()}
    if "z" in d:
        out["dz"] = d["z"]
    for k in ("C", "B", "x", "dt", "dt_bias", "A", "D", "state"):
        out["d" + k] = d[k]
    return out


def run(state):
    if own:
        return _run_own(state)
    kind = state["kind"]
    if kind == "draw":
        return _plain_draw(state)
    if kind == "clip":
        return _plain_clip(state)
    with torch.no_grad():
        return (_plain_conv if kind.startswith("conv") else _plain_scan)(state, kind.endswith("train"))


# --------------------------------------------------------------------- work --
def work(case):
    kind, size = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind == "draw":
        cells = case["rows"] * case["vocab"]
        return {"bytes": cells * (size + (1 if case["legal"] < 1.0 else 0)) + case["rows"] * 16, "flops": 4 * cells}
    if kind == "clip":
        e = case["elements"]
        return {"bytes": 2 * e * size, "flops": 3 * e}
    b, n, d = case["batch"], case["length"], case["channels"]
    cells, train = b * n * d, kind.endswith("train")
    if kind.startswith("conv"):
        w = case["width"]
        bytes_ = cells * size * (4 if train else 2) + b * (w - 1) * d * size * (3 if train else 2) + d * (w + 1) * 4
        return {"bytes": bytes_ + (b * n if case["resets"] else 0), "flops": cells * (2 * w + 6) * (3 if train else 1)}
    m, z = case["states"], 1 if case["gate"] else 0
    bytes_ = cells * size * (3 + z) + 2 * b * n * m * size + 2 * b * d * m * 4 + d * (m + 2) * 4
    if train:
        bytes_ += cells * size * (3 + z) + 2 * b * n * m * size + b * d * m * 4 + d * (m + 2) * 4
    return {"bytes": bytes_ + (b * n if case["resets"] else 0), "flops": cells * (m * (7 + (20 if train else 0)) + 20)}


# -------------------------------------------------------------------- exact --
def _exact_conv(s, train):
    x, w, bias, dy = s["x"].double(), s["weight"].double(), s["bias"].double(), s["dy"].double()
    b, n, d = x.shape
    width = w.shape[1]
    r = s["resets"] if s["resets"] is not None else torch.zeros(b, n, dtype=torch.bool, device=_DEV)
    rows = [s["state"][:, j].double() for j in range(width - 1)]       # oldest first
    src = [torch.ones(b, dtype=torch.bool, device=_DEV)] * (width - 1)  # is that row still in sight?
    y, pre_all, seen_all = torch.empty_like(x), torch.empty_like(x), []
    for t in range(n):
        src = [m & ~r[:, t] for m in src]
        win = rows + [x[:, t]]
        seen = src + [torch.ones_like(r[:, t])]
        pre = bias + sum(win[k] * seen[k][:, None] * w[:, k] for k in range(width))
        pre_all[:, t] = pre
        y[:, t] = pre / (1.0 + torch.exp(-pre)) if s["silu"] else pre
        seen_all.append(seen)
        rows, src = win[1:], seen[1:]
    out = {"y": y, "state": torch.stack([q * m[:, None] for q, m in zip(rows, src)], 1)}
    if train:
        g = dy
        if s["silu"]:
            q = 1.0 / (1.0 + torch.exp(-pre_all))
            g = dy * (q + pre_all * q * (1.0 - q))
        dx = torch.zeros(b, n + width - 1, d, dtype=torch.float64, device=_DEV)
        dw = torch.zeros_like(w)
        full = torch.cat([s["state"].double(), x], 1)
        for t in range(n):
            for k in range(width):
                m = seen_all[t][k][:, None]
                dx[:, t + k] += g[:, t] * w[:, k] * m
                dw[:, k] += (g[:, t] * full[:, t + k] * m).sum(0)
        out |= {"dweight": dw, "dbias": g.sum((0, 1)), "dx": dx[:, width - 1:], "dstate": dx[:, :width - 1]}
    return out


def _exact_scan(s, train):
    x, raw, A = s["x"].double(), s["dt"].double() + s["dt_bias"].double(), s["A"].double()
    B, C, D, dout = s["B"].double(), s["C"].double(), s["D"].double(), s["dy"].double()
    b, n, d = x.shape
    step = torch.logaddexp(raw, torch.zeros_like(raw))
    h = s["state"].double()
    z = s["z"].double() if s["z"] is not None else None
    live = 1.0 - s["resets"].double() if s["resets"] is not None else torch.ones(b, n, dtype=torch.float64, device=_DEV)
    y = torch.empty_like(x)
    hist = torch.empty(n + 1, *h.shape, dtype=torch.float64, device=_DEV) if train else None
    for t in range(n):
        if train:
            hist[t] = h
        h = torch.exp(step[:, t, :, None] * A) * live[:, t, None, None] * h \
            + (step[:, t] * x[:, t])[..., None] * B[:, t, None, :]
        y[:, t] = torch.matmul(h, C[:, t, :, None])[..., 0] + D * x[:, t]
    q = 1.0 / (1.0 + torch.exp(-z)) if z is not None else None
    out = {"y": y * z * q if z is not None else y, "state": h}
    if not train:
        return out
    hist[n] = h
    if z is not None:
        out["dz"] = dout * y * (q + z * q * (1.0 - q))
    dy = dout * z * q if z is not None else dout
    g = torch.zeros_like(h)
    o = {"dC": torch.empty_like(C), "dB": torch.empty_like(B), "dx": torch.empty_like(x), "ddt": torch.empty_like(x),
         "ddt_bias": None, "dA": torch.zeros_like(A), "dD": (dy * x).sum((0, 1))}
    for t in range(n - 1, -1, -1):
        g = g + dy[:, t, :, None] * C[:, t, None, :]
        decay = torch.exp(step[:, t, :, None] * A) * live[:, t, None, None]
        kept = g * decay * hist[t]
        o["dC"][:, t] = (dy[:, t, :, None] * hist[t + 1]).sum(1)
        o["dB"][:, t] = (g * (step[:, t] * x[:, t])[..., None]).sum(1)
        gb = (g * B[:, t, None, :]).sum(-1)
        o["dx"][:, t] = step[:, t] * gb + D * dy[:, t]
        o["ddt"][:, t] = (x[:, t] * gb + (kept * A).sum(-1)) / (1.0 + torch.exp(-raw[:, t]))
        o["dA"] += (kept * step[:, t, :, None]).sum(0)
        g = g * decay
    o["ddt_bias"] = o["ddt"].sum((0, 1))
    return {**out, **o, "dstate": g}


def _exact_draw(s):
    """The log-probabilities in 64 bits; the tokens are whole numbers."""
    rows = s["logits"].double()
    n, v = rows.shape

    def of(key, i):
        return s[key][i].item() if torch.is_tensor(s[key]) else s[key]

    logp = []
    for i in range(n):
        x = rows[i] if s["mask"] is None else torch.where(s["mask"][i], rows[i], -math.inf)
        x, where = torch.sort(x, descending=True, stable=True)
        k = of("k", i)
        q = torch.exp((x[:k] if 0 < k < v else x) / of("temperature", i) - x[0] / of("temperature", i))
        if of("p", i) < 1.0:
            q = q[:int((q.cumsum(0) - q < of("p", i) * q.sum()).sum())]
        q = q[q >= min(of("m", i), 1.0)]
        at, by = where[:q.numel()].sort()
        c = q[by].cumsum(0)
        j = int((c <= s["uniform"][i].item() * c[-1]).sum().clamp(max=q.numel() - 1))
        logp.append(torch.log(q[by[j]] / c[-1]))
    return {"token": None, "logp": torch.stack(logp)}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "draw":
        return _exact_draw(s)
    if kind == "clip":
        norm = math.sqrt(sum(float((x.double() ** 2).sum()) for x in s["grads"]))
        scale = min(1.0, 1.0 / (norm + 1e-6))
        out = {k: v.double() for k, v in s["flats"].items()}
        at = dict.fromkeys(out, 0)
        for x in s["grads"]:
            k = "f32" if x.dtype == torch.float32 else case["dtype"]
            out[k][at[k]:at[k] + x.numel()] = x.double() * scale
            at[k] += -(-x.numel() // 64) * 64
        return {"norm": torch.tensor(norm, dtype=torch.float64, device=_DEV), **out}
    train = kind.endswith("train")
    return _exact_conv(s, train) if kind.startswith("conv") else _exact_scan(s, train)
