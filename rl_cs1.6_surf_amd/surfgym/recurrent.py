"""Operators of a recurrent policy, next to the renders it sees.

The reference's trainer gives its policy a past by stacking frames, and draws
actions and clips gradients with torch. These are the operators a policy with
a memory needs instead, as HIP kernels behind the same C ABI as the renderer
(include/sdfr.h; csrc/conv.hip, scan.hip, draw.hip, clip.hip):

* :func:`causal_conv` and :func:`selective_scan`, the two halves of a selective
  state space memory, over a rollout's decisions or a prompt's tokens, with
  gradients (torch autograd), and their ``_step`` forms for one decision of
  every env;
* :func:`draw_actions`, one action or token a row from logits and a given
  uniform number a row: temperature, top-k, top-p, min-p, a mask of legal ones;
* :func:`clip_grad_norm`, the global gradient norm over many tensors, and
  clipping to it.

Activations are float32, float16 or bfloat16 device tensors, all of a call
alike; parameters and the scan's states are float32. Work goes onto the current
stream, nothing waits for the host, and calls may be captured into a graph.
There is no CPU path: a missing native library is an error.
"""
from __future__ import annotations

import ctypes

import torch

from . import _sdfr, vision

__all__ = ["causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step", "draw_actions",
           "clip_grad_norm"]

_CODES = {torch.float32: _sdfr.F32, torch.float16: _sdfr.F16, torch.bfloat16: _sdfr.BF16}


# ------------------------------------------------------------------ helpers --
def _check(rc: int, what: str) -> None:
    if rc != 0:
        raise _sdfr.SdfrError(f"{what} failed ({rc}): "
                              f"{_sdfr.load().sdfr_recurrent_last_error().decode('utf-8', 'replace')}")


def _call(device, entry: str, *args) -> None:
    """A C entry on the device's current stream; the device is switched only where it has to be."""
    fn = getattr(_sdfr.load(), entry)
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, vision._current_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, vision._current_stream(device))
    if rc != 0:
        _check(rc, entry)


def _workspace(nbytes: int, device):
    if nbytes < 0:
        _check(nbytes, "workspace size")
    return torch.empty(max(int(nbytes), 64), dtype=torch.uint8, device=device)


def _activation(name, t, shape, like=None):
    """``t`` with a unit last stride (copied only where it has none)."""
    if not torch.is_tensor(t) or t.device.type != "cuda":
        raise ValueError(f"{name} must be a tensor on a ROCm GPU; there is no CPU path")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype not in _CODES:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} is {t.dtype} on {t.device}, x {like.dtype} on {like.device}")
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _parameter(name, t, shape, like):
    if t is None:
        return None
    if not torch.is_tensor(t) or t.dtype != torch.float32 or t.device != like.device:
        raise ValueError(f"{name} must be a float32 tensor on {like.device}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t.contiguous()


def _resets(t, shape, like):
    if t is None:
        return None
    if not torch.is_tensor(t) or t.dtype not in (torch.bool, torch.uint8) or t.device != like.device:
        raise ValueError(f"resets must be a bool or uint8 tensor on {like.device}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"resets must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t


def _state(name, t, shape, dtype, like):
    if t is None:
        return None
    if not torch.is_tensor(t) or t.dtype != dtype or t.device != like.device:
        raise ValueError(f"{name} must be a {dtype} tensor on {like.device}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t.contiguous()


def _target(name, t, shape, dtype, like, dense):
    """A tensor the caller gives for an output: written where it is, so never copied."""
    if not torch.is_tensor(t) or t.dtype != dtype or t.device != like.device or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be a {dtype} tensor of shape {tuple(shape)} on {like.device}")
    if not t.is_contiguous() if dense else t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must be " + ("contiguous" if dense else "unit-strided in its last dimension"))
    return t


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _rows(t):
    """(pointer, batch stride, step stride) of a (batch, length, ...) tensor, or of none."""
    return (t.data_ptr(), t.stride(0), t.stride(1)) if t is not None else (None, 0, 0)


# -------------------------------------------------------------- convolution --
def _conv_desc(x, weight, bias, silu, resets, state, y, state_out):
    b, n, d = x.shape
    return _sdfr.Conv(*_rows(x), weight.data_ptr(), _ptr(bias), *_rows(resets), _ptr(state), *_rows(y),
                      _ptr(state_out), n, b, d, weight.shape[1], _CODES[x.dtype], int(bool(silu)))


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _conv(x, weight, bias, state, resets, silu):
    b, n, d = x.shape
    y = torch.empty((b, n, d), dtype=x.dtype, device=x.device)
    state_out = torch.empty((b, weight.shape[1] - 1, d), dtype=x.dtype, device=x.device)
    _call(x.device, "sdfr_conv", _conv_desc(x, weight, bias, silu, resets, state, y, state_out))
    return y, state_out


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, resets, silu):
        y, state_out = _conv(x, weight, bias, state, resets, silu)
        ctx.save_for_backward(x, weight, bias, state, resets)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return y, state_out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dstate_out):
        x, weight, bias, state, resets = ctx.saved_tensors
        b, n, d = x.shape
        dy = torch.zeros_like(x) if dy is None else _activation("the gradient of y", dy, x.shape, x)
        if dstate_out is not None:
            dstate_out = dstate_out.contiguous()
        dx = torch.empty((b, n, d), dtype=x.dtype, device=x.device)
        dweight = torch.empty_like(weight)
        dbias = torch.empty_like(bias) if bias is not None else None
        dstate = torch.empty_like(state) if state is not None else None
        desc = _conv_desc(x, weight, bias, ctx.silu, resets, state, dx, None)
        ws = _workspace(_sdfr.load().sdfr_conv_grad_workspace_bytes(desc), x.device)
        grad = _sdfr.ConvGrad(*_rows(dy), _ptr(dstate_out), dx.data_ptr(), _ptr(dstate), dweight.data_ptr(),
                              _ptr(dbias))
        _call(x.device, "sdfr_conv_grad", desc, grad, ws.data_ptr(), ws.numel())
        return dx, dweight, dbias, dstate, None, None


def causal_conv(x, weight, bias=None, *, silu: bool = True, resets=None, state=None, return_state: bool = False):
    """Short causal convolution of each channel: ``x`` (batch, length, channels), ``weight``
    (channels, width) whose last column weighs the present input, width 1 to 8, ``bias`` (channels);
    through SiLU unless ``silu`` is false.

    ``resets`` (batch, length) is true where a sequence begins: nothing from before is seen from there.
    ``state`` (batch, width - 1, channels), of ``x``'s type, holds the inputs before the first (oldest first;
    zeros without one); with ``return_state`` the result is ``(y, state)``, the second to be handed to the
    call that goes on. Differentiable in x, weight, bias and state.
    """
    if not torch.is_tensor(x) or x.dim() != 3:
        raise ValueError("x must be a (batch, length, channels) tensor")
    b, n, d = x.shape
    x = _activation("x", x, (b, n, d))
    if not torch.is_tensor(weight) or weight.dim() != 2 or not 1 <= weight.shape[1] <= 8:
        raise ValueError("weight must be (channels, width) with a width of 1 to 8")
    width = weight.shape[1]
    weight = _parameter("weight", weight, (d, width), x)
    bias = _parameter("bias", bias, (d,), x)
    resets = _resets(resets, (b, n), x)
    state = _state("state", state, (b, width - 1, d), x.dtype, x)
    if b == 0 or n == 0 or d == 0:
        y = x * 1.0
        out = state if state is not None else x.new_zeros((b, width - 1, d))
    else:
        go = _CausalConv.apply if _wants_grad(x, weight, bias, state) else _conv
        y, out = go(x, weight, bias, state, resets, silu)
    return (y, out) if return_state else y


@torch.no_grad()
def causal_conv_step(x, state, weight, bias=None, *, silu: bool = True, resets=None, out=None, state_out=None):
    """:func:`causal_conv` for one step of every sequence: ``x`` (batch, channels), ``state`` (batch, width - 1,
    channels), which is moved on in place unless ``state_out`` names another place for it; ``resets`` (batch,).
    Returns y (batch, channels), written to ``out`` if given."""
    if not torch.is_tensor(x) or x.dim() != 2:
        raise ValueError("x must be a (batch, channels) tensor")
    b, d = x.shape
    x = _activation("x", x, (b, d))
    if not torch.is_tensor(weight) or weight.dim() != 2 or not 1 <= weight.shape[1] <= 8:
        raise ValueError("weight must be (channels, width) with a width of 1 to 8")
    width = weight.shape[1]
    weight = _parameter("weight", weight, (d, width), x)
    bias = _parameter("bias", bias, (d,), x)
    state = _target("state", state, (b, width - 1, d), x.dtype, x, True)
    state_out = state if state_out is None else _target("state_out", state_out, (b, width - 1, d), x.dtype, x, True)
    resets = _resets(resets, (b,), x)
    y = torch.empty((b, d), dtype=x.dtype, device=x.device) if out is None \
        else _target("out", out, (b, d), x.dtype, x, False)
    if b and d:
        desc = _sdfr.Conv(x.data_ptr(), x.stride(0), 0, weight.data_ptr(), _ptr(bias), _ptr(resets),
                          resets.stride(0) if resets is not None else 0, 0, state.data_ptr(), y.data_ptr(),
                          y.stride(0), 0, state_out.data_ptr(), 1, b, d, width, _CODES[x.dtype], int(bool(silu)))
        _call(x.device, "sdfr_conv", desc)
    return y


# --------------------------------------------------------------------- scan --
def _scan_desc(x, dt, A, B, C, D, z, dt_bias, softplus, resets, state, y, state_out, marks):
    b, n, d = x.shape
    return _sdfr.Scan(*_rows(x), *_rows(dt), *_rows(z), *_rows(B), *_rows(C), A.data_ptr(), _ptr(D),
                      _ptr(dt_bias), *_rows(resets), _ptr(state), _ptr(state_out), _ptr(marks), *_rows(y), n, b, d,
                      A.shape[1], _CODES[x.dtype], int(bool(softplus)))


def _scan(x, dt, A, B, C, D, z, dt_bias, state, resets, softplus, keep=False):
    """y, the final state, and with ``keep`` what the gradients start from."""
    b, n, d = x.shape
    lib = _sdfr.load()
    y = torch.empty((b, n, d), dtype=x.dtype, device=x.device)
    state_out = torch.empty((b, d, A.shape[1]), dtype=torch.float32, device=x.device)
    marks = None
    desc = _scan_desc(x, dt, A, B, C, D, z, dt_bias, softplus, resets, state, y, state_out, None)
    if keep:
        marks = _workspace(lib.sdfr_scan_marks_bytes(desc), x.device)
        desc.marks = marks.data_ptr()
    ws = _workspace(lib.sdfr_scan_workspace_bytes(desc, 0), x.device)
    _call(x.device, "sdfr_scan", desc, ws.data_ptr(), ws.numel())
    return (y, state_out, marks) if keep else (y, state_out)


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, state, resets, softplus):
        y, state_out, marks = _scan(x, dt, A, B, C, D, z, dt_bias, state, resets, softplus, keep=True)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, state, resets, marks)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, state_out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dstate_out):
        x, dt, A, B, C, D, z, dt_bias, state, resets, marks = ctx.saved_tensors
        b, n, d = x.shape
        dout = torch.zeros_like(x) if dout is None else _activation("the gradient of y", dout, x.shape, x)
        if dstate_out is not None:
            dstate_out = dstate_out.contiguous()

        def like(t):
            return torch.empty(t.shape, dtype=t.dtype, device=t.device) if t is not None else None

        dx, ddt, dz, dB, dC = like(x), like(dt), like(z), like(B), like(C)
        dA, dD, dbias, dstate = like(A), like(D), like(dt_bias), like(state)
        desc = _scan_desc(x, dt, A, B, C, D, z, dt_bias, ctx.softplus, resets, state, dx, None, marks)
        ws = _workspace(_sdfr.load().sdfr_scan_workspace_bytes(desc, 1), x.device)
        grad = _sdfr.ScanGrad(*_rows(dout), _ptr(dstate_out), dx.data_ptr(), ddt.data_ptr(), _ptr(dz),
                              dB.data_ptr(), dC.data_ptr(), dA.data_ptr(), _ptr(dD), _ptr(dbias), _ptr(dstate))
        _call(x.device, "sdfr_scan_grad", desc, grad, ws.data_ptr(), ws.numel())
        return dx, ddt, dA, dB, dC, dD, dz, dbias, dstate, None, None


def _rates(A):
    if not torch.is_tensor(A) or A.dim() != 2 or not 1 <= A.shape[1] <= 32:
        raise ValueError("A must be (channels, states) with 1 to 32 states")
    return A.shape[1]


def selective_scan(x, dt, A, B, C, *, D=None, z=None, dt_bias=None, softplus: bool = True, resets=None, state=None,
                   return_state: bool = False):
    """Selective state space scan. Per channel d and state n, with step = softplus(dt + dt_bias) (or dt + dt_bias):

        h[t] = exp(step A[d, n]) h[t-1] + step x[t] B[t, n]
        y[t] = sum_n C[t, n] h[t] + D[d] x[t],  times z[t] sigmoid(z[t]) if there is a z

    ``x``, ``dt``, ``z`` (batch, length, channels), ``B``, ``C`` (batch, length, states), ``A`` (channels, states)
    with 1 to 32 states, ``D``, ``dt_bias`` (channels). ``resets`` (batch, length) is true where a sequence begins:
    the state is zero before it. ``state`` (batch, channels, states) float32 is what the scan starts from (zeros
    without one); with ``return_state`` the result is ``(y, state)``. Differentiable in everything but ``resets``.
    """
    if not torch.is_tensor(x) or x.dim() != 3:
        raise ValueError("x must be a (batch, length, channels) tensor")
    b, n, d = x.shape
    m = _rates(A)
    x = _activation("x", x, (b, n, d))
    dt = _activation("dt", dt, (b, n, d), x)
    z = _activation("z", z, (b, n, d), x) if z is not None else None
    B = _activation("B", B, (b, n, m), x)
    C = _activation("C", C, (b, n, m), x)
    A = _parameter("A", A, (d, m), x)
    D = _parameter("D", D, (d,), x)
    dt_bias = _parameter("dt_bias", dt_bias, (d,), x)
    resets = _resets(resets, (b, n), x)
    state = _state("state", state, (b, d, m), torch.float32, x)
    if b == 0 or n == 0 or d == 0:
        y = x * 1.0
        out = state if state is not None else torch.zeros((b, d, m), dtype=torch.float32, device=x.device)
    else:
        go = _SelectiveScan.apply if _wants_grad(x, dt, A, B, C, D, z, dt_bias, state) else _scan
        y, out = go(x, dt, A, B, C, D, z, dt_bias, state, resets, softplus)
    return (y, out) if return_state else y


@torch.no_grad()
def selective_scan_step(x, dt, A, B, C, state, *, D=None, z=None, dt_bias=None, softplus: bool = True, resets=None,
                        out=None, state_out=None):
    """:func:`selective_scan` for one step of every sequence: ``x``, ``dt``, ``z`` (batch, channels), ``B``, ``C``
    (batch, states), ``resets`` (batch,), ``state`` (batch, channels, states) float32, which is moved on in place
    unless ``state_out`` names another place for it. Returns y (batch, channels), written to ``out`` if given."""
    if not torch.is_tensor(x) or x.dim() != 2:
        raise ValueError("x must be a (batch, channels) tensor")
    b, d = x.shape
    m = _rates(A)
    x = _activation("x", x, (b, d))
    dt = _activation("dt", dt, (b, d), x)
    z = _activation("z", z, (b, d), x) if z is not None else None
    B = _activation("B", B, (b, m), x)
    C = _activation("C", C, (b, m), x)
    A = _parameter("A", A, (d, m), x)
    D = _parameter("D", D, (d,), x)
    dt_bias = _parameter("dt_bias", dt_bias, (d,), x)
    state = _target("state", state, (b, d, m), torch.float32, x, True)
    state_out = state if state_out is None else _target("state_out", state_out, (b, d, m), torch.float32, x, True)
    resets = _resets(resets, (b,), x)
    y = torch.empty((b, d), dtype=x.dtype, device=x.device) if out is None \
        else _target("out", out, (b, d), x.dtype, x, False)
    if b and d:
        desc = _sdfr.Scan(x.data_ptr(), x.stride(0), 0, dt.data_ptr(), dt.stride(0), 0, _ptr(z),
                          z.stride(0) if z is not None else 0, 0, B.data_ptr(), B.stride(0), 0, C.data_ptr(),
                          C.stride(0), 0, A.data_ptr(), _ptr(D), _ptr(dt_bias), _ptr(resets),
                          resets.stride(0) if resets is not None else 0, 0, state.data_ptr(), state_out.data_ptr(),
                          None, y.data_ptr(), y.stride(0), 0, 1, b, d, m, _CODES[x.dtype], int(bool(softplus)))
        _call(x.device, "sdfr_scan", desc, None, 0)
    return y


# --------------------------------------------------------------------- draw --
def _setting(name, v, rows, dtype, like):
    """(per-row tensor or None, the one value)."""
    if not torch.is_tensor(v):
        return None, v
    if v.device != like.device or tuple(v.shape) != (rows,) or v.dtype.is_floating_point != dtype.is_floating_point:
        raise ValueError(f"{name} must be a number or a {dtype} tensor of shape ({rows},) on {like.device}")
    return v.to(dtype).contiguous(), 0


@torch.no_grad()
def draw_actions(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask=None):
    """One index a row of ``logits`` (rows, vocab), drawn by ``uniform`` (rows,) float32 in [0, 1): the first index
    at which the running sum of the kept probabilities passes it. Returns ``(token, logp)``, int64 and float32: the
    index and its log-probability among the kept.

    ``temperature`` divides the logits (0: the largest, lowest index first); ``top_k`` keeps the likeliest k (0:
    all), ties to the lowest index; ``top_p`` keeps of those the ones before which less than ``top_p`` of their
    probability lies; ``min_p`` keeps those that are at least ``min_p`` times as likely as the likeliest. Each is a
    number or a tensor of one a row. ``mask`` (rows, vocab) bool is true where an index may be drawn; what a masked
    logit holds does not matter. A row that leaves nothing to draw gives -1 and logp 0, one with a NaN -1 and NaN.
    An answer does not go by batch or order: weights are whole multiples of 2^-40, whose sums are exact.
    """
    if not torch.is_tensor(logits) or logits.dim() != 2:
        raise ValueError("logits must be a (rows, vocab) tensor")
    rows, vocab = logits.shape
    logits = _activation("logits", logits, (rows, vocab))
    dev = logits.device
    if not torch.is_tensor(uniform) or uniform.device != dev or uniform.dtype != torch.float32 \
            or tuple(uniform.shape) != (rows,):
        raise ValueError(f"uniform must be a float32 tensor of shape ({rows},) on {dev}")
    uniform = uniform.contiguous()
    if mask is not None:
        if not torch.is_tensor(mask) or mask.dtype not in (torch.bool, torch.uint8) or mask.device != dev \
                or tuple(mask.shape) != (rows, vocab):
            raise ValueError(f"mask must be a bool tensor of shape ({rows}, {vocab}) on {dev}")
        if vocab > 1 and mask.stride(1) != 1:
            mask = mask.contiguous()
    t, t1 = _setting("temperature", temperature, rows, torch.float32, logits)
    k, k1 = _setting("top_k", top_k, rows, torch.int32, logits)
    p, p1 = _setting("top_p", top_p, rows, torch.float32, logits)
    m, m1 = _setting("min_p", min_p, rows, torch.float32, logits)
    token = torch.empty(rows, dtype=torch.int64, device=dev)
    logp = torch.empty(rows, dtype=torch.float32, device=dev)
    desc = _sdfr.Draw(logits.data_ptr(), logits.stride(0), _ptr(mask), mask.stride(0) if mask is not None else 0,
                      uniform.data_ptr(), _ptr(t), _ptr(k), _ptr(p), _ptr(m), t1, min(k1, 0x7fffffff), p1, m1,
                      token.data_ptr(), logp.data_ptr(), rows, vocab, _CODES[logits.dtype])
    _call(dev, "sdfr_draw", desc)
    return token, logp


# --------------------------------------------------------------------- clip --
def _dense(name, t):
    if not torch.is_tensor(t) or t.device.type != "cuda" or t.dtype not in _CODES:
        raise ValueError(f"{name} must be float32, float16 or bfloat16 tensors on a ROCm GPU; there is no CPU path")
    if not t.is_contiguous() and not torch._prims_common.is_non_overlapping_and_dense(t):
        raise ValueError(f"{name} must hold each of their elements once, without gaps")
    return t


@torch.no_grad()
def clip_grad_norm(grads, max_norm: float, *, out=None, eps: float = 1e-6):
    """The 2-norm over all elements of ``grads`` (tensors of any of the three types, mixed), a float32 scalar on the
    device, and each of them times min(1, max_norm / (norm + eps)): in place, or into the tensors of ``out``
    (``grads`` then stay as they are). A norm that is infinite or NaN goes into the gradients as such."""
    grads = [_dense("grads", g) for g in ([grads] if torch.is_tensor(grads) else grads) if g is not None]
    if not grads:
        raise ValueError("no gradients")
    dev = grads[0].device
    into = grads if out is None else [_dense("out", o) for o in ([out] if torch.is_tensor(out) else out)]
    if len(into) != len(grads):
        raise ValueError(f"{len(grads)} gradients, {len(into)} places for them")
    table = (_sdfr.Tensor * len(grads))()
    for row, g, o in zip(table, grads, into):
        if g.device != dev:
            raise ValueError(f"gradients on {dev} and {g.device}")
        if o is not g and (o.dtype != g.dtype or o.shape != g.shape or o.stride() != g.stride() or o.device != dev):
            raise ValueError("out must match the gradients in type, shape, strides and device")
        row.in_, row.out, row.size, row.dtype = g.data_ptr(), o.data_ptr(), g.numel(), _CODES[g.dtype]
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = _workspace(_sdfr.load().sdfr_clip_workspace_bytes(table, len(grads)), dev)
    _call(dev, "sdfr_clip", table, len(grads), float(max_norm), float(eps), norm.data_ptr(), ws.data_ptr(),
          ws.numel())
    return norm
