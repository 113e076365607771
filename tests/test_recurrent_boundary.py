"""The C boundary of a recurrent policy's operators without a GPU: struct layouts as the header's, and every refusal
before anything is launched."""
from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from surfgym import _sdfr, recurrent

ROOT = Path(__file__).resolve().parents[1]
FAKE = 64 * 1024   # never dereferenced: every case fails before a launch


def test_structs_match_the_header_layout(tmp_path):
    structs = {"SdfrConv": _sdfr.Conv, "SdfrConvGrad": _sdfr.ConvGrad, "SdfrScan": _sdfr.Scan,
               "SdfrScanGrad": _sdfr.ScanGrad, "SdfrDraw": _sdfr.Draw, "SdfrTensor": _sdfr.Tensor}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "sdfr.h"', "int main(void){"]
    for cname, cls in structs.items():
        lines.append(f'printf("{cname} sizeof %zu\\n", sizeof({cname}));')
        for field, _ in cls._fields_:
            lines.append(f'printf("{cname} {field} %zu\\n", offsetof({cname}, {field.rstrip("_")}));')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout
    for line in got.splitlines():
        cname, field, value = line.split()
        cls = structs[cname]
        at = getattr(cls, field + "_" if field == "in" else field, None)
        assert int(value) == (ctypes.sizeof(cls) if field == "sizeof" else at.offset), line


def _conv(**kw):
    a = dict(x=FAKE, x_b=40, x_t=8, weight=FAKE, y=FAKE, y_b=40, y_t=8, length=5, batch=2, channels=8, width=4,
             dtype=_sdfr.BF16, silu=1)
    return _sdfr.Conv(**(a | kw))


def _scan(**kw):
    a = dict(x=FAKE, x_b=40, x_t=8, dt=FAKE, dt_b=40, dt_t=8, B=FAKE, B_b=80, B_t=16, C=FAKE, C_b=80, C_t=16, A=FAKE,
             y=FAKE, y_b=40, y_t=8, length=5, batch=2, channels=8, states=16, dtype=_sdfr.F32, softplus=1)
    return _sdfr.Scan(**(a | kw))


def _refused(rc, code, needle):
    msg = _sdfr.load().sdfr_recurrent_last_error().decode()
    assert rc == code and needle in msg, (rc, msg)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(width=0), -2, "width"), (dict(width=9), -2, "width"), (dict(dtype=_sdfr.F64), -3, "dtype"),
    (dict(channels=0), -2, "sizes"), (dict(batch=-1), -2, "sizes"), (dict(weight=None), -1, "weight"),
    (dict(x=None), -1, "null"), (dict(y=None), -1, "null"), (dict(length=0), -2, "length"),
    (dict(channels=1 << 25), -2, "large"), (dict(length=1 << 40), -2, "large"),
    (dict(length=17, state=FAKE, state_out=FAKE), -2, "in place")])
def test_convolution_refuses(kw, code, needle):
    lib = _sdfr.load()
    _refused(lib.sdfr_conv(_conv(**kw), None), code, needle)
    assert lib.sdfr_conv(_conv(batch=0), None) == 0


def test_convolution_gradient_refuses():
    lib = _sdfr.load()
    need = lib.sdfr_conv_grad_workspace_bytes(_conv())
    assert need > 0
    grad = _sdfr.ConvGrad(dy=FAKE, dx=FAKE, dweight=FAKE)
    _refused(lib.sdfr_conv_grad(_conv(), None, FAKE, need, None), -1, "descriptor")
    _refused(lib.sdfr_conv_grad(_conv(), _sdfr.ConvGrad(dy=FAKE, dx=FAKE), FAKE, need, None), -1, "null")
    _refused(lib.sdfr_conv_grad(_conv(), grad, None, need, None), -1, "workspace")
    _refused(lib.sdfr_conv_grad(_conv(), grad, FAKE, need - 1, None), -2, "workspace")
    _refused(lib.sdfr_conv_grad(_conv(), grad, FAKE + 4, need, None), -2, "aligned")
    _refused(lib.sdfr_conv_grad(_conv(batch=0), grad, FAKE, need, None), -2, "nothing")


@pytest.mark.parametrize("kw,code,needle", [
    (dict(states=0), -2, "states"), (dict(states=33), -2, "states"), (dict(dtype=_sdfr.I32), -3, "dtype"),
    (dict(channels=0), -2, "sizes"), (dict(length=-1), -2, "sizes"), (dict(A=None), -1, "rates"),
    (dict(dt=None), -1, "null"), (dict(C=None), -1, "null"), (dict(length=0), -2, "length"),
    (dict(channels=1 << 25), -2, "large"), (dict(batch=1 << 30, channels=1 << 20), -2, "large")])
def test_scan_refuses(kw, code, needle):
    lib = _sdfr.load()
    _refused(lib.sdfr_scan(_scan(**kw), FAKE, 1 << 40, None), code, needle)
    assert lib.sdfr_scan(_scan(batch=0), None, 0, None) == 0


def test_scan_workspace_and_gradient_refuse():
    lib = _sdfr.load()
    need, more = (lib.sdfr_scan_workspace_bytes(_scan(marks=FAKE), g) for g in (0, 1))
    assert 0 < need < more
    assert lib.sdfr_scan_workspace_bytes(_scan(length=1), 0) == 0
    assert lib.sdfr_scan_marks_bytes(_scan()) > 0
    _refused(lib.sdfr_scan(_scan(), None, 0, None), -1, "workspace")
    _refused(lib.sdfr_scan(_scan(), FAKE, need - 1, None), -2, "workspace")
    _refused(lib.sdfr_scan(_scan(), FAKE + 8, need, None), -2, "aligned")
    grad = dict(dout=FAKE, dx=FAKE, ddt=FAKE, dB=FAKE, dC=FAKE, dA=FAKE)
    _refused(lib.sdfr_scan_grad(_scan(marks=FAKE), None, FAKE, more, None), -1, "descriptor")
    _refused(lib.sdfr_scan_grad(_scan(), _sdfr.ScanGrad(**grad), FAKE, more, None), -1, "null")
    _refused(lib.sdfr_scan_grad(_scan(marks=FAKE, z=FAKE), _sdfr.ScanGrad(**grad), FAKE, more, None), -1, "null")
    _refused(lib.sdfr_scan_grad(_scan(marks=FAKE), _sdfr.ScanGrad(**(grad | dict(dA=None))), FAKE, more, None), -1,
             "null")
    _refused(lib.sdfr_scan_grad(_scan(marks=FAKE), _sdfr.ScanGrad(**grad), FAKE, more - 1, None), -2, "workspace")
    _refused(lib.sdfr_scan_grad(_scan(marks=FAKE, length=0), _sdfr.ScanGrad(**grad), FAKE, more, None), -2, "nothing")


@pytest.mark.parametrize("kw,code,needle", [
    (dict(vocab=0), -2, "vocabulary"), (dict(vocab=(1 << 18) + 1), -2, "vocabulary"), (dict(rows=-1), -2, "rows"),
    (dict(dtype=_sdfr.U8), -3, "dtype"), (dict(logits=None), -1, "null"), (dict(token=None), -1, "null")])
def test_draw_refuses(kw, code, needle):
    a = dict(logits=FAKE, logits_row=9, uniform=FAKE, temperature1=1.0, top_p1=1.0, token=FAKE, logp=FAKE, rows=2,
             vocab=9, dtype=_sdfr.F32)
    lib = _sdfr.load()
    _refused(lib.sdfr_draw(_sdfr.Draw(**(a | kw)), None), code, needle)
    assert lib.sdfr_draw(_sdfr.Draw(**(a | dict(rows=0))), None) == 0


def test_clip_refuses():
    lib = _sdfr.load()

    def one(**kw):
        return (_sdfr.Tensor * 1)(_sdfr.Tensor(**(dict(in_=FAKE, out=FAKE, size=10, dtype=_sdfr.F32) | kw)))

    need = lib.sdfr_clip_workspace_bytes(one(), 1)
    assert need > 0
    for args, code, needle in [((one(dtype=_sdfr.I64), 1, 1.0, 1e-6, FAKE, FAKE, need), -3, "dtype"),
                               ((one(size=-1), 1, 1.0, 1e-6, FAKE, FAKE, need), -2, "size"),
                               ((one(out=None), 1, 1.0, 1e-6, FAKE, FAKE, need), -1, "null"),
                               ((None, 1, 1.0, 1e-6, FAKE, FAKE, need), -1, "null"),
                               ((one(), -1, 1.0, 1e-6, FAKE, FAKE, need), -2, "count"),
                               ((one(), 1, -1.0, 1e-6, FAKE, FAKE, need), -2, "negative"),
                               ((one(), 1, float("nan"), 1e-6, FAKE, FAKE, need), -2, "negative"),
                               ((one(), 1, 1.0, 1e-6, None, FAKE, need), -1, "null"),
                               ((one(), 1, 1.0, 1e-6, FAKE, FAKE, need - 1), -2, "workspace"),
                               ((one(), 1, 1.0, 1e-6, FAKE, FAKE + 4, need), -2, "aligned")]:
        _refused(lib.sdfr_clip(*args, None), code, needle)


def test_python_refuses_the_cpu_instead_of_falling_back():
    x = torch.zeros(2, 5, 8)
    for f in (lambda: recurrent.causal_conv(x, torch.ones(8, 4)),
              lambda: recurrent.causal_conv_step(x[:, 0], torch.zeros(2, 3, 8), torch.ones(8, 4)),
              lambda: recurrent.selective_scan(x, x, torch.ones(8, 4), x[..., :4], x[..., :4]),
              lambda: recurrent.selective_scan_step(x[:, 0], x[:, 0], torch.ones(8, 4), x[:, 0, :4], x[:, 0, :4],
                                                    torch.zeros(2, 8, 4)),
              lambda: recurrent.draw_actions(x[0], torch.zeros(5)),
              lambda: recurrent.clip_grad_norm([x], 1.0)):
        with pytest.raises(ValueError, match="no CPU path"):
            f()
