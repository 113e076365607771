"""ctypes binding of libsdfr.so (include/sdfr.h).

Written the way the reference binds its C core (python/surfgym/core.py:1-19,
:444-448): explicit argtypes for every entry point and a refusal to run
against a library whose ABI version differs from the one this file mirrors.

torch is imported before the library is opened so that the HIP runtime torch
already loaded is the one libsdfr.so binds to: device pointers and streams
then pass between the two unchanged.
"""
from __future__ import annotations

import ctypes
import struct
from pathlib import Path

import torch  # noqa: F401  (load torch's HIP runtime first, see above)

PKG_ROOT = Path(__file__).resolve().parents[1]
LIB_PATH = PKG_ROOT / "lib" / "libsdfr.so"

ABI_VERSION = 15
NOALLOC_SCRATCH_BYTES = 24 << 20   # SDFR_NOALLOC_SCRATCH_BYTES

# element types (SDFR_* in sdfr.h)
F32, F16, BF16, I32, I64, U8, F64, U16, R16 = 0, 1, 2, 3, 4, 5, 6, 7, 8
LAYOUT_LINEAR, LAYOUT_BRICK4 = 0, 1
CAM_EQUIANGULAR, CAM_PINHOLE = 0, 1
SCHED_PERSISTENT, SCHED_TILES = 0, 1
ORDER_LAUNCH, ORDER_LOOKAHEAD = 0, 1
FACES_AUTO, FACES_ON, FACES_OFF = 0, 1, 2

EXPORTS = ("sdfr_abi_version", "sdfr_last_error", "sdfr_grid_create", "sdfr_grid_destroy",
           "sdfr_grid_bytes", "sdfr_grid_attach_surfnz", "sdfr_grid_set_schedule",
           "sdfr_grid_set_tile_order", "sdfr_grid_set_border_faces", "sdfr_grid_set_march_events",
           "sdfr_render_rays_per_lane",
           "sdfr_workspace_bytes", "sdfr_render", "sdfr_render_noalloc", "sdfr_ray_dirs",
           "sdfr_grid_read",
           "sdfr_edt_workspace_bytes",
           "sdfr_edt", "sdfr_edt_last_error", "sdfr_goal_workspace_bytes", "sdfr_goal_bake",
           "sdfr_goal_sample", "sdfr_goal_yaw", "sdfr_goal_last_error",
           "sdfr_conv", "sdfr_conv_grad_workspace_bytes", "sdfr_conv_grad",
           "sdfr_scan_workspace_bytes", "sdfr_scan_marks_bytes", "sdfr_scan", "sdfr_scan_grad",
           "sdfr_draw", "sdfr_clip_workspace_bytes", "sdfr_clip", "sdfr_recurrent_last_error")


class GridDesc(ctypes.Structure):
    _fields_ = [("nx", ctypes.c_int32), ("ny", ctypes.c_int32), ("nz", ctypes.c_int32),
                ("mins", ctypes.c_float * 3), ("cell", ctypes.c_float)]


class Cam(ctypes.Structure):
    _fields_ = [("width", ctypes.c_int32), ("height", ctypes.c_int32),
                ("hfov_deg", ctypes.c_double), ("vfov_deg", ctypes.c_double),
                ("tan_half_h", ctypes.c_double), ("tan_half_v", ctypes.c_double),
                ("range", ctypes.c_float), ("near", ctypes.c_float),
                ("hit_eps", ctypes.c_float), ("min_step", ctypes.c_float),
                ("max_steps", ctypes.c_int32), ("camera", ctypes.c_int32)]


class Poses(ctypes.Structure):
    _fields_ = [("origin", ctypes.c_void_p), ("origin_stride", ctypes.c_int64),
                ("yaw_deg", ctypes.c_void_p), ("yaw_stride", ctypes.c_int64),
                ("pitch_deg", ctypes.c_void_p), ("pitch_stride", ctypes.c_int64),
                ("ducked", ctypes.c_void_p), ("ducked_stride", ctypes.c_int64),
                ("ducked_dtype", ctypes.c_int32), ("n_envs", ctypes.c_int32)]


class Image(ctypes.Structure):
    _fields_ = [("out", ctypes.c_void_p), ("env_stride", ctypes.c_int64),
                ("dtype", ctypes.c_int32), ("channels", ctypes.c_int32),
                ("taps", ctypes.c_void_p)]


class GoalInfo(ctypes.Structure):
    _fields_ = [("reach_max", ctypes.c_float), ("sentinel", ctypes.c_float),
                ("quant", ctypes.c_float), ("sweeps", ctypes.c_int32),
                ("n_seed", ctypes.c_int64), ("tile_visits", ctypes.c_int64)]


_KINDS = {"p": ctypes.c_void_p, "q": ctypes.c_int64, "i": ctypes.c_int32, "f": ctypes.c_float}


def _fields(text: str):
    """ctypes fields from "name:kind" words; p pointer, q int64, i int32, f float."""
    return [(n, _KINDS[k]) for n, k in (w.split(":") for w in text.split())]


def _packer(text: str):
    """The same layout as a function from the fields' values to its bytes: a fifth of what filling a ctypes structure
    of 20 to 40 fields takes, in calls whose time is the host's. Null pointers are 0."""
    return struct.Struct("@" + "".join(w.split(":")[1] for w in text.split()).replace("p", "P")).pack


_CONV = ("x:p x_b:q x_t:q weight:p bias:p resets:p resets_b:q resets_t:q state:p "
         "y:p y_b:q y_t:q state_out:p length:q batch:i channels:i width:i dtype:i silu:i")
_CONV_GRAD = "dy:p dy_b:q dy_t:q dstate_out:p dx:p dstate:p dweight:p dbias:p"
_SCAN = ("x:p x_b:q x_t:q dt:p dt_b:q dt_t:q z:p z_b:q z_t:q B:p B_b:q B_t:q C:p C_b:q C_t:q "
         "A:p skip:p dt_bias:p resets:p resets_b:q resets_t:q state:p state_out:p marks:p "
         "y:p y_b:q y_t:q length:q batch:i channels:i states:i dtype:i softplus:i")
_SCAN_GRAD = "dout:p dout_b:q dout_t:q dstate_out:p dx:p ddt:p dz:p dB:p dC:p dA:p dskip:p ddt_bias:p dstate:p"
_DRAW = ("logits:p logits_row:q mask:p mask_row:q uniform:p temperature:p top_k:p top_p:p "
         "min_p:p temperature1:f top_k1:i top_p1:f min_p1:f token:p logp:p rows:i vocab:i dtype:i")


class Conv(ctypes.Structure):
    _fields_ = _fields(_CONV)
    pack = staticmethod(_packer(_CONV))


class ConvGrad(ctypes.Structure):
    _fields_ = _fields(_CONV_GRAD)
    pack = staticmethod(_packer(_CONV_GRAD))


class Scan(ctypes.Structure):
    _fields_ = _fields(_SCAN)
    pack = staticmethod(_packer(_SCAN))


class ScanGrad(ctypes.Structure):
    _fields_ = _fields(_SCAN_GRAD)
    pack = staticmethod(_packer(_SCAN_GRAD))


class Draw(ctypes.Structure):
    _fields_ = _fields(_DRAW)
    pack = staticmethod(_packer(_DRAW))


class Tensor(ctypes.Structure):
    _fields_ = _fields("in_:p out:p size:q dtype:i")


class SdfrError(RuntimeError):
    pass


_lib = None


def load(path: Path | str | None = None):
    """Open libsdfr.so once, declare its entry points, check the ABI."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = Path(path) if path is not None else LIB_PATH
    if not p.exists():
        raise SdfrError(f"native renderer {p} is not built (run __graft_entry__.build()); "
                        "there is no fallback path")
    lib = ctypes.CDLL(str(p))
    vp, i32, i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
    lib.sdfr_abi_version.restype = i32
    lib.sdfr_abi_version.argtypes = []
    lib.sdfr_last_error.restype = ctypes.c_char_p
    lib.sdfr_last_error.argtypes = []
    lib.sdfr_grid_create.restype = vp
    lib.sdfr_grid_create.argtypes = [ctypes.POINTER(GridDesc), vp, i32, i32, i32, i32, vp,
                                     ctypes.c_char_p, i32]
    lib.sdfr_grid_destroy.restype = None
    lib.sdfr_grid_destroy.argtypes = [vp]
    lib.sdfr_grid_bytes.restype = i64
    lib.sdfr_grid_bytes.argtypes = [vp]
    lib.sdfr_grid_attach_surfnz.restype = i32
    lib.sdfr_grid_attach_surfnz.argtypes = [vp, vp, i32, vp]
    lib.sdfr_grid_set_schedule.restype = i32
    lib.sdfr_grid_set_schedule.argtypes = [vp, i32, i32, i32]
    lib.sdfr_grid_set_tile_order.restype = i32
    lib.sdfr_grid_set_tile_order.argtypes = [vp, i32, i64]
    lib.sdfr_grid_set_border_faces.restype = i32
    lib.sdfr_grid_set_border_faces.argtypes = [vp, i32]
    lib.sdfr_grid_set_march_events.restype = i32
    lib.sdfr_render_rays_per_lane.restype = i32
    lib.sdfr_render_rays_per_lane.argtypes = [vp, ctypes.POINTER(Cam), i32]
    lib.sdfr_grid_set_march_events.argtypes = [vp, vp, vp]
    lib.sdfr_workspace_bytes.restype = i64
    lib.sdfr_workspace_bytes.argtypes = [ctypes.POINTER(Cam), i32]
    lib.sdfr_render.restype = i32
    lib.sdfr_render.argtypes = [vp, ctypes.POINTER(Cam), ctypes.POINTER(Poses),
                                ctypes.POINTER(Image), vp, i64, vp]
    lib.sdfr_render_noalloc.restype = i32
    lib.sdfr_render_noalloc.argtypes = [vp, ctypes.POINTER(Cam), ctypes.POINTER(Poses),
                                        ctypes.POINTER(Image), vp]
    lib.sdfr_grid_read.restype = i32
    lib.sdfr_grid_read.argtypes = [vp, vp, vp]
    lib.sdfr_ray_dirs.restype = i32
    lib.sdfr_ray_dirs.argtypes = [ctypes.POINTER(Cam), ctypes.POINTER(Poses), vp, vp]
    lib.sdfr_edt_workspace_bytes.restype = i64
    lib.sdfr_edt_workspace_bytes.argtypes = [i32, i32, i32]
    lib.sdfr_edt.restype = i32
    lib.sdfr_edt.argtypes = [vp, i32, i32, i32, ctypes.c_float, vp, i32, vp, i64, vp]
    lib.sdfr_edt_last_error.restype = ctypes.c_char_p
    lib.sdfr_edt_last_error.argtypes = []
    lib.sdfr_goal_workspace_bytes.restype = i64
    lib.sdfr_goal_workspace_bytes.argtypes = [i32, i32, i32]
    lib.sdfr_goal_bake.restype = i32
    lib.sdfr_goal_bake.argtypes = [vp, i32, i32, i32, ctypes.c_float, ctypes.POINTER(ctypes.c_int32),
                                   ctypes.POINTER(ctypes.c_int32), i32, vp, vp,
                                   ctypes.POINTER(GoalInfo), vp, i64, vp]
    lib.sdfr_goal_sample.restype = i32
    lib.sdfr_goal_sample.argtypes = [vp, i32, ctypes.c_float, i32, i32, i32,
                                     ctypes.POINTER(ctypes.c_double), ctypes.c_double,
                                     ctypes.c_double, vp, i32, i64, i64, vp, vp]
    lib.sdfr_goal_yaw.restype = i32
    lib.sdfr_goal_yaw.argtypes = lib.sdfr_goal_sample.argtypes
    lib.sdfr_goal_last_error.restype = ctypes.c_char_p
    lib.sdfr_goal_last_error.argtypes = []
    lib.sdfr_conv.restype = i32
    lib.sdfr_conv.argtypes = [ctypes.POINTER(Conv), vp]
    lib.sdfr_conv_grad_workspace_bytes.restype = i64
    lib.sdfr_conv_grad_workspace_bytes.argtypes = [ctypes.POINTER(Conv)]
    lib.sdfr_conv_grad.restype = i32
    lib.sdfr_conv_grad.argtypes = [ctypes.POINTER(Conv), ctypes.POINTER(ConvGrad), vp, i64, vp]
    lib.sdfr_scan_workspace_bytes.restype = i64
    lib.sdfr_scan_workspace_bytes.argtypes = [ctypes.POINTER(Scan), i32]
    lib.sdfr_scan_marks_bytes.restype = i64
    lib.sdfr_scan_marks_bytes.argtypes = [ctypes.POINTER(Scan)]
    lib.sdfr_scan.restype = i32
    lib.sdfr_scan.argtypes = [ctypes.POINTER(Scan), vp, i64, vp]
    lib.sdfr_scan_grad.restype = i32
    lib.sdfr_scan_grad.argtypes = [ctypes.POINTER(Scan), ctypes.POINTER(ScanGrad), vp, i64, vp]
    lib.sdfr_draw.restype = i32
    lib.sdfr_draw.argtypes = [ctypes.POINTER(Draw), vp]
    lib.sdfr_clip_workspace_bytes.restype = i64
    lib.sdfr_clip_workspace_bytes.argtypes = [ctypes.POINTER(Tensor), i32]
    lib.sdfr_clip.restype = i32
    lib.sdfr_clip.argtypes = [ctypes.POINTER(Tensor), i32, ctypes.c_double, ctypes.c_double, vp, vp, i64, vp]
    lib.sdfr_recurrent_last_error.restype = ctypes.c_char_p
    lib.sdfr_recurrent_last_error.argtypes = []
    got = lib.sdfr_abi_version()
    if got != ABI_VERSION:
        raise SdfrError(f"{p} reports ABI {got}, this binding mirrors ABI {ABI_VERSION}: "
                        "rebuild the library")
    if path is None:
        _lib = lib
    return lib


_packed: dict = {}


def packed(name: str):
    """An entry point of the loaded library that takes its descriptors as packed bytes (``Conv.pack(...)``)."""
    fn = _packed.get(name)
    if fn is None:
        lib = load()
        fn = lib[name]              # another function object than lib.<name>, with argument types of its own
        like = getattr(lib, name)
        fn.restype = like.restype
        fn.argtypes = [ctypes.c_char_p if hasattr(t, "contents") else t for t in like.argtypes]
        _packed[name] = fn
    return fn


def last_error(lib=None) -> str:
    lib = lib or load()
    return lib.sdfr_last_error().decode("utf-8", "replace")


def check(rc: int, what: str, lib=None) -> None:
    if rc != 0:
        raise SdfrError(f"{what} failed ({rc}): {last_error(lib)}")
