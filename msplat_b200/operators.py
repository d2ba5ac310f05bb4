"""Dropout and 4-bit colours on torch CUDA tensors: the operators that the
training step (engine.set_step_options) and the packed renderer
(engine.PackedGaussians) are made of, as calls of their own.

Every call runs on torch's current stream of its tensors' device, allocates
only its outputs (none where `out` is given) and does not wait.  Tensors are
float32 unless stated; a wrong shape, type, layout or device raises
ValueError before anything runs.  Autograd does not record the calls: a tensor
that requires a gradient is refused unless gradients are off (torch.no_grad());
the backward passes are calls of their own.  What is written into `out` counts
as modified in place; it must not overlap an input (but dropout works in
place).  No counterpart in the reference.
"""
from __future__ import annotations

import numpy as np
import torch

from . import _lib

REST_BASES = (0, 3, 8, 15, 24)      # SH coefficients beside dc, per channel, by degree
RECORD_BYTES = (8, 16, 24, 32, 48)  # bytes of a Gaussian's record, by degree
MAX_VIEWS = 64
MAX_INT = 2**31 - 1                 # largest count that the C-ABI takes as an int

# The current device's number and the handle of its current stream;
# torch.cuda.current_stream() builds a Stream object around the latter, which
# took 3.2 us of a 14 us call.  (A torch without CUDA has neither, and no
# tensor that passes the checks.)
_device_now = getattr(torch._C, "_cuda_getDevice", None)
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_F32 = np.dtype(np.float32)
_bound = {}     # the library's functions by name, once called


def _check(t, name: str, shape, dtype=torch.float32, device=None) -> None:
    if (isinstance(t, torch.Tensor) and t.dtype is dtype and t.is_cuda and t.shape == shape
            and t.is_contiguous() and (device is None or t.device == device) and not t.requires_grad):
        return
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor of {dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, not {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    _unrecorded(t, name)


def _unrecorded(t, name: str) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which this call does not record: "
                         "call it under torch.no_grad(), and its backward pass on the gradient")


# For outputs that the caller handed in, several at once
# (torch.autograd.graph.increment_version, which takes twice its time).
_written = torch._C._increment_version


def _count(n: int, name: str) -> None:
    """Refuses a count that the binding would cut down to 32 bits."""
    if n > MAX_INT:
        raise ValueError(f"{name} must be at most {MAX_INT}, not {n}")


def _run(fn: str, device, *args) -> None:
    call = _bound.get(fn) or _bound.setdefault(fn, getattr(_lib.load(), fn))
    index = device.index
    if index == _device_now():
        rc = call(*args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            rc = call(*args, _stream_of(index))
    if rc:
        _lib.check(rc, fn)


def _rows(t, name: str):
    """A tensor as (rows, cols, row stride): two dimensions with unit column
    stride, or contiguous of any number of dimensions (rows of the last
    one; one column where there is a single dimension)."""
    if t.is_neg():   # the sign is not in memory yet
        raise ValueError(f"{name} is a negated view: pass {name}.resolve_neg()")
    if t.dim() == 2 and (t.shape[1] <= 1 or t.stride(1) == 1):
        rows, cols = t.shape
        stride = t.stride(0) if rows > 1 else max(cols, 1)
        if stride >= cols:
            return rows, cols, stride
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous, or two-dimensional with contiguous rows")
    if t.dim() < 2:
        return t.numel(), 1, 1
    cols = t.shape[-1]
    return (t.numel() // cols if cols else 0), cols, cols


def dropout(x, rate: float, seed: int, step: int, whole_rows: bool = False, out=None):
    """msplat_dropout: x / (1 - rate) where kept, 0 where dropped; a draw per
    element, or per row of the last dimension (per element of a
    one-dimensional x).  A function of (seed, step) and the position alone:
    called on the gradient of the result it is the backward pass.  `out` may
    be x itself."""
    if not isinstance(x, torch.Tensor) or x.dtype != torch.float32 or not x.is_cuda:
        raise ValueError("x must be a CUDA tensor of torch.float32")
    if not 0.0 <= rate < 1.0:
        raise ValueError(f"the rate must be in [0, 1), not {rate}")
    _unrecorded(x, "x")
    rows, cols, xs = _rows(x, "x")
    _count(cols, "the columns of x")
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        ys = cols
    else:
        if not isinstance(out, torch.Tensor) or out.dtype != torch.float32 or out.device != x.device:
            raise ValueError("out must be a float32 tensor on x's device")
        if out.shape != x.shape:
            raise ValueError(f"out must have shape {tuple(x.shape)}, not {tuple(out.shape)}")
        _unrecorded(out, "out")
        ys = _rows(out, "out")[2]
        _written((out,))
    if rows and cols:
        _run("msplat_dropout", x.device, rows, cols, x.data_ptr(), xs, out.data_ptr(), ys, rate,
             int(seed) & (2**64 - 1), int(step) & (2**64 - 1), int(bool(whole_rows)))
    return out


def _degree_of(rest_bases: int) -> int:
    if rest_bases not in REST_BASES:
        raise ValueError(f"features_rest has {rest_bases} bases; SH degrees 0 to 4 have {REST_BASES}")
    return REST_BASES.index(rest_bases)


def _check_degree(degree: int) -> None:
    if degree not in (0, 1, 2, 3, 4):
        raise ValueError(f"the SH degree must be 0 to 4, not {degree}")


def mx4_pack(features_dc, features_rest, out=None):
    """msplat_mx4_pack: the 4-bit colour records (N, record bytes) uint8 of
    features_dc (N, 3) and features_rest (N, B, 3)."""
    if not isinstance(features_rest, torch.Tensor) or features_rest.dim() != 3:
        raise ValueError("features_rest must be a tensor of shape (N, B, 3)")
    n, bases = features_rest.shape[:2]
    degree = _degree_of(bases)
    _count(n, "the Gaussians")
    _check(features_rest, "features_rest", (n, bases, 3))
    dev = features_rest.device
    _check(features_dc, "features_dc", (n, 3), device=dev)
    shape = (n, RECORD_BYTES[degree])
    if out is None:
        out = features_dc.new_empty(shape, dtype=torch.uint8)
    else:
        _check(out, "out", shape, torch.uint8, dev)
        _written((out,))
    _run("msplat_mx4_pack", dev, n, degree, features_dc.data_ptr(), features_rest.data_ptr(),
         out.data_ptr())
    return out


def _check_records(records, degree: int):
    _check_degree(degree)
    if not isinstance(records, torch.Tensor) or records.dim() != 2:
        raise ValueError("records must be a tensor of shape (N, record bytes)")
    n = records.shape[0]
    _count(n, "the Gaussians")
    _check(records, "records", (n, RECORD_BYTES[degree]), torch.uint8)
    return n, records.device


def mx4_unpack(records, degree: int, out=None):
    """msplat_mx4_unpack: (features_dc (N, 3), features_rest (N, B, 3)) that
    the records stand for; `out` is such a pair."""
    n, dev = _check_records(records, degree)
    shapes = ((n, 3), (n, REST_BASES[degree], 3))
    if out is None:
        out = tuple(records.new_empty(s, dtype=torch.float32) for s in shapes)
    else:
        for t, s, name in zip(out, shapes, ("out[0]", "out[1]"), strict=True):
            _check(t, name, s, device=dev)
        _written(out)
    _run("msplat_mx4_unpack", dev, n, degree, records.data_ptr(), out[0].data_ptr(),
         out[1].data_ptr())
    return out


def _views(cam_pos):
    """Camera positions as C-ordered float32 (V, 3) in host bytes, and V."""
    if type(cam_pos) is not np.ndarray and isinstance(cam_pos, torch.Tensor):
        raise ValueError("cam_pos is host data: an array or nested list of shape (V, 3)")
    cams = np.asarray(cam_pos, _F32)
    shape = cams.shape
    if len(shape) != 2 or shape[1] != 3 or shape[0] > MAX_VIEWS:
        raise ValueError(f"cam_pos must have shape (V, 3), V <= {MAX_VIEWS}, not {shape}")
    return cams.tobytes(), shape[0]


def _use(degrees_to_use, degree: int) -> int:
    if degrees_to_use is None:
        return degree
    if not 0 <= degrees_to_use <= degree or degrees_to_use != int(degrees_to_use):
        raise ValueError(f"degrees_to_use must be 0 to {degree}, not {degrees_to_use}")
    return int(degrees_to_use)


def _radii(radii, views: int, n: int, dev):
    if radii is None:
        return None
    _check(radii, "radii", (views, n), torch.int32, dev)
    return radii.data_ptr()


def mx4_colors(records, degree: int, means, cam_pos, degrees_to_use=None, radii=None, out=None):
    """msplat_mx4_colors: raw SH colours (V, N, 3) of the records seen from
    cam_pos (V, 3; host).  Where radii (V, N) int32 is given and not positive,
    `out` keeps what it held (0 in a new one)."""
    n, dev = _check_records(records, degree)
    use = _use(degrees_to_use, degree)
    _check(means, "means", (n, 3), device=dev)
    cams, views = _views(cam_pos)
    rp = _radii(radii, views, n, dev)
    if out is None:
        out = (means.new_empty if radii is None else means.new_zeros)((views, n, 3))
    else:
        _check(out, "out", (views, n, 3), device=dev)
        _written((out,))
    _run("msplat_mx4_colors", dev, n, degree, use, means.data_ptr(), records.data_ptr(), views,
         cams, rp, out.data_ptr())
    return out


def mx4_colors_backward(v_colors, degree: int, means, cam_pos, degrees_to_use=None, radii=None,
                        out=None):
    """msplat_mx4_colors_backward: the gradients (v_dc (N, 3), v_rest
    (N, B, 3)) of the coefficients from v_colors (V, N, 3); `out` is such a
    pair."""
    _check_degree(degree)
    use = _use(degrees_to_use, degree)
    cams, views = _views(cam_pos)
    if not isinstance(means, torch.Tensor) or means.dim() != 2:
        raise ValueError("means must be a tensor of shape (N, 3)")
    n, dev = means.shape[0], means.device
    _count(n, "the Gaussians")
    _check(means, "means", (n, 3))
    _check(v_colors, "v_colors", (views, n, 3), device=dev)
    rp = _radii(radii, views, n, dev)
    shapes = ((n, 3), (n, REST_BASES[degree], 3))
    if out is None:
        out = (torch.empty_like(means), means.new_empty(shapes[1]))
    else:
        for t, s, name in zip(out, shapes, ("out[0]", "out[1]"), strict=True):
            _check(t, name, s, device=dev)
        _written(out)
    _run("msplat_mx4_colors_backward", dev, n, degree, use, means.data_ptr(), views,
         cams, rp, v_colors.data_ptr(), out[0].data_ptr(), out[1].data_ptr())
    return out
