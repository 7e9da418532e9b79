"""Training a content encoder's unit head over libvfr_retrieval.so.

A content encoder learns to tell a frame's unit, the k-means cluster
(`vfr.training.kmeans`, `vfr.training.assign`) its features fall in.  The
operators here are that head on the device: layer norm of the frames, softmax
cross entropy against the codebook without keeping the logits, the gradients
of both, and 8-bit checkpoints that keep an activation until the backward
pass.  They are plain calls, forward and backward each its own, without
hooks into torch's autograd.

Tensors are contiguous CUDA tensors of one device, [rows, width] with width
up to 4,096.  The work runs on `stream` (default: the current stream of that
device) and the results belong to it; inputs made on another stream must be
ready before the call, as with any CUDA work.  Calls allocate only through
torch, so they can be captured into CUDA graphs.
"""
from __future__ import annotations

import ctypes
import dataclasses
import functools

import torch

from .lib import Stream, call, load_library

BLOCK = 128  # elements of a row that share one exponent
_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # VFR_F32, VFR_BF16, VFR_F16


@dataclasses.dataclass
class Checkpoint:
    """An activation in 8 bits: e4m3 `packed` [rows, width] (torch
    float8_e4m3fn), times 2^(byte - 127) per 128 elements of a row,
    `exponents` [rows, ceil(width / 128)] (uint8); `dtype` is the type it was
    packed from."""
    packed: torch.Tensor
    exponents: torch.Tensor
    dtype: torch.dtype


def _code(dtype) -> int:
    code = _CODES.get(dtype)
    if code is None:
        raise ValueError(f"expected float32, bfloat16 or float16, not {dtype}")
    return code


def _matrix(name, t) -> int:
    """Checks a matrix argument and returns its type's code."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == 2 and t.is_contiguous()):
        raise ValueError(f"{name}: expected a contiguous CUDA tensor [rows, width]")
    return _code(t.dtype)


def _like(name, t, shape, dtype, device):
    if not (isinstance(t, torch.Tensor) and t.dtype == dtype and t.shape == shape and t.device == device
            and t.is_contiguous()):
        raise ValueError(f"{name}: expected a contiguous {dtype} tensor {list(shape)} on {device}")


def _ptr(t):
    return None if t is None else t.data_ptr() or None


# The current stream's handle without a Stream object, where torch offers it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _launch(run, device, stream, inputs):
    """run(stream argument) with the tensors' device current.  With a stream
    of the caller's, what run allocates belongs to that stream, and the inputs
    are kept until its work is done."""
    index = device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return _launch(run, device, stream, inputs)
    if stream is None:
        return run(ctypes.byref(Stream(_raw_stream(index))))
    if stream.device != device:
        raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
    with torch.cuda.stream(stream):
        out = run(ctypes.byref(Stream(stream.cuda_stream)))
    for t in inputs:
        if t is not None:
            t.record_stream(stream)
    return out


@functools.lru_cache(maxsize=256)
def _workspace_size(query, *args) -> int:
    """Bytes a workspace query gives; its last argument is the device index
    (the current device, which the answer depends on)."""
    size = ctypes.c_size_t(0)
    call(getattr(load_library(), query), *args[:-1], ctypes.byref(size))
    return size.value


def _workspace(size, device):
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _blocks(width):
    return (width + BLOCK - 1) // BLOCK


def _empty_checkpoint(x):
    rows, width = x.shape
    return Checkpoint(torch.empty((rows, width), dtype=torch.float8_e4m3fn, device=x.device),
                      torch.empty((rows, _blocks(width)), dtype=torch.uint8, device=x.device), x.dtype)


def _check_checkpoint(c):
    p = c.packed
    if not (isinstance(p, torch.Tensor) and p.is_cuda and p.dim() == 2 and p.is_contiguous()
            and p.dtype == torch.float8_e4m3fn):
        raise ValueError("checkpoint: expected a contiguous CUDA float8_e4m3fn tensor [rows, width]")
    _like("checkpoint exponents", c.exponents, (p.shape[0], _blocks(p.shape[1])), torch.uint8, p.device)
    return c


def checkpoint_pack(x, stream=None) -> Checkpoint:
    """`x` in 8 bits (`vfr_checkpoint_pack`)."""
    code = _matrix("x", x)

    def run(s):
        out = _empty_checkpoint(x)
        call(load_library().vfr_checkpoint_pack, _ptr(x), x.shape[0], x.shape[1], code, _ptr(out.packed),
             _ptr(out.exponents), s)
        return out

    return _launch(run, x.device, stream, (x,))


def checkpoint_unpack(checkpoint: Checkpoint, dtype=None, stream=None):
    """The checkpoint's values, in `dtype` (default: the type it was packed
    from; float32 holds them exactly, but for magnitudes from 1.9375 * 2^127 on,
    which come out as infinities)."""
    c = _check_checkpoint(checkpoint)
    dtype = c.dtype if dtype is None else dtype
    code = _code(dtype)

    def run(s):
        x = torch.empty_like(c.packed, dtype=dtype)
        call(load_library().vfr_checkpoint_unpack, _ptr(c.packed), _ptr(c.exponents), x.shape[0], x.shape[1], code,
             _ptr(x), s)
        return x

    return _launch(run, c.packed.device, stream, (c.packed, c.exponents))


def layer_norm(x, gamma=None, beta=None, eps: float = 1e-5, checkpoint: bool = False, stream=None):
    """(y, mean, rstd) of the rows of `x` (`vfr_layer_norm`): y of x's type,
    mean and rstd float32 [rows]; gamma and beta float32 [width].  With
    `checkpoint`, also x's `Checkpoint`, written in the same pass."""
    code = _matrix("x", x)
    rows, width = x.shape
    device = x.device
    if gamma is not None:
        _like("gamma", gamma, (width,), torch.float32, device)
    if beta is not None:
        _like("beta", beta, (width,), torch.float32, device)

    def run(s):
        y = torch.empty_like(x)
        mean = torch.empty(rows, dtype=torch.float32, device=device)
        rstd = torch.empty_like(mean)
        saved = _empty_checkpoint(x) if checkpoint else None
        call(load_library().vfr_layer_norm, _ptr(x), _ptr(gamma), _ptr(beta), rows, width, code, eps, _ptr(y),
             _ptr(mean), _ptr(rstd), _ptr(saved.packed) if saved else None, _ptr(saved.exponents) if saved else None,
             s)
        return (y, mean, rstd, saved) if checkpoint else (y, mean, rstd)

    return _launch(run, device, stream, (x, gamma, beta))


def layer_norm_backward(dy, x, mean, rstd, gamma=None, params: bool = True, stream=None):
    """(dx, dgamma, dbeta) of `layer_norm`, from the input `x` or its
    `Checkpoint`: dx of dy's type, dgamma and dbeta float32 [width] (None
    without `params`)."""
    code = _matrix("dy", dy)
    rows, width = dy.shape
    device = dy.device
    packed = exponents = None
    if isinstance(x, Checkpoint):
        _check_checkpoint(x)
        _like("checkpoint", x.packed, dy.shape, torch.float8_e4m3fn, device)
        packed, exponents, x = x.packed, x.exponents, None
    else:
        _like("x", x, dy.shape, dy.dtype, device)
    _like("mean", mean, (rows,), torch.float32, device)
    _like("rstd", rstd, (rows,), torch.float32, device)
    if gamma is not None:
        _like("gamma", gamma, (width,), torch.float32, device)

    def run(s):
        dx = torch.empty_like(dy)
        dgamma = dbeta = workspace = None
        size = 0
        if params:
            dgamma = torch.empty(width, dtype=torch.float32, device=device)
            dbeta = torch.empty_like(dgamma)
            size = _workspace_size("vfr_layer_norm_workspace", rows, width, device.index)
            workspace = _workspace(size, device)
        call(load_library().vfr_layer_norm_backward, _ptr(dy), _ptr(x), _ptr(packed), _ptr(exponents), _ptr(mean),
             _ptr(rstd), _ptr(gamma), rows, width, code, _ptr(dx), _ptr(dgamma), _ptr(dbeta), _ptr(workspace), size,
             s)
        return dx, dgamma, dbeta

    return _launch(run, device, stream, (dy, x, packed, exponents, mean, rstd, gamma))


def _check_units(x, units, labels, bias) -> int:
    code = _matrix("x", x)
    _matrix("units", units)
    if units.dtype != x.dtype or units.device != x.device or units.shape[1] != x.shape[1]:
        raise ValueError("units: expected the type, device and width of x")
    _like("labels", labels, (x.shape[0],), torch.int32, x.device)
    if bias is not None:
        _like("bias", bias, (units.shape[0],), torch.float32, x.device)
    return code


def unit_loss(x, units, labels, scale: float = 1.0, bias=None, stream=None):
    """(loss, lse), float32 [rows], of frames `x` [rows, width] over the
    codebook `units` [k, width] (`vfr_unit_loss`; float32 or bfloat16), with
    logits scale x units^T + bias.  labels: int32 [rows]; one outside [0, k)
    is none (loss 0).  bias: float32 [k]; -inf leaves a unit out."""
    code = _check_units(x, units, labels, bias)
    rows, width = x.shape
    k, device = units.shape[0], x.device

    def run(s):
        loss = torch.empty(rows, dtype=torch.float32, device=device)
        lse = torch.empty_like(loss)
        size = _workspace_size("vfr_unit_loss_workspace", rows, k, width, code, 0, device.index)
        workspace = _workspace(size, device)
        call(load_library().vfr_unit_loss, _ptr(x), _ptr(units), _ptr(bias), _ptr(labels), rows, k, width, code,
             scale, _ptr(loss), _ptr(lse), _ptr(workspace), size, s)
        return loss, lse

    return _launch(run, device, stream, (x, units, labels, bias))


def unit_loss_backward(x, units, labels, lse, dloss, scale: float = 1.0, bias=None, stream=None):
    """(dx, dunits, dbias) of `unit_loss` from its lse and the gradient
    `dloss` (float32 [rows]) of each row's loss; dbias is None without bias."""
    code = _check_units(x, units, labels, bias)
    rows, width = x.shape
    k, device = units.shape[0], x.device
    _like("lse", lse, (rows,), torch.float32, device)
    _like("dloss", dloss, (rows,), torch.float32, device)

    def run(s):
        dx = torch.empty_like(x)
        dunits = torch.empty_like(units)
        dbias = None if bias is None else torch.empty_like(bias)
        size = _workspace_size("vfr_unit_loss_workspace", rows, k, width, code, 1, device.index)
        workspace = _workspace(size, device)
        call(load_library().vfr_unit_loss_backward, _ptr(x), _ptr(units), _ptr(bias), _ptr(labels), _ptr(lse),
             _ptr(dloss), rows, k, width, code, scale, _ptr(dx), _ptr(dunits), _ptr(dbias), _ptr(workspace), size, s)
        return dx, dunits, dbias

    return _launch(run, device, stream, (x, units, labels, lse, dloss, bias))
