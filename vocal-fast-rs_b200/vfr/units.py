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

import contextlib
import ctypes
import dataclasses

from .lib import call, load_library, stream_struct

BLOCK = 128  # elements of a row that share one exponent
F32, BF16, F16 = 0, 1, 2


@dataclasses.dataclass
class Checkpoint:
    """An activation in 8 bits: e4m3 `packed` [rows, width] (torch
    float8_e4m3fn), times 2^(byte - 127) per 128 elements of a row,
    `exponents` [rows, ceil(width / 128)] (uint8); `dtype` is the type it was
    packed from."""
    packed: "torch.Tensor"  # noqa: F821
    exponents: "torch.Tensor"  # noqa: F821
    dtype: "torch.dtype"  # noqa: F821


def _code(dtype) -> int:
    import torch

    codes = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
    if dtype not in codes:
        raise ValueError(f"expected float32, bfloat16 or float16, not {dtype}")
    return codes[dtype]


def _matrix(name, t):
    import torch

    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == 2 and t.is_contiguous()):
        raise ValueError(f"{name}: expected a contiguous CUDA tensor [rows, width]")
    _code(t.dtype)
    return t


def _like(name, t, shape, dtype, device):
    import torch

    if not (isinstance(t, torch.Tensor) and t.device == device and t.dtype == dtype and tuple(t.shape) == tuple(shape)
            and t.is_contiguous()):
        raise ValueError(f"{name}: expected a contiguous {dtype} tensor {list(shape)} on {device}")
    return t


def _ptr(t):
    return None if t is None or t.numel() == 0 else t.data_ptr()


@contextlib.contextmanager
def _launch(device, stream, inputs):
    """The device and stream of a call: allocations inside belong to the
    stream, and inputs of another stream are kept until its work is done."""
    import torch

    with torch.cuda.device(device):
        current = torch.cuda.current_stream(device)
        s = current if stream is None else stream
        if s.device != device:
            raise ValueError(f"the stream is on {s.device}, the tensors on {device}")
        if s == current:
            yield stream_struct(s)
            return
        with torch.cuda.stream(s):
            yield stream_struct(s)
        for t in inputs:
            if t is not None:
                t.record_stream(s)


def _workspace(size, device):
    import torch

    return torch.empty(max(size, 1), dtype=torch.uint8, device=device)


def _blocks(width):
    return (width + BLOCK - 1) // BLOCK


def _empty_checkpoint(x):
    import torch

    rows, width = x.shape
    return Checkpoint(torch.empty((rows, width), dtype=torch.float8_e4m3fn, device=x.device),
                      torch.empty((rows, _blocks(width)), dtype=torch.uint8, device=x.device), x.dtype)


def _check_checkpoint(c):
    import torch

    p = c.packed
    if not (isinstance(p, torch.Tensor) and p.is_cuda and p.dim() == 2 and p.is_contiguous()
            and p.dtype == torch.float8_e4m3fn):
        raise ValueError("checkpoint: expected a contiguous CUDA float8_e4m3fn tensor [rows, width]")
    _like("checkpoint exponents", c.exponents, (p.shape[0], _blocks(p.shape[1])), torch.uint8, p.device)
    return c


def checkpoint_pack(x, stream=None) -> Checkpoint:
    """`x` in 8 bits (`vfr_checkpoint_pack`)."""
    _matrix("x", x)
    with _launch(x.device, stream, (x,)) as s:
        out = _empty_checkpoint(x)
        call(load_library().vfr_checkpoint_pack, _ptr(x), x.shape[0], x.shape[1], _code(x.dtype), _ptr(out.packed),
             _ptr(out.exponents), ctypes.byref(s))
    return out


def checkpoint_unpack(checkpoint: Checkpoint, dtype=None, stream=None):
    """The checkpoint's values, in `dtype` (default: the type it was packed
    from; exact in float32)."""
    import torch

    c = _check_checkpoint(checkpoint)
    dtype = c.dtype if dtype is None else dtype
    code = _code(dtype)
    rows, width = c.packed.shape
    with _launch(c.packed.device, stream, (c.packed, c.exponents)) as s:
        x = torch.empty((rows, width), dtype=dtype, device=c.packed.device)
        call(load_library().vfr_checkpoint_unpack, _ptr(c.packed), _ptr(c.exponents), rows, width, code, _ptr(x),
             ctypes.byref(s))
    return x


def layer_norm(x, gamma=None, beta=None, eps: float = 1e-5, checkpoint: bool = False, stream=None):
    """(y, mean, rstd) of the rows of `x` (`vfr_layer_norm`): y of x's type,
    mean and rstd float32 [rows]; gamma and beta float32 [width].  With
    `checkpoint`, also x's `Checkpoint`, written in the same pass."""
    import torch

    _matrix("x", x)
    rows, width = x.shape
    for name, t in (("gamma", gamma), ("beta", beta)):
        if t is not None:
            _like(name, t, (width,), torch.float32, x.device)
    with _launch(x.device, stream, (x, gamma, beta)) as s:
        y = torch.empty_like(x)
        mean = torch.empty(rows, dtype=torch.float32, device=x.device)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        saved = _empty_checkpoint(x) if checkpoint else None
        call(load_library().vfr_layer_norm, _ptr(x), _ptr(gamma), _ptr(beta), rows, width, _code(x.dtype), float(eps),
             _ptr(y), _ptr(mean), _ptr(rstd), _ptr(saved.packed) if saved else None,
             _ptr(saved.exponents) if saved else None, ctypes.byref(s))
    return (y, mean, rstd, saved) if checkpoint else (y, mean, rstd)


def layer_norm_backward(dy, x, mean, rstd, gamma=None, params: bool = True, stream=None):
    """(dx, dgamma, dbeta) of `layer_norm`, from the input `x` or its
    `Checkpoint`: dx of dy's type, dgamma and dbeta float32 [width] (None
    without `params`)."""
    import torch

    _matrix("dy", dy)
    rows, width = dy.shape
    packed = exponents = None
    if isinstance(x, Checkpoint):
        _check_checkpoint(x)
        packed = _like("checkpoint", x.packed, dy.shape, torch.float8_e4m3fn, dy.device)
        exponents, x = x.exponents, None
    else:
        _like("x", x, dy.shape, dy.dtype, dy.device)
    for name, t in (("mean", mean), ("rstd", rstd)):
        _like(name, t, (rows,), torch.float32, dy.device)
    if gamma is not None:
        _like("gamma", gamma, (width,), torch.float32, dy.device)
    L = load_library()
    with _launch(dy.device, stream, (dy, x, packed, exponents, mean, rstd, gamma)) as s:
        dx = torch.empty_like(dy)
        dgamma = dbeta = workspace = None
        size = ctypes.c_size_t(0)
        if params:
            dgamma = torch.empty(width, dtype=torch.float32, device=dy.device)
            dbeta = torch.empty(width, dtype=torch.float32, device=dy.device)
            call(L.vfr_layer_norm_workspace, rows, width, ctypes.byref(size))
            workspace = _workspace(size.value, dy.device)
        call(L.vfr_layer_norm_backward, _ptr(dy), _ptr(x), _ptr(packed), _ptr(exponents), _ptr(mean), _ptr(rstd),
             _ptr(gamma), rows, width, _code(dy.dtype), _ptr(dx), _ptr(dgamma), _ptr(dbeta), _ptr(workspace),
             size.value, ctypes.byref(s))
    return dx, dgamma, dbeta


def _check_units(x, units, labels, bias):
    import torch

    _matrix("x", x)
    _matrix("units", units)
    if units.dtype != x.dtype or units.device != x.device or units.shape[1] != x.shape[1]:
        raise ValueError("units: expected the type, device and width of x")
    _like("labels", labels, (x.shape[0],), torch.int32, x.device)
    if bias is not None:
        _like("bias", bias, (units.shape[0],), torch.float32, x.device)


def _unit_workspace(x, units, backward):
    size = ctypes.c_size_t(0)
    call(load_library().vfr_unit_loss_workspace, x.shape[0], units.shape[0], x.shape[1], _code(x.dtype),
         int(backward), ctypes.byref(size))
    return _workspace(size.value, x.device), size.value


def unit_loss(x, units, labels, scale: float = 1.0, bias=None, stream=None):
    """(loss, lse), float32 [rows], of frames `x` [rows, width] over the
    codebook `units` [k, width] (`vfr_unit_loss`; float32 or bfloat16), with
    logits scale x units^T + bias.  labels: int32 [rows]; one outside [0, k)
    is none (loss 0).  bias: float32 [k]; -inf leaves a unit out."""
    import torch

    _check_units(x, units, labels, bias)
    rows, width = x.shape
    with _launch(x.device, stream, (x, units, labels, bias)) as s:
        loss = torch.empty(rows, dtype=torch.float32, device=x.device)
        lse = torch.empty(rows, dtype=torch.float32, device=x.device)
        workspace, size = _unit_workspace(x, units, False)
        call(load_library().vfr_unit_loss, _ptr(x), _ptr(units), _ptr(bias), _ptr(labels), rows, units.shape[0],
             width, _code(x.dtype), float(scale), _ptr(loss), _ptr(lse), _ptr(workspace), size, ctypes.byref(s))
    return loss, lse


def unit_loss_backward(x, units, labels, lse, dloss, scale: float = 1.0, bias=None, stream=None):
    """(dx, dunits, dbias) of `unit_loss` from its lse and the gradient
    `dloss` (float32 [rows]) of each row's loss; dbias is None without bias."""
    import torch

    _check_units(x, units, labels, bias)
    rows, width = x.shape
    for name, t in (("lse", lse), ("dloss", dloss)):
        _like(name, t, (rows,), torch.float32, x.device)
    with _launch(x.device, stream, (x, units, labels, lse, dloss, bias)) as s:
        dx = torch.empty_like(x)
        dunits = torch.empty_like(units)
        dbias = None if bias is None else torch.empty_like(bias)
        workspace, size = _unit_workspace(x, units, True)
        call(load_library().vfr_unit_loss_backward, _ptr(x), _ptr(units), _ptr(bias), _ptr(labels), _ptr(lse),
             _ptr(dloss), rows, units.shape[0], width, _code(x.dtype), float(scale), _ptr(dx), _ptr(dunits),
             _ptr(dbias), _ptr(workspace), size, ctypes.byref(s))
    return dx, dunits, dbias
