"""Unit-head operators (`vfr.units`): layer norm and its gradients, 8-bit
activation checkpoints, softmax cross entropy over a codebook of units and
its gradients.  No counterpart in the reference: each result is compared with
a plain f64 statement of its formula.

Tolerances are worst-case error bounds of the arithmetic, elementwise, in
u = 2^-24 (half an f32 step) and h(t), half a step of the output type:
* a row's sums add 32 values a lane, then at most 7 levels of lanes and
  warps: 40 u of the sum of magnitudes, taken as 64 with the few products;
* a sum over rows, in any order: (rows + 16) u of the sum of magnitudes;
* a dot product of depth d, f32 accumulation in any order that may truncate
  instead of rounding: (6 d + 16) 2u of the sum of magnitudes (f32 operands
  are three bf16 terms, six products; what is dropped is below 2^-25);
* a softmax gradient G = dloss (p - y): p (dz + 8 u) + |G| (h + 2 u), dz
  the logit's error, h a bf16 half step where the products take it in bf16.
"""
import ctypes
import math

import pytest

U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def _dtype(name):
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _within(got, want, tol):
    """Elementwise |got - want| <= tol; NaN where and only where wanted.  A
    value within its tolerance of the type's overflow (half a step past its
    largest: 65,520 in f16) may be an infinity."""
    import torch

    edge = torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 4)
    got = got.double()
    over = torch.isinf(got) & (want.abs() + tol >= edge) & (torch.sign(got) == torch.sign(want))
    want = torch.where(over, got, want)
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    ok = torch.isfinite(want)
    over = (got - want).abs()[ok] - tol.expand_as(want)[ok]
    assert over.numel() == 0 or over.max().item() <= 0.0, f"off by {over.max().item()} over the bound"


# ------------------------------------------------------------- f64 statements


def ref_norm(x, gamma, beta, eps):
    v = x.double()
    mean = v.mean(1, keepdim=True)
    rstd = (((v - mean) ** 2).mean(1, keepdim=True) + eps) ** -0.5
    n = (v - mean) * rstd
    g = 1.0 if gamma is None else gamma.double()
    b = 0.0 if beta is None else beta.double()
    return n * g + b, mean[:, 0], rstd[:, 0], n


def ref_norm_grad(dy, values, mean, rstd, gamma):
    d, m, r = dy.double(), mean.double()[:, None], rstd.double()[:, None]
    n = (values.double() - m) * r
    g = d if gamma is None else d * gamma.double()
    dx = r * (g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True))
    return dx, (d * n).sum(0), d.sum(0), n, g


def ref_pack(x):
    """(values, exponent bytes) of the checkpoint of x, element by element."""
    import numpy as np
    import torch

    v = x.double().cpu().numpy()
    rows, width = v.shape
    out = np.empty_like(v)
    exponents = np.empty((rows, (width + 127) // 128), np.uint8)
    codes = np.array([math.ldexp(8 + m, e - 3) for e in range(-6, 9) for m in range(8)][:-1]
                     + [math.ldexp(m, -9) for m in range(8)])  # every e4m3 magnitude but NaN
    codes = np.unique(codes)
    assert codes[-1] == 448.0
    fraction = np.array([int(round(math.ldexp(math.frexp(c)[0], 4))) if c >= 2.0 ** -6 else int(c * 2 ** 9)
                         for c in codes])
    for r in range(rows):
        for b in range(exponents.shape[1]):
            block = v[r, 128 * b:128 * b + 128]
            top = np.abs(block[np.isfinite(block)]).max(initial=0.0)
            s = -127
            while top > 448.0 * 2.0 ** s:
                s += 1
            exponents[r, b] = s + 127
            scaled = np.abs(block) * 2.0 ** -s
            i = np.clip(np.searchsorted(codes, scaled), 1, len(codes) - 1)
            low, high = codes[i - 1], codes[i]
            with np.errstate(invalid="ignore"):
                take_high = (scaled - low > high - scaled) | ((scaled - low == high - scaled)
                                                              & (fraction[i] % 2 == 0))
            q = np.where(take_high, high, low)
            out[r, 128 * b:128 * b + 128] = np.where(np.isfinite(block), np.sign(block) * q * 2.0 ** s, np.nan)
    return torch.from_numpy(out), torch.from_numpy(exponents)


def ref_logits(x, units, scale, bias):
    import torch

    z = x.double() @ units.double().t() * scale
    if bias is not None:
        z = z + bias.double()
        z = torch.where(torch.isneginf(bias.double())[None, :].expand_as(z), torch.full_like(z, -math.inf), z)
    return z


def ref_loss(x, units, labels, scale, bias):
    import torch

    z = ref_logits(x, units, scale, bias)
    lse = torch.logsumexp(z, 1)
    loss = torch.zeros_like(lse)
    hit = torch.nonzero((labels >= 0) & (labels < units.shape[0]))[:, 0]
    zt = z[hit, labels[hit].long()]
    loss[hit] = torch.where(torch.isneginf(zt), torch.full_like(zt, math.inf), lse[hit] - zt)
    return loss, lse


def ref_loss_grad(x, units, labels, lse, dloss, scale, bias):
    """dx, dunits, dbias, and what their bounds need: p times |dloss|, G, and
    the frames and units as the products see them."""
    import torch

    valid = (labels >= 0) & (labels < units.shape[0])
    xs = torch.where(valid[:, None], x.double(), torch.zeros_like(x.double()))
    ws = units.double()
    if bias is not None:
        ws = torch.where(torch.isneginf(bias)[:, None], torch.zeros_like(ws), ws)
    z = ref_logits(xs, ws, scale, bias)
    p = torch.where(torch.isneginf(z), torch.zeros_like(z), torch.exp(z - lse.double()[:, None]))
    y = torch.zeros_like(p)
    hit = torch.nonzero(valid)[:, 0]
    y[hit, labels[hit].long()] = 1.0
    if bias is not None:
        y[:, torch.isneginf(bias)] = 0.0
    w = torch.where(valid, dloss.double(), torch.zeros_like(dloss.double()))[:, None]
    w = torch.where(valid[:, None], w, torch.zeros_like(w))
    p = torch.where(valid[:, None], p, torch.zeros_like(p))
    G = w * (p - y)
    return G @ ws * scale, G.t() @ xs * scale, G.sum(0), w.abs() * p, G, xs, ws


def check_loss(x, units, labels, scale, bias, loss, lse):
    import torch

    want_loss, want_lse = ref_loss(x, units, labels, scale, bias)
    ok = (labels >= 0) & (labels < units.shape[0])
    depth = (6 * x.shape[1] + 16) * 2 * U
    b = torch.zeros(units.shape[0], device=x.device, dtype=torch.float64)
    ws = units.double().abs()
    if bias is not None:
        off = torch.isneginf(bias)
        b = torch.where(off, b, bias.double().abs())
        ws = torch.where(off[:, None], torch.zeros_like(ws), ws)
    size = x.double().abs() @ ws.t() * abs(scale) + b
    dz = (depth + 4 * U) * size.amax(1)
    # the sum of k exponentials in any order, its logarithm, and the exponent's rounding
    tol = dz + (units.shape[0] + 16) * U + 4 * U * (want_lse.abs().nan_to_num(posinf=0.0, neginf=0.0) + size.amax(1))
    live = torch.isfinite(x.double()).all(1)
    _within(lse[live], want_lse[live], tol[live])
    live |= ~ok
    _within(loss[live], want_loss[live].nan_to_num(nan=0.0, posinf=math.inf), 2 * tol[live].nan_to_num())


def check_loss_grad(name, x, units, labels, lse, dloss, scale, bias, dx, dunits, dbias):
    import torch

    rdx, rdw, rdb, p, g, xa, wa = ref_loss_grad(x, units, labels, lse, dloss, scale, bias)
    g, xa, wa = g.abs(), xa.abs(), wa.abs()
    b = 0.0 if bias is None else torch.where(torch.isneginf(bias), torch.zeros_like(bias), bias).double().abs()
    size = (xa @ wa.t()) * abs(scale) + b
    rows, k, width = x.shape[0], units.shape[0], x.shape[1]
    finite_lse = lse.double().abs().nan_to_num(posinf=0.0, neginf=0.0)[:, None]
    dz = (6 * width + 32) * 2 * U * size + 4 * U * finite_lse
    half = HALF["bf16"] if name == "bf16" else 2 * U
    under = 2.0 ** -126 * (1 + dloss.double().abs().nan_to_num())[:, None]
    eg = p * (dz + 8 * U) + g * (half + 2 * U) + under
    tiny = 1e-36
    _within(dx, rdx, abs(scale) * ((eg + (6 * k + 16) * 2 * U * g) @ wa) + HALF[name] * rdx.abs() + tiny)
    _within(dunits, rdw, abs(scale) * ((eg + (6 * rows + 16) * 2 * U * g).t() @ xa) + HALF[name] * rdw.abs() + tiny)
    if bias is not None:
        eb = p * (dz + 8 * U) + 2 * U * g + under
        _within(dbias, rdb, (eb + (rows + 16) * U * g).sum(0) + tiny)


# ------------------------------------------------------------- CPU


def _call(name, *args):
    from vfr import lib

    L = lib.load_library()
    lib.call(getattr(L, name), *args)


P16 = ctypes.c_void_p(256)  # never dereferenced: each call below is refused first


def _stream():
    from vfr import lib

    return ctypes.byref(lib.Stream(None))


@pytest.mark.parametrize("change,message", [
    (dict(width=0), "row width must be in 1..4096"),
    (dict(width=4097), "row width must be in 1..4096"),
    (dict(rows=-1), "row count must be in"),
    (dict(rows=2 ** 31), "row count must be in"),
    (dict(dtype=3), "unknown element type"),
    (dict(eps=-1.0), "eps must be finite and not negative"),
    (dict(eps=float("nan")), "eps must be finite and not negative"),
    (dict(x=None), "null layer norm binding"),
    (dict(mean=None), "null layer norm binding"),
    (dict(packed=P16), "both its packed and its exponent buffer"),
    (dict(x=ctypes.c_void_p(258)), "misaligned layer norm binding"),
    (dict(gamma=ctypes.c_void_p(258)), "misaligned layer norm binding"),
    (dict(stream=None), "null CUDA stream binding"),
])
def test_layer_norm_refusals(native, change, message):
    from vfr import lib

    a = dict(x=P16, gamma=None, beta=None, rows=4, width=8, dtype=0, eps=1e-5, y=P16, mean=P16, rstd=P16, packed=None,
             exponents=None, stream=_stream())
    a.update(change)
    with pytest.raises(lib.NativeError, match=message):
        _call("vfr_layer_norm", *a.values())


@pytest.mark.parametrize("change,message", [
    (dict(dy=None), "null layer norm binding"),
    (dict(x=None), "null layer norm binding"),
    (dict(packed=P16, exponents=P16), "not both"),
    (dict(exponents=P16), "both its packed and its exponent buffer"),
    (dict(dtype=-1), "unknown element type"),
    (dict(workspace=ctypes.c_void_p(8)), "misaligned layer norm binding"),
])
def test_layer_norm_backward_refusals(native, change, message):
    from vfr import lib

    a = dict(dy=P16, x=P16, packed=None, exponents=None, mean=P16, rstd=P16, gamma=None, rows=4, width=8, dtype=0,
             dx=P16, dgamma=P16, dbeta=P16, workspace=P16, bytes=1 << 20, stream=_stream())
    a.update(change)
    with pytest.raises(lib.NativeError, match=message):
        _call("vfr_layer_norm_backward", *a.values())


@pytest.mark.parametrize("change,message", [
    (dict(dtype=2), "takes f32 or bf16"),
    (dict(k=0), "unit count must be positive"),
    # tiles past the last row or unit must keep 32-bit coordinates
    (dict(k=2 ** 30 + 1), "frames and units must number 2\\^30 at most"),
    (dict(k=2 ** 31 - 1), "frames and units must number 2\\^30 at most"),
    (dict(rows=2 ** 30 + 1), "frames and units must number 2\\^30 at most"),
    (dict(width=4097), "row width must be in 1..4096"),
    (dict(scale=float("inf")), "logit scale must be finite"),
    (dict(scale=float("nan")), "logit scale must be finite"),
    (dict(scale=-2e30), "logit scale must be finite"),
    (dict(units=None), "null unit loss binding"),
    (dict(labels=None), "null unit loss binding"),
    (dict(labels=ctypes.c_void_p(2)), "misaligned unit loss binding"),
    (dict(workspace=ctypes.c_void_p(16)), "misaligned unit loss binding"),
    (dict(stream=None), "null CUDA stream binding"),
])
def test_unit_loss_refusals(native, change, message):
    from vfr import lib

    a = dict(x=P16, units=P16, bias=None, labels=P16, rows=4, k=8, width=8, dtype=0, scale=1.0, loss=P16, lse=P16,
             workspace=None, bytes=0, stream=_stream())
    a.update(change)
    with pytest.raises(lib.NativeError, match=message):
        _call("vfr_unit_loss", *a.values())
    b = dict(x=P16, units=P16, bias=None, labels=P16, lse=P16, dloss=P16, rows=4, k=8, width=8, dtype=0, scale=1.0,
             dx=P16, dunits=P16, dbias=None, workspace=None, bytes=0, stream=_stream())
    b.update(change)
    with pytest.raises(lib.NativeError, match=message):
        _call("vfr_unit_loss_backward", *b.values())


def test_checkpoint_refusals(native):
    from vfr import lib

    for args, message in [((None, 4, 8, 0, P16, P16), "null checkpoint binding"),
                          ((P16, 4, 8, 7, P16, P16), "unknown element type"),
                          ((ctypes.c_void_p(257), 4, 8, 1, P16, P16), "misaligned checkpoint binding")]:
        with pytest.raises(lib.NativeError, match=message):
            _call("vfr_checkpoint_pack", *args, _stream())
    with pytest.raises(lib.NativeError, match="null checkpoint binding"):
        _call("vfr_checkpoint_unpack", P16, None, 4, 8, 0, P16, _stream())


def test_python_refuses_host_tensors_and_shapes():
    import torch

    from vfr import units as u

    x = torch.zeros(4, 8)
    for f in (lambda: u.layer_norm(x), lambda: u.checkpoint_pack(x), lambda: u.layer_norm_backward(x, x, x, x),
              lambda: u.unit_loss(x, x, torch.zeros(4, dtype=torch.int32)),
              lambda: u.checkpoint_unpack(u.Checkpoint(x, x, torch.float32))):
        with pytest.raises(ValueError, match="CUDA"):
            f()


def test_reference_statements_agree_with_differences():
    """The f64 gradients above against central differences."""
    import torch

    torch.manual_seed(0)
    x, w = torch.randn(5, 6).double(), torch.randn(7, 6).double()
    bias = torch.randn(7).double()
    bias[2] = -math.inf
    labels = torch.tensor([0, 6, -1, 3, 9], dtype=torch.int32)
    dloss = torch.randn(5).double()
    _, lse = ref_loss(x, w, labels, 0.7, bias)
    dx, dw, db = ref_loss_grad(x, w, labels, lse, dloss, 0.7, bias)[:3]
    f = lambda x, w, b: (ref_loss(x, w, labels, 0.7, b)[0] * dloss).sum()  # noqa: E731
    h = 1e-6
    for t, grad, at in ((x, dx, 0), (w, dw, 1), (bias, db, 2)):
        for i in range(t.numel()):
            if not math.isfinite(t.view(-1)[i]):
                assert grad.reshape(-1)[i] == 0
                continue
            args = [x, w, bias]
            up, down = t.clone(), t.clone()
            up.view(-1)[i] += h
            down.view(-1)[i] -= h
            args[at] = up
            a = f(*args)
            args[at] = down
            assert abs((a - f(*args)) / (2 * h) - grad.reshape(-1)[i]) < 1e-7
    gamma = torch.randn(6).double()
    dy = torch.randn(5, 6).double()
    _, mean, rstd, _ = ref_norm(x, gamma, None, 1e-5)
    dx, dg, db = ref_norm_grad(dy, x, mean, rstd, gamma)[:3]
    f = lambda x, g: (ref_norm(x, g, None, 1e-5)[0] * dy).sum()  # noqa: E731
    for t, grad, at in ((x, dx, 0), (gamma, dg, 1)):
        for i in range(t.numel()):
            args = [x, gamma]
            up, down = t.clone(), t.clone()
            up.view(-1)[i] += h
            down.view(-1)[i] -= h
            args[at] = up
            a = f(*args)
            args[at] = down
            assert abs((a - f(*args)) / (2 * h) - grad.reshape(-1)[i]) < 1e-6


def test_reference_checkpoint_against_torch_rounding():
    import torch

    torch.manual_seed(1)
    x = torch.randn(3, 300) * torch.exp(2 * torch.randn(3, 300))
    values, e = ref_pack(x)
    scale = torch.exp2(e.double() - 127).repeat_interleave(128, 1)[:, :300]
    assert torch.equal(values, (x / scale).to(torch.float8_e4m3fn).double() * scale)
    assert torch.equal(ref_pack(torch.zeros(1, 5))[1], torch.zeros(1, 1, dtype=torch.uint8))


# ------------------------------------------------------------- GPU


def _frames(torch, rows, width, dtype, seed, align=True):
    """Frames with channel offsets and loud channels; with align False, one
    element off a 16-byte boundary."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g) + 2.0 * torch.randn(1, width, generator=g)
    x[:, ::17] *= 30.0
    x = x.to(_dtype(dtype))
    if align:
        return x.cuda()
    buf = torch.empty(rows * width + 1, dtype=x.dtype, device="cuda")
    buf[1:] = x.flatten().cuda()
    return buf[1:].view(rows, width)


SHAPES = [(1, 1), (1, 768), (2, 2), (3, 7), (34, 768), (65, 127), (140, 256), (33, 129), (17, 1023), (9, 1024),
          (9, 1025), (5, 1032), (7, 2048), (3, 4095), (4, 4096), (2999, 513), (5000, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("affine,align", [(True, True), (False, False)])
def test_layer_norm(cuda, rows, width, dtype, affine, align):
    from vfr import units as u

    torch = cuda
    x = _frames(torch, rows, width, dtype, rows + width, align)
    gamma = torch.randn(width, device="cuda") if affine else None
    beta = torch.randn(width, device="cuda") if affine else None
    y, mean, rstd, saved = u.layer_norm(x, gamma, beta, 1e-5, checkpoint=True)
    plain = u.layer_norm(x, gamma, beta, 1e-5)
    assert all(torch.equal(a, b) for a, b in zip(plain, (y, mean, rstd)))
    wy, wm, wr, n = ref_norm(x, gamma, beta, 1e-5)
    v = x.double()
    size = v.abs().mean(1)
    _within(mean, wm, 64 * U * size)
    # d(rstd)/rstd = half the variance's relative error; the mean's error adds its square
    rel = 64 * U + (64 * U * size * wr) ** 2
    _within(rstd, wr, rel * wr)
    g = 1.0 if gamma is None else gamma.double().abs()
    b = 0.0 if beta is None else beta.double().abs()
    tol = g * (wr[:, None] * 64 * U * size[:, None] + n.abs() * (rel[:, None] + 8 * U)) + 4 * U * (wy.abs() + b)
    _within(y, wy, tol + HALF[dtype] * (wy.abs() + tol) + 2.0 ** -25)
    if rows * width <= 20000:
        values, e = ref_pack(x)
        assert torch.equal(saved.exponents.cpu(), e)
        assert torch.equal(u.checkpoint_unpack(saved, torch.float32).cpu().double(), values)
    packed = u.checkpoint_pack(x)
    assert torch.equal(packed.packed.view(torch.uint8), saved.packed.view(torch.uint8))
    assert torch.equal(packed.exponents, saved.exponents)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("affine,align", [(True, True), (False, False)])
def test_layer_norm_backward(cuda, rows, width, dtype, affine, align):
    from vfr import units as u

    torch = cuda
    x = _frames(torch, rows, width, dtype, rows * width, align)
    dy = torch.randn(rows, width, device="cuda").to(_dtype(dtype))
    gamma = torch.randn(width, device="cuda") if affine else None
    _, mean, rstd = u.layer_norm(x, gamma)
    saved = u.checkpoint_pack(x)
    for source, values in ((x, x), (saved, u.checkpoint_unpack(saved, torch.float32))):
        dx, dgamma, dbeta = u.layer_norm_backward(dy, source, mean, rstd, gamma)
        wx, wg, wb, n, g = ref_norm_grad(dy, values, mean, rstd, gamma)
        r = rstd.double()[:, None]
        tol = 64 * U * r * (g.abs() + g.abs().mean(1, keepdim=True) + n.abs() * (g * n).abs().mean(1, keepdim=True))
        # n's own error: the subtraction of the mean and the product, each half a step
        en = 4 * U * n.abs()
        tol = tol + r * (en * (g * n).abs().mean(1, keepdim=True) + n.abs() * (g.abs() * en).mean(1, keepdim=True))
        _within(dx, wx, tol + HALF[dtype] * (wx.abs() + tol) + 2.0 ** -25)
        d = dy.double().abs()
        _within(dgamma, wg, (rows + 16) * U * (d * n.abs()).sum(0) + (d * en).sum(0))
        _within(dbeta, wb, (rows + 16) * U * d.sum(0))
        only = u.layer_norm_backward(dy, source, mean, rstd, gamma, params=False)
        assert torch.equal(only[0], dx) and only[1] is None and only[2] is None
        again = u.layer_norm_backward(dy, source, mean, rstd, gamma)
        assert torch.equal(again[1], dgamma) and torch.equal(again[2], dbeta)


@pytest.mark.gpu
def test_layer_norm_unaligned_parameters(cuda):
    """gamma, beta, dy or the checkpoint off a 16-byte boundary, each alone."""
    from vfr import units as u

    torch = cuda

    def moved(t):
        buf = torch.empty(t.numel() * t.element_size() + 4, dtype=torch.uint8, device="cuda")
        out = buf[4:].view(t.dtype).view(t.shape)
        out.copy_(t)
        return out

    x = _frames(torch, 77, 768, "f32", 5)
    gamma, beta = torch.randn(768, device="cuda"), torch.randn(768, device="cuda")
    dy = torch.randn(77, 768, device="cuda")
    y, mean, rstd, saved = u.layer_norm(x, gamma, beta, checkpoint=True)
    wy, _, _, n = ref_norm(x, gamma, beta, 1e-5)
    size = x.double().abs().mean(1, keepdim=True) * rstd.double()[:, None]
    tol = gamma.double().abs() * (64 * U * size + n.abs() * 80 * U) + 8 * U * (wy.abs() + beta.double().abs())
    for g, b in ((moved(gamma), beta), (gamma, moved(beta))):
        _within(u.layer_norm(x, g, b)[0], wy, tol + 64 * U * (64 * U * size) ** 2 + 2.0 ** -25)
    other = u.Checkpoint(moved(saved.packed.view(torch.uint8)).view(torch.float8_e4m3fn), saved.exponents, saved.dtype)
    assert torch.equal(u.checkpoint_unpack(other, torch.float32), u.checkpoint_unpack(saved, torch.float32))
    for source in (x, saved, other):
        values = x if source is x else u.checkpoint_unpack(saved, torch.float32)
        wx, wg, wb, n, g = ref_norm_grad(dy, values, mean, rstd, gamma)
        r = rstd.double()[:, None]
        tol = 80 * U * r * (g.abs() + g.abs().mean(1, keepdim=True) + 2 * n.abs() * (g * n).abs().mean(1, keepdim=True)
                            + n.abs().mean(1, keepdim=True) * g.abs()) + 2.0 ** -25
        for d, gm in ((dy, gamma), (moved(dy), gamma), (dy, moved(gamma))):
            dx, dgamma, dbeta = u.layer_norm_backward(d, source, mean, rstd, gm)
            _within(dx, wx, tol + 2 * U * wx.abs())
            _within(dgamma, wg, 100 * U * (dy.double().abs() * n.abs()).sum(0))
            _within(dbeta, wb, 100 * U * dy.double().abs().sum(0))


@pytest.mark.gpu
def test_first_call_may_be_captured(cuda):
    """A process whose first calls of the operators are inside a capture."""
    import os
    import subprocess
    import sys

    code = """
import torch
from vfr import units as u
x = torch.randn(300, 256, device="cuda").bfloat16()
w = torch.randn(400, 256, device="cuda").bfloat16()
labels = torch.arange(300, dtype=torch.int32, device="cuda")
dloss = torch.ones(300, device="cuda")
def step():
    y, mean, rstd, saved = u.layer_norm(x, checkpoint=True)
    loss, lse = u.unit_loss(y, w, labels, 0.1)
    dy, dw, _ = u.unit_loss_backward(y, w, labels, lse, dloss, 0.1)
    return loss, dw, u.layer_norm_backward(dy, saved, mean, rstd)[0]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = step()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, step()))
print("same")
"""
    from vfr import lib

    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": lib.PKG})
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("width", [8, 129, 4096])
def test_checkpoint_special_values(cuda, dtype, width):
    """Ties of the rounding, the format's ends, zeros of both signs,
    infinities and NaN, blocks of very large and very small values."""
    from vfr import units as u

    torch = cuda
    t = _dtype(dtype)
    top = torch.finfo(t).max
    patterns = torch.tensor([448.0, 449.0, 17.0, 19.0, -18.0, 1.0625, 1.1875, 0.0, -0.0, 2.0 ** -9, 2.0 ** -10,
                             3 * 2.0 ** -10, -2.0 ** -6, float("inf"), -float("inf"), float("nan")])
    x = patterns.repeat(math.ceil(12 * width / patterns.numel()))[:12 * width].view(12, width).clone()
    scales = torch.tensor([1.0, 2.0, 2.0 ** -3, 1.7, 130.0, 2.0 ** -14, 0.0, top / 512, 2.0 ** -20, 1e-3, 3.0, 100.0])
    x = (x * scales[:, None]).to(t)
    x[11] = float("nan")
    x[10] = top
    dx = x.cuda()
    c = u.checkpoint_pack(dx)
    values, e = ref_pack(x)
    assert torch.equal(c.exponents.cpu(), e)
    got = u.checkpoint_unpack(c, torch.float32).cpu().double()
    # the values rounded to f32: its largest number becomes 256 * 2^120 = 2^128, past f32's range
    values = values.float().double()
    assert torch.equal(torch.isnan(got), torch.isnan(values))
    assert torch.equal(got.nan_to_num(), values.nan_to_num())
    back = u.checkpoint_unpack(c)
    assert back.dtype == t
    assert torch.equal(back.cpu().nan_to_num(), got.to(t).nan_to_num())


@pytest.mark.gpu
def test_empty_and_single(cuda):
    from vfr import units as u

    torch = cuda
    x = torch.empty(0, 96, device="cuda")
    y, mean, rstd, saved = u.layer_norm(x, checkpoint=True)
    assert y.shape == (0, 96) and mean.numel() == 0 and saved.exponents.shape == (0, 1)
    for source in (x, saved):
        dx, dgamma, dbeta = u.layer_norm_backward(x, source, mean, rstd)
        assert dx.shape == (0, 96) and not dgamma.any() and not dbeta.any()
    assert u.checkpoint_unpack(u.checkpoint_pack(x)).shape == (0, 96)
    w = torch.randn(5, 96, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    loss, lse = u.unit_loss(x, w, none)
    assert loss.numel() == 0 and lse.numel() == 0
    dx, dw, db = u.unit_loss_backward(x, w, none, lse, loss, bias=torch.zeros(5, device="cuda"))
    assert dx.shape == (0, 96) and not dw.any() and not db.any()


def _head(torch, rows, k, width, dtype, seed, masked=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(k, width, generator=g)
    labels = torch.randint(0, k, (rows,), generator=g, dtype=torch.int32)
    x = torch.randn(rows, width, generator=g) + 0.3 * w[labels.long()]
    bias = torch.randn(k, generator=g)
    if masked:
        bias[torch.randperm(k, generator=g)[:masked]] = -math.inf
    labels[::5] = -1
    if rows > 3:
        labels[3] = k
    dloss = torch.randn(rows, generator=g)
    t = _dtype(dtype)
    return x.to(t).cuda(), w.to(t).cuda(), labels.cuda(), bias.cuda(), dloss.cuda(), 2.0 / math.sqrt(width)


UNIT_SHAPES = [(1, 1, 1), (1, 511, 768), (2, 3, 5), (34, 511, 768), (127, 255, 64), (128, 256, 64), (129, 257, 65),
               (140, 504, 256), (300, 1000, 72), (257, 129, 1000), (1000, 33, 8), (5, 2000, 4096), (700, 640, 200),
               (64, 64, 128), (1, 5000, 96), (3000, 2, 16),
               # several rounds of tiles, ragged on every side; the gradients'
               # products of (6200, ...) and below run on CTA pairs in bf16 (a
               # tile of 256 x 256 for each of 74 pairs at least)
               (9001, 4611, 256), (6200, 7000, 450), (4500, 4700, 700), (10001, 9001, 770)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k,width", UNIT_SHAPES)
@pytest.mark.parametrize("biased", [True, False])
def test_unit_loss(cuda, rows, k, width, dtype, biased):
    from vfr import units as u

    torch = cuda
    x, w, labels, bias, dloss, scale = _head(torch, rows, k, width, dtype, rows + k, masked=k // 4)
    if not biased:
        bias = None
    loss, lse = u.unit_loss(x, w, labels, scale, bias)
    check_loss(x, w, labels, scale, bias, loss, lse)
    out = u.unit_loss_backward(x, w, labels, lse, dloss, scale, bias)
    check_loss_grad(dtype, x, w, labels, lse, dloss, scale, bias, *out)
    again = u.unit_loss_backward(x, w, labels, lse, dloss, scale, bias)
    for a, b in zip(out, again):
        assert a is None and b is None or torch.equal(a, b)
    l2, s2 = u.unit_loss(x, w, labels, scale, bias)
    assert torch.equal(l2, loss) and torch.equal(s2, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("width", [64, 100])
def test_unit_loss_masked_places_hold_anything(cuda, dtype, width):
    """NaN and infinities in frames without a label and in units left out
    reach no result but those frames' lse."""
    from vfr import units as u

    torch = cuda
    rows, k = 300, 400
    x, w, labels, bias, dloss, scale = _head(torch, rows, k, width, dtype, 5, masked=60)
    none = torch.nonzero((labels < 0) | (labels >= k))[:, 0]
    x[none[::2]] = float("nan")
    x[none[1::2]] = float("inf")
    dloss[none] = float("nan")
    off = torch.nonzero(torch.isneginf(bias))[:, 0]
    w[off[::2]] = float("nan")
    w[off[1::2]] = -float("inf")
    loss, lse = u.unit_loss(x, w, labels, scale, bias)
    check_loss(x, torch.where(torch.isneginf(bias)[:, None], torch.zeros_like(w), w), labels, scale, bias, loss, lse)
    assert not loss[none].any()
    dx, dw, db = u.unit_loss_backward(x, w, labels, lse, dloss, scale, bias)
    check_loss_grad(dtype, x, w, labels, torch.where(torch.isnan(lse), torch.zeros_like(lse), lse),
                    torch.where(torch.isnan(dloss), torch.zeros_like(dloss), dloss), scale, bias, dx, dw, db)
    assert not dx[none].any() and not db[off].any() and not dw[off].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_unit_loss_all_units_left_out_and_lowest_bias(cuda, dtype):
    from vfr import units as u

    torch = cuda
    x, w, labels, bias, dloss, scale = _head(torch, 70, 90, 64, dtype, 8)
    gone = torch.full_like(bias, -math.inf)
    loss, lse = u.unit_loss(x, w, labels, scale, gone)
    valid = (labels >= 0) & (labels < 90)
    assert torch.isneginf(lse).all() and torch.isposinf(loss[valid]).all() and not loss[~valid].any()
    dx, dw, db = u.unit_loss_backward(x, w, labels, lse, dloss, scale, gone)
    # p = 0 everywhere: G is -dloss at the labels; the units' rows take no part
    assert not dx.any()
    check_loss_grad(dtype, x, w, labels, lse, dloss, scale, gone, dx, dw, db)
    # the lowest finite bias leaves a unit out of the softmax without the mask's meaning
    low = bias.clone()
    low[::3] = torch.finfo(torch.float32).min
    labels = torch.where(labels % 3 == 0, labels + 1, labels).int()
    loss, lse = u.unit_loss(x, w, labels, scale, low)
    gone = torch.where(low < -1e38, torch.full_like(low, -math.inf), low)
    want = u.unit_loss(x, w, labels, scale, gone)
    assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])
    # a label on such a unit: the loss is the bias's size (f32 holds no more of it)
    on = torch.full_like(labels, 3)
    loss, lse2 = u.unit_loss(x, w, on, scale, low)
    assert torch.equal(lse2, lse) and torch.equal(loss, torch.full_like(loss, torch.finfo(torch.float32).max))
    # every unit at the lowest: equal logits, as natural f32 logits would be
    low[:] = torch.finfo(torch.float32).min
    loss, lse = u.unit_loss(x, w, labels, scale, low)
    valid = (labels >= 0) & (labels < 90)
    assert torch.equal(lse, torch.full_like(lse, torch.finfo(torch.float32).min)) and not loss[valid].any()
    dx, dw, db = u.unit_loss_backward(x, w, labels, lse, dloss, scale, low)
    assert all(torch.isfinite(t).all() for t in (dx, dw, db))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_unit_loss_extreme_logits(cuda, dtype):
    """Logits of several thousand, equal logits, and one unit far above."""
    from vfr import units as u

    torch = cuda
    x, w, labels, bias, dloss, _ = _head(torch, 200, 300, 64, dtype, 9)
    for scale in (300.0, 0.0, -50.0):
        loss, lse = u.unit_loss(x, w, labels, scale, bias)
        check_loss(x, w, labels, scale, bias, loss, lse)
        out = u.unit_loss_backward(x, w, labels, lse, dloss, scale, bias)
        check_loss_grad(dtype, x, w, labels, lse, dloss, scale, bias, *out)


@pytest.mark.gpu
def test_unit_loss_unaligned_frames(cuda):
    """Bases that fit no 16-byte copy, in both types."""
    from vfr import units as u

    torch = cuda
    for dtype in ("f32", "bf16"):
        x, w, labels, bias, dloss, scale = _head(torch, 150, 270, 64, dtype, 10)
        moved = []
        for t in (x, w):
            buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
            buf[1:] = t.flatten()
            moved.append(buf[1:].view_as(t))
        loss, lse = u.unit_loss(x, w, labels, scale, bias)
        l2, s2 = u.unit_loss(*moved, labels, scale, bias)
        assert torch.equal(loss, l2) and torch.equal(lse, s2)
        a = u.unit_loss_backward(x, w, labels, lse, dloss, scale, bias)
        b = u.unit_loss_backward(*moved, labels, lse, dloss, scale, bias)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
def test_unit_gradient_against_differences(cuda):
    """The sum of the device losses moves along a direction as the device
    gradients say.  Central differences of step t err by t^2 / 6 of a third
    cumulant (of a variable within [-D, D]: below 0.77 D^3, D the largest
    change of a logit), and each loss and gradient by its bound."""
    from vfr import units as u

    torch = cuda
    x, w, labels, bias, _, scale = _head(torch, 40, 60, 32, "f32", 12)
    _, lse = u.unit_loss(x, w, labels, scale, bias)
    one = torch.ones(40, device="cuda")
    dx, dw, db = u.unit_loss_backward(x, w, labels, lse, one, scale, bias)
    g = torch.Generator().manual_seed(3)
    ex, ew, eb = (torch.randn(t.shape, generator=g).cuda() for t in (x, w, bias))
    for dirs, grad in (((ex, 0 * ew, 0 * eb), (dx * ex).double().sum()), ((0 * ex, ew, 0 * eb), (dw * ew).double().sum()),
                       ((0 * ex, 0 * ew, eb), (db * eb).double().sum())):
        t = 2.0 ** -6
        up = u.unit_loss(x + t * dirs[0], w + t * dirs[1], labels, scale, bias + t * dirs[2])[0].double().sum()
        down = u.unit_loss(x - t * dirs[0], w - t * dirs[1], labels, scale, bias - t * dirs[2])[0].double().sum()
        dz = (dirs[0].double() @ w.double().t() + x.double() @ dirs[1].double().t()) * scale + dirs[2].double()
        third = dz.abs().amax(1).pow(3).sum()
        size = ((x.double().abs() @ w.double().abs().t()) * scale + bias.double().abs()).amax(1)
        noise = (2 * ((6 * 32 + 40) * 2 * U * size + 80 * U)).sum() / t
        own = (2 * ((6 * 32 + 40) * 2 * U * size + 400 * U) * dz.abs().amax(1)).sum()
        assert abs((up - down) / (2 * t) - grad) <= third * t * t / 6 + noise + own


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_unit_loss_several_pieces(cuda, dtype):
    """A batch whose gradient takes the units in more than one piece; sampled
    rows and units against f64."""
    from vfr import units as u

    torch = cuda
    rows, k, width = (150_000, 4000, 64) if dtype == "bf16" else (50_000, 4000, 64)
    x, w, labels, bias, dloss, scale = _head(torch, rows, k, width, dtype, 11, masked=100)
    dloss = dloss / rows
    loss, lse = u.unit_loss(x, w, labels, scale, bias)
    dx, dw, db = u.unit_loss_backward(x, w, labels, lse, dloss, scale, bias)
    pick = torch.arange(0, rows, 997, device="cuda")
    check_loss(x[pick], w, labels[pick], scale, bias, loss[pick], lse[pick])
    rdx, _, _, p, g, xa, wa = ref_loss_grad(x[pick], w, labels[pick], lse[pick], dloss[pick], scale, bias)
    g, xa, wa = g.abs(), xa.abs(), wa.abs()
    half = HALF["bf16"] if dtype == "bf16" else 2 * U
    safe = torch.where(torch.isneginf(bias), torch.zeros_like(bias), bias).double().abs()
    dz = (6 * width + 32) * 2 * U * (xa @ wa.t() * scale + safe) + 4 * U * lse[pick].double().abs()[:, None]
    eg = p * (dz + 8 * U) + g * (half + 2 * U)
    _within(dx[pick], rdx, scale * ((eg + (6 * k + 16) * 2 * U * g) @ wa) + HALF[dtype] * rdx.abs() + 1e-36)
    units_pick = torch.tensor([0, 1, 255, 256, 1023, 1024, 2047, 2048, 3500, 3998, 3999], device="cuda")
    wdw = torch.zeros(len(units_pick), width, dtype=torch.float64, device="cuda")
    wdb = torch.zeros(len(units_pick), dtype=torch.float64, device="cuda")
    tdw, tdb = torch.zeros_like(wdw), torch.zeros_like(wdb)
    for lo in range(0, rows, 20000):
        s = slice(lo, lo + 20000)
        _, _, _, p, full, xs, _ = ref_loss_grad(x[s], w, labels[s], lse[s], dloss[s], scale, bias)
        g, xa = full.abs(), xs.abs()
        dz = (6 * width + 32) * 2 * U * (xa @ wa.t() * scale + safe) + 4 * U * lse[s].double().abs()[:, None]
        eg = (p * (dz + 8 * U) + g * (half + 2 * U + (6 * rows + 16) * 2 * U))[:, units_pick]
        eb = (p * (dz + 8 * U) + g * (2 * U + (rows + 16) * U))[:, units_pick]
        wdw += full[:, units_pick].t() @ xs * scale
        wdb += full[:, units_pick].sum(0)
        tdw += eg.t() @ xa * scale
        tdb += eb.sum(0)
    _within(dw[units_pick], wdw, tdw + HALF[dtype] * wdw.abs() + 1e-36)
    _within(db[units_pick], wdb, tdb + 1e-36)


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    """More than 2^31 elements in the frames: the last rows of every operator
    equal the same rows computed alone."""
    from vfr import units as u

    torch = cuda
    rows, width = 2_100_000, 1032
    x = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda").normal_()
    tail = x[-300:].clone()
    gamma = torch.randn(width, device="cuda")
    y, mean, rstd, saved = u.layer_norm(x, gamma, checkpoint=True)
    ty, tm, tr, tsaved = u.layer_norm(tail, gamma, checkpoint=True)
    assert torch.equal(y[-300:], ty) and torch.equal(mean[-300:], tm) and torch.equal(rstd[-300:], tr)
    assert torch.equal(saved.packed[-300:].view(torch.uint8), tsaved.packed.view(torch.uint8))
    assert torch.equal(saved.exponents[-300:], tsaved.exponents)
    dx, _, _ = u.layer_norm_backward(y, saved, mean, rstd, gamma)
    tdx, _, _ = u.layer_norm_backward(ty, tsaved, tm, tr, gamma)
    assert torch.equal(dx[-300:], tdx)
    del dx, saved
    back = u.checkpoint_unpack(u.checkpoint_pack(y))
    assert torch.equal(back[-300:], u.checkpoint_unpack(u.checkpoint_pack(ty)))
    del y, back
    w = torch.randn(20, width, device="cuda").bfloat16()
    labels = torch.randint(0, 20, (rows,), dtype=torch.int32, device="cuda")
    loss, lse = u.unit_loss(x, w, labels, 0.1)
    check_loss(tail, w, labels[-300:], 0.1, None, loss[-300:], lse[-300:])
    dloss = torch.zeros(rows, device="cuda")
    dloss[-300:] = 1.0
    dx, dw, _ = u.unit_loss_backward(x, w, labels, lse, dloss, 0.1)
    check_loss_grad("bf16", tail, w, labels[-300:], lse[-300:], dloss[-300:], 0.1, None, dx[-300:], dw, None)
    assert not dx[:1000].any()


@pytest.mark.gpu
def test_unit_head_together(cuda):
    """The head as it is trained: a codebook from k-means, units from its
    assignment, layer norm with a checkpoint, the loss, the gradients back to
    the frames, a step of the codebook; against f64 of the same step."""
    from vfr import units as u
    from vfr.training import assign, kmeans

    torch = cuda
    g = torch.Generator().manual_seed(21)
    centres = 2.0 * torch.randn(24, 96, generator=g)
    frames = (centres[torch.randint(0, 24, (900,), generator=g)] + 0.5 * torch.randn(900, 96, generator=g)).cuda()
    book, _ = kmeans(frames, 24, 6)
    lists, _ = assign(book, frames)
    assert lists.dtype == torch.int32
    gamma, beta = torch.ones(96, device="cuda"), torch.zeros(96, device="cuda")
    y, mean, rstd, saved = u.layer_norm(frames, gamma, beta, checkpoint=True)
    scale = 0.25
    bias = -0.5 * scale * (book * book).sum(1)
    loss, lse = u.unit_loss(y, book, lists, scale, bias)
    check_loss(y, book, lists, scale, bias, loss, lse)
    dloss = torch.full((900,), 1.0 / 900, device="cuda")
    dy, dbook, dbias = u.unit_loss_backward(y, book, lists, lse, dloss, scale, bias)
    check_loss_grad("f32", y, book, lists, lse, dloss, scale, bias, dy, dbook, dbias)
    dx, dgamma, dbeta = u.layer_norm_backward(dy, saved, mean, rstd, gamma)
    wx, wg, wb, n, gg = ref_norm_grad(dy, u.checkpoint_unpack(saved, torch.float32), mean, rstd, gamma)
    r = rstd.double()[:, None]
    _within(dx, wx, 72 * U * r * (gg.abs() + gg.abs().mean(1, keepdim=True)
                                  + 2 * n.abs() * (gg * n).abs().mean(1, keepdim=True)) + 2 * U * wx.abs())
    _within(dgamma, wg, 940 * U * (dy.double().abs() * n.abs()).sum(0))
    _within(dbeta, wb, 940 * U * dy.double().abs().sum(0))
    # the checkpoint's rounding: half an e4m3 step of each element moves n by at most 2^-4 |x| rstd
    exact = ref_norm_grad(dy, frames, mean, rstd, gamma)[1]
    _within(dgamma, exact, (dy.double().abs() * (frames.double().abs() * r * 2.0 ** -4 + 2.0 ** -10)).sum(0)
            + 940 * U * (dy.double().abs() * n.abs()).sum(0))
    book2 = book - 0.1 * dbook
    assert torch.isfinite(u.unit_loss(y, book2, lists, scale, bias)[0]).all()


@pytest.mark.gpu
def test_streams_and_graphs(cuda):
    """A side stream given as an argument, and two captured graphs replayed
    in turn on new inputs, equal the plain calls."""
    from vfr import units as u

    torch = cuda

    def step(x, w, labels, bias, dloss, gamma, stream=None):
        y, mean, rstd, saved = u.layer_norm(x, gamma, None, checkpoint=True, stream=stream)
        loss, lse = u.unit_loss(y, w, labels, 0.2, bias, stream=stream)
        dy, dw, db = u.unit_loss_backward(y, w, labels, lse, dloss, 0.2, bias, stream=stream)
        dx, dg, dbeta = u.layer_norm_backward(dy, saved, mean, rstd, gamma, stream=stream)
        return y, loss, lse, dy, dw, db, dx, dg, dbeta

    for dtype in ("bf16", "f32"):
        a = _head(torch, 300, 500, 128, dtype, 31)[:5]
        b = _head(torch, 300, 500, 128, dtype, 32)[:5]
        gamma = torch.randn(128, device="cuda")
        want_a, want_b = step(*a, gamma), step(*b, gamma)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        got = step(*a, gamma, stream=s)
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(p, q) for p, q in zip(got, want_a))
        held = [t.clone() for t in a]
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(*held, gamma)
            graphs.append((graph, out))
        for inputs, want in ((b, want_b), (a, want_a)):
            for t, v in zip(held, inputs):
                t.copy_(v)
            for graph, out in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for _, out in graphs:
                assert all(torch.equal(p, q) for p, q in zip(out, want))


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(cuda):
    from vfr import units as u

    torch = cuda
    sets = [_head(torch, 1500, 2000, 256, "bf16", 40 + i) for i in range(2)]
    want = []
    for x, w, labels, bias, dloss, scale in sets:
        loss, lse = u.unit_loss(x, w, labels, scale, bias)
        want.append((loss, lse, *u.unit_loss_backward(x, w, labels, lse, dloss, scale, bias)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for (x, w, labels, bias, dloss, scale), s in zip(sets, streams):
            loss, lse = u.unit_loss(x, w, labels, scale, bias, stream=s)
            got.append((loss, lse, *u.unit_loss_backward(x, w, labels, lse, dloss, scale, bias, stream=s)))
        torch.cuda.synchronize()
        for g, t in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(g, t))


@pytest.mark.gpu
def test_device_refusals(cuda):
    from vfr import lib
    from vfr import units as u

    torch = cuda
    x = torch.randn(8, 16, device="cuda")
    labels = torch.zeros(8, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="contiguous"):
        u.layer_norm(x.t())
    with pytest.raises(ValueError, match="contiguous"):
        u.layer_norm(x[:, ::2])
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        u.layer_norm(x.double())
    with pytest.raises(ValueError, match="gamma"):
        u.layer_norm(x, torch.ones(15, device="cuda"))
    with pytest.raises(ValueError, match="labels"):
        u.unit_loss(x, x, labels.long())
    with pytest.raises(ValueError, match="units"):
        u.unit_loss(x, x.bfloat16(), labels)
    with pytest.raises(lib.NativeError, match="f32 or bf16"):
        u.unit_loss(x.half(), x.half(), labels)
    with pytest.raises(lib.NativeError, match="1..4096"):
        u.layer_norm(torch.zeros(2, 4097, device="cuda"))
    L = lib.load_library()
    s = lib.stream_struct()
    y, m, r = torch.empty_like(x), torch.empty(8, device="cuda"), torch.empty(8, device="cuda")
    host = torch.zeros(8, 16)
    with pytest.raises(lib.NativeError, match="must be device memory"):
        lib.call(L.vfr_layer_norm, host.data_ptr(), None, None, 8, 16, 0, 1e-5, y.data_ptr(), m.data_ptr(),
                 r.data_ptr(), None, None, ctypes.byref(s))
    with pytest.raises(lib.NativeError, match="workspace is too small"):
        lib.call(L.vfr_layer_norm_backward, x.data_ptr(), x.data_ptr(), None, None, m.data_ptr(), r.data_ptr(), None,
                 8, 16, 0, y.data_ptr(), m.data_ptr(), None, y.data_ptr(), 4, ctypes.byref(s))
    with pytest.raises(lib.NativeError, match="workspace is too small"):
        lib.call(L.vfr_unit_loss_backward, x.data_ptr(), x.data_ptr(), None, labels.data_ptr(), m.data_ptr(),
                 r.data_ptr(), 8, 8, 16, 0, ctypes.c_float(1.0), y.data_ptr(), y.data_ptr(), None, y.data_ptr(), 16,
                 ctypes.byref(s))
