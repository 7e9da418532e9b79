"""Cases that measure the unit-head operators: layer norm and its gradients,
8-bit activation checkpoints, and the softmax cross entropy of frames over a
codebook of units with its gradients.

`run` computes a case in plain torch (f32, rounded once at the end) or, with
`own` set, through the library's Python calls (`vfr.units`).  `exact` states
the same results in f64.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_EPS = 1e-5
_BLOCK = 128  # elements of a row that share one checkpoint exponent


def listed():
    return [
        # One realtime block (34 HuBERT frames of an RVC v2 voice) through the
        # norm in front of the unit head: a call whose latency counts.
        {"name": "norm-block-f32", "kind": "norm", "rows": 34, "width": 768, "dtype": "f32"},
        # An offline batch of 30,000 frames, mixed-precision training.
        {"name": "norm-batch-bf16", "kind": "norm", "rows": 30000, "width": 768, "dtype": "bf16"},
        # Gradients of one utterance whose width fits no vector load.
        {"name": "norm-grad-ragged-f32", "kind": "norm_grad", "rows": 2999, "width": 513, "dtype": "f32"},
        # Gradients of the offline batch.
        {"name": "norm-grad-batch-bf16", "kind": "norm_grad", "rows": 30000, "width": 768, "dtype": "bf16"},
        # Norm forward with an 8-bit checkpoint of its input, then backward
        # from the checkpoint: a short v1 (256-wide) block in fp16 ...
        {"name": "norm-step-block-f16", "kind": "norm_step", "rows": 140, "width": 256, "dtype": "f16"},
        # ... and the offline batch in f32, where the checkpoint saves most.
        {"name": "norm-step-batch-f32", "kind": "norm_step", "rows": 30000, "width": 768, "dtype": "f32"},
        # One frame kept in 8 bits and read back.
        {"name": "checkpoint-row-f32", "kind": "checkpoint", "rows": 1, "width": 768, "dtype": "f32"},
        # A batch at the library's widest rows kept in 8 bits and read back.
        {"name": "checkpoint-batch-bf16", "kind": "checkpoint", "rows": 30000, "width": 4096, "dtype": "bf16"},
        # Loss of one realtime block over the 511 lists of a voice index.
        {"name": "units-block-f32", "kind": "units", "rows": 34, "units": 511, "width": 768, "dtype": "f32",
         "masked": 3},
        # Loss of an offline batch over a large codebook.
        {"name": "units-batch-bf16", "kind": "units", "rows": 30000, "units": 16384, "width": 768, "dtype": "bf16",
         "masked": 0},
        # Gradients in full precision at odd sizes, some units masked (empty clusters).
        {"name": "units-grad-ragged-f32", "kind": "units_grad", "rows": 1003, "units": 2003, "width": 768,
         "dtype": "f32", "masked": 17},
        # Gradients of the offline batch over the large codebook.
        {"name": "units-grad-batch-bf16", "kind": "units_grad", "rows": 30000, "units": 16384, "width": 768,
         "dtype": "bf16", "masked": 0},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "norm_step", "checkpoint", "units", "units_grad"])
    width = _log_int(rng, 8, 4096)
    if rng.random() < 0.5:
        width = rng.choice([256, 512, 768, 1024])
    if kind in ("units", "units_grad"):
        dtype = rng.choice(["f32", "bf16"])
        rows = _log_int(rng, 1, 30000)
        units = _log_int(rng, 2, 16384)
        # the f32 cases stay below the largest bf16 one
        limit = 30000 * 16384 * 768 // (8 if dtype == "f32" else 1)
        while rows * units * width > limit:
            rows, units = max(1, rows * 2 // 3), max(2, units * 2 // 3)
        masked = rng.choice([0, 0, units // 50, units // 3])
        return {"kind": kind, "rows": rows, "units": units, "width": width, "dtype": dtype, "masked": masked}
    return {"kind": kind, "rows": _log_int(rng, 1, 30000), "width": width,
            "dtype": rng.choice(["f32", "bf16", "f16"])}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def prepare(case, seed):
    g = _generator(seed)
    rows, width, dtype = case["rows"], case["width"], _DTYPES[case["dtype"]]
    state = {"case": dict(case), "dtype": dtype}
    if case["kind"] in ("units", "units_grad"):
        k = case["units"]
        units = _randn(g, k, width)
        labels = torch.randint(0, k, (rows,), generator=g, device="cuda", dtype=torch.int64)
        # frames lean toward their unit, about as far as a half-trained head
        # (target logit 4 noise deviations above the mean)
        x = _randn(g, rows, width) + (4.0 / math.sqrt(width)) * units[labels]
        state["x"] = x.to(dtype)
        state["units"] = units.to(dtype)
        # logits: the inner product scaled to a deviation of 4, and the
        # squared-norm term that makes them a soft nearest-centroid choice
        scale = 4.0 / math.sqrt(width)
        bias = -0.05 * scale * (units * units).sum(1)
        masked = case["masked"]
        if masked:
            # empty clusters take no part
            bias[torch.randperm(k, generator=g, device="cuda")[:masked]] = -math.inf
        state["scale"], state["bias"] = scale, bias
        # frames of a batch's padding carry no label
        pad = torch.rand(rows, generator=g, device="cuda") < 0.04
        labels = torch.where(pad | torch.isinf(bias)[labels], torch.full_like(labels, -1), labels)
        state["labels"] = labels.to(torch.int32)
        if case["kind"] == "units_grad":
            state["dloss"] = torch.full((rows,), 1.0 / rows, device="cuda") * (
                0.5 + torch.rand(rows, generator=g, device="cuda"))
            # the forward pass's result, in the program's hands before the backward
            state["lse"] = _plain_units(state["x"], state["units"], state["labels"], scale, bias)[1]
        return state
    # frames: unit-scale channels with their own offsets, a few far larger
    x = _randn(g, rows, width) + 0.5 * _randn(g, 1, width)
    loud = torch.rand(width, generator=g, device="cuda") < 0.02
    x = torch.where(loud, 20.0 * x, x)
    state["x"] = x.to(dtype)
    if case["kind"] == "checkpoint":
        return state
    state["gamma"] = 1.0 + 0.2 * _randn(g, width)
    state["beta"] = 0.1 * _randn(g, width)
    if case["kind"] in ("norm_grad", "norm_step"):
        state["dy"] = _randn(g, rows, width).to(dtype)
    if case["kind"] == "norm_grad":
        _, state["mean"], state["rstd"] = _plain_norm(state["x"], state["gamma"], state["beta"])
    return state


# ------------------------------------------------------------- plain forms


def _plain_norm(x, gamma, beta):
    v = x.float()
    mean = v.sum(1, keepdim=True) / v.shape[1]
    c = v - mean
    var = (c * c).sum(1, keepdim=True) / v.shape[1]
    rstd = 1.0 / torch.sqrt(var + _EPS)
    y = c * rstd * gamma + beta
    return y.to(x.dtype), mean[:, 0], rstd[:, 0]


def _plain_norm_grad(dy, x, mean, rstd, gamma):
    d = dy.float()
    n = (x.float() - mean[:, None]) * rstd[:, None]
    g = d * gamma
    width = d.shape[1]
    a = g.sum(1, keepdim=True) / width
    b = (g * n).sum(1, keepdim=True) / width
    dx = (g - a - n * b) * rstd[:, None]
    return dx.to(dy.dtype), (d * n).sum(0), d.sum(0)


def _plain_checkpoint(x):
    """The values that the 8-bit checkpoint of x stands for (f32): per 128
    elements of a row a power of two 2^s, the smallest that brings the
    block's largest magnitude to at most 448, and each x / 2^s rounded to
    e4m3."""
    v = x.float()
    rows, width = v.shape
    blocks = (width + _BLOCK - 1) // _BLOCK
    p = torch.zeros(rows, blocks * _BLOCK, device=v.device)
    p[:, :width] = v
    p = p.view(rows, blocks, _BLOCK)
    bits = p.abs().amax(2, keepdim=True).view(torch.int32)
    e = (bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()
    s = e.clamp(min=0) - 127
    # 2^-s and 2^(s + 1) from their exponent bits: exact, and both normal numbers
    q = (p * ((127 - s) << 23).view(torch.float32)).to(torch.float8_e4m3fn).float()
    return (q * ((s + 128) << 23).view(torch.float32) * 0.5).view(rows, -1)[:, :width]


def _plain_units(x, units, labels, scale, bias):
    z = (x.float() @ units.float().t()) * scale + bias
    top = z.amax(1, keepdim=True)
    lse = (top + torch.log(torch.exp(z - top).sum(1, keepdim=True)))[:, 0]
    rows = torch.arange(x.shape[0], device=x.device)
    target = z[rows, labels.long().clamp(min=0)]
    return torch.where(labels >= 0, lse - target, torch.zeros_like(lse)), lse


def _plain_units_grad(x, units, labels, lse, dloss, scale, bias):
    xf, wf = x.float(), units.float()
    p = torch.exp((xf @ wf.t()) * scale + bias - lse[:, None])
    valid = labels >= 0
    rows = torch.arange(x.shape[0], device=x.device)
    p[rows[valid], labels[valid].long()] -= 1.0
    p = p * torch.where(valid, dloss, torch.zeros_like(dloss))[:, None]
    dbias = p.sum(0)
    dx = (p @ wf) * scale
    dw = (p.t() @ xf) * scale
    return dx.to(x.dtype), dw.to(units.dtype), dbias


def _units():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vocal-fast-rs_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from vfr import units

    return units


def run(state):
    kind = state["case"]["kind"]
    s = state
    if own:
        u = _units()
        if kind == "norm":
            return u.layer_norm(s["x"], s["gamma"], s["beta"], _EPS)
        if kind == "norm_grad":
            return u.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["gamma"])
        if kind == "norm_step":
            y, mean, rstd, saved = u.layer_norm(s["x"], s["gamma"], s["beta"], _EPS, checkpoint=True)
            return (y, *u.layer_norm_backward(s["dy"], saved, mean, rstd, s["gamma"]))
        if kind == "checkpoint":
            return u.checkpoint_unpack(u.checkpoint_pack(s["x"]), torch.float32)
        if kind == "units":
            return u.unit_loss(s["x"], s["units"], s["labels"], s["scale"], s["bias"])
        return u.unit_loss_backward(s["x"], s["units"], s["labels"], s["lse"], s["dloss"], s["scale"], s["bias"])
    if kind == "norm":
        return _plain_norm(s["x"], s["gamma"], s["beta"])
    if kind == "norm_grad":
        return _plain_norm_grad(s["dy"], s["x"], s["mean"], s["rstd"], s["gamma"])
    if kind == "norm_step":
        y, mean, rstd = _plain_norm(s["x"], s["gamma"], s["beta"])
        return (y, *_plain_norm_grad(s["dy"], _plain_checkpoint(s["x"]), mean, rstd, s["gamma"]))
    if kind == "checkpoint":
        return _plain_checkpoint(s["x"])
    if kind == "units":
        return _plain_units(s["x"], s["units"], s["labels"], s["scale"], s["bias"])
    return _plain_units_grad(s["x"], s["units"], s["labels"], s["lse"], s["dloss"], s["scale"], s["bias"])


def work(case):
    rows, width, es = case["rows"], case["width"], _BYTES[case["dtype"]]
    kind = case["kind"]
    cells = rows * width
    exponents = rows * ((width + _BLOCK - 1) // _BLOCK)
    if kind == "norm":
        return {"bytes": 2 * cells * es + 8 * width + 8 * rows, "flops": 8 * cells}
    if kind == "norm_grad":
        return {"bytes": 3 * cells * es + 12 * width + 8 * rows, "flops": 13 * cells}
    if kind == "norm_step":
        # x and dy in, y and dx out; the checkpoint written and read once
        return {"bytes": 4 * cells * es + 2 * (cells + exponents) + 16 * width, "flops": 23 * cells}
    if kind == "checkpoint":
        # the checkpoint written and read once, the values out in f32
        return {"bytes": cells * (es + 4) + 2 * (cells + exponents), "flops": 3 * cells}
    k = case["units"]
    if kind == "units":
        return {"bytes": (cells + k * width) * es + 4 * k + 12 * rows, "flops": 2 * cells * k}
    # the logits again from the kept log-sum, then both products
    return {"bytes": 2 * (cells + k * width) * es + 8 * k + 12 * rows, "flops": 6 * cells * k}


# ------------------------------------------------------------- definitions in 64 bits


def _exact_moments(x):
    v = x.double()
    mean = v.mean(1)
    var = ((v - mean[:, None]) ** 2).mean(1)
    return v, mean, (var + _EPS) ** -0.5


def _exact_norm_grad(dy, values, mean, rstd, gamma):
    d, n = dy.double(), (values - mean[:, None]) * rstd[:, None]
    g = d * gamma.double()
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True))
    return dx, (d * n).sum(0), d.sum(0)


def _power(e):
    """2^e in f64 from its exponent bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_checkpoint(x):
    v = x.double()
    out = torch.empty_like(v)
    for lo in range(0, v.shape[1], _BLOCK):
        b = v[:, lo:lo + _BLOCK]
        # top = m 2^e with m in [1/2, 1): the smallest s with top <= (7/8) 2^(s + 9)
        m, e = torch.frexp(b.abs().amax(1, keepdim=True))
        s = e - 9 + (m > 0.875).int()
        s = torch.where(m > 0, s, torch.full_like(s, -127)).clamp(min=-127)
        r = b * _power(-s)
        # e4m3: 3 fraction bits, smallest exponent -6
        step = _power((torch.frexp(r)[1] - 1).clamp(min=-6) - 3)
        out[:, lo:lo + _BLOCK] = torch.round(r / step) * step * _power(s)
    return out


def _exact_logits(s, lo, hi):
    z = s["x"][lo:hi].double() @ s["units"].double().t()
    return z.mul_(s["scale"]).add_(s["bias"].double())


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "checkpoint":
        return _exact_checkpoint(s["x"])
    if kind == "norm":
        v, mean, rstd = _exact_moments(s["x"])
        return (v - mean[:, None]) * rstd[:, None] * s["gamma"].double() + s["beta"].double(), mean, rstd
    if kind == "norm_grad":
        return _exact_norm_grad(s["dy"], s["x"].double(), s["mean"].double(), s["rstd"].double(), s["gamma"])
    if kind == "norm_step":
        v, mean, rstd = _exact_moments(s["x"])
        y = (v - mean[:, None]) * rstd[:, None] * s["gamma"].double() + s["beta"].double()
        return (y, *_exact_norm_grad(s["dy"], _exact_checkpoint(s["x"]), mean, rstd, s["gamma"]))
    rows, step = case["rows"], 4096
    labels = s["labels"].long()
    if kind == "units":
        loss = torch.zeros(rows, dtype=torch.float64, device="cuda")
        lse = torch.zeros_like(loss)
        for lo in range(0, rows, step):
            hi = min(rows, lo + step)
            z = _exact_logits(s, lo, hi)
            lse[lo:hi] = torch.logsumexp(z, 1)
            t = labels[lo:hi]
            hit = torch.nonzero(t >= 0)[:, 0]
            loss[lo + hit] = lse[lo + hit] - z[hit, t[hit]]
        return loss, lse
    w = s["units"].double()
    dx = torch.zeros(rows, case["width"], dtype=torch.float64, device="cuda")
    dw = torch.zeros_like(w)
    dbias = torch.zeros(w.shape[0], dtype=torch.float64, device="cuda")
    for lo in range(0, rows, step):
        hi = min(rows, lo + step)
        g = _exact_logits(s, lo, hi).sub_(s["lse"][lo:hi, None].double()).exp_()
        t = labels[lo:hi]
        hit = torch.nonzero(t >= 0)[:, 0]
        g[hit, t[hit]] -= 1.0
        g *= (s["dloss"][lo:hi].double() * (t >= 0).double())[:, None]
        dx[lo:hi] = g @ w * s["scale"]
        dw += g.t() @ s["x"][lo:hi].double() * s["scale"]
        dbias += g.sum(0)
    return dx, dw, dbias
