"""Plain 64-bit forms of a layer's products (projection, choice of experts, experts) with
bounds on what fp32 sums and one rounding may differ by, for their tests. Written from
the formulas."""
import math

import numpy as np
import torch

U = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def act(name, x):
    """(act(x), bound of the device's relative error, bound of its slope)."""
    if name.startswith("silu"):
        z = x
    elif name.startswith("gelu"):
        z = 2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
    else:
        return x, torch.zeros_like(x)
    # x sigmoid(z): z (5 roundings and the constants' one each) and z log2(e) are off by
    # 8 half steps at most, which moves e^-z by 8 |z| of them and the sigmoid by as much at
    # most; exp2, the sum, the reciprocal and the product add 8 (two ulps for the two
    # hardware functions).
    y = x / (1 + torch.exp(-z.clamp(min=-700)))
    return y, U * (8 + 8 * z.abs()) * y.abs()


def linear(x, w, bias=None, activation="none", residual=None, out_dtype=None):
    """(result, bound) in 64 bits."""
    dt = out_dtype or x.dtype
    k = x.shape[1]
    xd, wd = x.double().cpu(), w.double().cpu()
    y = xd @ wd.t()
    # Products of 16-bit values are exact in fp32; k sums and the bias's.
    err = (k + 2) * U * (xd.abs() @ wd.abs().t())
    if bias is not None:
        y = y + bias.double().cpu()
        err = err + (k + 2) * U * bias.double().cpu().abs()
    if activation.endswith("_and_mul"):
        n = w.shape[0] // 2
        g, eg = act(activation, y[:, :n])
        eg = eg + 1.2 * err[:, :n]  # neither activation is steeper than 1.13
        u, eu = y[:, n:], err[:, n:]
        y, err = g * u, eg * u.abs() + eu * g.abs() + eg * eu
        err = err + U * y.abs()
    elif activation != "none":
        y, e = act(activation, y)
        err = e + 1.2 * err
    if residual is not None:
        y = y + residual.double().cpu()
        err = err + U * y.abs()
    # fp16 has denormals: half of the smallest step at least.
    return y, err * 1.01 + half_step(dt) * (y.abs() + err) + torch.finfo(dt).smallest_normal * half_step(dt) * 2


def check(got, want, bound, what=""):
    d = (got.double().cpu() - want).abs()
    bad = ~(d <= bound)
    if bad.any():
        i = tuple(int(v) for v in torch.nonzero(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: got "
                             f"{float(got[i])}, want {float(want[i])}, bound {float(bound[i]):.3g}")


def route(logits, top_k, renormalize):
    """(weights, experts) in 64 bits: stable order by falling logit, NaN last."""
    v = logits.double().cpu().numpy()
    key = np.where(np.isnan(v), np.inf, -v)
    nan = np.isnan(v)
    order = np.lexsort((np.broadcast_to(np.arange(v.shape[1]), v.shape), key, nan), axis=-1)
    ids = order[:, :top_k]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp(v - np.max(v, axis=1, keepdims=True))
        p = w / w.sum(1, keepdims=True)
        p = np.take_along_axis(p, ids, 1)
        if renormalize:
            p = p / p.sum(1, keepdims=True)
    return torch.from_numpy(p), torch.from_numpy(ids.astype(np.int32))


def experts(x, gate_up, down, weights, ids, residual=None, activation="silu_and_mul"):
    """(result, bound) in 64 bits, what lies between the projections unrounded."""
    T, H = x.shape
    E, I = gate_up.shape[0], down.shape[2]
    K = weights.shape[1]
    eps = half_step(x.dtype)
    y = torch.zeros(T, H, dtype=torch.float64)
    err, var = torch.zeros_like(y), torch.zeros_like(y)
    xc, wc, ic = x.double().cpu(), weights.double().cpu(), ids.cpu()
    size = torch.zeros_like(y)
    for e in range(E):
        t, j = torch.nonzero(ic == e, as_tuple=True)
        if len(t) == 0:
            continue
        w = gate_up[e].double().cpu()
        both = xc[t] @ w.t()
        eb = (H + 2) * U * (xc[t].abs() @ w.abs().t())
        g, eg = act(activation, both[:, :I])
        eg = eg + 1.2 * eb[:, :I]
        u, eu = both[:, I:], eb[:, I:]
        h = g * u
        eh = eg * u.abs() + eu * g.abs() + eg * eu + U * h.abs()
        d = down[e].double().cpu()
        f = wc[t, j][:, None]
        # A token may choose an expert twice.
        y.index_add_(0, t, f * (h @ d.t()))
        s = f.abs() * (h.abs() @ d.abs().t())
        size.index_add_(0, t, s)
        err.index_add_(0, t, f.abs() * (eh @ d.abs().t()) + (I + 4) * U * s)
        # h rounded to the type: independent errors of at most half a step of it (of its
        # smallest step, for fp16's denormals).
        step = eps * (h.abs() + eh) + torch.finfo(x.dtype).smallest_normal * eps
        var.index_add_(0, t, f ** 2 * ((step ** 2) @ (d ** 2).t()))
        # The weighted output may be rounded once more before the sum.
        var.index_add_(0, t, (eps * f * (h @ d.t())) ** 2)
    err = err + (K + 2) * U * size
    if residual is not None:
        y = y + residual.double().cpu()
        err = err + U * y.abs()
    # Independent errors bounded by s_i pass 8 sqrt(sum s_i^2) with a probability below
    # 2 e^-32 (Hoeffding).
    err = err + 8 * var.sqrt()
    return y, err * 1.01 + eps * (y.abs() + err) + torch.finfo(x.dtype).smallest_normal * eps * 2
