"""Plain 64-bit forms of the shared-prefix step's operators, for their tests:
scaled rotary tables, rotate and append, attention behind a shared prefix and the
verification of drafted tokens. Written from the formulas; torch float64 on
whatever device the inputs are, and numpy."""
import math

import numpy as np
import torch


def frequencies(rotary, base, kind="none", factor=1.0, original=0, beta_fast=32.0, beta_slow=1.0,
                low=1.0, high=4.0, attention=0.0):
    """(f [rotary / 2], factor of cos and sin)."""
    f = np.array([base ** (-2.0 * i / rotary) for i in range(rotary // 2)])
    m = 1.0
    if kind == "linear":
        f = f / factor
    elif kind == "ntk":
        b = base * factor ** (rotary / (rotary - 2))
        f = np.array([b ** (-2.0 * i / rotary) for i in range(rotary // 2)])
    elif kind == "yarn":
        pair = lambda t: rotary * math.log(original / (2 * math.pi * t)) / (2 * math.log(base))
        lo = max(math.floor(pair(beta_fast)), 0)
        hi = min(math.ceil(pair(beta_slow)), rotary - 1)
        for i in range(len(f)):
            g = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f[i] = f[i] * (g / factor + 1 - g)
        m = attention if attention > 0 else (0.1 * math.log(factor) + 1 if factor > 1 else 1.0)
    elif kind == "bands":
        for i in range(len(f)):
            turns = original * f[i] / (2 * math.pi)
            w = min(max((turns - low) / (high - low), 0.0), 1.0)
            f[i] = f[i] * ((1 - w) / factor + w)
    return f, m


def rotate(x, cos, sin, interleaved):
    """x [T, heads, d] rotated by cos, sin [T, rotary / 2], in 64 bits; also the sum of the
    absolute products of each element (what fp32 roundings are relative to)."""
    x, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    half = cos.shape[1]
    out, size = x.clone(), x.abs().clone()
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    size[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    size[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return out, size


def prefix_rows(q, kc, vc, prefix_indices, indices, kv_indptr, qo_indptr, scale):
    """{row: (o [Hq, D], sum_j p_j |v_j| [Hq, D])} of every query row, in 64 bits."""
    hq, hkv = q.shape[1], kc.shape[1]
    rows = {}
    for r in range(len(kv_indptr) - 1):
        own = indices[int(kv_indptr[r]):int(kv_indptr[r + 1])]
        slots = torch.cat([prefix_indices, own]).long()
        qo = int(qo_indptr[r + 1]) - int(qo_indptr[r])
        k = kc[slots].double().repeat_interleave(hq // hkv, 1).permute(1, 0, 2).contiguous()
        v = vc[slots].double().repeat_interleave(hq // hkv, 1).permute(1, 0, 2).contiguous()
        for i in range(qo):
            row = int(qo_indptr[r]) + i
            sees = len(slots) - qo + i + 1
            if sees <= 0:
                z = torch.zeros(q.shape[1:], dtype=torch.float64, device=q.device)
                rows[row] = (z, z)
                continue
            score = (k[:, :sees] * q[row].double()[:, None]).sum(-1) * scale
            p = torch.softmax(score, -1)[..., None]
            rows[row] = ((p * v[:, :sees]).sum(1), (p * v[:, :sees].abs()).sum(1))
    return rows


def verify(target, draft, tokens, indptr, accept_u, sample_u):
    """(tokens, accepted) as lists, numpy float64."""
    V = target.shape[1]
    out, accepted = [], []
    for r in range(len(indptr) - 1):
        d0, n = int(indptr[r]), int(indptr[r + 1]) - int(indptr[r])
        a = 0
        while a < n:
            x = int(tokens[d0 + a])
            if not 0 <= x < V:
                break
            qx = 1.0 if draft is None else float(draft[d0 + a, x])
            if not float(accept_u[d0 + a]) * qx < float(target[d0 + r + a, x]):
                break
            a += 1
        p = target[d0 + r + a].astype(np.float64)
        p = np.where(p > 0, p, 0.0)
        w = p
        if a < n:
            less = np.zeros(V)
            if draft is not None:
                less = draft[d0 + a].astype(np.float64)
            elif 0 <= int(tokens[d0 + a]) < V:
                less[int(tokens[d0 + a])] = np.inf
            w = target[d0 + r + a].astype(np.float64) - less
            w = np.where(w > 0, w, 0.0)
            if not w.sum() > 0:
                w = p
        if not w.sum() > 0:
            token = V - 1
        else:
            run = np.cumsum(w)
            past = np.nonzero(run > float(sample_u[r]) * run[-1])[0]
            token = int(past[0]) if len(past) else int(np.nonzero(w)[0][-1])
        out += [int(t) for t in tokens[d0:d0 + a]] + [token] + [-1] * (n - a)
        accepted.append(a)
    return out, accepted
