"""The products around a layer's attention, as a decoder's step runs them, measured one
by one:

  linear    a projection with what follows it: bias, activation (or gate and up
            projection joined by it), residual
  route     the experts of each token and their weights, from the router's logits
  experts   a mixture-of-experts layer behind the router: gate and up projection,
            activation, down projection, weighted sum

  listed()              the fixed cases
  draw(rng)             one more case of the same ranges
  prepare(case, seed)   inputs on the GPU
  run(state)            one pass and its outputs: elementary torch operations, or
                        (own) the framework's operators
  work(case)            bytes and operations a pass cannot do without
  exact(case, seed)     the outputs in 64 bits, written apart from run()

Widths are those of the framework's own workloads (hidden 4096 with 32 + 8 + 8 heads of
128 and an intermediate width of 12,288; hidden 2048 with experts of 768). Which experts
the tokens of a case share is drawn from the case's own `routing` number, so a case's
work is the same for every seed; the seed makes the data and says which token and which
expert is which.
"""
import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

ROOT = Path(__file__).resolve().parent.parent
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GATED = ("silu_and_mul", "gelu_and_mul")

own = False


def _backend():
    """The C++ backend module (the package's directory name is not a Python
    identifier, so it is loaded by path)."""
    name = "sglang_cpp_amd"
    if name not in sys.modules:
        pkg = ROOT / "sglang.cpp_amd"
        spec = importlib.util.spec_from_file_location(
            name, pkg / "__init__.py", submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name].backend.load()


# ------------------------------------------------------------------ cases

def _linear(tokens, n, k, activation="none", bias=False, residual=False, dtype="bf16",
            out="same"):
    return dict(kind="linear", tokens=tokens, n=n, k=k, activation=activation, bias=bias,
                residual=residual, dtype=dtype, out=out)


def _route(tokens, experts, top_k, dtype="fp32", renormalize=True):
    return dict(kind="route", tokens=tokens, experts=experts, top_k=top_k, dtype=dtype,
                renormalize=renormalize)


def _experts(tokens, experts, top_k, hidden, inter, routing, dtype="bf16"):
    return dict(kind="experts", tokens=tokens, experts=experts, top_k=top_k, hidden=hidden,
                inter=inter, routing=routing, dtype=dtype)


def listed():
    return [
        # The router's logits for a decode step of a few requests: launch latency.
        dict(name="linear_router_b7", **_linear(7, 128, 2048, out="fp32")),
        # One user's token through the joined q, k and v projection, with their bias.
        dict(name="linear_qkv_b1", **_linear(1, 6144, 4096, bias=True)),
        # A small batch's gate and up projection, the activation between them.
        dict(name="linear_mlp_b5", **_linear(5, 12_288, 4096, activation="silu_and_mul")),
        # A busy server's output projection back onto the residual stream.
        dict(name="linear_o_b48", **_linear(48, 4096, 4096, residual=True)),
        # A chunk of an odd number of tokens through the down projection.
        dict(name="linear_down_chunk", **_linear(333, 4096, 12_288, residual=True, dtype="fp16")),
        # A full prefill batch's gate and up projection.
        dict(name="linear_mlp_prefill", **_linear(8192, 12_288, 4096, activation="silu_and_mul")),
        # A decode step's tokens choose their experts.
        dict(name="route_b7", **_route(7, 128, 8)),
        # A full prefill batch's choice.
        dict(name="route_prefill", **_route(16_384, 128, 8, dtype="bf16")),
        # One user's token through its eight experts.
        dict(name="experts_b1", **_experts(1, 128, 8, 2048, 768, 1)),
        # A decode batch that reaches most experts with a token or two each.
        dict(name="experts_b24", **_experts(24, 128, 8, 2048, 768, 2)),
        # A chunk of an odd number of tokens: some fifty for each expert.
        dict(name="experts_chunk", **_experts(777, 128, 8, 2048, 768, 3)),
        # A full prefill batch.
        dict(name="experts_prefill", **_experts(8192, 128, 8, 2048, 768, 4)),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width of `lo` to `hi`: mostly whole 64s, some whole 8s, a few odd ones."""
    unit = rng.choice((64, 64, 64, 8, 8, 1))
    return max(lo, _log_int(rng, lo, hi) // unit * unit)


def draw(rng):
    kind = rng.choice(("linear", "linear", "linear", "route", "experts", "experts"))
    if kind == "linear":
        act = rng.choice(("none", "none", "silu", "gelu", "silu_and_mul", "gelu_and_mul"))
        return _linear(_log_int(rng, 1, 8192), _width(rng, 64, 12_288), _width(rng, 64, 12_288 if
                       act not in GATED else 4096), act, rng.random() < 0.4, rng.random() < 0.4,
                       rng.choice(("bf16", "fp16")), "fp32" if rng.random() < 0.15 else "same")
    if kind == "route":
        experts = rng.choice((8, 16, 60, 64, 128, 128, 256))
        return _route(_log_int(rng, 1, 16_384), experts, rng.randint(1, min(8, experts)),
                      rng.choice(("fp32", "bf16", "fp16")), rng.random() < 0.7)
    experts, top_k, hidden, inter = rng.choice((
        (128, 8, 2048, 768), (128, 8, 2048, 768), (64, 6, 2048, 1408), (60, 4, 2048, 1408),
        (8, 2, 4096, 1792), (32, 8, 1024, 512), (16, 1, 1000, 360)))
    return _experts(_log_int(rng, 1, 8192), experts, top_k, hidden, inter, rng.randrange(1 << 20),
                    rng.choice(("bf16", "bf16", "fp16")))


# ------------------------------------------------------------------ routing

def _choice(case):
    """[tokens, top_k] experts of a case, some more popular than others."""
    rng = np.random.default_rng(case["routing"])
    score = rng.standard_normal((case["tokens"], case["experts"])) \
        + 0.5 * rng.standard_normal(case["experts"])
    return np.argsort(-score, axis=1, kind="stable")[:, :case["top_k"]]


# ------------------------------------------------------------------ prepare

def _prepare_linear(case, g):
    T, n, k, dt = case["tokens"], case["n"], case["k"], DTYPES[case["dtype"]]
    rows = 2 * n if case["activation"] in GATED else n
    make = lambda *shape: torch.randn(shape, generator=g, device=DEV)
    return dict(x=make(T, k).to(dt), weight=(make(rows, k) / math.sqrt(k)).to(dt),
                bias=make(rows).to(dt) if case["bias"] else None,
                residual=make(T, n).to(dt) if case["residual"] else None,
                out_dtype=torch.float32 if case["out"] == "fp32" else dt)


def _prepare_route(case, g):
    logits = torch.randn((case["tokens"], case["experts"]), generator=g, device=DEV)
    return dict(logits=(2 * logits).to(DTYPES[case["dtype"]]))


def _prepare_experts(case, g):
    T, E, H, I, dt = (case["tokens"], case["experts"], case["hidden"], case["inter"],
                      DTYPES[case["dtype"]])
    chosen = torch.from_numpy(_choice(case)).to(DEV)
    token = torch.randperm(T, generator=g, device=DEV)
    expert = torch.randperm(E, generator=g, device=DEV)
    make = lambda *shape: torch.randn(shape, generator=g, device=DEV)
    weights = torch.softmax(make(T, case["top_k"]), -1).sort(-1, descending=True).values
    return dict(x=make(T, H).to(dt), gate_up=(make(E, 2 * I, H) / math.sqrt(H)).to(dt),
                down=(make(E, H, I) / math.sqrt(I)).to(dt), weights=weights.contiguous(),
                experts=expert[chosen[token]].int().contiguous())


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    make = {"linear": _prepare_linear, "route": _prepare_route, "experts": _prepare_experts}
    return dict(make[case["kind"]](case, g), case=case)


# ------------------------------------------------------------------ plain forms

def _silu(x):
    return x / (1 + (-x).exp())


def _gelu(x):
    return 0.5 * x * (1 + (0.7978845608028654 * (x + 0.044715 * x * x * x)).tanh())


def _plain_linear(s):
    c = s["case"]
    y = s["x"].float() @ s["weight"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    act = c["activation"]
    if act in GATED:
        y = (_silu if act == "silu_and_mul" else _gelu)(y[:, :c["n"]]) * y[:, c["n"]:]
    elif act != "none":
        y = (_silu if act == "silu" else _gelu)(y)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["out_dtype"])


def _plain_route(s):
    c, logits = s["case"], s["logits"].float()
    best = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :c["top_k"]]
    e = (logits - logits.amax(-1, keepdim=True)).exp()
    p = (e / e.sum(-1, keepdim=True)).gather(-1, best)
    if c["renormalize"]:
        p = p / p.sum(-1, keepdim=True)
    return dict(weights=p, experts=best.int())


def _plain_experts(s):
    c = s["case"]
    T, K, H, I = c["tokens"], c["top_k"], c["hidden"], c["inter"]
    flat = s["experts"].reshape(-1).long()
    order = torch.sort(flat, stable=True).indices
    counts = torch.bincount(flat, minlength=c["experts"]).tolist()
    y = torch.empty((T * K, H), device=DEV)
    at = 0
    for e, n in enumerate(counts):
        if n == 0:
            continue
        rows = order[at:at + n]
        at += n
        h = s["x"][rows // K].float() @ s["gate_up"][e].float().t()
        y[rows] = (_silu(h[:, :I]) * h[:, I:]) @ s["down"][e].float().t()
    return (y.view(T, K, H) * s["weights"][..., None]).sum(1).to(s["x"].dtype)


# ------------------------------------------------------------------ the framework's operators

def _own_linear(s):
    return _backend().linear(s["x"], s["weight"], bias=s["bias"],
                             activation=s["case"]["activation"], residual=s["residual"],
                             out_dtype=s["out_dtype"])


def _own_route(s):
    c = s["case"]
    weights, experts = _backend().moe_route(s["logits"], c["top_k"], renormalize=c["renormalize"])
    return dict(weights=weights, experts=experts)


def _own_experts(s):
    return _backend().moe_experts(s["x"], s["gate_up"], s["down"], s["weights"], s["experts"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"linear": _own_linear, "route": _own_route, "experts": _own_experts}[kind](state)
    return {"linear": _plain_linear, "route": _plain_route, "experts": _plain_experts}[kind](state)


# ------------------------------------------------------------------ work

def work(case):
    kind, T = case["kind"], case["tokens"]
    if kind == "linear":
        n, k = case["n"], case["k"]
        rows = 2 * n if case["activation"] in GATED else n
        out = 4 if case["out"] == "fp32" else 2
        return {"bytes": 2 * (T * k + rows * k + (rows if case["bias"] else 0)
                              + (T * n if case["residual"] else 0)) + out * T * n,
                "flops": 2 * T * rows * k}
    if kind == "route":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": T * (size * case["experts"] + 8 * case["top_k"]),
                "flops": 3 * T * case["experts"]}
    chosen = _choice(case)
    H, I = case["hidden"], case["inter"]
    return {"bytes": 6 * len(np.unique(chosen)) * H * I + 4 * T * H + 8 * chosen.size,
            "flops": 6 * chosen.size * H * I}


# ------------------------------------------------------------------ exact

def _act64(name, x):
    if name.startswith("silu"):
        return x * torch.sigmoid(x)
    if name.startswith("gelu"):
        return x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))
    return x


def _exact_linear(case, s):
    T, n, act = case["tokens"], case["n"], case["activation"]
    out = torch.empty((T, n), dtype=torch.float64, device=DEV)
    x = s["x"].double()
    for a in range(0, n, 4096):  # a part of the columns at a time
        b = min(n, a + 4096)
        part = lambda first: torch.nn.functional.linear(
            x, s["weight"][first + a:first + b].double(),
            None if s["bias"] is None else s["bias"][first + a:first + b].double())
        y = _act64(act, part(0))
        if act in GATED:
            y = y * part(n)
        out[:, a:b] = y if s["residual"] is None else y + s["residual"][:, a:b].double()
    return out


def _exact_route(case, s):
    v = s["logits"].double().cpu().numpy()
    rank = np.lexsort((np.broadcast_to(np.arange(v.shape[1]), v.shape), -v), axis=-1)
    experts = rank[:, :case["top_k"]]
    w = np.exp(v - v.max(1, keepdims=True))
    p = np.take_along_axis(w, experts, 1)
    p = p / (p if case["renormalize"] else w).sum(1, keepdims=True)
    return dict(weights=torch.from_numpy(p), experts=torch.from_numpy(experts.astype(np.int32)))


def _exact_experts(case, s):
    I = case["inter"]
    x = s["x"].double()
    out = torch.zeros_like(x)
    for e in range(case["experts"]):
        token, slot = torch.nonzero(s["experts"] == e, as_tuple=True)
        if len(token) == 0:
            continue
        both = x[token] @ s["gate_up"][e].double().t()
        gate, up = both[:, :I], both[:, I:]
        y = (gate * torch.sigmoid(gate) * up) @ s["down"][e].double().t()
        out.index_add_(0, token, y * s["weights"][token, slot].double()[:, None])
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"linear": _exact_linear, "route": _exact_route,
            "experts": _exact_experts}[case["kind"]](case, state)
