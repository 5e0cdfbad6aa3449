"""The operators of a target model's step over a batch that shares a prompt, as
speculative decoding and parallel sampling run it, measured one by one:

  rope_table   the cos/sin table of a rotary embedding scaled for long contexts
  rope_append  q and k rotated (half or interleaved pairs, part of the head), k
               and v appended to the paged pool on the way
  prefix       attention over [shared prefix | the request's own suffix], the
               prefix's keys and values read once for the whole batch
  verify       drafted tokens accepted or rejected against the target's
               probabilities, and the token that follows them

  listed()              the fixed cases
  draw(rng)             one more case of the same ranges
  prepare(case, seed)   inputs on the GPU
  run(state)            one pass and its outputs: elementary torch operations, or
                        (own) the framework's operators
  work(case)            bytes and operations a pass cannot do without
  exact(case, seed)     the outputs in 64 bits, written apart from run()

Head counts, head size and vocabulary are those of the framework's own
workloads. Lengths are drawn from the case's own `lengths` number, so a case's
work is the same for every seed; the seed makes the data.
"""
import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

ROOT = Path(__file__).resolve().parent.parent
D = 128
VOCAB = 151_936
BASE = 1_000_000.0
PAGE = 16
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

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

def _table(positions, rotary, scaling, factor):
    return dict(kind="rope_table", positions=positions, rotary=rotary, scaling=scaling,
                factor=factor)


def _append(tokens, hq, hkv, rotary=D, interleaved=False, dtype="bf16", max_pos=40_960):
    return dict(kind="rope_append", tokens=tokens, hq=hq, hkv=hkv, rotary=rotary,
                interleaved=interleaved, dtype=dtype, max_pos=max_pos)


def _prefix(batch, prefix, hq, hkv, lengths, lo, hi, qo_lo=1, qo_hi=1):
    return dict(kind="prefix", batch=batch, prefix=prefix, hq=hq, hkv=hkv, lengths=lengths,
                lo=lo, hi=hi, qo_lo=qo_lo, qo_hi=qo_hi)


def _verify(batch, drafts_lo, drafts_hi, lengths, vocab=VOCAB, with_probs=True):
    return dict(kind="verify", batch=batch, drafts_lo=drafts_lo, drafts_hi=drafts_hi,
                lengths=lengths, vocab=vocab, with_probs=with_probs)


def listed():
    return [
        # The table of a model that rotates half of each head, made at load time.
        dict(name="table_part", **_table(4096, 64, "linear", 4.0)),
        # The table for a context stretched to 131,072 positions.
        dict(name="table_long", **_table(131_072, 128, "yarn", 4.0)),
        # A decode step of a few requests: launch latency.
        dict(name="append_decode_b7", **_append(7, 16, 8)),
        # A chunk of an odd number of new tokens, interleaved pairs over half of the head.
        dict(name="append_chunk_part", **_append(2047, 32, 8, rotary=64, interleaved=True,
                                                 dtype="fp16")),
        # A full prefill batch.
        dict(name="append_prefill", **_append(16_384, 32, 8)),
        # Four samples of one prompt on the smallest model, just begun.
        dict(name="prefix_b4", **_prefix(4, 1500, 16, 8, 1, 1, 60)),
        # A batch on one system prompt, ragged replies.
        dict(name="prefix_b32", **_prefix(32, 4001, 32, 8, 2, 16, 700)),
        # The target's pass over drafted tokens: several query tokens a request.
        dict(name="prefix_drafts_b64", **_prefix(64, 6000, 32, 4, 3, 8, 400, 2, 6)),
        # A full batch behind a long shared document.
        dict(name="prefix_b256", **_prefix(256, 16_384, 32, 8, 4, 32, 1024)),
        # One user's drafts.
        dict(name="verify_b1", **_verify(1, 4, 4, 1)),
        # A busy server's step, ragged draft counts.
        dict(name="verify_b48", **_verify(48, 0, 5, 2)),
        # A full batch whose drafts come from n-gram lookup, without probabilities.
        dict(name="verify_b256_lookup", **_verify(256, 2, 4, 3, with_probs=False)),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("rope_table", "rope_append", "rope_append", "prefix", "prefix", "prefix",
                       "verify", "verify"))
    seed = rng.randrange(1 << 20)
    hq, hkv = rng.choice(((16, 8), (32, 8), (32, 4)))
    if kind == "rope_table":
        return _table(_log_int(rng, 512, 131_072), rng.choice((32, 64, 96, 128)),
                      rng.choice(("none", "linear", "ntk", "yarn", "bands")),
                      float(rng.choice((2, 4, 8, 16))))
    if kind == "rope_append":
        return _append(_log_int(rng, 1, 16_384), hq, hkv, rotary=rng.choice((32, 64, 96, 128, 128)),
                       interleaved=rng.random() < 0.5, dtype=rng.choice(("bf16", "fp16")),
                       max_pos=rng.choice((8192, 40_960)))
    if kind == "prefix":
        batch = _log_int(rng, 1, 256)
        qo_hi = rng.choice((1, 1, rng.randint(2, 8)))
        if batch * qo_hi > 512:
            qo_hi = 1
        hi = max(qo_hi, _log_int(rng, 8, 1024))
        return _prefix(batch, _log_int(rng, 100, 16_000), hq, hkv, seed,
                       max(qo_hi, int(hi * rng.uniform(0.05, 1.0))), hi,
                       rng.randint(1, qo_hi), qo_hi)
    batch = _log_int(rng, 1, 256)
    hi = rng.randint(1, 8 if batch <= 96 else 4)
    return _verify(batch, rng.randint(0, hi), hi, seed,
                   vocab=rng.choice((VOCAB, VOCAB, 32_001, 50_257)),
                   with_probs=rng.random() < 0.7)


# ------------------------------------------------------------------ lengths

def _qo_and_suffix(case):
    """(query tokens, suffix tokens) of each request; a suffix holds its query tokens."""
    rng = np.random.default_rng(case["lengths"])
    qo = rng.integers(case["qo_lo"], case["qo_hi"] + 1, size=case["batch"])
    suffix = rng.integers(case["lo"], case["hi"] + 1, size=case["batch"])
    return qo.astype(np.int64), np.maximum(suffix, qo).astype(np.int64)


def _drafts(case):
    rng = np.random.default_rng(case["lengths"])
    return rng.integers(case["drafts_lo"], case["drafts_hi"] + 1,
                        size=case["batch"]).astype(np.int64)


def _indptr(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


# ------------------------------------------------------------------ frequencies

def _frequencies(rotary, base, scaling, factor, original):
    """(frequency of each pair, factor of cos and sin) in 64 bits."""
    i = torch.arange(rotary // 2, dtype=torch.float64, device=DEV)
    f = base ** (-2.0 * i / rotary)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "ntk":
        return (base * factor ** (rotary / (rotary - 2.0))) ** (-2.0 * i / rotary), 1.0
    if scaling == "yarn":
        at = [rotary * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))
              for turns in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rotary - 1)
        keep = 1 - ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return f / factor * (1 - keep) + f * keep, 0.1 * math.log(factor) + 1
    if scaling == "bands":
        turns = original * f / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f / factor * (1 - keep) + f * keep, 1.0
    return f, 1.0


# ------------------------------------------------------------------ prepare

def _prepare_table(case, g):
    # Another seed is another base: the table has no other input.
    base = BASE * (1 + 0.01 * float(torch.rand((), generator=g, device=DEV)))
    return dict(base=base, original=max(case["positions"] // 4, 64))


def _prepare_append(case, g):
    T, hq, hkv, dt = case["tokens"], case["hq"], case["hkv"], DTYPES[case["dtype"]]
    slots = (T + 40) // PAGE * PAGE + 512
    qkv = torch.randn((T, (hq + 2 * hkv) * D), generator=g, device=DEV).to(dt)
    q, k, v = qkv.split([hq * D, hkv * D, hkv * D], dim=1)
    f, _ = _frequencies(case["rotary"], BASE, "none", 1.0, 1)
    angle = torch.arange(case["max_pos"], dtype=torch.float64, device=DEV)[:, None] * f
    start = int(torch.randint(0, max(1, case["max_pos"] - T), (), generator=g, device=DEV))
    return dict(q=q.view(T, hq, D), k=k.view(T, hkv, D), v=v.view(T, hkv, D),
                k_cache=torch.randn((slots, hkv, D), generator=g, device=DEV).to(dt),
                v_cache=torch.randn((slots, hkv, D), generator=g, device=DEV).to(dt),
                cos=angle.cos().float(), sin=angle.sin().float(),
                positions=(start + torch.arange(T, device=DEV) % (case["max_pos"] - start)).int(),
                out_loc=torch.randperm(slots, generator=g, device=DEV)[:T].int())


def _prepare_prefix(case, g):
    qo, suffix = _qo_and_suffix(case)
    T, hq, hkv, P = int(qo.sum()), case["hq"], case["hkv"], case["prefix"]
    pages = np.concatenate([[-(-P // PAGE)], -(-suffix // PAGE)])
    order = torch.randperm(int(pages.sum()) + 1, generator=g, device=DEV).cpu().numpy()
    ends = np.cumsum(pages)
    rows = []
    for n, end, count in zip([P, *suffix], ends, pages):
        slots = order[end - count:end, None] * PAGE + np.arange(PAGE)[None, :]
        rows.append(slots.reshape(-1)[:n])
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)
    slots = (int(pages.sum()) + 1) * PAGE
    make = lambda *shape: torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16)
    state = dict(q=make(T, hq, D), k_cache=make(slots, hkv, D), v_cache=make(slots, hkv, D),
                 prefix_indices=dev(rows[0]), indices=dev(np.concatenate(rows[1:])),
                 kv_indptr=dev(_indptr(suffix)), qo_indptr=dev(_indptr(qo)),
                 longest=int(suffix.max()), max_qo=int(qo.max()), scale=D ** -0.5)
    if own:  # the plan and its workspace, which a program keeps from step to step
        state["attention"] = _backend().PrefixAttention(P, case["batch"], T, int(qo.max()), hq,
                                                        hkv, D)
    return state


def _prepare_verify(case, g):
    n = _drafts(case)
    B, total, V = case["batch"], int(n.sum()), case["vocab"]
    indptr = _indptr(n)
    rows = np.concatenate([np.arange(a, b) for a, b in zip(indptr[:-1] + np.arange(B),
                                                           indptr[1:] + np.arange(B))]
                          or [np.zeros(0)]).astype(np.int64)
    logits = 4 * torch.randn((total + B, V), generator=g, device=DEV)
    rows = torch.from_numpy(rows).to(DEV)
    # The draft model agrees with the target up to noise; its tokens are drawn from its own
    # probabilities.
    draft = torch.softmax(logits[rows] + 0.7 * torch.randn((total, V), generator=g, device=DEV), -1)
    noise = torch.rand((total, V), generator=g, device=DEV).clamp_min_(1e-20).log_().neg_()
    tokens = (draft / noise).argmax(-1).int() if total else torch.zeros(0, dtype=torch.int32,
                                                                         device=DEV)
    return dict(target=torch.softmax(logits, -1), draft=draft if case["with_probs"] else None,
                tokens=tokens, indptr=torch.from_numpy(indptr).to(DEV),
                accept_u=torch.rand(total, generator=g, device=DEV),
                sample_u=torch.rand(B, generator=g, device=DEV), most=int(n.max()))


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    make = {"rope_table": _prepare_table, "rope_append": _prepare_append,
            "prefix": _prepare_prefix, "verify": _prepare_verify}
    return dict(make[case["kind"]](case, g), case=case)


# ------------------------------------------------------------------ plain forms

def _plain_table(s):
    c = s["case"]
    f, m = _frequencies(c["rotary"], s["base"], c["scaling"], c["factor"], s["original"])
    angle = torch.arange(c["positions"], dtype=torch.float64, device=DEV)[:, None] * f
    return dict(cos=(angle.cos() * m).float(), sin=(angle.sin() * m).float())


def _rotate(x, cos, sin, rotary, interleaved):
    """x [T, heads, D] in 32 bits, its first `rotary` elements rotated by cos/sin [T, rotary / 2]."""
    x, c, s = x.float(), cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, x[..., rotary:]], -1)


def _plain_append(s):
    c, at = s["case"], s["positions"].long()
    cos, sin, slots = s["cos"][at], s["sin"][at], s["out_loc"].long()
    q = _rotate(s["q"], cos, sin, c["rotary"], c["interleaved"]).to(s["q"].dtype)
    s["k_cache"][slots] = _rotate(s["k"], cos, sin, c["rotary"], c["interleaved"]).to(s["k"].dtype)
    s["v_cache"][slots] = s["v"]
    return dict(q=q, k_cache=s["k_cache"], v_cache=s["v_cache"])


def _plain_prefix(s):
    c = s["case"]
    B, hq, hkv, P, Q, S = c["batch"], c["hq"], c["hkv"], c["prefix"], s["max_qo"], s["longest"]
    G = hq // hkv
    qo0, kv0 = s["qo_indptr"].long(), s["kv_indptr"].long()
    qo, kv = qo0[1:] - qo0[:-1], kv0[1:] - kv0[:-1]
    q = s["q"].float() * s["scale"]
    T = q.shape[0]
    # Every row over the prefix: [Hkv, T G, P].
    kp = s["k_cache"][s["prefix_indices"].long()].float().permute(1, 2, 0).contiguous()
    vp = s["v_cache"][s["prefix_indices"].long()].float().permute(1, 0, 2).contiguous()
    rows = q.view(T, hkv, G, D).permute(1, 0, 2, 3).reshape(hkv, T * G, D)
    score_p = rows @ kp
    # Every request's rows over its own suffix, both padded: [B, Hkv, Q G, S].
    tok = torch.arange(S, device=DEV)
    own_slots = s["indices"].long()[(kv0[:-1, None] + tok).clamp_max(len(s["indices"]) - 1)]
    ks = s["k_cache"][own_slots].float().permute(0, 2, 3, 1).contiguous()
    vs = s["v_cache"][own_slots].float().permute(0, 2, 1, 3).contiguous()
    i = torch.arange(Q, device=DEV)
    at = (qo0[:-1, None] + i).clamp_max(T - 1)
    padded = q[at].view(B, Q, hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, hkv, Q * G, D)
    sees = tok[None, None] <= (i[None, :] + (kv - qo)[:, None])[:, :, None]  # [B, Q, S]
    sees = sees & (tok < kv[:, None])[:, None]
    score_s = (padded @ ks).view(B, hkv, Q, G, S).masked_fill(~sees[:, None, :, None], -math.inf)
    # Back to one row per token, in [Hkv, T G] order.
    real = (i < qo[:, None]).reshape(-1)
    place = torch.nonzero(real)[:, 0]
    score_s = score_s.permute(1, 0, 2, 3, 4).reshape(hkv, B * Q, G, S)[:, place].reshape(hkv, T * G, S)
    top = torch.maximum(score_p.amax(-1), score_s.amax(-1))[..., None]
    wp, ws = (score_p - top).exp(), (score_s - top).exp()
    total = wp.sum(-1, keepdim=True) + ws.sum(-1, keepdim=True)
    back = torch.zeros((hkv, B * Q, G, S), device=DEV)
    back[:, place] = ws.view(hkv, T, G, S)
    from_s = back.view(hkv, B, Q * G, S).permute(1, 0, 2, 3).contiguous() @ vs
    from_s = from_s.permute(1, 0, 2, 3).reshape(hkv, B * Q, G, D)[:, place].reshape(hkv, T * G, D)
    o = (wp @ vp + from_s) / total
    return o.view(hkv, T, G, D).permute(1, 0, 2, 3).reshape(T, hq, D).to(s["q"].dtype)


def _plain_verify(s):
    d0 = s["indptr"].long()
    B, V = len(d0) - 1, s["target"].shape[1]
    n, r = d0[1:] - d0[:-1], torch.arange(B, device=DEV)
    total = len(s["tokens"])
    request = torch.repeat_interleave(r, n, output_size=total)
    draft_at = torch.arange(total, device=DEV)
    x = s["tokens"].long()
    p = s["target"][draft_at + request, x].double()
    q = 1.0 if s["draft"] is None else s["draft"][draft_at, x].double()
    ok = s["accept_u"].double() * q < p
    # Accepted: drafts before the first rejected one.
    place = draft_at - d0[request]
    accepted = n.scatter_reduce(0, request, torch.where(ok, n[request], place), "amin")
    rest = s["target"][d0[:-1] + r + accepted].double()
    if total:
        rejected = (accepted < n)[:, None]
        at = (d0[:-1] + accepted).clamp_max(total - 1)
        if s["draft"] is None:
            less = torch.zeros_like(rest).scatter_(1, x[at][:, None], math.inf)
        else:
            less = s["draft"][at].double()
        left = (rest - less).clamp_min(0)
        rest = torch.where(rejected & (left.sum(-1, keepdim=True) > 0), left, rest)
    run_sum = rest.cumsum(-1)
    past = run_sum > s["sample_u"].double()[:, None] * rest.sum(-1, keepdim=True)
    token = torch.where(past.any(-1), past.int().argmax(-1),
                        V - 1 - (rest > 0).flip(-1).int().argmax(-1))
    out = torch.full((total + B,), -1, dtype=torch.int32, device=DEV)
    kept = torch.where(place < accepted[request], s["tokens"], torch.full_like(s["tokens"], -1))
    out[draft_at + request] = kept
    out[d0[:-1] + r + accepted] = token.int()
    return dict(tokens=out, accepted=accepted.int())


# ------------------------------------------------------------------ the framework's operators

def _own_table(s):
    c = s["case"]
    be = _backend()
    scaling = be.RopeScaling(kind=c["scaling"], factor=c["factor"],
                             original_max_position=s["original"])
    cos, sin = be.rope_scaled_cache(c["positions"], c["rotary"], s["base"], scaling)
    return dict(cos=cos, sin=sin)


def _own_append(s):
    c = s["case"]
    q = _backend().rope_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["cos"],
                               s["sin"], s["positions"], s["out_loc"], c["interleaved"])
    return dict(q=q, k_cache=s["k_cache"], v_cache=s["v_cache"])


def _own_prefix(s):
    return s["attention"].forward(s["q"], s["k_cache"], s["v_cache"], s["prefix_indices"],
                                  s["indices"], s["kv_indptr"], s["qo_indptr"])


def _own_verify(s):
    tokens, accepted = _backend().verify_drafts(s["target"], s["draft"], s["tokens"], s["indptr"],
                                                s["accept_u"], s["sample_u"])
    return dict(tokens=tokens, accepted=accepted)


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rope_table": _own_table, "rope_append": _own_append, "prefix": _own_prefix,
                "verify": _own_verify}[kind](state)
    return {"rope_table": _plain_table, "rope_append": _plain_append, "prefix": _plain_prefix,
            "verify": _plain_verify}[kind](state)


# ------------------------------------------------------------------ work

def work(case):
    kind = case["kind"]
    if kind == "rope_table":
        n = case["positions"] * case["rotary"] // 2
        return {"bytes": 8 * n, "flops": 40 * n}
    if kind == "rope_append":
        rows = case["tokens"] * (case["hq"] + 2 * case["hkv"])
        table = min(case["tokens"], case["max_pos"]) * case["rotary"] * 4
        return {"bytes": rows * D * 4 + table + 8 * case["tokens"],
                "flops": 3 * case["tokens"] * (case["hq"] + case["hkv"]) * case["rotary"]}
    if kind == "prefix":
        qo, suffix = _qo_and_suffix(case)
        T = int(qo.sum())
        kv = case["prefix"] + int(suffix.sum())
        # Query i of a request sees all but the last qo - 1 - i tokens of its suffix.
        seen = int((qo * (case["prefix"] + suffix) - qo * (qo - 1) // 2).sum())
        return {"bytes": kv * (case["hkv"] * D * 4 + 4) + T * case["hq"] * D * 4,
                "flops": 4 * D * case["hq"] * seen}
    n = _drafts(case)
    # A target row and, where a request has drafts with probabilities, a draft row.
    rows = case["batch"] + (int((n > 0).sum()) if case["with_probs"] else 0)
    return {"bytes": 4 * rows * case["vocab"] + 16 * int(n.sum()) + 20 * case["batch"],
            "flops": 3 * rows * case["vocab"]}


# ------------------------------------------------------------------ exact

def _exact_table(case, s):
    i = np.arange(case["rotary"] // 2, dtype=np.float64)
    R, L, k = case["rotary"], s["original"], case["factor"]
    f = np.power(s["base"], -2 * i / R)
    m = 1.0
    if case["scaling"] == "linear":
        f = f / k
    elif case["scaling"] == "ntk":
        f = f * np.power(k, -2 * i / (R - 2))
    elif case["scaling"] == "yarn":
        lo, hi = (R / 2 * math.log(L / (2 * math.pi * t)) / math.log(s["base"]) for t in (32, 1))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), R - 1)
        w = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        f, m = f * (w / k + 1 - w), 1 + math.log(k) / 10
    elif case["scaling"] == "bands":
        w = np.clip((L * f / (2 * math.pi) - 1) / 3, 0, 1)
        f = f * ((1 - w) / k + w)
    turn = torch.outer(torch.arange(case["positions"], dtype=torch.float64, device=DEV),
                       torch.from_numpy(f).to(DEV))
    return dict(cos=m * torch.cos(turn), sin=m * torch.sin(turn))


def _exact_append(case, s):
    R = case["rotary"]
    pair = torch.arange(R // 2, device=DEV)
    first, second = (2 * pair, 2 * pair + 1) if case["interleaved"] else (pair, pair + R // 2)
    z = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None]

    def turned(x):
        x = x.double().clone()
        y = torch.complex(x[..., first], x[..., second]) * z
        x[..., first], x[..., second] = y.real, y.imag
        return x

    kc, vc, at = s["k_cache"].double(), s["v_cache"].double(), s["out_loc"].long()
    kc[at], vc[at] = turned(s["k"]), s["v"].double()
    return dict(q=turned(s["q"]), k_cache=kc, v_cache=vc)


def _exact_prefix(case, s):
    qo, suffix = _qo_and_suffix(case)
    q0, k0 = _indptr(qo), _indptr(suffix)
    hq, hkv = case["hq"], case["hkv"]
    G = hq // hkv
    o = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    for r in range(case["batch"]):
        slots = torch.cat([s["prefix_indices"], s["indices"][k0[r]:k0[r + 1]]]).long()
        k = s["k_cache"][slots].double().permute(1, 2, 0).contiguous()
        v = s["v_cache"][slots].double().permute(1, 0, 2).contiguous()
        for i in range(int(qo[r])):
            sees = len(slots) - int(qo[r]) + i + 1
            rows = s["q"][q0[r] + i].double().view(hkv, G, D)
            w = torch.softmax((rows @ k[..., :sees].contiguous()) / math.sqrt(D), -1)
            o[q0[r] + i] = (w @ v[:, :sees].contiguous()).reshape(hq, D)
    return o


def _exact_verify(case, s):
    ends = s["indptr"].cpu().numpy()
    x, u, last = (s[k].cpu().numpy() for k in ("tokens", "accept_u", "sample_u"))
    out = np.full(len(x) + case["batch"], -1, dtype=np.int32)
    accepted = np.zeros(case["batch"], dtype=np.int32)
    for r in range(case["batch"]):
        a, b = int(ends[r]), int(ends[r + 1])
        at, weights = a, None
        while at < b:
            p = s["target"][at + r].double().cpu().numpy()
            q = np.zeros_like(p)
            if s["draft"] is None:
                q[x[at]] = 1.0
            else:
                q = s["draft"][at].double().cpu().numpy()
            if float(u[at]) * q[x[at]] >= p[x[at]]:
                weights = np.maximum(p - q, 0)
                weights = weights if weights.sum() > 0 else p
                break
            out[at + r] = x[at]
            at += 1
        if weights is None:
            weights = s["target"][b + r].double().cpu().numpy()
        accepted[r] = at - a
        ran = np.cumsum(weights)
        out[at + r] = min(int(np.searchsorted(ran, float(last[r]) * ran[-1], side="right")),
                          int(np.nonzero(weights)[0][-1]))
    return dict(tokens=torch.from_numpy(out), accepted=torch.from_numpy(accepted))


def exact(case, seed):
    state = prepare(case, seed)
    return {"rope_table": _exact_table, "rope_append": _exact_append, "prefix": _exact_prefix,
            "verify": _exact_verify}[case["kind"]](case, state)
