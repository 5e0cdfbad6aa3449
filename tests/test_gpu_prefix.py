"""GPU tests (marked gpu) of attention behind a shared prefix against its 64-bit form.

Bound of a row: its output is rounded to bf16 (half a step, 2^-8 of it), each
weight P to bf16 before the product with V (2^-8 of sum_j p_j |v_j|), and scores are
fp32 sums of 128 products: 2^-16 of sum |q k| scale, about 13 for unit normals, which
moves weights by less than 2^-12. Together 2^-8 |o| + (2^-8 + 2^-11) sum p |v| + 1e-6."""
import math

import numpy as np
import pytest
import torch

import operator_refs as refs
from conftest import capi, pkg

pytestmark = pytest.mark.gpu


def make(dev, P, kv, qo, hq, hkv, seed, spare=3, kv_first=0, qo_first=0, tail=0):
    """Inputs: slots in random order, `spare` unlisted ones full of NaN; the requests'
    offsets start at kv_first / qo_first, `tail` rows follow the last request's."""
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    kv, qo = np.asarray(kv, np.int64), np.asarray(qo, np.int64)
    n = P + int(kv.sum())
    slots = n + spare
    order = torch.randperm(slots, generator=g, device=dev).int()
    rand = lambda *s: torch.randn(s, generator=g, device=dev).to(torch.bfloat16)
    kc, vc = rand(slots, hkv, 128), rand(slots, hkv, 128)
    kc[order[n:].long()] = float("nan")
    vc[order[n:].long()] = float("nan")
    ip = lambda x, first: torch.from_numpy((first + np.concatenate([[0], np.cumsum(x)])).astype(np.int32)).to(dev)
    lead = torch.full((kv_first,), int(order[-1]) if spare else 0, dtype=torch.int32, device=dev)
    T = qo_first + int(qo.sum()) + tail
    return dict(q=rand(T, hq, 128), kc=kc, vc=vc, pidx=order[:P].contiguous(),
                idx=torch.cat([lead, order[P:n]]).contiguous(), kvp=ip(kv, kv_first),
                qop=ip(qo, qo_first), P=P, B=len(kv), T=T, max_qo=max(1, int(qo.max(initial=0))),
                hq=hq, hkv=hkv, scale=128 ** -0.5)


def plan_of(x, **kw):
    return capi.prefix_plan(kw.get("P", x["P"]), kw.get("B", x["B"]), kw.get("T", x["T"]),
                            kw.get("max_qo", x["max_qo"]), x["hq"], x["hkv"], 128)


def run(x, plan=None, ws=None, o=None, q=None):
    plan = plan_of(x) if plan is None else plan
    if ws is None:
        ws = capi.prefix_workspace(plan, x["q"].device)
        ws.view(torch.uint8).fill_(0xFF)  # NaN everywhere: nothing is read before it is written
    o = torch.full_like(x["q"], 7.0) if o is None else o
    capi.prefix_attention(plan, x["q"] if q is None else q, x["kc"], x["vc"], x["pidx"], x["idx"],
                          x["kvp"], x["qop"], o, ws, x["scale"])
    return o


def check(x, o, skip=()):
    want = refs.prefix_rows(x["q"], x["kc"], x["vc"], x["pidx"], x["idx"], x["kvp"].cpu(),
                            x["qop"].cpu(), x["scale"])
    for t in range(x["T"]):
        if t in skip:
            continue
        if t not in want:
            assert (o[t] == 7.0).all(), f"row {t} belongs to no request"
            continue
        ref, size = want[t]
        err = (o[t].double() - ref).abs()
        bound = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -11) * size + 1e-6
        assert (err <= bound).all(), f"row {t}: {float((err - bound).max())} past the bound"


HEADS = [(16, 8), (32, 8), (32, 4), (1, 1), (15, 3), (16, 1), (64, 1), (26, 13), (16, 16), (12, 12)]


@pytest.mark.parametrize("hq,hkv", HEADS)
@pytest.mark.parametrize("P,kv,qo", [
    (1, [1], [1]),
    (300, [5, 70, 1, 33], [1, 1, 1, 1]),
    (129, [64, 7, 130], [2, 7, 5]),
    (1000, [17] * 9, [1] * 9),
])
def test_heads(dev, hq, hkv, P, kv, qo):
    x = make(dev, P, kv, qo, hq, hkv, P + hq)
    check(x, run(x))


@pytest.mark.parametrize("P,kv,qo", [
    (0, [5, 70], [1, 1]),                       # no prefix
    (0, [0, 3], [1, 2]),                        # a row that sees nothing
    (40, [0, 0, 0], [1, 1, 1]),                 # only the prefix
    (40, [0, 9, 0], [0, 0, 0]),                 # no rows at all
    (63, [3, 0, 65, 0, 1], [1, 0, 3, 1, 1]),    # empty requests between others
    (5, [1, 0, 2], [4, 7, 9]),                  # more query tokens than own ones: rows that see a part
    (3, [0, 1], [6, 5]),                        # ... of the prefix, or nothing
    (2000, [1], [1]),
    (15, [2049], [1]),
    (16, [4000, 3, 2], [1, 1, 1]),              # one long request over many units
    (17, [200, 900], [64, 33]),                 # the most query tokens
    (4097, [30] * 40, [1] * 40),                # several tiles of rows
    (777, [12] * 70, [3] * 70),
])
@pytest.mark.parametrize("hq,hkv", [(32, 8), (16, 2)])
def test_lengths(dev, P, kv, qo, hq, hkv):
    x = make(dev, P, kv, qo, hq, hkv, 11)
    check(x, run(x))


def test_many_requests(dev):
    """More requests than a wave has lanes, and than units."""
    rng = np.random.default_rng(3)
    kv = rng.integers(0, 4, 700)
    x = make(dev, 50, kv, np.minimum(1, kv), 4, 2, 12)
    check(x, run(x))


@pytest.mark.parametrize("hq,hkv,qo", [(8, 8, 1), (24, 4, 4)])
def test_many_requests_of_all_lengths(dev, hq, hkv, qo):
    """Units that begin and end anywhere in a list of 200 requests, empty ones among them."""
    rng = np.random.default_rng(qo)
    kv = rng.integers(0, 300, 200) * (rng.random(200) > 0.3)
    n = np.minimum(rng.integers(0, qo + 1, 200), kv)
    x = make(dev, 130, kv, n, hq, hkv, 22)
    check(x, run(x))


def test_offsets_past_zero_and_rows_behind(dev):
    """A part of a larger batch: offsets that start past 0, rows before and behind that
    belong to no request stay as they were."""
    x = make(dev, 90, [4, 50, 9], [1, 3, 2], 16, 8, 13, kv_first=21, qo_first=5, tail=4)
    check(x, run(x))


def test_a_plan_for_more_and_the_backend(dev):
    x = make(dev, 500, [4, 50, 9], [1, 3, 2], 32, 8, 14)
    big = plan_of(x, B=40, T=200, max_qo=16)
    check(x, run(x, big))
    b = pkg.backend.load().PrefixAttention(500, 3, x["T"], 3, 32, 8, 128)
    o = b.forward(x["q"], x["kc"], x["vc"], x["pidx"], x["idx"], x["kvp"], x["qop"])
    check(x, o)
    assert torch.equal(o, run(x))


@pytest.mark.parametrize("scale", [0.02, 0.15])
def test_other_scales(dev, scale):
    x = make(dev, 300, [20, 90, 1], [1, 2, 1], 16, 4, 24)
    x["scale"] = scale
    check(x, run(x))


def test_equals_decode_and_prefill_of_the_joined_sequences(dev):
    """Within both sides' bounds: the paged decode kernel over prefix + own tokens."""
    x = make(dev, 400, [20, 90, 1, 300], [1, 1, 1, 1], 32, 8, 15)
    parts = [torch.cat([x["pidx"], x["idx"][int(a):int(b)]]) for a, b in zip(x["kvp"][:-1], x["kvp"][1:])]
    ip = np.concatenate([[0], np.cumsum([len(p) for p in parts])]).astype(np.int32)
    plan = capi.decode_plan(ip, 32, 8, 128)
    o = torch.empty_like(x["q"])
    capi.paged_decode(plan, x["q"], x["kc"], x["vc"], torch.cat(parts), torch.from_numpy(ip).to(dev), o,
                      capi.decode_workspace(plan, dev))
    check(x, o)
    check(x, run(x))


def test_values_behind_a_row_never_reach_it(dev):
    """NaN and infinities in K and V of a request's later query tokens: earlier rows of
    the request and every other request are as without them."""
    for what in ("nan k", "nan v", "inf v", "-inf k"):
        x = make(dev, 200, [40, 25, 60], [4, 3, 1], 16, 8, 16)
        base = run(x)
        kvp = x["kvp"].cpu()
        bad = x["idx"][int(kvp[1]) - 1].long()  # request 0's last token: only its last row sees it
        cache = x["kc"] if what.endswith("k") else x["vc"]
        cache[bad] = float(what.split()[0])
        o = run(x)
        check(x, o, skip=(3,))
        seen = [t for t in range(x["T"]) if t != 3]
        if what.endswith("k"):
            assert torch.equal(o[seen], base[seen])
        if "nan" in what:
            assert o[3].isnan().all()
    # A visible one does reach: NaN in the prefix reaches every row.
    x["vc"][x["pidx"][17].long()] = float("nan")
    assert run(x).isnan().all()


def test_invalid_requests_get_nan_rows(dev):
    x = make(dev, 64, [9, 9, 9], [2, 2, 2], 16, 8, 17)
    good = run(x)
    x["qop"] = torch.tensor([0, 2, 4, 6], device=dev, dtype=torch.int32)
    # kv offsets that decrease: that request's rows are NaN.
    x["kvp"] = torch.tensor([0, 9, 5, 27], device=dev, dtype=torch.int32)
    o = run(x)
    assert o[2:4].isnan().all() and torch.equal(o[:2], good[:2])
    # More query tokens than the plan's.
    y = make(dev, 64, [9, 9], [2, 5], 16, 8, 18)
    o = run(y, plan_of(y, max_qo=4))
    assert o[2:].isnan().all() and not o[:2].isnan().any()
    # q offsets that decrease: rows 4 to 9 belong to no request (the third one, whose own
    # offsets hold, is the one that their place in the list points to).
    z = make(dev, 64, [40, 9, 9, 9], [4, 2, 2, 4], 16, 8, 20)
    z["qop"] = torch.tensor([0, 10, 2, 4, 12], device=dev, dtype=torch.int32)
    o = run(z, plan_of(z, max_qo=8))
    assert o[4:10].isnan().all()


def test_strided_rows_far_slots_and_a_side_stream(dev):
    """q a view of qkv rows, o with a padded stride; element offsets in the pool past
    2^32; all on a side stream."""
    hq, hkv = 16, 8
    x = make(dev, 70, [9, 30], [1, 2], hq, hkv, 19)
    slots = (1 << 32) // (hkv * 128) + 200
    kc = torch.zeros((slots, hkv, 128), device=dev, dtype=torch.bfloat16)
    vc = torch.zeros_like(kc)
    shift = slots - x["kc"].shape[0]
    kc[shift:], vc[shift:] = x["kc"], x["vc"]
    qkv = torch.randn((3, (hq + 2 * hkv) * 128), device=dev).to(torch.bfloat16)
    qkv[:, :hq * 128] = x["q"].reshape(3, -1)
    wide = torch.full((3, hq + 3, 136), 7.0, device=dev, dtype=torch.bfloat16)
    plain = run(x)
    y = {**x, "kc": kc, "vc": vc, "pidx": x["pidx"] + shift, "idx": x["idx"] + shift}
    plan = plan_of(y)
    ws = capi.prefix_workspace(plan, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(y, plan, ws, o=wide[:, :hq, :128], q=qkv[:, :hq * 128].view(3, hq, 128))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(wide[:, :hq, :128], plain)
    assert (wide[:, hq:] == 7).all() and (wide[..., 128:] == 7).all()


def test_captured_steps_share_a_workspace(dev):
    """Two graphs captured on one plan and workspace, replayed in turn while the
    requests grow, with eager calls of another batch in between."""
    hq, hkv, P, B = 32, 8, 333, 6
    x = make(dev, P, [200] * B, [1] * B, hq, hkv, 20)
    full = x["idx"].clone()
    plan = plan_of(x)
    ws = capi.prefix_workspace(plan, dev)
    outs = [torch.empty_like(x["q"]) for _ in range(2)]
    qs = [x["q"], torch.randn_like(x["q"])]
    graphs = []
    run(x, plan, ws)
    torch.cuda.synchronize()
    for o, q in zip(outs, qs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(x, plan, ws, o=o, q=q)
        graphs.append(g)
    other = make(dev, 50, [3, 4], [2, 1], 16, 8, 21)
    for step in (1, 2, 60, 199, 200):
        lens = np.array([step, 1 + step // 2, step, 7, 200, 1 + step // 3])
        ip = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        x["kvp"].copy_(torch.from_numpy(ip))
        new = torch.cat([full[200 * r:200 * r + n] for r, n in enumerate(lens)])
        x["idx"][:len(new)].copy_(new)
        for g, o, q in zip(graphs, outs, qs):
            g.replay()
            want = run({**x, "q": q})
            assert torch.equal(o, want)
            check(other, run(other))
        check(x, outs[0])


@pytest.mark.parametrize("B,qo,hq,hkv,P,own", [
    (9, 1, 32, 8, 65, 3),        # 36 rows of a kv head: a wave's and four more
    (33, 1, 32, 8, 640, 1),      # one token more than a row tile holds
    (65, 1, 32, 8, 63, 20),
    (257, 1, 16, 4, 1025, 2),
    (100, 8, 16, 2, 129, 9),     # 6,400 rows a kv head
    (300, 4, 64, 1, 130, 4),     # 76,800: more row tiles than workgroups
    (40, 1, 600, 600, 70, 2),    # more kv heads than workgroups for the prefix
    (45, 1, 39, 13, 200, 5),
])
def test_many_rows(dev, B, qo, hq, hkv, P, own):
    x = make(dev, P, [own + r % 3 for r in range(B)], [qo - r % qo for r in range(B)], hq, hkv, B)
    check(x, run(x))
    check(x, run(x, plan_of(x, B=B + 7, T=x["T"] + 300, max_qo=qo + 3)))  # a plan for more of everything


@pytest.mark.parametrize("seed", range(12))
def test_drawn_shapes(dev, seed):
    rng = np.random.default_rng(seed)
    hq, hkv = [(16, 8), (32, 8), (32, 4), (8, 8), (24, 3), (20, 5)][seed % 6]
    B = int(rng.integers(1, 60))
    qo = rng.integers(0, int(rng.choice([2, 5, 12])), B)
    kv = rng.integers(0, int(rng.choice([4, 80, 700])), B) + qo
    x = make(dev, int(rng.integers(0, 3000)), kv, qo, hq, hkv, 500 + seed)
    check(x, run(x))
