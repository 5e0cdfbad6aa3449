"""GPU tests (marked gpu) of the verification of drafted tokens against its 64-bit
form: whole numbers, so equal."""
import ctypes

import numpy as np
import pytest
import torch

import operator_refs as refs
from conftest import capi, pkg

pytestmark = pytest.mark.gpu


def batch(n, vocab, seed, sharp=3.0, noise=0.7, with_probs=True):
    rng = np.random.default_rng(seed)
    n = np.asarray(n, np.int64)
    B, total = len(n), int(n.sum())
    indptr = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    soft = lambda x: (lambda e: (e / e.sum(-1, keepdims=True)).astype(np.float32))(
        np.exp(x - x.max(-1, keepdims=True)))
    logits = sharp * rng.standard_normal((total + B, vocab))
    rows = np.array([i + r for r in range(B) for i in range(indptr[r], indptr[r + 1])], np.int64)
    draft = soft(logits[rows] + noise * rng.standard_normal((total, vocab))) if total else \
        np.zeros((0, vocab), np.float32)
    tokens = np.array([np.searchsorted(np.cumsum(d), rng.random() * d.sum()) for d in draft],
                      np.int32).clip(0, vocab - 1).reshape(-1)
    return dict(target=soft(logits), draft=draft if with_probs else None, tokens=tokens,
                indptr=indptr, accept=rng.random(total, np.float32), sample=rng.random(B, np.float32))


def run(x, dev, route="capi", target=None, draft=None):
    t = {k: None if v is None else torch.from_numpy(np.ascontiguousarray(v)).to(dev)
         for k, v in x.items()}
    if target is not None:
        t["target"] = target
    if draft is not None:
        t["draft"] = draft
    fn = capi.verify_drafts if route == "capi" else pkg.backend.load().verify_drafts
    tokens, accepted = fn(t["target"], t["draft"], t["tokens"], t["indptr"], t["accept"], t["sample"])
    return tokens.cpu().tolist(), accepted.cpu().tolist()


def check(x, dev, **kw):
    want = refs.verify(x["target"], x["draft"], x["tokens"], x["indptr"], x["accept"], x["sample"])
    assert run(x, dev, **kw) == want
    return want


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 1000, 1023, 4096, 4097, 32001, 151936])
@pytest.mark.parametrize("n", [[0], [1], [4], [3, 0, 5, 1], [2] * 17])
@pytest.mark.parametrize("with_probs", [True, False])
def test_verify(dev, vocab, n, with_probs):
    if vocab > 40000 and len(n) > 4:
        n = n[:4]
    for seed in range(3):
        x = batch(n, vocab, seed * 7 + vocab, with_probs=with_probs)
        check(x, dev)
        check(x, dev, route="backend")


def test_all_accepted_none_accepted_and_long_drafts(dev):
    """More drafts than a wave has lanes; acceptance forced both ways by the uniforms."""
    x = batch([70, 1, 130, 0], 300, 1, noise=0.0)
    x["accept"][:] = 0.0
    assert check(x, dev)[1] == [70, 1, 130, 0]
    x["accept"][69] = x["accept"][71 + 64] = 1.0  # p = q here: u = 1 rejects
    assert check(x, dev)[1] == [69, 1, 64, 0]


def test_borders_of_the_draw(dev):
    """u = 0 takes the first token with any weight, u just under 1 the last, u = 1 too;
    tokens without weight are never drawn."""
    V = 9000
    p = np.zeros((1, V), np.float32)
    at = [17, 18, 4095, 4096, 8191, 8999 - 5]
    p[0, at] = [0.125, 0.125, 0.25, 0.25, 0.125, 0.125]
    x = dict(target=p, draft=None, tokens=np.zeros(0, np.int32), indptr=np.zeros(2, np.int32),
             accept=np.zeros(0, np.float32), sample=np.zeros(1, np.float32))
    for u, want in ((0.0, 17), (0.124, 17), (0.125, 18), (0.25, 4095), (0.4999, 4095), (0.5, 4096),
                    (0.75, 8191), (0.875, 8994), (1 - 2.0 ** -24, 8994), (1.0, 8994)):
        x["sample"][:] = u
        assert check(x, dev)[0] == [want]


def test_degenerate_rows(dev):
    """p <= q everywhere: the draw is from p. No weight at all: vocab - 1. NaN rejects and
    weighs nothing. Drafts outside the vocabulary are rejected."""
    V = 70
    x = batch([1, 1, 1, 1, 2], V, 5)
    x["accept"][:] = 0.999999
    x["target"][0] = 0.5 * x["draft"][0]   # request 0: residual empty
    x["target"][2] = 0.0                   # request 1: nothing
    x["target"][4] = np.nan                # request 2: NaN
    x["tokens"][3] = V                     # request 3: outside
    x["tokens"][4] = -2
    want = check(x, dev)
    assert want[1] == [0, 0, 0, 0, 0] and want[0][2] == V - 1 and want[0][4] == V - 1
    x["draft"] = None
    check(x, dev)


def test_invalid_offsets_are_marked(dev):
    """A request whose offsets decrease or leave the drafts gets -1 and nothing else."""
    x = batch([2, 2, 2], 50, 6)
    ip = x["indptr"].copy()
    for bad in ([0, 2, 1, 6], [0, 2, 7, 6], [-1, 2, 4, 6]):
        x["indptr"] = np.array(bad, np.int32)
        tokens, accepted = run(x, dev)
        ok = [0 <= bad[r] <= bad[r + 1] <= 6 for r in range(3)]
        assert [a >= 0 for a in accepted] == ok
    x["indptr"] = ip
    check(x, dev)


def test_views_streams_and_graphs(dev):
    """Row strides past the vocabulary (and off the 16-byte grid), a side stream, and a
    captured call replayed with new inputs between eager ones."""
    x = batch([3, 1, 4], 5001, 9)
    for pad, shift in ((3, 0), (7, 1), (8, 4)):
        wide = torch.zeros((len(x["target"]), 5001 + pad + shift), device=dev)
        target = wide[:, shift:shift + 5001]
        target.copy_(torch.from_numpy(x["target"]))
        check(x, dev, target=target)
        wide_d = torch.zeros((len(x["draft"]), 5001 + pad), device=dev)
        draft = wide_d[:, :5001]
        draft.copy_(torch.from_numpy(x["draft"]))
        check(x, dev, target=target, draft=draft)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        check(x, dev)
    g = {k: torch.from_numpy(v).to(dev) for k, v in x.items()}
    ws = torch.empty(capi.lib().sgl_verify_workspace_bytes(3, 5001), dtype=torch.uint8, device=dev)
    call = lambda: capi.verify_drafts(g["target"], g["draft"], g["tokens"], g["indptr"], g["accept"],
                                      g["sample"], ws)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in range(4):
        y = batch([[3, 1, 4], [1, 3, 4], [8, 0, 0], [0, 0, 8]][seed], 5001, 20 + seed)
        for k in g:
            g[k].copy_(torch.from_numpy(y[k]))
        graph.replay()
        torch.cuda.synchronize()
        want = refs.verify(*(y[k] for k in ("target", "draft", "tokens", "indptr", "accept", "sample")))
        assert (out[0].cpu().tolist(), out[1].cpu().tolist()) == want
        check(batch([2, 2], 777, seed), dev)


def test_rows_past_32_bits(dev):
    """Rows 2^31 + 8 elements apart: the third one begins past 2^32."""
    x = batch([2], 4099, 12)
    wide = torch.empty((3, (1 << 31) + 8), device=dev)
    target = wide[:, :4099]
    target.copy_(torch.from_numpy(x["target"]))
    for accept in (x["accept"], np.zeros(2, np.float32), np.full(2, 0.999, np.float32)):
        check({**x, "accept": accept}, dev, target=target)


def test_tokens_follow_the_target(dev):
    """20,000 requests with one draft each: the first emitted token has the target's
    distribution. Each count is binomial; 5 standard deviations (and a half) bound it."""
    N, V = 20_000, 6
    rng = np.random.default_rng(0)
    p = np.array([0.05, 0.3, 0.1, 0.25, 0.2, 0.1], np.float32)
    q = np.array([0.3, 0.1, 0.2, 0.05, 0.05, 0.3], np.float32)
    x = dict(target=np.tile(p, (2 * N, 1)), draft=np.tile(q, (N, 1)),
             tokens=rng.choice(V, N, p=q.astype(np.float64) / q.astype(np.float64).sum()).astype(np.int32),
             indptr=np.arange(N + 1, dtype=np.int32), accept=rng.random(N, np.float32),
             sample=rng.random(N, np.float32))
    tokens, _ = run(x, dev)
    first = np.bincount(np.array(tokens)[::2], minlength=V)
    assert (np.abs(first - N * p) <= 5 * np.sqrt(N * p * (1 - p)) + 0.5).all()


@pytest.mark.parametrize("with_probs", [True, False])
@pytest.mark.parametrize("bad", [[0, 2, 1, 6], [0, 2, 7, 6], [-1, 2, 4, 6], [0, 2, 2 ** 31 - 1, -5], [3, 1, 4, 6]])
def test_invalid_requests_write_nothing_but_their_mark(dev, bad, with_probs):
    """Outputs full of a sentinel: a request whose offsets do not hold gets accepted = -1 and
    no token is written for it; the others, whose places do not meet, have their 64-bit
    results."""
    V, N, B, mark = 4099, 6, 3, -77
    x = batch([2, 2, 2], V, 13, with_probs=with_probs)
    t = {k: None if v is None else torch.from_numpy(v).to(dev) for k, v in x.items()}
    indptr = torch.tensor(bad, dtype=torch.int32, device=dev)
    tokens = torch.full((N + B,), mark, dtype=torch.int32, device=dev)
    accepted = torch.full((B,), mark, dtype=torch.int32, device=dev)
    size = capi.lib().sgl_verify_workspace_bytes(B, V)
    ws = torch.full((size,), 0x7F, dtype=torch.uint8, device=dev)
    args = capi.VerifyArgs(t["target"].data_ptr(), t["draft"].data_ptr() if with_probs else 0,
                           t["tokens"].data_ptr(), indptr.data_ptr(), t["accept"].data_ptr(),
                           t["sample"].data_ptr(), tokens.data_ptr(), accepted.data_ptr(), V, V, N, B, V)
    assert capi.lib().sgl_verify_drafts(ctypes.byref(args), ws.data_ptr(), size,
                                        torch.cuda.current_stream().cuda_stream) == 0
    want, counts = [mark] * (N + B), []
    for r in range(B):
        a, b = bad[r], bad[r + 1]
        if not 0 <= a <= b <= N:
            counts.append(-1)
            continue
        # The request alone: its own rows, drafts and random numbers.
        one, n = refs.verify(x["target"][a + r:b + r + 1], x["draft"][a:b] if with_probs else None,
                             x["tokens"][a:b], [0, b - a], x["accept"][a:b], x["sample"][r:r + 1])
        assert want[a + r:b + r + 1] == [mark] * (b - a + 1)
        want[a + r:b + r + 1] = one
        counts.append(n[0])
    assert accepted.cpu().tolist() == counts
    assert tokens.cpu().tolist() == want
