"""sgl_moe_route and sgl_moe_experts against 64-bit forms, the MLP layers made of them, and
a decoder layer's run of them behind the attention."""
import math

import numpy as np
import pytest
import torch

import layer_refs as ref
from conftest import capi, pkg

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ route

def check_route(logits, top_k, renormalize=True):
    weights, experts = capi.moe_route(logits, top_k, renormalize)
    want, ids = ref.route(logits, top_k, renormalize)
    assert weights.dtype == torch.float32 and experts.dtype == torch.int32
    assert torch.equal(experts.cpu(), ids)
    E = logits.shape[1]
    v = logits.double().cpu()
    finite = torch.isfinite(want).all(1)
    assert torch.equal(torch.isfinite(weights.cpu()).all(1), finite)
    assert torch.isnan(weights.cpu()[~finite]).all()
    # The difference to the largest is rounded once (2 half steps of it reach the sums'
    # ratio), expf is good to an ulp, two sums of E and top_k values, two divisions.
    spread = (v - v.max(1, keepdim=True).values).gather(1, ids.long()).abs().clamp(max=200)
    bound = want * ref.U * (2 * spread + 2 * 110 + E + top_k + 8) + 2.0 ** -148
    ref.check(weights[finite.to(weights.device)], want[finite], bound[finite])
    b = pkg.backend.load().moe_route(logits, top_k, renormalize)
    assert torch.equal(b[1], experts) and torch.equal(b[0].isnan(), weights.isnan())
    assert torch.equal(b[0].nan_to_num(), weights.nan_to_num())


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("E", [1, 2, 8, 15, 60, 64, 65, 128, 130, 256, 300, 512])
def test_route(dev, E, dtype):
    g = torch.Generator().manual_seed(E)
    for T in (1, 3, 4, 5, 63, 257):
        logits = (3 * torch.randn(T, E, generator=g)).to(DT[dtype]).to(dev)
        for k in {1, min(E, 2), min(E, 6), min(E, 8), min(E, 32)}:
            check_route(logits, k, renormalize=(T + k) % 2 == 0)


def test_route_of_equal_and_unusual_logits(dev):
    g = torch.Generator().manual_seed(3)
    coarse = torch.randint(-2, 3, (200, 128), generator=g).float()  # ties everywhere
    check_route(coarse.to(dev), 8)
    check_route(torch.zeros(5, 128, device=dev), 8)
    signed = torch.where(coarse > 0, torch.tensor(0.0), torch.tensor(-0.0))  # 0 equals -0
    check_route(signed.to(dev), 6)
    x = torch.randn(12, 60, generator=g)
    x[0, 7] = math.nan                     # a NaN not chosen: NaN weights all the same
    x[1] = math.nan
    x[2, 4] = math.inf
    x[3] = -math.inf
    x[4, 3:] = -math.inf                   # fewer finite logits than chosen
    x[5, 10:20] = -math.inf                # experts masked off
    x[6] = torch.finfo(torch.float32).min  # all at the lowest value
    x[7, 1:] = torch.finfo(torch.float32).min
    x[8] *= 1e30
    x[9] *= 1e-40
    for k in (1, 4, 8):
        for r in (True, False):
            check_route(x.to(dev), k, r)


def test_route_of_strided_rows(dev):
    g = torch.Generator().manual_seed(4)
    big = torch.randn(50, 200, generator=g).to(dev)
    for dt in (torch.float32, torch.bfloat16):
        for off in (0, 1, 8, 37):
            check_route(big.to(dt)[:, off:off + 128], 8)
    check_route(big[:0, :64], 8)
    check_route(big[::3, 1:65], 5)


# ------------------------------------------------------------------ experts

def make(dev, T, E, K, H, I, dtype="bf16", seed=0, spread=True):
    g = torch.Generator(device=dev).manual_seed(seed + T * 7 + E)
    dt = DT[dtype]
    r = lambda *s: torch.randn(s, generator=g, device=dev)
    score = r(T, E) + (r(E) if spread else 0)
    ids = score.topk(K, dim=1).indices.int() if T else torch.zeros(0, K, dtype=torch.int32, device=dev)
    return (r(T, H).to(dt), (r(E, 2 * I, H) / math.sqrt(H)).to(dt),
            (r(E, H, I) / math.sqrt(I)).to(dt), torch.softmax(r(T, K), 1), ids.contiguous())


def check_experts(a, residual=None, activation="silu_and_mul", **kw):
    got = capi.moe_experts(*a, residual=residual, activation=activation, **kw)
    want, bound = ref.experts(*a, residual, activation)
    ref.check(got, want, bound)
    return got


@pytest.mark.parametrize("E,K,H,I", [(8, 2, 128, 64), (16, 1, 200, 72), (32, 8, 256, 96),
                                     (60, 4, 264, 40), (5, 5, 64, 320), (1, 1, 96, 128),
                                     (128, 8, 192, 48)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_experts(dev, E, K, H, I, dtype):
    for i, T in enumerate((1, 2, 3, 4, 5, 8, 9, 16, 17, 33, 64, 100, 300, 700)):
        check_experts(make(dev, T, E, K, H, I, dtype), None,
                      ("silu_and_mul", "gelu_and_mul")[i % 2])


@pytest.mark.parametrize("H,I", [(1, 1), (7, 3), (63, 65), (100, 77), (129, 260)])
def test_experts_of_odd_widths(dev, H, I):
    for T in (1, 6, 40, 200):
        a = make(dev, T, 12, 3, H, I)
        r = torch.randn(T, H, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
        check_experts(a, r)


@pytest.mark.parametrize("T", [1, 7, 30, 90, 500])
def test_experts_of_the_model(dev, T):
    check_experts(make(dev, T, 128, 8, 2048, 768))


@pytest.mark.parametrize("T", [1, 4, 20, 130, 600])
def test_experts_with_a_residual_in_place(dev, T):
    a = make(dev, T, 16, 4, 256, 128)
    r = torch.randn(T, 256, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev)
    want, bound = ref.experts(*a, r.clone())
    assert capi.moe_experts(*a, residual=r, out=r) is r
    ref.check(r, want, bound)


@pytest.mark.parametrize("T", [1, 5, 24, 150, 520])
def test_slots_of_no_expert_and_experts_chosen_twice(dev, T):
    x, gu, d, w, ids = make(dev, T, 10, 4, 128, 96)
    g = torch.Generator().manual_seed(8)
    bad = torch.randint(0, 6, ids.shape, generator=g).to(dev)
    ids = torch.where(bad == 0, torch.full_like(ids, -1), ids)
    ids = torch.where(bad == 1, torch.full_like(ids, 10), ids)
    ids = torch.where(bad == 2, torch.full_like(ids, 2 ** 31 - 1), ids)
    ids = torch.where(bad == 3, ids[:, :1], ids)  # the first one again
    ids[T // 2] = -(2 ** 31)                       # a token of no expert at all
    w = torch.where(ids >= 10, torch.full_like(w, math.nan), w)
    got = capi.moe_experts(x, gu, d, w, ids.int().contiguous())
    clean = torch.where((ids >= 0) & (ids < 10), w, torch.zeros_like(w))
    want, bound = ref.experts(x, gu, d, clean, ids)
    ref.check(got, want, bound)
    assert (got[T // 2] == 0).all()


@pytest.mark.parametrize("T", [1, 12, 100, 400])
def test_all_tokens_at_one_expert(dev, T):
    x, gu, d, w, ids = make(dev, T, 9, 2, 136, 64)
    ids[:, 0], ids[:, 1] = 8, 0
    check_experts((x, gu, d, w, ids))
    ids[:, 1] = 8
    check_experts((x, gu, d, w, ids))


@pytest.mark.parametrize("T", [17, 40, 100])
def test_one_expert_of_many_for_all_tokens(dev, T):
    x, gu, d, w, ids = make(dev, T, 64, 2, 136, 64)
    ids[:, 0], ids[:, 1] = 63, torch.arange(T, device=dev) % 63
    check_experts((x, gu, d, w, ids))
    ids[:, 1] = 63
    check_experts((x, gu, d, w, ids))


def test_values_that_are_not_finite_stay_with_their_token(dev):
    for T in (3, 40, 300):
        x, gu, d, w, ids = make(dev, T, 8, 2, 128, 64)
        want, bound = ref.experts(x, gu, d, w, ids)
        x[T // 2, 5], w[0, 1] = math.nan, math.inf
        got = capi.moe_experts(x, gu, d, w, ids).cpu()
        ok = torch.ones(T, dtype=torch.bool)
        ok[[0, T // 2]] = False
        assert not torch.isfinite(got[T // 2]).any() and not torch.isfinite(got[0]).all()
        ref.check(got[ok], want[ok], bound[ok])


@pytest.mark.parametrize("off,pad", [(0, 8), (1, 3), (4, 4), (8, 0)])
def test_experts_of_strided_tensors(dev, off, pad):
    for T in (2, 30, 260):
        x, gu, d, w, ids = make(dev, T, 6, 3, 128, 64)
        r = torch.randn(T, 128, generator=torch.Generator().manual_seed(3)).to(x.dtype).to(dev)

        def spread(t):
            shape = list(t.shape[:-1]) + [t.shape[-1] + pad]
            flat = torch.full((math.prod(shape) + off + 8,), 7.0, dtype=t.dtype, device=dev)
            v = flat[off:off + math.prod(shape)].view(shape)[..., :t.shape[-1]]
            v.copy_(t)
            return v, flat

        out, flat = spread(torch.zeros_like(x))
        capi.moe_experts(spread(x)[0], spread(gu)[0], spread(d)[0], w, ids, spread(r)[0], out=out)
        want, bound = ref.experts(x, gu, d, w, ids, r)
        ref.check(out, want, bound)
        flat[off:off + T * (128 + pad)].view(T, -1)[:, :128] = 7.0
        assert (flat == 7.0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_terms_of_any_size(dev, dtype):
    """Weights and rows far apart in size: a slot's outputs, large or tiny, reach the sum with
    their own precision, and one that is infinite leaves its neighbours what they are."""
    for T in (3, 60, 400):
        x, gu, d, w, ids = make(dev, T, 8, 2, 128, 64, dtype)
        far = torch.tensor([1e-3, 1.0, 1e3] if dtype == "fp16" else [1e-20, 1.0, 1e20], device=dev)
        w = (w * far[torch.arange(T, device=dev) % 3][:, None]).contiguous()
        rows = torch.ones(128, device=dev)
        rows[::5], rows[1::7] = 2.0 ** -10, 2.0 ** 4
        d = (d.float() * rows[None, :, None]).to(d.dtype)
        if dtype == "fp16":
            w = w.clamp(max=100.0)
        check_experts((x, gu, d, w, ids))
        want, bound = ref.experts(x, gu, d, w, ids)
        d[3, 17] = math.inf
        got = capi.moe_experts(x, gu, d, w, ids).cpu()
        ok = torch.ones(T, 128, dtype=torch.bool)
        ok[(ids == 3).any(1).cpu(), 17] = False
        assert not torch.isfinite(got[~ok]).any()
        ref.check(got[ok], want[ok], bound[ok])


@pytest.mark.parametrize("T", [3, 60, 130, 400])
def test_terms_of_fp16_are_not_rounded(dev, T):
    """2,049 - 2,048, of which fp16 has the first only as 2,048 or 2,050."""
    x, gu, d, w, ids = make(dev, T, 2, 2, 128, 64, "fp16")
    x.zero_(), gu.zero_(), d.zero_()
    x[:, 5], gu[:, :64, 5], gu[:, 64:, 5] = 1, 32, 1   # silu(32) is 32 to 2^-40
    d[:, :, 3], d[0, :, 40] = 64, 2.0 ** -5
    w.copy_(torch.where(ids == 0, 1.0, -1.0))
    assert (capi.moe_experts(x, gu, d, w, ids) == 1).all()


@pytest.mark.parametrize("T,K", [(8192, 8), (9001, 8), (30001, 3), (140000, 1)])
def test_many_choices(dev, T, K):
    check_experts(make(dev, T, 40, K, 16, 8))


@pytest.mark.parametrize("T,E,K", [(1, 700, 6), (300, 700, 4), (1500, 1025, 2), (1, 64, 40), (3, 64, 40),
                                   (4, 64, 32), (4, 64, 33), (30, 200, 33), (100, 64, 40)])
def test_many_experts_and_many_of_a_token(dev, T, E, K):
    check_experts(make(dev, T, E, K, 72, 40))


@pytest.mark.parametrize("T", [3, 130, 1501])
def test_choices_at_any_place(dev, T):
    x, gu, d, w, ids = make(dev, T, 12, 3, 64, 32)
    for off in (1, 2, 3):
        at = torch.full((off + 3 * T,), 5, dtype=torch.int32, device=dev)
        weights = torch.zeros(off + 3 * T, device=dev)
        at[off:], weights[off:] = ids.view(-1), w.view(-1)
        check_experts((x, gu, d, weights[off:].view(T, 3), at[off:].view(T, 3)))


@pytest.mark.parametrize("T", [3, 20, 500])
def test_experts_past_32_bits(dev, T):
    """Weights whose elements, and rows of x whose bytes, pass 2^31."""
    x, gu, d, w, ids = make(dev, T, 4, 2, 64, 32)
    apart = 2 ** 30 + 8
    big = torch.empty(3 * apart + 64 * 64, dtype=x.dtype, device=dev)
    gate_up = big.as_strided((4, 64, 64), (apart, 64, 1))
    gate_up.copy_(gu)
    want = check_experts((x, gate_up, d, w, ids))
    down = big.as_strided((4, 64, 32), (apart, 32, 1))
    down.copy_(d)
    assert torch.equal(capi.moe_experts(x, gu, down, w, ids), want)


@pytest.mark.parametrize("T", [500, 1000, 1100])
def test_rows_of_experts_past_32_bits(dev, T):
    x, gu, d, w, ids = make(dev, T, 4, 2, 64, 32)
    far = torch.empty(T * 2 ** 20, dtype=x.dtype, device=dev).as_strided((T, 64), (2 ** 20, 1))
    far.copy_(x)
    check_experts((far, gu, d, w, ids))
    out = far[:, 16:]
    a = make(dev, T, 4, 2, 48, 32)
    want = capi.moe_experts(*a)
    assert torch.equal(capi.moe_experts(*a, out=out), want)


def test_experts_of_no_tokens(dev):
    a = make(dev, 0, 4, 2, 64, 32)
    assert capi.moe_experts(*a).shape == (0, 64)


@pytest.mark.parametrize("T", [1, 12, 90, 400])
def test_captured_replayed_and_two_at_once(dev, T):
    be = pkg.backend.load()
    x, gu, d, w, ids = make(dev, T, 16, 4, 256, 128)
    out = torch.empty_like(x)
    be.moe_experts(x, gu, d, w, ids, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        be.moe_experts(x, gu, d, w, ids, out=out)
    for i in range(4):
        new = make(dev, T, 16, 4, 256, 128, seed=i + 1)
        x.copy_(new[0]), w.copy_(new[3]), ids.copy_(new[4])
        want = be.moe_experts(x, gu, d, w, ids)
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    main, side = torch.cuda.current_stream(), torch.cuda.Stream()
    side.wait_stream(main)
    outs = []
    for i in range(8):
        with torch.cuda.stream(side if i % 2 else main):
            outs.append(be.moe_experts(x, gu, d, w, ids))
    main.wait_stream(side)
    assert all(torch.equal(o, want) for o in outs)


def test_argument_checks(dev):
    be = pkg.backend.load()
    x, gu, d, w, ids = make(dev, 4, 8, 2, 64, 32)
    bad = [(x.float(), gu, d, w, ids), (x, gu[:, :63], d, w, ids), (x, gu.half(), d, w, ids),
           (x, gu, d[:7], w, ids), (x, gu, d, w.half(), ids), (x, gu, d, w, ids.long()),
           (x, gu, d, w[:3], ids[:3]), (x, gu, d, w, ids[:, :1]), (x.cpu(), gu, d, w, ids)]
    for a in bad:
        for f in (capi.moe_experts, be.moe_experts):
            with pytest.raises((ValueError, RuntimeError)):
                f(*a)
    for f in (capi.moe_route, be.moe_route):
        for a in ((x.float(), 0), (x.float(), 65), (x.int(), 2), (x.float()[0], 2)):
            with pytest.raises((ValueError, RuntimeError)):
                f(*a)
    with pytest.raises(RuntimeError):
        be.MoEMLP(64, 32, 4, 5)
    with pytest.raises(RuntimeError):
        be.GatedMLP(64, 32, "silu")


# ------------------------------------------------------------------ layers

@pytest.mark.parametrize("T", [1, 20, 200])
def test_mlp_layers(dev, T):
    be = pkg.backend.load()
    g = torch.Generator().manual_seed(11)
    r = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16).to(dev)
    x, res = r(T, 256), r(T, 256)
    mlp = be.GatedMLP(256, 512, "gelu_and_mul")
    assert (mlp.forward(x) == 0).all()
    mlp.gate_up, mlp.down = r(1024, 256) / 16, r(256, 512) / 16
    h = be.linear(x, mlp.gate_up, activation="gelu_and_mul")
    want, bound = ref.linear(h, mlp.down, residual=res)
    ref.check(mlp.forward(x, res), want, bound)
    moe = be.MoEMLP(256, 96, 16, 4, True)
    moe.router, moe.gate_up, moe.down = r(16, 256) / 4, r(16, 192, 256) / 16, r(16, 256, 96) / 8
    logits = be.linear(x, moe.router, out_dtype=torch.float32)
    want, bound = ref.linear(x, moe.router, out_dtype=torch.float32)
    ref.check(logits, want, bound)
    weights, ids = ref.route(logits, 4, True)
    want, bound = ref.experts(x, moe.gate_up, moe.down, weights.float(), ids, res)
    ref.check(moe.forward(x, res), want, bound)


def test_mlp_layers_in_fp16_and_captured(dev):
    be = pkg.backend.load()
    g = torch.Generator().manual_seed(12)
    r = lambda *s: torch.randn(s, generator=g).to(torch.float16).to(dev)
    mlp, moe = be.GatedMLP(128, 192, "silu_and_mul"), be.MoEMLP(128, 64, 8, 2)
    mlp.gate_up, mlp.down = r(384, 128) / 12, r(128, 192) / 14
    moe.router, moe.gate_up, moe.down = r(8, 128) / 4, r(8, 128, 128) / 12, r(8, 128, 64) / 8
    for T in (1, 40, 300):
        x, out = r(T, 128), torch.empty(T, 128, dtype=torch.float16, device=dev)
        step = lambda: out.copy_(moe.forward(mlp.forward(x, x), x))
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for _ in range(3):
            x.copy_(r(T, 128))
            h = mlp.forward(x, x)
            want, bound = ref.linear(be.linear(x, mlp.gate_up, activation="silu_and_mul"), mlp.down,
                                     residual=x)
            ref.check(h, want, bound)
            want = moe.forward(h, x)
            out.fill_(9.0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


@pytest.mark.parametrize("decode", [True, False])
def test_decoder_layer(dev, decode):
    """norm, q/k/v projection, attention, output projection onto the residual, norm, experts,
    each against 64 bits from the same inputs, then the whole run again from a graph."""
    be, wl = pkg.backend.load(), pkg.workloads
    hq, hkv, D, H = 8, 2, 128, 512
    rng = np.random.default_rng(5)
    b = wl.make_paged_batch(rng, [30, 0, 200] if not decode else [30, 7, 200],
                            [37, 21, 233] if not decode else [31, 8, 201], 16, decode=decode)
    T = len(b.positions)
    g = torch.Generator().manual_seed(6)
    r = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16).to(dev)
    cache = be.MHAKVCache(hkv, 1, D, b.num_pages + 1, 16)
    cache.buffer().copy_(r(*cache.buffer().shape))
    table = torch.from_numpy(b.page_table).to(dev)
    att = be.HipAttnBackend(cache, hq, hkv, D)
    att.set_page_table(table)
    rope = be.RotaryEmbedding(D, D, 4096, 1e6)
    reqs = [be.Req(int(t), int(c), int(d)) for t, c, d in zip(b.table_idx, b.cached_lens, b.device_lens)]
    batch = be.Batch(not decode, reqs, torch.from_numpy(b.positions).to(dev),
                     torch.from_numpy(b.out_loc).to(dev))
    att.prepare_metadata(batch)
    layer = be.AttentionLayer(0, hq, hkv, D, att, rope)
    norm1, norm2 = be.RMSNorm(H, 1e-6), be.RMSNorm(H, 1e-6)
    qkv_w, qkv_b, o_w = r((hq + 2 * hkv) * D, H) / 22, r((hq + 2 * hkv) * D), r(H, hq * D) / 32
    moe = be.MoEMLP(H, 96, 16, 4)
    moe.router, moe.gate_up, moe.down = r(16, H) / 4, r(16, 192, H) / 22, r(16, H, 96) / 10
    hidden = r(T, H)

    def step():
        n = norm1.forward(hidden)
        qkv = be.linear(n, qkv_w, qkv_b)
        first = qkv.clone()
        o = layer.forward(qkv, batch.positions, batch)
        mid = be.linear(o, o_w, residual=hidden)
        m = norm2.forward(mid)
        return n, first, o, mid, m, moe.forward(m, mid)

    n, qkv, o, mid, m, out = step()
    ref.check(qkv, *ref.linear(n, qkv_w, qkv_b))
    ref.check(mid, *ref.linear(o, o_w, residual=hidden))
    logits = be.linear(m, moe.router, out_dtype=torch.float32)
    weights, ids = ref.route(logits, 4, True)
    ref.check(out, *ref.experts(m, moe.gate_up, moe.down, weights.float(), ids, mid))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = step()[-1]
    for _ in range(3):
        again.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, out)
