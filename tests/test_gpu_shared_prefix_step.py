"""GPU tests (marked gpu) of the target model's step over a batch that shares a prompt,
its operators one after the other as a speculative decoder calls them: the scaled
rotary table, rotate-and-append of the last tokens and the drafts, attention behind the
shared prefix, probabilities from logits, verification. And the layers that use them:
RotaryEmbedding and AttentionLayer with scaled, interleaved and partial rotations."""
import numpy as np
import pytest
import torch

import operator_refs as refs
from conftest import capi, pkg, wl

pytestmark = pytest.mark.gpu
D = 128


@pytest.fixture(scope="module")
def be():
    return pkg.backend.load()


class Step:
    """A batch of requests behind a shared prefix, n drafts each; a linear head of its own."""

    def __init__(self, be, dev, P, own, n, hq, hkv, vocab, seed, interleaved):
        g = torch.Generator(device=dev)
        g.manual_seed(seed)
        self.be, self.interleaved, self.hq, self.hkv, self.P = be, interleaved, hq, hkv, P
        own, n = np.asarray(own), np.asarray(n)
        self.qo = n + 1                      # the last token and the drafts
        self.kv = own + self.qo              # cached own tokens, then these
        T = int(self.qo.sum())
        randn = lambda *s: torch.randn(s, generator=g, device=dev)
        slots = P + int(self.kv.sum()) + 16
        self.kc, self.vc = (randn(slots, hkv, D).to(torch.bfloat16) for _ in range(2))
        order = torch.randperm(slots, generator=g, device=dev).int()
        ip = lambda x: torch.from_numpy(np.concatenate([[0], np.cumsum(x)]).astype(np.int32)).to(dev)
        self.prefix, self.indices = order[:P].contiguous(), order[P:P + int(self.kv.sum())].contiguous()
        self.kvp, self.qop, self.indptr = ip(self.kv), ip(self.qo), ip(n)
        at = np.concatenate([np.arange(e - q, e) for e, q in zip(np.cumsum(self.kv), self.qo)])
        self.out_loc = self.indices[torch.from_numpy(at).to(dev)].contiguous()
        pos = np.concatenate([np.arange(P + k - q, P + k) for k, q in zip(self.kv, self.qo)])
        self.pos = torch.from_numpy(pos.astype(np.int32)).to(dev)
        self.qkv = randn(T, (hq + 2 * hkv) * D).to(torch.bfloat16)
        self.head = randn(hq * D, vocab) / np.sqrt(hq * D) * 6
        self.table = be.rope_scaled_cache(P + 4096, 96, 1e6, be.RopeScaling("yarn", 4.0, 1024))
        self.attention = be.PrefixAttention(P, len(n), T, int(self.qo.max()), hq, hkv, D)
        total = int(n.sum())
        self.draft = torch.softmax(2 * randn(total, vocab), -1)
        self.tokens = torch.randint(0, vocab, (total,), generator=g, device=dev).int()
        self.u = torch.rand(total, generator=g, device=dev), torch.rand(len(n), generator=g, device=dev)
        self.temps = torch.full((T,), 0.8, device=dev)

    def heads(self):
        q, k, v = self.qkv.split([self.hq * D, self.hkv * D, self.hkv * D], 1)
        return q.view(-1, self.hq, D), k.view(-1, self.hkv, D), v.view(-1, self.hkv, D)

    def run(self):
        q, k, v = self.heads()
        self.rotated = self.be.rope_append(q, k, v, self.kc, self.vc, *self.table, self.pos,
                                           self.out_loc, self.interleaved)
        self.o = self.attention.forward(self.rotated, self.kc, self.vc, self.prefix, self.indices,
                                        self.kvp, self.qop)
        logits = self.o.reshape(len(self.o), -1).float() @ self.head
        self.probs = self.be.sampling_probs(logits, self.temps)
        return self.be.verify_drafts(self.probs, self.draft, self.tokens, self.indptr, *self.u)


@pytest.mark.parametrize("P,own,n,hq,hkv,interleaved", [
    (700, [3, 90, 0, 17], [4, 2, 0, 7], 32, 8, True),
    (64, [0, 1], [1, 3], 16, 8, False),
    (2050, [20] * 24, [3] * 24, 32, 4, True),
])
def test_step_of_operators(be, dev, P, own, n, hq, hkv, interleaved):
    s = Step(be, dev, P, own, n, hq, hkv, 3001, 1, interleaved)
    tokens, accepted = s.run()
    # The rotation and what the pool holds.
    f, m = refs.frequencies(96, 1e6, "yarn", 4.0, 1024)
    angle = s.pos.cpu().double()[:, None] * torch.from_numpy(f)
    cos, sin = (m * angle.cos()).to(dev), (m * angle.sin()).to(dev)
    q, k, v = s.heads()
    for got, src in ((s.rotated, q), (s.kc[s.out_loc.long()], k)):
        want, size = refs.rotate(src, cos, sin, interleaved)
        # fp32 table (6 x 2^-24 of m each), fp32 rotation, one rounding to bf16.
        assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * size).all()
    assert torch.equal(s.vc[s.out_loc.long()], v)
    # Attention over prefix + own tokens, the bound of its own tests.
    rows = refs.prefix_rows(s.rotated, s.kc, s.vc, s.prefix, s.indices, s.kvp.cpu(), s.qop.cpu(),
                            D ** -0.5)
    for t, (ref, size) in rows.items():
        bound = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -11) * size + 1e-6
        assert ((s.o[t].double() - ref).abs() <= bound).all()
    # The verification of what the target said.
    want = refs.verify(*(x.cpu().numpy() for x in (s.probs, s.draft, s.tokens, s.indptr, *s.u)))
    assert (tokens.cpu().tolist(), accepted.cpu().tolist()) == want


def test_drafts_of_the_target_itself_are_accepted(be, dev):
    """Drafts drawn from the target's own probabilities: all accepted whatever the
    uniforms below 1, and the next token drawn behind the last."""
    s = Step(be, dev, 500, [5, 40, 9], [3, 6, 1], 32, 8, 999, 2, True)
    s.run()
    rows = torch.tensor([i + r for r in range(3) for i in range(int(s.indptr[r]), int(s.indptr[r + 1]))],
                        device=dev)
    s.draft.copy_(s.probs[rows])
    s.tokens.copy_(s.probs[rows].argmax(-1))
    tokens, accepted = s.run()
    assert accepted.cpu().tolist() == [3, 6, 1]
    assert (tokens >= 0).all()


def test_step_captured(be, dev):
    """The step in one graph, replayed with new tokens, drafts and random numbers between
    eager steps of another batch: the bits of the eager step."""
    s = Step(be, dev, 900, [30, 4, 61, 8], [2, 3, 1, 4], 32, 8, 1501, 3, True)
    e = Step(be, dev, 900, [30, 4, 61, 8], [2, 3, 1, 4], 32, 8, 1501, 3, True)
    other = Step(be, dev, 77, [3, 1], [1, 2], 16, 8, 700, 4, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s.run()
    for i in range(4):
        g = torch.Generator(device=dev)
        g.manual_seed(100 + i)
        for x in (s.qkv, *s.u):
            x.copy_(torch.rand(x.shape, generator=g, device=dev))
        s.tokens.copy_(torch.randint(0, 1501, s.tokens.shape, generator=g, device=dev))
        for a, b in ((e.qkv, s.qkv), (e.u[0], s.u[0]), (e.u[1], s.u[1]), (e.tokens, s.tokens),
                     (e.kc, s.kc), (e.vc, s.vc)):
            a.copy_(b)
        graph.replay()
        other.run()
        want = e.run()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        assert torch.equal(s.kc.view(torch.int16), e.kc.view(torch.int16))


def test_two_steps_at_once(be, dev):
    """Two batches on two streams at the same time: the results of one after the other."""
    steps = [Step(be, dev, 400 + 100 * i, [9, 33], [2, 1], 32, 8, 801, 10 + i, bool(i)) for i in range(2)]
    want = []
    for s in steps:
        want.append(s.run())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(steps):
            with torch.cuda.stream(streams[i]):
                got[i] = s.run()
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("interleaved,rotary", [(True, D), (True, 64), (False, 64), (False, D)])
def test_rotary_embedding_module(be, dev, interleaved, rotary):
    rot = be.RotaryEmbedding(D, rotary, 5000, 1e4, be.RopeScaling("bands", 8.0, 1024), interleaved)
    g = torch.Generator(device=dev)
    g.manual_seed(5)
    q, k = (torch.randn((17, h, D), generator=g, device=dev).to(torch.bfloat16) for h in (6, 2))
    pos = torch.randint(0, 5000, (17,), generator=g, device=dev).int()
    q1, k1 = q.clone(), k.clone()
    rot.forward_inplace(pos, q1, k1)
    f, _ = refs.frequencies(rotary, 1e4, "bands", 8.0, 1024)
    angle = pos.cpu().double()[:, None] * torch.from_numpy(f)
    for got, src in ((q1, q), (k1, k)):
        want, size = refs.rotate(src, angle.cos().to(dev), angle.sin().to(dev), interleaved)
        assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * size).all()


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("interleaved,rotary", [(True, D), (False, 32)])
@pytest.mark.parametrize("norm", [True, False])
def test_attention_layer_with_other_rotations(be, dev, decode, interleaved, rotary, norm):
    """AttentionLayer with interleaved or partial rotation: the bits of norm, rotate and
    append, and attend called one by one; other head counts are refused before the pool is
    written."""
    hq, hkv, layers = 32, 8, 2
    b = wl.make_paged_batch(np.random.default_rng(7), [49, 8] if decode else [0, 40],
                            [50, 9] if decode else [33, 95], page_size=16, decode=decode)
    g = torch.Generator(device=dev)
    g.manual_seed(8)
    randn = lambda *s: torch.randn(s, generator=g, device=dev).to(torch.bfloat16)
    rot = be.RotaryEmbedding(D, rotary, 4096, 1e6, be.RopeScaling(), interleaved)
    qn = kn = None
    if norm:
        qn, kn = be.RMSNorm(D, 1e-6, 0), be.RMSNorm(D, 1e-6, 0)
        qn.weight, kn.weight = randn(D), randn(D)
    qkv = randn(int(b.qo_indptr[-1]), (hq + 2 * hkv) * D)
    fill = randn(2, layers, (b.num_pages + 1) * 16, hkv, D)
    outs = []
    for whole in (True, False):
        cache = be.MHAKVCache(hkv, layers, D, b.num_pages + 1, 16, 0)
        cache.buffer().copy_(fill)
        backend = be.HipAttnBackend(cache, hq, hkv, D)
        backend.set_page_table(torch.from_numpy(b.page_table).to(dev))
        reqs = [be.Req(int(b.table_idx[i]), int(b.cached_lens[i]), int(b.device_lens[i]))
                for i in range(b.batch_size)]
        batch = be.Batch(not decode, reqs, torch.from_numpy(b.positions).to(dev),
                         torch.from_numpy(b.out_loc).to(dev))
        backend.prepare_metadata(batch)
        x = qkv.clone()
        if whole:
            o = be.AttentionLayer(1, hq, hkv, D, backend, rot, qn, kn).forward(x, batch.positions, batch)
        else:
            q, k, v = (t.view(-1, h, D) for t, h in zip(x.split([hq * D, hkv * D, hkv * D], 1),
                                                       (hq, hkv, hkv)))
            if norm:
                be.fused_qk_rmsnorm_inplace_3d_strided(q, k, qn, kn)
            be.rope_append(q, k, v, cache.k_cache(1), cache.v_cache(1), rot.cos_cache(),
                           rot.sin_cache(), batch.positions, batch.out_loc, interleaved, q)
            o = backend.attend(q, 1, batch)
            other = be.AttentionLayer(1, hq, 4, D, backend, rot, qn, kn)
            before = cache.buffer().clone()
            with pytest.raises(RuntimeError, match="backend's"):
                other.forward(x[:, :(hq + 8) * D], batch.positions, batch)
            assert torch.equal(before.view(torch.int16), cache.buffer().view(torch.int16))
        outs.append((o, cache.buffer()))
    for a, c in zip(*outs):
        assert torch.equal(a.view(torch.int16), c.view(torch.int16))


def layer_parts(be, dev, decode):
    """A backend over a filled cache, one prepared batch and its qkv rows (32q/8kv)."""
    hq, hkv, layers = 32, 8, 2
    b = wl.make_paged_batch(np.random.default_rng(9), [49, 8] if decode else [0, 40],
                            [50, 9] if decode else [33, 95], page_size=16, decode=decode)
    g = torch.Generator(device=dev)
    g.manual_seed(9)
    cache = be.MHAKVCache(hkv, layers, D, b.num_pages + 1, 16, 0)
    cache.buffer().copy_(torch.randn(cache.buffer().shape, generator=g, device=dev))
    backend = be.HipAttnBackend(cache, hq, hkv, D)
    backend.set_page_table(torch.from_numpy(b.page_table).to(dev))
    reqs = [be.Req(int(b.table_idx[i]), int(b.cached_lens[i]), int(b.device_lens[i]))
            for i in range(b.batch_size)]
    batch = be.Batch(not decode, reqs, torch.from_numpy(b.positions).to(dev),
                     torch.from_numpy(b.out_loc).to(dev))
    backend.prepare_metadata(batch)
    T = int(b.qo_indptr[-1])
    qkv = torch.randn((T, (hq + 2 * hkv) * D), generator=g, device=dev).to(torch.bfloat16)
    norms = be.RMSNorm(D, 1e-6, 0), be.RMSNorm(D, 1e-6, 0)
    for n in norms:
        n.weight = torch.randn(D, generator=g, device=dev).to(torch.bfloat16)
    return cache, backend, batch, qkv, norms


@pytest.mark.parametrize("interleaved", [True, False])
def test_attention_layer_refuses_a_rotation_wider_than_the_head(be, dev, interleaved):
    """A rotary embedding of a larger head is refused when the layer is made; up to the
    head's width it is taken."""
    _, backend, _, _, norms = layer_parts(be, dev, True)
    wide = be.RotaryEmbedding(2 * D, D + 2, 4096, 1e6, be.RopeScaling(), interleaved)
    with pytest.raises(RuntimeError, match="rotary"):
        be.AttentionLayer(1, 32, 8, D, backend, wide, *norms)
    for rotary in (2, 64, D):
        be.AttentionLayer(1, 32, 8, D, backend,
                          be.RotaryEmbedding(2 * D, rotary, 4096, 1e6, be.RopeScaling(), interleaved), *norms)


def refused_calls(batch, qkv):
    """(name, qkv, positions, out_loc) that the layer refuses."""
    T, W = qkv.shape
    pos, loc = batch.positions, batch.out_loc
    wide = lambda first, more: torch.empty((T, W + more), device=qkv.device, dtype=qkv.dtype)[:, first:first + W].copy_(qkv)
    apart = lambda x: torch.stack([x, x], 1)[:, 0]
    yield "positions apart", qkv, apart(pos), loc
    yield "positions on the host", qkv, pos.cpu(), loc
    yield "positions of rank 2", qkv, pos[:, None], loc
    yield "slots apart", qkv, pos, apart(loc)
    yield "slots on the host", qkv, pos, loc.cpu()
    yield "rows off the 16-byte grid", wide(1, 8), pos, loc
    yield "rows a step off the grid", wide(0, 4), pos, loc


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("interleaved,rotary", [(True, D), (False, 32)])
@pytest.mark.parametrize("norm", [True, False])
def test_attention_layer_refuses_before_it_writes(be, dev, decode, interleaved, rotary, norm):
    """A call that interleaved or partial rotations refuse leaves the caller's rows and the
    pool as they were, so that it can be made again."""
    cache, backend, batch, qkv, norms = layer_parts(be, dev, decode)
    rot = be.RotaryEmbedding(D, rotary, 4096, 1e6, be.RopeScaling(), interleaved)
    layer = be.AttentionLayer(1, 32, 8, D, backend, rot, *(norms if norm else (None, None)))
    pool, pos, loc = cache.buffer().clone(), batch.positions, batch.out_loc
    bits = lambda x: x.view(torch.int16)
    touched = []
    for name, rows, p, slots in refused_calls(batch, qkv):
        before = rows.clone()
        batch.out_loc = slots
        with pytest.raises(RuntimeError):
            layer.forward(rows, p, batch)
        batch.out_loc = loc
        if not torch.equal(bits(rows.contiguous()), bits(before.contiguous())) or \
                not torch.equal(bits(cache.buffer()), bits(pool)):
            touched.append(name)
        cache.buffer().copy_(pool)
    assert not touched
    layer.forward(qkv, pos, batch)  # the same objects take the call that holds
