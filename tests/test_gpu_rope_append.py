"""GPU tests (marked gpu) of the scaled rotary tables and of the pass that rotates
q and k and appends k and v to the paged pool, against 64-bit forms.

Tables: the angle of a quarter turn's rest, at most pi / 4, takes three roundings
(2.5 x 2^-24 of it), the series leaves out 2e-9 and its last steps round twice,
the factor m once: below 6 x 2^-24 of m. The 64-bit angle is off by less than
2^-33. Rotation: two products and a sum in fp32 (at most 2 x 2^-24 of the absolute
products), then one rounding to the type: half a step, 2^-8 (bf16) or 2^-11 (fp16)
of the value, and for fp16 half its smallest step, 2^-25."""
import ctypes

import numpy as np
import pytest
import torch

import operator_refs as refs
from conftest import capi, pkg

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
SMALLEST = {"bf16": 0.0, "fp16": 2.0 ** -25}


def be():
    return pkg.backend.load()


@pytest.mark.parametrize("kind,extra", [
    ("none", {}), ("linear", {}), ("ntk", {}),
    ("yarn", {}), ("yarn", dict(beta_fast=16.0, beta_slow=2.0, attention_factor=1.25)),
    ("bands", {}), ("bands", dict(low_freq_factor=2.0, high_freq_factor=8.0))])
@pytest.mark.parametrize("max_pos,rotary", [(1, 2), (7, 6), (1000, 64), (513, 96), (2049, 128),
                                            (33, 512), (5, 508)])
def test_scaled_table(dev, kind, extra, max_pos, rotary):
    if kind == "ntk":
        rotary += 2 * (rotary == 2)  # two pairs at least: of one the exponent has no value
    factor, original = 4.0, 500
    sc = capi.rope_scaling(kind, factor, original, **extra)
    cos, sin = capi.rope_scaled_cache(max_pos, rotary, 10000.0, dev, sc)
    names = dict(low_freq_factor="low", high_freq_factor="high", attention_factor="attention")
    f, m = refs.frequencies(rotary, 10000.0, kind, factor, original,
                            **{names.get(k, k): v for k, v in extra.items()})
    angle = np.arange(max_pos)[:, None] * f[None]
    for got, want in ((cos, m * np.cos(angle)), (sin, m * np.sin(angle))):
        assert got.shape == (max_pos, rotary // 2) and got.dtype == torch.float32
        assert np.abs(got.cpu().double().numpy() - want).max() <= 6 * 2.0 ** -24 * m


def test_scaled_table_far_positions_and_backend(dev):
    b = be()
    sc = b.RopeScaling(kind="yarn", factor=8.0, original_max_position=32768)
    cos, sin = b.rope_scaled_cache(262_147, 128, 1e6, sc)
    f, m = refs.frequencies(128, 1e6, "yarn", 8.0, 32768)
    at = np.array([0, 1, 131_071, 200_001, 262_146])
    angle = at[:, None] * f[None]
    idx = torch.from_numpy(at).to(dev)
    assert np.abs(cos[idx].cpu().double().numpy() - m * np.cos(angle)).max() <= 6 * 2.0 ** -24 * m
    assert np.abs(sin[idx].cpu().double().numpy() - m * np.sin(angle)).max() <= 6 * 2.0 ** -24 * m
    c2, s2 = capi.rope_scaled_cache(262_147, 128, 1e6, dev, capi.rope_scaling("yarn", 8.0, 32768))
    assert torch.equal(cos, c2) and torch.equal(sin, s2)


def table(max_pos, rotary, dev):
    f, _ = refs.frequencies(rotary, 10000.0)
    angle = torch.arange(max_pos, dtype=torch.float64)[:, None] * torch.from_numpy(f)
    return angle.cos().float().to(dev), angle.sin().float().to(dev)


def make(dev, T, hq, hkv, d, rotary, dtype, seed, slots=None, max_pos=500):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rand = lambda *s: torch.randn(s, device=dev, generator=g).to(DT[dtype])
    slots = T + 9 if slots is None else slots
    cos, sin = table(max_pos, rotary, dev)
    return dict(q=rand(T, hq, d), k=rand(T, hkv, d), v=rand(T, hkv, d), kc=rand(slots, hkv, d),
                vc=rand(slots, hkv, d), cos=cos, sin=sin,
                pos=torch.randint(0, max_pos, (T,), device=dev, generator=g).int(),
                loc=torch.randperm(slots, device=dev, generator=g)[:T].int())


def check(x, q, kc, vc, before, interleaved, dtype, loc=None):
    """q rotated, the new rows of the caches, and every other row as it was."""
    loc = x["loc"] if loc is None else loc
    at = x["pos"].long()
    c, s = x["cos"][at], x["sin"][at]
    def near(got, src):
        want, size = refs.rotate(src, c, s, interleaved)
        # Elements past the rotated part are copies.
        r = 2 * x["cos"].shape[1]
        assert torch.equal(got[..., r:], src[..., r:])
        err = (got.double() - want).abs()[..., :r]
        bound = HALF_STEP[dtype] * want.abs() + 2.0 ** -22 * size + SMALLEST[dtype]
        assert (err <= bound[..., :r]).all(), float((err - bound[..., :r]).max())
    near(q, x["q"])
    new = loc.long()
    near(kc[new], x["k"])
    assert torch.equal(vc[new], x["v"])
    rest = torch.ones(kc.shape[0], dtype=torch.bool, device=kc.device)
    rest[new] = False
    assert torch.equal(kc[rest], before[0][rest]) and torch.equal(vc[rest], before[1][rest])


SHAPES = [(1, 1, 1, 128, 128), (7, 16, 8, 128, 128), (33, 32, 4, 128, 64), (5, 3, 1, 64, 64),
          (6, 4, 2, 64, 32), (9, 2, 2, 256, 192), (4, 5, 5, 80, 80), (3, 2, 1, 96, 64),
          (8, 4, 2, 128, 96), (11, 3, 3, 72, 40), (2, 1, 1, 6, 4), (2, 2, 1, 7, 2),
          (3, 1, 1, 1024, 512), (130, 8, 2, 128, 16), (300, 6, 2, 112, 112)]


@pytest.mark.parametrize("T,hq,hkv,d,rotary", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_append(dev, T, hq, hkv, d, rotary, interleaved, dtype):
    x = make(dev, T, hq, hkv, d, rotary, dtype, T * 31 + d)
    before = x["kc"].clone(), x["vc"].clone()
    q0 = x["q"].clone()
    q = capi.rope_append(x["q"], x["k"], x["v"], x["kc"], x["vc"], x["cos"], x["sin"], x["pos"],
                         x["loc"], interleaved)
    assert torch.equal(x["q"], q0)
    check(x, q, x["kc"], x["vc"], before, interleaved, dtype)
    # In place, with int64 slots and through the C++ backend: the same bits.
    kc, vc = before[0].clone(), before[1].clone()
    y = q0.clone()
    be().rope_append(y, x["k"], x["v"], kc, vc, x["cos"], x["sin"], x["pos"], x["loc"].long(),
                     interleaved, y)
    assert torch.equal(y, q) and torch.equal(kc, x["kc"]) and torch.equal(vc, x["vc"])


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_views(dev, interleaved):
    """q, k, v narrow views of a qkv row, caches with a padded slot stride, one by
    one also shifted off the 16-byte grid."""
    T, hq, hkv, d = 19, 8, 2, 128
    x = make(dev, T, hq, hkv, d, d, "bf16", 5)
    for shift in (0, 1, 8):
        w = (hq + 2 * hkv) * d
        qkv = torch.empty((T, w + 24), device=dev, dtype=torch.bfloat16)[:, shift:shift + w]
        q, k, v = (t.view(T, -1, d) for t in qkv.split([hq * d, hkv * d, hkv * d], 1))
        q.copy_(x["q"]), k.copy_(x["k"]), v.copy_(x["v"])
        wide = torch.randn((2, x["kc"].shape[0], hkv + 1, d + 8), device=dev).to(torch.bfloat16)
        kc, vc = wide[0][:, :hkv, shift // 8 * 8:][..., :d], wide[1][:, :hkv, shift // 8 * 8:][..., :d]
        before = kc.clone(), vc.clone()
        out = capi.rope_append(q, k, v, kc, vc, x["cos"], x["sin"], x["pos"], x["loc"], interleaved, q)
        assert out.data_ptr() == q.data_ptr()
        check(x, q, kc, vc, before, interleaved, "bf16")


@pytest.mark.parametrize("d,rotary", [(128, 128), (7, 2)])
def test_append_padding_and_far_positions(dev, d, rotary):
    """Slots outside the pool are not written, positions outside the table give NaN
    in the rotated elements and nowhere else."""
    T = 12
    x = make(dev, T, 4, 2, d, rotary, "bf16", 3)
    before = x["kc"].clone(), x["vc"].clone()
    loc, pos = x["loc"].clone(), x["pos"].clone()
    loc[3], loc[7], loc[11] = -1, x["kc"].shape[0], 2 ** 31 - 1
    pos[5], pos[6] = -1, x["cos"].shape[0]
    q = capi.rope_append(x["q"], x["k"], x["v"], x["kc"], x["vc"], x["cos"], x["sin"], pos, loc)
    for t in (5, 6):
        assert q[t][:, :rotary].isnan().all() and x["kc"][loc[t].long()][:, :rotary].isnan().all()
        assert torch.equal(q[t][:, rotary:], x["q"][t][:, rotary:])
        assert torch.equal(x["vc"][loc[t].long()], x["v"][t])
    good = [t for t in range(T) if t not in (3, 5, 6, 7, 11)]
    sub = {**x, "q": x["q"][good], "k": x["k"][good], "v": x["v"][good], "pos": x["pos"][good]}
    for t in (5, 6):  # their rows were looked at above
        before[0][loc[t].long()] = x["kc"][loc[t].long()] = 0
        before[1][loc[t].long()] = x["vc"][loc[t].long()] = 0
    check(sub, q[good], x["kc"], x["vc"], before, False, "bf16", loc[good])


def test_append_without_v_or_slots_rotates_in_place(dev):
    """out_loc None and the cache k itself: q and k rotated where they are."""
    x = make(dev, 21, 6, 3, 64, 48, "fp16", 8)
    q, k = x["q"].clone(), x["k"].clone()
    capi.rope_append(q, k, None, k, None, x["cos"], x["sin"], x["pos"], None, True, q)
    at = x["pos"].long()
    for got, src in ((q, x["q"]), (k, x["k"])):
        want, size = refs.rotate(src, x["cos"][at], x["sin"][at], True)
        assert ((got.double() - want).abs() <= HALF_STEP["fp16"] * want.abs() + 2.0 ** -22 * size
                + SMALLEST["fp16"]).all()


def test_append_empty_and_equals_the_fused_pass(dev):
    x = make(dev, 40, 16, 8, 128, 128, "bf16", 2)
    e = {k: x[k][:0] for k in ("q", "k", "v", "pos", "loc")}
    before = x["kc"].clone(), x["vc"].clone()
    out = capi.rope_append(e["q"], e["k"], e["v"], x["kc"], x["vc"], x["cos"], x["sin"], e["pos"],
                           e["loc"])
    assert out.shape == (0, 16, 128) and torch.equal(x["kc"], before[0])
    # Half layout over the whole head: the bits of the fused pass without norms.
    qkv = torch.cat([x[k].reshape(40, -1) for k in ("q", "k", "v")], 1).contiguous()
    kc, vc = before[0].clone(), before[1].clone()
    capi.fused_qknorm_rope_store(qkv, kc, vc, None, None, x["cos"], x["sin"], x["pos"], x["loc"],
                                 16, 8, 128, 1e-6)
    q = capi.rope_append(x["q"], x["k"], x["v"], x["kc"], x["vc"], x["cos"], x["sin"], x["pos"], x["loc"])
    assert torch.equal(q.reshape(40, -1), qkv[:, :16 * 128])
    assert torch.equal(kc, x["kc"]) and torch.equal(vc, x["vc"])


def test_append_far_slots_on_a_side_stream_and_in_a_graph(dev):
    """Slots whose element offsets pass 2^32; a side stream; a captured call replayed
    between eager ones."""
    slots, hkv, d, T = (1 << 32) // (8 * 128) + 64, 8, 128, 33
    kc = torch.zeros((slots, hkv, d), device=dev, dtype=torch.bfloat16)
    vc = torch.zeros_like(kc)
    x = make(dev, T, 16, hkv, d, d, "bf16", 4)
    loc = (slots - 1 - torch.arange(T, device=dev)).int()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q = capi.rope_append(x["q"], x["k"], x["v"], kc, vc, x["cos"], x["sin"], x["pos"], loc)
    torch.cuda.current_stream().wait_stream(side)
    rows = loc.long()
    assert not kc[:slots - T].any() and torch.equal(vc[rows], x["v"])
    out = torch.empty_like(x["q"])
    graph = torch.cuda.CUDAGraph()
    kc.zero_(), vc.zero_()
    with torch.cuda.graph(graph):
        capi.rope_append(x["q"], x["k"], x["v"], kc, vc, x["cos"], x["sin"], x["pos"], loc, False, out)
    for step in range(3):
        x["pos"].copy_((x["pos"] + step) % 500)
        x["v"].add_(1)
        graph.replay()
        eager = capi.rope_append(x["q"], x["k"], x["v"], x["kc"], x["vc"], x["cos"], x["sin"],
                                 x["pos"], x["loc"])
        assert torch.equal(out, eager) and torch.equal(vc[rows], x["v"])
        assert torch.equal(kc[rows], x["kc"][x["loc"].long()])


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_many_tokens(dev, interleaved):
    """A batch whose rows pass the size from which a thread has one token: the bits of the
    same call on its parts."""
    T = 4099
    x = make(dev, T, 32, 8, 128, 128, "bf16", 6)
    kc, vc = x["kc"].clone(), x["vc"].clone()
    q = capi.rope_append(x["q"], x["k"], x["v"], x["kc"], x["vc"], x["cos"], x["sin"], x["pos"],
                         x["loc"], interleaved)
    for a, b in ((0, 1000), (1000, 1001), (1001, T)):
        part = capi.rope_append(*(x[k][a:b] for k in ("q", "k", "v")), kc, vc, x["cos"], x["sin"],
                                x["pos"][a:b], x["loc"][a:b], interleaved)
        assert torch.equal(part, q[a:b])
    assert torch.equal(kc, x["kc"]) and torch.equal(vc, x["vc"])


def test_append_without_q_takes_any_q_strides(dev):
    """num_qo_heads 0: no q, whatever its pointers and strides say; k and v as with it."""
    x = make(dev, 9, 4, 2, 128, 64, "bf16", 12)
    kc, vc = x["kc"].clone(), x["vc"].clone()
    capi.rope_append(x["q"], x["k"], x["v"], x["kc"], x["vc"], x["cos"], x["sin"], x["pos"], x["loc"])
    for st in (0, 512):
        k2, v2 = kc.clone(), vc.clone()
        args = capi.RopeAppendArgs(
            k=x["k"].data_ptr(), v=x["v"].data_ptr(), k_cache=k2.data_ptr(), v_cache=v2.data_ptr(),
            cos=x["cos"].data_ptr(), sin=x["sin"].data_ptr(), positions=x["pos"].data_ptr(),
            out_loc=x["loc"].data_ptr(), tokens=9, num_slots=k2.shape[0], max_pos=x["cos"].shape[0],
            q_stride_token=st, q_stride_head=128, k_stride_token=256, k_stride_head=128,
            v_stride_token=256, v_stride_head=128, kv_stride_slot=256, kv_stride_head=128,
            num_qo_heads=0, num_kv_heads=2, head_dim=128, rotary_dim=64)
        stream = torch.cuda.current_stream().cuda_stream
        assert capi.lib().sgl_rope_append(ctypes.byref(args), stream) == 0
        assert torch.equal(k2, x["kc"]) and torch.equal(v2, x["vc"])
