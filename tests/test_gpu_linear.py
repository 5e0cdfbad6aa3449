"""sgl_linear against 64-bit sums: sizes from one token and one output on, odd ones, every
epilogue, strides and alignments, values that are not finite, other streams and graphs."""
import itertools
import math

import pytest
import torch

import layer_refs as ref
from conftest import capi, pkg

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def make(dev, T, n, k, dtype="bf16", gated=False, seed=0):
    g = torch.Generator().manual_seed(seed + 1000 * T + 10 * n + k)
    dt = DT[dtype]
    rows = 2 * n if gated else n
    r = lambda *s: torch.randn(s, generator=g)
    return ((r(T, k)).to(dt).to(dev), (r(rows, k) / math.sqrt(k)).to(dt).to(dev),
            r(rows).to(dt).to(dev), r(T, n).to(dt).to(dev))


def run(dev, T, n, k, dtype="bf16", activation="none", bias=False, residual=False, fp32=False):
    x, w, b, r = make(dev, T, n, k, dtype, activation.endswith("_and_mul"))
    b, r = b if bias else None, r if residual else None
    to = torch.float32 if fp32 else x.dtype
    got = capi.linear(x, w, b, activation, r, out_dtype=to)
    want, bound = ref.linear(x, w, b, activation, r, to)
    assert got.dtype == to and got.shape == (T, n)
    ref.check(got, want, bound, f"{T} x {n} x {k} {dtype} {activation}")


@pytest.mark.parametrize("k", [1, 7, 8, 40, 64, 72, 200, 1032, 2048])
@pytest.mark.parametrize("n", [1, 16, 100, 128, 1000])
def test_sizes_of_few_tokens(dev, n, k):
    for T in (1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 33, 48, 64):
        run(dev, T, n, k)


@pytest.mark.parametrize("T,n,k", [
    (65, 128, 64), (100, 257, 136), (128, 256, 512), (129, 300, 1000), (255, 512, 72),
    (256, 1024, 192), (257, 1000, 264), (333, 640, 1024), (512, 513, 71), (600, 2048, 640),
    (1000, 256, 2048), (1025, 1280, 328), (2049, 700, 256)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_sizes_of_many_tokens(dev, T, n, k, dtype):
    run(dev, T, n, k, dtype)
    run(dev, T, n, k, dtype, "silu_and_mul", bias=True, residual=True)


# Sizes that take each tile shape with the inputs whole and in parts, a part of a stage among them.
@pytest.mark.parametrize("T,n,k,gated", [
    (4100, 1000, 72, True), (4100, 500, 4104, True), (4100, 500, 9000, False),
    (4100, 500, 72, True), (400, 2500, 6000, True), (257, 2000, 9000, True),
    (257, 1000, 2056, True), (130, 500, 1032, True), (70, 64, 1000, False),
    (130, 500, 2056, True), (130, 500, 4104, True), (70, 64, 2056, False), (70, 64, 4104, False)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_tiles_and_parts(dev, T, n, k, gated, dtype):
    run(dev, T, n, k, dtype, "gelu_and_mul" if gated else "none", bias=True, residual=True)
    run(dev, T, n, k, dtype, "silu_and_mul" if gated else "silu", fp32=True)


@pytest.mark.parametrize("T", [80, 300, 1100])
def test_a_call_without_a_workspace(dev, T):
    """The C entry with no workspace: the inputs in one part, the same sums to rounding."""
    n, k = 512, 4096
    x, w, b, r = make(dev, T, n, k)
    out = torch.empty(T, n, dtype=x.dtype, device=dev)
    a = capi.LinearArgs(x.data_ptr(), w.data_ptr(), b.data_ptr(), r.data_ptr(), out.data_ptr(), T, n, k,
                        k, k, n, n, 0, 0, 1, 0)
    import ctypes
    assert capi.lib().sgl_linear_workspace_bytes(T, n, k, 1) > 0
    assert capi.lib().sgl_linear(ctypes.byref(a), None, 0,
                                 ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    ref.check(out, *ref.linear(x, w, b, "silu", r))


@pytest.mark.parametrize("T", [1, 20, 90])
def test_subnormal_values(dev, T):
    """fp16 values below its smallest normal one count with their own precision."""
    x, w, _, _ = make(dev, T, 64, 128, "fp16")
    x = (x.float() * 2.0 ** -20).half()
    want, bound = ref.linear(x, w, out_dtype=torch.float32)
    ref.check(capi.linear(x, w, out_dtype=torch.float32), want, bound)
    w = (w.float() * 2.0 ** -16).half()
    x = x.float().mul(2.0 ** 20).half()
    want, bound = ref.linear(x, w)
    ref.check(capi.linear(x, w), want, bound)


EPILOGUES = list(itertools.product(["none", "silu", "gelu", "silu_and_mul", "gelu_and_mul"],
                                   [False, True], [False, True], [False, True]))


@pytest.mark.parametrize("T,n,k", [(1, 96, 512), (6, 130, 256), (13, 64, 1024), (40, 260, 320),
                                   (150, 384, 256), (700, 512, 512)])
def test_epilogues(dev, T, n, k):
    for i, (activation, bias, residual, fp32) in enumerate(EPILOGUES):
        run(dev, T, n, k, ("bf16", "fp16")[i % 2], activation, bias, residual, fp32)


@pytest.mark.parametrize("T", [1, 7, 16, 50, 300, 800])
@pytest.mark.parametrize("off,pad", [(0, 8), (1, 3), (4, 0), (8, 64), (3, 5)])
def test_strided_and_unaligned_rows(dev, T, off, pad):
    n, k = 256, 320
    x, w, b, r = make(dev, T, n, k, gated=True)

    def spread(t):  # the same rows `pad` further apart, starting `off` elements in
        big = torch.full((t.shape[0] * (t.shape[1] + pad) + off + 8,), 7.0, dtype=t.dtype, device=dev)
        v = big[off:off + t.shape[0] * (t.shape[1] + pad)].view(t.shape[0], -1)[:, :t.shape[1]]
        v.copy_(t)
        return v, big

    (xs, _), (ws, _), (rs, _) = spread(x), spread(w), spread(r)
    out, big = spread(torch.zeros(T, n, dtype=x.dtype, device=dev))
    got = capi.linear(xs, ws, b, "silu_and_mul", rs, out=out)
    assert got is out
    want, bound = ref.linear(x, w, b, "silu_and_mul", r)
    ref.check(out, want, bound)
    rest = big.clone()
    rest[off:off + T * (n + pad)].view(T, -1)[:, :n] = 7.0
    assert (rest == 7.0).all()  # nothing between or behind the rows


@pytest.mark.parametrize("T", [1, 5, 24, 64, 200, 700])
def test_residual_in_place(dev, T):
    x, w, _, r = make(dev, T, 384, 512)
    want, bound = ref.linear(x, w, None, "none", r)
    assert capi.linear(x, w, residual=r, out=r) is r
    ref.check(r, want, bound)


@pytest.mark.parametrize("T", [3, 20, 90, 520])
def test_values_that_are_not_finite_stay_in_their_row_and_column(dev, T):
    x, w, _, _ = make(dev, T, 200, 456)
    want, bound = ref.linear(x, w)
    x[T // 2, 17], x[0, 3] = math.nan, math.inf
    w[111, 40], w[199, 455] = math.nan, -math.inf
    got = capi.linear(x, w).cpu()
    rows, cols = [0, T // 2], [111, 199]
    ok = torch.ones(T, 200, dtype=torch.bool)
    ok[rows], ok[:, cols] = False, False
    assert not torch.isfinite(got[~ok]).any()
    ref.check(got[ok], want[ok], bound[ok])


def test_activations_of_large_values(dev):
    v = torch.tensor([-3e38, -1e4, -200.0, -90.0, -20.0, 0.0, 20.0, 90.0, 1e4, 3e38])
    x = v.to(torch.bfloat16)[:, None].to(dev)
    w = torch.ones(1, 1, dtype=torch.bfloat16, device=dev)
    for name in ("silu", "gelu"):
        y = capi.linear(x, w, activation=name, out_dtype=torch.float32).cpu()[:, 0]
        want = torch.where(v > 0, x.cpu()[:, 0].float(), torch.zeros(()))
        assert torch.isfinite(y).all() and (y - want).abs().max() <= 1.001 * 20 * math.exp(-20)


def test_nothing_to_do(dev):
    x, w, _, _ = make(dev, 4, 16, 32)
    assert capi.linear(x[:0], w).shape == (0, 16)
    assert pkg.backend.load().linear(x[:0], w).shape == (0, 16)


@pytest.mark.parametrize("T,n", [(1, 700), (16, 13_000), (17, 40), (17, 13_000), (100, 40), (800, 40),
                                 (800, 700), (12_300, 5)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_inputs_of_odd_length(dev, T, n, dtype):
    for k in (31, 33, 333, 1025):
        run(dev, T, n, k, dtype, "silu_and_mul" if k == 333 else "gelu", k != 31, k != 33, k == 1025)


@pytest.mark.parametrize("n", [2 ** 27 - 16, 2 ** 27, 2 ** 27 + 5])
def test_more_outputs_than_a_grid_of_few_tokens(dev, n):
    x = torch.full((1, 1), 3.0, dtype=torch.bfloat16, device=dev)
    w = (torch.arange(n, device=dev) % 251 - 125).to(torch.bfloat16).view(n, 1)
    assert torch.equal(capi.linear(x, w).view(-1), (w * 3.0).view(-1))  # one rounding on both sides


@pytest.mark.parametrize("T", [1, 7, 20, 60, 300])
def test_logits_of_a_vocabulary(dev, T):
    x, w, _, _ = make(dev, T, 151_936, 128)
    want, bound = ref.linear(x, w, out_dtype=torch.float32)
    ref.check(capi.linear(x, w, out_dtype=torch.float32), want, bound)


def test_rows_past_32_bits(dev):
    # Weight and output rows beyond 2^32 bytes and 2^31 elements.
    n, k, T = 300_000, 8192, 3
    w = torch.zeros(n, k, dtype=torch.bfloat16, device=dev)
    x, _, _, _ = make(dev, T, 1, k)
    at = [0, 131_071, 262_143, 262_144, 299_999]
    g = torch.Generator().manual_seed(5)
    w[at] = torch.randn(5, k, generator=g).to(torch.bfloat16).to(dev)
    got = capi.linear(x, w, out_dtype=torch.float32)
    want, bound = ref.linear(x, w[at], out_dtype=torch.float32)
    ref.check(got[:, at], want, bound)
    assert int((got != 0).sum()) <= 5 * T
    del w, got
    wide = torch.empty(70_000, 40_000, dtype=torch.bfloat16, device=dev)  # 2.8e9 outputs
    x = torch.randn(70_000, 8, generator=g).to(torch.bfloat16).to(dev)
    w = torch.randn(40_000, 8, generator=g).to(torch.bfloat16).to(dev)
    capi.linear(x, w, out=wide)
    at = torch.tensor([0, 53_687, 53_688, 69_999])
    want, bound = ref.linear(x[at.to(dev)], w)
    ref.check(wide[at.to(dev)], want, bound)


@pytest.mark.parametrize("T", [2, 20, 130, 600])
def test_backend_and_streams(dev, T):
    be = pkg.backend.load()
    x, w, b, r = make(dev, T, 320, 576, gated=True)
    want = capi.linear(x, w, b, "gelu_and_mul", r)
    assert torch.equal(be.linear(x, w, b, "gelu_and_mul", r), want)
    main, side = torch.cuda.current_stream(), torch.cuda.Stream()
    side.wait_stream(main)
    outs = []
    for i in range(8):  # two calls at once, each with its own workspace
        with torch.cuda.stream(side if i % 2 else main):
            outs.append(be.linear(x, w, b, "gelu_and_mul", r))
    main.wait_stream(side)
    for o in outs:
        assert torch.equal(o, want)


@pytest.mark.parametrize("T", [1, 24, 150, 700])
def test_captured_and_replayed(dev, T):
    be = pkg.backend.load()
    x, w, b, r = make(dev, T, 512, 1024)
    out = torch.empty(T, 512, dtype=x.dtype, device=dev)
    be.linear(x, w, b, "silu", r, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        be.linear(x, w, b, "silu", r, out=out)
    for i in range(4):
        x.copy_(make(dev, T, 512, 1024, seed=i + 1)[0])
        want = be.linear(x, w, b, "silu", r)
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_argument_checks(dev):
    x, w, b, r = make(dev, 4, 16, 32)
    be = pkg.backend.load()
    bad = [dict(x=x.float()), dict(w=w[:, :31]), dict(w=w.half()), dict(b=b[:15]), dict(r=r[:, :15]),
           dict(activation="relu"), dict(w=w[:15], activation="silu_and_mul"), dict(x=x.cpu()),
           dict(x=x.t()), dict(out_dtype=torch.float16)]
    for kw in bad:
        a = dict(x=x, w=w, b=b, r=r, activation="none", out_dtype=None)
        a.update(kw)
        with pytest.raises((ValueError, RuntimeError)):
            capi.linear(a["x"], a["w"], a["b"], a["activation"], a["r"], out_dtype=a["out_dtype"])
        with pytest.raises((ValueError, RuntimeError)):
            be.linear(a["x"], a["w"], a["b"], a["activation"], a["r"], out_dtype=a["out_dtype"])
