"""Calls with more workgroups than one dimension of a grid holds (fewer than 2^32 threads), and
rows further apart than 32-bit offsets reach."""
import pytest
import torch

import layer_refs as ref
from conftest import capi, pkg
from test_gpu_moe import make as make_experts

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def pattern(n, k, dev):
    """[n, k] of small whole numbers that change from row to row and from column to column."""
    w = torch.empty(n, k, dtype=torch.bfloat16, device=dev)
    for a in range(0, n, 1 << 26):
        i = torch.arange(a, min(n, a + (1 << 26)), device=dev, dtype=torch.int32)
        for c in range(k):
            w[a:a + len(i), c] = ((i + 37 * c) % 251 - 125).to(torch.bfloat16)
    return w


# At 256 threads a workgroup: 32 (gated 16) outputs of the streams, 64 of the tiles of any layout.
@pytest.mark.parametrize("n,k,activation", [(2 ** 29 + 40, 8, "none"), (2 ** 28 + 24, 8, "silu_and_mul"),
                                            (2 ** 30 + 70, 1, "none")])
def test_outputs_past_a_grid(dev, n, k, activation):
    gated = activation != "none"
    w = pattern(2 * n if gated else n, k, dev)
    x = torch.zeros(1, k, dtype=torch.bfloat16, device=dev)
    x[0, 0], x[0, k - 1] = 2 ** -7, 2 ** -5
    out = torch.full((1, n + 64), 9.0, dtype=torch.bfloat16, device=dev)
    capi.linear(x, w, activation=activation, out=out[:, :n])
    assert (out[0, n:] == 9).all()
    for a in (0, n // 2 - 999, 2 ** 28 - 500, n - 5000):
        at = torch.arange(a, min(n, a + 5000), device=dev)
        rows = w[torch.cat((at, at + n)) if gated else at]
        ref.check(out[:, at], *ref.linear(x, rows, activation=activation))
    want = (w[:n].float() * x[0].float()).sum(1) if k == 1 else None
    if want is not None:
        assert torch.equal(out[0, :n], want.bfloat16())


def test_tokens_past_a_grid_choose(dev):
    T = 2 ** 28 + 19
    logits = pattern(T, 2, dev)
    weights, experts = capi.moe_route(logits, 1, False)
    assert torch.equal(experts[:, 0] == 1, logits[:, 1] > logits[:, 0])
    for a in (0, 2 ** 28 - 500, T - 1000):
        want, ids = ref.route(logits[a:a + 1000], 1, False)
        assert torch.equal(experts[a:a + 1000].cpu(), ids)
        bound = want * ref.U * 1024 + 2.0 ** -148  # differences of whole numbers below 2^8 are exact
        ref.check(weights[a:a + 1000], want, bound)


def test_tokens_past_a_grid_through_experts(dev):
    T = 2 ** 24 + 300
    x, gu, d, _, _ = make_experts(dev, 4, 3, 1, 8, 8)
    x = pattern(T, 8, dev) / 128
    ids = (torch.arange(T, device=dev, dtype=torch.int32) * 7 % 3).view(T, 1).contiguous()
    w = torch.full((T, 1), 0.75, device=dev)
    out = torch.full((T + 8, 8), 9.0, dtype=torch.bfloat16, device=dev)
    capi.moe_experts(x, gu, d, w, ids, residual=x, out=out[:T])
    assert (out[T:] == 9).all()
    for a in (0, 2 ** 23, 2 ** 24 - 700, T - 1000):
        s = slice(a, a + 1000)
        ref.check(out[s], *ref.experts(x[s], gu, d, w[s], ids[s], x[s]))
    # The pattern repeats after 251 rows, the experts after 3.
    assert torch.equal(out[753:T], out[:T - 753])


# 65,536 experts' tiles by 256 of outputs: 128 x 64 tiles (64 gated outputs), and any layout's (32).
@pytest.mark.parametrize("H,I", [(8, 16_384), (7, 8_190)])
def test_experts_past_a_grid(dev, H, I):
    E, T = 65_536, 1100
    at = torch.tensor([0, 1, 40_001, E - 1], device=dev)
    x, gu, d, w, ids = make_experts(dev, T, 4, 1, H, I)
    many_gu = torch.empty(E, 2 * I, H, dtype=x.dtype, device=dev)  # experts of no token are not read
    many_d = torch.empty(E, H, I, dtype=x.dtype, device=dev)
    many_gu[at], many_d[at] = gu, d
    got = capi.moe_experts(x, many_gu, many_d, w, at[ids.long()].int())
    ref.check(got, *ref.experts(x, gu, d, w, ids))


# Of x 2^30 - 1 elements are in the tiles' reach: 1,023 rows of the first, 262,143 of the second.
@pytest.mark.parametrize("T,H,I,stride,part", [(1100, 200, 72, 2 ** 20, 1023),
                                               (262_200, 4096, 72, 4096, 262_143)])
def test_rows_past_32_bit_offsets_are_calls_of_their_parts(dev, T, H, I, stride, part):
    x, gu, d, w, ids = make_experts(dev, T, 4, 2, H, I)
    far = torch.empty(T * stride, dtype=x.dtype, device=dev).as_strided((T, H), (stride, 1))
    far.copy_(x)
    out = x.clone()
    assert capi.moe_experts(far, gu, d, w, ids, residual=out, out=out) is out
    for s in (slice(0, part), slice(part, T)):
        want = capi.moe_experts(x[s], gu, d, w[s].contiguous(), ids[s].contiguous(), residual=x[s])
        assert torch.equal(out[s], want)
    for s in (slice(0, 50), slice(part - 20, part + 20), slice(T - 50, T)):
        ref.check(out[s], *ref.experts(x[s], gu, d, w[s], ids[s], x[s]))


def test_sizes_past_32_bits_are_refused(dev):
    """2^32 + 8 is not 8: nothing is launched for a size that its 32-bit argument would cut."""
    be = pkg.backend.load()
    logits = torch.empty(0, 16, dtype=torch.float32, device=dev)
    wide = torch.empty(0, 2 ** 32 + 8, dtype=torch.float32, device=dev)
    x, gu, d, _, _ = make_experts(dev, 1, 4, 2, 16, 8)
    choices = torch.empty(0, 2 ** 32 + 2, device=dev), torch.empty(0, 2 ** 32 + 2, dtype=torch.int32, device=dev)
    for f in (capi, be):
        for bad in ((logits, 2 ** 32 + 2), (logits, 17), (logits, 0), (wide, 2)):
            with pytest.raises((ValueError, RuntimeError)):
                f.moe_route(*bad)
        with pytest.raises((ValueError, RuntimeError)):
            f.moe_experts(x[:0], gu, d, *choices)
