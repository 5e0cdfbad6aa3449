"""The weighted outputs of a token's slots keep fp32's precision up to their sum, whatever their
neighbours' size and however many tokens there are. What lies between the projections is
exact in 16 bits here, so that nothing else is rounded before the result."""
import pytest
import torch

import layer_refs as ref
from conftest import capi

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def make(dev, T, E, K, H, I, dtype):
    """Inputs whose h has eight entries, powers of two that differ by expert; the others are zero."""
    g = torch.Generator().manual_seed(T + H)
    x, gu, d = torch.zeros(T, H), torch.zeros(E, 2 * I, H), torch.randn(E, H, I, generator=g)
    x[:, 5] = 1
    at = torch.arange(8) * (I // 8)
    gu[:, at, 5] = 32  # silu(32) is 32 to 2^-40
    sign = torch.randint(0, 2, (E, 8), generator=g) * 2 - 1
    gu[:, I + at, 5] = sign * 2.0 ** torch.randint(-6, -2, (E, 8), generator=g)
    ids = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]).int()
    w = torch.randn(T, K, generator=g)
    return (*(t.to(DT[dtype]).to(dev) for t in (x, gu, d)), w.to(dev), ids.to(dev))


def sums(x, gu, d, w, ids):
    """(result, bound) in 64 bits: products of 16-bit values are exact, I of them are summed
    (two more roundings for a sum over waves and its weight), K terms too, then one rounding to the
    type (half of its smallest step at least)."""
    I = d.shape[2]
    both = x.double().cpu() @ gu.double().cpu().transpose(1, 2)  # [E, T, 2 I]
    g = both[..., :I]
    assert set(g.unique().tolist()) == {0.0, 32.0}
    h = g * both[..., I:]
    dc, wc, ic = d.double().cpu(), w.double().cpu(), ids.cpu().long()
    y, size = torch.zeros(x.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64)
    for j in range(ids.shape[1]):
        for e in range(d.shape[0]):
            t = torch.nonzero(ic[:, j] == e)[:, 0]
            y[t] += wc[t, j, None] * (h[e, t] @ dc[e].t())
            size[t] += wc[t, j, None].abs() * (h[e, t].abs() @ dc[e].abs().t())
    eps = ref.half_step(x.dtype)
    return y, (I + ids.shape[1] + 4) * ref.U * size * 1.01 + eps * y.abs() * 1.01 \
        + torch.finfo(x.dtype).smallest_normal * eps * 2


@pytest.mark.parametrize("T", [1, 3, 60, 130, 400, 1100])
@pytest.mark.parametrize("H,I", [(192, 64), (200, 72)])
def test_small_outputs_beside_large_ones_bf16(dev, T, H, I):
    x, gu, d, w, ids = make(dev, T, 4, 2, H, I, "bf16")
    rows = 2.0 ** -(torch.arange(H, device=dev) * 7 % 48).float()
    d = (d.float() * rows[None, :, None]).bfloat16()
    ref.check(capi.moe_experts(x, gu, d, w, ids), *sums(x, gu, d, w, ids))


@pytest.mark.parametrize("T", [1, 3, 60, 130, 400, 1100])
def test_small_outputs_beside_large_ones_fp16(dev, T):
    x, gu, d, w, ids = make(dev, T, 4, 2, 192, 64, "fp16")
    rows = 2.0 ** (6 - (torch.arange(192, device=dev) * 7 % 16)).float()
    d = (d.float() * rows[None, :, None]).half()
    ref.check(capi.moe_experts(x, gu, d, w, ids), *sums(x, gu, d, w, ids))


@pytest.mark.parametrize("T", [3, 60, 130, 400, 1100])
def test_large_terms_that_cancel(dev, T):
    """65,537 - 65,536, of which no 16-bit type has the first."""
    x, gu, d, w, ids = make(dev, T, 2, 2, 128, 64, "bf16")
    gu.zero_(), d.zero_()
    gu[:, :64, 5], gu[:, 64:, 5] = 32, 1
    d[:, :, 3], d[0, :, 40] = 2.0 ** 11, 2.0 ** -5
    w.copy_(torch.where(ids == 0, 1.0, -1.0))
    assert (capi.moe_experts(x, gu, d, w, ids) == 1).all()
