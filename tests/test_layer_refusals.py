"""What the projections' and experts' entry points refuse, without a GPU: none of these
calls reaches the HIP runtime. Status codes: -1 invalid argument, -2 unsupported,
-3 capacity, -4 alignment."""
import ctypes

from conftest import capi


def linear(ws=None, ws_bytes=0, **kw):
    a = dict(x=256, weight=512, bias=None, residual=None, out=1024, tokens=4, n=8, k=16,
             x_stride_row=16, weight_stride_row=16, residual_stride_row=8, out_stride_row=8,
             dtype=0, out_dtype=0, activation=0, reserved=0)
    a.update(kw)
    return capi.lib().sgl_linear(ctypes.byref(capi.LinearArgs(**a)), ws, ws_bytes, None)


def test_linear_refusals():
    assert capi.lib().sgl_linear(None, None, 0, None) == -1
    assert linear(tokens=0) == 0 and linear(tokens=0, x=None, weight=None, out=None) == 0
    for name in ("x", "weight", "out"):
        assert linear(**{name: None}) == -1, name
    assert linear(tokens=-1) == linear(n=0) == linear(k=0) == linear(reserved=1) == -1
    assert linear(dtype=2) == linear(out_dtype=1) == linear(activation=5) == linear(activation=-1) == -2
    assert linear(tokens=2 ** 31) == linear(n=2 ** 31, out_stride_row=2 ** 31) == -2
    assert linear(k=2 ** 31, x_stride_row=2 ** 31, weight_stride_row=2 ** 31) == -2
    for name in ("x_stride_row", "weight_stride_row", "out_stride_row"):
        assert linear(**{name: 7}) == -1, name
    assert linear(residual=2048, residual_stride_row=7) == -1
    assert linear(out=256) == -1                                # over x
    assert linear(residual=1024, residual_stride_row=9) == -1   # in place, other strides
    assert linear(residual=1024, out_dtype=2) == -1             # in place, other type
    # More workgroups than a grid has.
    assert linear(tokens=2 ** 31 - 256, n=2 ** 31 - 256, out_stride_row=2 ** 31) == -2


def test_linear_workspace():
    need = capi.lib().sgl_linear_workspace_bytes
    for T in (1, 7, 64, 65, 300, 1000, 5000):
        for n, k in ((64, 64), (2048, 4096), (4096, 12288), (7, 9)):
            for act in range(5):
                b = need(T, n, k, act)
                assert b >= 0 and b % 16 == 0
                if b:
                    a = dict(tokens=T, n=n, k=k, x_stride_row=k, weight_stride_row=k,
                             out_stride_row=n, activation=act)
                    assert linear(4096, b - 1, **a) == -3
                    assert linear(4100, b, **a) == -4
    assert need(-1, 4, 4, 0) == need(4, 0, 4, 0) == need(4, 4, 0, 0) == need(4, 4, 4, 9) == 0


def route(**kw):
    a = dict(logits=256, stride=16, dtype=2, tokens=4, experts=16, top_k=4, renormalize=1,
             weights=512, ids=1024)
    a.update(kw)
    return capi.lib().sgl_moe_route(*a.values(), None)


def test_route_refusals():
    assert route(tokens=0, logits=None) == 0
    assert route(logits=None) == route(weights=None) == route(ids=None) == -1
    assert route(tokens=-1) == route(experts=0) == route(top_k=0) == route(top_k=17) == -1
    assert route(stride=15) == -1
    assert route(dtype=3) == route(dtype=-1) == -2
    assert route(experts=513, stride=600) == route(experts=64, stride=64, top_k=33) == -2


def moe(ws=4096, ws_bytes=1 << 40, **kw):
    a = dict(x=256, gate_up=512, down=768, weights=1024, experts=1280, residual=None, out=1536,
             tokens=4, x_stride_row=16, residual_stride_row=16, out_stride_row=16,
             gate_up_stride_expert=256, gate_up_stride_row=16, down_stride_expert=128,
             down_stride_row=8, top_k=2, num_experts=6, hidden=16, intermediate=8, dtype=0,
             activation=3)
    a.update(kw)
    return capi.lib().sgl_moe_experts(ctypes.byref(capi.MoeArgs(**a)), ws, ws_bytes, None)


def test_experts_refusals():
    assert capi.lib().sgl_moe_experts(None, None, 0, None) == -1
    assert moe(tokens=0, x=None, ws=None) == 0
    for name in ("x", "gate_up", "down", "weights", "experts", "out"):
        assert moe(**{name: None}) == -1, name
    assert moe(tokens=-1) == moe(top_k=0) == moe(num_experts=0) == moe(hidden=0) == moe(intermediate=0) == -1
    assert moe(dtype=2) == moe(activation=0) == moe(activation=2) == moe(activation=5) == -2
    assert moe(num_experts=65537) == moe(hidden=2 ** 21) == moe(intermediate=2 ** 21) == -2
    assert moe(tokens=2 ** 30, top_k=2) == -2
    for name in ("x_stride_row", "out_stride_row", "gate_up_stride_row", "down_stride_row",
                 "gate_up_stride_expert", "down_stride_expert"):
        assert moe(**{name: 7}) == -1, name
    assert moe(residual=2048, residual_stride_row=15) == -1
    assert moe(out=256) == -1 and moe(residual=1536, residual_stride_row=17) == -1
    need = capi.lib().sgl_moe_workspace_bytes(4, 2, 6, 16, 8)
    assert need > 0
    assert moe(ws=None) == moe(ws_bytes=need - 1) == -3
    assert moe(ws=4104, ws_bytes=need) == -4
    assert capi.lib().sgl_moe_workspace_bytes(-1, 2, 6, 16, 8) == 0
