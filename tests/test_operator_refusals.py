"""What the shared-prefix step's operators refuse, and their host logic, without a GPU:
of these calls only a valid plan reaches the HIP runtime, for the device's CUs (256 where
there is none). Status codes: -1 invalid argument, -2
unsupported, -3 capacity, -4 alignment."""
import ctypes
import math
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from conftest import capi, pkg


def table(max_pos=16, rotary=8, base=1e4, cos=16, sin=16, **kw):
    sc = capi.rope_scaling(kw.pop("kind"), **kw) if kw else None
    return capi.lib().sgl_rope_scaled_cache(cos, sin, max_pos, rotary, base,
                                            None if sc is None else ctypes.byref(sc), None)


def test_scaled_table_refusals():
    assert table(max_pos=0, cos=None, sin=None) == 0
    assert table(cos=None) == table(max_pos=-1) == table(rotary=7) == table(rotary=0) == -1
    assert table(base=0.0) == table(base=math.inf) == table(base=math.nan) == -1
    assert table(rotary=514) == -2
    assert table(max_pos=2 ** 31 - 1, rotary=4, base=1e-12) == -2  # quarter turns past 31 bits
    for kind in ("linear", "ntk", "yarn", "bands"):
        for factor in (0.0, -1.0, math.nan, math.inf):
            assert table(kind=kind, factor=factor, original_max_position=99) == -1
    assert table(kind="ntk", factor=2.0, rotary=2) == -1
    assert table(kind="yarn", factor=2.0) == table(kind="bands", factor=2.0) == -1  # no original length
    ok = dict(factor=2.0, original_max_position=99)
    assert table(kind="yarn", base=1.0, **ok) == -1
    assert table(kind="yarn", beta_slow=0.0, **ok) == table(kind="yarn", beta_fast=0.5, **ok) == -1
    assert table(kind="yarn", attention_factor=-1.0, **ok) == -1
    assert table(kind="bands", low_freq_factor=4.0, **ok) == table(kind="bands", low_freq_factor=0.0, **ok) == -1
    bad = capi.RopeScaling(9, 0, 2.0)
    assert capi.lib().sgl_rope_scaled_cache(16, 16, 4, 8, 1e4, ctypes.byref(bad), None) == -2
    with pytest.raises(ValueError):
        capi.rope_scaling("cubic")


def append(**kw):
    a = dict(q=16, q_out=32, k=48, v=64, k_cache=80, v_cache=96, cos=112, sin=128, positions=144,
             out_loc=160, tokens=4, num_slots=9, max_pos=5, num_qo_heads=4, num_kv_heads=2,
             head_dim=64, rotary_dim=64, dtype=0, index_dtype=0, flags=0)
    a.update(kw)
    return capi.lib().sgl_rope_append(ctypes.byref(capi.RopeAppendArgs(**a)), None)


def test_rope_append_refusals():
    lib = capi.lib()
    assert lib.sgl_rope_append(None, None) == -1
    assert append(tokens=0, q=None, k=None) == 0
    assert append(num_qo_heads=0, num_kv_heads=0) == 0
    for name in ("q", "q_out", "k", "k_cache", "cos", "sin", "positions", "v", "v_cache"):
        assert append(**{name: None}) == -1, name
    for name in ("tokens", "num_slots", "max_pos", "num_qo_heads", "num_kv_heads", "head_dim"):
        assert append(**{name: -1}) == -1, name
    assert append(rotary_dim=63) == append(rotary_dim=66) == append(rotary_dim=0) == -1
    assert append(dtype=2) == append(index_dtype=2) == append(head_dim=1025, rotary_dim=2) == -2
    assert append(flags=2) == -1
    assert append(q_out=16, q_stride_token=256, q_out_stride_token=512) == -1  # in place, other strides


def plan(P=100, B=4, T=8, qo=2, hq=8, hkv=2, d=128):
    p = capi.PrefixPlan()
    return capi.lib().sgl_prefix_plan(P, B, T, qo, hq, hkv, d, ctypes.byref(p)), p


def test_prefix_plan():
    assert capi.lib().sgl_prefix_plan(1, 1, 1, 1, 1, 1, 128, None) == -1
    for kw in (dict(P=-1), dict(B=-1), dict(T=-1), dict(qo=-1), dict(hq=0), dict(hkv=0), dict(hkv=3)):
        assert plan(**kw)[0] == -1, kw
    for kw in (dict(d=64), dict(qo=capi.PREFIX_MAX_QO + 1), dict(hq=65, hkv=1), dict(T=1 << 29),
               dict(T=1 << 24, hq=1, hkv=1), dict(P=(1 << 29) + 1), dict(B=(1 << 25) + 1)):
        assert plan(**kw)[0] == -2, kw
    st, p = plan()
    assert st == 0 and p.num_blocks >= 1 and p.max_units >= 1 and p.workspace_bytes > 0
    assert plan(P=0)[0] == plan(B=0, T=0, qo=0)[0] == 0
    # Room for every row's own piece (128 fp32 values), whichever way the prefix goes.
    for T in (1, 8, 16, 17, 64, 700):
        st, p = plan(T=T)
        assert p.workspace_bytes >= T * 8 * 512 and p.prefix_rows > 0


def attend(p, **kw):
    a = dict(q=16, qs=1024, qh=128, k=32, v=48, ks=256, kh=128, pidx=64, idx=64, kvp=80, qop=96, B=4,
             T=8, hq=8, hkv=2, d=128, o=112, os=1024, oh=128, ws=256, wsb=p.workspace_bytes, scale=0.1)
    a.update(kw)
    return capi.lib().sgl_prefix_attention(
        ctypes.byref(p), a["q"], a["qs"], a["qh"], a["k"], a["v"], a["ks"], a["kh"], a["pidx"],
        a["idx"], a["kvp"], a["qop"], a["B"], a["T"], a["hq"], a["hkv"], a["d"], a["scale"], a["o"],
        a["os"], a["oh"], a["ws"], a["wsb"], None)


def test_prefix_attention_refusals():
    _, p = plan()
    assert capi.lib().sgl_prefix_attention(None, *[None] * 1, 0, 0, None, None, 0, 0, None, None, None,
                                           None, 1, 1, 8, 2, 128, 0.1, None, 0, 0, None, 0, None) == -1
    assert attend(p, B=0) == attend(p, T=0, q=None) == 0
    for name in ("q", "k", "v", "pidx", "kvp", "qop", "o"):
        assert attend(p, **{name: None}) == -1, name
    assert attend(p, B=-1) == attend(p, T=-1) == attend(p, hq=16) == attend(p, d=64) == -1
    assert attend(p, B=5) == attend(p, T=9) == -3
    assert attend(p, ws=None) == attend(p, wsb=p.workspace_bytes - 1) == -3
    assert attend(p, q=18) == attend(p, o=24) == attend(p, k=40) == attend(p, qs=1020) == -4
    assert attend(p, kh=100) == attend(p, oh=129) == attend(p, ws=264) == -4
    assert attend(p, ks=0) == -2
    for scale in (0.0, -0.1, float("inf"), float("nan")):
        assert attend(p, scale=scale) == -1, scale
    # A plan that was not made by sgl_prefix_plan.
    q = capi.PrefixPlan.from_buffer_copy(p)
    q.num_blocks = 0
    assert attend(q) == -1
    q = capi.PrefixPlan.from_buffer_copy(p)
    q.prefix_rows += 1
    assert attend(q) == -1


def verify(n=3, B=2, V=10, **kw):
    a = dict(target_probs=16, draft_probs=32, draft_tokens=48, draft_indptr=64, accept_uniform=80,
             sample_uniform=96, tokens=112, accepted=128, target_stride_row=V, draft_stride_row=V,
             num_drafts=n, batch_size=B, vocab=V)
    ws, wsb = kw.pop("ws", 16), kw.pop("wsb", 1 << 30)
    a.update(kw)
    return capi.lib().sgl_verify_drafts(ctypes.byref(capi.VerifyArgs(**a)), ws, wsb, None)


def test_verify_refusals():
    lib = capi.lib()
    assert lib.sgl_verify_drafts(None, 16, 1 << 20, None) == -1
    assert verify(n=0, B=0) == 0 and verify(n=1, B=0) == -1
    for name in ("target_probs", "draft_tokens", "draft_indptr", "accept_uniform", "sample_uniform",
                 "tokens", "accepted"):
        assert verify(**{name: None}) == -1, name
    assert verify(n=-1) == verify(B=-1) == verify(V=0) == -1
    assert verify(target_stride_row=9) == verify(draft_stride_row=9) == -1
    assert verify(B=65536) == verify(V=(1 << 24) + 1) == verify(n=0x7fffffff) == -2
    assert verify(ws=None) == verify(wsb=8) == -3 and verify(ws=24) == -4
    assert lib.sgl_verify_workspace_bytes(0, 5) == lib.sgl_verify_workspace_bytes(3, 0) == 0
    assert lib.sgl_verify_workspace_bytes(3, 5) > 0


def test_host_tensors_are_refused():
    z = torch.zeros
    with pytest.raises(ValueError):
        capi.rope_append(z(1, 1, 8), z(1, 1, 8), None, z(1, 1, 8), None, z(1, 4), z(1, 4),
                         z(1, dtype=torch.int32), None)
    with pytest.raises(ValueError):
        capi.verify_drafts(z(1, 4), None, z(0, dtype=torch.int32), z(2, dtype=torch.int32), z(0), z(1))
    be = pkg.backend.load()
    with pytest.raises(RuntimeError):
        be.rope_append(z(1, 1, 8), z(1, 1, 8), None, z(1, 1, 8), None, z(1, 4), z(1, 4),
                       z(1, dtype=torch.int32), None)
    with pytest.raises(RuntimeError):
        be.verify_drafts(z(1, 4), None, z(0, dtype=torch.int32), z(2, dtype=torch.int32), z(0), z(1))
    with pytest.raises(RuntimeError):
        be.rope_scaled_cache(4, 7, 1e4)


def test_refused_prefix_plans_do_not_ask_the_device():
    """A refused plan is refused from its numbers alone: the runtime's own log of calls, in a
    process of its own, holds none behind the mark (a valid plan asks for the device's CUs)."""
    root = Path(__file__).resolve().parents[1]
    code = """
import ctypes, sys
import __graft_entry__ as entry
capi = entry.load_package().capi
lib, p = capi.lib(), capi.PrefixPlan()
print("mark", file=sys.stderr, flush=True)
sizes = [(-1, 4, 8, 2, 8, 2, 128), (100, 4, 8, 2, 8, 3, 128), (100, 4, 8, 2, 8, 2, 64), (100, 4, 1 << 29, 2, 8, 2, 128)]
print(*(lib.sgl_prefix_plan(*x, ctypes.byref(p)) for x in sizes), lib.sgl_prefix_plan(*sizes[0], None))
print("mark", file=sys.stderr, flush=True)
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300,
                          env={**os.environ, "AMD_LOG_LEVEL": "3"})
    assert done.returncode == 0 and done.stdout.split() == ["-1", "-1", "-2", "-2", "-1"], done.stderr[-2000:]
    between = done.stderr.split("mark\n")
    assert len(between) == 3 and "hip" not in between[1], between[1]
