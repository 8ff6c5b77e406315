"""Refusals of attention with score rules that need no GPU: the mask object and the C ABI's host-side checks."""
import ctypes

import pytest
import torch

from stof import _lib
from stof.ops import StofError
from stof.scores import ScoreMask, score_attn


def test_mask_object():
    i = torch.zeros(2, dtype=torch.int32)
    d = torch.zeros(2, 5, dtype=torch.int32)
    ScoreMask(causal=True, prefix=i, kv_len=i, docs=d, q_start="end")
    ScoreMask(docs=(d, torch.zeros(2, 9, dtype=torch.int32)), q_start=-4)
    for kw in (dict(kv_len=i.long()), dict(kv_len=d), dict(kv_len=[1, 2]), dict(prefix=i), dict(causal=True, prefix=i.float()),
               dict(docs=i), dict(docs=d.long()), dict(docs=d.t()), dict(docs=(d, None)), dict(q_start="start"), dict(q_start=1.0),
               dict(q_start=True), dict(q_start=1 << 30), dict(q_start="end"), dict(kv_len=torch.zeros(4, dtype=torch.int32)[::2])):
        with pytest.raises(StofError):
            ScoreMask(**kw)


def test_no_cpu_path():
    x = torch.zeros(1, 1, 1, 64, dtype=torch.float16)
    with pytest.raises(StofError):
        score_attn(x, x, x)


@pytest.fixture(params=["ctypes", "ext"])
def lib(request):
    h = _lib.lib(request.param)
    if h is None:
        pytest.skip("extension module not built")
    return h, request.param


P = 4096   # fake, 16-byte aligned, never dereferenced: validation fails first


def test_forward_argument_checks(lib):
    h, kind = lib
    s3 = lambda a, b, c: (a, b, c) if kind == "ext" else (ctypes.c_int64 * 3)(a, b, c)
    st = s3(4 * 8 * 64, 8 * 64, 64)

    def call(**kw):
        g = kw.get
        return h.stof_score_attn_fwd(g("q", P), P, P, P, None, g("table"), g("slopes"), None, g("kv_len"), g("dq"), g("dk"),
                                     g("scale", 0.125), g("cap", 0.0), g("radius", -1), 0, g("start", 0), g("end", 0),
                                     g("qs", st), st, st, st, g("B", 2), g("Hq", 4), g("Hkv", 2), g("Sq", 8), g("Sk", 8), g("D", 64),
                                     g("dtype", 0), g("form", -1), g("ws"), g("bytes", 0), None)
    assert call(q=None) == -1
    assert call(q=P + 2) == -4
    assert call(qs=s3(4 * 8 * 64, 8 * 64, 65)) == -4
    assert call(qs=s3(4 * 8 * 64, 8 * 64, 1 << 24)) == -2
    assert call(qs=s3(-64, 64, 64)) == -4
    for kw in (dict(B=0), dict(Hq=3), dict(Sq=0), dict(Sk=-1), dict(B=1 << 20, Hq=1 << 10, Sq=1 << 20), dict(start=1 << 30), dict(table=P)):
        assert call(**kw) == -2, kw
    for kw in (dict(D=96), dict(dtype=2), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(cap=-1.0), dict(cap=float("inf")),
               dict(cap=1025.0), dict(cap=1e-4), dict(scale=1e7),
               dict(table=P, radius=1025), dict(table=P, radius=4, slopes=P), dict(form=3)):
        assert call(**kw) == -3, kw
    assert call(dq=P) == -1 and call(end=1) == -1
    assert call(dq=P, dk=P) == -1                                  # documents need a workspace
    assert call(dq=P, dk=P, ws=P, bytes=8) == -2
    assert h.stof_score_attn_workspace_bytes(2, 4, 2, 8, 8, 64, 0, -1) == 0
    assert h.stof_score_attn_workspace_bytes(2, 4, 2, 100, 200, 64, 1, 0) == 2 * (2 + 4) * 16
    assert h.stof_score_attn_workspace_bytes(1, 8, 2, 1, 100000, 64, 0, -1) > 0     # split along the keys
    assert h.stof_score_attn_workspace_bytes(2, 4, 3, 8, 8, 64, 0, -1) == 0


def test_backward_argument_checks(lib):
    h, kind = lib
    st = (4 * 8 * 64, 8 * 64, 64) if kind == "ext" else (ctypes.c_int64 * 3)(4 * 8 * 64, 8 * 64, 64)

    def call(**kw):
        g = kw.get
        return h.stof_score_attn_bwd(g("dout", P), P, P, P, P, P, g("dq", P), P, P, g("dtable"), g("table"), None, None, g("kv_len"), None, None,
                                     0.125, 0.0, g("radius", -1), 0, 0, g("end", 0), st, st, st, st, st, 2, 4, 2, 8, g("Sk", 8), g("D", 64), 0,
                                     g("ws", P), g("bytes", 8), None)
    assert call(dout=None) == -1 and call(dq=None) == -1 and call(ws=None) == -1
    assert call(table=P, radius=4) == -1 and call(end=1) == -1
    assert call(D=32) == -3
    assert call(Sk=0) == -2
    assert call() == -2                                            # workspace too small
    need = h.stof_score_attn_bwd_workspace_bytes(2, 4, 2, 100, 200, 64, 16, 1)
    assert need >= 2 * (2 + 4) * 16 + 2 * 4 * 128 * 8 + 2 * 4 * 2 * 33 * 4
    assert h.stof_score_attn_bwd_workspace_bytes(2, 4, 3, 100, 200, 64, 16, 1) == 0
