"""The float64 oracle of attention with score rules against autograd, finite differences and the existing dense oracle."""
import math

import pytest
import torch

from oracle import attention as oa, scores as os_


def _inputs(B=2, Hq=4, Hkv=2, Sq=9, Sk=13, D=8, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    return n(B, Hq, Sq, D), n(B, Hkv, Sk, D), n(B, Hkv, Sk, D), n(B, Hq, Sq, D), n(Hq, 7)


RULES = [dict(), dict(causal=True), dict(causal=True, prefix=torch.tensor([3, 7])), dict(kv_len=torch.tensor([5, 0])),
         dict(kv_len=torch.tensor([13, 4]), q_start="end", causal=True), dict(q_start=-3, causal=True)]


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("cap", [None, 1.5])
@pytest.mark.parametrize("what", ["table", "slopes", "none"])
def test_gradients_against_autograd_and_differences(rule, cap, what):
    q, k, v, dout, tab = _inputs()
    kw = dict(cap=cap, bias=tab if what == "table" else None, slopes=torch.rand(4) if what == "slopes" else None, **rule)
    got = os_.score_attn(q, k, v, dout=dout, **kw)
    names = ["dq", "dk", "dv"] + (["dbias"] if what == "table" else [])
    args = [q, k, v] + ([tab] if what == "table" else [])

    def loss(*a):
        kk = dict(kw)
        if what == "table":
            kk["bias"] = a[3]
        return (os_.score_attn(*a[:3], **kk)["out"][0] * dout).sum()

    g = torch.Generator().manual_seed(5)
    for x, name in enumerate(names):
        d = torch.randn(args[x].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        up, dn = list(args), list(args)
        up[x], dn[x] = args[x] + h * d, args[x] - h * d
        want = (loss(*up) - loss(*dn)) / (2 * h)
        assert abs(float((got[name][0] * d).sum() - want)) <= 1e-6 * max(1.0, abs(float(want))), name
    if not cap and what == "none":
        # torch's own softmax and autograd on the rows that have keys
        ok, _ = os_.allowed(2, 9, 13, **rule)
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        s = (leaves[0] @ leaves[1].repeat_interleave(2, 1).transpose(-1, -2)) / math.sqrt(8)
        p = torch.softmax(s.masked_fill(~ok[:, None], -1e300), -1) * ok.any(-1)[:, None, :, None]
        out = p @ leaves[2].repeat_interleave(2, 1)
        assert torch.allclose(out, got["out"][0], atol=1e-12)
        for a, b in zip(torch.autograd.grad(out, leaves, dout), names):
            assert torch.allclose(a, got[b][0], atol=1e-10), b


def test_agrees_with_the_dense_mask_oracle():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, 2, 64, 16, generator=g) for _ in range(3))
    want = oa.dense_masked_attention(q, k, v, torch.ones(64, 64).tril().bool())
    got = os_.score_attn(q, k, v, causal=True)["out"][0]
    assert (got - want).abs().max() < 1e-5


def test_documents_and_positions_by_hand():
    docs = torch.tensor([[0, 0, 7, 7, -1, 0]], dtype=torch.int32)
    ok, pos = os_.allowed(1, 6, 6, docs=docs, causal=True)
    want = torch.tensor([[1, 0, 0, 0, 0, 0], [1, 1, 0, 0, 0, 0], [0, 0, 1, 0, 0, 0], [0, 0, 1, 1, 0, 0], [0] * 6, [1, 1, 0, 0, 0, 1]]).bool()
    assert torch.equal(ok[0], want)
    ok, pos = os_.allowed(2, 2, 5, kv_len=torch.tensor([4, 1]), q_start="end", causal=True)
    assert pos.tolist() == [[2, 3], [-1, 0]]
    assert ok.int().tolist() == [[[1, 1, 1, 0, 0], [1, 1, 1, 1, 0]], [[0] * 5, [1, 0, 0, 0, 0]]]
    one = os_.score_attn(torch.ones(1, 1, 1, 64), torch.ones(1, 1, 3, 64), torch.ones(1, 1, 3, 64), slopes=torch.tensor([1.0]))
    assert abs(float(one["lse"][0]) - (8 + math.log(1 + math.exp(-1) + math.exp(-2)))) < 1e-12
