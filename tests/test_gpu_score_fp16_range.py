"""Attention with score rules in fp16 where the range of the format matters: gradients of keys whose value rows are small, and
outputs that many keys of small probability make up together."""
import math

import pytest
import torch

from oracle import scores as os_
from stof.scores import score_attn

pytestmark = pytest.mark.gpu


def _within(got, want, name):
    value, bound = want
    got = got.double().cpu()
    err = (got - value).abs()
    assert bool(torch.isfinite(got).all()), f"{name}: {int((~torch.isfinite(got)).sum())} of {got.numel()} are not finite"
    assert not bool((err > bound).any()), f"{name}: {int((err > bound).sum())} beyond the bound, worst {float((err / bound).max()):.2f} of it"


@pytest.mark.parametrize("small", [1e-3, 1e-5, 0.0])
@pytest.mark.parametrize("cap", [None, 20.0])
@pytest.mark.parametrize("D,Hq,Hkv,Sq", [(64, 1, 1, 64), (64, 4, 1, 300), (128, 1, 1, 64), (128, 4, 1, 300)])   # query tiles unsplit | split
def test_gradient_of_a_heavily_attended_key_with_a_small_value_row(small, cap, D, Hq, Hkv, Sq):
    """dT_ij = P_ij (dP_ij - delta_i), and delta_i follows the other keys' values: it is not small where V_j is."""
    g = torch.Generator().manual_seed(31)
    n = lambda *s: torch.randn(*s, generator=g)
    Sk, sink = 150, 70
    along = torch.zeros(D)
    along[0] = 1.0
    q = (n(1, Hq, Sq, D) * 0.3 + along).half()
    k = n(1, Hkv, Sk, D).half()
    k[:, :, sink] = (along * 5.0 * math.sqrt(D)).half()         # about half of every query's probability
    v, dout = (n(1, Hkv, Sk, D).abs() + 0.5), (n(1, Hq, Sq, D).abs() + 0.5)
    v[:, :, sink] *= small
    v, dout = v.half(), dout.half()
    want = os_.score_attn(q, k, v, cap=cap, dout=dout)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(score_attn(*leaves, cap=cap), leaves, dout.cuda())
    for name, got in zip(("dq", "dk", "dv"), grads):
        _within(got, want[name], name)


@pytest.mark.parametrize("form", ["wide", "wide2", "rows"])
@pytest.mark.parametrize("D,N,top", [(64, 65536, 0), (64, 65541, 65540), (128, 65536, 30000), (64, 5000, 4999)])
def test_many_keys_of_small_probability(form, D, N, top):
    """One key at score 0 with a value of zeros, N - 1 at -17.5 with ones: each has the probability 2^-25.2 of the first, all of
    them together 1.6e-3 at 65536.  P is carried times 2^7 relative to a maximum that lags by up to 2^8, so a small P is off by at
    most 2^-25 / 2^7 = 2^-32 of the top; the scores are exact products, in log2 units off by 2 x 2^-24 x 25.  The sum of P is one
    of fp32: a wave of the wide forms adds N / 64 tiles to it, each with a rounding of at most 2^-24 of the sum (about 1, all
    alike here, so that they add up: 6.1e-5 at 65536)."""
    q, k, v = torch.zeros(1, 1, 1, D), torch.zeros(1, 1, N, D), torch.ones(1, 1, N, D)
    q[..., 0] = 1.0
    k[..., 0] = -17.5
    k[0, 0, top] = 0.0
    v[0, 0, top] = 0.0
    out, lse = score_attn(*(t.half().cuda() for t in (q, k, v)), scale=1.0, return_lse=True, launch_form=form)
    rest = (N - 1) * math.exp(-17.5)
    want = rest / (1.0 + rest)
    total = (N / 64 + 1) * 2.0 ** -24 * (1.0 + rest)
    bound = N * 2.0 ** -32 + (2.0 ** -11 + 2.0 ** -17 + total) * want + 2.0 ** -25
    assert bool(((out.double().cpu() - want).abs() <= bound).all()), (float(out[0, 0, 0, 0]), want, bound)
    assert abs(float(lse) - math.log1p(rest)) <= total + 2.0 ** -20 + 2.0 ** -17 * rest
