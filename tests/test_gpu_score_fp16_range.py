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
