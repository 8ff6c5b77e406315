"""Forward-mode derivatives: the score attention and the 8-bit operators have none and say so."""
import pytest
import torch

from stof.ops import StofError
from stof.quant import gemm_i8, linear_i8, quantize_rows_i8
from stof.scores import score_attn, score_attn_backward

pytestmark = pytest.mark.gpu
fw = torch.autograd.forward_ad
h = lambda *s, d=torch.float16: torch.zeros(*s, dtype=d, device="cuda")
dual = lambda t: fw.make_dual(t, torch.ones_like(t))


def test_score_attention():
    x, tab, slopes = h(1, 2, 8, 64), h(2, 5), h(2, d=torch.float32)
    with fw.dual_level():
        for call in (lambda: score_attn(dual(x), x, x), lambda: score_attn(x, dual(x), x), lambda: score_attn(x, x, dual(x)),
                     lambda: score_attn(x, x, x, bias=dual(tab)), lambda: score_attn(x, x, x, slopes=dual(slopes)),
                     lambda: score_attn(dual(x), x.clone().requires_grad_(), x),
                     lambda: score_attn_backward(dual(x), x, x, x, x, h(1, 2, 8, d=torch.float32))):
            with pytest.raises(StofError, match="tangent"):
                call()
        score_attn(x, x, x, bias=tab)           # no tangent: as ever


def test_8_bit_operators():
    x, w, s, b = h(4, 64), h(16, 64, d=torch.int8), h(16, d=torch.float32), h(16)
    with fw.dual_level():
        for call in (lambda: linear_i8(dual(x), w, s, b), lambda: linear_i8(x, w, dual(s), b), lambda: linear_i8(x, w, s, dual(b)),
                     lambda: quantize_rows_i8(dual(x)), lambda: gemm_i8(w[:4], dual(s[:4]), w, s, b), lambda: gemm_i8(w[:4], s[:4], w, dual(s), b),
                     lambda: gemm_i8(w[:4], s[:4], w, s, dual(b))):
            with pytest.raises(StofError, match="tangent"):
                call()
        linear_i8(x, w, s, b)
