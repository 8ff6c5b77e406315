"""The encoder layer with a score rule and with 8-bit linear operators: the operators together, as a model uses them."""
import subprocess
import sys

import pytest
import torch

from oracle import scores as os_
from stof import configs, fused, masks as pm
from stof.layer import CapturedForward, EncoderLayer, EncoderStack, eager_layer
from stof.ops import StofError
from stof.quant import linear_i8, quantize_rows_i8
from stof.scores import ScoreMask, score_attn

pytestmark = pytest.mark.gpu
D, H, F = 256, 4, 512


def _weights(seed=0, dtype=torch.float16):
    return {k: v.to(dtype).cuda() for k, v in configs.layer_weights(D, F, seed=seed).items()}


def _x(B, S, dtype=torch.float16, seed=1):
    return torch.randn(B, S, D, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _table(dtype=torch.float16):
    return torch.randn(H, 2 * 16 + 1, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()


@pytest.mark.parametrize("S", [64, 150])
def test_layer_with_a_table_and_key_lengths(S):
    """16-bit linear operators: against the plain layer in fp32 on the same fp16 inputs.  Rounding points as in the
    encoder tests (five fp16 tensors between kernels): the same bound, 2e-3 + 1e-2 |want|, on the rows that exist."""
    B = 3
    w, x, tab = _weights(), _x(B, S), _table()
    lens = torch.tensor([S, S // 2, 1], dtype=torch.int32)
    m = ScoreMask(kv_len=lens.cuda())
    got = EncoderLayer(w, H, scores=dict(bias=tab))(x, m)
    at = torch.arange(S)
    dense = tab.float().cpu()[:, (at[None, :] - at[:, None]).clamp(-16, 16) + 16]
    mask = (at[None, :] < lens[:, None])[:, None, :].expand(B, S, S).float()
    want = eager_layer(x.float().cpu(), {k: v.float().cpu() for k, v in w.items()}, mask, H, bias=dense)
    err = (got.float().cpu() - want).abs()
    assert bool((err <= 2e-3 + 1e-2 * want.abs()).all()), float(err.max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,S", [(1, 1), (2, 150)])
def test_int8_layer_is_its_operators_in_sequence(B, S, dtype):
    w, x, tab = _weights(dtype=dtype), _x(B, S, dtype), _table(dtype)
    docs = torch.zeros(B, S, dtype=torch.int32, device="cuda")
    docs[:, S // 2:] = 1
    m = ScoreMask(causal=True, docs=docs)
    layer = EncoderLayer(w, H, scores=dict(bias=tab, cap=20.0), linear="int8", gelu="tanh")
    got = layer(x, m)
    q8 = {k: quantize_rows_i8(w[k].t().contiguous()) for k in ("W_qkv", "W_o", "W_1", "W_2")}
    qkv = linear_i8(x, *q8["W_qkv"], w["b_qkv"])
    q, k, v = (t.view(B, S, H, D // H).permute(0, 2, 1, 3) for t in qkv.chunk(3, -1))
    a = score_attn(q, k, v, m, bias=tab, cap=20.0).permute(0, 2, 1, 3).reshape(B, S, D)
    h = fused.bias_residual_layernorm(linear_i8(a, *q8["W_o"]), w["b_o"], x, w["g1"], w["be1"], 1e-12)
    f = linear_i8(h, *q8["W_1"], w["b_1"], act="gelu_tanh")
    want = fused.bias_residual_layernorm(linear_i8(f, *q8["W_2"]), w["b_2"], h, w["g2"], w["be2"], 1e-12)
    assert torch.equal(got, want)
    for name, fn in layer.stages(x, m):
        fn()
    # and the attention inside it against the oracle on the projection the layer computed
    ref = os_.score_attn(q.cpu(), k.cpu(), v.cpu(), causal=True, docs=docs.cpu(), bias=tab.cpu(), cap=20.0)["out"]
    err = (a.view(B, S, H, D // H).permute(0, 2, 1, 3).double().cpu() - ref[0]).abs()
    assert bool((err <= ref[1]).all())


def test_int8_layer_on_a_block_mask():
    """8-bit linear operators around the block-masked attention, near the 16-bit layer: each linear operator's error is
    that of rounding rows of ~N(0,1) values (largest about 4) to steps of a/127, 4/127/sqrt(12) = 0.9 % of their
    size, and as much for the weights; four of them in sequence, LayerNorms between: 5 % in the 2-norm."""
    B, S = 2, 256
    w, x = _weights(), _x(2, 256)
    lut = pm.get_sparse_storage(configs.mask_c5(S).float()[None].cuda(), 64, 64)[1:]
    a, b = EncoderLayer(w, H)(x, lut), EncoderLayer(w, H, linear="int8")(x, lut)
    assert float((a.float() - b.float()).norm() / a.float().norm()) < 0.05


def test_stack_captured_into_a_graph():
    ws = [_weights(seed=s) for s in range(3)]
    x = _x(1, 40)
    stack = EncoderStack(ws, H, scores=dict(bias=_table()), linear="int8")
    m = ScoreMask(causal=True, kv_len=torch.tensor([40], dtype=torch.int32, device="cuda"))
    run = CapturedForward(stack, x, m)
    for seed in (5, 6, 7):
        y = _x(1, 40, seed=seed)
        want = stack(y, m)
        torch.cuda.synchronize()
        assert torch.equal(run(y), want)
        m.kv_len.fill_(40 - seed)          # read by the replay
        want = stack(y, m)
        torch.cuda.synchronize()
        assert torch.equal(run(y), want)


def test_refusals():
    w, x = _weights(), _x(1, 64)
    lut = pm.get_sparse_storage(torch.ones(1, 64, 64).cuda(), 64, 64)[1:]
    for kw in (dict(linear="int4"), dict(linear="int8", ln_fusion="cluster"), dict(linear="int8", ffn_chain=True), dict(scores=dict(window=4))):
        with pytest.raises(StofError):
            EncoderLayer(w, H, **kw)
    with pytest.raises(StofError):
        EncoderLayer(w, H, scores=dict(cap=3.0))(x, lut)


def test_end_to_end_command_with_table_and_int8():
    cmd = [sys.executable, "sc25-stof-ad_amd/examples/end2end.py", "--model", "t5", "--batch_size", "1", "--seq_len", "128", "--position_bias",
           "--linear", "int8", "--warmup_iters", "1", "--running_iters", "1"]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "STOF" in r.stdout and "max abs difference" in r.stdout, r.stdout + r.stderr


def test_stages_run_the_layer_s_own_attention():
    """A layer with a score rule refuses a LUT in ``stages`` as in ``forward``, and its stages give what ``forward`` gives."""
    w, x = _weights(), _x(1, 64)
    lut = pm.get_sparse_storage(torch.ones(1, 64, 64).cuda(), 64, 64)[1:]
    layer = EncoderLayer(w, H, scores=dict(cap=3.0))
    for call in (lambda: layer(x, lut), lambda: layer.stages(x, lut)):
        with pytest.raises(StofError, match="ScoreMask"):
            call()
    m = ScoreMask(causal=True)
    stages = dict(layer.stages(x, m))
    assert torch.equal(stages["attention"](), layer._attn(stages["qkv_gemm"](), m, 64)) and torch.equal(stages["ffn2_ln"](), layer(x, m))
    plain = EncoderLayer(w, H)
    stages = dict(plain.stages(x, lut))
    assert torch.equal(stages["attention"](), plain._attn(stages["qkv_gemm"](), lut, 64)) and torch.equal(stages["ffn2_ln"](), plain(x, lut))
