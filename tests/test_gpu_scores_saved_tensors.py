"""Gradients of attention with score rules whose saved tensors pass through hooks, against the float64 oracle."""
import pytest
import torch
import torch.utils.checkpoint

from oracle import scores as os_
from stof.scores import ScoreMask, score_attn

pytestmark = pytest.mark.gpu


def _within(got, want, name):
    value, bound = want
    assert bool(((got.double().cpu() - value).abs() <= bound).all()), name


HOOKS = {
    "host": lambda: torch.autograd.graph.save_on_cpu(pin_memory=False),
    "pinned host": lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
    "copied": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t),
    "heads and rows exchanged": lambda: torch.autograd.graph.saved_tensors_hooks(
        lambda t: t.transpose(1, 2).contiguous().transpose(1, 2) if t.dim() == 4 else t, lambda t: t),
}


@pytest.mark.parametrize("how", HOOKS)
@pytest.mark.parametrize("layout,D,dtype", [("bhsd", 64, torch.float16), ("bshd", 64, torch.bfloat16), ("bshd", 128, torch.float16)])
def test_views_of_a_packed_projection(how, layout, D, dtype):
    B, H, S = 2, 4, 130
    g = torch.Generator().manual_seed(41)
    qkv = torch.randn(B, S, 3 * H * D, generator=g).to(dtype)
    dout = torch.randn(B, H, S, D, generator=g).to(dtype)
    bias = torch.randn(H, 21, generator=g).to(dtype)
    docs = (torch.arange(S, dtype=torch.int32) // 50).expand(B, S).contiguous()
    split = lambda t: [t[..., n * H * D:(n + 1) * H * D].view(B, S, H, D).permute(0, 2, 1, 3) for n in range(3)]
    want = os_.score_attn(*split(qkv), dout=dout, causal=True, docs=docs, bias=bias)
    packed, tab = qkv.cuda().requires_grad_(), bias.cuda().requires_grad_()
    with HOOKS[how]():
        out = score_attn(*split(packed), ScoreMask(causal=True, docs=docs.cuda()), bias=tab, out_layout=layout)
    d = dout if layout == "bhsd" else dout.permute(0, 2, 1, 3).reshape(B, S, H * D)
    grad, dtab = torch.autograd.grad(out, (packed, tab), d.cuda())
    for n, got in zip(("dq", "dk", "dv"), split(grad)):
        _within(got, want[n], n)
    _within(dtab, want["dbias"], "dbias")


@pytest.mark.parametrize("how", HOOKS)
def test_expanded_keys_and_slopes(how):
    g = torch.Generator().manual_seed(42)
    n = lambda *s: torch.randn(*s, generator=g).half()
    q, k, v, dout, slopes = n(2, 4, 70, 64), n(2, 1, 90, 64), n(2, 1, 90, 64), n(2, 4, 70, 64), torch.rand(4, generator=g) * 0.1
    want = os_.score_attn(q, k.expand(2, 4, 90, 64), v.expand(2, 4, 90, 64), dout=dout, slopes=slopes)
    lq = q.cuda().requires_grad_()
    kx, vx = (t.cuda().expand(2, 4, 90, 64).detach().requires_grad_() for t in (k, v))
    with HOOKS[how]():
        out = score_attn(lq, kx, vx, slopes=slopes.cuda())
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (lq, kx, vx), dout.cuda())):
        _within(got, want[name], name)


def test_rule_of_the_forward_pass_when_the_mask_object_changes():
    """A mask object that is given other tensors or another causality between the passes: the gradients are of the rule that ran."""
    g = torch.Generator().manual_seed(5)
    n = lambda: torch.randn(2, 2, 90, 64, generator=g).half()
    q, k, v, dout = n(), n(), n(), n()
    docs = (torch.arange(90, dtype=torch.int32) // 20).expand(2, 90).contiguous()
    rule = dict(causal=True, kv_len=torch.tensor([90, 60], dtype=torch.int32), prefix=torch.tensor([0, 30], dtype=torch.int32), docs=docs)
    want = os_.score_attn(q, k, v, dout=dout, **rule)
    m = ScoreMask(causal=True, kv_len=rule["kv_len"].cuda(), prefix=rule["prefix"].cuda(), docs=docs.cuda())
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    out = score_attn(*leaves, m)
    m.causal, m.prefix, m.kv_len = 0, None, torch.tensor([3, 90], dtype=torch.int32, device="cuda")
    m.docs_q = m.docs_k = torch.zeros(2, 90, dtype=torch.int32, device="cuda")
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout.cuda())):
        _within(got, want[name], name)


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_checkpointed_step_has_the_gradients_of_a_plain_one(reentrant):
    """Activations formed again in the backward pass: the same bits."""
    B, H, S, D = 2, 4, 130, 64
    g = torch.Generator().manual_seed(43)
    packed = torch.randn(B, S, 3 * H * D, generator=g).half().cuda().requires_grad_()
    tab = torch.randn(H, 21, generator=g).half().cuda().requires_grad_()
    dout = torch.randn(B, S, H * D, generator=g).half().cuda()
    m = ScoreMask(causal=True, kv_len=torch.tensor([130, 70], dtype=torch.int32, device="cuda"))

    def step(x, t):
        return score_attn(*(x[..., n * H * D:(n + 1) * H * D].view(B, S, H, D).permute(0, 2, 1, 3) for n in range(3)), m, bias=t, out_layout="bshd")

    step(packed, tab).backward(dout)
    want = packed.grad.clone(), tab.grad.clone()
    packed.grad = tab.grad = None
    torch.utils.checkpoint.checkpoint(step, packed, tab, use_reentrant=reentrant).backward(dout)
    assert torch.equal(packed.grad, want[0]) and torch.equal(tab.grad, want[1])
