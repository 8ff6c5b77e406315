"""GPU parity of attention with score rules (stof.scores) against the float64 oracle, forward and backward,
element by element within the bound that the oracle derives from the roundings of the computation."""
import math

import pytest
import torch

from oracle import scores as os_
from stof import _lib
from stof.ops import StofError
from stof.scores import ScoreMask, score_attn, score_attn_backward

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _qkv(B, Hq, Hkv, Sq, Sk, D, dtype, seed=0, scale=1.0):
    g = _gen(seed)
    n = lambda *s: torch.randn(*s, generator=g)
    return ((n(B, Hq, Sq, D) * scale).to(dtype), n(B, Hkv, Sk, D).to(dtype), n(B, Hkv, Sk, D).to(dtype), n(B, Hq, Sq, D).to(dtype))


def _check(got, want, name):
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, name
    inf = torch.isinf(value)
    assert torch.equal(inf, torch.isinf(got)) and torch.equal(got[inf], value[inf]), f"{name}: infinities differ"
    err = torch.where(inf, 0.0, (got - value).abs())
    over = err > bound
    assert not bool(over.any()) and not bool(torch.isnan(got).any()), \
        f"{name}: {int(over.sum())} of {err.numel()} beyond the bound, worst {float((err / bound.clamp_min(1e-300)).nan_to_num().max()):.2f} of it, NaN {int(torch.isnan(got).sum())}"
    return float((err / bound.clamp_min(1e-300)).max()) if err.numel() else 0.0


def _mask(rule):
    c = lambda t: t.cuda() if torch.is_tensor(t) else tuple(x.cuda() for x in t) if isinstance(t, tuple) else t
    return ScoreMask(**{k: c(v) for k, v in rule.items()})


def _run(q, k, v, dout, rule, forms=("wide", "wide2", "rows"), train=True, **kw):
    """Every form of the forward pass, and the gradients through autograd, against the oracle."""
    want = os_.score_attn(q, k, v, dout=dout if train else None, **{**kw, **rule})
    cu = {n: (t.cuda() if torch.is_tensor(t) else t) for n, t in kw.items()}
    m = _mask(rule)
    for f in forms:
        out, lse = score_attn(q.cuda(), k.cuda(), v.cuda(), m, return_lse=True, launch_form=f, **cu)
        _check(out, want["out"], f"out ({f})")
        _check(lse, want["lse"], f"lse ({f})")
    if not train:
        return
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    if kw.get("bias") is not None:
        leaves.append(kw["bias"].cuda().requires_grad_())
        cu["bias"] = leaves[3]
    out = score_attn(*leaves[:3], m, **cu)
    grads = torch.autograd.grad(out, leaves, dout.cuda())
    for n, g in zip(("dq", "dk", "dv", "dbias"), grads):
        _check(g, want[n], n)


def _docs(B, S, seed):
    g = _gen(seed)
    d = torch.cumsum(torch.rand(B, S, generator=g) < 0.04, 1).to(torch.int32)
    d[:, S - S // 10:] = -1
    if S > 20:
        d[0, 7:11] = -1            # padding in the middle too
        d[-1, 15:19] = 0           # a document that comes back
    return d


def _rule(name, B, Sq, Sk):
    g = _gen(11)
    ints = lambda lo, hi: torch.randint(lo, hi + 1, (B,), generator=g, dtype=torch.int32)
    if name == "full":
        return {}
    if name == "causal":
        return dict(causal=True)
    if name == "prefix":
        return dict(causal=True, prefix=ints(0, Sk))
    if name == "lengths":
        return dict(kv_len=torch.cat([torch.tensor([0], dtype=torch.int32), ints(1, Sk)[1:]]))     # the first sample has no keys
    if name == "docs":
        return dict(docs=_docs(B, Sq, 3) if Sq == Sk else (_docs(B, Sq, 3), _docs(B, Sk, 4)))
    if name == "causal_docs_lengths":
        return dict(causal=True, kv_len=ints(1, Sk), docs=_docs(B, Sq, 3) if Sq == Sk else (_docs(B, Sq, 3), _docs(B, Sk, 4)))
    if name == "ahead":
        return dict(causal=True, q_start=-5)        # the first five rows see nothing
    raise KeyError(name)


@pytest.mark.parametrize("rule", ["full", "causal", "prefix", "lengths", "docs", "causal_docs_lengths", "ahead"])
@pytest.mark.parametrize("what", ["none", "table", "slopes"])
@pytest.mark.parametrize("dtype,D,cap", [("fp16", 64, None), ("bf16", 64, 20.0), ("fp16", 128, 20.0), ("bf16", 128, None)])
def test_rules_forward_and_backward(rule, what, dtype, D, cap):
    B, Hq, Hkv, S = 2, 4, 2, 197
    q, k, v, dout = _qkv(B, Hq, Hkv, S, S, D, DT[dtype], seed=1, scale=2.0)
    g = _gen(2)
    kw = dict(cap=cap)
    if what == "table":
        kw["bias"] = torch.randn(Hq, 2 * 20 + 1, generator=g).to(DT[dtype])
    if what == "slopes":
        kw["slopes"] = torch.rand(Hq, generator=g) * 0.1
    _run(q, k, v, dout, _rule(rule, B, S, S), **kw)


@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 64), (3, 65), (31, 33), (64, 64), (65, 1), (128, 130), (129, 127), (300, 70), (5, 700)])
@pytest.mark.parametrize("Hq,Hkv,D,dtype", [(3, 3, 64, "fp16"), (8, 1, 128, "bf16"), (6, 2, 64, "bf16")])
def test_lengths_and_head_groups(Sq, Sk, Hq, Hkv, D, dtype):
    q, k, v, dout = _qkv(2, Hq, Hkv, Sq, Sk, D, DT[dtype], seed=Sq + Sk)
    bias = torch.randn(Hq, 2 * 40 + 1, generator=_gen(1)).to(DT[dtype])
    _run(q, k, v, dout, dict(causal=True), bias=bias)


@pytest.mark.parametrize("radius", [0, 1, 31, 32, 100, 1024])
def test_table_radius(radius):
    q, k, v, dout = _qkv(1, 2, 1, 170, 230, 64, torch.float16, seed=4)
    bias = torch.randn(2, 2 * radius + 1, generator=_gen(radius)).to(torch.float16)
    _run(q, k, v, dout, {}, bias=bias)
    q, k, v, dout = _qkv(1, 2, 1, 70, 70, 128, torch.bfloat16, seed=4)
    _run(q, k, v, dout, dict(causal=True), bias=bias.to(torch.bfloat16), forms=("wide",))


@pytest.mark.parametrize("low,high", [(0.5, -0.5), (12.0, 3.0), (-40.0, 25.0), (2800.0, 0.0), (0.0, -2800.0), (2900.0, 2900.0), (-math.inf, 1.0), (2.0, -math.inf)])
@pytest.mark.parametrize("D,dtype,cap", [(64, "fp16", None), (64, "bf16", 20.0), (128, "bf16", None)])
def test_distances_far_beyond_the_table(low, high, D, dtype, cap):
    """Most pairs clip to an end of a short table: whole pieces of scores that share one entry, whatever it holds."""
    q, k, v, dout = _qkv(1, 4, 2, 330, 270, D, DT[dtype], seed=25)
    bias = torch.randn(4, 2 * 6 + 1, generator=_gen(26)).to(DT[dtype])
    bias[:, 0], bias[:, -1] = low, high
    finite = math.isfinite(low) and math.isfinite(high)
    _run(q, k, v, dout if finite else None, dict(q_start=0), bias=bias, cap=cap, train=finite)
    _run(q, k, v, dout if finite else None, dict(causal=True, q_start=-20), bias=bias, cap=cap, train=finite)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_table_entries_at_the_ends_of_the_format(dtype):
    """-inf closes a distance, a row whose every distance is closed gives zeros; the lowest finite value is
    a very small score and not a mask: a row with nothing else is a plain softmax over them."""
    lo = torch.finfo(DT[dtype]).min
    q, k, v, dout = _qkv(1, 3, 1, 80, 80, 64, DT[dtype], seed=6)
    bias = torch.zeros(3, 11).to(DT[dtype])
    bias[0, :] = -math.inf
    bias[0, 5] = 1.0                 # head 0: its own key only
    bias[1, :] = -math.inf           # head 1: nothing
    bias[2, :] = lo                  # head 2: everything, very low
    m = ScoreMask()
    for f in ("wide", "wide2", "rows"):
        out, lse = score_attn(q.cuda(), k.cuda(), v.cuda(), m, bias=bias.cuda(), return_lse=True, launch_form=f)
        assert torch.equal(out[0, 0].cpu(), v[0, 0]) and torch.equal(out[0, 1].cpu(), torch.zeros(80, 64, dtype=DT[dtype]))
        assert bool(torch.isinf(lse[0, 1]).all())
        if dtype == "bf16":          # scores below 2^127 / log2 e are absorbed: uniform
            want = v[0, 0].double().mean(0)
            assert float((out[0, 2].double().cpu() - want).abs().max()) <= 2.0 ** -8 * 2 * float(v.abs().double().mean(2).max())
        else:
            plain = score_attn(q.cuda(), k.cuda(), v.cuda(), m, launch_form=f)[0, 2].double().cpu()
            # q.k on top of -65504 keeps a spacing of 2^-8: scores half of it off
            assert float((out[0, 2].double().cpu() - plain).abs().max()) <= (2.0 ** -8 + 2.0 ** -10) * float(v.abs().max())
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, bias)]
    grads = torch.autograd.grad(score_attn(*leaves[:3], m, bias=leaves[3]), leaves, dout.cuda())
    assert all(bool(torch.isfinite(t).all()) for t in grads)
    assert not bool(grads[0][0, 1].any()) and not bool(grads[3][1].any())


@pytest.mark.parametrize("form", ["wide", "wide2", "rows"])
@pytest.mark.parametrize("D", [64, 128])
def test_what_no_query_may_use_is_not_read_as_a_value(form, D):
    """NaN and infinities past kv_len, at positions without a document and in padded query rows."""
    B, S = 2, 150
    q, k, v, dout = _qkv(B, 2, 2, S, S, D, torch.float16, seed=8)
    docs = _docs(B, S, 5)
    kv_len = torch.tensor([150, 77], dtype=torch.int32)
    rule = dict(docs=docs, kv_len=kv_len)
    want = os_.score_attn(q, k, v, dout=dout, **rule)
    dead = (docs < 0)[:, None, :, None]
    past = torch.arange(S)[None, :] >= kv_len[:, None]
    dead_k = dead | past[:, None, :, None]
    spoil = lambda t, where, x: torch.where(where, torch.tensor(x, dtype=t.dtype), t)
    q, dout = spoil(q, dead, math.nan), spoil(dout, dead, math.inf)
    k, v = spoil(k, dead_k, math.nan), spoil(v, dead_k, -math.inf)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    out, lse = score_attn(*leaves, _mask(rule), return_lse=True, launch_form=form)
    _check(out, want["out"], "out")
    _check(lse, want["lse"], "lse")
    for n, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout.cuda())):
        _check(g, want[n], n)


@pytest.mark.parametrize("form", ["wide", "wide2", "rows"])
def test_the_free_part_of_a_cache_behind_causality(form):
    """No key length given: what causality closes to every query is not read as a value either."""
    q, k, v, dout = _qkv(2, 2, 1, 40, 150, 64, torch.bfloat16, seed=18)
    rule = dict(causal=True, q_start=60, prefix=torch.tensor([0, 110], dtype=torch.int32))
    want = os_.score_attn(q, k, v, dout=dout, **rule)
    for t in (k, v):
        t[0, :, 100:] = math.nan
        t[1, :, 110:] = math.inf
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    out = score_attn(*leaves, _mask(rule), launch_form=form)
    _check(out, want["out"], "out")
    for n, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout.cuda())):
        _check(g, want[n], n)


@pytest.mark.parametrize("form", ["wide", "wide2", "rows"])
@pytest.mark.parametrize("D", [64, 128])
def test_nan_in_an_allowed_place_reaches_its_rows(form, D):
    """A query of NaN, and a NaN key that is the only one of its tile and split: NaN out and NaN lse, never a number."""
    q, k, v, _ = (t.cuda() for t in _qkv(2, 4, 2, 1, 8192, D, torch.float16, seed=21))
    q[0, 1] = math.nan
    for n in (8192, 257, 5):
        out, lse = score_attn(q, k, v, ScoreMask(kv_len=torch.full((2,), n, dtype=torch.int32, device="cuda")), launch_form=form, return_lse=True)
        bad = torch.zeros(2, 4, 1, dtype=torch.bool, device="cuda")
        bad[0, 1] = True
        assert torch.equal(out.isnan().all(-1), bad) and torch.equal(out.isnan().any(-1), bad) and torch.equal(lse.isnan(), bad)
    k[1, 0, 256] = math.nan
    out, lse = score_attn(q, k, v, ScoreMask(kv_len=torch.full((2,), 257, dtype=torch.int32, device="cuda")), launch_form=form, return_lse=True)
    bad[1, :2] = True
    assert torch.equal(out.isnan().all(-1), bad) and torch.equal(out.isnan().any(-1), bad) and torch.equal(lse.isnan(), bad)


def test_one_tensor_in_all_three_places():
    x, _, _, dout = _qkv(2, 3, 3, 90, 90, 64, torch.float16, seed=22)
    want = os_.score_attn(x, x, x, dout=dout, causal=True)
    leaf = x.cuda().requires_grad_()
    out = score_attn(leaf, leaf, leaf, ScoreMask(causal=True))
    _check(out, want["out"], "out")
    out.backward(dout.cuda())
    # (three rounded gradients summed by autograd in fp16: two more roundings of at most half a step of the partial sums)
    parts = [want[n] for n in ("dq", "dk", "dv")]
    room = sum(p[1] for p in parts) + 2 * 2.0 ** -11 * sum(p[0].abs() for p in parts)
    _check(leaf.grad, (sum(p[0] for p in parts), room), "dx")


def test_training_steps_on_two_streams_at_once():
    """Forward and backward passes that overlap on two streams: workspaces are each call's own."""
    sets = [[t.cuda() for t in _qkv(2, 8, 2, 300, 300, 64, torch.float16, seed=s)] for s in (23, 24)]
    bias = torch.randn(8, 129, generator=_gen(5)).half().cuda()
    docs = (torch.arange(300, dtype=torch.int32) // 70).expand(2, 300).contiguous().cuda()

    def step(t):
        out, lse = score_attn(*t[:3], ScoreMask(causal=True, docs=docs), bias=bias, return_lse=True)
        return (out,) + score_attn_backward(t[3], *t[:3], out, lse, ScoreMask(causal=True, docs=docs), bias=bias)
    want = [step(t) for t in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append(step(sets[n]))
    torch.cuda.synchronize()
    for n in range(2):
        for g in got[n]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[n]))


@pytest.mark.parametrize("B,Hq,Hkv,S,D", [(4, 4, 2, 300, 64), (8, 2, 1, 520, 128), (1, 16, 8, 260, 64), (2, 8, 8, 200, 64)])
def test_causal_work_placed_over_the_xcds(B, Hq, Hkv, S, D):
    """Key heads that divide over the eight XCDs: every tile of every head exactly once."""
    q, k, v, dout = _qkv(B, Hq, Hkv, S, S, D, torch.float16, seed=19)
    _run(q, k, v, dout, dict(causal=True))
    _run(q, k, v, dout, dict(kv_len=torch.randint(0, S + 1, (B,), generator=_gen(S), dtype=torch.int32)))


@pytest.mark.parametrize("B,Hq,Hkv,S,D", [(3, 12, 12, 300, 64), (2, 16, 4, 260, 128), (3, 8, 4, 200, 64), (5, 3, 1, 270, 64), (1, 12, 6, 520, 64), (8, 12, 12, 140, 64)])
def test_uneven_samples_placed_over_the_xcds(B, Hq, Hkv, S, D):
    q, k, v, dout = _qkv(B, Hq, Hkv, S, S, D, torch.bfloat16, seed=27)
    _run(q, k, v, dout, dict(causal=True))
    _run(q, k, v, dout, dict(causal=True, docs=_docs(B, S, 28)))
    _run(q, k, v, dout, dict(kv_len=torch.randint(0, S + 1, (B,), generator=_gen(S + 1), dtype=torch.int32)))


def test_gradient_of_an_expanded_scalar_and_of_broadcast_keys():
    """out.sum() hands an expanded gradient back; one key head expanded over four collects the sum of their gradients."""
    q, k, v, _ = _qkv(2, 4, 1, 50, 70, 64, torch.float16, seed=20)
    want = os_.score_attn(q, k, v, dout=torch.ones_like(q))
    lq, lk, lv = (t.cuda().requires_grad_() for t in (q, k, v))
    score_attn(lq, lk, lv).sum().backward()
    for t, n in ((lq, "dq"), (lk, "dk"), (lv, "dv")):
        _check(t.grad, want[n], n)
    lk2, lv2 = (t.cuda().requires_grad_() for t in (k, v))
    out = score_attn(q.cuda(), lk2.expand(2, 4, 70, 64), lv2.expand(2, 4, 70, 64))
    _check(out, want["out"], "out")
    out.sum().backward()
    # (four rounded gradients summed by autograd in fp16: three more roundings of at most half a step of the largest partial sum)
    for got, n in ((lk2.grad, "dk"), (lv2.grad, "dv")):
        value, bound = want[n]
        parts = os_.score_attn(q, k.expand(2, 4, 70, 64), v.expand(2, 4, 70, 64), dout=torch.ones_like(q))[n]
        room = parts[1].sum(1, keepdim=True) + 3 * 2.0 ** -11 * parts[0].abs().sum(1, keepdim=True)
        _check(got, (value, room), n)


@pytest.mark.parametrize("dscale", [2.0 ** -12, 1.0, 4096.0])
def test_fp16_gradients_of_small_and_large_losses(dscale):
    """A loss scaled by a power of two scales every gradient by it, inside the range of the format."""
    q, k, v, dout = _qkv(1, 2, 2, 200, 200, 64, torch.float16, seed=9)
    dout = (dout * dscale).half()
    _run(q, k, v, dout, dict(causal=True), forms=())
    _run(q, k, (v.float() * 16).half(), dout, {}, forms=())


def test_strided_views_layouts_and_rows_behind_the_last():
    """q, k, v as views of one packed projection, a cache with room behind the last key, outputs in both layouts, written
    between guard rows that stay as they were."""
    B, H, S, D = 2, 4, 100, 64
    qkv = torch.randn(B, S, 3 * H * D, generator=_gen(1)).half()
    q, k, v = (qkv[..., t * H * D:(t + 1) * H * D].view(B, S, H, D).permute(0, 2, 1, 3) for t in range(3))
    dout = torch.randn(B, H, S, D, generator=_gen(2)).half()
    want = os_.score_attn(q, k, v, dout=dout, causal=True)
    packed = qkv.cuda().requires_grad_()
    vq, vk, vv = (packed[..., t * H * D:(t + 1) * H * D].view(B, S, H, D).permute(0, 2, 1, 3) for t in range(3))
    for layout in ("bhsd", "bshd"):
        out = score_attn(vq, vk, vv, ScoreMask(causal=True), out_layout=layout)
        as_bhsd = out if layout == "bhsd" else out.view(B, S, H, D).permute(0, 2, 1, 3)
        _check(as_bhsd, want["out"], layout)
        d = dout.cuda() if layout == "bhsd" else dout.permute(0, 2, 1, 3).reshape(B, S, H * D).cuda()
        g, = torch.autograd.grad(out, packed, d)
        for t, n in enumerate(("dq", "dk", "dv")):
            _check(g[..., t * H * D:(t + 1) * H * D].view(B, S, H, D).permute(0, 2, 1, 3), want[n], f"{layout} {n}")
    big = torch.full((B, H, S + 40, D), 7.0, dtype=torch.float16, device="cuda")
    for f in ("wide", "wide2", "rows"):
        score_attn(vq.detach(), vk.detach(), vv.detach(), ScoreMask(causal=True), out=big[:, :, 20:20 + S], launch_form=f)
        _check(big[:, :, 20:20 + S], want["out"], f"out= ({f})")
        assert bool((big[:, :, :20] == 7).all()) and bool((big[:, :, 20 + S:] == 7).all())
    cache = torch.full((B, H, 512, D), math.nan, dtype=torch.float16, device="cuda")
    cache[:, :, :S] = k.cuda()
    vals = torch.full((B, 512, H, D), math.nan, dtype=torch.float16, device="cuda").permute(0, 2, 1, 3)
    vals[:, :, :S] = v.cuda()
    m = ScoreMask(causal=True, kv_len=torch.full((B,), S, dtype=torch.int32, device="cuda"), q_start="end")
    for f in ("wide", "wide2", "rows"):
        _check(score_attn(q.cuda(), cache, vals, m, launch_form=f), want["out"], f"cache ({f})")


@pytest.mark.parametrize("B,Hq,Hkv,D,Sk", [(1, 12, 12, 64, 512), (3, 8, 2, 128, 3000), (2, 32, 1, 64, 1025), (5, 16, 4, 64, 40)])
@pytest.mark.parametrize("what", ["none", "table", "slopes"])
def test_single_tokens(B, Hq, Hkv, D, Sk, what):
    """One query at the end of caches of uneven length, one of them empty."""
    dtype = torch.bfloat16 if D == 128 else torch.float16
    q, k, v, _ = _qkv(B, Hq, Hkv, 1, Sk, D, dtype, seed=Sk)
    kv_len = torch.randint(1, Sk + 1, (B,), generator=_gen(Sk), dtype=torch.int32)
    if B > 1:
        kv_len[0] = 0
    kw = dict(cap=30.0)
    if what == "table":
        kw["bias"] = torch.randn(Hq, 2 * 64 + 1, generator=_gen(1)).to(dtype)
    if what == "slopes":
        kw["slopes"] = torch.rand(Hq, generator=_gen(1)) * 0.05
    _run(q, k, v, None, dict(kv_len=kv_len, q_start="end"), train=False, forms=(None, "wide", "wide2", "rows"), **kw)


def test_a_sequence_token_by_token_equals_the_whole():
    """Run together, as a model uses them: a prompt, then tokens one at a time over the growing cache."""
    B, Hq, Hkv, D, n, cap = 2, 4, 2, 64, 90, 25.0
    q, k, v, _ = _qkv(B, Hq, Hkv, n, n, D, torch.float16, seed=12)
    bias = torch.randn(Hq, 2 * 16 + 1, generator=_gen(3)).half()
    want = os_.score_attn(q, k, v, causal=True, cap=cap, bias=bias)["out"]
    q, k, v, bias = (t.cuda() for t in (q, k, v, bias))
    ck, cv = (torch.full((B, Hkv, 128, D), math.nan, dtype=torch.float16, device="cuda") for _ in range(2))
    lens = torch.full((B,), 70, dtype=torch.int32, device="cuda")
    step = ScoreMask(causal=True, kv_len=lens, q_start="end")
    ck[:, :, :70], cv[:, :, :70] = k[:, :, :70], v[:, :, :70]
    outs = [score_attn(q[:, :, :70], ck, cv, step, cap=cap, bias=bias)]
    for t in range(70, n):
        ck[:, :, t], cv[:, :, t] = k[:, :, t], v[:, :, t]
        lens.add_(1)
        outs.append(score_attn(q[:, :, t:t + 1], ck, cv, step, cap=cap, bias=bias))
    _check(torch.cat(outs, 2), want, "token by token")


def test_same_inputs_same_bits():
    q, k, v, dout = (t.cuda() for t in _qkv(2, 4, 2, 333, 333, 64, torch.bfloat16, seed=13))
    bias = torch.randn(4, 65, generator=_gen(1)).bfloat16().cuda()
    m = ScoreMask(causal=True)
    first = None
    for _ in range(4):
        out, lse = score_attn(q, k, v, m, cap=30.0, bias=bias, return_lse=True)
        got = (out, lse, *score_attn_backward(dout, q, k, v, out, lse, m, cap=30.0, bias=bias))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_long_cache_past_32_bit_offsets():
    """A value cache whose last rows lie past 2^32 bytes: 700 000 positions of 4096 elements, of which a head takes 64."""
    S, W = 700_000, 4096
    try:
        cache = torch.empty(1, S, W, dtype=torch.float16, device="cuda")
    except torch.OutOfMemoryError:
        pytest.skip("not enough memory")
    view = cache.view(1, S, W // 64, 64).permute(0, 2, 1, 3)[:, 3:4]
    g = torch.Generator(device="cuda").manual_seed(1)
    view[:] = torch.randn(1, 1, S, 64, generator=g, device="cuda")
    q = torch.randn(1, 1, 1, 64, generator=g, device="cuda").half()
    p = torch.softmax((view[0, 0].double() @ q[0, 0, 0].double()) / 8, 0)
    want = p @ view[0, 0].double()
    size = float((p[:, None] * view[0, 0].double().abs()).sum(0).max())
    for f in ("wide", "wide2", "rows"):
        out = score_attn(q, view, view, launch_form=f)[0, 0, 0].double()
        # roundings of P and out, fp32 scores of at most 6: (64 + 8) 2^-24 * 6 * 8 twice; small P: 2^-25 each against a sum of S terms
        bound = (2.0 ** -11 + 2 * 72 * 48 * 2.0 ** -24) * size + 2.0 ** -11 * want.abs() + 2.0 ** -25
        assert bool(((out - want).abs() <= bound).all()), f


def test_other_stream_and_captured_graph():
    q, k, v, _ = (t.cuda() for t in _qkv(1, 8, 2, 1, 3000, 64, torch.float16, seed=14))
    lens = torch.full((1,), 3000, dtype=torch.int32, device="cuda")
    m = ScoreMask(kv_len=lens, q_start="end")
    slopes = (torch.arange(8) * 0.01).cuda()
    eager = lambda: score_attn(q, k, v, m, slopes=slopes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            eager()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):             # two graphs of the same call, replayed at the same time on two streams
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = eager()
        graphs.append((gr, out))
    for n in (3000, 1, 64, 2000):
        lens.fill_(n)
        want = eager()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want)


def test_backward_in_a_captured_graph():
    q, k, v, dout = (t.cuda() for t in _qkv(1, 2, 2, 130, 130, 64, torch.bfloat16, seed=15))
    m = ScoreMask(causal=True, docs=torch.zeros(1, 130, dtype=torch.int32, device="cuda"))

    def step():
        out, lse = score_attn(q, k, v, m, return_lse=True)
        return score_attn_backward(dout, q, k, v, out, lse, m)[:3]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = step()
    for seed in (1, 2, 3):
        q.copy_(torch.randn(q.shape, generator=_gen(seed)))
        want = step()
        torch.cuda.synchronize()
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradient_against_differences():
    """A directional derivative of the kernels' own forward pass: outputs carry a rounding of 2^-11 each, against steps
    of 2^-5: (L(+h) - L(-h)) / 2 h is off by at most sqrt(n) 2^-11 rms(out dout) / h (independent roundings; four times that
    is asked) plus the third order, h^2 / 6 of a third derivative taken from the oracle at two steps."""
    q, k, v, dout = _qkv(1, 2, 1, 60, 60, 64, torch.float16, seed=16)
    d = torch.randn(q.shape, generator=_gen(17)).half()
    h = 2.0 ** -5
    q64, m = q.double(), ScoreMask(causal=True)
    loss = lambda x: (score_attn(x.half().cuda(), k.cuda(), v.cuda(), m, cap=20.0).double().cpu() * dout.double()).sum()
    ref = lambda x: (os_.score_attn(x.half(), k, v, causal=True, cap=20.0)["out"][0] * dout.double()).sum()
    up, dn = (q64 + h * d.double()).half().double(), (q64 - h * d.double()).half().double()
    got = float(loss(up) - loss(dn))
    leaf = q.cuda().requires_grad_()
    g, = torch.autograd.grad(score_attn(leaf, k.cuda(), v.cuda(), m, cap=20.0), leaf, dout.cuda())
    want = float((g.double().cpu() * (up - dn)).sum())
    curve = abs(float(ref(up) - ref(dn)) - float((os_.score_attn(q, k, v, causal=True, cap=20.0, dout=dout)["dq"][0] * (up - dn)).sum()))
    out = os_.score_attn(q, k, v, causal=True, cap=20.0)["out"][0]
    noise = 4 * 2 * math.sqrt(out.numel()) * 2.0 ** -11 * float((out * dout.double()).pow(2).mean().sqrt())
    assert abs(got - want) <= noise + curve + 2.0 ** -10 * abs(want), (got, want, noise, curve)


def test_rule_tensor_changed_before_backward_is_noticed():
    q, k, v, dout = (t.cuda() for t in _qkv(1, 1, 1, 8, 8, 64, torch.float16))
    lens = torch.tensor([8], dtype=torch.int32, device="cuda")
    leaf = q.requires_grad_()
    out = score_attn(leaf, k, v, ScoreMask(kv_len=lens))
    lens.fill_(3)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.backward(dout)


def test_empty_calls():
    z = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")
    out, lse = score_attn(z(2, 4, 3, 64), z(2, 2, 0, 64), z(2, 2, 0, 64), return_lse=True)
    assert out.shape == (2, 4, 3, 64) and not bool(out.any()) and bool((lse == -math.inf).all())
    assert score_attn(z(0, 4, 3, 64), z(0, 2, 5, 64), z(0, 2, 5, 64)).shape == (0, 4, 3, 64)
    assert score_attn(z(2, 4, 0, 64), z(2, 2, 5, 64), z(2, 2, 5, 64)).shape == (2, 4, 0, 64)


def test_refusals():
    h = lambda *s, d=torch.float16: torch.zeros(*s, dtype=d, device="cuda")
    q, k = h(2, 4, 8, 64), h(2, 2, 16, 64)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    bad = [
        lambda: score_attn(q.cpu(), k.cpu(), k.cpu()),
        lambda: score_attn(q.float(), k.float(), k.float()),
        lambda: score_attn(q, k.bfloat16(), k),
        lambda: score_attn(q, h(2, 3, 16, 64), h(2, 3, 16, 64)),
        lambda: score_attn(q, k, h(2, 2, 17, 64)),
        lambda: score_attn(h(2, 4, 8, 32), h(2, 2, 16, 32), h(2, 2, 16, 32)),
        lambda: score_attn(q.transpose(2, 3), k, k),
        lambda: score_attn(q, k, k, scale=0.0),
        lambda: score_attn(q, k, k, cap=-1.0),
        lambda: score_attn(q, k, k, bias=h(4, 10)),
        lambda: score_attn(q, k, k, bias=h(4, 11, d=torch.float32)),
        lambda: score_attn(q, k, k, bias=h(4, 2051)),
        lambda: score_attn(q, k, k, bias=h(4, 11), slopes=h(4, d=torch.float32)),
        lambda: score_attn(q, k, k, slopes=h(4)),
        lambda: score_attn(q, k, k, slopes=h(4, d=torch.float32).requires_grad_()),
        lambda: score_attn(q, k, k, ScoreMask(kv_len=i32(3))),
        lambda: score_attn(q, k, k, ScoreMask(docs=i32(2, 8))),
        lambda: score_attn(q, k, k, ScoreMask(kv_len=i32(2).cpu())),
        lambda: score_attn(q, k, k, launch_form="other"),
        lambda: score_attn(q, k, k, out=h(2, 4, 8, 64, d=torch.bfloat16)),
        lambda: score_attn(q, k, k, out_layout="other"),
        lambda: score_attn(q.requires_grad_(), k, k, out=h(2, 4, 8, 64)),
        lambda: score_attn(h(2, 4, 8, 65)[..., :64], k, k),          # row stride not a multiple of 8
        lambda: score_attn(h(2 * 4 * 8 * 64 + 1)[1:].view(2, 4, 8, 64), k, k),   # not 16-byte aligned
    ]
    for n, call in enumerate(bad):
        with pytest.raises(StofError):
            call()
            pytest.fail(f"refusal {n} was accepted")


def test_slopes_kept_as_a_parameter():
    """Refused where a gradient would be asked for, taken under no_grad."""
    x = torch.randn(1, 4, 20, 64, generator=torch.Generator().manual_seed(1)).half().cuda()
    slopes = torch.nn.Parameter(torch.rand(4, generator=torch.Generator().manual_seed(2)).cuda())
    with pytest.raises(StofError, match="gradient"):
        score_attn(x, x, x, slopes=slopes)
    with torch.no_grad():
        assert torch.equal(score_attn(x, x, x, slopes=slopes), score_attn(x, x, x, slopes=slopes.detach()))


@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
def test_gradient_that_arrives_at_an_odd_address(layout):
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(2, 3, 70, 64, generator=g).half().cuda().requires_grad_() for _ in range(3))
    out = score_attn(q, k, v, ScoreMask(causal=True), out_layout=layout)
    flat = torch.randn(out.numel() + 1, generator=g).half().cuda()
    odd = flat[1:].view(out.shape)
    assert odd.is_contiguous() and odd.data_ptr() % 16
    want = torch.autograd.grad(out, (q, k, v), odd.clone(), retain_graph=True)
    got = torch.autograd.grad(out, (q, k, v), odd)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
