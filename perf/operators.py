"""Measured cases of the score-rule attention (``stof.scores``) and of the 8-bit linear operator (``stof.quant``).

A case is one call that a user's program makes; ``run`` computes it in elementary torch operations in
32 bits, or, with ``own`` set, through the framework's entry points on the same tensors.

Attention, q [B,Hq,Sq,D] (position of query i: p_i), k and v [B,Hkv,Sk,D], query head h reads key head h // (Hq / Hkv):

    t_ij = scale q_i . k_j;   t_ij = cap tanh(t_ij / cap)  with a cap
    s_ij = t_ij - slope_h |p_i - j|      or      t_ij + table[h, clip(j - p_i, -R, R) + R]
    allowed(i, j) = j < kv_len  and  (not causal or j <= p_i or j < prefix)  and  doc_i = doc_j >= 0
    out_i = sum_j softmax_j(s_ij over the allowed j) v_j,  zero for a row without allowed keys

"train" adds the gradients of sum(out * dout) with respect to q, k, v and the table; "decode" is one
query per sequence at position kv_len - 1 over a cache with room for more.

Linear, x [M,K] in 16 bits, wq [N,K] in 8 bits with a scale for each row:

    a_m = max_k |x_mk|;   xq_mk = round(127 x_mk / a_m), ties to even;   y_mn = act((a_m / 127) ws_n sum_k xq_mk wq_nk + bias_n)
"""
import math
import os
import sys

import torch

own = False

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _attn(name, op, b, hq, hkv, sq, sk, d, dtype, bias="none", cap=0.0, causal=False, prefix=False, docs=False, ragged=False):
    case = dict(op=op, b=b, hq=hq, hkv=hkv, sq=sq, sk=sk, d=d, dtype=dtype, bias=bias, cap=cap, causal=causal,
                prefix=prefix, docs=docs, ragged=ragged)
    return dict(case, name=name) if name else case


def _lin(name, m, k, n, dtype, act, bias=True):
    case = dict(op="linear", m=m, k=k, n=n, dtype=dtype, act=act, use_bias=bias)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one encoder layer's attention with a learned distance table, a single short request: paced by latency
        _attn("fwd_table_b1", "fwd", 1, 12, 12, 512, 512, 64, "fp16", bias="table"),
        # the same at serving batch, key padding of uneven lengths
        _attn("fwd_table_padded_b8", "fwd", 8, 12, 12, 1024, 1024, 64, "fp16", bias="table", ragged=True),
        # long causal prompt with capped scores, shared key heads, head size 128
        _attn("fwd_cap_causal_long", "fwd", 2, 16, 8, 4096, 4096, 128, "bf16", cap=50.0, causal=True),
        # documents packed into one odd-length row, distance slopes, causal inside each document
        _attn("fwd_docs_slopes_odd", "fwd", 2, 16, 16, 4001, 4001, 64, "bf16", bias="slopes", causal=True, docs=True),
        # training step of the distance-table layer: gradients of the table and of q, k, v
        _attn("train_table_b8", "train", 8, 12, 12, 512, 512, 64, "bf16", bias="table"),
        # training step on packed documents, capped, shared key heads
        _attn("train_cap_docs", "train", 2, 16, 4, 2048, 2048, 128, "bf16", cap=30.0, causal=True, docs=True),
        # training step of a prefix model, odd length, fp16 gradients
        _attn("train_prefix_odd", "train", 3, 8, 8, 1000, 1000, 64, "fp16", bias="slopes", causal=True, prefix=True),
        # one token of one sequence: the smallest serving step
        _attn("decode_b1", "decode", 1, 12, 12, 1, 512, 64, "fp16", bias="slopes", ragged=True),
        # one token of many long sequences of uneven length, shared key heads, capped
        _attn("decode_long", "decode", 16, 32, 8, 1, 16384, 128, "bf16", cap=50.0, ragged=True),
        # feed-forward projection of one token
        _lin("linear_token", 1, 1024, 4096, "fp16", "gelu"),
        # an odd number of ordinary rows, no activation
        _lin("linear_odd_rows", 777, 768, 2304, "bf16", "none"),
        # feed-forward projection of a full batch
        _lin("linear_batch", 8192, 1024, 4096, "fp16", "gelu"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["fp16", "bf16"])
    kind = rng.choice(["fwd", "train", "decode", "linear"])
    if kind == "linear":
        m, k, n = _log_int(rng, 1, 8192), 16 * _log_int(rng, 8, 256), 8 * _log_int(rng, 8, 512)
        m = min(m, max(1, 8192 * 1024 * 4096 // (k * n)))
        return _lin("", m, k, n, dtype, rng.choice(["none", "relu", "gelu"]), rng.random() < 0.8)
    d = rng.choice([64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 4])
    bias = rng.choice(["none", "table", "slopes"])
    cap = rng.choice([0.0, 30.0, 50.0])
    b = rng.randint(1, 8)
    if kind == "decode":
        sk = _log_int(rng, 64, 16384)
        return _attn("", "decode", b, hq, hkv, 1, sk, d, dtype, bias, cap, ragged=True)
    s = _log_int(rng, 48, 4096 if kind == "fwd" else 2048)
    b = max(1, min(b, (2 * 16 * 4096 * 4096 if kind == "fwd" else 2 * 16 * 2048 * 2048) // (hq * s * s)))
    causal = rng.random() < 0.6
    docs = rng.random() < 0.4
    sk = s
    if kind == "fwd" and not docs and rng.random() < 0.3:     # a prompt read in pieces: these queries are the last of sk positions
        sk = _log_int(rng, s, 4096)
        b = max(1, min(b, 2 * 16 * 4096 * 4096 // (hq * s * sk)))
    return _attn("", kind, b, hq, hkv, s, sk, d, dtype, bias, cap, causal, causal and not docs and rng.random() < 0.5, docs,
                 not causal and not docs and rng.random() < 0.5)


_RADIUS = 128   # distances told apart by a learned table, as in encoders that clip at 128


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    normal = lambda *shape, std=1.0: (torch.randn(*shape, generator=g, device="cuda") * std)
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        x = normal(m, k)
        x[:, :: max(1, k // 6)] *= 8.0    # activations have a few channels of larger size
        w = normal(n, k, std=0.02)
        ws = w.abs().amax(1) / 127
        wq = torch.round(w / ws[:, None]).clamp(-127, 127).to(torch.int8)
        bias = normal(n, std=0.02).to(dt) if case["use_bias"] else None
        return dict(case=case, x=x.to(dt), wq=wq, ws=ws, bias=bias)
    b, hq, hkv, sq, sk, d = (case[n] for n in ("b", "hq", "hkv", "sq", "sk", "d"))
    q, k, v = normal(b, hq, sq, d, std=4.0 if case["cap"] else 1.0).to(dt), normal(b, hkv, sk, d).to(dt), normal(b, hkv, sk, d).to(dt)
    s = dict(case=case, q=q, k=k, v=v, bias=None, slopes=None, prefix=None, kv_len=None, docs=None)
    ints = lambda lo, hi: torch.randint(lo, hi + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    if case["bias"] == "table":
        s["bias"] = normal(hq, 2 * _RADIUS + 1).to(dt)
    if case["bias"] == "slopes":
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, hq + 1, device="cuda", dtype=torch.float32) / hq)
    if case["prefix"]:
        s["prefix"] = ints(1, max(1, sq // 2))
    if case["ragged"]:
        s["kv_len"] = ints(max(1, sk // 4), sk)
    if case["docs"]:
        cut = torch.rand(b, sq, generator=g, device="cuda") < 6.0 / sq      # about seven documents a row
        docs = torch.cumsum(cut, 1).to(torch.int32)
        pad = sq - sq // 50                                                  # the row's last places are padding
        docs[:, pad:] = -1
        s["docs"] = docs
    if case["op"] == "train":
        s["dout"] = normal(b, hq, sq, d).to(dt)
    return s


# ---- plain forms

def _gelu(x):
    return 0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5)))


def _plain_linear(s):
    case, x = s["case"], s["x"].float()
    a = x.abs().amax(1, keepdim=True)
    xq = torch.round(x.double() * 127.0 / a.clamp_min(1e-38).double()).float()     # next to a border 32 bits would round some values the other way
    y = (xq @ s["wq"].float().t()) * (a / 127.0) * s["ws"][None, :]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if case["act"] == "gelu":
        y = _gelu(y)
    if case["act"] == "relu":
        y = torch.relu(y)
    return y.to(s["x"].dtype)


def _positions(s):
    """Query positions [B,1,Sq,1] and key positions [1,1,1,Sk]."""
    case = s["case"]
    i = torch.arange(case["sq"], device="cuda").view(1, 1, -1, 1)
    j = torch.arange(case["sk"], device="cuda").view(1, 1, 1, -1)
    if case["op"] == "decode":
        return i + s["kv_len"].view(-1, 1, 1, 1) - case["sq"], j
    return i + (case["sk"] - case["sq"]), j


def _allowed(s, p, j):
    ok = torch.ones_like(p >= j)
    if s["kv_len"] is not None:
        ok = ok & (j < s["kv_len"].view(-1, 1, 1, 1))
    if s["case"]["causal"]:
        past = j <= p
        if s["prefix"] is not None:
            past = past | (j < s["prefix"].view(-1, 1, 1, 1))
        ok = ok & past
    if s["docs"] is not None:
        dq, dk = s["docs"][:, None, :, None], s["docs"][:, None, None, :]
        ok = ok & (dq == dk) & (dq >= 0)
    return ok


def _plain_attn(s):
    case = s["case"]
    d, group = case["d"], case["hq"] // case["hkv"]
    q, k, v = s["q"].float(), s["k"].float().repeat_interleave(group, 1), s["v"].float().repeat_interleave(group, 1)
    p, j = _positions(s)
    raw = (q @ k.transpose(-1, -2).contiguous()) / math.sqrt(d)
    th = torch.tanh(raw / case["cap"]) if case["cap"] else None
    score = raw if th is None else case["cap"] * th
    if s["slopes"] is not None:
        score = score - s["slopes"].view(1, -1, 1, 1) * (p - j).abs()
    if s["bias"] is not None:
        at = (j - p).clamp(-_RADIUS, _RADIUS) + _RADIUS                     # [B or 1, 1, Sq, Sk]
        score = score + s["bias"].float()[:, at[:, 0]].transpose(0, 1)
    score = torch.where(_allowed(s, p, j), score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    prob = e / torch.where(total == 0, 1.0, total)
    out = prob @ v
    if case["op"] != "train":
        return out.to(s["q"].dtype)
    dout = s["dout"].float()
    share = lambda t: t.view(case["b"], case["hkv"], group, case["sk"], d).sum(2).to(s["q"].dtype)
    dv = share(prob.transpose(-1, -2).contiguous() @ dout)
    dprob = dout @ v.transpose(-1, -2).contiguous()
    ds = prob * (dprob - (prob * dprob).sum(-1, keepdim=True))
    back = [out.to(s["q"].dtype)]
    table = _table_gradient(ds.sum(0), case["sq"], case["sk"]).to(s["q"].dtype) if s["bias"] is not None else None
    if th is not None:
        ds = ds * (1.0 - th * th)
    ds = ds / math.sqrt(d)
    back += [(ds @ k).to(s["q"].dtype), share(ds.transpose(-1, -2).contiguous() @ q), dv]
    return back + ([table] if table is not None else [])


def _table_gradient(ds, sq, sk):
    """Sums of ds [H,Sq,Sk] (query i at position i) over the entries of equal clipped distance j - i: the
    rows are padded so that a diagonal becomes a column, whose sums are then gathered into the table."""
    h = ds.shape[0]
    wide = torch.nn.functional.pad(ds, (sq, 0)).reshape(h, -1)                    # row i: sq zeros, then its keys
    skew = torch.nn.functional.pad(wide, (0, sq)).view(h, sq, sq + sk + 1)[:, :, :sq + sk]   # row i moves i places to the left
    sums = skew.sum(1)                                                            # column c: distance c - sq
    sums = torch.nn.functional.pad(sums, (_RADIUS, _RADIUS + 1))                  # distance c - sq - R
    mid = sq + _RADIUS
    low, high = sums[:, :mid - _RADIUS + 1].sum(1, keepdim=True), sums[:, mid + _RADIUS:].sum(1, keepdim=True)
    return torch.cat([low, sums[:, mid - _RADIUS + 1:mid + _RADIUS], high], 1)


# ---- the framework's calls

def _package():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sc25-stof-ad_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    from stof import quant, scores
    return quant, scores


def _own(s):
    quant, scores = _package()
    case = s["case"]
    if case["op"] == "linear":
        return quant.linear_i8(s["x"], s["wq"], s["ws"], bias=s["bias"], act=case["act"])
    mask = scores.ScoreMask(causal=case["causal"], prefix=s["prefix"], kv_len=s["kv_len"], docs=s["docs"],
                            q_start="end" if case["op"] == "decode" else None)
    rule = dict(cap=case["cap"] or None, slopes=s["slopes"])
    if case["op"] != "train":
        return scores.score_attn(s["q"], s["k"], s["v"], mask, bias=s["bias"], **rule)
    leaves = [t.detach().requires_grad_() for t in (s["q"], s["k"], s["v"], s["bias"]) if t is not None]
    out = scores.score_attn(*leaves[:3], mask, bias=leaves[3] if len(leaves) > 3 else None, **rule)
    return [out.detach(), *torch.autograd.grad(out, leaves, s["dout"])]


def run(state):
    if own:
        return _own(state)
    return _plain_linear(state) if state["case"]["op"] == "linear" else _plain_attn(state)


# ---- floors

def _pairs(case):
    """Query-key pairs of one head that carry work (the padding of a ragged batch at its expected share)."""
    sq, sk = case["sq"], case["sk"]
    n = sq * (sk - sq) + sq * (sq + 1) / 2 if case["causal"] else sq * sk
    if case["prefix"] and sk == sq:
        n += (sq / 4) ** 2 / 2          # the part of an expected prefix of sq / 4 that lies after the diagonal
    if case["docs"]:
        n *= 0.27                       # about seven documents of random length: the expected sum of squared shares
    if case["ragged"]:
        n *= 0.625
    return case["b"] * n


def work(case):
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": 2 * m * k + n * k + 4 * n + 2 * m * n + (2 * n if case["use_bias"] else 0), "flops": 2 * m * k * n}
    b, hq, hkv, sq, sk, d = (case[n] for n in ("b", "hq", "hkv", "sq", "sk", "d"))
    keys = sk * (0.625 if case["ragged"] else 1.0)
    queries, cache = 2 * b * hq * sq * d, 2 * b * hkv * keys * d
    table = 2 * hq * (2 * _RADIUS + 1) if case["bias"] == "table" else 0
    flops = 4 * d * hq * _pairs(case)
    if case["op"] == "train":           # q, k, v, dout in; out and four gradients out; five products after the two of the forward pass
        return {"bytes": 4 * queries + 4 * cache + 2 * table, "flops": 3.5 * flops}
    return {"bytes": 2 * queries + 2 * cache + table, "flops": flops}


# ---- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        x, w = s["x"].double(), s["wq"].double() * s["ws"].double()[:, None]
        a = x.abs().max(dim=1).values
        steps = torch.round(x * 127.0 / torch.where(a == 0, 1.0, a)[:, None])
        y = torch.mm(steps * (a / 127.0)[:, None], w.t().contiguous())
        if s["bias"] is not None:
            y = y + s["bias"].double()
        return {"none": lambda t: t, "relu": lambda t: t.clamp_min(0), "gelu": lambda t: t * torch.special.ndtr(t)}[case["act"]](y)
    b, hq, hkv, sq, sk, d = (case[n] for n in ("b", "hq", "hkv", "sq", "sk", "d"))
    train = case["op"] == "train"
    out = torch.zeros(b, hq, sq, d, dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(out), *(torch.zeros(b, hkv, sk, d, dtype=torch.float64, device="cuda") for _ in range(2))
    dt = torch.zeros(hq, 2 * _RADIUS + 1, dtype=torch.float64, device="cuda")
    for n in range(b):
        keys = int(s["kv_len"][n]) if s["kv_len"] is not None else sk
        first = keys - sq if case["op"] == "decode" else sk - sq
        pos = torch.arange(first, first + sq, device="cuda")[:, None]
        key = torch.arange(keys, device="cuda")[None, :]
        ban = torch.zeros(sq, keys, dtype=torch.bool, device="cuda")
        if case["causal"]:
            ban |= key > pos
            if s["prefix"] is not None:
                ban[:, :int(s["prefix"][n])] = False
        if s["docs"] is not None:
            ids = s["docs"][n]
            ban |= (ids[:, None] != ids[None, :keys]) | (ids < 0)[:, None]
        lonely = ban.all(1, keepdim=True)
        for h in range(hq):
            m = h * hkv // hq
            leaf = [t.double().detach().requires_grad_(train) for t in (s["q"][n, h], s["k"][n, m, :keys], s["v"][n, m, :keys])]
            tab = s["bias"][h].double().detach().requires_grad_(train) if s["bias"] is not None else None
            z = torch.mm(leaf[0], leaf[1].t()) * d ** -0.5
            if case["cap"]:
                z = torch.tanh(z / case["cap"]) * case["cap"]
            if s["slopes"] is not None:
                z = z - (pos - key).abs() * s["slopes"][h].double()
            if tab is not None:
                z = z + tab[torch.clamp(key - pos, min=-_RADIUS, max=_RADIUS) + _RADIUS]
            prob = torch.softmax(z.masked_fill(ban & ~lonely, -math.inf), 1).masked_fill(lonely, 0.0)
            o = torch.mm(prob, leaf[2])
            out[n, h] = o.detach()
            if train:
                grads = torch.autograd.grad(o, leaf + ([tab] if tab is not None else []), s["dout"][n, h].double())
                dq[n, h] = grads[0]
                dk[n, m, :keys] += grads[1]
                dv[n, m, :keys] += grads[2]
                if tab is not None:
                    dt[h] += grads[3]
    if not train:
        return out
    return [out, dq, dk, dv] + ([dt] if s["bias"] is not None else [])
