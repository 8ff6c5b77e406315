"""Attention with score rules in float64 on the CPU, from the definition, with its gradients by the
formulas and, beside each result, how far a computation that rounds where the kernels do may be off.

Rounding model.  u = eps / 2 of the tensors' format.  The kernels round P (and dS) to the format before a
product and the result once; sums, scores and statistics are fp32.  A score is a sum of D products, scaled,
capped and biased in fp32: its error is at most (D + 8) 2^-24 (scale sum_d |q_d k_d| + |bias|) + 2^-20 |cap|
(exp2 and reciprocal at 1 ulp inside the cap), which makes a relative error of P of twice that (the
denominator has it too) plus 2^-20 for exp2, sum and division.  Called e_P below:
    out:   (u + e_P) sum_j P |v| + u |out|
    dv:    (u + e_P) sum_i P |dout| + u |dv|
    dS:    (u + 2^-22) |dS| + e_P P (|dP| + |delta|) + 2^-17 P (A + delta_A), A = sum_d |dout v|, delta_A = sum_j P A
           (dP: D products in fp32, <= 2^-17 A; delta: sums of P dP in fp32)
    dq:    scale sum_j err(dS) |k| + u |dq|,  dk likewise,  dtable: sum of err(dS) without its u + u |dtable|
and the smallest number of the format for results that vanish."""
import math

import torch


def allowed(B, Sq, Sk, causal=False, prefix=None, kv_len=None, docs=None, q_start=None):
    """[B,Sq,Sk] bool and the query positions [B,Sq]."""
    dq, dk = docs if isinstance(docs, (tuple, list)) else (docs, docs)
    ok = torch.zeros(B, Sq, Sk, dtype=torch.bool)
    pos = torch.zeros(B, Sq, dtype=torch.int64)
    j = torch.arange(Sk)
    for b in range(B):
        n = Sk if kv_len is None else min(max(int(kv_len[b]), 0), Sk)
        first = Sk - Sq if q_start is None else n - Sq if q_start == "end" else q_start
        for i in range(Sq):
            p = first + i
            pos[b, i] = p
            row = j < n
            if causal:
                row = row & ((j <= p) | (j < (0 if prefix is None else int(prefix[b]))))
            if docs is not None:
                row = row & (dk[b] == dq[b, i]) & (dq[b, i] >= 0)
            ok[b, i] = row
    return ok, pos


def score_attn(q, k, v, scale=None, cap=None, bias=None, slopes=None, dout=None, **mask):
    """dict of name -> (value, bound): out, lse and, with dout, dq, dk, dv, dbias; float64."""
    u = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * 2.0 ** (-9 if q.dtype == torch.float16 else 0)
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    ok, pos = allowed(B, Sq, Sk, **mask)
    ok = ok[:, None]
    live = ok.any(-1, keepdim=True)
    # what no query may use has no value: zeros stand for it, whatever the tensors hold
    used_k = ok.any(2).any(1)[:, None, :, None]
    wide = lambda t: torch.where(used_k, t.double(), 0.0).repeat_interleave(G, 1)
    Q, K, V = torch.where(live, q.double(), 0.0), wide(k), wide(v)
    s = scale * (Q @ K.transpose(-1, -2))
    err = (D + 8) * 2.0 ** -24 * scale * (Q.abs() @ K.abs().transpose(-1, -2))
    th = None
    if cap:
        th = torch.tanh(s / cap)
        s = cap * th
        err = err + 2.0 ** -20 * cap
    dist = torch.arange(Sk)[None, None, :] - pos[:, :, None]
    if slopes is not None:
        w = -slopes.double().view(1, Hq, 1, 1) * dist.abs()[:, None]
        s, err = s + w, err + 2.0 ** -21 * w.abs()
    if bias is not None:
        R = bias.shape[1] // 2
        at = dist.clamp(-R, R) + R
        w = bias.double()[:, at].transpose(0, 1)
        s, err = s + w, err + 2.0 ** -21 * w.abs().clamp(max=1e30)
    s = torch.where(ok, s, -math.inf)
    top = s.amax(-1, keepdim=True) if Sk else torch.full((B, Hq, Sq, 1), -math.inf, dtype=torch.float64)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    tot = e.sum(-1, keepdim=True)
    P = e / torch.where(tot == 0, 1.0, tot)
    lse = (torch.log(tot) + torch.where(top == -math.inf, 0.0, top))[..., 0]
    eP = 2 * torch.where(ok, err, 0.0).amax(-1, keepdim=True) + 2.0 ** -20 if Sk else torch.zeros(B, Hq, Sq, 1)
    out = P @ V
    floor = 2.0 ** -32 if q.dtype == torch.float16 else 0.0      # P times 2^7 by half the smallest fp16 number: what a small P may be off
    res = {"out": (out, ((u + eP) * P + floor * ok) @ V.abs() + u * out.abs() + tiny),
           "lse": (lse, eP[..., 0] + 2.0 ** -21 * lse.abs().nan_to_num(posinf=0.0))}
    if dout is None:
        return res
    dO = torch.where(live, dout.double(), 0.0)
    fold = lambda t: t.view(B, Hkv, G, Sk, D).sum(2)
    dV = fold(P.transpose(-1, -2) @ dO)
    dP = dO @ V.transpose(-1, -2)
    A = dO.abs() @ V.abs().transpose(-1, -2)
    delta, dA = (P * dP).sum(-1, keepdim=True), (P * A).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    eS = 2.0 ** -22 * dS.abs() + eP * P * (dP.abs() + delta.abs()) + 2.0 ** -17 * P * (A + dA)
    res["dv"] = (dV, fold(((u + eP) * P).transpose(-1, -2) @ dO.abs()) + u * dV.abs() + tiny)
    if bias is not None:
        dB, eB = torch.zeros_like(bias, dtype=torch.float64), torch.zeros_like(bias, dtype=torch.float64)
        for b in range(B):
            flat = at[b].reshape(-1)
            dB.index_add_(1, flat, dS[b].reshape(Hq, -1))
            eB.index_add_(1, flat, eS[b].reshape(Hq, -1))
        res["dbias"] = (dB, eB + u * dB.abs() + tiny)
    dT = dS if th is None else dS * (1 - th * th)
    eT = eS if th is None else eS * (1 - th * th) + 2.0 ** -20 * dS.abs()
    eT = eT + u * dT.abs()
    dQ, dK = scale * (dT @ K), fold(scale * (dT.transpose(-1, -2) @ Q))
    res["dq"] = (dQ, scale * (eT @ K.abs()) + u * dQ.abs() + tiny)
    res["dk"] = (dK, fold(scale * (eT.transpose(-1, -2) @ Q.abs())) + u * dK.abs() + tiny)
    return res
