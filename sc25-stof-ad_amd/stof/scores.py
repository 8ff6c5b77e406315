"""Attention whose scores follow a rule: capped by a tanh, biased by the distance of query and key, and
restricted by lengths, causality, prefixes and packed documents.  The reference's operators take 0/1
masks only (src/ops/package_op.py:10-74); this is the counterpart for layers whose scores are more than
scaled products, for training them and for serving them token by token.

    mask = ScoreMask(causal=True, docs=doc_ids)                # what a batch allows
    out = score_attn(q, k, v, mask, cap=50.0)                  # [B,Hq,S,D]; differentiable
    out = score_attn(q1, cache_k, cache_v, ScoreMask(kv_len=lengths, q_start="end"), slopes=slopes)

Query ``i`` of a sample stands at position ``p_i``, query head ``h`` reads key head ``h // (Hq // Hkv)``:

    t_ij = scale q_i.k_j,   cap tanh(t_ij / cap) with ``cap``
    s_ij = t_ij + bias[h, clip(j - p_i, -R, R) + R]   or   t_ij - slopes[h] |p_i - j|
    allowed: j < kv_len, and (causal) j <= p_i or j < prefix, and doc_i = doc_j >= 0
    out_i = softmax over the allowed j, times v;  zeros for a row without allowed keys

Everything runs in libstof_hip.so; there is no PyTorch fallback.
"""
import math

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import StofError, check
from .ops import _DTYPES, _ptr, _require, _stream

__all__ = ["ScoreMask", "score_attn", "score_attn_backward", "MAX_RADIUS"]

MAX_RADIUS = 1024
_FORMS = {None: -1, "auto": -1, "wide": 0, "rows": 1}


class ScoreMask:
    """Which keys a query may attend to.

    ``causal``   keys up to the query's own position
    ``prefix``   int32 ``[B]``: with ``causal``, the first ``prefix`` keys are open to every query
    ``kv_len``   int32 ``[B]``: keys from there on do not exist (padding, the free part of a cache)
    ``docs``     int32 ``[B,S]``, or a pair ``([B,Sq], [B,Sk])``: a query sees the keys of its own document;
                 negative = no document (padding)
    ``q_start``  position of the first query: None = ``Sk - Sq``, an int, or ``"end"`` = ``kv_len - Sq`` of
                 each sample (the queries are the last tokens of a cache)

    The tensors are read by the launches, not here: a serving loop keeps one object and writes new lengths
    into ``kv_len``.  Contents are not checked (that would synchronise); lengths are clamped to [0, Sk].
    Keys past ``kv_len`` and keys without a document are never used as values, whatever they hold.  A
    non-finite key or value that SOME query of a sample may attend to can reach other rows of its
    64 x 64 tile, as it does in a dense product."""

    __slots__ = ("causal", "prefix", "kv_len", "docs_q", "docs_k", "q_start")

    def __init__(self, causal=False, prefix=None, kv_len=None, docs=None, q_start=None):
        for name, t in (("prefix", prefix), ("kv_len", kv_len)):
            _require(t is None or (torch.is_tensor(t) and t.dtype == torch.int32 and t.dim() == 1 and t.is_contiguous()),
                     f"{name} must be a contiguous int32 tensor [B]")
        _require(prefix is None or causal, "a prefix opens keys that a causal rule closes: it needs causal=True")
        dq, dk = docs if isinstance(docs, (tuple, list)) else (docs, docs)
        for t in (dq, dk):
            _require(docs is None or (torch.is_tensor(t) and t.dtype == torch.int32 and t.dim() == 2 and t.is_contiguous()),
                     "docs must be a contiguous int32 tensor [B,S] or a pair of them")
        _require(q_start is None or q_start == "end" or (type(q_start) is int and abs(q_start) <= 1 << 29),
                 f"q_start must be None, an int or 'end', got {q_start!r}")
        _require(q_start != "end" or kv_len is not None, "q_start='end' needs kv_len")
        self.causal, self.prefix, self.kv_len, self.q_start = bool(causal), prefix, kv_len, q_start
        self.docs_q, self.docs_k = dq, dk

    def _check(self, B, Sq, Sk, dev):
        for name, t, shape in (("prefix", self.prefix, (B,)), ("kv_len", self.kv_len, (B,)),
                               ("docs", self.docs_q, (B, Sq)), ("docs", self.docs_k, (B, Sk))):
            if t is not None and (t.shape != shape or t.device != dev):
                raise StofError(f"{name} must be {list(shape)} on q's device, got {list(t.shape)} on {t.device}")


_NO_MASK = ScoreMask()


def _checked(q, k, v, mask, cap, scale, bias, slopes):
    """The argument checks of forward and backward; the rule's numbers as the C ABI takes them."""
    if not q.is_cuda:
        raise StofError("q must be a CUDA tensor (this path has no CPU implementation)")
    dt = _DTYPES.get(q.dtype)
    if dt is None:
        raise StofError(f"q must be float16 or bfloat16, got {q.dtype}")
    dev = q.device
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4 or t.stride(3) != 1:
            raise StofError(f"{name} must be [B,H,S,D] with contiguous D")
        if t.dtype != q.dtype or t.device != dev:
            raise StofError(f"{name} must have q's dtype and device")
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise StofError(f"k and v must be [{B},Hkv,Sk,{D}], got {list(k.shape)} and {list(v.shape)}")
    if Hkv == 0 or Hq % Hkv != 0:
        raise StofError(f"the number of query heads ({Hq}) must be a multiple of the number of key heads ({Hkv})")
    if D not in (64, 128):
        raise StofError(f"head size must be 64 or 128, got {D}")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < 1e30:
        raise StofError(f"scale must be positive, got {scale}")
    cap = 0.0 if cap is None else float(cap)
    if cap != 0.0 and not 1e-30 < cap < 1e30:
        raise StofError(f"cap must be positive, got {cap}")
    radius = -1
    if bias is not None:
        if slopes is not None:
            raise StofError("bias and slopes exclude each other")
        if not (bias.dim() == 2 and bias.shape[0] == Hq and bias.shape[1] % 2 == 1 and bias.is_contiguous()
                and bias.dtype == q.dtype and bias.device == dev):
            raise StofError(f"bias must be a contiguous [{Hq}, 2 R + 1] tensor of q's dtype and device")
        radius = bias.shape[1] // 2
        if radius > MAX_RADIUS:
            raise StofError(f"bias must tell apart at most {MAX_RADIUS} distances to each side, got {radius}")
    elif slopes is not None:
        if not (slopes.shape == (Hq,) and slopes.dtype == torch.float32 and slopes.is_contiguous() and slopes.device == dev):
            raise StofError(f"slopes must be a contiguous float32 [{Hq}] tensor on q's device")
        if slopes.requires_grad:
            raise StofError("slopes are constants of the rule: there is no gradient for them")
    mask._check(B, Sq, Sk, dev)
    q_end = 1 if mask.q_start == "end" else 0
    q_start = 0 if q_end else (Sk - Sq if mask.q_start is None else mask.q_start)
    return dt, scale, cap, radius, q_start, q_end


def _forward(q, k, v, mask, scale, cap, bias, slopes, out, out_layout, want_lse, launch_form):
    dt, scale, cap, radius, q_start, q_end = _checked(q, k, v, mask, cap, scale, bias, slopes)
    if launch_form not in _FORMS:
        raise StofError(f"launch form must be one of None, 'auto', 'wide', 'rows', got {launch_form!r}")
    form = _FORMS[launch_form]
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    dev = q.device
    if out_layout == "bhsd":
        if out is None:
            out = torch.empty((B, Hq, Sq, D), dtype=q.dtype, device=dev)
        elif out.shape != q.shape or out.stride(3) != 1:
            raise StofError("out must be [B,H,S,D] with contiguous D")
        ostr = (out.stride(0), out.stride(1), out.stride(2))
    elif out_layout == "bshd":
        if out is None:
            out = torch.empty((B, Sq, Hq * D), dtype=q.dtype, device=dev)
        elif out.shape != (B, Sq, Hq * D) or out.stride(2) != 1:
            raise StofError("out must be [B,S,H*D] with contiguous last dim")
        ostr = (out.stride(0), D, out.stride(1))
    else:
        raise StofError(f"unknown out_layout {out_layout!r}")
    if out.dtype != q.dtype or out.device != dev:
        raise StofError("out must have q's dtype and device")
    lse = torch.empty((B, Hq, Sq), dtype=torch.float32, device=dev) if want_lse else None
    if B == 0 or Hq == 0 or Sq == 0 or Sk == 0:
        out.zero_()
        if lse is not None:
            lse.fill_(-math.inf)
        return out, lse
    lib = _lib.lib()
    nbytes = lib.stof_score_attn_workspace_bytes(B, Hq, Hkv, Sq, Sk, D, radius, mask.docs_q is not None, form)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None   # this call's own: calls may overlap on other streams and graphs
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    args = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(lse), _ptr(bias), _ptr(slopes), _ptr(mask.prefix),
            _ptr(mask.kv_len), _ptr(mask.docs_q), _ptr(mask.docs_k), scale, cap, radius, int(mask.causal), q_start, q_end,
            _lib.i64x3(qs[0], qs[1], qs[2]), _lib.i64x3(ks[0], ks[1], ks[2]), _lib.i64x3(vs[0], vs[1], vs[2]), _lib.i64x3(*ostr),
            B, Hq, Hkv, Sq, Sk, D, dt, form, _ptr(ws), nbytes, _stream(dev))
    if dev.index == torch.cuda.current_device():
        check(lib.stof_score_attn_fwd(*args), "stof_score_attn_fwd")
    else:
        with torch.cuda.device(dev):
            check(lib.stof_score_attn_fwd(*args), "stof_score_attn_fwd")
    return out, lse


def _rows(t):
    """t as the kernels read it: unit stride in D, other strides multiples of 8, 16-byte aligned (else a copy)."""
    s = t.stride()
    if s[3] == 1 and not (s[0] % 8 or s[1] % 8 or s[2] % 8 or t.data_ptr() % 16):
        return t
    return t.contiguous()


def score_attn_backward(dout, q, k, v, out, lse, mask=None, scale=None, cap=None, bias=None, slopes=None):
    """Gradients of ``sum(out * dout)`` for ``out, lse = score_attn(..., return_lse=True)``: ``(dq, dk, dv, dbias)``,
    contiguous, ``dbias`` None without a table.  What autograd calls; on its own
    it is for training loops that keep their own graph of calls, a captured one among them.  ``dout`` and ``out``
    are ``[B,Hq,Sq,D]`` views; the rule must be the forward pass's."""
    mask = _NO_MASK if mask is None else mask
    dt, scale, cap, radius, q_start, q_end = _checked(q, k, v, mask, cap, scale, bias, slopes)
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    dev = q.device
    for name, t in (("dout", dout), ("out", out)):
        if t.shape != q.shape or t.dtype != q.dtype or t.device != dev:
            raise StofError(f"{name} must have q's shape, dtype and device")
    if lse.shape != (B, Hq, Sq) or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != dev:
        raise StofError(f"lse must be the float32 [{B}, {Hq}, {Sq}] tensor of the forward pass")
    new = lambda like: torch.empty(like.shape, dtype=q.dtype, device=dev)
    dq, dk, dv = new(q), new(k), new(v)
    db = new(bias) if bias is not None else None
    if B == 0 or Hq == 0 or Sq == 0 or Sk == 0:
        for t in (dq, dk, dv, db):
            if t is not None:
                t.zero_()
        return dq, dk, dv, db
    dout, out = _rows(dout), _rows(out)
    lib = _lib.lib()
    nbytes = lib.stof_score_attn_bwd_workspace_bytes(B, Hq, Hkv, Sq, Sk, D, radius, mask.docs_q is not None)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    s3 = lambda t: _lib.i64x3(*t.stride()[:3])
    args = (dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(db),
            _ptr(bias), _ptr(slopes), _ptr(mask.prefix), _ptr(mask.kv_len), _ptr(mask.docs_q), _ptr(mask.docs_k),
            scale, cap, radius, int(mask.causal), q_start, q_end, s3(dout), s3(q), s3(k), s3(v), s3(out),
            B, Hq, Hkv, Sq, Sk, D, dt, ws.data_ptr(), nbytes, _stream(dev))
    if dev.index == torch.cuda.current_device():
        check(lib.stof_score_attn_bwd(*args), "stof_score_attn_bwd")
    else:
        with torch.cuda.device(dev):
            check(lib.stof_score_attn_bwd(*args), "stof_score_attn_bwd")
    return dq, dk, dv, db


class _ScoreAttn(Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, slopes, mask, scale, cap, out_layout, launch_form):
        out, lse = _forward(q, k, v, mask, scale, cap, bias, slopes, None, out_layout, True, launch_form)
        # the rule's tensors are saved too, so that one changed in place before the backward pass is noticed
        ctx.save_for_backward(q, k, v, out, lse, bias, slopes, mask.prefix, mask.kv_len, mask.docs_q, mask.docs_k)
        ctx.rule = (mask, scale, cap, out_layout)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)          # no zeros for lse
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _dlse):
        if dout is None:
            return (None,) * 10
        q, k, v, out, lse, bias, slopes = ctx.saved_tensors[:7]
        mask, scale, cap, out_layout = ctx.rule
        if out_layout == "bshd":
            B, H, S, D = q.shape
            out, dout = (t.reshape(B, S, H, D).permute(0, 2, 1, 3) for t in (out, dout))
        need = ctx.needs_input_grad
        dq, dk, dv, db = score_attn_backward(dout, q, k, v, out, lse, mask, scale, cap, bias, slopes)
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, db if need[3] else None,
                None, None, None, None, None, None)


def score_attn(q, k, v, mask=None, scale=None, cap=None, bias=None, slopes=None, out=None, out_layout="bhsd",
               return_lse=False, launch_form=None):
    """Attention with a score rule (module docstring).  ``q`` ``[B,Hq,Sq,D]``, ``k`` and ``v`` ``[B,Hkv,Sk,D]``:
    fp16 or, all alike, bfloat16, head size 64 or 128, any lengths, unit stride in D and other strides
    multiples of 8.  ``mask``: a ``ScoreMask`` (None: every key).  ``scale``: default ``1/sqrt(D)``.
    ``bias``: learned distance table ``[Hq, 2R+1]`` of q's dtype, R up to 1024; ``slopes``: fp32 ``[Hq]``, constants.
    Returns ``[B,Hq,Sq,D]`` (``out_layout="bhsd"``) or ``[B,Sq,Hq*D]`` (``"bshd"``), with ``return_lse`` also the
    logarithm of the softmax's denominator, fp32 ``[B,Hq,Sq]``.  Differentiable in q, k, v and bias (through the
    output, not through lse).  ``launch_form``: None, "wide" (128-query tiles) or "rows" (32-row tiles with the
    keys split; single tokens and small grids) - the rule by sizes is in the library."""
    mask = _NO_MASK if mask is None else mask
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (bias is not None and bias.requires_grad)):
        if out is not None:
            raise StofError("out= has no gradient: leave it out, or call under torch.no_grad()")
        o, lse = _ScoreAttn.apply(q, k, v, bias, slopes, mask, scale, cap, out_layout, launch_form)
        return (o, lse) if return_lse else o
    o, lse = _forward(q, k, v, mask, scale, cap, bias, slopes, out, out_layout, return_lse, launch_form)
    return (o, lse) if return_lse else o
