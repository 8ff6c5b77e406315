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
from .ops import _DTYPES, _current_device, _refuse_tangents, _require, _stream

__all__ = ["ScoreMask", "score_attn", "score_attn_backward", "MAX_RADIUS", "MAX_CAP"]

MAX_RADIUS = 1024
MAX_CAP = 1024.0        # the cap is formed to 2^-22 of its size: a larger one would take more from the scores than 16-bit outputs show
_FORMS = {None: -1, "auto": -1, "wide": 0, "rows": 1, "wide2": 2}


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
    A backward pass uses the rule and the tensors of its forward pass: attributes assigned in between change nothing, a
    tensor written to in between is an error.
    Keys past ``kv_len``, keys that causality closes to every query of the sample and keys without a document are
    never used as values, whatever they hold (the free part of a cache).  A non-finite key or value that SOME
    query of a sample may attend to can reach other rows of its 64 x 64 tile, as it does in a dense product."""

    __slots__ = ("causal", "prefix", "kv_len", "docs_q", "docs_k", "q_start")

    def __init__(self, causal=False, prefix=None, kv_len=None, docs=None, q_start=None):
        for name, t in (("prefix", prefix), ("kv_len", kv_len)):
            if t is not None:
                _require(torch.is_tensor(t) and t.dtype == torch.int32 and t.dim() == 1 and t.is_contiguous(),
                         f"{name} must be a contiguous int32 tensor [B]")
        _require(prefix is None or causal, "a prefix opens keys that a causal rule closes: it needs causal=True")
        dq = dk = None
        if docs is not None:
            dq, dk = docs if isinstance(docs, (tuple, list)) else (docs, docs)
            for t in (dq, dk):
                _require(torch.is_tensor(t) and t.dtype == torch.int32 and t.dim() == 2 and t.is_contiguous(),
                         "docs must be a contiguous int32 tensor [B,S] or a pair of them")
        if q_start is not None:
            _require(q_start == "end" or (type(q_start) is int and abs(q_start) <= 1 << 29), "q_start must be None, an int or 'end'")
            _require(q_start != "end" or kv_len is not None, "q_start='end' needs kv_len")
        self.causal, self.prefix, self.kv_len, self.q_start = 1 if causal else 0, prefix, kv_len, q_start
        self.docs_q, self.docs_k = dq, dk

    def _check(self, B, Sq, Sk, dev):
        if self.kv_len is not None:
            _fits("kv_len", self.kv_len, (B,), dev)
        if self.prefix is not None:
            _fits("prefix", self.prefix, (B,), dev)
        if self.docs_q is not None:
            _fits("docs", self.docs_q, (B, Sq), dev)
            _fits("docs", self.docs_k, (B, Sk), dev)


def _fits(name, t, shape, dev):
    # (type and layout again: a mask object may have been given another tensor since it was made)
    if t.shape != shape or t.device != dev or t.dtype != torch.int32 or not t.is_contiguous():
        raise StofError(f"{name} must be a contiguous int32 {list(shape)} tensor on q's device, got {t.dtype} {list(t.shape)} on {t.device}")


_NO_MASK = ScoreMask()


def _refuse(q, k, v, scale, cap, bias, slopes):
    """The refusal of a call that ``_rule`` found wanting, by name."""
    if not q.is_cuda:
        raise StofError("q must be a CUDA tensor (this path has no CPU implementation)")
    if q.dtype not in _DTYPES:
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
    if not 1e-6 <= scale <= 1e6:
        raise StofError(f"scale must be between 1e-6 and 1e6, got {scale}")
    if cap != 0.0 and not 1e-3 <= cap <= MAX_CAP:
        raise StofError(f"cap must be between 1e-3 and {MAX_CAP}, got {cap}")
    if bias is not None and slopes is not None:
        raise StofError("bias and slopes exclude each other")
    if bias is not None:
        if not (bias.dim() == 2 and bias.shape[0] == Hq and bias.shape[1] % 2 == 1 and bias.is_contiguous()
                and bias.dtype == q.dtype and bias.device == dev):
            raise StofError(f"bias must be a contiguous [{Hq}, 2 R + 1] tensor of q's dtype and device")
        raise StofError(f"bias must tell apart at most {MAX_RADIUS} distances to each side, got {bias.shape[1] // 2}")
    if slopes is not None:
        if not (slopes.shape == (Hq,) and slopes.dtype == torch.float32 and slopes.is_contiguous() and slopes.device == dev):
            raise StofError(f"slopes must be a contiguous float32 [{Hq}] tensor on q's device")
        raise StofError("slopes are constants of the rule: there is no gradient for them (detach them, or call under torch.no_grad())")
    raise StofError("these tensors cannot be used together")


class _Rule:
    """A call's checked numbers, as the C ABI takes them: what the backward pass keeps of the rule beside its tensors.  (Not the
    mask object, which may hold another rule by then.)"""

    __slots__ = ("elem", "dt", "dev", "sizes", "scale", "cap", "radius", "causal", "q_start", "q_end")

    def __init__(self, q, k, v, mask, scale, cap, bias, slopes):
        # (one pass over the conditions: this runs on every call; which of them failed is found out by _refuse)
        dtype, dev = q.dtype, q.device
        qs, ks, vs = q.shape, k.shape, v.shape
        scale = (0.0 if len(qs) != 4 or qs[3] == 0 else 1.0 / math.sqrt(qs[3])) if scale is None else float(scale)
        cap = 0.0 if cap is None else float(cap)
        qt, kt, vt = q.stride(), k.stride(), v.stride()
        ok = (q.is_cuda and dtype in _DTYPES and len(qs) == 4 and len(ks) == 4 and vs == ks and qt[3] == 1 and kt[3] == 1 and vt[3] == 1
              and k.dtype == dtype and v.dtype == dtype and k.device == dev and v.device == dev and ks[0] == qs[0] and ks[3] == qs[3]
              and ks[1] > 0 and qs[1] % ks[1] == 0 and (qs[3] == 64 or qs[3] == 128) and 1e-6 <= scale <= 1e6
              and (cap == 0.0 or 1e-3 <= cap <= MAX_CAP))
        radius = -1
        if ok and bias is not None:
            n = bias.shape
            ok = (slopes is None and len(n) == 2 and n[0] == qs[1] and n[1] % 2 == 1 and n[1] <= 2 * MAX_RADIUS + 1 and bias.is_contiguous()
                  and bias.dtype == dtype and bias.device == dev)
            radius = n[-1] // 2
        elif ok and slopes is not None:
            ok = (slopes.shape == qs[1:2] and slopes.dtype == torch.float32 and slopes.is_contiguous() and slopes.device == dev
                  and not (slopes.requires_grad and torch.is_grad_enabled()))
        if not ok:
            _refuse(q, k, v, scale, cap, bias, slopes)
        B, Hq, Sq, D = qs
        Hkv, Sk = ks[1], ks[2]
        if mask is not _NO_MASK:
            mask._check(B, Sq, Sk, dev)
        start = mask.q_start
        self.elem, self.dt, self.dev, self.sizes = dtype, _DTYPES[dtype], dev, (B, Hq, Hkv, Sq, Sk, D)
        self.scale, self.cap, self.radius, self.causal = scale, cap, radius, mask.causal
        self.q_end = 1 if start == "end" else 0
        self.q_start = 0 if self.q_end else (Sk - Sq if start is None else start)


def _forward(q, k, v, r, mask, bias, slopes, out, out_layout, want_lse, launch_form):
    if launch_form not in _FORMS:
        raise StofError(f"launch form must be one of None, 'auto', 'wide', 'wide2', 'rows', got {launch_form!r}")
    form = _FORMS[launch_form]
    B, Hq, Hkv, Sq, Sk, D = sizes = r.sizes
    dev = r.dev
    if out_layout == "bhsd":
        if out is None:
            out = q.new_empty((B, Hq, Sq, D))
            ostr = (Hq * Sq * D, Sq * D, D)
        elif out.shape != q.shape or out.stride(3) != 1 or out.dtype != q.dtype or out.device != dev:
            raise StofError("out must be [B,H,S,D] with contiguous D, of q's dtype and device")
        else:
            ostr = out.stride()
    elif out_layout == "bshd":
        if out is None:
            out = q.new_empty((B, Sq, Hq * D))
            ostr = (Sq * Hq * D, D, Hq * D)
        elif out.shape != (B, Sq, Hq * D) or out.stride(2) != 1 or out.dtype != q.dtype or out.device != dev:
            raise StofError("out must be [B,S,H*D] with contiguous last dim, of q's dtype and device")
        else:
            ostr = (out.stride(0), D, out.stride(1))
    else:
        raise StofError(f"unknown out_layout {out_layout!r}")
    lse = torch.empty((B, Hq, Sq), dtype=torch.float32, device=dev) if want_lse else None
    if B == 0 or Hq == 0 or Sq == 0 or Sk == 0:
        out.zero_()
        if lse is not None:
            lse.fill_(-math.inf)
        return out, lse
    lib = _lib.lib()
    docs_q = mask.docs_q
    nbytes = lib.stof_score_attn_workspace_bytes(B, Hq, Hkv, Sq, Sk, D, docs_q is not None, form)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None   # this call's own: calls may overlap on other streams and graphs
    i64x3, qs, ks, vs = _lib.i64x3, q.stride(), k.stride(), v.stride()
    args = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _at(lse), _at(bias), _at(slopes), _at(mask.prefix),
            _at(mask.kv_len), _at(docs_q), _at(mask.docs_k), r.scale, r.cap, r.radius, r.causal, r.q_start, r.q_end,
            i64x3(qs[0], qs[1], qs[2]), i64x3(ks[0], ks[1], ks[2]), i64x3(vs[0], vs[1], vs[2]), i64x3(ostr[0], ostr[1], ostr[2]),
            *sizes, r.dt, form, _at(ws), nbytes, _stream(dev))
    if dev.index == _current_device():
        check(lib.stof_score_attn_fwd(*args), "stof_score_attn_fwd")
    else:
        with torch.cuda.device(dev):
            check(lib.stof_score_attn_fwd(*args), "stof_score_attn_fwd")
    return out, lse


def _at(t):
    return None if t is None else t.data_ptr()


def _rows(t):
    """t as the kernels read it and its strides: unit stride in D, other strides multiples of 8, rows at most 2^23 apart, 16-byte
    aligned (else a copy; ``contiguous()`` would return a contiguous tensor at an odd address as it is)."""
    s = t.stride()
    if s[3] != 1 or s[0] % 8 or s[1] % 8 or s[2] % 8 or s[2] > 1 << 23 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        s = t.stride()
    return t, _lib.i64x3(s[0], s[1], s[2])


def score_attn_backward(dout, q, k, v, out, lse, mask=None, scale=None, cap=None, bias=None, slopes=None):
    """Gradients of ``sum(out * dout)`` for ``out, lse = score_attn(..., return_lse=True)``: ``(dq, dk, dv, dbias)``,
    contiguous, ``dbias`` None without a table.  What autograd calls; on its own
    it is for training loops that keep their own graph of calls, a captured one among them.  ``dout`` and ``out``
    are ``[B,Hq,Sq,D]`` views; the rule must be the forward pass's."""
    mask = _NO_MASK if mask is None else mask
    r = _Rule(q, k, v, mask, scale, cap, bias, slopes)
    _refuse_tangents(dout, q, k, v, out, lse, bias, slopes)
    for name, t in (("dout", dout), ("out", out)):
        if t.shape != q.shape or t.dtype != q.dtype or t.device != r.dev:
            raise StofError(f"{name} must have q's shape, dtype and device")
    if lse.shape != q.shape[:3] or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != r.dev:
        raise StofError(f"lse must be the float32 {list(q.shape[:3])} tensor of the forward pass")
    return _backward(dout, r, q, k, v, out, lse, bias, slopes, mask.prefix, mask.kv_len, mask.docs_q, mask.docs_k)


def _backward(dout, r, q, k, v, out, lse, bias, slopes, prefix, kv_len, docs_q, docs_k):
    B, Hq, Hkv, Sq, Sk, D = sizes = r.sizes
    dev = r.dev
    dq, dk, dv = q.new_empty((B, Hq, Sq, D)), q.new_empty((B, Hkv, Sk, D)), q.new_empty((B, Hkv, Sk, D))
    db = torch.empty_like(bias) if bias is not None else None
    if B == 0 or Hq == 0 or Sq == 0 or Sk == 0:
        for t in (dq, dk, dv, db):
            if t is not None:
                t.zero_()
        return dq, dk, dv, db
    (dout, ds), (q, qs), (k, ks), (v, vs), (out, os_) = _rows(dout), _rows(q), _rows(k), _rows(v), _rows(out)
    lib = _lib.lib()
    nbytes = lib.stof_score_attn_bwd_workspace_bytes(B, Hq, Hkv, Sq, Sk, D, r.radius, docs_q is not None)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    args = (dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(),
            dv.data_ptr(), _at(db), _at(bias), _at(slopes), _at(prefix), _at(kv_len), _at(docs_q), _at(docs_k),
            r.scale, r.cap, r.radius, r.causal, r.q_start, r.q_end, ds, qs, ks, vs, os_, *sizes, r.dt, ws.data_ptr(), nbytes, _stream(dev))
    if dev.index == _current_device():
        check(lib.stof_score_attn_bwd(*args), "stof_score_attn_bwd")
    else:
        with torch.cuda.device(dev):
            check(lib.stof_score_attn_bwd(*args), "stof_score_attn_bwd")
    return dq, dk, dv, db


def _unpacked(saved, r, out_layout):
    """The saved tensors (``_ScoreAttn.forward``) as the backward pass takes them.  Saved-tensor hooks (activations kept on the
    host, copies) may hand back tensors that lie in memory otherwise than those of the forward pass."""
    B, Hq, Hkv, Sq, Sk, D = r.sizes
    keys = (B, Hkv, Sk, D)
    shapes = ((B, Hq, Sq, D), keys, keys, (B, Sq, Hq * D) if out_layout == "bshd" else (B, Hq, Sq, D), (B, Hq, Sq), (Hq, 2 * r.radius + 1), (Hq,),
              (B,), (B,), (B, Sq), (B, Sk))
    kinds = (r.elem, r.elem, r.elem, r.elem, torch.float32, r.elem, torch.float32, torch.int32, torch.int32, torch.int32, torch.int32)
    dev, tensors = r.dev, []
    for t, shape, kind in zip(saved, shapes, kinds):
        if t is not None:
            if t.shape != shape or t.dtype is not kind or t.device != dev:
                raise StofError(f"a saved tensor came back as {t.dtype} {list(t.shape)} on {t.device}; saved was {kind} {list(shape)} on {dev}")
            if len(shape) < 4 and (t.data_ptr() % 16 or not t.is_contiguous()):        # ([B,H,S,D] views: _backward reads their strides)
                t = t.clone(memory_format=torch.contiguous_format)
        tensors.append(t)
    return tensors


class _ScoreAttn(Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, slopes, rule, mask, out_layout, launch_form):
        out, lse = _forward(q, k, v, rule, mask, bias, slopes, None, out_layout, True, launch_form)
        # the rule's tensors are saved too: one changed in place before the backward pass is noticed, a mask object that
        # was given others by then changes nothing
        ctx.save_for_backward(q, k, v, out, lse, bias, slopes, mask.prefix, mask.kv_len, mask.docs_q, mask.docs_k)
        ctx.rule, ctx.out_layout = rule, out_layout
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)          # no zeros for lse
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _dlse):
        if dout is None:
            return (None,) * 9
        q, k, v, out, *rest = _unpacked(ctx.saved_tensors, ctx.rule, ctx.out_layout)
        if ctx.out_layout == "bshd":
            B, H, S, D = q.shape
            out, dout = (t.reshape(B, S, H, D).permute(0, 2, 1, 3) for t in (out, dout))
        need = ctx.needs_input_grad
        dq, dk, dv, db = _backward(dout, ctx.rule, q, k, v, out, *rest)
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, db if need[3] else None,
                None, None, None, None, None)


def score_attn(q, k, v, mask=None, scale=None, cap=None, bias=None, slopes=None, out=None, out_layout="bhsd",
               return_lse=False, launch_form=None):
    """Attention with a score rule (module docstring).  ``q`` ``[B,Hq,Sq,D]``, ``k`` and ``v`` ``[B,Hkv,Sk,D]``:
    fp16 or, all alike, bfloat16, head size 64 or 128, any lengths, unit stride in D and other strides
    multiples of 8.  ``mask``: a ``ScoreMask`` (None: every key).  ``scale``: default ``1/sqrt(D)``.
    ``bias``: learned distance table ``[Hq, 2R+1]`` of q's dtype, R up to 1024; ``slopes``: fp32 ``[Hq]``, constants
    (a parameter is taken under ``torch.no_grad()`` only).
    ``out`` must not overlap the inputs.  Returns ``[B,Hq,Sq,D]`` (``out_layout="bhsd"``) or ``[B,Sq,Hq*D]`` (``"bshd"``), with ``return_lse`` also the
    logarithm of the softmax's denominator, fp32 ``[B,Hq,Sq]``.  Differentiable in q, k, v and bias (through the
    output, not through lse; reverse mode only: forward-mode tangents are refused).  ``launch_form``: None, "wide" (128-query tiles), "wide2" (those with the keys
    in two parts; small grids) or "rows" (32-row tiles with the keys split; single tokens and smaller grids) - the rule by
    sizes is in the library."""
    mask = _NO_MASK if mask is None else mask
    r = _Rule(q, k, v, mask, scale, cap, bias, slopes)
    _refuse_tangents(q, k, v, bias, slopes)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (bias is not None and bias.requires_grad)):
        if out is not None:
            raise StofError("out= has no gradient: leave it out, or call under torch.no_grad()")
        o, lse = _ScoreAttn.apply(q, k, v, bias, slopes, r, mask, out_layout, launch_form)
    else:
        o, lse = _forward(q, k, v, r, mask, bias, slopes, out, out_layout, return_lse, launch_form)
    return (o, lse) if return_lse else o
