"""Linear operator in 8-bit integers: activations quantised per token as they arrive, weights per output
channel once, the product exact in 32-bit integers, scales, bias and activation in its epilogue.  The 8-bit
counterpart of ``fused.gemm_bias_act``.

    wq, ws = quantize_rows_i8(W)                       # once: W [N,K] in 16 bits (nn.Linear orientation)
    y = linear_i8(x, wq, ws, bias, act="gelu")          # x [..., K] in 16 bits -> [..., N]

    xq, xs = quantize_rows_i8(x)                       # several products on one x: quantise it once
    up, gate = (gemm_i8(xq, xs, *w, dtype=x.dtype) for w in (w_up, w_gate))

A row's scale is its largest magnitude / 127; values are ``round(127 x / max)``, ties to even, from the exact
quotient.  Rows of zeros have scale 0; a row with an infinity or NaN has scale NaN, so its outputs are NaN.
For inference: there is no gradient, and tensors that ask for one (x, scales, bias) or carry a forward-mode tangent are
refused; under ``torch.no_grad()`` parameters are taken."""
import torch

from . import _lib
from ._lib import StofError, check
from .fused import ACT, _DTYPES, _p, _stream
from .ops import _current_device, _refuse_tangents

__all__ = ["quantize_rows_i8", "gemm_i8", "linear_i8"]


def _call(dev, fn, what, *args):
    if dev.index == _current_device():
        rc = fn(*args)
        if rc:
            check(rc, what)
    else:
        with torch.cuda.device(dev):
            check(fn(*args), what)


def _elems(name, t):
    dt = _DTYPES.get(t.dtype) if t.is_cuda else None
    if dt is None:
        raise StofError(f"{name} must be a CUDA float16 or bfloat16 tensor")
    return dt


def _no_gradient(**tensors):
    """Refuses tensors (or None) that ask for a gradient or carry a forward-mode tangent."""
    for name, t in tensors.items():
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise StofError(f"{name} requires a gradient: the 8-bit operators have none (call them under torch.no_grad())")
    _refuse_tangents(*tensors.values())


def _rows2d(name, t, align):
    """[..., K] as (2-D view, row stride): unit stride in K, rows ``align`` elements aligned; a copy if it is neither."""
    if t.dim() == 0 or t.shape[-1] == 0:
        raise StofError(f"{name} must be [..., K] with K > 0")
    K = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(-1, K)
    s = t.stride(0) if t.shape[0] > 1 else K
    if t.stride(1) != 1 or s % align or s < K or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)     # (contiguous() returns rows at an odd address as they are)
        s = K
    return t, s


def quantize_rows_i8(x):
    """``x`` ``[..., K]`` (fp16 or bfloat16, K a multiple of 16) -> int8 ``[..., K]`` and its scales, fp32 ``[...]``."""
    dt = _elems("x", x)
    _no_gradient(x=x)
    K = x.shape[-1] if x.dim() else 0
    if K % 16 or K == 0 or K > 131056:
        raise StofError(f"K must be a multiple of 16 up to 131056, got {K}")
    x2, ldx = _rows2d("x", x, 8)
    M = x2.shape[0]
    xq = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    xs = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    if M:
        _call(x.device, _lib.lib().stof_quantize_rows_i8, "stof_quantize_rows_i8",
              x2.data_ptr(), xq.data_ptr(), xs.data_ptr(), M, K, ldx, K, dt, _stream(x))
    return xq, xs


def _weights(wq, w_scale, bias, K, dev, dtype, act):
    if not (wq.dtype == torch.int8 and wq.dim() == 2 and wq.device == dev and wq.shape[1] == K and wq.stride(1) == 1):
        raise StofError(f"wq must be an int8 [N, {K}] tensor on x's device with contiguous rows")
    N = wq.shape[0]
    if N == 0 or N % 8:
        raise StofError(f"N must be a multiple of 8, got {N}")
    if K % 16 or K == 0 or K > 131056:
        raise StofError(f"K must be a multiple of 16 up to 131056, got {K}")
    ldw = wq.stride(0) if N > 1 else K
    if not (w_scale.dtype == torch.float32 and w_scale.shape == (N,) and w_scale.is_contiguous() and w_scale.device == dev):
        raise StofError(f"w_scale must be a contiguous float32 [{N}] tensor on x's device")
    if bias is not None and not (bias.dtype == dtype and bias.shape == (N,) and bias.is_contiguous() and bias.device == dev):
        raise StofError(f"bias must be a contiguous [{N}] tensor of the output's dtype on x's device")
    if act not in ACT:
        raise StofError(f"act must be one of {sorted(ACT)}, got {act!r}")
    return N, ldw


def _output(out, shape, dtype, dev):
    if out is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    if out.shape != shape or out.dtype != dtype or out.device != dev or not out.is_contiguous():
        raise StofError(f"out must be a contiguous {list(shape)} tensor of dtype {dtype} on x's device")
    return out


def gemm_i8(xq, x_scale, wq, w_scale, bias=None, act="none", dtype=torch.float16, out=None):
    """``act((xq @ wq^T) * x_scale * w_scale + bias)`` on quantised rows: xq int8 ``[..., K]``, x_scale fp32 ``[...]``,
    wq int8 ``[N, K]``, w_scale fp32 ``[N]``, bias ``[N]`` of the output's ``dtype`` (fp16 or bfloat16)."""
    if not (xq.is_cuda and xq.dtype == torch.int8):
        raise StofError("xq must be a CUDA int8 tensor")
    if dtype not in _DTYPES:
        raise StofError(f"dtype must be float16 or bfloat16, got {dtype}")
    K = xq.shape[-1] if xq.dim() else 0
    N, ldw = _weights(wq, w_scale, bias, K, xq.device, dtype, act)
    x2, ldq = _rows2d("xq", xq, 16)
    M = x2.shape[0]
    if not (x_scale.dtype == torch.float32 and x_scale.shape == xq.shape[:-1] and x_scale.device == xq.device):
        raise StofError(f"x_scale must be a float32 {list(xq.shape[:-1])} tensor on xq's device")
    _no_gradient(x_scale=x_scale, w_scale=w_scale, bias=bias)
    x_scale = x_scale.contiguous()
    y = _output(out, xq.shape[:-1] + (N,), dtype, xq.device)
    if M:
        _call(xq.device, _lib.lib().stof_gemm_i8_bias_act, "stof_gemm_i8_bias_act",
              x2.data_ptr(), x_scale.data_ptr(), wq.data_ptr(), w_scale.data_ptr(), _p(bias), y.data_ptr(),
              M, N, K, ldq, ldw, N, ACT[act], _DTYPES[dtype], _stream(xq))
    return y


def linear_i8(x, wq, w_scale, bias=None, act="none", out=None):
    """``act(x @ (wq * w_scale)^T + bias)`` with x quantised per token: x ``[..., K]`` fp16 or bfloat16, wq int8 ``[N, K]``
    with scales fp32 ``[N]`` (``quantize_rows_i8``), bias ``[N]`` of x's dtype.  One launch up to 16 tokens
    whose quantised rows fit 64 KB of LDS (16 of them up to K = 4032), else two.  ``out`` must not overlap the inputs."""
    dt = _elems("x", x)
    K = x.shape[-1] if x.dim() else 0
    N, ldw = _weights(wq, w_scale, bias, K, x.device, x.dtype, act)
    _no_gradient(x=x, w_scale=w_scale, bias=bias)
    x2, ldx = _rows2d("x", x, 8)
    M = x2.shape[0]
    shape = (M, N) if x.dim() == 2 else x.shape[:-1] + (N,)
    y = x.new_empty(shape) if out is None else _output(out, shape, x.dtype, x.device)
    if M:
        lib = _lib.lib()
        nbytes = lib.stof_linear_i8_workspace_bytes(M, K)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None   # this call's own
        _call(x.device, lib.stof_linear_i8, "stof_linear_i8",
              x2.data_ptr(), wq.data_ptr(), w_scale.data_ptr(), _p(bias), y.data_ptr(), M, N, K, ldx, ldw, N, ACT[act], dt,
              _p(ws), nbytes, _stream(x))
    return y
