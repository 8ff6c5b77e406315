"""What the backward pass of the score attention hands to the library, without a GPU: a stand-in library notes the
arguments.  Tensors that come back from saved-tensor hooks may lie in memory otherwise than the ones that were saved."""
import ctypes

import pytest
import torch

from stof import _lib, scores
from stof.ops import StofError
from stof.scores import ScoreMask, score_attn

Q, K, V, DOUT, OUT, LSE = 1, 2, 3, 0, 4, 5                        # places in stof_score_attn_bwd's arguments
SLOPES, PREFIX, KV_LEN, DOCS_Q, DOCS_K, CAUSAL = 11, 12, 13, 14, 15, 19
STRIDES = {DOUT: 22, Q: 23, K: 24, V: 25, OUT: 26}


class OnGpu(torch.Tensor):
    """A CPU tensor that passes for one of the GPU; nothing reads its memory."""
    is_cuda = property(lambda self: True)


class Library:
    def __init__(self):
        self.bwd, self.read, self.values = None, {}, {}

    def stof_score_attn_workspace_bytes(self, *a):
        return 0

    stof_score_attn_bwd_workspace_bytes = stof_score_attn_workspace_bytes

    def stof_score_attn_fwd(self, *a):
        return 0

    def stof_score_attn_bwd(self, *a):
        self.bwd = a
        self.values = {at: list((kind * n).from_address(a[at])) for at, (kind, n) in self.read.items()}
        return 0


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(_lib, "lib", lambda binding=None: lib)
    monkeypatch.setattr(_lib, "i64x3", lambda a, b, c: (a, b, c))
    monkeypatch.setattr(scores, "_stream", lambda dev: 0)
    monkeypatch.setattr(scores, "_current_device", lambda: None)
    return lib


def _gpu(t):
    return t.as_subclass(OnGpu)


def _packed(B=2, H=4, S=100, D=64):
    qkv = torch.zeros(B, S, 3 * H * D, dtype=torch.float16)
    return [_gpu(qkv[..., n * H * D:(n + 1) * H * D].view(B, S, H, D).permute(0, 2, 1, 3)).detach().requires_grad_() for n in range(3)]


def _end(t):
    return t.data_ptr() + 2 * (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1)


REPACK = {
    "copied": lambda t: t.clone(memory_format=torch.contiguous_format),
    "as it was": lambda t: t,
    "heads and rows exchanged": lambda t: t.transpose(1, 2).contiguous().transpose(1, 2) if t.dim() == 4 else t.clone(),
    "head size not innermost": lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() == 4 else t.clone(),
}


@pytest.mark.parametrize("how", REPACK)
@pytest.mark.parametrize("keys", ["packed", "expanded", "permuted"])
def test_strides_are_those_of_the_tensors_that_are_read(library, how, keys):
    q, k, v = _packed()
    if keys == "expanded":
        k, v = (_gpu(torch.zeros(2, 1, 100, 64, dtype=torch.float16).expand(2, 4, 100, 64)).detach().requires_grad_() for _ in range(2))
    if keys == "permuted":
        k, v = (_gpu(torch.zeros(100, 2, 4, 64, dtype=torch.float16).permute(1, 2, 0, 3)).detach().requires_grad_() for _ in range(2))
    back = []

    def unpack(t):
        back.append(REPACK[how](t))
        return back[-1]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        out = score_attn(q, k, v, ScoreMask(causal=True))
    out.backward(torch.zeros_like(out))
    for at, shape in ((Q, q.shape), (K, k.shape), (V, v.shape), (OUT, q.shape)):
        st = library.bwd[STRIDES[at]]
        last = library.bwd[at] + 2 * (sum((n - 1) * s for n, s in zip(shape, st)) + shape[3])
        held = [t for t in back if t.dim() == 4 and t.shape == shape and library.bwd[at] == t.data_ptr() and st == t.stride()[:3] and last == _end(t)]
        # a tensor as it came back, or (D not innermost) a contiguous copy of one
        assert held or (how == "head size not innermost" and st == (shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3])), (at, st)


def _every_second(t):
    """The values of t at every second place of a larger tensor; 1, 2, 3, ... for lse, which nothing computes here."""
    if t.dim() == 4:
        return t
    wide = torch.full((*t.shape, 2), -7, dtype=t.dtype)
    wide[..., 0] = torch.arange(1, 1 + t.numel()).view(t.shape) if t.shape == (2, 4, 100) else t
    return _gpu(wide[..., 0])


def test_statistics_and_slopes_that_come_back_strided(library):
    library.read = {LSE: (ctypes.c_float, 800), SLOPES: (ctypes.c_float, 4)}
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, _every_second):
        out = score_attn(*_packed(), slopes=_gpu(torch.arange(1.0, 5.0)))
    out.backward(torch.zeros_like(out))
    for at, (_, n) in library.read.items():
        assert library.values[at] == list(range(1, n + 1)), at


@pytest.mark.parametrize("change", ["type", "shape", "device"])
@pytest.mark.parametrize("which", [torch.float16, torch.float32])
def test_tensors_of_another_kind_are_refused(library, change, which):
    change = {"type": lambda t: t.double(), "shape": lambda t: t[..., :1], "device": lambda t: t.to("meta")}[change]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t) if t.dtype == which else t):
        out = score_attn(*_packed())
    with pytest.raises(StofError, match="saved"):
        out.backward(torch.zeros_like(out))
    assert library.bwd is None


def test_rule_tensors_that_come_back_strided(library):
    i32 = lambda *s: _gpu(torch.arange(1, 1 + torch.Size(s).numel(), dtype=torch.int32).view(*s))
    mask = ScoreMask(causal=True, prefix=i32(2), kv_len=i32(2), docs=i32(2, 100))
    library.read = {PREFIX: (ctypes.c_int32, 2), KV_LEN: (ctypes.c_int32, 2), DOCS_Q: (ctypes.c_int32, 200), DOCS_K: (ctypes.c_int32, 200)}
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, _every_second):
        out = score_attn(*_packed(), mask)
    out.backward(torch.zeros_like(out))
    for at, (_, n) in library.read.items():
        assert library.values[at] == list(range(1, n + 1)), at


@pytest.mark.parametrize("change", ["type", "shape", "device"])
def test_rule_tensors_of_another_kind_are_refused(library, change):
    change = {"type": lambda t: t.long(), "shape": lambda t: t[..., :1], "device": lambda t: t.to("meta")}[change]
    mask = ScoreMask(kv_len=_gpu(torch.zeros(2, dtype=torch.int32)))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t) if t.dtype == torch.int32 else t):
        out = score_attn(*_packed(), mask)
    with pytest.raises(StofError, match="saved"):
        out.backward(torch.zeros_like(out))
    assert library.bwd is None


def test_a_mask_object_changed_between_the_passes(library):
    """The backward pass takes the rule of the forward pass, whatever the object holds by then."""
    i32 = lambda *s: _gpu(torch.arange(1, 1 + torch.Size(s).numel(), dtype=torch.int32).view(*s))
    mask = ScoreMask(causal=True, prefix=i32(2), kv_len=i32(2), docs=i32(2, 100))
    was = {PREFIX: mask.prefix.data_ptr(), KV_LEN: mask.kv_len.data_ptr(), DOCS_Q: mask.docs_q.data_ptr(), DOCS_K: mask.docs_k.data_ptr(), CAUSAL: 1}
    out = score_attn(*_packed(), mask)
    keep = [mask.prefix, mask.kv_len, mask.docs_q]
    mask.causal, mask.prefix, mask.kv_len, mask.docs_q, mask.docs_k = 0, None, i32(1), i32(2, 3), None
    out.backward(torch.zeros_like(out))
    assert {at: library.bwd[at] for at in was} == was and len(keep) == 3


def test_tensors_given_to_a_mask_object_later_are_checked(library):
    """Another type is read as other numbers, an expanded tensor past its end: both refused, as by the constructor."""
    q, k, v = (t.detach() for t in _packed())
    i32 = lambda *s: _gpu(torch.zeros(*s, dtype=torch.int32))
    for name, good, bad in (("kv_len", i32(2), i32(1).expand(2)), ("kv_len", i32(2), i32(2).long()), ("prefix", i32(2), i32(4)[::2]),
                            ("docs_q", i32(2, 100), i32(2, 1).expand(2, 100)), ("docs_k", i32(2, 100), i32(2, 100).short())):
        mask = ScoreMask(causal=True, kv_len=i32(2), prefix=i32(2), docs=i32(2, 100))
        setattr(mask, name, good)
        score_attn(q, k, v, mask)
        setattr(mask, name, bad)
        with pytest.raises(StofError):
            score_attn(q, k, v, mask)


def test_gradients_the_kernels_cannot_read_as_they_lie_are_copied(library):
    """Rows more than 2^23 elements apart, an odd address, an odd stride."""
    q, k, v = (_gpu(torch.zeros(1, 2, 3, 64, dtype=torch.float16)).requires_grad_() for _ in range(3))
    out = score_attn(q, k, v)
    base = torch.zeros(2 * (1 << 23) + 4096, dtype=torch.float16)
    for dout in (base.as_strided((1, 2, 3, 64), (64, 64, (1 << 23) + 8, 1)), base[1:385].view(1, 2, 3, 64), base.as_strided((1, 2, 3, 64), (400, 200, 65, 1))):
        torch.autograd.grad(out, (q, k, v), _gpu(dout), retain_graph=True)
        assert library.bwd[STRIDES[DOUT]] == (384, 192, 64) and library.bwd[DOUT] % 16 == 0
