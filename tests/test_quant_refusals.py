"""Host-side argument checks of the 8-bit entry points of the C ABI (no GPU: every call fails validation)."""
import pytest
import torch

from stof import _lib
from stof.ops import StofError
from stof.quant import linear_i8, quantize_rows_i8

P = 4096   # fake, 16-byte aligned, never dereferenced


@pytest.fixture(params=["ctypes", "ext"])
def lib(request):
    h = _lib.lib(request.param)
    if h is None:
        pytest.skip("extension module not built")
    return h


def test_no_cpu_path():
    with pytest.raises(StofError):
        quantize_rows_i8(torch.zeros(2, 16, dtype=torch.float16))
    with pytest.raises(StofError):
        linear_i8(torch.zeros(2, 16, dtype=torch.float16), torch.zeros(8, 16, dtype=torch.int8), torch.zeros(8))


def test_argument_checks(lib):
    q = lambda x=P, xq=P, sx=P, M=4, K=64, ldx=64, ldq=64, dt=0: lib.stof_quantize_rows_i8(x, xq, sx, M, K, ldx, ldq, dt, None)
    assert q(x=None) == -1 and q(xq=None) == -1 and q(sx=None) == -1
    assert q(x=P + 2) == -4 and q(ldx=65) == -4 and q(ldq=72) == -4
    assert q(M=0) == -2 and q(K=40) == -2 and q(K=131072) == -2 and q(ldx=56) == -2 and q(ldq=48) == -2
    assert q(dt=2) == -3
    g = lambda xq=P, sx=P, wq=P, sw=P, b=None, o=P, M=4, N=16, K=64, ldq=64, ldw=64, ldo=16, act=0, dt=0: \
        lib.stof_gemm_i8_bias_act(xq, sx, wq, sw, b, o, M, N, K, ldq, ldw, ldo, act, dt, None)
    assert g(xq=None) == -1 and g(sx=None) == -1 and g(wq=None) == -1 and g(sw=None) == -1 and g(o=None) == -1
    assert g(wq=P + 8) == -4 and g(b=P + 2) == -4 and g(ldw=72) == -4 and g(ldo=20) == -4
    assert g(N=12) == -2 and g(K=24) == -2 and g(ldw=48) == -2 and g(ldo=8) == -2 and g(M=1 << 40) == -2
    assert g(act=4) == -3 and g(dt=3) == -3
    ln = lambda x=P, M=40, ws=P, n=1 << 20, ldx=64: lib.stof_linear_i8(x, P, P, None, P, M, 16, 64, ldx, 64, 16, 0, 0, ws, n, None)
    assert ln(x=None) == -1 and ln(ws=None) == -1 and ln(ws=P + 4) == -4 and ln(n=40 * 64) == -2 and ln(ldx=68) == -4 and ln(ldx=56) == -2
    assert lib.stof_linear_i8_workspace_bytes(1, 64) == 0 and lib.stof_linear_i8_workspace_bytes(40, 64) == 40 * 64 + 160
    assert lib.stof_linear_i8_workspace_bytes(16, 8192) > 0        # the rows do not fit into a workgroup's LDS


def test_where_the_one_launch_form_ends(lib):
    """Up to 16 tokens whose quantised rows (K rounded up to 64, and 16 bytes) fit 64 KB; beyond, a workspace is asked for."""
    need = lib.stof_linear_i8_workspace_bytes
    for M, last in ((1, 65472), (2, 32704), (15, 4352), (16, 4032)):
        assert M * (last + 16) <= 65536 < M * (last + 64 + 16)
        assert need(M, last) == 0 and need(M, last + 16) == M * (last + 16) + (4 * M + 15) // 16 * 16
    assert need(17, 16) == 17 * 16 + 80
    assert lib.stof_linear_i8(P, P, P, None, P, 16, 16, 4096, 4096, 4096, 16, 0, 0, None, 0, None) == -1
