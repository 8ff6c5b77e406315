"""Calls of the score attention's C ABI that its Python wrapper does not make."""
import math

import pytest
import torch

from stof import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", [-1, 0, 1, 2])
@pytest.mark.parametrize("D,Sq,docs", [(64, 1, False), (64, 200, True), (128, 40, False)])
def test_no_keys_through_the_c_abi(form, D, Sq, docs):
    """Sk = 0: zeros and lse = -inf from every launch form."""
    B, H = 2, 4
    lib = _lib.lib()
    buf = torch.full((B, H, Sq + 2, D), 7.0, dtype=torch.float16, device="cuda")
    q = torch.ones(B, H, Sq, D, dtype=torch.float16, device="cuda")
    lse = torch.zeros(B, H, Sq, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    ids = torch.zeros(B, Sq, dtype=torch.int32, device="cuda")
    out = buf[:, :, 1:-1]
    n = lib.stof_score_attn_workspace_bytes(B, H, 2, Sq, 0, D, 1 if docs else 0, form)
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    st = _lib.strides3(q)
    rc = lib.stof_score_attn_fwd(q.data_ptr(), q.data_ptr(), q.data_ptr(), out.data_ptr(), lse.data_ptr(), None, None, None, lens.data_ptr(),
                                 ids.data_ptr() if docs else None, ids.data_ptr() if docs else None, 0.125, 0.0, -1, 1, 0, 0,
                                 st, st, st, _lib.strides3(out), B, H, 2, Sq, 0, D, 0, form, ws.data_ptr(), n,
                                 torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == 0
    assert not bool(out.any()) and bool((lse == -math.inf).all())
    assert bool((buf[:, :, 0] == 7).all()) and bool((buf[:, :, -1] == 7).all())
