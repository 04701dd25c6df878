"""The 8-bit activation tape: gradients through saturated units, kernels that are not exact in bf16, workspaces aligned as
floats are."""
import ctypes

import pytest
import torch

from music_generator_amd import _cabi, backend, ops
from test_gpu_tape8 import ALPHA, conv_case, conv_reference, derivative

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("n,h,w,cin,k", [(1, 8, 64, 32, 3), (3, 13, 131, 32, 2), (2, 5, 37, 128, 3)])
def test_workspace_aligned_as_floats(n, h, w, cin, k):
    """The same bits from a workspace at any multiple of 4 bytes, in the bf16 and the 8-bit form."""
    d, x, g, wt = conv_case(n, h, w, cin, k, seed=3)
    t = ops.tape8_pack(x.cuda())
    kept, g, wt = ops.tape8_unpack(t, torch.bfloat16), g.cuda(), wt.cuda()
    lib = _cabi.load()
    size = lib.mgx_conv_bwd_bf16_workspace(ctypes.byref(d))
    ws = torch.empty((size + 16,), dtype=torch.uint8, device="cuda")
    outs = []
    for shift in (0, 4, 8, 12):
        for tape in (False, True):
            dw, db, dx = torch.zeros_like(wt), torch.zeros((32,), device="cuda"), torch.empty_like(kept)
            rest = (g.data_ptr(), wt.data_ptr(), dw.data_ptr(), db.data_ptr(), dx.data_ptr(), ALPHA, ws.data_ptr() + shift, size,
                    backend.stream_ptr())
            if tape:
                code = lib.mgx_conv_bwd_tape8(ctypes.byref(d), t.codes.data_ptr(), t.exps.data_ptr(), *rest)
            else:
                code = lib.mgx_conv_bwd_bf16(ctypes.byref(d), kept.data_ptr(), *rest)
            assert code == _cabi.MGX_OK
            outs.append((dw, db, dx))
    for out in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out, outs[0]))
