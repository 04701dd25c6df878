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


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_derivative_of_saturated_units(dtype):
    """Pre-activations up to 30, most of them saturated.  In a block that reaches 1, y comes back as y' with |y - y'| <= 2^-8 and
    |y|, |y'| <= 1 (or y above 1, where f' = 1 / alpha, and y' = +-255/256): the derivative 1 + 1/alpha - y'^2 is off by
    |y - y'| |y + y'| <= 2^-7 at most, and by nearly that where y is +-1.  The product with 1, up to f' + 2^-7, is rounded to bf16
    once: 2^-8 of that."""
    pre = torch.randn((64, 500, 32), generator=torch.Generator().manual_seed(8)) * 10
    pre[..., 0] = 30.0                                 # H = 1 in every block
    y = (torch.tanh(pre) + pre / ALPHA).to(dtype)
    got = ops.mul_dact_tape8(torch.ones(y.shape, device="cuda"), ops.tape8_pack(y.cuda()), ALPHA).cpu().double()
    want = derivative(y.double())
    assert bool(((got - want).abs() <= 2.0 ** -7 + 2.0 ** -8 * (want + 2.0 ** -7)).all())
    at_one = 1.0 + 1.0 / ALPHA - (255.0 / 256.0) ** 2
    assert bool(((got[y.abs() >= 1].double() - at_one).abs() <= 2.0 ** -8 * at_one).all()) and int((y.abs() >= 1).sum()) > 1000


@gpu
@pytest.mark.parametrize("act", [True, False])
@pytest.mark.parametrize("n,h,w,cin,k", [(2, 9, 65, 32, 3), (3, 13, 131, 32, 2), (2, 5, 37, 128, 3)])
def test_kernels_that_are_not_exact_in_bf16(n, h, w, cin, k, act):
    """The data gradient takes the kernel rounded to bf16, 2^-8 of a weight at most, as mgx_conv_bwd_bf16 does; dw and db do not
    depend on it."""
    d, x, g, wt = conv_case(n, h, w, cin, k, seed=9)
    wt = wt * (1.0 + 2.0 ** -9 * torch.rand(wt.shape, generator=torch.Generator().manual_seed(10)))
    t = ops.tape8_pack(x.cuda())
    dw, db, dx = torch.zeros_like(wt).cuda(), torch.zeros((32,), device="cuda"), torch.empty(x.shape, dtype=torch.bfloat16, device="cuda")
    ops.conv_bwd_tape8(d, t, g.cuda(), wt.cuda(), dw, db, dx, ALPHA if act else 0.0)
    rx, rw, rb = conv_reference(x, g, wt, act)
    size = conv_reference(x, g.abs(), wt.abs(), act)[0]          # sum of |g w|, times f'
    # the weights, one rounding of dx, float32 sums of k k 32 terms
    assert bool(((dx.cpu().double() - rx).abs() <= (2.0 ** -8 + 288 * 2.0 ** -24) * size + 2.0 ** -8 * rx.abs()).all())
    lim = n * h * w * 2.0 ** -24 * 4 + 2.0 ** -22               # as with exact kernels
    assert float((dw.cpu().double() - rw).abs().max()) <= lim and float((db.cpu().double() - rb).abs().max()) <= lim
