"""Refusals of the 8-bit tape and of the cross entropy without logits at the C entries.  Every call is turned down from its
arguments, so no device is needed and no pointer is read."""
import ctypes
import itertools

import pytest

from music_generator_amd import _cabi, ops

P = 1 << 20             # an aligned address that nothing reads


def refuse(fn, good, bad, want):
    """`good` with each of `bad`'s changes in turn gives `want`."""
    for change in bad:
        args = dict(good, **change)
        assert fn(*args.values()) == want, change


@pytest.fixture
def lib():
    return _cabi.load()


def test_tape8_blocks(lib):
    assert [lib.mgx_tape8_blocks(n) for n in (-1, 0, 1, 32, 33, 2 ** 40)] == [0, 0, 1, 1, 2, 2 ** 35]


def test_tape8_pack_and_unpack(lib):
    for f in (0, 1):
        pack = dict(x=P, f32=f, codes=P, exps=P, n=100, stream=None)
        refuse(lib.mgx_tape8_pack, pack, [dict(x=None), dict(codes=None), dict(exps=None), dict(x=P + 2), dict(codes=P + 8), dict(n=-1)],
               _cabi.MGX_ERR_ARG)
        unpack = dict(codes=P, exps=P, y=P, f32=f, n=100, stream=None)
        refuse(lib.mgx_tape8_unpack, unpack, [dict(codes=None), dict(exps=None), dict(y=None), dict(y=P + 4), dict(codes=P + 1), dict(n=-5)],
               _cabi.MGX_ERR_ARG)
        product = dict(a=P, f32=f, codes=P, exps=P, alpha=2.0, out=P, n=100, stream=None)
        refuse(lib.mgx_mul_dact_tape8, product, [dict(a=None), dict(codes=None), dict(exps=None), dict(out=None), dict(a=P + 2), dict(out=P + 2),
                                                 dict(codes=P + 4), dict(alpha=0.0), dict(alpha=-1.0), dict(alpha=float("nan")), dict(n=-1)],
               _cabi.MGX_ERR_ARG)
    assert lib.mgx_tape8_pack(None, 0, None, None, 0, None) == _cabi.MGX_OK
    assert lib.mgx_tape8_unpack(None, None, None, 0, 0, None) == _cabi.MGX_OK


def test_conv_bwd_tape8(lib):
    def desc(**change):
        k = change.pop("k", 3)
        return ops.make_conv_desc(**{**dict(nimg=2, hin=9, win=40, cin=32, hout=9, wout=40, kh=k, kw=k, pt=(k - 1) // 2, pl=(k - 1) // 2, ngemm=32,
                                            cout=32, wtap=32 * 32, wsk=32, wsn=1, nbias=32), **change})

    d = desc()
    need = lib.mgx_conv_bwd_bf16_workspace(ctypes.byref(d))
    good = dict(d=ctypes.byref(d), codes=P, exps=P, g=P, w=P, dw=P, db=P, dx=P, alpha=0.0, ws=P, bytes=need, stream=None)
    refuse(lib.mgx_conv_bwd_tape8, good, [dict(d=None)] + [{k: None} for k in ("codes", "exps", "g", "w", "dw", "dx", "ws")]
           + [dict(codes=P + 8), dict(g=P + 2), dict(dx=P + 2), dict(w=P + 4), dict(alpha=-1.0), dict(alpha=float("nan"))]
           + [dict(d=ctypes.byref(x)) for x in (desc(cin=31), desc(cin=64), desc(k=5), desc(sh=2), desc(nimg=0), desc(nbias=16))], _cabi.MGX_ERR_ARG)
    refuse(lib.mgx_conv_bwd_tape8, good, [dict(bytes=need - 1), dict(bytes=0)], _cabi.MGX_ERR_WORKSPACE)


def test_dense_xent_sizes(lib):
    for bad in ((-1, 4, 4), (4, 0, 4), (4, 4, 0), (8000001, 4, 4), (4, 65001, 4), (4, 4, 8000001)):
        assert all(lib.mgx_dense_xent_workspace(*bad, f, d) == -1 for f, d in itertools.product((0, 1), (0, 1))), bad
        n, e, v = bad
        assert lib.mgx_dense_xent_fwd(P, 1, P, P, P, P, P, None, n, e, v, P, 1 << 40, None) == _cabi.MGX_ERR_ARG
        assert lib.mgx_dense_xent_bwd(P, 1, P, P, P, P, P, P, P, P, 0, n, e, v, P, 1 << 40, None) == _cabi.MGX_ERR_ARG
    for f, d in itertools.product((0, 1), (0, 1)):
        assert lib.mgx_dense_xent_workspace(0, 4, 4, f, d) == 0
        # the whole allowed range has a size, and more rows, features or classes never need less than a few
        sizes = [lib.mgx_dense_xent_workspace(*s, f, d) for s in ((1, 1, 1), (16, 65000, 8000000), (17, 65000, 8000000), (8000000, 1, 8000000),
                                                                  (8000000, 65000, 1), (8000000, 65000, 8000000))]
        assert all(s > 0 for s in sizes) and sizes[5] == max(sizes)


@pytest.mark.parametrize("n,e,v", [(1, 128, 4097), (16, 300, 1000), (17, 40, 300), (500, 128, 5000), (300, 301, 5001), (4000, 130, 12000)])
def test_dense_xent(lib, n, e, v):
    for f in (0, 1):
        fwd = dict(x=P, f32=f, w=P, b=P, labels=P, loss=P, lse=P, hits=None, n=n, e=e, v=v, ws=P, bytes=lib.mgx_dense_xent_workspace(n, e, v, f, 0),
                   stream=None)
        refuse(lib.mgx_dense_xent_fwd, fwd, [{k: None} for k in ("x", "w", "labels", "loss", "lse", "ws")]
               + [dict(x=P + 8), dict(w=P + 4), dict(ws=P + 4)], _cabi.MGX_ERR_ARG)
        refuse(lib.mgx_dense_xent_fwd, fwd, [dict(bytes=fwd["bytes"] - 1), dict(bytes=0)], _cabi.MGX_ERR_WORKSPACE)
        bwd = dict(x=P, f32=f, w=P, b=P, labels=P, lse=P, dloss=P, dx=P, dw=P, db=P, acc=0, n=n, e=e, v=v, ws=P,
                   bytes=lib.mgx_dense_xent_workspace(n, e, v, f, 1), stream=None)
        refuse(lib.mgx_dense_xent_bwd, bwd, [{k: None} for k in ("x", "w", "labels", "lse", "dloss", "ws")]
               + [dict(x=P + 8), dict(w=P + 4), dict(ws=P + 4)], _cabi.MGX_ERR_ARG)
        refuse(lib.mgx_dense_xent_bwd, bwd, [dict(bytes=bwd["bytes"] - 1), dict(bytes=0)], _cabi.MGX_ERR_WORKSPACE)


@pytest.mark.parametrize("rows,numbers", [(1, 10), (1, 0), (4, 1), (4, 40), (4, 5)])
@pytest.mark.parametrize("units,cin", [(9, 64), (80, 64)])
def test_class_numbers_of_another_count(rows, numbers, units, cin):
    """One class number for each row of features, for heads that store their logits and heads that do not: integer rows that are
    no one-hot rows of the model's classes must not be read as class numbers of other rows."""
    import torch

    from music_generator_amd.evaluacion import SoftmaxDense
    head = SoftmaxDense(units)
    head.cin = cin
    for features in (torch.zeros((rows, cin)), torch.zeros((rows, 1, 1, cin))):
        for backward in (False, True):
            with pytest.raises(_cabi.MgxError, match="class numbers"):
                head.loss(features, torch.zeros((numbers,), dtype=torch.int32), backward)


@pytest.mark.parametrize("precision", ["float32", "bfloat16"])
def test_tape_estimate_of_saved_derivatives(precision):
    """The 8-bit tape leaves saved bf16 derivatives in bf16: they cost the same with it and without."""
    import music_generator_amd as M
    model = M.define_discriminator(3)[2][0]
    M.backend.set_precision(precision)
    try:
        cost = []
        for tape8 in (False, True):
            M.backend.TAPE8 = tape8
            each = []
            for derivative in (False, True):
                M.backend.BF16_SAVE_DERIVATIVE = derivative
                each.append(model.tape_bytes_estimate(2))
            cost.append(each[1] - each[0])
        assert cost[0] == cost[1] and (cost[0] > 0) == (precision == "bfloat16")
    finally:
        M.backend.TAPE8 = M.backend.BF16_SAVE_DERIVATIVE = False
        M.backend.set_precision("float32")
