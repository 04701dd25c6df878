"""Softmax cross entropy of a Dense head without its logits, at the ends of its range, against the definition in float64 on
the CPU."""
import pytest
import torch

from test_gpu_dense_xent import case, check, reference, run

gpu = pytest.mark.gpu
LOWEST = -3.4028234663852886e38

# one size of every form: few rows, blocks of rows (two kernels), streamed with 64 and 128 features, split streams, wide
FORMS = [(3, 40, 300), (60, 70, 500), (40, 30, 33000), (100, 40, 777), (200, 128, 900), (2000, 100, 9000), (150, 300, 1000)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,e,v", FORMS)
@pytest.mark.parametrize("mask", [-1e5, -1e10, -5e9, -1e18, -1e20, -1e30])
def test_finite_masks(mask, n, e, v, dtype):
    """Classes masked with a finite bias, among them whole tiles and the whole first parts of a split stream."""
    x, w, b, labels, dloss = case(n, e, v, dtype, seed=100 + e, unlabelled=0)
    b[torch.rand((v,), generator=torch.Generator().manual_seed(1)) < 0.3] = mask
    b[:v // 3] = mask
    b[v - v // 5:] = mask
    open_ = (b != mask).nonzero()[:, 0]
    labels = open_[labels.long() % len(open_)].int()
    want = reference(x, w, b, labels, dloss)
    got = run(x, w, b, labels, dloss)
    check(got, want, dtype, float((x.double() @ w.double()).abs().max()))
    assert bool((got["dw"][:, b == mask] == 0).all()) and bool((got["db"][b == mask] == 0).all())
