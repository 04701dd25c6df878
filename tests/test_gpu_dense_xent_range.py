"""Softmax cross entropy of a Dense head without its logits, at the ends of its range, against the definition in float64 on
the CPU."""
import pytest
import torch

from test_gpu_dense_xent import case, check, reference, run

gpu = pytest.mark.gpu
LOWEST = -3.4028234663852886e38

# one size of every form: few rows, blocks of rows (two kernels), streamed with 64 and 128 features, split streams, wide
FORMS = [(3, 40, 300), (60, 70, 500), (40, 30, 33000), (100, 40, 777), (200, 128, 900), (2000, 100, 9000), (150, 300, 1000)]


def row_bounds(x, w, b, labels, dloss, dtype):
    """Per row: how far a loss or lse (beside 2^-23 of its own size) and the 2-norm of a dx may be off.  Logits are
    sums of float32 quality: 22 bits of each operand and one dropped product, 3 2^-22 of a term |x_k w_kj| at most, and 3 e / 16
    additions, half a unit of the sum so far each.  Both are of either sign, so that over the e terms of a logit they stay
    below 2^-22 of sum_k |x_k w_kj| (0.8 of it in emulation with up to 300 terms and 18 million logits; one float32 sum in the
    order of k comes to 1.5).  lse adds its own to the label's: `unit` is twice that of the row's largest sum, beside a few
    2^-23 for bias, exponential and logarithm.  A probability is off by unit relative to itself, and the label's p - 1 by
    unit however small it is.  A bf16 dx is rounded once (2^-8 of it at most), and its second product takes both
    operands to 11 bits: 2^-11 of a term each, terms |dz_ij| |w_kj|."""
    x64, w64 = x.double(), w.double()
    z = x64 @ w64
    unit = 2.0 ** -23 * 8 + 2.0 ** -21 * (x64.abs() @ w64.abs()).amax(dim=1)
    z = z + (b.double() if b is not None else 0.0)
    d = torch.softmax(z, dim=1)
    at = torch.arange(len(labels)), labels.long()
    d[at] -= 1.0
    d *= dloss.double()[:, None]
    dx = d @ w64.t()
    size = d.abs() @ w64.abs().t()
    off = 4 * unit * size.norm(dim=1) + unit * dloss.double().abs() * w64.norm(dim=0)[labels.long()]
    if dtype == torch.bfloat16:
        off = off + 2.0 ** -8 * dx.norm(dim=1) + 2.0 ** -10 * size.norm(dim=1)
    return unit, off


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


def gradients_close(got, want, unit, dtype):
    """dw, db and dx in the 2-norm as in check(), with nothing absolute: the operands may be of any size."""
    for k in ("dw", "db", "dx"):
        norm = float(want[k].norm())
        tol = 4 * unit + (2.0 ** -8 + 2.0 ** -10 if k == "dx" and dtype == torch.bfloat16 else 0.0)
        off = float((got[k].double() - want[k]).norm())
        assert off <= tol * norm + unit * want["slack"][k], (k, off / max(norm, 1e-300), tol)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,e,v", FORMS)
@pytest.mark.parametrize("scale_x,scale_w", [(1e-16, 1e-15), (1e-30, 1e-2), (1e-2, 1e-30), (1e-25, 1e3), (1e-32, 1e-32)])
def test_small_operands_beside_a_bias(scale_x, scale_w, n, e, v, dtype):
    """max |x| max |W| far below the bias: the logits are the biases, the gradients as exact as at any other size."""
    x, w, b, labels, dloss = case(n, e, v, torch.float32, seed=110 + e)
    args = ((x * scale_x).to(dtype), w * scale_w, b, labels, dloss * n)
    want, got = reference(*args), run(*args)
    unit = 2.0 ** -23 * (8 + 2 * 2.0)          # logits: the biases, up to 1.5
    for k in ("loss", "lse"):
        assert float((got[k].double() - want[k]).abs().max()) <= unit + 2.0 ** -23 * float(want[k].abs().max())
    gradients_close(got, want, unit, dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,e,v", FORMS)
@pytest.mark.parametrize("mask", [-1e25, -1e32, -3e38, LOWEST, float("-inf")])
def test_masked_labels(mask, n, e, v, dtype):
    """A row whose label is masked has the loss of that bias, and p - 1 = -1 at it; a mask of the lowest float or -inf leaves
    the class's column of W out of dx."""
    x, w, b, labels, dloss = case(n, e, v, dtype, seed=120 + e, unlabelled=0)
    b[7] = mask
    labels[labels == 7] = 8
    hidden = torch.arange(n) % 3 == 1
    labels[hidden] = 7
    w_used = w.clone()
    if mask <= LOWEST:
        w_used[:, 7] = 0.0
    want, got = reference(x, w_used, b, labels, dloss), run(x, w, b, labels, dloss)
    if mask == float("-inf"):
        assert bool(torch.isposinf(got["loss"][hidden]).all())
    else:
        # the bias into units of log 2 and back, the difference from lse: four roundings at most
        assert bool(((got["loss"].double() - want["loss"]).abs()[hidden] <= 2.0 ** -22 * want["loss"][hidden]).all()), float(got["loss"][1])
    unit = 2.0 ** -23 * (8 + 2 * float((x.double() @ w.double()).abs().max()))
    assert float((got["loss"].double() - want["loss"])[~hidden].abs().max()) <= unit + 2.0 ** -23 * float(want["loss"][~hidden].max())
    assert float((got["lse"].double() - want["lse"]).abs().max()) <= unit + 2.0 ** -23 * float(want["lse"].abs().max())
    gradients_close(got, want, unit, dtype)
    assert bool((got["hits"][hidden] == 0).all())


@gpu
@pytest.mark.parametrize("spread", [2.0, 8.0, 16.0, 32.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,e,v", FORMS)
def test_sharp_logits(n, e, v, dtype, spread):
    """Logits of standard deviation up to 32: each row's dx within its own bound."""
    x, w, b, labels, dloss = case(n, e, v, dtype, seed=130 + e, unlabelled=0, spread=spread)
    want, got = reference(x, w, b, labels, dloss), run(x, w, b, labels, dloss)
    unit, off = row_bounds(x, w, b, labels, dloss, dtype)
    for k in ("loss", "lse"):
        assert bool(((got[k].double() - want[k]).abs() <= unit + 2.0 ** -23 * want[k].abs()).all()), k
    short = (got["dx"].double() - want["dx"]).norm(dim=1) / off
    assert float(short.max()) <= 1.0, float(short.max())
    gradients_close({**got, "dx": want["dx"]}, want, float(unit.max()), dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,e,v", FORMS)
@pytest.mark.parametrize("size", [1e-33, 1e30])
def test_weights_of_any_size(size, n, e, v, dtype):
    x, w, b, labels, dloss = case(n, e, v, dtype, seed=140 + e)
    args = (x, w, b, labels, dloss * n * size)
    gradients_close(run(*args), reference(*args), 2.0 ** -23 * (8 + 2 * float((x.double() @ w.double()).abs().max())), dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,e,v", [f for f in FORMS if f[0] > 16])
@pytest.mark.parametrize("large", [1e6, 1e8])
def test_rows_of_very_different_size(large, n, e, v, dtype):
    """One labelled row has features `large` times the others', one as much smaller ones: no other row's loss or dx loses digits.
    With a weight of zero at the large row, neither do dw and db."""
    x, w, b, labels, dloss = case(n, e, v, dtype, seed=150 + e, unlabelled=0)
    k = n // 2
    x[k] *= large
    x[3] /= large
    rest = torch.arange(n) != k
    unit, off = row_bounds(x, w, b, labels, dloss, dtype)
    want, got = reference(x, w, b, labels, dloss), run(x, w, b, labels, dloss)
    for name in ("loss", "lse"):
        short = (got[name].double() - want[name]).abs() / (unit + 2.0 ** -23 * want[name].abs())
        assert float(short.max()) <= 1.0, (name, float(short.max()))
    short = ((got["dx"].double() - want["dx"]).norm(dim=1) / off)[rest]
    assert float(short.max()) <= 1.0, float(short.max())
    assert all(bool(got[name].isfinite().all()) for name in ("dx", "dw", "db"))
    dloss[k] = 0.0
    want, got = reference(x, w, b, labels, dloss), run(x, w, b, labels, dloss)
    gradients_close(got, want, float(unit[rest].max()), dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,e,v", FORMS)
def test_logits_beyond_the_digits_of_lse(n, e, v, dtype):
    """Logits around 1e8, where lse, a float32, is known to a few units only: no probability comes out above 1, and
    gradients stay finite."""
    x, w, b, labels, dloss = case(n, e, v, dtype, seed=160 + e, unlabelled=0)
    large = torch.arange(n) % 3 == 2
    x[large] *= 1e8
    got = run(x, w, b, labels, dloss)
    assert all(bool(got[name].isfinite().all()) for name in ("loss", "lse", "dx", "dw", "db"))
    # |dz| of a row sums to 2 at most
    assert float(got["db"].abs().sum()) <= 2.001 * float(dloss.sum())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,e,v", FORMS)
def test_logits_that_are_all_cancellation(n, e, v, dtype):
    """Features of 1e9 against columns of W whose halves cancel to the last digits: what is left of the logits are the roundings
    of terms a billion times larger.  The backward meets the forward's logits again: its probabilities sum to 1 and stay finite."""
    x, w, b, labels, dloss = case(n, e, v, dtype, seed=170 + e, unlabelled=0)
    half = e // 2
    x[:, :half] = (x[:, :half].float() * 1e9).to(dtype)
    x[:, half:] = -x[:, :half]
    w[half:] = w[:half] * (1.0 + 2.0 ** -22 * torch.randint(-1, 2, w[:half].shape, generator=torch.Generator().manual_seed(2)))
    got = run(x, w, b, labels, dloss)
    assert all(bool(got[name].isfinite().all()) for name in ("loss", "lse", "dx", "dw", "db"))
    # a row's dz sums to 0 but for the rounding of lse, 2^-22 of it, and the 11 and 22 bits of the planes in front of a float32 sum
    assert abs(float(got["db"].double().sum())) <= (2.0 ** -20 * float(got["lse"].abs().max()) + 2.0 ** -18) * float(dloss.sum())
    assert float(got["db"].abs().sum()) <= 2.001 * float(dloss.sum())
