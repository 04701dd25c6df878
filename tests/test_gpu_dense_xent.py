"""Softmax cross entropy of a Dense head without its logits: loss, gradients, masks, refusals, against the definition in
float64 on the CPU."""
import math

import numpy as np
import pytest
import torch

import music_generator_amd as M
from music_generator_amd import ops
from music_generator_amd._cabi import MgxError

gpu = pytest.mark.gpu


def case(n, e, v, dtype, seed=0, bias=True, unlabelled=0.1, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((n, e), generator=gen).to(dtype)
    w = torch.randn((e, v), generator=gen) * (spread / math.sqrt(e))
    b = torch.randn((v,), generator=gen) * 0.3 if bias else None
    labels = torch.randint(0, v, (n,), generator=gen, dtype=torch.int32)
    if unlabelled:
        labels[torch.rand((n,), generator=gen) < unlabelled] = -1
    dloss = (0.5 + torch.rand((n,), generator=gen)) / max(n, 1)
    return x, w, b, labels, dloss


def reference(x, w, b, labels, dloss):
    x64, w64 = x.double(), w.double()
    z = x64 @ w64 + (b.double() if b is not None else 0.0)
    lse = torch.logsumexp(z, dim=1)
    ok = (labels >= 0) & (labels < w.shape[1])
    at = labels.clamp(0, w.shape[1] - 1).long()
    picked = z.gather(1, at[:, None])[:, 0]
    loss = torch.where(ok, lse - picked, torch.zeros_like(lse))
    d = torch.exp(z - lse[:, None])
    at_label = torch.zeros_like(d)
    at_label[torch.arange(len(at)), at] = torch.where(ok, d[torch.arange(len(at)), at] * dloss.double().abs(), torch.zeros_like(lse))
    d[torch.arange(len(at)), at] -= 1.0
    d = torch.where(ok[:, None], d * dloss.double()[:, None], torch.zeros_like(d))
    x64 = torch.where(ok[:, None], x64, torch.zeros_like(x64))
    hits = (ok & (picked >= z.amax(dim=1))).int()
    slack = {"dx": at_label @ w64.abs().t(), "dw": x64.abs().t() @ at_label, "db": at_label.sum(dim=0)}
    return {"slack": {k: float(s.norm()) for k, s in slack.items()}, "loss": loss, "lse": torch.where(ok, lse, torch.zeros_like(lse)), "dx": d @ w64.t(), "dw": x64.t() @ d,
            "db": d.sum(dim=0), "hits": hits}


def run(x, w, b, labels, dloss, accumulate=False, dw=None, db=None):
    dev = [t.cuda() if t is not None else None for t in (x, w, b, labels, dloss)]
    x, w, b, labels, dloss = dev
    n, v = x.shape[0], w.shape[1]
    loss, lse, hits = torch.empty((n,)).cuda(), torch.empty((n,)).cuda(), torch.empty((n,), dtype=torch.int32).cuda()
    ops.dense_xent_fwd(x, w, b, labels, loss, lse, hits)
    dx = torch.full_like(x, float("nan"))
    dw = torch.full_like(w, float("nan")) if dw is None else dw.cuda()
    db = torch.full((v,), float("nan")).cuda() if db is None else db.cuda()
    ops.dense_xent_bwd(x, w, b, labels, lse, dloss, dx, dw, db, accumulate=accumulate)
    return {k: t.cpu() for k, t in (("loss", loss), ("lse", lse), ("dx", dx), ("dw", dw), ("db", db), ("hits", hits))}


def check(got, want, dtype, largest_logit):
    """Logits: operands of 22 bits and float32 sums, so a logit is off by a few 2^-23 of the largest one, and lse, a float32,
    by its rounding: `unit`.  A loss is off by that and one rounding, a probability by unit relative to itself, and so are
    the gradients (sums of terms of both signs: compared in the 2-norm) but for the label's term p - 1, which is off by
    unit p however small it is itself: `slack` is the gradient with p dloss at the labels, the size of that part.  A bf16 dx has one rounding, eps / 2 = 2^-8 of a value at most and so 2^-8 of the 2-norm, and its
    second product may take both operands to 11 bits (2^-11 of a term each, terms of both signs)."""
    unit = 2.0 ** -23 * (8 + 2 * largest_logit)
    assert float((got["loss"].double() - want["loss"]).abs().max()) <= unit + 2.0 ** -23 * float(want["loss"].abs().max())
    assert float((got["lse"].double() - want["lse"]).abs().max()) <= unit + 2.0 ** -23 * float(want["lse"].abs().max())
    for k in ("dw", "db", "dx"):
        norm = float(want[k].norm())
        off = float((got[k].double() - want[k]).norm())
        tol = 4 * unit + (2.0 ** -8 + 2.0 ** -10 if k == "dx" and dtype == torch.bfloat16 else 0.0)
        assert off <= tol * norm + unit * want["slack"][k] + 1e-30, (k, off / max(norm, 1e-300), tol)


SIZES = [(1, 1, 1), (1, 128, 4097), (2, 16, 2), (5, 33, 130), (64, 128, 256), (127, 64, 129), (129, 130, 1000), (300, 256, 511),
         (257, 500, 2049), (1000, 128, 3001), (17, 1000, 10001), (4, 1, 70000), (640, 32, 128)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,e,v", SIZES)
def test_loss_and_gradients(n, e, v, dtype):
    args = case(n, e, v, dtype, seed=n + e + v, bias=(n % 2 == 1))
    want = reference(*args)
    check(run(*args), want, dtype, float((args[0].double() @ args[1].double()).abs().max()))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_hits(dtype):
    x, w, b, labels, dloss = case(200, 64, 40, dtype, seed=3)
    z = x.double() @ w.double() + b.double()
    top = z.topk(2, dim=1)
    clear = top.values[:, 0] - top.values[:, 1] > 1e-3          # no tie within the logits' accuracy
    labels[::2] = top.indices[::2, 0].int()
    got, want = run(x, w, b, labels, dloss)["hits"], reference(x, w, b, labels, dloss)["hits"]
    assert torch.equal(got[clear], want[clear]) and int(want.sum()) >= 90


@gpu
@pytest.mark.parametrize("scale_x,scale_w", [(1e-6, 1e-3), (1e4, 1e-6), (3e-3, 2e3), (1e-20, 1e18)])
def test_magnitudes(scale_x, scale_w):
    """The planes follow the operands' magnitudes: the result is as exact for small and large ones."""
    x, w, b, labels, dloss = case(150, 96, 700, torch.float32, seed=8)
    args = (x * scale_x, w * scale_w, b, labels, dloss * 1e-5)
    z = args[0].double() @ args[1].double()
    check(run(*args), reference(*args), torch.float32, float(z.abs().max()) + 1)


@gpu
def test_confident_rows():
    """Rows whose label has nearly all the probability: dz = p - 1 is small and taken before any rounding to fewer bits, and a
    small loss keeps its digits (lse - z would lose those below 2^-24 lse)."""
    x, w, b, labels, dloss = case(128, 64, 300, torch.float32, seed=5, unlabelled=0, spread=1.0)
    w = w * 0.05
    for i in range(128):                           # the label's class points along the row
        labels[i] = i
        w[:, i] += x[i] * (14.0 / float(x[i].square().sum()))
    want = reference(x, w, b, labels, dloss)
    assert float(want["loss"].median()) < 1e-2
    got = run(x, w, b, labels, dloss)
    check(got, want, torch.float32, 20.0)
    # log of 1 + small exponentials: those are off by a few 2^-23 of a logit's 20, and the sum by half a unit, 2^-24, for
    # each addition behind the 1: at most 32 in a lane's part of the classes, and one for each of the parts joined to it
    # (300 classes: under 32)
    assert bool(((got["loss"].double() - want["loss"]).abs() <= 2.0 ** -23 * (1 + 32 + 48 * want["loss"])).all())


@gpu
@pytest.mark.parametrize("mask", [float("-inf"), -3.4028234663852886e38])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_classes(mask, dtype):
    x, w, b, labels, dloss = case(100, 40, 777, dtype, seed=6)
    b[torch.rand((777,), generator=torch.Generator().manual_seed(1)) < 0.5] = mask
    b[256:512] = mask                              # whole tiles
    b[640:] = mask
    labels = torch.where(b[labels.clamp(min=0).long()] == mask, torch.full_like(labels, -1), labels)
    assert int((labels >= 0).sum()) > 5
    want = reference(x, w, b, labels, dloss)
    got = run(x, w, b, labels, dloss)
    check(got, want, dtype, 6.0)
    assert bool((got["dw"][:, b == mask] == 0).all()) and bool((got["db"][b == mask] == 0).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_without_a_label_may_hold_anything(dtype):
    x, w, b, labels, dloss = case(90, 48, 200, dtype, seed=7, unlabelled=0.3)
    labels[3], labels[4], labels[5], labels[6] = 200, 2 ** 31 - 1, -2 ** 31, -1       # outside [0, v)
    want = reference(x, w, b, labels, dloss)
    bad = (labels < 0) | (labels >= 200)
    x[bad] = float("nan")
    x[4] = float("inf")
    dloss[5] = float("nan")
    got = run(x, w, b, labels, dloss)
    check(got, want, dtype, 6.0)
    assert bool((got["loss"][bad] == 0).all()) and bool((got["dx"][bad] == 0).all())


@gpu
def test_no_row_has_a_label():
    x, w, b, labels, dloss = case(70, 20, 150, torch.float32, seed=9)
    got = run(x, w, b, torch.full_like(labels, -1), dloss)
    for k in ("loss", "lse", "dx", "dw", "db"):
        assert bool((got[k] == 0).all()), k


@gpu
def test_a_row_that_is_not_finite_stays_in_its_row():
    x, w, b, labels, dloss = case(130, 24, 90, torch.float32, seed=10, unlabelled=0)
    want = reference(x, w, b, labels, dloss)
    x[7, 3] = float("nan")
    got = run(x, w, b, labels, dloss)
    others = torch.arange(130) != 7
    assert bool(got["loss"][7].isnan())
    assert float((got["loss"][others].double() - want["loss"][others]).abs().max()) < 1e-5
    assert float((got["dx"][others].double() - want["dx"][others]).norm() / want["dx"][others].norm()) < 1e-5


@gpu
def test_accumulation_and_missing_outputs():
    x, w, b, labels, dloss = case(100, 130, 300, torch.float32, seed=11)
    want = reference(x, w, b, labels, dloss)
    dw0, db0 = torch.ones_like(w), torch.full_like(b, -2.0)
    got = run(x, w, b, labels, dloss, accumulate=True, dw=dw0, db=db0)
    # sums near 1 and 2: half a unit of 2^-23 and 2^-22 beside the gradient's own error
    assert float((got["dw"].double() - 1 - want["dw"]).abs().max()) < 2.0 ** -22
    assert float((got["db"].double() + 2 - want["db"]).abs().max()) < 2.0 ** -21
    dev = [t.cuda() for t in (x, w, b, labels)]
    loss, lse = torch.empty((100,)).cuda(), torch.empty((100,)).cuda()
    ops.dense_xent_fwd(*dev, loss, lse)
    whole = run(x, w, b, labels, dloss)
    for pick in ("dx", "dw", "db"):
        out = {"dx": None, "dw": None, "db": None}
        out[pick] = torch.full_like({"dx": dev[0], "dw": dev[1], "db": dev[2]}[pick], 7.0)
        ops.dense_xent_bwd(*dev, lse, dloss.cuda(), out["dx"], out["dw"], out["db"])
        assert torch.equal(out[pick].cpu(), whole[pick])


@gpu
def test_same_bits_every_time():
    args = case(500, 128, 5000, torch.bfloat16, seed=12)
    a, b = run(*args), run(*args)
    assert all(torch.equal(a[k], b[k]) for k in a)


@gpu
def test_no_rows():
    w, b = torch.randn((16, 40)).cuda(), torch.randn((40,)).cuda()
    x, labels = torch.empty((0, 16)).cuda(), torch.empty((0,), dtype=torch.int32).cuda()
    none = torch.empty((0,)).cuda()
    ops.dense_xent_fwd(x, w, b, labels, none, none)
    dw, db = torch.ones_like(w), torch.ones_like(b)
    ops.dense_xent_bwd(x, w, b, labels, none, none, torch.empty_like(x), dw, db, accumulate=True)
    assert bool((dw == 1).all()) and bool((db == 1).all())
    ops.dense_xent_bwd(x, w, b, labels, none, none, torch.empty_like(x), dw, db)
    assert bool((dw == 0).all()) and bool((db == 0).all())


@gpu
def test_gradient_against_differences():
    """Central differences of the float64 definition along a random direction of every operand."""
    x, w, b, labels, dloss = case(40, 20, 100, torch.float32, seed=13)
    got = run(x, w, b, labels, dloss)
    step = 1e-5
    for k, (name, t) in enumerate((("dx", x), ("dw", w), ("db", b))):
        direction = torch.randn(t.shape, generator=torch.Generator().manual_seed(k)).double()
        ends = []
        for s in (step, -step):
            moved = [x.double(), w.double(), b.double()]
            moved[k] = moved[k] + s * direction
            ends.append(float((reference(moved[0], moved[1], moved[2], labels, dloss)["loss"] * dloss.double()).sum()))
        quotient = (ends[0] - ends[1]) / (2 * step)
        slope = float((got[name].double() * direction).sum())
        # quotient: step^2 relative, and 2^-52 of the loss over the step; slope: float32 gradients
        assert abs(quotient - slope) <= 1e-5 * float(got[name].double().norm() * direction.norm()) + 1e-9


@gpu
def test_captured_forward_and_backward_replay():
    args = case(200, 128, 1000, torch.bfloat16, seed=14)
    x, w, b, labels, dloss = [t.cuda() for t in args]
    loss, lse = torch.empty((200,)).cuda(), torch.empty((200,)).cuda()
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)

    def step():
        ops.dense_xent_fwd(x, w, b, labels, loss, lse)
        ops.dense_xent_bwd(x, w, b, labels, lse, dloss, dx, dw, db)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(3):
        x.copy_(case(200, 128, 1000, torch.bfloat16, seed=20 + seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (loss, dx, dw, db)]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, (loss, dx, dw, db)))


@gpu
def test_two_streams_at_once():
    sets = [[t.cuda() for t in case(300, 128, 2000, torch.float32, seed=30 + k)] for k in range(2)]
    want = [run(*[t.cpu() for t in s]) for s in sets]
    outs, streams = [], [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(3):
        outs = []
        for (x, w, b, labels, dloss), st in zip(sets, streams):
            with torch.cuda.stream(st):
                loss, lse = torch.empty((300,), device="cuda"), torch.empty((300,), device="cuda")
                dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
                ops.dense_xent_fwd(x, w, b, labels, loss, lse)
                ops.dense_xent_bwd(x, w, b, labels, lse, dloss, dx, dw, db)
                outs.append((loss, dx, dw, db))
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert all(torch.equal(g.cpu(), ref[k]) for g, k in zip(got, ("loss", "dx", "dw", "db")))


@gpu
def test_refusals():
    x, w, b, labels, dloss = [t.cuda() for t in case(8, 16, 40, torch.float32)]
    row = torch.empty((8,), device="cuda")
    good = dict(x=x, w=w, b=b, labels=labels, loss=row, lse=row)
    for bad in (dict(x=x.double()), dict(x=x.half()), dict(x=x.t()), dict(x=x[:, :8]), dict(x=x.view(8, 4, 4)), dict(x=x.cpu()),
                dict(w=w.to(torch.bfloat16)), dict(w=w.t()), dict(w=w[:, :30]), dict(b=b[:39].contiguous()), dict(labels=labels.long()),
                dict(labels=labels[:7].contiguous()), dict(loss=row[:7].contiguous()), dict(lse=row.double()),
                dict(hits=row), dict(x=torch.cat([x.view(-1), x.view(-1)])[1:129].view(8, 16))):
        with pytest.raises(MgxError):
            ops.dense_xent_fwd(**{**good, **bad})
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    good = dict(x=x, w=w, b=b, labels=labels, lse=row, dloss=dloss, dx=dx, dw=dw, db=db)
    for bad in (dict(dx=dx.to(torch.bfloat16)), dict(dx=dx[:7].contiguous()), dict(dw=dw[:15].contiguous()), dict(db=db[:3].contiguous()),
                dict(dloss=dloss[:3].contiguous()), dict(dw=dw.double()), dict(lse=row[:5].contiguous())):
        with pytest.raises(MgxError):
            ops.dense_xent_bwd(**{**good, **bad})
    with pytest.raises(MgxError):                  # more features than the library serves
        ops.dense_xent_fwd(torch.empty((1, 70000), device="cuda"), torch.empty((70000, 1), device="cuda"), None,
                           labels[:1], row[:1], row[:1])


# ---- the evaluator's fit on class numbers, with and without the 8-bit tape ----
def position_classifier(classes, precision="float32"):
    """A small evaluator-like trunk with a classifier on every position (no Flatten)."""
    from music_generator_amd.evaluacion import SoftmaxDense
    from music_generator_amd.graph import Input, Model
    from music_generator_amd.layers import Conv2D
    M.backend.set_precision(precision)
    M.clear_session()
    M.layers.set_init_seed(5)
    image = Input(shape=(8, 40, 2))
    t = Conv2D(128, (1, 1), padding="same", kernel_initializer="he_normal")(image)
    t = Conv2D(32, (3, 3), padding="same", kernel_initializer="he_normal")(t)
    t = Conv2D(128, (1, 1), padding="same", kernel_initializer="he_normal")(t)
    return Model(image, SoftmaxDense(classes)(t))


@pytest.fixture
def restore():
    yield
    M.backend.TAPE8 = False
    M.backend.set_precision("float32")


@gpu
def test_fit_on_class_numbers_equals_one_hot_labels(restore):
    from music_generator_amd import evaluacion as E
    rng = np.random.default_rng(0)
    x = rng.standard_normal((12, 4, 750, 2)).astype(np.float32)
    numbers = rng.integers(0, 9, 12)
    weights, history = [], []
    for y in (np.eye(9, dtype=np.float32)[numbers], numbers):
        M.clear_session()
        M.layers.set_init_seed(3)
        model = E.define_evaluator(1)[0]
        history.append(E.fit_evaluator(model, x, y, 1, 4, validation_data=(x, y)))
        weights.append(model.get_weights_dict())
    # three batches; the first two losses come from weights that agree to the rounding of one update, which Adam's division by
    # the root of the squared gradient turns into 2 lr = 2e-3 for a weight whose gradient is all rounding: compared in the mean
    assert abs(history[0]["loss"][0] - history[1]["loss"][0]) < 1e-3 * abs(history[0]["loss"][0])
    for k in weights[0]:
        moved = np.abs(weights[0][k] - weights[1][k])
        assert moved.max() <= 6.1e-3 and moved.mean() < 3e-4, k


@gpu
@pytest.mark.parametrize("precision", ["float32", "bfloat16"])
@pytest.mark.parametrize("tape8", [False, True])
def test_positions_with_many_classes(restore, precision, tape8):
    """Loss and gradients of a classifier on every position against the float64 definition behind the same features, and the
    whole fit running from the 8-bit tape."""
    from music_generator_amd import evaluacion as E
    classes = 1500
    model = position_classifier(classes, precision)
    M.backend.TAPE8 = tape8
    gen = torch.Generator().manual_seed(1)
    x = torch.randn((3, 8, 40, 2), generator=gen)
    labels = torch.randint(-1, classes, (3, 8, 40), generator=gen)
    trunk, head = E._split_head(model)
    model.bind_grads(0).zero_()
    features, tape = trunk.forward(x.cuda(), save=True)
    assert features.dtype == (torch.bfloat16 if precision == "bfloat16" else torch.float32)
    if tape8:
        assert any(isinstance(v, ops.Tape8) for s in tape for v in (s if isinstance(s, tuple) else (getattr(s, "x", None),)))
    loss, hits, count, dx = head.loss(features, E.class_numbers_to_device(labels))
    flat = features.cpu().reshape(-1, 128)
    lab = labels.reshape(-1).int()
    dl = (lab >= 0).double() / int((lab >= 0).sum())
    want = reference(flat, torch.from_numpy(head.kernel.numpy()), torch.from_numpy(head.bias.numpy()), lab, dl)
    got = {"loss": want["loss"], "lse": want["lse"], "dx": dx.cpu().reshape(-1, 128), "dw": head.kernel.grad.cpu().view(128, classes),
           "db": head.bias.grad.cpu()}
    largest = float((flat.double() @ torch.from_numpy(head.kernel.numpy()).double()).abs().max())
    check(got, want, features.dtype, largest)
    assert int(count) == int((lab >= 0).sum())
    # a float32 sum of the losses: half a unit a step at most
    assert abs(float(loss) - float(want["loss"].sum())) <= 960 * 2.0 ** -24 * float(want["loss"].sum()) + 960 * 2.0 ** -20
    trunk.backward(tape, dx, need_input_grad=False)
    assert all(bool(v.grad.isfinite().all()) and float(v.grad.abs().max()) > 0 for v in model.trainable_variables)
    hist = E.fit_evaluator(model, x.numpy(), labels.numpy(), 2, 2, validation_data=(x.numpy(), labels.numpy()))
    assert all(np.isfinite(hist[k]).all() for k in hist) and 0 <= hist["accuracy"][-1] <= 1


@gpu
def test_narrow_head_on_class_numbers(restore):
    """Fewer classes than features: the logits are stored; unlabelled samples, whatever they hold, leave no trace."""
    from music_generator_amd import evaluacion as E
    M.clear_session()
    model = E.define_evaluator(1)[0]
    _, head = E._split_head(model)
    gen = torch.Generator().manual_seed(2)
    x = torch.randn((6, head.cin), generator=gen)
    labels = torch.tensor([3, -1, 0, 8, 9, 5])
    w = torch.randn((head.cin, 9), generator=gen) / head.cin ** 0.5
    head.kernel.assign(w.numpy())
    lab = torch.where(labels < 9, labels, torch.full_like(labels, -1)).int()
    dl = (lab >= 0).double() / 4
    want = reference(x, w, torch.zeros((9,)), lab, dl)
    x[1], x[4] = float("nan"), 1e30
    model.bind_grads(0).zero_()
    loss, hits, count, dx = head.loss(x.cuda(), E.class_numbers_to_device(labels))
    got = {"loss": want["loss"], "lse": want["lse"], "dx": dx.cpu(), "dw": head.kernel.grad.cpu().view(-1, 9), "db": head.bias.grad.cpu()}
    # products over 384 000 float32 terms: sqrt(384 000) roundings of 2^-24 relative in the mean
    check(got, want, torch.float32, 40.0)
    assert int(count) == 4 and int(hits) == int(want["hits"].sum())
    assert abs(float(loss) - float(want["loss"].sum())) < 1e-4


@gpu
def test_probabilities_on_every_position(restore):
    model = position_classifier(30)
    p = model(torch.randn((2, 8, 40, 2)).cuda())
    assert tuple(p.shape) == (2, 8, 40, 30) and float((p.sum(dim=-1) - 1).abs().max()) < 1e-5


def test_class_numbers_are_told_by_their_type():
    from music_generator_amd import evaluacion as E
    assert E._class_numbers(np.array([1, 2])) and E._class_numbers(torch.tensor([1, 2]))
    assert not E._class_numbers(np.eye(3)) and not E._class_numbers(torch.eye(3))


def test_a_model_without_a_classifier_head_is_refused():
    from music_generator_amd import evaluacion as E
    with pytest.raises(ValueError):
        E._split_head(M.define_discriminator(1)[0][0])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,e,v", [(9, 20, 300), (90, 40, 700), (200, 128, 900), (150, 300, 1000)])
def test_weights_of_very_different_size(n, e, v, dtype):
    """dloss from 1e-7 to 1, of both signs, and zeros: the gradient of every single row is as exact as if it stood alone."""
    x, w, b, labels, dloss = case(n, e, v, dtype, seed=40 + e, unlabelled=0)
    gen = torch.Generator().manual_seed(41)
    dloss = torch.sign(torch.randn((n,), generator=gen)) * 10.0 ** (-7 * torch.rand((n,), generator=gen))
    dloss[::5] = 0.0
    want, got = reference(x, w, b, labels, dloss), run(x, w, b, labels, dloss)
    check(got, want, dtype, float((x.double() @ w.double()).abs().max()))
    unit = 2.0 ** -23 * (8 + 2 * float((x.double() @ w.double()).abs().max()))
    # one row: the bound of check() on that row; the label's term of a row is at most |dloss| |W[:, label]|
    slack = unit * dloss.double().abs() * w.double().norm(dim=0)[labels.long()]
    tol = 4 * unit + (2.0 ** -8 + 2.0 ** -10 if dtype == torch.bfloat16 else 0.0)
    off = (got["dx"].double() - want["dx"]).norm(dim=1)
    assert bool((off <= tol * want["dx"].norm(dim=1) + slack + 1e-30).all()), float((off / want["dx"].norm(dim=1).clamp(min=1e-30)).max())
    assert bool((got["dx"][dloss == 0] == 0).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("n,e,v", [(3000, 130, 12000), (300, 1000, 9000), (17, 700, 20000), (2000, 100, 9000), (2000, 33, 9000), (20, 128, 30000),
                                   (16, 600, 3000), (17, 600, 3000)])
def test_parts_and_pieces(n, e, v, dtype, accumulate):
    """Sizes whose classes come in several pieces (the first) or whose products are split, with labels at every end."""
    x, w, b, labels, dloss = case(n, e, v, dtype, seed=50 + e)
    labels[0], labels[1], labels[2] = 0, v - 1, v // 2
    want = reference(x, w, b, labels, dloss)
    if accumulate:
        gen = torch.Generator().manual_seed(51)
        dw, db = torch.randn(w.shape, generator=gen) * 1e-3, torch.randn(b.shape, generator=gen) * 1e-3
        want["dw"], want["db"] = want["dw"] + dw.double(), want["db"] + db.double()
        got = run(x, w, b, labels, dloss, accumulate=True, dw=dw, db=db)
    else:
        got = run(x, w, b, labels, dloss)
    check(got, want, dtype, float((x.double() @ w.double()).abs().max()))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,e,v", [(9, 40, 300), (90, 40, 700), (90, 33, 700), (200, 128, 900), (150, 300, 1000), (150, 301, 1000)])
def test_unlabelled_rows_may_hold_large_values(n, e, v, dtype):
    """Rows without a label (below 0 or above the classes) change no bit of the others, whatever finite values they hold: they
    have no part in the scales of the planes either."""
    x, w, b, labels, dloss = case(n, e, v, dtype, seed=60 + e, unlabelled=0)
    off = torch.arange(n) % 3 == 1
    labels[off] = torch.where(torch.arange(n) % 2 == 0, -7, v)[off].int()
    clean_x, clean_d = x.clone(), dloss.clone()
    clean_x[off], clean_d[off] = 0.0, 0.0
    x[off], dloss[off] = 3e30, -2e30
    got, want = run(x, w, b, labels, dloss), run(clean_x, w, b, labels, clean_d)
    assert all(torch.equal(got[k], want[k]) for k in want)
    check(got, reference(clean_x, w, b, labels, clean_d), dtype, float((clean_x.double() @ w.double()).abs().max()))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [float("-inf"), -3.4028234663852886e38])
@pytest.mark.parametrize("n,e,v", [(1, 40, 301), (9, 300, 300), (90, 40, 700), (90, 33, 701), (200, 128, 900), (150, 300, 1001), (150, 301, 1000)])
def test_masked_classes_may_hold_anything(n, e, v, mask, dtype):
    """A masked class changes no bit of the rest, whatever its column of W holds: NaN, infinities, large finite values."""
    x, w, b, labels, dloss = case(n, e, v, dtype, seed=70 + e, unlabelled=0)
    off = torch.arange(v) % 4 == 1
    b[off] = mask
    labels = torch.where(off[labels.long()], labels - 1, labels)
    clean = w.clone()
    clean[:, off] = 0.0
    for fill in (3e30, float("inf"), float("nan")):
        w[:, off] = fill
        got, want = run(x, w, b, labels, dloss), run(x, clean, b, labels, dloss)
        assert all(torch.equal(got[k], want[k]) for k in want), fill
    check(got, reference(x, clean, b, labels, dloss), dtype, float((x.double() @ clean.double()).abs().max()))
    assert bool((got["dw"][:, off] == 0).all()) and bool((got["db"][off] == 0).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("n,e,v", [(17, 1, 1), (17, 16, 33), (32, 15, 4097), (33, 63, 300), (64, 129, 1000), (65, 300, 2049), (96, 128, 130),
                                   (97, 1000, 4001), (128, 257, 31), (100, 17, 40000), (128, 1000, 5000),
                                   (20, 70, 40003), (60, 130, 32770), (70, 40, 32768), (128, 20, 33001)])
def test_blocks_of_rows(n, e, v, dtype, accumulate):
    """17 to 128 rows: every count of row blocks, features and classes that end inside a tile, rows of W with and without whole
    16-byte pieces."""
    x, w, b, labels, dloss = case(n, e, v, dtype, seed=80 + e)
    labels[0], labels[1], labels[2] = 0, v - 1, v // 2
    want = reference(x, w, b, labels, dloss)
    largest = float((x.double() @ w.double()).abs().max())
    if accumulate:
        gen = torch.Generator().manual_seed(81)
        dw, db = torch.randn(w.shape, generator=gen) * 1e-3, torch.randn(b.shape, generator=gen) * 1e-3
        want["dw"], want["db"] = want["dw"] + dw.double(), want["db"] + db.double()
        check(run(x, w, b, labels, dloss, accumulate=True, dw=dw, db=db), want, dtype, largest)
    else:
        check(run(x, w, b, labels, dloss), want, dtype, largest)


@gpu
def test_integer_one_hot_rows_are_one_hot_rows():
    """One-hot labels of an integer type, which have the shape of the model's output, are what they were with float rows."""
    from music_generator_amd import evaluacion
    from music_generator_amd.graph import Input, Model
    from music_generator_amd.layers import Flatten

    gen = np.random.default_rng(5)
    x = gen.uniform(-1, 1, (6, 2, 8, 4)).astype(np.float32)
    hot = np.eye(5, dtype=np.int64)[gen.integers(0, 5, 6)]
    M.clear_session()
    t = Input(shape=(2, 8, 4))
    model = Model(t, evaluacion.SoftmaxDense(5)(Flatten()(t)))
    a = evaluacion.evaluate(model, x, hot.astype(np.float32), 4)
    assert evaluacion.evaluate(model, x, hot, 4) == a == evaluacion.evaluate(model, x, torch.from_numpy(hot), 4)
    b = evaluacion.evaluate(model, x, hot.argmax(axis=1), 4)
    assert b["accuracy"] == a["accuracy"] and b["loss"] == pytest.approx(a["loss"], rel=1e-5)
    start = [v.numpy().copy() for v in model.trainable_variables]
    runs = []
    for y in (hot.astype(np.float32), hot, hot.argmax(axis=1)):
        for v, value in zip(model.trainable_variables, start):
            v.assign(value)
        runs.append(evaluacion.fit_evaluator(model, x, y, 2, 4))
    assert runs[0] == runs[1]
    assert runs[2]["loss"] == pytest.approx(runs[0]["loss"], rel=1e-4)


@gpu
@pytest.mark.parametrize("n,e,v,dtype", [(3, 300, 7500000, torch.float32), (100, 300, 7500001, torch.float32), (200, 300, 7500000, torch.float32),
                                         (150, 128, 8000000, torch.bfloat16), (8000000, 128, 300, torch.bfloat16),
                                         (8000000, 290, 140, torch.bfloat16)])
def test_offsets_beyond_32_bits(n, e, v, dtype):
    """Operands of more than 2^32 bytes: loss, lse and gradients of some rows and classes, the last ones among them, against
    float64 on the device.  Tolerances of check(), per row and class."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((n, e), generator=gen, device="cuda").to(dtype)
    w = torch.randn((e, v), generator=gen, device="cuda") / e ** 0.5
    b = torch.randn((v,), generator=gen, device="cuda") * 0.3
    labels = torch.randint(0, v, (n,), generator=gen, device="cuda", dtype=torch.int32)
    labels[-1] = v - 1
    dloss = torch.rand((n,), generator=gen, device="cuda") + 0.5
    loss, lse = torch.empty((n,), device="cuda"), torch.empty((n,), device="cuda")
    ops.dense_xent_fwd(x, w, b, labels, loss, lse)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    ops.dense_xent_bwd(x, w, b, labels, lse, dloss, dx, dw, db)
    rows = torch.unique(torch.cat([torch.randint(0, n, (20,), generator=gen, device="cuda"), torch.tensor([0, n - 1], device="cuda")]))
    cols = torch.unique(torch.cat([torch.randint(0, v, (20,), generator=gen, device="cuda"), torch.tensor([0, v - 1], device="cuda")]))
    xr, lr = x[rows].double(), labels[rows].long()
    z = torch.empty((len(rows), v), dtype=torch.float64, device="cuda")
    for c in range(0, v, 500000):
        z[:, c:c + 500000] = xr @ w[:, c:c + 500000].double() + b[c:c + 500000].double()
    unit = 2.0 ** -23 * (8 + 2 * float(z.abs().max()))
    want = torch.logsumexp(z, dim=1)
    at = z.gather(1, lr[:, None])[:, 0]
    assert float((lse[rows].double() - want).abs().max()) <= unit + 2.0 ** -23 * float(want.abs().max())
    assert float((loss[rows].double() - (want - at)).abs().max()) <= unit + 2.0 ** -23 * float(want.abs().max())
    z = torch.exp(z - want[:, None])
    z[torch.arange(len(rows), device="cuda"), lr] -= 1.0
    z *= dloss[rows].double()[:, None]
    dxr = torch.zeros((len(rows), e), dtype=torch.float64, device="cuda")
    for c in range(0, v, 500000):
        dxr += z[:, c:c + 500000] @ w[:, c:c + 500000].double().t().contiguous()
    del z
    slack = unit * dloss[rows].double() * w[:, lr].double().norm(dim=0)
    tol = 4 * unit + (2.0 ** -8 + 2.0 ** -10 if dtype == torch.bfloat16 else 0.0)
    assert bool(((dx[rows].double() - dxr).norm(dim=1) <= tol * dxr.norm(dim=1) + slack).all())
    # classes: every row's probability of them, from the kernel's lse (checked above on the rows)
    dwc, dbc = torch.zeros((e, len(cols)), dtype=torch.float64, device="cuda"), torch.zeros((len(cols),), dtype=torch.float64, device="cuda")
    size = torch.zeros((len(cols),), dtype=torch.float64, device="cuda")
    wc, bc = w[:, cols].double(), b[cols].double()
    for i in range(0, n, 500000):
        xi = x[i:i + 500000].double()
        hot = (labels[i:i + 500000, None].long() == cols[None]).double()
        d = (torch.exp(xi @ wc + bc - lse[i:i + 500000].double()[:, None]) - hot) * dloss[i:i + 500000].double()[:, None]
        dwc += xi.t().contiguous() @ d
        dbc += d.sum(dim=0)
        size += d.abs().sum(dim=0)          # terms of both signs: a float32 sum and 2^-24 of the scale are relative to these
    most = float(x[:500000].abs().max())
    assert bool(((db[cols].double() - dbc).abs() <= 4 * unit * size + 2.0 ** -24 * 1.5).all())
    assert bool(((dw[:, cols].double() - dwc).abs().amax(dim=0) <= (4 * unit * size + 2.0 ** -24 * 1.5) * most).all())
    del x, w, dx, dw
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("n,e,v,dtype", [(2, 40, 500, torch.float32), (13, 30, 600, torch.bfloat16), (90, 200, 33000, torch.float32),
                                         (60, 70, 500, torch.bfloat16), (140, 60, 700, torch.float32), (140, 200, 700, torch.bfloat16)])
def test_two_captured_graphs_of_every_form(n, e, v, dtype):
    """Each form captured twice, into graphs of their own, replayed on two streams at once and again: every replay gives the
    bits of an eager call on the same values."""
    sets = []
    for seed in (90, 91):
        x, w, b, labels, dloss = [t.cuda() for t in case(n, e, v, dtype, seed=seed)]
        outs = [torch.empty((n,)).cuda(), torch.empty((n,)).cuda(), torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)]

        def step(x=x, w=w, b=b, labels=labels, dloss=dloss, outs=outs):
            ops.dense_xent_fwd(x, w, b, labels, outs[0], outs[1])
            ops.dense_xent_bwd(x, w, b, labels, outs[1], dloss, outs[2], outs[3], outs[4])

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        sets.append((graph, step, outs, torch.cuda.Stream()))
    for _ in range(3):
        torch.cuda.synchronize()
        for graph, _, _, st in sets:
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for graph, step, outs, _ in sets:
            got = [t.clone() for t in outs]
            for t in outs:
                t.fill_(5.0)
            step()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, outs))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,e,v", [(1, 30, 400), (4, 30, 400), (16, 30, 400), (60, 30, 400), (100, 140, 33000), (200, 140, 400)])
def test_hits_of_every_form(n, e, v, dtype):
    x, w, b, labels, dloss = case(n, e, v, dtype, seed=95, unlabelled=0)
    z = x.double() @ w.double() + b.double()
    top = z.topk(2, dim=1)
    clear = top.values[:, 0] - top.values[:, 1] > 1e-3          # no tie within the logits' accuracy
    labels[::2] = top.indices[::2, 0].int()
    labels[n // 2] = -1
    got, want = run(x, w, b, labels, dloss)["hits"], reference(x, w, b, labels, dloss)["hits"]
    assert torch.equal(got[clear], want[clear]) and int(got[n // 2]) == 0
