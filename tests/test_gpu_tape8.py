"""The 8-bit activation tape: format, special blocks, products with the recovered derivative, the fused convolution
backward that reads it, refusals.  The reference is the definition in float64 on the CPU."""
import numpy as np
import pytest
import torch

import music_generator_amd as M
from music_generator_amd import ops
from music_generator_amd._cabi import MgxError

gpu = pytest.mark.gpu
ALPHA = 20000.0


def kept_reference(x):
    """Values the tape of x stands for, float64, from the definition."""
    v = x.detach().cpu().double().reshape(-1)
    n = v.numel()
    v = torch.nn.functional.pad(v, (0, -n % 32)).view(-1, 32)
    big = v.abs().max(dim=1, keepdim=True).values
    m, ex = torch.frexp(torch.where(torch.isfinite(big), big, torch.ones_like(big)))
    top = torch.ldexp(torch.ones_like(m), torch.where(m <= 0.5 * (1 + 2.0 ** -8), ex - 1, ex).clamp(min=-118))
    q = ((v * 128.0 / top).floor().clamp(-128.0, 127.0) + 0.5) * top / 128.0
    q = torch.where(big == 0, torch.zeros_like(q), q)
    q = torch.where(torch.isfinite(v).all(dim=1, keepdim=True), q, torch.full_like(q, float("nan")))
    return q.view(-1)[:n].view(x.shape)


def derivative(y):
    return torch.clamp(1.0 + 1.0 / ALPHA - y * y, min=1.0 / ALPHA)


def activations(shape, seed, dtype):
    pre = torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * 1.2
    return (torch.tanh(pre) + pre / ALPHA).to(dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 7, 31, 32, 33, 256, 1000, 4 * 1501 * 32, 300001])
def test_kept_values_are_the_definition(n, dtype):
    x = activations((n,), n, dtype).cuda()
    t = ops.tape8_pack(x)
    assert t.nbytes() == 33 * ((n + 31) // 32)
    want = kept_reference(x)
    for out in (torch.float32, torch.bfloat16):
        assert torch.equal(ops.tape8_unpack(t, out).cpu().double(), want)      # eight significant bits: exact in both
    assert ops.tape8_unpack(t).dtype == dtype
    # |tanh(v) + v / alpha| <= 1 + |v| / alpha, |v| < 7 here: less than a 256th past 1, so H <= 1; values up to H come back
    # within H / 256, those above it within H / 128
    v = x.cpu().double()
    assert float(v.abs().max()) <= 1 + 2.0 ** -8
    assert bool(((want - v).abs() <= torch.where(v.abs() <= 1, 2.0 ** -8, 2.0 ** -7)).all())


@gpu
def test_special_blocks():
    x = torch.zeros((12, 32))
    x[1] = torch.linspace(-1, 1, 32)                 # both ends of the range
    x[2, 5] = float("nan")
    x[3, 9] = float("-inf")
    x[4] = 1e-42                                     # below the smallest normal number
    x[5, 3] = 3.3e38                                 # above 2^127
    x[6] = 2.0 ** torch.arange(-20, 12)
    x[7, 31] = -2.0 ** -100
    x[8] = -0.0
    x[9, 0] = 2.0 ** -118
    x[10] = torch.nextafter(torch.tensor(1.0), torch.tensor(2.0))
    x[11] = -1e-7                                    # floor, not rounding towards zero
    x[11, 0] = 1.0
    x = torch.cat([x, torch.zeros((3, 32))])
    x[12, 0], x[12, 1] = -1.0 - 2.0 ** -8, 1.0 + 2.0 ** -8       # the border of the rule for H, both signs
    x[13, 0] = 1.0 + 2.0 ** -8 + 2.0 ** -23
    x[14, 0], x[14, 1] = 1.0 + 2.0 ** -7, 0.3
    for y in (x, x.to(torch.bfloat16)):
        got = ops.tape8_unpack(ops.tape8_pack(y.cuda()), torch.float32).cpu().double()
        assert torch.equal(torch.nan_to_num(got, 77.0), torch.nan_to_num(kept_reference(y), 77.0))
        assert got[2].isnan().all() and got[3].isnan().all()
        assert (got[0] == 0).all() and (got[8] == 0).all()
        assert got[1, 0] == -got[1, 31] == -255.0 / 256.0
        assert got[12, 0] == -got[12, 1] == -255.0 / 256.0 or y.dtype == torch.bfloat16


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [5, 32, 8 * 1500 * 32, 100003])
def test_product_with_the_recovered_derivative(n, dtype):
    y = activations((n,), 3, torch.bfloat16).cuda()
    a = (torch.randn((n,), generator=torch.Generator().manual_seed(4)) * 1e-3).to(dtype).cuda()
    got = ops.mul_dact_tape8(a, ops.tape8_pack(y), ALPHA).cpu().double()
    want = a.cpu().double() * derivative(kept_reference(y))
    # one rounding to bf16 (2^-8 of the value covers it and the float32 steps: 1 + 1/alpha and 1 - y^2 are 2^-24 off
    # where the derivative is at least 2^-8, the smallest distance of a kept y from 1)
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 1e-30).all())


@gpu
def test_non_finite_blocks_reach_the_gradient():
    y = torch.zeros((64,), dtype=torch.bfloat16)
    y[3] = float("inf")
    got = ops.mul_dact_tape8(torch.ones((64,)).cuda(), ops.tape8_pack(y.cuda()), ALPHA).cpu()
    assert got[:32].isnan().all() and got[32:].isfinite().all()


def conv_case(n, h, w, cin, k, seed):
    gen = torch.Generator().manual_seed(seed)
    x = activations((n, h, w, cin), seed, torch.bfloat16)
    g = torch.randn((n, h, w, 32), generator=gen).to(torch.bfloat16)
    # kernels that are exact in bf16, so that the data gradient has one rounding only
    wt = (torch.randn((k, k, cin, 32), generator=gen) / (k * cin ** 0.5)).to(torch.bfloat16).float()
    p = (k - 1) // 2
    d = ops.make_conv_desc(nimg=n, hin=h, win=w, cin=cin, hout=h, wout=w, kh=k, kw=k, pt=p, pl=p, ngemm=32, cout=32,
                           wsk=32, wsn=1, wtap=cin * 32, nbias=32)
    return d, x, g, wt


def conv_reference(x, g, wt, act):
    """Gradients of the 'same' convolution by autograd in float64 on the kept values."""
    q = kept_reference(x)
    k = wt.shape[0]
    p0, p1 = (k - 1) // 2, k - 1 - (k - 1) // 2
    xi = q.permute(0, 3, 1, 2).clone().requires_grad_(True)
    wi = wt.double().permute(3, 2, 0, 1).clone().requires_grad_(True)
    bi = torch.zeros((32,), dtype=torch.float64, requires_grad=True)
    y = torch.nn.functional.conv2d(torch.nn.functional.pad(xi, (p0, p1, p0, p1)), wi, bi)
    dx, dw, db = torch.autograd.grad(y, (xi, wi, bi), g.double().permute(0, 3, 1, 2))
    dx = dx.permute(0, 2, 3, 1)
    return dx * derivative(q) if act else dx, dw.permute(2, 3, 1, 0), db


@gpu
@pytest.mark.parametrize("act", [True, False])
@pytest.mark.parametrize("n,h,w,cin,k", [(1, 8, 64, 32, 3), (1, 1, 1, 32, 3), (2, 9, 65, 32, 3), (3, 13, 131, 32, 2),
                                         (1, 1, 7, 32, 2), (1, 8, 32, 128, 3), (2, 5, 37, 128, 3), (1, 3, 1501, 32, 3)])
def test_convolution_backward(n, h, w, cin, k, act):
    d, x, g, wt = conv_case(n, h, w, cin, k, seed=n * 100 + h + w)
    t = ops.tape8_pack(x.cuda())
    dw0 = torch.randn((k, k, cin, 32), generator=torch.Generator().manual_seed(1))
    dw, db = dw0.cuda(), torch.full((32,), 0.5).cuda()
    dx = torch.empty((n, h, w, cin), dtype=torch.bfloat16, device="cuda")
    ops.conv_bwd_tape8(d, t, g.cuda(), wt.cuda(), dw, db, dx, ALPHA if act else 0.0)
    rx, rw, rb = conv_reference(x, g, wt, act)
    # dx: one rounding to bf16, and float32 sums of 9 * 32 products of magnitude ~ 1 / (3 sqrt(cin))
    assert bool(((dx.cpu().double() - rx).abs() <= 2.0 ** -8 * rx.abs() + 288 * 2.0 ** -24).all())
    # dw, db: exact products, float32 sums of P terms of magnitude ~ 1: P ulp at most, sqrt(P) in practice
    lim = n * h * w * 2.0 ** -24 * 4 + 2.0 ** -22
    assert float((dw.cpu().double() - dw0.double() - rw).abs().max()) <= lim
    assert float((db.cpu().double() - 0.5 - rb).abs().max()) <= lim


@gpu
def test_convolution_backward_equals_the_bf16_kernel_on_the_kept_values():
    d, x, g, wt = conv_case(2, 17, 200, 32, 3, seed=5)
    t = ops.tape8_pack(x.cuda())
    kept = ops.tape8_unpack(t)
    out = []
    for f, xin in ((ops.conv_bwd_tape8, t), (ops.conv_bwd_bf16, kept)):
        dw, db = torch.zeros_like(wt).cuda(), torch.zeros((32,)).cuda()
        dx = torch.empty_like(kept)
        f(d, xin, g.cuda(), wt.cuda(), dw, db, dx, ALPHA)
        out.append((dw, db, dx))
    for a, b in zip(*out):
        assert torch.equal(a, b)


@gpu
def test_captured_pack_and_backward_replay():
    d, x, g, wt = conv_case(1, 8, 100, 32, 3, seed=6)
    xd, gd, wd = x.cuda(), g.cuda(), wt.cuda()
    dw, db, dx = torch.zeros_like(wd), torch.zeros((32,), device="cuda"), torch.empty_like(xd)

    def step():
        dw.zero_()
        db.zero_()
        ops.conv_bwd_tape8(d, ops.tape8_pack(xd), gd, wd, dw, db, dx, ALPHA)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(3):
        xd.copy_(activations(tuple(x.shape), 50 + seed, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in (dw, db, dx)]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (dw, db, dx)))


@gpu
def test_empty_tensor():
    t = ops.tape8_pack(torch.empty((0, 32), device="cuda"))
    assert t.nbytes() == 0 and tuple(ops.tape8_unpack(t).shape) == (0, 32)


@gpu
def test_refusals():
    x = torch.zeros((4, 8, 16, 32), dtype=torch.bfloat16, device="cuda")
    t = ops.tape8_pack(x)
    d, _, g, wt = conv_case(4, 8, 16, 32, 3, seed=0)
    g, wt = g.cuda(), wt.cuda()
    dw, db, dx = torch.zeros_like(wt), torch.zeros((32,), device="cuda"), torch.empty_like(x)
    for bad in (x.permute(0, 3, 1, 2), x.half(), x.double(), x.cpu()):
        with pytest.raises(MgxError):
            ops.tape8_pack(bad)
    with pytest.raises(MgxError):
        ops.tape8_pack(x.view(-1)[1:])                                   # not 16-byte aligned
    with pytest.raises(MgxError):
        ops.tape8_unpack(t, torch.float16)
    with pytest.raises(MgxError):
        ops.tape8_unpack(ops.Tape8((4, 8, 16, 33), t.dtype, t.codes, t.exps))
    with pytest.raises(MgxError):
        ops.mul_dact_tape8(x[:2], t, ALPHA)
    with pytest.raises(MgxError):
        ops.mul_dact_tape8(x, t, 0.0)
    with pytest.raises(MgxError):
        ops.conv_bwd_tape8(d, ops.tape8_pack(x[:2].contiguous()), g, wt, dw, db, dx)
    with pytest.raises(MgxError):
        ops.conv_bwd_tape8(d, t, g.float(), wt, dw, db, dx)
    with pytest.raises(MgxError):
        ops.conv_bwd_tape8(d, t, g, wt, dw, db, dx, act_alpha=-1.0)
    with pytest.raises(MgxError):
        ops.conv_bwd_tape8(d, t, g, wt, dw, torch.zeros((16,), device="cuda"), dx)


# ---- the tape of a model (backend.TAPE8) ----
@pytest.fixture
def tape8():
    M.backend.TAPE8 = True
    yield
    M.backend.TAPE8 = False
    M.backend.set_precision("float32")


def discriminator(stage, fade, precision):
    M.backend.set_precision(precision)
    M.clear_session()
    return M.define_discriminator(stage + 1)[stage][int(fade)]


def whole_again(tape):
    """The tape with every 8-bit form replaced by the tensor it stands for (one per Tape8, as a tape shares them)."""
    seen = {}

    def back(v, dtype=None):
        if isinstance(v, ops.Tape8):
            return seen.setdefault((id(v), dtype), ops.tape8_unpack(v, dtype))
        if isinstance(v, tuple):      # a subclass marks the float32 copy of a bf16 input
            return tuple(back(u) for u in v) if type(v) is tuple else type(v)([back(u, torch.float32) for u in v])
        if hasattr(v, "premultiplied"):
            v.x, v.yact = back(v.x), back(v.yact)
        return v
    for i, entry in enumerate(tape):
        tape[i] = back(entry)
    return tape


def tape_bytes(tape):
    seen = {}

    def count(v):
        if isinstance(v, ops.Tape8):
            seen[v.codes.data_ptr()] = v.nbytes()
        elif isinstance(v, torch.Tensor):
            seen[v.data_ptr()] = v.numel() * v.element_size()
        elif isinstance(v, (tuple, list)):
            for u in v:
                count(u)
        elif hasattr(v, "premultiplied"):
            for u in (v.x, v.yact, v.dact):
                count(u)
    count(list(tape))
    return sum(seen.values())


def gradients(model, tape, dy, **kw):
    flat = model.bind_grads()
    flat.zero_()
    dx = model.backward(tape, dy, **kw)
    return flat.clone(), dx


@gpu
@pytest.mark.parametrize("precision,fade", [("bfloat16", False), ("bfloat16", True), ("float32", True)])
def test_model_backward_from_the_8_bit_tape(tape8, precision, fade):
    """The sweep over the bytes gives the bits of the same sweep over the tensors they stand for, the forward is
    untouched, and the tape is a half (bf16) or a quarter (float32) of what it was."""
    d = discriminator(1, fade, precision)
    x = torch.randn((4, 8, 1500, 2), generator=torch.Generator().manual_seed(2)).cuda()
    dy = torch.full((4, 1), 0.25).cuda()
    M.backend.TAPE8 = False
    y0, full = d.forward(x, save=True)
    full_bytes, estimate0 = tape_bytes(full), d.tape_bytes_estimate(4)
    g0, dx0 = gradients(d, full, dy, need_input_grad=True)
    M.backend.TAPE8 = True
    y1, tape = d.forward(x, save=True)
    assert torch.equal(y0, y1)
    assert tape_bytes(tape) < (0.65 if precision == "bfloat16" else 0.35) * full_bytes
    assert d.tape_bytes_estimate(4) < 0.65 * estimate0
    g1, dx1 = gradients(d, tape, dy, need_input_grad=True)
    g2, dx2 = gradients(d, whole_again(d.forward(x, save=True)[1]), dy, need_input_grad=True)
    assert torch.equal(g1, g2) and torch.equal(dx1, dx2)
    # the gradients of activations off by at most 2^-8: a kept value is off by 2^-7 / sqrt(12) = 0.23 % of 1 in the mean
    # and its derivative by 2 |y| of that; the activations' root mean square is about 0.6, so a layer adds 0.4 % (its
    # input in the weight gradient) and 0.6 % (derivative), and the 20 layers of the sweep 20 * 0.6 % at most
    for a, b in ((g1, g0), (dx1, dx0)):
        assert float((a - b).norm() / b.norm()) < 20 * 0.006


@gpu
def test_sweep_without_weight_gradients(tape8):
    d = discriminator(1, False, "bfloat16")
    x = torch.randn((4, 8, 1500, 2), generator=torch.Generator().manual_seed(3)).cuda()
    dy = torch.full((4, 1), 0.25).cuda()
    dx = d.backward(d.forward(x, save=True)[1], dy, need_input_grad=True, need_weight_grads=False)
    want = d.backward(whole_again(d.forward(x, save=True)[1]), dy, need_input_grad=True, need_weight_grads=False)
    assert torch.equal(dx, want)


@gpu
def test_weight_gradient_against_differences(tape8):
    """Difference quotient of the last convolution's kernel: its gradient uses the kept input, its derivative and nothing
    in front of it, so the quotient of the exact forward is met to the rounding of that one layer."""
    d = discriminator(0, False, "float32")
    x = torch.randn((4, 4, 750, 2), generator=torch.Generator().manual_seed(4)).cuda()
    conv = [l for l in d.layers if type(l).__name__ == "Conv2D"][-1]
    direction = torch.randn((conv.kernel.size,), generator=torch.Generator().manual_seed(5)).cuda()
    direction /= direction.norm()
    dy = torch.ones((4, 1)).cuda()
    _, tape = d.forward(x, save=True)
    gradients(d, tape, dy)
    slope = float((conv.kernel.grad.double() * direction.double()).sum())
    w0, step, ends = conv.kernel.value().clone(), 1e-2, []
    for s in (step, -step):
        conv.kernel.value().copy_(w0 + s * direction)
        ends.append(float(d(x).double().sum()))
    conv.kernel.value().copy_(w0)
    quotient = (ends[0] - ends[1]) / (2 * step)
    norm = float(conv.kernel.grad.double().norm())
    # 1 % of the gradient's length covers the 0.4 % and 0.6 % of one layer's input and derivative; the quotient's own
    # float32 noise is 4 outputs of 2^-24 relative over 2 step
    assert abs(quotient - slope) <= 0.01 * norm + 4 * abs(ends[0]) * 2.0 ** -24 / step


@gpu
@pytest.mark.parametrize("use_graph", [False, True])
def test_train_step(tape8, use_graph):
    """Fade-in steps train from the 8-bit tape, eagerly and replayed: finite metrics, other bits than from the ordinary
    tape, and a graph of its own for each kind of tape."""
    def build():
        M.backend.set_precision("bfloat16")
        M.clear_session()
        M.layers.set_init_seed(7)
        d, g = M.define_discriminator(2), M.define_generator(2)
        gan = M.define_composite(d, g, (1, 100, 2))[1][1]
        gan.set_train_steps(10)
        gan.use_graph = use_graph
        return gan
    real = torch.randn((4, 8, 1500, 2), generator=torch.Generator().manual_seed(6)).cuda()
    runs = []
    for eight in (False, True):
        M.backend.TAPE8 = eight
        gan = build()
        torch.manual_seed(11)
        out = []
        for _ in range(4):
            out.append({k: float(v) for k, v in gan.train_step(real).items()})
        runs.append(out)
        assert all(np.isfinite(list(m.values())).all() for m in out)
    assert runs[0] != runs[1]                       # the gradients are not the same bits
    if use_graph:
        M.backend.TAPE8 = False                     # another key: an eager step, then a capture of its own
        before = len(gan._graphs)
        gan.train_step(real)
        assert len(gan._graphs) == before + 1


@gpu
def test_two_captured_graphs_share_nothing():
    """Two backward calls captured into graphs of their own and replayed on two streams at once: each call's scratch memory is
    its own, also after later calls asked for more."""
    sets = []
    for seed, (n, h, w) in enumerate(((2, 16, 700), (1, 24, 900))):
        d, x, g, wt = conv_case(n, h, w, 32, 3, seed + 30)
        t, g, wt = ops.tape8_pack(x.cuda()), g.cuda(), wt.cuda()
        dx, dw, db = torch.empty_like(g), torch.zeros_like(wt), torch.zeros((32,)).cuda()

        def step(d=d, t=t, g=g, wt=wt, dx=dx, dw=dw, db=db):
            dw.zero_()
            db.zero_()
            ops.conv_bwd_tape8(d, t, g, wt, dw, db, dx, ALPHA)

        step()
        torch.cuda.synchronize()
        want = [v.clone() for v in (dx, dw, db)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        sets.append((graph, (dx, dw, db), want, torch.cuda.Stream(), (t, g, wt)))      # a replay reads the captured tensors
    d, x, g, wt = conv_case(2, 64, 3000, 32, 3, 40)
    ops.conv_bwd_tape8(d, ops.tape8_pack(x.cuda()), g.cuda(), wt.cuda(), torch.zeros_like(wt).cuda(), torch.zeros((32,)).cuda(),
                       torch.empty_like(g).cuda(), ALPHA)
    for _ in range(3):
        for graph, outs, _, st, _ in sets:
            for v in outs:
                v.fill_(7.0)
        torch.cuda.synchronize()
        for graph, _, _, st, _ in sets:
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for _, outs, want, _, _ in sets:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


@gpu
def test_offsets_beyond_32_bits():
    """Six clips of the full resolution (2.36e9 values): packing, unpacking and the derivative's product at both ends and
    where the 32-bit offsets end, and the convolution's data gradient of the last clip against a call with that clip alone."""
    n, h, w = 6, 256, 48000
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty((n, h, w, 32), dtype=torch.bfloat16, device="cuda")
    g = torch.empty_like(x)
    for i in range(n):
        x[i] = torch.tanh(torch.randn((h, w, 32), generator=gen, device="cuda"))
        g[i] = torch.randn((h, w, 32), generator=gen, device="cuda")
    t = ops.tape8_pack(x)
    y = ops.tape8_unpack(t)
    flat, back = x.view(-1), y.view(-1)
    for at in (0, 2 ** 30 - 4096, 2 ** 31 - 4096, flat.numel() - 8192):
        part = ops.tape8_pack(flat[at:at + 8192].contiguous())
        assert torch.equal(part.codes, t.codes[at:at + 8192]) and torch.equal(part.exps, t.exps[at // 32:at // 32 + 256])
        assert torch.equal(back[at:at + 8192], ops.tape8_unpack(part))
        product = ops.mul_dact_tape8(g.view(-1)[at:at + 8192].contiguous(), part, ALPHA)
    del y, back
    whole = ops.mul_dact_tape8(g, t, ALPHA)
    assert torch.equal(whole.view(-1)[-8192:], product)
    del whole
    wt = (torch.randn((3, 3, 32, 32), generator=gen, device="cuda") / 17.0)
    dw, db, dx = torch.zeros_like(wt), torch.zeros((32,), device="cuda"), torch.empty_like(x)

    def desc(images):
        return ops.make_conv_desc(nimg=images, hin=h, win=w, cin=32, hout=h, wout=w, kh=3, kw=3, pt=1, pl=1, ngemm=32, cout=32, wsk=32, wsn=1,
                                  wtap=32 * 32, nbias=32)

    ops.conv_bwd_tape8(desc(n), t, g, wt, dw, db, dx, ALPHA)
    one = torch.empty_like(x[:1])
    sums = torch.zeros_like(wt)
    for i in range(n):
        ops.conv_bwd_tape8(desc(1), ops.tape8_pack(x[i:i + 1]), g[i:i + 1], wt, sums, torch.zeros_like(db), one, ALPHA)
        assert torch.equal(dx[i:i + 1], one), i
    # the same terms added in another order: sums over 7.4e7 positions whose float32 partial sums are off by 2^-24 a level
    assert float((dw - sums).norm()) <= 2.0 ** -16 * float(sums.norm())
    del x, g, dx, t
    torch.cuda.empty_cache()
