"""The linear cross entropy against float64, within bounds by arithmetic
(linear_ce_reference.py): sizes from one row, one column and one class up to
several tiles, pieces of the vocabulary, ignored rows that hold NaN, labels that
are no class, strides, streams and graphs."""
import pytest
import torch

import orda_hip as H
from orda_hip.autograd import linear_cross_entropy_autograd

from linear_ce_reference import Exact

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def inputs(n, h, v, dtype, seed=0, ignored=0.0, scale=2.0):
    g = torch.Generator().manual_seed(1000 * seed + n + 7 * h + 13 * v)
    x = torch.randn(n, h, generator=g).to(DT[dtype])
    w = (torch.randn(v, h, generator=g) * scale / h ** 0.5).to(DT[dtype])
    y = torch.randint(0, v, (n,), generator=g)
    if ignored:
        y[torch.rand(n, generator=g) < ignored] = -100
    gn, gl = torch.randn(n, generator=g), torch.randn(n, generator=g) * 0.1
    return [t.cuda() for t in (x, w, y, gn, gl)]


def both(x, w, y, gn, gl, **kw):
    nll, lse = H.linear_cross_entropy(x, w, y, **kw)
    gh, gw = H.linear_cross_entropy_backward(x, w, y, lse, gn, gl, **kw)
    return nll, lse, gh, gw


def check(x, w, y, gn, gl, **kw):
    nll, lse, gh, gw = both(x, w, y, gn, gl, **kw)
    kw.pop("vocab_piece", None)
    e = Exact(x, w, y, **kw)
    e.check_losses(nll, lse)
    e.check_gradients(gh, gw, gn, gl)


SHAPES = [(1, 1, 1), (1, 8, 3), (2, 64, 256), (17, 72, 257), (64, 64, 300), (100, 33, 1000),
          (129, 520, 513), (257, 128, 777), (300, 200, 5001), (513, 264, 4097), (31, 1000, 12289)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n, h, v", SHAPES)
def test_against_float64(n, h, v, dtype):
    check(*inputs(n, h, v, dtype))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n, h, v", [(5, 40, 100), (257, 128, 777), (300, 200, 5001), (700, 96, 1500)])
@pytest.mark.parametrize("ignored", [0.1, 0.6, 0.97])
def test_ignored_rows_and_smoothing(n, h, v, dtype, ignored):
    check(*inputs(n, h, v, dtype, seed=1, ignored=ignored), label_smoothing=0.1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("piece", [1, 256, 700, 5000, 10000])
def test_pieces_of_the_vocabulary(dtype, piece):
    check(*inputs(300, 200, 5001, dtype, seed=2, ignored=0.2), label_smoothing=0.05, vocab_piece=piece)


@pytest.mark.parametrize("n, h, v", [(1, 8, 300), (17, 72, 257), (129, 520, 513), (300, 33, 1001), (700, 1000, 2300)])
@pytest.mark.parametrize("ignored", [0.0, 0.5])
def test_fp32_over_planes(n, h, v, ignored):
    """fp32 in pieces of the vocabulary takes three-plane operands whatever its
    size (small calls in one piece keep their logits)."""
    check(*inputs(n, h, v, "f32", seed=6, ignored=ignored), label_smoothing=0.1, vocab_piece=256)


@pytest.mark.parametrize("n, h, v, ignored", [(5000, 4096, 600, 0.1), (5000, 4096, 600, 0.4), (17000, 40, 300, 0.3),
                                              (16384, 24, 70, 0.02), (8200, 1032, 500, 0.0)])
def test_many_rows(n, h, v, ignored):
    """Whole rounds of tiles with a split tail, and more rows than a workgroup
    counts for itself."""
    check(*inputs(n, h, v, "bf16", seed=4, ignored=ignored), vocab_piece=256)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_no_row_left(dtype):
    x, w, y, gn, gl = inputs(70, 48, 300, dtype)
    y.fill_(-100)
    x.fill_(float("nan"))
    nll, lse, gh, gw = both(x, w, y, gn, gl)
    for t in (nll, lse, gh, gw):
        assert (t == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_no_rows(dtype):
    x, w, y, gn, gl = inputs(3, 48, 300, dtype)
    nll, lse, gh, gw = both(x[:0], w, y[:0], gn[:0], gl[:0])
    assert nll.shape == lse.shape == (0,) and gh.shape == (0, 48)
    assert (gw == 0).all() and gw.shape == w.shape


def test_no_rows_of_more_classes_than_one_launch_holds():
    """The zeros of 2^26 classes are 2^32 threads, which HIP takes in no one launch."""
    v = 2 ** 26 + 5
    w = torch.zeros(v, 1, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(0, 1, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(0, dtype=torch.int64, device="cuda")
    torch.full((v, 1), 7.0, dtype=torch.bfloat16, device="cuda")   # what the gradient's memory held before
    _, lse = H.linear_cross_entropy(x, w, y)
    _, gw = H.linear_cross_entropy_backward(x, w, y, lse, lse, grad_hidden=False)
    assert gw.shape == w.shape and (gw == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_masked_rows_are_not_read(dtype, what):
    x, w, y, gn, gl = inputs(150, 64, 700, dtype, ignored=0.4)
    x[y == -100] = what
    gn[y == -100] = what
    gl[y == -100] = what
    nll, lse, gh, gw = both(x, w, y, gn, gl)
    zero = torch.zeros((), device="cuda")
    e = Exact(x, w, y)
    e.check_losses(nll, lse)
    e.check_gradients(gh, gw, torch.where(y == -100, zero, gn), torch.where(y == -100, zero, gl))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_ignore_index_may_be_a_class(dtype):
    x, w, y, gn, gl = inputs(64, 64, 7, dtype)
    check(x, w, y, gn, gl, ignore_index=3)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_label_that_is_no_class(dtype):
    x, w, y, gn, gl = inputs(40, 64, 300, dtype)
    y[3], y[17] = 300, -1
    nll, lse, gh, gw = both(x, w, y, gn, gl)
    Exact(x, w, y).check_losses(nll, lse)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[3, 17]] = True
    assert torch.isnan(gh[bad]).all() and not torch.isnan(gh[~bad]).any()
    assert torch.isnan(gw).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strides_and_int32_labels(dtype):
    x, w, y, gn, gl = inputs(200, 96, 500, dtype, ignored=0.3)
    xs = torch.randn(200, 131, device="cuda").to(x.dtype)
    xs[:, 5:101] = x
    ws = torch.randn(500, 101, device="cuda").to(w.dtype)
    ws[:, 3:99] = w
    ys = torch.stack([y, y + 1], 1).to(torch.int32)[:, 0]
    gs = torch.stack([gn, gl], 1)
    want = both(x, w, y, gn, gl)
    for a, b in zip(want, both(xs[:, 5:101], ws[:, 3:99], ys, gs[:, 0], gs[:, 1])):
        assert torch.equal(a, b)
    for a, b in zip(want, both(x.t().contiguous().t(), w.t().contiguous().t(), y, gn, gl)):
        assert torch.equal(a, b)


def test_large_logits():
    """Logits of several hundred: the losses stay finite and right."""
    x, w, y, gn, gl = inputs(64, 128, 1000, "f32", scale=200.0)
    check(x, w, y, gn, gl)
    nll, lse = H.linear_cross_entropy(x * 1e20, w * 1e20, y)   # infinite logits
    assert not torch.isfinite(lse).any() and not torch.isfinite(nll).any()


@pytest.mark.parametrize("dtype, piece", [("bf16", None), ("f32", None), ("f32", 256)])
@pytest.mark.parametrize("n", [1, 40, 100])
def test_logits_at_the_end_of_the_range(n, dtype, piece):
    """A class 2^127 above the others is the whole sum; beyond, it counts as infinite; classes as far below add
    nothing; all so far below are minus infinity."""
    x = torch.zeros(n, 64, dtype=DT[dtype], device="cuda")
    x[:, 0] = 2.0 ** 64
    w = torch.zeros(600, 64, dtype=DT[dtype], device="cuda")
    y = torch.full((n,), 300, device="cuda")
    for top, low, want in ((2.0 ** 63, 0.0, 2.0 ** 127), (1.9 * 2.0 ** 63, 0.0, float("inf")),
                           (2.0 ** 63, -1.75 * 2.0 ** 63, 2.0 ** 127), (-1.75 * 2.0 ** 63, -1.875 * 2.0 ** 63, -float("inf")),
                           (-2.0 ** 63, -1.875 * 2.0 ** 63, -2.0 ** 127)):
        w[:, 0] = low
        w[300, 0] = top
        nll, lse = H.linear_cross_entropy(x, w, y, vocab_piece=piece)
        assert (lse == want).all(), (top, low, lse[:3])
        if abs(want) < float("inf"):
            assert (nll == 0).all()


@pytest.mark.parametrize("want", [(True, False), (False, True), (False, False)])
def test_single_gradients(want):
    x, w, y, gn, gl = inputs(100, 64, 700, "bf16", ignored=0.3)
    _, lse, gh, gw = both(x, w, y, gn, gl)
    a, b = H.linear_cross_entropy_backward(x, w, y, lse, gn, gl, grad_hidden=want[0], grad_weight=want[1])
    assert (a is None) != want[0] and (b is None) != want[1]
    assert a is None or torch.equal(a, gh)
    assert b is None or torch.equal(b, gw)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("which", ["nll", "lse", "both"])
def test_autograd(dtype, which):
    x, w, y, gn, gl = inputs(120, 72, 600, dtype, ignored=0.3)
    x.requires_grad_(True)
    w.requires_grad_(True)
    nll, lse = linear_cross_entropy_autograd(x, w, y, label_smoothing=0.1)
    loss = (nll * gn).sum() if which == "nll" else (lse * gl).sum() if which == "lse" else (nll * gn + lse * gl).sum()
    loss.backward()
    e = Exact(x.detach(), w.detach(), y, label_smoothing=0.1)
    e.check_gradients(x.grad, w.grad, gn if which != "lse" else None, gl if which != "nll" else None)


def test_autograd_partial_and_unused():
    x, w, y, gn, gl = inputs(50, 64, 300, "bf16")
    x.requires_grad_(True)
    nll, lse = linear_cross_entropy_autograd(x, w, y)
    nll.sum().backward()
    assert x.grad is not None
    with torch.no_grad():
        nll2, _ = linear_cross_entropy_autograd(x, w, y)
    assert torch.equal(nll2, nll.detach()) and not nll2.requires_grad


def test_autograd_reports_changed_inputs():
    x, w, y, gn, gl = inputs(50, 64, 300, "bf16")
    w.requires_grad_(True)
    nll, _ = linear_cross_entropy_autograd(x, w, y)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        nll.sum().backward()


def test_no_second_derivative():
    """A gradient of the gradient is reported, not silently zero."""
    x, w, y, gn, gl = inputs(20, 64, 300, "f32")
    x.requires_grad_(True)
    gn.requires_grad_(True)
    nll, _ = linear_cross_entropy_autograd(x, w, y)
    (gx,) = torch.autograd.grad(nll, x, gn, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.sum().backward()


def test_batched_gradients_refused():
    x, w, y, gn, gl = inputs(20, 64, 300, "bf16")
    x.requires_grad_(True)
    nll, _ = linear_cross_entropy_autograd(x, w, y)
    with pytest.raises((H.OrdaError, RuntimeError)):
        torch.autograd.grad(nll, x, torch.eye(20, device="cuda"), is_grads_batched=True)


def test_gradient_against_differences():
    """Central differences of the library's own losses along its gradient: with
    |change of a logit| <= D per unit, the third derivative of each row's loss is
    at most 4 D^3 (a third central moment of a variable within [-D, D]
    is at most (2D)^3 / 2), so a step t errs by t^2/6 of that, and by the losses'
    own error over t."""
    x, w, y, gn, gl = inputs(60, 48, 500, "f32", scale=1.0)
    nll, lse = H.linear_cross_entropy(x, w, y)
    gh, _ = H.linear_cross_entropy_backward(x, w, y, lse, gn, gl)
    ux = 0.2 * gh / gh.abs().max()
    e = Exact(x, w, y)
    t = 2.0 ** -2

    def f(s):
        a, b = H.linear_cross_entropy(x + s * t * ux, w, y)
        return (a.double() * gn.double() + b.double() * gl.double()).sum().item()
    got = (f(1) - f(-1)) / (2 * t)
    want = (gh.double() * ux.double()).sum().item()
    D = (ux.double().cpu() @ e.w.t()).abs().amax(1)
    weight = (gn.abs() + gl.abs()).double().cpu()
    step = (4 * D ** 3 * weight).sum().item() * t * t / 6
    noise = ((e.dnll + e.dlse) * weight).sum().item() / t
    assert abs(got - want) <= step + 2 * noise
    assert abs(want) > 10 * (step + 2 * noise)   # the test can tell


def test_another_stream_and_two_at_once():
    x, w, y, gn, gl = inputs(500, 256, 4000, "bf16", ignored=0.3)
    want = both(x, w, y, gn, gl)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for s in (a, b, a, b):
        with torch.cuda.stream(s):
            got.append(both(x, w, y, gn, gl))
    torch.cuda.synchronize()
    for g in got:
        for p, q in zip(want, g):
            assert torch.equal(p, q)


def test_captured_and_replayed():
    x, w, y, gn, gl = inputs(300, 128, 3000, "bf16", ignored=0.3)
    both(x, w, y, gn, gl)   # warm up
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = both(x, w, y, gn, gl)
    with torch.cuda.graph(g2):
        o2 = both(x, w, y, gn, gl, label_smoothing=0.1)
    for seed in (11, 12, 13):
        for t, s in zip((x, w, y, gn, gl), inputs(300, 128, 3000, "bf16", seed=seed, ignored=0.1 * (seed - 10))):
            t.copy_(s)
        want1, want2 = both(x, w, y, gn, gl), both(x, w, y, gn, gl, label_smoothing=0.1)
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        for p, q in zip(want1 + want2, o1 + o2):
            assert torch.equal(p, q)


def test_repeated_calls_agree_bit_for_bit():
    args = inputs(700, 512, 9000, "bf16", ignored=0.3)
    first = both(*args)
    for _ in range(3):
        for p, q in zip(first, both(*args)):
            assert torch.equal(p, q)


def test_refusals():
    x, w, y, gn, gl = inputs(20, 64, 300, "bf16")
    for bad in (dict(hidden=x[0]), dict(weight=w[:, :63]), dict(labels=y[:-1]), dict(labels=y.float()),
                dict(hidden=x.half()), dict(weight=w.float()), dict(weight=w.cpu()), dict(label_smoothing=2.0),
                dict(vocab_piece=0), dict(hidden=x[:, :0], weight=w[:, :0]), dict(weight=w[:0])):
        kw = dict(hidden=x, weight=w, labels=y)
        kw.update(bad)
        with pytest.raises(H.OrdaError):
            H.linear_cross_entropy(**kw)
    lse = torch.zeros(20, device="cuda")
    for bad in (dict(lse=None), dict(lse=lse[:5]), dict(grad_nll=gn.double()), dict(grad_lse=gl[:3]),
                dict(grad_nll=gn.cpu())):
        kw = dict(hidden=x, weight=w, labels=y, lse=lse, grad_nll=gn)
        kw.update(bad)
        with pytest.raises(H.OrdaError):
            H.linear_cross_entropy_backward(**kw)


def test_a_weight_at_a_wide_pitch():
    """Columns of a table 2^23 + 72 wide: 300 rows lie 5 GB apart."""
    table = torch.empty((300, 2 ** 23 + 72), dtype=torch.bfloat16, device="cuda")
    w = table[:, 8:72]
    w.copy_(torch.randn(300, 64, generator=torch.Generator().manual_seed(1)).mul_(0.2))
    h = torch.randn(70, 64, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    y = torch.randint(0, 300, (70,), generator=torch.Generator().manual_seed(3)).cuda()
    nll, lse = H.linear_cross_entropy(h, w, y)
    Exact(h, w.contiguous(), y).check_losses(nll, lse)
    g = torch.ones_like(nll)
    got = H.linear_cross_entropy_backward(h, w, y, lse, g)
    for a, b in zip(got, H.linear_cross_entropy_backward(h, w.contiguous(), y, lse, g)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v, h", [(1000, 64), (4339, 520), (997, 200), (129, 8), (33, 1304), (2000, 264), (700, 1003), (301, 67)])
@pytest.mark.parametrize("n", [1, 16, 17, 32, 33, 64, 65])
def test_few_rows(n, v, h, dtype):
    """Rows by waves of 16 classes (up to 64 of them) beside the tiles' (65): widths of parts of 128 columns,
    vocabularies of parts of 16 and 64 classes, ignored and bad labels, both outputs' gradients."""
    g = torch.Generator().manual_seed(n * 7 + v)
    x = (torch.randn(n, h, generator=g)).to(dtype).cuda()
    w = (torch.randn(v, h, generator=g) * 0.2).to(dtype).cuda()
    y = torch.randint(0, v, (n,), generator=g)
    y[-1] = v - 1
    if n > 8:
        y[::5] = -100
    y = y.cuda()
    exact = Exact(x, w, y, label_smoothing=0.1)
    nll, lse = H.linear_cross_entropy(x, w, y, label_smoothing=0.1)
    exact.check_losses(nll, lse)
    gn, gl = torch.randn(n, generator=g).cuda(), torch.randn(n, generator=g).cuda()
    gh, gw = H.linear_cross_entropy_backward(x, w, y, lse, gn, gl, label_smoothing=0.1)
    exact.check_gradients(gh, gw, gn, gl)
    pieces = H.linear_cross_entropy(x, w, y, label_smoothing=0.1, vocab_piece=256)
    exact.check_losses(*pieces)


@pytest.mark.parametrize("n", [1, 40, 200])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_few_rows_of_infinite_logits(n, value):
    """One class whose logit is infinite or NaN in every row: lse is what logsumexp gives."""
    x = torch.zeros(n, 64, dtype=torch.bfloat16, device="cuda")
    x[:, :2] = 1.0
    w = torch.randn(500, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    w[77, 0] = value
    y = torch.full((n,), 3, device="cuda")
    nll, lse = H.linear_cross_entropy(x, w, y)
    logits = (w[:, 0].double() + w[:, 1].double()).cpu()
    want = torch.logsumexp(logits, 0)
    # (two exact terms a logit; 2^-22 an exponential, 64 + 1 additions, the maximum twice)
    bound = 2.0 ** -22 + 70 * 2.0 ** -24 + 6 * 2.0 ** -24 * 8
    if torch.isfinite(want):
        assert ((lse.double().cpu() - want).abs() <= bound).all()
        assert ((nll.double().cpu() - (want - logits[3])).abs() <= bound + 2.0 ** -24 * 16).all()
    else:
        assert torch.equal(lse.double().cpu(), want.expand(n)) or (torch.isnan(want) and torch.isnan(lse).all())
        assert torch.equal(nll.isnan(), lse.isnan())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("at", [0, 1, 3])
@pytest.mark.parametrize("n, h, v", [(5, 2426, 300), (90, 2051, 333), (5, 1543, 77), (3, 4099, 130), (200, 2050, 65)])
def test_widths_that_are_copied(n, h, v, at, dtype):
    """Weights whose rows begin anywhere, wider than a wave's vectors, between NaN on both sides."""
    g = torch.Generator().manual_seed(n + h)
    frame = torch.full((v, h + 9), float("nan"), dtype=dtype, device="cuda")
    w = frame[:, at:at + h]
    w.copy_((torch.randn(v, h, generator=g) * 0.1).to(dtype))
    x = torch.randn(n, h, generator=g).to(dtype).cuda()
    y = torch.randint(0, v, (n,), generator=g).cuda()
    exact = Exact(x, w, y)
    nll, lse = H.linear_cross_entropy(x, w, y)
    exact.check_losses(nll, lse)
    gn = torch.randn(n, generator=g).cuda()
    gh, gw = H.linear_cross_entropy_backward(x, w, y, lse, gn)
    exact.check_gradients(gh, gw, gn, torch.zeros_like(gn))


@pytest.mark.parametrize("n, h, v", [(3, 4096, 44000), (64, 1000, 180001)])
def test_few_fp32_rows_of_a_large_weight(n, h, v):
    """Weights that three planes would cut into pieces: few rows stream them whole, odd vocabularies too."""
    g = torch.Generator(device="cuda").manual_seed(n + h)
    x = torch.randn(n, h, generator=g, device="cuda")
    w = torch.randn(v, h, generator=g, device="cuda") * (2.0 / h ** 0.5)
    y = torch.randint(0, v, (n,), generator=g, device="cuda")
    y[0] = v - 1
    if n > 8:
        y[1::5] = -100
    gn, gl = torch.randn(n, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda")
    check(x, w, y, gn, gl, label_smoothing=0.1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n, h, v", [(1, 200, 997), (16, 264, 2000), (17, 1003, 700), (33, 67, 301), (64, 520, 1025), (5, 72, 513)])
def test_few_rows_in_pieces(n, h, v, dtype):
    """Gradients of few rows over pieces of 256 classes, the last one shorter: labels past the first piece,
    grad_hidden added from piece to piece, weights copied by pieces (odd widths)."""
    x, w, y, gn, gl = inputs(n, h, v, dtype, seed=7)
    y[-1] = v - 1
    if n > 8:
        y[::5] = -100
    check(x, w, y, gn, gl, label_smoothing=0.1, vocab_piece=256)


@pytest.mark.parametrize("n, h, v, dtype, ignored", [(12545, 8192, 300, "bf16", 0.0), (12545, 8192, 300, "bf16", 0.4),
                                                     (20000, 6208, 260, "bf16", 0.1), (12545, 2688, 300, "f32", 0.0),
                                                     (12545, 2688, 300, "f32", 0.3)])
def test_rows_in_bands(n, h, v, dtype, ignored):
    """Batches whose rows overflow the last cache walk their tiles in bands of 32 M-tiles, with a count of rows that
    only the device knows: whole bands and rows past them, and (0.4 ignored) fewer rows than a band."""
    check(*inputs(n, h, v, dtype, seed=8, ignored=ignored), vocab_piece=256)
