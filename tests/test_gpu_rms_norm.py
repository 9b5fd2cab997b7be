"""The norm, its output in e4m3 and its gradients against float64.

U is a rounding of fp32. The factor s of a row is formed in 64 bits and rounded
once; a value t·s·(w + o) has then at most four more roundings, and one to its type.
"""
import pytest
import torch
import torch.utils.checkpoint

import orda_hip as H
from orda_hip.autograd import rms_norm_autograd

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -24
EPS = 1e-6
TINY = 1e-37


def normal(shape, dtype, seed=0, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed + 17 * len(shape) + 3 * shape[0] + 7 * shape[-1])
    return (torch.randn(shape, generator=g) * std + mean).to(DT[dtype]).cuda()


def total_of(x, r):
    return x if r is None else (x.float() + r.float()).to(x.dtype)


def formula(t, w, offset, eps=EPS):
    """In 64 bits on the CPU (weights as float32 values added to a float32 offset)."""
    t, w = t.double().cpu(), w.double().cpu()
    s = (t.square().mean(-1, keepdim=True) + eps).rsqrt()
    return t * s * (w + offset), s


def check_out(out, t, w, offset=0.0, eps=EPS):
    v, _ = formula(t, w, offset, eps)
    assert out.dtype == t.dtype and out.shape == t.shape
    bound = (ROUND[out.dtype] + 6 * U) * v.abs() + TINY
    bad = ~((out.double().cpu() - v).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} off, the first at {bad.nonzero()[0].tolist()}"


# each form of the kernel (few and many rows, one to eight vectors a thread, rows read
# twice), whole and partial vectors of eight, fewer columns than one
SHAPES = [(1, 1), (3, 5), (1, 8), (2, 9), (1, 4096), (5, 1531), (300, 1500), (7, 2048), (9, 2049), (4, 8192), (3, 8200),
          (2, 32768), (2, 32769), (3, 40000), (1025, 64), (1030, 1024), (1025, 1027), (1100, 2048), (1027, 4096), (1025, 4090),
          (1026, 8192), (1025, 5001), (1025, 16384)]


@pytest.mark.parametrize("dtype, weight", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("n, h", SHAPES)
def test_forward(n, h, dtype, weight):
    x, w = normal((n, h), dtype), normal((h,), weight, std=0.2, mean=1.0)
    check_out(H.rms_norm(x, w, eps=EPS), x, w)
    r = normal((n, h), dtype, seed=1, std=4.0)
    out, t = H.rms_norm(x, w, residual=r, eps=EPS, weight_offset=1.0)
    assert torch.equal(t, total_of(x, r))
    check_out(out, t, w, 1.0)


def quantized(v):
    """Codes and scales of float32 values, on the CPU."""
    r, c = v.shape
    b = torch.nn.functional.pad(v, (0, -c % 128)).view(r, -1, 128)
    top = b.abs().amax(2)
    s = (top / torch.full_like(top, 448.0)).clamp_min(2.0 ** -126)
    q = (b / s[:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return q.reshape(r, -1)[:, :c], s


@pytest.mark.parametrize("dtype, weight", [("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("n, h", SHAPES)
def test_fp8(n, h, dtype, weight):
    """Bit for bit: values are formed in 64 bits and rounded to fp32 once (another
    order of the 64-bit sum moves one across a border once in 1e8)."""
    x, w, r = normal((n, h), dtype), normal((h,), weight, std=0.2), normal((n, h), dtype, seed=1, std=3.0)
    codes, scales, t = H.rms_norm_fp8(x, w, residual=r, eps=EPS, weight_offset=1.0)
    assert torch.equal(t, total_of(x, r)) and codes.shape == x.shape
    want, s = quantized(formula(t, w, 1.0)[0].float())
    assert torch.equal(scales.cpu(), s)
    assert torch.equal(codes.cpu().view(torch.uint8), want)
    codes, scales = H.rms_norm_fp8(x, w, eps=EPS)
    want, s = quantized(formula(x, w, 0.0)[0].float())
    assert torch.equal(scales.cpu(), s) and torch.equal(codes.cpu().view(torch.uint8), want)


def check_grads(gx, gw, g, t, w, gt=None, offset=0.0, eps=EPS):
    """d = Σ g·q·t is a sum of h terms in fp32, at most h/64 + 64 in a row of additions;
    the weight's gradient one of n terms, each with three roundings."""
    n, h = t.shape
    g64, t64, q = g.double().cpu(), t.double().cpu(), w.double().cpu() + offset
    s = (t64.square().mean(1, keepdim=True) + eps).rsqrt()
    gq = g64 * q
    k = (gq * t64).mean(1, keepdim=True) * s * s
    k_mag = (gq * t64).abs().mean(1, keepdim=True) * s * s
    ref = s * (gq - t64 * k)
    if gx is not None:
        err = s * (5 * U * (gq.abs() + t64.abs() * k.abs()) + t64.abs() * k_mag * (h / 64 + 70) * U)
        if gt is not None:
            ref = ref + gt.double().cpu()
            err = err + U * ref.abs()
        bound = err + ROUND[gx.dtype] * (ref.abs() + err) + TINY
        bad = ~((gx.double().cpu() - ref).abs() <= bound)
        assert gx.dtype == t.dtype and not bad.any(), f"grad_x: {int(bad.sum())} off, the first at {bad.nonzero()[0].tolist()}"
    if gw is not None:
        terms = g64 * t64 * s
        ref, mag = terms.sum(0), terms.abs().sum(0)
        err = (n + 6) * U * mag
        bound = err + ROUND[gw.dtype] * (ref.abs() + err) + TINY
        bad = ~((gw.double().cpu() - ref).abs() <= bound)
        assert gw.dtype == w.dtype and not bad.any(), f"grad_weight: {int(bad.sum())} off, at {bad.nonzero()[0].tolist()}"


GRAD_SHAPES = [(1, 1), (3, 5), (1, 4096), (17, 512), (33, 513), (300, 1500), (9, 2049), (700, 2048), (1000, 1531), (1030, 4096),
               (5, 8192), (300, 8192), (260, 5001), (3, 16384), (2, 16385), (40, 20000), (5000, 96), (4100, 256)]


@pytest.mark.parametrize("dtype, weight", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("n, h", GRAD_SHAPES)
def test_gradients(n, h, dtype, weight):
    t, w, g = normal((n, h), dtype, std=2.0), normal((h,), weight, std=0.2), normal((n, h), dtype, seed=2, std=0.1)
    gt = normal((n, h), dtype, seed=3, std=0.1)
    gx, gw = H.rms_norm_backward(g, t, w, grad_total=gt, eps=EPS, weight_offset=1.0)
    check_grads(gx, gw, g, t, w, gt, 1.0)
    gx, none = H.rms_norm_backward(g, t, w, eps=EPS, grad_weight=False)
    assert none is None
    check_grads(gx, None, g, t, w)
    none, gw2 = H.rms_norm_backward(g, t, w, eps=EPS, weight_offset=1.0, grad_x=False)
    assert none is None and torch.equal(gw2, gw)


@pytest.mark.parametrize("n, h", [(3, 40), (5, 300), (2, 1500)])
def test_gradient_against_differences(n, h):
    """Along a direction d of x and w: (L(+e) - L(-e)) / 2e in fp32, where L = Σ g·out is
    added up in 64 bits. What the difference itself is off is measured on the formula in
    64 bits; each of the two sums is off by six roundings of its terms."""
    x, w, g = normal((n, h), "f32"), normal((h,), "f32", std=0.2, mean=1.0), normal((n, h), "f32", seed=2)
    dx, dw = normal((n, h), "f32", seed=5), normal((h,), "f32", seed=6, std=0.2)
    e = 2.0 ** -8

    def off(sign):   # exact in fp32 only up to its rounding: the formula gets the same values
        return x + sign * e * dx, w + sign * e * dw
    gpu, exact, mag = [], [], 0.0
    for sign in (1, -1):
        xs, ws = off(sign)
        gpu.append((H.rms_norm(xs, ws, eps=EPS).double().cpu() * g.double().cpu()).sum())
        v = formula(xs, ws, 0.0)[0] * g.double().cpu()
        exact.append(v.sum())
        mag += float(v.abs().sum())
    gx, gw = H.rms_norm_backward(g, x, w, eps=EPS)
    along = (gx.double() * dx.double()).sum().cpu() + (gw.double() * dw.double()).sum().cpu()
    x64, w64 = x.double().cpu().requires_grad_(True), w.double().cpu().requires_grad_(True)
    s = (x64.square().mean(-1, keepdim=True) + EPS).rsqrt()
    rx, rw = torch.autograd.grad((x64 * s * w64 * g.double().cpu()).sum(), [x64, w64])
    true = (rx * dx.double().cpu()).sum() + (rw * dw.double().cpu()).sum()
    step = abs((exact[0] - exact[1]) / (2 * e) - true)
    # the gradients' own error, as in check_grads with every term at its magnitude
    own = (h / 64 + 80 + n) * U * ((rx.abs() + (g.cpu().double() * w64).abs() * s) * dx.double().cpu().abs()).sum() * 4 \
        + (n + 6) * U * ((g.cpu().double() * x64 * s).abs().sum(0) * dw.double().cpu().abs()).sum()
    assert abs((gpu[0] - gpu[1]) / (2 * e) - along) <= step + 6 * U * mag / (2 * e) + own


def test_strides_shapes_and_empty():
    x, w, r = normal((40, 300), "bf16"), normal((300,), "bf16"), normal((40, 300), "bf16", seed=1)
    want, t = H.rms_norm(x, w, residual=r)
    codes, scales, _ = H.rms_norm_fp8(x, w, residual=r)
    g = normal((40, 300), "bf16", seed=2)
    gx, gw = H.rms_norm_backward(g, t, w, grad_total=x)

    def frame(m):
        f = torch.full((40, 333), 9.0, dtype=m.dtype, device="cuda")
        f[:, 5:305] = m
        return f[:, 5:305]
    for view in (frame, lambda m: m.t().contiguous().t()):
        out, total = H.rms_norm(view(x), w, residual=view(r))
        assert torch.equal(out, want) and torch.equal(total, t)
        c, s, total = H.rms_norm_fp8(view(x), w, residual=view(r))
        assert torch.equal(c.float(), codes.float()) and torch.equal(s, scales) and torch.equal(total, t)
        a, b = H.rms_norm_backward(view(g), view(t), w, grad_total=view(x))
        assert torch.equal(a, gx) and torch.equal(b, gw)
    out, total = H.rms_norm(x.view(2, 20, 300), w, residual=r.view(2, 20, 300))
    assert out.shape == (2, 20, 300) and torch.equal(out.view(40, 300), want) and total.shape == out.shape
    a, b = H.rms_norm_backward(g.view(2, 20, 300), t.view(2, 20, 300), w, grad_total=x.view(2, 20, 300))
    assert torch.equal(a.view(40, 300), gx) and torch.equal(b, gw)
    assert torch.equal(H.rms_norm(x[0], w), H.rms_norm(x[:1], w)[0])
    wide = torch.stack([w, w], 1)
    assert torch.equal(H.rms_norm(x, wide[:, 0]), H.rms_norm(x, w))
    # rows that begin at any multiple of two bytes, and a broadcast one
    for at in (1, 3, 6):
        flat = torch.zeros(40 * 300 + at, dtype=torch.bfloat16, device="cuda")
        flat[at:] = x.reshape(-1)
        assert torch.equal(H.rms_norm(flat[at:].view(40, 300), w, residual=r)[0], want)
    assert torch.equal(H.rms_norm(x[:1].expand(40, 300), w), H.rms_norm(x[:1], w).expand(40, 300))
    assert H.rms_norm(x[:0], w).shape == (0, 300) and H.rms_norm_fp8(x[:0], w)[1].shape == (0, 3)
    a, b = H.rms_norm_backward(x[:0], x[:0], w)
    assert a.shape == (0, 300) and (b == 0).all() and b.shape == (300,)
    assert H.rms_norm(x[:, :0], w[:0]).shape == (40, 0) and H.rms_norm(x.view(2, 20, 300)[..., :0], w[:0]).shape == (2, 20, 0)
    assert H.rms_norm_backward(x[:, :0], x[:, :0], w[:0])[1].shape == (0,)


@pytest.mark.parametrize("h", [100, 4096, 40000])
def test_extremes(h):
    """Rows of zeros, of values whose squares leave fp32's range, and of infinities and NaN."""
    x, w = normal((6, h), "f32"), normal((h,), "f32", std=0.2, mean=1.0)
    x[0] = 0
    x[1] *= 1e30
    x[2] *= 1e-30
    assert (H.rms_norm(x, w)[0] == 0).all()
    check_out(H.rms_norm(x, w), x, w)
    check_out(H.rms_norm(x[1:], w, eps=0.0), x[1:], w, eps=0.0)
    assert torch.isnan(H.rms_norm(x, w, eps=0.0)[0]).all()   # 0 / 0
    codes, scales = H.rms_norm_fp8(x, w)
    want, s = quantized(formula(x, w, 0.0)[0].float())
    assert torch.equal(scales.cpu(), s) and torch.equal(codes.cpu().view(torch.uint8), want)
    x[3, h // 2], x[4, 1] = float("nan"), float("inf")
    out = H.rms_norm(x, w)
    assert torch.isnan(out[3]).all()
    assert torch.isnan(out[4, 1]) and (out[4, 2:] == 0).all()
    check_out(out[[0, 1, 2, 5]], x[[0, 1, 2, 5]], w)
    scales = H.rms_norm_fp8(x, w)[1]
    assert torch.isnan(scales[3]).all() and torch.isnan(scales[4, 0]) and torch.isfinite(scales[[0, 1, 2, 5]]).all()
    # a row's NaN stays in its row of grad_x, and is in all of the weight's gradient
    g = normal((6, h), "f32", seed=2)
    gx, gw = H.rms_norm_backward(g, x, w)
    assert torch.isnan(gx[3]).all() and torch.isfinite(gx[[0, 5]]).all() and torch.isnan(gw).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("residual", [True, False])
def test_autograd(dtype, residual):
    x, w = normal((2, 30, 136), dtype).requires_grad_(True), normal((136,), dtype, mean=1.0).requires_grad_(True)
    r = normal((2, 30, 136), dtype, seed=1).requires_grad_(True) if residual else None
    g, gt = normal((2, 30, 136), dtype, seed=2), normal((2, 30, 136), dtype, seed=3)
    got = rms_norm_autograd(x, w, residual=r, eps=EPS)
    if residual:
        out, t = got
        torch.autograd.backward([out, t], [g, gt])
        assert torch.equal(x.grad, r.grad)
    else:
        out, t = got, x
        out.backward(g)
    check_grads(x.grad.view(60, 136), w.grad, g.view(60, 136), t.detach().view(60, 136), w.detach(),
                gt.view(60, 136) if residual else None)
    if not residual:
        return
    # each output alone, a gradient that is broadcast, inputs that want none
    x.grad = w.grad = r.grad = None
    out, t = rms_norm_autograd(x, w, residual=r, eps=EPS)
    t.sum().backward()
    assert (x.grad == 1).all() and (r.grad == 1).all() and (w.grad is None or (w.grad == 0).all())
    x.grad = w.grad = r.grad = None
    out, t = rms_norm_autograd(x, w, residual=r, eps=EPS)
    out.sum().backward()
    check_grads(x.grad.view(60, 136), w.grad, torch.ones_like(g).view(60, 136), t.detach().view(60, 136), w.detach())
    out, t = rms_norm_autograd(x.detach(), w.detach(), residual=r, eps=EPS)
    (gr,) = torch.autograd.grad(out, r, g)
    check_grads(gr.view(60, 136), None, g.view(60, 136), t.detach().view(60, 136), w.detach())
    out, t = rms_norm_autograd(x.detach(), w, residual=r.detach(), eps=EPS)
    (gw,) = torch.autograd.grad(out, w, g)
    check_grads(None, gw, g.view(60, 136), t.detach().view(60, 136), w.detach())
    with torch.no_grad():
        assert torch.equal(rms_norm_autograd(x, w, residual=r)[0], H.rms_norm(x, w, residual=r)[0])
    out, _ = rms_norm_autograd(x, w, residual=r)
    gv = g.clone().requires_grad_(True)
    (gx,) = torch.autograd.grad(out, x, gv, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.sum().backward()


def test_a_change_in_place_is_reported():
    x, w = normal((4, 64), "f32").requires_grad_(True), normal((64,), "f32").requires_grad_(True)
    out = rms_norm_autograd(x, w)
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


@pytest.mark.parametrize("n, h", [(1, 4096), (2000, 520), (40, 20000)])
def test_other_streams_and_graphs(n, h):
    x, w, r, g = normal((n, h), "bf16"), normal((h,), "bf16"), normal((n, h), "bf16", seed=1), normal((n, h), "bf16", seed=2)

    def step():
        out, t = H.rms_norm(x, w, residual=r)
        codes, scales, _ = H.rms_norm_fp8(x, w, residual=r)
        return out, t, codes.float(), scales, *H.rms_norm_backward(g, t, w, grad_total=x)
    want = step()
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)] * 2:
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    for o in got:
        assert all(torch.equal(a, b) for a, b in zip(o, want))
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    for seed in (1, 2, 3):
        x.copy_(normal((n, h), "bf16", seed=10 * seed))
        g.copy_(normal((n, h), "bf16", seed=10 * seed + 1))
        want = step()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_offsets_past_32_bits():
    """Rows behind the first 2^32 bytes and values of the inputs."""
    n, h = 2 ** 20 + 5, 2 ** 12
    x = torch.zeros((n, h), dtype=torch.bfloat16, device="cuda")
    w = normal((h,), "bf16")
    last = normal((6, h), "bf16", seed=4)
    x[-6:] = last
    out = H.rms_norm(x, w)
    check_out(out[-6:], last, w)
    assert (out[:-6] == 0).all()
    del out
    codes, scales = H.rms_norm_fp8(x, w)
    want, s = quantized(formula(last, w, 0.0)[0].float())
    assert torch.equal(scales[-6:].cpu(), s) and torch.equal(codes[-6:].cpu().view(torch.uint8), want)
    del codes, scales
    gx, gw = H.rms_norm_backward(x, x, w)
    check_grads(gx[-6:], gw, last, last, w)
    assert (gx[:-6] == 0).all()


def test_refusals():
    x, w = normal((4, 64), "bf16"), normal((64,), "bf16")
    for a, kw in (((x.half(), w), {}), ((x, w.half()), {}), ((x, w[:63]), {}), ((x, w.view(1, 64)), {}), ((x, w.cpu()), {}),
                  ((x.cpu(), w), {}), ((x, w), dict(residual=x[:3])), ((x, w), dict(residual=x.float())),
                  ((x, w), dict(eps=-1.0)), ((x, w), dict(weight_offset=float("nan"))), ((x[0, 0], w), {})):
        for f in (H.rms_norm, H.rms_norm_fp8):
            with pytest.raises(H.OrdaError):
                f(*a, **kw)
    for a, kw in (((x[:3], x, w), {}), ((x.float(), x, w), {}), ((None, x, w), {}), ((x, x, w), dict(grad_total=x[:2])),
                  ((x, x, w[:60]), {}), ((x.cpu(), x, w), {})):
        with pytest.raises(H.OrdaError):
            H.rms_norm_backward(*a, **kw)


@pytest.mark.parametrize("n", [20, 3000])
def test_a_second_backward_and_one_that_wants_less(n):
    """Small and large backward calls, of which the first has its gradients' memory made by the forward."""
    h = 1024
    x, w = normal((n, h), "f32").requires_grad_(True), normal((h,), "f32", mean=1.0).requires_grad_(True)
    g, g2 = normal((n, h), "f32", seed=2), normal((n, h), "f32", seed=3)
    out = rms_norm_autograd(x, w)
    first = torch.autograd.grad(out, [x, w], g, retain_graph=True)
    kept = [t.clone() for t in first]
    second = torch.autograd.grad(out, [x, w], g2, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, kept))
    check_grads(*second, g2, x.detach(), w.detach())
    (gx,) = torch.autograd.grad(out, [x], g, retain_graph=True)
    assert torch.equal(gx, first[0])
    (gw,) = torch.autograd.grad(out, [w], g)
    assert torch.equal(gw, first[1])


@pytest.mark.parametrize("n", [5, 1500, 5000])   # (the last is over the bytes up to which grad_x is made ready)
def test_tensors_that_move_between_forward_and_backward(n):
    """Saved tensors kept on the host meanwhile, and a weight whose memory is exchanged, as
    sharded training does it: the gradients of those that the backward is given."""
    x, r, w = (normal(s, "f32", seed=i) for i, s in enumerate([(n, 1000), (n, 1000), (1000,)]))
    g = normal((n, 1000), "f32", seed=3)
    want_x, want_w = H.rms_norm_backward(g, x + r, w)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    with torch.autograd.graph.save_on_cpu():
        out, _ = rms_norm_autograd(a, b, residual=r)
    out.backward(g)
    assert torch.equal(a.grad, want_x) and torch.equal(b.grad, want_w)
    a.grad = b.grad = None
    out, _ = rms_norm_autograd(a, b, residual=r)
    old, b.data = b.data, b.data.clone()
    old.fill_(float("nan"))
    out.backward(g)
    assert torch.equal(a.grad, want_x) and torch.equal(b.grad, want_w)


def test_nothing_but_the_saved_tensors_is_held():
    """A forward whose saved tensors are put elsewhere leaves no rows behind."""
    x, w = normal((4096, 2048), "f32").requires_grad_(True), normal((2048,), "f32").requires_grad_(True)
    r = normal((4096, 2048), "f32", seed=1)
    rms_norm_autograd(x, w, residual=r)[0].sum().backward()   # (what torch allocates once)
    x.grad = w.grad = None
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.save_on_cpu():
        out = rms_norm_autograd(x, w, residual=r)[0]
    assert torch.cuda.memory_allocated() - before <= out.numel() * 4 + (1 << 20)


@pytest.mark.parametrize("kw", [dict(eps="1e-6"), dict(eps=None), dict(weight_offset=[1.0])], ids=str)
def test_options_that_are_no_numbers(kw):
    x, w = normal((3, 8), "f32"), normal((8,), "f32")
    for call in (H.rms_norm, H.rms_norm_fp8, rms_norm_autograd, lambda x, w, **kw: H.rms_norm_backward(x, x, w, **kw)):
        with pytest.raises(H.OrdaError, match="numbers"):
            call(x, w, **kw)


def test_autograd_of_unusual_calls():
    """Shapes, strides and uses beside the usual ones, against torch's gradients in 64 bits. Both gradients are sums
    of at most 100 terms of magnitude 30 or less: 1e-4 is 500 roundings of fp32 of them."""
    def check(x, w, r=None, offset=0.0, both=False):
        own = [None if a is None else a.detach().requires_grad_(True) for a in (x, w, r)]
        ref = [None if a is None else a.detach().double().requires_grad_(True) for a in (x, w, r)]
        y = rms_norm_autograd(own[0], own[1], residual=own[2], weight_offset=offset, eps=EPS)
        y, t = y if r is not None else (y, None)
        t64 = ref[0] if r is None else ref[0] + ref[2]
        y64 = t64 * (t64.square().mean(-1, keepdim=True) + EPS).rsqrt() * (ref[1] + offset)
        g = torch.linspace(-1, 1, y.numel(), device="cuda").reshape(y.shape)
        ((y * g).sum() + ((t * g).sum() if both else 0)).backward()
        ((y64 * g.double()).sum() + ((t64 * g.double()).sum() if both else 0)).backward()
        for a, b in zip(own, ref):
            assert a is None or (a.grad.shape == a.shape and ((a.grad.double() - b.grad).abs() <= 1e-4).all())

    def rnd(*shape):
        return normal(shape, "f32")
    check(rnd(0, 8), rnd(8))
    check(rnd(8), rnd(8), rnd(8), 1.0, True)
    check(rnd(2, 3, 4, 16), rnd(16), rnd(2, 3, 4, 16), 0.0, True)
    check(rnd(3, 1), rnd(1))
    check(rnd(16, 5).t(), rnd(16))
    check(rnd(6, 20)[:, 3:17], rnd(28)[::2], rnd(6, 21)[:, 1:15], 1.0, True)
    # one tensor in both places, and a broadcast one
    x, w = rnd(5, 33).requires_grad_(True), rnd(33).requires_grad_(True)
    y, t = rms_norm_autograd(x, w, residual=x)
    gx = torch.autograd.grad(y.sum() + t.sum(), x)[0]
    alone = torch.autograd.grad(sum(o.sum() for o in rms_norm_autograd(x, w, residual=x.detach())), x)[0]
    assert torch.equal(gx, 2 * alone)
    row = rnd(1, 33).requires_grad_(True)
    rms_norm_autograd(row.expand(7, 33), w).sum().backward()
    assert row.grad.shape == (1, 33)
    # the sum alone is used; a part of the gradients is asked for
    r = rnd(5, 33).requires_grad_(True)
    _, t = rms_norm_autograd(x, w, residual=r)
    gx, gr, gw = torch.autograd.grad(t.sum(), [x, r, w])
    assert (gx == 1).all() and (gr == 1).all() and (gw == 0).all()
    y = rms_norm_autograd(x, w)
    part = torch.autograd.grad(y.sum(), [w], retain_graph=True)[0]
    assert torch.equal(part, torch.autograd.grad(y.sum(), [x, w])[1])
    # recomputed in the backward
    want = torch.autograd.grad(rms_norm_autograd(x, w).tanh().sum(), [x, w])
    for reentrant in (True, False):
        x.grad = w.grad = None
        torch.utils.checkpoint.checkpoint(lambda x: rms_norm_autograd(x, w).tanh(), x, use_reentrant=reentrant).sum().backward()
        assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])
