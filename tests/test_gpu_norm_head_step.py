"""The norm, the clipping and the drawing of tokens in runs, as the steps around a head
use them: serving (norm in e4m3, the head's product, tokens) and training (lookup, norm,
linear cross entropy, gradients, clipping). Each operator's values are tested against
float64 where it stands alone; here what one gives the next is checked on the way."""
import threading

import pytest
import torch

import orda_hip as H
from linear_ce_reference import Exact
from orda_hip.autograd import embedding_autograd, linear_cross_entropy_autograd, rms_norm_autograd
from test_gpu_clip import check_norm, check_scaled, norm_of
from test_gpu_sampling import reference

pytestmark = pytest.mark.gpu
SCALE = 8.0   # a power of two: no rounding of its own
U = 2.0 ** -24


def normal(shape, seed, std, dtype, mean=0.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std + mean).to(dtype).cuda()


def widened(codes, scales):
    """The values of codes with a scale for each 128 columns, float64."""
    return codes.double().cpu() * scales.double().cpu().repeat_interleave(128, -1)[..., :codes.size(-1)]


def serving(dtype, n, h, v):
    head = H.quantize_fp8_blocks(normal((v, h), 1, 0.08, torch.bfloat16), block_rows=128)
    return (normal((n, h), 2, 1.0, dtype), normal((n, h), 3, 2.0, dtype), normal((h,), 4, 0.2, dtype), head,
            torch.rand(n, generator=torch.Generator().manual_seed(5)).cuda(),
            (0.5 + torch.rand(n, generator=torch.Generator().manual_seed(6))).cuda())


def serve(p, **filters):
    x, r, w, head, u, t = p
    codes, scales, total = H.rms_norm_fp8(x, w, residual=r, weight_offset=1.0)
    logits = H.fp8_block_matmul(codes, scales, *head, out_dtype=torch.float32)
    return codes, scales, total, logits, *H.sample_tokens(logits, u, temperature=t, **filters)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, h, v", [(1, 512, 4000), (5, 300, 1111), (130, 512, 2050)])
def test_a_serving_step(n, h, v, dtype):
    p = serving(dtype, n, h, v)
    x, r, w, head, u, t = p
    filters = dict(top_k=40, top_p=0.9, min_p=0.01)
    codes, scales, total, logits, tokens, logprobs = serve(p, **filters)
    assert torch.equal(total, (x.float() + r.float()).to(dtype))
    # half a step of e4m3 (2^-4, or 2^-10 of the scale below its normal range) and six roundings of fp32
    a, t64 = widened(codes, scales), total.double().cpu()
    value = t64 * (t64.square().mean(1, keepdim=True) + 1e-6).rsqrt() * (w.double().cpu() + 1.0)
    small = scales.double().cpu().repeat_interleave(128, 1)[:, :h] * 2.0 ** -10
    assert ((a - value).abs() <= 1.001 * torch.maximum(value.abs() * 2.0 ** -4, small) + 6 * U * value.abs()).all()
    # the product of what the norm gave: sums of h terms in fp32, scaled by block
    b_codes, b_scales = head
    b = b_codes.double().cpu() * b_scales.double().cpu().repeat_interleave(128, 0)[:v].repeat_interleave(128, 1)[:, :h]
    exact, bound = a @ b.t(), a.abs() @ b.abs().t()
    assert ((logits.double().cpu() - exact).abs() <= (h + 8) * U * bound).all()
    # the tokens of those logits
    for i in range(n):
        token, logp = reference(logits[i].double().cpu().numpy(), float(u[i]), float(t[i]), 40, 0.9, 0.01)
        assert int(tokens[i]) == token
        assert abs(float(logprobs[i]) - logp) <= U * abs(logp) + 1e-11


def tied(dtype, n=150, v=700, h=64):
    """ids, labels (some ignored, some tokens repeated), weight, body, the norm's weight."""
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, v, (n,), generator=g).cuda()
    ids[n - n // 2:] = ids[: n // 2]
    labels = torch.randint(0, v, (n,), generator=g)
    labels[::7] = -100
    return ids, labels.cuda(), normal((v, h), 4, 0.1, dtype), normal((h, h), 5, 0.1, dtype), normal((h,), 6, 0.1, dtype)


def forward(ids, labels, w, b, g):
    x = embedding_autograd(ids, w, scale=SCALE)
    y, total = rms_norm_autograd(torch.tanh(x @ b), g, residual=x, weight_offset=1.0)
    nll, lse = linear_cross_entropy_autograd(y, w, labels)
    loss = nll.sum() / (labels != -100).sum() + 1e-4 * (lse ** 2).sum() + 1e-3 * total.float().square().mean()
    return x, y, total, nll, lse, loss


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_training_step(dtype):
    ids, labels, *leaves = tied(dtype)
    w, b, g = (t.clone().requires_grad_(True) for t in leaves)
    x, y, total, nll, lse, loss = forward(ids, labels, w, b, g)
    for t in (y, total):
        t.retain_grad()
    Exact(y.detach(), leaves[0], labels).check_losses(nll.detach(), lse.detach())
    loss.backward()
    # the norm's gradients from those that came to it
    gx, gg = H.rms_norm_backward(y.grad, total.detach(), leaves[2], grad_total=total.grad, weight_offset=1.0)
    assert torch.equal(g.grad, gg)
    d = torch.tanh(x.detach() @ leaves[1])
    if dtype == torch.float32:
        # tanh' and a product of 150 terms: 2^-24 each
        back = gx * (1 - d * d)
        want = x.detach().double().t().cpu() @ back.double().cpu()
        bound = x.detach().double().abs().t().cpu() @ back.double().abs().cpu()
        assert ((b.grad.double().cpu() - want).abs() <= 160 * U * bound).all()
    # clipped, in place, as the optimizer reads them
    grads = [w.grad, b.grad, g.grad]
    old = [t.clone() for t in grads]
    norm = norm_of(old)
    check_norm(H.clip_gradients([w.grad, None, b.grad, g.grad], 0.25 * norm), norm)
    for new, t in zip(grads, old):
        check_scaled(new, t, norm, 0.25 * norm)


def test_the_loss_falls_by_its_gradient():
    """The directional derivative of the run's loss, in float64 on the host, against the gradients (fp32). The
    step of 1e-5 makes the central difference off by 1e-10 relative of the third derivative and 1e-11 / 1e-5 of
    rounding; the products' 6 * (64 + 2) * 2^-24 * sum |y||w| <= 2.4e-5 * (8 * 1.5) * 1.5 = 4.3e-4 in a logit, thus
    9e-4 of each probability: 1e-2 of the magnitudes that the derivative sums."""
    ids, labels, *leaves = tied(torch.float32)
    params = [t.clone().requires_grad_(True) for t in leaves]
    forward(ids, labels, *params)[-1].backward()
    i, y, keep = ids.cpu(), labels.cpu(), (labels != -100).cpu()

    def loss(w, b, g):
        x = SCALE * w[i]
        t = torch.tanh(x @ b) + x
        n = t * (t.square().mean(1, keepdim=True) + 1e-6).rsqrt() * (g + 1.0)
        z = (n @ w.t())[keep]
        return (torch.nn.functional.cross_entropy(z, y[keep]) + 1e-4 * (torch.logsumexp(z, 1) ** 2).sum()
                + 1e-3 * t.square().mean())

    at = [t.double().cpu() for t in leaves]
    grads = [p.grad.double().cpu() for p in params]
    for k in range(3):
        step = [torch.zeros_like(t) for t in at]
        step[k] = grads[k] / grads[k].norm()
        e = 1e-5
        slope = float(loss(*(t + e * s for t, s in zip(at, step))) - loss(*(t - e * s for t, s in zip(at, step)))) / (2 * e)
        got = float((grads[k] * step[k]).sum())
        assert abs(got - slope) <= 1e-2 * float((grads[k].abs() * step[k].abs()).sum()), (k, got, slope)


def bits(t):
    return t.contiguous().reshape(-1).view(torch.uint8)


def captured(step):
    """(a graph of the step, what it gives)."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = step()
    torch.cuda.current_stream().wait_stream(s)
    return graph, got


@pytest.mark.parametrize("filters", [dict(top_k=40, top_p=0.9), dict(top_p=0.95), dict()], ids=str)
def test_a_serving_step_captured(filters):
    """One graph, its inputs changed between replays, with eager steps in between."""
    p = serving(torch.bfloat16, 3, 512, 4000)
    graph, got = captured(lambda: serve(p, **filters))
    for k in range(4):
        for t, seed in ((p[0], 20), (p[1], 30)):
            t.copy_(normal(t.shape, seed + k, 1.0 + k, torch.bfloat16))
        p[4].copy_(torch.rand(3, generator=torch.Generator().manual_seed(40 + k)))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, serve(p, **filters)):
            assert torch.equal(bits(a), bits(b))


def gradients(p, max_norm=0.05):
    """A step's gradients without autograd, clipped."""
    ids, labels, w, b, g = p
    x = H.embedding(ids, w, scale=SCALE)
    y, total = H.rms_norm(x, g, residual=x, weight_offset=1.0)
    nll, lse = H.linear_cross_entropy(y, w, labels)
    gy, gw = H.linear_cross_entropy_backward(y, w, labels, lse, torch.ones_like(nll), 1e-3 * lse)
    gt, gg = H.rms_norm_backward(gy, total, g, weight_offset=1.0)
    H.embedding_backward(gt, ids, w.size(0), scale=SCALE, out=gw, accumulate=True)
    return H.clip_gradients([gw, gg], max_norm), gw, gg


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_captured(dtype):
    p = tied(dtype)
    graph, got = captured(lambda: gradients(p))
    for k in range(4):
        p[0].copy_((p[0] * 7 + k) % 700)
        p[2].copy_(normal(p[2].shape, 50 + k, 0.1, dtype))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, gradients(p)):
            assert torch.equal(a, b)


def test_calls_on_two_streams_at_once():
    """Each call's scratch is its own: interleaved on two streams, the results of one after the other."""
    a = (serving(torch.bfloat16, 40, 512, 4000), tied(torch.bfloat16, n=700, v=3000, h=256))
    b = (serving(torch.float32, 7, 300, 1111), tied(torch.float32))
    want = [(*serve(p, top_p=0.95), *gradients(q)) for p, q in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(6):
        for s, (p, q) in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append((*serve(p, top_p=0.95), *gradients(q)))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(bits(x), bits(y)) for x, y in zip(out, want[i % 2]))


def test_threads_at_once():
    """Calls of several threads, each on a stream of its own, refused ones (with their own messages) among them."""
    errors = []

    def work(seed):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                x, w = normal((300, 700), seed, 1.0, torch.float32), normal((700,), seed, 0.2, torch.float32)
                logits, u = normal((20, 5000), seed, 2.0, torch.float32), torch.full((20,), 0.37, device="cuda")
                first = None
                for _ in range(20):
                    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
                    rms_norm_autograd(a, b)[0].square().sum().backward()
                    tokens, logprobs = H.sample_tokens(logits, u, top_p=0.9)
                    grads = [a.grad.clone(), b.grad.clone()]
                    now = [a.grad, b.grad, tokens, logprobs, H.clip_gradients(grads, 0.5), *grads]
                    with pytest.raises(H.OrdaError, match="weight must be"):
                        H.rms_norm(x, w[:5])
                    with pytest.raises(H.OrdaError, match="temperature must be"):
                        H.sample_tokens(logits, u, temperature=-1.0)
                    with pytest.raises(H.OrdaError, match="eps must be"):
                        H.rms_norm(x, w, eps=-1.0)
                    first = first or now
                    assert all(torch.equal(p, q) for p, q in zip(first, now))
        except BaseException as e:   # (pytest sees the main thread's alone)
            errors.append(repr(e))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
