"""The operators in a run, as a tied student trained beside a teacher whose head is
held in 8 bits uses them: lookup, body, teacher's logits, distillation loss and
linear cross entropy of the same hidden rows, and one weight that the head's and the
lookup's gradients meet in. Each operator's values are tested against float64 where
it stands alone; here the run's results must be, bit for bit, those of its parts on
the same tensors."""
import pytest
import torch

import orda_hip as H
from linear_ce_reference import Exact
from orda_hip.autograd import distillation_loss_autograd, embedding_autograd, linear_cross_entropy_autograd

pytestmark = pytest.mark.gpu
SCALE = 8.0   # a power of two: no rounding of its own


def normal(shape, seed, std, dtype):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def parts(dtype, n=150, v=700, h=64, ht=320):
    """ids, labels (some ignored, some tokens repeated), weight, body, teacher's rows and its head in e4m3."""
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, v, (n,), generator=g).cuda()
    ids[n - n // 2:] = ids[: n // 2]
    labels = torch.randint(0, v, (n,), generator=g)
    labels[::7] = -100
    head = H.quantize_fp8_blocks(normal((v, ht), 6, 0.1, dtype), block_rows=128)
    return (ids, labels.cuda(), normal((v, h), 4, 0.1, dtype), normal((h, h), 5, 0.1, dtype),
            normal((n, ht), 7, 1.0, dtype), head)


def teacher_logits(rows, head):
    return H.fp8_block_matmul(*H.quantize_fp8_blocks(rows), *head, out_dtype=torch.float32)


def sums(a, b, c):
    """a + b + c in each order that a leaf may be added to."""
    return [(a + b) + c, (a + c) + b, (b + c) + a]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_tied_step(dtype):
    ids, labels, weight, body, rows, head = parts(dtype)
    opts = H.LossOptions(student_ce_weight=0.0, kd_weight=0.5, temperature=2.0)
    w, b = weight.clone().requires_grad_(True), body.clone().requires_grad_(True)
    x = embedding_autograd(ids, w, scale=SCALE, padding_idx=0)
    hidden = torch.tanh(x @ b)
    hidden.retain_grad()
    x.retain_grad()
    logits = teacher_logits(rows, head)
    kd, _ = distillation_loss_autograd(hidden, w, labels, H.Teacher.Precomputed(logits), opts)
    nll, lse = linear_cross_entropy_autograd(hidden, w, labels, label_smoothing=0.1)
    Exact(hidden.detach(), weight, labels, label_smoothing=0.1).check_losses(nll.detach(), lse.detach())
    count = (labels != -100).sum()
    loss = kd + nll.sum() / count + 1e-4 * (lse ** 2).sum()
    loss.backward()
    # the same from the parts
    d = hidden.detach()
    out = H.distillation_loss(d, weight, labels, H.Teacher.Precomputed(logits), opts)
    assert kd.item() == out.loss
    kd_h, kd_w = out.grad_student_hidden.to(dtype), out.grad_weight.to(dtype)
    g_nll = torch.ones_like(nll) / count
    g_lse = 1e-4 * (2 * lse.detach())
    ce_h, ce_w = H.linear_cross_entropy_backward(d, weight, labels, lse.detach(), g_nll, g_lse, label_smoothing=0.1)
    assert torch.equal(hidden.grad, kd_h + ce_h)
    em_w = H.embedding_backward(x.grad, ids, weight.size(0), scale=SCALE, padding_idx=0)
    assert any(torch.equal(w.grad, s) for s in sums(kd_w, ce_w, em_w))
    # added in place, as a step without autograd does it
    both = (kd_w + ce_w).clone()
    H.embedding_backward(x.grad, ids, weight.size(0), scale=SCALE, padding_idx=0, out=both, accumulate=True)
    if dtype == torch.float32:
        assert torch.equal(both, (kd_w + ce_w) + em_w)
    untouched = torch.ones(weight.size(0), dtype=torch.bool, device="cuda")
    untouched[ids[ids != 0]] = False
    assert torch.equal(both[untouched], (kd_w + ce_w)[untouched])


def test_the_loss_falls_by_its_gradient():
    """The directional derivative of the run's loss, in float64 on the host from the run's own formulas, against
    the gradient the run gives (fp32). The reference's step is 1e-5 of the weight: its central difference is off
    by 1e-10 relative of the third derivative and 1e-11 / 1e-5 of rounding; the gradient by the products'
    6 * (64 + 2) * 2^-24 * sum |h||w| <= 2.4e-5 * 64 * 1 * 0.5 = 8e-4 in a logit, thus 2e-3 of each probability:
    1e-2 of the magnitudes that the derivative sums."""
    ids, labels, weight, body, rows, head = parts(torch.float32)
    w = weight.clone().requires_grad_(True)
    x = embedding_autograd(ids, w, scale=SCALE)
    hidden = torch.tanh(x @ body)
    logits = teacher_logits(rows, head)
    opts = H.LossOptions(student_ce_weight=0.0, kd_weight=0.5, temperature=2.0)
    kd, _ = distillation_loss_autograd(hidden, w, labels, H.Teacher.Precomputed(logits), opts)
    nll, lse = linear_cross_entropy_autograd(hidden, w, labels)
    keep = (labels != -100).cpu()
    (kd + nll.sum() / keep.sum().item() + 1e-4 * (lse ** 2).sum()).backward()

    i, y, t, bd = ids.cpu(), labels.cpu(), logits.double().cpu(), body.double().cpu()

    def loss(wt):
        z = torch.tanh(SCALE * wt[i] @ bd) @ wt.t()
        z, y1, q = z[keep], y[keep], t[keep]
        ce = torch.nn.functional.cross_entropy(z, y1)
        ls, lt = torch.log_softmax(z / 2, 1), torch.log_softmax(q / 2, 1)
        kl = (lt.exp() * (lt - ls)).sum(1).mean() * 4
        return 0.5 * kl + ce + 1e-4 * (torch.logsumexp(z, 1) ** 2).sum()

    w64 = weight.double().cpu()
    direction = w.grad.double().cpu()
    direction /= direction.norm()
    e = 1e-5
    slope = float((loss(w64 + e * direction) - loss(w64 - e * direction)) / (2 * e))
    got = float((w.grad.double().cpu() * direction).sum())
    mags = float((w.grad.double().cpu().abs() * direction.abs()).sum())
    assert abs(got - slope) <= 1e-2 * mags, (got, slope)


def test_a_serving_step_captured():
    """Lookup, teacher's logits and the scored tokens in one graph, its inputs changed between replays."""
    ids, labels, weight, _, rows, head = parts(torch.bfloat16, n=3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())

    def step():
        x = H.embedding(ids, weight, scale=SCALE)
        nll, lse = H.linear_cross_entropy(x, weight, labels)
        return x, nll, lse, teacher_logits(rows, head)

    with torch.cuda.stream(s):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = step()
    torch.cuda.current_stream().wait_stream(s)
    for k in range(4):
        ids.copy_(torch.tensor([k, 5 * k, 699 - k]).cuda())
        labels.copy_(torch.tensor([k, -100, 3 * k + 1]).cuda())
        rows.copy_(normal(rows.shape, 20 + k, 1.0, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_calls_on_two_streams_at_once():
    """Each call's scratch is its own: interleaved on two streams, the results of one after the other."""
    a, b = parts(torch.bfloat16, n=700, v=3000, h=256), parts(torch.float32, n=90, v=900, h=64)

    def calls(p):
        ids, labels, weight, _, rows, head = p
        x = H.embedding(ids, weight, scale=SCALE)
        nll, lse = H.linear_cross_entropy(x, weight, labels)
        gh, gw = H.linear_cross_entropy_backward(x, weight, labels, lse, torch.ones_like(nll), lse)
        return x, nll, lse, gh, gw, H.embedding_backward(gh, ids, weight.size(0)), teacher_logits(rows, head)

    want = [calls(a), calls(b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(6):
        for s, p in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(calls(p))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(x, y) for x, y in zip(out, want[i % 2]))
