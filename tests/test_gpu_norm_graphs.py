"""The norm's autograd in captured graphs, and what it holds between forward and backward."""
import pytest
import torch

import orda_hip as H
from orda_hip.autograd import rms_norm_autograd

pytestmark = pytest.mark.gpu


def normal(shape, seed, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, h", [(1024, 1600), (300, 3000)])
def test_forwards_hold_nothing_but_the_saved_tensors(n, h, dtype):
    """16 norms of a few MB whose saved tensors are put elsewhere: of the device's memory they
    keep their results alone (each up to the allocator's 512 bytes)."""
    x, w = normal((n, h), 1, dtype=dtype).requires_grad_(True), normal((h,), 2, dtype=dtype).requires_grad_(True)
    r = normal((n, h), 3, dtype=dtype)
    rms_norm_autograd(x, w, residual=r)[0].sum().backward()   # (what torch allocates once)
    x.grad = w.grad = None
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.save_on_cpu():
        outs = [rms_norm_autograd(x, w, residual=r)[0] for _ in range(16)]
    assert torch.cuda.memory_allocated() - before <= 16 * (outs[0].numel() * outs[0].element_size() + 512) + (1 << 20)


def leaves(n, h, dtype):
    return [normal(s, i, dtype=dtype).requires_grad_(True) for i, s in enumerate([(n, h), (h,), (n, h)])]


def on_a_stream():
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    return s


def gradients(x, w, r, g, gt, **kw):
    out, t = rms_norm_autograd(x, w, residual=r, weight_offset=1.0)
    return (out, t, *torch.autograd.grad([out, t], [x, w, r], [g, gt], **kw))


def check(got, x, w, r, g, gt):
    x, w, r = x.detach(), w.detach(), r.detach()
    out, t = H.rms_norm(x, w, residual=r, weight_offset=1.0)
    gx, gw = H.rms_norm_backward(g, t, w, grad_total=gt, weight_offset=1.0)
    for a, b in zip(got, (out, t, gx, gw, gx)):
        assert torch.equal(a, b)


def change(k, *tensors):
    with torch.no_grad():
        for i, t in enumerate(tensors):
            t.copy_(normal(t.shape, 100 * k + i, 1.0 + k))


SIZES = [(1, 4096), (300, 1500), (1000, 1531), (40, 20000), (3000, 4096)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, h", SIZES)
def test_forward_and_backward_captured(n, h, dtype):
    x, w, r = leaves(n, h, dtype)
    g, gt = normal((n, h), 8, dtype=dtype), normal((n, h), 9, dtype=dtype)
    s = on_a_stream()
    with torch.cuda.stream(s):
        gradients(x, w, r, g, gt)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = gradients(x, w, r, g, gt)
    torch.cuda.current_stream().wait_stream(s)
    for k in range(4):
        change(k, x, w, r, g, gt)
        graph.replay()
        torch.cuda.synchronize()
        check([t.detach() for t in got], x, w, r, g, gt)


@pytest.mark.parametrize("earlier", [False, True], ids=["its first", "a later one"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, h", SIZES)
def test_a_backward_captured_alone(n, h, dtype, earlier):
    """The forward ran before; each replay takes new gradients into its results, and writes
    nothing but the graph's own memory: not what the stream has allocated since."""
    g, gt = normal((n, h), 8, dtype=dtype), normal((n, h), 9, dtype=dtype)
    s = on_a_stream()
    with torch.cuda.stream(s):
        gradients(*leaves(n, h, dtype), g, gt)   # (kernels are loaded)
        x, w, r = leaves(n, h, dtype)
        out, t = rms_norm_autograd(x, w, residual=r, weight_offset=1.0)

        def back():
            return torch.autograd.grad([out, t], [x, w, r], [g, gt], retain_graph=True)
        if earlier:
            back()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = back()
        size = x.numel() * x.element_size()
        others = [torch.full((b,), 77, dtype=torch.uint8, device="cuda")
                  for b in (size, size, size // 2, 4 * 256 * h, 4 * 256 * h, 4 * h, 2 * h, 4 * h, 2 * h) for _ in range(2)]
    torch.cuda.current_stream().wait_stream(s)
    for k in range(4):
        change(k, g, gt)
        graph.replay()
        torch.cuda.synchronize()
        check([out.detach(), t.detach(), *got], x, w, r, g, gt)
        assert all((o == 77).all() for o in others)
