"""The norm's step, drawn tokens and clipping from several threads at once, each on a stream of its own, against
what the same inputs gave before the threads began."""
import threading

import pytest
import torch

import orda_hip as H
from orda_hip.autograd import rms_norm_autograd

pytestmark = pytest.mark.gpu


def normal(shape, seed, std):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).cuda()


def inputs(seed):
    n = 100 + 50 * seed   # (sizes of their own: a scratch of another thread's call would show)
    return (normal((n, 700), seed, 1.0), normal((700,), seed + 10, 0.2), normal((20 + seed, 5000), seed + 20, 2.0),
            torch.rand(20 + seed, generator=torch.Generator().manual_seed(seed)).cuda())


def step(x, w, logits, u):
    a, b, r = (t.clone().requires_grad_(True) for t in (x, w, x))
    out, total = rms_norm_autograd(a, b, residual=r)
    assert out.shape == x.shape
    (out.square().sum() + total.sum()).backward()
    grads = [a.grad.clone(), b.grad.clone()]
    return [out.detach(), total.detach(), a.grad, b.grad, r.grad, *H.sample_tokens(logits, u, top_p=0.9),
            *H.sample_tokens(logits, u, top_k=3000, top_p=0.9), H.clip_gradients(grads, 0.5), *grads]


def test_threads_give_what_one_thread_gives():
    data = [inputs(seed) for seed in range(4)]
    want = [[t.clone() for t in step(*d)] for d in data]
    assert all((w[2] != 0).all(1).all() for w in want)   # every row has a gradient
    torch.cuda.synchronize()
    errors, start = [], threading.Barrier(4)

    def work(i):
        try:
            start.wait(30)
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(25):
                    got = step(*data[i])
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
                    with pytest.raises(H.OrdaError, match="weight must be"):
                        H.rms_norm(data[i][0], data[i][1][:5])
                    with pytest.raises(H.OrdaError, match="temperature must be"):
                        H.sample_tokens(*data[i][2:], temperature=-1.0)
        except BaseException as e:   # (pytest sees the main thread's alone)
            errors.append((i, repr(e)))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
