"""The norm's backward on what saved tensors' hooks give back: its values where they are the saved ones, whatever
their place, and an error, not a read past them, where they are of another type, size or place."""
import pytest
import torch

import orda_hip as H
from orda_hip.autograd import rms_norm_autograd

pytestmark = pytest.mark.gpu


def gradients(unpack, n=300, h=1500, residual=True):
    gen = torch.Generator().manual_seed(1)
    x, r, w, g = (torch.randn(s, generator=gen).cuda() for s in ((n, h), (n, h), (h,), (n, h)))
    r = r if residual else None
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        out = rms_norm_autograd(a, b, residual=r)
    out = out[0] if residual else out
    return torch.autograd.grad(out, [a, b], g), H.rms_norm_backward(g, x + r if residual else x, w)


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("unpack", [lambda t: t.clone(), lambda t: t.t().contiguous().t(), lambda t: torch.stack([t, t], -1)[..., 0]],
                         ids=["a copy", "columns", "apart"])
def test_the_same_values_elsewhere(unpack, residual):
    got, want = gradients(unpack, residual=residual)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("unpack", [
    lambda t: t.bfloat16(), lambda t: t.bfloat16() if t.dim() == 2 else t, lambda t: t[:1], lambda t: t[..., :8],
    lambda t: t.cpu(), lambda t: t if t.dim() == 2 else t[:8], lambda t: t.double(), lambda t: t.to_sparse(),
    lambda t: t[:, :700].reshape(700, 300).contiguous() if t.dim() == 2 else t], ids=range(9))
def test_other_values_are_refused(unpack):
    with pytest.raises((H.OrdaError, RuntimeError)):
        gradients(unpack)
