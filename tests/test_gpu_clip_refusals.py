"""Refused calls of the clipping leave gradients and destinations as they were."""
import pytest
import torch

import orda_hip as H

pytestmark = pytest.mark.gpu


def test_a_refused_call_writes_nothing():
    # (over its limit: a call that went through would scale it)
    g = torch.linspace(1, 2, 64 * 32, device="cuda").view(64, 32)
    o, want_grad = torch.full_like(g, 7.0), torch.full_like(g, 7.0).requires_grad_(True)
    kept = [(t, t.detach().clone()) for t in (g, o, want_grad)]
    for grads, kw in (([g, g], {}), ([g, g[3]], {}), ([g, g.half()], {}), ([g, g.cpu()], {}), ([g], dict(max_norm=-1.0)),
                      ([g], dict(max_norm=float("nan"))), ([g], dict(max_norm="1")), ([g], dict(eps=-1.0)), ([g], dict(eps="0")),
                      ([g, g[:, ::2]], {}), ([g, g[:1].expand(64, 32)], {}), ([g], dict(out=[g])), ([g], dict(out=[o.t()])),
                      ([g], dict(out=[o[:32]])), ([g], dict(out=[o.half()])), ([g], dict(out=[o, o])), ([g, None], dict(out=[o, o])),
                      ([g, g.clone()], dict(out=[o, o])), ([g, g.clone()], dict(out=[o, g])), ([g], dict(out=[want_grad])),
                      ([g, g.clone()], dict(out=[o, o.cpu()]))):
        with pytest.raises(H.OrdaError):
            H.clip_gradients(grads, kw.pop("max_norm", 1.0), **kw)
        torch.cuda.synchronize()
        assert all(torch.equal(t, old) for t, old in kept), (grads, kw)


def test_parameters_in_their_gradients_place_are_refused():
    p = torch.nn.Parameter(torch.linspace(1, 2, 300, device="cuda").view(20, 15))
    q = torch.ones(7, device="cuda")
    old = p.detach().clone()
    for grads in ([p], [q, p], [q, p.detach().t()[3:], p]):
        with pytest.raises(H.OrdaError, match="leaf that requires"):
            H.clip_gradients(grads, 0.5)
    torch.cuda.synchronize()
    assert torch.equal(p.detach(), old) and (q == 1).all()
    # read alone, without recording, or a gradient with a history of its own
    norm = float(H.gradient_norm([p, q]))
    out = [torch.empty_like(old)]
    H.clip_gradients([p], norm / 2, out=out)
    with torch.no_grad():
        H.clip_gradients([p], norm / 2)
    assert torch.equal(p.detach(), out[0]) and not torch.equal(out[0], old)
    g = p * 2
    want = [torch.empty_like(old)]
    H.clip_gradients([g], 1.0, out=want)
    H.clip_gradients([g], 1.0)
    assert torch.equal(g.detach(), want[0])
