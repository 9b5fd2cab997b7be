"""Limits of zero and without end, with norms of zero and without end."""
import math

import pytest
import torch

import orda_hip as H

pytestmark = pytest.mark.gpu
INF = math.inf


def clipped(values, limit, eps, dtype):
    g = torch.zeros(5000, dtype=dtype, device="cuda")
    g[100:100 + len(values)] = torch.tensor(values)
    h = torch.ones(33, 7, dtype=dtype, device="cuda") if any(values) else torch.zeros(33, 7, dtype=dtype, device="cuda")
    old = [g.clone(), h.clone()]
    out = [torch.full_like(g, 5.0), torch.full_like(h, 5.0)]
    norm = H.clip_gradients([g, h], limit, eps=eps, out=out)
    assert torch.equal(torch.stack([norm, H.clip_gradients([g, h], limit, eps=eps)]).isnan(), norm.isnan().expand(2))
    for a, b in zip((g, h), out):
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0))
    return float(norm), (g, h), old


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_limits(dtype):
    for limit, eps in ((INF, 0.0), (INF, 1e-6)):   # none: whatever the norm, but for a NaN
        for values in ([], [3.0, -4.0], [INF, 1.0], [-INF]):
            norm, got, old = clipped(values, limit, eps, dtype)
            assert all(torch.equal(a, b) for a, b in zip(got, old)) and (norm == INF) == any(map(math.isinf, values))
        norm, got, _ = clipped([1.0, math.nan], limit, eps, dtype)
        assert math.isnan(norm) and all(a.isnan().all() for a in got)
    for limit in (0.0, 1.0):   # zeros stay zeros
        for eps in (0.0, 1e-6):
            norm, got, _ = clipped([], limit, eps, dtype)
            assert norm == 0 and all((a == 0).all() for a in got)
    for eps in (0.0, 1e-6):
        norm, got, _ = clipped([3.0], 0.0, eps, dtype)
        assert norm > 0 and all((a == 0).all() for a in got)
        norm, got, old = clipped([INF, 2.0], 1.0, eps, dtype)
        assert norm == INF and got[0][100].isnan() and (got[0][101:] == 0).all() and (got[1] == 0).all()
