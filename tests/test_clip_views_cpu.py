"""What the clipping takes a gradient's memory for, without a GPU: rows, columns and pitch
from sizes and strides alone, and no copy on the way."""
import pytest
import torch

import orda_hip as H
from orda_hip.operators import _view

FRAME = torch.empty(50, 400)


@pytest.fixture
def no_copies(monkeypatch):
    def copied(*args, **kw):
        raise AssertionError("a copy")
    for name in ("contiguous", "clone", "reshape", "to"):
        monkeypatch.setattr(torch.Tensor, name, copied)


@pytest.mark.parametrize("g, want", [
    (FRAME, (1, 20000, 20000)), (FRAME.t(), (1, 20000, 20000)), (FRAME[:, 3:200], (50, 197, 400)),
    (FRAME[:, 3:200].t(), (50, 197, 400)), (FRAME.t()[7:30], (50, 23, 400)), (FRAME[3:9], (1, 2400, 2400)),
    (FRAME[:1, ::2], (200, 1, 2)), (FRAME[:, :1], (50, 1, 400)), (FRAME[:0, ::2], (1, 0, 0)),
    (torch.empty(4, 6, 5, 3).to(memory_format=torch.channels_last), (1, 360, 360))])
def test_views(g, want, no_copies):
    assert _view(g, "g") == want


@pytest.mark.parametrize("g", [FRAME[:, ::2], FRAME[:1].expand(50, 400), FRAME.t()[::3], FRAME.view(5, 10, 400)[:, :, 3:9],
                               FRAME.as_strided((50, 400), (200, 1))])
def test_no_views(g, no_copies):
    with pytest.raises(H.OrdaError, match="dense"):
        _view(g, "g")
