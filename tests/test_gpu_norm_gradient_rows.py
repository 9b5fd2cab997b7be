"""The norm's gradients of long rows, of which a workgroup has several: bf16 rows of 8193 to 16384
columns, whose next row is under way while one is summed up, and longer ones (fp32 from 8193 on)
in bands of rows, the last of which may be shorter."""
import pytest
import torch

import orda_hip as H
from test_gpu_rms_norm import EPS, check_grads, normal

pytestmark = pytest.mark.gpu


# bf16 up to 16384 columns: one to three rows a workgroup; 20000: bands of 3 rows, the last of 1; 33000: of 9, of 5
@pytest.mark.parametrize("dtype, weight", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("n, h", [(260, 16384), (520, 8200), (300, 10001), (515, 16383), (250, 20000), (300, 16391), (500, 33000)])
def test_gradients_of_several_long_rows(n, h, dtype, weight):
    t, w, g = normal((n, h), dtype, std=2.0), normal((h,), weight, std=0.2), normal((n, h), dtype, seed=2, std=0.1)
    gt = normal((n, h), dtype, seed=3, std=0.1)
    gx, gw = H.rms_norm_backward(g, t, w, grad_total=gt, eps=EPS, weight_offset=1.0)
    check_grads(gx, gw, g, t, w, gt, 1.0)
    gx, none = H.rms_norm_backward(g, t, w, eps=EPS, grad_weight=False)
    assert none is None
    check_grads(gx, None, g, t, w)
    again = H.rms_norm_backward(g, t, w, eps=EPS)
    assert torch.equal(again[0], gx)
    check_grads(None, again[1], g, t, w)
