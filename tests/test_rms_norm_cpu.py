"""The norm's refusals, without a GPU: the C entry points check their arguments
before any device call."""
import ctypes as C

import pytest
import torch

import orda_hip as H
from orda_hip import _lib as L


def mat(rows, cols, **kw):
    t = L.Tensor(data=256, rows=rows, cols=cols, dtype=L.BF16, location=L.DEVICE)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def args(**kw):
    a = dict(x=mat(4, 256), weight=mat(1, 256), eps=1e-6)
    a.update(kw)
    return L.RmsNormC(**a)


def codes(rows=4, cols=256, **kw):
    d = dict(codes=256, rows=rows, cols=cols, ld=cols, scales=256, scale_row=1, scale_col=rows, block_rows=1)
    d.update(kw)
    return L.Fp8MatrixC(**d)


ARGS = [(dict(x=mat(4, 256, dtype=L.I8)), "float32 or bfloat16"), (dict(x=mat(4, 256, location=L.HOST)), "device"),
        (dict(x=mat(4, 256, data=None)), "null"), (dict(x=mat(-4, 256)), "negative"), (dict(x=mat(4, 256, ld=255)), "ld < cols"),
        (dict(x=mat(4, 1 << 21), weight=mat(1, 1 << 21)), "at most"), (dict(weight=mat(1, 255)), "weight must be"),
        (dict(weight=mat(2, 256)), "weight must be"), (dict(weight=mat(1, 256, data=None)), "null"),
        (dict(residual=mat(4, 256, dtype=L.F32)), "dtype"), (dict(residual=mat(5, 256)), "residual must be"),
        (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(weight_offset=float("inf")), "weight_offset")]


@pytest.mark.parametrize("kw, message", ARGS + [
    (dict(total=mat(4, 255)), "total must be"), (dict(total=mat(4, 256, dtype=L.F32)), "dtype"),
    (dict(out=mat(3, 256)), "out must be"), (dict(out=mat(4, 256, dtype=L.F32)), "dtype"),
    (dict(out=mat(4, 256, data=None)), "null")])
def test_forward_refused(kw, message):
    kw = dict(kw)
    total, out = kw.pop("total", mat(4, 256)), kw.pop("out", mat(4, 256))
    err = C.create_string_buffer(512)
    rc = L.load().orda_rms_norm_forward(0, None, C.byref(args(**kw)), C.byref(total), C.byref(out), err, 512)
    assert rc == L.ORDA_ERR_INVALID and message in err.value.decode()


@pytest.mark.parametrize("kw, message", ARGS + [
    (dict(out=codes(block_rows=128)), "block_rows 1"), (dict(out=codes(cols=255)), "shape"), (dict(out=codes(ld=260)), "8"),
    (dict(out=codes(codes=260)), "8-byte"), (dict(out=codes(scales=None)), "null"), (dict(out=codes(scale_col=-1)), "strides")])
def test_fp8_refused(kw, message):
    kw = dict(kw)
    out = kw.pop("out", codes())
    err = C.create_string_buffer(512)
    rc = L.load().orda_rms_norm_fp8(0, None, C.byref(args(**kw)), None, C.byref(out), err, 512)
    assert rc == L.ORDA_ERR_INVALID and message in err.value.decode()


@pytest.mark.parametrize("kw, message", [c for c in ARGS if "residual" not in c[0]] + [
    (dict(residual=mat(4, 256)), "no residual"), (dict(g=mat(4, 255)), "grad_out must be"),
    (dict(g=mat(4, 256, dtype=L.F32)), "dtype"), (dict(gt=mat(3, 256)), "grad_total must be"),
    (dict(gx=mat(3, 256)), "grad_x must be"), (dict(gw=mat(1, 256, dtype=L.F32)), "dtype"), (dict(gw=mat(4, 256)), "grad_weight must be"),
    (dict(ws=264), "aligned"), (dict(ws_bytes=100), "workspace"), (dict(ws=None), "workspace")])
def test_backward_refused(kw, message):
    kw = dict(kw)
    g, gt, gx, gw = kw.pop("g", mat(4, 256)), kw.pop("gt", mat(4, 256)), kw.pop("gx", mat(4, 256)), kw.pop("gw", mat(1, 256))
    ws, ws_bytes = kw.pop("ws", 256), kw.pop("ws_bytes", 1 << 40)
    err = C.create_string_buffer(512)
    rc = L.load().orda_rms_norm_backward(0, None, C.byref(args(**kw)), C.byref(g), C.byref(gt), C.byref(gx), C.byref(gw), ws,
                                         ws_bytes, err, 512)
    assert rc == L.ORDA_ERR_INVALID and message in err.value.decode()


@pytest.mark.parametrize("n, h", [(0, 4096), (1, 1), (1, 4096), (8192, 4096), (1 << 30, 64), (100, 1 << 20), (1 << 20, 20000)])
def test_workspace_is_bounded(n, h):
    """At most 512 rows of fp32; long rows (more than 16384 columns): two values a row, and as many partial rows as
    give 1024 tiles of 2048 columns."""
    out, err = C.c_int64(), C.create_string_buffer(512)
    assert L.load().orda_rms_norm_backward_workspace(n, h, C.byref(out), err, 512) == L.ORDA_OK
    assert out.value % 256 == 0
    if h <= 16384:
        assert out.value <= min(n, 512) * h * 4 + 255
    else:
        assert out.value <= 8 * n + 256 + min(n, -(-1024 // -(-h // 2048))) * h * 4 + 255


def test_python_refuses_cpu_tensors():
    x, w = torch.zeros(3, 8), torch.zeros(8)
    for call in (lambda: H.rms_norm(x, w), lambda: H.rms_norm_fp8(x, w), lambda: H.rms_norm_backward(x, x, w)):
        with pytest.raises(H.OrdaError, match="GPU tensor"):
            call()
