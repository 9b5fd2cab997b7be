"""The e4m3 operators' refusals, without a GPU: the C entry points check their
arguments before any device call."""
import ctypes as C

import pytest
import torch

import orda_hip as H
from orda_hip import _lib as L


def mat(rows, cols, block_rows, **kw):
    d = dict(codes=256, rows=rows, cols=cols, ld=cols, scales=256, scale_row=-(-cols // 128), scale_col=1,
             block_rows=block_rows)
    d.update(kw)
    return L.Fp8MatrixC(**d)


def tensor(rows, cols, **kw):
    d = dict(data=256, rows=rows, cols=cols, dtype=L.BF16, location=L.DEVICE)
    d.update(kw)
    return L.Tensor(**d)


def matmul(a, b, out, ws=256, ws_bytes=1 << 40):
    err = C.create_string_buffer(512)
    rc = L.load().orda_fp8_block_matmul(0, None, C.byref(a), C.byref(b), C.byref(out), ws, ws_bytes, err, 512)
    return rc, err.value.decode()


@pytest.mark.parametrize("kw, message", [
    (dict(a=mat(4, 256, 128)), "block_rows 1"), (dict(b=mat(300, 256, 1)), "block_rows 128"),
    (dict(a=mat(4, 256, 2)), "1 or 128"), (dict(a=mat(4, 255, 1)), "columns"), (dict(a=mat(-4, 256, 1)), "negative"),
    (dict(a=mat(4, 256, 1, codes=None)), "null"), (dict(b=mat(300, 256, 128, scales=None)), "null"),
    (dict(a=mat(4, 256, 1, ld=255)), "pitch"), (dict(a=mat(4, 256, 1, ld=1 << 21)), "pitch"),
    (dict(a=mat(4, 256, 1, scale_row=-1)), "strides"), (dict(a=mat(4, 256, 1, scale_row=1 << 23)), "strides"),
    (dict(a=mat(4, 0, 1), b=mat(300, 0, 128)), "columns"),
    (dict(a=mat(4, 1 << 21, 1), b=mat(300, 1 << 21, 128)), "at most"),
    (dict(out=tensor(4, 299)), "out must be"), (dict(out=tensor(4, 300, dtype=L.I8)), "float32 or bfloat16"),
    (dict(out=tensor(4, 300, location=L.HOST)), "device"), (dict(ws=264), "aligned"),
    (dict(a=mat(4, 250, 1), b=mat(300, 250, 128), ws_bytes=100), "workspace"),
])
def test_product_refused(kw, message):
    d = dict(a=mat(4, 256, 1), b=mat(300, 256, 128), out=tensor(4, 300))
    d.update(kw)
    rc, err = matmul(**d)
    assert rc == L.ORDA_ERR_INVALID and message in err


@pytest.mark.parametrize("kw, message", [
    (dict(m=tensor(4, 256, dtype=L.I8)), "float32 or bfloat16"), (dict(m=tensor(4, 256, location=L.HOST)), "device"),
    (dict(out=mat(5, 256, 1)), "shape"), (dict(out=mat(4, 256, 3)), "1 or 128"), (dict(out=mat(4, 256, 1, ld=260)), "8"),
    (dict(out=mat(4, 256, 1, codes=260)), "8-byte"), (dict(m=tensor(4, 256, data=None)), "null"),
])
def test_quantiser_refused(kw, message):
    d = dict(m=tensor(4, 256), out=mat(4, 256, 1))
    d.update(kw)
    err = C.create_string_buffer(512)
    rc = L.load().orda_quant_fp8_blocks(0, None, C.byref(d["m"]), C.byref(d["out"]), err, 512)
    assert rc == L.ORDA_ERR_INVALID and message in err.value.decode()


def test_python_refuses_cpu_tensors():
    with pytest.raises(H.OrdaError, match="GPU tensor"):
        H.quantize_fp8_blocks(torch.zeros(4, 256))
    c = torch.zeros(4, 256).to(torch.float8_e4m3fn)
    with pytest.raises(H.OrdaError, match="GPU tensor"):
        H.fp8_block_matmul(c, torch.ones(4, 2), c, torch.ones(1, 2))
