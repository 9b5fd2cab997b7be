"""The embedding's refusals, without a GPU: the C entry points check their
arguments before any device call."""
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


def forward(w, out, ids=256, ids_bytes=8, n=4):
    err = C.create_string_buffer(512)
    rc = L.load().orda_embedding(0, None, ids, ids_bytes, n, C.byref(w), 1.0, C.byref(out), err, 512)
    return rc, err.value.decode()


def backward(g, out, ids=256, ids_bytes=8, n=4, ws=256, ws_bytes=1 << 40):
    err = C.create_string_buffer(512)
    rc = L.load().orda_embedding_backward(0, None, ids, ids_bytes, n, C.byref(g), -1, 1.0, 0, C.byref(out), ws,
                                          ws_bytes, err, 512)
    return rc, err.value.decode()


@pytest.mark.parametrize("kw, message", [
    (dict(ids=None), "null"), (dict(ids_bytes=2), "int32 or int64"), (dict(n=-1), "ids"), (dict(n=5), "out must be"),
    (dict(w=mat(9, 8, dtype=L.I8)), "float32 or bfloat16"), (dict(w=mat(9, 8, location=L.HOST)), "device"),
    (dict(w=mat(9, 8, data=None)), "null"), (dict(w=mat(9, 8, ld=4)), "ld < cols"), (dict(w=mat(-1, 8)), "negative"),
    (dict(out=mat(4, 8, dtype=L.F32)), "dtype"), (dict(out=mat(4, 9)), "out must be"),
    (dict(w=mat(9, 1 << 21), out=mat(4, 1 << 21)), "at most"),
])
def test_lookup_refused(kw, message):
    a = dict(w=mat(9, 8), out=mat(4, 8))
    a.update(kw)
    rc, err = forward(**a)
    assert rc == L.ORDA_ERR_INVALID and message in err


@pytest.mark.parametrize("kw, message", [
    (dict(ids=None), "null"), (dict(ids_bytes=1), "int32 or int64"), (dict(n=3), "grad must be"),
    (dict(g=mat(4, 9)), "grad must be"), (dict(g=mat(4, 8, dtype=L.I8)), "float32 or bfloat16"),
    (dict(out=mat(9, 8, dtype=L.I8)), "float32 or bfloat16"), (dict(out=mat(9, 8, location=L.HOST)), "device"),
    (dict(ws=264), "aligned"), (dict(ws_bytes=0), "workspace"), (dict(ws=None), "workspace"),
])
def test_gradient_refused(kw, message):
    a = dict(g=mat(4, 8), out=mat(9, 8))
    a.update(kw)
    rc, err = backward(**a)
    assert rc == L.ORDA_ERR_INVALID and message in err


@pytest.mark.parametrize("n", [0, 1, 32, 33, 2048, 2049, 4096, 65536, 1 << 20])
def test_workspace_grows_with_the_tokens(n):
    out, err = C.c_int64(), C.create_string_buffer(512)
    assert L.load().orda_embedding_backward_workspace(n, 131072, 4096, L.BF16, C.byref(out), err, 512) == L.ORDA_OK
    # pairs, twice where they are sorted in passes (with 512 counts for every 4096), and two fp32 rows a
    # chunk: of 8 tokens, or more where that makes over 512 chunks, up to 256 tokens
    assert out.value >= 8 * n
    chunks = min(n / 8 + 1, max(513, n / 256 + 1))
    assert out.value <= 16 * n + (n / 4096 + 1) * 2048 + 2 * chunks * 4096 * 4 + 6 * 256


@pytest.mark.parametrize("n", [1 << 17, (1 << 17) + 1, 1 << 24, 1 << 30])
def test_workspace_of_many_tokens(n):
    """Pairs twice, 512 counts for every 4096 of them and, where a launch sums these, one row more; two fp32 rows for
    each chunk of 256."""
    out, err = C.c_int64(), C.create_string_buffer(512)
    assert L.load().orda_embedding_backward_workspace(n, 131072, 8, L.BF16, C.byref(out), err, 512) == L.ORDA_OK
    rows = -(-n // 4096) + (1 if n > 1 << 17 else 0)
    up = lambda b: -(-b // 256) * 256
    assert out.value == 4 * up(4 * n) + rows * 2048 + up(-(-n // 256) * 2 * 512 * 4)


def test_python_refuses_cpu_tensors():
    with pytest.raises(H.OrdaError, match="GPU tensor"):
        H.embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(5, 8))
    with pytest.raises(H.OrdaError, match="GPU tensor"):
        H.embedding_backward(torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64), 5)
