"""Refusals of drawing tokens, without a GPU: the C entry points check their
arguments before any device call."""
import ctypes as C

import pytest
import torch

import orda_hip as H
from orda_hip import _lib as L


def logits(rows=4, cols=1000, **kw):
    t = L.Tensor(data=256, rows=rows, cols=cols, dtype=L.BF16, location=L.DEVICE)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("kw, message", [
    (dict(logits=logits(dtype=L.I8)), "float32 or bfloat16"), (dict(logits=logits(location=L.HOST)), "device"),
    (dict(logits=logits(data=None)), "null"), (dict(logits=logits(rows=-1)), "negative"), (dict(logits=logits(ld=999)), "ld < cols"),
    (dict(logits=logits(cols=(1 << 20) + 1)), "at most"), (dict(logits=logits(rows=(1 << 20) + 1)), "at most"),
    (dict(logits=logits(cols=0)), "columns"), (dict(uniform=None), "null"), (dict(tokens=None), "null"),
    (dict(temperature=-1.0), "temperature"), (dict(temperature=NAN), "temperature"), (dict(temperature=INF), "temperature"),
    (dict(top_p=-0.1), "top_p"), (dict(top_p=1.1), "top_p"), (dict(top_p=NAN), "top_p"), (dict(min_p=-0.1), "min_p"),
    (dict(min_p=1.5), "min_p"), (dict(min_p=NAN), "min_p"), (dict(ws=264), "aligned"), (dict(ws=None), "workspace"),
    (dict(ws_bytes=64), "workspace")])
def test_refused(kw, message):
    kw = dict(kw)
    tokens, ws, ws_bytes = kw.pop("tokens", 256), kw.pop("ws", 256), kw.pop("ws_bytes", 1 << 40)
    a = dict(logits=logits(), uniform=256, temperature=1.0, top_p=1.0, min_p=0.0, top_k=0)
    a.update(kw)
    err = C.create_string_buffer(512)
    rc = L.load().orda_sample_tokens(0, None, C.byref(L.SamplingC(**a)), tokens, None, ws, ws_bytes, err, 512)
    assert rc == L.ORDA_ERR_INVALID and message in err.value.decode()


@pytest.mark.parametrize("n, v", [(0, 1000), (1, 1), (1, 131072), (512, 131072), (1 << 20, 64), (3, 1 << 20)])
def test_workspace(n, v):
    """Of every 64 tokens a key, of every 1024 a key and a sum; and a row's last 1024 where they are fewer."""
    for dtype, es in ((L.F32, 4), (L.BF16, 2)):
        out, err = C.c_int64(), C.create_string_buffer(512)
        assert L.load().orda_sample_tokens_workspace(n, v, dtype, C.byref(out), err, 512) == L.ORDA_OK
        need = n * (-(-v // 64) * 4 + -(-v // 1024) * 12 + (1024 * es if v % 1024 else 0))
        assert need <= out.value < need + 4 * 256


def test_python_refuses_cpu_tensors():
    with pytest.raises(H.OrdaError, match="GPU tensor"):
        H.sample_tokens(torch.zeros(2, 8), torch.zeros(2))
