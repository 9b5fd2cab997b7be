"""The gradient norm's and clipping's refusals and scratch, without a GPU: the C
entry points check their arguments before any device call."""
import ctypes as C

import pytest
import torch

import orda_hip as H
from orda_hip import _lib as L

BASE = 1 << 20


def mat(rows, cols, at=0, **kw):
    t = L.Tensor(data=BASE + at, rows=rows, cols=cols, dtype=L.F32, location=L.DEVICE)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def table(*pairs):
    a = (L.GradientC * max(1, len(pairs)))()
    for e, (src, dst) in zip(a, pairs):
        e.src = src
        if dst is not None:
            e.dst = dst
    return a


def clip(a, count, max_norm=1.0, eps=1e-6, norm=256, ws=256, ws_bytes=1 << 40):
    err = C.create_string_buffer(512)
    rc = L.load().orda_clip_gradients(0, None, a, count, max_norm, eps, norm, ws, ws_bytes, err, 512)
    return rc, err.value.decode()


FAR = 1 << 30


@pytest.mark.parametrize("pairs, message", [
    ([(mat(2, 8, dtype=L.I8), None)], "float32 or bfloat16"), ([(mat(2, 8, location=L.HOST), None)], "device"),
    ([(mat(2, 8, data=None), None)], "null"), ([(mat(2, 8, ld=7), None)], "ld < cols"), ([(mat(-2, 8), None)], "negative"),
    ([(mat(1 << 40, 2), None)], "2^40"), ([(mat(1 << 30, 1 << 10), None), (mat(1, 8, FAR), None)], "2^40"),
    ([(mat(2, 8), mat(2, 9, FAR))], "destination"), ([(mat(2, 8), mat(2, 8, FAR, dtype=L.I8))], "float32 or bfloat16"),
    ([(mat(2, 8), mat(2, 8, FAR, location=L.HOST))], "device"),
    ([(mat(2, 8), mat(2, 8, FAR)), (mat(2, 8, 2 * FAR), None)], "all gradients"),
    # the same gradient twice, parts of one another, a destination on another's gradient
    ([(mat(2, 8), None), (mat(2, 8), None)], "share memory"), ([(mat(2, 8), None), (mat(1, 4, 60), None)], "share memory"),
    ([(mat(2, 8), mat(2, 8, FAR)), (mat(2, 8, 64), mat(2, 8, FAR + 32))], "share memory"),
    ([(mat(2, 8), mat(2, 8, 32))], "share memory"),
    ([(mat(4, 8, ld=20), None), (mat(4, 8, 28, ld=20), None)], "share memory"),   # columns 0-7 and 7-14 of one frame
    ([(mat(4, 8, ld=20), None), (mat(4, 8, 60, ld=20), None)], "share memory"),   # 0-7, and 15-19 with the next row's 0-2
])
def test_clip_refused(pairs, message):
    rc, err = clip(table(*pairs), len(pairs))
    assert rc == L.ORDA_ERR_INVALID and message in err


@pytest.mark.parametrize("kw, message", [
    (dict(count=-1), "at most"), (dict(count=(1 << 20) + 1), "at most"), (dict(max_norm=-1.0), "max_norm"),
    (dict(max_norm=float("nan")), "max_norm"), (dict(eps=-1.0), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(norm=None), "null"), (dict(ws=264), "aligned"), (dict(ws=None), "workspace"), (dict(ws_bytes=0), "workspace"),
    (dict(a=None), "null")])
def test_clip_arguments_refused(kw, message):
    d = dict(a=table((mat(2, 8), None)), count=1)
    d.update(kw)
    rc, err = clip(**d)
    assert rc == L.ORDA_ERR_INVALID and message in err


@pytest.mark.parametrize("pairs", [
    [(mat(4, 8, ld=20), None), (mat(4, 8, 32, ld=20), None)],     # columns 0-7 and 8-15 of one frame
    [(mat(4, 8, ld=20), None), (mat(4, 4, 64, ld=20), None)],     # 0-7 and 16-19
    [(mat(4, 8), None), (mat(4, 8, 128), None)],                  # end to end
    [(mat(2, 8), None), (mat(0, 8), None), (mat(8, 0), None)],    # without values
])
def test_gradients_beside_one_another_pass_the_checks(pairs):
    """(A workspace that is too small is found after them.)"""
    rc, err = clip(table(*pairs), len(pairs), ws_bytes=0)
    assert rc == L.ORDA_ERR_INVALID and "workspace" in err


@pytest.mark.parametrize("count", [0, 1, 57, 1000, 1 << 20])
def test_workspace_has_a_sum_for_each_workgroup(count):
    out, err = C.c_int64(), C.create_string_buffer(512)
    assert L.load().orda_clip_gradients_workspace(count, C.byref(out), err, 512) == L.ORDA_OK
    assert 8 * min(count, 1) <= out.value <= 8 * (4096 + count / 32 + 1) + 256


def test_python_refuses():
    with pytest.raises(H.OrdaError, match="GPU tensor"):
        H.clip_gradients([torch.zeros(4)], 1.0)
    for call in (lambda: H.gradient_norm([]), lambda: H.gradient_norm([None]), lambda: H.clip_gradients([], 1.0)):
        with pytest.raises(H.OrdaError, match="no gradients"):
            call()
    with pytest.raises(H.OrdaError, match="out must have"):
        H.clip_gradients([torch.zeros(4)], 1.0, out=[])
