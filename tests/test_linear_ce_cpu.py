"""The linear cross entropy's refusals, without a GPU: the Python checks, and the
C entry points' checks of their arguments (made before any device call)."""
import ctypes as C

import pytest
import torch

import orda_hip as H
from orda_hip import _lib as L


def args(n=4, h=8, v=16, **kw):
    a = L.LinearCeC(hidden=L.Tensor(data=256, rows=n, cols=h, dtype=L.BF16, location=L.DEVICE),
                    weight=L.Tensor(data=256, rows=v, cols=h, dtype=L.BF16, location=L.DEVICE),
                    labels=256, n_labels=n, ignore_index=-100)
    for k, x in kw.items():
        if "." in k:
            t, f = k.split(".")
            setattr(getattr(a, t), f, x)
        else:
            setattr(a, k, x)
    return a


def workspace(a, backward=0):
    n, err = C.c_int64(), C.create_string_buffer(512)
    rc = L.load().orda_linear_ce_workspace(C.byref(a), backward, C.byref(n), err, 512)
    return rc, n.value, err.value.decode()


@pytest.mark.parametrize("change, message", [
    ({"weight.cols": 9}, "columns"),
    ({"n_labels": 3}, "labels"),
    ({"weight.dtype": L.F32}, "dtype"),
    ({"hidden.dtype": L.I8}, "float32 or bfloat16"),
    ({"hidden.location": L.HOST}, "device"),
    ({"weight.location": L.HOST}, "device"),
    ({"hidden.rows": -1}, "negative"),
    ({"hidden.data": None}, "null"),
    ({"weight.ld": 7}, "ld < cols"),
    ({"label_smoothing": -0.1}, "label_smoothing"),
    ({"label_smoothing": 1.5}, "label_smoothing"),
    ({"label_smoothing": float("nan")}, "label_smoothing"),
    ({"vocab_piece": -1}, "vocab_piece"),
    ({"weight.rows": 0}, "> 0"),
    ({"hidden.cols": 0, "weight.cols": 0}, "> 0"),
    ({"hidden.cols": 2 ** 21, "weight.cols": 2 ** 21}, "at most"),
])
def test_arguments_refused(change, message):
    a = args(**change)
    rc, _, err = workspace(a)
    assert rc == L.ORDA_ERR_INVALID and message in err
    err = C.create_string_buffer(512)
    rc = L.load().orda_linear_ce_forward(0, None, C.byref(a), 256, 256, 256, 1 << 40, err, 512)
    assert rc == L.ORDA_ERR_INVALID and message in err.value.decode()


def test_null_and_small_workspaces_refused():
    lib, a, err = L.load(), args(), C.create_string_buffer(512)
    assert workspace(a)[0] == L.ORDA_OK
    need = workspace(a)[1]
    assert lib.orda_linear_ce_forward(0, None, C.byref(a), 256, 256, 256, need - 1, err, 512) == L.ORDA_ERR_INVALID
    assert "workspace" in err.value.decode()
    assert lib.orda_linear_ce_forward(0, None, C.byref(a), 256, 256, 264, need, err, 512) == L.ORDA_ERR_INVALID
    assert "aligned" in err.value.decode()
    assert lib.orda_linear_ce_forward(0, None, C.byref(a), None, 256, 256, need, err, 512) == L.ORDA_ERR_INVALID
    assert lib.orda_linear_ce_workspace(None, 0, None, err, 512) == L.ORDA_ERR_INVALID
    g = L.Tensor(data=256, rows=4, cols=8, dtype=L.F32, location=L.DEVICE)
    rc = lib.orda_linear_ce_backward(0, None, C.byref(a), 256, 256, None, C.byref(g), None, 256, 1 << 40, err, 512)
    assert rc == L.ORDA_ERR_INVALID and "dtype" in err.value.decode()
    g = L.Tensor(data=256, rows=5, cols=8, dtype=L.BF16, location=L.DEVICE)
    rc = lib.orda_linear_ce_backward(0, None, C.byref(a), 256, 256, None, None, C.byref(g), 256, 1 << 40, err, 512)
    assert rc == L.ORDA_ERR_INVALID and "grad_weight" in err.value.decode()


def test_scratch_follows_the_piece():
    """Smaller pieces take less scratch (beside the partial sums of products that
    are split); a piece is whole 256s; a default call of a large batch stays near
    a GiB beside its rows."""
    big = dict(n=8192, h=4096, v=131072)
    sizes = [workspace(args(**big, vocab_piece=p), 3)[1] for p in (1, 256, 16384, 65536, 131072)]
    assert sizes[0] == sizes[1] < sizes[2] < sizes[3] < sizes[4]
    assert workspace(args(**big), 3)[1] < 3 << 29
    assert workspace(args(**big), 0)[1] < 3 << 28
    # no rows: nothing to hold
    assert workspace(args(n=0, **{"hidden.data": None}))[:2] == (L.ORDA_OK, 0)


@pytest.mark.parametrize("n, h, v, piece", [(1, 1, 1, 0), (100, 33, 1000, 0), (64, 64, 300, 256), (5000, 4096, 600, 256),
                                            (4915, 4096, 131072, 65536), (700, 520, 50257, 0), (17000, 40, 300, 0)])
@pytest.mark.parametrize("dtype", [L.BF16, L.F32])
def test_the_scratch_asked_for_is_the_scratch_laid_out(n, h, v, piece, dtype):
    """A call with exactly the bytes that were asked for gets past the check of
    the layout it will use (and ends at a device that does not exist); with 256
    fewer it does not."""
    a = args(n=n, h=h, v=v, vocab_piece=piece, **{"hidden.dtype": dtype, "weight.dtype": dtype})
    lib, err = L.load(), C.create_string_buffer(512)
    need = workspace(a)[1]
    for less, want in ((0, L.ORDA_ERR_HIP), (256, L.ORDA_ERR_INVALID)):
        assert lib.orda_linear_ce_forward(9999, None, C.byref(a), 256, 256, 256, need - less, err, 512) == want
    gh = L.Tensor(data=256, rows=n, cols=h, dtype=dtype, location=L.DEVICE)
    gw = L.Tensor(data=256, rows=v, cols=h, dtype=dtype, location=L.DEVICE)
    for which, out in ((1, (gh, None)), (2, (None, gw)), (3, (gh, gw))):
        need = workspace(a, which)[1]
        for less, want in ((0, L.ORDA_ERR_HIP), (256, L.ORDA_ERR_INVALID)):
            rc = lib.orda_linear_ce_backward(9999, None, C.byref(a), 256, 256, None,
                                             *(C.byref(t) if t is not None else None for t in out), 256, need - less,
                                             err, 512)
            assert rc == want, err.value


@pytest.mark.parametrize("dtype", [L.BF16, L.F32])
def test_operands_stay_within_32_bit_offsets(dtype):
    """A tile of a product's operand is 256 rows at 32-bit byte offsets: batches whose transpose passes them are
    refused, larger pieces cut, weights at larger pitches copied."""
    both = {"hidden.dtype": dtype, "weight.dtype": dtype}
    top = 2 ** 21
    assert workspace(args(n=top, v=300, **both), 3)[0] == L.ORDA_OK
    rc, _, err = workspace(args(n=top + 1, v=300, **both), 3)
    assert rc == L.ORDA_ERR_INVALID and "2^21 rows" in err
    # the gradient of a piece's logits is the largest part of the scratch
    cut = workspace(args(n=512, v=4 * top, vocab_piece=top, **both), 3)[1]
    assert cut >= 512 * top * 2
    assert workspace(args(n=512, v=4 * top, vocab_piece=2 * top, **both), 3)[1] == cut
    assert workspace(args(n=1, v=4 * top, **both), 3)[1] <= workspace(args(n=1, v=4 * top, vocab_piece=top, **both), 3)[1]
    if dtype == L.BF16:
        wide = workspace(args(v=1000, **{"weight.ld": 2 ** 20}), 3)[1]
        assert workspace(args(v=1000, **{"weight.ld": 2 ** 20 + 8}), 3)[1] >= wide + 1000 * 8 * 2


def test_python_refuses_cpu_tensors():
    h, w, y = torch.zeros(2, 8), torch.zeros(3, 8), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(H.OrdaError, match="GPU tensor"):
        H.linear_cross_entropy(h, w, y)
    with pytest.raises(H.OrdaError, match="GPU tensor"):
        H.linear_cross_entropy_backward(h, w, y, torch.zeros(2), torch.zeros(2))


@pytest.mark.parametrize("v, h", [(32000, 4096), (44000, 4096), (50257, 4096), (131072, 2048), (131072, 4096), (2 ** 20, 512)])
@pytest.mark.parametrize("n", [1, 16, 64])
def test_few_fp32_rows_take_no_planes(n, v, h):
    """Few fp32 rows stream the weight whatever its size: the scratch holds the rows and 16 bytes of statistics for
    each of them and 64 classes (with gradients their logits' rows and split products), not the weight."""
    f32 = {"hidden.dtype": L.F32, "weight.dtype": L.F32}
    need = workspace(args(n=n, h=h, v=v, **f32))[1]
    assert need <= 2 * n * (v / 64 + 1) * 16 + 4 * 64 * h + (1 << 16)
    whole = workspace(args(n=n, h=h, v=v, vocab_piece=v // 256 * 256 + 256, **f32))[1]
    assert need == whole
    assert workspace(args(n=n, h=h, v=v, **f32), 2)[1] <= 4 * n * (v + 2048) * 2 + 4 * 64 * 2 * h + (1 << 20)
    assert workspace(args(n=n, h=h, v=v, **f32), 3)[1] <= 1 << 30


@pytest.mark.parametrize("n", [2 ** 20, 2 ** 21])
def test_a_piece_is_one_launch(n):
    """HIP takes fewer than 2^32 threads in a launch, 256 for each tile of 128 or 256 rows by 256 classes: larger
    pieces are cut, which the statistics' scratch (16 bytes a row and tile) shows."""
    need = workspace(args(n=n, h=64, v=2 ** 21, vocab_piece=2 ** 21))[1]
    tiles = (2 ** 24 - 1) // (n // 128)
    assert n * tiles * 16 // 2 <= need <= n * (tiles * 16 + 64 * 2 + 64)


@pytest.mark.parametrize("n, h, v", [(2048, 2048, 32000), (1024, 4096, 32000), (900, 4096, 32000), (4096, 1024, 30000)])
def test_large_fp32_gradients_take_planes(n, h, v):
    """The form that keeps its logits is for small calls: a grad_hidden of 48 to 64 tiles of 256 over a whole
    vocabulary goes over planes (6 bytes for each element of the weight, and of the logits), as both gradients do."""
    f32 = {"hidden.dtype": L.F32, "weight.dtype": L.F32}
    for which in (1, 2, 3):
        assert workspace(args(n=n, h=h, v=v, **f32), which)[1] >= 6 * v * (h + n)


def test_asked_for_pieces_are_kept():
    """vocab_piece bounds the scratch of fp32 calls too: smaller pieces, less of it."""
    f32 = {"hidden.dtype": L.F32, "weight.dtype": L.F32}
    sizes = [workspace(args(n=512, h=4096, v=131072, vocab_piece=p, **f32), 3)[1] for p in (256, 4096, 16384, 65536)]
    assert sizes == sorted(sizes) and sizes[0] < sizes[-1]


@pytest.mark.parametrize("n, h, v, piece", [(3, 4096, 44000, 0), (64, 1000, 180001, 0), (64, 2426, 131072, 0), (1, 512, 2 ** 21, 0),
                                            (1, 64, 2 ** 21 + 300, 0), (2048, 2048, 32000, 0), (1000, 4096, 50257, 0)])
def test_the_scratch_of_large_fp32_calls_is_the_scratch_laid_out(n, h, v, piece):
    """As above, at and past the vocabularies that the planes' scratch cuts into pieces."""
    test_the_scratch_asked_for_is_the_scratch_laid_out(n, h, v, piece, L.F32)
