"""Operators beside the distillation loss, on GPU tensors.

* ``linear_cross_entropy`` / ``linear_cross_entropy_backward``: row losses of a
  language-model head without keeping its logits.
* ``embedding`` / ``embedding_backward``: rows of the same weight by token id,
  and their share of its gradient.
* ``quantize_fp8_blocks`` / ``fp8_block_matmul``: matrices in e4m3 with a scale for
  each block of 128, and their product (a teacher's logits from a head held in 8
  bits, for ``Teacher.Precomputed``). Not differentiable.

Every call queues its kernels on torch's current stream of the inputs' device
and returns without waiting; outputs and scratch come from torch's allocator, so
the calls follow the stream and may be captured into a graph (each captured
graph then owns its scratch). Their differentiable forms are in
``orda_hip.autograd``. They have no counterpart in the reference, whose loss is
a weighted mean with the gradients in the same call (src/api.rs:188-422).
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional, Tuple

from . import _lib as L
from .types import OrdaError


_module = None


def _torch():
    global _module
    if _module is None:
        import torch
        _module = torch
    return _module


def _gpu_tensor(x, what: str):
    """x itself, where it is a tensor in GPU memory of its own (not a wrapper
    such as functorch makes, whose memory the library cannot read)."""
    torch = _torch()
    kind = type(x)
    if (kind is not torch.Tensor and kind is not torch.nn.Parameter) or not x.is_cuda:
        if not isinstance(x, torch.Tensor) or not x.is_cuda:
            raise OrdaError(f"{what} must be a GPU tensor")
        raise OrdaError(f"{what} must be a plain tensor with memory of its own")
    try:
        plain = x.data_ptr() != 0 or x.numel() == 0
    except RuntimeError:
        plain = False
    if not plain or x.layout is not torch.strided or x.is_neg():
        raise OrdaError(f"{what} must be a plain tensor with memory of its own")
    return x


def _same_device(device, **tensors):
    for name, t in tensors.items():
        if t.device != device:
            raise OrdaError(f"{name} is on {t.device}, not on {device}")


def _matrix(x, what: str):
    """x as a 2-D tensor with adjacent columns and rows that do not overlap (a
    copy where it is none)."""
    if x.dim() != 2:
        raise OrdaError(f"{what} must be 2-D")
    if x.is_contiguous():
        return x
    (r, c), (sr, sc) = x.shape, x.stride()
    return x.contiguous() if (c > 1 and sc != 1) or (r > 1 and sr < c) else x


def _overlap(a, b) -> bool:
    """Whether the memory of two matrices overlaps."""
    def span(x):
        return x.data_ptr(), x.data_ptr() + (((x.size(0) - 1) * x.stride(0) + x.size(1)) * x.element_size()
                                             if x.numel() else 0)
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


_DTYPES = None


def _dtype(x, what: str) -> int:
    global _DTYPES
    if _DTYPES is None:
        torch = _torch()
        _DTYPES = {torch.float32: L.F32, torch.bfloat16: L.BF16}
    if x.dtype not in _DTYPES:
        raise OrdaError(f"{what} must be float32 or bfloat16, got {x.dtype}")
    return _DTYPES[x.dtype]


def _desc(x, what: str) -> L.Tensor:
    """orda_tensor of a _matrix."""
    r, c = x.shape
    return L.Tensor(x.data_ptr(), r, c, x.stride(0) if r > 1 else c, _dtype(x, what), L.DEVICE)


def _call(fn, *args):
    err = C.create_string_buffer(512)
    rc = fn(*args, err, 512)
    if rc != L.ORDA_OK:
        raise OrdaError(err.value.decode(), rc)


def _stream(device):
    """The handle of torch's current stream (a Stream object costs 2 us more)."""
    return _torch()._C._cuda_getCurrentRawStream(device.index)


def _bytes(n: int, device):
    torch = _torch()
    return torch.empty(n, dtype=torch.uint8, device=device)


@functools.lru_cache(maxsize=1024)
def _embed_bytes(n: int, rows: int, cols: int, dtype: int) -> int:
    b = C.c_int64()
    _call(L.load().orda_embedding_backward_workspace, n, rows, cols, dtype, C.byref(b))
    return b.value


# ------------------------------------------------------------------ linear cross entropy
def _ce_args(hidden, weight, labels, ignore_index, label_smoothing, vocab_piece):
    """(orda_linear_ce, the tensors it points into)."""
    torch = _torch()
    h = _matrix(_gpu_tensor(hidden, "hidden"), "hidden")
    w = _matrix(_gpu_tensor(weight, "weight"), "weight")
    y = _gpu_tensor(labels, "labels")
    if y.dim() != 1:
        raise OrdaError("labels must be 1-D")
    if y.dtype not in (torch.int64, torch.int32):
        raise OrdaError(f"labels must be int64 or int32, got {y.dtype}")
    _same_device(h.device, weight=w, labels=y)
    if y.dtype != torch.int64 or not y.is_contiguous():
        y = y.to(torch.int64).contiguous()
    if vocab_piece is not None and vocab_piece < 1:
        raise OrdaError("vocab_piece must be >= 1")
    a = L.LinearCeC(hidden=_desc(h, "hidden"), weight=_desc(w, "weight"), labels=y.data_ptr(),
                    n_labels=y.numel(), ignore_index=ignore_index, label_smoothing=label_smoothing,
                    vocab_piece=vocab_piece or 0)
    return a, (h, w, y)


def _ce_workspace(lib, a, backward: int, device):
    n = C.c_int64()
    _call(lib.orda_linear_ce_workspace, C.byref(a), backward, C.byref(n))
    return _bytes(n.value, device)


def linear_cross_entropy(hidden, weight, labels, *, ignore_index: int = -100,
                         label_smoothing: float = 0.0, vocab_piece: Optional[int] = None) -> Tuple:
    """Row losses of the logits ``x = hidden @ weight.T``, which are formed a
    piece of the vocabulary at a time and not kept.

    ``hidden`` [N, H] and ``weight`` [V, H] are float32 or bfloat16 GPU tensors,
    ``labels`` [N] int64 or int32. Returns float32 ``(nll, lse)``, each [N]:

    * ``lse[r] = log(sum_v exp(x[r, v]))``
    * ``nll[r] = lse[r] - (1 - e) x[r, y] - (e / V) sum_v x[r, v]`` with
      ``e = label_smoothing``

    Rows labelled ``ignore_index`` are not read and have ``nll = lse = 0``; a
    label that is no class makes its row's ``nll`` NaN. ``vocab_piece`` sets the
    columns of a piece (whole 256s; default: what 1 GiB of scratch holds).
    """
    torch = _torch()
    a, (h, w, y) = _ce_args(hidden, weight, labels, ignore_index, label_smoothing, vocab_piece)
    lib = L.load()
    ws = _ce_workspace(lib, a, 0, h.device)
    nll = torch.empty(h.size(0), dtype=torch.float32, device=h.device)
    lse = torch.empty_like(nll)
    _call(lib.orda_linear_ce_forward, h.device.index, _stream(h.device), C.byref(a), nll.data_ptr(),
          lse.data_ptr(), ws.data_ptr(), ws.numel())
    return nll, lse


def _row_gradient(g, n: int, device, what: str):
    """A float32 [n] gradient with adjacent elements, or None."""
    if g is None:
        return None
    torch = _torch()
    g = _gpu_tensor(g, what)
    _same_device(device, **{what: g})
    if g.dtype != torch.float32 or tuple(g.shape) != (n,):
        raise OrdaError(f"{what} must be float32 [{n}]")
    return g.contiguous()


def linear_cross_entropy_backward(hidden, weight, labels, lse, grad_nll, grad_lse=None, *,
                                  ignore_index: int = -100, label_smoothing: float = 0.0,
                                  vocab_piece: Optional[int] = None, grad_hidden: bool = True,
                                  grad_weight: bool = True) -> Tuple:
    """Gradients of a loss with respect to ``hidden`` and ``weight`` (in their
    types; None where not asked for), given its gradients into ``nll`` and
    ``lse`` of ``linear_cross_entropy`` (float32 [N], either may be None: 0) and
    the ``lse`` that call returned. Ignored rows have zero gradients whatever
    comes in for them; a label that is no class makes its row of ``grad_hidden``
    and all of ``grad_weight`` NaN.
    """
    torch = _torch()
    a, (h, w, y) = _ce_args(hidden, weight, labels, ignore_index, label_smoothing, vocab_piece)
    lib = L.load()
    n = h.size(0)
    if lse is None:
        raise OrdaError("lse must be a GPU tensor")
    lse = _row_gradient(lse, n, h.device, "lse")
    gn = _row_gradient(grad_nll, n, h.device, "grad_nll")
    gl = _row_gradient(grad_lse, n, h.device, "grad_lse")
    ws = _ce_workspace(lib, a, int(grad_hidden) + 2 * int(grad_weight), h.device)
    gh = torch.empty(h.shape, dtype=h.dtype, device=h.device) if grad_hidden else None
    gw = torch.empty(w.shape, dtype=w.dtype, device=w.device) if grad_weight else None
    _call(lib.orda_linear_ce_backward, h.device.index, _stream(h.device), C.byref(a), lse.data_ptr(),
          gn.data_ptr() if gn is not None else None, gl.data_ptr() if gl is not None else None,
          C.byref(_desc(gh, "grad_hidden")) if gh is not None else None,
          C.byref(_desc(gw, "grad_weight")) if gw is not None else None, ws.data_ptr(), ws.numel())
    return gh, gw


# ------------------------------------------------------------------ embedding
def _ids(ids, device, what: str = "ids"):
    """ids as a contiguous 1-D int32 or int64 GPU tensor."""
    torch = _torch()
    ids = _gpu_tensor(ids, what)
    if ids.dtype not in (torch.int64, torch.int32):
        raise OrdaError(f"{what} must be int64 or int32, got {ids.dtype}")
    _same_device(device, **{what: ids})
    return ids if ids.dim() == 1 and ids.is_contiguous() else ids.reshape(-1).contiguous()


def embedding(ids, weight, *, scale: float = 1.0):
    """``scale * weight[ids]``: ``ids`` (int64 or int32, any shape) select rows of
    ``weight`` [V, H] (float32 or bfloat16); the product is rounded once to the
    weight's type. Returns ``[*ids.shape, H]``. An id that is no row gives a row
    of NaN."""
    torch = _torch()
    w = _matrix(_gpu_tensor(weight, "weight"), "weight")
    wd = _desc(w, "weight")
    i = _ids(ids, w.device)
    out = torch.empty((i.numel(), w.size(1)), dtype=w.dtype, device=w.device)
    _call(L.load().orda_embedding, w.device.index, _stream(w.device), i.data_ptr(), i.element_size(),
          i.numel(), C.byref(wd), scale, C.byref(_desc(out, "out")))
    return out if ids.dim() == 1 else out.view(*ids.shape, w.size(1))


def embedding_backward(grad, ids, num_rows: int, *, scale: float = 1.0,
                       padding_idx: Optional[int] = None, out=None, accumulate: bool = False):
    """Gradient of ``embedding`` with respect to its weight: row ``v`` is ``scale *
    sum(grad[t] for ids[t] == v)``, added in the order of the tokens in fp32 and
    rounded once.

    ``grad`` is ``[*ids.shape, H]``, float32 or bfloat16. The result is
    ``[num_rows, H]`` in grad's type, or goes to ``out`` (float32 or bfloat16, 2-D
    with adjacent columns); with ``accumulate`` it is added to ``out``, of which
    only the rows that an id names are read and written (a tied weight's
    gradient, after its other use). Tokens equal to ``padding_idx`` (counted from
    the end where negative), and ids that are no row, add nothing.
    """
    g = _gpu_tensor(grad, "grad")
    i = _ids(ids, g.device)
    if g.dim() != ids.dim() + 1 or g.shape[:-1] != ids.shape:
        raise OrdaError(f"grad must be [*ids.shape, H], got {list(g.shape)} for ids {list(ids.shape)}")
    if num_rows < 0:
        raise OrdaError("num_rows must be >= 0")
    pad = _padding_row(padding_idx, num_rows)
    if out is None:
        if accumulate:
            raise OrdaError("accumulate needs out")
        return _embed_grad(g, i, num_rows, scale, pad)
    torch = _torch()
    out = _gpu_tensor(out, "out")
    _same_device(g.device, out=out)
    if tuple(out.shape) != (num_rows, g.size(-1)):
        raise OrdaError(f"out must be [{num_rows}, {g.size(-1)}]")
    if _matrix(out, "out") is not out:
        raise OrdaError("out must have adjacent columns and rows that do not overlap")
    if out.requires_grad and torch.is_grad_enabled():
        raise OrdaError("out must not require a gradient")
    if _overlap(out, g.reshape(-1, g.size(-1)) if g.numel() else g.new_empty((0, 0))):
        raise OrdaError("out must not share memory with grad")
    if _overlap(out, i.reshape(1, -1)):
        raise OrdaError("out must not share memory with ids")
    _embed_grad(g, i, num_rows, scale, pad, out, accumulate)
    torch.autograd.graph.increment_version(out)   # written in place
    return out


def _padding_row(padding_idx, num_rows: int) -> int:
    if padding_idx is None:
        return -1
    pad = padding_idx + num_rows if padding_idx < 0 else padding_idx
    if not 0 <= pad < num_rows:
        raise OrdaError(f"padding_idx must be a row of {num_rows}, got {padding_idx}")
    return pad


def _embed_grad(g, i, num_rows: int, scale: float, pad: int, out=None, accumulate: bool = False):
    """embedding_backward on checked tensors (g [*, H], i 1-D)."""
    torch = _torch()
    h = g.size(-1)
    if g.dim() != 2:
        g = g.reshape(-1, h) if h else g.new_empty((i.numel(), 0))
    g = _matrix(g, "grad")
    gd = _desc(g, "grad")
    if out is None:
        out = torch.empty((num_rows, h), dtype=g.dtype, device=g.device)
    n = i.numel()
    b = _embed_bytes(n, num_rows, h, gd.dtype)
    ws = _bytes(b, g.device)
    _call(L.load().orda_embedding_backward, g.device.index, _stream(g.device), i.data_ptr(), i.element_size(), n,
          C.byref(gd), pad, scale, accumulate, C.byref(_desc(out, "out")), ws.data_ptr(), b)
    return out


# ------------------------------------------------------------------ e4m3 with block scales
_FP8_PITCH, _FP8_STRIDE = 2 ** 20 + 16, 2 ** 22   # the most that orda_fp8_matrix takes between rows of codes, of scales


def _fp8_desc(codes, scales, block_rows: int, what: str):
    """(orda_fp8_matrix, the tensors it points into) of codes [R, C] and scales
    [ceil(R / block_rows), ceil(C / 128)]."""
    torch = _torch()
    c = _gpu_tensor(codes, what)
    if c.dtype != torch.float8_e4m3fn:
        raise OrdaError(f"{what} must be float8_e4m3fn, got {c.dtype}")
    c = _matrix(c, what)
    if c.size(0) > 1 and c.stride(0) > _FP8_PITCH:
        c = c.contiguous()
    s = _gpu_tensor(scales, f"{what}'s scales")
    _same_device(c.device, **{f"{what}'s scales": s})
    shape = (-(-c.size(0) // block_rows), -(-c.size(1) // 128))
    if s.dtype != torch.float32 or tuple(s.shape) != shape:
        raise OrdaError(f"{what}'s scales must be float32 {list(shape)}")
    if shape[0] > 1 and s.stride(0) > _FP8_STRIDE:
        s = s.contiguous()
    d = L.Fp8MatrixC(codes=c.data_ptr(), rows=c.size(0), cols=c.size(1),
                     ld=c.stride(0) if c.size(0) > 1 else -(-c.size(1) // 16) * 16,
                     scales=s.data_ptr(), scale_row=s.stride(0) if shape[0] > 1 else 0,
                     scale_col=s.stride(1) if shape[1] > 1 else 0, block_rows=block_rows)
    return d, (c, s)


def quantize_fp8_blocks(m, *, block_rows: int = 1) -> Tuple:
    """``(codes, scales)`` of ``m`` [R, C] (float32 or bfloat16): float8_e4m3fn codes
    [R, C] and one float32 scale for each block of 128 columns and ``block_rows``
    rows (1 or 128), [ceil(R / block_rows), ceil(C / 128)].

    ``scale = max(amax / 448, 2**-126)`` and ``code = m / scale`` rounded to nearest
    even, both quotients in float32; a block with an infinity or a NaN has the
    scale NaN and codes NaN. The rows of ``codes`` lie a multiple of 16 bytes apart,
    and the scales of single rows block by block, as ``fp8_block_matmul`` reads
    them best.
    """
    torch = _torch()
    m = _matrix(_gpu_tensor(m, "m"), "m")
    md = _desc(m, "m")
    if block_rows not in (1, 128):
        raise OrdaError(f"block_rows must be 1 or 128, got {block_rows}")
    r, c = m.shape
    pitch = -(-c // 16) * 16
    codes = torch.empty((r, pitch), dtype=torch.float8_e4m3fn, device=m.device)[:, :c]
    rb, cb = -(-r // block_rows), -(-c // 128)
    scales = (torch.empty((cb, rb), dtype=torch.float32, device=m.device).t() if block_rows == 1
              else torch.empty((rb, cb), dtype=torch.float32, device=m.device))
    d = L.Fp8MatrixC(codes=codes.data_ptr(), rows=r, cols=c, ld=pitch, scales=scales.data_ptr(),
                     scale_row=1 if block_rows == 1 else cb, scale_col=rb if block_rows == 1 else 1,
                     block_rows=block_rows)
    _call(L.load().orda_quant_fp8_blocks, m.device.index, _stream(m.device), C.byref(md), C.byref(d))
    return codes, scales


def fp8_block_matmul(a, a_scales, b, b_scales, *, out_dtype=None):
    """``A @ B.T`` of quantised matrices: ``a`` [M, K] with a scale for each row and 128
    columns (``a_scales`` [M, ceil(K / 128)]), ``b`` [N, K] for each 128 rows and 128
    columns (``b_scales`` [ceil(N / 128), ceil(K / 128)]), as ``quantize_fp8_blocks``
    makes them with ``block_rows`` 1 and 128, or a checkpoint holds them. Blocks are
    added in float32 and rounded once to ``out_dtype`` (bfloat16, the default, or
    float32); the sum over a block of 128 is float32 for float32 outputs, and held
    to fewer bits for bfloat16 ones (off by 1.5e-5 of the root of the sum of the
    products' squares, at most 1e-4).
    Returns [M, N]. Codes whose memory or pitch is not 16-byte aligned, or whose
    rows lie over 2^20 + 16 bytes apart, are copied first."""
    torch = _torch()
    ad, (a, _sa) = _fp8_desc(a, a_scales, 1, "a")
    bd, (b, _sb) = _fp8_desc(b, b_scales, 128, "b")
    _same_device(a.device, b=b)
    out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise OrdaError(f"out_dtype must be bfloat16 or float32, got {out_dtype}")
    lib = L.load()
    n = C.c_int64()
    _call(lib.orda_fp8_block_matmul_workspace, C.byref(ad), C.byref(bd), C.byref(n))
    ws = _bytes(n.value, a.device)
    out = torch.empty((a.size(0), b.size(0)), dtype=out_dtype, device=a.device)
    _call(lib.orda_fp8_block_matmul, a.device.index, _stream(a.device), C.byref(ad), C.byref(bd),
          C.byref(_desc(out, "out")), ws.data_ptr(), ws.numel())
    return out
