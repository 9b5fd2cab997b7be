"""Operators beside the distillation loss, on GPU tensors.

* ``linear_cross_entropy`` / ``linear_cross_entropy_backward``: row losses of a
  language-model head without keeping its logits.
* ``embedding`` / ``embedding_backward``: rows of the same weight by token id,
  and their share of its gradient.
* ``quantize_fp8_blocks`` / ``fp8_block_matmul``: matrices in e4m3 with a scale for
  each block of 128, and their product (a teacher's logits from a head held in 8
  bits, for ``Teacher.Precomputed``). Not differentiable.
* ``rms_norm`` / ``rms_norm_backward``: the norm before the head, with the
  residual's addition; ``rms_norm_fp8``: its output in e4m3, for ``fp8_block_matmul``.
* ``sample_tokens``: tokens drawn from the head's logits.
* ``clip_gradients`` / ``gradient_norm``: the norm of all gradients together, and
  their scaling to a limit.

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
import math
import operator
import struct
import threading
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


def _is_matrix(x) -> bool:
    """Whether a 2-D tensor has adjacent columns and rows that do not overlap."""
    if x.is_contiguous():
        return True
    (r, c), (sr, sc) = x.shape, x.stride()
    return not ((c > 1 and sc != 1) or (r > 1 and sr < c))


def _matrix(x, what: str):
    """x as a 2-D tensor with adjacent columns and rows that do not overlap (a
    copy where it is none)."""
    if x.dim() != 2:
        raise OrdaError(f"{what} must be 2-D")
    return x if _is_matrix(x) else x.contiguous()


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


# Structures packed into one buffer, and a message's place for each thread: a call of a
# few tensors costs half of what ctypes' structures and a new message take.
_TENSOR = "Qqqqii"                                                  # orda_tensor
_NORM = struct.Struct("=" + 3 * _TENSOR + "dd")                     # orda_rms_norm
_ROWS = struct.Struct("=" + _TENSOR)
_ADDRESS = struct.Struct("=Q")
_NORM_OUT = struct.Struct("=" + 2 * _TENSOR)                        # total, out
_NORM_FP8 = struct.Struct("=" + _TENSOR + "QqqqQqqi4x")             # total, orda_fp8_matrix
_NORM_GRADS = struct.Struct("=" + 4 * _TENSOR)                      # grad_out, grad_total, grad_x, grad_weight
_NO_TENSOR = (0, 0, 0, 0, 0, 0)


_thread = threading.local()


def _message() -> int:
    try:
        return _thread.message
    except AttributeError:
        _thread.buffer = C.create_string_buffer(512)
        _thread.message = C.addressof(_thread.buffer)
        return _thread.message


def _packed(data: bytes):
    """A buffer that holds data, and its address."""
    buf = bytearray(data)
    return buf, C.addressof(C.c_char.from_buffer(buf))


def _check(rc: int):
    if rc != L.ORDA_OK:
        raise OrdaError(C.string_at(_message()).decode(), rc)


def _fields(x, what: str):
    """orda_tensor of a _matrix."""
    r, c = x.shape
    return x.data_ptr(), r, c, x.stride(0) if r > 1 else c, _dtype(x, what), L.DEVICE


def _row_fields(x, what: str):
    """orda_tensor of a contiguous vector as one row."""
    n = x.numel()
    return x.data_ptr(), 1, n, n, _dtype(x, what), L.DEVICE


# ------------------------------------------------------------------ root-mean-square norm
def _rows(x, h: int, what: str):
    """x [..., h] as a _matrix."""
    if x.dim() == 2:
        return _matrix(x, what)
    return _matrix(x.reshape(-1, h) if h else x.new_empty((math.prod(x.shape[:-1]), 0)), what)


def _norm_args(x, weight, residual, eps: float, weight_offset: float):
    """(orda_rms_norm, x as a matrix, weight, residual as they are pointed to)."""
    x = _gpu_tensor(x, "x")
    if x.dim() < 1:
        raise OrdaError("x must be [..., H]")
    h = x.size(-1)
    w = _gpu_tensor(weight, "weight")
    index = x.get_device()
    if w.get_device() != index:
        raise OrdaError(f"weight is on {w.device}, not on {x.device}")
    if w.dim() != 1 or w.size(0) != h:
        raise OrdaError(f"weight must be [{h}]")
    w = w.contiguous()
    m, r = _rows(x, h, "x"), None
    if residual is not None:
        r = _gpu_tensor(residual, "residual")
        if r.get_device() != index:
            raise OrdaError(f"residual is on {r.device}, not on {x.device}")
        if r.shape != x.shape or r.dtype != x.dtype:
            raise OrdaError("residual must have the shape and dtype of x")
        r = _rows(r, h, "residual")
    try:
        a = _NORM.pack(*_fields(m, "x"), *(_fields(r, "residual") if r is not None else _NO_TENSOR),
                       *_row_fields(w, "weight"), eps, weight_offset)
    except (struct.error, OverflowError, TypeError):
        raise OrdaError("eps and weight_offset must be numbers") from None
    return a, m, w, r


def _like(m):
    """An empty matrix of a _matrix's shape and type, row by row."""
    torch = _torch()
    return torch.empty_like(m) if m.is_contiguous() else torch.empty(m.shape, dtype=m.dtype, device=m.device)


def _norm_forward(x, weight, residual, eps: float, weight_offset: float):
    """rms_norm's result and sum (None without a residual) as matrices, and the arguments."""
    a, m, w, _r = args = _norm_args(x, weight, residual, eps, weight_offset)
    out = _like(m)
    n, h = m.shape
    kind, total = _DTYPES[m.dtype], None
    if residual is not None:
        total = _like(m)
        outs = _NORM_OUT.pack(total.data_ptr(), n, h, h, kind, L.DEVICE, out.data_ptr(), n, h, h, kind, L.DEVICE)
    else:
        outs = _NORM_OUT.pack(0, 0, 0, 0, 0, 0, out.data_ptr(), n, h, h, kind, L.DEVICE)
    _buf, p = _packed(a + outs)
    index = m.get_device()
    _check(L.load().orda_rms_norm_forward(index, _torch()._C._cuda_getCurrentRawStream(index), p, p + _NORM.size,
                                          p + _NORM.size + _ROWS.size, _message(), 512))
    return out, total, args


def rms_norm(x, weight, *, residual=None, eps: float = 1e-6, weight_offset: float = 0.0):
    """``t / sqrt(mean(t**2) + eps) * (weight + weight_offset)`` over the last dimension
    of ``t = x + residual`` (``t = x`` without a residual).

    ``x`` and ``residual`` are [..., H], float32 or bfloat16, ``weight`` [H] either of
    them. ``t`` is rounded to x's type, the mean formed in 64 bits, the result
    rounded once to x's type. A root below 3e-39 (of ``eps`` 0) counts as 0. Returns the
    result, with a residual ``(result, t)``.
    """
    out, total, _ = _norm_forward(x, weight, residual, eps, weight_offset)
    if x.dim() != 2:
        out, total = out.view(x.shape), total.view(x.shape) if total is not None else None
    return out if total is None else (out, total)


def rms_norm_fp8(x, weight, *, residual=None, eps: float = 1e-6, weight_offset: float = 0.0) -> Tuple:
    """``rms_norm`` with its result in e4m3: ``(codes, scales)``, with a residual
    ``(codes, scales, t)``. The codes [N, H] of x's N rows and the scales [N, ceil(H / 128)]
    are those that ``quantize_fp8_blocks`` gives of the result in float32 (which is not
    rounded to x's type before), laid out as ``fp8_block_matmul`` reads them best."""
    torch = _torch()
    a, m, _w, _r = _norm_args(x, weight, residual, eps, weight_offset)
    n, h = m.shape
    device = m.device
    pitch, cb = -(-h // 16) * 16, -(-h // 128)
    codes = torch.empty((n, pitch), dtype=torch.float8_e4m3fn, device=device)
    scales = torch.empty((cb, n), dtype=torch.float32, device=device)
    total = _like(m) if residual is not None else None
    t = _fields(total, "total") if total is not None else _NO_TENSOR
    _buf, p = _packed(a + _NORM_FP8.pack(*t, codes.data_ptr(), n, h, pitch, scales.data_ptr(), 1, n, 1))
    _check(L.load().orda_rms_norm_fp8(device.index, _stream(device), p, p + _NORM.size, p + _NORM.size + _ROWS.size,
                                      _message(), 512))
    if pitch != h:
        codes = codes[:, :h]
    return (codes, scales.t()) if total is None else (codes, scales.t(), total.view(x.shape))


@functools.lru_cache(maxsize=1024)
def _norm_bytes(n: int, h: int) -> int:
    b = C.c_int64()
    _call(L.load().orda_rms_norm_backward_workspace, n, h, C.byref(b))
    return b.value


def rms_norm_backward(grad_out, total, weight, *, grad_total=None, eps: float = 1e-6, weight_offset: float = 0.0,
                      grad_x: bool = True, grad_weight: bool = True) -> Tuple:
    """``(grad_x, grad_weight)`` of ``rms_norm``, given the gradient into its result, ``total``
    (``t`` as it returned it; ``x`` where there was no residual) and, where the sum is
    used beside the norm, the gradient into ``t``. ``grad_x``, in x's type, is also the
    residual's gradient; ``grad_weight`` is summed over the rows in float32, in an order
    that the sizes fix, and rounded once to the weight's type. None where not asked for.
    """
    a, t, w, _ = _norm_args(total, weight, None, eps, weight_offset)
    if grad_out is None:
        raise OrdaError("grad_out must be a GPU tensor")
    for g, what in ((grad_out, "grad_out"), (grad_total, "grad_total")):
        if g is not None and (_gpu_tensor(g, what).shape != total.shape or g.dtype != t.dtype):
            raise OrdaError(f"{what} must have the shape and dtype of total")
    gx, gw = _NormGrad(a, t, w, grad_x, grad_weight).run(t, w, grad_out, grad_total)
    return gx.view(total.shape) if gx is not None else None, gw


def _without_residual(a: bytes) -> bytes:
    """orda_rms_norm of a contiguous sum, given that of the rows."""
    n, h = _ROWS.unpack_from(a)[1:3]
    return a[:24] + struct.pack("=q", h) + a[32:40] + bytes(40) + a[80:]


class _NormGrad:
    """A backward call of a matrix like t, a weight like w and orda_rms_norm, made ready:
    its arguments but for the addresses. It holds no device memory; gradients and scratch
    are made when it runs, from the pool of the stream or the graph that it runs in."""
    __slots__ = "buf", "at", "want_x", "want_w", "bytes", "device", "shape", "values", "dtype", "weight"

    def __init__(self, a: bytes, t, w, want_x: bool, want_w: bool):
        self.shape, self.values = t.shape, t.numel()
        n, h = t.shape
        self.device, self.dtype, self.weight = t.device, t.dtype, w.dtype
        self.want_x, self.want_w = want_x, want_w
        self.bytes = _norm_bytes(n, h)
        kind = _DTYPES[t.dtype]
        self.buf, self.at = _packed(a + _NORM_GRADS.pack(0, n, h, h, kind, L.DEVICE, 0, n, h, h, kind, L.DEVICE,
                                                         0, n, h, h, kind, L.DEVICE,
                                                         0, 1, h, h, _DTYPES[w.dtype], L.DEVICE))

    def takes(self, t, w) -> bool:
        """Whether they are as the sum and the weight that it was made for, but for their place."""
        return (t.dtype is self.dtype and w.dtype is self.weight and t.numel() == self.values
                and w.shape == self.shape[1:] and t.is_contiguous() and w.is_contiguous())

    def run(self, t, w, g, gt):
        """(grad_x, grad_weight), given a sum and a weight that it `takes` and plain gradients
        of t's number of values and dtype."""
        torch, buf, put = _torch(), self.buf, _ADDRESS.pack_into
        index, gx, gw = self.device.index, None, None
        if not index == t.get_device() == w.get_device() == g.get_device() or (gt is not None and gt.get_device() != index):
            raise OrdaError(f"weight and gradients must be on {self.device}")
        if not g.is_contiguous():
            g = _rows(g, self.shape[1], "grad_out")
            _ROWS.pack_into(buf, 136, *_fields(g, "grad_out"))
        if gt is not None:
            if not gt.is_contiguous():
                gt = _rows(gt, self.shape[1], "grad_total")
                _ROWS.pack_into(buf, 176, *_fields(gt, "grad_total"))
            put(buf, 176, gt.data_ptr())
        put(buf, 0, t.data_ptr())
        put(buf, 80, w.data_ptr())
        put(buf, 136, g.data_ptr())
        if self.want_x:
            gx = torch.empty(self.shape, dtype=self.dtype, device=self.device)
            put(buf, 216, gx.data_ptr())
        if self.want_w:
            gw = torch.empty_like(w)
            put(buf, 256, gw.data_ptr())
        ws = _bytes(self.bytes, self.device)
        at = self.at
        _check(L.load().orda_rms_norm_backward(index, torch._C._cuda_getCurrentRawStream(index), at, at + 136, at + 176,
                                               at + 216, at + 256, ws.data_ptr(), self.bytes, _message(), 512))
        return gx, gw


# ------------------------------------------------------------------ gradient norm and clipping
def _view(g, what: str):
    """(rows, cols, pitch) of a tensor's memory: one row where it is dense, in
    whatever order of its dimensions."""
    n = g.numel()
    if g.is_contiguous():
        return 1, n, n
    at = 1
    for stride, size in sorted((s, k) for k, s in zip(g.shape, g.stride()) if k > 1):
        if stride != at:
            break
        at *= size
    else:
        return 1, n, n
    if g.dim() == 2 and _is_matrix(g):
        return g.size(0), g.size(1), g.stride(0)
    if g.dim() == 2 and _is_matrix(g.t()):
        return g.size(1), g.size(0), g.stride(1)
    raise OrdaError(f"{what} must be dense, or a matrix with adjacent columns or rows")


@functools.lru_cache(maxsize=64)
def _gradient_table(n: int):
    return struct.Struct("=" + n * 2 * _TENSOR)   # orda_gradient


def _plain_gradients(grads, out, index, unwritten):
    """The table of contiguous gradients and destinations, as most are (37 us for 37 of
    both, 56 with the checks below); None where one is anything else. unwritten: leaves
    that require a gradient are refused."""
    torch = _torch()
    kinds = torch.Tensor, torch.nn.Parameter
    dtypes = {torch.float32: L.F32, torch.bfloat16: L.BF16}
    recording = torch.is_grad_enabled()
    fields = []
    try:
        for g, o in zip(grads, grads if out is None else out):
            if type(g) not in kinds or g.get_device() != index or not g.is_contiguous() or g.is_neg():
                return None
            if unwritten and g.requires_grad and g.is_leaf:
                return None
            p, n = g.data_ptr(), g.numel()
            if not p and n:
                return None
            fields += p, 1, n, n, dtypes[g.dtype], 1
            if out is None:
                fields += _NO_TENSOR
                continue
            if (type(o) not in kinds or o.get_device() != index or not o.is_contiguous() or o.is_neg()
                    or o.shape != g.shape or (recording and o.requires_grad)):
                return None
            p = o.data_ptr()
            if not p and n:
                return None
            fields += p, 1, n, n, dtypes[o.dtype], 1
    except (KeyError, RuntimeError):
        return None
    return fields


def _gradients(grads, out, scale: bool):
    """(orda_gradient array, the gradients, device, destinations). scale: they are written."""
    torch = _torch()
    grads = list(grads)
    if out is None:
        grads = [g for g in grads if g is not None]
        to = (None,) * len(grads)
    else:
        out = to = list(out)
        if len(out) != len(grads):
            raise OrdaError(f"out must have {len(grads)} tensors")
    if not grads:
        raise OrdaError("there are no gradients")
    device = _gpu_tensor(grads[0], "gradient 0").device
    recording = torch.is_grad_enabled()
    unwritten = scale and recording and out is None
    fields = _plain_gradients(grads, out, device.index, unwritten)
    if fields is not None:
        return _gradient_table(len(grads)).pack(*fields), grads, device, out
    fields = []
    for i, (g, o) in enumerate(zip(grads, to)):
        _same_device(device, **{f"gradient {i}": _gpu_tensor(g, f"gradient {i}")})
        r, c, ld = _view(g, f"gradient {i}")
        if unwritten and g.requires_grad and g.is_leaf:
            raise OrdaError(f"gradient {i} is a leaf that requires a gradient: it is not written in place")
        fields += g.data_ptr(), r, c, ld, _dtype(g, f"gradient {i}"), L.DEVICE
        if out is None:
            fields += _NO_TENSOR
            continue
        _same_device(device, **{f"out {i}": _gpu_tensor(o, f"out {i}")})
        if o.shape != g.shape or not ((o.is_contiguous() and g.is_contiguous()) or o.stride() == g.stride()):
            raise OrdaError(f"out {i} must have the shape and strides of gradient {i}")
        if recording and o.requires_grad:
            raise OrdaError(f"out {i} must not require a gradient")
        fields += o.data_ptr(), r, c, ld, _dtype(o, f"out {i}"), L.DEVICE
    return _gradient_table(len(grads)).pack(*fields), grads, device, out


@functools.lru_cache(maxsize=64)
def _clip_bytes(n: int) -> int:
    b = C.c_int64()
    _call(L.load().orda_clip_gradients_workspace, n, C.byref(b))
    return b.value


def gradient_norm(grads):
    """The 2-norm of all gradients together, a 0-dim float32 tensor. Gradients are
    float32 or bfloat16 GPU tensors of any shape, dense in any order or matrices
    with adjacent columns; None is skipped. Squares and sums are formed in 64 bits."""
    torch = _torch()
    a, grads, device, _ = _gradients(grads, None, False)
    b = _clip_bytes(len(grads))
    ws = _bytes(b, device)
    norm = torch.empty((), dtype=torch.float32, device=device)
    _call(L.load().orda_gradient_norm, device.index, _stream(device), a, len(grads), norm.data_ptr(), ws.data_ptr(), b)
    return norm


def clip_gradients(grads, max_norm: float, *, eps: float = 1e-6, out=None):
    """Scales all gradients by ``min(1, max_norm / (norm + eps))`` and returns their
    ``gradient_norm`` before that.

    In place, where nothing is written if the factor is 1; or to the tensors of ``out``,
    of the same shapes and strides, float32 or bfloat16, whatever the factor (the
    gradients then stay as they are, and none may be None). A norm that is NaN makes
    all of them NaN; the factor is 1 wherever ``norm + eps <= max_norm``, infinite ones
    included. Does not wait for the device. Tensors that are written share no
    memory with others of the call, and while torch records none is a leaf that requires
    a gradient (a parameter in its gradient's place)."""
    torch = _torch()
    a, grads, device, out = _gradients(grads, out, True)
    b = _clip_bytes(len(grads))
    ws = _bytes(b, device)
    norm = torch.empty((), dtype=torch.float32, device=device)
    try:
        _call(L.load().orda_clip_gradients, device.index, _stream(device), a, len(grads), max_norm, eps, norm.data_ptr(),
              ws.data_ptr(), b)
    except (C.ArgumentError, OverflowError):
        raise OrdaError("max_norm and eps must be numbers") from None
    torch.autograd.graph.increment_version(grads if out is None else out)   # written in place
    return norm


# ------------------------------------------------------------------ drawing tokens
_SAMPLING = struct.Struct("=" + _TENSOR + "5Q3fi")   # orda_sampling


def _per_row(value, n: int, shape, device, what: str, dtype, none):
    """(tensor or None, the one value)."""
    if value is None:
        return None, none
    if type(value) is float or type(value) is int:
        return None, value
    torch = _torch()
    if not isinstance(value, torch.Tensor):
        return None, value
    v = _gpu_tensor(value, what)
    _same_device(device, **{what: v})
    if v.shape != shape:
        raise OrdaError(f"{what} must be a number or of shape {list(shape)}")
    if dtype == torch.int32:
        if v.dtype not in (torch.int32, torch.int64):
            raise OrdaError(f"{what} must be int32 or int64, got {v.dtype}")
        if v.dtype == torch.int64:
            v = v.clamp(0, 2 ** 31 - 1).to(torch.int32)
    elif v.dtype != torch.float32:
        raise OrdaError(f"{what} must be float32, got {v.dtype}")
    return v.reshape(-1).contiguous(), none


@functools.lru_cache(maxsize=1024)
def _sample_bytes(n: int, v: int, dtype: int) -> int:
    b = C.c_int64()
    _call(L.load().orda_sample_tokens_workspace, n, v, dtype, C.byref(b))
    return b.value


def sample_tokens(logits, uniform, *, temperature=1.0, top_k=None, top_p=None, min_p=None) -> Tuple:
    """One token of each row of ``logits`` [..., V] (float32 or bfloat16) by that row's
    number of ``uniform`` [...] (float32, in [0, 1)): ``(tokens, logprobs)``, int64 and
    float32 [...].

    A token's mass is ``exp((x - max) / temperature)``. Of the tokens in descending order
    (equal logits: the lowest first) are kept the first ``top_k``; of those the ones whose
    mass before them is below ``top_p`` times the mass of all of those; of those the ones
    whose mass is at least ``min_p`` times the largest; the first always. The token is the
    first in the vocabulary's order up to which the kept masses add to more than
    ``uniform`` times their sum, its log-probability that of its share of the sum.
    ``temperature`` 0 gives the largest logit, the lowest such token, with log-probability
    0. Masses and sums are formed in 64 bits.

    Each parameter is a number, or a tensor [...] with a row's own (float32, ``top_k``
    int32 or int64); ``None`` and ``top_k <= 0`` filter nothing. A row with a NaN, without
    a logit over -infinity, or with a parameter of a tensor that is out of range
    (temperature negative or not finite, ``top_p`` or ``min_p`` NaN, ``uniform`` outside
    [0, 1]) gets token -1 and log-probability NaN.
    """
    torch = _torch()
    x = _gpu_tensor(logits, "logits")
    if x.dim() < 1:
        raise OrdaError("logits must be [..., V]")
    shape, v = x.shape[:-1], x.size(-1)
    if v < 1:
        raise OrdaError("logits must have columns")
    m = _rows(x, v, "logits")
    n = m.size(0)
    u = _gpu_tensor(uniform, "uniform")
    _same_device(m.device, uniform=u)
    if u.dtype != torch.float32 or u.shape != shape:
        raise OrdaError(f"uniform must be float32 {list(shape)}")
    if u.dim() != 1 or not u.is_contiguous():
        u = u.reshape(-1).contiguous()
    d = m.device
    t, t1 = _per_row(temperature, n, shape, d, "temperature", torch.float32, 1.0)
    k, k1 = _per_row(top_k, n, shape, d, "top_k", torch.int32, 0)
    p, p1 = _per_row(top_p, n, shape, d, "top_p", torch.float32, 1.0)
    q, q1 = _per_row(min_p, n, shape, d, "min_p", torch.float32, 0.0)
    f = _fields(m, "logits")
    try:
        a = _SAMPLING.pack(*f, u.data_ptr(), t.data_ptr() if t is not None else 0, p.data_ptr() if p is not None else 0,
                           q.data_ptr() if q is not None else 0, k.data_ptr() if k is not None else 0, t1, p1, q1,
                           max(0, min(operator.index(k1), 2 ** 31 - 1)))
    except (struct.error, OverflowError, TypeError):
        raise OrdaError("temperature, top_p and min_p must be numbers within float32, top_k a whole number") from None
    b = _sample_bytes(n, v, f[4])
    ws = _bytes(b, d)
    tokens = torch.empty(shape, dtype=torch.int64, device=d)
    logprobs = torch.empty_like(u) if len(shape) == 1 else torch.empty(shape, dtype=torch.float32, device=d)
    _buf, at = _packed(a)
    _check(L.load().orda_sample_tokens(d.index, _stream(d), at, tokens.data_ptr(), logprobs.data_ptr(), ws.data_ptr(), b,
                                       _message(), 512))
    return tokens, logprobs
