"""Operators on compressed weights: products with a 2-D float16 or bfloat16 weight that stays a blob.

A model whose weights are kept compressed in GPU memory is used through these calls instead of
decompress_tensor followed by a product: the weight is decoded a piece of rows at a time into a
bounded scratch buffer (or, for a single token, only in the decoder's registers) and is frozen, so
gradients go to the other operands.  The reference has no counterpart.

Blobs must be on the GPU of the other operands.  A blob that compress_tensor(..., readback_to_cpu=
False) or upload_blob returned carries its header, and the calls neither read anything back nor
synchronise, so they can be captured into a CUDA graph; another GPU blob costs one header read per
call.  Decoding errors are reported by last_decode_status(), as for decompress_tensor (a malformed
chunk counts as zeros); after a backward pass that decoded, it reports that pass and its forward pass,
to the thread that called the operator.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._codec import (_CODES, _FIXED, _FLAG_REORDER, _FLAG_STORED, _MAX_NDIM, _REORDER, _check_device, _gpu,
                     _known_header, _on, _parse_header, _remember, _set_status, _statuses, _stream, _upload)

_ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}
_MAX_TOP = 256
_MAX_DIM = 1 << 31
_MIN_TEMPERATURE, _MAX_TEMPERATURE = 2.0**-20, 2.0**20  # its square and inverse stay far inside float32
_ENTRIES = {name: (getattr(_lib.lib, name + "_temp_bytes"), getattr(_lib.lib, name))
            for name in ("zn_linear", "zn_linear_grad", "zn_loss")}


def upload_blob(blob: torch.Tensor, *, compute_device: torch.device | str | None = None) -> torch.Tensor:
    """A GPU blob with its header remembered, from a blob on the CPU or the GPU (returned as it is
    when it is a GPU blob that carries its header already): what a program that loads blobs from
    storage does once, so that decompressing or multiplying with them reads nothing back."""
    compute_device = _check_device(compute_device)
    _check_blob(blob)
    device = _gpu(blob, compute_device)
    if blob.device == device and _known_header(blob) is not None:
        return blob
    dtype, shape, flags, chunk_bytes, _, n = _read_header(blob)
    # A tensor of inference mode has no version counter, which the record needs.
    with _on(device), torch.inference_mode(False):
        if blob.is_cuda:
            out = blob.detach().to(device, non_blocking=True).clone(memory_format=torch.contiguous_format)
        else:
            src = blob.detach().contiguous()
            out = _upload(src, device)
            if src.is_pinned():  # asynchronous, but the caller may reuse the blob once we return
                torch.cuda.current_stream(device).synchronize()
    return _remember(out, dtype, shape, flags, chunk_bytes, n)


def _check_blob(blob: torch.Tensor) -> None:
    if blob.dtype != torch.uint8 or blob.dim() != 1:
        raise ValueError("blob must be a 1-D uint8 tensor")


def _read_header(blob: torch.Tensor) -> tuple:
    """(dtype, shape, flags, chunk_bytes, n_comp, n) of a blob without a record, checked."""
    if blob.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a blob without a remembered header cannot be read during stream capture: "
                           "pass it through upload_blob first")
    prefix = blob.detach()[: _FIXED.size + 8 * _MAX_NDIM].cpu().contiguous()
    dtype, shape, flags, chunk_bytes, n_comp, n = _parse_header(prefix.numpy())
    stored = bool(flags & _FLAG_STORED)
    if any(d < 0 for d in shape) or math.prod(shape) != n or (not stored and n and chunk_bytes <= 0):
        raise ValueError("not a cuzipnn blob")
    if stored and blob.numel() < _FIXED.size + 8 * len(shape) + n * dtype.itemsize:
        raise ValueError("blob is truncated")
    return dtype, tuple(shape), flags, chunk_bytes, n_comp, n


class _Weight:
    """A blob as the weight of a product with `x`: its fields checked against `x` (no GPU work), then,
    by place(), its description for the C calls."""

    __slots__ = ("blob", "rows", "cols", "device", "dtype", "chunk_bytes", "desc")

    def __init__(self, blob: torch.Tensor, x: torch.Tensor, name: str):
        _check_blob(blob)
        known = _known_header(blob)
        if known is not None:
            dtype, shape, flags, chunk_bytes, _ = known
        else:
            dtype, shape, flags, chunk_bytes, _, _ = _read_header(blob)
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"the blob holds {dtype}: float16 or bfloat16 weights are supported")
        if x.dtype != dtype:
            raise TypeError(f"{name} has dtype {x.dtype}, the blob holds {dtype}")
        if len(shape) != 2 or not all(0 < d < _MAX_DIM for d in shape):
            raise ValueError(f"the blob holds a tensor of shape {tuple(shape)}, a weight has two nonempty dimensions")
        stored = bool(flags & _FLAG_STORED)
        if not stored and (bool(flags & _FLAG_REORDER) != (dtype in _REORDER) or chunk_bytes % 8):
            raise ValueError("not a cuzipnn blob")
        self.rows, self.cols = shape
        if x.dim() < 1 or x.shape[-1] != self.cols:
            raise ValueError(f"{name} has shape {tuple(x.shape)}, the weight has {self.cols} columns")
        if x.numel() // self.cols >= _MAX_DIM:
            raise ValueError(f"{name} has too many rows")
        self.device, self.dtype = x.device, dtype
        self.chunk_bytes = 0 if stored else chunk_bytes
        self.blob = blob

    def place(self, name: str) -> None:
        if self.device.type != "cuda":
            raise ValueError(f"{name} must be a CUDA tensor")
        if self.blob.device != self.device:
            raise ValueError(f"the blob is on {self.blob.device}, {name} on {self.device}")
        b = self.blob
        if not b.is_contiguous() or b.data_ptr() % 8:
            with _on(self.device):
                self.blob = b = b.clone(memory_format=torch.contiguous_format)
        self.desc = _lib.Weight(b.data_ptr(), b.numel(), self.rows, self.cols, self.chunk_bytes, _CODES[self.dtype])

    def call(self, name: str, query: tuple, args: tuple, status: int) -> None:
        """Run entry point `name` on the device's current stream: scratch from <name>_temp_bytes
        (with the `query` arguments), then (weight, *args, status, scratch, stream).  `status`: the
        address of its status word."""
        w = ctypes.byref(self.desc)
        temp_bytes, run = _ENTRIES[name]
        nbytes = temp_bytes(w, *query)
        temp = torch.empty(nbytes or 1, dtype=torch.uint8, device=self.device)
        status_code = run(w, *args, status, temp.data_ptr(), nbytes, _stream(self.device))
        if status_code:
            _lib.check(status_code, name)


def _rows(t: torch.Tensor, cols: int) -> tuple[torch.Tensor, int]:
    """`t` as rows of `cols` adjacent elements, and the pitch between them (a copy if it must be)."""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    if t.is_contiguous() and t.shape[0] > 1:
        return t, cols
    if (cols > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < cols):
        t = t.contiguous()
    # One row has any pitch: the next multiple of 8, which the kernels read in place.
    return t, t.stride(0) if t.shape[0] > 1 else (cols + 7) & ~7


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _check_tangent(name: str, t: torch.Tensor) -> None:
    """Operands with a forward-mode tangent: they need no gradient, so the tangent would be lost."""
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{name} carries a forward-mode derivative: operators on blobs have none")


def _linear_forward(w: _Weight, x, shape, bias, act: int, residual, want_slope: bool, status):
    y = torch.empty(shape, dtype=w.dtype, device=w.device)
    slope = torch.empty(shape, dtype=torch.float16, device=w.device) if want_slope else None
    x2, ldx = _rows(x, w.cols)
    r2, ldr = (None, 0) if residual is None else _rows(residual, w.rows)
    b = None if bias is None else bias.contiguous()
    tokens = x2.shape[0]
    if tokens:
        w.call("zn_linear", (x2.data_ptr(), ldx, tokens),
               (x2.data_ptr(), ldx, tokens, _ptr(b), act, _ptr(r2), ldr, y.data_ptr(), _ptr(slope)), status.data_ptr())
    else:
        status.zero_()
    return y, slope


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, blob, bias, residual, w, shape, act):
        status = torch.empty(2, dtype=torch.int32, device=w.device)  # of this pass, and of the backward pass
        want = act != 0 and (ctx.needs_input_grad[0] or ctx.needs_input_grad[2])
        y, slope = _linear_forward(w, x, shape, bias, act, residual, want, status)
        _set_status(w.device, status, 1)
        ctx.w, ctx.status, ctx.statuses, ctx.x_shape = w, status, _statuses(), x.shape
        ctx.save_for_backward(blob, slope)  # the blob: an in-place change before backward raises
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w = ctx.w
        _, slope = ctx.saved_tensors
        need_x, _, need_b, need_r = ctx.needs_input_grad[:4]
        dx = torch.empty(ctx.x_shape, dtype=w.dtype, device=w.device) if need_x else None
        db = torch.empty(w.rows, dtype=w.dtype, device=w.device) if need_b else None
        if not dy.numel():
            return dx, None, db.zero_() if need_b else None, dy if need_r else None, None, None, None
        if need_x or need_b:
            with _on(w.device):
                g, ldy = _rows(dy, w.rows)
                w.call("zn_linear_grad",
                       (g.data_ptr(), ldy, g.shape[0], int(slope is not None), int(need_x), int(need_b)),
                       (g.data_ptr(), ldy, g.shape[0], _ptr(slope), _ptr(dx), _ptr(db)),
                       ctx.status.data_ptr() + 4)
                if need_x:  # it decoded; the engine's thread reports to the one that called the layer
                    ctx.statuses[w.device.index] = (ctx.status, 2, _stream(w.device))
        return dx, None, db, dy if need_r else None, None, None, None


def blob_linear(
    x: torch.Tensor,
    blob: torch.Tensor,
    *,
    bias: torch.Tensor | None = None,
    activation: str | None = None,
    residual: torch.Tensor | None = None,
) -> torch.Tensor:
    """activation(x W^T + bias) + residual with the compressed weight W [rows, cols] of `blob`.

    `x` is [..., cols] on the blob's GPU, of the weight's dtype (float16 or bfloat16), with any
    strides; the result is [..., rows].  `bias` [rows] and `residual` (exactly the result's shape)
    have the same dtype and device.  `activation` is None, "relu", "gelu" (erf), "gelu_tanh" or
    "silu".  Products are summed in 32 bits and the result is rounded once.

    Differentiable in x, bias and residual (the weight is frozen).  With an activation the forward
    pass keeps its derivative for the backward pass, in 16 bits (off by 2^-11 of itself at most; below
    2^-29 by 2^-40), and there the input's gradient is taken of the product of both in the dtype.  The
    weight is decoded again there."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(map(str, _ACTIVATIONS))}, not {activation!r}")
    w = _Weight(blob, x, "x")
    _check_tangent("x", x)
    shape = (*x.shape[:-1], w.rows)
    for name, t, expected in (("bias", bias, (w.rows,)), ("residual", residual, shape)):
        if t is None:
            continue
        if t.dtype != w.dtype:
            raise TypeError(f"{name} has dtype {t.dtype}, the blob holds {w.dtype}")
        if t.shape != expected:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {expected}")
        if t.device != w.device:
            raise ValueError(f"{name} is on {t.device}, x on {w.device}")
        _check_tangent(name, t)
    w.place("x")
    act = _ACTIVATIONS[activation]
    with _on(w.device):
        if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)
                                        or (residual is not None and residual.requires_grad)):
            return _Linear.apply(x, blob, bias, residual, w, shape, act)
        status = torch.empty(1, dtype=torch.int32, device=w.device)
        y, _ = _linear_forward(w, x, shape, bias, act, residual, False, status)
        _set_status(w.device, status)
        return y


def _loss_forward(w: _Weight, hidden, ids, logits, top, ignore_index, temperature, reduction, want_grad, status):
    """(loss, the rows' own gradients in 32 bits or None, state)"""
    h, ldh = _rows(hidden, w.cols)
    tokens = h.shape[0]
    loss = torch.empty(tokens if reduction == 2 else (), dtype=torch.float32, device=w.device)
    unit = torch.empty((tokens, w.cols), dtype=torch.float32, device=w.device) if want_grad else None
    state = torch.empty(_lib.lib.zn_loss_state_bytes(tokens, top) or 1, dtype=torch.uint8, device=w.device)
    if tokens:
        w.call("zn_loss", (h.data_ptr(), ldh, tokens, top, int(want_grad)),
               (h.data_ptr(), ldh, tokens, ids.data_ptr(), _ptr(logits), top, ignore_index, temperature, reduction,
                loss.data_ptr(), _ptr(unit), state.data_ptr()), status.data_ptr())
    else:
        loss.zero_()
        status.zero_()
    return loss, unit, state


class _Loss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, w, ids, logits, top, ignore_index, temperature, reduction):
        status = torch.empty(1, dtype=torch.int32, device=w.device)
        loss, unit, state = _loss_forward(w, hidden, ids, logits, top, ignore_index, temperature, reduction, True,
                                          status)
        _set_status(w.device, status)
        ctx.args = (_CODES[w.dtype], w.dtype, hidden.shape, top, reduction)
        ctx.save_for_backward(unit, state)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        unit, state = ctx.saved_tensors
        code, dtype, shape, top, reduction = ctx.args
        dh = torch.empty(shape, dtype=dtype, device=unit.device)
        if dh.numel():
            with _on(unit.device):
                g = grad.float().contiguous()
                _lib.check(_lib.lib.zn_loss_grad(code, unit.shape[0], unit.shape[1], top, reduction, state.data_ptr(),
                                                 unit.data_ptr(), g.data_ptr(), dh.data_ptr(), _stream(unit.device)),
                           "zn_loss_grad")
        return dh, *(None,) * 7


def _loss(hidden, w, ids, logits, top, ignore_index, temperature, reduction, shape):
    _check_tangent("hidden", hidden)
    w.place("hidden")
    red = _REDUCTIONS[reduction]
    args = (ids, logits, top, ignore_index, temperature, red)
    with _on(w.device):
        if torch.is_grad_enabled() and hidden.requires_grad:
            loss = _Loss.apply(hidden, w, *args)
        else:
            status = torch.empty(1, dtype=torch.int32, device=w.device)
            loss, _, _ = _loss_forward(w, hidden, *args, False, status)
            _set_status(w.device, status)
        return loss.reshape(shape) if red == 2 else loss


def _check_reduction(reduction: str) -> None:
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, not {reduction!r}")


def _check_ids(name: str, t: torch.Tensor, shape: tuple[int, ...], w: _Weight) -> None:
    if t.dtype != torch.int64:
        raise TypeError(f"{name} must be int64, not {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    if t.device != w.device:
        raise ValueError(f"{name} is on {t.device}, hidden on {w.device}")


def blob_cross_entropy(
    hidden: torch.Tensor,
    blob: torch.Tensor,
    targets: torch.Tensor,
    *,
    ignore_index: int = -100,
    reduction: str = "mean",
) -> torch.Tensor:
    """Softmax cross entropy of the logits hidden W^T with the compressed head W [vocabulary, cols]
    of `blob`, without keeping the logits.

    `hidden` is [..., cols] (the weight's dtype, any strides), `targets` int64 [...].  Returns
    float32: the mean over the rows whose target is not ignore_index (0 when there is none), their
    "sum", or with "none" one loss per row (0 where ignored).  Any other target outside the
    vocabulary makes the row's loss and gradient NaN.

    Differentiable in hidden: where hidden requires a gradient, the forward pass computes it with the
    loss, in the same pass over the vocabulary, a piece at a time, and keeps it in 32 bits (tokens x
    cols).  The softmax's weights are rounded to the dtype before the product with a piece, except
    at the row's own target (sums are in 32 bits), where softmax - 1 is taken from the other weights'
    sum, so that confident rows are as exact as others; in float16, weights below about 2^-33 of the
    largest vanish.  Ignored rows get zero gradients whatever they hold."""
    _check_reduction(reduction)
    w = _Weight(blob, hidden, "hidden")
    shape = tuple(hidden.shape[:-1])
    _check_ids("targets", targets, shape, w)
    ignore_index = int(ignore_index)
    if not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError(f"ignore_index must be an int64, not {ignore_index}")
    ids = targets.detach().reshape(-1).contiguous()
    return _loss(hidden, w, ids, None, 1, ignore_index, 1.0, reduction, shape)


def blob_distillation(
    hidden: torch.Tensor,
    blob: torch.Tensor,
    teacher_logits: torch.Tensor,
    teacher_ids: torch.Tensor,
    *,
    temperature: float = 1.0,
    reduction: str = "mean",
) -> torch.Tensor:
    """Distillation loss temperature^2 * KL(q || softmax(hidden W^T / temperature)) per row, from a
    teacher's top logits, with the compressed head W [vocabulary, cols] of `blob` and without keeping
    the student's logits.

    `teacher_ids` int64 and `teacher_logits` (a float type) are [..., top] with top in [1, 256]: the
    ids of the teacher's best tokens, in any order, and their logits; q is their softmax at the same
    temperature, over these entries alone.  An id < 0 marks an empty entry (rows may be of different
    lengths) and an id given twice counts twice.  A row without entries, or whose logits are all
    -inf, does not count: its loss and gradient are 0 and a "mean" leaves it out (0 when no row
    counts).  An id past the vocabulary makes the row's loss and gradient NaN.

    Returns float32, "mean", "sum" or per row ("none").  Differentiable in hidden, as
    blob_cross_entropy; the teacher is a constant."""
    _check_reduction(reduction)
    temperature = float(temperature)
    if not _MIN_TEMPERATURE <= temperature <= _MAX_TEMPERATURE:
        raise ValueError(f"temperature must be between {_MIN_TEMPERATURE} and {_MAX_TEMPERATURE}, not {temperature}")
    w = _Weight(blob, hidden, "hidden")
    if teacher_ids.dim() < 1 or not 1 <= teacher_ids.shape[-1] <= _MAX_TOP:
        raise ValueError(f"teacher_ids must have between 1 and {_MAX_TOP} entries per row")
    shape, top = tuple(hidden.shape[:-1]), teacher_ids.shape[-1]
    _check_ids("teacher_ids", teacher_ids, (*shape, top), w)
    if not teacher_logits.dtype.is_floating_point:
        raise TypeError(f"teacher_logits must be a float type, not {teacher_logits.dtype}")
    if tuple(teacher_logits.shape) != (*shape, top):
        raise ValueError(f"teacher_logits has shape {tuple(teacher_logits.shape)}, expected {(*shape, top)}")
    if teacher_logits.device != w.device:
        raise ValueError(f"teacher_logits is on {teacher_logits.device}, hidden on {w.device}")
    ids = teacher_ids.detach().reshape(-1, top).contiguous()
    logits = teacher_logits.detach().reshape(-1, top)
    if logits.dtype == torch.float64:  # less their maximum first, or 32 bits would lose the small differences of large ones
        peak = logits.masked_fill(ids < 0, -math.inf).amax(1, keepdim=True)
        logits = logits - torch.where(peak.isfinite(), peak, 0.0)
    logits = logits.float().contiguous()
    return _loss(hidden, w, ids, logits, top, 0, temperature, reduction, shape)
