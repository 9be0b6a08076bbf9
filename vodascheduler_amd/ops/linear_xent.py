"""Softmax cross-entropy of a vocabulary head without its logits (csrc/hip/linear_xent.hip).

``linear_cross_entropy(x, weight, labels, bias, num_classes, ignore_index)`` is
``softmax_cross_entropy(x @ weight.T + bias, labels, num_classes, ignore_index)`` (ops/xent.py) in one
op: the head's product and its loss together, so that the [rows, vocab] logits never reach memory.
It returns the same ``(loss, correct, n_valid)``: the mean loss over the labelled rows, the number of
those whose first-maximum class is the label, and their count, all device tensors (no host sync,
hipGraph-capturable).

* The forward keeps two numbers a row, and the labelled rows of ``x`` together (in a buffer of all rows' size:
  how many are labelled stays on the device; fp32: three planes, 6 bytes an element), with the bias in fp32.
  The backward computes the logits again, piece by piece of the vocabulary, and leaves their gradient in a
  workspace of at most ``G_BYTES`` (512 MB; one piece has at least 256 columns); beside it stand the split sums
  of dx and dw and, in fp32, the planes of ``weight``.  BERT-base's MLM head over 8192 positions would keep
  0.5 GB of bf16 logits and as much gradient.
* A row whose label is ``ignore_index`` or lies outside [0, num_classes) is left out before any
  product: it costs nothing, its gradient is exactly zero, and nothing that it holds (NaN, uninitialised
  padding) reaches the loss or a gradient.  A loss with every row ignored is 0 (PyTorch: NaN).
* ``weight`` rows from ``num_classes`` on are padding: outside the softmax, gradient zero.  A bias of
  -inf takes a class out.
* Types: bf16 or fp32 ``x`` and ``weight`` alike, ``bias`` of either; fp32 runs at fp32 accuracy (three
  bf16 planes an operand, which hold an element of 2^-110 or more by itself, whatever stands beside it) wherever
  the products stay finite.  An infinite or NaN input of a labelled row or of a class's
  weights makes the loss NaN or infinite, and such a row counts as not correct.  Anything else is refused on a GPU.
* Gradients of a weight and bias that the fused optimizer owns are summed straight into its flat
  buffer (ops/dense.py's contract), else returned.  Sums have a fixed order: the same call gives the
  same bits.  Only first derivatives.

The reference's head is a Dense layer with a softmax over the vocabulary and a sparse cross-entropy
(examples/py/tensorflow2/neural_machine_translation_with_transformer.py:191-315).
"""
from __future__ import annotations

from contextlib import nullcontext

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from ..utils.flat import flat_grad
from . import _native as N
from .dense import _direct, _ready


# most for G of one piece of the vocabulary in the backward.  Smaller pieces take more time: at 512 / 256 / 128 / 64 MB
# a translation batch (10240 x 256 x 15000) ran in 477 / 513 / 576 / 695 us
G_BYTES = 512 << 20


def _valid(labels: torch.Tensor, classes: int, ignore_index: int) -> torch.Tensor:
    return (labels != ignore_index) & (labels >= 0) & (labels < classes)


def linear_cross_entropy_ref(x: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                             bias: torch.Tensor | None = None, num_classes: int | None = None,
                             ignore_index: int = -100) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """PyTorch reference of :func:`linear_cross_entropy` (fp32; fp64 for fp64 inputs)."""
    C = weight.shape[0] if num_classes is None else num_classes
    dt = torch.promote_types(x.dtype, torch.float32)
    x, labels = x.reshape(-1, x.shape[-1]), labels.reshape(-1)
    rows = _valid(labels, C, ignore_index).nonzero()[:, 0]
    y = labels[rows]
    with torch.autocast(x.device.type, enabled=False):
        z = F.linear(x[rows].to(dt), weight[:C].to(dt), None if bias is None else bias[:C].to(dt))
        loss = F.cross_entropy(z, y, reduction="sum") / max(1, rows.numel())
    correct = (z.detach().argmax(1) == y).sum()
    return loss, correct, torch.tensor(rows.numel(), device=x.device)


def _rows16(w: torch.Tensor) -> torch.Tensor:
    """w with 16-byte rows of whole 16-byte vectors (bf16): w itself, or a zero-padded copy."""
    ld, step = w.stride()
    width = w.shape[1]
    if step == 1 and ld % 8 == 0 and ld >= width and width % 8 == 0 and w.data_ptr() % 16 == 0:
        return w
    # (not F.pad: it keeps a single row's stride, whatever that is)
    out = w.new_zeros(w.shape[0], -(-width // 8) * 8)
    out[:, :width] = w
    return out


# torch's own accessor, where it has one: 0.5 us instead of 3.5 in a call whose whole forward takes 30
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_HERE = nullcontext()


def _on(device: torch.device):
    """Context with the GPU ``device`` current (nothing to do where it is already)."""
    return _HERE if device.index == _current_device() else torch.cuda.device(device)


class _LinearXentFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, labels, C, ignore):
        h = N.hip()
        rows, K = x.shape
        V = weight.shape[0]
        f32 = x.dtype == torch.float32
        dev = x.device
        with _on(dev):
            nf, nb, kp, vpad, nd = h.linear_xent_sizes(rows, K, C, V, f32, G_BYTES)
            w = weight if f32 else _rows16(weight)
            ws = torch.empty(max(nf, 256), dtype=torch.uint8, device=dev)
            # what the backward needs, in one buffer, each part 256-byte aligned: x's compact rows, the
            # padded bias, each row's place, the labels, (max, 1 / sum), the device scalars
            at = [0]
            for n in ((6 if f32 else 2) * rows * kp, 4 * vpad, 4 * rows, 4 * rows, 8 * rows, nd):
                at.append(at[-1] + -(-n // 256) * 256)
            keep = torch.empty(at[-1], dtype=torch.uint8, device=dev)
            p = keep.data_ptr()
            p = [p + a for a in at]
            planes = torch.empty(6 * C * kp, dtype=torch.uint8, device=dev) if f32 else None
            loss = torch.empty((), dtype=torch.float32, device=dev)
            correct = torch.empty((), dtype=torch.int64, device=dev)
            n = torch.empty((), dtype=torch.int64, device=dev)
            h.linear_xent_fwd(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), N.ptr(bias),
                              N.DT_F32 if bias is None else N.dtype_code(bias.dtype), labels.data_ptr(), ignore, rows,
                              K, C, V, N.dtype_code(x.dtype), ws.data_ptr(), p[0], p[1], p[2], p[3], p[4], p[5],
                              N.ptr(planes), loss.data_ptr(), correct.data_ptr(), n.data_ptr(), N.stream_of(x))
        ctx.save_for_backward(weight, keep)
        ctx.at, ctx.dims, ctx.nb, ctx.kp = at, (rows, K, C, V), nb, kp
        ctx.params, ctx.g_bytes = (weight, bias), G_BYTES
        ctx.x_dtype = x.dtype
        ctx.mark_non_differentiable(correct, n)
        ctx.set_materialize_grads(False)  # no zero gradients for the two counts
        return loss, correct, n

    @staticmethod
    @once_differentiable
    def backward(ctx, gloss, _gc, _gn):
        if gloss is None:
            return None, None, None, None, None, None
        weight, keep = ctx.saved_tensors
        rows, K, C, V = ctx.dims
        wp, bp = ctx.params
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dev = weight.device
        f32 = ctx.x_dtype == torch.float32
        dx = dw = db = None
        with _on(dev):
            p = keep.data_ptr()
            p = [p + a for a in ctx.at]
            w = weight if f32 else _rows16(weight)
            if need_x:
                dx = torch.empty(rows, K, dtype=ctx.x_dtype, device=dev)
            # into the optimizer's flat gradients where it owns every gradient that is asked for
            direct = (need_w or need_b) and all(_direct(t) and flat_grad(t).dtype in (torch.float32, torch.bfloat16)
                                                for t, need in ((wp, need_w), (bp, need_b)) if need)
            if need_w:
                dw = flat_grad(wp) if direct else torch.empty(V, K, dtype=weight.dtype, device=dev)
            if need_b:
                db = flat_grad(bp) if direct else torch.empty(V, dtype=bp.dtype, device=dev)
            if not direct and C < V:
                for t in (dw, db):
                    if t is not None:
                        t[C:].zero_()
            ws = torch.empty(max(ctx.nb, 256), dtype=torch.uint8, device=dev)
            planes = torch.empty(6 * C * ctx.kp, dtype=torch.uint8, device=dev) if f32 else None
            N.hip().linear_xent_bwd(w.data_ptr(), w.stride(0), rows, K, C, V, N.dtype_code(ctx.x_dtype), ws.data_ptr(),
                                    p[0], p[1], p[2], p[3], p[4], p[5], N.ptr(planes), gloss.data_ptr(), N.ptr(dx),
                                    N.ptr(dw), dw.stride(0) if need_w else K, N.ptr(db),
                                    N.dtype_code(dw.dtype) if need_w else N.DT_F32,
                                    N.dtype_code(db.dtype) if need_b else N.DT_F32, bool(direct), ctx.g_bytes,
                                    N.stream_of(weight))
        if direct:
            if need_w:
                _ready(wp)
            if need_b:
                _ready(bp)
            dw = db = None
        return dx, dw, db, None, None, None


def _check(x, weight, labels, bias, C) -> None:
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_cross_entropy: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not multiply")
    if labels.numel() != x.numel() // max(1, x.shape[-1]):
        raise ValueError(f"linear_cross_entropy: {labels.numel()} labels for x {tuple(x.shape)}")
    if labels.dtype.is_floating_point or labels.dtype.is_complex or labels.dtype == torch.bool:
        raise TypeError(f"linear_cross_entropy: labels must be integers, got {labels.dtype}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"linear_cross_entropy: bias {tuple(bias.shape)} for weight {tuple(weight.shape)}")
    if x.shape[-1] < 1 or not 1 <= C <= weight.shape[0]:
        raise ValueError(f"linear_cross_entropy: {C} classes of weight {tuple(weight.shape)}")
    dev = x.device
    for t, nm in ((weight, "weight"), (labels, "labels"), (bias, "bias")):
        if t is not None and t.device != dev:
            raise ValueError(f"linear_cross_entropy: {nm} on {t.device}, x on {x.device}")


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                         bias: torch.Tensor | None = None, num_classes: int | None = None,
                         ignore_index: int = -100) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(loss, correct, n_valid)`` of the head ``x [.., K] @ weight [V, K].T + bias [V]`` over its first
    ``num_classes`` classes against integer ``labels`` (one a row of x); see the module docstring."""
    C = weight.shape[0] if num_classes is None else int(num_classes)
    _check(x, weight, labels, bias, C)
    dev = x.device
    if x.dtype != weight.dtype and torch.is_autocast_enabled(x.device.type):
        x = x.to(weight.dtype)
    # (a reshape that changes nothing would still be a node of the backward)
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if labels.dim() != 1:
        labels = labels.reshape(-1)
    if not x.is_cuda:
        return linear_cross_entropy_ref(x2, weight, labels, bias, C, ignore_index)
    if x.dtype not in (torch.float32, torch.bfloat16) or weight.dtype != x.dtype:
        raise TypeError(f"linear_cross_entropy: x and weight must both be fp32 or bf16, got {x.dtype}, {weight.dtype}")
    if bias is not None and bias.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"linear_cross_entropy: bias must be fp32 or bf16, got {bias.dtype}")
    if x2.shape[0] == 0:  # no rows: a zero that still has (zero) gradients
        with torch.autocast(dev.type, enabled=False):
            loss = F.linear(x2.float(), weight.float(), None if bias is None else bias.float()).sum()
        return loss, labels.new_zeros((), dtype=torch.int64), labels.new_zeros((), dtype=torch.int64)
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    if weight.stride(1) != 1:
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if labels.dtype != torch.int64 or not labels.is_contiguous():
        labels = labels.to(torch.int64).contiguous()
    return _LinearXentFn.apply(x2, weight, bias, labels, C, int(ignore_index))
