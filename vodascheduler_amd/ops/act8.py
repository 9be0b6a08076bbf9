"""Linear layer that keeps its input in 8 bits for the backward (csrc/hip/act8.hip).

``linear_act8(x, weight, bias, act)`` is ``F.linear(act(x), weight, bias)`` with ``act`` None or
``"gelu"`` (tanh form).  The product reads ``x`` itself; what autograd keeps is a checkpoint of ``x``:
e4m3 with one power-of-two scale for 32 features, 33 bytes for 32 features against 64 (bf16) or 128
(fp32), and with ``act="gelu"`` neither the GELU's output.  With ``c`` the value the checkpoint stands for

    dx = (dy W) act'(c)        dW = dy^T act(c)        db = sum dy

so ``dx`` of the plain form is exact and ``dW`` sees ``x`` to within e4m3's half step (2^-4 of a value).
BERT-base's FFN keeps 0.79 + 3.17 KB a token this way instead of 1.5 + 6 + 6 KB (bf16).

``act8_pack`` / ``act8_unpack`` are the checkpoint by itself: ``scale`` is the smallest power of two (at
least 2^-126) that keeps the block's largest finite value within 448, so the only rounding is e4m3's
(what would round past fp32's range stays at 240 2^120); infinities and NaN come back as NaN.

Types: bf16 or fp32 ``x`` and ``weight`` alike (fp32 at fp32 accuracy wherever the products stay
finite: three bf16 planes hold an element of 2^-110 or more by itself, whatever stands beside it; an infinite one gives NaN or infinity where it
takes part), ``bias`` of either.  Any sizes and row strides.  Gradients that the
fused optimizer owns go straight into its flat buffer (ops/dense.py's contract).  Without a gradient of
``weight`` and without the GELU no checkpoint is kept.  Only first derivatives.  ``Act8Linear`` is the
layer, with ``FusedLinear``'s parameters.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from ..utils.flat import flat_grad
from . import _native as N
from .dense import FusedLinear, _direct, _ready, colsum_accumulate_
from .ffn import gelu_tanh_grad_ref
from .linear_xent import _on, _rows16

BLOCK = 32
E4M3_MAX = 448.0
_F8, _E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _pack_ref(x2: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    rows, width = x2.shape
    kq = -(-width // BLOCK) * BLOCK
    v = F.pad(x2.float(), (0, kq - width)).view(rows, kq // BLOCK, BLOCK)
    fin = torch.isfinite(v)
    mant, exp = torch.frexp(torch.where(fin, v, 0).abs().amax(2, keepdim=True))  # [0.5, 1) 2^exp
    exp = torch.where(mant > 0, exp - 9 + (mant > E4M3_MAX / 512), -126).clamp(min=-126)
    most = torch.where(exp == 120, 240.0, E4M3_MAX)  # 256 2^120 is past fp32
    v = torch.minimum(torch.maximum(torch.ldexp(v, -exp), -most), most)
    q = torch.where(fin, v, torch.nan).to(_F8).view(rows, kq)
    return q, (exp.view(rows, kq // BLOCK) + 127).to(torch.uint8).view(_E8)


def _unpack_ref(q: torch.Tensor, scale: torch.Tensor, width: int, dtype: torch.dtype) -> torch.Tensor:
    v = q.float().view(*scale.shape, BLOCK)
    exp = scale.view(torch.uint8).to(torch.int32) - 127
    return torch.ldexp(v, exp[..., None]).flatten(-2)[..., :width].to(dtype)


def act8_pack(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Checkpoint of ``x`` [.., width]: ``(q [.., kq] float8_e4m3fn, scale [.., kq / 32]
    float8_e8m0fnu)``, kq = width rounded up to whole blocks of 32 (the rest is zero)."""
    _check_float("act8_pack", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"act8_pack: nothing to pack in {tuple(x.shape)}")
    x2 = x.detach().reshape(-1, x.shape[-1])
    rows, width = x2.shape
    kq = -(-width // BLOCK) * BLOCK
    if not x.is_cuda or rows == 0:
        q, s = _pack_ref(x2)
    else:
        if x2.stride(1) != 1:
            x2 = x2.contiguous()
        with _on(x.device):
            q = torch.empty(rows, kq, dtype=_F8, device=x.device)
            s = torch.empty(rows, kq // BLOCK, dtype=_E8, device=x.device)
            N.hip().act8_pack(x2.data_ptr(), x2.stride(0), rows, width, N.dtype_code(x.dtype), q.data_ptr(),
                              s.data_ptr(), N.stream_of(x))
    return q.view(*x.shape[:-1], kq), s.view(*x.shape[:-1], kq // BLOCK)


def act8_unpack(q: torch.Tensor, scale: torch.Tensor, width: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values a checkpoint stands for, [.., width] (exact in bf16 too, for values bf16 reaches)."""
    if q.dim() < 1 or q.dtype != _F8 or scale.dtype != _E8 or q.shape[:-1] != scale.shape[:-1] or q.device != scale.device:
        raise ValueError("act8_unpack: q and scale are not a checkpoint of act8_pack")
    if q.shape[-1] != BLOCK * scale.shape[-1] or not 0 < width <= q.shape[-1] or width <= q.shape[-1] - BLOCK:
        raise ValueError(f"act8_unpack: width {width} of a checkpoint {tuple(q.shape)}, {tuple(scale.shape)}")
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"act8_unpack: fp32 or bf16, got {dtype}")
    rows = scale.numel() // scale.shape[-1]
    if not q.is_cuda or rows == 0:
        return _unpack_ref(q, scale, width, dtype)
    q, scale = q.contiguous(), scale.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    with _on(q.device):
        out = torch.empty(*q.shape[:-1], width, dtype=dtype, device=q.device)
        N.hip().act8_values(q.data_ptr(), scale.data_ptr(), rows, width, N.dtype_code(dtype), out.data_ptr(),
                            N.stream_of(q))
    return out


def _check_float(who: str, x: torch.Tensor) -> None:
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{who}: fp32 or bf16, got {x.dtype}")


def _planes(w: torch.Tensor) -> torch.Tensor:
    """Workspace for the three planes of an fp32 weight."""
    return torch.empty(6 * w.shape[0] * (-(-w.shape[1] // 8) * 8), dtype=torch.uint8, device=w.device)


class _LinearAct8Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, gelu, sink_in, bias_handoff):
        rows, K = x.shape
        out = weight.shape[0]
        dev = x.device
        f32 = x.dtype == torch.float32
        ctx.params = (weight, bias)
        ctx.gelu, ctx.dims, ctx.x_dtype = gelu, (rows, K, out), x.dtype
        ctx.sink_in, ctx.bias_handoff = sink_in, bias_handoff
        # for dw, and for the GELU's slope in dx
        keep = ctx.needs_input_grad[1] or gelu and ctx.needs_input_grad[0]
        if not x.is_cuda:
            wide = x.float()
            with torch.autocast("cpu", enabled=False):
                y = F.linear(F.gelu(wide, approximate="tanh") if gelu else wide, weight.float(),
                             None if bias is None else bias.float()).to(x.dtype)
            q, s = _pack_ref(x) if keep else (None, None)
            ctx.save_for_backward(weight, q, s)
            return y
        h = N.hip()
        with _on(dev):
            dt = N.dtype_code(x.dtype)
            # bf16 rows of whole aligned vectors go into the product as they are
            copy = bool(f32 or gelu or x.data_ptr() % 16 or x.stride(0) % 8 or K % 8)
            nf, _, kq, _ = h.linear_act8_sizes(rows, K, out, dt, copy, gelu)
            w = weight if f32 else _rows16(weight)
            ws = torch.empty(max(nf, 256), dtype=torch.uint8, device=dev)
            y = torch.empty(rows, out, dtype=x.dtype, device=dev)
            q = torch.empty(rows, kq, dtype=_F8, device=dev) if keep else None
            s = torch.empty(rows, kq // BLOCK, dtype=_E8, device=dev) if keep else None
            planes = _planes(w) if f32 else None
            h.linear_act8_fwd(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), N.ptr(bias),
                              N.DT_F32 if bias is None else N.dtype_code(bias.dtype), y.data_ptr(), N.ptr(q),
                              N.ptr(s), rows, K, out, dt, gelu, copy, N.ptr(planes), ws.data_ptr(), N.stream_of(x))
        ctx.save_for_backward(weight, q, s)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, q, s = ctx.saved_tensors
        rows, K, out = ctx.dims
        wp, bp = ctx.params
        gelu, dt = ctx.gelu, ctx.x_dtype
        need_x, need_w, need_b = ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[2]
        if bp is None:
            need_b = False
        hb = ctx.bias_handoff
        if need_b and hb is not None and hb.done:
            need_b = False  # summed into the flat gradient by the next op's backward
            hb.done = False
        if dy.dtype != dt:
            dy = dy.to(dt)
        if dy.stride(1) != 1 or dy.stride(0) < out:
            dy = dy.contiguous()  # (an expanded gradient's rows overlap)
        acc = ctx.sink_in.take() if ctx.sink_in is not None and need_x else None
        if acc is not None:
            acc = acc.reshape(rows, K).to(dt).contiguous()
        dx = dw = db = None
        if not dy.is_cuda:
            c = None if q is None else _unpack_ref(q, s, K, torch.float32)
            g = dy.float()
            with torch.autocast("cpu", enabled=False):
                if need_x:
                    dx = g @ weight.float()
                    if gelu:
                        dx = dx * gelu_tanh_grad_ref(c)
                    dx = dx.to(dt) if acc is None else (dx + acc.float()).to(dt)
                if need_w:
                    dw = (g.t() @ (F.gelu(c, approximate="tanh") if gelu else c)).to(weight.dtype)
                if need_b:
                    db = g.sum(0).to(bp.dtype)
            return dx, dw, db, None, None, None
        dev = dy.device
        f32 = dt == torch.float32
        h = N.hip()
        with _on(dev):
            if not f32:
                dy = _rows16(dy)
            _, nb, _, _ = h.linear_act8_sizes(rows, K, out, N.dtype_code(dt), True, gelu)
            w = weight if f32 else _rows16(weight)
            if need_x:
                dx = acc if acc is not None else torch.empty(rows, K, dtype=dt, device=dev)
            # into the optimizer's flat gradients where it owns every gradient that is asked for
            direct = need_w and all(_direct(t) and flat_grad(t).dtype in (torch.float32, torch.bfloat16)
                                    for t, need in ((wp, True), (bp, need_b)) if need)
            if need_w:
                dw = flat_grad(wp) if direct else torch.empty(out, K, dtype=weight.dtype, device=dev)
                if need_b:
                    db = flat_grad(bp) if direct else torch.empty(out, dtype=bp.dtype, device=dev)
            elif need_b:
                db = torch.zeros(dy.shape[1], dtype=torch.float32, device=dev)
                colsum_accumulate_(dy, db)
                db = db[:out].to(bp.dtype)
            ws = torch.empty(max(nb, 256), dtype=torch.uint8, device=dev)
            planes = _planes(w) if f32 and need_x else None
            if need_x or need_w:
                h.linear_act8_bwd(dy.data_ptr(), dy.stride(0), w.data_ptr(), w.stride(0), N.ptr(q), N.ptr(s),
                                  N.ptr(dx), acc is not None, N.ptr(dw), dw.stride(0) if need_w else K,
                                  N.ptr(db) if need_w else 0, N.dtype_code(dw.dtype) if need_w else N.DT_F32,
                                  N.dtype_code(db.dtype) if db is not None else N.DT_F32, bool(direct), rows, K, out,
                                  N.dtype_code(dt), gelu, N.ptr(planes), ws.data_ptr(), N.stream_of(dy))
        if direct:
            _ready(wp)
            if need_b:
                _ready(bp)
            dw = db = None
        return dx, dw, db, None, None, None


def linear_act8(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, act: str | None = None,
                sink_in=None, bias_handoff=None) -> torch.Tensor:
    """``F.linear(act(x), weight, bias)`` for x [.., K], weight [N, K], bias [N], its backward from an
    8-bit checkpoint of x (module docstring).  ``sink_in`` / ``bias_handoff``: as ``FusedLinear``'s."""
    if act not in (None, "gelu"):
        raise ValueError(f"linear_act8: act is None or 'gelu', got {act!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or weight.numel() == 0:
        raise ValueError(f"linear_act8: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not multiply")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"linear_act8: bias {tuple(bias.shape)} for weight {tuple(weight.shape)}")
    if x.dtype != weight.dtype and torch.is_autocast_enabled(x.device.type):
        x = x.to(weight.dtype)
    _check_float("linear_act8", x)
    if weight.dtype != x.dtype:
        raise TypeError(f"linear_act8: x and weight must both be fp32 or bf16, got {x.dtype}, {weight.dtype}")
    if bias is not None and bias.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"linear_act8: bias must be fp32 or bf16, got {bias.dtype}")
    dev = x.device
    for t, nm in ((weight, "weight"), (bias, "bias")):
        if t is not None and t.device != dev:
            raise ValueError(f"linear_act8: {nm} on {t.device}, x on {x.device}")
    # (a reshape that changes nothing would still be a node of the backward)
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if x2.shape[0] == 0:
        with torch.autocast(dev.type, enabled=False):
            return F.linear(F.gelu(x, approximate="tanh") if act else x, weight, None if bias is None else bias.to(x.dtype))
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    if weight.stride(1) != 1:
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    y = _LinearAct8Fn.apply(x2, weight, bias, act == "gelu", sink_in, bias_handoff)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], weight.shape[0])


class Act8Linear(FusedLinear):
    """``FusedLinear`` (same parameters) whose backward works from an 8-bit checkpoint of its input;
    ``act="gelu"``: of the GELU's input, the GELU being part of the layer."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, act: str | None = None, **kw):
        super().__init__(in_features, out_features, bias=bias, **kw)
        self.act = act

    def forward(self, x, sink_in=None, bias_handoff=None):
        return linear_act8(x, self.weight, self.bias, self.act, sink_in, bias_handoff)
