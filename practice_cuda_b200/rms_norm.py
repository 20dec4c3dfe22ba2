"""Root-mean-square norm with the residual's addition and an FP8 output.

``h = x + residual`` (held in ``x``'s type: the residual that later layers
read), ``y = h / sqrt(mean(h^2) + eps) * weight``, and the FP8 quantization
of ``y`` with the scales that the FP8 linears read (1x128 blocks, or one per
row), in one pass over ``x`` and ``residual``.  The reference has no norm of
its own; its training linears quantize their input in a pass apart
(``fp8_training/fp8_bench/modules/bmm_linear.py:229-310``).

* :func:`rms_norm_quant` -- forward, without autograd.
* :func:`rms_norm_backward` -- its gradients.
* :func:`rms_norm` -- differentiable, with the FP8 output beside ``y``.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .registry import QuantResult

_QUANT_MODES = {None: 0, "block": 1, "row": 2}
_BLOCK = 128
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


@dataclass
class RMSNormResult:
    """What one forward pass wrote (``None``: not asked for)."""

    y: Optional[torch.Tensor]  # [..., dim], x's type
    quant: Optional[QuantResult]  # tensor [rows, dim] fp8, dequant_scale [rows, ceil(dim / 128)] or [rows]
    residual: torch.Tensor  # h: x + residual, or x itself without a residual
    rstd: torch.Tensor  # [rows] fp32


def _rows(t: torch.Tensor, dim: int) -> torch.Tensor:
    """``t`` as [rows, dim] with contiguous rows; copied only where no view is."""
    t = t if t.ndim == 2 else t.reshape(-1, dim)
    return t if t.stride(1) == 1 or dim == 1 else t.contiguous()


def _check_weight(weight: torch.Tensor, x: torch.Tensor, what: str) -> torch.Tensor:
    dim = x.shape[-1]
    if weight.ndim != 1 or weight.shape[0] != dim:
        raise ValueError(f"{what}: weight must have shape ({dim},), got {tuple(weight.shape)}")
    if weight.dtype not in _FLOATS:
        raise ValueError(f"{what}: weight must be bf16, fp16 or fp32, got {weight.dtype}")
    if weight.device != x.device:
        raise ValueError(f"{what}: weight is on {weight.device}, x on {x.device}")
    return weight if weight.stride(0) == 1 else weight.contiguous()


def _check_like(t: torch.Tensor, x: torch.Tensor, name: str, what: str) -> None:
    if t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{what}: {name} must match {tuple(x.shape)} {x.dtype} on {x.device}, "
                         f"got {tuple(t.shape)} {t.dtype} on {t.device}")


def _check_input(x: torch.Tensor, name: str, what: str) -> None:
    _lib.require_cuda(x, name)
    if x.ndim < 1 or x.shape[-1] == 0:
        raise ValueError(f"{what}: {name} needs a last dimension of at least one element, got {tuple(x.shape)}")
    if x.dtype not in _FLOATS:
        raise ValueError(f"{what}: {name} must be bf16, fp16 or fp32, got {x.dtype}")


def rms_norm_quant(
    x: torch.Tensor,
    weight: torch.Tensor,
    residual: Optional[torch.Tensor] = None,
    *,
    eps: float = 1e-5,
    quant: Optional[str] = "block",
    fp8_dtype: torch.dtype = torch.float8_e4m3fn,
    pow2_scales: bool = False,
    return_y: bool = False,
    quant_eps: float = 1e-12,
) -> RMSNormResult:
    """Norm of ``x`` (+ ``residual``), its FP8 quantization and, with
    ``return_y``, the normalised rows in ``x``'s type.

    ``quant``: ``"block"`` (1x128 blocks, the scales of
    ``b200_per_block_quant``; ``pow2_scales`` for its power-of-two ones),
    ``"row"`` (one scale per row, the scales of ``b200_per_channel_quant``)
    or ``None`` (``y`` alone).  ``y`` is quantized unrounded, so the FP8
    values do not pass through ``x``'s type.  Runs on the current stream;
    no autograd.
    """
    what = "rms_norm_quant"
    _check_input(x, "x", what)
    weight = _check_weight(weight, x, what)
    if quant not in _QUANT_MODES:
        raise ValueError(f'{what}: quant must be "block", "row" or None, got {quant!r}')
    if pow2_scales and quant != "block":
        raise ValueError(f"{what}: power-of-two scales go with 1x128 blocks")
    if quant is not None and fp8_dtype not in (torch.float8_e4m3fn, torch.float8_e5m2):
        raise ValueError(f"{what}: fp8_dtype must be float8_e4m3fn or float8_e5m2, got {fp8_dtype}")
    dim = x.shape[-1]
    x2 = _rows(x, dim)
    rows, device = x2.shape[0], x.device
    with _lib.on_device(device):
        h = y = q = scale = None
        xp, rp, hp, yp, qp, scp = x2.data_ptr(), None, None, None, None, None
        rs = q_code = ss = sb = 0
        if residual is not None:
            _check_like(residual, x, "residual", what)
            r2 = _rows(residual, dim)
            h = _like(x2)
            rp, rs, hp = r2.data_ptr(), r2.stride(0), h.data_ptr()
        if return_y or quant is None:
            y = _like(x2)
            yp = y.data_ptr()
        if quant is not None:
            q = _like(x2, fp8_dtype)
            if quant == "block":
                ss, sb = -(-dim // _BLOCK), 1
                scale = x2.new_empty((rows, ss), dtype=torch.float32)
            else:
                ss = 1
                scale = x2.new_empty((rows,), dtype=torch.float32)
            qp, q_code, scp = q.data_ptr(), _lib.PCB_DTYPE[fp8_dtype], scale.data_ptr()
        rstd = x2.new_empty((rows,), dtype=torch.float32)
        status = _lib.lib().pcb_rms_norm_fwd(
            xp, _lib.PCB_DTYPE[x.dtype], rows, dim, x2.stride(0), rp, rs,
            weight.data_ptr(), _lib.PCB_DTYPE[weight.dtype], eps, hp, dim, yp, dim, qp, q_code, dim, scp, ss, sb,
            _QUANT_MODES[quant], int(pow2_scales), quant_eps, rstd.data_ptr(), _lib.stream_ptr(device))
        if status:
            _lib.check(status, "pcb_rms_norm_fwd")
    if x2 is not x:
        y = y.view(x.shape) if y is not None else None
        h = h.view(x.shape) if h is not None else None
    return RMSNormResult(y, _quant_result(q, scale, quant, pow2_scales) if q is not None else None,
                         h if h is not None else x, rstd)


def _like(t: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """A contiguous tensor of t's [rows, dim]."""
    if t.is_contiguous():
        return torch.empty_like(t) if dtype is None else torch.empty_like(t, dtype=dtype)
    return t.new_empty(t.shape) if dtype is None else t.new_empty(t.shape, dtype=dtype)


def _quant_result(q: torch.Tensor, scale: torch.Tensor, quant: str, pow2_scales: bool) -> QuantResult:
    meta = {"logical_shape": tuple(q.shape), "fp8_dtype": str(q.dtype)}
    if pow2_scales:
        meta["scale_format"] = "e8m0"
    if quant == "block":
        meta.update(block_m=1, block_n=_BLOCK)
        return QuantResult(q, scale, "b200_rms_norm", "block", meta)
    meta.update(channel_axis=-2)
    return QuantResult(q, scale, "b200_rms_norm", "channel", meta)


def rms_norm_backward(
    dy: torch.Tensor,
    h: torch.Tensor,
    weight: torch.Tensor,
    rstd: torch.Tensor,
    *,
    dresidual: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Gradients ``(dx, dweight)`` of :func:`rms_norm_quant`'s ``y`` from the
    ``residual`` (h) and ``rstd`` that it returned.

    ``dresidual`` is the gradient that reaches ``h`` itself.  ``dx`` is the
    gradient of ``x`` and of the residual input alike.  ``dweight`` (the
    weight's type) is summed in a fixed order.
    """
    what = "rms_norm_backward"
    _check_input(h, "h", what)
    _check_like(dy, h, "dy", what)
    weight = _check_weight(weight, h, what)
    dim = h.shape[-1]
    h2, dy2 = _rows(h, dim), _rows(dy, dim)
    rows, device = h2.shape[0], h.device
    if rstd.shape != (rows,) or rstd.dtype != torch.float32 or rstd.device != device:
        raise ValueError(f"{what}: rstd must be fp32 of shape ({rows},) on {device}, "
                         f"got {rstd.dtype} {tuple(rstd.shape)} on {rstd.device}")
    rstd = rstd.contiguous()
    with _lib.on_device(device):
        dhp, dhs = None, 0
        if dresidual is not None:
            _check_like(dresidual, h, "dresidual", what)
            dh2 = _rows(dresidual, dim)
            dhp, dhs = dh2.data_ptr(), dh2.stride(0)
        dx = _like(h2)
        dw = torch.empty_like(weight)
        lib = _lib.lib()
        nbytes = lib.pcb_rms_norm_bwd_workspace_bytes(rows, dim)
        workspace = h2.new_empty((nbytes,), dtype=torch.uint8)
        status = lib.pcb_rms_norm_bwd(
            dy2.data_ptr(), dy2.stride(0), h2.data_ptr(), h2.stride(0), _lib.PCB_DTYPE[h.dtype], rows, dim, dhp, dhs,
            weight.data_ptr(), _lib.PCB_DTYPE[weight.dtype], rstd.data_ptr(), dx.data_ptr(), dim, dw.data_ptr(),
            workspace.data_ptr(), nbytes, _lib.stream_ptr(device))
        if status:
            _lib.check(status, "pcb_rms_norm_bwd")
    return dx if h2 is h else dx.view(h.shape), dw


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, quant, fp8_dtype, pow2_scales):
        r = rms_norm_quant(x, weight, residual, eps=eps, quant=quant, fp8_dtype=fp8_dtype, pow2_scales=pow2_scales,
                           return_y=True)
        ctx.save_for_backward(r.residual, weight, r.rstd)
        ctx.has_residual = residual is not None
        ctx.set_materialize_grads(False)
        q, scale = (r.quant.tensor, r.quant.dequant_scale) if r.quant is not None else (None, None)
        if q is not None:
            ctx.mark_non_differentiable(q, scale)
        return r.y, r.residual if residual is not None else None, q, scale

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh, _dq, _dscale):
        h, weight, rstd = ctx.saved_tensors
        if dy is None:  # y was not used: h alone carries a gradient
            return dh, None, dh if ctx.has_residual else None, None, None, None, None
        dx, dw = rms_norm_backward(dy, h, weight, rstd, dresidual=dh)
        return dx, dw, dx if ctx.has_residual else None, None, None, None, None


def rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    residual: Optional[torch.Tensor] = None,
    *,
    eps: float = 1e-5,
    quant: Optional[str] = None,
    fp8_dtype: torch.dtype = torch.float8_e4m3fn,
    pow2_scales: bool = False,
) -> tuple[torch.Tensor, torch.Tensor, Optional[QuantResult]]:
    """Differentiable (once) norm: ``(y, h, quant)``.

    ``y`` and ``h`` (``x + residual``, or ``x``) carry gradients; ``quant`` is
    the FP8 quantization of ``y`` for the linears that read it (``None``
    unless ``quant`` names a scheme), through which no gradient flows.
    """
    y, h, q, scale = _RMSNorm.apply(x, weight, residual, eps, quant, fp8_dtype, pow2_scales)
    result = _quant_result(q, scale, quant, pow2_scales) if q is not None else None
    return y, h if h is not None else x, result
