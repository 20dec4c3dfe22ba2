"""Softmax cross entropy of an output projection, without its logits.

``linear_cross_entropy(x, weight, target)`` is
``cross_entropy(x @ weight.T, target)`` with the projection and the loss in
one: the logits leave the tensor cores as each token's softmax statistics, and
the backward pass computes them again in pieces of the vocabulary, so that no
more than one piece of their gradient exists at a time.  The reference computes
the whole logits and their loss in torch
(``fp8_training/fp8_bench/bench/bench_fsdp2.py:120-187``).
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable

from . import _lib

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_ALIGN = 8  # elements: 16 bytes, what a tensor map asks of a row
_LINE = 64  # elements: 128 bytes
# Rows that do not start on 128-byte lines are read with twice the requests.  With
# gradients wanted, x is copied to rows that do from so many tokens on (kept for the
# backward pass), since every tile of all three products reads it again: on a B200 loss
# and gradients of 1021 tokens of 50001 x 2056 fp16 take 749 us so and 786 us with x as
# it is, 2048 tokens of 32000 x 4104 bf16 1656 and 1804 us, 4096 tokens of 32000 x 520
# 676 and 685 us; 1021 tokens of 4001 x 264 78 and 76 us, and where tokens are left out
# of large products, whose packed x lies on lines already, it costs up to 3 %.  Fewer
# tokens would gain alike (512 of 50001 x 2056: 419 and 450 us).  The weight is not
# worth its copy: with it those calls take 859, 1786 and 716 us, and 770 instead of 645
# us with 30 % of the 1021 tokens left out.
_LINES_FROM = 768


def _aligned_rows(t: torch.Tensor, whole_lines: bool) -> torch.Tensor:
    """``t`` with contiguous rows that start on 16-byte boundaries, or with
    ``whole_lines`` on 128-byte ones: a copy with padded rows where they do not."""
    rows, cols = t.shape
    row = _LINE if whole_lines else _ALIGN
    if t.stride(1) == 1 and t.stride(0) % row == 0 and t.stride(0) >= cols and t.data_ptr() % (2 * row) == 0:
        return t
    padded = t.new_empty((rows, -(-cols // _LINE) * _LINE))
    view = padded[:, :cols]
    if t.stride(1) == 1 or cols == 1:
        status = _lib.lib().pcb_repack_u16(t.data_ptr(), rows, cols, t.stride(0), padded.data_ptr(), padded.stride(0),
                                           _lib.stream_ptr(t.device))
        if status:
            _lib.check(status, "pcb_repack_u16")
    else:
        view.copy_(t)
    return view


def _check(x, weight, target, reduction, piece):
    what = "linear_cross_entropy"
    _lib.require_cuda(x, "x")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{what}: x must be bf16 or fp16, got {x.dtype}")
    if weight.dtype != x.dtype:
        raise ValueError(f"{what}: weight must have x's type {x.dtype}, got {weight.dtype}")
    if x.ndim < 1 or weight.ndim != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"{what}: x [..., dim] and weight [vocab, dim] do not fit: "
                         f"{tuple(x.shape)} and {tuple(weight.shape)}")
    if weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError(f"{what}: weight has no elements: {tuple(weight.shape)}")
    if target.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: target must be int64 or int32, got {target.dtype}")
    if target.shape != x.shape[:-1]:
        raise ValueError(f"{what}: target must have shape {tuple(x.shape[:-1])}, got {tuple(target.shape)}")
    if weight.device != x.device or target.device != x.device:
        raise ValueError(f"{what}: x is on {x.device}, weight on {weight.device}, target on {target.device}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f'{what}: reduction must be "mean", "sum" or "none", got {reduction!r}')
    if piece is not None and piece < 1:
        raise ValueError(f"{what}: vocab_piece must be positive, got {piece}")


def _forward(x, weight, target, ignore_index, reduction, train):
    """loss, and what the backward pass reads."""
    tokens, dim = x.shape
    vocab = weight.shape[0]
    device = x.device
    lib = _lib.lib()
    with _lib.on_device(device):
        lines = train and tokens >= _LINES_FROM
        x2, w2 = _aligned_rows(x, lines), _aligned_rows(weight, False)
        loss = x.new_empty((tokens,) if reduction == 0 else (), dtype=torch.float32)
        stats = x.new_empty((2 * tokens + 1,), dtype=torch.float32)  # [2, tokens], count
        if tokens == 0:
            loss.fill_(float("nan") if reduction == 2 else 0.0)
        nbytes = lib.pcb_linear_ce_fwd_workspace_bytes(tokens, vocab)
        workspace = x.new_empty((nbytes,), dtype=torch.uint8)
        at = stats.data_ptr()
        packed_bytes = lib.pcb_linear_ce_packed_bytes(tokens, vocab, dim)
        packed = x.new_empty((packed_bytes,), dtype=torch.uint8) if packed_bytes else None
        status = lib.pcb_linear_ce_packed_fwd(
            x2.data_ptr(), x2.stride(0), w2.data_ptr(), w2.stride(0), _lib.PCB_DTYPE[x.dtype], tokens, vocab, dim,
            target.data_ptr(), ignore_index, reduction, loss.data_ptr(), at, at + 8 * tokens,
            packed.data_ptr() if packed_bytes else None, packed_bytes,
            workspace.data_ptr(), nbytes, _lib.stream_ptr(device))
        if status:
            _lib.check(status, "pcb_linear_ce_packed_fwd")
    return loss, x2, w2, stats, packed


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction, piece):
        loss, x2, w2, stats, packed = _forward(x, weight, target, ignore_index, reduction, True)
        ctx.save_for_backward(x2, w2, target, stats, packed)
        ctx.args = (ignore_index, reduction, piece)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        x2, w2, target, stats, packed = ctx.saved_tensors
        ignore_index, reduction, piece = ctx.args
        tokens, dim = x2.shape
        vocab = w2.shape[0]
        device = x2.device
        want_dx, want_dw = ctx.needs_input_grad[:2]
        lib = _lib.lib()
        with _lib.on_device(device):
            dloss = dloss.to(torch.float32).contiguous()
            dx = x2.new_empty((tokens, dim)) if want_dx else None
            dw = x2.new_empty((vocab, dim)) if want_dw else None
            nbytes = lib.pcb_linear_ce_packed_bwd_workspace_bytes(tokens, vocab, dim, piece, want_dx, want_dw)
            workspace = x2.new_empty((nbytes,), dtype=torch.uint8)
            at = stats.data_ptr()
            status = lib.pcb_linear_ce_packed_bwd(
                x2.data_ptr(), x2.stride(0), w2.data_ptr(), w2.stride(0), _lib.PCB_DTYPE[x2.dtype], tokens, vocab, dim,
                target.data_ptr(), ignore_index, reduction, at, at + 8 * tokens,
                packed.data_ptr() if packed is not None else None, packed.numel() if packed is not None else 0,
                dloss.data_ptr(), dx.data_ptr() if want_dx else None, dim, dw.data_ptr() if want_dw else None, dim,
                piece, workspace.data_ptr(), nbytes, _lib.stream_ptr(device))
            if status:
                _lib.check(status, "pcb_linear_ce_packed_bwd")
        return dx, dw, None, None, None, None


def linear_cross_entropy(
    x: torch.Tensor,
    weight: torch.Tensor,
    target: torch.Tensor,
    *,
    reduction: str = "mean",
    ignore_index: int = -100,
    vocab_piece: Optional[int] = None,
) -> torch.Tensor:
    """Cross entropy of the logits ``x @ weight.T`` (x [..., dim], weight
    [vocab, dim], both bf16 or both fp16) against ``target`` [...], in fp32.

    ``reduction``, ``ignore_index`` and the mean over no token at all (NaN,
    with zero gradients) are those of ``torch.nn.functional.cross_entropy``.
    Differentiable (once, in reverse mode) in ``x`` and ``weight``; a gradient that
    is not needed is not computed.  ``vocab_piece`` bounds the columns of the logits' gradient
    that exist at a time in the backward pass (rounded down to a multiple of
    256, at least 256; default: as many as fit 128 MiB, at least 2048).

    What ``x`` holds for tokens that are left out (NaN, say) reaches nothing.
    Tokens left out of large products (512 tokens or more, ``tokens * vocab * dim``
    of 2^36 or more) take no part in them: the others are packed, which keeps a
    copy of ``x`` until the backward pass.

    A target outside the vocabulary that is not ``ignore_index`` makes its
    loss NaN and sets the device error word (``_lib.device_error``).
    """
    _check(x, weight, target, reduction, vocab_piece)
    shape = target.shape
    x2 = x if x.ndim == 2 else x.reshape(-1, x.shape[-1])
    t = target if target.ndim == 1 else target.reshape(-1)
    t = t.to(torch.int64).contiguous()
    code = _REDUCTIONS[reduction]
    train = torch.is_grad_enabled() and (x2.requires_grad or weight.requires_grad)
    # A tangent of forward mode goes to the autograd function too, which refuses it.
    if train or unpack_dual(x2).tangent is not None or unpack_dual(weight).tangent is not None:
        loss = _LinearCrossEntropy.apply(x2, weight, t, int(ignore_index), code, int(vocab_piece or 0))
    else:
        loss = _forward(x2, weight, t, int(ignore_index), code, False)[0]
    return loss.view(shape) if code == 0 and len(shape) != 1 else loss
