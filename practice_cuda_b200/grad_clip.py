"""Global norm of a model's gradients, and clipping by it.

``norm = sqrt(sum g^2)`` over every tensor given (or the largest magnitude),
then ``g * min(1, max_norm / (norm + eps))``: two launches for up to 1000
tensors of mixed types, nothing read back by the host.  The reference trains
without clipping (``fp8_training/fp8_bench/bench/bench_fsdp2.py:120-187``).

* :func:`grad_norm` -- the norm alone.
* :func:`clip_grad_norm` -- norm and clipping of a list of tensors, in place
  or into other tensors.
* :func:`clip_grad_norm_` -- the gradients of a model's parameters, FSDP2
  shards included.
"""

from __future__ import annotations

import math
from array import array
from typing import Iterable, Optional, Sequence, Union

import torch
import torch.distributed as dist

from . import _lib

_NORM_TYPES = {2.0: 0, math.inf: 1}
# Called through map(): one pass over many small tensors is what a call costs.
_pointer, _numel, _device, _contiguous = (
    torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device, torch.Tensor.is_contiguous)
_DTYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _norm_code(norm_type: float, what: str) -> int:
    try:
        return _NORM_TYPES[float(norm_type)]
    except (KeyError, ValueError, TypeError):
        raise ValueError(f"{what}: norm_type must be 2 or inf, got {norm_type!r}") from None


def _as_list(tensors: Union[torch.Tensor, Iterable[torch.Tensor]], what: str):
    """The tensors and their types."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        raise ValueError(f"{what}: no tensors (their device is where the norm goes)")
    first = tensors[0]
    dtypes = [t.dtype for t in tensors]
    for dtype in set(dtypes):
        if dtype not in _DTYPE_CODES:
            raise ValueError(f"{what}: gradients must be bf16, fp16 or fp32, got {dtype}")
    if len(set(map(_device, tensors))) != 1:
        raise ValueError(f"{what}: gradients on {sorted({str(t.device) for t in tensors})}")
    _lib.require_cuda(first, "gradients")
    return tensors, dtypes


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill one stretch of memory, in whatever order."""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _same_order(a: torch.Tensor, b: torch.Tensor) -> bool:
    return (a.is_contiguous() and b.is_contiguous()) or a.stride() == b.stride()


class _Table:
    """The host arrays of one call: pointers, sizes and types."""

    def __init__(self, tensors: Sequence[torch.Tensor], dtypes: Sequence[torch.dtype]):
        self.pointers = array("Q", map(_pointer, tensors))
        self.sizes = array("q", map(_numel, tensors))
        self.types = array("i", [_DTYPE_CODES[t] for t in dtypes])
        self.count = len(tensors)

    def args(self) -> tuple[int, int, int]:
        return self.sizes.buffer_info()[0], self.types.buffer_info()[0], self.count


def _workspace(count: int, device: torch.device) -> tuple[torch.Tensor, int]:
    nbytes = _lib.lib().pcb_grad_norm_workspace_bytes(count)
    return torch.empty(nbytes, device=device, dtype=torch.uint8), nbytes


def grad_norm(tensors: Union[torch.Tensor, Iterable[torch.Tensor]], *, norm_type: float = 2.0) -> torch.Tensor:
    """The norm over all tensors: a 0-dim fp32 tensor on their device."""
    what = "grad_norm"
    code = _norm_code(norm_type, what)
    tensors, dtypes = _as_list(tensors, what)
    device = tensors[0].device
    with _lib.on_device(device):
        # A view whose elements do not fill one stretch of memory is copied.
        tensors = [t if t.is_contiguous() or _dense(t) else t.contiguous() for t in tensors]
        table = _Table(tensors, dtypes)
        norm = torch.empty((), device=device, dtype=torch.float32)
        workspace, nbytes = _workspace(table.count, device)
        status = _lib.lib().pcb_grad_norm(table.pointers.buffer_info()[0], *table.args(), code, norm.data_ptr(),
                                          workspace.data_ptr(), nbytes, _lib.stream_ptr(device))
        if status:
            _lib.check(status, "pcb_grad_norm")
    return norm


def _targets(tensors, dtypes, out: Sequence[torch.Tensor], what: str) -> list[torch.Tensor]:
    out = [out] if isinstance(out, torch.Tensor) else list(out)
    if len(out) != len(tensors):
        raise ValueError(f"{what}: {len(out)} outputs for {len(tensors)} gradients")
    if ([o.shape for o in out] != [t.shape for t in tensors] or [o.dtype for o in out] != dtypes
            or set(map(_device, out)) != {tensors[0].get_device()}):
        for t, o in zip(tensors, out):
            if o.shape != t.shape or o.dtype != t.dtype or o.device != t.device:
                raise ValueError(f"{what}: an output is {tuple(o.shape)} {o.dtype} on {o.device}, "
                                 f"its gradient {tuple(t.shape)} {t.dtype} on {t.device}")
    return out


def _check_writable(out: Sequence[torch.Tensor], what: str) -> None:
    for o in out:
        if not _dense(o) and any(s == 0 and n > 1 for s, n in zip(o.stride(), o.shape)):
            raise ValueError(f"{what}: cannot write to an expanded tensor of shape {tuple(o.shape)}")


def _check_apart(out: Sequence[torch.Tensor], what: str) -> None:
    """Refuse a tensor that is written twice.  (The library refuses dense tensors that
    overlap; these, of which some are not, are written one after the other.)"""
    pointers = [o.data_ptr() for o in out if o.numel()]
    if len(set(pointers)) != len(pointers):
        raise ValueError(f"{what}: gradients or outputs overlap: each element may be scaled once only")


def _check_status(status: int, entry: str, what: str) -> None:
    if status == _lib.PCB_ERR_INVALID:
        raise ValueError(f"{what}: {_lib.lib().pcb_last_error_text().decode()}")
    if status:
        _lib.check(status, entry)


def clip_grad_norm(
    tensors: Union[torch.Tensor, Iterable[torch.Tensor]],
    max_norm: float,
    *,
    norm_type: float = 2.0,
    eps: float = 1e-6,
    out: Optional[Sequence[torch.Tensor]] = None,
    error_if_nonfinite: bool = False,
    group: Optional["dist.ProcessGroup"] = None,
) -> torch.Tensor:
    """Scale ``tensors`` by ``min(1, max_norm / (norm + eps))`` and return
    the norm before it (0-dim fp32, on the device).

    In place, or into ``out`` (one tensor each, of the same shape and type).  Each
    element is scaled once: a tensor that stands in the list twice, tensors that
    overlap, and outputs that overlap another gradient are refused.
    A non-finite norm makes the gradients NaN or 0, as the product says;
    ``error_if_nonfinite`` raises instead, before anything is written, and
    waits for the GPU to know.  With ``group``, the tensors are this process's
    shards: the norm is that of all processes' shards together.
    """
    what = "clip_grad_norm"
    code = _norm_code(norm_type, what)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"{what}: max_norm must not be negative, got {max_norm}")
    tensors, dtypes = _as_list(tensors, what)
    in_place = out is None
    out = tensors if in_place else _targets(tensors, dtypes, out, what)
    device = tensors[0].device
    lib = _lib.lib()
    with _lib.on_device(device):
        # Views that do not fill one stretch of memory, or whose output lies in
        # another order, pass through a contiguous copy.
        src, dst, direct = tensors, out, None
        if not (all(map(_contiguous, out)) and (in_place or all(map(_contiguous, tensors)))):
            _check_writable(out, what)
            _check_apart(out, what)
            direct = [_dense(t) and _dense(o) and _same_order(t, o) for t, o in zip(tensors, out)]
            src = [t if d else t.contiguous() for t, d in zip(tensors, direct)]
            dst = [o if d else torch.empty_like(t) for t, o, d in zip(src, out, direct)]
        table = _Table(src, dtypes)
        targets = table.pointers if dst is src else array("Q", map(_pointer, dst))
        pointers, targets_at = table.pointers.buffer_info()[0], targets.buffer_info()[0]
        stream = _lib.stream_ptr(device)
        if group is None and not error_if_nonfinite:
            norm = torch.empty((), device=device, dtype=torch.float32)
            workspace, nbytes = _workspace(table.count, device)
            status = lib.pcb_grad_clip(pointers, targets_at, *table.args(), code, max_norm, eps, norm.data_ptr(),
                                       workspace.data_ptr(), nbytes, stream)
            if status:
                _check_status(status, "pcb_grad_clip", what)
        else:
            norm = grad_norm(src, norm_type=norm_type)
            if group is not None:
                norm = join_norms(norm, norm_type, group)
            if error_if_nonfinite and not bool(torch.isfinite(norm)):
                raise RuntimeError(f"{what}: the gradients' norm is {norm.item()}")
            status = lib.pcb_grad_scale(pointers, targets_at, *table.args(), norm.data_ptr(), max_norm, eps, stream)
            if status:
                _check_status(status, "pcb_grad_scale", what)
        if direct is not None:
            for t, o, d in zip(dst, out, direct):
                if not d:
                    o.copy_(t)
        # A graph may have saved any of them, whether or not they require a gradient:
        # it is to see that they have changed, as after an in-place operation of torch.
        torch.autograd.graph.increment_version(out)
    return norm


def join_norms(norm: torch.Tensor, norm_type: float, group: Optional["dist.ProcessGroup"]) -> torch.Tensor:
    """The norm over the shards of every process of ``group`` from each one's own."""
    if float(norm_type) == math.inf:
        # NaN has to survive the maximum: processes vote on it beside the value.
        pair = torch.stack([torch.nan_to_num(norm, nan=0.0, posinf=math.inf), torch.isnan(norm).to(norm.dtype)])
        dist.all_reduce(pair, op=dist.ReduceOp.MAX, group=group)
        return torch.where(pair[1] > 0, torch.full_like(pair[0], math.nan), pair[0])
    squares = norm.double().square()
    dist.all_reduce(squares, op=dist.ReduceOp.SUM, group=group)
    return squares.sqrt().to(norm.dtype)


def clip_grad_norm_(
    parameters: Union[torch.Tensor, Iterable[torch.Tensor]],
    max_norm: float,
    *,
    norm_type: float = 2.0,
    eps: float = 1e-6,
    error_if_nonfinite: bool = False,
) -> torch.Tensor:
    """Clip the gradients of ``parameters`` in place by their global norm.

    Parameters without a gradient are left out.  DTensor gradients (FSDP2
    shards) are clipped shard by shard and their norm is joined over the
    device mesh they share; mixing sharded and plain gradients, several
    meshes, or gradients that are not sharded over the whole mesh is refused.
    """
    what = "clip_grad_norm_"
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.zeros(())
    locals_, group = _local_shards(grads, what)
    norm = clip_grad_norm(locals_, max_norm, norm_type=norm_type, eps=eps, error_if_nonfinite=error_if_nonfinite,
                          group=group)
    if group is not None:  # the shards' versions are their own
        torch.autograd.graph.increment_version(grads)
    return norm


def _local_shards(grads: list[torch.Tensor], what: str):
    from torch.distributed.tensor import DTensor, Shard

    sharded = [g for g in grads if isinstance(g, DTensor)]
    if not sharded:
        return grads, None
    mesh = sharded[0].device_mesh
    if len(sharded) != len(grads) or any(g.device_mesh != mesh for g in sharded):
        raise ValueError(f"{what}: gradients must all be sharded over one device mesh, or all be plain tensors")
    if mesh.ndim != 1 or any(not isinstance(g.placements[0], Shard) for g in sharded):
        raise ValueError(f"{what}: sharded gradients need a one-dimensional mesh and a Shard placement")
    return [g.to_local() for g in sharded], mesh.get_group()
