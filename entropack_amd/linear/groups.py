"""Rows grouped by an id: the plan that products by expert and adapters by request share, and the weighted return.

`group_rows(ids, groups)` sorts the entries of `ids` (one per token, or k per token) by group on the device and returns a
`RowGroups`; `linear.grouped` multiplies each group with its own weight, `linear.adapters` adds each group's low-rank
update, and `combine_rows` brings grouped rows back to their tokens. Sizes of groups stay on the device: nothing here
synchronises, and every call may be captured into a graph (the ids may then change between replays). The reference has no
counterpart: its layers have one weight each (entropack/linear/linear.py:18-230).

Capturing a training step: run forward and backward inside the same capture, and let no eager graph over the same leaves
live meanwhile (torch ties a leaf's gradient accumulation to the stream it was first used on).
"""
from __future__ import annotations

import dataclasses
import functools

import torch
from torch.autograd import forward_ad

from ..backends import hip as _hip

MAX_GROUPS = 896                   # a thread per group and 64 KiB of LDS in the sorting kernel
MAX_ENTRIES = 1 << 30
_BF16, _F32 = 0, 2
_ROW_KINDS = {torch.bfloat16: _BF16, torch.float32: _F32}


def device_of(name: str, *tensors: torch.Tensor | None) -> torch.device:
    """The one GPU all operands are on."""
    device = None
    for tensor in tensors:
        if tensor is None:
            continue
        if tensor.device.type != "cuda":
            raise RuntimeError(f"{name} runs on the GPU, got a tensor on {tensor.device}")
        if device is None:
            device = tensor.device
        elif tensor.device != device:
            raise ValueError(f"{name}: all operands must be on one device, got {device} and {tensor.device}")
    return device


def refuse_tangents(name: str, *tensors: torch.Tensor | None) -> None:
    """The operators have gradients, no Jacobian-vector products. A tensor with a tangent need not ask for a gradient, so a call on it could
    return a result whose tangent is missing: such a call raises. (The level is asked for first: outside of one no tensor has a tangent.)"""
    if forward_ad._current_level < 0:
        return
    if any(tensor is not None and forward_ad.unpack_dual(tensor).tangent is not None for tensor in tensors):
        raise RuntimeError(f"{name} has no forward-mode derivative (jvp); detach the operand or take the gradient in reverse mode")


def matrix(tensor: torch.Tensor, pieces: int) -> torch.Tensor:
    """`tensor` ([.., columns]) as the kernels read it: columns contiguous, rows and groups whole numbers of 16 bytes apart and
    not overlapping, the first row 16-byte aligned. Rows of a number of columns that is no multiple of `pieces` are padded
    with zeros. A tensor that lies so already is returned as it is; anything else is copied."""
    shape = tensor.shape
    columns = shape[-1]
    if columns % pieces:
        return torch.nn.functional.pad(tensor, (0, pieces - columns % pieces))
    if 1 not in shape and tensor.is_contiguous():                # the usual case by one call; a dimension of one may have any stride
        return tensor if tensor.data_ptr() % 16 == 0 else tensor.clone(memory_format=torch.contiguous_format)
    fits = tensor.stride(-1) == 1 and tensor.data_ptr() % 16 == 0
    least = columns
    for dim in range(tensor.dim() - 2, -1, -1):
        fits = fits and tensor.stride(dim) >= least and tensor.stride(dim) % pieces == 0
        least = tensor.stride(dim) * (tensor.shape[dim] - 1) + least
    return tensor if fits else tensor.clone(memory_format=torch.contiguous_format)


def rows_of(tensor: torch.Tensor) -> torch.Tensor:
    """`tensor` ([.., columns]) for kernels that take any address: columns contiguous, rows and groups not overlapping."""
    if 1 not in tensor.shape and tensor.is_contiguous():
        return tensor
    fits = tensor.stride(-1) == 1
    least = tensor.shape[-1]
    for dim in range(tensor.dim() - 2, -1, -1):
        fits = fits and tensor.stride(dim) >= least
        least = tensor.stride(dim) * (tensor.shape[dim] - 1) + least
    return tensor if fits else tensor.clone(memory_format=torch.contiguous_format)


def first_order(backward):
    """`once_differentiable` where a graph of the gradients is asked for, without its two context managers where none is (3 us)."""
    checked = torch.autograd.function.once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        refuse_tangents("the gradient of an operator on grouped rows", *grads)
        return checked(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


@dataclasses.dataclass(frozen=True, eq=False)
class RowGroups:
    """What `group_rows` made of a tensor of ids. Made by `group_rows` only: the kernels take its indices as they are.

    Attributes:
        order: int32 [entries], the entries (token * per_row + pick) sorted by group, those of no group last.
        offsets: int32 [groups + 1], the first place of every group; places from offsets[groups] on have no group.
        place: int32 [entries], the inverse of `order`.
        rows: int32 [entries], the token of every place (`order` itself for one id per token).
        groups: number of groups.
        tokens, per_row: the ids' shape; entries = tokens * per_row.
    """
    order: torch.Tensor
    offsets: torch.Tensor
    place: torch.Tensor
    rows: torch.Tensor
    groups: int
    tokens: int
    per_row: int

    @property
    def entries(self) -> int:
        return self.tokens * self.per_row

    @property
    def device(self) -> torch.device:
        return self.order.device


def group_rows(ids: torch.Tensor, groups: int) -> RowGroups:
    """Sorts the entries of `ids` (int32 or int64, [tokens] or [tokens, k], on the GPU) by group.

    Ids outside [0, groups), such as -1 for padding, belong to no group: the products give those rows zero (the adapters
    leave them as they are), the weighted return skips them. The sort is stable, so the result is the same in every run.
    """
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"group_rows takes int32 or int64 ids, got {ids.dtype}")
    if ids.dim() not in (1, 2):
        raise ValueError(f"group_rows takes ids of shape [tokens] or [tokens, k], got {tuple(ids.shape)}")
    if isinstance(groups, bool) or not isinstance(groups, int) or not 1 <= groups <= MAX_GROUPS:
        raise ValueError(f"groups must be an integer from 1 to {MAX_GROUPS}, got {groups!r}")
    tokens, per_row = ids.shape[0], 1 if ids.dim() == 1 else ids.shape[1]
    if per_row < 1:
        raise ValueError("group_rows needs at least one id per token")
    entries = tokens * per_row
    if entries > MAX_ENTRIES:
        raise ValueError(f"group_rows takes at most {MAX_ENTRIES} entries, got {entries}")
    device = device_of("group_rows", ids)
    order = torch.empty(entries, dtype=torch.int32, device=device)
    place = torch.empty(entries, dtype=torch.int32, device=device)
    rows = torch.empty(entries, dtype=torch.int32, device=device) if per_row > 1 else order
    if entries == 0:
        return RowGroups(order, torch.zeros(groups + 1, dtype=torch.int32, device=device), place, rows, groups, tokens, per_row)
    offsets = torch.empty(groups + 1, dtype=torch.int32, device=device)
    flat = ids.contiguous()
    room = _hip.library().ep_hip_group_rows_workspace(entries, groups)
    workspace = torch.empty(room, dtype=torch.uint8, device=device) if room else None
    _hip.launch("ep_hip_group_rows", device,
                flat.data_ptr(), flat.element_size(), entries, groups, per_row, order.data_ptr(), offsets.data_ptr(), place.data_ptr(),
                rows.data_ptr() if per_row > 1 else None, None if workspace is None else workspace.data_ptr(), room)
    return RowGroups(order, offsets, place, rows, groups, tokens, per_row)


def kept_rows(groups: RowGroups) -> int:
    """Address of the number of places that have a group."""
    return groups.offsets.data_ptr() + 4 * groups.groups


def sum_entries(rows: torch.Tensor, tokens: int, per_row: int) -> torch.Tensor:
    """[entries, width] rows in the order of the entries (f32 or bf16) added up per token, rounded to bf16 once."""
    out = torch.empty(tokens, rows.shape[1], dtype=torch.bfloat16, device=rows.device)
    if out.numel():
        _hip.launch("ep_hip_combine_rows", rows.device,
                    rows.data_ptr(), _ROW_KINDS[rows.dtype], rows.stride(0), None, None, None, 0, per_row, tokens, rows.shape[1],
                    out.data_ptr(), out.stride(0))
    return out


def _combine(y, weight, groups: RowGroups):
    """The tokens' sums; y and the weights as the kernels read them."""
    rows = rows_of(y)
    ready = None if weight is None else weight.contiguous()
    width = y.shape[1]
    out = torch.empty(groups.tokens, width, dtype=torch.bfloat16, device=y.device)
    if out.numel():
        _hip.launch("ep_hip_combine_rows", y.device,
                    rows.data_ptr(), _BF16, rows.stride(0), groups.place.data_ptr(), kept_rows(groups),
                    None if ready is None else ready.data_ptr(), 0 if ready is None else _ROW_KINDS[ready.dtype], groups.per_row,
                    groups.tokens, width, out.data_ptr(), width)
    return out, rows, ready


class _CombineRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weight, groups):
        out, rows, ready = _combine(y, weight, groups)
        ctx.groups = groups
        ctx.save_for_backward(rows, ready)
        return out

    @staticmethod
    @first_order
    def backward(ctx, grad):
        rows, ready = ctx.saved_tensors
        groups, (need_y, need_weight, _) = ctx.groups, ctx.needs_input_grad
        entries, width = rows.shape
        grad_y = torch.empty(entries, width, dtype=torch.bfloat16, device=grad.device) if need_y else None
        grad_weight = torch.empty(ready.shape, dtype=ready.dtype, device=grad.device) if need_weight else None
        if entries and width:
            slope = rows_of(grad)
            _hip.launch("ep_hip_combine_rows_grad", grad.device,
                        slope.data_ptr(), slope.stride(0), rows.data_ptr(), rows.stride(0), groups.place.data_ptr(), kept_rows(groups),
                        None if ready is None else ready.data_ptr(), 0 if ready is None else _ROW_KINDS[ready.dtype], groups.per_row,
                        groups.tokens, width, None if grad_y is None else grad_y.data_ptr(), width,
                        None if grad_weight is None else grad_weight.data_ptr())
        elif grad_weight is not None:
            grad_weight.zero_()
        return grad_y, grad_weight, None


def combine_rows(y: torch.Tensor, groups: RowGroups, weight: torch.Tensor | None = None) -> torch.Tensor:
    """Grouped rows back to their tokens: out[t] = sum over t's entries of weight[t, j] * y[place of the entry].

    Args:
        y: bf16 [entries, width] in grouped order, as `grouped_linear` returns it.
        groups: the plan of `group_rows`.
        weight: f32 or bf16, the shape of the ids, or None for ones (the router's weights).

    Entries of no group add nothing, whatever y and weight hold there. Sums are f32, rounded to bf16 once. Differentiable
    in y and weight, in reverse mode.
    """
    if not isinstance(groups, RowGroups):
        raise TypeError(f"combine_rows takes the plan that group_rows returns, got {type(groups).__name__}")
    if y.dtype != torch.bfloat16:
        raise TypeError(f"combine_rows takes bfloat16 rows, got {y.dtype}")
    if y.dim() != 2 or y.shape[0] != groups.entries:
        raise ValueError(f"combine_rows takes {groups.entries} rows (one per entry), got shape {tuple(y.shape)}")
    if weight is not None:
        if weight.dtype not in _ROW_KINDS:
            raise TypeError(f"combine_rows takes float32 or bfloat16 weights, got {weight.dtype}")
        if tuple(weight.shape) not in ({(groups.tokens, groups.per_row)} | ({(groups.tokens,)} if groups.per_row == 1 else set())):
            raise ValueError(f"combine_rows takes weights of shape {(groups.tokens, groups.per_row)}, got {tuple(weight.shape)}")
    device_of("combine_rows", y, groups.order, weight)
    refuse_tangents("combine_rows", y, weight)
    if torch.is_grad_enabled() and (y.requires_grad or (weight is not None and weight.requires_grad)):
        return _CombineRows.apply(y, weight, groups)
    return _combine(y, weight, groups)[0]


__all__ = ["RowGroups", "combine_rows", "group_rows"]
