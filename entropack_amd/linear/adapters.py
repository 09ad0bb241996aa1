"""Low-rank adapters of many requests beside a shared, compressed projection.

`low_rank_update(y, x, down, up, groups, scale)` adds to the shared projection's output y each row's own update,
scale[a] * (x down[a]^T) up[a]^T, for rows that name their adapter (`group_rows(ids, adapters)`, made once per step and used
by every layer). `AdaptedLinear` wraps a compressed layer with a bank of adapters; the compressed weight stays frozen, the
adapters train. The reference has no counterpart.
"""
from __future__ import annotations

import torch

from ..backends import hip as _hip
from .groups import MAX_GROUPS, RowGroups, device_of, first_order, matrix, refuse_tangents, rows_of
from .linear import CompressedLinear


MAX_RANK = 4096


def _update(y, x, down, up, scale, groups: RowGroups):
    """The updated rows; the narrow rows between the two products (three bf16 parts and zeros, of the rank rounded up to 16 each);
    x, down and up as the kernels read them."""
    rank, outer = up.shape[2], up.shape[1]
    planes = torch.empty(groups.entries, 4 * (-(-rank // 16) * 16), dtype=torch.bfloat16, device=x.device)
    out = torch.empty(groups.entries, outer, dtype=torch.bfloat16, device=x.device)
    rows, narrow, wide, base = matrix(x, 8), matrix(down, 8), rows_of(up), rows_of(y)
    _hip.launch("ep_hip_low_rank_update", x.device,
                rows.data_ptr(), rows.stride(0), narrow.data_ptr(), narrow.stride(1), narrow.stride(0), wide.data_ptr(), wide.stride(1), wide.stride(0),
                None if scale is None else scale.data_ptr(), base.data_ptr(), base.stride(0), planes.data_ptr(), out.data_ptr(), outer,
                groups.order.data_ptr(), groups.offsets.data_ptr(), groups.entries, groups.groups, rank, x.shape[1], outer)
    return out, planes, rows, narrow, wide


class _LowRankUpdate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, down, up, scale, groups):
        out, planes, rows, narrow, wide = _update(y, x, down, up, scale, groups)
        ctx.groups, ctx.inner = groups, x.shape[1]
        ctx.save_for_backward(rows, narrow, wide, scale, planes if ctx.needs_input_grad[3] else None)
        return out

    @staticmethod
    @first_order
    def backward(ctx, grad):
        rows, narrow, wide, scale, planes = ctx.saved_tensors
        groups, inner, device, (need_y, need_x, need_down, need_up) = ctx.groups, ctx.inner, grad.device, ctx.needs_input_grad[:4]
        if not (need_x or need_down or need_up):
            return grad, None, None, None, None, None
        adapters, outer, rank = wide.shape
        grad_x = torch.empty(groups.entries, inner, dtype=torch.bfloat16, device=device) if need_x else None
        grad_down = torch.empty(adapters, rank, inner, dtype=torch.bfloat16, device=device) if need_down else None
        grad_up = torch.empty(adapters, outer, rank, dtype=torch.bfloat16, device=device) if need_up else None
        room = _hip.library().ep_hip_low_rank_grad_workspace_for(groups.entries, adapters, rank, inner, outer, need_x, need_down, need_up)
        workspace = torch.empty(room, dtype=torch.uint8, device=device)
        slope = matrix(grad, 8)
        _hip.launch("ep_hip_low_rank_update_grad", device,
                    slope.data_ptr(), slope.stride(0), rows.data_ptr(), rows.stride(0), narrow.data_ptr(), narrow.stride(1), narrow.stride(0),
                    wide.data_ptr(), wide.stride(1), wide.stride(0), None if scale is None else scale.data_ptr(),
                    None if planes is None else planes.data_ptr(), None if grad_x is None else grad_x.data_ptr(), inner,
                    None if grad_down is None else grad_down.data_ptr(), None if grad_up is None else grad_up.data_ptr(),
                    groups.order.data_ptr(), groups.offsets.data_ptr(), groups.entries, adapters, rank, inner, outer,
                    workspace.data_ptr(), room)
        return grad if need_y else None, grad_x, grad_down, grad_up, None, None


def low_rank_update(y: torch.Tensor, x: torch.Tensor, down: torch.Tensor, up: torch.Tensor, groups: RowGroups,
                    scale: torch.Tensor | None = None) -> torch.Tensor:
    """y[t] + scale[a] * (x[t] @ down[a].T) @ up[a].T with a = the adapter of row t; rows without one come back as y.

    Args:
        y: bf16 [tokens, out_features], the shared projection's output.
        x: bf16 [tokens, in_features], its input.
        down: bf16 [adapters, rank, in_features]. up: bf16 [adapters, out_features, rank].
        groups: the plan of `group_rows(ids, adapters)` with one id per token.
        scale: f32 [adapters] or None for ones; it gets no gradient, and one that wants it is refused while gradients are recorded.

    Sums and the narrow rows between the two products are f32; the result is rounded to bf16 once. An infinity or NaN in a row's adapter makes that row's results NaN where it reaches them. Differentiable in y, x, down and
    up, in reverse mode.
    """
    if not isinstance(groups, RowGroups):
        raise TypeError(f"low_rank_update takes the plan that group_rows returns, got {type(groups).__name__}")
    for name, tensor in (("y", y), ("x", x), ("down", down), ("up", up)):
        if tensor.dtype != torch.bfloat16:
            raise TypeError(f"low_rank_update takes bfloat16 operands, got {name} in {tensor.dtype}")
    if groups.per_row != 1:
        raise ValueError(f"low_rank_update takes one adapter per row, the plan has {groups.per_row}")
    if down.dim() != 3 or up.dim() != 3 or down.shape[0] != groups.groups or up.shape[0] != groups.groups or down.shape[1] != up.shape[2]:
        raise ValueError(f"low_rank_update takes down [{groups.groups}, rank, in_features] and up [{groups.groups}, out_features, rank], "
                         f"got {tuple(down.shape)} and {tuple(up.shape)}")
    if tuple(x.shape) != (groups.tokens, down.shape[2]) or tuple(y.shape) != (groups.tokens, up.shape[1]):
        raise ValueError(f"low_rank_update takes x of shape {(groups.tokens, down.shape[2])} and y of shape {(groups.tokens, up.shape[1])}, "
                         f"got {tuple(x.shape)} and {tuple(y.shape)}")
    if 0 in down.shape or 0 in up.shape:
        raise ValueError("low_rank_update needs at least one feature and rank one")
    if down.shape[1] > MAX_RANK:
        raise ValueError(f"low_rank_update takes ranks up to {MAX_RANK}, got {down.shape[1]}")
    refuse_tangents("low_rank_update", y, x, down, up, scale)
    if scale is not None:
        if tuple(scale.shape) != (groups.groups,):
            raise ValueError(f"low_rank_update takes one scale per adapter, got shape {tuple(scale.shape)}")
        if scale.requires_grad and torch.is_grad_enabled():
            raise ValueError("low_rank_update gives no gradient of the scale: detach it")
        scale = scale if scale.dtype == torch.float32 and scale.is_contiguous() else scale.float().contiguous()
    device_of("low_rank_update", y, x, down, up, groups.order, scale)
    if groups.tokens == 0:
        return y + (x.sum() + down.sum() + up.sum()) * 0
    if torch.is_grad_enabled() and (y.requires_grad or x.requires_grad or down.requires_grad or up.requires_grad):
        return _LowRankUpdate.apply(y, x, down, up, scale, groups)
    return _update(y, x, down, up, scale, groups)[0]


class AdaptedLinear(torch.nn.Module):
    """A compressed linear layer with a bank of low-rank adapters, one of them (or none) per activation row.

    Args:
        base: a `CompressedLinear` or a subclass of it; its weight stays frozen.
        adapters: how many the bank holds. rank: of every adapter; a smaller one is stored padded with zeros.

    `down` starts with small random values and `up` with zeros, so that a new adapter changes nothing until it is trained or set;
    both are trainable parameters. `scale` is a buffer of ones. Casting the layer (`.to(dtype)`, `.half()`, ..) casts none of the three: the
    kernels take the adapters in bf16 and the scales in f32.
    """

    def __init__(self, base: CompressedLinear, adapters: int, rank: int):
        super().__init__()
        if not isinstance(base, CompressedLinear):
            raise TypeError(f"AdaptedLinear takes a compressed linear layer, got {type(base).__name__}")
        for name, value, most in (("adapters", adapters, MAX_GROUPS), ("rank", rank, MAX_RANK)):
            if isinstance(value, bool) or not isinstance(value, int) or not 1 <= value <= most:
                raise ValueError(f"{name} must be an integer from 1 to {most}, got {value!r}")
        self.base = base
        device = base.device
        self.down = torch.nn.Parameter(torch.randn(adapters, rank, base.in_features, device=device).mul_(base.in_features ** -0.5).bfloat16())
        self.up = torch.nn.Parameter(torch.zeros(adapters, base.out_features, rank, dtype=torch.bfloat16, device=device))
        self.register_buffer("scale", torch.ones(adapters, device=device))

    @property
    def adapters(self) -> int:
        return self.down.shape[0]

    @property
    def rank(self) -> int:
        return self.down.shape[1]

    def _apply(self, fn, recurse=True):
        def keep(tensor):
            moved = fn(tensor)
            return moved if moved.dtype == tensor.dtype else tensor.to(device=moved.device)

        if recurse:
            self.base._apply(fn)
        return super()._apply(keep, recurse=False)

    @torch.no_grad()
    def set_adapter(self, index: int, down: torch.Tensor, up: torch.Tensor, scale: float = 1.0) -> None:
        """Stores one adapter: down [r, in_features], up [out_features, r], r at most the bank's rank."""
        if not 0 <= index < self.adapters:
            raise IndexError(f"adapter {index} of a bank of {self.adapters}")
        rank = down.shape[0]
        if rank > self.rank or tuple(down.shape) != (rank, self.base.in_features) or tuple(up.shape) != (self.base.out_features, rank):
            raise ValueError(f"an adapter of this bank has down [r, {self.base.in_features}] and up [{self.base.out_features}, r] with r up to "
                             f"{self.rank}, got {tuple(down.shape)} and {tuple(up.shape)}")
        fresh_down, fresh_up = torch.zeros_like(self.down[index]), torch.zeros_like(self.up[index])    # the source may be a part of this slot
        fresh_down[:rank].copy_(down)
        fresh_up[:, :rank].copy_(up)
        self.down[index].copy_(fresh_down)
        self.up[index].copy_(fresh_up)
        self.scale[index] = scale

    def forward(self, x: torch.Tensor, groups: RowGroups) -> torch.Tensor:
        """base(x) plus every row's update; x [.., in_features] in bf16, `groups` one id per row of x."""
        y = self.base(x)
        rows = low_rank_update(y.reshape(-1, y.shape[-1]), x.reshape(-1, x.shape[-1]), self.down, self.up, groups, self.scale)
        return rows.reshape(y.shape)

    def extra_repr(self) -> str:
        return f"adapters={self.adapters}, rank={self.rank}"


__all__ = ["AdaptedLinear", "low_rank_update"]
