"""Products of grouped rows with the weight of their group: a mixture of experts whose weights are stored compressed.

`grouped_linear` (bf16, differentiable) and `grouped_int8_linear` (W8A8) are the products on dense weights;
`CompressedGroupedLinear` holds one compressed layer per expert, decodes them all in one batched pass and multiplies.
The plan of a step comes from `group_rows`, the way back to the tokens is `combine_rows` (`linear/groups.py`):

    groups = ep.group_rows(expert_ids, experts.groups)            # ids [tokens, k]
    hidden = torch.nn.functional.silu(gate(x, groups)) * up(x, groups)
    y = ep.combine_rows(down(hidden, groups, x_grouped=True), groups, router_weights)

The reference has no counterpart: its layers have one weight each (entropack/linear/linear.py:18-230, 447-490).
"""
from __future__ import annotations

import torch

from ..backends import hip as _hip
from ..compression import BatchDecompressor
from . import kernels
from .groups import MAX_GROUPS, RowGroups, device_of, first_order, matrix, refuse_tangents, rows_of, sum_entries
from .linear import FORWARD_MODES, CompressedINT8Linear, CompressedLinear


def _check_groups(name: str, x: torch.Tensor, weight: torch.Tensor, groups: RowGroups, bias, x_grouped: bool) -> None:
    if not isinstance(groups, RowGroups):
        raise TypeError(f"{name} takes the plan that group_rows returns, got {type(groups).__name__}")
    if weight.dim() != 3 or weight.shape[0] != groups.groups:
        raise ValueError(f"{name} takes a weight of shape [{groups.groups}, out_features, in_features], got {tuple(weight.shape)}")
    rows = groups.entries if x_grouped else groups.tokens
    if x.dim() != 2 or x.shape[0] != rows:
        raise ValueError(f"{name} takes {rows} rows of x ({'one per entry' if x_grouped else 'one per token'}), got shape {tuple(x.shape)}")
    if x.shape[1] != weight.shape[2] or x.shape[1] == 0 or weight.shape[1] == 0:
        raise ValueError(f"{name}: x has {x.shape[1]} features, the weight is {tuple(weight.shape)}")
    if bias is not None and tuple(bias.shape) != tuple(weight.shape[:2]):
        raise ValueError(f"{name} takes a bias of shape {tuple(weight.shape[:2])}, got {tuple(bias.shape)}")


def _forward(x, weight, bias, groups: RowGroups, x_grouped: bool) -> torch.Tensor:
    outer = weight.shape[1]
    y = torch.empty(groups.entries, outer, dtype=torch.bfloat16, device=x.device)
    if y.numel():
        rows, w = matrix(x, 8), matrix(weight, 8)
        ready = None if bias is None else bias.contiguous()
        _hip.launch("ep_hip_grouped_gemm_bf16", x.device,
                    rows.data_ptr(), rows.stride(0), rows.shape[0], w.data_ptr(), w.stride(1), w.stride(0),
                    None if ready is None else ready.data_ptr(), y.data_ptr(), outer, _hip.FLOAT_KINDS[torch.bfloat16],
                    None if x_grouped else groups.rows.data_ptr(), groups.offsets.data_ptr(), groups.entries,
                    groups.groups, outer, rows.shape[1])
    return y


def _grad_rows(grad, weight, groups: RowGroups, x_grouped: bool) -> torch.Tensor:
    """The gradient of x. A token with several entries takes the sum of their gradients: those stay in f32 until they are
    added, so that the result is rounded once."""
    inner = weight.shape[2]
    summed = not x_grouped and groups.per_row > 1
    out = torch.empty(groups.entries, inner, dtype=torch.float32 if summed else torch.bfloat16, device=grad.device)
    if out.numel():
        dy, w = matrix(grad, 8), matrix(weight, 8)
        if w.shape[2] != inner:                                  # padded columns would be written past the rows of out
            out = torch.empty(groups.entries, w.shape[2], dtype=out.dtype, device=grad.device)
        _hip.launch("ep_hip_grouped_grad_rows_bf16", grad.device,
                    dy.data_ptr(), dy.stride(0), w.data_ptr(), w.stride(1), w.stride(0), out.data_ptr(), out.stride(0),
                    _hip.FLOAT_KINDS[out.dtype], None if x_grouped else groups.order.data_ptr(), groups.offsets.data_ptr(),
                    groups.entries, groups.groups, w.shape[1], w.shape[2])
    if summed:
        out = sum_entries(out, groups.tokens, groups.per_row)
    return out if out.shape[1] == inner else out[:, :inner].contiguous()


def _grad_weight(grad, x, weight, groups: RowGroups, x_grouped: bool) -> torch.Tensor:
    if groups.entries == 0:
        return torch.zeros(weight.shape, dtype=weight.dtype, device=weight.device)
    dy, rows = matrix(grad, 8), matrix(x, 8)
    outer, inner = dy.shape[1], rows.shape[1]
    out = torch.empty(groups.groups, outer, inner, dtype=torch.bfloat16, device=grad.device)
    room = _hip.library().ep_hip_grouped_grad_weight_workspace(groups.entries, groups.groups, outer, inner)
    workspace = torch.empty(room, dtype=torch.uint8, device=grad.device) if room else None
    _hip.launch("ep_hip_grouped_grad_weight_bf16", grad.device,
                dy.data_ptr(), dy.stride(0), rows.data_ptr(), rows.stride(0), rows.shape[0], out.data_ptr(), inner, outer * inner,
                _hip.FLOAT_KINDS[torch.bfloat16], None if x_grouped else groups.rows.data_ptr(),
                groups.offsets.data_ptr(), groups.entries, groups.groups, outer, inner,
                None if workspace is None else workspace.data_ptr(), room)
    return out if tuple(out.shape) == tuple(weight.shape) else out[:, :weight.shape[1], :weight.shape[2]].contiguous()


def _grad_bias(grad, groups: RowGroups, dtype: torch.dtype) -> torch.Tensor:
    outer = grad.shape[1]
    if groups.entries == 0:
        return torch.zeros(groups.groups, outer, dtype=dtype, device=grad.device)
    dy = rows_of(grad)
    out = torch.empty(groups.groups, outer, dtype=dtype, device=grad.device)
    _hip.launch("ep_hip_grouped_column_sums_bf16", grad.device,
                dy.data_ptr(), dy.stride(0), groups.offsets.data_ptr(), groups.groups, outer, out.data_ptr(), _hip.FLOAT_KINDS[dtype])
    return out


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, x_grouped):
        ctx.groups, ctx.x_grouped = groups, x_grouped
        ctx.save_for_backward(x, weight)
        return _forward(x, weight, bias, groups, x_grouped)

    @staticmethod
    @first_order
    def backward(ctx, grad):
        x, weight = ctx.saved_tensors
        need_x, need_weight, need_bias = ctx.needs_input_grad[:3]
        return (_grad_rows(grad, weight, ctx.groups, ctx.x_grouped) if need_x else None,
                _grad_weight(grad, x, weight, ctx.groups, ctx.x_grouped) if need_weight else None,
                _grad_bias(grad, ctx.groups, torch.bfloat16) if need_bias else None, None, None)


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, groups: RowGroups, bias: torch.Tensor | None = None, *,
                   x_grouped: bool = False) -> torch.Tensor:
    """y[p] = x[token of place p] @ weight[g].T (+ bias[g]) for every place p of every group g; [entries, out_features] bf16 in
    grouped order. Places of no group are zero.

    Args:
        x: bf16 [tokens, in_features]; each token's row is read once per entry. With `x_grouped`, [entries, in_features] in
            grouped order, such as an earlier product's result.
        weight: bf16 [groups, out_features, in_features]; groups and rows may be strided (views of an arena).
        groups: the plan of `group_rows`.
        bias: bf16 [groups, out_features] or None.

    Sums are f32, rounded to bf16 once. Differentiable in x, weight and bias, in reverse mode. Feature counts that are no multiple of 8 are
    padded, which copies the operand.
    """
    _check_groups("grouped_linear", x, weight, groups, bias, x_grouped)
    for name, tensor in (("x", x), ("weight", weight), ("bias", bias)):
        if tensor is not None and tensor.dtype != torch.bfloat16:
            raise TypeError(f"grouped_linear takes bfloat16 operands, got {name} in {tensor.dtype}")
    device_of("grouped_linear", x, weight, groups.order, bias)
    refuse_tangents("grouped_linear", x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _GroupedLinear.apply(x, weight, bias, groups, x_grouped)
    return _forward(x, weight, bias, groups, x_grouped)


def grouped_int8_linear(x: torch.Tensor, weight: torch.Tensor, groups: RowGroups, x_scale: torch.Tensor, weight_scale: torch.Tensor,
                        bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16, *, x_grouped: bool = False) -> torch.Tensor:
    """The W8A8 form of `grouped_linear`: (x codes . weight codes) in int32, times both rows' scales, plus bias.

    Args:
        x: int8 [tokens, in_features] (or [entries, ..] in grouped order with `x_grouped`), as `quantize_rows` gives it.
        weight: int8 [groups, out_features, in_features].
        x_scale: f32, one per row of x. weight_scale: f32 [groups, out_features].
        bias: [groups, out_features] or None. out_dtype: bfloat16, float16 or float32.

    Nothing gets a gradient; scales and biases that want one are refused while gradients are recorded.
    """
    _check_groups("grouped_int8_linear", x, weight, groups, bias, x_grouped)
    if x.dtype != torch.int8 or weight.dtype != torch.int8:
        raise TypeError(f"grouped_int8_linear takes int8 codes, got {x.dtype} and {weight.dtype}")
    if out_dtype not in _hip.FLOAT_KINDS:
        raise TypeError(f"grouped_int8_linear returns bfloat16, float16 or float32, not {out_dtype}")
    if x_scale.numel() != x.shape[0] or tuple(weight_scale.shape) != tuple(weight.shape[:2]):
        raise ValueError(f"grouped_int8_linear takes {x.shape[0]} activation scales and weight scales of shape {tuple(weight.shape[:2])}, "
                         f"got {tuple(x_scale.shape)} and {tuple(weight_scale.shape)}")
    for name, tensor in (("x_scale", x_scale), ("weight_scale", weight_scale), ("bias", bias)):
        if tensor is not None and tensor.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"grouped_int8_linear gives no gradient of {name}: detach it")
    device = device_of("grouped_int8_linear", x, weight, groups.order, x_scale, weight_scale, bias)
    refuse_tangents("grouped_int8_linear", x_scale, weight_scale, bias)
    outer = weight.shape[1]
    y = torch.empty(groups.entries, outer, dtype=out_dtype, device=device)
    if y.numel() == 0:
        return y
    rows, w = matrix(x, 16), matrix(weight, 16)
    ready = None if bias is None else bias.detach().to(out_dtype).contiguous()
    scale_x, scale_w = x_scale.detach().float().contiguous(), weight_scale.detach().float().contiguous()
    _hip.launch("ep_hip_grouped_gemm_i8", device,
                rows.data_ptr(), rows.stride(0), rows.shape[0], w.data_ptr(), w.stride(1), w.stride(0), scale_x.data_ptr(), scale_w.data_ptr(),
                None if ready is None else ready.data_ptr(), y.data_ptr(), outer, _hip.FLOAT_KINDS[out_dtype],
                None if x_grouped else groups.rows.data_ptr(), groups.offsets.data_ptr(), groups.entries, groups.groups,
                outer, rows.shape[1])
    return y


class _CompressedGrouped(torch.autograd.Function):
    """The forward on decoded weights with the gradients of the activations and of the biases; the weights are decoded again for the
    first (they are frozen and get no gradient), as in the layers' own fused forward."""

    @staticmethod
    def forward(ctx, x, biases, layer, groups, x_grouped):
        ctx.layer, ctx.groups, ctx.x_grouped = layer, groups, x_grouped
        ctx.bias_dtype = biases.dtype if biases is not None and biases.dtype in _hip.FLOAT_KINDS else torch.float32      # of int8 experts, any
        return layer._product(x.detach(), biases, groups, x_grouped)

    @staticmethod
    @first_order
    def backward(ctx, grad):
        need_x, need_biases = ctx.needs_input_grad[:2]
        return (_grad_rows(grad, ctx.layer.dequantize(grad.device).to(grad.dtype), ctx.groups, ctx.x_grouped) if need_x else None,
                _grad_bias(grad, ctx.groups, ctx.bias_dtype) if need_biases else None, None, None, None)


class CompressedGroupedLinear(torch.nn.Module):
    """The same projection of every expert of a mixture, each expert's weight compressed in a layer of its own.

    `experts`: `CompressedLinear` layers (bf16 containers) or `CompressedINT8Linear` layers, one class, one shape, with
    biases in all of them or in none, with the default `forward_mode` and no `DecodeAhead` attached (this layer decodes and multiplies by
    itself, and would use neither). They stay ordinary submodules: `state_dict` holds `experts.<i>.weight.entropack_quant_state`
    and so on. A forward decodes all experts (in one pass when their weights are `lattice_rans` containers), then runs
    `grouped_linear` or, for int8 experts, the row quantiser and `grouped_int8_linear`. Differentiable in x and in the biases (which the
    layers keep frozen unless asked otherwise). The first forward
    plans the decode, which copies to the device: run one before capturing a graph. The plan is made again when a container changes or the
    layer moves; of experts kept on the host it holds a copy of the containers on the device.
    """

    def __init__(self, experts):
        super().__init__()
        experts = list(experts)
        if not experts:
            raise ValueError("CompressedGroupedLinear needs at least one expert")
        if len(experts) > MAX_GROUPS:
            raise ValueError(f"CompressedGroupedLinear takes at most {MAX_GROUPS} experts, got {len(experts)}")
        first = experts[0]
        kind = CompressedINT8Linear if isinstance(first, CompressedINT8Linear) else CompressedLinear
        for expert in experts:
            if type(expert) is not type(first) or type(first) not in (CompressedLinear, CompressedINT8Linear):
                raise TypeError("CompressedGroupedLinear takes CompressedLinear layers or CompressedINT8Linear layers, all of one class, "
                                f"got {type(expert).__name__} beside {type(first).__name__}")
            if (expert.in_features, expert.out_features) != (first.in_features, first.out_features):
                raise ValueError("the experts' shapes differ")
            if (expert.bias is None) != (first.bias is None):
                raise ValueError("biases in all experts or in none")
            if kind is CompressedLinear and expert.container_dtype != torch.bfloat16:
                raise TypeError(f"grouped products run in bfloat16, got an expert of {expert.container_dtype}")
            if kind is CompressedINT8Linear and expert._convrot_group != first._convrot_group:
                raise ValueError("the experts' rotation groups differ")
        self.experts = torch.nn.ModuleList(experts)
        self.in_features, self.out_features = first.in_features, first.out_features
        self._check_settings()
        self._int8 = kind is CompressedINT8Linear
        self._decoder = None            # (device, the experts' payloads it was planned for, BatchDecompressor)

    @classmethod
    def from_linears(cls, linears, *, int8: bool = False, **kwargs) -> "CompressedGroupedLinear":
        """Compresses one `torch.nn.Linear` per expert; keyword arguments go to the layers' `from_linear`."""
        layer_class = CompressedINT8Linear if int8 else CompressedLinear
        return cls([layer_class.from_linear(linear, **kwargs) for linear in linears])

    def __getstate__(self):
        # A decode plan holds addresses of this object's containers: a copy makes its own.
        return {**self.__dict__, "_decoder": None}

    def _apply(self, fn, recurse=True):
        self._decoder = None            # it keeps the containers that are about to be left behind
        return super()._apply(fn, recurse=recurse)

    def _load_from_state_dict(self, *args, **kwargs):
        self._decoder = None
        super()._load_from_state_dict(*args, **kwargs)

    @property
    def groups(self) -> int:
        return len(self.experts)

    def _check_settings(self) -> None:
        """Refuses experts that were told to work in another way than this layer does."""
        for expert in self.experts:
            if expert.forward_mode != FORWARD_MODES[0]:
                raise ValueError(f"CompressedGroupedLinear decodes its experts and multiplies, forward_mode {FORWARD_MODES[0]!r}, got an expert with {expert.forward_mode!r}")
            if expert._decode_ahead is not None:
                raise ValueError("CompressedGroupedLinear decodes its experts by itself, got one that is attached to a DecodeAhead: close that first")

    def _stacked(self, device: torch.device) -> torch.Tensor:
        """All experts' containers decoded: [experts, out_features, in_features] in the containers' dtype."""
        self._check_settings()
        containers = [expert._container() for expert in self.experts]
        if any(container.compress_method != "lattice_rans" for container in containers):
            return torch.stack([expert.codes(device) if self._int8 else expert.dequantize(device).to(expert.container_dtype) for expert in self.experts])
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        held = self._decoder
        if held is None or held[0] != device or any(container.buffers["payload"] is not payload for container, payload in zip(containers, held[1])):
            here = [container.to(device=device, dtype=expert.container_dtype) for container, expert in zip(containers, self.experts)]
            held = self._decoder = (device, [container.buffers["payload"] for container in containers], BatchDecompressor(here, self.experts[0]._decode_config))
        arena = torch.empty(held[2].arena_bytes, dtype=torch.uint8, device=device)
        views = held[2](arena)
        if any(view.untyped_storage().data_ptr() != arena.data_ptr() for view in views):
            return torch.stack(views)                        # a type the decode stores as another and converts
        size, row = views[0].element_size(), views[0].stride(0)
        apart = row * self.out_features if len(views) == 1 else (views[1].data_ptr() - views[0].data_ptr()) // size    # one shape, so even steps
        return torch.as_strided(views[0], (len(views), self.out_features, self.in_features), (apart, row, 1))

    def _product(self, x: torch.Tensor, biases: torch.Tensor | None, groups: RowGroups, x_grouped: bool) -> torch.Tensor:
        weight = self._stacked(x.device)
        if not self._int8:
            return grouped_linear(x, weight, groups, biases, x_grouped=x_grouped)
        first = self.experts[0]
        rows = x.contiguous()
        codes, scale = kernels.rotate_quantize_rows(rows, first._convrot_group) if first.use_convrot else kernels.quantize_rows(rows)
        scales = torch.stack([expert._scale(x.device) for expert in self.experts])
        return grouped_int8_linear(codes, weight, groups, scale, scales, biases, x.dtype, x_grouped=x_grouped)

    def dequantize(self, device=None) -> torch.Tensor:
        """The dense weights [experts, out_features, in_features]."""
        if self._int8:
            return torch.stack([expert.dequantize(device) for expert in self.experts])
        return self._stacked(torch.device(device) if device is not None else self.experts[0].device)

    def forward(self, x: torch.Tensor, groups: RowGroups, *, x_grouped: bool = False) -> torch.Tensor:
        """`grouped_linear` with the experts' weights: bf16 x, [entries, out_features] in grouped order."""
        if x.dtype != torch.bfloat16:
            raise TypeError(f"CompressedGroupedLinear runs in bfloat16, got {x.dtype}")
        device_of("CompressedGroupedLinear", x)
        refuse_tangents("CompressedGroupedLinear", x)
        if not isinstance(groups, RowGroups):
            raise TypeError(f"CompressedGroupedLinear takes the plan that group_rows returns, got {type(groups).__name__}")
        if groups.groups != self.groups:
            raise ValueError(f"the plan has {groups.groups} groups, the layer {self.groups} experts")
        rows = groups.entries if x_grouped else groups.tokens
        if x.dim() != 2 or tuple(x.shape) != (rows, self.in_features):
            raise ValueError(f"CompressedGroupedLinear takes x of shape {(rows, self.in_features)}, got {tuple(x.shape)}")
        if groups.entries == 0:
            return x.new_zeros(0, self.out_features) + x.sum() * 0
        biases = None if self.experts[0].bias is None else torch.stack([expert._bias_on(x.device) for expert in self.experts])
        if torch.is_grad_enabled() and (x.requires_grad or (biases is not None and biases.requires_grad)):
            return _CompressedGrouped.apply(x, biases, self, groups, x_grouped)
        return self._product(x, biases, groups, x_grouped)

    def extra_repr(self) -> str:
        return f"experts={self.groups}, in_features={self.in_features}, out_features={self.out_features}"


__all__ = ["CompressedGroupedLinear", "grouped_int8_linear", "grouped_linear"]
