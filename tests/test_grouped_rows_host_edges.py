"""The operators on grouped rows without a device, continued: derivatives that they do not give, layers moved, cast and put together in
ways they cannot serve, sizes beyond a launch. Kernels are replaced by nothing where a call would reach them: what is tested is what
the call refuses, or what it hands on."""
import pytest
import torch
from torch.autograd import forward_ad

import entropack_amd as ep
from entropack_amd.backends import hip
from entropack_amd.linear import adapters, grouped, groups


def _plan(tokens=3, per_row=2, count=4):
    entries = tokens * per_row
    index = torch.arange(entries, dtype=torch.int32)
    return ep.RowGroups(index, torch.full((count + 1,), entries, dtype=torch.int32), index.clone(), index // per_row, count, tokens, per_row)


def _bf16(*shape):
    return torch.ones(*shape, dtype=torch.bfloat16)


@pytest.fixture
def no_device(monkeypatch):
    """The operators on host tensors, every kernel replaced by nothing; yields the names of those that were called."""
    called = []
    monkeypatch.setattr(hip, "launch", lambda name, *rest: called.append(name))
    for module in (adapters, grouped, groups):
        monkeypatch.setattr(module, "device_of", lambda name, *tensors: torch.device("cpu"))
    return called


OPERATORS = [("grouped_linear", lambda x, w, b: ep.grouped_linear(x, w, _plan(), b), (_bf16(3, 8), _bf16(4, 5, 8), _bf16(4, 5))),
             ("combine_rows", lambda y, w: ep.combine_rows(y, _plan(), w), (_bf16(6, 8), torch.ones(3, 2))),
             ("low_rank_update", lambda y, x, d, u: ep.low_rank_update(y, x, d, u, _plan(per_row=1)), (_bf16(3, 10), _bf16(3, 8), _bf16(4, 2, 8), _bf16(4, 10, 2))),
             ("low_rank_update's scale", lambda s: ep.low_rank_update(_bf16(3, 10), _bf16(3, 8), _bf16(4, 2, 8), _bf16(4, 10, 2), _plan(per_row=1), s), (torch.ones(4),)),
             ("grouped_int8_linear", lambda sx, sw, b: ep.grouped_int8_linear(torch.ones(3, 16, dtype=torch.int8), torch.ones(4, 5, 16, dtype=torch.int8), _plan(), sx, sw, b),
              (torch.ones(3), torch.ones(4, 5), _bf16(4, 5)))]


@pytest.mark.parametrize("name,run,operands", OPERATORS, ids=[o[0] for o in OPERATORS])
@pytest.mark.parametrize("recording", [True, False], ids=["grad", "no_grad"])
def test_forward_mode_derivatives_are_refused_not_dropped(no_device, name, run, operands, recording):
    run(*operands)                                                                       # without tangents the call is fine
    for which in range(len(operands)):
        def of_one(t):
            return run(*[t if i == which else o for i, o in enumerate(operands)])

        with torch.set_grad_enabled(recording):
            before = len(no_device)
            with forward_ad.dual_level():
                assert forward_ad.unpack_dual(run(*operands)).tangent is None                # nor does a level without tangents matter
                with pytest.raises((RuntimeError, ValueError), match="forward-mode|jvp|JVP"):
                    of_one(forward_ad.make_dual(operands[which], torch.ones_like(operands[which])))
            with pytest.raises((RuntimeError, ValueError)):
                torch.func.jvp(of_one, (operands[which],), (torch.ones_like(operands[which]),))
            with pytest.raises((RuntimeError, ValueError)):
                torch.func.vmap(of_one)(operands[which].unsqueeze(0).expand(2, *operands[which].shape).clone())


def test_a_mixtures_forward_mode_derivative_is_refused(no_device):
    experts = ep.CompressedGroupedLinear([ep.CompressedLinear(8, 5) for _ in range(4)])
    experts._stacked = lambda device: _bf16(4, 5, 8)
    assert experts(_bf16(3, 8), _plan()).shape == (6, 5)
    with forward_ad.dual_level(), pytest.raises((RuntimeError, ValueError), match="forward-mode|jvp|JVP"):
        experts(forward_ad.make_dual(_bf16(3, 8), _bf16(3, 8)), _plan())


@pytest.mark.parametrize("name,run,operands", OPERATORS[:3], ids=[o[0] for o in OPERATORS[:3]])
def test_a_gradient_with_a_tangent_is_refused(no_device, name, run, operands):
    leaves = [t.clone().requires_grad_(True) for t in operands]
    out = run(*leaves)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        torch.autograd.grad(out, leaves[0], forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))


@pytest.mark.parametrize("of_x", [False, True], ids=["biases alone", "and x"])
def test_a_mixture_hands_its_biases_their_gradients(no_device, monkeypatch, of_x):
    monkeypatch.setattr(grouped, "_grad_rows", lambda grad, weight, plan, x_grouped: torch.full((3, 8), 2.0, dtype=grad.dtype))
    monkeypatch.setattr(grouped, "_grad_bias", lambda grad, plan, dtype: torch.arange(20.0, dtype=grad.dtype).reshape(4, 5))
    layer = ep.CompressedGroupedLinear([ep.CompressedLinear(8, 5) for _ in range(4)])
    layer._stacked = lambda device: _bf16(4, 5, 8)
    biases = [expert.bias.requires_grad_(True) for expert in layer.experts]
    x = _bf16(3, 8).requires_grad_(of_x)
    layer(x, _plan()).sum().backward()
    assert torch.equal(torch.stack([bias.grad for bias in biases]), torch.arange(20.0).reshape(4, 5).bfloat16())
    assert (x.grad is not None) == of_x


def test_biases_of_any_float_type_get_their_gradient(no_device, monkeypatch):
    asked = []
    monkeypatch.setattr(grouped, "_grad_bias", lambda grad, plan, dtype: asked.append(dtype) or torch.ones(4, 5, dtype=dtype))
    monkeypatch.setattr(grouped.kernels, "quantize_rows", lambda rows: (torch.ones(rows.shape, dtype=torch.int8), torch.ones(len(rows))))
    for dtype, sums in ((torch.float64, torch.float32), (torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16)):
        layer = ep.CompressedGroupedLinear([ep.CompressedINT8Linear(16, 5) for _ in range(4)]).to(dtype)
        layer._stacked = lambda device: torch.ones(4, 5, 16, dtype=torch.int8)
        biases = [expert.bias.requires_grad_(True) for expert in layer.experts]
        layer(_bf16(3, 16), _plan()).sum().backward()
        assert asked.pop() == sums and all(bias.grad.dtype == dtype and bias.grad.eq(1).all() for bias in biases)


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(), lambda m: torch.nn.Sequential(m).half()[0]], ids=["bf16", "half", "double", "inside a model"])
def test_casting_an_adapted_layer_leaves_its_bank_as_the_kernels_take_it(cast):
    layer = ep.AdaptedLinear(ep.CompressedLinear(16, 8), 3, 4)
    layer.set_adapter(1, torch.randn(4, 16), torch.randn(8, 4), scale=1.0 / 3.0)
    down, up, scale = layer.down.detach().clone(), layer.up.detach().clone(), layer.scale.clone()
    parameters = list(layer.parameters())
    cast(layer)
    assert layer.down.dtype == layer.up.dtype == torch.bfloat16 and layer.scale.dtype == torch.float32
    assert torch.equal(layer.down, down) and torch.equal(layer.up, up) and torch.equal(layer.scale, scale) and layer.down.requires_grad
    assert all(a is b for a, b in zip(parameters, layer.parameters()))              # an optimiser's own
    meta = layer.to("meta")
    assert meta.down.device.type == meta.scale.device.type == "meta" and meta.scale.dtype == torch.float32
    empty = meta.to_empty(device="cpu")
    assert empty.up.device.type == "cpu" and empty.up.dtype == torch.bfloat16


def test_an_adapter_set_from_a_part_of_its_own_slot():
    layer = ep.AdaptedLinear(ep.CompressedLinear(16, 8), 2, 4)
    layer.set_adapter(1, torch.randn(4, 16), torch.randn(8, 4))
    down, up = layer.down[1].detach().clone(), layer.up[1].detach().clone()
    layer.set_adapter(1, layer.down[1, 1:3], layer.up[1, :, 1:3], scale=2.0)         # two of its four ranks kept
    assert torch.equal(layer.down[1, :2], down[1:3]) and torch.equal(layer.up[1, :, :2], up[:, 1:3])
    assert layer.down[1, 2:].eq(0).all() and layer.up[1, :, 2:].eq(0).all() and layer.scale.tolist() == [1.0, 2.0]


def test_a_bank_that_no_forward_could_use_is_refused():
    base = ep.CompressedLinear(16, 8)
    for count, rank in ((groups.MAX_GROUPS + 1, 1), (1, 4097)):
        with pytest.raises(ValueError, match="from 1 to"):
            ep.AdaptedLinear(base, count, rank)
    assert ep.AdaptedLinear(base, groups.MAX_GROUPS, 1).adapters == 896 and ep.AdaptedLinear(base, 1, 4096).rank == 4096
    experts = [ep.CompressedLinear(16, 8) for _ in range(groups.MAX_GROUPS + 1)]
    with pytest.raises(ValueError, match="at most 896"):
        ep.CompressedGroupedLinear(experts)
    assert ep.CompressedGroupedLinear(experts[:-1]).groups == 896


def test_a_mixture_that_moves_or_is_loaded_lets_go_of_its_decode_plan():
    layer = ep.CompressedGroupedLinear([ep.CompressedLinear(16, 8) for _ in range(2)])
    for change in (lambda: layer.cpu(), lambda: layer.to(torch.bfloat16), lambda: torch.nn.Sequential(layer).cpu(),
                   lambda: layer.load_state_dict(layer.state_dict(), strict=False), lambda: torch.nn.Sequential(layer).load_state_dict({}, strict=False)):
        layer._decoder = object()
        change()
        assert layer._decoder is None


def test_a_mixture_plans_once_wherever_its_containers_are(monkeypatch):
    """Neither containers on another device than x nor a cast, which both need new tensors for the decode, make a plan per call."""
    config, made = ep.EntroPackLossyConfig(target_bpp=4.0, execution_backend="eager"), []

    class Plan:
        arena_bytes = 2 * 8 * 16 * 2

        def __init__(self, containers, config):
            made.append([container.dtype for container in containers])

        def __call__(self, arena):
            return list(arena.view(torch.bfloat16).view(2, 8, 16).unbind(0))

    monkeypatch.setattr(grouped, "BatchDecompressor", Plan)
    layer = ep.CompressedGroupedLinear.from_linears([torch.nn.Linear(16, 8, dtype=torch.bfloat16) for _ in range(2)], config=config)
    layer.float()
    for _ in range(3):
        assert layer._stacked(torch.device("cpu")).shape == (2, 8, 16)
    assert made == [[torch.bfloat16] * 2]
    layer._stacked(torch.device("meta"))                                               # another device, another plan
    assert len(made) == 2
    layer.experts[1].compress_weight(torch.randn(8, 16))                               # another container, another plan
    layer._stacked(torch.device("meta"))
    layer._stacked(torch.device("meta"))
    assert len(made) == 3


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_a_mixture_refuses_experts_with_settings_that_it_would_not_follow(int8):
    kind = ep.CompressedINT8Linear if int8 else ep.CompressedLinear
    for mode in ("fused", "fused_through_lds"):
        with pytest.raises(ValueError, match="forward_mode"):
            ep.CompressedGroupedLinear([kind(16, 8), kind(16, 8, forward_mode=mode)])
    attached = kind(16, 8)
    attached._decode_ahead = object()
    with pytest.raises(ValueError, match="DecodeAhead"):
        ep.CompressedGroupedLinear([kind(16, 8), attached])
    layer = ep.CompressedGroupedLinear([kind(16, 8) for _ in range(2)])               # set afterwards: the forward refuses
    layer.experts[1].forward_mode = "fused"
    with pytest.raises(ValueError, match="forward_mode"):
        layer.dequantize() if not int8 else layer._stacked(torch.device("cpu"))
    layer.experts[1].forward_mode, layer.experts[0]._decode_ahead = "decode_then_gemm", object()
    with pytest.raises(ValueError, match="DecodeAhead"):
        layer._stacked(torch.device("cpu"))


def test_operands_whose_gradient_is_not_given_are_refused_only_while_gradients_are_recorded(no_device):
    name, run, operands = OPERATORS[4]
    for which in range(len(operands)):
        leaf = operands[which].clone().requires_grad_(True)
        with pytest.raises(ValueError, match="gives no gradient"):
            run(*[leaf if i == which else o for i, o in enumerate(operands)])
        with torch.no_grad():
            assert run(*[leaf if i == which else o for i, o in enumerate(operands)]).shape == (6, 5)
    scaled = lambda s: OPERATORS[3][1](s)
    with pytest.raises(ValueError, match="gives no gradient"):
        scaled(torch.ones(4, requires_grad=True))
    with torch.no_grad():
        assert scaled(torch.ones(4, requires_grad=True)).shape == (3, 10)


def test_launches_of_too_many_work_items_are_refused_before_they_are_made():
    """A launch has fewer than 2^32 work items. Nothing is launched, so no device is needed and no address is followed."""
    lib, at = hip.library(), 4096
    update = lambda rows, count: lib.ep_hip_low_rank_update(at, 16, at, 16, 64, at, 4, 64, None, at, 16, at, at, 16, at, at, rows, count, 4, 16, 16, None)
    grad = lambda rows, count: lib.ep_hip_low_rank_update_grad(at, 16, at, 16, at, 16, 64, at, 4, 64, None, at, at, 16, at, at, at, at, rows, count, 4, 16, 16, at, 1 << 62, None)
    sums = lambda count, columns: lib.ep_hip_grouped_column_sums_bf16(at, columns, at, count, columns, at, 0, None)
    for call in (update, grad):
        for rows, count in ((1 << 30, 1), (1 << 28, 2), ((1 << 28) - 14000, 896)):
            assert call(rows, count) == hip.EUNSUPPORTED
    assert sums(1, 1 << 30) == hip.EUNSUPPORTED and sums(500, 1 << 21) == hip.EUNSUPPORTED
    # 100 entries in 30 groups by 2^25 columns, 16 rows and 16 columns per block of 256 threads
    assert lib.ep_hip_grouped_gemm_bf16(at, 16, 100, at, 16, 64, None, at, 1 << 25, 0, at, at, 100, 30, 1 << 25, 16, None) == hip.EUNSUPPORTED


@pytest.mark.parametrize("entries,count,rank,inner,outer", [(1024, 64, 64, 8192, 8192), (1000, 896, 64, 4096, 4096), (7, 3, 5, 72, 40), (5000, 2, 16, 4096, 1024)])
def test_workspace_of_the_adapters_gradients_holds_what_is_asked_for(entries, count, rank, inner, outer):
    room = lambda *wanted: hip.library().ep_hip_low_rank_grad_workspace_for(entries, count, rank, inner, outer, *wanted)
    line = 256
    whole = lambda n, unit: -(-n // unit) * unit
    turned_up, turned_down = 2 * count * rank * whole(outer, 8), 2 * count * inner * whole(rank, 8)
    planes = entries * whole(rank, 16) * 8
    assert room(1, 0, 0) <= turned_up + turned_down + planes + 3 * line                # nothing of the weights' gradients
    down_parts, up_parts = room(0, 1, 0) - room(1, 0, 0) + whole(turned_down, line), room(0, 0, 1)
    assert room(0, 1, 0) == whole(turned_up, line) + whole(planes, line) + down_parts
    assert room(1, 1, 1) == room(1, 0, 0) + down_parts + up_parts == hip.library().ep_hip_low_rank_grad_workspace(entries, count, rank, inner, outer)
    assert room(0, 0, 0) == 0
    # The sums: an f32 matrix per chunk of 128 places or more, one at least for every adapter with places.
    chunks = min(count, entries) + entries // 128
    assert up_parts <= 4 * chunks * whole(rank, 16) * outer + line and down_parts <= 4 * chunks * whole(rank, 16) * inner + line
    at = 4096
    for gx, gd, gu in ((at, None, None), (None, at, None), (None, None, at), (at, at, None)):
        wanted = [int(p is not None) for p in (gx, gd, gu)]
        assert hip.library().ep_hip_low_rank_update_grad(at, whole(outer, 8), at, whole(inner, 8), at, whole(inner, 8), 0, at, rank, 0, None, at, gx, inner, gd, gu, at, at, entries, count,
                                                         rank, inner, outer, at, room(*wanted) - 1, None) == hip.EINVAL
