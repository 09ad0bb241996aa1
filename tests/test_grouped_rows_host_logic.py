"""The operators on grouped rows without a device: what they refuse, in Python and at the C entry points."""
import pytest
import torch

import entropack_amd as ep
from entropack_amd.backends import hip
from entropack_amd.linear.groups import matrix


def _plan(tokens=3, per_row=2, groups=4):
    entries = tokens * per_row
    index = torch.arange(entries, dtype=torch.int32)
    return ep.RowGroups(index, torch.full((groups + 1,), entries, dtype=torch.int32), index.clone(), index // per_row, groups, tokens, per_row)


def _bf16(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_group_rows_refuses():
    with pytest.raises(TypeError):
        ep.group_rows(torch.zeros(4), 2)
    with pytest.raises(TypeError):
        ep.group_rows(torch.zeros(4, dtype=torch.int16), 2)
    with pytest.raises(ValueError):
        ep.group_rows(torch.zeros(2, 2, 2, dtype=torch.int64), 2)
    with pytest.raises(ValueError):
        ep.group_rows(torch.zeros(4, 0, dtype=torch.int64), 2)
    for groups in (0, -1, 897, 2.0, True):
        with pytest.raises(ValueError):
            ep.group_rows(torch.zeros(4, dtype=torch.int64), groups)
    with pytest.raises(RuntimeError, match="GPU"):
        ep.group_rows(torch.zeros(4, dtype=torch.int64), 2)


def test_grouped_linear_refuses():
    plan = _plan()
    with pytest.raises(TypeError):
        ep.grouped_linear(_bf16(3, 8), _bf16(4, 5, 8), torch.zeros(3))
    with pytest.raises(ValueError):
        ep.grouped_linear(_bf16(3, 8), _bf16(5, 5, 8), plan)                       # groups
    with pytest.raises(ValueError):
        ep.grouped_linear(_bf16(6, 8), _bf16(4, 5, 8), plan)                       # rows per token
    with pytest.raises(ValueError):
        ep.grouped_linear(_bf16(3, 8), _bf16(4, 5, 8), plan, x_grouped=True)       # rows per entry
    with pytest.raises(ValueError):
        ep.grouped_linear(_bf16(3, 8), _bf16(4, 5, 16), plan)                      # features
    with pytest.raises(ValueError):
        ep.grouped_linear(_bf16(3, 0), _bf16(4, 5, 0), plan)
    with pytest.raises(ValueError):
        ep.grouped_linear(_bf16(3, 8), _bf16(4, 5, 8), plan, _bf16(5))
    with pytest.raises(TypeError):
        ep.grouped_linear(_bf16(3, 8).float(), _bf16(4, 5, 8), plan)
    with pytest.raises(TypeError):
        ep.grouped_linear(_bf16(3, 8), _bf16(4, 5, 8), plan, _bf16(4, 5).float())
    with pytest.raises(RuntimeError, match="GPU"):
        ep.grouped_linear(_bf16(3, 8), _bf16(4, 5, 8), plan)


def test_grouped_int8_linear_refuses():
    plan = _plan()
    x, w = torch.zeros(3, 16, dtype=torch.int8), torch.zeros(4, 5, 16, dtype=torch.int8)
    with pytest.raises(TypeError):
        ep.grouped_int8_linear(x.float(), w, plan, torch.ones(3), torch.ones(4, 5))
    with pytest.raises(TypeError):
        ep.grouped_int8_linear(x, w, plan, torch.ones(3), torch.ones(4, 5), out_dtype=torch.int8)
    with pytest.raises(ValueError):
        ep.grouped_int8_linear(x, w, plan, torch.ones(6), torch.ones(4, 5))
    with pytest.raises(ValueError):
        ep.grouped_int8_linear(x, w, plan, torch.ones(3), torch.ones(5))
    with pytest.raises(RuntimeError, match="GPU"):
        ep.grouped_int8_linear(x, w, plan, torch.ones(3), torch.ones(4, 5))


def test_combine_rows_refuses():
    plan = _plan()
    with pytest.raises(TypeError):
        ep.combine_rows(_bf16(6, 8), None)
    with pytest.raises(TypeError):
        ep.combine_rows(_bf16(6, 8).float(), plan)
    with pytest.raises(ValueError):
        ep.combine_rows(_bf16(3, 8), plan)
    with pytest.raises(ValueError):
        ep.combine_rows(_bf16(6, 8), plan, torch.ones(6))
    with pytest.raises(TypeError):
        ep.combine_rows(_bf16(6, 8), plan, torch.ones(3, 2, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="GPU"):
        ep.combine_rows(_bf16(6, 8), plan, torch.ones(3, 2))


def test_low_rank_update_refuses():
    plan = _plan(tokens=3, per_row=1)
    y, x, down, up = _bf16(3, 10), _bf16(3, 8), _bf16(4, 2, 8), _bf16(4, 10, 2)
    with pytest.raises(TypeError):
        ep.low_rank_update(y, x, down, up, None)
    with pytest.raises(TypeError):
        ep.low_rank_update(y, x.float(), down, up, plan)
    with pytest.raises(ValueError):
        ep.low_rank_update(_bf16(6, 10), _bf16(6, 8), down, up, _plan())           # two ids per row
    with pytest.raises(ValueError):
        ep.low_rank_update(y, x, down, _bf16(4, 10, 3), plan)
    with pytest.raises(ValueError):
        ep.low_rank_update(y, x, down, _bf16(5, 10, 2), plan)
    with pytest.raises(ValueError):
        ep.low_rank_update(y, _bf16(2, 8), down, up, plan)
    with pytest.raises(ValueError):
        ep.low_rank_update(_bf16(3, 9), x, down, up, plan)
    with pytest.raises(ValueError):
        ep.low_rank_update(y, x, _bf16(4, 0, 8), _bf16(4, 10, 0), plan)
    with pytest.raises(ValueError):
        ep.low_rank_update(y, x, _bf16(4, 4097, 8), _bf16(4, 10, 4097), plan)
    with pytest.raises(ValueError):
        ep.low_rank_update(y, x, down, up, plan, torch.ones(3))
    with pytest.raises(ValueError):
        ep.low_rank_update(y, x, down, up, plan, torch.ones(4, requires_grad=True))
    with pytest.raises(RuntimeError, match="GPU"):
        ep.low_rank_update(y, x, down, up, plan, torch.ones(4))


def test_modules_refuse():
    config = ep.EntroPackLossyConfig(target_bpp=4.0, execution_backend="eager")
    plain, wide = ep.CompressedLinear(16, 8), ep.CompressedLinear(32, 8)
    with pytest.raises(ValueError):
        ep.CompressedGroupedLinear([])
    with pytest.raises(TypeError):
        ep.CompressedGroupedLinear([torch.nn.Linear(16, 8)])
    with pytest.raises(ValueError):
        ep.CompressedGroupedLinear([plain, wide])
    with pytest.raises(ValueError):
        ep.CompressedGroupedLinear([plain, ep.CompressedLinear(16, 8, bias=False)])
    with pytest.raises(TypeError):
        ep.CompressedGroupedLinear([plain, ep.CompressedINT8Linear(16, 8)])
    with pytest.raises(TypeError):
        ep.CompressedGroupedLinear([ep.CompressedLinear(16, 8, dtype=torch.float32, config=config)])
    experts = ep.CompressedGroupedLinear([ep.CompressedLinear(16, 8) for _ in range(4)])
    with pytest.raises(RuntimeError, match="GPU"):
        experts(_bf16(3, 16), _plan())
    with pytest.raises(TypeError):
        experts(torch.zeros(3, 16), _plan())
    with pytest.raises(TypeError):
        ep.AdaptedLinear(torch.nn.Linear(16, 8), 2, 4)
    for adapters, rank in ((0, 4), (2, 0), (2, True), (1.0, 4)):
        with pytest.raises(ValueError):
            ep.AdaptedLinear(plain, adapters, rank)
    bank = ep.AdaptedLinear(plain, 2, 4)
    with pytest.raises(IndexError):
        bank.set_adapter(2, _bf16(4, 16), _bf16(8, 4))
    with pytest.raises(ValueError):
        bank.set_adapter(0, _bf16(5, 16), _bf16(8, 5))
    bank.set_adapter(1, torch.ones(3, 16), torch.ones(8, 3), scale=0.5)
    assert bank.scale.tolist() == [1.0, 0.5]
    assert bank.down[1, :3].eq(1).all() and bank.down[1, 3:].eq(0).all() and bank.up[1, :, :3].eq(1).all() and bank.up[1, :, 3:].eq(0).all()


def test_matrix_copies_only_what_the_kernels_cannot_read():
    whole = _bf16(6, 32)
    assert matrix(whole, 8) is whole
    part = whole[:, :24]
    assert matrix(part, 8) is part                                       # rows 32 elements apart
    for awkward in (whole[:, 1:25], _bf16(32, 6).t(), _bf16(1, 8).expand(5, 8), _bf16(7, 36)[:, :32], _bf16(3, 4, 8).transpose(0, 1)):
        ready = matrix(awkward, 8)
        assert ready.is_contiguous() and ready.data_ptr() % 16 == 0 and ready.shape[:-1] == awkward.shape[:-1] and ready.shape[-1] % 8 == 0
    padded = matrix(torch.ones(3, 5, dtype=torch.bfloat16), 8)
    assert padded.shape == (3, 8) and padded[:, :5].eq(1).all() and padded[:, 5:].eq(0).all()


def test_entry_points_refuse_bad_arguments():
    """Every check below fails before anything is launched, so no device is needed; the addresses are never followed."""
    lib, at, odd = hip.library(), 4096, 4104
    call = lambda name, good, **bad: getattr(lib, name)(*[bad.get(key, value) for key, value in good])
    sort = [("ids", at), ("id_bytes", 8), ("entries", 9000), ("groups", 4), ("per_row", 1), ("order", at), ("offsets", at), ("place", at), ("rows", None), ("work", at), ("room", 1 << 20), ("stream", None)]
    for bad in ({"ids": None}, {"id_bytes": 2}, {"entries": 0}, {"groups": 0}, {"per_row": 0}, {"order": None}, {"offsets": None}, {"place": None}, {"work": None}, {"room": 8}):
        assert call("ep_hip_group_rows", sort, **bad) == hip.EINVAL, bad
    for bad in ({"groups": 897}, {"entries": (1 << 30) + 1}):
        assert call("ep_hip_group_rows", sort, **bad) == hip.EUNSUPPORTED, bad
    assert lib.ep_hip_group_rows_workspace(10, 4) == 0 and lib.ep_hip_group_rows_workspace(1 << 20, 4) == 256 * 5 * 4

    product = [("x", at), ("ldx", 16), ("x_rows", 4), ("w", at), ("ldw", 16), ("w_group", 64), ("bias", None), ("y", at), ("ldy", 4), ("kind", 0), ("rows", at),
               ("offsets", at), ("entries", 8), ("groups", 2), ("N", 4), ("K", 16), ("stream", None)]
    for bad in ({"x": None}, {"x": odd}, {"w": odd}, {"w": None}, {"y": None}, {"ldx": 12}, {"ldx": 8}, {"ldw": 20}, {"w_group": 60}, {"w_group": -8}, {"ldy": 3}, {"kind": 3},
                {"offsets": None}, {"entries": 0}, {"groups": 0}, {"N": 0}, {"K": 0}, {"K": 12}, {"rows": None, "x_rows": 7}, {"N": 1 << 31}):
        assert call("ep_hip_grouped_gemm_bf16", product, **bad) == hip.EINVAL, bad
    codes = [("x", at), ("ldx", 16), ("x_rows", 4), ("w", at), ("ldw", 16), ("w_group", 64), ("sx", at), ("sw", at), ("bias", None), ("y", at), ("ldy", 4), ("kind", 0),
             ("rows", at), ("offsets", at), ("entries", 8), ("groups", 2), ("N", 4), ("K", 16), ("stream", None)]
    for bad in ({"sx": None}, {"sw": None}, {"ldx": 24}, {"K": 8}, {"w_group": 72}, {"kind": -1}):
        assert call("ep_hip_grouped_gemm_i8", codes, **bad) == hip.EINVAL, bad
    rows = [("dy", at), ("lddy", 8), ("w", at), ("ldw", 16), ("w_group", 128), ("dx", at), ("lddx", 16), ("kind", 0), ("order", at), ("offsets", at), ("entries", 8), ("groups", 2),
            ("N", 8), ("K", 16), ("stream", None)]
    for bad in ({"dy": odd}, {"w": None}, {"dx": None}, {"lddx": 8}, {"N": 9}, {"K": 12}, {"lddy": 4}, {"offsets": None}):
        assert call("ep_hip_grouped_grad_rows_bf16", rows, **bad) == hip.EINVAL, bad
    weight = [("dy", at), ("lddy", 8), ("x", at), ("ldx", 16), ("x_rows", 8), ("dw", at), ("lddw", 16), ("dw_group", 128), ("kind", 0), ("rows", at), ("offsets", at),
              ("entries", 8), ("groups", 2), ("N", 8), ("K", 16), ("work", None), ("room", 0), ("stream", None)]
    long = {"entries": 10000, "x_rows": 10000}                     # two small weights, many rows: the sums of chunks take a workspace
    room = lib.ep_hip_grouped_grad_weight_workspace(10000, 2, 8, 16)
    assert room > 0 and lib.ep_hip_grouped_grad_weight_workspace(8, 2, 8, 16) == 0 and lib.ep_hip_grouped_grad_weight_workspace(1 << 20, 8, 4096, 4096) == 0
    for bad in ({**long, "work": at, "room": room - 1}, {**long, "work": odd, "room": room}, {**long, "room": room}, {"dy": odd}, {"x": odd}, {"dw": None}, {"lddw": 8}, {"N": 4}, {"K": 12}, {"dw_group": -1}, {"rows": None, "x_rows": 7}):
        assert call("ep_hip_grouped_grad_weight_bf16", weight, **bad) == hip.EINVAL, bad
    sums = [("dy", at), ("lddy", 8), ("offsets", at), ("groups", 2), ("N", 8), ("out", at), ("kind", 0), ("stream", None)]
    for bad in ({"dy": None}, {"lddy": 4}, {"groups": 0}, {"N": 0}, {"out": None}, {"kind": 7}):
        assert call("ep_hip_grouped_column_sums_bf16", sums, **bad) == hip.EINVAL, bad

    update = [("x", at), ("ldx", 16), ("down", at), ("ldd", 16), ("down_group", 64), ("up", at), ("ldu", 4), ("up_group", 64), ("scale", None), ("y", at), ("ldy", 16), ("planes", at), ("out", at),
              ("ldo", 16), ("order", at), ("offsets", at), ("entries", 8), ("groups", 2), ("rank", 4), ("K", 16), ("N", 16), ("stream", None)]
    for bad in ({"x": odd}, {"x": None}, {"ldx": 12}, {"ldx": 8}, {"down": None}, {"ldd": 20}, {"down_group": 4}, {"down_group": -8}, {"up": None}, {"ldu": 3}, {"up_group": -1}, {"ldy": 8},
                {"planes": odd}, {"planes": None}, {"out": None}, {"ldo": 8}, {"order": None}, {"offsets": None}, {"entries": 0}, {"groups": 0}, {"rank": 0}, {"rank": 4097}, {"K": 0}, {"N": 0},
                {"N": 1 << 30}, {"K": 17}):
        assert call("ep_hip_low_rank_update", update, **bad) == hip.EINVAL, bad
    grad = [("grad", at), ("ldg", 16), ("x", at), ("ldx", 16), ("down", at), ("ldd", 16), ("down_group", 64), ("up", at), ("ldu", 4), ("up_group", 64), ("scale", None), ("planes", at),
            ("gx", at), ("ldgx", 16), ("gd", at), ("gu", at), ("order", at), ("offsets", at), ("entries", 8), ("groups", 2), ("rank", 4), ("K", 16), ("N", 16), ("work", at), ("room", 1 << 30),
            ("stream", None)]
    for bad in ({"grad": odd}, {"grad": None}, {"ldg": 8}, {"ldg": 20}, {"x": None}, {"ldx": 8}, {"down": None}, {"ldd": 8}, {"up": None}, {"ldu": 3}, {"planes": None}, {"planes": odd}, {"ldgx": 8},
                {"gx": None, "gd": None, "gu": None}, {"order": None}, {"entries": 0}, {"rank": 0}, {"work": None}, {"work": 128}, {"room": 64}):
        assert call("ep_hip_low_rank_update_grad", grad, **bad) == hip.EINVAL, bad

    combine = [("y", at), ("kind", 0), ("ldy", 8), ("place", at), ("kept", at), ("weight", at), ("weight_kind", 2), ("per_row", 2), ("tokens", 4), ("width", 8), ("out", at), ("ldo", 8), ("stream", None)]
    for bad in ({"y": None}, {"kind": 1}, {"ldy": 4}, {"kept": None}, {"weight_kind": 1}, {"per_row": 0}, {"tokens": 0}, {"width": 0}, {"out": None}, {"ldo": 4}):
        assert call("ep_hip_combine_rows", combine, **bad) == hip.EINVAL, bad
    grads = [("grad", at), ("ldg", 8), ("y", at), ("ldy", 8), ("place", at), ("kept", at), ("weight", at), ("weight_kind", 2), ("per_row", 2), ("tokens", 4), ("width", 8), ("gy", at), ("ldgy", 8),
             ("gw", at), ("stream", None)]
    for bad in ({"grad": None}, {"place": None}, {"kept": None}, {"gy": None, "gw": None}, {"y": None}, {"ldgy": 4}, {"weight_kind": 1}, {"width": 0}, {"tokens": 0}):
        assert call("ep_hip_combine_rows_grad", grads, **bad) == hip.EINVAL, bad
