"""GPU parity of the operators on grouped rows, against plain implementations in 64 bits.

Tolerances. Products of two bf16 numbers are exact in f32; a sum of K of them in any order is off by at most K steps of
2^-23 relative to the sum of the magnitudes (a whole unit in the last place per addition, whichever way the matrix cores
round), and the one rounding to bf16 by half a step, 2^-8 of the value. `_bound` is that. Where a second product follows, the
bound of the first is carried through the magnitudes; the two-part narrow rows of the adapters add 2^-16.
"""
import copy
import pytest
import torch

import entropack_amd as ep
from entropack_amd.linear import kernels

pytestmark = pytest.mark.gpu
HALF_BF16, STEP_F32 = 2.0 ** -8, 2.0 ** -23


def _bound(value, magnitudes, terms):
    return HALF_BF16 * value.abs() + (1 + HALF_BF16) * (terms + 2) * STEP_F32 * magnitudes + 1e-37


def _within(got, expect, bound):
    got, off = got.double(), (got.double() - expect).abs()
    assert torch.isfinite(got).all()
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert worst <= 0.0, f"off by {worst} more than the bound; largest difference {off.max().item()}"


def _members(ids, groups):
    flat = ids.reshape(-1).cpu()
    return [torch.nonzero(flat == g).reshape(-1).cuda() for g in range(groups)]


def _ids(tokens, per_row, groups, kind, seed=0, dtype=torch.int64):
    source = torch.Generator().manual_seed(seed)
    shape = (tokens, per_row) if per_row else (tokens,)
    if kind == "even":
        ids = torch.randint(0, groups, shape, generator=source)
    elif kind == "padded":
        ids = torch.randint(0, groups, shape, generator=source)
        ids[torch.rand(tokens, generator=source) < 0.3] = -1
    elif kind == "one":                                    # every row in the last group
        ids = torch.full(shape, groups - 1)
    elif kind == "none":
        ids = torch.full(shape, -1)
    elif kind == "outside":                                # ids beyond the groups count as none
        ids = torch.randint(-2, groups + 3, shape, generator=source)
    elif kind == "skewed":
        ids = (torch.rand(shape, generator=source) ** 4 * groups).long()
    return ids.to(dtype).cuda()


def _plain_places(ids, groups):
    flat = ids.reshape(-1).cpu().long()
    key = torch.where((flat < 0) | (flat >= groups), groups, flat)
    order = torch.sort(key, stable=True).indices
    offsets = torch.tensor([int((key < g).sum()) for g in range(groups + 1)])
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel())
    return order, offsets, place


@pytest.mark.parametrize("tokens,per_row,groups", [(1, 0, 1), (1, 8, 3), (63, 1, 2), (64, 0, 64), (65, 2, 65), (1000, 3, 7), (4096, 1, 100), (4097, 1, 5), (2049, 4, 896),
                                                   (20001, 8, 128), (300000, 5, 33), (1024, 0, 9), (1025, 0, 896), (4096, 2, 64), (8193, 0, 3), (8192, 2, 64), (1 << 20, 0, 17),
                                                   ((1 << 20) + 1, 0, 2)])
@pytest.mark.parametrize("kind", ["even", "padded", "one", "none", "outside", "skewed"])
def test_group_rows(tokens, per_row, groups, kind):
    print("case", tokens, per_row, groups, kind, flush=True)
    for dtype in (torch.int64, torch.int32):
        ids = _ids(tokens, per_row, groups, kind, dtype=dtype)
        plan = ep.group_rows(ids, groups)
        order, offsets, place = _plain_places(ids, groups)
        assert torch.equal(plan.rows.cpu().long(), order // (per_row or 1))
        assert torch.equal(plan.order.cpu().long(), order) and torch.equal(plan.offsets.cpu().long(), offsets) and torch.equal(plan.place.cpu().long(), place)
        assert (plan.tokens, plan.per_row, plan.entries, plan.groups) == (tokens, per_row or 1, order.numel(), groups)


def test_group_rows_takes_strided_ids_wide_values_and_none_at_all():
    ids = torch.randint(0, 9, (5, 700), device="cuda").t()
    for given, want in ((ids, ids.contiguous()), (ids[::2], ids[::2].contiguous())):
        assert torch.equal(ep.group_rows(given, 9).order, ep.group_rows(want, 9).order)
    far = torch.tensor([2 ** 32 + 1, 1, -2 ** 40, 0], device="cuda")                  # the low 32 bits of the first are 1
    assert ep.group_rows(far, 4).offsets.tolist() == [0, 1, 2, 2, 2]
    empty = ep.group_rows(torch.zeros(0, 4, dtype=torch.int64, device="cuda"), 3)
    assert empty.entries == 0 and empty.offsets.tolist() == [0, 0, 0, 0]


# tokens, ids per token, groups, in, out, ids
PRODUCTS = [(1, 2, 8, 264, 100, "even"), (1, 0, 1, 8, 1, "even"), (5, 4, 64, 512, 129, "padded"), (40, 2, 3, 72, 257, "even"), (33, 1, 4, 1024, 64, "one"),
            (7, 3, 5, 128, 40, "none"), (129, 2, 5, 320, 130, "outside"), (300, 2, 4, 136, 264, "skewed"), (1100, 2, 3, 200, 384, "padded"), (700, 0, 2, 1096, 520, "even"),
            (64, 8, 4, 33, 65, "even"), (513, 4, 6, 2048, 128, "skewed"), (260, 1, 896, 64, 72, "even"), (2100, 1, 1, 448, 1000, "one"),
            (4100, 2, 6, 2064, 1041, "padded"), (2100, 2, 4, 2048, 2304, "even"), (4200, 0, 3, 1032, 2056, "one"), (4300, 2, 3, 1024, 2056, "even"), (5000, 2, 4, 2056, 2100, "skewed"),
            (9000, 0, 2, 136, 72, "padded"), (7001, 2, 3, 128, 128, "skewed"), (5000, 2, 1, 264, 9, "outside"), (5000, 2, 2, 520, 264, "one")]


def _product_operands(case, x_grouped, seed=3):
    tokens, per_row, groups, inner, outer, kind = case
    ids = _ids(tokens, per_row, groups, kind)
    plan = ep.group_rows(ids, groups)
    source = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(plan.entries if x_grouped else tokens, inner, device="cuda", generator=source).bfloat16()
    w = (torch.randn(groups, outer, inner, device="cuda", generator=source) * 0.05).bfloat16()
    kept = int(plan.offsets[-1])
    where = plan.order.long() // plan.per_row if not x_grouped else torch.arange(plan.entries, device="cuda")
    spans = [(g, int(plan.offsets[g]), int(plan.offsets[g + 1])) for g in range(groups)]
    return plan, x, w, where, spans, kept


@pytest.mark.parametrize("case", PRODUCTS, ids=str)
@pytest.mark.parametrize("x_grouped", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
def test_grouped_linear(case, x_grouped, with_bias):
    print("case", case, x_grouped, with_bias, flush=True)
    plan, x, w, where, spans, kept = _product_operands(case, x_grouped)
    bias = torch.randn(w.shape[:2], device="cuda").bfloat16() if with_bias else None
    y = ep.grouped_linear(x, w, plan, bias, x_grouped=x_grouped)
    assert y.shape == (plan.entries, w.shape[1]) and y.dtype == torch.bfloat16 and y.is_contiguous()
    expect, size = torch.zeros(y.shape, dtype=torch.float64, device="cuda"), torch.zeros(y.shape, dtype=torch.float64, device="cuda")
    for g, first, last in spans:
        rows = x[where[first:last]].double()
        expect[first:last] = rows @ w[g].double().t() + (bias[g].double() if with_bias else 0.0)
        size[first:last] = rows.abs() @ w[g].double().abs().t() + (bias[g].double().abs() if with_bias else 0.0)
    _within(y, expect, _bound(expect, size, x.shape[1] + 1))
    assert y[kept:].eq(0).all()


@pytest.mark.parametrize("case", PRODUCTS, ids=str)
@pytest.mark.parametrize("x_grouped", [False, True])
def test_grouped_linear_gradients(case, x_grouped):
    print("case", case, x_grouped, flush=True)
    plan, x, w, where, spans, kept = _product_operands(case, x_grouped)
    bias = torch.randn(w.shape[:2], device="cuda").bfloat16()
    leaves = [t.requires_grad_(True) for t in (x, w, bias)]
    y = ep.grouped_linear(x, w, plan, bias, x_grouped=x_grouped)
    grad = torch.randn(y.shape, device="cuda").bfloat16()
    grad[kept:] = float("nan")                              # rows of no group reach no gradient
    grad_x, grad_w, grad_b = torch.autograd.grad(y, leaves, grad)
    with torch.no_grad():
        want_x, size_x = torch.zeros(x.shape, dtype=torch.float64, device="cuda"), torch.zeros(x.shape, dtype=torch.float64, device="cuda")
        most = 0
        for g, first, last in spans:
            rows, dy, weight = x[where[first:last]].double(), grad[first:last].double(), w[g].double()
            most = max(most, last - first)
            want_x.index_add_(0, where[first:last], dy @ weight)
            size_x.index_add_(0, where[first:last], dy.abs() @ weight.abs())
            _within(grad_w[g], dy.t() @ rows, _bound(dy.t() @ rows, dy.abs().t() @ rows.abs(), last - first))
            _within(grad_b[g], dy.sum(0), _bound(dy.sum(0), dy.abs().sum(0), last - first))
        # one sum per entry and the entries' sum, all in f32
        _within(grad_x, want_x, _bound(want_x, size_x, w.shape[1] + plan.per_row))
    assert grad_x.dtype == grad_w.dtype == grad_b.dtype == torch.bfloat16


def test_grouped_linear_gradient_agrees_with_differences():
    """The product is linear in x and in w: <dy, F(x + v) - F(x)> = <grad_x, v> up to the roundings of both sides."""
    plan, x, w, where, spans, kept = _product_operands((150, 2, 4, 128, 96, "padded"), False)
    x.requires_grad_(True), w.requires_grad_(True)
    dy = torch.randn(plan.entries, 96, device="cuda").bfloat16()
    grad_x, grad_w = torch.autograd.grad(ep.grouped_linear(x, w, plan), (x, w), dy)
    with torch.no_grad():
        base = ep.grouped_linear(x, w, plan).double()
        for leaf, grad, other in ((x, grad_x, lambda v: ep.grouped_linear(v, w, plan)), (w, grad_w, lambda v: ep.grouped_linear(x, v, plan))):
            step = (torch.randn_like(leaf, dtype=torch.float32) * leaf.float().std()).bfloat16()
            moved = (leaf.float() + step.float()).bfloat16()
            taken = moved.double() - leaf.double()                        # what bf16 made of the step
            change = other(moved).double() - base
            left, right = (dy.double() * change).sum(), (grad.double() * taken).sum()
            # half a step on every element of F(x + v), F(x) and the gradient, plus the f32 sums (128 terms, far below)
            bound = (dy.double().abs() * (other(moved).double().abs() + base.abs())).sum() * HALF_BF16 * 1.01 + (grad.double().abs() * taken.abs()).sum() * HALF_BF16 * 1.01
            assert (left - right).abs() <= bound
            assert right.abs() > 0


def test_grouped_linear_takes_strided_operands():
    tokens, groups, inner, outer = 50, 3, 96, 72
    plan = ep.group_rows(_ids(tokens, 2, groups, "padded"), groups)
    wide = torch.randn(tokens, 160, device="cuda").bfloat16()
    arena = torch.randn(groups, outer + 5, 128, device="cuda").bfloat16() * 0.1
    views = [(wide[:, :inner], arena[:, :outer, :inner]), (wide[:, 3:3 + inner], arena[:, 5:, 1:1 + inner]), (wide.t()[:inner, :].t(), arena[:, :outer, :inner].transpose(1, 2).contiguous().transpose(1, 2)),
             (wide[:1, :inner].expand(tokens, inner), arena[:1, :outer, :inner].expand(groups, outer, inner))]
    for x, w in views:
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        xc, wc = x.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True), w.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
        got, want = ep.grouped_linear(x, w, plan), ep.grouped_linear(xc, wc, plan)
        assert torch.equal(got, want)
        for dy in (torch.ones((), device="cuda", dtype=torch.bfloat16).expand(got.shape), torch.randn(outer, plan.entries, device="cuda").bfloat16().t()):
            for a, b in zip(torch.autograd.grad(got, (x, w), dy, retain_graph=True), torch.autograd.grad(want, (xc, wc), dy.contiguous(), retain_graph=True)):
                assert torch.equal(a, b)


def test_values_of_rows_without_a_group_reach_nothing():
    groups, inner, outer = 4, 128, 96
    ids = _ids(60, 2, groups, "padded")
    dropped = ids[:, 0] < 0
    plan = ep.group_rows(ids, groups)
    x, w = torch.randn(60, inner, device="cuda").bfloat16(), torch.randn(groups, outer, inner, device="cuda").bfloat16()
    spoiled = x.clone()
    spoiled[dropped] = float("nan")
    assert torch.equal(ep.grouped_linear(spoiled, w, plan), ep.grouped_linear(x, w, plan))
    x.requires_grad_(True), w.requires_grad_(True), spoiled.requires_grad_(True)
    dy = torch.randn(plan.entries, outer, device="cuda").bfloat16()
    for a, b in zip(torch.autograd.grad(ep.grouped_linear(spoiled, w, plan), (spoiled, w), dy), torch.autograd.grad(ep.grouped_linear(x, w, plan), (x, w), dy)):
        assert torch.equal(a, b)
    # An infinity stays in its own row's outputs, a spoiled weight in its own group's.
    x = x.detach().clone()
    at = int(torch.nonzero(~dropped)[0])
    clean = ep.grouped_linear(x, w.detach(), plan)
    x[at, 5] = float("inf")
    hit = (plan.order.long() // 2) == at
    y = ep.grouped_linear(x, w.detach(), plan)
    assert torch.equal(y[~hit], clean[~hit]) and not torch.isfinite(y[hit]).any()


@pytest.mark.parametrize("case", PRODUCTS, ids=str)
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_grouped_int8_linear(case, out_dtype):
    """Exact: the sums are integers, and the roundings after them are made one by one in a fixed order."""
    print("case", case, out_dtype, flush=True)
    tokens, per_row, groups, inner, outer, kind = case
    plan = ep.group_rows(_ids(tokens, per_row, groups, kind), groups)
    source = torch.Generator(device="cuda").manual_seed(1)
    for x_grouped, with_bias in ((False, True), (True, False)):
        rows = plan.entries if x_grouped else tokens
        x = torch.randint(-127, 128, (rows, inner), device="cuda", generator=source, dtype=torch.int8)
        w = torch.randint(-127, 128, (groups, outer, inner), device="cuda", generator=source, dtype=torch.int8)
        sx = 0.01 + torch.rand(rows, device="cuda", generator=source) * 0.02
        sw = 0.0002 + torch.rand(groups, outer, device="cuda", generator=source) * 0.0003
        bias = torch.randn(groups, outer, device="cuda", generator=source).to(out_dtype) if with_bias else None
        y = ep.grouped_int8_linear(x, w, plan, sx, sw, bias, out_dtype, x_grouped=x_grouped)
        where = torch.arange(plan.entries, device="cuda") if x_grouped else plan.order.long() // plan.per_row
        expect = torch.zeros(plan.entries, outer, device="cuda")
        for g in range(groups):
            first, last = int(plan.offsets[g]), int(plan.offsets[g + 1])
            sums = (x[where[first:last]].double() @ w[g].double().t()).float()
            expect[first:last] = sums * sx[where[first:last]].unsqueeze(1) * sw[g]
            if with_bias:
                expect[first:last] += bias[g].float()
        assert y.dtype == out_dtype and torch.equal(y, expect.to(out_dtype))


COMBINES = [(1, 1, 3, 8), (1, 8, 4, 1), (17, 3, 5, 100), (64, 2, 8, 2048), (300, 9, 20, 72), (50, 17, 20, 33), (1000, 4, 16, 264)]


@pytest.mark.parametrize("tokens,per_row,groups,width", COMBINES)
@pytest.mark.parametrize("kind", ["even", "padded", "none"])
@pytest.mark.parametrize("weights", [torch.float32, torch.bfloat16, None], ids=str)
def test_combine_rows_and_gradients(tokens, per_row, groups, width, kind, weights):
    print("case", tokens, per_row, groups, width, kind, weights, flush=True)
    ids = _ids(tokens, per_row, groups, kind)
    plan = ep.group_rows(ids, groups)
    kept = int(plan.offsets[-1])
    y = torch.randn(plan.entries, width, device="cuda").bfloat16()
    y[kept:] = float("nan")
    y.requires_grad_(True)
    counts = (plan.place.long() < kept).reshape(tokens, per_row)
    weight = None
    if weights is not None:
        weight = torch.rand(tokens, per_row, device="cuda").to(weights)
        weight[~counts] = float("inf")
        weight.requires_grad_(True)
    out = ep.combine_rows(y, plan, weight)
    grad = torch.randn(tokens, width, device="cuda").bfloat16()
    leaves = [y] if weight is None else [y, weight]
    grads = torch.autograd.grad(out, leaves, grad)
    with torch.no_grad():
        rows = torch.where(counts.unsqueeze(2), y[plan.place.long()].reshape(tokens, per_row, width).double(), 0.0)
        share = counts.double() if weight is None else torch.where(counts, weight.double(), 0.0)
        expect, size = (rows * share.unsqueeze(2)).sum(1), (rows.abs() * share.unsqueeze(2)).sum(1)
        _within(out, expect, _bound(expect, size, per_row))
        want_y = (share.unsqueeze(2) * grad.double().unsqueeze(1)).reshape(-1, width)
        got_y = grads[0][plan.place.long()]
        _within(got_y, want_y, HALF_BF16 * want_y.abs() + STEP_F32 * want_y.abs() + 1e-37)
        if weight is not None:
            want_w, size_w = (rows * grad.double().unsqueeze(1)).sum(2), (rows.abs() * grad.double().abs().unsqueeze(1)).sum(2)
            rounding = 0.0 if weights == torch.float32 else HALF_BF16 * want_w.abs()
            _within(grads[1], want_w, rounding + (1 + HALF_BF16) * (width + 2) * STEP_F32 * size_w + 1e-37)
            assert grads[1].dtype == weights
            with torch.enable_grad():
                only = torch.autograd.grad(ep.combine_rows(y.detach(), plan, weight), weight, grad)[0]
            assert torch.equal(only, grads[1])


# rows, adapters, rank, in, out, ids
UPDATES = [(1, 1, 1, 8, 1, "even"), (1, 5, 16, 4096, 100, "even"), (7, 3, 4, 264, 72, "padded"), (64, 64, 8, 512, 257, "even"), (65, 4, 16, 1024, 264, "padded"), (33, 2, 12, 72, 130, "none"),
           (500, 3, 33, 200, 520, "skewed"), (300, 2, 64, 33, 65, "outside"), (1500, 4, 32, 264, 384, "padded"), (260, 896, 16, 64, 72, "even"), (700, 1, 128, 128, 256, "one"), (90, 6, 24, 2048, 64, "even")]


@pytest.mark.parametrize("case", UPDATES, ids=str)
@pytest.mark.parametrize("with_scale", [True, False])
def test_low_rank_update_and_gradients(case, with_scale):
    print("case", case, with_scale, flush=True)
    tokens, adapters, rank, inner, outer, kind = case
    ids = _ids(tokens, 0, adapters, kind)
    plan = ep.group_rows(ids, adapters)
    source = torch.Generator(device="cuda").manual_seed(2)
    make = lambda *shape, scale=1.0: (torch.randn(*shape, device="cuda", generator=source) * scale).bfloat16()
    y, x, down, up = make(tokens, outer), make(tokens, inner), make(adapters, rank, inner, scale=inner ** -0.5), make(adapters, outer, rank, scale=rank ** -0.5)
    scale = 0.5 + torch.rand(adapters, device="cuda", generator=source) if with_scale else None
    leaves = [t.requires_grad_(True) for t in (y, x, down, up)]
    out = ep.low_rank_update(y, x, down, up, plan, scale)
    grad = make(tokens, outer)
    grad_y, grad_x, grad_down, grad_up = torch.autograd.grad(out, leaves, grad)
    two_parts = 2.0 ** -16
    with torch.no_grad():
        want, size, want_x, size_x = y.double(), y.double().abs(), torch.zeros(x.shape, dtype=torch.float64, device="cuda"), torch.zeros(x.shape, dtype=torch.float64, device="cuda")
        narrow_f, narrow_b = (inner + 3) * STEP_F32 + two_parts, (outer + 3) * STEP_F32 + two_parts          # relative errors of the narrow rows
        for a, rows in enumerate(_members(ids, adapters)):
            s = 1.0 if scale is None else scale[a].double()
            xs, dn, u, dy = x[rows].double(), down[a].double(), up[a].double(), grad[rows].double()
            h, h_size = s * (xs @ dn.t()), s * (xs.abs() @ dn.abs().t())
            want[rows] += h @ u.t()
            size[rows] += (h_size @ u.abs().t()) * (1 + narrow_f / ((2 * rank + 17) * STEP_F32))       # so that the bound's factor carries both
            g, g_size = s * (dy @ u), s * (dy.abs() @ u.abs())
            want_x[rows] = g @ dn
            size_x[rows] = (g_size @ dn.abs()) * (1 + narrow_b / ((2 * rank + 17) * STEP_F32))
            n = 2 * rows.numel() + 2
            _within(grad_down[a], g.t() @ xs, HALF_BF16 * (g.t() @ xs).abs() + (1 + HALF_BF16) * (n * STEP_F32 + narrow_b) * (g_size.t() @ xs.abs()) + 1e-37)
            _within(grad_up[a], dy.t() @ h, HALF_BF16 * (dy.t() @ h).abs() + (1 + HALF_BF16) * (n * STEP_F32 + narrow_f) * (dy.abs().t() @ h_size) + 1e-37)
        _within(out, want, _bound(want, size, 2 * rank + 15))
        _within(grad_x, want_x, _bound(want_x, size_x, 2 * rank + 15))
        none = (ids < 0) | (ids >= adapters)
        assert torch.equal(out[none], y[none]) and grad_x[none].eq(0).all()
    assert torch.equal(grad_y, grad)


def test_low_rank_update_agrees_with_differences():
    """The update is linear in x: <dout, F(x + v) - F(x)> = <grad_x, v> up to the roundings of both sides."""
    plan = ep.group_rows(_ids(200, 0, 3, "padded"), 3)
    y, x = torch.zeros(200, 96, device="cuda").bfloat16(), torch.randn(200, 128, device="cuda").bfloat16().requires_grad_(True)
    down, up = (torch.randn(3, 16, 128, device="cuda") * 0.1).bfloat16(), (torch.randn(3, 96, 16, device="cuda") * 0.25).bfloat16()
    dout = torch.randn(200, 96, device="cuda").bfloat16()
    base = ep.low_rank_update(y, x, down, up, plan)
    grad = torch.autograd.grad(base, x, dout)[0].double()
    with torch.no_grad():
        moved = (x.float() + torch.randn(x.shape, device="cuda")).bfloat16()
        taken = moved.double() - x.double()
        after = ep.low_rank_update(y, moved, down, up, plan).double()
        left, right = (dout.double() * (after - base.double())).sum(), (grad * taken).sum()
        bound = ((dout.double().abs() * (after.abs() + base.double().abs())).sum() + (grad.abs() * taken.abs()).sum()) * HALF_BF16 * 1.05      # 5 % for the f32 sums and the two-part rows
        assert (left - right).abs() <= bound and right.abs() > 0


def test_low_rank_update_strided_misaligned_and_spoiled_rows():
    plan = ep.group_rows(_ids(90, 0, 4, "padded"), 4)
    none = _ids(90, 0, 4, "padded") < 0
    wide = torch.randn(90, 300, device="cuda").bfloat16()
    down, up = torch.randn(4, 8, 128, device="cuda").bfloat16() * 0.1, torch.randn(4, 64, 8, device="cuda").bfloat16()
    for x, y in ((wide[:, :128], wide[:, 128:192]), (wide[:, 1:129], wide[:, 131:195]), (wide.t()[:128].t(), wide[:1, 200:264].expand(90, 64))):
        got = ep.low_rank_update(y, x, down, up, plan)
        assert torch.equal(got, ep.low_rank_update(y.contiguous(), x.contiguous(), down, up, plan))
        spoiled = x.clone()
        spoiled[none] = float("nan")
        assert torch.equal(got, ep.low_rank_update(y, spoiled, down, up, plan))
    big = torch.randn(4, 70, 24, device="cuda").bfloat16()
    assert torch.equal(ep.low_rank_update(wide[:, :64], wide[:, :128], down, big[:, 3:67, 1:9], plan), ep.low_rank_update(wide[:, :64], wide[:, :128], down, big[:, 3:67, 1:9].contiguous(), plan))


def test_dimensions_of_one_with_any_stride():
    """torch leaves the stride of a dimension of size one free, and calls such a tensor contiguous."""
    plan = ep.group_rows(torch.ones(1, dtype=torch.int64, device="cuda"), 3)
    x, y = torch.randn(64, 1, device="cuda").bfloat16().t(), torch.randn(40, 1, device="cuda").bfloat16().t()
    down, up = torch.randn(3, 64, 1, device="cuda").bfloat16().transpose(1, 2), torch.randn(3, 1, 40, device="cuda").bfloat16().transpose(1, 2)
    weight, dout = torch.randn(3, 64, 1, device="cuda").bfloat16().transpose(1, 2), torch.randn(40, 1, device="cuda").bfloat16().t()
    plain = lambda *tensors: [t.clone(memory_format=torch.contiguous_format).requires_grad_(True) for t in tensors]

    def both(run, grad, *operands):
        odd = [t.detach().requires_grad_(True) for t in operands]
        got = run(*odd)
        even = plain(*operands)
        want = run(*even)
        assert torch.equal(got, want)
        for a, b in zip(torch.autograd.grad(got, odd, grad), torch.autograd.grad(want, even, grad.clone(memory_format=torch.contiguous_format))):
            assert a.shape == b.shape and torch.equal(a, b)

    both(lambda y, x, d, u: ep.low_rank_update(y, x, d, u, plan), dout, y, x, down, up)
    both(lambda x, w, b: ep.grouped_linear(x, w, plan, b), dout[:, :1], x, weight, torch.randn(3, 1, device="cuda").bfloat16())
    both(lambda y: ep.combine_rows(y, plan), dout, y)


def test_empty_batches():
    plan = ep.group_rows(torch.zeros(0, 2, dtype=torch.int64, device="cuda"), 3)
    x, w = torch.zeros(0, 16, device="cuda").bfloat16().requires_grad_(True), torch.randn(3, 8, 16, device="cuda").bfloat16().requires_grad_(True)
    y = ep.grouped_linear(x, w, plan)
    gx, gw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == (0, 8) and gx.shape == (0, 16) and gw.eq(0).all()
    assert ep.combine_rows(y, plan, torch.zeros(0, 2, device="cuda")).shape == (0, 8)
    assert ep.grouped_int8_linear(torch.zeros(0, 16, dtype=torch.int8, device="cuda"), torch.zeros(3, 8, 16, dtype=torch.int8, device="cuda"), plan, torch.zeros(0, device="cuda"),
                                  torch.ones(3, 8, device="cuda")).shape == (0, 8)
    one = ep.group_rows(torch.zeros(0, dtype=torch.int64, device="cuda"), 3)
    out = ep.low_rank_update(torch.zeros(0, 8, device="cuda").bfloat16(), x, torch.randn(3, 4, 16, device="cuda").bfloat16(), torch.randn(3, 8, 4, device="cuda").bfloat16(), one)
    assert out.shape == (0, 8)


def _dense(outer, inner, seed, bias=True):
    torch.manual_seed(seed)
    layer = torch.nn.Linear(inner, outer, bias=bias, dtype=torch.bfloat16)
    layer.weight.data.mul_(2.0)
    return layer


@pytest.mark.parametrize("config", [ep.EntroPackLossyConfig(target_bpp=4.0), ep.TileANSConfig()], ids=["lattice_rans", "tile_ans"])
def test_mixture_of_compressed_experts(config):
    """A whole expert layer as a model runs it: route, two projections, gate, the third projection, the weighted return; forward
    and the gradient of the activations, against the same layer on the dense decoded weights in 64 bits."""
    experts, inner, middle, tokens, per_row = 5, 264, 136, 70, 2
    gate, up, down = [ep.CompressedGroupedLinear.from_linears([_dense(o, i, 10 * k + e) for e in range(experts)], config=config).cuda()
                      for k, (o, i) in enumerate([(middle, inner), (middle, inner), (inner, middle)])]
    ids = _ids(tokens, per_row, experts, "padded")
    share = torch.rand(tokens, per_row, device="cuda", requires_grad=True)
    x = torch.randn(tokens, inner, device="cuda").bfloat16().requires_grad_(True)
    dout = torch.randn(tokens, inner, device="cuda").bfloat16()

    def run(x, share):
        plan = ep.group_rows(ids, experts)
        hidden = torch.nn.functional.silu(gate(x, plan)) * up(x, plan)
        return ep.combine_rows(down(hidden, plan, x_grouped=True), plan, share)

    out = run(x, share)
    grads = torch.autograd.grad(out, (x, share), dout)
    for layer in (gate, up, down):                 # the plan of the decode is made once
        assert (layer._decoder is None) == isinstance(config, ep.TileANSConfig)
    dense = [layer.dequantize().double() for layer in (gate, up, down)]
    biases = [torch.stack([e.bias for e in layer.experts]).double() for layer in (gate, up, down)]
    xd, sd = x.detach().double().requires_grad_(True), share.detach().double().requires_grad_(True)
    rows = []
    for t in range(tokens):
        total = xd.new_zeros(inner)
        for j in range(per_row):
            e = int(ids[t, j])
            if e < 0:
                continue
            hidden = torch.nn.functional.silu(dense[0][e] @ xd[t] + biases[0][e]) * (dense[1][e] @ xd[t] + biases[1][e])
            total = total + sd[t, j] * (dense[2][e] @ hidden + biases[2][e])
        rows.append(total)
    want = torch.stack(rows)
    want_grads = torch.autograd.grad(want, (xd, sd), dout.double())
    # Seven roundings to bf16 lie on the longest path (three products, silu, the gate, the return, the gradient), each of 2^-8 at
    # most, and the gate's two factors count twice: 16 of them bound the relative error of the whole, taken over all elements.
    for got, expect in ((out, want), *zip(grads, want_grads)):
        assert ((got.double() - expect).norm() / expect.norm()).item() <= 16 * HALF_BF16
    with torch.no_grad():
        assert torch.equal(run(x, share), out)


def test_experts_follow_their_checkpoints_and_int8_experts():
    experts, inner, outer, tokens = 3, 256, 96, 40
    first = ep.CompressedGroupedLinear.from_linears([_dense(outer, inner, e) for e in range(experts)], config=ep.EntroPackLossyConfig(target_bpp=4.0)).cuda()
    other = ep.CompressedGroupedLinear.from_linears([_dense(outer, inner, 50 + e) for e in range(experts)], config=ep.EntroPackLossyConfig(target_bpp=4.0)).cuda()
    plan = ep.group_rows(_ids(tokens, 1, experts, "padded"), experts)
    x = torch.randn(tokens, inner, device="cuda").bfloat16()
    before, wanted = first(x, plan), other(x, plan)
    assert torch.equal(before, ep.grouped_linear(x, first.dequantize(), plan, torch.stack([e.bias for e in first.experts])))
    held = first._decoder
    assert torch.equal(first(x, plan), before) and first._decoder is held                # no second plan for the same weights
    first.load_state_dict(other.state_dict())
    assert torch.equal(first(x, plan), wanted) and not torch.equal(before, wanted)

    for options in ({"config": ep.EntroPackLossyConfig(target_bpp=5.0)}, {}, {"use_convrot": True}):
        layer = ep.CompressedGroupedLinear.from_linears([_dense(outer, inner, e) for e in range(experts)], int8=True, **options).cuda()
        y = layer(x, plan)
        for g, expert in enumerate(layer.experts):                                       # the same codes as each layer by itself
            rows = plan.order[int(plan.offsets[g]):int(plan.offsets[g + 1])].long()
            assert torch.equal(y[int(plan.offsets[g]):int(plan.offsets[g + 1])], expert(x[rows]))
        leaf = x.clone().requires_grad_(True)
        dy = torch.randn(tokens, outer, device="cuda").bfloat16()
        grad = torch.autograd.grad(layer(leaf, plan), leaf, dy)[0]
        want = torch.autograd.grad(ep.grouped_linear(leaf, layer.dequantize(), plan), leaf, dy)[0]
        assert torch.equal(grad, want)


def test_adapted_layer_trains_beside_its_compressed_weight():
    inner, outer, tokens, adapters, rank = 256, 192, 45, 3, 8
    for base in (ep.CompressedLinear.from_linear(_dense(outer, inner, 1), config=ep.EntroPackLossyConfig(target_bpp=4.0), forward_mode="fused").cuda(),
                 ep.CompressedINT8Linear.from_linear(_dense(outer, inner, 1)).cuda()):
        layer = ep.AdaptedLinear(base, adapters, rank).cuda()
        ids = _ids(tokens, 0, adapters, "padded")
        plan = ep.group_rows(ids, adapters)
        x = torch.randn(5, 9, inner, device="cuda").bfloat16().requires_grad_(True)
        assert torch.equal(layer(x, plan), base(x))                                   # fresh adapters change nothing
        layer.set_adapter(1, torch.randn(6, inner) * 0.1, torch.randn(outer, 6) * 0.1, scale=0.5)
        layer.set_adapter(2, torch.randn(rank, inner) * 0.1, torch.randn(outer, rank) * 0.1)
        out = layer(x, plan)
        dout = torch.randn(out.shape, device="cuda").bfloat16()
        out.backward(dout)
        rows = x.detach().reshape(-1, inner)
        with torch.no_grad():
            assert torch.equal(out.reshape(-1, outer), ep.low_rank_update(base(rows), rows, layer.down, layer.up, plan, layer.scale))
            want = layer.base.dequantize().double().t() @ dout.reshape(-1, outer).double().t()
            for a, members in enumerate(_members(ids, adapters)):
                want[:, members] += layer.scale[a].double() * layer.down[a].double().t() @ (layer.up[a].double().t() @ dout.reshape(-1, outer)[members].double().t())
        # two gradients rounded to bf16 and their sum rounded again: three half steps of the largest part
        assert ((x.grad.reshape(-1, inner).double().t() - want).norm() / want.norm()).item() <= 3 * HALF_BF16
        assert layer.down.grad is not None and layer.up.grad is not None and layer.up.grad.abs().sum() > 0
        again = ep.AdaptedLinear(base, adapters, rank).cuda()
        again.load_state_dict(layer.state_dict())
        with torch.no_grad():
            assert torch.equal(again(x, plan), layer(x, plan))


def test_another_stream_and_a_replayed_graph():
    """The same work on a stream of its own, and captured once (the sort of the ids included) and replayed with new ids and
    inputs, eager work and synchronisations between the replays; every replay equals the eager call."""
    tokens, per_row, groups, inner, outer = 96, 2, 5, 256, 200
    w = (torch.randn(groups, outer, inner, device="cuda") * 0.1).bfloat16().requires_grad_(True)
    codes, scale_w = torch.randint(-127, 128, (groups, outer, inner), device="cuda", dtype=torch.int8), torch.rand(groups, outer, device="cuda") * 0.01
    down, up = (torch.randn(groups, 16, inner, device="cuda") * 0.1).bfloat16().requires_grad_(True), torch.randn(groups, inner, 16, device="cuda").bfloat16().requires_grad_(True)
    ids, x, share = torch.zeros(tokens, per_row, dtype=torch.int64, device="cuda"), torch.zeros(tokens, inner, device="cuda").bfloat16(), torch.zeros(tokens, per_row, device="cuda")

    def step(x, ids, share):
        leaf = x.detach().requires_grad_(True)
        plan, one = ep.group_rows(ids, groups), ep.group_rows(ids[:, 0], groups)
        out = ep.combine_rows(ep.grouped_linear(leaf, w, plan), plan, share)
        lifted = ep.low_rank_update(leaf, leaf, down, up, one)
        q, s = kernels.quantize_rows(x)
        return [out, lifted, ep.grouped_int8_linear(q, codes, plan, s, scale_w),
                *torch.autograd.grad((out, lifted), (leaf, w, down, up), (torch.ones_like(out), torch.ones_like(lifted)))]

    def fill(seed):
        x.copy_(torch.randn(tokens, inner, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        ids.copy_(_ids(tokens, per_row, groups, "padded", seed))
        share.copy_(torch.rand(tokens, per_row, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))

    # Results are kept detached: an eager graph over w, down and up that lived through the capture would tie their gradients to
    # the eager stream, and the captured backward would draw that stream into the capture.
    fill(0)
    eager = [t.detach().clone() for t in step(x, ids, share)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [t.detach().clone() for t in step(x, ids, share)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(there, eager))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            held = [t.detach() for t in step(x, ids, share)]
    torch.cuda.current_stream().wait_stream(side)
    for replay in range(4):
        fill(replay)
        for tensor in held:
            tensor.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(got, step(x, ids, share))), replay
        assert torch.isfinite(torch.randn(1 << 20, device="cuda").sum()).item()


def test_layers_copied_captured_and_used_on_two_streams_at_once():
    experts, inner, outer, tokens = 3, 256, 192, 33
    config = ep.EntroPackLossyConfig(target_bpp=4.0)
    mixture = ep.CompressedGroupedLinear.from_linears([_dense(outer, inner, e) for e in range(experts)], config=config).cuda()
    adapted = ep.AdaptedLinear(ep.CompressedLinear.from_linear(_dense(outer, inner, 7), config=config).cuda(), experts, 8).cuda()
    adapted.set_adapter(1, torch.randn(8, inner) * 0.1, torch.randn(outer, 8) * 0.1)
    x, ids = torch.randn(tokens, inner, device="cuda").bfloat16(), _ids(tokens, 0, experts, "padded")

    def run(mixture, adapted, x, ids):
        plan = ep.group_rows(ids, experts)
        return ep.combine_rows(mixture(x, plan), plan), adapted(x, plan)

    with torch.no_grad():
        want = run(mixture, adapted, x, ids)
        twins = copy.deepcopy(mixture), copy.deepcopy(adapted)
        assert twins[0]._decoder is None and mixture._decoder is not None
        assert all(torch.equal(a, b) for a, b in zip(run(*twins, x, ids), want))
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for turn in range(6):
            with torch.cuda.stream(streams[turn % 2]):
                got.append(run(mixture, adapted, x, ids))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for result in got for a, b in zip(result, want))
        fixed, fixed_ids = x.clone(), ids.clone()
        graphs = []
        for _ in range(2):                                # two graphs of the same layers
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                graphs.append((graph, run(mixture, adapted, fixed, fixed_ids)))
        for seed in range(3):
            fixed.copy_(torch.randn(tokens, inner, device="cuda"))
            fixed_ids.copy_(_ids(tokens, 0, experts, "padded", seed))
            expect = run(mixture, adapted, fixed, fixed_ids)
            for graph, held in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for _, held in graphs:
                assert all(torch.equal(a, b) for a, b in zip(held, expect)), seed


def test_any_subset_of_gradients_and_none_of_second_order():
    groups, tokens, inner, outer, rank = 3, 50, 72, 40, 5
    source = torch.Generator(device="cuda").manual_seed(5)
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=source).bfloat16()
    one, two = ep.group_rows(_ids(tokens, 0, groups, "padded"), groups), ep.group_rows(_ids(tokens, 2, groups, "padded"), groups)
    share = torch.rand(tokens, 2, device="cuda", generator=source)
    cases = [(lambda y, x, d, u: ep.low_rank_update(y, x, d, u, one), (randn(tokens, outer), randn(tokens, inner), randn(groups, rank, inner), randn(groups, outer, rank))),
             (lambda x, w, b: ep.grouped_linear(x, w, two, b), (randn(tokens, inner), randn(groups, outer, inner), randn(groups, outer))),
             (lambda y, w: ep.combine_rows(y, two, w), (randn(two.entries, outer), share)), (lambda y, w: ep.combine_rows(y, two, w), (randn(two.entries, outer), share.bfloat16()))]
    for run, operands in cases:
        full = [t.clone().requires_grad_(True) for t in operands]
        out = run(*full)
        dout = randn(*out.shape)
        want = torch.autograd.grad(out, full, dout)
        for chosen in range(1, 1 << len(operands)):
            leaves = [t.clone().requires_grad_(bool(chosen >> i & 1)) for i, t in enumerate(operands)]
            asked = [leaf for leaf in leaves if leaf.requires_grad]
            got = torch.autograd.grad(run(*leaves), asked, dout)
            assert all(torch.equal(a, want[i]) for a, i in zip(got, [i for i in range(len(operands)) if chosen >> i & 1])), chosen
        first = torch.autograd.grad(run(*full), full[0], dout.requires_grad_(True), create_graph=True)[0]
        assert torch.equal(first, want[0])
        with pytest.raises(RuntimeError, match="once_differentiable"):
            first.sum().backward()


def test_operands_past_two_to_the_31_elements():
    """300000 rows of 8192: the last of them lie past 32 bits of elements. Few rows have a group; they are spread over the whole."""
    tokens, wide, narrow, groups, rank = 300_000, 8192, 64, 3, 16
    rows = torch.tensor([0, 1, 70_000, 140_001, 262_143, 262_144, 262_145, 299_998, 299_999], device="cuda")
    ids = torch.full((tokens,), -1, dtype=torch.int64, device="cuda")
    ids[rows] = torch.arange(len(rows), device="cuda") % groups
    plan = ep.group_rows(ids, groups)
    x = torch.zeros(tokens, wide, dtype=torch.bfloat16, device="cuda")
    x[rows] = torch.randn(len(rows), wide, device="cuda").bfloat16()
    x.requires_grad_(True)
    weight = (torch.randn(groups, narrow, wide, device="cuda") * 0.05).bfloat16().requires_grad_(True)
    kept, group, place = len(rows), ids[rows], plan.place.long()[rows]
    y = ep.grouped_linear(x, weight, plan)
    dy = torch.zeros_like(y)
    dy[:kept] = torch.randn(kept, narrow, device="cuda").bfloat16()
    gx, gw = torch.autograd.grad(y, (x, weight), dy)
    # Against 64 bits: the mean rows per group choose the kernel and with it the order of the sums, so that the same rows in a small
    # batch need not give the same bits.
    xd, wd, dyd = x.detach()[rows].double(), weight.detach().double()[group], dy[place].double()
    times = lambda a, b: (a.unsqueeze(1) @ b).squeeze(1)
    want, size = times(xd, wd.transpose(1, 2).contiguous()), times(xd.abs(), wd.abs().transpose(1, 2).contiguous())
    _within(y[place], want, _bound(want, size, wide))
    _within(gx[rows], times(dyd, wd), _bound(times(dyd, wd), times(dyd.abs(), wd.abs()), narrow))
    for g in range(groups):
        mine = group == g
        _within(gw[g], dyd[mine].t() @ xd[mine], _bound(dyd[mine].t() @ xd[mine], dyd[mine].abs().t() @ xd[mine].abs(), kept))
    assert y[kept:].eq(0).all()
    assert gx[:70_000][2:].eq(0).all() and gx[262_146:299_998].eq(0).all()
    del gx, y, dy

    down, up = (torch.randn(groups, rank, narrow, device="cuda") * 0.1).bfloat16(), torch.randn(groups, wide, rank, device="cuda").bfloat16()
    thin = torch.randn(tokens, narrow, device="cuda").bfloat16()
    with torch.no_grad():
        out = ep.low_rank_update(x, thin, down, up, plan)
        hidden, hidden_size = times(thin[rows].double(), down.double()[group].transpose(1, 2)), times(thin[rows].double().abs(), down.double()[group].abs().transpose(1, 2))
        u = up.double()[group].transpose(1, 2)
        want = x[rows].double() + times(hidden, u)
        # the narrow sums' own error and their two parts' 2^-16, carried through |up|, besides the second product's
        carried = times(narrow * STEP_F32 * hidden_size + 2.0 ** -16 * hidden.abs(), u.abs()) * 1.01
        _within(out[rows], want, _bound(want, x[rows].double().abs() + times(hidden.abs(), u.abs()), 2 * rank + 1) + carried)
        out[rows] = x[rows]
        assert torch.equal(out, x)
        del out
        back = ep.low_rank_update(thin, x, torch.ones(groups, 1, wide, device="cuda").bfloat16(), torch.ones(groups, narrow, 1, device="cuda").bfloat16(), plan)
        sums = x[rows].double().sum(1, keepdim=True)
        want = thin[rows].double() + sums
        _within(back[rows], want, _bound(want, x[rows].double().abs().sum(1, keepdim=True) + thin[rows].double().abs(), wide + 3) + 2.0 ** -16 * 1.01 * sums.abs())
        combined = ep.combine_rows(x, plan)                  # here x holds places: those of a group are the first
        assert torch.equal(combined[rows], x[plan.place.long()[rows]]) and combined[2:70_000].eq(0).all()
