"""GPU tests of the operators on grouped rows where results are small against what they are sums of, where operands lie oddly, at
sizes that other kernels serve, and through the entry points of the C library. Against plain implementations in 64 bits.

Tolerances: products of two bf16 numbers are exact in f32; every addition of a sum, in any order and whichever way the matrix cores
round, is off by at most a whole unit in the last place, 2^-23 of the sum of the magnitudes; a rounding to bf16 by half a step, 2^-8 of
the value.
"""
import weakref

import pytest
import torch

import entropack_amd as ep
from entropack_amd.backends import hip

pytestmark = pytest.mark.gpu
HALF_BF16, STEP_F32 = 2.0 ** -8, 2.0 ** -23


def whole(columns):
    """Columns of a row in whole pieces of 16 bytes."""
    return (columns + 7) // 8 * 8


def _within(got, expect, bound):
    off = (got.double() - expect).abs()
    assert torch.isfinite(got.double()).all()
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert worst <= 0.0, f"off by {worst} more than the bound; largest difference {off.max().item()}"


@pytest.mark.parametrize("tokens", [20, 40], ids=["few rows", "many rows"])       # 16 rows per block in the product with `up`, and 64
def test_narrow_rows_of_an_adapter_lose_nothing(tokens):
    """One feature, rank one: h = s (x d) is one product of three numbers, exact but for the rounding of an f32. y is the update's negative
    rounded to bf16, so that what is left is some 2^-9 of the update and shows what of it was lost on the way. Three parts' products
    and y make four additions; with the rounding of h eight steps bound them, of |y| + |update|."""
    outer = 4096
    source = torch.Generator(device="cuda").manual_seed(7)
    make = lambda *shape: torch.randn(*shape, device="cuda", generator=source).bfloat16()
    plan = ep.group_rows(torch.zeros(tokens, dtype=torch.int64, device="cuda"), 1)
    x, down, up, scale = make(tokens, 1), make(1, 1, 1), make(1, outer, 1), 0.5 + torch.rand(1, device="cuda", generator=source)
    update = (scale.double() * x.double() * down[0, 0, 0].double()) * up[0, :, 0].double()
    y = (-update).bfloat16()
    out = ep.low_rank_update(y, x, down, up, plan, scale)
    want = y.double() + update
    _within(out, want, HALF_BF16 * want.abs() + 8 * STEP_F32 * (y.double().abs() + update.abs()))


def test_narrow_rows_of_an_adapters_gradients_lose_nothing():
    """The same for the gradients: each is a sum of two terms that cancel to some 2^-9 of either. Of x: two ranks, whose second row of
    `down` is chosen so; of `down` and `up`: two tokens, the second's row of the other operand chosen so."""
    wide = 4096
    source = torch.Generator(device="cuda").manual_seed(8)
    make = lambda *shape: torch.randn(*shape, device="cuda", generator=source).bfloat16()
    scale = 0.5 + torch.rand(1, device="cuda", generator=source)
    s = scale.double()

    def gradients(x, down, up, dout):
        plan = ep.group_rows(torch.zeros(len(x), dtype=torch.int64, device="cuda"), 1)
        leaves = [t.requires_grad_(True) for t in (x, down, up)]
        return torch.autograd.grad(ep.low_rank_update(torch.zeros_like(dout), *leaves, plan, scale), leaves, dout)

    def check(got, first, second):                           # two terms of three parts each: eight additions and two roundings of an f32
        want = first + second
        assert want.abs().median() < 2.0 ** -8 * first.abs().median()
        _within(got, want, HALF_BF16 * want.abs() + 10 * STEP_F32 * (first.abs() + second.abs()))

    # gradient of x: e_0 down[0] + e_1 down[1] with e_r = s dout up[r]
    dout, up, x = make(1, 1), make(1, 1, 2), make(1, wide)
    e = s * dout.double()[0, 0] * up.double()[0, 0]
    down = make(1, 2, wide)
    down[0, 1] = (-e[0] * down[0, 0].double() / e[1]).bfloat16()
    check(gradients(x, down, up, dout)[0][0], e[0] * down[0, 0].double(), e[1] * down[0, 1].double())

    # gradient of down: e_0 x[0] + e_1 x[1] with e_t = s dout[t] up
    dout, up, x, down = make(2, 1), make(1, 1, 1), make(2, wide), make(1, 1, wide)
    e = s * dout.double()[:, 0] * up.double()[0, 0, 0]
    x[1] = (-e[0] * x[0].double() / e[1]).bfloat16()
    check(gradients(x, down, up, dout)[1][0, 0], e[0] * x[0].double(), e[1] * x[1].double())

    # gradient of up: h_0 dout[0] + h_1 dout[1] with h_t = s x[t] down
    dout, up, x, down = make(2, wide), make(1, wide, 1), make(2, 1), make(1, 1, 1)
    h = s * x.double()[:, 0] * down.double()[0, 0, 0]
    dout[1] = (-h[0] * dout[0].double() / h[1]).bfloat16()
    check(gradients(x, down, up, dout)[2][0, :, 0], h[0] * dout[0].double(), h[1] * dout[1].double())


def _linears(experts, outer, inner, bias=True):
    torch.manual_seed(4)
    return [torch.nn.Linear(inner, outer, bias=bias, dtype=torch.bfloat16) for _ in range(experts)]


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("of_x", [False, True], ids=["biases alone", "and x"])
def test_biases_of_compressed_experts_that_train_get_their_gradient(int8, of_x):
    experts, outer, inner, tokens = 3, 72, 128, 40
    options = {"int8": True} if int8 else {"config": ep.EntroPackLossyConfig(target_bpp=4.0)}
    layer = ep.CompressedGroupedLinear.from_linears(_linears(experts, outer, inner), **options).cuda()
    ids = torch.randint(-1, experts, (tokens, 2), generator=torch.Generator().manual_seed(1)).cuda()
    plan = ep.group_rows(ids, experts)
    x = torch.randn(tokens, inner, device="cuda").bfloat16()
    frozen = layer(x, plan)
    biases = [expert.bias.requires_grad_(True) for expert in layer.experts]
    leaves = biases + ([x.requires_grad_(True)] if of_x else [])
    y = layer(x, plan)
    assert torch.equal(y, frozen)
    dy = torch.randn(y.shape, device="cuda").bfloat16()
    grads = torch.autograd.grad(y, leaves, dy)
    for g in range(experts):
        rows = dy[int(plan.offsets[g]):int(plan.offsets[g + 1])].double()
        _within(grads[g], rows.sum(0), HALF_BF16 * rows.sum(0).abs() + len(rows) * STEP_F32 * rows.abs().sum(0) * 1.01)
    if of_x:
        plain = x.detach().requires_grad_(True)
        want = torch.autograd.grad(ep.grouped_linear(plain, layer.dequantize().bfloat16(), plan), plain, dy)[0]
        assert torch.equal(grads[experts], want)
    with torch.no_grad():
        assert torch.equal(layer(x, plan), frozen)


def test_biases_in_f32_get_gradients_that_were_not_rounded_to_bf16():
    """int8 experts of an f32 model keep f32 biases; the sums of the bf16 gradient's columns are f32."""
    experts, outer, inner, tokens = 2, 40, 64, 300
    torch.manual_seed(4)
    layer = ep.CompressedGroupedLinear.from_linears([torch.nn.Linear(inner, outer) for _ in range(experts)], int8=True).cuda()
    biases = [expert.bias.requires_grad_(True) for expert in layer.experts]
    assert biases[0].dtype == torch.float32
    plan = ep.group_rows(torch.arange(tokens, device="cuda") % experts, experts)
    y = layer(torch.randn(tokens, inner, device="cuda").bfloat16(), plan)
    dy = torch.randn(y.shape, device="cuda").bfloat16()
    for g, grad in enumerate(torch.autograd.grad(y, biases, dy)):
        rows = dy[int(plan.offsets[g]):int(plan.offsets[g + 1])].double()
        assert grad.dtype == torch.float32
        _within(grad, rows.sum(0), len(rows) * STEP_F32 * rows.abs().sum(0))


def test_a_mixture_on_the_host_plans_once_and_one_that_leaves_the_device_lets_go():
    experts, outer, inner, tokens = 3, 72, 128, 40
    layer = ep.CompressedGroupedLinear.from_linears(_linears(experts, outer, inner), config=ep.EntroPackLossyConfig(target_bpp=4.0))
    plan = ep.group_rows(torch.arange(tokens, device="cuda") % (experts + 1), experts)
    x = torch.randn(tokens, inner, device="cuda").bfloat16()
    there = layer(x, plan)
    held = layer._decoder
    assert torch.equal(layer(x, plan), there) and layer._decoder is held
    leaf = x.clone().requires_grad_(True)
    layer(leaf, plan).sum().backward()
    assert layer._decoder is held
    layer.cuda()
    assert layer._decoder is None and torch.equal(layer(x, plan), there)
    again = layer._decoder
    assert torch.equal(layer.dequantize("cuda"), layer.dequantize()) and layer._decoder is again
    del again
    payload = weakref.ref(layer.experts[0].weight.buffers["payload"])
    del held
    layer.cpu()
    assert payload() is None
    assert torch.equal(layer(x, plan), there)


@pytest.mark.parametrize("width", [8, 257], ids=["a block per token", "a thread per element"])
def test_weighted_return_of_more_tokens_than_a_launch_takes(width):
    """2^24 + 37 tokens: the gradient's blocks of one token each, and at width 257 the forward's threads too, pass 2^32 work items. One entry
    per token and no weight: the return and its gradient copy rows, exactly. With weights: a power of two each, exact again."""
    tokens, count = (1 << 24) + 37, 5
    source = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.randint(-1, count, (tokens,), device="cuda", generator=source)
    plan = ep.group_rows(ids, count)
    place, none = plan.place.long(), ids < 0
    y = torch.empty(tokens, width, dtype=torch.bfloat16, device="cuda").normal_(generator=source)
    for weight in (None, torch.exp2(torch.randint(-3, 3, (tokens,), device="cuda", generator=source).float())):
        leaves = [y.requires_grad_(True)] + ([] if weight is None else [weight.requires_grad_(True)])
        out = ep.combine_rows(y, plan, weight)
        dout = torch.empty_like(out).normal_(generator=source)
        grads = torch.autograd.grad(out, leaves, dout)
        with torch.no_grad():
            for first in range(0, tokens, 1 << 21):
                some = slice(first, first + (1 << 21))
                factor = 1.0 if weight is None else weight[some].unsqueeze(1)
                dead = none[some].unsqueeze(1)
                rows = y[place[some]].float()
                assert torch.equal(out[some], torch.where(dead, 0.0, factor * rows).bfloat16())
                assert torch.equal(grads[0][place[some]], torch.where(dead, 0.0, factor * dout[some].float()).bfloat16())
                if weight is not None:
                    dot, size = (rows.double() * dout[some].double()).sum(1), (rows.double() * dout[some].double()).abs().sum(1)
                    _within(grads[1][some], torch.where(none[some], 0.0, dot), (width + 2) * STEP_F32 * size)
        del out, dout, grads


@pytest.mark.parametrize("wanted", range(1, 8))
@pytest.mark.parametrize("tokens,count,rank,inner,outer", [(50, 3, 5, 72, 40), (700, 20, 33, 264, 130)])
def test_gradients_of_adapters_keep_to_the_workspace_of_what_is_asked_for(wanted, tokens, count, rank, inner, outer):
    """The entry point itself, its workspace between two guards and full of NaN, so that nothing can be read that was not written."""
    lib = hip.library()
    source = torch.Generator(device="cuda").manual_seed(2)
    make = lambda *shape: torch.randn(*shape, device="cuda", generator=source).bfloat16()
    plan = ep.group_rows(torch.randint(-1, count, (tokens,), device="cuda", generator=source), count)
    y, x, down, up, dout = make(tokens, outer), make(tokens, inner), make(count, rank, inner), make(count, outer, rank), make(tokens, whole(outer))
    dout[:, outer:] = 0
    leaves = [t.requires_grad_(True) for t in (x, down, up)]
    want = torch.autograd.grad(ep.low_rank_update(y, *leaves, plan), leaves, dout[:, :outer])
    x, down, up = (t.detach() for t in leaves)
    stream = torch.cuda.current_stream().cuda_stream
    planes = torch.empty(lib.ep_hip_low_rank_planes_bytes(tokens, rank), dtype=torch.uint8, device="cuda")
    out = torch.empty(tokens, outer, dtype=torch.bfloat16, device="cuda")
    shape = (plan.order.data_ptr(), plan.offsets.data_ptr(), tokens, count, rank, inner, outer)
    hip.check("forward", lib.ep_hip_low_rank_update(x.data_ptr(), inner, down.data_ptr(), inner, rank * inner, up.data_ptr(), rank, outer * rank, None, y.data_ptr(), outer, planes.data_ptr(),
                                                    out.data_ptr(), outer, *shape, stream))
    flags = [wanted & 1, wanted >> 1 & 1, wanted >> 2 & 1]
    room, guard = lib.ep_hip_low_rank_grad_workspace_for(tokens, count, rank, inner, outer, *flags), 4096
    space = torch.full((room + 2 * guard,), 0xFF, dtype=torch.uint8, device="cuda")
    got = [torch.full_like(t, float("nan")) if flag else None for t, flag in zip((x, down, up), flags)]
    at = [None if t is None else t.data_ptr() for t in got]
    hip.check("gradients", lib.ep_hip_low_rank_update_grad(dout.data_ptr(), dout.stride(0), x.data_ptr(), inner, down.data_ptr(), inner, rank * inner, up.data_ptr(), rank, outer * rank, None,
                                                           planes.data_ptr(), at[0], inner, at[1], at[2], *shape, space.data_ptr() + guard, room, stream))
    assert space[:guard].eq(0xFF).all() and space[guard + room:].eq(0xFF).all()
    assert all(torch.equal(a, b) for a, b, flag in zip(got, want, flags) if flag)


# rows, adapters, rank, in, out, ids: what the kernels for many rows take (64 rows per block of the expand with 16, 32 and 64 ranks at a
# time, the shrink from 2048 rows on), and chunks of the weights' gradients of many steps that do not divide the groups' rows.
MANY_ROWS = [(4099, 4, 16, 1032, 1041, "skewed"), (2500, 2, 8, 264, 72, "padded"), (5000, 3, 16, 4096, 4096, "padded"), (2048, 1, 4, 520, 1032, "even"), (6000, 5, 32, 2056, 1000, "skewed"),
             (3000, 2, 64, 4096, 520, "padded"), (2300, 3, 100, 264, 2064, "even"), (9000, 2, 17, 4100, 4099, "even"), (5000, 64, 16, 1032, 1032, "skewed")]


@pytest.mark.parametrize("case", MANY_ROWS, ids=str)
def test_low_rank_update_of_many_rows_and_gradients(case):
    """The narrow rows h are f32: off by their own sum and the scale's product, (inner + 2) steps of their magnitudes. They enter the second
    product whole, as three parts each: 3 rank additions and y's. A weight's gradient adds the places of a chunk in three sums, those, and
    the chunks: 2 n + 2 additions cover it."""
    print("case", case, flush=True)
    tokens, count, rank, inner, outer, kind = case
    source = torch.Generator(device="cuda").manual_seed(6)
    make = lambda *shape, scale=1.0: (torch.randn(*shape, device="cuda", generator=source) * scale).bfloat16()
    ids = torch.randint(0, count, (tokens,), device="cuda", generator=source)
    if kind == "skewed":
        ids = (torch.rand(tokens, device="cuda", generator=source) ** 3 * count).long()
    elif kind == "padded":
        ids[torch.rand(tokens, device="cuda", generator=source) < 0.3] = -1
    plan = ep.group_rows(ids, count)
    y, x, down, up, dout = make(tokens, outer), make(tokens, inner), make(count, rank, inner, scale=inner ** -0.5), make(count, outer, rank, scale=rank ** -0.5), make(tokens, outer)
    scale = 0.5 + torch.rand(count, device="cuda", generator=source)
    leaves = [t.requires_grad_(True) for t in (y, x, down, up)]
    out = ep.low_rank_update(*leaves, plan, scale)
    grad_y, grad_x, grad_down, grad_up = torch.autograd.grad(out, leaves, dout)
    assert torch.equal(grad_y, dout)
    narrow_f, narrow_b, second = (inner + 2) * STEP_F32, (outer + 2) * STEP_F32, (3 * rank + 2) * STEP_F32 * (1 + HALF_BF16)
    whole_of = lambda value, error: HALF_BF16 * value.abs() + (1 + HALF_BF16) * error + 1e-37
    with torch.no_grad():
        for a in range(count):
            rows = torch.nonzero(ids == a).reshape(-1)
            s, xs, dn, u, dy = scale[a].double(), x[rows].double(), down[a].double(), up[a].double(), dout[rows].double()
            h, h_size = s * (xs @ dn.t()), s * (xs.abs() @ dn.abs().t())
            want = y[rows].double() + h @ u.t()
            _within(out[rows], want, whole_of(want, (second + narrow_f) * (h_size @ u.abs().t()) + STEP_F32 * y[rows].double().abs()))
            e, e_size = s * (dy @ u), s * (dy.abs() @ u.abs())
            _within(grad_x[rows], e @ dn, whole_of(e @ dn, (second + narrow_b) * (e_size @ dn.abs())))
            many = (2 * len(rows) + 2) * STEP_F32 * (1 + HALF_BF16)
            _within(grad_down[a], e.t() @ xs, whole_of(e.t() @ xs, (many + narrow_b) * (e_size.t() @ xs.abs())))
            _within(grad_up[a], dy.t() @ h, whole_of(dy.t() @ h, (many + narrow_f) * (dy.abs().t() @ h_size)))
        none = ids < 0
        assert torch.equal(out[none], y[none]) and grad_x[none].eq(0).all()


def _odd_views(t):
    """The same values lying oddly: a wider row's part, misaligned by an element, transposed, every other row."""
    rows, columns = t.shape
    wide = torch.empty(rows, columns + 24, dtype=t.dtype, device=t.device)
    part, shifted, turned, sparse = wide[:, :columns], torch.empty_like(wide)[:, 3:3 + columns], torch.empty(columns, rows, dtype=t.dtype, device=t.device).t(), \
        torch.empty(2 * rows, columns, dtype=t.dtype, device=t.device)[::2]
    return [view.copy_(t) for view in (part, shifted, turned, sparse)]


@pytest.mark.parametrize("tokens,per_row,width", [(33, 2, 264), (70, 3, 33), (5, 9, 2048)])
def test_combine_rows_of_operands_that_lie_oddly(tokens, per_row, width):
    """Sums per element do not depend on how the operands lie: outputs and rows' gradients are equal. The weights' gradient is a dot product
    whose lanes follow the loads: within its bound."""
    count = 4
    source = torch.Generator(device="cuda").manual_seed(9)
    ids = torch.randint(-1, count, (tokens, per_row), device="cuda", generator=source)
    plan = ep.group_rows(ids, count)
    y = torch.randn(tokens * per_row, width, device="cuda", generator=source).bfloat16()
    weight = torch.rand(tokens, per_row, device="cuda", generator=source)
    dout = torch.randn(tokens, width, device="cuda", generator=source).bfloat16()

    def run(y, weight, dout):
        y, weight = y.detach().requires_grad_(True), weight.detach().requires_grad_(True)
        out = ep.combine_rows(y, plan, weight)
        return (out.detach(), *torch.autograd.grad(out, (y, weight), dout))

    def check(got, want, y, dout):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[2].shape == weight.shape
        rows = torch.where((ids >= 0).unsqueeze(2), y[plan.place.long()].reshape(tokens, per_row, width).double(), 0.0)
        dot, size = (rows * dout.double().unsqueeze(1)).sum(2), (rows.abs() * dout.double().abs().unsqueeze(1)).sum(2)
        _within(got[2], dot, (width + 2) * STEP_F32 * size)

    want = run(y, weight, dout)
    check(want, want, y, dout)
    for odd_y in _odd_views(y):
        check(run(odd_y, weight, dout), want, y, dout)
    for odd_dout in _odd_views(dout):
        check(run(y, weight, odd_dout), want, y, dout)
    for odd_weight in _odd_views(weight):
        check(run(y, odd_weight, dout), want, y, dout)
    ones = torch.ones((), device="cuda", dtype=torch.bfloat16)
    check(run(y, weight, ones.expand(tokens, width)), run(y, weight, torch.ones_like(dout)), y, torch.ones_like(dout))        # a sum's gradient
    check(run(y[:1].expand_as(y), weight, dout), run(y[:1].expand_as(y).contiguous(), weight, dout), y[:1].expand_as(y), dout)
    check(run(y, weight[:1, :1].expand_as(weight), dout), run(y, weight[:1, :1].expand_as(weight).contiguous(), dout), y, dout)


HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 0.0}


# entries' tokens, ids per token, groups, K, N: the kernels for few rows, 128 x 128 and 256 x 256 tiles, sums of chunks
@pytest.mark.parametrize("tokens,per_row,count,inner,outer", [(40, 2, 30, 72, 104), (30, 2, 4, 264, 72), (700, 1, 2, 264, 520), (4200, 1, 3, 1032, 2056), (9000, 1, 2, 136, 72)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_products_through_the_c_library_in_every_output_type(tokens, per_row, count, inner, outer, dtype):
    """Outputs of f16 and f32, which the Python functions do not ask for, in rows wider than they are: what lies behind a row stays."""
    print("case", tokens, per_row, count, inner, outer, dtype, flush=True)
    lib, kind, stream, margin = hip.library(), hip.FLOAT_KINDS[dtype], torch.cuda.current_stream().cuda_stream, 16
    source = torch.Generator(device="cuda").manual_seed(5)
    make = lambda *shape: torch.randn(*shape, device="cuda", generator=source).bfloat16()
    plan = ep.group_rows(torch.randint(-1, count, (tokens, per_row), device="cuda", generator=source), count)
    entries, kept = plan.entries, int(plan.offsets[-1])
    x, w, dy = make(tokens, inner), make(count, outer, inner) * 0.05, make(entries, outer)
    bias = torch.randn(count, outer, device="cuda", generator=source).to(dtype)
    mark = 7.0
    room = lambda *shape: torch.full((*shape[:-1], shape[-1] + margin), mark, dtype=dtype, device="cuda")
    y, dx, dw, db = room(entries, outer), room(entries, inner), room(count, outer, inner), torch.full((count, outer), mark, dtype=dtype, device="cuda")
    common = (plan.offsets.data_ptr(), entries, count, outer, inner)
    hip.check("forward", lib.ep_hip_grouped_gemm_bf16(x.data_ptr(), inner, tokens, w.data_ptr(), inner, outer * inner, bias.data_ptr(), y.data_ptr(), outer + margin, kind, plan.rows.data_ptr(),
                                                      *common, stream))
    hip.check("rows", lib.ep_hip_grouped_grad_rows_bf16(dy.data_ptr(), outer, w.data_ptr(), inner, outer * inner, dx.data_ptr(), inner + margin, kind, plan.order.data_ptr(), *common, stream))
    bytes_ = lib.ep_hip_grouped_grad_weight_workspace(entries, count, outer, inner)
    space = torch.full((bytes_,), 0xFF, dtype=torch.uint8, device="cuda")
    hip.check("weight", lib.ep_hip_grouped_grad_weight_bf16(dy.data_ptr(), outer, x.data_ptr(), inner, tokens, dw.data_ptr(), inner + margin, outer * (inner + margin), kind,
                                                            plan.rows.data_ptr(), *common, space.data_ptr() if bytes_ else None, bytes_, stream))
    hip.check("bias", lib.ep_hip_grouped_column_sums_bf16(dy.data_ptr(), outer, plan.offsets.data_ptr(), count, outer, db.data_ptr(), kind, stream))
    for tensor in (y, dx, dw):
        assert tensor[..., -margin:].eq(mark).all()
    y, dx, dw, half = y[..., :outer], dx[..., :inner], dw[..., :inner], HALF_STEP[dtype]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-37                          # half of f16's least step
    check = lambda got, want, size, terms: _within(got, want, half * want.abs() + (1 + half) * (terms + 2) * STEP_F32 * size + tiny)
    for g in range(count):
        first, last = int(plan.offsets[g]), int(plan.offsets[g + 1])
        order, rows, weight, slope = plan.order[first:last].long(), x[plan.rows[first:last].long()].double(), w[g].double(), dy[first:last].double()
        check(y[first:last], rows @ weight.t() + bias[g].double(), rows.abs() @ weight.abs().t() + bias[g].double().abs(), inner + 1)
        check(dx[order], slope @ weight, slope.abs() @ weight.abs(), outer)
        check(dw[g], slope.t() @ rows, slope.abs().t() @ rows.abs(), 2 * (last - first))
        check(db[g], slope.sum(0), slope.abs().sum(0), last - first)
    assert y[kept:].eq(0).all() and dx[plan.order[kept:].long()].eq(0).all()


@pytest.mark.parametrize("tokens,outer", [(20, 72), (20, 33), (300, 264), (300, 65)])
def test_update_through_the_c_library_without_a_shared_output(tokens, outer):
    lib, stream, inner, rank, count = hip.library(), torch.cuda.current_stream().cuda_stream, 64, 8, 3
    source = torch.Generator(device="cuda").manual_seed(5)
    make = lambda *shape: torch.randn(*shape, device="cuda", generator=source).bfloat16()
    ids = torch.randint(-1, count, (tokens,), device="cuda", generator=source)
    plan = ep.group_rows(ids, count)
    x, down, up = make(tokens, inner), make(count, rank, inner), make(count, outer, rank)
    assert lib.ep_hip_low_rank_planes_bytes(tokens, rank) == tokens * 64 * 2 and lib.ep_hip_low_rank_planes_bytes(tokens, 33) == tokens * 3 * 64 * 2
    planes = torch.full((lib.ep_hip_low_rank_planes_bytes(tokens, rank) + 256,), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.full((tokens, outer + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    hip.check("update", lib.ep_hip_low_rank_update(x.data_ptr(), inner, down.data_ptr(), inner, rank * inner, up.data_ptr(), rank, outer * rank, None, None, 0, planes.data_ptr(), out.data_ptr(),
                                                   outer + 8, plan.order.data_ptr(), plan.offsets.data_ptr(), tokens, count, rank, inner, outer, stream))
    want = ep.low_rank_update(torch.zeros(tokens, outer, dtype=torch.bfloat16, device="cuda"), x, down, up, plan)
    assert torch.equal(out[:, :outer], want) and out[:, outer:].eq(7.0).all() and out[ids < 0][:, :outer].eq(0).all()
    assert planes[-256:].eq(0xFF).all()
