"""What is measured of the operators on grouped rows: products by expert, row grouping, the weighted return, low-rank adapters.

Every activation row (or each of its k copies) carries an id that picks the weight it meets. `order` lists the entries
sorted by id, entries of one id in their original order and entries without a group (id -1: padding of a batch) last;
`offsets[g]` is the first place of group g in that list and `place` the inverse of `order`.
"""
import math

import torch

own = False


# ---- cases ---------------------------------------------------------------------------------------------------------

def listed():
    return [
        # One decode step of a small serving batch: 32 tokens, four experts each, a tenth of the slots padding.
        {"name": "group-decode", "op": "group", "tokens": 32, "top": 4, "groups": 64, "padding": 0.1},
        # A whole prompt batch, eight experts per token.
        {"name": "group-prompt", "op": "group", "tokens": 16411, "top": 8, "groups": 128, "padding": 0.0},
        # The experts' outputs of a decode step brought back to the tokens.
        {"name": "combine-decode", "op": "combine", "tokens": 32, "top": 4, "groups": 64, "width": 2048, "padding": 0.1, "train": False},
        # The same in a training step, with the gradients of the outputs and of the router's weights.
        {"name": "combine-train", "op": "combine", "tokens": 8111, "top": 2, "groups": 16, "width": 4096, "padding": 0.05, "train": True},
        # A single token through two of eight large experts: latency and the stream of two weights.
        {"name": "experts-one-token", "op": "experts", "tokens": 1, "top": 2, "groups": 8, "width": 4096, "outputs": 4096, "padding": 0.0, "train": False},
        # A decode step over many small experts: about one row each.
        {"name": "experts-decode", "op": "experts", "tokens": 18, "top": 4, "groups": 64, "width": 2048, "outputs": 1408, "padding": 0.1, "train": False},
        # A prompt batch through large experts: bound by the matrix cores.
        {"name": "experts-prompt", "op": "experts", "tokens": 8011, "top": 2, "groups": 8, "width": 4096, "outputs": 4096, "padding": 0.0, "train": False},
        # A training step of one projection: outputs, gradient of the activations and of every expert's weight.
        {"name": "experts-train", "op": "experts", "tokens": 4093, "top": 2, "groups": 16, "width": 2048, "outputs": 4096, "padding": 0.05, "train": True},
        # The W8A8 form of the prompt case.
        {"name": "experts-int8-prompt", "op": "experts-int8", "tokens": 4001, "top": 2, "groups": 8, "width": 4096, "outputs": 4096, "padding": 0.0},
        # A decode step of a server that holds 48 adapters: every token its own, some tokens none.
        {"name": "adapters-decode", "op": "adapters", "tokens": 61, "groups": 48, "rank": 16, "width": 4096, "outputs": 4096, "requests": 61, "padding": 0.1, "train": False},
        # Prompts of 24 requests packed into one batch.
        {"name": "adapters-prompt", "op": "adapters", "tokens": 7993, "groups": 16, "rank": 32, "width": 4096, "outputs": 4096, "requests": 24, "padding": 0.05, "train": False},
        # Four adapters trained side by side on a frozen projection.
        {"name": "adapters-train", "op": "adapters", "tokens": 4099, "groups": 4, "rank": 16, "width": 4096, "outputs": 4096, "requests": 16, "padding": 0.0, "train": True},
    ]


def _spread(rng, low, high):
    """An integer between low and high, even on a logarithmic scale."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _draw_any(rng):
    op = rng.choice(("group", "combine", "experts", "experts", "experts-int8", "adapters", "adapters"))
    padding = rng.choice((0.0, 0.0, 0.05, 0.3))
    if op == "group":
        return {"op": op, "tokens": _spread(rng, 1, 16411), "top": rng.randint(1, 8), "groups": _spread(rng, 2, 256), "padding": padding}
    if op == "combine":
        return {"op": op, "tokens": _spread(rng, 1, 8111), "top": rng.randint(1, 8), "groups": _spread(rng, 2, 128),
                "width": _spread(rng, 64, 8192), "padding": padding, "train": rng.random() < 0.5}
    width = 8 * _spread(rng, 16, 1024)
    outputs = 8 * _spread(rng, 16, 1024)
    if op == "adapters":
        tokens = _spread(rng, 1, 8192)
        return {"op": op, "tokens": tokens, "groups": _spread(rng, 1, 64), "rank": rng.choice((4, 8, 16, 24, 32, 64)), "width": width,
                "outputs": outputs, "requests": rng.randint(1, min(tokens, 64)), "padding": padding, "train": rng.random() < 0.4}
    case = {"op": op, "tokens": _spread(rng, 1, 8192), "top": rng.randint(1, 8), "groups": _spread(rng, 2, 64), "width": width,
            "outputs": outputs if rng.random() < 0.7 else outputs - rng.randint(1, 7), "padding": padding}
    if op == "experts":
        case["train"] = rng.random() < 0.4
        if case["train"]:
            case["outputs"] = outputs
    return case


def draw(rng):
    largest = [work(case) for case in listed()]
    top_bytes, top_flops = max(w["bytes"] for w in largest), max(w["flops"] for w in largest)
    while True:
        case = _draw_any(rng)
        cost = work(case)
        if cost["bytes"] <= top_bytes and cost["flops"] <= top_flops:
            return case


def work(case):
    tokens, groups = case["tokens"], case["groups"]
    entries = tokens * case.get("top", 1)
    kept = entries * (1.0 - case["padding"])
    if case["op"] == "group":
        return {"bytes": 16 * entries + 4 * (groups + 1), "flops": entries}
    if case["op"] == "combine":
        width = case["width"]
        size, flops = 2 * width * (kept + tokens) + 4 * entries, 2 * kept * width
        if case["train"]:
            size, flops = size + 2 * width * (tokens + entries) + 4 * entries, flops + 4 * kept * width
        return {"bytes": int(size), "flops": int(flops)}
    width, outputs = case["width"], case["outputs"]
    if case["op"] == "adapters":
        rank = case["rank"]
        hit = groups * (1.0 - (1.0 - 1.0 / groups) ** (case["requests"] * (1.0 - case["padding"])))
        size = 2 * tokens * (width + 2 * outputs) + 2 * hit * rank * (width + outputs)
        flops = 2 * kept * rank * (width + outputs)
        if case["train"]:        # the output's gradient read, those of x, down and up written
            size, flops = size + 2 * tokens * (outputs + width) + 2 * groups * rank * (width + outputs), 3 * flops
        return {"bytes": int(size), "flops": int(flops)}
    hit = groups * (1.0 - (1.0 - 1.0 / groups) ** kept)
    if case["op"] == "experts-int8":
        return {"bytes": int(tokens * (width + 4) + hit * outputs * (width + 4) + 2 * entries * outputs), "flops": int(2 * kept * width * outputs)}
    size = 2 * (tokens * width + hit * outputs * width + entries * outputs)
    flops = 2 * kept * width * outputs
    if case["train"]:            # the output's gradient read, those of x and of the weights written
        size, flops = size + 2 * (entries * outputs + tokens * width + groups * outputs * width), 3 * flops
    return {"bytes": int(size), "flops": int(flops)}


# ---- inputs --------------------------------------------------------------------------------------------------------

def _normal(source, *shape, scale=1.0):
    return torch.empty(*shape, device="cuda").normal_(0.0, scale, generator=source)


def _expert_ids(case, source):
    """k different groups per token, some groups far more popular than others; padded tokens carry -1."""
    tokens, groups = case["tokens"], case["groups"]
    popularity = _normal(source, 1, groups, scale=0.7)
    logits = _normal(source, tokens, groups) + popularity
    value, ids = torch.topk(logits, min(case["top"], groups), dim=1)
    if ids.shape[1] < case["top"]:           # fewer groups than picks: the last one again
        ids = torch.cat([ids, ids[:, -1:].expand(-1, case["top"] - ids.shape[1])], dim=1)
        value = torch.cat([value, value[:, -1:].expand(-1, case["top"] - value.shape[1])], dim=1)
    padded = torch.rand(tokens, 1, device="cuda", generator=source) < case["padding"]
    return torch.where(padded, torch.full_like(ids, -1), ids).contiguous(), torch.softmax(value, dim=1)


def _request_ids(case, source):
    """Packed requests of uneven length, each with one adapter or, for a share of them, none."""
    tokens, requests = case["tokens"], case["requests"]
    share = torch.rand(requests, device="cuda", generator=source) + 0.1
    edge = (torch.cumsum(share, 0) / share.sum() * (tokens - requests)).long() + torch.arange(1, requests + 1, device="cuda")
    edge[-1] = tokens
    request = torch.searchsorted(edge, torch.arange(tokens, device="cuda"), right=True)
    adapter = torch.randint(0, case["groups"], (requests,), device="cuda", generator=source)
    none = torch.rand(requests, device="cuda", generator=source) < case["padding"]
    return torch.where(none, torch.full_like(adapter, -1), adapter)[request].contiguous()


def _inputs(case, seed):
    source = torch.Generator(device="cuda")
    source.manual_seed(seed)
    op, tokens, groups = case["op"], case["tokens"], case["groups"]
    made = {}
    if op == "adapters":
        width, outputs, rank = case["width"], case["outputs"], case["rank"]
        made["ids"] = _request_ids(case, source)
        made["x"] = _normal(source, tokens, width).bfloat16()
        made["y"] = _normal(source, tokens, outputs).bfloat16()
        made["down"] = _normal(source, groups, rank, width, scale=width ** -0.5).bfloat16()
        made["up"] = _normal(source, groups, outputs, rank, scale=rank ** -0.5).bfloat16()
        made["scale"] = 0.5 + torch.rand(groups, device="cuda", generator=source)
        if case["train"]:
            made["grad"] = _normal(source, tokens, outputs, scale=0.1).bfloat16()
        return made
    made["ids"], made["weight"] = _expert_ids(case, source)
    entries = made["ids"].numel()
    if op == "combine":
        made["y"] = _normal(source, entries, case["width"]).bfloat16()
        if case["train"]:
            made["grad"] = _normal(source, tokens, case["width"], scale=0.1).bfloat16()
    elif op == "experts":
        made["x"] = _normal(source, tokens, case["width"]).bfloat16()
        made["w"] = torch.empty(groups, case["outputs"], case["width"], device="cuda", dtype=torch.bfloat16).normal_(0.0, 0.02, generator=source)
        if case["train"]:
            made["grad"] = _normal(source, entries, case["outputs"], scale=0.1).bfloat16()
    elif op == "experts-int8":
        made["x"] = torch.randint(-127, 128, (tokens, case["width"]), device="cuda", dtype=torch.int8, generator=source)
        made["w"] = torch.randint(-127, 128, (groups, case["outputs"], case["width"]), device="cuda", dtype=torch.int8, generator=source)
        made["scale_x"] = 0.01 + 0.02 * torch.rand(tokens, device="cuda", generator=source)
        made["scale_w"] = 0.0002 + 0.0003 * torch.rand(groups, case["outputs"], device="cuda", generator=source)
    return made


def _plain_groups(ids, groups):
    flat = ids.reshape(-1)
    key = torch.where((flat < 0) | (flat >= groups), torch.full_like(flat, groups), flat)
    order = torch.sort(key, stable=True).indices
    counts = (key.unsqueeze(0) == torch.arange(groups, device=key.device).unsqueeze(1)).sum(1)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=key.device), torch.cumsum(counts, 0)])
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    return order, offsets, place


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["op"] != "group":        # the plan of the step: made once, used by every product of the layer or model
        if own:
            import entropack_amd as ep
            state["groups"] = ep.group_rows(state["ids"], case["groups"])
        else:
            order, offsets, place = _plain_groups(state["ids"], case["groups"])
            state.update(order=order, place=place, edges=offsets.tolist())
    if own and case.get("train"):
        for name in {"combine": ("y", "weight"), "experts": ("x", "w"), "adapters": ("x", "down", "up")}[case["op"]]:
            state[name].requires_grad_(True)
    return state


# ---- the passes ----------------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    import entropack_amd as ep
    case = state["case"]
    op = case["op"]
    if op == "group":
        groups = ep.group_rows(state["ids"], case["groups"])
        return {"order": groups.order, "offsets": groups.offsets, "place": groups.place}
    groups = state["groups"]
    if op == "combine":
        out = ep.combine_rows(state["y"], groups, state["weight"])
        if not case["train"]:
            return {"out": out}
        grad_y, grad_weight = torch.autograd.grad(out, (state["y"], state["weight"]), state["grad"])
        return {"out": out.detach(), "grad_y": grad_y, "grad_weight": grad_weight}
    if op == "experts":
        out = ep.grouped_linear(state["x"], state["w"], groups)
        if not case["train"]:
            return {"out": out}
        grad_x, grad_w = torch.autograd.grad(out, (state["x"], state["w"]), state["grad"])
        return {"out": out.detach(), "grad_x": grad_x, "grad_w": grad_w}
    if op == "experts-int8":
        return {"out": ep.grouped_int8_linear(state["x"], state["w"], groups, state["scale_x"], state["scale_w"], out_dtype=torch.bfloat16)}
    out = ep.low_rank_update(state["y"], state["x"], state["down"], state["up"], groups, state["scale"])
    if not case["train"]:
        return {"out": out}
    grad_x, grad_down, grad_up = torch.autograd.grad(out, (state["x"], state["down"], state["up"]), state["grad"])
    return {"out": out.detach(), "grad_x": grad_x, "grad_down": grad_down, "grad_up": grad_up}


def _run_plain(state):
    case = state["case"]
    op = case["op"]
    if op == "group":
        return {name: value.int() for name, value in zip(("order", "offsets", "place"), _plain_groups(state["ids"], case["groups"]))}
    order, place, edges = state["order"], state["place"], state["edges"]
    spans = [(g, edges[g], edges[g + 1]) for g in range(case["groups"]) if edges[g + 1] > edges[g]]
    if op == "combine":
        top = case["top"]
        kept = (place < edges[-1]).reshape(-1, top)
        weight = torch.where(kept, state["weight"], torch.zeros_like(state["weight"]))
        picked = torch.where(kept.unsqueeze(2), state["y"][place].reshape(-1, top, case["width"]).float(), torch.zeros((), device=place.device))
        out = {"out": (picked * weight.unsqueeze(2)).sum(1).bfloat16()}
        if case["train"]:
            grad = state["grad"].float()
            out["grad_y"] = torch.empty_like(state["y"])
            out["grad_y"][place] = (weight.unsqueeze(2) * grad.unsqueeze(1)).reshape(-1, case["width"]).bfloat16()
            out["grad_weight"] = (picked * grad.unsqueeze(1)).sum(2)
        return out
    if op == "experts":
        x, w = state["x"], state["w"]
        source = order // case["top"]
        y = torch.zeros(order.numel(), case["outputs"], device=x.device)
        for g, first, last in spans:
            y[first:last] = x[source[first:last]].float() @ w[g].float().t()
        out = {"out": y.bfloat16()}
        if case["train"]:
            grad_rows = torch.zeros(order.numel(), case["width"], device=x.device)
            out["grad_w"] = torch.zeros_like(w)
            for g, first, last in spans:
                grad = state["grad"][first:last].float()
                grad_rows[first:last] = grad @ w[g].float()
                out["grad_w"][g] = (grad.t() @ x[source[first:last]].float()).bfloat16()
            out["grad_x"] = grad_rows[place].reshape(-1, case["top"], case["width"]).sum(1).bfloat16()
        return out
    if op == "experts-int8":
        source = order // case["top"]
        y = torch.zeros(order.numel(), case["outputs"], device=order.device)
        for g, first, last in spans:            # the integer sums pass 2^24: taken in 64 bits
            sums = (state["x"][source[first:last]].double() @ state["w"][g].double().t()).float()
            y[first:last] = sums * state["scale_x"][source[first:last]].unsqueeze(1) * state["scale_w"][g]
        return {"out": y.bfloat16()}
    x, down, up, scale = state["x"], state["down"], state["up"], state["scale"]
    y = state["y"].float()
    grads = {}
    if case["train"]:
        grads = {"grad_x": torch.zeros_like(x), "grad_down": torch.zeros_like(down), "grad_up": torch.zeros_like(up)}
    for g, first, last in spans:
        rows = order[first:last]
        narrow = x[rows].float() @ down[g].float().t()
        y[rows] += scale[g] * (narrow @ up[g].float().t())
        if case["train"]:
            grad = state["grad"][rows].float()
            grad_narrow = scale[g] * (grad @ up[g].float())
            grads["grad_x"][rows] = (grad_narrow @ down[g].float()).bfloat16()
            grads["grad_down"][g] = (grad_narrow.t() @ x[rows].float()).bfloat16()
            grads["grad_up"][g] = (scale[g] * (grad.t() @ narrow)).bfloat16()
    return {"out": y.bfloat16(), **grads}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    op, groups = case["op"], case["groups"]
    if op == "group":            # whole numbers: the plain form's are the definition
        return None
    made = _inputs(case, seed)
    ids = made["ids"].reshape(-1)
    members = [torch.nonzero(ids == g).reshape(-1) for g in range(groups)]
    if op == "adapters":
        x, out = made["x"].double(), made["y"].double()
        grads = {}
        if case["train"]:
            grads = {"grad_x": torch.zeros_like(x), "grad_down": made["down"].double(), "grad_up": made["up"].double()}
        for g, rows in enumerate(members):
            down, up, scale = made["down"][g].double(), made["up"][g].double(), made["scale"][g].double()
            out[rows] += scale * torch.mm(torch.mm(x[rows], down.t()), up.t())
            if case["train"]:
                grad = made["grad"][rows].double()
                grads["grad_x"][rows] = scale * torch.mm(torch.mm(grad, up), down)
                grads["grad_down"][g] = scale * torch.mm(torch.mm(up.t(), grad.t()), x[rows])
                grads["grad_up"][g] = scale * torch.mm(grad.t(), torch.mm(x[rows], down.t()))
        return {"out": out, **grads}
    top, entries = case["top"], ids.numel()
    token = torch.arange(entries, device="cuda") // top
    first, start = torch.zeros(entries, dtype=torch.int64, device="cuda"), 0       # the place of every entry
    for rows in members + [torch.nonzero((ids < 0) | (ids >= groups)).reshape(-1)]:
        first[rows] = start + torch.arange(rows.numel(), device="cuda")
        start += rows.numel()
    if op == "combine":
        out = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")
        weight = made["weight"].reshape(-1).double()
        result = {"out": out}
        if case["train"]:
            result["grad_y"] = torch.zeros(entries, case["width"], dtype=torch.float64, device="cuda")
            result["grad_weight"] = torch.zeros(entries, dtype=torch.float64, device="cuda")
        for j in range(top):
            rows = torch.arange(j, entries, top, device="cuda")
            rows = rows[(ids[rows] >= 0) & (ids[rows] < groups)]
            values = made["y"][first[rows]].double()
            out[token[rows]] += weight[rows].unsqueeze(1) * values
            if case["train"]:
                grad = made["grad"][token[rows]].double()
                result["grad_y"][first[rows]] = weight[rows].unsqueeze(1) * grad
                result["grad_weight"][rows] = torch.einsum("rw,rw->r", grad, values)
        if case["train"]:
            result["grad_weight"] = result["grad_weight"].reshape(-1, top)
        return result
    x = made["x"].double()
    if op == "experts-int8":
        x = x * made["scale_x"].double().unsqueeze(1)
    out = torch.zeros(entries, case["outputs"], dtype=torch.float64, device="cuda")
    result = {"out": out}
    if case.get("train"):
        result["grad_x"] = torch.zeros_like(x)
        result["grad_w"] = torch.zeros(made["w"].shape, dtype=torch.float64, device="cuda")
    for g, rows in enumerate(members):
        if rows.numel() == 0:
            continue
        w = made["w"][g].double()
        if op == "experts-int8":
            w = w * made["scale_w"][g].double().unsqueeze(1)
        out[first[rows]] = torch.mm(x[token[rows]], w.t())
        if case.get("train"):
            grad = made["grad"][first[rows]].double()
            result["grad_x"].index_add_(0, token[rows], torch.mm(grad, w))
            result["grad_w"][g] = torch.mm(grad.t(), x[token[rows]])
    return result
