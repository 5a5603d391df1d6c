"""The operators on rows chosen by an index, as cases to time and to check.

A model meets such rows twice: where tokens (or the nodes of a graph) become
vectors, and where a mixture layer sends each token to a few experts and brings
the results back.  The operators are

    embed         rows of a table, looked up and scaled
    embed_grad    its gradient: the rows' sums by token, dense over the table
    route         softmax of the router's scores and the top_k experts of each token
    route_grad    its gradient
    dispatch      tokens copied into the order of their experts
    combine       the experts' rows brought back and summed with weights (without
                  weights: the gradient of dispatch)
    combine_grad  the gradient of combine, for the rows and for the weights

Every case is one of them with its sizes.  ``run`` computes it with elementary
torch operations, or, where ``own`` is set, through the package's entry points.
An index outside its range is an empty place (a padded token, an expert that
another GPU holds): it gives a row of zeros and takes no gradient, or is dropped.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}

MAX_ELEMENTS = 1 << 27  # of the rows moved or of the table, in a drawn case


def listed():
    """The listed cases: the smallest calls, ordinary ones, the largest and ragged ones."""
    return [
        # One step of a server that answers 16 requests: one token each, a bf16 table, scaled by the root of the width.
        dict(name="embed step", op="embed", tokens=16, rows=32768, width=4096, dtype="bf16", index="i64", scale=64.0, empty=0.0),
        # A training batch of 16384 tokens over a large vocabulary, a few of them padding.
        dict(name="embed batch", op="embed", tokens=16384, rows=131072, width=4096, dtype="bf16", index="i32", scale=1.0, empty=0.05),
        # The same batch's gradient, kept in 32 bits for the optimizer, as wide as half the table above.
        dict(name="embed_grad batch", op="embed_grad", tokens=16384, rows=131072, width=2048, dtype="bf16", out="f32", index="i32",
             scale=1.0, empty=0.05),
        # Ragged everything: rows that begin at odd addresses, a batch and a table that no tile divides.
        dict(name="embed_grad ragged", op="embed_grad", tokens=50003, rows=10007, width=515, dtype="f16", out="f16", index="i64",
             scale=22.5, empty=0.1),
        # Routing while serving: a few dozen tokens, scores in 16 bits (ties are common), weights that keep their share of all experts.
        dict(name="route step", op="route", tokens=32, experts=64, top_k=6, dtype="bf16", normalize=False, masked=0),
        # Routing a training batch over many experts; a few of them are switched off by scores of -inf.
        dict(name="route batch", op="route", tokens=16384, experts=256, top_k=8, dtype="f32", normalize=True, masked=3),
        # Its gradient, where the weights are shares of all experts: dense over the scores.
        dict(name="route_grad batch", op="route_grad", tokens=16384, experts=256, top_k=8, dtype="f32", normalize=False, masked=3),
        # A serving step's tokens to the experts of one GPU out of two.
        dict(name="dispatch step", op="dispatch", tokens=32, experts=64, top_k=6, width=2048, dtype="bf16", index="i32", align=1, shards=2),
        # A training batch, each expert's rows begun at a tile of 128.
        dict(name="dispatch batch", op="dispatch", tokens=8192, experts=64, top_k=8, width=4096, dtype="bf16", index="i32", align=128,
             shards=1),
        # Back again with the weights, and the layer's residual added on the way.
        dict(name="combine batch", op="combine", tokens=8192, experts=64, top_k=8, width=4096, dtype="bf16", weighted=True, add=True,
             align=128, shards=1),
        # The gradient of dispatch on a ragged layer in 32 bits, half of the experts elsewhere.
        dict(name="combine ragged", op="combine", tokens=3001, experts=13, top_k=3, width=1111, dtype="f32", weighted=False, add=False,
             align=1, shards=2),
        # The gradient of combine for a training batch.
        dict(name="combine_grad batch", op="combine_grad", tokens=8192, experts=64, top_k=8, width=2048, dtype="bf16", align=128, shards=1),
    ]


def draw(rng):
    """One more case: an operator, and sizes spread over the logarithm of their ranges."""
    def log(low, high):
        return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))

    op = rng.choice(["embed", "embed_grad", "route", "route_grad", "dispatch", "combine", "combine_grad"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op in ("embed", "embed_grad"):
        width = log(16, 8192)
        if rng.random() < 0.6:
            width = (width + 7) // 8 * 8
        case = dict(op=op, tokens=log(1, min(131072, MAX_ELEMENTS // width)), rows=log(100, min(262144, MAX_ELEMENTS // width)),
                    width=width, dtype=dtype)
        if op == "embed_grad":
            case["out"] = rng.choice([dtype, "f32"])
        return dict(case, index=rng.choice(["i32", "i64"]), scale=rng.choice([1.0, 0.25, round(math.sqrt(width), 3)]),
                    empty=rng.choice([0.0, 0.05, 0.5]))
    experts = log(2, 384)
    top_k = min(experts, rng.choice([1, 2, 3, 4, 6, 8, 10]))
    if op in ("route", "route_grad"):
        return dict(op=op, tokens=log(1, 16384), experts=experts, top_k=top_k, dtype=dtype, normalize=rng.random() < 0.5,
                    masked=rng.choice([0, 0, 1, experts // 2]))
    width = log(16, 8192)
    if rng.random() < 0.6:
        width = (width + 7) // 8 * 8
    # (at the most as many rows as the largest listed batch has)
    case = dict(op=op, tokens=log(1, min(16384, MAX_ELEMENTS // width // top_k)), experts=experts, top_k=top_k, width=width, dtype=dtype,
                align=rng.choice([1, 1, 16, 128]), shards=rng.choice([1, 1, 2, 4]))
    if op == "dispatch":
        case["index"] = rng.choice(["i32", "i64"])
    if op == "combine":
        case.update(weighted=rng.random() < 0.7, add=rng.random() < 0.4)
    if case["align"] * experts * width > MAX_ELEMENTS // 2:
        case["align"] = 1
    return case


def dispatched_rows(slots, experts, align):
    """Rows that the tokens of ``slots`` places can fill at the most when every expert begins at a multiple of ``align``."""
    return (slots + min(experts, slots) * (align - 1)) // align * align


# ---------------------------------------------------------------------------------------------- inputs

def _tokens(case, gen):
    """Tokens as text has them: the r-th most frequent about 1/r as often as the first, spread over the table, some empty (-1)."""
    n, rows = case["tokens"], case["rows"]
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    rank = torch.exp(u * math.log(rows + 1.0)).long().sub_(1).clamp_(0, rows - 1)
    token = (rank * 7919 + 13) % rows if rows % 7919 else rank
    if case["empty"]:
        token = torch.where(torch.rand(n, generator=gen, device="cuda") < case["empty"], torch.full_like(token, -1), token)
    return token.to(torch.int32 if case["index"] == "i32" else torch.int64)


def _scores(case, experts, gen):
    """Router scores: some experts are more popular than others, ``masked`` of them are off."""
    s = torch.randn(case["tokens"], experts, generator=gen, device="cuda") + 0.7 * torch.randn(experts, generator=gen, device="cuda")
    if case.get("masked"):
        s[:, torch.randperm(experts, generator=gen, device="cuda")[: case["masked"]]] = -math.inf
    return s


def _chosen(case, gen):
    """Experts of each token as this GPU numbers them (those of other GPUs lie outside [0, experts)), and weights that sum to one."""
    every = case["experts"] * case["shards"]
    scores = _scores(case, every, gen)
    value, expert = torch.sort(scores, dim=1, descending=True, stable=True)
    k = case["top_k"]
    return expert[:, :k].contiguous(), torch.softmax(value[:, :k], 1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(DTYPES[case["dtype"]])

    state = dict(case=case)
    if op in ("embed", "embed_grad"):
        state["tokens"] = _tokens(case, gen)
        if op == "embed":
            state["table"] = normal(case["rows"], case["width"], std=0.02)
        else:
            state["grad"] = normal(case["tokens"], case["width"], std=0.01)
        return state
    if op in ("route", "route_grad"):
        state["scores"] = _scores(case, case["experts"], gen).to(DTYPES[case["dtype"]])
        if op == "route_grad":
            state["weights"], state["chosen"] = _route(state["scores"], case["top_k"], case["normalize"])
            state["grad"] = torch.randn(case["tokens"], case["top_k"], generator=gen, device="cuda")
        return state
    chosen, weights = _chosen(case, gen)
    rows = dispatched_rows(chosen.numel(), case["experts"], case["align"])
    if op == "dispatch":
        state["chosen"] = chosen.to(torch.int32 if case["index"] == "i32" else torch.int64)
        state["x"] = normal(case["tokens"], case["width"])
        state["rows"] = torch.zeros(rows, case["width"], dtype=DTYPES[case["dtype"]], device="cuda")
        return state
    position, offsets, counts = _order(chosen, case["experts"], case["align"])
    state.update(position=position, offsets=offsets, counts=counts, y=normal(rows, case["width"]))
    if op == "combine":
        state["weights"] = weights if case["weighted"] else None
        state["add"] = normal(case["tokens"], case["width"]) if case["add"] else None
    else:
        state["weights"] = weights
        state["grad"] = normal(case["tokens"], case["width"])
        state["grad_rows"] = torch.zeros_like(state["y"])
    if own:
        import powersparse_b200 as psb
        state["plan"] = psb.DispatchPlan(position, offsets, counts)
    return state


# ---------------------------------------------------------------------------------------------- plain forms

def _embed(table, tokens, scale):
    inside = (tokens >= 0) & (tokens < table.shape[0])
    row = table[torch.where(inside, tokens, 0).long()].float() * scale
    return torch.where(inside[:, None], row, 0.0).to(table.dtype)


def _embed_grad(grad, tokens, rows, scale, dtype):
    inside = (tokens >= 0) & (tokens < rows)
    out = torch.zeros(rows + 1, grad.shape[1], device=grad.device)
    out.index_add_(0, torch.where(inside, tokens, rows).long(), grad.float() * scale)
    return out[:rows].to(dtype)


def _route(scores, top_k, normalize):
    x = scores.float()
    value, expert = torch.sort(x, dim=1, descending=True, stable=True)  # stable: of equal scores the lowest index is first
    top = value[:, :1]
    e = torch.exp(value - torch.where(top == -math.inf, 0.0, top))
    total = (e[:, :top_k] if normalize else e).sum(1, keepdim=True)
    value, e = value[:, :top_k], e[:, :top_k]
    on = value > -math.inf
    return torch.where(on, e / total, 0.0), torch.where(on, expert[:, :top_k], -1).int()


def _route_grad(grad, scores, chosen, weights, normalize):
    on = chosen >= 0
    g = torch.where(on, grad, 0.0)
    inner = (g * weights).sum(1, keepdim=True)
    out = torch.zeros(scores.shape[0], scores.shape[1] + 1, device=scores.device)
    at = torch.where(on, chosen, scores.shape[1]).long()
    if normalize:
        out.scatter_(1, at, weights * (g - inner))
        return out[:, :-1].to(scores.dtype)
    x = scores.float()
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(1, keepdim=True)
    p = e / torch.where(total > 0, total, 1.0)
    out.scatter_(1, at, g)
    return (p * (out[:, :-1] - inner)).to(scores.dtype)


def _order(chosen, experts, align):
    """Place of each (token, choice) among the rows in expert order (-1: dropped), where each expert begins, how many rows it has."""
    flat = chosen.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    sorted_key, slot = torch.sort(key, stable=True)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device).index_add_(0, key, torch.ones_like(key))
    first = torch.cumsum(counts, 0) - counts
    padded = (counts + align - 1) // align * align
    begin = torch.cumsum(padded, 0) - padded
    place = begin[sorted_key] + torch.arange(len(flat), device=flat.device) - first[sorted_key]
    position = torch.empty_like(key)
    position[slot] = torch.where(sorted_key < experts, place, -1)
    return position.view(chosen.shape).int(), begin.int(), counts[:-1].int()


def _dispatch(x, chosen, experts, align, rows):
    position, offsets, counts = _order(chosen, experts, align)
    out = torch.zeros(rows + 1, x.shape[1], dtype=x.dtype, device=x.device)
    at = torch.where(position >= 0, position, rows).long()
    for j in range(chosen.shape[1]):
        out[at[:, j]] = x
    return out[:rows], position, offsets, counts


def _combine(y, position, weights, add):
    out = torch.zeros(position.shape[0], y.shape[1], device=y.device) if add is None else add.float()
    for j in range(position.shape[1]):
        at = position[:, j]
        row = y[torch.where(at >= 0, at, 0).long()].float()
        if weights is not None:
            row = row * weights[:, j: j + 1]
        out = out + torch.where((at >= 0)[:, None], row, 0.0)
    return out.to(y.dtype)


def _combine_grad(grad, y, position, weights):
    rows = y.shape[0]
    grad_y = torch.zeros(rows + 1, y.shape[1], dtype=y.dtype, device=y.device)
    grad_weights = torch.zeros_like(weights)
    g = grad.float()
    for j in range(position.shape[1]):
        at = position[:, j]
        on = at >= 0
        grad_y[torch.where(on, at, rows).long()] = (g * weights[:, j: j + 1]).to(y.dtype)
        grad_weights[:, j] = torch.where(on, (g * y[torch.where(on, at, 0).long()].float()).sum(1), 0.0)
    return grad_y[:rows], grad_weights


def run(state):
    """One pass through the operator of the state's case."""
    case = state["case"]
    op = case["op"]
    if own:
        import powersparse_b200 as psb
        if op == "embed":
            return psb.embedding(state["table"], state["tokens"], scale=case["scale"])
        if op == "embed_grad":
            return psb.embedding_grad(state["grad"], state["tokens"], case["rows"], scale=case["scale"], dtype=DTYPES[case["out"]])
        if op == "route":
            return tuple(psb.route(state["scores"], case["top_k"], normalize=case["normalize"]))
        if op == "route_grad":
            return psb.route_grad(state["grad"], state["scores"], state["weights"], state["chosen"], normalize=case["normalize"])
        if op == "dispatch":
            rows, plan = psb.dispatch(state["x"], state["chosen"], case["experts"], align=case["align"], out=state["rows"])
            return rows, plan.position, plan.offsets, plan.counts
        if op == "combine":
            return psb.combine(state["y"], state["plan"], weights=state["weights"], add=state["add"])
        return tuple(psb.combine_grad(state["grad"], state["y"], state["plan"], state["weights"], out=state["grad_rows"]))
    if op == "embed":
        return _embed(state["table"], state["tokens"], case["scale"])
    if op == "embed_grad":
        return _embed_grad(state["grad"], state["tokens"], case["rows"], case["scale"], DTYPES[case["out"]])
    if op == "route":
        return _route(state["scores"], case["top_k"], case["normalize"])
    if op == "route_grad":
        return _route_grad(state["grad"], state["scores"], state["chosen"], state["weights"], case["normalize"])
    if op == "dispatch":
        return _dispatch(state["x"], state["chosen"], case["experts"], case["align"], state["rows"].shape[0])
    if op == "combine":
        return _combine(state["y"], state["position"], state["weights"], state["add"])
    return _combine_grad(state["grad"], state["y"], state["position"], state["weights"])


# ---------------------------------------------------------------------------------------------- the definition in 64 bits

def _exact_order(chosen, experts, align):
    flat = chosen.reshape(-1).cpu().long()
    position = torch.full_like(flat, -1)
    offsets, counts, at = [0], [], 0
    for e in range(experts):
        slots = (flat == e).nonzero()[:, 0]
        position[slots] = at + torch.arange(len(slots))
        counts.append(len(slots))
        at += -(-len(slots) // align) * align
        offsets.append(at)
    return tuple(t.to(chosen.device) for t in (position.view(chosen.shape).int(), torch.tensor(offsets, dtype=torch.int32),
                                               torch.tensor(counts, dtype=torch.int32)))


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "embed":
        table, tokens = state["table"], state["tokens"].long()
        out = torch.zeros(len(tokens), table.shape[1], dtype=torch.float64, device="cuda")
        full = (tokens > -1).nonzero()[:, 0]
        out[full] = table[tokens[full]].double() * case["scale"]
        return out
    if op == "embed_grad":
        tokens = state["tokens"].long()
        full = (tokens > -1).nonzero()[:, 0]
        token, by = torch.sort(tokens[full], stable=True)
        out = torch.zeros(case["rows"], case["width"], dtype=torch.float64, device="cuda")
        unique, count = torch.unique_consecutive(token, return_counts=True)
        for begin in range(0, case["width"], 256):
            part = state["grad"][full[by], begin: begin + 256].double()
            run_of = torch.repeat_interleave(torch.arange(len(unique), device="cuda"), count)
            sums = torch.zeros(len(unique), part.shape[1], dtype=torch.float64, device="cuda")
            sums.scatter_add_(0, run_of[:, None].expand_as(part), part)
            out[unique, begin: begin + 256] = sums * case["scale"]
        return out
    if op in ("route", "route_grad"):
        x = state["scores"].double()
        off = x == -math.inf
        k = case["top_k"]
        left, chosen = x.clone(), []
        index = torch.arange(case["experts"], device="cuda")
        for _ in range(k):
            best = left.max(1).values
            first = torch.where((left == best[:, None]) & ~torch.isinf(left), index, case["experts"]).amin(1)
            chosen.append(torch.where(first < case["experts"], first, -1))
            left = left.masked_fill(index == first[:, None], -math.inf)
        chosen = torch.stack(chosen, 1)
        among = (index[None, None] == chosen[:, :, None]).any(1) if case["normalize"] else ~off
        e = torch.where(among, torch.exp(x - x.masked_fill(off, -1e300).amax(1, keepdim=True)), 0.0)
        p = e / e.sum(1, keepdim=True).clamp_min(1e-300)
        if op == "route":
            return torch.where(chosen >= 0, p.gather(1, chosen.clamp_min(0)), 0.0), chosen.int()
        g = torch.zeros_like(p)
        for j in range(k):
            g += (index == chosen[:, j: j + 1]) * state["grad"][:, j: j + 1].double()
        return p * (g - (g * p).sum(1, keepdim=True))
    if op == "dispatch":
        position, offsets, counts = _exact_order(state["chosen"], case["experts"], case["align"])
        out = torch.zeros(state["rows"].shape, dtype=torch.float64, device="cuda")
        token, choice = (position >= 0).nonzero(as_tuple=True)
        out[position[token, choice].long()] = state["x"][token].double()
        return out, position, offsets, counts
    position = state["position"]
    token, choice = (position >= 0).nonzero(as_tuple=True)
    at = position[token, choice].long()
    if op == "combine":
        y = torch.cat([state["y"], torch.zeros_like(state["y"][:1])])
        w = torch.ones(position.shape, dtype=torch.float64, device="cuda") if state["weights"] is None else state["weights"].double()
        out = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")
        for j in range(case["top_k"]):  # a position of -1 takes the last row, of zeros
            out.addcmul_(y[position[:, j].long()].double(), w[:, j: j + 1])
        return out if state["add"] is None else out + state["add"].double()
    grad_y = torch.zeros(state["y"].shape, dtype=torch.float64, device="cuda")
    grad_weights = torch.zeros(position.shape, dtype=torch.float64, device="cuda")
    for begin in range(0, len(token), 8192):
        t, j, a = (v[begin: begin + 8192] for v in (token, choice, at))
        g = state["grad"][t].double()
        grad_y[a] = state["weights"][t, j].double()[:, None] * g
        grad_weights[t, j] = torch.einsum("ij,ij->i", g, state["y"][a].double())
    return grad_y, grad_weights


# ---------------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    op, t = case["op"], case["tokens"]
    if op in ("embed", "embed_grad"):
        full = t * (1.0 - case["empty"])
        index = t * (4 if case["index"] == "i32" else 8)
        row = case["width"] * BYTES[case["dtype"]]
        if op == "embed_grad":
            return dict(bytes=full * row + index + case["rows"] * case["width"] * BYTES[case["out"]], flops=full * case["width"])
        # Distinct rows expected: rank r is drawn with probability log((r + 2) / (r + 1)) / log(rows + 1).
        r = torch.arange(case["rows"], dtype=torch.float64)
        distinct = float((1.0 - torch.exp(full * torch.log1p(-torch.log((r + 2) / (r + 1)) / math.log(case["rows"] + 1.0)))).sum())
        return dict(bytes=distinct * row + index + t * row, flops=full * case["width"])
    k, size = case["top_k"], BYTES[case["dtype"]]
    if op in ("route", "route_grad"):
        e = case["experts"]
        scores = t * e * size
        if op == "route":
            return dict(bytes=scores + t * k * 8, flops=4 * t * e)
        return dict(bytes=(1 if case["normalize"] else 2) * scores + t * k * 12, flops=t * (2 * k if case["normalize"] else 6 * e))
    row = case["width"] * size
    slots = t * k / case["shards"]
    if op == "dispatch":
        return dict(bytes=t * row + slots * row + t * k * ((4 if case["index"] == "i32" else 8) + 4), flops=0)
    if op == "combine":
        return dict(bytes=slots * row + (2 if case["add"] else 1) * t * row + t * k * (8 if case["weighted"] else 4),
                    flops=2 * slots * case["width"])
    return dict(bytes=t * row + 2 * slots * row + t * k * 12, flops=3 * slots * case["width"])
