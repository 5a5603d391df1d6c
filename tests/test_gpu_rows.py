"""GPU tests: the operators on rows chosen by an index against their formulas in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of FP32, half(T) half a step of the
stored type relative to the value (finfo.eps / 2), tiny(T) half of its smallest
subnormal.  A sum of m terms in FP32, in whatever order, is off by at most
m * u * sum |terms| to first order (products included); the factor 1.01 covers the
higher orders (m * u < 1e-2 in every test).
"""
import math
import os
import subprocess
import sys
import threading

import pytest
import torch

import powersparse_b200 as psb
import powersparse_b200.torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
U = 2.0 ** -24


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def check(got, want, slack=0.0, tag=""):
    """|got - want| <= half a step of got's type at want + slack (the FP32 part, absolute)."""
    assert got.shape == want.shape and want.dtype == torch.float64
    got64 = got.double()
    room = 1.01 * (want.abs() * half(got.dtype) + slack * (1 + half(got.dtype))) + tiny(got.dtype)
    bad = ~((got64 - want).abs() <= room)
    assert not bad.any(), (tag, int(bad.sum()), bad.nonzero()[:3].tolist(), got64[bad][:3].tolist(), want[bad][:3].tolist())


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def strided(t, extra, offset=0):
    """t's values in a tensor whose rows are `extra` elements further apart, begun at element `offset`."""
    rows, width = t.shape
    buf = torch.full((rows * (width + extra) + offset + 1,), math.nan, device="cuda", dtype=t.dtype)
    view = buf[offset: offset + rows * (width + extra)].view(rows, width + extra)[:, :width]
    view.copy_(t)
    return view


# ------------------------------------------------------------------------------------ embedding

WIDTHS = [1, 2, 7, 8, 33, 128, 515, 1024, 4104]


def embedding64(table, tokens, scale):
    t = tokens.reshape(-1).long()
    inside = (t >= 0) & (t < table.shape[0])
    out = table.double()[t.clamp(0, table.shape[0] - 1)] * scale
    return out.masked_fill(~inside[:, None], 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_embedding(dtype, width):
    g = gen(width)
    for n, rows, index in ((1, 1, torch.int64), (5, 3, torch.int32), (257, 1000, torch.int64)):
        table = randn(g, rows, width, dtype=dtype)
        tokens = torch.randint(-2, rows + 2, (n,), generator=g, device="cuda").to(index)
        scale = 22.5
        want = embedding64(table, tokens, torch.tensor(scale, dtype=F32).double().item())
        check(psb.embedding(table, tokens, scale), want, want.abs() * U)
        assert torch.equal(psb.embedding(table, tokens).double(), embedding64(table, tokens, 1.0))  # a copy is exact
        out = strided(torch.zeros(n, width, device="cuda", dtype=dtype), 3)
        psb.embedding(strided(table, 5, 1), tokens, scale, out=out)
        check(out, want, want.abs() * U)


def test_embedding_shapes_and_far_tokens():
    table = randn(gen(0), 10, 24, dtype=BF16)
    tokens = torch.tensor([[0, 9, 2**40], [-2**40, 2**32 + 1, 3]], device="cuda")  # 2^32 + 1 is not row 1
    out = psb.embedding(table, tokens)
    assert out.shape == (2, 3, 24)
    assert torch.equal(out.view(6, 24).double(), embedding64(table, tokens, 1.0))
    assert psb.embedding(table, tokens[:0]).shape == (0, 3, 24)
    # What stands in rows that no token names has no effect, inf and NaN included.
    table[1:3] = math.nan
    table[5] = math.inf
    assert torch.equal(psb.embedding(table, tokens).view(6, 24)[[0, 1, 5]], table[[0, 9, 3]])
    assert not psb.embedding(table, tokens).isnan().any()


def test_embedding_offsets_pass_32_bits():
    rows, width = 600_000, 4096  # 2.4e9 elements
    table = torch.empty(rows, width, device="cuda", dtype=BF16)
    tokens = torch.tensor([0, rows - 1, 524_288, 524_287, rows], device="cuda")
    for i, t in enumerate(tokens[:-1].tolist()):
        table[t] = i + 1
    out = psb.embedding(table, tokens)
    assert out.double().mean(1).tolist() == [1, 2, 3, 4, 0]
    grad = torch.ones(5, width, device="cuda", dtype=BF16)
    psb.embedding_grad(grad, tokens, rows, out=table, scale=3.0)
    assert table[tokens[:-1]].double().mean(1).tolist() == [3, 3, 3, 3]
    assert table.count_nonzero().item() == 4 * width


def grad64(grad, tokens, rows, scale, padding=None):
    t = tokens.reshape(-1).long()
    on = (t >= 0) & (t < rows) & (t != (-1 if padding is None else padding))
    g = grad.double()[on] * scale
    out = torch.zeros(rows, grad.shape[1], dtype=torch.float64, device="cuda").index_add_(0, t[on], g)
    size = torch.zeros_like(out).index_add_(0, t[on], g.abs())
    many = torch.zeros(rows, dtype=torch.float64, device="cuda").index_add_(0, t[on], torch.ones_like(t[on], dtype=torch.float64))
    return out, size * (many[:, None] + 2) * U


def batch(g, kind, n, rows, index=torch.int64):
    if kind == "one":
        t = torch.full((n,), rows // 2, device="cuda")
    elif kind == "empty":
        t = torch.full((n,), -1, device="cuda")
    elif kind == "skewed":
        t = (rows ** torch.rand(n, generator=g, device="cuda")).long() - 1
    elif kind == "distinct":
        t = torch.randperm(rows, generator=g, device="cuda")[:n]
    elif kind == "sorted":
        t = torch.arange(n, device="cuda") * rows // max(n, 1)
    else:
        t = torch.randint(-3, rows + 3, (n,), generator=g, device="cuda")
    return t.to(index)


@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("width", [1, 8, 33, 128, 515, 1032])
def test_embedding_grad(dtype, out, width):
    g = gen(width)
    for kind, n, rows, index in (("any", 1, 1, torch.int32), ("any", 3, 7, torch.int64), ("skewed", 333, 50, torch.int32),
                                 ("distinct", 200, 257, torch.int64), ("one", 1000, 300, torch.int64), ("empty", 64, 20, torch.int32),
                                 ("skewed", 5000, 3000, torch.int64), ("sorted", 4097, 100, torch.int32)):
        tokens, grad = batch(g, kind, n, rows, index), randn(g, n, width, dtype=dtype)
        want, slack = grad64(grad, tokens, rows, 0.75)
        check(psb.embedding_grad(grad, tokens, rows, 0.75, dtype=out), want, slack, (kind, n, rows))
        dst = strided(torch.full((rows, width), 7.0, device="cuda", dtype=out), 2, 1)
        psb.embedding_grad(strided(grad, 3), tokens, rows, 0.75, out=dst)
        check(dst, want, slack, (kind, "strided"))


@pytest.mark.parametrize("kind", ["any", "skewed", "one", "distinct", "sorted", "empty"])
@pytest.mark.parametrize("n,rows", [(31, 9), (65, 5000), (2047, 300), (2048, 40000), (20000, 40000), (70001, 70001),
                                    (16384, 1025), (40000, 3_000_000), (9000, 512), (2049, 1023), (131072, 700_000), (131073, 1_000_000)])
def test_embedding_grad_order_of_large_batches(kind, n, rows):
    g = gen(n + rows)
    if kind == "distinct" and n > rows:
        n = rows
    tokens, grad = batch(g, kind, n, rows), randn(g, n, 16, dtype=BF16)
    want, slack = grad64(grad, tokens, rows, 1.0)
    got = psb.embedding_grad(grad, tokens, rows, dtype=F32)
    check(got, want, slack)
    assert torch.equal(got, psb.embedding_grad(grad, tokens, rows, dtype=F32))  # the same bits again


@pytest.mark.parametrize("n,width", [(2100, 40), (20000, 40), (20000, 1032), (40000, 1032)])
@pytest.mark.parametrize("lengths", [(1, 15, 16, 17), (16, 32, 48), (31, 33, 1), (30, 2, 32, 1), (47, 17, 1), (64, 63, 65, 1), (200, 5), (33,)])
def test_embedding_grad_of_runs_about_the_chunks_borders(n, width, lengths):
    """Runs of every length about one, two and more chunks (of 8 to 64) of the sorted batch, begun at every place in one."""
    g = gen(n)
    runs = torch.tensor(lengths * (n // sum(lengths) + 1), device="cuda")
    tokens = torch.repeat_interleave(torch.arange(len(runs), device="cuda"), runs)[:n]
    tokens = tokens[torch.randperm(n, generator=g, device="cuda")]
    tokens = torch.where(tokens % 5 == 4, tokens + len(runs), tokens)  # some outside
    grad = randn(g, n, width, dtype=BF16)
    want, slack = grad64(grad, tokens, len(runs), 1.0)
    check(psb.embedding_grad(grad, tokens, len(runs), dtype=F32), want, slack)


@pytest.mark.parametrize("n", [100, 3000])
@pytest.mark.parametrize("offset,extra", [(0, 0), (0, 1), (1, 0), (1, 1), (2, 2), (1, 3), (2, 6), (4, 4)])
def test_embedding_grad_in_32_bits_at_every_alignment(n, offset, extra):
    """16-bit rows that allow words while the 32-bit rows of the result begin elsewhere, and the other way round."""
    g = gen(offset)
    for width in (2, 6, 8, 64, 132):
        tokens, grad = batch(g, "skewed", n, 70), randn(g, n, width, dtype=F16)
        want, slack = grad64(grad, tokens, 70, 1.0)
        for a, b in (((0, 0), (extra, offset)), ((extra, offset), (0, 0)), ((2, 2), (extra, offset))):
            dst = strided(torch.full((70, width), 7.0, device="cuda"), *b)
            psb.embedding_grad(strided(grad, *a), tokens, 70, out=dst)
            check(dst, want, slack, (width, a, b))


def test_empty_places_are_plus_zero_whatever_the_scale():
    tokens = torch.tensor([-1, 3, 9], device="cuda")
    for scale in (-1.5, math.inf, math.nan):
        out = psb.embedding(torch.ones(9, 16, device="cuda"), tokens, scale)
        assert (out[[0, 2]].view(torch.int32) == 0).all()


def test_embedding_grad_of_a_large_table_with_rows_apart():
    """The gradient that is cleared in parts (above 144 MiB), in a wider buffer whose other columns stay."""
    g = gen(3)
    tokens, grad = batch(g, "skewed", 5000, 300_000), randn(g, 5000, 130)
    buf = torch.full((300_000, 133), 7.0, device="cuda")
    psb.embedding_grad(grad, tokens, 300_000, out=buf[:, 1:131])
    want, slack = grad64(grad, tokens, 300_000, 1.0)
    check(buf[:, 1:131], want, slack)
    assert (buf[:, 0] == 7).all() and (buf[:, 131:] == 7).all()


def test_embedding_grad_of_a_million_tokens_and_many_passes():
    g = gen(5)
    n, rows = 1_100_000, 5_000_000
    tokens, grad = batch(g, "skewed", n, rows), randn(g, n, 4)
    want, slack = grad64(grad, tokens, rows, 1.0)
    check(psb.embedding_grad(grad, tokens, rows), want, slack)
    rows = 2**31 - 2  # four digit passes; the sums go to the rows that occur, the others stay untouched
    tokens = torch.tensor([3, 7, 3, 2**20, 7, 3, -1, 2**31 - 2, 2**31], device="cuda")
    out = torch.zeros(2**20 + 1, 8, device="cuda")
    lib = psb.load_library()
    s = torch.cuda.current_stream().cuda_stream
    for times in (1, 1000):
        many = tokens.repeat(times)
        out.zero_()
        ws = torch.empty(lib.ps_embedding_grad_workspace(9 * times, rows, 8) + 1, dtype=torch.uint8, device="cuda")
        grad = randn(g, 9 * times, 8)
        assert lib.ps_embedding_grad(grad.data_ptr(), 0, 8, many.data_ptr(), 1, 9 * times, 1.0, -1, 1, out.data_ptr(), 0, 8, rows, 8,
                                     ws.data_ptr(), ws.numel(), s) == psb.PS_OK
        want, slack = grad64(grad, many, 2**20 + 1, 1.0)
        check(out, want, slack)


def test_embedding_grad_padding_accumulate_and_no_tokens():
    g = gen(9)
    tokens, grad = batch(g, "skewed", 3000, 100), randn(g, 3000, 40, dtype=BF16)
    want, slack = grad64(grad, tokens, 100, 2.0, padding=0)
    out = psb.embedding_grad(grad, tokens, 100, 2.0, padding=0, dtype=F32)
    check(out, want, slack)
    assert not out[0].any()
    before = randn(g, 100, 40)
    after = before.clone()
    assert psb.embedding_grad(grad, tokens, 100, 2.0, padding=0, out=after, accumulate=True) is after
    # one more addition in FP32: half a step of the result
    check(after, before.double() + want, slack + (before.double() + want).abs() * U)
    untouched = want.abs().sum(1) == 0
    assert untouched.any() and torch.equal(after[untouched], before[untouched])
    none = tokens[:0]
    assert not psb.embedding_grad(grad[:0], none, 100).any()
    psb.embedding_grad(grad[:0], none, 100, out=after, accumulate=True)
    assert torch.equal(after[untouched], before[untouched])
    # NaN and inf at empty places reach nothing; at a token they reach its row alone.
    tokens[5], tokens[6] = -1, 55
    grad[5], grad[6] = math.nan, math.inf
    out = psb.embedding_grad(grad, tokens, 100)
    assert out[55].isinf().all() and out.isfinite().all(1).sum() == 99


# ------------------------------------------------------------------------------------ router

def route64(logits, k, normalize):
    x = logits.double()
    t, experts = x.shape
    index = torch.arange(experts, device="cuda")
    left, chosen = x.clone(), []
    for _ in range(k):
        best = left.amax(1)
        at = torch.where((left == best[:, None]) & (left > -math.inf), index, experts).amin(1)
        left = left.masked_fill(index == at[:, None], -math.inf)
        chosen.append(torch.where(at < experts, at, -1))
    chosen = torch.stack(chosen, 1)
    on = x > -math.inf
    if normalize:
        on &= (index[None, None] == chosen[:, :, None]).any(1)
    top = torch.where(on, x, -1e300).amax(1, keepdim=True)
    e = torch.where(on, torch.exp(torch.where(on, x, top) - top), 0.0)
    p = e / e.sum(1, keepdim=True).clamp_min(1e-300)
    return p, torch.where(chosen >= 0, p.gather(1, chosen.clamp_min(0)), 0.0), chosen


def softmax_slack(logits):
    """Relative error of a share: x - max rounds by u * |x - max| <= u * spread (in the share's own exponent and, weighted, in
    the sum), expf is off by 2 steps (4u) in both, the sum of E terms by E * u, the division by u."""
    x = logits.double()
    finite = torch.where(x > -math.inf, x, math.nan)
    spread = (finite.nan_to_num(-1e300).amax(1) - finite.nan_to_num(1e300).amin(1)).clamp_min(0)
    return (2 * spread + 8 + x.shape[1] + 2)[:, None] * U


EXPERTS = [(1, 1), (2, 1), (3, 3), (8, 2), (31, 4), (32, 32), (33, 5), (64, 6), (100, 32), (256, 8), (257, 9), (512, 10), (1024, 32)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("experts,k", EXPERTS)
def test_route_and_its_gradient(dtype, normalize, experts, k):
    g = gen(experts)
    for tokens in (1, 7, 130):
        logits = randn(g, tokens, experts, dtype=dtype)
        if tokens == 130:
            logits[3:9] = -math.inf                                        # no expert at all
            logits[20:60, ::2] = -math.inf                                 # half of them off
            logits[60:80] = (logits[60:80].float() * 2).round().to(dtype)  # many ties
            logits[80:90] = 0.0
            logits[85:90, 1::2] = -0.0                                     # equal to +0
            logits[90:95] *= 20
            logits[95] = torch.finfo(dtype).min                            # the lowest value is a score like any other
            logits[96, : experts // 2] = torch.finfo(dtype).min
        p, want, chosen64 = route64(logits, k, normalize)
        weights, chosen = psb.route(logits, k, normalize)
        assert torch.equal(chosen.long(), chosen64)
        slack = softmax_slack(torch.where(logits == torch.finfo(dtype).min, -math.inf, logits))
        # shares below the smallest normal number lose bits, expf's included
        check(weights, want, want * slack + 2.0 ** -126)
        view = strided(logits, 3, 1)
        again = psb.route(view, k, normalize)
        assert torch.equal(again[0], weights) and torch.equal(again[1], chosen)

        grad = randn(g, tokens, k)
        dense = torch.zeros(tokens, experts + 1, dtype=torch.float64, device="cuda")
        dense.scatter_(1, torch.where(chosen64 >= 0, chosen64, experts), grad.double())
        dense, on = dense[:, :-1], chosen64 >= 0
        inner = (grad.double() * weights.double() * on).sum(1, keepdim=True)
        size = (grad.double() * weights.double() * on).abs().sum(1, keepdim=True)
        grad_slack = p * (dense.abs() + size) * (slack + (k + 4) * U) + 2.0 ** -126 * (dense.abs() + size + 1)
        if normalize:  # p is the weights as they were stored
            p = torch.zeros(tokens, experts + 1, dtype=torch.float64, device="cuda")
            p = p.scatter_(1, torch.where(on, chosen64, experts), weights.double())[:, :-1]
        want = p * (dense - inner)
        got = psb.route_grad(grad, logits, weights, chosen, normalize)
        check(got, want, grad_slack)
        out = strided(torch.full_like(logits, 5.0), 1)
        psb.route_grad(grad, view, weights, chosen, normalize, out=out)
        assert torch.equal(out, got)


def test_route_with_nan_and_inf():
    logits = randn(gen(1), 5, 40)
    logits[0, 7] = math.nan
    logits[1, 3] = math.inf
    logits[2] = math.nan
    logits[3, :38] = -math.inf
    for normalize in (True, False):
        weights, chosen = psb.route(logits, 4, normalize)
        assert 7 not in chosen[0].tolist() and weights[0].isnan().all()
        assert chosen[1, 0] == 3 and weights[1, 0].isnan()
        assert chosen[2].tolist() == [-1] * 4
        assert sorted(chosen[3, :2].tolist()) == [38, 39] and chosen[3, 2:].tolist() == [-1, -1]
        assert weights[3, 2:].tolist() == [0, 0] and abs(weights[3].sum().item() - 1) < 1e-6
        assert weights[4].isfinite().all()
        grad = torch.ones(5, 4, device="cuda")
        grad[3, 2:] = math.nan  # beside a choice of -1: not used
        got = psb.route_grad(grad, logits, weights, chosen, normalize)
        assert got[3:].isfinite().all() and got[0].isnan().any()


def test_route_gradient_with_a_choice_that_stands_twice():
    """route never gives one, but a caller may: the gradients of both places add up, as the formula says."""
    logits = randn(gen(8), 3, 40)
    chosen = torch.tensor([[5, 5, 7], [1, 0, 1], [9, 9, 9]], dtype=torch.int32, device="cuda")
    weights, grad = torch.rand(3, 3, generator=gen(9), device="cuda"), randn(gen(10), 3, 3)
    p = torch.softmax(logits.double(), 1)
    inner = (grad.double() * weights.double()).sum(1, keepdim=True)
    dense = torch.zeros_like(p).scatter_add_(1, chosen.long(), grad.double())
    size = grad.double().abs().sum(1, keepdim=True) * 2
    check(psb.route_grad(grad, logits, weights, chosen, False), p * (dense - inner), p * size * (softmax_slack(logits) + 8 * U))
    share = weights.double() * (grad.double() - inner)
    want = torch.zeros_like(p).scatter_add_(1, chosen.long(), share)
    check(psb.route_grad(grad, logits, weights, chosen, True), want, size * 8 * U)


def test_route_gradient_against_differences():
    logits = randn(gen(2), 6, 12)
    grad = randn(gen(3), 6, 3).double()
    for normalize in (True, False):
        weights, chosen = psb.route(logits, 3, normalize)
        got = psb.route_grad(grad.float(), logits, weights, chosen, normalize).double()
        h = 2.0 ** -10
        for e in range(12):
            up, down = logits.double(), logits.double()
            up[:, e] += h
            down[:, e] -= h

            def value(x):  # the choice held fixed, as the gradient holds it
                p = torch.softmax(x, 1).gather(1, chosen.long())
                return ((p / p.sum(1, keepdim=True) if normalize else p) * grad.float().double()).sum(1)
            # the difference quotient is off by h^2 / 6 of a third derivative (below 10 * |grad|), the kernel by FP32
            assert ((value(up) - value(down)) / (2 * h) - got[:, e]).abs().max() < 10 * grad.abs().max() * (h * h + 100 * U)


# ------------------------------------------------------------------------------------ dispatch and combine

def order64(chosen, experts, align):
    flat = chosen.reshape(-1).tolist()
    slots = [[] for _ in range(experts)]
    for s, e in enumerate(flat):
        if 0 <= e < experts:
            slots[e].append(s)
    position, offsets = [-1] * len(flat), [0]
    for e in range(experts):
        for i, s in enumerate(slots[e]):
            position[s] = offsets[-1] + i
        offsets.append(offsets[-1] + -(-len(slots[e]) // align) * align)
    return position, offsets, [len(s) for s in slots]


def choices(g, tokens, k, experts, kind, index):
    if kind == "one":
        c = torch.full((tokens, k), experts - 1, device="cuda")
    elif kind == "none":
        c = torch.full((tokens, k), -1, device="cuda")
    elif kind == "far":
        c = torch.randint(0, 2 * experts, (tokens, k), generator=g, device="cuda") - experts // 2
    else:
        c = torch.randint(0, experts, (tokens, k), generator=g, device="cuda")  # an expert may come twice
    return c.to(index)


LAYERS = [(1, 1, 1, 1, "any"), (1, 8, 64, 16, "any"), (5, 2, 3, 4, "far"), (33, 6, 64, 1, "any"), (200, 32, 40, 8, "one"),
          (129, 3, 1024, 1, "far"), (77, 2, 5, 7, "none"), (700, 4, 16, 128, "any"), (3000, 3, 13, 1, "far"), (9000, 8, 384, 16, "any"),
          (2048, 1, 8, 1, "one"), (341, 6, 9, 2, "any"), (342, 6, 9, 2, "any")]


@pytest.mark.parametrize("tokens,k,experts,align,kind", LAYERS)
@pytest.mark.parametrize("dtype,width", [(F32, 1), (F32, 20), (BF16, 64), (F16, 33), (BF16, 2056), (F16, 6)])
def test_dispatch_and_combine(tokens, k, experts, align, kind, dtype, width):
    if tokens * k * width > 2**26:
        width = 16
    g = gen(tokens + width)
    index = torch.int64 if tokens % 2 else torch.int32
    chosen = choices(g, tokens, k, experts, kind, index)
    x = randn(g, tokens, width, dtype=dtype)
    position, offsets, counts = order64(chosen, experts, align)
    at = torch.tensor(position, device="cuda").view(tokens, k)
    token, choice = (at >= 0).nonzero(as_tuple=True)
    slot = at[token, choice]
    end = offsets[-1]
    room = psb.dispatch_rows(tokens * k, experts, align)
    assert end <= room

    want = torch.zeros(room, width, dtype=dtype, device="cuda")
    want[slot] = x[token]
    rows, plan = psb.dispatch(x, chosen, experts, align)
    assert plan.position.tolist() == at.tolist() and plan.offsets.tolist() == offsets and plan.counts.tolist() == counts
    assert torch.equal(rows, want)
    out = strided(torch.full((room + 3, width), 9.0, device="cuda", dtype=dtype), 5, 1)
    psb.dispatch(strided(x, 2), chosen, experts, align, out=out)
    assert torch.equal(out[:end], want[:end]) and (out[end:] == 9).all()  # the rows behind the last expert stay

    # back, with weights and something added; rows that no token has hold NaN
    y = randn(g, room, width, dtype=dtype)
    used = torch.zeros(room, dtype=torch.bool, device="cuda").index_fill_(0, slot, True)
    y[~used] = math.nan
    weights = torch.rand(tokens, k, generator=g, device="cuda")
    weights[at < 0] = math.nan
    add = randn(g, tokens, width, dtype=dtype)
    for w, a in ((weights, None), (None, None), (weights, add), (None, add)):
        sum64 = torch.zeros(tokens, width, dtype=torch.float64, device="cuda")
        size = sum64.clone()
        term = y[slot].double() * (1.0 if w is None else w[token, choice].double()[:, None])
        sum64.index_add_(0, token, term)
        size.index_add_(0, token, term.abs())
        if a is not None:
            sum64, size = sum64 + a.double(), size + a.double().abs()
        check(psb.combine(y, plan, w, a), sum64, size * (k + 2) * U)
        dst = strided(torch.zeros(tokens, width, device="cuda", dtype=dtype) if a is None else a, 3, 1)
        psb.combine(strided(y, 1), plan, w, None if a is None else dst, out=dst)  # add may be out itself
        check(dst, sum64, size * (k + 2) * U)
    if kind != "none":
        assert torch.equal(psb.dispatch_grad(y, plan), psb.combine(y, plan))

    # gradients of combine
    grad = randn(g, tokens, width, dtype=dtype)
    grad_y, grad_w = psb.combine_grad(grad, y, plan, weights)
    want_y = torch.zeros(room, width, dtype=torch.float64, device="cuda")
    want_y[slot] = weights[token, choice].double()[:, None] * grad[token].double()
    check(grad_y, want_y, want_y.abs() * U)
    want_w = torch.zeros(tokens, k, dtype=torch.float64, device="cuda")
    term = grad[token].double() * y[slot].double()
    want_w[token, choice] = term.sum(1)
    size = torch.zeros_like(want_w)
    size[token, choice] = term.abs().sum(1)
    check(grad_w, want_w, size * (width / 32 + 24) * U)  # a lane adds at most width / 32 + 8 products, then at most 13 sums
    out = strided(torch.full((room, width), 9.0, device="cuda", dtype=dtype), 1, 1)
    again = psb.combine_grad(strided(grad, 1), strided(y, 2), plan, weights, out=out)
    assert again[0] is out and (out[end:] == 9).all()
    check(out[:end], want_y[:end], want_y[:end].abs() * U)
    check(again[1], want_w, size * (width / 32 + 24) * U)


def test_no_tokens():
    x = torch.empty(0, 16, device="cuda", dtype=BF16)
    rows, plan = psb.dispatch(x, torch.empty(0, 4, dtype=torch.int32, device="cuda"), 8, 128)
    assert rows.shape == (0, 16) and plan.offsets.tolist() == [0] * 9 and plan.counts.tolist() == [0] * 8
    assert psb.combine(rows, plan).shape == (0, 16)
    y = torch.full((5, 16), 2.0, device="cuda", dtype=BF16)
    grad_y, grad_w = psb.combine_grad(x, y, plan, torch.empty(0, 4, device="cuda"))
    assert not grad_y.any() and grad_w.shape == (0, 4)
    weights, chosen = psb.route(torch.empty(0, 8, device="cuda"), 2)
    assert weights.shape == chosen.shape == (0, 2)
    assert psb.route_grad(weights, torch.empty(0, 8, device="cuda"), weights, chosen).shape == (0, 8)


def test_a_plan_that_points_outside_is_not_followed():
    """Positions and bounds from anywhere: nothing outside the given tensors is read or written."""
    far = 2**31 - 1
    position = torch.tensor([[0, far], [-5, 1], [3, 4]], dtype=torch.int32, device="cuda")
    plan = psb.DispatchPlan(position, torch.tensor([-7, far, -1], dtype=torch.int32, device="cuda"),
                            torch.tensor([far, -far], dtype=torch.int32, device="cuda"))
    y = torch.ones(4, 8, device="cuda")
    w = torch.ones(3, 2, device="cuda")
    assert psb.combine(y, plan, w)[:, 0].tolist() == [1, 1, 1]
    grad_y, grad_w = psb.combine_grad(torch.ones(3, 8, device="cuda"), y, plan, w, out=torch.full_like(y, 9.0))
    assert grad_w.tolist() == [[8, 0], [0, 8], [8, 0]]


def test_dispatch_offsets_pass_32_bits():
    tokens, k, width = 70_000, 8, 4096  # 2.3e9 elements in expert order
    x = torch.empty(tokens, width, device="cuda", dtype=BF16)
    x[:] = (torch.arange(tokens, device="cuda") % 251)[:, None].to(BF16)
    chosen = torch.arange(k, dtype=torch.int32, device="cuda").repeat(tokens, 1)
    rows, plan = psb.dispatch(x, chosen, k)
    assert plan.counts.tolist() == [tokens] * k
    for e in range(k):
        assert torch.equal(rows[e * tokens: (e + 1) * tokens: 997], x[::997])
    assert torch.equal(rows[-1], x[-1])
    w = torch.full((tokens, k), 0.125, device="cuda")
    assert torch.equal(psb.combine(rows, plan, w), x)
    del x
    grad = torch.ones(tokens, width, device="cuda", dtype=BF16)
    grad_y, grad_w = psb.combine_grad(grad, rows, plan, w, out=rows)  # each element is read before it is written
    assert (grad_w[-1] == (tokens - 1) % 251 * width).all() and (grad_y[-1] == 0.125).all() and (grad_y[::1001] == 0.125).all()


# ------------------------------------------------------------------------------------ as they are used

def layer(x, logits, experts_w, k, align, ops=torch.ops.powersparse):
    weights, chosen = ops.route(logits, k, True)
    rows, position, offsets, counts = ops.dispatch(x, chosen, experts_w.shape[0], align)
    begin = offsets.tolist()
    y = torch.cat([torch.tanh(rows[a:b] @ w) for a, b, w in zip(begin, begin[1:], experts_w)] + [rows[begin[-1]:]])
    return ops.combine(y, position, offsets, counts, weights, x)


@pytest.mark.parametrize("align", [1, 4])
def test_a_model_of_them_and_its_gradients(align):
    """tokens -> embedding -> router -> dispatch -> experts -> combine with the residual, and back, against autograd in
    64 bits.  All values are of the order of one and fewer than 500 FP32 roundings lie on any path: 1e-4."""
    g = gen(11)
    vocab, width, experts, k = 50, 24, 6, 2
    tokens = torch.randint(-1, vocab, (4, 20), generator=g, device="cuda")
    leaves = [randn(g, vocab, width), randn(g, width, experts) * 0.3, randn(g, experts, width, width) * 0.2]
    ours = [t.clone().requires_grad_() for t in leaves]
    h = torch.ops.powersparse.embedding(ours[0], tokens, 1.5, 3).view(-1, width)
    out = layer(h, h @ ours[1], ours[2], k, align)
    (out * 0.5).sum().backward()  # an expanded gradient

    ref = [t.double().requires_grad_() for t in leaves]
    flat = tokens.reshape(-1)
    h = ref[0][flat.clamp_min(0)] * 1.5 * (flat >= 0)[:, None]
    h = torch.where((flat == 3)[:, None], h.detach(), h)  # token 3 is padding: no gradient through it
    logits = h @ ref[1]
    value, chosen = logits.topk(k, 1)
    weights = torch.softmax(value, 1)
    every = torch.tanh(torch.einsum("td,edf->tef", h, ref[2]))
    want = h + (every.gather(1, chosen[:, :, None].expand(-1, -1, width)) * weights[:, :, None]).sum(1)
    (want * 0.5).sum().backward()
    # logits that tie (the rows of padding are all zero) choose the same experts in both, up to order; compare all
    live = (flat >= 0)
    assert (out.double() - want)[live].abs().max() < 1e-4
    for a, b in zip(ours, ref):
        assert (a.grad.double() - b.grad).abs().max() < 1e-4 * max(1.0, b.grad.abs().max().item())
    assert not ours[0].grad[3].any()


def test_gradients_against_differences():
    """The registered ops' gradients against central differences of the ops themselves (all linear but route, whose own
    test is above): the difference of a linear map is its gradient up to rounding."""
    g = gen(4)
    ops = torch.ops.powersparse
    chosen = torch.tensor([[0, 2], [1, 1], [-1, 0], [2, 5]], device="cuda")
    x, w, add = randn(g, 4, 6).requires_grad_(), randn(g, 4, 2).requires_grad_(), randn(g, 4, 6).requires_grad_()
    probe = randn(g, 4, 6)

    def f(x, w, add):
        rows, position, offsets, counts = ops.dispatch(x, chosen, 3, 2)
        return (ops.combine(rows * rows, position, offsets, counts, w, add) * probe).sum()
    f(x, w, add).backward()
    for t in (x, w, add):
        d = randn(g, *t.shape)
        h = 2.0 ** -6
        args = [[u.detach() + (s * h * d if u is t else 0) for u in (x, w, add)] for s in (1, -1)]
        quotient = (f(*args[0]) - f(*args[1])).item() / (2 * h)
        # f is a polynomial of degree two in each argument, so the quotient is exact; its values round by some u * |f| / h
        assert abs(quotient - (t.grad * d).sum().item()) < 64 * U / h * 100


def test_opcheck():
    g = gen(6)
    ops = torch.ops.powersparse
    which = ("test_schema", "test_faketensor", "test_autograd_registration")
    table, tokens = randn(g, 20, 8).requires_grad_(), torch.randint(0, 20, (7,), generator=g, device="cuda")
    torch.library.opcheck(ops.embedding.default, (table, tokens, 2.0, 4), test_utils=which)
    torch.library.opcheck(ops.embedding_grad.default, (randn(g, 7, 8), tokens, 20), test_utils=which)
    logits = randn(g, 7, 10).requires_grad_()
    torch.library.opcheck(ops.route.default, (logits, 3, False), test_utils=which)
    x, chosen = randn(g, 7, 8).requires_grad_(), torch.randint(0, 5, (7, 3), generator=g, device="cuda")
    torch.library.opcheck(ops.dispatch.default, (x, chosen, 5, 4), test_utils=which)
    rows, plan = psb.dispatch(x.detach(), chosen, 5, 4)
    weights = torch.rand(7, 3, device="cuda").requires_grad_()
    torch.library.opcheck(ops.combine.default, (rows.requires_grad_(), *plan, weights, x), test_utils=which)


def run_all(s):
    """Every operator once, on tensors of the dictionary `s`."""
    out = [psb.embedding(s["table"], s["tokens"], 2.0)]
    out.append(psb.embedding_grad(out[0], s["tokens"], len(s["table"]), 0.5, dtype=F32))
    weights, chosen = psb.route(s["logits"], 4)
    rows, plan = psb.dispatch(out[0], chosen, s["logits"].shape[1], 8)
    y = psb.combine(rows, plan, weights, out[0])
    grads = psb.combine_grad(y, rows, plan, weights)
    out += [weights, chosen, rows, *plan, y, *grads, psb.dispatch_grad(grads[0], plan),
            psb.route_grad(grads[1], s["logits"], weights, chosen)]
    return out


def inputs(seed, n=600):
    g = gen(seed)
    return dict(table=randn(g, 300, 72, dtype=BF16), tokens=torch.randint(-1, 300, (n,), generator=g, device="cuda"),
                logits=randn(g, n, 48, dtype=BF16))


def test_replayed_graphs_streams_and_two_at_once():
    """Captured and replayed with new inputs, on a side stream, and two graphs whose replays overlap: the same bits as
    eager calls."""
    sets = [inputs(s) for s in (1, 2, 3, 4)]
    want = [run_all(s) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_all(sets[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))

    held, graphs, outs = [dict(inputs(9)), dict(inputs(10))], [], []
    for h in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run_all(h))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rounds in ((0, 1), (2, 3), (3, 0)):
        for h, i in zip(held, rounds):
            for key in h:
                h[key].copy_(sets[i][key])
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for out, i in zip(outs, rounds):
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


def mixed(s, side):
    """The operators between kernels, copies and fills of torch, on two streams: each reads what the one before has just
    written and overwrites what the one before that still read."""
    main = torch.cuda.current_stream()
    x = psb.embedding(s["table"], s["tokens"], 2.0)
    kept = []
    for i in range(6):
        x.mul_(-0.5)
        weights, chosen = psb.route(x[:, :48].contiguous(), 4)
        rows, plan = psb.dispatch(x, chosen, 48, 8)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            y = torch.empty_like(rows)
            y.copy_(rows)
            grads = psb.combine_grad(x, y, plan, weights, out=y)
        out = torch.zeros_like(x)
        psb.combine(rows, plan, weights, out=out, add=x)
        main.wait_stream(side)
        x.copy_(out)
        x.add_(psb.dispatch_grad(grads[0], plan))
        rows.zero_()
        grad = psb.embedding_grad(x, s["tokens"], 300, 0.5, dtype=F32)
        kept += [out, grads[1].clone(), grad.clone()]
        y.fill_(3.0)
    return kept + [x]


def test_between_other_kernels_copies_and_streams():
    """Eager, with a wait after every call, and captured: the same bits."""
    for n in (600, 3000):
        s, side = inputs(31, n), torch.cuda.Stream()
        with pytest.MonkeyPatch.context() as patch:
            for name in ("embedding", "route", "dispatch", "combine", "combine_grad", "dispatch_grad", "embedding_grad"):
                def waited(*args, call=getattr(psb, name), **kwargs):
                    torch.cuda.synchronize()
                    result = call(*args, **kwargs)
                    torch.cuda.synchronize()
                    return result
                patch.setattr(psb, name, waited)
            want = mixed(s, side)
        torch.cuda.synchronize()
        for _ in range(5):
            got = mixed(s, side)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = mixed(s, side)
        for _ in range(5):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_capture_before_any_eager_call():
    """In a process of its own, each operator's first call is a captured one."""
    code = """
import torch, sys
sys.path.insert(0, %r)
import test_gpu_rows as t
s = t.inputs(1)
many = t.inputs(2, 3000)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = t.run_all(s) + t.run_all(many)
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, t.run_all(s) + t.run_all(many)))
print("captured first")
""" % os.path.dirname(os.path.abspath(__file__))
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                         cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert "captured first" in run.stdout, run.stderr[-2000:]


def test_training_step_captured_and_replayed():
    """Forward and backward of the registered ops in a graph: gradients of each replay's inputs."""
    g = gen(21)
    vocab, width, experts, k, n = 40, 16, 4, 2, 24
    table, gate = randn(g, vocab, width).requires_grad_(), (randn(g, width, experts) * 0.3).requires_grad_()
    tokens = torch.randint(-1, vocab, (n,), generator=g, device="cuda")
    ops = torch.ops.powersparse

    def step():
        h = ops.embedding(table, tokens, 1.5)
        weights, chosen = ops.route(h @ gate, k, False)
        rows, position, offsets, counts = ops.dispatch(h, chosen, experts, 8)
        out = ops.combine(torch.tanh(rows), position, offsets, counts, weights, h)
        return torch.autograd.grad((out * out).sum(), (table, gate))
    want = []
    batches = [torch.randint(-1, vocab, (n,), generator=g, device="cuda") for _ in range(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for b in batches:
            tokens.copy_(b)
            want.append([t.clone() for t in step()])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for b, w in zip(batches, want):
        tokens.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        # The same kernels on the same numbers, but torch's products (16 and 24 terms of order one: off by 24 * u, under
        # 2e-6, each; three lie on a path) may be made by another kernel.
        assert all(torch.allclose(a, c, rtol=1e-5, atol=1e-5) for a, c in zip(got, w))


def test_calls_from_two_threads():
    sets = [inputs(s, 2500) for s in (1, 2)]
    want = [run_all(s) for s in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = run_all(sets[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_default_stream_by_its_handles():
    s = inputs(3)
    torch.cuda.synchronize()
    for handle in (0, 1):
        out = psb.embedding(s["table"], s["tokens"], 2.0, stream=handle)
        torch.cuda.synchronize()
        assert torch.equal(out, psb.embedding(s["table"], s["tokens"], 2.0))
    with pytest.raises(ValueError, match="handle"):
        psb.embedding(s["table"], s["tokens"], stream=7)


def test_explicit_stream_owns_what_the_call_allocates():
    s = inputs(7)
    want = run_all(s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = psb.embedding(s["table"], s["tokens"], 2.0, stream=side)
    b = psb.embedding_grad(a, s["tokens"], 300, 0.5, dtype=F32, stream=side.cuda_stream)
    weights, chosen = psb.route(s["logits"], 4, stream=side)
    rows, plan = psb.dispatch(a, chosen, 48, 8, stream=side)
    y = psb.combine(rows, plan, weights, a, stream=side)
    side.synchronize()
    for got, ref in ((a, want[0]), (b, want[1]), (weights, want[2]), (chosen, want[3]), (rows, want[4]), (y, want[8])):
        assert torch.equal(got, ref)


def test_refusals():
    g = gen(0)
    x, i = randn(g, 6, 8), torch.zeros(6, 2, dtype=torch.int32, device="cuda")
    _, plan = psb.dispatch(x, i, 4)
    y, w = randn(g, 12, 8), torch.ones(6, 2, device="cuda")
    t = i[:, 0].contiguous()
    for call in (lambda: psb.embedding(x.double(), t), lambda: psb.embedding(x.t(), t), lambda: psb.embedding(x, t.float()),
                 lambda: psb.embedding(x, i[:, 0]), lambda: psb.embedding(x, t.cpu()), lambda: psb.embedding(x[0], t),
                 lambda: psb.embedding(x[:0], t), lambda: psb.embedding(x, t, out=x[:5]), lambda: psb.embedding(x, t, out=x.half()),
                 lambda: psb.embedding(x[:1].expand(6, 8), t), lambda: psb.embedding(x[:, :0], t),
                 lambda: psb.embedding_grad(x[:5], t, 4), lambda: psb.embedding_grad(x, t, 0),
                 lambda: psb.embedding_grad(x, t, 4, dtype=BF16), lambda: psb.embedding_grad(x.half(), t, 4, dtype=BF16),
                 lambda: psb.embedding_grad(x, t, 4, accumulate=True), lambda: psb.embedding_grad(x, t, 4, padding=4),
                 lambda: psb.embedding_grad(x, t, 4, out=x), lambda: psb.embedding_grad(x, t, 2**31),
                 lambda: psb.route(x, 0), lambda: psb.route(x, 9), lambda: psb.route(torch.zeros(2, 1025, device="cuda"), 2),
                 lambda: psb.route(torch.zeros(2, 64, device="cuda"), 33), lambda: psb.route_grad(w, x, w, i.long()),
                 lambda: psb.route_grad(w[:5], x, w, i), lambda: psb.route_grad(w, x, w.half(), i),
                 lambda: psb.dispatch(x, i[:5], 4), lambda: psb.dispatch(x, t, 4), lambda: psb.dispatch(x, i, 0),
                 lambda: psb.dispatch(x, i, 4, align=0), lambda: psb.dispatch(x, i, 4, out=y[:11]),
                 lambda: psb.dispatch(x, i, 4, out=y[:, :7]), lambda: psb.dispatch(x, i.t().contiguous().t(), 4),
                 lambda: psb.dispatch(x, torch.zeros(6, 33, dtype=torch.int32, device="cuda"), 4),
                 lambda: psb.combine(y, plan, w.half()), lambda: psb.combine(y, plan, w[:5]), lambda: psb.combine(y, plan, add=x[:5]),
                 lambda: psb.combine(y, plan, add=x.half()), lambda: psb.combine(y, plan._replace(position=i.long())),
                 lambda: psb.combine(y, plan, out=x[:, :4]), lambda: psb.combine_grad(x[:5], y, plan, w),
                 lambda: psb.combine_grad(x, y, plan, w, out=y[:11]), lambda: psb.combine_grad(x.half(), y, plan, w),
                 lambda: psb.combine_grad(x, y, plan._replace(offsets=plan.counts), w)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------------------------ contracts of single functions

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("experts", [8, 40, 257])
def test_a_nan_reaches_every_weight_and_gradient_of_its_row(dtype, normalize, experts):
    logits = randn(gen(1), 9, experts, dtype=dtype)
    logits[0] = math.nan                                      # nothing else: no choice is left
    logits[1], logits[1, 3] = -math.inf, math.nan             # nor here
    logits[2, 5] = math.nan
    logits[3, 2:], logits[3, 6] = -math.inf, math.nan         # fewer choices than top_k
    logits[4, 1:], logits[4, 0] = -math.inf, math.inf
    logits[5, [1, 4]] = math.inf
    logits[6] = -math.inf                                     # no expert at all, and no NaN
    logits[7, 2:] = -math.inf
    weights, chosen = psb.route(logits, 4, normalize)
    assert chosen[:2].eq(-1).all() and chosen[6].eq(-1).all() and chosen[3, 2:].eq(-1).all() and chosen[4, 1:].eq(-1).all()
    assert weights[:6].isnan().all()
    assert not weights[6].any() and not weights[7, 2:].any() and weights[7:].isfinite().all()
    for grad in (torch.ones_like(weights), torch.where(chosen < 0, math.nan, 1.0)):  # beside a choice of -1 it is not used
        got = psb.route_grad(grad, logits, weights, chosen, normalize)
        assert got[:6].isnan().all() and not got[6].any() and got[7:].isfinite().all()


def test_route_of_the_most_tokens():
    """2^31 - 1 tokens, where a block count in 32 bits would overflow; one expert, so every weight is one."""
    n = 2**31 - 1
    logits = torch.zeros(n, 1, device="cuda", dtype=BF16)
    logits[n - 1] = math.nan
    weights, chosen = psb.route(logits, 1)
    for part in (slice(0, 2**30), slice(2**30, n - 1)):
        assert (weights[part] == 1).all() and not chosen[part].any()
    assert weights[n - 1].isnan() and chosen[n - 1] == -1
    # normalize=False: p = 1 and the sum of g w is g, so the gradient is zero but for the last row
    grad = psb.route_grad(weights, logits, weights, chosen, False)
    for part in (slice(0, 2**30), slice(2**30, n - 1)):
        assert not grad[part].any()
    assert grad[n - 1].isnan()


def test_embedding_op_refuses_a_padding_outside_the_table_in_the_forward_pass():
    table, tokens = randn(gen(0), 6, 8).requires_grad_(), torch.arange(6, device="cuda")
    for padding in (-1, 6):
        with pytest.raises(ValueError, match="padding"):
            torch.ops.powersparse.embedding(table, tokens, 1.0, padding)


def test_negated_views_are_refused_by_the_functions_and_resolved_by_the_ops():
    """Such a view has the negative bit set and its elements in memory with the other sign."""
    x, i = randn(gen(0), 6, 8), torch.arange(6, device="cuda")
    lazy = torch._neg_view(x)
    assert lazy.is_neg()
    w, c = psb.route(x, 2)
    _, plan = psb.dispatch(x, c, 8)
    y = randn(gen(1), 12, 8)
    for call in (lambda: psb.embedding(lazy, i), lambda: psb.embedding(x, i, out=torch._neg_view(torch.empty_like(x))),
                 lambda: psb.embedding_grad(lazy, i, 6), lambda: psb.route(lazy, 2), lambda: psb.route_grad(torch._neg_view(w), x, w, c),
                 lambda: psb.dispatch(lazy, c, 8), lambda: psb.combine(y, plan, torch._neg_view(w)), lambda: psb.combine(y, plan, add=lazy),
                 lambda: psb.combine_grad(lazy, y, plan, w), lambda: psb.embedding(x, torch._neg_view(i))):
        with pytest.raises(ValueError, match="negated"):
            call()
    assert torch.equal(torch.ops.powersparse.embedding(lazy, i), -x)


def test_a_given_out_counts_as_changed():
    """autograd refuses a backward pass through a tensor that a call has written since, as with torch's own out=."""
    s = inputs(1)
    x = psb.embedding(s["table"], s["tokens"])
    weights, chosen = psb.route(s["logits"], 4)
    rows, plan = psb.dispatch(x, chosen, 48)
    table = torch.zeros_like(s["table"])
    scores = torch.empty_like(s["logits"])
    grad_w = torch.ones_like(weights)
    for out, call in ((x, lambda: psb.embedding(s["table"], s["tokens"], out=x)),
                      (table, lambda: psb.embedding_grad(x, s["tokens"], 300, out=table)),
                      (table, lambda: psb.embedding_grad(x, s["tokens"], 300, out=table, accumulate=True)),
                      (scores, lambda: psb.route_grad(grad_w, s["logits"], weights, chosen, out=scores)),
                      (rows, lambda: psb.dispatch(x, chosen, 48, out=rows)),
                      (x, lambda: psb.combine(rows, plan, weights, out=x)),
                      (x, lambda: psb.dispatch_grad(rows, plan, out=x)),
                      (rows, lambda: psb.combine_grad(x, rows, plan, weights, out=rows))):
        before = out._version
        call()
        assert out._version > before
    leaf = torch.ones(300, 72, device="cuda", requires_grad=True)
    held = leaf * 2
    loss = (held * held).sum()
    psb.embedding(s["table"].float(), torch.arange(300, device="cuda"), out=held.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        out = torch.empty_like(x)
        psb.embedding(s["table"], s["tokens"], out=out)
    assert torch.equal(psb.embedding(s["table"], s["tokens"], out=out), psb.embedding(s["table"], s["tokens"]))


@pytest.mark.parametrize("tokens,k,experts,align,kind", [
    (2049, 1, 1, 1, "any"), (1025, 2, 1, 128, "far"), (2049, 1, 1024, 1, "any"), (700, 3, 1024, 16, "far"), (1024, 4, 1024, 128, "any"),
    (4097, 1, 1024, 3, "one"), (2731, 3, 1024, 1, "none"), (8193, 1, 1023, 2, "far"), (65537, 2, 1024, 1, "any"), (65537, 2, 1, 7, "far"),
    (4300, 32, 2, 1, "any")])
def test_order_of_many_slots_at_the_least_and_the_most_experts(tokens, k, experts, align, kind):
    """More than 2048 slots (a sort in clusters of 4, 8 and 16 blocks, beyond 131072 by strips that are walked twice)."""
    test_dispatch_and_combine(tokens, k, experts, align, kind, BF16, 16)


class Guarded:
    """Tensors inside larger buffers whose other elements hold a number that no call may change (in what is written) or a
    NaN that would reach the result (in what is read)."""

    def __init__(self):
        self.kept = []

    def read(self, t, extra=0):
        buf = torch.full((t.shape[0] + 64, t.shape[1] + extra), math.nan, device="cuda", dtype=t.dtype)
        view = buf[32: 32 + t.shape[0], : t.shape[1]]
        view.copy_(t)
        return view

    def write(self, rows, width, dtype, extra=0):
        buf = torch.full((rows + 64, width + extra), -77.0, device="cuda", dtype=dtype)
        self.kept.append((buf, rows, width))
        return buf[32: 32 + rows, :width]

    def untouched(self):
        return all((b[:32] == -77).all() and (b[32 + r:] == -77).all() and (b[:, w:] == -77).all() for b, r, w in self.kept)


@pytest.mark.parametrize("dtype,width,extra", [(F32, 8, 0), (F32, 1111, 3), (BF16, 64, 0), (BF16, 514, 2), (F16, 515, 0), (F16, 33, 5),
                                               (BF16, 2056, 8)])
@pytest.mark.parametrize("k", [1, 2, 5, 8])
def test_a_plan_that_points_outside_with_what_stands_around(dtype, width, extra, k):
    """As above, with everything inside larger buffers: values as the formulas have them, nothing read or changed outside."""
    g, guard = gen(width + k), Guarded()
    tokens, rows = 37, 60
    at = torch.arange(tokens * k, device="cuda") * 7 % (5 * rows // 4)  # rows of y; from `rows` on they are outside
    if tokens * k > rows:  # no row of grad_y from two places
        at = torch.where(torch.arange(tokens * k, device="cuda") < rows, at, rows + at)
    bad = torch.tensor([rows, -1, 2**31 - 1, -2**31, rows + 1, -rows], device="cuda")
    pick = torch.rand(tokens * k, generator=g, device="cuda") < 0.3
    at = torch.where(pick, bad[torch.arange(tokens * k, device="cuda") % len(bad)], at).view(tokens, k)
    nothing = torch.tensor([2**31 - 1, -9, -2**31], dtype=torch.int32, device="cuda")  # by these bounds no row is to be cleared
    plan = psb.DispatchPlan(at.to(torch.int32).contiguous(), nothing, torch.tensor([2**31 - 1, -2**31], dtype=torch.int32, device="cuda"))
    y, add, grad = (randn(g, n, width, dtype=dtype) for n in (rows, tokens, tokens))
    weights = torch.rand(tokens, k, generator=g, device="cuda")
    token, choice = ((at >= 0) & (at < rows)).nonzero(as_tuple=True)
    slot = at[token, choice]
    assert len(slot) and len(slot.unique()) == len(slot)
    weights[(at < 0) | (at >= rows)] = math.nan
    term = y[slot].double() * weights[token, choice].double()[:, None]
    want = add.double().index_add(0, token, term)
    size = add.double().abs().index_add(0, token, term.abs())
    out = guard.write(tokens, width, dtype, extra)
    psb.combine(guard.read(y, extra), plan, weights, guard.read(add), out=out)
    check(out, want, size * (k + 2) * U)
    plain = torch.zeros(tokens, width, dtype=torch.float64, device="cuda")
    out = guard.write(tokens, width, dtype, extra)
    psb.dispatch_grad(guard.read(y, extra), plan, out=out)
    check(out, plain.index_add(0, token, y[slot].double()), plain.index_add(0, token, y[slot].double().abs()) * (k + 2) * U)

    grad_y = guard.write(rows, width, dtype, extra)
    grad_y.fill_(5.0)
    want_y = torch.full((rows, width), 5.0, dtype=torch.float64, device="cuda")
    want_y[slot] = weights[token, choice].double()[:, None] * grad[token].double()
    got, grad_w = psb.combine_grad(guard.read(grad), guard.read(y, extra), plan, weights, out=grad_y)
    check(got, want_y, want_y.abs() * U)
    want_w, size = torch.zeros(tokens, k, dtype=torch.float64, device="cuda"), torch.zeros(tokens, k, dtype=torch.float64, device="cuda")
    term = grad[token].double() * y[slot].double()
    want_w[token, choice], size[token, choice] = term.sum(1), term.abs().sum(1)
    check(grad_w, want_w, size * (width / 32 + 24) * U)
    # bounds from anywhere, all of them to be cleared
    for offsets in ([-2**31, 2**31 - 1, -2**31], [0, -5, 2**31 - 1], [2**31 - 1] * 3, [-1] * 3):
        for counts in ([0, 0], [-2**31, 2**31 - 1], [2**31 - 1, -1]):
            grad_y = guard.write(rows, width, dtype, extra)
            psb.combine_grad(guard.read(grad), guard.read(y, extra), psb.DispatchPlan(
                plan.position, *(torch.tensor(v, dtype=torch.int32, device="cuda") for v in (offsets, counts))), weights, out=grad_y)
    assert guard.untouched()


@pytest.mark.parametrize("dtype,width,extra", [(F32, 20, 0), (F32, 131, 3), (BF16, 64, 8), (BF16, 130, 2), (F16, 33, 0)])
def test_what_stands_around_the_outputs_stays(dtype, width, extra):
    guard = Guarded()
    for n, rows in ((3, 5), (700, 90), (2048, 3000), (2049, 3000), (9000, 257)):
        g = gen(n)
        table, tokens = randn(g, rows, width, dtype=dtype), torch.randint(-rows, 2 * rows, (n,), generator=g, device="cuda")
        out = guard.write(n, width, dtype, extra)
        psb.embedding(guard.read(table, extra), tokens, out=out)
        assert torch.equal(out.double(), embedding64(table, tokens, 1.0))
        want, slack = grad64(out, tokens, rows, 1.0)
        grad = guard.write(rows, width, F32, extra)
        psb.embedding_grad(guard.read(out, extra), tokens, rows, out=grad)
        check(grad, want, slack)
        psb.embedding_grad(guard.read(out, extra), tokens, rows, out=grad, accumulate=True)
        chosen = torch.randint(-20, 60, (n, 3), generator=g, device="cuda")
        position, offsets, _ = order64(chosen, 40, 8)
        need = psb.dispatch_rows(n * 3, 40, 8)
        room = guard.write(need, width, dtype, extra)
        _, plan = psb.dispatch(guard.read(out, extra), chosen, 40, 8, out=room)
        assert plan.position.view(-1).tolist() == position
        assert (room[offsets[-1]:] == -77).all() and not (room[:offsets[-1]] == -77).all(1).any()
        logits = randn(g, n, 40, dtype=dtype)
        w, c = psb.route(guard.read(logits, extra), 3)
        scores = guard.write(n, 40, dtype, extra)
        psb.route_grad(torch.rand(n, 3, generator=g, device="cuda"), guard.read(logits, extra), w, c, out=scores)
        assert (scores != -77).all()
    assert guard.untouched()


@pytest.mark.parametrize("shards", [4, 16])
def test_fresh_outputs_where_most_experts_are_elsewhere(shards):
    """A batch on a GPU that holds few of the experts: all rows behind the last one are zeros in what a call allocates."""
    g = gen(shards)
    tokens, k, experts, width = 8192, 8, 64, 136
    chosen = torch.randint(0, experts, (tokens, k), generator=g, device="cuda") - experts // shards
    mine = experts // shards
    x = randn(g, tokens, width, dtype=BF16)
    for align in (1, 128):
        junk = torch.full((psb.dispatch_rows(tokens * k, mine, align), width), math.nan, device="cuda", dtype=BF16)
        del junk  # so that the allocation finds something
        rows, plan = psb.dispatch(x, chosen, mine, align)
        end = plan.offsets[-1].item()
        assert plan.counts.sum().item() == ((chosen >= 0) & (chosen < mine)).sum().item() < tokens * k // 2
        assert end < len(rows) // 2 and not rows[end:].any()
        token, choice = (plan.position >= 0).nonzero(as_tuple=True)
        slot = plan.position[token, choice].long()
        assert torch.equal(rows[slot], x[token])
        weights = torch.rand(tokens, k, generator=g, device="cuda")
        junk = torch.full_like(rows, math.nan)
        del junk
        grad_y, grad_w = psb.combine_grad(x, rows, plan, weights)
        want = torch.zeros(len(rows), width, dtype=torch.float64, device="cuda")
        want[slot] = weights[token, choice].double()[:, None] * x[token].double()
        check(grad_y, want, want.abs() * U)
        assert not grad_w[plan.position < 0].any()


@pytest.mark.parametrize("weighted", [True, False])
def test_combine_gradient_where_not_every_input_takes_one(weighted):
    """The registered op with weights, rows or something added that take no gradient: the same gradients for the others."""
    g = gen(13)
    ops = torch.ops.powersparse
    chosen = torch.randint(-1, 7, (50, 3), generator=g, device="cuda")
    x, add = randn(g, 50, 24), randn(g, 50, 24)
    weights = torch.rand(50, 3, generator=g, device="cuda") if weighted else None
    _, plan = psb.dispatch(x, chosen, 7, 4)
    y = randn(g, psb.dispatch_rows(150, 7, 4), 24)
    probe = randn(g, 50, 24)
    grad_y, grad_w = psb.combine_grad(probe, y, plan, weights if weighted else torch.ones(50, 3, device="cuda"))
    wants = dict(y=grad_y, weights=grad_w, add=probe)
    for names in (("y",), ("weights",), ("add",), ("y", "add"), ("y", "weights"), ("weights", "add"), ("y", "weights", "add")):
        if not weighted and "weights" in names:
            continue
        args = {n: t.clone().requires_grad_(n in names) for n, t in (("y", y), ("weights", weights), ("add", add)) if t is not None}
        out = ops.combine(args["y"], *plan, args.get("weights"), args["add"])
        assert torch.equal(out, psb.combine(y, plan, weights, add))
        (out * probe).sum().backward()
        for n, t in args.items():
            assert (t.grad is not None) == (n in names)
            assert n not in names or torch.equal(t.grad, wants[n])


@pytest.mark.parametrize("kind", ["one", "skewed", "distinct", "any", "empty"])
@pytest.mark.parametrize("n,width,rows", [(1, 5 * 2**20, 2), (1, 5 * 2**20 + 8, 3), (2, 5 * 2**19 + 1, 3), (33, 163841, 40), (200, 26300, 257),
                                          (1024, 5120, 1500), (1025, 5120, 1500), (2048, 2560, 3000), (2048, 2568, 3000),
                                          (2047, 2563, 2047)])
def test_embedding_grad_of_few_tokens_in_wide_rows(kind, n, width, rows):
    """About the border of 5 * 2^20 elements between the one launch and the sort, which fewer than 2049 tokens reach by wide rows alone."""
    g = gen(n)
    tokens, grad = batch(g, kind, n, rows), randn(g, n, width, dtype=BF16)
    want, slack = grad64(grad, tokens, rows, 0.5)
    for out in (BF16, F32):
        check(psb.embedding_grad(grad, tokens, rows, 0.5, dtype=out), want, slack)
    dst = torch.zeros(rows, width, device="cuda")
    psb.embedding_grad(grad, tokens, rows, 0.5, out=dst, accumulate=True)
    check(dst, want, slack)


@pytest.mark.parametrize("handle", [False, True])
def test_explicit_stream_of_every_function_with_outputs_given(handle):
    """More than 2048 tokens (a workspace on that stream), a torch stream or its handle, and every ``out``."""
    s = inputs(17, 3000)
    want = run_all(s)
    grad_scores = psb.route_grad(want[10], s["logits"], want[2], want[3])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    on = side.cuda_stream if handle else side
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # what is given belongs to that stream too
        x, table, scores = torch.empty_like(want[0]), torch.empty_like(want[1]), torch.empty_like(s["logits"])
        rows, y, grad_y, grad_x = (torch.zeros_like(want[i]) for i in (4, 8, 9, 11))
    psb.embedding(s["table"], s["tokens"], 2.0, out=x, stream=on)
    psb.embedding_grad(x, s["tokens"], 300, 0.5, out=table, stream=on)
    weights, chosen = psb.route(s["logits"], 4, stream=on)
    _, plan = psb.dispatch(x, chosen, 48, 8, out=rows, stream=on)
    psb.combine(rows, plan, weights, x, out=y, stream=on)
    _, grad_w = psb.combine_grad(y, rows, plan, weights, out=grad_y, stream=on)
    psb.dispatch_grad(grad_y, plan, out=grad_x, stream=on)
    psb.route_grad(grad_w, s["logits"], weights, chosen, out=scores, stream=on)
    side.synchronize()
    for got, ref in zip((x, table, weights, chosen, rows, *plan, y, grad_y, grad_w, grad_x, scores), [*want[:12], grad_scores]):
        assert torch.equal(got, ref)
