"""The operators beside the layer at their edges: calls whose result would be wrong without a word are refused, and
sizes, tables and cuts that the plain tests do not reach.  Bounds as in test_matmul.py and test_expert_rows.py.
"""
import os
import re

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.fx.experimental.proxy_tensor import make_fx

import mini_mega_b200 as mm
from mini_mega_b200 import _lib

E4 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def built():
    _lib.build()


def _plan(device="cpu"):
    """4 tokens x 2 pairs on 3 experts, all of them on expert 0."""
    place = torch.arange(8, dtype=torch.int32, device=device)
    return mm.ExpertPlan(place.view(4, 2), place.clone(), torch.tensor([0, 8, 8, 8], dtype=torch.int32, device=device))


def _dual(t):
    return fwAD.make_dual(t, torch.ones_like(t))


# ------------------------------------------------- tangents and tracers, which a result made here would lose
def _followed(device):
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device=device)   # noqa: E731
    plan, off = _plan(device), torch.zeros(4, dtype=torch.int32, device=device)
    out = lambda rows, cols: z(rows, cols, dtype=torch.bfloat16)   # noqa: E731
    return {
        "sort": (lambda t: mm.sort_tokens_by_expert(t, plan), z(4, 8)),
        "sort that asks for a gradient": (lambda t: mm.sort_tokens_by_expert(t.requires_grad_(), plan), z(4, 8)),
        "sort with scales": (lambda t: mm.sort_tokens_by_expert(t, plan, z(4, 1, dtype=torch.uint8))[0], z(4, 128, dtype=E4)),
        "unsort, rows": (lambda t: mm.unsort_tokens_by_expert(t, plan), z(8, 8)),
        "unsort with weights, rows": (lambda t: mm.unsort_tokens_by_expert(t, plan, z(4, 2)), z(8, 8)),
        "unsort, weights": (lambda t: mm.unsort_tokens_by_expert(z(8, 8), plan, t), z(4, 2)),
        "product, x": (lambda t: mm.fp8_matmul(t, z(8, 128, dtype=E4)), z(4, 128, dtype=E4)),
        "product, w": (lambda t: mm.fp8_matmul(z(4, 128, dtype=E4), t), z(8, 128, dtype=E4)),
        "product, out": (lambda t: mm.fp8_matmul(z(4, 128, dtype=E4), z(8, 128, dtype=E4), out=t), out(4, 8)),
        "grouped product, x": (lambda t: mm.fp8_grouped_matmul(t, z(3, 8, 128, dtype=E4), off), z(4, 128, dtype=E4)),
    }


@pytest.mark.parametrize("name", list(_followed("cpu")))
def test_a_tangent_is_refused_not_dropped(name):
    call, t = _followed("cpu")[name]
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        call(_dual(t))
    with fwAD.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):   # torch carries tangents on there
        call(_dual(t))
    with fwAD.dual_level(), fwAD._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="CUDA"):   # nothing to lose
        call(_dual(t))


@pytest.mark.parametrize("name", list(_followed("cpu")))
def test_a_tracer_is_refused_not_given_a_constant(name):
    call, t = _followed("cpu")[name]
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, (t,))
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(call)(t)


def test_a_plan_is_not_traced():
    idx = torch.zeros((4, 2), dtype=torch.int64)
    for trace in (lambda f: torch.jit.trace(f, (idx,)), lambda f: make_fx(f)(idx)):
        with pytest.raises(RuntimeError, match="traced"):
            trace(lambda i: mm.plan_tokens_by_expert(i, 3))


@pytest.mark.gpu
def test_a_tangent_of_an_incoming_gradient_is_refused():
    plan, w = _plan("cuda"), torch.rand((4, 2), device="cuda")
    x, rows = torch.randn((4, 8), device="cuda", requires_grad=True), torch.randn((8, 8), device="cuda", requires_grad=True)
    for y, leaf in ((mm.sort_tokens_by_expert(x, plan), x), (mm.unsort_tokens_by_expert(rows, plan), rows),
                    (mm.unsort_tokens_by_expert(rows, plan, w), rows)):
        dy = torch.ones_like(y)
        with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, leaf, _dual(dy), retain_graph=True)
        torch.autograd.grad(y, leaf, dy)
    for name, (call, t) in _followed("cuda").items():
        with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            call(_dual(t))
        with fwAD.dual_level():   # a level without tangents
            call(t)


# --------------------------------------------------------- bounded waits and the kernels before a product
def _product_roles():
    """The text of every warp role of the product kernel, comments taken out."""
    path = os.path.join(os.path.dirname(os.path.abspath(_lib.__file__)), "csrc", "mxk_matmul.cuh")
    text = open(path).read()
    text = text[text.index("void mm_body("):text.index("nobody leaves while a partner")]
    parts = re.split(r"// -{20,} (TMA producer|MMA issuer|scale-tile builders|epilogue)\n", text)
    return {name: re.sub(r"//.*", "", body) for name, body in zip(parts[1::2], parts[2::2])}


@pytest.mark.parametrize("role, first", [("TMA producer", r"\bload\(sw"), ("MMA issuer", r"\bfor \(int t = unit"),
                                         ("scale-tile builders", r"\bload_word\(wx"), ("epilogue", r"\bfor \(int t = unit")])
def test_no_bounded_wait_of_a_product_begins_under_the_kernel_before_it(role, first):
    """A product may begin while the kernel in front of it still runs, for however long that takes; its waits are bounded.
    So each role has to pass grid_wait() ahead of its first load, or ahead of its first wait for somebody else's (the
    producer and the builders first wait for slots that are free at the start).  Read from the source: showing it on a GPU
    would take a kernel in front that runs for longer than the bound."""
    body = _product_roles()[role]
    assert "grid_wait();" in body and body.index("grid_wait();") < re.search(first, body).start()


# ------------------------------------------------------------------------------ sizes whose products pass 32 bits
@pytest.mark.gpu
@pytest.mark.parametrize("blocks", [(1 << 22) - 1, 1 << 22])
def test_scales_of_very_wide_rows(blocks):
    """600 rows of 2^22 bytes (one column of CTAs, which takes all 600 in one batch) with as many scale bytes, at an odd
    width copied byte by byte: 600 (2^22 - 1) = 2.5e9 copies of one CTA are more than 31 bits count."""
    tokens, hidden = 600, 1 << 22
    g = torch.Generator(device="cuda").manual_seed(blocks)
    idx = torch.randint(0, 3, (tokens, 1), device="cuda", generator=g)
    x = torch.randint(0, 256, (tokens, hidden), device="cuda", generator=g, dtype=torch.uint8)
    sf = torch.randint(0, 256, (tokens, blocks), device="cuda", generator=g, dtype=torch.uint8)
    plan = mm.plan_tokens_by_expert(idx, 2)
    rows, rows_sf = mm.sort_tokens_by_expert(x, plan, sf)
    order, end = torch.sort(idx[:, 0], stable=True).indices, int((idx < 2).sum())
    for first in range(0, end, 100):
        at = order[first:min(first + 100, end)]
        assert torch.equal(rows[first:first + len(at)], x[at]) and torch.equal(rows_sf[first:first + len(at)], sf[at])
    assert not rows[end:].any() and not rows_sf[end:].any()


# ---------------------------------------------------------- pairs dropped from the tables after the plan was made
def _over_capacity(tokens, topk, experts, capacity, both_tables):
    """A plan whose pairs beyond `capacity` of an expert are then dropped: (the tables, the pair of every row or -1)."""
    g = torch.Generator(device="cuda").manual_seed(tokens + topk)
    idx = torch.randint(-1, experts, (tokens, topk), device="cuda", generator=g)
    plan = mm.plan_tokens_by_expert(idx, experts)
    place = torch.arange(tokens * topk, device="cuda")
    owner = torch.searchsorted(plan.offsets[1:].contiguous(), place.int(), right=True).clamp(max=experts - 1)
    left = (plan.pair_of_row >= 0) & (place - plan.offsets[owner] < capacity)
    row = plan.row_of_pair
    dropped = (row >= 0) & ~left[row.clamp(min=0).long()]
    named = torch.where(left, plan.pair_of_row, -1)
    return plan._replace(row_of_pair=torch.where(dropped, -1, row), pair_of_row=named if both_tables else plan.pair_of_row), named.long()


def _soil(shape, dtype):
    """Leaves the allocator with a freed block of this size that holds NaN."""
    torch.full(shape, float("nan"), device="cuda").to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("both_tables", [False, True])
@pytest.mark.parametrize("tokens, topk, experts, capacity, hidden, dtype", [
    (40, 4, 5, 20, 64, torch.bfloat16), (300, 8, 16, 100, 127, torch.float16), (1000, 6, 60, 70, 1001, torch.float32),
    (1, 8, 2, 2, 6144, torch.bfloat16), (1, 8, 2, 1, 6144, torch.bfloat16), (4096, 256, 3, 200000, 3, torch.float16)])
def test_rows_of_pairs_dropped_after_the_plan_are_zero(tokens, topk, experts, capacity, hidden, dtype, both_tables):
    """In the sorted rows and in every gradient of rows: whatever stands there takes part in the experts' products and in
    the gradients of their weights."""
    plan, named = _over_capacity(tokens, topk, experts, capacity, both_tables)
    g = torch.Generator(device="cuda").manual_seed(5)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)   # noqa: E731
    x, w = rnd(tokens, hidden).to(dtype), rnd(tokens, topk)
    at, held = named.clamp(min=0), (named >= 0)[:, None]
    spread = torch.where(held, x[at // topk], torch.zeros((), dtype=dtype, device="cuda"))
    _soil((tokens * topk, hidden), dtype)
    assert torch.equal(mm.sort_tokens_by_expert(x, plan), spread)
    rows, weights = rnd(tokens * topk, hidden).to(dtype).requires_grad_(), w.requires_grad_()
    want = torch.where(held, (w.detach().view(-1)[at][:, None] * x[at // topk].float()).to(dtype), torch.zeros((), dtype=dtype, device="cuda"))
    y = mm.unsort_tokens_by_expert(rows, plan, weights)
    _soil((tokens * topk, hidden), dtype)
    drows, dw = torch.autograd.grad(y, (rows, weights), x)
    assert torch.equal(drows, want) and bool((dw[plan.row_of_pair < 0] == 0).all())   # one FP32 product, rounded once
    y = mm.unsort_tokens_by_expert(rows, plan)
    _soil((tokens * topk, hidden), dtype)
    assert torch.equal(torch.autograd.grad(y, rows, x)[0], spread)


@pytest.mark.gpu
@pytest.mark.parametrize("both_tables", [False, True])
@pytest.mark.parametrize("blocks", [1, 7, 48])
def test_scales_of_pairs_dropped_after_the_plan_are_zero(blocks, both_tables):
    plan, named = _over_capacity(100, 4, 6, 50, both_tables)
    x = torch.randint(1, 100, (100, 128 * blocks), device="cuda", dtype=torch.uint8)
    sf = torch.randint(1, 100, (100, blocks), device="cuda", dtype=torch.uint8)
    torch.full((400, 128 * blocks), 255, device="cuda", dtype=torch.uint8), torch.full((400, blocks), 255, device="cuda", dtype=torch.uint8)
    rows, rows_sf = mm.sort_tokens_by_expert(x, plan, sf)
    held = (named >= 0)[:, None]
    assert torch.equal(rows, torch.where(held, x[named.clamp(min=0) // 4], 0)) and torch.equal(rows_sf, torch.where(held, sf[named.clamp(min=0) // 4], 0))


# ------------------------------------------------------------------- a training step whose bound holds by construction
@pytest.mark.gpu
def test_training_step_with_the_routing_held():
    """Sort, two products with a relu between them, unsort, and all gradients, FP32 against 64 bits.  Routing and weights are
    inputs, the same ones in every run, so the run on magnitudes adds up the magnitude of every term that the signed run adds (relu
    passes all of them, at least what it passes there): a result that is a chain of n roundings of 2^-24 is off by at most
    n 2^-24 (1 + n 2^-24) of it, element for element.  n: both depths, topk, the rows (gradients of the experts' weights), one
    product each.  No relu may change its side: the values there are farther from zero than their own bound."""
    tokens, topk, experts, hidden, inter = 50, 3, 5, 24, 32
    g = torch.Generator().manual_seed(8)
    rnd = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    x, w1, w2, dy = rnd(tokens, hidden), rnd(experts, inter, hidden), rnd(experts, hidden, inter), rnd(tokens, hidden)
    weights, idx = torch.softmax(rnd(tokens, topk), 1), torch.randint(-1, experts, (tokens, topk), generator=g)
    idx[5] = -1
    flat = idx.view(-1)
    order = torch.sort(torch.where(flat < 0, experts, flat), stable=True).indices
    offsets = [0] + torch.tensor([int((flat == e).sum()) for e in range(experts)]).cumsum(0).tolist()
    inner = []

    def step(x, weights, w1, w2, dy, sort, unsort):
        rows = sort(x)
        parts = [rows[a:b] @ w1[e].t() for e, (a, b) in enumerate(zip(offsets, offsets[1:]))]
        inner.append(torch.cat(parts).detach().double().cpu())
        out = torch.cat([p.relu() @ w2[e].t() for e, p in enumerate(parts)] + [rows.new_zeros(rows.shape[0] - offsets[-1], hidden)])
        y = unsort(out, weights)
        return (y.detach(), *torch.autograd.grad(y, (x, weights, w1, w2), dy))

    def plain_unsort(out, weights):
        n = offsets[-1]
        parts = out[:n] * weights.reshape(-1)[order[:n], None]
        return torch.zeros(tokens, hidden, dtype=out.dtype).index_add(0, order[:n] // topk, parts)

    plan = mm.plan_tokens_by_expert(idx.cuda(), experts)
    assert plan.offsets.tolist() == offsets
    leaves = (x, weights, w1, w2)
    plain = lambda f, d: step(*[f(t.double()).requires_grad_() for t in leaves], d, lambda t: t[order // topk], plain_unsort)   # noqa: E731
    want, mass = plain(lambda t: t, dy.double()), plain(torch.abs, dy.double().abs())
    got = step(*[t.cuda().requires_grad_() for t in leaves], dy.cuda(), lambda t: mm.sort_tokens_by_expert(t, plan),
               lambda out, w: mm.unsort_tokens_by_expert(out, plan, w))
    assert bool((inner[0].abs() > hidden * 2.0 ** -23 * inner[1]).all())
    n = hidden + inter + topk + offsets[-1] + 5
    for name, a, b, m in zip(("y", "x", "weights", "w1", "w2"), got, want, mass):
        tol = n * 2.0 ** -24 * (1 + n * 2.0 ** -24) * m
        assert bool(((a.double().cpu() - b).abs() <= tol).all()), name


# ------------------------------------------------------------------------------- weights of one row, apart
def test_experts_of_one_row_may_be_apart():
    w, off = torch.zeros((3, 1, 160), dtype=E4)[..., :128], torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):     # of its layout there is nothing to say
        mm.fp8_grouped_matmul(torch.zeros((4, 128), dtype=E4), w, off)
    for bad in (torch.zeros((1, 1, 128), dtype=E4).expand(3, 1, 128), torch.zeros((3, 1, 136), dtype=E4)[..., :128]):
        with pytest.raises(ValueError, match="w needs"):
            mm.fp8_grouped_matmul(torch.zeros((4, 128), dtype=E4), bad, off)


@pytest.mark.gpu
def test_experts_of_one_row_apart():
    g = torch.Generator(device="cuda").manual_seed(1)
    small = lambda *s: torch.randint(-3, 4, s, device="cuda", generator=g).float().to(E4)   # noqa: E731
    x, w = small(50, 272), small(4, 3, 304)[:, 1:2, 16:288]
    off = torch.tensor([0, 20, 20, 45, 50], dtype=torch.int32, device="cuda")
    want = torch.cat([x[a:b].double() @ w[e].double().t() for e, (a, b) in enumerate(zip(off.tolist(), off.tolist()[1:]))])
    assert torch.equal(mm.fp8_grouped_matmul(x, w, off), want.to(torch.bfloat16))
