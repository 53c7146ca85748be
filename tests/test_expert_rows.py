"""Tokens sorted by expert and back: the plan's tables against a plain Python counting sort, the copies bit for
bit, the sums and gradients against 64-bit arithmetic, refusals (on the CPU: every check comes before the device).

Tolerances.  u = half a step of the result's type relative to the value (2^-8 bf16, 2^-11 fp16, 2^-24 fp32).
  * sort, drows of the plain sum: copies, equal bits.
  * y and dx: k products and sums in FP32, each off by at most 2^-24 of a partial sum that is at most
    A = sum |w| |rows|: |d| <= u |want| + (k + 1) 2^-24 A (1 + u).
  * drows: one FP32 product rounded once more: |d| <= (u + 2^-24) |want| (1 + u).
  * dweights: H products summed in FP32, in whatever order at most H additions deep:
    |d| <= (H + 1) 2^-24 sum |dy| |rows|.
"""
import numpy as np
import pytest
import torch

import mini_mega_b200 as mm
from mini_mega_b200 import _lib

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}   # smallest subnormal


def plain_plan(idx, experts, first=0):
    """Counting sort in plain Python: row_of_pair, pair_of_row, offsets."""
    flat = [int(e) - first for e in np.asarray(idx).reshape(-1)]
    lists = [[] for _ in range(experts)]
    for p, e in enumerate(flat):
        if 0 <= e < experts:
            lists[e].append(p)
    row_of_pair, pair_of_row, offsets, row = [-1] * len(flat), [-1] * len(flat), [0], 0
    for group in lists:
        for p in group:
            row_of_pair[p], pair_of_row[row] = row, p
            row += 1
        offsets.append(row)
    return (torch.tensor(row_of_pair, dtype=torch.int32).view(np.asarray(idx).shape),
            torch.tensor(pair_of_row, dtype=torch.int32), torch.tensor(offsets, dtype=torch.int32))


def routing(seed, tokens, topk, experts, drop=0.0, hot=False):
    rng = np.random.default_rng(seed)
    idx = rng.integers(0, experts, (tokens, topk))
    if hot:
        idx[rng.random((tokens, topk)) < 0.7] = experts // 2
    if drop:
        idx[rng.random((tokens, topk)) < drop] = -1
    return torch.from_numpy(idx)


def table_device(idx, experts, first=0):
    return mm.ExpertPlan(*[t.cuda() for t in plain_plan(idx, experts, first)])


# ------------------------------------------------------------------------------ refusals
def _cpu_plan(tokens=4, topk=2, experts=3):
    return mm.ExpertPlan(*plain_plan(np.zeros((tokens, topk), np.int64), experts))


@pytest.fixture(scope="module")
def built():
    _lib.build()


@pytest.mark.parametrize("make, err", [
    (lambda: mm.plan_tokens_by_expert(torch.zeros(4, 2), 3), TypeError),
    (lambda: mm.plan_tokens_by_expert(torch.zeros(4, dtype=torch.int64), 3), ValueError),
    (lambda: mm.plan_tokens_by_expert(torch.zeros((4, 0), dtype=torch.int64), 3), ValueError),
    (lambda: mm.plan_tokens_by_expert(torch.zeros((4, 257), dtype=torch.int64), 3), ValueError),
    (lambda: mm.plan_tokens_by_expert(torch.zeros((4, 2), dtype=torch.int64), 0), ValueError),
    (lambda: mm.plan_tokens_by_expert(torch.zeros((4, 2), dtype=torch.int64), 1025), ValueError),
    (lambda: mm.plan_tokens_by_expert(torch.zeros((4, 2), dtype=torch.int64), 3, -1), ValueError),
    (lambda: mm.plan_tokens_by_expert(torch.zeros((1, 1), dtype=torch.int64).expand(1 << 23, 256), 3), ValueError),
    (lambda: mm.plan_tokens_by_expert(torch.zeros((4, 2), dtype=torch.int64), 3), ValueError),   # a CPU tensor
    (lambda: mm.sort_tokens_by_expert(torch.zeros(5, 8), _cpu_plan()), ValueError),
    (lambda: mm.sort_tokens_by_expert(torch.zeros(4, 0), _cpu_plan()), ValueError),
    (lambda: mm.sort_tokens_by_expert(torch.zeros(4, 8, dtype=torch.float64), _cpu_plan()), TypeError),
    (lambda: mm.sort_tokens_by_expert(torch.zeros(4, 8), _cpu_plan(), torch.zeros(4, 1, dtype=torch.uint8)), TypeError),
    (lambda: mm.sort_tokens_by_expert(torch.zeros(4, 8, dtype=torch.uint8), _cpu_plan(), torch.zeros(3, 1, dtype=torch.uint8)), ValueError),
    (lambda: mm.sort_tokens_by_expert(torch.zeros(4, 8), _cpu_plan()), ValueError),
    (lambda: mm.sort_tokens_by_expert(torch.zeros(4, 8), _cpu_plan()._replace(offsets=torch.zeros(1, dtype=torch.int32))), ValueError),
    (lambda: mm.sort_tokens_by_expert(torch.zeros(4, 8), _cpu_plan()._replace(offsets=torch.zeros(4))), TypeError),
    (lambda: mm.sort_tokens_by_expert(torch.zeros(4, 8), _cpu_plan()._replace(pair_of_row=torch.zeros(7, dtype=torch.int32))), ValueError),
    (lambda: mm.sort_tokens_by_expert(torch.zeros(2, 8), _cpu_plan()._replace(row_of_pair=torch.zeros(2, 4, dtype=torch.int32).t())), ValueError),
    (lambda: mm.unsort_tokens_by_expert(torch.zeros(7, 8), _cpu_plan()), ValueError),
    (lambda: mm.unsort_tokens_by_expert(torch.zeros(8, 8, dtype=torch.uint8), _cpu_plan()), TypeError),
    (lambda: mm.unsort_tokens_by_expert(torch.zeros(8, 8), _cpu_plan(), torch.zeros(4, 2, dtype=torch.bfloat16)), TypeError),
    (lambda: mm.unsort_tokens_by_expert(torch.zeros(8, 8), _cpu_plan(), torch.zeros(2, 4)), ValueError),
    (lambda: mm.unsort_tokens_by_expert(torch.zeros(8, 8), _cpu_plan(), torch.zeros(4, 2)), ValueError),
])
def test_refusals(built, make, err):
    with pytest.raises(err):
        make()


def test_c_abi_refuses_before_it_launches():
    _lib.build()
    L = _lib.lib()
    one = 16   # a pointer that is never followed: every call below is refused on its sizes
    assert L.mxk_plan_tokens(one, 8, 2, 4, 2, 0, 1025, one, one, one, None) == -1
    assert L.mxk_plan_tokens(one, 3, 2, 4, 2, 0, 8, one, one, one, None) == -1
    assert L.mxk_plan_tokens(None, 8, 2, 4, 2, 0, 8, one, one, one, None) == -1
    assert L.mxk_sort_tokens(one, 16, 0, None, 0, 0, 4, 2, 8, one, one, one, None, None) == -1
    assert L.mxk_sort_tokens(one, 16, 16, one, 1, 1, 4, 2, 8, one, one, one, None, None) == -1
    assert L.mxk_unsort_tokens(one, 3, 16, None, 0, 4, 2, 8, one, one, None) == -1
    assert L.mxk_unsort_tokens(17, 0, 16, None, 0, 4, 2, 8, one, one, None) == -1
    assert L.mxk_unsort_tokens_grad(one, 16, None, 16, 0, one, 2, 4, 2, 8, 8, one, one, one, one, None) == -1
    # addresses off their element's alignment, which would fault
    assert L.mxk_plan_tokens(20, 8, 2, 4, 2, 0, 8, one, one, one, None) == -1
    assert L.mxk_plan_tokens(18, 4, 2, 4, 2, 0, 8, one, one, one, None) == -1
    for tables in ((18, 16, 16), (16, 18, 16), (16, 16, 18)):
        assert L.mxk_plan_tokens(one, 8, 2, 4, 2, 0, 8, *tables, None) == -1
    assert L.mxk_sort_tokens(one, 16, 16, None, 0, 0, 4, 2, 8, 18, one, one, None, None) == -1
    assert L.mxk_sort_tokens(one, 16, 16, None, 0, 0, 4, 2, 8, one, 18, one, None, None) == -1
    assert L.mxk_unsort_tokens(one, 0, 16, 18, 2, 4, 2, 8, one, one, None) == -1
    assert L.mxk_unsort_tokens(one, 0, 16, one, 2, 4, 2, 8, 18, one, None) == -1
    for k in (5, 11, 12, 14):
        args = [one, 16, one, 16, 0, one, 2, 4, 2, 8, 8, one, one, one, one, None]
        args[k] = 18
        assert L.mxk_unsort_tokens_grad(*args) == -1, k
    assert len(L.mxk_last_error()) > 0


# ---------------------------------------------------------------------------------- plan
@pytest.mark.gpu
@pytest.mark.parametrize("tokens, topk, experts, drop, hot", [
    (1, 1, 1, 0.0, False), (1, 8, 256, 0.0, False), (16, 8, 32, 0.3, False), (31, 3, 7, 0.1, False),
    (128, 8, 256, 0.0, False), (512, 8, 64, 0.0, True), (513, 8, 64, 0.1, True), (4096, 8, 1024, 0.05, False),
    (5000, 7, 1000, 0.0, True), (40000, 8, 33, 0.02, True), (700, 256, 5, 0.0, False), (64, 4, 9, 1.0, False),
])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_plan(tokens, topk, experts, drop, hot, dtype):
    idx = routing(tokens + topk, tokens, topk, experts, drop, hot)
    plan = mm.plan_tokens_by_expert(idx.to(dtype).cuda(), experts)
    for got, want in zip(plan, plain_plan(idx, experts)):
        assert torch.equal(got.cpu(), want)


@pytest.mark.gpu
def test_plan_of_one_ranks_experts_strides_and_far_ids():
    idx = routing(3, 200, 6, 64)
    idx[5, 1], idx[6, 0], idx[7, 2] = 2 ** 62, -2 ** 62, 2 ** 32 + 20     # no expert of anybody
    wide = torch.full((200, 11), 17, dtype=torch.int64)
    wide[:, :6] = idx
    for view in (wide.cuda()[:, :6], idx.cuda(), idx.t().contiguous().cuda().t()):
        plan = mm.plan_tokens_by_expert(view, 16, first_expert=16)
        for got, want in zip(plan, plain_plan(idx, 16, 16)):
            assert torch.equal(got.cpu(), want)


@pytest.mark.gpu
def test_no_tokens():
    plan = mm.plan_tokens_by_expert(torch.zeros((0, 4), dtype=torch.int64, device="cuda"), 5)
    assert plan.offsets.tolist() == [0] * 6 and plan.row_of_pair.shape == (0, 4)
    x = torch.zeros((0, 64), device="cuda", requires_grad=True)
    rows = mm.sort_tokens_by_expert(x, plan)
    y = mm.unsort_tokens_by_expert(rows, plan, torch.zeros((0, 4), device="cuda"))
    y.sum().backward()
    assert rows.shape == (0, 64) and y.shape == (0, 64) and x.grad.shape == (0, 64)


# ---------------------------------------------------------------------------------- sort
def _random(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    if dtype.is_floating_point and dtype.itemsize > 1:
        return torch.randn(shape, generator=g).to(dtype)
    return torch.randint(0, 256, shape, generator=g, dtype=torch.uint8).view(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.uint8])
@pytest.mark.parametrize("tokens, topk, experts, hidden, drop", [
    (1, 1, 1, 1, 0.0), (1, 8, 256, 6144, 0.0), (3, 2, 4, 127, 0.4), (37, 5, 9, 1000, 0.1), (300, 8, 16, 16, 0.0),
    (129, 3, 12, 8, 0.2), (2, 1, 3, 40000, 0.0), (9, 2, 3, 64, 1.0),
])
def test_sort_is_a_copy(dtype, tokens, topk, experts, hidden, drop):
    idx = routing(hidden, tokens, topk, experts, drop)
    x = _random((tokens, hidden), dtype, 1)
    row_of_pair, pair_of_row, offsets = plain_plan(idx, experts)
    rows = mm.sort_tokens_by_expert(x.cuda(), table_device(idx, experts)).cpu()
    want = x.view(torch.uint8).view(tokens, -1)[pair_of_row.clamp(min=0) // topk]
    want[pair_of_row < 0] = 0
    assert torch.equal(rows.view(torch.uint8).view(tokens * topk, -1), want)


@pytest.mark.gpu
@pytest.mark.parametrize("blocks", [1, 3, 8, 48, 56])
def test_sort_carries_scales_and_reads_views(blocks):
    tokens, topk, experts = 21, 4, 6
    idx = routing(blocks, tokens, topk, experts, 0.15)
    x = _random((tokens, 128 * blocks + 16), torch.float8_e4m3fn, 2)
    sf = _random((tokens, blocks + 5), torch.uint8, 3)
    _, pair_of_row, _ = plain_plan(idx, experts)
    rows, rows_sf = mm.sort_tokens_by_expert(x.cuda()[:, 16:], table_device(idx, experts), sf.cuda()[:, 2:2 + blocks])
    at, held = pair_of_row.clamp(min=0) // topk, (pair_of_row >= 0)[:, None]
    zero = torch.zeros((), dtype=torch.uint8)
    assert torch.equal(rows.cpu().view(torch.uint8), torch.where(held, x.view(torch.uint8)[at, 16:], zero))
    assert torch.equal(rows_sf.cpu(), torch.where(held, sf[at, 2:2 + blocks], zero))


@pytest.mark.gpu
def test_entries_out_of_range_count_as_dropped():
    idx = routing(8, 12, 3, 4)
    plan = table_device(idx, 4)
    bad = plan.row_of_pair.clone()
    bad[2, 1], bad[3, 0], bad[4, 2] = 36, 2 ** 31 - 1, -2 ** 31
    hole = torch.where((bad < 0) | (bad >= 36), -1, bad)
    x, w = torch.randn(12, 50, device="cuda"), torch.rand(12, 3, device="cuda")
    rows = torch.randn(36, 50, device="cuda")
    one, two = plan._replace(row_of_pair=bad), plan._replace(row_of_pair=hole)
    assert torch.equal(mm.unsort_tokens_by_expert(rows, one, w), mm.unsort_tokens_by_expert(rows, two, w))
    held = hole.view(-1)[hole.view(-1) >= 0].long()
    assert torch.equal(mm.sort_tokens_by_expert(x, one)[held], mm.sort_tokens_by_expert(x, two)[held])
    wild = plan._replace(offsets=torch.tensor([0, 9, -5, 2 ** 31 - 1, 2 ** 31 - 1], dtype=torch.int32, device="cuda"))
    assert torch.equal(mm.sort_tokens_by_expert(x, wild), mm.sort_tokens_by_expert(x, plan))


# --------------------------------------------------------------------- sums and gradients
def _close(got, want, tol):
    d = (got.double().cpu() - want).abs()
    assert bool((d <= tol).all()), f"{int((d > tol).sum())} of {d.numel()} off, worst by a factor of {float((d / tol.clamp_min(1e-300)).max()):.3g}"


SHAPES = [(1, 1, 1, 1, 0.0), (1, 8, 64, 6144, 0.0), (5, 3, 4, 127, 0.4), (40, 8, 9, 1000, 0.1), (33, 11, 16, 130, 0.2),
          (260, 2, 12, 8, 0.1), (9, 2, 3, 64, 1.0), (3, 17, 8, 9000, 0.1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens, topk, experts, hidden, drop", SHAPES)
def test_unsort_and_its_gradients(dtype, tokens, topk, experts, hidden, drop):
    idx = routing(hidden + topk, tokens, topk, experts, drop)
    row_of_pair, pair_of_row, offsets = plain_plan(idx, experts)
    rows, dy = _random((tokens * topk, hidden), dtype, 4), _random((tokens, hidden), dtype, 5)
    w = _random((tokens, topk), torch.float32, 6)
    held, at = row_of_pair >= 0, row_of_pair.clamp(min=0).long()
    u, tiny = U[dtype], TINY[dtype]

    gr, gw = rows.cuda().requires_grad_(), w.cuda().requires_grad_()
    plan = table_device(idx, experts)
    y = mm.unsort_tokens_by_expert(gr, plan, gw)
    drows, dw = torch.autograd.grad(y, (gr, gw), dy.cuda())

    parts = torch.where(held, w, 0.0).double()[:, :, None] * rows.double()[at]
    want, mass = parts.sum(1), parts.abs().sum(1)
    _close(y, want, u * want.abs() + (topk + 1) * 2.0 ** -24 * mass * (1 + u) + tiny)
    factor = torch.where(pair_of_row >= 0, w.view(-1)[pair_of_row.clamp(min=0).long()], 0.0).double()
    want = factor[:, None] * dy.double()[pair_of_row.clamp(min=0).long() // topk]
    _close(drows, want, (u + 2.0 ** -24) * (1 + u) * want.abs() + tiny)
    dots = dy.double()[:, None, :] * rows.double()[at]
    want, mass = torch.where(held, dots.sum(2), 0.0), dots.abs().sum(2)
    _close(dw, want, (hidden + 1) * 2.0 ** -24 * mass + TINY[torch.float32])
    # each gradient alone, and the plain sum with its gradient
    only_r, = torch.autograd.grad(mm.unsort_tokens_by_expert(gr, plan, w.cuda()), gr, dy.cuda())
    only_w, = torch.autograd.grad(mm.unsort_tokens_by_expert(rows.cuda(), plan, gw), gw, dy.cuda())
    assert torch.equal(only_r, drows) and torch.equal(only_w, dw)
    plain = mm.unsort_tokens_by_expert(gr, plan)
    parts = torch.where(held[:, :, None], rows.double()[at], 0.0)
    _close(plain, parts.sum(1), u * parts.sum(1).abs() + (topk + 1) * 2.0 ** -24 * parts.abs().sum(1) * (1 + u) + tiny)
    spread, = torch.autograd.grad(plain, gr, dy.cuda())
    assert torch.equal(spread.cpu(), torch.where((pair_of_row >= 0)[:, None], dy[pair_of_row.clamp(min=0).long() // topk], torch.zeros((), dtype=dtype)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens, topk, experts, hidden, drop", SHAPES)
def test_gradient_of_sort(dtype, tokens, topk, experts, hidden, drop):
    idx = routing(hidden + topk, tokens, topk, experts, drop)
    row_of_pair, _, _ = plain_plan(idx, experts)
    drows = _random((tokens * topk, hidden), dtype, 7)
    x = _random((tokens, hidden), dtype, 8).cuda().requires_grad_()
    dx, = torch.autograd.grad(mm.sort_tokens_by_expert(x, table_device(idx, experts)), x, drows.cuda())
    parts = torch.where((row_of_pair >= 0)[:, :, None], drows.double()[row_of_pair.clamp(min=0).long()], 0.0)
    want = parts.sum(1)
    _close(dx, want, U[dtype] * want.abs() + (topk + 1) * 2.0 ** -24 * parts.abs().sum(1) * (1 + U[dtype]) + TINY[dtype])


@pytest.mark.gpu
def test_gradients_against_differences():
    """(f(v + h d) - f(v - h d)) / 2h is exact for a form that is linear in v up to FP32 rounding: with h = 1 the
    difference of two sums is off by at most 2 (n + 2) 2^-24 of their mass, n = 2000 terms, |value| <= 10 each."""
    idx = routing(11, 20, 4, 5, 0.2).cuda()
    plan = mm.plan_tokens_by_expert(idx, 5)
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)   # noqa: E731
    x, w, c = rnd(20, 25).requires_grad_(), rnd(20, 4).requires_grad_(), rnd(20, 25)
    f = lambda x_, w_: (mm.unsort_tokens_by_expert(mm.sort_tokens_by_expert(x_, plan) * 1.5, plan, w_).double() * c).sum()   # noqa: E731
    gx, gw = torch.autograd.grad(f(x, w), (x, w))
    for v, grad, ahead in ((x, gx, lambda d: f(x + d, w) - f(x - d, w)), (w, gw, lambda d: f(x, w + d) - f(x, w - d))):
        d = rnd(*v.shape)
        diff = float(ahead(d).detach()) / 2
        assert abs(diff - float((grad.double() * d).sum())) <= 2 * 2002 * 2.0 ** -24 * 500 * 10


@pytest.mark.gpu
def test_second_derivatives():
    """Sort and plain unsort are linear: differentiating their gradients again works; the weighted sum refuses."""
    plan = table_device(routing(4, 6, 3, 4, 0.2), 4)
    x = torch.randn(6, 20, device="cuda", requires_grad=True)
    c = torch.randn(6, 20, device="cuda", requires_grad=True)
    y = mm.unsort_tokens_by_expert(mm.sort_tokens_by_expert(x, plan), plan)       # x times its number of kept pairs
    gx, = torch.autograd.grad(y, x, c, create_graph=True)
    kept = (plan.row_of_pair >= 0).sum(1, keepdim=True).float()
    gc, = torch.autograd.grad(gx.sum(), c)
    assert torch.equal(gc, kept.expand(6, 20))
    rows = torch.randn(18, 20, device="cuda", requires_grad=True)
    y = mm.unsort_tokens_by_expert(rows, plan, torch.rand(6, 3, device="cuda"))
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y, rows, c, create_graph=True)


@pytest.mark.gpu
def test_masked_places_do_not_matter():
    """NaN and infinity behind the last row, and in rows and tokens whose pairs are dropped, reach no result."""
    idx = routing(12, 16, 4, 6, 0.3)
    idx[3] = -1                                   # a token without any expert
    plan = table_device(idx, 6)
    end = int(plan.offsets[-1])
    rows = torch.randn(64, 70, device="cuda").bfloat16()
    rows[end:] = float("nan")
    rows.requires_grad_()
    w = torch.rand(16, 4, device="cuda")
    w[idx.cuda() < 0] = float("inf")
    w.requires_grad_()
    y = mm.unsort_tokens_by_expert(rows, plan, w)
    assert bool(torch.isfinite(y).all()) and bool((y[3] == 0).all())
    dy = torch.randn(16, 70, device="cuda").bfloat16()
    dy[3] = float("nan")
    drows, dw = torch.autograd.grad(y, (rows, w), dy)
    assert bool(torch.isfinite(drows).all()) and bool((drows[end:] == 0).all())
    assert bool(torch.isfinite(dw).all()) and bool((dw[idx.cuda() < 0] == 0).all())
    # and where a pair is kept, NaN and infinity pass through
    rows2 = torch.ones(64, 70, device="cuda")
    rows2[0, 0], rows2[1, 1] = float("nan"), float("inf")
    y2 = mm.unsort_tokens_by_expert(rows2, plan, torch.ones(16, 4, device="cuda"))
    t0, t1 = (int(plan.pair_of_row[i]) // 4 for i in (0, 1))
    assert bool(torch.isnan(y2[t0, 0])) and bool(torch.isinf(y2[t1, 1]))


@pytest.mark.gpu
def test_gradients_of_broadcast_and_strided_inputs():
    idx = routing(13, 10, 3, 4, 0.1)
    plan = table_device(idx, 4)
    base = torch.randn(1, 48, device="cuda", requires_grad=True)
    rows = mm.sort_tokens_by_expert(base.expand(10, 48), plan)        # one row for every token
    y = mm.unsort_tokens_by_expert(rows, plan)
    y.sum().backward()                                                # an expanded gradient
    kept = int((idx >= 0).sum())
    assert torch.equal(base.grad, torch.full((1, 48), float(kept), device="cuda"))
    wide = torch.randn(30, 96, device="cuda")
    w = torch.rand(3, 10, device="cuda").t()                          # weights laid out the other way
    dy = torch.randn(48, 10, device="cuda").t()
    for strided in (wide[:, 16:64], wide[:, 1:49], wide[:, ::2]):
        a, b = strided.detach().requires_grad_(), strided.contiguous().detach().requires_grad_()
        wa, wb = w.detach().requires_grad_(), w.contiguous().detach().requires_grad_()
        ya, yb = mm.unsort_tokens_by_expert(a, plan, wa), mm.unsort_tokens_by_expert(b, plan, wb)
        assert torch.equal(ya, yb)
        (ra, ga), (rb, gb) = torch.autograd.grad(ya, (a, wa), dy), torch.autograd.grad(yb, (b, wb), dy.contiguous())
        assert torch.equal(ra, rb)
        # the dots' order of summation follows the width of the loads, which follows the alignment: two FP32 sums of
        # H products, each within (H + 1) 2^-24 of the mass of the exact one
        at = plan.row_of_pair.clamp(min=0).long()
        mass = (dy.double().abs()[:, None] * b.double().abs()[at]).sum(2).cpu()
        _close(ga, gb.double().cpu(), 2 * 49 * 2.0 ** -24 * mass)


@pytest.mark.gpu
def test_rows_behind_two_to_the_31_elements():
    """Element offsets of the last rows pass 32 bits: 270000 rows of 8192 bytes."""
    tokens, topk, hidden = 270000, 1, 8192
    idx = torch.zeros((tokens, topk), dtype=torch.int64, device="cuda")
    idx[: tokens // 2] = 1
    plan = mm.plan_tokens_by_expert(idx, 2)
    x = torch.zeros((tokens, hidden), dtype=torch.uint8, device="cuda")
    x[:, 0] = torch.arange(tokens, device="cuda") % 251
    x[:, -1] = torch.arange(tokens, device="cuda") % 241
    rows = mm.sort_tokens_by_expert(x, plan)
    at = plan.pair_of_row.long()
    assert torch.equal(rows[:, 0], x[at, 0]) and torch.equal(rows[:, -1], x[at, -1])
    back = mm.unsort_tokens_by_expert(rows.view(torch.float16), plan)
    # a sum of one value: equal as numbers (0 + -0 is +0, a NaN keeps no payload)
    want = x.view(torch.float16)
    assert bool(((back == want) | (torch.isnan(back) & torch.isnan(want))).all())


# ------------------------------------------------------------------- streams, graphs, repeats
@pytest.mark.gpu
def test_captured_replayed_and_run_on_two_streams():
    g = torch.Generator(device="cuda").manual_seed(5)
    idx = torch.randint(-1, 16, (64, 4), device="cuda", generator=g)
    x = torch.randn(64, 512, device="cuda", generator=g).bfloat16()
    w = torch.rand(64, 4, device="cuda", generator=g)
    dy = torch.randn(64, 512, device="cuda", generator=g).bfloat16()

    def step(idx, x, w, dy):
        plan = mm.plan_tokens_by_expert(idx, 16)
        xs, ws = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = mm.unsort_tokens_by_expert(mm.sort_tokens_by_expert(xs, plan), plan, ws)
        return (y.detach(), *torch.autograd.grad(y, (xs, ws), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(idx, x, w, dy)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step(idx, x, w, dy)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (6, 7):
        g.manual_seed(seed)
        idx.copy_(torch.randint(-1, 16, (64, 4), device="cuda", generator=g))
        x.copy_(torch.randn(64, 512, device="cuda", generator=g))
        graph.replay()
        want = step(idx, x, w, dy)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step(idx, x, w, dy)
        again = step(idx, x, w, dy)
        torch.cuda.synchronize()
        for a, b, c, d in zip(held, want, other, again):
            assert torch.equal(a, b) and torch.equal(c, b) and torch.equal(d, b)


@pytest.mark.gpu
def test_capture_with_a_live_graph_of_the_same_leaf_is_refused():
    idx = routing(1, 8, 2, 3).cuda()
    plan = mm.plan_tokens_by_expert(idx, 3)
    x = torch.randn(8, 32, device="cuda", requires_grad=True)
    alive = mm.sort_tokens_by_expert(x, plan)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph):
            mm.sort_tokens_by_expert(x, plan)
    torch.cuda.synchronize()
    alive.sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2.0))
    del alive
    x.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad, = torch.autograd.grad(mm.sort_tokens_by_expert(x, plan).sum(), x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(grad, torch.full_like(x, 2.0))
