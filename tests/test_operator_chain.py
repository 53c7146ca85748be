"""The operators beside the layer used together: the layer taken apart against the layer itself, and a
training step through sort, the experts' products and unsort against 64-bit arithmetic.

Tolerances.
  * apart against the layer: the same products and the same E4M3 requantisation, but the first product is rounded to bf16
    (2^-8 relative) before SwiGLU.  SwiGLU passes at most 2.2 times that on (its factor silu has slope below 1.1), so a hidden
    value is off by at most 2^-6.8; the two requantised values then differ only where a border lies between them, with
    probability at most 2^-6.8 / 2^-4 per value (steps are 2^-4 .. 2^-3 of a value), and by one step of at most 2^-3: a
    root mean square of 2^-3 sqrt(2^-2.8) = 0.047 of the hidden values, and as much, relatively, of the sums over them.
    The bf16 rows and the result add 2^-8.  Bound: 2^-4 in relative L2.
  * training step: FP32 all through; every result is a chain of at most n additions and products of terms whose
    magnitudes sum to `mass`: |d| <= n 2^-24 mass, with n the longest chain (depth of both products, topk, rows).
"""
import numpy as np
import pytest
import torch

import mini_mega_b200 as mm
from mini_mega_b200 import quant
from oracle import oracle as orc

pytestmark = pytest.mark.gpu


def _apart(x, x_sf, idx, weights, l1, l2, experts, first=0):
    plan = mm.plan_tokens_by_expert(idx, experts, first)
    rows = mm.sort_tokens_by_expert(x, plan, x_sf)
    h = mm.fp8_grouped_matmul(rows, l1, plan.offsets).float()
    inter = h.shape[1] // 2
    a = torch.nn.functional.silu(h[:, :inter]) * h[:, inter:]
    out = mm.fp8_grouped_matmul(quant.per_token_cast_to_fp8(a), l2, plan.offsets)
    return mm.unsort_tokens_by_expert(out, plan, weights)


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.view(dtype)


@pytest.mark.parametrize("tokens, experts, topk, hidden, inter", [(1, 8, 2, 512, 256), (40, 8, 2, 512, 256), (300, 4, 3, 768, 384)])
def test_layer_taken_apart(tokens, experts, topk, hidden, inter):
    case = orc.gen_case(1, experts, topk, hidden, inter, tokens, seed=tokens, routing="logits", scaled=True)
    buf = mm.get_symm_buffer_for_mega_moe(None, experts, tokens, topk, hidden, inter)
    try:
        x, x_sf = _dev(case.x[0][:tokens], torch.float8_e4m3fn), _dev(case.x_sf[0][:tokens])
        idx, weights = _dev(case.topk_idx[0][:tokens]), _dev(case.topk_w[0][:tokens])
        buf.x[:tokens].copy_(x)
        buf.x_sf[:tokens].copy_(x_sf)
        buf.topk_idx[:tokens].copy_(idx)
        buf.topk_weights[:tokens].copy_(weights)
        l1, l2 = mm.transform_weights_for_mega_moe((_dev(case.w1), _dev(case.w1_sf)), (_dev(case.w2), _dev(case.w2_sf)))
        y = torch.empty((tokens, hidden), dtype=torch.bfloat16, device="cuda")
        mm.fp8_mega_moe(y, l1, l2, buf)
        got = _apart(x, x_sf, idx, weights, l1, l2, experts)
        torch.cuda.synchronize()
        assert buf.status().status == 0 and mm.matmul_status() == 0
        assert orc.rel_l2(got.float().cpu().numpy(), y.float().cpu().numpy()) <= 2.0 ** -4
        # two halves of the experts, as two ranks would hold them, add up to the whole (their sums are rounded apart)
        half = experts // 2
        part = sum(_apart(x, x_sf, idx, weights, tuple(t[f:f + half] for t in l1), tuple(t[f:f + half] for t in l2), half, f).float()
                   for f in (0, half))
        assert orc.rel_l2(part.cpu().numpy(), got.float().cpu().numpy()) <= 2.0 ** -7
    finally:
        buf.destroy()


def test_capture_of_the_whole_run_follows_its_inputs():
    """Plan, sort, both products and unsort in one graph: another routing and other tokens at replay."""
    case = orc.gen_case(1, 8, 2, 512, 256, 64, seed=3, routing="logits", scaled=True)
    x, x_sf = _dev(case.x[0][:64], torch.float8_e4m3fn), _dev(case.x_sf[0][:64])
    idx, weights = _dev(case.topk_idx[0][:64]), _dev(case.topk_w[0][:64])
    l1, l2 = (_dev(case.w1).view(torch.float8_e4m3fn), _dev(case.w1_sf)), (_dev(case.w2).view(torch.float8_e4m3fn), _dev(case.w2_sf))
    _apart(x, x_sf, idx, weights, l1, l2, 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _apart(x, x_sf, idx, weights, l1, l2, 8)
    for _ in range(3):
        idx.copy_(torch.randint(-1, 8, idx.shape, device="cuda"))
        x.view(torch.uint8).copy_(x.view(torch.uint8)[torch.randperm(64, device="cuda")])
        graph.replay()
        assert torch.equal(held, _apart(x, x_sf, idx, weights, l1, l2, 8))


def test_branches_that_join_and_copies_in_a_graph():
    """Kernels behind copies from the host, on three streams, and with two predecessors: eager and captured."""
    gen = torch.Generator().manual_seed(9)
    tokens, hidden, topk, experts, cols = 300, 512, 8, 16, 384
    host_idx = torch.randint(0, experts, (tokens, topk), generator=gen).pin_memory()
    host_x = torch.randint(-8, 9, (tokens, hidden), generator=gen).to(torch.bfloat16).pin_memory()
    q = torch.randint(-3, 4, (tokens, hidden), generator=gen).float().cuda().to(torch.float8_e4m3fn)
    w = torch.randint(-3, 4, (cols, hidden), generator=gen).float().cuda().to(torch.float8_e4m3fn)
    all_w = w.expand(experts, cols, hidden).contiguous()
    idx, x = torch.zeros((tokens, topk), dtype=torch.int64, device="cuda"), torch.zeros((tokens, hidden), dtype=torch.bfloat16, device="cuda")
    streams = torch.cuda.Stream(), torch.cuda.Stream()

    def run():
        here = torch.cuda.current_stream()
        idx.copy_(host_idx, non_blocking=True)
        plan = mm.plan_tokens_by_expert(idx, experts)
        for s in streams:
            s.wait_stream(here)
        with torch.cuda.stream(streams[0]):
            x.copy_(host_x, non_blocking=True)
            dense = mm.fp8_matmul(q, w)
        with torch.cuda.stream(streams[1]):
            grouped = mm.fp8_grouped_matmul(mm.sort_tokens_by_expert(q, plan), all_w, plan.offsets)
        here.wait_stream(streams[0])
        rows = mm.sort_tokens_by_expert(x, plan)
        here.wait_stream(streams[1])
        return dense, rows, mm.unsort_tokens_by_expert(rows, plan), mm.unsort_tokens_by_expert(grouped, plan)

    product = (q.double() @ w.double().t()).to(torch.bfloat16)
    order = torch.sort(host_idx.reshape(-1), stable=True).indices // topk
    want = (product, host_x[order].cuda(), (host_x.float() * topk).to(torch.bfloat16).cuda(), (product.float() * topk).to(torch.bfloat16))
    run()
    torch.cuda.synchronize()
    for got, w_ in zip(run(), want):
        torch.cuda.synchronize()
        assert torch.equal(got, w_)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for _ in range(10):
        for t in (idx, x, *held):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for got, w_ in zip(held, want):
            assert torch.equal(got, w_)
    assert mm.matmul_status() == 0


def test_inference_mode_and_sign_flag_views():
    """Tables, rows and results made in inference mode; inputs that are views with their sign in a flag."""
    case = orc.gen_case(1, 8, 2, 512, 256, 33, seed=5, routing="logits", scaled=True)
    x, x_sf = _dev(case.x[0][:33], torch.float8_e4m3fn), _dev(case.x_sf[0][:33])
    idx, weights = _dev(case.topk_idx[0][:33]), _dev(case.topk_w[0][:33])
    l1, l2 = (_dev(case.w1).view(torch.float8_e4m3fn), _dev(case.w1_sf)), (_dev(case.w2).view(torch.float8_e4m3fn), _dev(case.w2_sf))
    want = _apart(x, x_sf, idx, weights, l1, l2, 8)
    with torch.inference_mode():
        plan = mm.plan_tokens_by_expert(idx, 8)
        got = _apart(x, x_sf, idx, weights, l1, l2, 8)
        out = torch.zeros((33, 512), dtype=torch.bfloat16, device="cuda")
        assert mm.fp8_matmul(x, l1[0][0], out=out) is not None
        assert plan.offsets.is_inference() and out.is_inference()
        assert torch.equal(out, mm.fp8_matmul(x, l1[0][0]))
        assert torch.equal(got, want)
    flagged = torch.view_as_complex(torch.arange(33 * 20 * 2, device="cuda").float().view(33, 20, 2)).conj().imag
    assert flagged.is_neg()
    plan = mm.plan_tokens_by_expert(idx, 8)
    rows = mm.sort_tokens_by_expert(flagged, plan)
    assert torch.equal(rows, mm.sort_tokens_by_expert(flagged.resolve_neg().contiguous(), plan))
    sign = torch.view_as_complex(torch.ones((33, 2, 2), device="cuda")).conj().imag
    assert torch.equal(mm.unsort_tokens_by_expert(rows, plan, sign), -mm.unsort_tokens_by_expert(rows, plan))


def test_training_step():
    tokens, topk, experts, hidden, inter = 50, 3, 5, 24, 32
    g = torch.Generator().manual_seed(8)
    rnd = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    x, router = rnd(tokens, hidden), rnd(experts, hidden)
    w1, w2, dy = rnd(experts, inter, hidden), rnd(experts, hidden, inter), rnd(tokens, hidden)

    def step(x, router, w1, w2, dy, sort, unsort):
        top, idx = (x @ router.t()).topk(topk, dim=1)
        weights = torch.softmax(top, dim=1)
        idx = torch.where(torch.arange(tokens, device=x.device)[:, None] % 7 == 3, -1, idx)   # some tokens dropped whole
        rows, offsets, back = sort(x, idx)
        out = torch.cat([(rows[a:b] @ w1[e].t()).relu() @ w2[e].t() for e, (a, b) in enumerate(zip(offsets, offsets[1:]))]
                        + [rows.new_zeros(rows.shape[0] - offsets[-1], hidden)])
        y = unsort(out, back, weights)
        return (y.detach(), *torch.autograd.grad(y, (x, router, w1, w2), dy))

    def plain_sort(x, idx):
        flat = idx.reshape(-1)
        order = torch.sort(torch.where(flat < 0, experts, flat), stable=True).indices
        counts = [int((flat == e).sum()) for e in range(experts)]
        return x[order // topk], [0] + torch.tensor(counts).cumsum(0).tolist(), (order, sum(counts))

    def plain_unsort(out, back, weights):
        order, n = back
        parts = out[:n] * weights.reshape(-1)[order[:n], None]
        return torch.zeros(tokens, hidden, dtype=out.dtype).index_add(0, order[:n] // topk, parts)

    def own_sort(x, idx):
        plan = mm.plan_tokens_by_expert(idx, experts)
        return mm.sort_tokens_by_expert(x, plan), plan.offsets.tolist(), plan

    want = step(*[t.double().requires_grad_() for t in (x, router, w1, w2)], dy.double(), plain_sort, plain_unsort)
    got = step(*[t.cuda().requires_grad_() for t in (x, router, w1, w2)], dy.cuda(), own_sort, mm.unsort_tokens_by_expert)
    mass = step(*[t.double().abs().requires_grad_() for t in (x, router, w1, w2)], dy.double().abs(), plain_sort, plain_unsort)
    for name, a, b, m in zip(("y", "x", "router", "w1", "w2"), got, want, mass):
        # the router's gradient runs through the softmax and a difference, its mass is taken four times
        tol = 4 * (hidden + inter + topk + tokens * topk) * 2.0 ** -24 * float(m.abs().max() + b.abs().max())
        assert float((a.double().cpu() - b).abs().max()) <= tol, name
