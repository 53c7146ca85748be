"""The operators around the MoE layer: what is measured, over which sizes, and their plain forms.

Four operators, each in the sizes that the layer and its benchmark run:

  sort     plan + rows of the tokens gathered in expert order (and its gradient)
  unsort   the sorted rows summed back per token with the routing weights (and its gradients)
  matmul   8-bit product with one power-of-two scale per 128 columns of x and per 128 x 128 block,
           or per row and 128 columns, of w
  grouped  the same product of sorted rows with each expert's own weights

`own` false: elementary torch operations, in 32 bits, rounded once.  `own` true: the package's calls.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}
_F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def listed():
    return [
        # one token of a decode step, 8-bit rows with their scales, as the layer's input is kept
        dict(name="sort_t1_fp8", op="sort", tokens=1, hidden=6144, topk=8, experts=256, dtype="fp8", drop=0.0, grad=False),
        # the decode job: 128 tokens over 256 experts
        dict(name="sort_t128_bf16", op="sort", tokens=128, hidden=6144, topk=8, experts=256, dtype="bf16", drop=0.0, grad=False),
        # the prefill-sized layer's dispatch: 4096 tokens, 8-bit rows with their scales
        dict(name="sort_t4096_fp8", op="sort", tokens=4096, hidden=7168, topk=8, experts=32, dtype="fp8", drop=0.0, grad=False),
        # a training step in 32 bits, a width that no vector divides, some pairs over an expert's capacity
        dict(name="sort_grad_t1000_fp32", op="sort", tokens=1000, hidden=1001, topk=6, experts=60, dtype="fp32", drop=0.1, grad=True),
        # the combine of a decode step of one rank
        dict(name="unsort_t16_bf16", op="unsort", tokens=16, hidden=6144, topk=8, experts=256, dtype="bf16", drop=0.0, grad=False),
        # the combine of the prefill-sized layer
        dict(name="unsort_t4096_bf16", op="unsort", tokens=4096, hidden=7168, topk=8, experts=32, dtype="bf16", drop=0.0, grad=False),
        # combine and its gradients in a training step
        dict(name="unsort_grad_t2048_bf16", op="unsort", tokens=2048, hidden=6144, topk=8, experts=64, dtype="bf16", drop=0.05, grad=True),
        # gate and up projection of a dense (shared) expert for one token
        dict(name="matmul_t1", op="matmul", rows=1, cols=4096, depth=6144, w_scale="block", x_type="e4m3", w_type="e4m3"),
        # the same projection over a prefill
        dict(name="matmul_t4096", op="matmul", rows=4096, cols=4096, depth=7168, w_scale="block", x_type="e4m3", w_type="e4m3"),
        # a weight gradient: both factors scaled along the tokens, ragged sizes, the output gradient in e5m2
        dict(name="matmul_wgrad_ragged", op="matmul", rows=2043, cols=1111, depth=4016, w_scale="row", x_type="e5m2", w_type="e4m3"),
        # one rank's experts in a decode step: 16 tokens on each of 8 ranks land on 32 experts
        dict(name="grouped_decode", op="grouped", rows=128, cols=4096, depth=6144, experts=32, skew=0.0),
        # one rank's experts over a prefill, unevenly loaded
        dict(name="grouped_prefill", op="grouped", rows=32768, cols=4096, depth=7168, experts=32, skew=0.3),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sort", "unsort", "matmul", "grouped"])
    if op in ("sort", "unsort"):
        while True:
            c = dict(op=op, tokens=_log_int(rng, 1, 4096), hidden=_log_int(rng, 128, 7168), topk=rng.randint(1, 8),
                     experts=_log_int(rng, 8, 256), dtype=rng.choice(["bf16", "fp16", "fp32"] + (["fp8"] if op == "sort" else [])),
                     drop=rng.choice([0.0, 0.1]), grad=rng.random() < 0.5)
            if c["dtype"] == "fp8":
                c.update(hidden=-(-c["hidden"] // 128) * 128, grad=False)
            elif rng.random() < 0.5:
                c["hidden"] = -(-c["hidden"] // 64) * 64
            size = c["tokens"] * c["topk"] * c["hidden"] * _BYTES[c["dtype"]]
            if size * (3 if c["grad"] else 1) <= 4096 * 8 * 7168 * 2:
                return c
    if op == "matmul":
        while True:
            c = dict(op=op, rows=_log_int(rng, 1, 8192), cols=_log_int(rng, 64, 7168), depth=16 * _log_int(rng, 8, 448),
                     w_scale=rng.choice(["block", "row"]), x_type=rng.choice(["e4m3", "e4m3", "e5m2"]), w_type="e4m3")
            if rng.random() < 0.5:
                c.update(cols=-(-c["cols"] // 128) * 128, depth=-(-c["depth"] // 128) * 128)
            if c["rows"] * c["cols"] * c["depth"] <= 4096 * 4096 * 7168:
                return c
    while True:
        c = dict(op=op, rows=_log_int(rng, 8, 32768), cols=_log_int(rng, 128, 4096), depth=16 * _log_int(rng, 16, 448),
                 experts=_log_int(rng, 1, 32), skew=rng.choice([0.0, 0.3]))
        if rng.random() < 0.7:
            c.update(cols=-(-c["cols"] // 128) * 128, depth=-(-c["depth"] // 128) * 128)
        if c["rows"] * c["cols"] * c["depth"] <= 32768 * 4096 * 7168:
            return c


# ------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _routing(g, tokens, topk, experts, drop):
    """Distinct experts per token drawn from logits with a popularity per expert; a share of the pairs is dropped (-1)."""
    k = min(topk, experts)
    logits = torch.randn(tokens, experts, generator=g, device="cuda") + 0.5 * torch.randn(experts, generator=g, device="cuda")
    top, idx = logits.topk(k, dim=1)
    weights = torch.softmax(top, dim=1)
    if drop:
        idx = torch.where(torch.rand(tokens, k, generator=g, device="cuda") < drop, -1, idx)
    return idx.contiguous(), weights.contiguous()


def _tables(idx, experts):
    """The plan's three tables: row of every pair, pair of every row, first row of every expert."""
    flat = idx.reshape(-1)
    key = torch.where(flat < 0, experts, flat)
    order = torch.sort(key, stable=True).indices
    counts = (key[:, None] == torch.arange(experts + 1, device=key.device)).sum(0)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=key.device)
    offsets[1:] = counts[:experts].cumsum(0)
    place = torch.arange(flat.numel(), dtype=torch.int32, device=key.device)
    row_of_pair = torch.empty_like(place)
    row_of_pair[order] = place
    row_of_pair = torch.where(flat < 0, -1, row_of_pair).view(idx.shape)
    pair_of_row = torch.where(place < offsets[-1], order.to(torch.int32), -1)
    return row_of_pair, pair_of_row, offsets


def _values(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _bytes8(g, shape, dtype=torch.float8_e4m3fn):
    """8-bit values as a quantiser leaves them: the largest of a block of 128 near the type's largest."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1, shape[-1])
    step = max(1, (1 << 28) // shape[-1])
    for i in range(0, flat.shape[0], step):
        part = flat[i:i + step]
        part.copy_((torch.randn(part.shape, generator=g, device="cuda") * 110.0).clamp_(-448.0, 448.0))
    return out


def _exponents(g, shape):
    """Scales 2^-10 .. 2^-5 as biased exponent bytes."""
    return torch.randint(117, 123, shape, generator=g, device="cuda", dtype=torch.uint8)


def prepare(case, seed):
    g = _generator(seed)
    c = dict(case)
    if c["op"] == "sort":
        s = dict(case=c, experts=c["experts"])
        s["idx"], _ = _routing(g, c["tokens"], c["topk"], c["experts"], c["drop"])
        pairs = s["idx"].numel()
        if c["dtype"] == "fp8":
            s["x"] = _bytes8(g, (c["tokens"], c["hidden"]))
            s["x_sf"] = _exponents(g, (c["tokens"], c["hidden"] // 128))
        else:
            s["x"] = _values(g, (c["tokens"], c["hidden"]), _DTYPES[c["dtype"]]).requires_grad_(c["grad"])
        if c["grad"]:
            s["drows"] = _values(g, (pairs, c["hidden"]), _DTYPES[c["dtype"]])
        return s
    if c["op"] == "unsort":
        idx, weights = _routing(g, c["tokens"], c["topk"], c["experts"], c["drop"])
        s = dict(case=c, weights=weights.requires_grad_(c["grad"]), plan=_tables(idx, c["experts"]))
        s["rows"] = _values(g, (idx.numel(), c["hidden"]), _DTYPES[c["dtype"]]).requires_grad_(c["grad"])
        if c["grad"]:
            s["dy"] = _values(g, (c["tokens"], c["hidden"]), _DTYPES[c["dtype"]])
        return s
    blocks = -(-c["depth"] // 128)
    if c["op"] == "matmul":
        w_blocks = -(-c["cols"] // 128) if c["w_scale"] == "block" else c["cols"]
        return dict(case=c,
                    x=(_bytes8(g, (c["rows"], c["depth"]), _F8[c["x_type"]]), _exponents(g, (c["rows"], blocks))),
                    w=(_bytes8(g, (c["cols"], c["depth"]), _F8[c["w_type"]]), _exponents(g, (w_blocks, blocks))))
    share = torch.softmax(c["skew"] * torch.randn(c["experts"], generator=g, device="cuda"), 0)
    owner = torch.multinomial(share, c["rows"], replacement=True, generator=g)
    counts = (owner[:, None] == torch.arange(c["experts"], device="cuda")).sum(0)
    offsets = torch.zeros(c["experts"] + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    return dict(case=c, offsets=offsets, most=int(counts.max()),
                x=(_bytes8(g, (c["rows"], c["depth"])), _exponents(g, (c["rows"], blocks))),
                w=(_bytes8(g, (c["experts"], c["cols"], c["depth"])),
                   _exponents(g, (c["experts"], -(-c["cols"] // 128), blocks))))


# -------------------------------------------------------------------------- plain forms
def _plain_sort(s):
    row_of_pair, pair_of_row, offsets = _tables(s["idx"], s["experts"])
    k = s["idx"].shape[1]
    at = torch.clamp(pair_of_row, min=0) // k
    held = pair_of_row >= 0
    x = s["x"].detach()
    out = dict(row_of_pair=row_of_pair, offsets=offsets)
    if "x_sf" in s:
        out["rows"] = torch.where(held[:, None], x.view(torch.uint8)[at], 0).view(x.dtype)
        out["rows_sf"] = torch.where(held[:, None], s["x_sf"][at], 0)
        return out
    out["rows"] = torch.where(held[:, None], x[at], 0.0)
    if "drows" in s:
        out["dx"] = _plain_gather_sum(s["drows"], row_of_pair, None)
    return out


def _plain_gather_sum(rows, row_of_pair, weights):
    """sum_j weights[t, j] * rows[row_of_pair[t, j]] in 32 bits, j ascending, rounded once."""
    held = row_of_pair >= 0
    at = torch.clamp(row_of_pair, min=0)
    factor = held.float() if weights is None else torch.where(held, weights, 0.0)
    return (rows[at].float() * factor[:, :, None]).sum(1).to(rows.dtype)


def _plain_unsort(s):
    row_of_pair, pair_of_row, _ = s["plan"]
    rows, weights = s["rows"].detach(), s["weights"].detach()
    out = dict(y=_plain_gather_sum(rows, row_of_pair, weights))
    if "dy" in s:
        k = row_of_pair.shape[1]
        pair = torch.clamp(pair_of_row, min=0)
        held = pair_of_row >= 0
        factor = torch.where(held, weights.reshape(-1)[pair], 0.0)
        out["drows"] = (s["dy"][pair // k].float() * factor[:, None]).to(rows.dtype)
        dot = (s["dy"].float()[:, None, :] * rows[torch.clamp(row_of_pair, min=0)].float()).sum(2)
        out["dweights"] = torch.where(row_of_pair >= 0, dot, 0.0)
    return out


def _power(e):
    return torch.exp2(e.float() - 127.0)


def _spread(sf, depth, rows=None):
    """Scale bytes per 128 columns (and per 128 rows, where `rows` is given) as a factor of every element."""
    f = _power(sf).repeat_interleave(128, dim=-1)[..., :depth]
    return f if rows is None else f.repeat_interleave(128, dim=-2)[..., :rows, :]


def _plain_matmul(s):
    (x, x_sf), (w, w_sf) = s["x"], s["w"]
    block = s["case"]["w_scale"] == "block"
    a = x.float() * _spread(x_sf, x.shape[1])
    b = w.float() * _spread(w_sf, w.shape[1], w.shape[0] if block else None)
    return dict(out=(a @ b.t()).to(torch.bfloat16))


def _plain_grouped(s):
    (x, x_sf), (w, w_sf) = s["x"], s["w"]
    experts, cols, depth = w.shape
    a = x.float() * _spread(x_sf, depth)
    b = w.float() * _spread(w_sf, depth, cols)
    offsets = s["offsets"].long()
    # every expert's rows padded to the longest group, one batched product, and back
    at = offsets[:-1, None] + torch.arange(s["most"], device=x.device)
    padded = torch.where((at < offsets[1:, None])[:, :, None], a[torch.clamp(at, max=x.shape[0] - 1)], 0.0)
    full = torch.bmm(padded, b.transpose(1, 2)).view(-1, cols)
    place = torch.arange(x.shape[0], device=x.device)
    owner = (place[:, None] >= offsets[None, 1:]).sum(1)
    return dict(out=full[owner * s["most"] + place - offsets[owner]].to(torch.bfloat16))


# ------------------------------------------------------------------------ the package's
def _own_sort(s):
    import mini_mega_b200 as mm

    plan = mm.plan_tokens_by_expert(s["idx"], s["experts"])
    out = dict(row_of_pair=plan.row_of_pair, offsets=plan.offsets)
    if "x_sf" in s:
        out["rows"], out["rows_sf"] = mm.sort_tokens_by_expert(s["x"], plan, s["x_sf"])
        return out
    rows = mm.sort_tokens_by_expert(s["x"], plan)
    out["rows"] = rows.detach()
    if "drows" in s:
        (out["dx"],) = torch.autograd.grad(rows, s["x"], s["drows"])
    return out


def _own_unsort(s):
    import mini_mega_b200 as mm

    y = mm.unsort_tokens_by_expert(s["rows"], mm.ExpertPlan(*s["plan"]), s["weights"])
    out = dict(y=y.detach())
    if "dy" in s:
        out["drows"], out["dweights"] = torch.autograd.grad(y, (s["rows"], s["weights"]), s["dy"])
    return out


def _own_matmul(s):
    import mini_mega_b200 as mm

    return dict(out=mm.fp8_matmul(s["x"], s["w"]))


def _own_grouped(s):
    import mini_mega_b200 as mm

    return dict(out=mm.fp8_grouped_matmul(s["x"], s["w"], s["offsets"]))


_PLAIN = {"sort": _plain_sort, "unsort": _plain_unsort, "matmul": _plain_matmul, "grouped": _plain_grouped}
_OWN = {"sort": _own_sort, "unsort": _own_unsort, "matmul": _own_matmul, "grouped": _own_grouped}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ----------------------------------------------------------------- in 64 bits, and the work
def _exact_dequant(q, sf, rows_per_scale=1):
    v = q.double()
    for b in range(sf.shape[-1]):
        part = torch.ldexp(torch.ones((), dtype=torch.float64, device=q.device), sf[..., b].to(torch.int32) - 127)
        if rows_per_scale > 1:
            part = part.repeat_interleave(rows_per_scale, dim=-1)[..., :q.shape[-2]]
        v[..., b * 128:(b + 1) * 128] *= part[..., None]
    return v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sort":
        flat = s["idx"].reshape(-1).tolist()
        k = s["idx"].shape[1]
        lists = [[] for _ in range(case["experts"])]
        for p, e in enumerate(flat):
            if e >= 0:
                lists[e].append(p)
        pairs = [p for group in lists for p in group]
        order = torch.tensor(pairs, dtype=torch.int64, device="cuda")
        x = s["x"].detach().double()
        rows = torch.zeros(len(flat), case["hidden"], dtype=torch.float64, device="cuda")
        rows[:len(pairs)] = x[order // k]
        out = dict(row_of_pair=None, offsets=None, rows=rows)
        if "x_sf" in s:
            out["rows_sf"] = None
        if "drows" in s:
            out["dx"] = torch.zeros_like(x).index_add_(0, order // k, s["drows"][:len(pairs)].double())
        return out
    if case["op"] == "unsort":
        row_of_pair = s["plan"][0]
        rows, weights = s["rows"].detach().double(), s["weights"].detach().double()
        tokens, k = row_of_pair.shape
        y = torch.zeros(tokens, case["hidden"], dtype=torch.float64, device="cuda")
        drows, dweights = torch.zeros_like(rows), torch.zeros_like(weights)
        for j in range(k):
            t = (row_of_pair[:, j] >= 0).nonzero()[:, 0]
            r = row_of_pair[t, j].long()
            y[t] += weights[t, j, None] * rows[r]
            if "dy" in s:
                dy = s["dy"][t].double()
                drows[r] = weights[t, j, None] * dy
                dweights[t, j] = torch.einsum("th,th->t", dy, rows[r])
        return dict(y=y, drows=drows, dweights=dweights) if "dy" in s else dict(y=y)
    (x, x_sf), (w, w_sf) = s["x"], s["w"]
    a = _exact_dequant(x, x_sf)
    if case["op"] == "matmul":
        return dict(out=a @ _exact_dequant(w, w_sf, 128 if case["w_scale"] == "block" else 1).t())
    out = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device="cuda")
    first = s["offsets"].tolist()
    for e in range(w.shape[0]):
        if first[e + 1] > first[e]:
            out[first[e]:first[e + 1]] = a[first[e]:first[e + 1]] @ _exact_dequant(w[e], w_sf[e], 128).t()
    return dict(out=out)


def work(case):
    c = case
    if c["op"] in ("sort", "unsort"):
        size = _BYTES[c["dtype"]]
        pairs = c["tokens"] * min(c["topk"], c["experts"])
        x, rows = c["tokens"] * c["hidden"] * size, pairs * c["hidden"] * size
        if c["op"] == "sort":
            scales = (c["tokens"] + pairs) * (c["hidden"] // 128) if c["dtype"] == "fp8" else 0
            b = 12 * pairs + 4 * (c["experts"] + 1) + x + rows + scales + (x + rows if c["grad"] else 0)
            return dict(bytes=b, flops=pairs * c["hidden"] if c["grad"] else 0)
        b = 8 * pairs + x + rows
        flops = 2 * pairs * c["hidden"]
        if c["grad"]:
            b += 8 * pairs + x + rows + rows + 4 * pairs
            flops += 3 * pairs * c["hidden"]
        return dict(bytes=b, flops=flops)
    blocks = -(-c["depth"] // 128)
    m, n, k = c["rows"], c["cols"], c["depth"]
    w_rows = n if c.get("w_scale") == "row" else -(-n // 128)
    groups = min(c.get("experts", 1), m)   # at most this many experts have rows
    return dict(bytes=m * (k + blocks) + groups * (n * k + w_rows * blocks) + 2 * m * n, flops=2.0 * m * n * k)
