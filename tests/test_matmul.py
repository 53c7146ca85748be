"""8-bit products with block scales, dense and grouped, against 64-bit arithmetic on the dequantised operands.

Tolerances.  `exact` cases use small integers and scales of 2^-2 .. 2^2: every product and partial sum is a multiple of
2^-4 below 2^20, so FP32 holds all of them and only the rounding to bf16 is left: equal bits.
Other cases: the tensor core adds the 32 products of one instruction and the accumulator after aligning them to
the largest; each of the at most 33 terms loses less than 2^-23 of a value that is at most A = sum |x w|.  Over K / 32
instructions that is at most 33 K / 32 * 2^-23 A, then one rounding of 2^-8: |d| <= 2^-8 |want| + 33 K / 32 * 2^-23 A (1 + 2^-8).
"""
import ctypes

import pytest
import torch

import mini_mega_b200 as mm
from mini_mega_b200 import _lib

E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2


# ------------------------------------------------------------------------------ refusals
def _x(rows=4, depth=256, dtype=E4):
    return torch.zeros((rows, depth), dtype=dtype)


def _sf(*shape):
    return torch.full(shape, 127, dtype=torch.uint8)


_OFF = torch.zeros(4, dtype=torch.int32)


def _inference_out():
    with torch.inference_mode():
        return torch.zeros((4, 4), dtype=torch.bfloat16)


@pytest.fixture(scope="module")
def built():
    _lib.build()


@pytest.mark.parametrize("make, err", [
    (lambda: mm.fp8_matmul(torch.zeros(4, 256), _x()), TypeError),
    (lambda: mm.fp8_matmul(_x(), torch.zeros(4, 256, dtype=torch.bfloat16)), TypeError),
    (lambda: mm.fp8_matmul((_x(), torch.ones(4, 2)), _x()), TypeError),
    (lambda: mm.fp8_matmul(_x(depth=128), _x()), ValueError),
    (lambda: mm.fp8_matmul(_x(depth=120), _x(depth=120)), ValueError),
    (lambda: mm.fp8_matmul(_x(depth=0), _x(depth=0)), ValueError),
    (lambda: mm.fp8_matmul(_x(), _x(rows=0)), ValueError),
    (lambda: mm.fp8_matmul(_x()[0], _x()), ValueError),
    (lambda: mm.fp8_matmul((_x(), _sf(4, 3)), _x()), ValueError),
    (lambda: mm.fp8_matmul((_x(), _sf(2, 4).t()), _x()), ValueError),
    (lambda: mm.fp8_matmul(_x(), (_x(rows=300), _sf(2, 2))), ValueError),
    (lambda: mm.fp8_matmul(_x(), (_x(rows=300), _sf(2, 3).t())), ValueError),
    (lambda: mm.fp8_matmul(_x(depth=512)[:, ::2], _x()), ValueError),
    (lambda: mm.fp8_matmul(_x(depth=264)[:, :256], _x()), ValueError),
    (lambda: mm.fp8_matmul(_x(depth=272)[:, 8:264], _x()), ValueError),
    (lambda: mm.fp8_matmul(_x(rows=1).expand(4, 256), _x()), ValueError),
    (lambda: mm.fp8_matmul(_x(), _x(), out=torch.zeros(4, 4)), ValueError),
    (lambda: mm.fp8_matmul(_x(), _x(), out=torch.zeros((4, 5), dtype=torch.bfloat16)), ValueError),
    (lambda: mm.fp8_matmul(_x(), _x(), out=torch.zeros((4, 8), dtype=torch.bfloat16)[:, ::2]), ValueError),
    (lambda: mm.fp8_matmul(_x(), _x(), out=_inference_out()), ValueError),
    (lambda: mm.fp8_matmul(_x(), _x()), ValueError),                       # CPU tensors
    (lambda: mm.fp8_matmul(_x().float().requires_grad_().to(E4), _x()), TypeError),      # no gradient would come back
    (lambda: mm.fp8_matmul(_x(), _x().requires_grad_()), TypeError),
    (lambda: mm.fp8_grouped_matmul(_x().requires_grad_(), torch.zeros((3, 8, 256), dtype=E4), _OFF), TypeError),
    (lambda: mm.fp8_grouped_matmul(_x(), _x(), _OFF), ValueError),         # w without an expert dimension
    (lambda: mm.fp8_grouped_matmul(_x(), torch.zeros((3, 8, 256), dtype=E4), None), TypeError),
    (lambda: mm.fp8_grouped_matmul(_x(), torch.zeros((4, 8, 256), dtype=E4), _OFF), ValueError),
    (lambda: mm.fp8_grouped_matmul(_x(), torch.zeros((3, 8, 256), dtype=E4), _OFF.long()), ValueError),
    (lambda: mm.fp8_grouped_matmul(_x(), torch.zeros((6, 8, 256), dtype=E4)[::2], _OFF), ValueError),
    (lambda: mm.fp8_grouped_matmul(_x(), (torch.zeros((3, 8, 256), dtype=E4), _sf(1, 2)), _OFF), ValueError),
    (lambda: mm.fp8_grouped_matmul(_x(), torch.zeros((3, 8, 256), dtype=E4), _OFF), ValueError),
])
def test_refusals(built, make, err):
    with pytest.raises(err):
        make()


def test_ctypes_mirror_matches_the_header(tmp_path):
    """Size and field offsets of MxkMatmulArgs as gcc lays it out against the ctypes mirror."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src, args = tmp_path / "s.c", _lib.MxkMatmulArgs
    names = [f[0] for f in args._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mxk_b200.h"\nint main(void) {\n  printf("%zu", sizeof(MxkMatmulArgs));\n'
                   + "".join(f'  printf(" %zu", offsetof(MxkMatmulArgs, {n}));\n' for n in names) + "  return 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), "-o", str(tmp_path / "s"), str(src)], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(args)] + [getattr(args, n).offset for n in names]


def test_c_abi_refuses_before_it_launches():
    _lib.build()
    L = _lib.lib()
    good = dict(x=16, w=16, out=16, x_stride=128, w_stride=128, out_stride=8, rows=4, cols=8, depth=128, experts=1)
    for change in (dict(x=0), dict(w=0), dict(out=0), dict(rows=-1), dict(cols=0), dict(depth=120), dict(depth=8), dict(x_stride=112),
                   dict(w_stride=136), dict(x=24), dict(out=17), dict(out_stride=7), dict(x_format=2), dict(w_format=5),
                   dict(offsets=16, experts=1025), dict(max_spins=1), dict(max_spins=-1), dict(max_spins=7999999),
                   dict(offsets=18)):
        assert L.mxk_fp8_matmul(ctypes.byref(_lib.MxkMatmulArgs(**{**good, **change})), None) == -1, change
        assert b"fp8_matmul" in L.mxk_last_error()
    assert L.mxk_fp8_matmul(None, None) == -1
    assert L.mxk_matmul_status(None) == -1


# ------------------------------------------------------------------------------- products
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _data(g, shape, dtype, exact):
    if exact:
        return torch.randint(-3, 4, shape, generator=g, device="cuda").float().to(dtype)
    return (torch.randn(shape, generator=g, device="cuda") * 60).clamp(-440, 440).to(dtype)


def _scales(g, shape, exact):
    return torch.randint(126 if exact else 110, 129 if exact else 140, shape, generator=g, device="cuda", dtype=torch.uint8)


def _dequant(q, sf, block_rows):
    v = q.double()
    if sf is None:
        return v
    f = torch.exp2(sf.double() - 127).repeat_interleave(128, -1)[..., :q.shape[-1]]
    return v * (f.repeat_interleave(128, -2)[..., :q.shape[-2], :] if block_rows else f)


def _check(out, a, b, exact):
    want = a @ b.t()
    if exact:
        assert torch.equal(out, want.to(torch.bfloat16))
        return
    mass = a.abs() @ b.abs().t()
    tol = 2.0 ** -8 * want.abs() + 33 * a.shape[1] / 32 * 2.0 ** -23 * mass * (1 + 2.0 ** -8)
    d = (out.double() - want).abs()
    assert bool((d <= tol).all()), f"{int((d > tol).sum())} of {d.numel()} off, worst by {float((d / tol).max()):.3g}"


DENSE = [(1, 128, 128), (1, 4096, 2048), (1, 1, 16), (3, 130, 144), (16, 512, 6144), (17, 384, 640), (32, 100, 1040), (33, 256, 512),
         (64, 640, 4096), (100, 1000, 272), (128, 2048, 384), (129, 257, 128), (200, 128, 1024), (240, 512, 512), (241, 300, 656),
         (500, 777, 2064), (1000, 1536, 768), (2500, 512, 144)]


@pytest.mark.gpu
@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("form", ["block", "row", "raw"])
@pytest.mark.parametrize("rows, cols, depth", DENSE)
def test_dense(rows, cols, depth, form, exact):
    g = _gen(rows * 7 + cols + depth)
    blocks = (depth + 127) // 128
    x, w = _data(g, (rows, depth), E4, exact), _data(g, (cols, depth), E4, exact)
    xs, ws = (None, None) if form == "raw" else (_scales(g, (rows, blocks), exact),
                                                 _scales(g, (cols if form == "row" else (cols + 127) // 128, blocks), exact))
    out = mm.fp8_matmul(x if xs is None else (x, xs), w if ws is None else (w, ws))
    _check(out, _dequant(x, xs, False), _dequant(w, ws, form == "block"), exact)
    assert mm.matmul_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("xt", [E4, E5])
@pytest.mark.parametrize("wt", [E4, E5])
@pytest.mark.parametrize("rows", [5, 300])
def test_formats(xt, wt, rows):
    g = _gen(rows)
    x, w = _data(g, (rows, 400), xt, False), _data(g, (210, 400), wt, False)
    xs, ws = _scales(g, (rows, 4), False), _scales(g, (210, 4), False)
    _check(mm.fp8_matmul((x, xs), (w, ws)), _dequant(x, xs, False), _dequant(w, ws, False), False)
    if wt == E4 and xt == E4:
        assert torch.equal(mm.fp8_matmul((x.view(torch.uint8), xs), (w.view(torch.uint8), ws)), mm.fp8_matmul((x, xs), (w, ws)))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [7, 200])
def test_views_and_rows_that_must_not_change(rows):
    g = _gen(rows + 1)
    x, w = _data(g, (rows, 512 + 32), E4, True), _data(g, (300, 512 + 64), E4, True)
    xs = _scales(g, (rows, 9), True)
    ws = _scales(g, (3, 4), True)
    out = torch.full((rows + 2, 300 + 3), 7.0, dtype=torch.bfloat16, device="cuda")
    got = mm.fp8_matmul((x[:, 16:528], xs[:, 3:7]), (w[:, 48:560], ws), out=out[1:-1, 1:301])
    assert got.data_ptr() == out[1:-1, 1:301].data_ptr()
    _check(got, _dequant(x[:, 16:528], xs[:, 3:7], False), _dequant(w[:, 48:560], ws, True), True)
    rest = out.clone()
    rest[1:-1, 1:301] = 7.0
    assert bool((rest == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 150])
def test_special_values(rows):
    """NaN bytes reach exactly their row and column; the scale byte 255 is NaN; extreme scales multiply out."""
    x, w = torch.ones((rows, 256), device="cuda").to(E4), torch.ones((140, 256), device="cuda").to(E4)
    x.view(torch.uint8)[1, 200], w.view(torch.uint8)[130, 3] = 0x7F, 0x7F
    out = mm.fp8_matmul(x, w)
    nan = torch.zeros((rows, 140), dtype=torch.bool, device="cuda")
    nan[1], nan[:, 130] = True, True
    assert torch.equal(torch.isnan(out), nan) and bool((out[~nan] == 256).all())
    x, w = torch.ones((rows, 256), device="cuda").to(E4), torch.ones((140, 256), device="cuda").to(E4)
    xs, ws = torch.full((rows, 2), 127, dtype=torch.uint8, device="cuda"), torch.full((140, 2), 127, dtype=torch.uint8, device="cuda")
    xs[2, 1] = 255
    xs[0], ws[5] = 127 + 60, 127 - 100
    out = mm.fp8_matmul((x, xs), (w, ws)).float()
    assert bool(torch.isnan(out[2]).all()) and not bool(torch.isnan(out[:2]).any())
    assert float(out[0, 0]) == 2.0 ** 68 and float(out[0, 5]) == 2.0 ** -32 and float(out[1, 5]) == 2.0 ** -92


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 150])
def test_scales_on_one_operand_and_at_the_ends_of_their_range(rows):
    g = _gen(rows + 5)
    x, w = _data(g, (rows, 272), E4, True), _data(g, (140, 272), E4, True)
    xs, ws = _scales(g, (rows, 3), True), _scales(g, (2, 3), True)
    plain = x.double() @ w.double().t()
    assert torch.equal(mm.fp8_matmul((x, xs), w), (_dequant(x, xs, False) @ w.double().t()).to(torch.bfloat16))
    assert torch.equal(mm.fp8_matmul(x, (w, ws)), (x.double() @ _dequant(w, ws, True).t()).to(torch.bfloat16))
    for a, b in ((0, 254), (1, 253), (254, 0), (60, 194), (254, 20), (3, 150)):   # 2^(a - 127) 2^(b - 127) is a bf16 factor
        xs.fill_(a)
        ws.fill_(b)
        want = plain * 2.0 ** (a + b - 254)
        assert torch.equal(mm.fp8_matmul((x, xs), (w, ws)), want.to(torch.bfloat16)), (a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 140])
def test_infinities_of_e5m2(rows):
    x = torch.ones((rows, 128), device="cuda").to(E5)
    w = torch.ones((130, 128), device="cuda").to(E5)
    x[0, 5], x[1, 7], w[3, 9], w[4, 5] = float("inf"), float("-inf"), float("inf"), float("-inf")
    want = x.double() @ w.double().t()
    out = mm.fp8_matmul(x, w).double()
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out[~torch.isnan(want)], want[~torch.isnan(want)])


@pytest.mark.gpu
def test_given_result_is_noticed_by_autograd():
    x = torch.ones((4, 128), device="cuda").to(E4)
    held = torch.ones((4, 4), device="cuda", dtype=torch.bfloat16)
    factor = torch.ones((4, 4), device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = (factor * held).sum()
    mm.fp8_matmul(x, x, out=held)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with pytest.raises(ValueError, match="gradient"):
        mm.fp8_matmul(x, x, out=factor)


# -------------------------------------------------------------------------------- grouped
GROUPED = [  # rows of every expert, behind: rows of nobody; cols, depth
    ([5], 0, 128, 128), ([0, 0, 3], 0, 256, 256), ([1] * 32, 0, 384, 512), ([4, 0, 1, 30, 2, 0], 5, 200, 1040),
    ([16, 17, 15, 33, 0, 47], 0, 512, 656), ([100, 3, 0, 260], 9, 300, 384), ([300, 241, 0, 17, 480, 1000], 3, 640, 272),
    ([0, 0, 0], 7, 130, 128), ([2000, 1, 1], 0, 257, 144), ([50] * 70, 11, 128, 128), ([9, 700], 2, 130, 2064)]


@pytest.mark.gpu
@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("form", ["block", "row", "raw"])
@pytest.mark.parametrize("counts, behind, cols, depth", GROUPED)
def test_grouped(counts, behind, cols, depth, form, exact):
    g = _gen(sum(counts) + cols)
    rows, experts, blocks = sum(counts) + behind, len(counts), (depth + 127) // 128
    x, w = _data(g, (rows, depth), E4, exact), _data(g, (experts, cols, depth), E4, exact)
    xs = ws = None
    if form != "raw":
        xs = _scales(g, (rows, blocks), exact)
        ws = _scales(g, (experts, cols if form == "row" else (cols + 127) // 128, blocks), exact)
    offsets = torch.tensor([0] + counts, device="cuda").cumsum(0).int()
    arg_x, arg_w = (x, w) if xs is None else ((x, xs), (w, ws))
    out = mm.fp8_grouped_matmul(arg_x, arg_w, offsets)
    given = torch.full((rows, cols), 7.0, dtype=torch.bfloat16, device="cuda")
    mm.fp8_grouped_matmul(arg_x, arg_w, offsets, out=given)
    a, r = _dequant(x, xs, False), 0
    for e, n in enumerate(counts):
        _check(out[r:r + n], a[r:r + n], _dequant(w[e], None if ws is None else ws[e], form == "block"), exact)
        r += n
    assert bool((out[r:] == 0).all()) and bool((given[r:] == 7.0).all()) and torch.equal(given[:r], out[:r])
    assert mm.matmul_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("per_expert", [8, 60, 400])
def test_wild_offsets_stay_inside(per_expert):
    """Offsets out of range or out of order: clamped and made ascending, rows outside every group zero."""
    g = _gen(per_expert)
    rows, experts, cols, depth = per_expert * 5, 5, 192, 256
    x, w = _data(g, (rows, depth), E4, True), _data(g, (experts, cols, depth), E4, True)
    for raw in ([-9, rows // 3, rows // 4, rows // 2, rows + 50, 2 ** 31 - 1], [rows // 5, 7, -2 ** 31, rows // 2, rows // 2, rows - 1]):
        off, top = [], 0
        for v in raw:
            top = max(top, min(max(v, 0), rows))
            off.append(top)
        out = mm.fp8_grouped_matmul(x, w, torch.tensor(raw, dtype=torch.int32, device="cuda"))
        want = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
        for e in range(experts):
            want[off[e]:off[e + 1]] = (x[off[e]:off[e + 1]].double() @ w[e].double().t()).to(torch.bfloat16)
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_captured_replayed_on_two_streams_and_without_rows():
    g = _gen(2)
    w = _data(g, (6, 640, 512), E4, False)
    cases = [(_data(g, (40, 512), E4, False), torch.tensor([0, 9, 9, 20, 31, 31, 40], dtype=torch.int32, device="cuda")),
             (_data(g, (1500, 512), E4, False), torch.tensor([0, 300, 301, 301, 900, 1200, 1480], dtype=torch.int32, device="cuda"))]
    calls = [lambda x=x, o=o: mm.fp8_grouped_matmul(x, w, o) for x, o in cases] + [lambda x=x: mm.fp8_matmul(x, w[2]) for x, _ in cases]
    want = [c() for c in calls]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for c in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = c()
        graphs.append((graph, held))
    for _ in range(3):
        for graph, _ in graphs:
            graph.replay()
        with torch.cuda.stream(side):
            beside = [c() for c in calls]
        here = [c() for c in calls]
        torch.cuda.synchronize()
        for i, (_, held) in enumerate(graphs):
            assert torch.equal(held, want[i]) and torch.equal(beside[i], want[i]) and torch.equal(here[i], want[i])
    # the offsets are read when the graph runs
    offsets = cases[0][1]
    offsets.copy_(torch.tensor([0, 0, 25, 25, 26, 40, 40], dtype=torch.int32))
    graphs[0][0].replay()
    assert torch.equal(graphs[0][1], mm.fp8_grouped_matmul(cases[0][0], w, offsets))
    empty = torch.empty((0, 512), dtype=E4, device="cuda")
    assert mm.fp8_matmul(empty, w[0]).shape == (0, 640)
    assert mm.fp8_grouped_matmul(empty, w, torch.zeros(7, dtype=torch.int32, device="cuda")).shape == (0, 640)
    assert mm.matmul_status() == 0


@pytest.mark.gpu
def test_results_behind_two_to_the_31_elements():
    """Element offsets of the last output rows pass 32 bits: 270000 rows of 8192 columns."""
    rows, cols = 270000, 8192
    g = _gen(9)
    x, w = _data(g, (rows, 16), E4, True), _data(g, (cols, 16), E4, True)
    out = mm.fp8_matmul(x, w)
    for at in (0, 131072, 262143, 262144, 269999):
        assert torch.equal(out[at], (x[at].double() @ w.double().t()).to(torch.bfloat16))
    offsets = torch.tensor([0, 5, 262150, rows], dtype=torch.int32, device="cuda")
    w3 = _data(g, (3, cols, 16), E4, True)
    mm.fp8_grouped_matmul(x, w3, offsets, out=out)
    for at, e in ((4, 0), (5, 1), (262149, 1), (262150, 2), (269999, 2)):
        assert torch.equal(out[at], (x[at].double() @ w3[e].double().t()).to(torch.bfloat16))


@pytest.mark.gpu
def test_many_experts_and_long_depth():
    g = _gen(10)
    counts = [(7 * e) % 5 for e in range(1024)]
    rows = sum(counts)
    x, w = _data(g, (rows, 144), E4, True), _data(g, (1024, 40, 144), E4, True)
    offsets = torch.tensor([0] + counts, device="cuda").cumsum(0).int()
    out = mm.fp8_grouped_matmul(x, w, offsets)
    owner = torch.repeat_interleave(torch.arange(1024, device="cuda"), torch.tensor(counts, device="cuda"))
    want = torch.einsum("rk,rnk->rn", x.double(), w.double()[owner])
    assert torch.equal(out, want.to(torch.bfloat16))
    # 65536 columns of depth: 1 and 300 rows
    w = _data(g, (200, 65536), E4, True)
    for n in (1, 300):
        x = _data(g, (n, 65536), E4, True)
        assert torch.equal(mm.fp8_matmul(x, w), (x.double() @ w.double().t()).to(torch.bfloat16))


@pytest.mark.gpu
def test_results_do_not_depend_on_timing():
    """The same bits on every run, splits of the depth included."""
    g = _gen(11)
    for rows, cols, depth in ((1, 512, 7168), (33, 1024, 4096), (700, 640, 2064)):
        x, w = _data(g, (rows, depth), E4, False), _data(g, (cols, depth), E4, False)
        first = mm.fp8_matmul(x, w)
        for _ in range(20):
            assert torch.equal(mm.fp8_matmul(x, w), first)
