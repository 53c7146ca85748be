"""8-bit products in every way they are cut: CTA pairs and single CTAs, the depth whole and in 2, 4 and 8 splits, dense and
grouped, and split products of which a cluster gets a second tile (unevenly loaded groups: the cut follows the mean).
The sizes are chosen by the cut that the library reports for them, and a test without a device holds that choice fast.
Data, reference and bounds are those of test_matmul.py.
"""
import ctypes

import pytest
import torch

import mini_mega_b200 as mm
from mini_mega_b200 import _lib
from test_matmul import E4, E5, _check, _data, _dequant, _gen, _scales

SMS = 148   # CTAs of a launch at most

DENSE = [  # rows, cols, depth; pair, splits
    (2048, 4096, 2048, 1, 1), (2043, 4001, 2064, 1, 1), (687, 4744, 4544, 1, 1), (1554, 1424, 1392, 1, 1), (2092, 1041, 1776, 1, 1),
    (580, 5484, 1936, 1, 1), (1762, 1977, 2064, 1, 1),
    (3, 358, 1424, 0, 2), (23, 3769, 2816, 0, 2), (134, 2289, 5776, 0, 2), (1, 4096, 6144, 0, 4), (81, 1286, 5616, 0, 4),
    (128, 2048, 6144, 0, 4), (1, 22, 5200, 0, 8), (84, 513, 7344, 0, 8)]

GROUPED = [  # rows of every expert, behind: rows of nobody; cols, depth; pair, splits
    ([0, 1, 189, 230, 196, 63, 159], 4, 1290, 672, 1, 1), ([0, 1, 580, 93, 38], 0, 1967, 704, 1, 1),
    ([0, 1, 31, 297, 276, 99, 252, 260, 285, 237, 280], 0, 855, 784, 1, 1), ([0, 1, 214, 275, 139, 319, 150, 313, 299], 0, 1089, 992, 1, 1),
    ([300, 0, 1, 513, 1200, 7, 0, 255], 5, 4096, 2064, 1, 1),
    ([0, 1, 52, 18, 37, 60, 10, 4], 4, 625, 5008, 0, 2), ([0, 1, 55, 36, 44, 33, 41], 0, 146, 7408, 0, 4),
    ([0, 1, 57, 3], 2, 406, 4912, 0, 4), ([0, 1, 17, 8, 58], 0, 101, 4080, 0, 8)]

TWICE = [  # the same, with more tiles than clusters
    ([204, 1, 1], 0, 1920, 4608, 0, 2), ([643, 6, 1, 4, 5, 3], 3, 967, 9040, 0, 2), ([1145] + [1] * 10, 0, 512, 12864, 0, 2),
    ([2, 4, 1, 197], 0, 1505, 7648, 0, 2), ([940] + [4] * 8, 0, 640, 8704, 0, 2), ([6, 6, 3, 6, 4, 1, 1, 1182, 3, 5, 3], 2, 213, 7792, 0, 4),
    ([3, 6, 5, 4, 5, 4, 4, 1116, 6, 5, 0, 4, 2, 1, 3, 6, 2, 1, 3, 3, 6, 6, 3], 0, 55, 6080, 0, 4)]


def cut_of(rows, cols, depth, experts=1, grouped=False):
    out = (ctypes.c_int32 * 3)()
    _lib.check(_lib.lib().mxk_matmul_cut(rows, cols, depth, experts, int(grouped), out))
    return tuple(out)


def test_the_sizes_reach_the_cuts_they_are_meant_for():
    _lib.build()
    for rows, cols, depth, pair, splits in DENSE:
        got = cut_of(rows, cols, depth)
        assert (got[0], got[2]) == (pair, splits), (rows, cols, depth, got)
    for table, twice in ((GROUPED, False), (TWICE, True)):
        for counts, behind, cols, depth, pair, splits in table:
            got = cut_of(sum(counts) + behind, cols, depth, len(counts), True)
            assert (got[0], got[2]) == (pair, splits), (counts, cols, depth, got)
            tiles = sum(-(-n // got[1]) for n in counts) * -(-cols // (256 if pair else 128))
            assert twice == (splits > 1 and tiles > SMS // ((1 + pair) * splits)), (counts, cols, depth, got, tiles)
    whole_and_split = {(1, 1), (0, 2), (0, 4), (0, 8)}
    assert {case[-2:] for case in DENSE} == whole_and_split == {case[-2:] for case in GROUPED}
    assert len({cut_of(*case[:3])[1] for case in DENSE if case[3]}) >= 5   # accumulators, and so scale slots, of several widths


def test_the_cut_refuses_what_the_product_refuses():
    _lib.build()
    L, out = _lib.lib(), (ctypes.c_int32 * 3)()
    for sizes in ((0, 8, 128, 1, 0), (4, 0, 128, 1, 0), (4, 8, 120, 1, 0), (4, 8, 128, 1025, 1), (4, 8, 128, 0, 1), ((1 << 30) + 1, 8, 128, 1, 0)):
        assert L.mxk_matmul_cut(*sizes, out) == -1, sizes
    assert L.mxk_matmul_cut(4, 8, 128, 1, 0, None) == -1


def _operands(g, rows, w_shape, depth, form, exact, x_type=E4):
    blocks, cols = (depth + 127) // 128, w_shape[-1]
    x, w = _data(g, (rows, depth), x_type, exact), _data(g, (*w_shape, depth), E4, exact)
    if form == "raw":
        return x, w, None, None
    return x, w, _scales(g, (rows, blocks), exact), _scales(g, (*w_shape[:-1], cols if form == "row" else (cols + 127) // 128, blocks), exact)


@pytest.mark.gpu
@pytest.mark.parametrize("form, exact, x_type", [("block", True, E4), ("row", True, E4), ("raw", True, E4), ("block", False, E4), ("row", False, E5)])
@pytest.mark.parametrize("rows, cols, depth, pair, splits", DENSE)
def test_dense(rows, cols, depth, pair, splits, form, exact, x_type):
    x, w, xs, ws = _operands(_gen(rows + cols + depth), rows, (cols,), depth, form, exact, x_type)
    out = mm.fp8_matmul(x if xs is None else (x, xs), w if ws is None else (w, ws))
    _check(out, _dequant(x, xs, False), _dequant(w, ws, form == "block"), exact)
    assert mm.matmul_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("form, exact, x_type", [("block", True, E4), ("row", True, E4), ("raw", True, E4), ("block", False, E4), ("row", False, E5)])
@pytest.mark.parametrize("counts, behind, cols, depth, pair, splits", GROUPED + TWICE)
def test_grouped(counts, behind, cols, depth, pair, splits, form, exact, x_type):
    rows, experts = sum(counts) + behind, len(counts)
    x, w, xs, ws = _operands(_gen(rows + cols + depth), rows, (experts, cols), depth, form, exact, x_type)
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
@pytest.mark.parametrize("counts, behind, cols, depth, pair, splits", TWICE + GROUPED[:1])
def test_the_same_bits_on_every_run(counts, behind, cols, depth, pair, splits):
    """Beside and behind one another, and behind a product that leaves its CTAs at other times."""
    rows = sum(counts) + behind
    x, w, xs, ws = _operands(_gen(cols), rows, (len(counts), cols), depth, "block", False)
    offsets = torch.tensor([0] + counts, device="cuda").cumsum(0).int()
    call = lambda: mm.fp8_grouped_matmul((x, xs), (w, ws), offsets)   # noqa: E731
    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for i in range(20):
        outs.append(call())
        mm.fp8_matmul(x[:1 + i], w[0])
        with torch.cuda.stream(side):
            outs.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    assert mm.matmul_status() == 0
