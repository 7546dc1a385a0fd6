"""Wide numbers to fp8 codes with power-of-two scales, by rows and transposed by expert: codes and scales are exact."""
import zlib

import numpy as np
import pytest
import torch

from expert_util import F8, TOP, offsets_of, places, quantized

pytestmark = pytest.mark.gpu

WIDE = [torch.float32, torch.bfloat16, torch.float16]


def generator(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def wide(gen, rows, cols, dtype):
    x = torch.randn((rows, cols), generator=gen, device="cuda") * torch.exp2(torch.randint(-9, 4, (rows, 1), generator=gen, device="cuda").float())
    return x.to(dtype)


def same(got, want):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 8), (5, 7), (1, 4096), (9, 1032), (1500, 4096), (1030, 1024), (4, 4104), (3, 16384), (2, 16392), (7, 4095), (2, 20000)])
def test_rows(pkg, dtype, fmt, rows, cols):
    """Every kernel: a wave to a row, four waves, any length; lengths that are not whole pieces."""
    x = wide(generator("rows", rows, cols), rows, cols, dtype)
    v, s = quantized(x, fmt, 1)
    got, scales = pkg.quantize_rows(x, fmt)
    assert got.dtype == F8[fmt] and torch.equal(scales.double(), s)
    same(got, v)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("cols", [72, 75, 1040, 4100])
def test_rows_hard_numbers(pkg, dtype, fmt, cols):
    """Zeros, infinities, NaNs, the type's largest and smallest numbers, maxima on and beside a power of two times the
    largest code."""
    gen = generator("hard", cols)
    x = wide(gen, 12, cols, dtype)
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    x[0] = 0
    x[1] = -0.0
    x[2, 3], x[2, 5], x[2, cols - 1] = float("inf"), float("-inf"), float("nan")
    x[3] = float("nan")
    x[4] = float("inf")
    x[5, cols // 2] = big
    x[6] = 0
    x[6, 1] = -big
    x[7] = 0
    x[7, cols - 2] = small
    for r, m in ((8, 0.875), (9, 0.875 * (1 + torch.finfo(dtype).eps)), (10, 0.875 * (1 - torch.finfo(dtype).eps)), (11, 1.0)):
        x[r] = (x[r].float().clamp(-0.5, 0.5)).to(dtype)
        x[r, r] = m
    v, s = quantized(x, fmt, 1)
    got, scales = pkg.quantize_rows(x, fmt)
    assert torch.equal(scales.double(), s)
    same(got, v)
    nan = torch.isnan(x)
    assert (got.view(torch.uint8)[nan] == 0x7F).all()
    assert (got.view(torch.uint8)[1] == 0x80).all()
    assert (got[4].float() == TOP[fmt]).all()


@pytest.mark.parametrize("fmt", [0, 1])
def test_rows_codes_equal_the_host_codec(pkg, fmt):
    """Every rounding: all midpoints and their neighbours, scale 1, against the library's host conversion."""
    from conftest import finite_codes
    v = np.sort(pkg.decode(finite_codes(fmt), fmt))
    mid = (v[1:].astype(np.float64) + v[:-1]) / 2
    pts = np.concatenate([v, mid, np.nextafter(mid.astype(np.float32), np.float32(1e9)), np.nextafter(mid.astype(np.float32), np.float32(-1e9))]).astype(np.float32)
    pts = pts[np.abs(pts) <= TOP[fmt]]
    pts = np.concatenate([pts, np.full(-pts.size % 8, TOP[fmt], np.float32)])
    got, scales = pkg.quantize_rows(torch.from_numpy(pts[None]).cuda(), fmt)
    assert float(scales[0]) == 1.0
    assert np.array_equal(got.view(torch.uint8).cpu().numpy()[0], pkg.encode(pts, fmt))


@pytest.mark.parametrize("cols", [64, 65, 2048, 4096])
def test_rows_gathered_and_strided(pkg, cols):
    gen = generator("gather", cols)
    store = wide(gen, 40, cols + 24, torch.bfloat16)
    index = torch.randint(0, 40, (1200,), generator=gen, dtype=torch.int32, device="cuda")
    index[3], index[7], index[11] = -1, 40, 2 ** 31 - 1
    for shift in (0, 8, 3):                                  # rows that start on 16 bytes, and that do not
        x = store[:, shift:shift + cols]
        got, scales = pkg.quantize_rows(x, 0, row_index=index)
        there = (index >= 0) & (index < 40)
        rows = torch.where(there[:, None], x[index.clamp(0, 39).long()], torch.zeros((), dtype=x.dtype, device="cuda"))
        v, s = quantized(rows, 0, 1)
        assert torch.equal(scales.double(), s)
        same(got, v)


def check_columns(pkg, x, counts, fmt, index=None, first=0):
    off = offsets_of(counts, first)
    got, scales = pkg.quantize_columns(x, off, fmt, row_index=index)
    rows = x if index is None else torch.where(((index >= 0) & (index < x.shape[0]))[:, None], x[index.clamp(0, x.shape[0] - 1).long()], torch.zeros((), dtype=x.dtype, device="cuda"))
    at, cs, used = places(off.tolist(), rows.shape[0])
    want = torch.zeros(got.shape, dtype=torch.float64, device="cuda")
    for g, (p, c) in enumerate(zip(at, cs)):
        v, s = quantized(rows[int(off[g]):int(off[g]) + c], fmt, 0) if c else (None, torch.ones(x.shape[1], dtype=torch.float64, device="cuda"))
        assert torch.equal(scales[g].double(), s)
        if c:
            want[:, p:p + c] = v.t()
    same(got, want)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("cols", [1, 64, 72, 200, 75])
@pytest.mark.parametrize("counts", [[1], [0, 5, 0, 131, 128, 0], [300, 1, 0, 1000], [i % 4 for i in range(67)]])
def test_columns(pkg, dtype, fmt, cols, counts):
    gen = generator("columns", cols, counts)
    check_columns(pkg, wide(gen, sum(counts), cols, dtype), counts, fmt)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("cols", [64, 75])
def test_columns_hard_numbers(pkg, dtype, cols):
    gen = generator("hard columns", cols)
    x = wide(gen, 150, cols, dtype)
    big = torch.finfo(dtype).max
    x[:, 0] = 0
    x[100, 1], x[101, 2], x[102, 3] = float("nan"), float("inf"), float("-inf")
    x[:, 4] = float("nan")
    x[5, 5] = big
    for fmt in (0, 1):
        check_columns(pkg, x, [20, 0, 100, 30], fmt)


def test_columns_gathered_strided_and_rows_outside(pkg):
    gen = generator("columns gather")
    store = wide(gen, 50, 160, torch.float16)
    index = torch.randint(0, 50, (333,), generator=gen, dtype=torch.int32, device="cuda")
    index[0], index[300] = -5, 50
    for shift in (0, 8, 5):
        x = store[:, shift:shift + 136]
        check_columns(pkg, x, [100, 0, 233], 0, index=index)
        check_columns(pkg, x, [10, 3, 20], 1, first=7)               # rows in front of the first and behind the last expert


def test_smallest_numbers(pkg):
    """Subnormal fp32 and fp16: scales stop at 2^-126."""
    x = torch.zeros((4, 72), device="cuda")
    x[0, 3], x[0, 4] = 1e-40, -3e-41
    x[1, 0], x[1, 71] = 2.0 ** -149, 2.0 ** -126
    x[2, 5] = 2.0 ** -126 * 448
    x[3, 5] = 2.0 ** -120
    for fmt in (0, 1):
        v, s = quantized(x, fmt, 1)
        got, scales = pkg.quantize_rows(x, fmt)
        assert torch.equal(scales.double(), s)
        same(got, v)
        check_columns(pkg, x, [2, 2], fmt)
    h = torch.zeros((2, 64), device="cuda", dtype=torch.float16)
    h[0, 1], h[0, 2], h[1, 63] = 6e-8, -3e-7, 6e-8
    v, s = quantized(h, 0, 1)
    got, scales = pkg.quantize_rows(h)
    assert torch.equal(scales.double(), s)
    same(got, v)


@pytest.mark.parametrize("rows,cols,gathered", [((1 << 26) + 5, 8, False), ((1 << 24) + 3, 3, False), ((1 << 24) + 3, 3, True), ((1 << 23) + 1, 1032, True)])
def test_more_rows_than_a_grid_holds(pkg, rows, cols, gathered):
    gen = generator("rows %d" % rows)
    x = torch.randn((1000 if gathered else rows, cols), generator=gen, device="cuda", dtype=torch.bfloat16)
    index = torch.arange(rows, device="cuda", dtype=torch.int32).remainder_(1001) if gathered else None      # (1000: a row of zeros)
    got, scales = pkg.quantize_rows(x, 0, row_index=index)
    for lo in (0, (1 << 23) - 4, rows - 9):
        at = slice(lo, lo + 9)
        part = x[at] if index is None else torch.cat([x, torch.zeros_like(x[:1])])[index[at].long()]
        v, s = quantized(part, 0, 1)
        lo_end = min(rows, lo + 9)
        assert torch.equal(scales[lo:lo_end].double(), s)
        same(got[lo:lo_end], v)


def test_no_rows(pkg):
    x = torch.zeros((0, 72), device="cuda")
    codes, scales = pkg.quantize_rows(x)
    assert codes.shape == (0, 72) and scales.shape == (0,)
    codes, scales = pkg.quantize_rows(torch.ones((5, 72), device="cuda"), row_index=torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert codes.shape == (0, 72) and scales.shape == (0,)
    codes, scales = pkg.quantize_columns(x, torch.zeros(4, dtype=torch.int32, device="cuda"))
    assert codes.shape == (72, 0) and torch.equal(scales, torch.ones((3, 72), device="cuda"))


def test_columns_of_many_experts(pkg):
    gen = generator("1024")
    counts = [0] * 1024
    for g, c in ((0, 3), (1, 1), (64, 600), (1022, 5), (1023, 130)):
        counts[g] = c
    check_columns(pkg, wide(gen, sum(counts), 200, torch.bfloat16), counts, 0)


def test_long_experts(pkg):
    """More rows of one expert than a workgroup holds at a time, several times over."""
    gen = generator("long")
    for dtype in WIDE:
        check_columns(pkg, wide(gen, 3000, 136, dtype), [1, 2500, 0, 499], 1)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("counts,cols", [([5000], 200), ([3000, 0, 1, 4100], 75), ([0, 0, 2600], 513), ([1025], 1)])
def test_few_experts_with_many_rows(pkg, dtype, counts, cols):
    """The walks split over the rows: infinities, NaNs and largest numbers in one part, columns of zeros, subnormals alone."""
    gen = generator("split", cols)
    rows = sum(counts)
    x = wide(gen, rows, cols, dtype)
    x[rows // 3, 0], x[rows - 1, cols // 2] = float("inf"), float("nan")
    if cols > 3:
        x[:, 1] = 0
        x[:, 2] = torch.finfo(dtype).tiny / 2
        x[rows // 2, 3] = torch.finfo(dtype).max
    for fmt in (0, 1):
        check_columns(pkg, x, counts, fmt)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("shift,cols", [(1, 64), (3, 61), (1, 1000), (5, 4097), (1, 9000)])
def test_any_place_and_length(pkg, dtype, shift, cols):
    """Rows that start anywhere and are not whole pieces, what surrounds them stays out; codes that start anywhere."""
    gen = generator("place", shift, cols)
    rows = 37
    store = torch.full((rows * (cols + 2) + 16,), float("inf"), dtype=dtype, device="cuda")
    x = store[shift:shift + rows * (cols + 2)].view(rows, cols + 2)[:, :cols]
    x.copy_(wide(gen, rows, cols, dtype))
    v, s = quantized(x, 0, 1)
    room = torch.full((rows * cols + 16,), 0x55, dtype=torch.uint8, device="cuda")
    out = room[shift:shift + rows * cols].view(F8[0]).view(rows, cols)
    got, scales = pkg.quantize_rows(x, 0, codes=out)
    assert torch.equal(scales.double(), s)
    same(got, v)
    assert (room[:shift] == 0x55).all() and (room[shift + rows * cols:] == 0x55).all()
    check_columns(pkg, x, [20, 0, 17], 0)


def test_calls_captured_and_replayed(pkg):
    gen = generator("graph")
    x = wide(gen, 256, 512, torch.bfloat16)
    off = offsets_of([100, 0, 156])
    codes, scales = pkg.quantize_rows(x)
    codes_t, scales_t = pkg.quantize_columns(x, off)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.quantize_rows(x, codes=codes, scales=scales)
        pkg.quantize_columns(x, off, codes=codes_t, scales=scales_t)
    for cut in ([256, 0, 0], [3, 250, 3], [0, 0, 0]):
        x.copy_(wide(gen, 256, 512, torch.bfloat16))
        off.copy_(offsets_of(cut))
        graph.replay()
        torch.cuda.synchronize()
        v, s = pkg.quantize_rows(x)
        vt, st = pkg.quantize_columns(x, off)
        assert torch.equal(v.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(s, scales)
        assert torch.equal(vt.view(torch.uint8), codes_t.view(torch.uint8)) and torch.equal(st, scales_t)


def test_split_columns_captured_and_replayed(pkg):
    """Few experts with many rows, replayed with other numbers and another cut: scales sink as well as rise."""
    gen = generator("split graph")
    rows, cols = 4096, 130
    x = wide(gen, rows, cols, torch.bfloat16)
    off = offsets_of([4000, 96])
    codes, scales = pkg.quantize_columns(x, off)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.quantize_columns(x, off, codes=codes, scales=scales)
    for turn, counts in enumerate(([4000, 96], [10, 4086], [4096, 0], [0, 1700])):
        x.copy_(wide(gen, rows, cols, torch.bfloat16) * 2.0 ** (-3 * turn))
        off.copy_(offsets_of(counts))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, want_s = pkg.quantize_columns(x, off)
        assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales, want_s)
        check_columns(pkg, x, counts, 0)


@pytest.mark.parametrize("fmt", [0, 1])
def test_indices_into_nothing(pkg, fmt):
    """A padded batch that has no token: every index is outside a matrix without rows, and stands for a row of zeros."""
    x = torch.empty((0, 200), dtype=torch.bfloat16, device="cuda")
    index = torch.full((70,), -1, dtype=torch.int32, device="cuda")
    off = offsets_of([40, 0, 30])
    for stream in (None, torch.cuda.Stream()):
        c, s = torch.full((70, 200), 3.0, device="cuda").to(F8[fmt]), torch.full((70,), 5.0, device="cuda")
        torch.cuda.synchronize()
        assert pkg.quantize_rows(x, fmt, row_index=index, codes=c, scales=s, stream=stream) == (c, s)
        ct, st = pkg.quantize_columns(x, off, fmt, row_index=index, stream=stream)
        torch.cuda.synchronize()
        assert not c.view(torch.uint8).any() and (s == 1).all()
        assert ct.shape == (200, pkg.grouped_ld(70, 3)) and not ct.view(torch.uint8).any() and st.shape == (3, 200) and (st == 1).all()
    # the same from a matrix that has rows
    some = torch.ones((5, 200), dtype=torch.bfloat16, device="cuda")
    want = pkg.quantize_columns(some, off, fmt, row_index=index)
    assert torch.equal(want[0].view(torch.uint8), ct.view(torch.uint8)) and torch.equal(want[1], st)
    # an index is checked all the same
    for bad in (index.long(), index.cpu(), index[::2]):
        with pytest.raises(pkg.Fp8GemmError):
            pkg.quantize_rows(x, fmt, row_index=bad)
        with pytest.raises(pkg.Fp8GemmError):
            pkg.quantize_columns(x, off, fmt, row_index=bad)
