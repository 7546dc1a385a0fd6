"""Products with 4-bit weights, one matrix and one per expert, against 64-bit sums."""
import zlib

import pytest
import torch

from expert_util import E2M1, F8, offsets_of, pow2, rounding, scale_values, w4_values

pytestmark = pytest.mark.gpu

SCALES = [torch.float32, torch.bfloat16, torch.float16, torch.uint8]
XS = [torch.bfloat16, torch.float16, F8[0], F8[1]]


def generator(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def weights(gen, lead, n, k, run, w_fmt, scale, zeros):
    w = torch.randint(0, 256, lead + (n, k // 2), generator=gen, dtype=torch.uint8, device="cuda")
    shape = lead + (n, k // run)
    if scale == torch.uint8:
        s = torch.randint(118, 131, shape, generator=gen, dtype=torch.uint8, device="cuda")
    else:
        s = (torch.rand(shape, generator=gen, device="cuda") + 0.1).to(scale)
    z = torch.randint(0, 16, shape, generator=gen, dtype=torch.uint8, device="cuda") if zeros else None
    return w, s, z


def tolerance(x, v, w_abs, dtype, y):
    """fp32 sums in any order over k products; the integer path adds (16 + q) x and -(16 + zero) x: at most 31 + 31
    per unit of scale instead of |q - zero|."""
    k = x.shape[1]
    return 2 * (k + 64) * 2.0 ** -24 * (x.abs() @ w_abs.t().contiguous()) + rounding(y, dtype) * 1.0001


def run_case(pkg, m, k, n, run, w_fmt, scale, zeros, x_type, dtype, key):
    gen = generator(m, k, n, run, key)
    w, s, z = weights(gen, (), n, k, run, w_fmt, scale, zeros)
    x = torch.randn((m, k), generator=gen, device="cuda").to(x_type)
    sx = pow2(torch.randint(-3, 4, (m,), generator=gen, device="cuda")).float() if x_type in F8.values() else None
    y = pkg.gemv_w4(x, w, s, run, w_fmt=w_fmt, zeros=z, x_scale=sx, out_dtype=dtype)
    v = w4_values(w, s, run, w_fmt, z)
    bound = (62.0 if w_fmt == 0 else 6.0) * scale_values(s).repeat_interleave(run, -1)
    xd = x.double() * (sx[:, None].double() if sx is not None else 1.0)
    ref = xd @ v.t().contiguous()
    err = (y.double() - ref).abs()
    tol = tolerance(xd, v, bound, dtype, ref)
    assert torch.isfinite(y.float()).all()
    assert (err <= tol).all(), "worst err/tol %g" % float((err / tol).max())


@pytest.mark.parametrize("w_fmt,zeros", [(0, False), (0, True), (1, False)])
@pytest.mark.parametrize("run", [32, 64, 96, 128, 384])
@pytest.mark.parametrize("m", [1, 2, 5, 16, 17, 33, 64, 70])
def test_rows_and_runs(pkg, w_fmt, zeros, run, m):
    """Every row block, runs shorter and longer than an MFMA's k, a K that ends inside a ring stage, columns that end
    inside a tile."""
    run_case(pkg, m, 1152, 75, run, w_fmt, torch.float16, zeros, torch.bfloat16, torch.float32, "rows")


@pytest.mark.parametrize("w_fmt", [0, 1])
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("x_type", XS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("run", [32, 128])
def test_types(pkg, w_fmt, scale, x_type, dtype, run):
    run_case(pkg, 3, 512, 40, run, w_fmt, scale, w_fmt == 0, x_type, dtype, "types")


@pytest.mark.parametrize("k", [32, 64, 96, 256, 288, 1024, 4128, 8192, 28672])
@pytest.mark.parametrize("n", [1, 15, 16, 130, 1100])
@pytest.mark.parametrize("m", [1, 16])
def test_lengths(pkg, k, n, m):
    """From a single run to lengths that are staged in several pieces."""
    for w_fmt in (0, 1):
        run_case(pkg, m, k, n, 32, w_fmt, torch.float32, w_fmt == 0, torch.bfloat16, torch.float32, "lengths")
        if k % 128 == 0:
            run_case(pkg, m, k, n, 128, w_fmt, torch.float16, False, torch.float16, torch.float32, "lengths")


@pytest.mark.parametrize("w_fmt", [0, 1])
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("x_type", XS)
@pytest.mark.parametrize("m", [20, 50])
@pytest.mark.parametrize("run", [32, 128])
def test_types_with_many_rows(pkg, w_fmt, scale, x_type, m, run):
    """The kernel for more rows of x, one and two blocks of columns a wave, two and four waves along K (which: n and k)."""
    run_case(pkg, m, 768, 40, run, w_fmt, scale, w_fmt == 0, x_type, torch.float32, "many")
    run_case(pkg, m, 384, 16900, run, w_fmt, scale, w_fmt == 0, x_type, torch.bfloat16, "many")
    run_case(pkg, m, 1920, 70, run, w_fmt, scale, w_fmt == 0, x_type, torch.float32, "many")


@pytest.mark.parametrize("k", [32, 64, 256, 288, 1056, 2048, 8192, 28672])
@pytest.mark.parametrize("m,n", [(17, 1), (32, 200), (64, 129), (130, 63)])
def test_lengths_with_many_rows(pkg, k, m, n):
    """K from a part of a piece to scales that are staged in several parts."""
    for w_fmt in (0, 1):
        run_case(pkg, m, k, n, 32, w_fmt, torch.float32, w_fmt == 0, torch.bfloat16, torch.float32, "lengths")
        if k % 128 == 0:
            run_case(pkg, m, k, n, 128, w_fmt, torch.float16, False, torch.float16, torch.float32, "lengths")


@pytest.mark.parametrize("counts", [[33, 0, 1, 20], [200, 0, 7], [16, 17, 15, 32, 31], [129, 64]])
@pytest.mark.parametrize("w_fmt,run,scale,x_type", [(0, 128, torch.float16, torch.float16), (1, 32, torch.uint8, torch.bfloat16), (0, 64, torch.bfloat16, F8[1]), (1, 32, torch.float32, F8[0])])
def test_experts_with_many_rows(pkg, counts, w_fmt, run, scale, x_type):
    """Passes over more rows than are held at once; rows in front of the first expert and behind the last stay."""
    gen = generator("many", counts, run)
    e, n, k = len(counts), 150, 1152
    w, s, z = weights(gen, (e,), n, k, run, w_fmt, scale, w_fmt == 0)
    m = sum(counts) + 5
    off = offsets_of(counts, 2)
    x = torch.randn((m, k), generator=gen, device="cuda").to(x_type)
    y = torch.full((m, n), 9.0, device="cuda")
    pkg.gemv_w4(x, w, s, run, w_fmt=w_fmt, zeros=z, row_offsets=off, out=y)
    for g in range(e):
        lo, hi = int(off[g]), int(off[g + 1])
        if hi > lo:
            ref = x[lo:hi].double() @ w4_values(w[g], s[g], run, w_fmt, None if z is None else z[g]).t().contiguous()
            bound = (62.0 if w_fmt == 0 else 6.0) * scale_values(s[g]).repeat_interleave(run, -1)
            assert ((y[lo:hi].double() - ref).abs() <= tolerance(x[lo:hi].double(), None, bound, torch.float32, ref)).all()
    assert (y[:2] == 9.0).all() and (y[int(off[e]):] == 9.0).all()


def test_operands_that_end_with_their_memory(pkg):
    """What lies behind x and W, NaNs here, stays out of the results (a K that ends inside a piece)."""
    gen = generator("end")
    for m in (3, 20, 50):
        for k, n in ((288, 33), (32, 65), (1056, 150)):
            w, s, z = weights(gen, (), n, k, 32, 0, torch.float16, True)
            x = torch.randn((m, k), generator=gen, device="cuda").to(torch.bfloat16)
            want = pkg.gemv_w4(x, w, s, 32, zeros=z)
            store = torch.full((m * k + 4096,), float("nan"), dtype=torch.bfloat16, device="cuda")
            x2 = store[:m * k].view(m, k).copy_(x)
            s2 = torch.full((s.numel() + 4096,), float("nan"), dtype=s.dtype, device="cuda")[:s.numel()].view(s.shape).copy_(s)
            assert torch.equal(pkg.gemv_w4(x2, w, s2, 32, zeros=z), want)


@pytest.mark.parametrize("x_type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("run", [32, 128])
def test_every_nibble_in_every_place(pkg, x_type, run):
    """One-hot rows of x: each output is one weight, exactly."""
    for w_fmt, zeros in ((0, None), (0, True), (1, None)):
        n, k = 33, 256
        w = (torch.arange(n * k // 2, device="cuda") * 37 % 256).to(torch.uint8).view(n, k // 2)
        s = pow2(torch.arange(n * (k // run), device="cuda") % 9 - 4).float().view(n, k // run)
        z = (torch.arange(n * (k // run), device="cuda") % 16).to(torch.uint8).view(n, k // run) if zeros else None
        v = w4_values(w, s, run, w_fmt, z)
        for k0 in range(0, k, 64):
            x = torch.zeros((64, k), dtype=x_type, device="cuda")
            x[torch.arange(64), torch.arange(k0, k0 + 64)] = 1
            assert torch.equal(pkg.gemv_w4(x, w, s, run, w_fmt=w_fmt, zeros=z).double(), v[:, k0:k0 + 64].t())


def test_scale_bytes(pkg):
    """Every power of two that a scale byte can name, NaN for 255: one-hot rows, fp32 results."""
    n, k = 256, 32
    w = torch.full((n, k // 2), 0x22, dtype=torch.uint8, device="cuda")         # e2m1 1.0
    s = torch.arange(256, device="cuda").to(torch.uint8).view(n, 1)
    for x_type in (torch.bfloat16, torch.float16):
        x = torch.zeros((1, k), dtype=x_type, device="cuda")
        x[0, 5] = 1
        y = pkg.gemv_w4(x, w, s, 32, w_fmt=1)[0].double()
        assert torch.isnan(y[255])
        want = pow2(torch.arange(255, device="cuda") - 127)
        # (2^-127 is a subnormal fp32 number, which a product may flush)
        assert torch.equal(y[1:255], want[1:]) and float(y[0]) in (0.0, 2.0 ** -127)


def test_nan_and_infinity_stay_in_their_row(pkg):
    gen = generator("nan")
    for w_fmt in (0, 1):
        w, s, _ = weights(gen, (), 48, 512, 128, w_fmt, torch.float16, False)
        x = torch.randn((20, 512), generator=gen, device="cuda").to(torch.bfloat16)
        x[3, 100], x[19, 7] = float("nan"), float("inf")
        y = pkg.gemv_w4(x, w, s, 128, w_fmt=w_fmt)
        odd = ~torch.isfinite(y)
        assert torch.isnan(y[3]).all()
        rest = [r for r in range(20) if r not in (3, 19)]
        assert not odd[rest].any()
        clean = x.clone()
        clean[3, 100] = clean[19, 7] = 0
        assert torch.equal(pkg.gemv_w4(clean, w, s, 128, w_fmt=w_fmt)[rest], y[rest])


@pytest.mark.parametrize("counts", [[1], [0, 1, 0, 3, 17, 0], [70, 0, 2], [1] * 40])
@pytest.mark.parametrize("w_fmt,run,scale", [(0, 128, torch.float16), (1, 32, torch.uint8), (0, 32, torch.bfloat16)])
def test_experts(pkg, counts, w_fmt, run, scale):
    gen = generator("experts", counts, run)
    e, n, k = len(counts), 100, 640
    w, s, z = weights(gen, (e,), n, k, run, w_fmt, scale, w_fmt == 0)
    m = sum(counts) + 5
    off = offsets_of(counts, 2)
    x = torch.randn((m, k), generator=gen, device="cuda").to(torch.bfloat16)
    y = torch.full((m, n), 9.0, device="cuda")
    pkg.gemv_w4(x, w, s, run, w_fmt=w_fmt, zeros=z, row_offsets=off, out=y)
    for g in range(e):
        lo, hi = int(off[g]), int(off[g + 1])
        if hi > lo:
            v = w4_values(w[g], s[g], run, w_fmt, None if z is None else z[g])
            ref = x[lo:hi].double() @ v.t().contiguous()
            sd = scale_values(s[g]).repeat_interleave(run, -1) * (62.0 if w_fmt == 0 else 6.0)
            assert ((y[lo:hi].double() - ref).abs() <= tolerance(x[lo:hi].double(), v, sd, torch.float32, ref)).all()
    assert (y[:2] == 9.0).all() and (y[int(off[-1]):] == 9.0).all()


def test_many_experts_and_results_anywhere(pkg):
    gen = generator("1024")
    counts = [0] * 1024
    for g, c in ((0, 3), (1, 1), (500, 40), (1023, 2)):
        counts[g] = c
    n, k, run = 40, 256, 64
    w, s, z = weights(gen, (1024,), n, k, run, 0, torch.float16, True)
    off = offsets_of(counts)
    m = sum(counts)
    x = torch.randn((m, k), generator=gen, device="cuda").to(torch.float16)
    for dtype in (torch.float32, torch.bfloat16):
        store = torch.full((m * n + 9,), 3.0, dtype=dtype, device="cuda")
        y = store[3:3 + m * n].view(m, n)
        pkg.gemv_w4(x, w, s, run, zeros=z, row_offsets=off, out=y)
        for g in (0, 1, 500, 1023):
            lo, hi = int(off[g]), int(off[g + 1])
            ref = x[lo:hi].double() @ w4_values(w[g], s[g], run, 0, z[g]).t().contiguous()
            bound = 62.0 * s[g].double().repeat_interleave(run, -1)
            assert ((y[lo:hi].double() - ref).abs() <= tolerance(x[lo:hi].double(), None, bound, dtype, ref)).all()
        assert (store[:3] == 3.0).all() and (store[3 + m * n:] == 3.0).all()


def test_experts_with_more_rows_than_the_average(pkg):
    """One expert has nearly all rows: x is staged in pieces where the plan had it whole."""
    gen = generator("skew")
    for n, k, run, w_fmt, scale, x_type in ((96, 8192, 128, 0, torch.float16, torch.bfloat16), (4096, 4096, 32, 1, torch.uint8, torch.bfloat16), (96, 28672, 128, 1, torch.float32, torch.float16)):
        counts = [0, 1, 61, 0, 2, 0, 0, 0]
        w, s, z = weights(gen, (8,), n, k, run, w_fmt, scale, w_fmt == 0)
        off = offsets_of(counts)
        x = torch.randn((64, k), generator=gen, device="cuda").to(x_type)
        y = pkg.gemv_w4(x, w, s, run, w_fmt=w_fmt, zeros=z, row_offsets=off)
        for g in (1, 2, 4):
            lo, hi = int(off[g]), int(off[g + 1])
            ref = x[lo:hi].double() @ w4_values(w[g], s[g], run, w_fmt, None if z is None else z[g]).t().contiguous()
            bound = (62.0 if w_fmt == 0 else 6.0) * scale_values(s[g]).repeat_interleave(run, -1)
            assert ((y[lo:hi].double() - ref).abs() <= tolerance(x[lo:hi].double(), None, bound, torch.float32, ref)).all()


def test_odd_places_of_scales(pkg):
    """Scales and zero points that cannot be read 16 bytes at a time: off 16 bytes, rows that are not whole pieces."""
    gen = generator("odd")
    for k, run in ((1024, 32), (1152, 128), (1024, 128)):
        n = 50
        w, s, z = weights(gen, (), n, k, run, 0, torch.float16, True)
        x = torch.randn((5, k), generator=gen, device="cuda").to(torch.bfloat16)
        want = pkg.gemv_w4(x, w, s, run, zeros=z)
        for shift in (1, 4):
            s2 = torch.zeros(s.numel() + 8, dtype=s.dtype, device="cuda")[shift:shift + s.numel()].view(s.shape).copy_(s)
            z2 = torch.zeros(z.numel() + 8, dtype=z.dtype, device="cuda")[shift:shift + z.numel()].view(z.shape).copy_(z)
            assert torch.equal(pkg.gemv_w4(x, w, s2, run, zeros=z2), want)


def test_captured_and_replayed_with_other_rows(pkg):
    gen = generator("graph")
    w, s, z = weights(gen, (4,), 256, 512, 64, 0, torch.float16, True)
    x = torch.randn((24, 512), generator=gen, device="cuda").to(torch.float16)
    off = offsets_of([6, 6, 6, 6])
    y = pkg.gemv_w4(x, w, s, 64, zeros=z, row_offsets=off)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.gemv_w4(x, w, s, 64, zeros=z, row_offsets=off, out=y)
    for cut in ([24, 0, 0, 0], [0, 1, 22, 1], [0, 0, 0, 24]):
        off.copy_(offsets_of(cut))
        x.copy_(torch.randn((24, 512), generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, pkg.gemv_w4(x, w, s, 64, zeros=z, row_offsets=off))


def test_weights_beyond_32_bits(pkg):
    """Offsets into the weights, their scales and the outputs past 2^32 bytes: the last experts of a large set."""
    gen = generator("large")
    e, n, k, run = 40, 28672, 8192, 128                        # 4.7 GB of weights
    w = torch.randint(0, 256, (e, n, k // 2), generator=gen, dtype=torch.uint8, device="cuda")
    s = (torch.rand((e, n, k // run), generator=gen, device="cuda") + 0.5).to(torch.float16)
    x = torch.randn((3, k), generator=gen, device="cuda").to(torch.bfloat16)
    off = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    off[38:] = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")       # one row each for experts 37, 38, 39
    y = pkg.gemv_w4(x, w, s, run, row_offsets=off)
    for r, g in enumerate((37, 38, 39)):
        v = w4_values(w[g, -2000:], s[g, -2000:], run, 0)
        ref = x[r:r + 1].double() @ v.t().contiguous()
        bound = 62.0 * s[g, -2000:].double().repeat_interleave(run, -1)
        assert ((y[r:r + 1, -2000:].double() - ref).abs() <= tolerance(x[r:r + 1].double(), v, bound, torch.float32, ref)).all()


def test_many_rows_captured_and_replayed(pkg):
    gen = generator("many graph")
    n, k, run = 200, 2304, 64
    w, s, z = weights(gen, (3,), n, k, run, 0, torch.float16, True)
    x = torch.randn((90, k), generator=gen, device="cuda").to(torch.bfloat16)
    off = offsets_of([40, 0, 50])
    y = torch.zeros((90, n), device="cuda")
    pkg.gemv_w4(x, w, s, run, zeros=z, row_offsets=off, out=y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.gemv_w4(x, w, s, run, zeros=z, row_offsets=off, out=y)
    for counts in ([40, 0, 50], [1, 88, 1], [0, 0, 90], [30, 30, 30]):
        x.copy_(torch.randn((90, k), generator=gen, device="cuda"))
        off.copy_(offsets_of(counts))
        y.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, pkg.gemv_w4(x, w, s, run, zeros=z, row_offsets=off))
        for g in range(3):
            lo, hi = int(off[g]), int(off[g + 1])
            if hi > lo:
                ref = x[lo:hi].double() @ w4_values(w[g], s[g], run, 0, z[g]).t().contiguous()
                bound = 62.0 * scale_values(s[g]).repeat_interleave(run, -1)
                assert ((y[lo:hi].double() - ref).abs() <= tolerance(x[lo:hi].double(), None, bound, torch.float32, ref)).all()


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("x_type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("w_fmt", [1, 0])
def test_scale_bytes_with_every_weight(pkg, w_fmt, x_type, many):
    """Every scale byte with every 4-bit weight and numbers of x from one end of the type to the other: one-hot rows, exact
    wherever weight, scale and their product are numbers that the header speaks of."""
    k = 64
    powers = [-126, -100, -60, -20, -1, 0, 1, 20, 60, 100, 115, 127] if x_type == torch.bfloat16 else list(range(-14, 16, 3))
    if w_fmt == 0:
        powers = [p for p in powers if p <= 115]           # (16 + q) x has to stay a number
    m = 40 if many else len(powers)
    place = torch.tensor([r * 7 % k for r in range(m)], device="cuda")
    exps = torch.tensor([powers[r % len(powers)] for r in range(m)], device="cuda")
    x = torch.zeros((m, k), dtype=torch.float64, device="cuda")
    x[torch.arange(m), place] = pow2(exps)
    # column: one byte and one weight, the weight in every place of the row
    byte, code = (t.flatten() for t in torch.meshgrid(torch.arange(256, device="cuda"), torch.arange(16, device="cuda"), indexing="ij"))
    w = (code * 17).to(torch.uint8)[:, None].expand(-1, k // 2).contiguous()
    s = byte.to(torch.uint8)[:, None].expand(-1, 2).contiguous()
    y = pkg.gemv_w4(x.to(x_type), w, s, 32, w_fmt=w_fmt).double()
    value = torch.tensor(E2M1 + [-t for t in E2M1], dtype=torch.float64, device="cuda")[code] if w_fmt == 1 else code.double() - 8.0
    assert torch.isnan(y[:, byte == 255]).all()
    want = pow2(exps)[:, None] * (value * pow2(byte - 127))[None, :]
    ok = (byte < 255)[None, :] & ((want == 0) | ((want.abs() >= 2.0 ** -126) & (want.abs() < 2.0 ** 128)))
    if w_fmt == 1 and x_type == torch.bfloat16:
        ok &= ((value * pow2(byte - 127)).abs() < 2.0 ** 128)[None, :]        # as a bf16 number it would be an infinity
    assert torch.equal(y[ok], want[ok]), "%d of %d differ" % (int((y[ok] != want[ok]).sum()), int(ok.sum()))
