"""Products of rows grouped by expert and their weight gradient, through the C ABI, against 64-bit sums."""
import zlib

import pytest
import torch

from expert_util import F8, codes, fp8_product, offsets_of, places, pow2, rounding

pytestmark = pytest.mark.gpu

PAIRS = [(0, 0), (1, 1), (0, 1), (1, 0)]
ROWS_VARIANTS, WGRAD_VARIANTS = [-1, 0, 13, 14, 15, 17, 18, 19], [-1, 13, 15, 18, 19]
WHOLE_K_TILES = (14, 15, 17)             # not compiled for a K that is not a multiple of 128
# rows of each expert: empty ones at either end and between, single rows, more rows than any tile, less than one
COUNTS = {"one": [1], "ragged": [0, 3, 0, 130, 1, 64, 0], "tall": [300, 0, 513], "many": [i % 5 for i in range(70)], "none": [0, 0, 0]}


def generator(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def powers(gen, *shape):
    return pow2(torch.randint(-4, 5, shape, generator=gen, device="cuda")).float()


def check(out, ref, tol):
    assert torch.isfinite(out.float()).all()
    err = (out.double() - ref).abs()
    assert (err <= tol).all(), "worst err/tol %g" % float((err / tol).max())


def case(gen, counts, k, n, fa, fb, behind=0):
    off = offsets_of(counts)
    m = max(1, sum(counts) + behind)
    return off, codes(gen, (m, k), fa), codes(gen, (len(counts), n, k), fb)


def check_rows(out, off, a, b, sa, sb, dtype):
    for g in range(b.shape[0]):
        lo, hi = int(off[g]), int(off[g + 1])
        if hi == lo:
            continue
        y, tol = fp8_product(a[lo:hi].double(), b[g].double())
        f = 1.0
        if sa is not None:
            f = f * sa[lo:hi, None].double()
        if sb is not None:
            f = f * (sb[g].double() if sb.dim() == 2 else sb[g].double())
        check(out[lo:hi], y * f, tol * (f if torch.is_tensor(f) else 1.0) + rounding(y * f, dtype) * 1.0001)


@pytest.mark.parametrize("variant", ROWS_VARIANTS)
@pytest.mark.parametrize("counts", list(COUNTS))
@pytest.mark.parametrize("k,n", [(128, 256), (272, 130), (512, 301), (1024, 4), (384, 260)])
def test_grouped_every_kernel(pkg, variant, counts, k, n):
    """Every compiled tile shape, ragged rows, columns that overhang tiles and are not whole quads, a K that overhangs its
    last tile, an odd count of K tiles."""
    if variant in (13, 14) and k <= 128:
        pytest.skip("the 16x16x128 tile needs two K tiles")
    if variant in WHOLE_K_TILES and k % 128:
        pytest.skip("whole K tiles only")
    gen = generator("rows", counts, k, n)
    off, a, b = case(gen, COUNTS[counts], k, n, 0, 0, behind=3)
    sa, sb = powers(gen, a.shape[0]), powers(gen, b.shape[0], n)
    out = torch.full((a.shape[0], n), 777.0, dtype=torch.bfloat16, device="cuda")
    pkg.gemm_grouped(a, b, off, a_scale=sa, b_scale=sb, out=out, variant=variant)
    check_rows(out, off, a, b, sa, sb, torch.bfloat16)
    assert (out[int(off[-1]):] == 777.0).all()                 # rows behind the last expert


@pytest.mark.parametrize("fa,fb", PAIRS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("variant", ROWS_VARIANTS)
def test_grouped_types_and_pairings(pkg, fa, fb, dtype, variant):
    gen = generator("types", fa, fb)
    off, a, b = case(gen, [70, 0, 33], 256, 192, fa, fb)
    sb = powers(gen, 3)
    out = pkg.gemm_grouped(a, b, off, b_scale=sb, out_dtype=dtype, variant=variant)        # one scale an expert, none for rows
    check_rows(out, off, a, b, None, sb, dtype)
    out = pkg.gemm_grouped(a, b, off, out_dtype=dtype, variant=variant)
    check_rows(out, off, a, b, None, None, dtype)


@pytest.mark.parametrize("k,n,shift", [(100, 70, 0), (1, 1, 0), (17, 33, 0), (64, 40, 1), (256, 64, 3)])
def test_grouped_any_k_and_alignment(pkg, k, n, shift):
    """Rows that are not whole 16-byte pieces, and operands that do not start on one, run on the general kernel."""
    gen = generator("any", k, n, shift)
    counts = [5, 0, 40, 1]
    off, a, b = case(gen, counts, k, n, 0, 1)
    store = torch.zeros(b.numel() + shift, dtype=torch.uint8, device="cuda")
    store[shift:] = b.view(torch.uint8).flatten()
    bs = store[shift:].view(F8[1]).view(b.shape)
    out = pkg.gemm_grouped(a, bs, off, out_dtype=torch.float32)
    check_rows(out, off, a, b, None, None, torch.float32)


@pytest.mark.parametrize("variant", ROWS_VARIANTS)
def test_grouped_nan_stays_in_its_rows_and_columns(pkg, variant):
    """A NaN code in one expert's matrix reaches that expert's rows only, one in a row only that row."""
    gen = generator("nan")
    off, a, b = case(gen, [20, 30, 14], 256, 128, 0, 0)
    b.view(torch.uint8)[1, 5, 7] = 0x7F
    a.view(torch.uint8)[60, 9] = 0x7F
    out = pkg.gemm_grouped(a, b, off, out_dtype=torch.float32, variant=variant)
    want = torch.zeros_like(out, dtype=torch.bool)
    want[20:50, 5] = True
    want[60] = True
    assert torch.equal(torch.isnan(out), want)


def test_grouped_offsets_that_are_no_cut_of_the_rows(pkg):
    """Offsets outside the matrix are clamped, one below an earlier one is raised to it; on every kernel."""
    gen = generator("bad")
    a, b = codes(gen, (100, 256), 0), codes(gen, (4, 128, 256), 0)
    bad = torch.tensor([-7, 40, 10, 2000, 50], dtype=torch.int32, device="cuda")
    meant = torch.tensor([0, 40, 40, 100, 100], dtype=torch.int32, device="cuda")
    for variant in ROWS_VARIANTS:
        out = pkg.gemm_grouped(a, b, bad, out_dtype=torch.float32, variant=variant)
        assert torch.equal(out, pkg.gemm_grouped(a, b, meant, out_dtype=torch.float32, variant=variant))
    first = torch.tensor([30, 40, 50, 60, 70], dtype=torch.int32, device="cuda")
    for variant in ROWS_VARIANTS:
        out = torch.full((100, 128), 5.0, device="cuda")
        pkg.gemm_grouped(a, b, first, out=out, variant=variant)
        check_rows(out, first, a, b, None, None, torch.float32)
        assert (out[:30] == 5.0).all() and (out[70:] == 5.0).all()


def test_grouped_equals_the_gemm_of_each_expert(pkg):
    """Several rounds of tiles per workgroup; against the dense entry point on each expert's rows."""
    gen = generator("rounds")
    counts = [700, 0, 1500, 33, 900, 1200]
    off, a, b = case(gen, counts, 512, 2560, 0, 0)
    ref = torch.cat([pkg.gemm(a[int(off[g]):int(off[g + 1])].contiguous(), b[g].contiguous()) for g in range(6) if counts[g]])
    size = torch.cat([a[int(off[g]):int(off[g + 1])].float().abs() @ b[g].float().abs().t() for g in range(6)])
    for variant in [13, 14, 15, 17, 18, 19]:
        out = pkg.gemm_grouped(a, b, off, variant=variant)
        # each is off its sum by fp32 reordering and by 2^-13 of twice the largest product for each of 8 in a group (expert_util)
        assert ((out - ref).abs() <= 2 * (2 * 512 * 2.0 ** -24 + 2.0 ** -9) * size).all()


@pytest.mark.parametrize("variant", [13, 14, 15, 17, 18, 19])
def test_grouped_every_element_of_a_wide_store(pkg, variant):
    """fp32 results leave four at a time, and the registers they leave from are used again at once: many ragged tiles, every
    element, several times over (the store reads its registers late)."""
    gen = generator("stores")
    counts = [700, 0, 1500, 33, 900, 1200]
    off, a, b = case(gen, counts, 512, 2560, 0, 0)
    ref = torch.cat([a[int(off[g]):int(off[g + 1])].double() @ b[g].double().t().contiguous() for g in range(6)])
    # |a b| summed: fp32 reordering, and 2^-13 of twice the largest product for each of 8 in a group (expert_util)
    size = torch.cat([a[int(off[g]):int(off[g + 1])].double().abs() @ b[g].double().abs().t().contiguous() for g in range(6)])
    tol = 2 * 512 * 2.0 ** -24 * size + 2.0 ** -9 * size
    for _ in range(8):
        out = torch.full(ref.shape, float("nan"), device="cuda")
        pkg.gemm_grouped(a, b, off, out=out, variant=variant)
        check(out, ref, tol)


def test_grouped_output_beyond_31_bits(pkg):
    gen = generator("large")
    counts = [70001, 1, 0, 30]
    off, a, b = case(gen, counts, 128, 32768, 0, 0)
    out = torch.empty((sum(counts), 32768), dtype=torch.bfloat16, device="cuda")
    assert out.numel() > 2 ** 31
    for variant in [18, 19]:
        out[-40:] = 0
        pkg.gemm_grouped(a, b, off, out=out, variant=variant)
        rows = torch.tensor([0, 12345, 65535, 65536, 69999, 70000], device="cuda")
        y, tol = fp8_product(a.float()[rows].double(), b[0, :512].double())
        check(out[rows][:, :512], y, tol + rounding(y, torch.bfloat16) * 1.0001)
        for g in (1, 3):
            lo, hi = int(off[g]), int(off[g + 1])
            y, tol = fp8_product(a[lo:hi].double(), b[g, -512:].double())
            check(out[lo:hi, -512:], y, tol + rounding(y, torch.bfloat16) * 1.0001)


def test_grouped_captured_and_replayed_with_other_offsets(pkg):
    """A captured call reads the offsets when it runs: replayed with other cuts, eager work between."""
    gen = generator("graph")
    off, a, b = case(gen, [100, 28, 0, 72], 256, 256, 0, 0)
    for variant in ROWS_VARIANTS:
        out = torch.zeros((200, 256), device="cuda")
        pkg.gemm_grouped(a, b, off, out=out, variant=variant)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pkg.gemm_grouped(a, b, off, out=out, variant=variant)
        for cut in ([0, 0, 200, 0], [50, 50, 50, 50], [1, 198, 0, 1]):
            off.copy_(offsets_of(cut))
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, pkg.gemm_grouped(a, b, off, variant=variant))
            a.view(torch.uint8)[0, 0] ^= 1
        off.copy_(offsets_of([100, 28, 0, 72]))


def test_grouped_on_two_streams_at_once(pkg):
    gen = generator("streams")
    off, a, b = case(gen, [400, 100, 524], 1024, 1024, 0, 0)
    ref = pkg.gemm_grouped(a, b, off)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [torch.zeros_like(ref) for _ in range(8)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        pkg.gemm_grouped(a, b, off, out=o, stream=s1 if i % 2 else s2)
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_grouped_output_anywhere(pkg, dtype):
    """Results that do not start on 16 bytes; what lies around them stays."""
    gen = generator("place")
    off, a, b = case(gen, [40, 0, 25], 256, 132, 0, 0)
    for variant in ROWS_VARIANTS:
        for shift in (1, 2, 5):
            store = torch.full((65 * 132 + 16,), 3.0, dtype=dtype, device="cuda")
            out = store[shift:shift + 65 * 132].view(65, 132)
            pkg.gemm_grouped(a, b, off, out=out, variant=variant)
            check_rows(out, off, a, b, None, None, dtype)
            assert (store[:shift] == 3.0).all() and (store[shift + 65 * 132:] == 3.0).all()


def test_grouped_many_experts(pkg):
    """The largest number of experts, most of them without rows, rows in the first and the last."""
    gen = generator("1024")
    counts = [0] * 1024
    for g, c in ((0, 3), (1, 1), (63, 2), (64, 70), (500, 1), (1022, 5), (1023, 130)):
        counts[g] = c
    off = offsets_of(counts)
    m = sum(counts)
    a, b = codes(gen, (m, 256), 0), codes(gen, (1024, 64, 256), 0)
    for variant in ROWS_VARIANTS:
        out = pkg.gemm_grouped(a, b, off, out_dtype=torch.float32, variant=variant)
        check_rows(out, off, a, b, None, None, torch.float32)


# ---------------------------------------------------------------- weight gradient
def transposed(gen, counts, m, fmt, extra=0):
    """(m, ld) codes with every expert's tokens in whole runs of 128, zeros behind them; NaN codes where nothing may be read."""
    off = offsets_of(counts)
    at, counts, used = places(off.tolist(), sum(counts))
    ld = (max(1, sum(counts)) + 127 * len(counts)) // 128 * 128 + extra
    t = torch.zeros((m, ld), device="cuda").to(F8[fmt])
    for p, c in zip(at, counts):
        t.view(torch.uint8)[:, p:p + c] = codes(gen, (m, c), fmt).view(torch.uint8)
    t.view(torch.uint8)[:, used:] = 0x7F
    return off, t, at, counts


def check_wgrad(out, at, counts, a, b, sa, sb, dtype, before=None):
    for g, (p, c) in enumerate(zip(at, counts)):
        y, tol = fp8_product(a[:, p:p + c].double(), b[:, p:p + c].double()) if c else (torch.zeros_like(out[g], dtype=torch.float64), torch.zeros_like(out[g], dtype=torch.float64))
        f = (sa[g][:, None].double() if sa is not None else 1.0) * (sb[g].double() if sb is not None else torch.ones(b.shape[0], dtype=torch.float64, device="cuda"))
        y, tol = y * f, tol * f
        if before is not None:
            y = y + before[g].double()
            tol = tol + y.abs() * 2.0 ** -24
        check(out[g], y, tol + rounding(y, dtype) * 1.0001)


@pytest.mark.parametrize("variant", WGRAD_VARIANTS)
@pytest.mark.parametrize("counts", list(COUNTS))
@pytest.mark.parametrize("m,n", [(256, 256), (130, 300), (1, 1), (33, 4), (260, 127)])
def test_wgrad_every_kernel(pkg, variant, counts, m, n):
    if counts == "many" and m * n > 20000:
        pytest.skip("covered by the smaller sizes")
    gen = generator("wgrad", counts, m, n)
    off, a, at, cs = transposed(gen, COUNTS[counts], m, 1, extra=128)
    _, b, _, _ = transposed(gen, COUNTS[counts], n, 0, extra=128)
    rows = max(1, sum(cs))
    sa, sb = powers(gen, len(cs), m), powers(gen, len(cs), n)
    out = pkg.gemm_grouped_wgrad(a, b, off, rows, a_scale=sa, b_scale=sb, out_dtype=torch.bfloat16, variant=variant)
    check_wgrad(out, at, cs, a, b, sa, sb, torch.bfloat16)
    out = pkg.gemm_grouped_wgrad(a, b, off, rows, out_dtype=torch.float32, variant=variant)
    check_wgrad(out, at, cs, a, b, None, None, torch.float32)
    # added to what is there: an expert without rows keeps its matrix
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        held = torch.randn(out.shape, generator=gen, device="cuda").to(dtype)
        into = held.clone()
        pkg.gemm_grouped_wgrad(a, b, off, rows, a_scale=sa, out=into, accumulate=True, variant=variant)
        check_wgrad(into, at, cs, a, b, sa, None, dtype, before=held)
        for g, c in enumerate(cs):
            assert c or torch.equal(into[g], held[g])


@pytest.mark.parametrize("fa,fb", PAIRS)
@pytest.mark.parametrize("variant", [13, 15, 18, 19])
def test_wgrad_pairings(pkg, fa, fb, variant):
    gen = generator("wgrad pairs", fa, fb)
    off, a, at, cs = transposed(gen, [129, 2, 500], 192, fa)
    _, b, _, _ = transposed(gen, [129, 2, 500], 140, fb)
    out = pkg.gemm_grouped_wgrad(a, b, off, 631, out_dtype=torch.float16, variant=variant)
    check_wgrad(out, at, cs, a, b, None, None, torch.float16)


def test_wgrad_many_tiles_per_workgroup(pkg):
    """More tiles than the chip holds at once, experts of very different length."""
    gen = generator("wgrad rounds")
    counts = [1500, 0, 7, 300, 1]
    off, a, at, cs = transposed(gen, counts, 2100, 0)
    _, b, _, _ = transposed(gen, counts, 1900, 0)
    for variant in (13, 15, 18, 19):
        out = pkg.gemm_grouped_wgrad(a, b, off, sum(counts), variant=variant)
        for g, (p, c) in enumerate(zip(at, cs)):
            if not c:
                assert (out[g] == 0).all()
                continue
            pick = torch.randint(0, 2100, (64,), generator=gen, device="cuda")
            y, tol = fp8_product(a.float()[pick, p:p + c].double(), b[:, p:p + c].double())
            check(out[g][pick], y, tol + rounding(y, torch.float32) * 1.0001)


def test_wgrad_captured_and_replayed(pkg):
    gen = generator("wgrad graph")
    counts = [200, 0, 56]
    off, a, at, cs = transposed(gen, counts, 128, 0)
    _, b, _, _ = transposed(gen, counts, 256, 0)
    for variant in (13, 15, 18, 19):
        out = torch.zeros((3, 128, 256), device="cuda")
        pkg.gemm_grouped_wgrad(a, b, off, 256, out=out, variant=variant)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pkg.gemm_grouped_wgrad(a, b, off, 256, out=out, variant=variant)
        for _ in range(3):
            a.view(torch.uint8)[:, :200] = codes(gen, (128, 200), 0).view(torch.uint8)
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, pkg.gemm_grouped_wgrad(a, b, off, 256, variant=variant))


def test_wgrad_operands_that_end_with_their_memory(pkg):
    """Experts with fewer tokens than the tile's schedule walks, operands that fill their allocation to its last byte: the
    whole of both is one K tile, and nothing behind it may be touched."""
    gen = generator("wgrad end")
    for counts in ([32], [0, 128], [128, 0, 0]):
        off, a, at, cs = transposed(gen, counts, 16384, 0)
        a, rows = a[:, :128].contiguous(), 128
        _, b, _, _ = transposed(gen, counts, 16384, 0)
        ld = pkg.grouped_ld(rows, 1)
        assert ld == 128 and a.numel() == 2 << 20
        b = b[:, :128].contiguous()
        one = torch.tensor([0, sum(counts)], dtype=torch.int32, device="cuda")
        pick = torch.randint(0, 16384, (64,), generator=gen, device="cuda")
        y, tol = fp8_product(a.float()[pick].double(), b.double())
        for variant in (13, 15, 18, 19):
            check(pkg.gemm_grouped_wgrad(a, b, one, rows, variant=variant)[0][pick], y, tol + rounding(y, torch.float32) * 1.0001)


def test_wgrad_many_experts_and_results_beyond_31_bits(pkg):
    gen = generator("wgrad many")
    counts = [0] * 1024
    for g, c in ((0, 3), (64, 129), (1023, 7)):
        counts[g] = c
    off, a, at, cs = transposed(gen, counts, 2048, 0)
    _, b, _, _ = transposed(gen, counts, 1152, 0)
    for variant in (13, 15, 18, 19):
        out = torch.full((1024, 2048, 1152), 5.0, dtype=torch.bfloat16, device="cuda")
        assert out.numel() > 2 ** 31
        pkg.gemm_grouped_wgrad(a, b, off, sum(counts), out=out, variant=variant)
        for g in (0, 64, 1023):
            y, tol = fp8_product(a[-64:, at[g]:at[g] + cs[g]].double(), b[-100:, at[g]:at[g] + cs[g]].double())
            check(out[g, -64:, -100:], y, tol + rounding(y, torch.bfloat16) * 1.0001)
        for g in (1, 63, 500, 1022):
            assert not out[g].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_wgrad_output_anywhere(pkg, dtype):
    gen = generator("wgrad place")
    off, a, at, cs = transposed(gen, [100, 0, 30], 130, 0)
    _, b, _, _ = transposed(gen, [100, 0, 30], 68, 0)
    size = 3 * 130 * 68
    for variant in (13, 15, 18, 19):
        for shift in (1, 3):
            store = torch.full((size + 16,), 3.0, dtype=dtype, device="cuda")
            out = store[shift:shift + size].view(3, 130, 68)
            pkg.gemm_grouped_wgrad(a, b, off, 130, out=out, variant=variant)
            check_wgrad(out, at, cs, a, b, None, None, dtype)
            assert (store[:shift] == 3.0).all() and (store[shift + size:] == 3.0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [256, 131])
def test_wgrad_scales_of_experts_without_tokens(pkg, n, dtype):
    """Scales that are no numbers, at experts that have no tokens: zeros, or what was there to its last bit."""
    gen = generator("wgrad no tokens")
    counts, m = [0, 200, 0, 0, 3, 0], 300
    off, a, at, cs = transposed(gen, counts, m, 1)
    _, b, _, _ = transposed(gen, counts, n, 0)
    sa, sb = powers(gen, len(cs), m), powers(gen, len(cs), n)
    odd = torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda")
    for g, c in enumerate(cs):
        if not c:
            sa[g] = odd[torch.arange(m, device="cuda") % 3]
            sb[g] = odd[(torch.arange(n, device="cuda") + g) % 3]
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    held = torch.randn((len(cs), m, n), generator=gen, device="cuda").to(dtype)
    held[:, ::7] = -0.0
    held[:, 1::7] = float("inf")
    held[:, 2::7] = float("nan")
    for variant in WGRAD_VARIANTS:
        for x, y in ((sa, sb), (sa, None), (None, sb)):
            out = torch.full((len(cs), m, n), 5.0, dtype=dtype, device="cuda")
            pkg.gemm_grouped_wgrad(a, b, off, sum(cs), a_scale=x, b_scale=y, out=out, variant=variant)
            into = held.clone()
            pkg.gemm_grouped_wgrad(a, b, off, sum(cs), a_scale=x, b_scale=y, out=into, accumulate=True, variant=variant)
            for g, c in enumerate(cs):
                if not c:
                    assert not out[g].view(bits).any(), (variant, g)
                    assert torch.equal(into[g].view(bits), held[g].view(bits)), (variant, g)
            check_wgrad(out[[1, 4]], [at[1], at[4]], [cs[1], cs[4]], a, b, None if x is None else x[[1, 4]], None if y is None else y[[1, 4]], dtype)


def test_scales_with_exchanged_axes_are_refused(pkg):
    gen = generator("axes")
    off, a, b = case(gen, [3, 0, 5], 128, 64, 0, 0)
    with pytest.raises(pkg.Fp8GemmError):
        pkg.gemm_grouped(a, b, off, b_scale=powers(gen, 64, 3))
    _, at, _, _ = transposed(gen, [3, 0, 5], 48, 0)
    _, bt, _, _ = transposed(gen, [3, 0, 5], 64, 0)
    for sa, sb in ((powers(gen, 48, 3), None), (None, powers(gen, 64, 3))):
        with pytest.raises(pkg.Fp8GemmError):
            pkg.gemm_grouped_wgrad(at, bt, off, 8, a_scale=sa, b_scale=sb)
