"""Products with 4-bit weights on numbers whose sums are exact, so that results have to be equal: a length, a layout or a
place at which a piece of K is lost, repeated or scaled wrongly cannot hide behind a tolerance.

x holds whole numbers up to 3 and the scales are 1/2, 1 or 2.  Whatever the order, every sum is then a multiple of 1/4 (e2m1;
1/2 for integers) and below 2^24 such units: e2m1 28672 * 6 * 3 * 2 / (1/4) = 4.1e6, integers 28672 * 15 * 3 * 2 / (1/2) =
5.2e6, and a run's sum of (16 + q) x at most 128 * 31 * 3 = 11904.  All are fp32 numbers."""
import zlib

import pytest
import torch

from expert_util import F8, W4_LAYOUTS, offsets_of, scale_values, w4_values

pytestmark = pytest.mark.gpu

X_TYPES = {1: torch.bfloat16, 2: torch.float16, 3: F8[0], 4: F8[1]}
SCALE_TYPES = {0: torch.float32, 1: torch.bfloat16, 2: torch.float16, 5: torch.uint8}


def generator(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def whole(gen, lead, m, n, k, x_type, w_fmt, run, scale):
    """x, w, scales, zeros as the header lays them out."""
    x = torch.randint(-3, 4, (m, k), generator=gen, device="cuda", dtype=torch.int8).to(torch.float32).to(X_TYPES[x_type])
    w = torch.randint(0, 256, lead + (n, k // 2), generator=gen, dtype=torch.uint8, device="cuda")
    s = torch.randint(126, 129, lead + (n, k // run), generator=gen, dtype=torch.uint8, device="cuda")
    z = torch.randint(0, 16, lead + (n, k // run), generator=gen, dtype=torch.uint8, device="cuda") if w_fmt == 0 else None
    return x, w, s if scale == 5 else scale_values(s).to(SCALE_TYPES[scale]), z


def product(x, w, s, run, w_fmt, z):
    """(m, n) in 64 bits, some columns at a time."""
    out = torch.empty((x.shape[0], w.shape[0]), dtype=torch.float64, device="cuda")
    step = max(1, (1 << 27) // x.shape[1])
    for c in range(0, w.shape[0], step):
        out[:, c:c + step] = x.double() @ w4_values(w[c:c + step], s[c:c + step], run, w_fmt, None if z is None else z[c:c + step]).t().contiguous()
    return out


def check_experts(y, off, x, w, s, run, w_fmt, z):
    for g in range(w.shape[0]):
        lo, hi = int(off[g]), int(off[g + 1])
        if hi > lo:
            want = product(x[lo:hi], w[g], s[g], run, w_fmt, None if z is None else z[g])
            assert torch.equal(y[lo:hi].double(), want), "expert %d: %d of %d differ" % (g, int((y[lo:hi].double() != want).sum()), want.numel())


@pytest.mark.parametrize("k", [32, 96, 256, 288, 1056, 4128, 8192, 28672])
@pytest.mark.parametrize("m", [1, 3, 16, 17, 32, 64, 130])
def test_every_length(pkg, m, k):
    """From a part of a stage to lengths that are staged in several pieces; every 256 k matter to the result."""
    for x_type, w_fmt, run, scale in ((1, 0, 32, 0), (2, 0, 128, 2), (1, 1, 32, 5), (1, 1, 128, 5), (2, 1, 32, 2), (4, 0, 32, 1)):
        if k % run:
            continue
        for n in (1, 16, 130):
            gen = generator("length", m, k, n, x_type, w_fmt, run)
            x, w, s, z = whole(gen, (), m, n, k, x_type, w_fmt, run, scale)
            want = product(x, w, s, run, w_fmt, z)
            assert torch.equal(pkg.gemv_w4(x, w, s, run, w_fmt=w_fmt, zeros=z).double(), want), (x_type, w_fmt, run, n)
            if n == 130:
                v = w4_values(w, s, run, w_fmt, z)
                for k0 in range(0, k, 256):
                    assert (x[:, k0:k0 + 256].double() @ v[:, k0:k0 + 256].t().contiguous()).any()


@pytest.mark.parametrize("index", range(len(W4_LAYOUTS)))
def test_every_layout(pkg, index):
    """All waves along K, blocks of columns one behind the other, scales of one, several and all blocks, K in pieces."""
    groups, m, k, n, x_type, w_fmt, run, scale, layout = W4_LAYOUTS[index]
    assert pkg.w4_plan(m, k, n, x_type, w_fmt, run, scale, groups) == layout
    gen = generator("layout", index)
    x, w, s, z = whole(gen, (groups,) if groups > 1 else (), m, n, k, x_type, w_fmt, run, scale)
    if groups == 1:
        y = pkg.gemv_w4(x, w, s, run, w_fmt=w_fmt, zeros=z)
        assert torch.equal(y.double(), product(x, w, s, run, w_fmt, z))
        return
    cuts = [[m // groups + (g < m % groups) for g in range(groups)], [0] * (groups - 1) + [m], [m - 1] + [0] * (groups - 2) + [1]]
    for counts in cuts:                                # as planned; all rows, and all but one, to one expert
        off = offsets_of(counts)
        y = torch.full((m, n), float("nan"), device="cuda")
        pkg.gemv_w4(x, w, s, run, w_fmt=w_fmt, zeros=z, row_offsets=off, out=y)
        check_experts(y, off, x, w, s, run, w_fmt, z)


@pytest.mark.parametrize("groups,counts", [(8, [0, 1, 21, 0, 2, 0, 0, 0]), (8, [16, 0, 0, 1, 0, 0, 7, 0]), (32, [1] * 12 + [0, 12] + [0] * 18)])
@pytest.mark.parametrize("n,k,x_type,w_fmt,run,scale", [(96, 4096, 1, 0, 128, 2), (96, 8192, 1, 0, 32, 0), (4096, 4096, 1, 1, 32, 5), (130, 8192, 2, 1, 128, 2), (1100, 2048, 1, 0, 32, 2)])
def test_experts_with_more_rows_than_planned(pkg, groups, counts, n, k, x_type, w_fmt, run, scale):
    """An expert has more rows than the layout took it to have: the streaming kernel stages x anew, where it does not fit in
    pieces of K (16 rows of 8192 are more than a CU's LDS)."""
    m = sum(counts)
    layout = pkg.w4_plan(m, k, n, x_type, w_fmt, run, scale, groups)
    assert layout[0] == 16 and layout[5] < min(16, max(counts))
    gen = generator("skew", groups, counts, n, k)
    x, w, s, z = whole(gen, (groups,), m + 5, n, k, x_type, w_fmt, run, scale)
    off = offsets_of(counts, 2)
    y = torch.full((m + 5, n), 9.0, device="cuda")
    pkg.gemv_w4(x, w, s, run, w_fmt=w_fmt, zeros=z, row_offsets=off, out=y)
    check_experts(y, off, x, w, s, run, w_fmt, z)
    assert (y[:2] == 9.0).all() and (y[m + 2:] == 9.0).all()


@pytest.mark.parametrize("counts", [[0, 1, 61, 0, 2, 0, 0, 0], [200, 0, 7], [33, 0, 1, 20]])
@pytest.mark.parametrize("n,k,x_type,w_fmt,run,scale", [(96, 8192, 1, 0, 128, 2), (2100, 4096, 1, 1, 32, 5), (96, 28672, 2, 1, 32, 0), (200, 1056, 3, 0, 32, 1)])
def test_experts_with_many_rows(pkg, counts, n, k, x_type, w_fmt, run, scale):
    """The kernel for more rows, several passes over an expert's rows, scales of K in parts."""
    m, groups = sum(counts), len(counts)
    assert pkg.w4_plan(m, k, n, x_type, w_fmt, run, scale, groups)[0] > 16
    gen = generator("tall", counts, n, k)
    x, w, s, z = whole(gen, (groups,), m, n, k, x_type, w_fmt, run, scale)
    off = offsets_of(counts)
    y = torch.full((m, n), float("nan"), device="cuda")
    pkg.gemv_w4(x, w, s, run, w_fmt=w_fmt, zeros=z, row_offsets=off, out=y)
    check_experts(y, off, x, w, s, run, w_fmt, z)


def test_weights_beyond_32_bits(pkg):
    """Offsets into the weights past 2^32 bytes: the last experts of a large set, several blocks of columns a workgroup."""
    gen = generator("large")
    e, n, k, run = 40, 28672, 8192, 128                        # 4.7 GB of weights
    x, w, s, _ = whole(gen, (e,), 3, n, k, 1, 1, run, 2)
    off = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    off[38:] = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")       # one row each for experts 37, 38, 39
    y = pkg.gemv_w4(x, w, s, run, w_fmt=1, row_offsets=off)
    check_experts(y, off, x, w, s, run, 1, None)


@pytest.mark.parametrize("m", [3, 20, 50])
@pytest.mark.parametrize("k,n,run", [(288, 33, 32), (32, 65, 32), (1056, 150, 96), (384, 17, 128)])
def test_weights_and_zeros_that_end_with_their_memory(pkg, m, k, n, run):
    """What lies behind W and the zero points, whatever its bits, stays out of the results (every byte is a number, so two
    fills are compared), and what lies behind x and the scales is no number at all."""
    gen = generator("end", m, k, n)
    x, w, s, z = whole(gen, (), m, n, k, 1, 0, run, 2)
    want = product(x, w, s, run, 0, z)

    def embedded(t, fill):
        store = torch.full((t.numel() + 8192,), fill, dtype=t.dtype, device="cuda")
        return store[:t.numel()].view(t.shape).copy_(t)

    for byte in (0x00, 0xFF, 0x77):
        y = pkg.gemv_w4(embedded(x, float("nan")), embedded(w, byte), embedded(s, float("nan")), run, zeros=embedded(z, byte))
        assert torch.equal(y.double(), want)
        y = pkg.gemv_w4(embedded(x, float("nan")), embedded(w, byte), embedded(s, float("inf")), run, w_fmt=1)
        assert torch.equal(y.double(), product(x, w, s, run, 1, None))
