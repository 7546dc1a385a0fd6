"""The operators for layers with experts together, as a layer uses them: tokens gathered by expert and quantised, the product,
the gradients of input and matrices, a decoding step on 4-bit matrices; eager, and captured into one HIP graph."""
import zlib

import pytest
import torch

from expert_util import codes, fp8_product, offsets_of, places, rounding, w4_values

pytestmark = pytest.mark.gpu

TOKENS, TOP, EXPERTS, K, N = 300, 2, 8, 256, 384


def generator(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def route(gen, off, index):
    """Two experts for every token: off (EXPERTS + 1) and index (TOKENS * TOP) are filled in place."""
    want = torch.randn((TOKENS, EXPERTS), generator=gen, device="cuda") + torch.linspace(1, -1, EXPERTS, device="cuda")
    expert = want.topk(TOP, dim=1).indices.flatten()
    order = torch.argsort(expert, stable=True)
    index.copy_((order // TOP).to(torch.int32))
    off[1:] = torch.cumsum(torch.bincount(expert, minlength=EXPERTS), 0).to(torch.int32)


class Layer:
    """y = x W[expert]^T on quantised operands, and its gradients."""

    def __init__(self, pkg, gen):
        self.pkg = pkg
        self.w = torch.randn((EXPERTS, N, K), generator=gen, device="cuda").to(torch.bfloat16)
        flat = lambda t: pkg.quantize_rows(t.reshape(-1, t.shape[-1]).contiguous())  # noqa: E731
        c, s = flat(self.w)
        self.wq, self.ws = c.view(EXPERTS, N, K), s.view(EXPERTS, N)
        c, s = flat(self.w.transpose(1, 2))
        self.wtq, self.wts = c.view(EXPERTS, K, N), s.view(EXPERTS, K)

    def step(self, x, dy, off, index):
        pkg = self.pkg
        xq, xs = pkg.quantize_rows(x, pkg.E4M3, row_index=index)
        y = pkg.gemm_grouped(xq, self.wq, off, a_scale=xs, b_scale=self.ws, out_dtype=torch.bfloat16)
        dyq, dys = pkg.quantize_rows(dy, pkg.E5M2)
        dx = pkg.gemm_grouped(dyq, self.wtq, off, a_scale=dys, b_scale=self.wts, out_dtype=torch.bfloat16)
        dyt, dyts = pkg.quantize_columns(dy, off, pkg.E5M2)
        xt, xts = pkg.quantize_columns(x, off, pkg.E4M3, row_index=index)
        dw = pkg.gemm_grouped_wgrad(dyt, xt, off, index.numel(), a_scale=dyts, b_scale=xts, out_dtype=torch.float32)
        return {"xq": xq, "xs": xs, "y": y, "dyq": dyq, "dys": dys, "dx": dx, "dyt": dyt, "dyts": dyts, "xt": xt, "xts": xts, "dw": dw}


def check_step(layer, off, r):
    at, counts, _ = places(off.tolist(), TOKENS * TOP)
    for g, c in enumerate(counts):
        lo = int(off[g])
        for a, sa, b, sb, out in ((r["xq"], r["xs"], layer.wq, layer.ws, r["y"]), (r["dyq"], r["dys"], layer.wtq, layer.wts, r["dx"])):
            y, tol = fp8_product(a[lo:lo + c].double(), b[g].double())
            f = sa[lo:lo + c, None].double() * sb[g].double()
            assert ((out[lo:lo + c].double() - y * f).abs() <= tol * f + rounding(y * f, torch.bfloat16) * 1.0001).all()
        y, tol = fp8_product(r["dyt"][:, at[g]:at[g] + c].double(), r["xt"][:, at[g]:at[g] + c].double())
        f = r["dyts"][g][:, None].double() * r["xts"][g].double()
        assert ((r["dw"][g].double() - y * f).abs() <= tol * f + rounding(y * f, torch.float32) * 1.0001).all()


def test_layer_forward_and_gradients(pkg):
    gen = generator("layer")
    layer = Layer(pkg, gen)
    x = torch.randn((TOKENS, K), generator=gen, device="cuda").to(torch.bfloat16)
    dy = (0.01 * torch.randn((TOKENS * TOP, N), generator=gen, device="cuda")).to(torch.bfloat16)
    off, index = torch.zeros(EXPERTS + 1, dtype=torch.int32, device="cuda"), torch.zeros(TOKENS * TOP, dtype=torch.int32, device="cuda")
    route(gen, off, index)
    r = layer.step(x, dy, off, index)
    check_step(layer, off, r)
    # the matrices' gradient against differences: the loss sum(dy * y) on the operands that the gradient saw, along a
    # random direction; it is linear in the matrices, so the difference is the derivative up to the products' tolerance
    at, counts, _ = places(off.tolist(), TOKENS * TOP)
    for g, c in enumerate(counts):
        a = r["dyt"][:, at[g]:at[g] + c].double() * r["dyts"][g][:, None].double()
        b = r["xt"][:, at[g]:at[g] + c].double() * r["xts"][g][:, None].double()
        d = torch.randn((N, K), generator=gen, device="cuda").double()
        loss = lambda w: (a.t().contiguous() * (b.t().contiguous() @ w.t().contiguous())).sum()  # noqa: E731
        w = layer.w[g].double()
        diff = (loss(w + 0.5 * d) - loss(w - 0.5 * d))
        _, tol = fp8_product(r["dyt"][:, at[g]:at[g] + c].double(), r["xt"][:, at[g]:at[g] + c].double())
        tol = tol * r["dyts"][g][:, None].double() * r["xts"][g].double() + r["dw"][g].double().abs() * 2.0 ** -23
        # (64-bit rounding of the two losses: their terms are at most ~1e5 in sum)
        assert (diff - (r["dw"][g].double() * d).sum()).abs() <= (tol * d.abs()).sum() + 1e-9


def test_layer_captured_and_replayed_with_other_routes(pkg):
    gen = generator("graph")
    layer = Layer(pkg, gen)
    x = torch.randn((TOKENS, K), generator=gen, device="cuda").to(torch.bfloat16)
    dy = torch.randn((TOKENS * TOP, N), generator=gen, device="cuda").to(torch.bfloat16)
    off, index = torch.zeros(EXPERTS + 1, dtype=torch.int32, device="cuda"), torch.zeros(TOKENS * TOP, dtype=torch.int32, device="cuda")
    route(gen, off, index)
    layer.step(x, dy, off, index)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = layer.step(x, dy, off, index)
    for _ in range(4):
        x.copy_(torch.randn((TOKENS, K), generator=gen, device="cuda"))
        route(gen, off, index)
        graph.replay()
        torch.cuda.synchronize()
        eager = layer.step(x, dy, off, index)
        for key in r:
            same = r[key].view(torch.uint8) if r[key].element_size() == 1 else r[key]
            assert torch.equal(same, eager[key].view(same.dtype) if same.dtype == torch.uint8 else eager[key]), key


def test_decoding_step_in_four_bits(pkg):
    """Hidden state to codes, gathered for its experts, through 4-bit matrices."""
    gen = generator("decode")
    run = 32
    w = torch.randint(0, 256, (EXPERTS, N, K // 2), generator=gen, dtype=torch.uint8, device="cuda")
    s = torch.randint(120, 128, (EXPERTS, N, K // run), generator=gen, dtype=torch.uint8, device="cuda")
    h = torch.randn((3, K), generator=gen, device="cuda").to(torch.bfloat16)
    index = torch.tensor([2, 0, 1, 0, 2, 1], dtype=torch.int32, device="cuda")
    off = offsets_of([1, 0, 2, 0, 0, 3, 0, 0])
    xq, xs = pkg.quantize_rows(h, pkg.E4M3, row_index=index)
    for x, scale in ((xq, xs), (h[index.long()].contiguous(), None)):
        y = pkg.gemv_w4(x, w, s, run, w_fmt=pkg.W4_E2M1, x_scale=scale, row_offsets=off, out_dtype=torch.bfloat16)
        xd = x.double() * (1.0 if scale is None else scale[:, None].double())
        for g in range(EXPERTS):
            lo, hi = int(off[g]), int(off[g + 1])
            if hi > lo:
                v = w4_values(w[g], s[g], run, 1)
                ref = xd[lo:hi] @ v.t().contiguous()
                tol = 2 * K * 2.0 ** -24 * (xd[lo:hi].abs() @ v.abs().t().contiguous()) + rounding(ref, torch.bfloat16) * 1.0001
                assert ((y[lo:hi].double() - ref).abs() <= tol).all()


def test_operands_on_another_stream_and_wrong_places(pkg):
    """Launches go to the current stream, or the one named; operands of two kinds of memory are refused."""
    gen = generator("streams")
    a, b = codes(gen, (64, 128), 0), codes(gen, (2, 64, 128), 0)
    off = offsets_of([30, 34])
    want = pkg.gemm_grouped(a, b, off)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.gemm_grouped(a, b, off)
    named = pkg.gemm_grouped(a, b, off, stream=side)
    side.synchronize()
    assert torch.equal(want, got) and torch.equal(want, named)
    for bad in (lambda: pkg.gemm_grouped(a, b, off.cpu()), lambda: pkg.gemm_grouped(a, b.cpu(), off), lambda: pkg.gemm_grouped(a, b, off.long()), lambda: pkg.gemm_grouped(a[:, :64], b, off),
                lambda: pkg.gemm_grouped(a.t(), b, off), lambda: pkg.gemm_grouped(a, b, off[:2]), lambda: pkg.gemm_grouped(a, b, off, a_scale=torch.ones(63, device="cuda")),
                lambda: pkg.gemm_grouped(a, b, off, out=torch.empty(64, 65, device="cuda")), lambda: pkg.gemm_grouped(a, b, off, out_dtype=torch.float64),
                lambda: pkg.quantize_rows(torch.zeros(4, 8, device="cuda", dtype=torch.float64)), lambda: pkg.quantize_rows(torch.zeros(8, device="cuda").expand(4, 8)),
                lambda: pkg.quantize_rows(torch.zeros(4, 8, device="cuda"), fmt=7), lambda: pkg.gemm_grouped_wgrad(a, a, off, 64), lambda: pkg.gemm_grouped_wgrad(a, a, off, 64, accumulate=True),
                lambda: pkg.gemv_w4(a.to(torch.bfloat16), b.view(torch.uint8)[0], torch.ones(64, 4, device="cuda"), 32),
                lambda: pkg.gemv_w4(a.to(torch.bfloat16), b.view(torch.uint8)[0, :, :64].contiguous(), torch.ones(64, 3, device="cuda"), 32)):
        with pytest.raises((pkg.Fp8GemmError, TypeError)):
            bad()


def test_a_step_without_tokens(pkg):
    """No token came: empty products, gradients of zeros, or nothing added."""
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    x, g = (torch.zeros((0, c), dtype=torch.bfloat16, device="cuda") for c in (64, 32))
    w = codes(generator("no tokens"), (3, 32, 64), 0)
    xc, xs = pkg.quantize_rows(x)
    assert pkg.gemm_grouped(xc, w, off, a_scale=xs, out_dtype=torch.bfloat16).shape == (0, 32)
    xt, xts = pkg.quantize_columns(x, off)
    gt, gts = pkg.quantize_columns(g, off)
    dw = pkg.gemm_grouped_wgrad(gt, xt, off, 0, a_scale=gts, b_scale=xts)
    assert dw.shape == (3, 32, 64) and not dw.any()
    held = torch.full((3, 32, 64), 2.0, device="cuda")
    pkg.gemm_grouped_wgrad(gt, xt, off, 0, out=held, accumulate=True)
    assert (held == 2.0).all()
    w4 = torch.zeros((3, 32, 32), dtype=torch.uint8, device="cuda")
    assert pkg.gemv_w4(x, w4, torch.ones((3, 32, 2), device="cuda"), 32, row_offsets=off).shape == (0, 32)


def test_results_on_a_named_stream_are_its_memory(pkg):
    """Work still queued on the current stream does not reach memory that another stream's call was given."""
    gen = generator("named")
    x = torch.randn((4096, 4096), generator=gen, device="cuda").to(torch.bfloat16)
    want, want_s = pkg.quantize_rows(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        late = torch.empty((4096, 4096), dtype=torch.uint8, device="cuda")
        for _ in range(8):
            late.fill_(0x55)
        del late                                                # (its writes may still be queued)
        got, got_s = pkg.quantize_rows(x, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8)) and torch.equal(got_s, want_s)


def test_sizes_that_an_int_cuts_off(pkg):
    """Rows, columns and lengths of 2^32 and more are refused, not taken for what is left of them in 32 bits."""
    wraps = (1 << 32) + 256
    one = offsets_of([1])
    flat = torch.empty((1, wraps), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(pkg.Fp8GemmError):
        pkg.quantize_rows(flat)
    with pytest.raises(pkg.Fp8GemmError):
        pkg.quantize_columns(flat, one)
    with pytest.raises(pkg.Fp8GemmError):
        pkg.quantize_rows(flat.view(wraps, 1))
    eight = flat.view(torch.float8_e4m3fn)[:, :wraps]
    few = torch.zeros((1, 256), dtype=torch.float8_e4m3fn, device="cuda")
    for a, b in ((eight, eight), (few[:, :1].contiguous(), eight.view(wraps, 1))):
        with pytest.raises(pkg.Fp8GemmError):
            pkg.gemm_grouped(a, b[None], one)
        with pytest.raises(pkg.Fp8GemmError):
            pkg.gemm(a, b)
        with pytest.raises(pkg.Fp8GemmError):
            pkg.gemm_ex(a, b)
    with pytest.raises(pkg.Fp8GemmError):
        pkg.gemm_grouped_wgrad(few, few, one, wraps)
    with pytest.raises(pkg.Fp8GemmError):
        pkg.gemm_grouped_wgrad(eight, eight, one, 1)
    w = flat.view(torch.uint8)[:, :wraps // 2]
    with pytest.raises(pkg.Fp8GemmError):
        pkg.gemv_w4(flat, w, torch.empty((1, wraps // 256), device="cuda"), 256)


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("rows,experts,cols", [(300, 4, 96), (300, 70, 40), (5000, 2, 64)])
def test_offsets_that_are_no_cut(pkg, rows, experts, cols, seed):
    """Offsets below zero, beyond the rows and out of order, some experts in front of the first row of the others: every
    operator goes by the same cut, each offset clamped to the rows and raised to the largest before it."""
    gen = generator("no cut", rows, experts, seed)
    bad = torch.randint(-rows // 3, rows + rows // 3, (experts + 1,), generator=gen, device="cuda")
    if seed % 2:
        bad = torch.sort(bad).values + torch.randint(-9, 10, (experts + 1,), generator=gen, device="cuda")
    meant = torch.cummax(bad.clamp(0, rows), 0).values.to(torch.int32)
    bad = bad.to(torch.int32)
    x = torch.randn((rows, cols), generator=gen, device="cuda").to(torch.bfloat16)
    dy = torch.randn((rows, 136), generator=gen, device="cuda").to(torch.float16)
    got = [pkg.quantize_columns(t, bad, fmt) for t, fmt in ((x, pkg.E4M3), (dy, pkg.E5M2))]
    want = [pkg.quantize_columns(t, meant, fmt) for t, fmt in ((x, pkg.E4M3), (dy, pkg.E5M2))]
    for (c, s), (c2, s2) in zip(got, want):
        assert torch.equal(c.view(torch.uint8), c2.view(torch.uint8)) and torch.equal(s, s2)
    off = meant.tolist()
    at, counts, used = places(off, rows)
    (xc, xs), (yc, ys) = got
    assert not xc.view(torch.uint8)[:, used:].any()
    dw = pkg.gemm_grouped_wgrad(yc, xc, bad, rows, a_scale=ys, b_scale=xs)
    for g, (p, c) in enumerate(zip(at, counts)):
        y, tol = fp8_product(yc[:, p:p + c].double(), xc[:, p:p + c].double()) if c else (torch.zeros_like(dw[g], dtype=torch.float64),) * 2
        f = ys[g][:, None].double() * xs[g].double()
        assert ((dw[g].double() - y * f).abs() <= tol * f + rounding(y * f, torch.float32) * 1.0001).all()
    # 4-bit matrices, with the kernel for few rows an expert and the one for many
    n, k, run = 48, 64, 32
    w = torch.randint(0, 256, (experts, n, k // 2), generator=gen, dtype=torch.uint8, device="cuda")
    s = torch.ones((experts, n, k // run), device="cuda")
    h = torch.randint(-3, 4, (rows, k), generator=gen, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    y = torch.full((rows, n), 9.0, device="cuda")
    pkg.gemv_w4(h, w, s, run, row_offsets=bad, out=y)
    for g in range(experts):
        lo, hi = off[g], off[g + 1]
        assert hi == lo or torch.equal(y[lo:hi].double(), h[lo:hi].double() @ w4_values(w[g], s[g], run, 0).t().contiguous())
    assert (y[:off[0]] == 9.0).all() and (y[off[-1]:] == 9.0).all()
