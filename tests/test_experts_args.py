"""Refusals of the entry points for layers with experts: before anything touches the GPU."""
import ctypes

import pytest

INVALID = 1      # hipErrorInvalidValue
P = ctypes.c_void_p(0x1000)
ODD = ctypes.c_void_p(0x1001)


def call(fn, good, **change):
    args = dict(good)
    args.update(change)
    return fn(*args.values())


def refused(fn, good, changes):
    for change in changes:
        assert call(fn, good, **change) == INVALID, change


GROUPED = dict(groups=4, m=100, k=256, n=128, row_offsets=P, a=P, a_fmt=0, b=P, b_fmt=0, out=P, out_type=0, a_scale=None, b_scale=None, per_column=0, stream=None)
WGRAD = dict(groups=4, rows=100, m=64, n=64, row_offsets=P, a_t=P, a_fmt=0, b_t=P, b_fmt=0, ld=512, out=P, out_type=0, a_scale=None, b_scale=None, accumulate=0, stream=None)
QROWS = dict(rows=10, cols=64, x=P, x_type=1, x_stride=64, x_rows=10, row_index=None, fmt=0, codes=P, scales=P, stream=None)
QCOLS = dict(groups=4, rows=100, cols=64, row_offsets=P, x=P, x_type=1, x_stride=64, x_rows=100, row_index=None, fmt=0, codes_t=P, ld=512, scales=P, stream=None)
W4 = dict(m=1, k=256, n=64, x=P, x_type=1, x_scale=None, w=P, w_fmt=0, run=128, w_scales=P, scale_type=2, w_zeros=None, y=P, y_type=1, stream=None)


def test_grouped(pkg):
    changes = [dict(groups=0), dict(groups=1025), dict(groups=-1), dict(m=0), dict(k=0), dict(n=-3), dict(row_offsets=None), dict(a=None), dict(b=None), dict(out=None), dict(a_fmt=2), dict(b_fmt=-1),
               dict(out_type=3), dict(out_type=-1), dict(out=ODD), dict(out=ODD, out_type=1)]
    refused(pkg.lib().fp8gemm_grouped, GROUPED, changes)
    tuned = dict(GROUPED)
    del tuned["stream"]
    tuned.update(variant=18, stream=None)
    # shapes that a kernel cannot run, and numbers that name none
    refused(pkg.lib().fp8gemm_grouped_tuned, tuned, [dict(variant=1), dict(variant=5), dict(variant=99), dict(variant=13, k=128), dict(variant=14, k=272), dict(variant=18, k=100), dict(variant=15, a=ODD), dict(variant=13, k=(1 << 23) + 16)])


def test_wgrad(pkg):
    changes = [dict(groups=0), dict(groups=1025), dict(rows=0), dict(m=0), dict(n=0), dict(row_offsets=None), dict(a_t=None), dict(b_t=None), dict(out=None), dict(a_fmt=5), dict(b_fmt=5), dict(out_type=7),
               dict(ld=384), dict(ld=513), dict(ld=(1 << 23) + 128), dict(rows=1000), dict(a_t=ODD), dict(b_t=ODD), dict(out=ODD)]
    refused(pkg.lib().fp8gemm_grouped_wgrad, WGRAD, changes)
    tuned = dict(WGRAD)
    del tuned["stream"]
    tuned.update(variant=18, stream=None)
    refused(pkg.lib().fp8gemm_grouped_wgrad_tuned, tuned, [dict(variant=0), dict(variant=5), dict(variant=17)])


def test_quantize(pkg):
    common = [dict(rows=0), dict(cols=0), dict(x=None), dict(x_type=3), dict(x_type=-1), dict(x_stride=63), dict(x_rows=0), dict(fmt=2), dict(scales=None), dict(x=ODD), dict(x_rows=9)]
    refused(pkg.lib().fp8gemm_quantize_rows, QROWS, common + [dict(codes=None)])
    refused(pkg.lib().fp8gemm_quantize_columns, QCOLS, common + [dict(codes_t=None), dict(codes_t=ODD), dict(row_offsets=None), dict(groups=0), dict(groups=2000), dict(ld=256), dict(ld=500), dict(rows=1 << 24, x_rows=1 << 24)])


def test_sizes_beyond_the_grids(pkg):
    """More than 2^30 of anything, or more workgroups than a grid holds."""
    big = (1 << 30) + 1
    refused(pkg.lib().fp8gemm_grouped, GROUPED, [dict(m=big), dict(k=big), dict(n=big), dict(m=2 ** 31 - 1), dict(m=1 << 30, n=1 << 30)])
    refused(pkg.lib().fp8gemm_grouped, dict(GROUPED, a=ODD), [dict(m=1 << 21, n=1 << 21), dict(m=1 << 30, n=1 << 30)])
    refused(pkg.lib().fp8gemm_grouped_wgrad, WGRAD, [dict(m=big), dict(n=big), dict(m=2 ** 31 - 1), dict(m=1 << 30, n=1 << 30), dict(rows=2 ** 31 - 1)])
    refused(pkg.lib().fp8gemm_quantize_rows, QROWS, [dict(rows=big, x_rows=2 ** 31 - 1), dict(cols=big, x_stride=big)])
    refused(pkg.lib().fp8gemm_quantize_columns, dict(QCOLS, groups=1024, ld=131200), [dict(cols=1 << 24, x_stride=1 << 24), dict(cols=2 ** 31 - 1, x_stride=1 << 40)])
    refused(pkg.lib().fp8gemm_gemv_w4, W4, [dict(m=big), dict(n=big), dict(n=2 ** 31 - 1), dict(m=2 ** 31 - 1)])


def test_padded_length(pkg):
    """Whole runs of 128 for every expert, whatever the cut; 0 for what is no length."""
    ld = pkg.lib().fp8gemm_grouped_ld
    for rows, groups in ((1, 1), (128, 1), (129, 1), (100, 4), (1, 1024), (4096, 8), (5, 7)):
        worst = 128 * (min(groups, rows) - 1) + -(-(rows - min(groups, rows) + 1) // 128) * 128      # as many experts as possible with one row
        assert ld(rows, groups) % 128 == 0 and ld(rows, groups) >= worst
    assert ld(0, 1) == 0 and ld(1, 0) == 0 and ld(1, 1025) == 0 and ld(1 << 24, 1) == 0


def test_w4(pkg):
    changes = [dict(m=0), dict(k=0), dict(n=0), dict(run=0), dict(run=48), dict(run=96), dict(run=16), dict(x=None), dict(w=None), dict(w_scales=None), dict(y=None), dict(w_fmt=2), dict(w_fmt=1, w_zeros=P),
               dict(x_type=0), dict(x_type=5), dict(scale_type=3), dict(scale_type=6), dict(y_type=3), dict(x=ODD), dict(w=ODD), dict(y=ODD), dict(w_scales=ODD), dict(k=1 << 24)]
    refused(pkg.lib().fp8gemm_gemv_w4, W4, changes)
    grouped = dict(groups=4, m=1, k=256, n=64, row_offsets=P)
    grouped.update({key: W4[key] for key in list(W4)[3:]})
    refused(pkg.lib().fp8gemm_grouped_w4, grouped, changes + [dict(row_offsets=None), dict(groups=0), dict(groups=1025)])


def test_python_checks_need_no_gpu(pkg):
    """Tensors that are not on a GPU, or do not fit, are refused before a call is made."""
    import torch
    a, b = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(2, 16, 32, dtype=torch.uint8)
    off = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(pkg.Fp8GemmError):
        pkg.gemm_grouped(a, b, off, a_fmt=0, b_fmt=0)
    with pytest.raises(pkg.Fp8GemmError):
        pkg.gemm_grouped_wgrad(a, b[0], off, 8, a_fmt=0, b_fmt=0)
    with pytest.raises(pkg.Fp8GemmError):
        pkg.quantize_rows(torch.zeros(4, 64))
    with pytest.raises(pkg.Fp8GemmError):
        pkg.quantize_rows(torch.zeros(4, 64).t())
    with pytest.raises(pkg.Fp8GemmError):
        pkg.quantize_columns(torch.zeros(4, 64), off)
    with pytest.raises(pkg.Fp8GemmError):
        pkg.gemv_w4(torch.zeros(1, 64, dtype=torch.bfloat16), torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2), 32)


WRAPS = (1 << 32) + 256         # what is left of it in 32 bits is a size that every operator takes


def test_sizes_that_an_int_cuts_off(pkg):
    """A size beyond an int would reach the C entry points as its low 32 bits: refused before."""
    import torch
    for rows, groups in ((WRAPS, 1), (5, WRAPS), (1 << 31, 1), (-WRAPS, 1)):
        with pytest.raises(pkg.Fp8GemmError):
            pkg.grouped_ld(rows, groups)
    with pytest.raises(pkg.Fp8GemmError):
        pkg.plan(WRAPS, 256, 256)
    off = torch.empty(WRAPS + 1, dtype=torch.int32, device="meta")
    with pytest.raises(pkg.Fp8GemmError):
        pkg._offsets(off)
    pkg._setup()
    for shape, index in (((1, WRAPS), None), ((WRAPS, 1), None), ((4, 8), WRAPS), ((WRAPS, 1), 4)):
        x = torch.empty(shape, dtype=torch.bfloat16, device="meta")
        with pytest.raises(pkg.Fp8GemmError):
            pkg._wide_matrix(x, None if index is None else torch.empty(index, dtype=torch.int32, device="meta"))
    assert pkg._wide_matrix(torch.empty((1, 1 << 30), dtype=torch.bfloat16, device="meta"), None) == (1, 1, 1 << 30, pkg.OUT_BF16, 1 << 30)
    # what the entry points do before any device is looked at
    a = torch.empty((4, 64), dtype=torch.float8_e4m3fn, device="meta")
    with pytest.raises(pkg.Fp8GemmError):
        pkg.GEMM(4, 64, WRAPS, a, a, a)


def test_w4_layouts(pkg):
    """The calls that the GPU tests make to reach every layout still reach it (a host decision)."""
    from expert_util import W4_LAYOUTS
    kinds = set()
    for groups, m, k, n, x_type, w_fmt, run, scale, layout in W4_LAYOUTS:
        assert pkg.w4_plan(m, k, n, x_type, w_fmt, run, scale, groups) == layout
        rows, wk, cols, blocks, at_once, planned, ring = layout
        assert rows == 16 and wk * cols == 128 and ring in (2, 4) and planned <= 16
        kinds.add((wk, "pieces" if at_once == 0 else ("one" if blocks == 1 else ("all" if at_once >= blocks else ("several" if at_once > 1 else "each")))))
    assert kinds >= {(wk, kind) for wk in (1, 2, 4, 8) for kind in ("pieces", "one", "all", "each")}
    assert {(wk, "several") for wk in (1, 2, 4, 8)} <= kinds
    # more rows: 32 or 64 at a time, the scales of all of K or of a part
    assert pkg.w4_plan(17, 4096, 4096)[0] == 32 and pkg.w4_plan(33, 4096, 4096)[0] == 64 and pkg.w4_plan(64, 4096, 4096, groups=8)[0] == 32
    assert pkg.w4_plan(64, 28672, 129, run=32, scale_type=pkg.T_F32)[4] < 28672 <= pkg.w4_plan(64, 28672, 129, run=128)[4]
    for bad in (dict(m=0, k=256, n=64), dict(m=1, k=256, n=64, run=48), dict(m=1, k=256, n=64, groups=2000), dict(m=1, k=256, n=64, x_type=0)):
        with pytest.raises(pkg.Fp8GemmError):
            pkg.w4_plan(**bad)


def test_scales_lie_by_expert(pkg):
    """A matrix of scales with its axes exchanged holds as many numbers: refused, not read as if it were the other one."""
    import torch
    pkg._setup()
    good = torch.ones((4, 6))
    assert pkg._floats(good, 24, "b_scale", 4) == good.data_ptr()
    assert pkg._floats(good.view(24), 24, "b_scale", 4) == good.data_ptr()
    assert pkg._floats(torch.ones((24, 1)), 24, "a_scale") and pkg._floats(None, 24, "a_scale", 4) is None
    for bad in (torch.ones((6, 4)), torch.ones((1, 24)), torch.ones((4, 5)), good.t(), good.double()):
        with pytest.raises(pkg.Fp8GemmError):
            pkg._floats(bad, 24, "b_scale", 4)


def test_results_without_a_kernel_go_by_their_stream_too(pkg):
    """A stream of another device is refused where an empty batch needs no launch, as it is where there is one."""
    import torch

    class Stream:
        device = torch.device("cuda", 5)

    pkg._setup()
    t = torch.ones(3)
    with pytest.raises(pkg.Fp8GemmError):
        pkg._fill(t, 0.0, Stream())
    assert (t == 1).all()
    pkg._fill(t, 2.0, None)
    assert (t == 2).all()
