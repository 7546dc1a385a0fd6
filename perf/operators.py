"""Operators of a mixture-of-experts layer in 8- and 4-bit formats: what is measured, and their plain forms.

Tokens are sorted by expert: expert g owns rows row_offsets[g] .. row_offsets[g + 1] of a matrix of rows.

  quantize_rows      rows (optionally gathered by index) to 8-bit codes, one power-of-two scale a row
  quantize_columns   the same matrix transposed, one scale per expert and column: the operand of the weight gradient
  grouped            out[row] = a_scale[row] * b_scale[expert] * (codes of the row) . (codes of its expert's matrix)^T
  wgrad              out[expert] = (rows of the gradient)^T (rows of the input), a sum over the expert's rows
  w4                 y[row] = W[expert] x[row], W in 4 bits with one scale per run of its row

The scale s of a run of numbers is the smallest power of two with  max |x| <= s * (largest finite code), over its
finite numbers; 1 where they are all zero.  A code is the nearest one to x / s, ties to even.
"""
import importlib
import math

import numpy as np
import torch

own = False

F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
WIDE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TOP = {"e4m3": 448.0, "e5m2": 57344.0}          # both are 0.875 times a power of two
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
PAD = 128                                       # an expert's rows fill whole runs of this many columns when transposed


def _pkg():
    return importlib.import_module("tensor-core-fp8_amd")


# ---------------------------------------------------------------- cases
def listed():
    return [
        # activations of eight tokens on their way into an 8-bit layer: only the latency of a call counts
        {"name": "rows-decode", "op": "quantize_rows", "rows": 8, "cols": 4096, "tokens": 0, "x": "bf16", "fmt": "e4m3"},
        # a prefill's tokens gathered for the two experts each has
        {"name": "rows-gather", "op": "quantize_rows", "rows": 32768, "cols": 4096, "tokens": 16384, "x": "bf16", "fmt": "e4m3"},
        # a small layer's output gradient, transposed for the weight gradient
        {"name": "columns-small", "op": "quantize_columns", "rows": 4099, "cols": 2048, "experts": 8, "x": "bf16", "fmt": "e5m2"},
        # a large layer's input, transposed for the weight gradient
        {"name": "columns-large", "op": "quantize_columns", "rows": 32768, "cols": 4096, "experts": 32, "x": "bf16", "fmt": "e4m3"},
        # serving, eight tokens with two experts each: bound by reading the chosen experts' weights
        {"name": "grouped-decode", "op": "grouped", "rows": 16, "experts": 32, "k": 4096, "n": 2048, "a": "e4m3", "b": "e4m3", "out": "bf16", "skew": 0.5},
        # serving, a mixed batch: a hundred rows an expert, ragged
        {"name": "grouped-batch", "op": "grouped", "rows": 3001, "experts": 32, "k": 2048, "n": 4096, "a": "e4m3", "b": "e4m3", "out": "bf16", "skew": 1.0},
        # training, forward
        {"name": "grouped-train", "op": "grouped", "rows": 32768, "experts": 16, "k": 4096, "n": 8192, "a": "e4m3", "b": "e4m3", "out": "bf16", "skew": 0.5},
        # training, the input's gradient: the same product with the gradient's format and the transposed weights
        {"name": "grouped-backward", "op": "grouped", "rows": 8192, "experts": 8, "k": 8192, "n": 4096, "a": "e5m2", "b": "e4m3", "out": "bf16", "skew": 0.5},
        # the weights' gradient of a small layer with short, odd runs of rows
        {"name": "wgrad-small", "op": "wgrad", "rows": 2051, "experts": 16, "m": 2048, "n": 1024, "a": "e5m2", "b": "e4m3", "out": "bf16", "skew": 1.0},
        # ... and of a large one
        {"name": "wgrad-large", "op": "wgrad", "rows": 32768, "experts": 16, "m": 8192, "n": 4096, "a": "e5m2", "b": "e4m3", "out": "bf16", "skew": 0.5},
        # one token through a large dense layer in 4-bit integers
        {"name": "w4-token", "op": "w4", "rows": 1, "experts": 1, "k": 8192, "n": 28672, "w": "int4", "zeros": True, "run": 128, "scale": "f16", "x": "bf16", "out": "bf16", "skew": 0.0},
        # twelve tokens with two experts each through 4-bit floating-point weights
        {"name": "w4-experts", "op": "w4", "rows": 24, "experts": 32, "k": 4096, "n": 4096, "w": "e2m1", "zeros": False, "run": 32, "scale": "e8m0", "x": "bf16", "out": "bf16", "skew": 0.5},
    ]


def _log(rng, low, high, of=1):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / of)) * of))


def draw(rng):
    op = rng.choice(["quantize_rows", "quantize_columns", "grouped", "grouped", "wgrad", "w4", "w4"])
    f8 = lambda: rng.choice(["e4m3", "e5m2"])  # noqa: E731
    if op == "quantize_rows":
        rows = _log(rng, 1, 32768)
        return {"op": op, "rows": rows, "cols": _log(rng, 200, 4096, rng.choice([1, 16, 128])), "tokens": rng.choice([0, 1 + rows // 2]), "x": rng.choice(list(WIDE)), "fmt": f8()}
    if op == "quantize_columns":
        return {"op": op, "rows": _log(rng, 100, 16384), "cols": _log(rng, 200, 4096, rng.choice([1, 16, 128])), "experts": rng.choice([1, 3, 8, 32]), "x": rng.choice(list(WIDE)), "fmt": f8()}
    if op == "grouped":
        return {"op": op, "rows": _log(rng, 1, 16384), "experts": rng.choice([1, 5, 8, 16, 64]), "k": _log(rng, 256, 4096, rng.choice([16, 128])), "n": _log(rng, 200, 8192, rng.choice([1, 16, 128])),
                "a": f8(), "b": "e4m3", "out": rng.choice(["bf16", "f16"]), "skew": rng.choice([0.0, 0.5, 1.5])}
    if op == "wgrad":
        return {"op": op, "rows": _log(rng, 100, 16384), "experts": rng.choice([1, 5, 8, 16]), "m": _log(rng, 256, 4096, rng.choice([1, 128])), "n": _log(rng, 256, 4096, rng.choice([4, 128])),
                "a": f8(), "b": "e4m3", "out": rng.choice(["bf16", "f16"]), "skew": rng.choice([0.0, 0.5, 1.5])}
    w = rng.choice(["int4", "e2m1"])
    run = rng.choice([32, 64, 128])
    experts = rng.choice([1, 1, 8, 32])
    return {"op": op, "rows": _log(rng, 1, 64), "experts": experts, "k": _log(rng, 512, 8192, 128), "n": _log(rng, 200, 28672 if experts == 1 else 4096, rng.choice([1, 16, 128])), "w": w,
            "zeros": w == "int4" and rng.random() < 0.5, "run": run, "scale": rng.choice(["f16", "bf16", "f32"] if w == "int4" else ["e8m0", "f16"]), "x": rng.choice(["bf16", "f16", "e4m3"]),
            "out": rng.choice(["bf16", "f16", "f32"]), "skew": rng.choice([0.0, 1.0])}


# ---------------------------------------------------------------- inputs
def _offsets(case, rng):
    """How many rows each expert has: shares that differ by `skew` (standard deviation of their logarithm), every row drawn on its own."""
    e = case["experts"]
    share = np.exp(rng.standard_normal(e) * case.get("skew", 0.5))
    count = rng.multinomial(case["rows"], share / share.sum())
    return np.concatenate([[0], np.cumsum(count)]).astype(np.int32)


def padded_columns(rows, experts):
    """Columns of a transposed operand: enough for every expert's rows in whole runs of PAD."""
    return (rows + (PAD - 1) * experts) // PAD * PAD


def _places(offsets):
    """The column of each row in a transposed operand (numpy int64)."""
    count = np.diff(offsets).astype(np.int64)
    start = np.concatenate([[0], np.cumsum((count + PAD - 1) // PAD * PAD)[:-1]])
    return np.concatenate([np.arange(c) + s for c, s in zip(count, start)]) if count.sum() else np.zeros(0, np.int64)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = {"device": "cuda"}
    normal = lambda *s: torch.randn(*s, generator=gen, **dev)  # noqa: E731
    power = lambda *s: torch.exp2(torch.randint(-6, -2, s, generator=gen, **dev).float())  # noqa: E731
    state = {"case": case}
    op = case["op"]
    if op in ("quantize_rows", "quantize_columns"):
        many = case.get("tokens") or case["rows"]
        # tokens of different size, and a few channels that stand out, as activations have them
        x = normal(many, case["cols"]) * torch.exp2(2 * normal(many, 1)) * torch.exp2(torch.clamp(3 * normal(1, case["cols"]), -4, 6))
        state["x"] = x.to(WIDE[case["x"]])
        if case.get("tokens"):
            state["index"] = torch.randint(0, case["tokens"], (case["rows"],), generator=gen, dtype=torch.int32, **dev)
    if op != "quantize_rows":
        off = _offsets(case, rng)
        state["offsets"] = torch.from_numpy(off).cuda()
        state["most"] = int(np.diff(off).max())
    if op == "grouped":
        state["a"] = normal(case["rows"], case["k"]).mul_(16).to(F8[case["a"]])
        state["b"] = normal(case["experts"], case["n"], case["k"]).mul_(16).to(F8[case["b"]])
        state["a_scale"], state["b_scale"] = power(case["rows"]), power(case["experts"], case["n"])
    if op == "wgrad":
        at, ld = torch.from_numpy(_places(off)).cuda(), padded_columns(case["rows"], case["experts"])
        for key, side in (("a", "m"), ("b", "n")):
            t = torch.zeros(case[side], ld, **dev)
            t[:, at] = normal(case[side], case["rows"]).mul_(16)
            state[key] = t.to(F8[case[key]])
            state[key + "_scale"] = power(case["experts"], case[side])
    if op == "w4":
        e, n, k = case["experts"], case["n"], case["k"]
        state["w"] = torch.randint(0, 256, (e, n, k // 2), generator=gen, dtype=torch.uint8, **dev)
        runs = (e, n, k // case["run"])
        if case["scale"] == "e8m0":
            state["w_scale"] = torch.randint(117, 124, runs, generator=gen, dtype=torch.uint8, **dev)
        else:
            state["w_scale"] = (0.002 * (1 + torch.rand(runs, generator=gen, **dev))).to(WIDE[case["scale"]])
        if case["zeros"]:
            state["w_zero"] = torch.randint(6, 11, runs, generator=gen, dtype=torch.uint8, **dev)
        x = normal(case["rows"], k)
        state["x"] = x.mul_(16).to(F8[case["x"]]) if case["x"] in F8 else x.to(WIDE[case["x"]])
        if case["x"] in F8:
            state["x_scale"] = power(case["rows"])
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    return {"quantize_rows": _plain_rows, "quantize_columns": _plain_columns, "grouped": _plain_grouped, "wgrad": _plain_wgrad, "w4": _plain_w4}[case["op"]](case, state)


def _own(case, s):
    pkg, op = _pkg(), case["op"]
    if op == "quantize_rows":
        return pkg.quantize_rows(s["x"], pkg.E4M3 if case["fmt"] == "e4m3" else pkg.E5M2, row_index=s.get("index"))
    if op == "quantize_columns":
        return pkg.quantize_columns(s["x"], s["offsets"], pkg.E4M3 if case["fmt"] == "e4m3" else pkg.E5M2)
    if op == "grouped":
        return pkg.gemm_grouped(s["a"], s["b"], s["offsets"], a_scale=s["a_scale"], b_scale=s["b_scale"], out_dtype=WIDE[case["out"]])
    if op == "wgrad":
        return pkg.gemm_grouped_wgrad(s["a"], s["b"], s["offsets"], case["rows"], a_scale=s["a_scale"], b_scale=s["b_scale"], out_dtype=WIDE[case["out"]])
    one = case["experts"] == 1
    drop = lambda t: t[0] if one and t is not None else t  # noqa: E731
    return pkg.gemv_w4(s["x"], drop(s["w"]), drop(s["w_scale"]), case["run"], w_fmt=pkg.W4_INT if case["w"] == "int4" else pkg.W4_E2M1, zeros=drop(s.get("w_zero")), x_scale=s.get("x_scale"),
                       row_offsets=None if one else s["offsets"], out_dtype=WIDE[case["out"]])


def _power_of_two(largest, fmt):
    m, e = torch.frexp(largest)                       # largest = m 2^e, m in [0.5, 1)
    s = torch.ldexp(torch.ones_like(largest), e - int(math.log2(TOP[fmt] / 0.875)) + (m > 0.875).to(e.dtype))
    return torch.where(largest == 0, torch.ones_like(s), s)


def _plain_rows(case, s):
    x = s["x"].float()
    if "index" in s:
        x = x[s["index"].long()]
    scale = _power_of_two(x.abs().amax(1), case["fmt"])
    return (x / scale[:, None]).to(F8[case["fmt"]]), scale


def _groups(s, rows):
    """The expert of each row, and the row's number inside it."""
    row = torch.arange(rows, device="cuda")
    group = torch.searchsorted(s["offsets"][1:].long(), row, right=True)
    return group, row - s["offsets"].long()[group]


def _plain_columns(case, s):
    x, rows, e = s["x"].float(), case["rows"], case["experts"]
    group, inside = _groups(s, rows)
    largest = torch.zeros(e, case["cols"], device="cuda").scatter_reduce_(0, group[:, None].expand_as(x), x.abs(), "amax")
    scale = _power_of_two(largest, case["fmt"])
    count = torch.diff(s["offsets"].long())
    filled = (count + PAD - 1) // PAD * PAD
    out = torch.zeros(padded_columns(rows, e), case["cols"], device="cuda")
    out[(torch.cumsum(filled, 0) - filled)[group] + inside] = x / scale[group]
    return out.t().contiguous().to(F8[case["fmt"]]), scale


def _spread(s, x, experts):
    """Rows sorted by expert -> (experts, most rows of any, columns), zeros behind an expert's last row."""
    group, inside = _groups(s, x.shape[0])
    out = torch.zeros(experts, max(1, s["most"]), x.shape[1], device="cuda")
    out[group, inside] = x
    return out, group, inside


def _plain_grouped(case, s):
    a, group, inside = _spread(s, s["a"].float(), case["experts"])
    y = torch.bmm(a, s["b"].float().transpose(1, 2).contiguous())[group, inside]
    return (y * s["a_scale"][:, None] * s["b_scale"][group]).to(WIDE[case["out"]])


def _plain_wgrad(case, s):
    rows, e = case["rows"], case["experts"]
    group, inside = _groups(s, rows)
    filled = (torch.diff(s["offsets"].long()) + PAD - 1) // PAD * PAD
    at = (torch.cumsum(filled, 0) - filled)[group] + inside
    a, _, _ = _spread(s, s["a"].float()[:, at].t(), e)
    b, _, _ = _spread(s, s["b"].float()[:, at].t(), e)
    y = torch.bmm(a.transpose(1, 2).contiguous(), b)
    return (y * s["a_scale"][:, :, None] * s["b_scale"][:, None, :]).to(WIDE[case["out"]])


def _plain_w4(case, s):
    q = torch.stack((s["w"] & 15, s["w"] >> 4), -1).flatten(-2)
    if case["w"] == "e2m1":
        v = torch.tensor(E2M1 + tuple(-t for t in E2M1), device="cuda")[q.long()]
    else:
        zero = s["w_zero"].float() if "w_zero" in s else torch.full(s["w_scale"].shape, 8.0, device="cuda")
        v = q.float() - zero.repeat_interleave(case["run"], -1)
    scale = torch.exp2(s["w_scale"].float() - 127) if case["scale"] == "e8m0" else s["w_scale"].float()
    v = v * scale.repeat_interleave(case["run"], -1)
    x, group, inside = _spread(s, s["x"].float(), case["experts"])
    y = torch.bmm(x, v.transpose(1, 2).contiguous())[group, inside]
    return (y * s["x_scale"][:, None] if "x_scale" in s else y).to(WIDE[case["out"]])


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    op, wide = case["op"], {"f32": 4, "bf16": 2, "f16": 2}
    if op == "quantize_rows":
        many = case["tokens"] or case["rows"]
        return {"bytes": min(many, case["rows"]) * case["cols"] * wide[case["x"]] + case["rows"] * (case["cols"] + 4) + (4 * case["rows"] if case["tokens"] else 0), "flops": 3 * case["rows"] * case["cols"]}
    if op == "quantize_columns":
        e = case["experts"]
        return {"bytes": case["rows"] * case["cols"] * wide[case["x"]] + case["cols"] * (padded_columns(case["rows"], e) + 4 * e) + 4 * e, "flops": 3 * case["rows"] * case["cols"]}
    busy = min(case["rows"], case["experts"])         # experts with rows, at most
    if op == "grouped":
        r, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": r * k + busy * n * (k + 4) + 4 * r + r * n * wide[case["out"]], "flops": 2 * r * k * n}
    if op == "wgrad":
        r, m, n = case["rows"], case["m"], case["n"]
        return {"bytes": r * (m + n) + case["experts"] * (4 * (m + n) + m * n * wide[case["out"]]), "flops": 2 * r * m * n}
    r, k, n = case["rows"], case["k"], case["n"]
    runs = n * (k // case["run"])
    each = n * k // 2 + runs * ({"e8m0": 1, "f32": 4}.get(case["scale"], 2) + (1 if case["zeros"] else 0))
    return {"bytes": busy * each + r * k * (1 if case["x"] in F8 else 2) + r * n * wide[case["out"]], "flops": 2 * r * k * n}


# ---------------------------------------------------------------- from the definitions, in 64 bits
def _nearest(x, fmt):
    """x (float64) to the nearest number of an 8-bit format, ties to even: numpy."""
    bits, low = (3, -6) if fmt == "e4m3" else (2, -14)
    _, e = np.frexp(x)
    step = np.ldexp(1.0, np.maximum(e - 1, low) - bits)
    return np.clip(np.rint(x / step) * step, -TOP[fmt], TOP[fmt])


def _scale64(largest, fmt):
    with np.errstate(divide="ignore"):
        return np.where(largest == 0, 1.0, np.exp2(np.ceil(np.log2(largest / TOP[fmt]))))


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    off = s["offsets"].cpu().numpy() if "offsets" in s else None
    if op in ("quantize_rows", "quantize_columns"):
        x = s["x"].double().cpu().numpy()
        if op == "quantize_rows":
            x = x[s["index"].cpu().numpy()] if "index" in s else x
            scale = _scale64(np.abs(x).max(1), case["fmt"])
            return _nearest(x / scale[:, None], case["fmt"]), scale
        out, scales, at = np.zeros((case["cols"], padded_columns(case["rows"], case["experts"]))), np.ones((case["experts"], case["cols"])), 0
        for g in range(case["experts"]):
            part = x[off[g]:off[g + 1]]
            if len(part):
                scales[g] = _scale64(np.abs(part).max(0), case["fmt"])
                out[:, at:at + len(part)] = _nearest(part / scales[g], case["fmt"]).T
            at += -(-len(part) // PAD) * PAD
        return out, scales
    if op == "grouped":
        out = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device="cuda")
        for g in range(case["experts"]):
            lo, hi = int(off[g]), int(off[g + 1])
            if hi > lo:
                out[lo:hi] = (s["a"][lo:hi].double() * s["a_scale"][lo:hi, None].double()) @ (s["b"][g].double() * s["b_scale"][g][:, None].double()).t().contiguous()
        return out
    if op == "wgrad":
        out, at = torch.zeros(case["experts"], case["m"], case["n"], dtype=torch.float64, device="cuda"), 0
        for g in range(case["experts"]):
            count = int(off[g + 1] - off[g])
            if count:
                a, b = s["a"][:, at:at + count].double(), s["b"][:, at:at + count].double()
                out[g] = (a @ b.t().contiguous()) * s["a_scale"][g][:, None].double() * s["b_scale"][g].double()
            at += -(-count // PAD) * PAD
        return out
    out, run_ = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device="cuda"), case["run"]
    for g in range(case["experts"]):
        lo, hi = int(off[g]), int(off[g + 1])
        if hi == lo:
            continue
        byte = s["w"][g]
        q = torch.empty(case["n"], case["k"], dtype=torch.float64, device="cuda")
        q[:, 0::2], q[:, 1::2] = (byte % 16).double(), torch.div(byte, 16, rounding_mode="floor").double()
        if case["w"] == "e2m1":                       # sign, two bits of exponent, one of mantissa
            sign, e, m = torch.where(q >= 8, -1.0, 1.0), torch.floor(q % 8 / 2), q % 2
            q = sign * torch.where(e == 0, m / 2, torch.exp2(e - 1) * (1 + m / 2))
        q = q.view(case["n"], -1, run_)
        if case["w"] == "int4":
            q = q - (s["w_zero"][g].double()[:, :, None] if case["zeros"] else 8.0)
        w_scale = torch.exp2(s["w_scale"][g].double() - 127) if case["scale"] == "e8m0" else s["w_scale"][g].double()
        w = (q * w_scale[:, :, None]).view(case["n"], case["k"])
        x = s["x"][lo:hi].double() * (s["x_scale"][lo:hi, None].double() if "x_scale" in s else 1.0)
        out[lo:hi] = x @ w.t().contiguous()
    return out
