"""Cases and expectations shared by the CPU and GPU tests of the layer operators (the fused linear
product, rotary positions, the queries' and keys' norm with rotation): float64 definitions and
the error that f32 arithmetic and one final rounding allow, element by element."""

import numpy as np

HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}      # a rounding is off by at most this
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -133, "f32": 2.0 ** -149}        # half the smallest subnormal


def _act(z, name):
    """(value, |derivative| bound, relative evaluation error) of an activation, in float64."""
    if name is None:
        return z, 1.0, 0.0
    if name == "relu":
        return np.maximum(z, 0.0), 1.0, 0.0
    # sigmoid = 1 / (1 + 2^t), t = -x log2 e rounded (|x| below 2^7 where the value is not 0: 2^-24 * 2^7 * 1.45
    # in the exponent), ex2.approx 2^-22, the sum 2^-24, rcp.approx 2^-23, the product 2^-24: below 2^-15.
    # gelu's argument adds four roundings of its own relative to u: 2^-22 * 2^7
    if name == "silu":
        return z / (1 + np.exp(-z)), 1.1, 2.0 ** -15
    u = np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)
    return z / (1 + np.exp(-2 * u)), 1.13, 2.0 ** -14


def linear_expected(x, w, bias, res, N, act, gated, out_dtype):
    """(want, allowed error) in float64.  Each 16-deep step of the tensor cores adds its products to the
    f32 sum with an error of at most 2^-22 of the terms' absolute sum so far: (K / 16 + 4) steps with
    the bias and the joins of a cut sum.  That error passes the activation (its derivative's bound),
    the gate's product and the residual, and the result is rounded once."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    K = x.shape[1]
    with np.errstate(all="ignore"):
        z, mag = x @ w.T, np.abs(x) @ np.abs(w).T
        if bias is not None:
            z, mag = z + bias.astype(np.float64), mag + np.abs(bias.astype(np.float64))
        err = (K / 16 + 8) * 2.0 ** -22 * mag
        y, d, r = _act(z[:, :N], act)
        e = d * err[:, :N] + r * np.abs(y)
        if gated:
            u, eu = z[:, N:], err[:, N:]
            y, e = y * u, e * np.abs(u) + eu * np.abs(y) + e * eu
        e = e + 2.0 ** -24 * np.abs(y)
        if res is not None:
            y = y + res.astype(np.float64)
            e = e + 2.0 ** -24 * np.abs(y)
        return y, e + HALF_STEP[out_dtype] * (np.abs(y) + e) + TINY[out_dtype]


def heads_expected(x, spec, table, before):
    """{output: (want, allowed error)} in float64 of a heads kernel on numpy inputs ``x`` (f32 values);
    ``spec``: heads, kv, D, R, dtype, interleaved, values, heads_first, inverse, norm.  ``before``:
    the outputs' contents, which rows of a position outside the table keep.

    The norm: the squares' sum is off by at most (D / 32 + 8) roundings of its own size (each lane's
    share, then the warp's), the division, root, reciprocal and two products by 2^-23 each with the
    root halving what comes before it: (D / 64 + 12) 2^-24 of |n|.  The rotation adds two products
    and a sum: 3 * 2^-24 of |a cos| + |b sin|.  Then one rounding to the type."""
    h, kv, D, R = spec["heads"], spec["kv"], spec["D"], spec["R"]
    pos = x["pos"]
    live = (pos >= 0) & (pos < table)
    p = np.clip(pos, 0, table - 1)
    cos, sin = (x[t].astype(np.float64)[p][:, :, None] for t in ("cos", "sin"))
    if spec["inverse"]:
        sin = -sin
    i0, i1 = (np.arange(0, R, 2), np.arange(1, R, 2)) if spec["interleaved"] else (np.arange(R // 2),
                                                                                    np.arange(R // 2, R))
    out = {}
    for name, lo, hi in (("q", 0, h), ("k", h, h + kv), ("v", h + kv, h + 2 * kv)):
        if lo == hi or (name == "v" and not spec["values"]):
            continue
        y = x["qkv"][:, :, lo:hi].astype(np.float64)
        e = np.zeros_like(y)
        if name != "v":
            with np.errstate(all="ignore"):
                if spec["norm"]:
                    y = y / np.sqrt((y * y).mean(-1, keepdims=True) + spec.get("eps", 1e-6)) \
                        * x["w" + name].astype(np.float64)
                    e = (D / 64 + 12) * 2.0 ** -24 * np.abs(y)
                a, b, ea, eb = y[..., i0], y[..., i1], e[..., i0], e[..., i1]
                y, e = y.copy(), e.copy()
                y[..., i0], y[..., i1] = a * cos - b * sin, b * cos + a * sin
                mag = 3 * 2.0 ** -24
                e[..., i0] = ea * abs(cos) + eb * abs(sin) + mag * (abs(a * cos) + abs(b * sin))
                e[..., i1] = eb * abs(cos) + ea * abs(sin) + mag * (abs(b * cos) + abs(a * sin))
                e = e + HALF_STEP[spec["dtype"]] * (np.abs(y) + e) + TINY[spec["dtype"]]
        keep = np.broadcast_to(live[:, :, None, None], y.shape)
        if spec["heads_first"]:
            y, e, keep = (np.ascontiguousarray(t.transpose(0, 2, 1, 3)) for t in (y, e, keep))
        out[name] = np.where(keep, y, before[name]), np.where(keep, e, 0.0)
    return out


def check(got, want, allowed, what):
    """Every element within its allowed error; NaN exactly where it is expected."""
    got = np.asarray(got, dtype=np.float64).reshape(want.shape)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), f"{what}: NaN in other places"
    with np.errstate(invalid="ignore"):
        bad = ~nan & ~(np.abs(got - want) <= allowed) & ~(np.isinf(want) & (got == want))
    if bad.any():
        i = tuple(int(v) for v in np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} elements off, first {i}: "
                             f"{got[i]!r} against {want[i]!r}, allowed {allowed[i]:.3e}")


# (M, N, K, dtype, out_dtype, bias, activation, residual, gated)
LINEAR = [
    (1, 64, 64, "f16", "f16", False, None, False, False),
    (1, 8, 8, "bf16", "bf16", True, None, True, False),
    (1, 4096, 1024, "bf16", "bf16", False, None, True, False),
    (3, 136, 200, "f16", "f32", True, "relu", False, False),
    (16, 1000, 520, "bf16", "bf16", False, "silu", False, True),
    (17, 128, 1032, "f16", "f16", True, "gelu_tanh", True, False),
    (40, 256, 64, "bf16", "f32", False, None, True, True),
    (64, 192, 320, "f16", "f16", True, "silu", True, True),
    (100, 1416, 72, "bf16", "bf16", True, None, False, False),
    (127, 72, 4104, "f16", "f16", False, None, False, False),
    (128, 264, 128, "bf16", "bf16", False, "gelu_tanh", True, True),
    (129, 120, 256, "f16", "f16", False, "relu", True, False),
    (255, 1000, 136, "bf16", "bf16", True, "gelu_tanh", False, False),
    (333, 520, 264, "f16", "f16", True, None, True, False),
    (512, 1536, 512, "bf16", "bf16", False, "silu", False, True),
    (1000, 2056, 520, "f16", "f16", True, "gelu_tanh", True, False),
    (1793, 1928, 328, "bf16", "bf16", True, "silu", True, True),
    (2048, 2048, 1024, "f16", "f32", False, None, True, False),
    (2049, 1000, 64, "bf16", "bf16", True, "relu", True, False),
    (2560, 2560, 1024, "bf16", "bf16", True, None, False, False),
    (1300, 264, 16384, "bf16", "bf16", True, None, True, False),       # bands of four and of two rows of tiles
]

# sizes whose last wave of tiles is cut: (whole strips of tiles or -1, tiles in halves, width of the units)
TAILS = [((1119, 5632, 136, "bf16", "bf16", False, "relu", True, False), (-1, 36, 128)),
         ((1119, 5592, 264, "bf16", "bf16", True, None, True, False), (-1, 36, 128)),
         ((1285, 4656, 264, "f16", "f16", True, "silu", True, False), (10, 0, 192)),
         ((1302, 4784, 136, "bf16", "f32", False, None, True, False), (12, 0, 192)),
         ((2338, 3592, 72, "f16", "f16", False, None, False, False), (7, 0, 128)),
         ((258, 4832, 200, "bf16", "bf16", True, "silu", True, True), (-1, 2, 128)),
         ((264, 4800, 200, "f16", "f16", False, "gelu_tanh", False, True), (37, 0, 128)),
         ((259, 4912, 136, "bf16", "f32", True, "silu", False, True), (0, 0, 192)),
         ((200, 1000, 136, "f16", "f16", False, "silu", True, True), (0, 0, 128)),
         ((1285, 4656, 16384, "bf16", "bf16", True, None, True, False), (10, 0, 192))]      # in bands of four rows

# (B, S, heads, kv, D, R, dtype, interleaved, values, heads_first, inverse, norm)
HEADS = [
    (1, 1, 1, 0, 2, 2, "f32", False, False, False, False, False),
    (1, 1, 32, 8, 128, 128, "bf16", False, True, False, False, False),
    (7, 1, 12, 4, 128, 128, "f16", False, False, True, False, True),
    (2, 5, 3, 1, 64, 64, "f32", True, True, True, True, False),
    (3, 33, 4, 2, 80, 40, "f16", False, True, True, False, True),
    (3, 33, 4, 2, 80, 40, "bf16", True, True, False, False, True),
    (1, 100, 5, 5, 96, 96, "f32", False, True, False, True, False),
    (2, 77, 16, 1, 256, 64, "bf16", True, False, True, False, True),
    (1, 129, 2, 2, 256, 256, "f32", False, True, True, False, True),
    (2, 9, 3, 3, 10, 6, "f16", False, True, True, False, True),
    (1, 50, 6, 0, 32, 16, "bf16", False, False, False, True, False),
    (1, 3, 2, 1, 512, 256, "f16", True, True, True, False, True),
    (1, 700, 32, 8, 128, 64, "f16", True, True, True, False, False),
    (2, 300, 8, 2, 64, 64, "bf16", False, True, True, False, True),
    (1, 4, 2, 2, 1000, 500, "f32", False, True, False, False, True),
]
HEADS_FIELDS = ("B", "S", "heads", "kv", "D", "R", "dtype", "interleaved", "values", "heads_first", "inverse", "norm")


def heads_spec(case):
    return dict(zip(HEADS_FIELDS, case))


def heads_package(synth, path, spec, table):
    build = synth.qk_norm_rope_package if spec["norm"] else synth.rope_package
    more = {} if spec["norm"] else {"inverse": spec["inverse"]}
    return build(path, spec["B"], spec["S"], spec["heads"], spec["kv"], spec["D"], rotary=spec["R"],
                 interleaved=spec["interleaved"], dtype=spec["dtype"], table=table, values=spec["values"],
                 heads_first=spec["heads_first"], **more)


def custom_epilogue_package(path, M, N, K):
    """linear[M, N] = row <= col ? max(scale[0] * z + shift[col], cap[row, col]) : -1, with f32 scale, shift and
    cap: an epilogue that no builder writes, of a constant load, a vector over columns, an array over
    elements and a selection by coordinates."""
    from thompiler import ir, schedules, synth
    L, V, B, assign = schedules.L, schedules.V, schedules.B, schedules.assign
    row = schedules.clamped(V("row"), M) if M % 64 else V("row")
    col = schedules.clamped(V("col"), N) if N % 64 else V("col")
    f32 = schedules.F32T
    epi = ir.Lambda(("z", "row", "col"), (
        ir.Load(("sc",), "scale", (L(0),), f32), ir.Load(("sh",), "shift", (col,), f32),
        ir.Load(("cp",), "cap", (row, col), f32), ir.Let("minus", L(-1.0, "float"), f32),
        assign("zs", "multiply", "z", "sc"), assign("zt", "add", "zs", "sh"), assign("zm", "maximum", "zt", "cp"),
        ir.Select("y", (ir.Branch(V("zm"), B("<=", V("row"), V("col"))), ir.Branch(V("minus"), None)))), ("y",))
    body = schedules.linear_body(M, N, K, "f16", False, epi)
    tiles = -(-M // 64) * -(-N // 64)
    inputs = {"x": ((M, K), "f16", None), "w": ((N, K), "f16", {"dist": "normal", "std": K ** -0.5}),
              "scale": ((1,), "f32", None), "shift": ((N,), "f32", None), "cap": ((M, N), "f32", None)}
    return synth._layer_write(path, "custom", "custom", "k_linear", body, inputs, {"linear": ((M, N), "f32", None)},
                              -(-tiles // 8) * 8, 128, 2e-2, 2e-3, smem=2 * 64 * 64 * 2,
                              aligned=dict.fromkeys((*inputs, "linear"), 16))


def custom_expected(x):
    z = x["x"].astype(np.float64) @ x["w"].astype(np.float64).T
    mag = np.abs(x["x"].astype(np.float64)) @ np.abs(x["w"].astype(np.float64)).T
    s = float(x["scale"].reshape(-1)[0])
    t = s * z + x["shift"].astype(np.float64)
    # the product's steps (as in linear_expected), then a product and a sum in f32
    err = abs(s) * (x["x"].shape[1] / 16 + 8) * 2.0 ** -22 * mag + 2.0 ** -23 * (np.abs(s * z) + np.abs(t))
    rows, cols = np.indices(t.shape)
    keep = rows <= cols
    return np.where(keep, np.maximum(t, x["cap"]), -1.0), np.where(keep, err + 2.0 ** -24 * np.abs(t), 0.0)
