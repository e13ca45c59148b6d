"""Statement trees of the layer operators: the fused linear product and the rotary heads.

``synth`` writes packages with these bodies, and the tuned families recognise a kernel by
rebuilding the body for the sizes, names and epilogue they read off it and comparing the two
trees, so a family takes exactly the kernels whose meaning it implements.  Each tree is also
what the generic lowering runs, statement by statement.

Ragged sizes.  A copy or an epilogue's load whose coordinate may pass the end of its axis reads
the last element of that axis instead (``clamped``), and the value is not stored: rows past M
and columns past N are masked by the RegStore's guards, and K's last slab is padded with zeros
in shared memory.
"""

from __future__ import annotations

from thompiler import ir

F32T = ir.DataType("f32", "float32", 4)
F16T = ir.DataType("f16", "float16", 2)
BF16T = ir.DataType("bf16", "bfloat16", 2)
I32T = ir.DataType("i32", "int32", 4)
TYPES = {t.name: t for t in (F32T, F16T, BF16T, I32T)}

V, B, E = ir.Var, ir.BinaryExpr, ir.ElementwiseImpl


def L(v, dt="int"):
    return ir.Literal(v, dt)


def axis(name, n):
    return ir.Axis(name, ir.Dim(n), None)


def assign(name, op, *args, dt=F32T):
    return ir.Assign(name, E(op), tuple(args), dt)


def clamped(e, n: int):
    """``e``, or the last index of an axis of ``n`` where ``e`` lies past it."""
    return ir.TernaryExpr(B("<", e, L(n)), e, L(n - 1))


def _load(name, buf, index, dtype):
    """One element as an f32 value (bf16 elements widen as they are loaded, f16 ones by a copy)."""
    if dtype == "f16":
        return [ir.Load((name + "h",), buf, index, F16T), ir.Assign(name, E("copy"), (name + "h",), F32T)]
    return [ir.Load((name,), buf, index, TYPES[dtype])]


def _write(buf, index, value, dtype):
    """One f32 value, rounded once to the buffer's type."""
    if dtype == "f16":
        return [ir.Assign(value + "h", E("copy"), (value,), F16T),
                ir.Write(buf, index, (value + "h",), F16T, False, "NONE")]
    return [ir.Write(buf, index, (value,), TYPES[dtype], False, "NONE")]


# ---- linear -----------------------------------------------------------------------------

ACTIVATIONS = ("relu", "silu", "gelu_tanh")
# gelu's tanh form by way of sigmoid: 0.5 z (1 + tanh u) = z sigmoid(2 u), u = sqrt(2/pi) (z + 0.044715 z^3);
# 1 + tanh u cancels for negative z, the sigmoid does not
GELU_C1 = 1.5957691216057308
GELU_C3 = GELU_C1 * 0.044715


def activation(z: str, name: str | None) -> tuple[list, str]:
    """Statements that apply an activation to the f32 value ``z``, and the result's name."""
    if name is None:
        return [], z
    if name == "relu":                                  # z < 0 ? 0 : z keeps a NaN; max(z, 0) would hide it
        return [ir.Let("none", L(0.0, "float"), F32T),
                ir.Select("act", (ir.Branch(V("none"), B("<", V(z), L(0.0, "float"))), ir.Branch(V(z), None)))], "act"
    if name == "silu":
        return [assign("sg", "sigmoid", z), assign("act", "multiply", z, "sg")], "act"
    if name == "gelu_tanh":
        return [ir.Let("gc1", L(GELU_C1, "float"), F32T), ir.Let("gc3", L(GELU_C3, "float"), F32T),
                assign("gz2", "multiply", z, z), assign("gz3", "multiply", "gz2", "gc3"),
                assign("gp", "add", "gz3", "gc1"), assign("gu", "multiply", "gp", z),
                assign("sg", "sigmoid", "gu"), assign("act", "multiply", z, "sg")], "act"
    raise ValueError(f"activation {name!r} (one of {', '.join(ACTIVATIONS)} or None)")


def linear_epilogue(M: int, N: int, dtype: str, bias: bool, act: str | None, residual: bool, gated: bool):
    """What follows the product, per element: z (+ bias), the activation, times the second product's
    element u (+ its bias) when gated, + residual.  None when nothing does."""
    if not (bias or act or residual or gated):
        return None
    row = clamped(V("row"), M) if M % 64 else V("row")
    col = clamped(V("col"), N) if N % 64 else V("col")
    body, z, u = [], "z", "u"
    if bias:
        body += [*_load("bz", "bias", (col,), dtype), assign("zb", "add", z, "bz")]
        z = "zb"
    more, z = activation(z, act)
    body += more
    if gated:
        if bias:
            body += [*_load("bu", "bias", (B("+", col, L(N)),), dtype), assign("ub", "add", u, "bu")]
            u = "ub"
        body.append(assign("gated", "multiply", z, u))
        z = "gated"
    if residual:
        body += [*_load("rz", "res", (row, col), dtype), assign("sum", "add", z, "rz")]
        z = "sum"
    return ir.Lambda(("z", "u", "row", "col") if gated else ("z", "row", "col"), tuple(body), (z,))


def linear_body(M: int, N: int, K: int, ab: str, gated: bool, epilogue, x: str = "x", w: str = "w",
                out: str = "linear"):
    """out[M, N] = epilogue(x[M, K] @ w[N, K]^T) on the warp-level tensor cores, f32 sums; gated:
    w[2N, K], the epilogue also takes the element of the product with w's second N rows.

    A 64 x 64 output tile per CTA of 4 warps, each warp a 16 x 64 strip; K in slabs of 64 staged
    with 16-byte copies under the 128-byte swizzle (the shared arrays hold raw 16-bit elements,
    f16 or bf16)."""
    DT = TYPES[ab]
    tid = B("+", B("*", V("a0_u"), L(32)), V("_lane"))
    slabs = [("_a_smem", x, "a0_b", M, 0), ("_b_smem", w, "a1_b", N, 0)]
    frags = [ir.RegFragment("_a", "a", (16, 8, 16), DT, 1, None),
             ir.RegFragment("_b", "b", (16, 8, 16), DT, 8, None),
             ir.RegFragment("_c", "c", (16, 8, 16), F32T, 8, None)]
    if gated:
        slabs.append(("_d_smem", w, "a1_b", N, N))
        frags += [ir.RegFragment("_e", "b", (16, 8, 16), DT, 8, None),
                  ir.RegFragment("_d", "c", (16, 8, 16), F32T, 8, None)]
    body = [*frags, *(ir.Smem(s[0], (64, 64), "__half", 1024) for s in slabs)]
    if K % 64:
        body.append(ir.Let("zero", L(0.0, "float"), F16T))
    copies = []
    for i in range(4):
        chunk = B("+", tid, L(128 * i))
        row, c8 = B("/", chunk, L(8)), B("*", B("%", chunk, L(8)), L(8))
        k = B("+", V("_ks"), c8)
        for smem, src, block, n, first in slabs:
            r = B("+", B("*", V(block), L(64)), row)
            if n % 64:
                r = clamped(r, n)
            if first:
                r = B("+", r, L(first))
            copy = ir.CpAsyncCopy(smem, (L(0), L(0)), src, (r, k), 16, "B128", (row, c8), None)
            if K % 64:
                copy = ir.Cond(B("<", k, L(K)), (copy,),
                               tuple(ir.Write(smem, (row, c), ("zero",) * 4, F16T, False, "B128")
                                     for c in (c8, B("+", c8, L(4)))))
            copies.append(copy)
    inner = [ir.LdmatrixLoad("_a", "_a_smem", (B("*", V("a0_u"), L(16)), V("_kk")), "a", 64, "B128", True, None,
                             None, False, None, False, None, (), 0, "m16n8k16", None)]
    pairs = [("_c", "_b", "_b_smem")] + ([("_d", "_e", "_d_smem")] if gated else [])
    for c, b, smem in pairs:
        for j in range(4):
            inner.append(ir.LdmatrixLoad(f"{b}[{2 * j}]", smem, (L(16 * j), V("_kk")), "b", 64, "B128", True, None,
                                         None, True, f"{b}[{2 * j + 1}]", False, None, (), 0, "m16n8k16", None))
        inner.append(ir.Loop(axis("_r0", 8), (ir.MmaSyncPtx(f"{c}[_r0]", "_a", f"{b}[_r0]", (16, 8, 16), ab, "f32",
                                                           False, None, None),), True, False))
    body.append(ir.StridedLoop(axis("_ks", K), L(0), L(64), (
        *copies, ir.CpAsyncCommit(), ir.CpAsyncWait(0), ir.Sync(0, None, False),
        ir.StridedLoop(axis("_kk", 64), L(0), L(16), tuple(inner), False, None, False),
        ir.Sync(0, None, False)), False, None, False))
    for j in range(8):
        body.append(ir.RegStore(out, (B("+", B("*", V("a0_b"), L(64)), B("*", V("a0_u"), L(16))),
                                      B("+", B("*", V("a1_b"), L(64)), L(8 * j))), f"_c[{j}]", (16, 8, 16), 0,
                                epilogue, (f"_d[{j}]",) if gated else (), L(M) if M % 64 else None,
                                L(N) if N % 64 else None, False, "m16n8k16", False, None, "NONE", None, None))
    return ir.Tile((axis("a0_b", -(-M // 64)), axis("a1_b", -(-N // 64)), axis("a0_u", 4), axis("_lane", 32)),
                   tuple(body), 128, 0, None, None, "m")


# ---- rotary heads ---------------------------------------------------------------------------

def heads_vector(D: int, R: int, nbytes: int) -> int:
    """Elements of a head (of D, R of them rotating) that the tuned kernel moves at a time: 16 bytes, or
    the largest power of two that divides the rotating half and the rest's."""
    V = 16 // nbytes
    while (R // 2) % V or ((D - R) // 2) % V:
        V //= 2
    return V


def heads_body(Bn: int, S: int, heads: int, kv: int, D: int, R: int, P: int, dtype: str, interleaved: bool,
               values: bool, heads_first: bool, inverse: bool, eps: float | None):
    """The heads of qkv[B, S, heads + kv (+ kv), D] into q, k (and v): one head of one token per warp.

    Queries and keys: y = x (norm: x * rsqrt(mean(x^2) + eps) * w, wq or wk), then of the leading R
    elements each pair (a, b) becomes (a cos - b sin, b cos + a sin), with row pos[b, s] of the
    tables cos / sin [P, R/2]; the pairs are (i, i + R/2), or (2i, 2i + 1) when interleaved;
    inverse: by the negative angle.  Values are copied.  A token whose position is outside
    [0, P) leaves its rows of the outputs as they were."""
    b, s, h, lane, p = V("a_b"), V("a_s"), V("a_h"), V("_lane"), V("p")
    half = R // 2

    def at(first, n, d):
        hh = B("-", h, L(first)) if first else h
        return (b, hh, s, d) if heads_first else (b, s, hh, d)

    def x(name, d):
        return _load(name, "qkv", (b, s, h, d), dtype)

    def copy(buf, first):
        return [ir.StridedLoop(axis("d", D), lane, L(32), (*x("xv", V("d")), *_write(buf, at(first, kv, V("d")), "xv",
                                                                                      dtype)), False, None, False)]

    def turned(buf, first, n, w):
        out, names = [], {}
        if eps is not None:
            out += [ir.StridedLoop(axis("d0", D), lane, L(32), (
                        *x("xs", V("d0")), assign("sq", "multiply", "xs", "xs"),
                        ir.Accum("acc", "sq", E("add"), F32T, ("d0",), None)), False, None, True),
                    ir.WarpShuffle(("acc",), ("acc__o",), (assign("acc", "add", "acc", "acc__o", dt=None),), 32, F32T),
                    ir.Let("count", L(float(D), "float"), F32T), ir.Let("eps", L(float(eps), "float"), F32T),
                    assign("mean", "divide", "acc", "count"), assign("meps", "add", "mean", "eps"),
                    assign("root", "sqrt", "meps"), assign("rstd", "reciprocal", "root")]

        def normed(name, d):
            st = x(name, d)
            if eps is None:
                return st, name
            return st + [assign(name + "r", "multiply", name, "rstd"), *_load(name + "w", w, (d,), dtype),
                         assign(name + "n", "multiply", name + "r", name + "w")], name + "n"
        i = V("i")
        d0, d1 = ((B("*", i, L(2)), B("+", B("*", i, L(2)), L(1))) if interleaved else (i, B("+", i, L(half))))
        s0, n0 = normed("xa", d0)
        s1, n1 = normed("xb", d1)
        first_op, second_op = ("add", "subtract") if inverse else ("subtract", "add")
        out.append(ir.StridedLoop(axis("i", half), lane, L(32), (
            *s0, *s1, ir.Load(("c",), "cos", (p, i), F32T), ir.Load(("sn",), "sin", (p, i), F32T),
            assign("ac", "multiply", n0, "c"), assign("bs", "multiply", n1, "sn"), assign("ya", first_op, "ac", "bs"),
            assign("bc", "multiply", n1, "c"), assign("as", "multiply", n0, "sn"), assign("yb", second_op, "bc", "as"),
            *_write(buf, at(first, n, d0), "ya", dtype), *_write(buf, at(first, n, d1), "yb", dtype)),
            False, None, False))
        if R < D:
            st, nm = normed("xt", V("dt"))
            out.append(ir.StridedLoop(axis("dt", D), B("+", lane, L(R)), L(32),
                                      (*st, *_write(buf, at(first, n, V("dt")), nm, dtype)), False, None, False))
        return out

    rows = tuple(turned("q", 0, heads, "wq"))
    if kv:
        rest = tuple(turned("k", heads, kv, "wk"))
        if values:
            rest = (ir.Cond(B("<", h, L(heads + kv)), rest, tuple(copy("v", heads + kv))),)
        rows = (ir.Cond(B("<", h, L(heads)), rows, rest),)
    n = heads + kv * (2 if values else 1)
    return ir.Tile((axis("a_b", Bn), axis("a_s", S), axis("a_h", n), axis("_lane", 32)), (
        ir.Load(("p",), "pos", (b, s), I32T),
        ir.Cond(B("&&", B(">=", p, L(0)), B("<", p, L(P))), rows, ())), 128, 0, None, None, "m")
