"""The layer operators on the GPU, under their own launch, under meta.json's and compiled without
the tuned families (the generic lowering of the same tree), against their float64 definitions.  Outputs lie inside larger buffers
whose other contents must not change; rows of empty slots keep what they held."""

import numpy as np
import pytest

from layer_cases import (HEADS, LINEAR, TAILS, check, custom_epilogue_package, custom_expected, heads_expected,
                         heads_package, heads_spec, linear_expected)
from thompiler import synth
from thompiler.device import DeviceKernel
from thompiler.families.tuning import TUNING

pytestmark = pytest.mark.gpu

PAD = 4096                                                # elements on either side of an output
SENTINEL = 7.0


def _t(dtype):
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[dtype]


def _out(shape, dtype):
    """(whole buffer, the output's view in its middle)."""
    import torch
    n = int(np.prod(shape))
    whole = torch.full((n + 2 * PAD,), SENTINEL, device="cuda", dtype=_t(dtype))
    return whole, whole[PAD:PAD + n].view(shape)


def _untouched(whole):
    assert bool((whole[:PAD] == SENTINEL).all()) and bool((whole[-PAD:] == SENTINEL).all())


def _stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def _np(t):
    return t.float().cpu().numpy()


def _kernel(d, launch):
    return DeviceKernel(next(d.glob("*.ir.json")), honour_meta=launch == "meta", tuned=launch != "generic")


def _linear_inputs(case, seed=0):
    import torch
    M, N, K, dtype, out, bias, act, res, gated = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = 2 * N if gated else N
    t = {"x": torch.randn(M, K, device="cuda", generator=g).to(_t(dtype)),
         "w": (torch.randn(rows, K, device="cuda", generator=g) * K ** -0.5).to(_t(dtype))}
    if bias:
        t["bias"] = torch.randn(rows, device="cuda", generator=g).to(_t(dtype))
    if res:
        t["res"] = torch.randn(M, N, device="cuda", generator=g).to(_t(dtype))
    return t


def _linear_check(case, t, got, what):
    M, N, K, dtype, out, bias, act, res, gated = case
    x = {n: _np(v) for n, v in t.items()}
    want, allowed = linear_expected(x["x"], x["w"], x.get("bias"), x.get("res"), N, act, gated, out)
    check(_np(got), want, allowed, what)


@pytest.mark.parametrize("launch", ["own", "meta", "generic", "stream", "rows", "split", "pair"])
@pytest.mark.parametrize("case", LINEAR, ids=str)
def test_linear(tmp_path, monkeypatch, case, launch):
    """``stream``, ``rows``, ``split`` and ``pair`` force one of the tuned kernels, also at sizes it is not chosen for."""
    import torch
    M, N = case[:2]
    if launch in ("stream", "rows", "split", "pair"):
        monkeypatch.setattr(TUNING, "linear_kernel", launch)
    k = _kernel(synth.linear_package(tmp_path, *case), launch)
    if launch in ("stream", "rows", "split", "pair") and not k.family.endswith(launch):
        pytest.skip(f"no {launch} plan for this size")
    t = _linear_inputs(case)
    whole, y = _out((M, N), case[4])
    ptrs = {n: v.data_ptr() for n, v in dict(t, linear=y).items()}
    k(ptrs, _stream())
    torch.cuda.synchronize()
    assert k.error_word() == 0
    _untouched(whole)
    _linear_check(case, t, y, f"{k.family} {launch}")
    first = y.clone()
    y.fill_(float("nan"))
    k(ptrs, _stream())                                    # the same bits again
    torch.cuda.synchronize()
    assert torch.equal(first, y)
    k.close()


@pytest.mark.parametrize("case,cut", TAILS, ids=str)
def test_pair_tails(tmp_path, monkeypatch, case, cut):
    import torch
    from thompiler.families.linear import LinearPair, Product
    from thompiler.load import load
    monkeypatch.setattr(TUNING, "linear_kernel", "pair")
    d = synth.linear_package(tmp_path, *case)
    assert min(LinearPair.plans(Product.read(load(next(d.glob("*.ir.json"))))))[3:] == cut
    k = _kernel(d, "own")
    _family(k, "pair")
    M, N = case[:2]
    t = _linear_inputs(case)
    whole, y = _out((M, N), case[4])
    k({n: v.data_ptr() for n, v in dict(t, linear=y).items()}, _stream())
    torch.cuda.synchronize()
    assert k.error_word() == 0
    _untouched(whole)
    rows = sorted(r for r in {0, 127, 128, 255, 256, M - 1, *range(0, M, 61), *range(max(0, M - 130), M, 17)} if r < M)
    some = {n: v[rows] if n in ("x", "res") else v for n, v in t.items()}
    _linear_check((len(rows), *case[1:]), some, y[rows], f"{cut}")
    assert bool(y.float().isfinite().all())
    k.close()


@pytest.mark.parametrize("kernel", ["generic", "stream", "rows", "split", "pair"])
@pytest.mark.parametrize("M,N,K", [(20, 200, 264), (32, 64, 64), (600, 328, 200)])
def test_custom_epilogue(tmp_path, monkeypatch, kernel, M, N, K):
    """Epilogues of other statements, buffers and types than the builder's are replayed by every kernel."""
    import torch
    from thompiler import problems
    if kernel != "generic":
        monkeypatch.setattr(TUNING, "linear_kernel", kernel)
    d = custom_epilogue_package(tmp_path, M, N, K)
    k = _kernel(d, "generic" if kernel == "generic" else "own")
    if kernel not in k.family:
        pytest.skip(f"no {kernel} plan for this size")
    x = problems.make_inputs(problems.load_package(d))
    t = {n: torch.from_numpy(v).cuda() for n, v in x.items()}
    whole, y = _out((M, N), "f32")
    k({n: v.data_ptr() for n, v in dict(t, linear=y).items()}, _stream())
    torch.cuda.synchronize()
    assert k.error_word() == 0
    _untouched(whole)
    want, allowed = custom_expected(x)
    check(_np(y), want, allowed, k.family)
    k.close()


def _heads_inputs(spec, table, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, S, D, R = spec["B"], spec["S"], spec["D"], spec["R"]
    n = spec["heads"] + spec["kv"] * (2 if spec["values"] else 1)
    a = torch.rand(table, R // 2, device="cuda", generator=g) * 6.28
    t = {"cos": torch.cos(a), "sin": torch.sin(a),
         "pos": torch.randint(0, table, (B, S), device="cuda", generator=g, dtype=torch.int32),
         "qkv": torch.randn(B, S, n, D, device="cuda", generator=g).to(_t(spec["dtype"]))}
    if spec["norm"]:
        t["wq"] = (torch.rand(D, device="cuda", generator=g) + 0.5).to(_t(spec["dtype"]))
        if spec["kv"]:
            t["wk"] = (torch.rand(D, device="cuda", generator=g) + 0.5).to(_t(spec["dtype"]))
    return t


def _heads_outputs(spec):
    B, S, D = spec["B"], spec["S"], spec["D"]
    out = {}
    for name, n in (("q", spec["heads"]), ("k", spec["kv"]), ("v", spec["kv"] if spec["values"] else 0)):
        if n:
            out[name] = _out((B, n, S, D) if spec["heads_first"] else (B, S, n, D), spec["dtype"])
    return out


def _heads_check(spec, table, t, out, what):
    x = {n: v.cpu().numpy() if n == "pos" else _np(v) for n, v in t.items()}
    want = heads_expected(x, spec, table, {n: SENTINEL for n in out})
    for name, (w, allowed) in want.items():
        whole, view = out[name]
        _untouched(whole)
        check(_np(view), w, allowed, f"{what} {name}")


@pytest.mark.parametrize("launch", ["own", "meta", "generic"])
@pytest.mark.parametrize("case", HEADS, ids=str)
def test_heads(tmp_path, case, launch):
    import torch
    spec, table = heads_spec(case), 1000
    k = _kernel(heads_package(synth, tmp_path, spec, table), launch)
    t = _heads_inputs(spec, table)
    if t["pos"].numel() > 2:                              # empty slots, and positions past the table
        t["pos"].view(-1)[-1] = -1
        t["pos"].view(-1)[1] = table
        t["pos"].view(-1)[0] = -2 ** 31
    out = _heads_outputs(spec)
    k(dict({n: v.data_ptr() for n, v in t.items()}, **{n: v.data_ptr() for n, (_, v) in out.items()}), _stream())
    torch.cuda.synchronize()
    _heads_check(spec, table, t, out, f"{k.family} {launch}")
    k.close()


# ---- as they are used --------------------------------------------------------------------------

ODD_HEADS = [(2, 9, 3, 2, 7, 4, "f32", False, True, True, False, False), (1, 33, 2, 1, 33, 32, "bf16", True, True, False, False, True),
             (3, 4, 1, 1, 129, 2, "f16", False, False, True, True, False)]


@pytest.mark.parametrize("case", ODD_HEADS, ids=str)
def test_heads_of_odd_length(tmp_path, case):
    """An odd number of elements a head has no pairs to move at a time: the generic lowering serves it."""
    import torch
    spec, table = heads_spec(case), 50
    k = _kernel(heads_package(synth, tmp_path, spec, table), "own")
    assert k.family == "generic"
    t, out = _heads_inputs(spec, table), _heads_outputs(spec)
    t["pos"][-1, -1] = -1
    k(dict({n: v.data_ptr() for n, v in t.items()}, **{n: v.data_ptr() for n, (_, v) in out.items()}), _stream())
    torch.cuda.synchronize()
    _heads_check(spec, table, t, out, "odd")
    k.close()


def _family(k, *names):
    assert any(n in k.family for n in names), k.family


@pytest.mark.parametrize("dtype", ["f16"])
def test_a_layer(tmp_path, dtype):
    """The dense path of a layer on one stream, eagerly and as a captured graph with fresh inputs: projection
    with bias, norm and rotation into the attention kernel's layout, attention, projection onto the
    residual stream, gated projection, projection onto the residual stream.  Each output is compared
    with its float64 definition on what the kernel before it wrote, so a kernel that starts too
    early shows."""
    import torch
    from thompiler import rotary
    B, S, H, D = 1, 256, 4, 64
    C, F, T = H * D, 512, B * S

    def linear(name, *a, **kw):
        return DeviceKernel(synth.linear_package(tmp_path / name, *a, dtype=dtype, **kw) / "k_linear.ir.json")
    k_qkv = linear("qkv", T, 3 * C, C, bias=True)
    k_rot = DeviceKernel(synth.qk_norm_rope_package(tmp_path / "rot", B, S, H, H, D, dtype=dtype, table=S + 100,
                                                    values=True, heads_first=True) / "k_qk_norm_rope.ir.json")
    k_att = DeviceKernel(synth.attention_package(tmp_path / "att", B, H, S, D) / "k_attention.ir.json")
    k_out = linear("out", T, C, C, residual=True)
    k_up = linear("up", T, F, C, activation="silu", gated=True)
    k_down = linear("down", T, C, F, residual=True)
    _family(k_rot, "rotary-heads")
    for k in (k_qkv, k_out, k_up, k_down):
        _family(k, "linear")
    g = torch.Generator(device="cuda").manual_seed(11)

    def new(*shape):
        return torch.empty(*shape, device="cuda", dtype=torch.float16)
    par = {n: (torch.randn(*s, device="cuda", generator=g) * sc).half() for n, s, sc in (
        ("wqkv", (3 * C, C), C ** -0.5), ("bqkv", (3 * C,), 0.5), ("wq", (D,), 1.0), ("wk", (D,), 1.0),
        ("wout", (C, C), C ** -0.5), ("wup", (2 * F, C), C ** -0.5), ("wdown", (C, F), F ** -0.5))}
    cos, sin = (torch.from_numpy(t).cuda() for t in rotary.tables(S + 100, D))
    pos = (torch.arange(S, device="cuda", dtype=torch.int32) + 100).repeat(B, 1)
    scale = torch.tensor([D ** 0.5], device="cuda")
    x, qkv, q, kk, v, o = new(T, C), new(T, 3 * C), *(new(B, H, S, D) for _ in range(4))
    o2, h, up, y = new(T, C), new(T, C), new(T, F), new(T, C)

    def p(**t):
        return {n: a.data_ptr() for n, a in t.items()}

    def run():
        s = _stream()
        k_qkv(p(x=x, w=par["wqkv"], bias=par["bqkv"], linear=qkv), s)
        k_rot(p(cos=cos, sin=sin, pos=pos, qkv=qkv, wq=par["wq"], wk=par["wk"], q=q, k=kk, v=v), s)
        k_att(p(div_c1=scale, q=q, k=kk, v=v, attn=o), s)
        o2.copy_(o.permute(0, 2, 1, 3).reshape(T, C))
        k_out(p(x=o2, w=par["wout"], res=x, linear=h), s)
        k_up(p(x=h, w=par["wup"], linear=up), s)
        k_down(p(x=up, w=par["wdown"], res=h, linear=y), s)

    def verify(what):
        import numpy as np
        n = {k: _np(t) for k, t in dict(par, x=x, qkv=qkv, q=q, k=kk, v=v, o=o, o2=o2, h=h, up=up, y=y).items()}
        for name, a, w, b, r, N, act, gated in (
                ("qkv", "x", "wqkv", "bqkv", None, 3 * C, None, False), ("h", "o2", "wout", None, "x", C, None, False),
                ("up", "h", "wup", None, None, F, "silu", True), ("y", "up", "wdown", None, "h", C, None, False)):
            want, allowed = linear_expected(n[a], n[w], n[b] if b else None, n[r] if r else None, N, act, gated, dtype)
            check(n[name], want, allowed, f"{what} {name}")
        spec = dict(B=B, S=S, heads=H, kv=H, D=D, R=D, dtype=dtype, interleaved=False, values=True, heads_first=True,
                    inverse=False, norm=True)
        src = {"cos": cos.cpu().numpy(), "sin": sin.cpu().numpy(), "pos": pos.cpu().numpy(),
               "qkv": n["qkv"].reshape(B, S, 3 * H, D), "wq": n["wq"], "wk": n["wk"]}
        for name, (want, allowed) in heads_expected(src, spec, S + 100, {t: 0.0 for t in "qkv"}).items():
            check(n[name], want, allowed, f"{what} {name}")
        s_ = n["q"].astype(np.float64) @ n["k"].astype(np.float64).transpose(0, 1, 3, 2) / D ** 0.5
        e_ = np.exp(s_ - s_.max(-1, keepdims=True))
        want = (e_ / e_.sum(-1, keepdims=True)) @ n["v"].astype(np.float64)
        assert np.allclose(n["o"], want, rtol=2e-2, atol=2e-3), what
        for k in (k_qkv, k_att, k_out, k_up, k_down):
            assert k.error_word() == 0

    def refill():
        x.copy_(torch.randn(T, C, device="cuda", generator=g))
        for t in (qkv, q, kk, v, o, o2, h, up, y):
            t.fill_(float("nan"))

    for i in range(3):
        refill()
        run()
        torch.cuda.synchronize()
        verify(f"eager {i}")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in range(3):
        refill()
        graph.replay()
        torch.cuda.synchronize()
        verify(f"replay {i}")
    del graph
    for k in (k_qkv, k_rot, k_att, k_out, k_up, k_down):
        k.close()


@pytest.mark.parametrize("kernel,M,N", [("stream", 5, 512), ("stream", 16, 1024), ("rows", 5, 512), ("rows", 200, 512),
                                        ("split", 300, 512), ("split", 20, 1024), ("pair", 300, 512)])
def test_chain_reads_what_the_launch_before_wrote(tmp_path, monkeypatch, kernel, M, N):
    """Launches that overlap, each reading the one before it, in a graph replayed many times: the bits of the
    same calls made one by one.  (Loads that the assembler may move above the wait for the previous kernel
    fail this at every replay.)"""
    import torch
    monkeypatch.setattr(TUNING, "linear_kernel", kernel)
    layers = 40
    case = (M, N, N, "bf16", "bf16", False, "silu", True, False)
    k = _kernel(synth.linear_package(tmp_path, *case), "own")
    _family(k, kernel)
    t = _linear_inputs(case)
    ws = [(torch.randn(N, N, device="cuda") * N ** -0.5).to(torch.bfloat16) for _ in range(layers)]
    ys = [torch.empty(M, N, device="cuda", dtype=torch.bfloat16) for _ in ws]

    def call(src, w, y):
        k({"x": src.data_ptr(), "w": w.data_ptr(), "res": t["res"].data_ptr(), "linear": y.data_ptr()}, _stream())
    refs, src = [], t["x"]
    for w, y in zip(ws, ys):
        call(src, w, y)
        torch.cuda.synchronize()
        refs.append(y.clone())
        src = y
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        src = t["x"]
        for w, y in zip(ws, ys):
            call(src, w, y)
            src = y
    for i in range(50):
        for y in ys:
            y.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for n, (a, b) in enumerate(zip(ys, refs)):
            assert torch.equal(a, b), f"replay {i}, layer {n}"
    assert k.error_word() == 0
    del graph
    k.close()


def test_heads_chain(tmp_path):
    """The same for rotations: forward and inverse in turn, each of the one before it."""
    import torch
    spec = heads_spec((1, 64, 8, 0, 128, 128, "f32", False, False, False, False, False))
    ks = [_kernel(heads_package(synth, tmp_path / str(inv), dict(spec, inverse=inv), 64), "own") for inv in (False, True)]
    t = _heads_inputs(spec, 64)
    ys = [torch.empty_like(t["qkv"]) for _ in range(40)]

    def run(sync=False):
        src = t["qkv"]
        for i, y in enumerate(ys):
            ks[i % 2]({"cos": t["cos"].data_ptr(), "sin": t["sin"].data_ptr(), "pos": t["pos"].data_ptr(),
                       "qkv": src.data_ptr(), "q": y.data_ptr()}, _stream())
            if sync:
                torch.cuda.synchronize()
            src = y
    run(True)
    refs = [y.clone() for y in ys]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in range(50):
        for y in ys:
            y.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ys, refs)), i
    del graph
    for k in ks:
        k.close()


@pytest.mark.parametrize("kernel", ["stream", "rows"])
def test_few_row_kernels_share_a_graph_with_many_weights(tmp_path, monkeypatch, kernel):
    """One compiled kernel for all layers of a model: twenty weights captured into one graph with no call
    on them before the capture (nothing is kept for a buffer), replayed with new activations."""
    import torch
    monkeypatch.setattr(TUNING, "linear_kernel", kernel)
    M, N = 5, 512
    case = (M, N, N, "bf16", "bf16", False, "silu", True, False)
    k = _kernel(synth.linear_package(tmp_path, *case), "own")
    _family(k, kernel)
    t = _linear_inputs(case)
    ws = [torch.randn(N, N, device="cuda").mul_(N ** -0.5).to(torch.bfloat16) for _ in range(20)]
    ys = [torch.empty(M, N, device="cuda", dtype=torch.bfloat16) for _ in ws]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        src = t["x"]
        for w, y in zip(ws, ys):                          # each layer's result is the next one's input
            k({"x": src.data_ptr(), "w": w.data_ptr(), "res": t["res"].data_ptr(), "linear": y.data_ptr()}, _stream())
            src = y
    for seed in (1, 2):
        t["x"].copy_(_linear_inputs(case, seed)["x"])
        for y in ys:
            y.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        src = t["x"]
        for i, (w, y) in enumerate(zip(ws, ys)):
            _linear_check(case, {"x": src, "w": w, "res": t["res"]}, y, f"layer {i}")
            src = y
    assert k.error_word() == 0
    del graph
    k.close()


def test_pair_kernel_serves_many_weights(tmp_path, monkeypatch):
    """The kernel for many rows keeps 128 sets of tensor maps: 150 weights one after another re-encode the
    oldest, a hundred of them then share a graph."""
    import torch
    monkeypatch.setattr(TUNING, "linear_kernel", "pair")
    M, N = 200, 264
    case = (M, N, N, "bf16", "bf16", False, None, True, False)
    k = _kernel(synth.linear_package(tmp_path, *case), "own")
    _family(k, "pair")
    t = _linear_inputs(case)
    ws = [(torch.randn(N, N, device="cuda") * N ** -0.5).to(torch.bfloat16) for _ in range(150)]
    ys = [torch.empty(M, N, device="cuda", dtype=torch.bfloat16) for _ in ws]
    for w in ws:
        w.fill_diagonal_(0.5)

    def run(first, last):
        for w, y in zip(ws[first:last], ys[first:last]):
            k({"x": t["x"].data_ptr(), "w": w.data_ptr(), "res": t["res"].data_ptr(), "linear": y.data_ptr()},
              _stream())

    def verify(first, last):
        for i in range(first, last):
            _linear_check(case, {"x": t["x"], "w": ws[i], "res": t["res"]}, ys[i], f"weight {i}")
    run(0, 150)
    torch.cuda.synchronize()
    verify(0, 150)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(50, 150)
    t["x"].copy_(_linear_inputs(case, 1)["x"])
    for y in ys:
        y.fill_(float("nan"))
    run(0, 50)                                            # others around it leave the graph's sets alone
    graph.replay()
    torch.cuda.synchronize()
    assert k.error_word() == 0
    verify(0, 150)
    del graph
    k.close()


@pytest.mark.parametrize("kernel", ["split", "pair"])
def test_refuses_buffers_without_maps(tmp_path, monkeypatch, kernel):
    """A launch in the kernel's own geometry on buffers whose tensor maps nobody bound writes nothing and says
    so in the error word (the generic lowering needs meta.json's grid)."""
    import torch
    monkeypatch.setattr(TUNING, "linear_kernel", kernel)
    case = (200, 264, 264, "bf16", "bf16", False, None, False, False)
    k = _kernel(synth.linear_package(tmp_path, *case), "own")
    t = _linear_inputs(case)
    y = torch.full((200, 264), SENTINEL, device="cuda", dtype=torch.bfloat16)
    ptrs = {n: v.data_ptr() for n, v in dict(t, linear=y).items()}
    k.fn.launch(k.plan.grid, k.plan.block, k.plan.smem, [ptrs[n] for n in k.arg_order], _stream())
    torch.cuda.synchronize()
    assert k.error_word() == 1 << 4 and bool((y == SENTINEL).all())
    k(ptrs, _stream())
    torch.cuda.synchronize()
    _linear_check(case, t, y, k.family)
    k.close()


@pytest.mark.parametrize("launch", ["generic", "stream", "rows", "split", "pair"])
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
def test_residual_in_place_and_shared_inputs(tmp_path, monkeypatch, launch, gated):
    """``res`` may be ``linear`` itself (every element is read by the thread that then stores it), and x."""
    import torch
    if launch != "generic":
        monkeypatch.setattr(TUNING, "linear_kernel", launch)
    for M in (20, 24):
        case = (M, 1032, 1032, "bf16", "bf16", True, "silu", True, gated)
        k = _kernel(synth.linear_package(tmp_path / str(M), *case), "generic" if launch == "generic" else "own")
        assert launch in k.family
        t = _linear_inputs(case)
        want = dict(t, res=t["res"].clone())
        ptrs = {n: v.data_ptr() for n, v in t.items()}
        k(dict(ptrs, linear=ptrs["res"]), _stream())
        torch.cuda.synchronize()
        _linear_check(case, want, t["res"], f"{k.family} in place")
        y = torch.empty_like(t["res"])
        k(dict(ptrs, res=ptrs["x"], linear=y.data_ptr()), _stream())
        torch.cuda.synchronize()
        _linear_check(case, dict(t, res=t["x"]), y, f"{k.family} x + f(x)")
        assert k.error_word() == 0
        k.close()


def test_residual_in_place_many_tiles(tmp_path):
    """The same over tiles that share rows and columns of several CTAs."""
    import torch
    case = (1300, 2056, 520, "f16", "f16", False, None, True, False)
    k = _kernel(synth.linear_package(tmp_path, *case), "own")
    t = _linear_inputs(case)
    before = t["res"].clone()
    for _ in range(3):
        t["res"].copy_(before)
        ptrs = {n: v.data_ptr() for n, v in t.items()}
        k(dict(ptrs, linear=ptrs["res"]), _stream())
        torch.cuda.synchronize()
        _linear_check(case, dict(t, res=before), t["res"], k.family)
    k.close()


@pytest.mark.parametrize("kernel", ["stream", "rows", "split", "pair"])
def test_two_streams_at_once(tmp_path, monkeypatch, kernel):
    """Calls of one kernel in flight on two streams, on buffers of their own."""
    import torch
    monkeypatch.setattr(TUNING, "linear_kernel", kernel)
    case = (24, 2048, 1024, "f16", "f16", True, "gelu_tanh", True, False)
    k = _kernel(synth.linear_package(tmp_path, *case), "own")
    _family(k, kernel)
    sets = [_linear_inputs(case, s) for s in (1, 2)]
    outs = [torch.full((24, 2048), float("nan"), device="cuda", dtype=torch.float16) for _ in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        for t, y, s in zip(sets, outs, streams):
            k({n: v.data_ptr() for n, v in dict(t, linear=y).items()}, s.cuda_stream)
    torch.cuda.synchronize()
    assert k.error_word() == 0
    for t, y in zip(sets, outs):
        _linear_check(case, t, y, kernel)
    k.close()


@pytest.mark.parametrize("kernel", ["stream", "rows", "split", "pair", "generic"])
def test_not_finite(tmp_path, monkeypatch, kernel):
    """NaN and infinities stay in the rows and columns they belong to: a NaN row of x, an infinite row of w,
    an infinite residual; the padding of K, M and N adds none."""
    import torch
    if kernel != "generic":
        monkeypatch.setattr(TUNING, "linear_kernel", kernel)
    case = (20, 200, 136, "bf16", "bf16", True, "silu", True, False)
    k = _kernel(synth.linear_package(tmp_path, *case), "generic" if kernel == "generic" else "own")
    t = _linear_inputs(case)
    t["x"][3, 7] = float("nan")
    t["w"][199, 135] = float("inf")
    t["x"][:, 135] = t["x"][:, 135].abs() + 0.5           # inf * x stays +inf: silu(+inf) = +inf
    t["res"][5, 11] = float("-inf")
    y = torch.zeros(20, 200, device="cuda", dtype=torch.bfloat16)
    k({n: v.data_ptr() for n, v in dict(t, linear=y).items()}, _stream())
    torch.cuda.synchronize()
    got = _np(y)
    assert np.isnan(got[3]).all() and np.isposinf(np.delete(got[:, 199], 3)).all() and np.isneginf(got[5, 11])
    rest = np.ones_like(got, dtype=bool)
    rest[3], rest[:, 199], rest[5, 11] = False, False, False
    assert np.isfinite(got[rest]).all()
    clean = dict(t)
    clean["x"], clean["w"], clean["res"] = t["x"].clone(), t["w"].clone(), t["res"].clone()
    clean["x"][3, 7], clean["w"][199, 135], clean["res"][5, 11] = 0, 0, 0
    x = {n: _np(v) for n, v in clean.items()}
    want, allowed = linear_expected(x["x"], x["w"], x["bias"], x["res"], 200, "silu", False, "bf16")
    check(np.where(rest, got, want), want, allowed, kernel)
    k.close()


@pytest.mark.parametrize("act", ["relu", "gelu_tanh"])
@pytest.mark.parametrize("kernel", ["stream", "rows", "split", "pair", "generic"])
def test_activations_keep_nan(tmp_path, monkeypatch, kernel, act):
    """A NaN row of x is a NaN row of the result, not the zeros of a maximum."""
    import torch
    if kernel != "generic":
        monkeypatch.setattr(TUNING, "linear_kernel", kernel)
    case = (9, 72, 64, "f16", "f32", False, act, False, False)
    k = _kernel(synth.linear_package(tmp_path, *case), "generic" if kernel == "generic" else "own")
    t = _linear_inputs(case)
    t["x"][4, 63] = float("nan")
    y = torch.zeros(9, 72, device="cuda")
    k({n: v.data_ptr() for n, v in dict(t, linear=y).items()}, _stream())
    torch.cuda.synchronize()
    assert k.error_word() == 0
    assert bool(y[4].isnan().all()) and int(y.isnan().sum()) == 72
    k.close()


def test_heads_not_finite(tmp_path):
    """Of a head that rotates half of its elements, a NaN in the rest stays where it is; with the norm it
    takes the head and no other."""
    import torch
    spec = heads_spec((1, 6, 3, 1, 64, 32, "bf16", True, True, False, False, False))
    for norm in (False, True):
        spec["norm"] = norm
        k = _kernel(heads_package(synth, tmp_path / str(norm), spec, 100), "own")
        t = _heads_inputs(spec, 100)
        t["qkv"][0, 2, 1, 40] = float("nan")              # a query head's unrotated part
        t["qkv"][0, 3, 0, 5] = float("inf")               # a rotated pair
        t["qkv"][0, 4, 4, 9] = float("nan")               # a value
        out = _heads_outputs(spec)
        k(dict({n: v.data_ptr() for n, v in t.items()}, **{n: v.data_ptr() for n, (_, v) in out.items()}), _stream())
        torch.cuda.synchronize()
        q, kk, v = (_np(out[n][1]) for n in ("q", "k", "v"))
        bad = np.argwhere(~np.isfinite(q))
        heads = {(int(s), int(h)) for _, s, h, _ in bad}
        assert heads == {(2, 1), (3, 0)}
        if not norm:
            assert {int(d) for _, s, _, d in bad if s == 2} == {40}
            assert {int(d) for _, s, _, d in bad if s == 3} == {4, 5}
        assert np.isfinite(kk).all() and np.argwhere(~np.isfinite(v)).tolist() == [[0, 4, 0, 9]]
        k.close()


def test_misaligned_buffers(tmp_path):
    """A buffer that does not start on the boundary its vectors need is refused before the launch, by name; one
    that starts on a later such boundary is served."""
    import torch
    from thompiler.runner import RunnerError
    for M in (4, 100, 700):
        case = (M, 64, 64, "f16", "f16", True, None, True, False)
        k = _kernel(synth.linear_package(tmp_path / str(M), *case), "own")
        t = _linear_inputs(case)
        y = torch.zeros(M * 64 + 16, device="cuda", dtype=torch.float16)
        ptrs = {n: v.data_ptr() for n, v in dict(t, linear=y).items()}
        for name in ptrs:
            with pytest.raises(RunnerError, match=f"buffer '{name}' .* not 16-byte aligned"):
                k(dict(ptrs, **{name: ptrs[name] + 8}), _stream())
        for name in ptrs:
            u, at = dict(t), y[:M * 64]
            if name in u:
                u[name] = torch.empty(t[name].numel() + 8, device="cuda", dtype=torch.float16)[8:].view(t[name].shape)
                u[name].copy_(t[name])
            else:
                at = y[8:8 + M * 64]
            y.fill_(float("nan"))
            k({n: v.data_ptr() for n, v in dict(u, linear=at).items()}, _stream())
            torch.cuda.synchronize()
            assert k.error_word() == 0
            _linear_check(case, t, at.view(M, 64), f"{k.family} {name}")
        k.close()
    for D, R, step in ((64, 64, 8), (80, 40, 4), (10, 6, 1)):
        spec = heads_spec((1, 33, 4, 2, D, R, "f16", False, True, True, False, True))
        k = _kernel(heads_package(synth, tmp_path / f"h{D}", spec, 100), "own")
        t = _heads_inputs(spec, 100)
        for name in ("qkv", "wq", "wk", "q", "k", "v"):
            out, u = _heads_outputs(spec), dict(t)
            ptrs = {n: v.data_ptr() for n, v in t.items()}
            ptrs.update({n: v.data_ptr() for n, (_, v) in out.items()})
            if step > 1:
                with pytest.raises(RunnerError, match=f"buffer '{name}' .* not {2 * step}-byte aligned"):
                    k(dict(ptrs, **{name: ptrs[name] + step}), _stream())
            whole, src = None, out[name][1] if name in out else t[name]
            whole = torch.full((src.numel() + 2 * PAD,), SENTINEL, device="cuda", dtype=torch.float16)
            view = whole[PAD + step:PAD + step + src.numel()].view(src.shape)
            view.copy_(src)
            k(dict(ptrs, **{name: view.data_ptr()}), _stream())
            torch.cuda.synchronize()
            assert k.error_word() == 0
            if name in out:
                out[name][1].copy_(view)
            _heads_check(spec, 100, t, out, f"{name} at {step}")
        k.close()


def test_offsets_past_32_bits(tmp_path):
    """Rows and products of more than 2^31 elements: the last ones are right."""
    import torch
    spec = heads_spec((1, 400000, 32, 16, 96, 96, "bf16", False, True, False, False, False))
    assert 400000 * 64 * 96 > 2 ** 31
    k = _kernel(heads_package(synth, tmp_path / "h", spec, 16), "own")
    _family(k, "rotary-heads")
    S, tail = 400000, 3
    qkv = torch.zeros(1, S, 64, 96, device="cuda", dtype=torch.bfloat16)
    qkv[:, -tail:] = torch.randn(1, tail, 64, 96, device="cuda").to(torch.bfloat16)
    small = dict(spec, S=tail)
    t = _heads_inputs(small, 16)
    t["qkv"] = qkv[:, -tail:].contiguous()
    pos = torch.zeros(1, S, device="cuda", dtype=torch.int32)
    pos[:, -tail:] = t["pos"]
    out = {n: torch.full((1, S, h, 96), SENTINEL, device="cuda", dtype=torch.bfloat16)
           for n, h in (("q", 32), ("k", 16), ("v", 16))}
    ptrs = {n: v.data_ptr() for n, v in dict(t, qkv=qkv, pos=pos, **out).items()}
    k(ptrs, _stream())
    torch.cuda.synchronize()
    x = {n: v.cpu().numpy() if n == "pos" else _np(v) for n, v in t.items()}
    for name, (want, allowed) in heads_expected(x, small, 16, {n: SENTINEL for n in out}).items():
        check(_np(out[name][:, -tail:]), want, allowed, name)
    k.close()
    del qkv, out, pos
    torch.cuda.empty_cache()
    M, N, K = 33000, 65536, 64
    case = (M, N, K, "f16", "f16", False, None, True, False)
    k = _kernel(synth.linear_package(tmp_path / "l", *case), "own")
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w = (torch.randn(n, K, device="cuda", generator=g).half() for n in (M, N))
    y = torch.full((M, N), float("nan"), device="cuda", dtype=torch.float16)
    res = torch.zeros(M, N, device="cuda", dtype=torch.float16)
    res[-2:] = torch.randn(2, N, device="cuda", generator=g).half()
    k({"x": x.data_ptr(), "w": w.data_ptr(), "res": res.data_ptr(), "linear": y.data_ptr()}, _stream())
    torch.cuda.synchronize()
    assert k.error_word() == 0
    for rows in (slice(0, 2), slice(M - 2, M)):
        want, allowed = linear_expected(_np(x[rows]), _np(w), None, _np(res[rows]), N, None, False, "f16")
        check(_np(y[rows]), want, allowed, "linear")
    k.close()


def test_rotation_inverse_undoes_and_is_the_gradient(tmp_path):
    """inverse(rope(x)) = x; and for a linear map, <g, rope(x)> = <inverse(g), x>: the inverse rotation is
    the gradient, checked against differences of the forward kernel too."""
    import torch
    spec = heads_spec((2, 17, 4, 0, 64, 48, "f32", True, False, False, False, False))
    fwd = _kernel(heads_package(synth, tmp_path / "f", spec, 64), "own")
    bwd = _kernel(heads_package(synth, tmp_path / "b", dict(spec, inverse=True), 64), "own")
    t = _heads_inputs(spec, 64)

    def call(k, x):
        y = torch.zeros_like(x)
        k({"cos": t["cos"].data_ptr(), "sin": t["sin"].data_ptr(), "pos": t["pos"].data_ptr(), "qkv": x.data_ptr(),
           "q": y.data_ptr()}, _stream())
        torch.cuda.synchronize()
        return y
    x = t["qkv"]
    y = call(fwd, x)
    # each pair: two products and a sum twice over, of values below 2^3: 2^-24 * 8 * 8
    assert (call(bwd, y) - x).abs().max().item() <= 2.0 ** -18
    g = torch.randn_like(x)
    dx = call(bwd, g).double()
    lhs, rhs = (g.double() * y.double()).sum().item(), (dx * x.double()).sum().item()
    assert abs(lhs - rhs) <= 2.0 ** -20 * (g.double().abs() * y.double().abs()).sum().item()
    for i in (0, 777, 2049, x.numel() - 1):               # differences: the map is linear, so a step of 1 is exact
        e = x.clone()
        e.view(-1)[i] += 1.0
        step = (e.view(-1)[i] - x.view(-1)[i]).item()
        diff = ((call(fwd, e).double() - y.double()) * g.double()).sum().item() / step
        # the rotated pair of the changed element differs by roundings of values below 2^3
        assert abs(diff - dx.view(-1)[i].item()) <= 2.0 ** -18 * (1 + g.abs().max().item())
    fwd.close()
    bwd.close()
