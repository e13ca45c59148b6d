"""The layer operators on the GPU, under their own launch, under meta.json's and compiled without
the tuned families (the generic lowering of the same tree), against their float64 definitions.  Outputs lie inside larger buffers
whose other contents must not change; rows of empty slots keep what they held."""

import numpy as np
import pytest

from layer_cases import HEADS, LINEAR, check, heads_expected, heads_package, heads_spec, linear_expected
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


@pytest.mark.parametrize("launch", ["own", "meta", "generic", "rows", "pair"])
@pytest.mark.parametrize("case", LINEAR, ids=str)
def test_linear(tmp_path, monkeypatch, case, launch):
    """``rows`` and ``pair`` force one of the two tuned kernels, also at sizes it is not chosen for."""
    import torch
    M, N = case[:2]
    if launch in ("rows", "pair"):
        monkeypatch.setattr(TUNING, "linear_kernel", launch)
    k = _kernel(synth.linear_package(tmp_path, *case), launch)
    if launch in ("rows", "pair") and not k.family.endswith(launch):
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
