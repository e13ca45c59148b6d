"""The layer operators on the CPU: the packages' statement trees, run by the oracle's interpreter
(every access bounds-checked), give the operators' float64 definitions within what f32 arithmetic
and one rounding allow; the builders refuse what they do not take; every module assembles without
spills; the rotary tables follow their formulas."""

import re
import shutil
import subprocess

import numpy as np
import pytest

from layer_cases import (HEADS, LINEAR, TAILS, check, custom_epilogue_package, custom_expected, heads_expected,
                         heads_package, heads_spec, linear_expected)
from oracle.interp import run_package as oracle_run
from thompiler import ir, load, problems, rotary, synth
from thompiler.compiler import compile_kernel


def _ir(d):
    return next(d.glob("*.ir.json"))


@pytest.mark.parametrize("case", [c for c in LINEAR if c[3] == "f16" and c[0] * c[1] * c[2] < 2 ** 24], ids=str)
def test_linear_tree_is_the_definition(tmp_path, case):
    M, N, K, dtype, out, bias, act, res, gated = case
    d = synth.linear_package(tmp_path, M, N, K, dtype, out, bias, act, res, gated)
    x = problems.make_inputs(problems.load_package(d))
    want, allowed = linear_expected(x["x"], x["w"], x.get("bias"), x.get("res"), N, act, gated, out)
    check(oracle_run(d)["linear"], want, allowed, "linear")


@pytest.mark.parametrize("case", [c for c in HEADS if c[6] != "bf16" and c[1] < 200], ids=str)
def test_heads_tree_is_the_definition(tmp_path, case):
    spec, table = heads_spec(case), 23
    d = heads_package(synth, tmp_path, spec, table)
    x = problems.make_inputs(problems.load_package(d))
    x["pos"].flat[-1] = -1                               # an empty slot, and a position past the table
    if x["pos"].size > 2:
        x["pos"].flat[1] = table
    got = oracle_run(d, x)
    zeros = {n: 0.0 for n in ("q", "k", "v")}
    want = heads_expected(x, spec, table, zeros)
    assert set(got) == set(want)
    for name, (w, allowed) in want.items():
        check(got[name], w, allowed, name)


def test_custom_epilogue_tree(tmp_path):
    d = custom_epilogue_package(tmp_path, 40, 72, 136)
    x = problems.make_inputs(problems.load_package(d))
    want, allowed = custom_expected(x)
    check(oracle_run(d)["linear"], want, allowed, "linear")


def test_tree_survives_the_reader(tmp_path):
    """The written text reads back as the tree the builder made (families compare the two)."""
    from thompiler import schedules
    epi = schedules.linear_epilogue(70, 72, "bf16", True, "gelu_tanh", True, True)
    tree = schedules.linear_body(70, 72, 136, "bf16", True, epi)
    assert ir.parse_stmt(synth.to_repr(tree)) == tree
    tree = schedules.heads_body(2, 3, 4, 2, 80, 40, 9, "f16", True, True, True, False, 1e-5)
    assert ir.parse_stmt(synth.to_repr(tree)) == tree


@pytest.mark.parametrize("kw,text", [
    (dict(M=0, N=64, K=64), "M = 0"), (dict(M=4, N=60, K=64), "multiples of 8"), (dict(M=4, N=64, K=60), "multiples of 8"),
    (dict(M=4, N=64, K=64, dtype="f32"), "dtype 'f32'"), (dict(M=4, N=64, K=64, dtype="f16", out_dtype="bf16"), "dtype"),
    (dict(M=4, N=64, K=64, activation="gelu"), "activation 'gelu'"), (dict(M=2.0, N=64, K=64), "M = 2.0"),
    (dict(M=4, N=-8, K=64), "N = -8")])
def test_linear_refusals(tmp_path, kw, text):
    with pytest.raises(ValueError, match=text):
        synth.linear_package(tmp_path, **kw)
    assert not list(tmp_path.glob("*"))


@pytest.mark.parametrize("kw,text", [
    (dict(rotary=33), "rotary = 33"), (dict(rotary=130), "rotary = 130"), (dict(rotary=0), "rotary = 0"),
    (dict(dtype="f64"), "dtype 'f64'"), (dict(kv_heads=0, values=True), "values without kv_heads"),
    (dict(kv_heads=-1), "kv_heads = -1"), (dict(S=0), "S = 0"), (dict(table=0), "table = 0"), (dict(D=0), "D = 0"),
    (dict(heads=0), "heads = 0")])
def test_heads_refusals(tmp_path, kw, text):
    args = dict(B=1, S=4, heads=4, kv_heads=2, D=128)
    for build in (synth.rope_package, synth.qk_norm_rope_package):
        with pytest.raises(ValueError, match=re.escape(text)):
            build(tmp_path, **dict(args, **kw))
    assert not list(tmp_path.glob("*"))


def test_norm_refuses_a_negative_eps(tmp_path):
    for eps in (-1e-6, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            synth.qk_norm_rope_package(tmp_path, 1, 4, 4, 2, 128, eps=eps)


def _ptxas(ptx, tmp_path):
    if shutil.which("ptxas") is None:
        pytest.skip("ptxas not on PATH")
    f = tmp_path / "k.ptx"
    f.write_text(ptx)
    r = subprocess.run(["ptxas", "-arch=sm_100a", "-v", str(f), "-o", str(tmp_path / "k.cubin")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert "0 bytes spill stores" in r.stderr and "0 bytes stack frame" in r.stderr, r.stderr


@pytest.mark.parametrize("tuned", [True, False], ids=["tuned", "generic"])
@pytest.mark.parametrize("case", [LINEAR[i] for i in (1, 3, 4, 7, 12, 16, 17)], ids=str)
def test_linear_assembles(tmp_path, case, tuned):
    d = synth.linear_package(tmp_path, *case)
    _ptxas(compile_kernel(load.load(str(_ir(d))), tuned=tuned), tmp_path)


@pytest.mark.parametrize("kernel", ["stream", "rows", "split", "pair"])
@pytest.mark.parametrize("case", [LINEAR[i] for i in (4, 5, 7)] + [(20, 264, 200, "bf16", "f32", True, "relu", True, False)],
                         ids=str)
def test_each_linear_kernel_assembles(tmp_path, monkeypatch, case, kernel):
    from thompiler.emitter import read_sidecar
    from thompiler.families.tuning import TUNING
    monkeypatch.setattr(TUNING, "linear_kernel", kernel)
    ptx = compile_kernel(load.load(str(_ir(synth.linear_package(tmp_path, *case)))))
    if not (kernel == "stream" and case[0] > 24):
        assert read_sidecar(ptx)["family"].endswith(kernel)
    _ptxas(ptx, tmp_path)


@pytest.mark.parametrize("tuned", [True, False], ids=["tuned", "generic"])
@pytest.mark.parametrize("case", HEADS, ids=str)
def test_heads_assemble(tmp_path, case, tuned):
    d = heads_package(synth, tmp_path, heads_spec(case), 64)
    _ptxas(compile_kernel(load.load(str(_ir(d))), tuned=tuned), tmp_path)


def test_misaligned_buffer_is_refused_by_name(tmp_path):
    """The check precedes everything of the launch, so it answers without a GPU."""
    from types import SimpleNamespace

    from thompiler import runner
    if not runner.LIB_PATH.exists():
        pytest.skip("runner library not built")
    for d in (synth.linear_package(tmp_path / "l", 4, 64, 64, bias=True, residual=True),
              synth.qk_norm_rope_package(tmp_path / "h", 1, 4, 4, 2, 128, values=True),
              synth.rope_package(tmp_path / "r", 1, 4, 4, 2, 80, rotary=40)):
        import json
        kmeta = json.loads((d / "meta.json").read_text())["kernels"][0]
        k = runner.Launch(SimpleNamespace(handle=1, name=kmeta["entry"], module=SimpleNamespace(handle=0)),
                          SimpleNamespace(grid=(1, 1, 1), block=(128, 1, 1), smem=0, pdl=True), kmeta, None)
        want = {a["name"]: a["align"] for a in kmeta["args"] if "align" in a}
        assert set(want) == set(kmeta["arg_order"]) - {"pos"}
        good = {n: 4096 * (i + 1) for i, n in enumerate(kmeta["arg_order"])}
        for name, align in want.items():
            with pytest.raises(runner.RunnerError, match=f"buffer '{name}' .* not {align}-byte aligned") as e:
                k(dict(good, **{name: good[name] + align // 2}))
            assert e.value.stage == "request"
    assert min(want.values()) == 8                        # the last one moves four f16 elements at a time


@pytest.mark.parametrize("kernel", ["stream", "rows", "split", "pair", "heads"])
def test_waits_for_the_previous_kernel(tmp_path, monkeypatch, kernel):
    """Launches may overlap the previous kernel's end: no access to global data, and in the kernel whose CTAs
    share SMs with others' no tensor memory taken, before the wait for it; the next kernel may come
    only after that memory is taken."""
    from test_pdl_order import GLOBAL, HOST_TABLES, _body
    from thompiler.emitter import read_sidecar
    from thompiler.families.tuning import TUNING
    monkeypatch.setattr(TUNING, "linear_kernel", kernel)
    d = (synth.qk_norm_rope_package(tmp_path, 2, 64, 4, 2, 128, values=True) if kernel == "heads" else
         synth.linear_package(tmp_path, 16, 512, 512, bias=True, residual=True))
    ptx = compile_kernel(load.load(str(_ir(d))))
    assert kernel in (read_sidecar(ptx) or {})["family"] and read_sidecar(ptx)["pdl"] is True
    lines = [ln.strip() for ln in _body(ptx)]
    # the tables that the host writes in stream order, by name or through a register that points into one
    tables = (*HOST_TABLES, *(f"[{m[1]}+" for ln in lines if (m := re.match(r"mov\.u64 (%\w+), thc_tmap_ptr;", ln))))
    generic = next(i for i, ln in enumerate(lines) if "generic lowering of the same IR" in ln)
    assert next(ln for ln in lines[generic + 1:] if ln and not ln.startswith("//")) == "griddepcontrol.wait;"
    # no load whose data would have to be constant while the previous kernel still writes
    assert not [ln for ln in lines if "ld.global.nc" in ln and not any(x in ln for x in tables)]
    lines = lines[:generic]
    at = lambda text: [i for i, ln in enumerate(lines) if text in ln]        # noqa: E731
    waits, first = at("griddepcontrol.wait"), at("griddepcontrol.wait")[0]
    for ln in lines[:first]:
        # prefetches into L2 read nothing; a refused launch only records its error
        assert (not GLOBAL.match(ln) or any(x in ln for x in tables) or "atom.global.or.b32" in ln
                or "prefetch.global.L2" in ln), ln
    if kernel == "rows":
        (alloc,), (trigger,) = at("tcgen05.alloc"), at("griddepcontrol.launch_dependents")
        assert len(waits) == 2 and waits[0] < alloc < trigger
        assert not any("$L_" in ln and ln.endswith(":") for ln in lines[waits[-1]:alloc])     # one straight piece
        assert waits[-1] < alloc


# ---- storage types -----------------------------------------------------------------------

def test_bf16_bits_round_to_nearest_even():
    torch = pytest.importorskip("torch")
    x = np.random.default_rng(1).standard_normal(4096).astype(np.float32)
    x[:9] = [0.0, -0.0, np.inf, -np.inf, 1.00390625, 1.01171875, 3.4e38, 1e-40, 65535.0]
    bits = problems.to_bf16(x)
    want = torch.from_numpy(x).bfloat16().view(torch.int16).numpy().view(np.uint16)
    assert np.array_equal(bits, want)
    assert np.isnan(problems.from_bf16(problems.to_bf16(np.float32([np.nan]))))[0]
    assert np.array_equal(problems.from_bf16(bits), torch.from_numpy(x).bfloat16().float().numpy())


# ---- rotary tables -------------------------------------------------------------------------

def test_rotary_tables_plain_and_far():
    cos, sin = rotary.tables(131073, 64)
    assert cos.dtype == sin.dtype == np.float32 and cos.shape == (131073, 32)
    from math import cos as c, sin as s
    for p in (0, 1, 4095, 65535, 65536, 131072):
        for i in (0, 1, 17, 31):
            a = p * 10000.0 ** (-2 * i / 64)
            assert abs(cos[p, i] - c(a)) <= 2.0 ** -24 and abs(sin[p, i] - s(a)) <= 2.0 ** -24


def test_rotary_scalings():
    R, base, f = 128, 10000.0, 4.0
    plain = rotary.frequencies(R)
    assert np.allclose(rotary.frequencies(R, scaling="linear", factor=f), plain / f, rtol=1e-15)
    ntk = rotary.frequencies(R, scaling="ntk", factor=f)
    assert ntk[0] == 1.0 and np.isclose(ntk[-1], plain[-1] / f, rtol=1e-12)
    parts = rotary.frequencies(R, scaling="parts", factor=f, original=4096, fast=32, slow=1)
    turns = 4096 * plain / (2 * np.pi)
    assert np.array_equal(parts[turns > 32], plain[turns > 32])
    assert np.allclose(parts[turns < 1], plain[turns < 1] / f, rtol=1e-15)
    mid = (turns >= 1) & (turns <= 32)
    g = (turns[mid] - 1) / 31
    assert mid.any() and np.allclose(parts[mid], plain[mid] * ((1 - g) / f + g), rtol=1e-15)
    cos, _ = rotary.tables(4, R, scaling="parts", factor=f, original=4096, scale=1.25)
    assert np.all(cos[0] == np.float32(1.25))


@pytest.mark.parametrize("kw", [dict(rotary=7), dict(rotary=0), dict(rotary=8, scaling="dynamic"),
                                dict(rotary=8, scaling="parts", factor=2.0), dict(rotary=8, factor=0.5),
                                dict(rotary=8, base=0.0),
                                dict(rotary=8, scaling="parts", original=64, fast=1.0, slow=2.0)])
def test_rotary_refusals(kw):
    with pytest.raises(ValueError):
        rotary.frequencies(**kw)
    with pytest.raises(ValueError):
        rotary.tables(0, 8)


@pytest.mark.parametrize("index,tuned", [
    (("col",), True), (("col<72",), True), (("col<16",), False), (("col<72", 72), True), (("col<16", 72), False),
    (("row<40", "col<72"), True), (("row<8", "col"), False), (("row", "col<64"), False), (("col", "row"), False)], ids=str)
def test_epilogue_index_is_taken_for_what_it_is(tmp_path, index, tuned):
    """An epilogue's load that is clamped short of C's sizes reads other elements than the row's and column's
    own: the tuned kernels leave it to the generic lowering."""
    from thompiler import schedules
    from thompiler.emitter import read_sidecar
    M, N, K = 40, 72, 64
    V, L, f32 = schedules.V, schedules.L, schedules.F32T

    def at(t):
        name, _, n = t.partition("<")
        return schedules.clamped(V(name), int(n)) if n else V(name)
    if len(index) == 2 and isinstance(index[1], int):
        idx, shape = (schedules.B("+", at(index[0]), L(index[1])),), (2 * N,)
    else:
        idx, shape = tuple(at(t) for t in index), (N,) if len(index) == 1 else (M, N)
    epi = ir.Lambda(("z", "row", "col"), (ir.Load(("e",), "extra", idx, f32),
                                                    schedules.assign("y", "add", "z", "e")), ("y",))
    inputs = {"x": ((M, K), "f16", None), "w": ((N, K), "f16", None), "extra": (shape, "f32", None)}
    d = synth._layer_write(tmp_path, "extra", "extra", "k_linear", schedules.linear_body(M, N, K, "f16", False, epi),
                           inputs, {"linear": ((M, N), "f32", None)}, 8, 128, 2e-2, 2e-3, smem=2 * 64 * 64 * 2)
    side = read_sidecar(compile_kernel(load.load(str(_ir(d))))) or {}
    assert ("linear" in side.get("family", "")) == tuned


@pytest.mark.parametrize("act", ["relu", "silu", "gelu_tanh"])
def test_activations_keep_nan(tmp_path, act):
    """A NaN in x reaches its row of the result through every activation, and no other row."""
    d = synth.linear_package(tmp_path, 3, 72, 64, activation=act)
    x = problems.make_inputs(problems.load_package(d))
    x["x"][1, 5] = np.nan
    got = oracle_run(d, x)["linear"]
    assert np.isnan(got[1]).all() and np.isfinite(got[[0, 2]]).all()


@pytest.mark.parametrize("case,cut", TAILS, ids=str)
def test_cut_tails_cover_every_column_once(tmp_path, monkeypatch, case, cut):
    """The units of a cut tail are C's columns after the whole tiles, each once, and nothing in the kernel's
    index arithmetic divides by a count that the cut made zero."""
    from thompiler.families.linear import LinearPair, Product
    from thompiler.families.matmul_pair import PM
    from thompiler.families.tuning import TUNING
    monkeypatch.setattr(TUNING, "linear_kernel", "pair")
    k = load.load(str(_ir(synth.linear_package(tmp_path, *case))))
    f = LinearPair(Product.read(k))
    M, N = case[:2]
    strips, halves, width = cut
    assert (f.strips if strips >= 0 else -1, f.hrem, f.tail_cols) == cut and f.tiles_m == -(-M // PM)
    if strips >= 0:
        per_row = (f.units - f.full_tiles) // f.tiles_m
        assert f.full_tiles == strips * f.tiles_m and f.units == f.full_tiles + per_row * f.tiles_m
        left = N - strips * f.tile_cols
        assert (per_row - 1) * f.tail_out() < left <= per_row * f.tail_out()
    else:
        assert f.full_tiles + halves == f.tiles_m * -(-N // f.tile_cols) and f.units == f.full_tiles + 2 * halves
        assert 2 * f.tail_out() == f.tile_cols
    assert f.HN % f.b_box == 0 and (f.tail_cols // 2) % f.b_box == 0
    ptx = compile_kernel(k)
    assert "tcgen05-linear-pair" in ptx and not re.findall(r"\b(?:div|rem)\.u32 [^;]*, 0;", ptx)
