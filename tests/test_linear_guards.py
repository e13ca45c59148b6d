"""What the fused linear product's kernels refuse by themselves, on the CPU: operands off the 16-byte
boundary that their copies need, whatever meta.json says of alignment, and launch geometries that the
package's own does not allow."""

import json
import re
from types import SimpleNamespace

import pytest

from thompiler import ir, load, runner, schedules, synth
from thompiler.compiler import compile_kernel
from thompiler.emitter import read_sidecar
from thompiler.families.tuning import TUNING

KERNELS = ("stream", "rows", "split", "pair")


def _package(out, M, N, K, grid, epilogue=None, inputs=None):
    """A linear product without ``align`` records, launched with ``grid`` CTAs by meta.json."""
    return synth._layer_write(out, "linear", "linear", "k_linear",
                              schedules.linear_body(M, N, K, "f16", False, epilogue),
                              {"x": ((M, K), "f16", None), "w": ((N, K), "f16", None), **(inputs or {})},
                              {"linear": ((M, N), "f16", None)}, grid, 128, 2e-2, 2e-3, smem=2 * 64 * 64 * 2)


def _info(d):
    return load.load(str(next(d.glob("*.ir.json"))))


def _extra(M, N):
    """An epilogue that adds a vector over the columns, and its input."""
    epi = ir.Lambda(("z", "row", "col"), (ir.Load(("e",), "extra", (schedules.clamped(ir.Var("col"), N),), schedules.F32T),
                                          schedules.assign("y", "add", "z", "e")), ("y",))
    return epi, {"extra": ((N,), "f32", None)}


@pytest.mark.parametrize("kernel", KERNELS)
def test_kernel_checks_its_operands(tmp_path, monkeypatch, kernel):
    """Before any branch to a path that copies from them, x and w are tested and sent to the refusal."""
    monkeypatch.setattr(TUNING, "linear_kernel", kernel)
    ptx = compile_kernel(_info(_package(tmp_path / "p", 16, 512, 512, 64)))
    assert read_sidecar(ptx)["family"].endswith("linear-" + kernel)
    body = ptx[ptx.index(".entry"):]
    to = set()
    for name in ("x", "w"):
        m = re.search(rf"and\.b64 (%rd\d+), %g_{name}, 15;\s*setp\.ne\.u64 (%p\d+), \1, 0;\s*@\2 bra (\$\w+);", body)
        assert m, name
        assert not re.search(r"\bbra\b|cp\.async|ld\.global", body[:m.start()].replace(f"bra {m[3]}", ""))
        to.add(m[3])
    (bad,) = to
    assert re.match(r"\s*(griddepcontrol\.wait;\s*)?mov\.u64 %rd\d+, thc_error;\s*atom\.global\.or\.b32 %r\d+, \[%rd\d+\], 16;\s*ret;",
                    body[body.index(bad + ":") + len(bad) + 1:])


@pytest.mark.parametrize("kernel", KERNELS)
def test_call_is_refused_without_align_in_meta(tmp_path, monkeypatch, kernel):
    """The launch record carries the boundaries: ``Launch`` refuses before anything is issued."""
    if not runner.LIB_PATH.exists():
        pytest.skip("runner library not built")
    monkeypatch.setattr(TUNING, "linear_kernel", kernel)
    epi, more = _extra(16, 512)
    d = _package(tmp_path / "p", 16, 512, 512, 64, epi, more)
    kmeta = json.loads((d / "meta.json").read_text())["kernels"][0]
    assert not any("align" in a for a in kmeta["args"])
    side = read_sidecar(compile_kernel(_info(d)))
    plan = runner.plan_launch(SimpleNamespace(sidecar=side), kmeta)
    plan.tmaps = []
    wide = {"x", "w"} | ({"extra", "linear"} if kernel in ("split", "pair") else set())
    assert {n for n, a in plan.align.items() if a == 16} == wide
    k = runner.Launch(SimpleNamespace(handle=1, name="k_linear", module=SimpleNamespace(handle=0)), plan, kmeta, None)
    good = {n: 4096 * (i + 1) for i, n in enumerate(kmeta["arg_order"])}
    for name in wide:
        with pytest.raises(runner.RunnerError, match=f"buffer '{name}' .* not 16-byte aligned") as e:
            k(dict(good, **{name: good[name] + 8}))
        assert e.value.stage == "request"


@pytest.mark.parametrize("kernel", ["", *KERNELS])
@pytest.mark.parametrize("M,N,K,grid", [(40, 72, 4096, 2), (130, 72, 4096, 6), (40, 200, 8192, 4), (300, 200, 2048, 20),
                                        (64, 64, 4096, 1), (300, 64, 4096, 5), (2048, 576, 512, 288), (600, 960, 512, 150)])
def test_clusters_divide_metas_grid(tmp_path, monkeypatch, kernel, M, N, K, grid):
    """A cluster's shape belongs to the entry, so meta.json's launch runs in it too."""
    monkeypatch.setattr(TUNING, "linear_kernel", kernel)
    ptx = compile_kernel(_info(_package(tmp_path / "p", M, N, K, grid)))
    shapes = [int(x) for x in re.findall(r"\.reqnctapercluster (\d+)", ptx)]
    assert all(grid % s == 0 for s in shapes), shapes
    side = read_sidecar(ptx) or {}
    assert side.get("cluster", [1])[0] in (shapes or [1])
    if not shapes and M > 24:                             # neither a cluster's kernel nor the one for a handful of rows
        assert "linear-rows" in side["family"] if "family" in side else "griddepcontrol" not in ptx


@pytest.mark.parametrize("kernel", ["", *KERNELS])
@pytest.mark.parametrize("M,N,K,more", [(16, 64, 16 << 20, {}), (256, 64, 5 << 20, {}), (1, 64, 1 << 27, {}),
                                        (20, 16, 1 << 28, {}), (3, 64, 1 << 26, dict(gated=True)), (200, 64, 4 << 20, {}),
                                        (1, 1 << 30, 8, dict(residual=True, out_dtype="f32"))], ids=str)
def test_offsets_fit_their_fields(tmp_path, monkeypatch, kernel, M, N, K, more):
    """Immediate offsets of addresses are signed 32-bit numbers, and so fit the operands of 32-bit
    instructions, at the longest rows too."""
    monkeypatch.setattr(TUNING, "linear_kernel", kernel)
    ptx = compile_kernel(_info(synth.linear_package(tmp_path / "p", M, N, K, **more)))
    side = read_sidecar(ptx) or {}
    assert "linear" in side.get("family", "") or K > 64 << 20
    # a wait lasts about a second: no CTA-pair tile of more than 2^20 K blocks
    assert K <= 64 << 20 or side.get("cluster", [1])[0] == 1
    assert max(int(x) for x in re.findall(r"\+(\d+)\]", ptx)) < 2 ** 31
    for op, n in re.findall(r"\t(?:@!?%p\d+ )?(\w+\.[\w.]*(?:u32|s32|b32)) [^;]*?, (\d+)(?:, %\w+)?;", ptx):
        assert int(n) < 2 ** 32, (op, n)


def test_wide_f32_rows_of_an_epilogue(tmp_path, monkeypatch):
    """An f32 array of C's shape whose rows are 4 GB: its row pitch is no 32-bit number."""
    monkeypatch.setattr(TUNING, "linear_kernel", "pair")
    M, N = 2, 1 << 30
    epi = ir.Lambda(("z", "row", "col"), (ir.Load(("e",), "extra", (schedules.clamped(ir.Var("row"), M), ir.Var("col")),
                                                  schedules.F32T), schedules.assign("y", "add", "z", "e")), ("y",))
    ptx = compile_kernel(_info(_package(tmp_path / "p", M, N, 8, 1 << 24, epi, {"extra": ((M, N), "f32", None)})))
    tuned = ptx[:ptx.index("generic lowering of the same IR")]
    assert "tcgen05-linear-pair" in ptx and not re.search(rf"\.u32 [^;]*\b{4 * N};", tuned)


@pytest.mark.parametrize("kernel", [*KERNELS, "heads"])
def test_a_refused_launch_waits_for_the_previous_kernel(tmp_path, monkeypatch, kernel):
    """A kernel behind a refused launch waits for that launch alone; were it to end at once, the kernel behind
    it would run beside the one before it."""
    monkeypatch.setattr(TUNING, "linear_kernel", kernel)
    ptx = compile_kernel(_info(synth.rope_package(tmp_path / "p", 2, 64, 4, 2, 128) if kernel == "heads" else
                               synth.linear_package(tmp_path / "p", 16, 512, 512)))
    lines = [ln.strip() for ln in ptx.splitlines()]
    records = [i for i, ln in enumerate(lines) if "atom.global.or.b32" in ln and ln.endswith(", 16;")
               and lines[i + 1] == "ret;"]
    assert records
    for i in records:
        start = max(j for j in range(i) if lines[j].endswith(":"))
        assert lines[start + 1] == "griddepcontrol.wait;", lines[start:i + 1]
