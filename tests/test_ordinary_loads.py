"""Loads of a kernel that may begin while the one before it still writes (programmatic dependent
launch).  ``ld.global.nc`` promises data that is constant for the kernel's lifetime, and the assembler
may move such a load above griddepcontrol.wait: a module with that wait has none, but for the
tensor-map tables that the host alone writes and a body that only ordinary launches reach."""

import re

import pytest

from conftest import GOLDEN
from thompiler import load, synth
from thompiler.compiler import compile_kernel
from thompiler.emitter import read_sidecar

CASES = [
    ("softmax", lambda d: synth.row_package(d, "softmax", 256, 4096)),
    ("rmsnorm", lambda d: synth.row_package(d, "rmsnorm", 64, 1024)),
    ("l2norm", lambda d: synth.row_package(d, "l2norm", 64, 128)),
    ("rowsum", lambda d: synth.row_package(d, "rowsum", 64, 1024)),
    ("sum", lambda d: synth.sum_package(d, 1 << 20)),
    ("mean", lambda d: GOLDEN / "r03_mean"),
    ("matmul pair", lambda d: synth.matmul_package(d, 1024, 1024, 512)),
    ("matmul", lambda d: synth.matmul_package(d, 384, 320, 512)),
    ("attention", lambda d: synth.attention_package(d, 1, 2, 512, 128)),
    ("f32 matmul", lambda d: GOLDEN / "m01_matmul_512"),
    ("linear", lambda d: synth.linear_package(d, 40, 512, 512, bias=True)),
    ("rope", lambda d: synth.rope_package(d, 2, 64, 4, 2, 128)),
]


def _ptx(d) -> str:
    return compile_kernel(load.load(str(sorted(d.glob("*.ir.json"))[0])))


def _constant_loads(ptx: str) -> list[str]:
    """The ld.global.nc of anything but the tensor-map tables (by name, or through a register that points
    into one)."""
    lines = [ln.strip() for ln in ptx.splitlines()]
    tables = ["thc_tmap_ptr"] + [f"[{m[1]}+" for ln in lines if (m := re.match(r"mov\.u64 (%\w+), thc_tmap_ptr;", ln))]
    return [ln for ln in lines if re.search(r"\bld\.global\.nc\b", ln) and not any(x in ln for x in tables)]


@pytest.mark.parametrize("name,make", CASES, ids=[c[0] for c in CASES])
def test_overlapping_kernels_read_with_ordinary_loads(tmp_path, name, make):
    ptx = _ptx(make(tmp_path / "p"))
    assert "griddepcontrol.wait" in ptx and read_sidecar(ptx)["pdl"] is True
    assert not _constant_loads(ptx)


@pytest.mark.parametrize("make", [lambda d: synth.pointwise_package(d, 1 << 20, "relu_mul"),
                                  lambda d: synth.pointwise_package(d, 1 << 20, "add"),
                                  lambda d: GOLDEN / "p02_scale_shift", lambda d: GOLDEN / "p01_vector_add"],
                         ids=["relu_mul", "add", "p02", "p01"])
def test_pointwise_launch_that_overlaps_has_a_body_of_its_own(tmp_path, make):
    """The recorded launch (a CTA more than meta.json's) takes the body with ordinary loads; meta.json's takes
    the other one, and is not launched to overlap."""
    from thompiler import runner
    d = make(tmp_path / "p")
    info = load.load(str(sorted(d.glob("*.ir.json"))[0]))
    ptx = compile_kernel(info)
    side = read_sidecar(ptx)
    assert "family: pointwise-vector" in ptx
    grid = info.grid[0]
    assert side["grid"] == [grid + 1, 1, 1] and side["block"] == list(info.block) and side["pdl"] is True
    m = re.search(rf"mov\.u32 (%r\d+), %nctaid\.x;\s*setp\.ne\.u32 (%p\d+), \1, {grid + 1};\s*griddepcontrol\.wait;\s*"
                  r"@\2 bra (\$\w+);", ptx)
    own, _, rest = ptx[m.end():].partition(f"{m[3]}:")
    meta, _, generic = rest.partition("generic lowering of the same IR")
    assert "ld.global." in own and not _constant_loads(own) and not _constant_loads(generic)
    assert _constant_loads(meta)

    class Module:
        sidecar = side
    kmeta = {"grid": list(info.grid), "block": list(info.block), "smem_bytes": info.dynamic_smem_bytes}
    assert runner.plan_launch(Module, kmeta).pdl and not runner.plan_launch(Module, kmeta, honour_meta=True).pdl
