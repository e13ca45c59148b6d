"""Kernels launched to overlap a fused linear product read what it wrote, eagerly and in a CUDA graph:
every intermediate holds NaN before each pass, and each pass gives the bits of the same calls made
one by one, with a synchronisation after each."""

import pytest

from conftest import GOLDEN
from thompiler import synth
from thompiler.device import DeviceKernel
from thompiler.families.tuning import TUNING

pytestmark = pytest.mark.gpu


def _kernel(d):
    k = DeviceKernel(sorted(d.glob("*.ir.json"))[0])
    assert k.plan.pdl
    return k


@pytest.mark.parametrize("linear", ["stream", "rows", "split", "pair"])
@pytest.mark.parametrize("cols", [512, 1024, 4096])
def test_norms_and_pointwise_after_a_linear_product(tmp_path, monkeypatch, linear, cols):
    import torch
    monkeypatch.setattr(TUNING, "linear_kernel", linear)
    M, K, layers = 16, 512, 24
    lin = _kernel(synth.linear_package(tmp_path / "l", M, cols, K, out_dtype="f32"))
    assert lin.family.endswith("linear-" + linear)
    rms = _kernel(synth.row_package(tmp_path / "r", "rmsnorm", M, cols))
    soft = _kernel(synth.row_package(tmp_path / "s", "softmax", M, cols))
    l2 = _kernel(synth.row_package(tmp_path / "n", "l2norm", M, cols))
    add = _kernel(synth.pointwise_package(tmp_path / "p", M * cols, "add"))
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(M, K, device="cuda", generator=g).half()
    w = [(torch.randn(cols, K, device="cuda", generator=g) * K ** -0.5).half() for _ in range(layers)]
    scale = torch.rand(cols, device="cuda", generator=g) + 0.5
    count, eps = torch.tensor([float(cols)], device="cuda"), torch.tensor([1e-6], device="cuda")
    buf = [[torch.empty(M, cols, device="cuda") for _ in range(6)] for _ in w]

    def chain(sync=False):
        s = torch.cuda.current_stream().cuda_stream
        for wi, (y, a, b, c, d, e) in zip(w, buf):
            for k, p in ((lin, dict(x=x, w=wi, linear=y)), (rms, dict(mean_count=count, add_c1=eps, x=y, w=scale, mul_1=a)),
                         (soft, dict(x=a, softmax=b)), (l2, dict(x=a, div=c)), (add, dict(x0=b, x1=c, add=d)),
                         (add, dict(x0=d, x1=y, add=e))):
                k({n: t.data_ptr() for n, t in p.items()}, s)
                if sync:
                    torch.cuda.synchronize()

    flat = [t for row in buf for t in row]
    chain(sync=True)
    refs = [t.clone() for t in flat]
    assert all(torch.isfinite(r).all() for r in refs)
    want = buf[0][0].double()
    want = want * torch.rsqrt((want * want).mean(-1, keepdim=True) + 1e-6) * scale.double()
    # f32 sums of ``cols`` squares: relative error at most cols 2^-24, half of it after the root; then a few roundings
    assert ((buf[0][1].double() - want).abs() <= (cols * 2.0 ** -25 + 2.0 ** -20) * want.abs()).all()

    def check(run):
        for t in flat:
            t.fill_(float("nan"))
        run()
        torch.cuda.synchronize()
        for i, (t, r) in enumerate(zip(flat, refs)):
            assert torch.equal(t, r), f"layer {i // 6}, buffer {i % 6}"
    check(chain)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain()
    for _ in range(20):
        check(graph.replay)
    assert lin.error_word() == 0
    del graph
    for k in (lin, rms, soft, l2, add):
        k.close()


def test_f32_matmul_after_a_linear_product(tmp_path):
    import torch
    lin = _kernel(synth.linear_package(tmp_path / "l", 512, 512, 256, out_dtype="f32"))
    mm = _kernel(GOLDEN / "m01_matmul_512")
    assert mm.family == "simt-matmul-f32"
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(512, 256, device="cuda", generator=g).half()
    w = [(torch.randn(512, 256, device="cuda", generator=g) / 16).half() for _ in range(8)]
    buf = [[torch.empty(512, 512, device="cuda") for _ in range(2)] for _ in w]

    def chain(sync=False):
        s = torch.cuda.current_stream().cuda_stream
        for wi, (y, z) in zip(w, buf):
            lin({"x": x.data_ptr(), "w": wi.data_ptr(), "linear": y.data_ptr()}, s)
            if sync:
                torch.cuda.synchronize()
            mm({"x0": y.data_ptr(), "x1": y.data_ptr(), "matmul": z.data_ptr()}, s)
            if sync:
                torch.cuda.synchronize()

    flat = [t for row in buf for t in row]
    chain(sync=True)
    refs = [t.clone() for t in flat]
    y = buf[0][0].double()
    assert ((buf[0][1].double() - y @ y).abs() <= 512 * 2.0 ** -24 * (y.abs() @ y.abs())).all()    # 512 f32 additions
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain()
    for run in (chain, *[graph.replay] * 20):
        for t in flat:
            t.fill_(float("nan"))
        run()
        torch.cuda.synchronize()
        assert all(torch.equal(t, r) for t, r in zip(flat, refs))
    del graph
    lin.close()
    mm.close()
