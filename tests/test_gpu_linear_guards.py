"""Linear products whose package is launched with a grid that clusters do not divide, under their own
launch and meta.json's, against the float64 product; products of very long rows, and of very many columns."""

import pytest

from test_linear_guards import _package
from thompiler import synth
from thompiler.device import DeviceKernel
from thompiler.families.tuning import TUNING

pytestmark = pytest.mark.gpu


def _bound(x, w):
    """K f32 additions, then one rounding to f16 (half a step, or half the smallest subnormal)."""
    x, w = x.double(), w.double()
    want = x @ w.t()
    return want, x.shape[1] * 2.0 ** -24 * (x.abs() @ w.abs().t()) + 2.0 ** -11 * want.abs() + 2.0 ** -25


@pytest.mark.parametrize("meta", [False, True], ids=["own", "meta"])
@pytest.mark.parametrize("M,N,K,grid", [(40, 72, 4096, 2), (130, 72, 512, 6), (300, 64, 1024, 5), (300, 200, 2048, 20),
                                        (64, 64, 264, 1), (3000, 64, 512, 47)])
def test_any_grid_of_metas(tmp_path, M, N, K, grid, meta):
    import torch
    k = DeviceKernel(next(_package(tmp_path / "p", M, N, K, grid).glob("*.ir.json")), honour_meta=meta)
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn(M, K, device="cuda", generator=g).half()
    w = (torch.randn(N, K, device="cuda", generator=g) * K ** -0.5).half()
    y = torch.full((M, N), float("nan"), device="cuda", dtype=torch.float16)
    k({"x": x.data_ptr(), "w": w.data_ptr(), "linear": y.data_ptr()}, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want, allowed = _bound(x, w)
    assert ((y.double() - want).abs() <= allowed).all()
    assert k.error_word() == 0
    k.close()


@pytest.mark.parametrize("M,N,K,kernel", [(16, 64, 16 << 20, ""), (16, 64, 16 << 20, "pair"), (1, 24, 16 << 20, ""),
                                          (256, 64, (5 << 20) + 8, "")])
def test_long_rows(tmp_path, monkeypatch, M, N, K, kernel):
    """Rows past the reach of an address' immediate offset.  Entries of -1, 0 and 1: about 4 K / 9 products, fewer
    than 2^24, are not zero, so f32 holds every partial sum exactly, whatever the order."""
    import torch
    monkeypatch.setattr(TUNING, "linear_kernel", kernel)
    k = DeviceKernel(next(synth.linear_package(tmp_path / "p", M, N, K, out_dtype="f32").glob("*.ir.json")))
    g = torch.Generator(device="cuda").manual_seed(K + M)

    def entries(rows):
        return torch.randint(-1, 2, (rows, K), device="cuda", generator=g, dtype=torch.int8).half()
    x, w = entries(M), entries(N)
    y = torch.full((M, N), float("nan"), device="cuda")
    k({"x": x.data_ptr(), "w": w.data_ptr(), "linear": y.data_ptr()}, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = torch.zeros(M, N, device="cuda", dtype=torch.float64)
    for at in range(0, K, 1 << 20):
        want += x[:, at:at + (1 << 20)].double() @ w[:, at:at + (1 << 20)].double().t()
    assert torch.equal(y.double(), want)
    assert k.error_word() == 0
    k.close()


@pytest.mark.parametrize("M,N,K", [(1, 50264, 264), (25, 50264, 264), (64, 128256, 64), (300, 37904, 72)])
def test_many_columns(tmp_path, M, N, K):
    """The widths of an output head, past the columns that the kernel for few rows takes."""
    import torch
    k = DeviceKernel(next(synth.linear_package(tmp_path / "p", M, N, K).glob("*.ir.json")))
    g = torch.Generator(device="cuda").manual_seed(N)
    x = torch.randn(M, K, device="cuda", generator=g).half()
    w = (torch.randn(N, K, device="cuda", generator=g) * K ** -0.5).half()
    y = torch.full((M, N), float("nan"), device="cuda", dtype=torch.float16)
    k({"x": x.data_ptr(), "w": w.data_ptr(), "linear": y.data_ptr()}, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want, allowed = _bound(x, w)
    assert ((y.double() - want).abs() <= allowed).all()
    assert k.error_word() == 0
    k.close()
