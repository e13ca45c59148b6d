"""Linear products whose package is launched with a grid that clusters do not divide, under their own
launch and meta.json's, against the float64 product."""

import pytest

from test_linear_guards import _package
from thompiler.device import DeviceKernel

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
