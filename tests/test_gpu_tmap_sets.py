"""Which set of tensor maps a call on new buffers re-encodes.  A kernel takes the lowest set whose recorded
addresses are its parameters', and another stream may be rewriting a set meanwhile: a set is left alone while
its old addresses mixed with the new ones could make up the buffers of a launch in flight, and a launch in a
captured graph is in flight for as long as the graph lives."""

import pytest

from thompiler import runner, synth
from thompiler.device import DeviceKernel
from thompiler.families.kit import TMAP_SETS
from thompiler.families.tuning import TUNING

pytestmark = pytest.mark.gpu

M, N, K = 256, 128, 64


@pytest.fixture
def kernel(tmp_path):
    k = DeviceKernel(synth.matmul_package(tmp_path / "mm", M, N, K) / "k_matmul_f16.ir.json")
    assert k.module.sidecar["tmap_sets"] == TMAP_SETS
    yield k
    k.close()


def _buffers(count):
    import torch
    return [[torch.randn(*s, device="cuda", dtype=t) * 0.1 for s, t in (((M, K), torch.float16), ((N, K), torch.float16),
                                                                        ((M, N), torch.float32))] for _ in range(count)]


def _ptrs(a, b, c):
    return {"x0": a.data_ptr(), "x1": b.data_ptr(), "matmul": c.data_ptr()}


def _captured(k, t):
    """A graph with one launch on ``t``: its set is encoded, and its eager launch known to be over."""
    import torch
    k(_ptrs(*t), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    other = _buffers(1)[0]
    k(_ptrs(*other), torch.cuda.current_stream().cuda_stream)     # a bind that sees that launch's event done
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k(_ptrs(*t), torch.cuda.current_stream().cuda_stream)
    return graph, other


def test_a_graphs_buffers_are_not_mixed_up(kernel):
    import torch
    s = torch.cuda.current_stream().cuda_stream
    (a, b, c), *rest = _buffers(TMAP_SETS + 2)
    graph, other = _captured(kernel, (a, b, c))                      # sets 0 (the graph's) and 1
    a2, b2, c2 = rest[-1]
    first = kernel.tmaps.bind(_ptrs(a, b2, c), s)                    # the graph's a and c, another b
    torch.cuda.synchronize()
    kernel.tmaps.bind(_ptrs(*other), s)                              # used since: not the oldest
    used = {0, first, kernel.tmaps.bind(_ptrs(*other), s)}
    for t in rest[:TMAP_SETS - 3]:
        used.add(kernel.tmaps.bind(_ptrs(*t), s))
    torch.cuda.synchronize()
    assert used == set(range(TMAP_SETS))
    # on the way from (a, b2, c) to (a2, b, c2) that oldest set could read (a, b, c): not at the first such call
    # (which sees that the graph's set was last launched eagerly) nor at later ones
    for a3, _, c3 in rest[-3:]:
        assert kernel.tmaps.bind(_ptrs(a3, b, c3), s) not in (0, first)
        torch.cuda.synchronize()
    # with nothing of the graph's among the new addresses it is the one to go
    assert kernel.tmaps.bind(_ptrs(a2, b2, c2), s) == first
    torch.cuda.synchronize()
    c.fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    assert (c.double() - a.double() @ b.double().t()).abs().max().item() < 1e-4
    assert kernel.error_word() == 0
    del graph


def test_no_set_left_is_refused(kernel):
    """Every set but one pinned, that one open to the mix-up: the call is refused, and a call without it is not."""
    import torch
    s = torch.cuda.current_stream().cuda_stream
    bufs = _buffers(TMAP_SETS)
    for t in bufs[:-1]:
        kernel(_ptrs(*t), s)
    a, b, c = bufs[0]
    a2, b2, c2 = bufs[-1]
    kernel(_ptrs(a, b2, c), s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for t in bufs[:-1]:
            kernel(_ptrs(*t), torch.cuda.current_stream().cuda_stream)
    kernel(_ptrs(a, b2, c), s)
    torch.cuda.synchronize()
    with pytest.raises(runner.RunnerError, match="could alias one a captured graph reads"):
        kernel(_ptrs(a2, b, c2), s)
    kernel(_ptrs(a2, b2, c2), s)
    torch.cuda.synchronize()
    assert (c2.double() - a2.double() @ b2.double().t()).abs().max().item() < 1e-4
    for t in bufs[:-1]:
        t[2].fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in bufs[:-1]:
        assert (c.double() - a.double() @ b.double().t()).abs().max().item() < 1e-4
    assert kernel.error_word() == 0
    del graph


def test_threads_share_the_last_free_set(tmp_path, monkeypatch):
    """Graphs keep every set but one, and two threads call the kernel on buffers of their own, each on its own
    stream: a call's maps stay its own from their binding to its launch.  (A launch whose set is taken from it
    records bit 4 of the error word and writes nothing.)"""
    import threading

    import torch
    from thompiler.families.linear import LinearPair
    monkeypatch.setattr(TUNING, "linear_kernel", "pair")
    monkeypatch.setattr(LinearPair, "map_sets", 32)
    rows, cols, depth, calls = 64, 128, 64, 400
    k = DeviceKernel(next(synth.linear_package(tmp_path / "p", rows, cols, depth, out_dtype="f32").glob("*.ir.json")))
    assert k.family == "tcgen05-linear-pair" and k.module.sidecar["tmap_sets"] == 32

    def buffers(n):
        """Entries of -1, 0 and 1: exact sums."""
        draw = lambda *shape: torch.randint(-1, 2, (n, *shape), device="cuda").half()   # noqa: E731
        return draw(rows, depth), draw(cols, depth), torch.empty(n, rows, cols, device="cuda")

    def call(x, w, y, stream):
        k({"x": x.data_ptr(), "w": w.data_ptr(), "linear": y.data_ptr()}, stream)
    kept = list(zip(*buffers(31)))
    for t in kept:
        call(*t, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for t in kept:
            call(*t, torch.cuda.current_stream().cuda_stream)
    streams = [torch.cuda.Stream() for _ in range(2)]
    own = [buffers(calls) for _ in streams]
    own = [(x, w, y.fill_(float("nan"))) for x, w, y in own]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            for x, w, y in zip(*own[i]):
                call(x, w, y, streams[i].cuda_stream)
            streams[i].synchronize()
        except Exception as e:                                # noqa: BLE001 - reported by the test
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    assert k.error_word() == 0
    for x, w, y in own:
        assert torch.equal(y, x.float() @ w.float().transpose(1, 2))
    for x, w, y in kept:
        y.fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    for x, w, y in kept:
        assert torch.equal(y, x.float() @ w.float().t())
    del graph
    k.close()
