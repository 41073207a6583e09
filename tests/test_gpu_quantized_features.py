"""The feature cache in 8 bits (SnapshotGraph.quantized_features) from more than one stream."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import ogl_amd  # noqa: F401
    from ogl_amd import ops as _ops
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return _ops


def toy():
    from ogl_amd import synthetic
    _, _, dyn, _, _ = synthetic.load("toy", device="cuda")
    for _ in range(8):
        dyn.evolve()
    return dyn.get_graph()


def test_two_streams_share_the_table(ops):
    """Rows added on a stream with work in front of them, read at once on another that does not wait for it, from another view; and the other way round."""
    from ogl_amd.graph.snapshot_graph import SnapshotGraph
    g = toy()
    n, cut = g.n_present, g.cut
    want = ops.quantize_rows(g.feat_table)
    view, side = SnapshotGraph.shared(g), torch.cuda.Stream()
    work = torch.randn(2048, 2048, device="cuda")
    torch.cuda.synchronize()
    for present, writer, reader in ((n // 3, side, torch.cuda.current_stream()), (n, torch.cuda.current_stream(), side)):
        for v in (g, view):
            v.set_snapshot(present, min(cut, present))
        torch.cuda.synchronize()
        with torch.cuda.stream(writer):
            busy = work
            for _ in range(8):
                busy = (busy @ work).clamp(-1, 1)
            g.quantized_features()
        with torch.cuda.stream(reader):
            q = view.quantized_features()
            codes, scales = q.codes.clone(), q.scales.clone()
        torch.cuda.synchronize()
        assert torch.equal(codes, want.codes[:present]) and torch.equal(scales, want.scales[:present])
        del busy


def test_captured_after_the_rows_are_there(ops):
    """A first call inside a capture is refused; after one outside it, the rows are read by every replay, with eager work in between."""
    g = toy()
    n, cut = g.n_present, g.cut
    at = torch.arange(0, n, 2, device="cuda")
    x = torch.zeros(n, 8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):                                           # (it records the caller's own work all the same)
        with pytest.raises(RuntimeError, match="before the capture"):
            g.quantized_features()
        y = x + 1
    graph.replay()
    want = ops.quant_rows_read(g.quantized_features(), at)
    graph.replay()
    assert torch.equal(ops.quant_rows_read(g.quantized_features(), at), want) and float(want.abs().max()) > 0
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        z = ops.quant_rows_read(g.quantized_features(), at)
    for step in range(3):
        z.zero_()
        second.replay()
        graph.replay()
        assert torch.equal(z, want) and (y == 1).all()
        assert torch.equal(ops.quant_rows_read(g.quantized_features(), at), want)
