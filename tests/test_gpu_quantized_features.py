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
