"""SnapshotGraph.quantized_features: what its calls leave behind on the host, with the device's queue played by a list."""
import threading
import time

import pytest
import torch

import ogl_amd  # noqa: F401
from ogl_amd import ops as real_ops
from ogl_amd.graph import snapshot_graph
from ogl_amd.graph.snapshot_graph import SnapshotGraph

N, WIDTH = 12, 40


class Device:
    """Launches queue up until the host waits for the stream that they are on."""

    def __init__(self, monkeypatch):
        self.queued, self.written, self.capturing = [], [], False
        dev = self

        class Ops:
            QuantRows = real_ops.QuantRows

            @staticmethod
            def quant_rows(n, width, **kw):
                time.sleep(0.02)                                        # (another thread gets its turn here)
                dev.queued += ["zeros"] * (n > 0)
                return real_ops.quant_rows(n, width, device="cpu")

            @staticmethod
            def quant_rows_write(rows, x, start=0):
                dev.queued.append((start, start + x.shape[0]))
                time.sleep(0.02)

        class Stream:
            def synchronize(self):
                dev.written += dev.queued
                dev.queued.clear()

            def __eq__(self, other):
                return True

        class On:
            def __init__(self, device):
                pass

            def __enter__(self):
                pass

            def __exit__(self, *exc):
                return False

        monkeypatch.setattr(snapshot_graph, "ops", Ops)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: dev.capturing)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
        monkeypatch.setattr(torch.cuda, "device", On)


def graph(present=N):
    g = SnapshotGraph.__new__(SnapshotGraph)
    g.device, g.n_total, g.n_present = torch.device("cpu"), N, present
    g.feat_table = torch.zeros(N, WIDTH)
    g._quantized = snapshot_graph._QuantizedFeatures()
    return g


def view(other, present):
    g = graph(present)
    g.feat_table, g._quantized = other.feat_table, other._quantized
    return g


def test_rows_are_written_before_anyone_is_told(monkeypatch):
    """A caller on another stream finds the rows counted as written and adds nothing: they have to be there by then, not queued behind this stream."""
    dev = Device(monkeypatch)
    g = graph(5)
    assert g.quantized_features().n == 5
    assert dev.queued == [] and dev.written == ["zeros", (0, 5)]
    other = view(g, N)
    assert other.quantized_features().n == N
    assert dev.queued == [] and dev.written == ["zeros", (0, 5), (5, N)]
    g.quantized_features(), other.quantized_features()
    assert dev.queued == [] and len(dev.written) == 3                    # (nothing is written twice)


def test_a_table_without_rows_yet(monkeypatch):
    """Its zero fill must not reach the device behind rows that another stream writes."""
    dev = Device(monkeypatch)
    g = graph(0)
    assert g.quantized_features().n == 0 and dev.queued == []
    assert view(g, 3).quantized_features().n == 3 and dev.queued == []


def test_two_threads_make_one_table(monkeypatch):
    dev = Device(monkeypatch)
    g = graph()
    other, got = view(g, N), [None, None]

    def call(i, v):
        got[i] = v.quantized_features()
    threads = [threading.Thread(target=call, args=a) for a in enumerate((g, other))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert dev.written == ["zeros", (0, N)] and got[0].codes.data_ptr() == got[1].codes.data_ptr()


@pytest.mark.parametrize("present", [0, 5])
def test_a_first_call_inside_a_capture_keeps_nothing(monkeypatch, present):
    """A table allocated there would live in the graph's memory, its zero fill a node of the graph: cleared again at every replay."""
    dev = Device(monkeypatch)
    dev.capturing = True
    g = graph(present)
    if present:
        with pytest.raises(RuntimeError, match="before the capture"):
            g.quantized_features()
    else:
        assert g.quantized_features().n == 0
    assert g._quantized.rows is None and g._quantized.written == 0 and (0, present) not in dev.queued
    dev.capturing = False
    dev.queued.clear()
    assert view(g, N).quantized_features().n == N and dev.written == ["zeros", (0, N)]
    dev.capturing = True
    assert g.quantized_features().n == present and dev.queued == []
    g.n_present = N
    assert g.quantized_features().n == N
