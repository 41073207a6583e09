"""The row operators refuse what they cannot do, before anything reaches a GPU."""
import ctypes
import os
import re

import pytest
import torch

import ogl_amd  # noqa: F401
from ogl_amd import _lib, ops


def cache(n=4, width=40, group=None, fmt="int8"):
    return ops.quant_rows(n, width, group, fmt, device="cpu")


def test_header_symbols_exported_and_bound():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {}
    for header in ("ogl_hip.h", "ogl_rows.h"):
        src = re.sub(r"/\*.*?\*/", "", open(os.path.join(root, "include", header)).read(), flags=re.S)
        names[header] = set(re.findall(r"\b(ogl_[a-z0-9_]+)\s*\(", src))
    assert names["ogl_rows.h"] == set(_lib.ROW_SIGNATURES) and not names["ogl_rows.h"] & names["ogl_hip.h"]
    h = _lib.lib()
    for n in names["ogl_rows.h"]:
        assert getattr(h, n).argtypes == _lib.ROW_SIGNATURES[n][1]


def test_quant_rows_layout():
    c = cache(5, 130, 64)
    assert c.codes.shape == (5, 192) and c.scales.shape == (5, 3) and c.shape == (5, 130) and c.format == 0 and c.nbytes == 5 * 192 + 60
    assert cache(5, 130, 500).group == 130 and cache(0, 1).scales.shape == (0, 1)
    assert cache(2, 64, fmt="e4m3").codes.dtype == torch.float8_e4m3fn


@pytest.mark.parametrize("kw", [dict(fmt="int4"), dict(group=12), dict(group=0), dict(group=-8), dict(width=0), dict(n=-1)])
def test_quant_rows_refuses(kw):
    with pytest.raises(ValueError):
        cache(**kw)


def test_quant_rows_container_refuses():
    codes, scales = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 1)
    ops.QuantRows(codes, scales, 64)
    for bad in [(codes.float(), scales, 40), (codes[:, :60], scales, 40), (codes, scales, 65), (codes, scales, 0), (codes, scales[:3], 40),
                (codes, scales.double(), 40), (codes.t().contiguous().t(), scales, 40), (codes, torch.zeros(4, 2), 40), (codes[0], scales, 40)]:
        with pytest.raises(ValueError):
            ops.QuantRows(*bad)
    with pytest.raises(ValueError):
        ops.QuantRows(codes, torch.zeros(4, 4), 40, 12)
    flat = torch.zeros(4 * 64 + 64, dtype=torch.int8)
    off = 1 if flat.data_ptr() % 64 == 0 else 0
    with pytest.raises(ValueError, match="aligned"):
        ops.QuantRows(flat[off:off + 256].view(4, 64), scales, 40)


def test_cpu_tensors_are_refused():
    c = cache()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.quant_rows_write(c, torch.zeros(4, 40))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.quant_rows_read(c)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.quantize_rows(torch.zeros(4, 40))
    with pytest.raises(ValueError):
        ops.quant_rows_write(c, torch.zeros(4, 40, dtype=torch.float64))
    with pytest.raises(ValueError):
        ops.quant_rows_write(c, torch.zeros(40))
    with pytest.raises(ValueError):
        ops.quant_rows_read(c, dtype=torch.int8)


def test_c_entries_check_their_arguments():
    h = _lib.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64
    ok = dict(x=p, ldx=40, t=0, m=3, w=40, slots=None, start=0, codes=p, ldc=64, f=0, scales=p, n=4, g=40, ws=None, nb=0)

    def write(**kw):
        a = dict(ok, **kw)
        return h.ogl_quant_rows_write(a["x"], a["ldx"], a["t"], a["m"], a["w"], a["slots"], a["start"], a["codes"], a["ldc"], a["f"], a["scales"],
                                      a["n"], a["g"], a["ws"], a["nb"], None)

    for kw in [dict(x=None), dict(ldx=39), dict(t=3), dict(t=-1), dict(m=-1), dict(w=0), dict(start=2), dict(start=-1), dict(codes=None), dict(ldc=72),
               dict(ldc=0), dict(f=2), dict(scales=None), dict(n=-1), dict(g=12), dict(g=0), dict(codes=p + 8), dict(x=p + 2), dict(m=2 ** 31, slots=p),
               dict(start=2 ** 62)]:
        assert write(**kw) == -1, kw
    assert write(m=0) == 0 and write(n=0, m=0) == 0
    assert write(m=1000, slots=p) == -4 and write(m=1000, slots=p, ws=p, nb=15) == -4      # more rows than the scan takes: a workspace
    assert h.ogl_quant_rows_workspace_bytes(1000, 4, 1) == 16 and h.ogl_quant_rows_workspace_bytes(1000, 4, 0) == 0
    assert h.ogl_quant_rows_workspace_bytes(256, 4, 1) == 0 and h.ogl_quant_rows_workspace_bytes(-1, 4, 1) == -1

    def read(**kw):
        a = dict(dict(ok, out=p, ldo=40, rows=None), **kw)
        return h.ogl_quant_rows_read(a["codes"], a["ldc"], a["f"], a["scales"], a["n"], a["w"], a["g"], a["rows"], a["m"], a["out"], a["ldo"], a["t"], None)

    for kw in [dict(m=5), dict(m=-1), dict(ldo=39), dict(out=None), dict(t=3), dict(codes=None), dict(g=12), dict(out=p + 1, t=1), dict(m=2 ** 31, rows=p)]:
        assert read(**kw) == -1, kw
    assert read(m=0) == 0


def test_linear_refuses():
    x, w = cache(4, 40), cache(6, 40)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.linear_int8(x, w)
    for a, kw in [((x, cache(6, 41)), {}), ((cache(4, 40, 8), w), {}), ((x, cache(6, 40, fmt="e4m3")), {}), ((x, torch.zeros(6, 40)), {}),
                  ((x, w), dict(dtype=torch.float64)), ((x, w), dict(bias=torch.zeros(5))), ((x, w), dict(bias=torch.zeros(6, dtype=torch.float16))),
                  ((torch.zeros(4, 40), w), dict(x_rows=torch.zeros(2, dtype=torch.int64))), ((cache(1, 131072), cache(1, 131072)), {})]:
        with pytest.raises(ValueError):
            ops.linear_int8(*a, **kw)
    with pytest.raises(RuntimeError, match="inference only"):
        ops.linear_int8(x, w, bias=torch.zeros(6, requires_grad=True))
    with pytest.raises(RuntimeError, match="inference only"):
        ops.linear_int8(torch.zeros(4, 40, requires_grad=True), w)


def test_linear_c_entry_checks_its_arguments():
    h = _lib.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64
    ok = dict(x=p, ldx=64, sx=p, rows=None, nrows=4, M=3, K=40, w=p, ldw=64, sw=p, N=6, bias=None, relu=0, y=p, ldy=8, t=0)

    def call(**kw):
        a = dict(ok, **kw)
        return h.ogl_linear_i8(a["x"], a["ldx"], a["sx"], a["rows"], a["nrows"], a["M"], a["K"], a["w"], a["ldw"], a["sw"], a["N"], a["bias"],
                               a["relu"], a["y"], a["ldy"], a["t"], None)

    for kw in [dict(x=None), dict(sx=None), dict(w=None), dict(sw=None), dict(y=None), dict(ldx=72), dict(ldx=0), dict(ldw=32), dict(K=65), dict(K=0),
               dict(K=131072, ldx=131072, ldw=131072), dict(M=5), dict(M=-1), dict(N=-1), dict(nrows=-1), dict(nrows=0, rows=p), dict(ldy=5), dict(t=3),
               dict(x=p + 16), dict(w=p + 16), dict(y=p + 2), dict(y=p + 1, t=1)]:
        assert call(**kw) == -1, kw
    assert call(M=0) == 0 and call(N=0) == 0


def test_linear_c_entry_refuses_tables_beyond_its_offsets():
    h = _lib.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64
    for nrows, ldx, n, ldw in [(2 ** 32, 64, 6, 64), (4, 2 ** 37, 6, 64), (2 ** 20, 2 ** 18, 6, 64), (4, 64, 2 ** 30, 256), (4, 64, 6, 2 ** 36)]:
        assert h.ogl_linear_i8(p, ldx, p, None, nrows, 3, 40, p, ldw, p, n, None, 0, p, n, 0, None) == -1


def test_group_norm_refuses():
    x = torch.zeros(4, 12)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.group_norm(x, 3)
    for a, kw in [((torch.zeros(12), 3), {}), ((x, 5), {}), ((x, 0), {}), ((x.double(), 3), {}), ((x, 3), dict(activation="tanh")), ((x, 3), dict(eps=-1.0)),
                  ((x, 3, torch.ones(11)), {}), ((x, 3, torch.ones(12, dtype=torch.bfloat16)), {}), ((x, 3, torch.ones(24)[::2]), {}),
                  ((x.half(), 3, torch.ones(12), torch.ones(12).half()), {}), ((torch.zeros(4, 0), 1), {})]:
        with pytest.raises(ValueError):
            ops.group_norm(*a, **kw)


def test_group_norm_c_entries_check_their_arguments():
    h = _lib.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64
    ok = dict(x=p, xb=12, xl=12, t=0, B=4, L=1, C=12, G=3, w=p, b=p, pt=0, eps=1e-5, act=1, y=p, yb=12, yl=12, mean=p, rstd=p, ws=p, nb=1 << 30, dy=p, dw=p, db=p)

    def fwd(**kw):
        a = dict(ok, **kw)
        return h.ogl_group_norm_fwd(a["x"], a["xb"], a["xl"], a["t"], a["B"], a["L"], a["C"], a["G"], a["w"], a["b"], a["pt"], a["eps"], a["act"], a["y"],
                                    a["yb"], a["yl"], a["mean"], a["rstd"], a["ws"], a["nb"], None)

    def bwd(**kw):
        a = dict(ok, **kw)
        return h.ogl_group_norm_bwd(a["dy"], a["xb"], a["xl"], a["x"], a["xb"], a["xl"], a["t"], a["B"], a["L"], a["C"], a["G"], a["w"], a["b"], a["pt"],
                                    a["act"], a["mean"], a["rstd"], a["y"], a["yb"], a["yl"], a["dw"], a["db"], a["ws"], a["nb"], None)

    common = [dict(x=None), dict(t=3), dict(B=-1), dict(L=-1), dict(L=2 ** 31), dict(C=0), dict(G=0), dict(G=5), dict(pt=1), dict(act=4), dict(act=-1),
              dict(xb=11), dict(L=2, xl=11), dict(yb=11), dict(C=2 ** 23, G=1, xb=2 ** 23, yb=2 ** 23), dict(x=p + 2), dict(w=p + 2), dict(rstd=None)]
    for kw in common + [dict(y=None), dict(eps=-1.0), dict(eps=float("nan")), dict(mean=None)]:
        assert fwd(**kw) == -1, kw
    for kw in common + [dict(dy=None), dict(mean=None), dict(B=0), dict(L=0), dict(dw=p + 2)]:
        assert bwd(**kw) == -1, kw
    assert fwd(B=0) == 0 and fwd(L=0) == 0
    assert bwd(y=None, dw=None, db=None) == 0                                  # nothing is wanted
    assert bwd(ws=None) == -4 and bwd(nb=8) == -4
    assert fwd(B=1, L=2000, ws=None) == -4 and fwd(B=1, L=2000, nb=8) == -4     # tiles of positions: partial sums
    size = h.ogl_group_norm_workspace_bytes
    assert size(4, 1, 12, 3, 0, 0) == 0 and size(4, 1, 12, 3, 0, 1) > 0 and size(1, 2000, 12, 3, 0, 0) > 0
    assert size(4, 1, 12, 5, 0, 0) == -1 and size(0, 1, 12, 3, 0, 1) == 0
