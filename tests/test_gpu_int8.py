"""Rows kept in 8 bits against their definition in 64 bits.

Codes, scales and values are compared for EQUALITY: a scale is the float32 nearest amax / Q (one correctly rounded division), a code is the exact
quotient x / s rounded to nearest even — x and s have 24 bits, so where the quotient is not on a border between two codes it is at least 2^-33
of itself away from it, and a 64-bit quotient (error 2^-53) decides every case as the exact one does — and a value is one float32 product.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

Q = {"int8": 127.0, "e4m3": 448.0}
FLOOR = 2.0 ** -80


@pytest.fixture(scope="module")
def ops():
    import ogl_amd  # noqa: F401
    from ogl_amd import ops as _ops
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return _ops


def e4m3_grid():
    return torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def nearest(t, grid):
    hi = torch.searchsorted(grid, t).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - t, t - grid[lo]
    return torch.where(torch.where(up == down, hi % 2 == 0, up < down), grid[hi], grid[lo])


def oracle_rows(x, fmt, group):
    """(codes as the numbers they are, scales) of CPU rows, in 64 bits."""
    x = x.double()
    m, w = x.shape
    group = min(group or w, w)
    codes, scales = torch.zeros(m, w, dtype=torch.float64), torch.zeros(m, -(-w // group))
    grid = torch.arange(128, dtype=torch.float64) if fmt == "int8" else e4m3_grid()
    for g, lo in enumerate(range(0, w, group)):
        v = x[:, lo:lo + group]
        amax = v.abs().amax(1, keepdim=True)
        ok = torch.isfinite(v).all(1, keepdim=True)
        s = (amax.clamp(min=FLOOR) / Q[fmt]).float()
        s = torch.where(ok, s, torch.full_like(s, math.nan))
        t = torch.where(ok, v / s.double(), torch.zeros_like(v))
        codes[:, lo:lo + group] = torch.sign(t) * nearest(t.abs(), grid)
        scales[:, g] = s[:, 0]
    return codes, scales


def expand(scales, group, w):
    return torch.repeat_interleave(scales, group, dim=1)[:, :w]


def make(m, w, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(m, w, generator=gen) * torch.exp(2 * torch.randn(m, 1, generator=gen))).to(dtype)


def check_cache(cache, codes, scales, rows=slice(None)):
    w = cache.width
    got = cache.codes.cpu()
    assert torch.equal(got[rows, :w].float(), codes.float())
    assert (got[rows, w:].view(torch.int8) == 0).all()                   # what the products read behind the last column
    assert torch.equal(torch.nan_to_num(cache.scales.cpu()[rows], nan=-1.0), torch.nan_to_num(scales, nan=-1.0))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,w,group", [(1, 1, None), (3, 7, None), (5, 8, None), (70, 9, 8), (33, 64, 16), (130, 100, 24), (17, 602, None), (9, 602, 96),
                                       (300, 128, 64), (5, 513, None), (4, 1100, 512), (3, 2048, None), (3, 2049, None), (2, 5001, None), (2, 6000, 2056),
                                       (6, 1024, 128), (2, 200, 4096)])
def test_write_and_read_equal_the_definition(ops, fmt, dtype, m, w, group):
    x = make(m, w, dtype, seed=m * 1000 + w)
    x[m // 2] = 0                                                            # an empty row: amax 0
    codes, scales = oracle_rows(x, fmt, group)
    cache = ops.quantize_rows(x.cuda(), group, fmt)
    assert cache.shape == (m, w) and cache.codes.shape[1] % 64 == 0
    check_cache(cache, codes, scales)
    values = codes.float() * expand(scales, cache.group, w)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        got = ops.quant_rows_read(cache, dtype=out)
        assert got.dtype == out and torch.equal(got.cpu(), values.to(out))
    ids = torch.tensor([m - 1, -1, 0, m, 0, 2 ** 40, m // 2])
    got = ops.quant_rows_read(cache, ids.cuda()).cpu()
    for row, i in zip(got, ids.tolist()):
        assert torch.equal(row, values[i] if 0 <= i < m else torch.zeros(w))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("scale", [1.0, 1.1, 0.37, 3e-20, 1.7e30])
def test_borders_between_codes(ops, fmt, scale):
    """Elements at, and one float next to, every border between two codes."""
    s = torch.tensor(scale).float()
    amax = (s.double() * Q[fmt]).float()
    s = (amax.double() / Q[fmt]).float()
    grid = torch.arange(128, dtype=torch.float64) if fmt == "int8" else e4m3_grid()
    mid = ((grid[1:] + grid[:-1]) / 2 * s.double()).float()
    x = torch.cat([mid, torch.nextafter(mid, torch.tensor(math.inf)), torch.nextafter(mid, torch.tensor(0.0))])
    x = torch.cat([x, -x, amax.reshape(1)]).reshape(1, -1)
    codes, scales = oracle_rows(x, fmt, None)
    assert float(scales[0, 0]) == float(s)
    check_cache(ops.quantize_rows(x.cuda(), None, fmt), codes, scales)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_extreme_values(ops, fmt):
    inf, nan = math.inf, math.nan
    x = torch.zeros(9, 48)
    x[0, 3] = inf; x[1, 20] = -inf; x[2, 40] = nan; x[3] = 3.4028234663852886e38; x[4] = 1e-45; x[5, ::2] = -1e-38
    x[6] = 1e-30; x[7, 0] = 65504.0; x[8, :16] = torch.linspace(-1e-24, 1e-24, 16)
    codes, scales = oracle_rows(x, fmt, 16)
    cache = ops.quantize_rows(x.cuda(), 16, fmt)
    check_cache(cache, codes, scales)
    got = ops.quant_rows_read(cache).cpu()
    bad = torch.isnan(expand(scales, 16, 48))
    assert torch.equal(torch.isnan(got), bad) and int(bad.sum()) == 48              # the three groups that hold one, nothing else
    want = codes.float() * expand(scales, 16, 48)
    assert torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("m,n", [(40, 30), (256, 90), (257, 90), (3000, 700)])
@pytest.mark.parametrize("w,group", [(40, None), (602, None), (128, 16), (2600, None)])
def test_slots_repeat_skip_and_leave_the_rest(ops, m, n, w, group):
    """Of a slot's rows the last stands, slots outside the cache are skipped, other rows keep what they held (both forms of finding the last)."""
    gen = torch.Generator().manual_seed(m + w)
    old = make(n, w, torch.float32, 5)
    x = make(m, w, torch.bfloat16, 6)
    slots = torch.randint(-2, n + 2, (m,), generator=gen)
    slots[slots == 3] = 4                                                           # a row that nobody writes
    slots[m - 1], slots[0] = 2 ** 40, -2 ** 40
    c0, s0 = oracle_rows(old, "int8", group)
    c1, s1 = oracle_rows(x, "int8", group)
    for i, t in enumerate(slots.tolist()):
        if 0 <= t < n:
            c0[t], s0[t] = c1[i], s1[i]
    cache = ops.quantize_rows(old.cuda(), group)
    for _ in range(2):                                                              # a second call finds nothing of the first in its workspace
        ops.quant_rows_write(cache, x.cuda(), slots=slots.cuda())
        check_cache(cache, c0, s0)


def test_strided_rows_and_ranges(ops):
    wide = make(20, 300, torch.float32, 7).cuda()
    view = wide[1::3, 5:106]                                                         # 7 rows, stride 900, 20 bytes off an aligned address
    codes, scales = oracle_rows(view.cpu(), "int8", None)
    cache = ops.quant_rows(12, 101)
    ops.quant_rows_write(cache, view, start=4)
    check_cache(cache, codes, scales, slice(4, 11))
    assert (cache.codes[:4] == 0).all() and (cache.codes[11:] == 0).all() and (cache.scales[11:] == 0).all()
    ops.quant_rows_write(cache, wide.t()[:101, :5].t(), start=0)                     # columns far apart: copied first
    check_cache(cache, *oracle_rows(wide.cpu().t()[:101, :5].t(), "int8", None), slice(0, 5))
    ops.quant_rows_write(cache, view[:0], start=12)
    ops.quant_rows_write(cache, view[:0], slots=torch.empty(0, dtype=torch.int64, device="cuda"))
    assert ops.quant_rows_read(cache, torch.empty(0, dtype=torch.int64, device="cuda")).shape == (0, 101)
    empty = ops.quant_rows(0, 101)
    ops.quant_rows_write(empty, view, slots=torch.zeros(7, dtype=torch.int64, device="cuda"))
    assert ops.quant_rows_read(empty).shape == (0, 101)
    assert (ops.quant_rows_read(empty, torch.tensor([0, 1], device="cuda")) == 0).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("w,group", [(602, None), (1031, 128), (270, 8), (100, None)])
def test_many_rows_read(ops, fmt, dtype, w, group):
    """Enough rows for every form of the reading kernel: the product in float32, rounded once more to the type; ids outside the cache are zero rows."""
    n, m = 5000, 4 * 2048 * 256 * 8 // w + 3
    gen = torch.Generator(device="cuda").manual_seed(w)
    cache = ops.quantize_rows(torch.randn(n, w, device="cuda", generator=gen), group, fmt)
    rows = torch.randint(-3, n + 3, (m,), device="cuda", generator=gen)
    rows[0], rows[-1] = 2 ** 40, -2 ** 40
    got = ops.quant_rows_read(cache, rows, dtype)
    ok = ((rows >= 0) & (rows < n)).unsqueeze(1)
    at = rows.clamp(0, n - 1)
    at = torch.where(ok[:, 0], at, torch.zeros_like(at))
    scales = torch.repeat_interleave(cache.scales, cache.group, dim=1)[:, :w]
    want = torch.where(ok, cache.codes[:, :w].float()[at] * scales[at], torch.zeros((), device="cuda")).to(dtype)
    assert torch.equal(got, want)
    assert not torch.signbit(got[~ok[:, 0]]).any()


def test_rows_behind_four_gigabytes(ops):
    """Row offsets that pass 32 bits."""
    n, w = 4_300_000, 1000                                                           # 4.4 GB of codes
    cache = ops.quant_rows(n, w)
    x = make(3, w, torch.float32, 8)
    slots = torch.tensor([n - 1, 7, 4_200_000])
    ops.quant_rows_write(cache, x.cuda(), slots=slots.cuda())
    codes, scales = oracle_rows(x, "int8", None)
    check = ops.quant_rows_read(cache, torch.cat([slots, torch.tensor([n - 2, 4_200_000 - 2 ** 32 // 1024])]).cuda()).cpu()
    assert torch.equal(check[:3], codes.float() * scales) and (check[3:] == 0).all()


def test_captured_write_and_read(ops):
    """Replays of a captured write + read follow the inputs, between eager calls on the same cache."""
    n, w, m = 600, 96, 400
    cache = ops.quant_rows(n, w, 32, "e4m3")
    x, slots, rows = torch.zeros(m, w, device="cuda"), torch.zeros(m, dtype=torch.int64, device="cuda"), torch.arange(n, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.quant_rows_write(cache, x, slots=slots)
        ops.quant_rows_read(cache, rows)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.quant_rows_write(cache, x, slots=slots)
        out = ops.quant_rows_read(cache, rows)
    c0, s0 = torch.zeros(n, w, dtype=torch.float64), torch.zeros(n, 3)
    cache.codes.view(torch.int8).zero_(); cache.scales.zero_()
    for step in range(4):
        xs = make(m, w, torch.float32, 20 + step)
        gen = torch.Generator().manual_seed(step)
        ss = torch.randint(-1, n, (m,), generator=gen)
        x.copy_(xs); slots.copy_(ss)
        g.replay()
        c1, s1 = oracle_rows(xs, "e4m3", 32)
        for i, t in enumerate(ss.tolist()):
            if t >= 0:
                c0[t], s0[t] = c1[i], s1[i]
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), c0.float() * expand(s0, 32, w))
        ops.quant_rows_write(cache, xs[:1].cuda(), start=step)                         # the program's own eager work in between
        c0[step], s0[step] = c1[0], s1[0]


# ---- the product ---------------------------------------------------------------------------------------------------------------------------------
def random_cache(ops, n, k, seed, big=False):
    gen = torch.Generator().manual_seed(seed)
    codes = torch.zeros(n, -(-k // 64) * 64, dtype=torch.int8)
    codes[:, :k] = 127 if big else torch.randint(-128, 128, (n, k), generator=gen, dtype=torch.int8)
    scales = torch.rand(n, 1, generator=gen) + 0.1
    return ops.QuantRows(codes.cuda(), scales.cuda(), k)


def linear_oracle(x, w, bias, relu, rows, dtype):
    """(result, bound) in 64 bits.  The sum is exact in both; float32 roundings behind it: of the sum, of sx sw, of their product (2^-24 each of the
    product p), of the addition (2^-24 of |p| + |b|, itself off by at most 3 * 2^-24 |p|): below 2^-24 (5 |p| + |b|); then one to ``dtype``,
    at most half its eps of the value."""
    xc, sx = x.codes.cpu()[:, :x.width].double(), x.scales.cpu().double()
    if rows is not None:
        ok = (rows >= 0) & (rows < x.shape[0])
        at = torch.where(ok, rows, torch.zeros_like(rows))
        xc, sx = xc[at] * ok.unsqueeze(1), sx[at] * ok.unsqueeze(1)
    p = (xc @ w.codes.cpu()[:, :w.width].double().t()) * sx * w.scales.cpu().double().t()
    b = torch.zeros(w.shape[0], dtype=torch.float64) if bias is None else bias.cpu().double()
    y = p + b
    bound = 2.0 ** -24 * (5 * p.abs() + b.abs())
    y = y.clamp(min=0) if relu else y
    if dtype != torch.float32:
        bound = bound + torch.finfo(dtype).eps / 2 * (y.abs() + bound)
    return y, bound + 1e-30


def check_linear(ops, M, N, K, dtype=torch.float32, relu=False, with_bias=True, n_rows=None, seed=0, big=False):
    x, w = random_cache(ops, n_rows or M, K, seed + 1, big), random_cache(ops, N, K, seed + 2, big)
    gen = torch.Generator().manual_seed(seed)
    bias = (torch.randn(N, generator=gen) * 50).cuda() if with_bias else None
    rows = torch.randint(-2, n_rows + 2, (M,), generator=gen) if n_rows else None
    got = ops.linear_int8(x, w, bias, relu, None if rows is None else rows.cuda(), dtype)
    assert got.shape == (M, N) and got.dtype == dtype
    want, bound = linear_oracle(x, w, bias, relu, rows, dtype)
    assert (got.cpu().double() - want).abs().sub(bound).max() <= 0


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 130, 256, 300])
@pytest.mark.parametrize("N,K", [(1, 1), (3, 64), (15, 65), (16, 128), (17, 129), (41, 600), (65, 191), (130, 257), (600, 602)])
def test_linear_equals_the_definition(ops, M, N, K):
    check_linear(ops, M, N, K, relu=(M + N) % 2 == 1, with_bias=K % 2 == 0, seed=M)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K,n_rows", [(5, 70, 100, 40), (100, 600, 602, 3000), (1000, 257, 320, 77), (4096, 4100, 192, 999)])
def test_linear_gathers_rows(ops, dtype, M, N, K, n_rows):
    x_scale = 1e-3 if dtype == torch.float16 else 1.0                                  # (float16 ends at 65504)
    x, w = random_cache(ops, n_rows, K, 3), random_cache(ops, N, K, 4)
    x.scales.mul_(x_scale)
    rows = torch.randint(-2, n_rows + 2, (M,), generator=torch.Generator().manual_seed(1))
    rows[0], rows[-1] = 2 ** 40, -1
    got = ops.linear_int8(x, w, None, False, rows.cuda(), dtype)
    want, bound = linear_oracle(x, w, None, False, rows, dtype)
    assert (got.cpu().double() - want).abs().sub(bound).max() <= 0
    assert (got[0] == 0).all() and (got[-1] == 0).all()


@pytest.mark.parametrize("M,N,K", [(4097, 4099, 64), (4100, 4111, 129), (9000, 2048, 1000), (62500, 600, 602), (2048, 8192, 4096)])
def test_linear_large(ops, M, N, K):
    """Against the same product on the GPU in 64 bits (exact sums there too: |sum| < 2^53)."""
    x, w = random_cache(ops, M, K, 5), random_cache(ops, N, K, 6)
    got = ops.linear_int8(x, w, None, True)
    p = x.codes[:, :K].double() @ w.codes[:, :K].double().t() * x.scales.double() * w.scales.double().t()
    assert (got.double() - p.clamp(min=0)).abs().sub(2.0 ** -24 * 5 * p.abs()).max() <= 0


@pytest.mark.parametrize("M,N", [(3, 20), (70, 70)])
def test_linear_longest_sum(ops, M, N):
    """131071 columns of the largest code: 2114123119 of 2^31 - 1."""
    check_linear(ops, M, N, 131071, big=True)


def test_linear_of_a_nan_row_and_of_float_rows(ops):
    x = make(6, 100, torch.float32, 1)
    x[2, 5] = math.nan
    w = ops.quantize_rows(make(30, 100, torch.float32, 2).cuda())
    y = ops.linear_int8(x.cuda(), w, relu=True)
    assert torch.isnan(y[2]).all() and not torch.isnan(y[[0, 1, 3, 4, 5]]).any()
    assert torch.equal(torch.nan_to_num(y), torch.nan_to_num(ops.linear_int8(ops.quantize_rows(x.cuda()), w, relu=True)))


def test_linear_empty(ops):
    w = random_cache(ops, 8, 40, 1)
    assert ops.linear_int8(random_cache(ops, 0, 40, 2), w).shape == (0, 8)
    assert ops.linear_int8(random_cache(ops, 5, 40, 2), random_cache(ops, 0, 40, 1)).shape == (5, 0)
    with pytest.raises(ValueError, match="empty table"):
        ops.linear_int8(random_cache(ops, 0, 40, 2), w, x_rows=torch.zeros(3, dtype=torch.int64, device="cuda"))


def test_linear_captured(ops):
    w = random_cache(ops, 600, 602, 1)
    x, rows = random_cache(ops, 900, 602, 2), torch.zeros(300, dtype=torch.int64, device="cuda")
    ops.linear_int8(x, w, x_rows=rows)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.linear_int8(x, w, x_rows=rows)
    for step in range(4):
        ids = torch.randint(0, 900, (300,), generator=torch.Generator().manual_seed(step))
        rows.copy_(ids)
        x.scales.mul_(0.5)
        g.replay()
        assert torch.equal(y, ops.linear_int8(x, w, x_rows=ids.cuda()))
