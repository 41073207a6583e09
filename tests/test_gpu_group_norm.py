"""Group norm with an activation against its definition in 64 bits, forward and backward.

Tolerances.  u = 2^-24.  Every value is compared with the 64-bit result v of the same (already rounded) inputs.
  y:   h = (x - mean) rstd.  The mean of m values is off by at most a few u times max|x| (sums joined pairwise or by threads of <= a few hundred
       terms: bounded here by 64 u max|x|), the variance by the same relative to its scale; with max|h| = H, max|w| = W the error of z is below
       64 u (|x|max rstd + H) W + 2 u |b|, the activations have slopes of at most 1.13 and errors of a few u of z: 256 u (1 + |x|max rstd + H)(1 + W)
       holds with a factor to spare, plus half a step of the output type.
  dx:  rstd (dz w - s1 - h s2): the same relative errors against the largest term: 1024 u rstd (1 + H)(1 + |x|max rstd + H) D W^2 with D = max|dy|.
  dw, db: sums of N = B L terms of at most D H: the rounding of a float32 sum over threads, rows and blocks, each a chain of at most
       N^(1/2) + 64 terms or so: below 16 u (sqrt(N) + 64) sum|terms| / sqrt(N) .. bounded by u (64 + 4 sqrt(N)) sum|terms|, terms off by 64 u (...) too.
These are bounds on rounding, loose by design; the relative 2-norm (checked to 3e-6 in float32) is what would show a wrong term.
"""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ACTS = {None: lambda z: z, "relu": torch.relu, "silu": F.silu, "gelu": F.gelu}


@pytest.fixture(scope="module")
def ops():
    import ogl_amd  # noqa: F401
    from ogl_amd import ops as _ops
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return _ops


def oracle(x, G, w, b, eps, act, dy=None):
    """float64 on the CPU, from the definition; gradients by autograd over it."""
    x = x.detach().double().cpu().requires_grad_(dy is not None)
    C = x.shape[-1]
    w = torch.ones(C, dtype=torch.float64) if w is None else w.detach().double().cpu()
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.detach().double().cpu()
    w.requires_grad_(dy is not None), b.requires_grad_(dy is not None)
    B = x.shape[0]
    v = x.reshape(B, -1, G, C // G)
    mean = v.mean((1, 3), keepdim=True)
    var = ((v - mean) ** 2).mean((1, 3), keepdim=True)
    h = (v - mean) / torch.sqrt(var + eps)
    z = (h.reshape(x.shape) * w + b)
    y = ACTS[act](z)
    if dy is None:
        return y, None, (h, z, 1 / torch.sqrt(var + eps))
    grads = torch.autograd.grad(y, (x, w, b), dy.detach().double().cpu())
    return y.detach(), grads, (h.detach(), z.detach(), (1 / torch.sqrt(var + eps)).detach())


def check(ops, shape, G, dtype=torch.float32, act=None, p_dtype=None, affine=(True, True), seed=0, mean=0.3, eps=1e-5, strided=False):
    gen = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = (torch.randn(shape, generator=gen) * 1.5 + mean).to(dtype).cuda()
    dy = torch.randn(shape, generator=gen).to(dtype).cuda()
    w = (torch.rand(C, generator=gen) + 0.5).to(p_dtype or torch.float32).cuda() if affine[0] else None
    b = (torch.randn(C, generator=gen) * 0.2).to(p_dtype or torch.float32).cuda() if affine[1] else None
    if strided:                                                            # rows further apart, off any alignment
        wide = torch.zeros((*shape[:-1], C + 13), dtype=dtype, device="cuda")
        wide[..., 5:5 + C] = x
        x = wide[..., 5:5 + C]
    if act == "relu":
        # no z within rounding of the kink: its slope would be either side's
        _, _, (h, z, rstd) = oracle(x, G, w, b, eps, act)
        near = (z.abs() < 1e-4).cuda()
        dy = torch.where(near, torch.zeros_like(dy), dy)
    leaves = [t for t in (x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_()
    y = ops.group_norm(x, G, w, b, eps, act)
    assert y.shape == x.shape and y.dtype == dtype
    grads = torch.autograd.grad(y, leaves, dy)
    want, (dx0, dw0, db0), (h, z, rstd) = oracle(x, G, w, b, eps, act, dy)
    half = torch.finfo(dtype).eps / 2
    xm, rm, H = float(x.detach().abs().max()), float(rstd.max()), float(h.abs().max())
    W, D = float(w.detach().abs().max()) if w is not None else 1.0, float(dy.abs().max())
    spread = 1 + xm * rm + H
    err = (y.detach().cpu().double() - want).abs()
    assert (err <= 256 * U * spread * (1 + W) + half * want.abs()).all(), float(err.max())
    got = dict(zip([i for i, t in enumerate((x, w, b)) if t is not None], grads))
    assert got[0].dtype == dtype and got[0].shape == x.shape
    err = (got[0].cpu().double() - dx0).abs()
    assert (err <= 1024 * U * rm * (1 + H) * spread * D * W * W + half * dx0.abs()).all(), float(err.max())
    N = want.numel() / C
    for i, v, top in ((1, dw0, H), (2, db0, 1.0)):
        if i in got:
            assert got[i].dtype == (p_dtype or torch.float32)
            err = (got[i].cpu().double() - v).abs()
            bound = (U * (64 + 4 * N ** 0.5) + 256 * U * spread) * N * D * top * 1.2 + torch.finfo(got[i].dtype).eps / 2 * v.abs()
            assert (err <= bound).all(), float(err.max())
    if dtype == torch.float32 and (p_dtype or torch.float32) == torch.float32 and mean == 0.3 and want.numel() // (shape[0] * G) >= 8:
        for a, v in [(y.detach(), want), (got[0], dx0)] + [(got[i], v) for i, v in ((1, dw0), (2, db0)) if i in got and N >= 8]:
            norm = float(v.norm())
            assert norm == 0 or float((a.cpu().double() - v).norm()) <= 3e-6 * max(norm, 1e-3 * D * W * v.numel() ** 0.5)
    # inference gives the same values, and so does a second backward (no atomics)
    with torch.no_grad():
        assert torch.equal(ops.group_norm(x, G, w, b, eps, act), y.detach())
    again = torch.autograd.grad(ops.group_norm(x, G, w, b, eps, act), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


ROWS = [((1, 1), 1), ((1, 4), 1), ((3, 6), 3), ((5, 7), 1), ((7, 12), 12), ((832, 32), 4), ((50, 600), 30), ((41, 600), 8), ((33, 602), 2), ((9, 602), 1),
        ((130, 128), 1), ((5, 1030), 1), ((4, 2050), 2), ((3, 4096), 1), ((2, 4100), 1), ((2, 9000), 1), ((3, 40000), 2), ((700, 24), 8), ((1, 512), 32)]
MAPS = [((1, 2, 1), 1), ((2, 3, 5), 5), ((1, 1, 8), 2), ((3, 7, 12), 4), ((2, 64, 320), 32), ((2, 9, 9, 96), 3), ((1, 4096, 40), 8), ((1, 1000, 512), 32),
        ((4, 33, 33, 64), 32), ((1200, 5, 16), 4), ((2, 100, 1200), 1), ((1, 300, 2400), 1), ((1, 2000, 2400), 1), ((2, 17, 5000), 1), ((2, 3, 600), 300),
        ((1, 2500, 7), 7), ((2, 2, 2, 2, 6), 2), ((1100, 2, 2100), 1), ((2, 50, 3000), 1000)]


@pytest.mark.parametrize("shape,G", ROWS + MAPS)
def test_float32_every_shape(ops, shape, G):
    check(ops, shape, G, act="silu", seed=sum(shape))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,G", [((1030, 2, 8), 2), ((1030, 3, 9), 3), ((1024, 7, 40), 5), ((2050, 4, 6), 1), ((1500, 2, 250), 1), ((1100, 50, 12), 4),
                                     ((1024, 2, 1000), 125), ((9001, 2, 5), 5)])
def test_many_small_maps(ops, dtype, shape, G):
    check(ops, shape, G, dtype, act="silu", seed=sum(shape))


@pytest.mark.parametrize("act", [None, "relu", "gelu"])
@pytest.mark.parametrize("shape,G", [((65, 96), 6), ((2, 40, 64), 8), ((1, 1500, 48), 4), ((3, 2, 4500), 1)])
def test_activations(ops, act, shape, G):
    check(ops, shape, G, act=act)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("own_params", [True, False])
@pytest.mark.parametrize("shape,G", [((70, 600), 30), ((33, 75), 3), ((9, 1100), 1), ((5, 5000), 1), ((2, 12000), 1), ((3, 100, 320), 32), ((1, 3000, 72), 9),
                                     ((1, 600, 4800), 2), ((1500, 3, 24), 8)])
def test_half_types(ops, dtype, own_params, shape, G):
    check(ops, shape, G, dtype=dtype, act="gelu", p_dtype=dtype if own_params else None)


@pytest.mark.parametrize("shape,G", [((40, 60), 6), ((2, 70, 60), 6), ((1, 1500, 60), 6)])
@pytest.mark.parametrize("affine", [(True, False), (False, True), (False, False)])
def test_without_weight_or_bias(ops, shape, G, affine):
    check(ops, shape, G, act="silu", affine=affine)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,G", [((40, 61), 1), ((6, 50, 61), 61), ((1, 1500, 62), 2), ((3, 9, 9, 20), 4)])
def test_strided_and_misaligned_rows(ops, dtype, shape, G):
    check(ops, shape, G, dtype=dtype, act="silu", strided=True)


@pytest.mark.parametrize("shape,G", [((200, 256), 4), ((2, 500, 64), 8), ((1, 6000, 64), 8), ((2, 40, 4800), 2)])
def test_a_mean_far_from_zero(ops, shape, G):
    """mean 1000, deviation 1.5: the variance comes from differences, so its digits stay."""
    check(ops, shape, G, mean=1000.0)
    gen = torch.Generator().manual_seed(1)
    x = (torch.randn(shape, generator=gen) + 1000.0).cuda()
    want = oracle(x, G, None, None, 1e-5, None)[0]
    got = ops.group_norm(x, G).cpu().double()
    assert float((got - want).norm() / want.norm()) < 1e-4           # a step of x is 6e-5 of its deviation; E[x^2] - E[x]^2 would be off by 6e-2


def test_differences(ops):
    """The gradient against central differences of the kernel's own forward (float32, step 1e-2: truncation ~1e-4, rounding ~1e-5 of a sum of 96)."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(2, 6, 8, generator=gen).cuda().requires_grad_()
    dy = torch.randn(2, 6, 8, generator=gen).cuda()
    w, b = (torch.rand(8, generator=gen) + 0.5).cuda(), torch.randn(8, generator=gen).cuda()
    (dx,) = torch.autograd.grad(ops.group_norm(x, 2, w, b, 1e-5, "gelu"), x, dy)
    step = 1e-2
    with torch.no_grad():
        for at in [(0, 0, 0), (0, 5, 7), (1, 2, 3), (1, 4, 6)]:
            p, q = x.clone(), x.clone()
            p[at] += step
            q[at] -= step
            diff = ((ops.group_norm(p, 2, w, b, 1e-5, "gelu") - ops.group_norm(q, 2, w, b, 1e-5, "gelu")) * dy).sum() / (2 * step)
            assert abs(float(diff) - float(dx[at])) < 2e-3 * max(1.0, abs(float(dx[at])))


def test_infinities_and_nans_stay_in_their_group(ops):
    x = torch.randn(4, 10, 12, generator=torch.Generator().manual_seed(0)).cuda()
    clean = ops.group_norm(x, 3)
    x[1, 4, 5], x[2, 0, 0], x[3, 9, 11] = float("nan"), float("inf"), float("-inf")
    y = ops.group_norm(x, 3)
    bad = torch.zeros_like(x, dtype=torch.bool)
    bad[1, :, 4:8] = bad[2, :, 0:4] = bad[3, :, 8:12] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])
    r = torch.randn(5, 600, generator=torch.Generator().manual_seed(0)).cuda()
    clean = ops.group_norm(r, 30)
    r[2, 599] = float("inf")
    y = ops.group_norm(r, 30)
    assert torch.isnan(y[2, 580:]).all() and torch.equal(y[:2], clean[:2]) and torch.equal(y[2, :580], clean[2, :580])


@pytest.mark.parametrize("shape", [(0, 8), (0, 5, 8), (3, 0, 8)])
def test_empty(ops, shape):
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    w, b = torch.ones(8, device="cuda", requires_grad=True), torch.zeros(8, device="cuda", requires_grad=True)
    y = ops.group_norm(x, 2, w, b, activation="silu")
    assert y.shape == shape
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert dx.shape == shape and (dw == 0).all() and (db == 0).all()


def test_only_some_gradients(ops):
    x = torch.randn(30, 40, device="cuda")
    w, b = torch.ones(40, device="cuda", requires_grad=True), torch.zeros(40, device="cuda")
    y = ops.group_norm(x, 4, w, b, activation="silu")
    (dw,) = torch.autograd.grad(y.sum(), w)
    xg = x.clone().requires_grad_()
    wd = w.detach()
    (dx,) = torch.autograd.grad(ops.group_norm(xg, 4, wd, b, activation="silu").sum(), xg)
    xb = x.clone().requires_grad_()
    both = torch.autograd.grad(ops.group_norm(xb, 4, w, b, activation="silu").sum(), (xb, w))
    assert torch.equal(dx, both[0]) and torch.equal(dw, both[1])
    m = torch.randn(2, 900, 40, device="cuda")
    (dw,) = torch.autograd.grad(ops.group_norm(m, 4, w, b).sum(), w)       # tiles, no dx
    assert torch.isfinite(dw).all()


def test_twice_differentiating_is_refused(ops):
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    (dx,) = torch.autograd.grad((ops.group_norm(x, 2) ** 2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), x)


@pytest.mark.parametrize("shape,G", [((500, 96), 6), ((2, 1500, 96), 6), ((1500, 4, 24), 3)])
def test_captured(ops, shape, G):
    """Forward and backward in a graph, replayed with the program's own eager calls in between: each replay equals the eager result."""
    gen = torch.Generator().manual_seed(0)
    x, dy = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
    w, b = torch.ones(shape[-1], device="cuda"), torch.zeros(shape[-1], device="cuda")

    def body():
        y, stats = ops.group_norm_fwd(x, G, w, b, 1e-5, 2, True)
        return (y, *ops.group_norm_bwd(dy, x, G, w, b, stats, 2))
    body()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = body()
    for step in range(4):
        x.copy_(torch.randn(shape, generator=gen)), dy.copy_(torch.randn(shape, generator=gen)), w.copy_(torch.rand(shape[-1], generator=gen))
        g.replay()
        assert all(torch.equal(p, q) for p, q in zip(out, body()))
