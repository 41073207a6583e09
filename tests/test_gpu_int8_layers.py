"""Group norm, rows in 8 bits and their product where the framework uses them: layers, per-pass tables, train steps, custom ops, and a run of them
together.  What must be the same arithmetic is compared bit for bit; the run together against 64 bits, with the bounds derived there."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import ogl_amd  # noqa: F401
    from ogl_amd import ops as _ops
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return _ops


def toy(name="toy", evolve=8):
    from ogl_amd import synthetic
    feat_size, targets, dyn, n_classes, _ = synthetic.load(name, device="cuda")
    for _ in range(evolve):
        dyn.evolve()
    return feat_size, targets, dyn, n_classes


def norm_twin(x, norm):
    """float64 group norm + activation of the rows x, from the definition, on the CPU."""
    v = x.double().cpu()
    w, b = norm.weight.detach().double().cpu(), norm.bias.detach().double().cpu()
    g = v.view(v.shape[0], norm.num_groups, -1)
    mean, var = g.mean(2, keepdim=True), g.var(2, unbiased=False, keepdim=True)
    z = ((g - mean) / torch.sqrt(var + norm.eps)).view_as(v) * w + b
    return {None: lambda t: t, "relu": torch.relu, "silu": F.silu, "gelu": F.gelu}[norm.activation](z)


# ---- a run together ------------------------------------------------------------------------------------------------------------------------------
def test_norm_rows_and_product_together(ops):
    """Normalised, activated, appended to a cache, gathered from it by the product and read back, captured and replayed with eager work in between.
    The product against 64 bits of what the cache holds: an exact sum, then 2^-24 each for the sum, the two scales' product, their product and the
    addition (5 * 2^-24 of the product's size and 2^-24 of the bias), as for the operator alone.  The rows read back against the normalised rows: half a
    code, max|row| / 127 / 2, and 3 roundings of 2^-24 (scale, product, quotient's border)."""
    m, width, n_out, slots_n = 300, 96, 70, 1000
    gen = torch.Generator().manual_seed(0)
    x, slots = torch.zeros(m, width, device="cuda"), torch.zeros(m, dtype=torch.int64, device="cuda")
    w, b = (torch.rand(width, generator=gen) + 0.5).cuda(), torch.randn(width, generator=gen).cuda()
    weight, bias = ops.quantize_rows(torch.randn(n_out, width, generator=gen).cuda()), torch.randn(n_out, generator=gen).cuda()
    cache = ops.quant_rows(slots_n, width)

    def body():
        y = ops.group_norm(x, 6, w, b, activation="gelu")
        ops.quant_rows_write(cache, y, slots=slots)
        return y, ops.linear_int8(cache, weight, bias, True, slots), ops.quant_rows_read(cache, slots)
    body()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = body()
    for step in range(4):
        x.copy_(torch.randn(m, width, generator=gen) * 3)
        slots.copy_(torch.randperm(slots_n, generator=gen)[:m])
        graph.replay()
        got = [t.clone() for t in out]
        for t, e in zip(got, body()):
            assert torch.equal(t, e)
        y, p, back = (t.cpu().double() for t in got)
        assert ((back - y).abs() <= y.abs().amax(1, keepdim=True) * (1 / 254 + 3 * 2 ** -24)).all()
        at = slots.cpu()
        q = cache.codes.cpu()[at, :width].double() @ weight.codes.cpu()[:, :width].double().t() * cache.scales.cpu()[at].double() * weight.scales.cpu().double().t()
        want = (q + bias.cpu().double()).clamp(min=0)
        assert ((p - want).abs() <= 2 ** -24 * (5 * q.abs() + bias.cpu().double().abs())).all()


def test_two_graphs_share_a_cache(ops):
    """Each captured write has its own workspace: replayed at once on two streams, on slots of their own with repeats, both leave the last rows."""
    n, w, m = 4000, 64, 900                                                             # (m > 256: the owner table is in use)
    cache = ops.quant_rows(n, w)
    gen = torch.Generator().manual_seed(3)
    xs = [torch.randn(m, w, generator=gen).cuda() for _ in range(2)]
    ids = [(torch.randint(0, n // 2, (m,), generator=gen) + i * (n // 2)).cuda() for i in range(2)]
    ops.quant_rows_write(cache, xs[0], slots=ids[0])
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.quant_rows_write(cache, xs[i], slots=ids[i])
        graphs.append(g)
    for step in range(3):
        cache.codes.zero_(), cache.scales.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            last = {int(t): k for k, t in enumerate(ids[i].tolist())}
            want = ops.quantize_rows(xs[i][torch.tensor(list(last.values()), device="cuda")])
            at = torch.tensor(list(last), device="cuda")
            assert torch.equal(cache.codes[at], want.codes) and torch.equal(cache.scales[at], want.scales)
        for t in xs:
            t.mul_(0.5).add_(0.25)


def test_on_another_stream(ops):
    side = torch.cuda.Stream()
    x = torch.randn(2000, 96, device="cuda")
    want = ops.group_norm(x, 6)
    wq = ops.quantize_rows(x[:70].clone())
    wl = ops.linear_int8(want, wq)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        y = ops.group_norm(x, 6)
        z = ops.linear_int8(y, wq)
    side.synchronize()
    assert torch.equal(y, want) and torch.equal(z, wl)


# ---- outputs large enough to be stored past the caches --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("width", [600, 602])
def test_rows_of_large_outputs(ops, width):
    """The same bits as in calls too small for it (rows do not depend on each other; the gradients of weight and bias are sums over all rows)."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    n, h = 30_000, 15_000                                                              # 72 MB; halves of 36 MB
    x, dy = (torch.randn(n, width, device="cuda", generator=gen) for _ in range(2))
    w, b = torch.rand(width, device="cuda", generator=gen), torch.rand(width, device="cuda", generator=gen)
    y, stats = ops.group_norm_fwd(x, 2, w, b, 1e-5, 2, True)
    dx = ops.group_norm_bwd(dy, x, 2, w, b, stats, 2)[0]
    cache = ops.quantize_rows(x)
    back = ops.quant_rows_read(cache)
    for s in (slice(0, h), slice(h, n)):
        ys, st = ops.group_norm_fwd(x[s], 2, w, b, 1e-5, 2, True)
        assert torch.equal(y[s], ys) and torch.equal(stats[:, s], st)
        assert torch.equal(dx[s], ops.group_norm_bwd(dy[s], x[s], 2, w, b, st, 2)[0])
        assert torch.equal(back[s], ops.quant_rows_read(cache, torch.arange(s.start, s.stop, device="cuda")))


def test_map_of_large_outputs(ops):
    """2400 samples of 30 x 384, a block each whatever their number: the same bits in halves too small for it."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(2400, 30, 24 * 16, device="cuda", generator=gen)                   # 110 MB; halves of 55 MB
    y = ops.group_norm(x, 4, activation="silu")
    for s in (slice(0, 1200), slice(1200, 2400)):
        assert torch.equal(y[s], ops.group_norm(x[s], 4, activation="silu"))


# ---- offsets that pass 32 bits --------------------------------------------------------------------------------------------------------------------
def test_products_and_reads_behind_four_gigabytes(ops):
    """Rows of a table of 4.4 GB: the same bits as from a small table that holds the same rows."""
    n, w, k = 4_300_000, 1000, 64
    gen = torch.Generator().manual_seed(0)
    small = ops.quantize_rows(torch.randn(k, w, generator=gen).cuda())
    at = torch.randint(0, n, (k,), generator=gen)
    at[0], at[1], at[2] = n - 1, 2 ** 32 // 1024, 2 ** 31 // 1024
    at = torch.unique(at)
    table = ops.quant_rows(n, w)
    table.codes[at.cuda()], table.scales[at.cuda()] = small.codes[:len(at)], small.scales[:len(at)]
    weight = ops.quantize_rows(torch.randn(70, w, generator=gen).cuda())
    for m in (5, 60, 300, 9000):
        pick = torch.randint(0, len(at), (m,), generator=gen)
        far, near = at[pick].cuda(), pick.cuda()
        assert torch.equal(ops.linear_int8(table, weight, x_rows=far), ops.linear_int8(small, weight, x_rows=near))
        assert torch.equal(ops.quant_rows_read(table, far), ops.quant_rows_read(small, near))
    wide = ops.quantize_rows(torch.randn(9000, w, generator=gen).cuda())                 # (large tiles of the product)
    pick = torch.randint(0, len(at), (9000,), generator=gen)
    assert torch.equal(ops.linear_int8(table, wide, x_rows=at[pick].cuda()), ops.linear_int8(small, wide, x_rows=pick.cuda()))


def test_norm_behind_four_gigabytes(ops):
    """Rows and samples whose offsets pass 2^31 elements: the same bits as in a call on the last of them alone."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    w, b = torch.rand(1000, device="cuda", generator=gen), torch.rand(1000, device="cuda", generator=gen)
    x = torch.randn(2_300_000, 1000, device="cuda", generator=gen, dtype=torch.bfloat16)
    y, stats = ops.group_norm_fwd(x, 4, w, b, 1e-5, 2, True)
    dx = ops.group_norm_bwd(x, x, 4, w, b, stats, 2)[0]
    last = slice(2_200_000, None)
    y1, st1 = ops.group_norm_fwd(x[last], 4, w, b, 1e-5, 2, True)
    assert torch.equal(y[last], y1) and torch.equal(stats[:, last], st1)
    assert torch.equal(dx[last], ops.group_norm_bwd(x[last], x[last], 4, w, b, st1, 2)[0])
    x = x[:2_200_000].view(1100, 2000, 1000)
    y, stats = ops.group_norm_fwd(x, 4, w, b, 1e-5, 2, True)
    dx = ops.group_norm_bwd(x, x, 4, w, b, stats, 2)[0]
    last = slice(70, None)
    y1, st1 = ops.group_norm_fwd(x[last], 4, w, b, 1e-5, 2, True)
    assert torch.equal(y[last], y1) and torch.equal(stats[:, last], st1)
    assert torch.equal(dx[last], ops.group_norm_bwd(x[last], x[last], 4, w, b, st1, 2)[0])


# ---- products of middle size ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K,gather", [(2001, 1700, 1100, False), (300, 12200, 1030, True), (1537, 2049, 1024, True)])
def test_linear_of_middle_size(ops, dtype, M, N, K, gather):
    """Sums of K products exact in 64 bits on the GPU too (below 2^53), bounds as for the operator's other tests."""
    gen = torch.Generator().manual_seed(M)
    n = 777 if gather else M
    x, w = ops.quant_rows(n, K), ops.quant_rows(N, K)
    for q, scale in ((x, 1e-2), (w, 1e-2)):
        q.codes[:, :K] = torch.randint(-128, 128, (q.n, K), generator=gen, dtype=torch.int8).cuda()
        q.scales.copy_((torch.rand(q.n, 1, generator=gen) + 0.1) * scale)
    bias = torch.randn(N, generator=gen).cuda()
    rows = torch.randint(0, n, (M,), generator=gen).cuda() if gather else None
    got = ops.linear_int8(x, w, bias, True, rows, dtype)
    at = rows if gather else torch.arange(M, device="cuda")
    p = x.codes[at, :K].double() @ w.codes[:, :K].double().t() * x.scales[at].double() * w.scales.double().t()
    want = (p + bias.double()).clamp(min=0)
    bound = 2.0 ** -24 * (5 * p.abs() + bias.double().abs())
    if dtype != torch.float32:
        bound = bound + torch.finfo(dtype).eps / 2 * (want + bound) + 2.0 ** -25      # (2^-25: half the smallest float16)
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("M", [16, 17, 33, 64, 65])
@pytest.mark.parametrize("N", [4090, 4100])
def test_linear_of_few_rows_and_many_columns(ops, M, N):
    """Exact sums in every form, so the same bits as rows of a product that takes another one (as many rows as its tiles ask for)."""
    gen = torch.Generator().manual_seed(M)
    x, w = ops.quantize_rows(torch.randn(300, 333, generator=gen).cuda()), ops.quantize_rows(torch.randn(N, 333, generator=gen).cuda())
    bias = torch.randn(N, generator=gen).cuda()
    whole = ops.linear_int8(x, w, bias, True)
    assert torch.equal(ops.linear_int8(x, w, bias, True, torch.arange(M, device="cuda")), whole[:M])
    p = x.codes[:M, :333].double() @ w.codes[:, :333].double().t() * x.scales[:M].double() * w.scales.double().t()
    want = (p + bias.double()).clamp(min=0)
    assert ((whole[:M].double() - want).abs() <= 2.0 ** -24 * (5 * p.abs() + bias.double().abs())).all()


def test_linear_into_a_given_matrix(ops):
    gen = torch.Generator().manual_seed(1)
    x, w = ops.quantize_rows(torch.randn(200, 100, generator=gen).cuda()), ops.quantize_rows(torch.randn(70, 100, generator=gen).cuda())
    wide = torch.full((202, 90), 7.0, device="cuda")
    out = wide[1:201, 3:73]
    assert ops.linear_int8(x, w, out=out) is out
    assert torch.equal(out, ops.linear_int8(x, w))
    assert (wide[0] == 7).all() and (wide[201] == 7).all() and (wide[:, :3] == 7).all() and (wide[:, 73:] == 7).all()
    for bad in (wide[:200, :69], wide[:200, :70].double(), torch.zeros(70, 200, device="cuda").t()):
        with pytest.raises(ValueError):
            ops.linear_int8(x, w, out=bad)


# ---- layers ---------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("mode,pool", [("pool", None), ("maxpool", 9), ("meanpool", 12)])
def test_tables_from_rows_in_8_bits(ops, mode, pool):
    """The per-pass tables are the product of the quantised rows and weights, whole, by rows and into given blocks; a pass against them runs."""
    from ogl_amd import sampling
    from ogl_amd.graphsage import GatheredRows, GraphSAGE
    feat_size, _, dyn, n_classes = toy()
    g = dyn.get_graph()
    torch.manual_seed(2)
    model = GraphSAGE(feat_size, 16, n_classes, 1, F.relu, 0, mode, edge_feats=0, pool_feats=pool).cuda().eval()
    layer = model.layers[0]
    q = ops.quantize_rows(g.ndata["feat"])
    with torch.no_grad():
        p0, s0 = layer.project_tables(q)
        w_self, b_self = (layer.fc_self.weight, layer.fc_self.bias + layer.fc_neigh.bias) if mode == "pool" else \
            (layer.fc_neigh.weight[:, :feat_size], layer.fc_neigh.bias)
        assert torch.equal(p0, ops.linear_int8(q, ops.quantize_rows(layer.fc_pool.weight), layer.fc_pool.bias, True))
        assert torch.equal(s0, ops.linear_int8(q, ops.quantize_rows(w_self.contiguous()), b_self))
        rows = torch.arange(3, g.n_present - 2, device="cuda")
        blocks = torch.zeros_like(p0)[3:-2], torch.zeros_like(s0)[3:-2]
        layer.project_tables(q, rows=rows, out=blocks)
        assert torch.equal(blocks[0], p0[3:-2]) and torch.equal(blocks[1], s0[3:-2])
        smp = sampling.MultiLayerNeighborSampler([6, 6])
        for i, sd, b in sampling.NodeDataLoader(g, torch.arange(60), smp, batch_size=60, relabel_input=False):
            assert torch.isfinite(model(b, GatheredRows(q, None, (p0, s0)))).all()


def test_features_are_quantised_as_the_stream_grows(ops):
    from ogl_amd.graph.snapshot_graph import SnapshotGraph
    _, _, dyn, _ = toy()
    g = dyn.get_graph()
    n, cut = g.n_present, g.cut
    view = SnapshotGraph.shared(g)
    want = ops.quantize_rows(g.feat_table)
    for present in (5, 0, n // 2, n):
        g.set_snapshot(present, min(cut, present))
        q = g.quantized_features()
        assert q.n == present and torch.equal(q.codes, want.codes[:present]) and torch.equal(q.scales, want.scales[:present])
    view.set_snapshot(7, 7)
    assert view.quantized_features().codes.data_ptr() == g.quantized_features().codes.data_ptr()
    # rows that are there are not written again: the cache grows
    q = g.quantized_features()
    q.codes[3] = 1
    assert (g.quantized_features().codes[3] == 1).all()


def test_evaluation_with_quantised_features(ops):
    """A strategy that asks for it evaluates against the tables of quantised features: the logits of a pass against those tables."""
    from ogl_amd import sampling
    from ogl_amd.graphsage import GraphSAGE
    from ogl_amd.graphsage.model import RandomHipSupervisedGraphSage
    feat_size, labels, dyn, n_classes = toy()
    g = dyn.get_graph()
    torch.manual_seed(2)
    model = GraphSAGE(feat_size, 16, n_classes, 1, F.relu, 0, "pool", edge_feats=0).cuda()
    st = RandomHipSupervisedGraphSage(model, 1, 16, labels, 5, cuda=True, batch_full=32)
    seeds = np.arange(g.n_present)
    logits = {}
    for quantized in (False, True):
        st.quantize_features = quantized
        sampling.seed(5)
        logits[quantized] = np.concatenate(st._run_custom_eval(g, None, None, seeds))
    st.quantize_features = False
    plain = g.ndata["feat"]
    with torch.no_grad():
        tables = model.layers[0].project_tables(g.quantized_features())
    original = model.layers[0].project_tables

    def given(table, rows=None, out=None):
        assert table is g.ndata["feat"] and out is not None
        at = slice(None) if rows is None else rows
        out[0].copy_(tables[0][at]), out[1].copy_(tables[1][at])
        return out
    model.layers[0].project_tables = given
    sampling.seed(5)
    want = np.concatenate(st._run_custom_eval(g, None, None, seeds))
    model.layers[0].project_tables = original
    assert plain is g.ndata["feat"]
    np.testing.assert_array_equal(logits[True], want)
    assert not np.array_equal(logits[True], logits[False])                             # (it did take another path)


@pytest.mark.parametrize("mode", ["pool", "mean", "gcn", "meanpool", "maxpool"])
@pytest.mark.parametrize("fmt,group", [("int8", None), ("e4m3", 16)])
def test_a_layer_reads_rows_in_8_bits_back(ops, mode, fmt, group):
    """Forward and loss on a table of 8-bit rows equal those on the rows it stands for."""
    from ogl_amd import sampling
    from ogl_amd.graphsage import GatheredRows, GraphSAGE
    feat_size, _, dyn, n_classes = toy()
    g = dyn.get_graph()
    torch.manual_seed(2)
    model = GraphSAGE(feat_size, 16, n_classes, 1, F.relu, 0, mode, edge_feats=0, pool_feats=9).cuda()
    q = ops.quantize_rows(g.ndata["feat"], group, fmt)
    sampling.seed(3)
    for i, sd, b in sampling.NodeDataLoader(g, torch.arange(50), sampling.MultiLayerNeighborSampler([4, 4]), batch_size=50):
        rows = ops.quant_rows_read(q, i)
        labels = ops.gather_i64(g.ndata["target"], sd.cuda())
        with torch.no_grad():
            assert torch.equal(model(b, GatheredRows(q, i)), model(b, rows))
            assert torch.equal(model.layers[0](b[0], GatheredRows(q, i)), model.layers[0](b[0], rows))
        loss = model.forward_loss(b, GatheredRows(q, i), labels)[0]
        want = model.forward_loss(b, rows, labels)[0]
        assert torch.equal(loss, want)
        loss.backward()
        assert all(torch.isfinite(p.grad).all() for p in model.parameters() if p.grad is not None)
        model.zero_grad()


@pytest.mark.parametrize("mode", ["pool", "mean"])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_layer_norm_module(ops, mode, act):
    """A layer's norm is group norm of the layer's rows: against 64 bits of those rows.  Bound: the statistics of 4 values and the affine step are a few
    float32 roundings each (64 * 2^-24 of the largest intermediate, the activation's slope at most 1.13): 256 * 2^-24 (1 + |x| rstd + |h|)."""
    from ogl_amd import sampling
    from ogl_amd.graphsage import GraphSAGE, GroupNorm
    feat_size, _, dyn, n_classes = toy()
    g = dyn.get_graph()
    torch.manual_seed(2)
    model = GraphSAGE(feat_size, 16, n_classes, 1, F.relu, 0, mode, edge_feats=0, norm=lambda width: GroupNorm(4, width, activation=act)).cuda()
    assert model.layers[1].norm is None and "layers.0.norm.weight" in model.state_dict()
    layer, norm = model.layers[0], model.layers[0].norm
    with torch.no_grad():
        norm.weight.uniform_(0.5, 1.5), norm.bias.uniform_(-1, 1)
    for i, sd, b in sampling.NodeDataLoader(g, torch.arange(50), sampling.MultiLayerNeighborSampler([4, 4]), batch_size=50):
        x = ops.gather_rows(g.ndata["feat"], i)
        taken = []
        hook = norm.register_forward_pre_hook(lambda module, args: taken.append(args[0].detach()))
        got = layer(b[0], x)
        hook.remove()
        (rows,) = taken
        want = norm_twin(rows, norm)
        v = rows.double().cpu().view(len(rows), 4, -1)
        rstd = 1 / torch.sqrt(v.var(2, unbiased=False) + norm.eps)
        spread = 1 + float((v.abs().amax(2) * rstd).max()) * 2 + 2
        assert ((got.detach().cpu().double() - want).abs() <= 256 * 2.0 ** -24 * spread * 2.5).all()
        assert torch.equal(got, ops.group_norm(rows, 4, norm.weight, norm.bias, norm.eps, act))
        got.sum().backward()
        assert norm.weight.grad is not None and layer.fc_neigh.weight.grad is not None


def test_group_norm_module_refuses():
    from ogl_amd.graphsage import GroupNorm
    for args in ((0, 8), (3, 8), (8, 0)):
        with pytest.raises(ValueError):
            GroupNorm(*args)
    with pytest.raises(ValueError):
        GroupNorm(2, 8, activation="tanh")
    m = GroupNorm(2, 8, affine=False, activation="silu")
    assert m.weight is None and "silu" in repr(m)
    with pytest.raises(ValueError):
        m(torch.zeros(3, 9))


def test_train_steps_with_a_norm_captured_and_eager(ops):
    """The strategies' captured steps replay the norm's forward and backward: the losses of the eager steps.  The same operations on rows padded to a
    bucket (their gradients are exact zeros) in another summation order: 2e-4 of the loss, as for the layers without a norm."""
    from ogl_amd import sampling
    from ogl_amd.graphsage import GraphSAGE, GroupNorm
    from ogl_amd.graphsage.model import RandomHipSupervisedGraphSage
    feat_size, labels, dyn, n_classes = toy()
    g = dyn.get_graph()
    seeds = np.random.default_rng(0).choice(g.n_present, 64, replace=False).astype(np.int64)
    losses = {}
    for graphs in (False, True):
        torch.manual_seed(9)
        model = GraphSAGE(feat_size, 16, n_classes, 1, None, 0, "pool", edge_feats=0, norm=lambda width: GroupNorm(4, width, activation="silu")).cuda()
        st = RandomHipSupervisedGraphSage(model, 4, 16, labels, 5, cuda=True, batch_full=64)
        st.use_graphs = graphs
        st.build_optimizer()
        rec = []
        st.step_hook = lambda info, rec=rec: rec.append((info["form"], float(info["loss"])))
        sampling.seed(4)
        for _ in range(3):
            st._train_batches(g, seeds, 16)
        losses[graphs] = rec
        assert all(torch.isfinite(p).all() for p in model.parameters())
        assert not torch.equal(model.layers[0].norm.weight, torch.ones(16, device="cuda"))
    assert {f for f, _ in losses[False]} == {"eager"} and "eager" not in {f for f, _ in losses[True]}
    np.testing.assert_allclose([l for _, l in losses[True]], [l for _, l in losses[False]], rtol=2e-4)


def test_every_row_entry_point_is_reached(ops):
    """Training with a norm, evaluation on quantised features and a cache written by ids call every symbol of include/ogl_rows.h."""
    from ogl_amd import _lib, sampling
    from ogl_amd.graphsage import GatheredRows, GraphSAGE, GroupNorm
    from ogl_amd.graphsage.model import RandomHipSupervisedGraphSage
    ops._norm_workspace.cache_clear()
    real, seen = _lib.lib(), set()

    class Proxy:
        def __getattr__(self, name):
            seen.add(name)
            return getattr(real, name)
    _lib._lib = Proxy()
    try:
        feat_size, labels, dyn, n_classes = toy()
        g = dyn.get_graph()
        model = GraphSAGE(feat_size, 16, n_classes, 1, None, 0, "pool", edge_feats=0, norm=lambda width: GroupNorm(4, width, activation="relu")).cuda()
        st = RandomHipSupervisedGraphSage(model, 1, 16, labels, 5, cuda=True, batch_full=32)
        st.use_graphs, st.quantize_features = False, True
        st.build_optimizer()
        st._train_batches(g, np.arange(16), 16)
        st._run_custom_eval(g, None, None, np.arange(g.n_present))
        cache = ops.quant_rows(40, feat_size)
        ids = torch.arange(300, device="cuda") % 40
        ops.quant_rows_write(cache, g.ndata["feat"][:1].expand(300, -1), slots=ids)
        GatheredRows(cache, ids).materialize()
    finally:
        _lib._lib = real
    assert set(_lib.ROW_SIGNATURES) <= seen, set(_lib.ROW_SIGNATURES) - seen


# ---- custom ops -----------------------------------------------------------------------------------------------------------------------------------
def test_custom_ops(ops):
    import ogl_amd.torch_ops  # noqa: F401
    T = torch.ops.ogl
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(40, 96, generator=gen).cuda()
    for group, fmt in ((None, "int8"), (32, "e4m3")):
        codes, scales = T.quantize_rows(x, group, fmt)
        q = ops.quantize_rows(x, group, fmt)
        assert torch.equal(codes.view(torch.int8), q.codes.view(torch.int8)) and torch.equal(scales, q.scales)
        T.quant_rows_write(codes, scales, 96, group, x[:5] * 2, torch.tensor([9, 3, 9, -1, 50]).cuda())
        ops.quant_rows_write(q, x[:5] * 2, slots=torch.tensor([9, 3, 9, -1, 50]).cuda())
        assert torch.equal(codes.view(torch.int8), q.codes.view(torch.int8)) and torch.equal(scales, q.scales)
        rows = torch.tensor([9, 0, 39]).cuda()
        assert torch.equal(T.quant_rows_read(codes, scales, 96, group, rows, torch.bfloat16), ops.quant_rows_read(q, rows, torch.bfloat16))
    codes, scales = T.quantize_rows(x)
    w, bias = ops.quantize_rows(torch.randn(33, 96, generator=gen).cuda()), torch.randn(33, generator=gen).cuda()
    assert torch.equal(T.linear_int8(codes, scales, w.codes, w.scales, 96, bias, True), ops.linear_int8(x, w, bias, True))
    xg, wt = x.clone().requires_grad_(), torch.ones(96, device="cuda", requires_grad=True)
    y = T.group_norm(xg, 6, wt, None, 1e-5, "gelu")
    assert torch.equal(y, ops.group_norm(x, 6, wt, None, activation="gelu"))
    got = torch.autograd.grad(y, (xg, wt), torch.ones_like(y))
    want = torch.autograd.grad(ops.group_norm(xg, 6, wt, None, activation="gelu"), (xg, wt), torch.ones_like(y))
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    for call in (lambda: T.group_norm(x.cpu(), 6), lambda: T.quantize_rows(x.cpu()), lambda: T.quant_rows_read(codes.cpu(), scales.cpu(), 96)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
