"""The row operators under two ranks (gloo rendezvous, both on cuda:0): per-pass tables of 8-bit features, projected by vertex range and exchanged, and a
layer's group norm in the gradient exchange, each against one rank on the same seeds."""
import os
import random
import sys

import numpy as np
import pytest
import torch

from test_gpu_parallel import _free_port

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run(rank, world, port, out_path):
    sys.path.insert(0, ROOT)
    import torch.distributed as dist
    import torch.nn.functional as F
    import ogl_amd  # noqa: F401
    from ogl_amd import sampling, synthetic
    from ogl_amd.graph import TrainTestGraph
    from ogl_amd.graphsage import GraphSAGE, GroupNorm
    from ogl_amd.graphsage.model import RandomHipSupervisedGraphSage
    if world > 1:
        os.environ["MASTER_ADDR"] = "127.0.0.1"; os.environ["MASTER_PORT"] = str(port)
        dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.cuda.set_device(0)
    np.random.seed(3); random.seed(3); torch.manual_seed(3); sampling.seed(3)     # identical on every rank
    feat_size, labels, graph, n_classes, graph_test = synthetic.load("toy", device="cuda")
    gu = TrainTestGraph(graph, split=0.15, start_prior_alpha=4, end_prior_alpha=50, scale=1, max_priority=10)
    for _ in range(3):
        gu.evolve()
    g = gu.get_graph()
    model = GraphSAGE(feat_size, 8, n_classes, 1, F.relu, 0, "pool", edge_feats=0, norm=lambda width: GroupNorm(2, width)).cuda()
    st = RandomHipSupervisedGraphSage(model, 2, 7, labels, 5, cuda=True, batch_full=32)
    st.build_optimizer()
    # plain SGD for the comparison: Adam turns the summation-order noise of a near-zero gradient into a full lr step
    st.optimizer = torch.optim.SGD(model.parameters(), lr=0.05)
    assert (st.gsync is not None) == (world > 1)
    id2s, s2id = gu.get_original_to_subgraph_map(), gu.get_subgraph_to_original_map()
    res = {}
    st.quantize_features = True
    model.eval()
    seeds = np.arange(g.n_present)
    for partition in (False, True):
        st.partition_features = partition
        with torch.no_grad():
            P, S = st._projection_tables(g, model.layers[0])
        res["tables", partition] = [t[:g.n_present].cpu().clone() for t in (P, S)]
        sampling.seed(5)
        res["confusion", partition] = st._eval_confusion(g, s2id, id2s, seeds)
    fixed = np.asarray(sorted(gu.get_train_set()))[:14]                    # 2 batches of 7: 4 + 3 by rank
    model.train()
    sampling.seed(6)
    st._run_custom_train(g, s2id, id2s, id2s[fixed], gu)
    res["params"] = {k: p.detach().cpu().clone() for k, p in model.named_parameters()}
    if world > 1:
        mine = torch.cat([p.reshape(-1) for p in res["params"].values()])
        other = [torch.empty_like(mine) for _ in range(world)]
        dist.all_gather(other, mine)
        assert all(torch.equal(o, other[0]) for o in other)
        dist.barrier()
        dist.destroy_process_group()
    if rank == 0:
        torch.save(res, out_path)


def test_two_ranks_match_one_rank(tmp_path):
    import torch.multiprocessing as mp
    ctx = mp.get_context("spawn")
    one, two = str(tmp_path / "one.pt"), str(tmp_path / "two.pt")
    p = ctx.Process(target=_run, args=(0, 1, 0, one)); p.start(); p.join(100)
    assert p.exitcode == 0
    port = _free_port()
    procs = [ctx.Process(target=_run, args=(r, 2, port, two)) for r in range(2)]
    for q in procs:
        q.start()
    for q in procs:
        q.join(100)
    assert [q.exitcode for q in procs] == [0, 0]
    a, b = torch.load(one, weights_only=False), torch.load(two, weights_only=False)
    for partition in (False, True):                                        # (exact sums: the same bits whoever projects a row)
        for x, y in zip(a["tables", False], b["tables", partition]):
            assert torch.equal(x, y)
        (cm1, n1), (cm2, n2) = a["confusion", False], b["confusion", partition]
        assert n1 == n2 and np.array_equal(cm1, cm2)
    assert any("norm" in k for k in a["params"])
    for k, v in a["params"].items():
        torch.testing.assert_close(v, b["params"][k], rtol=1e-4, atol=1e-5)
