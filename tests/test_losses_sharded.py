"""BCSRGraphConv.classifier on row-sharded graphs: gloo ranks on the CPU against the single-process result."""
import os
import socket

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _worker(rank, world, port, out):
    """The product kernel is CUDA-only: the CPU oracle takes its place; the layer, its autograd function, the
    sharded graph and the gathers of both directions are the shipped code."""
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        import scipy.sparse as sps
        import oracle
        from graph_rws_b200 import BCSRGraph, core
        from graph_rws_b200.layers import BCSRGraphConv
        from graph_rws_b200.parallel import RowShardedGraph, partition_windows_by_tiles, shard_bcsr

        def cpu_spmm(wo, cols, vals, dense, **kw):
            return torch.from_numpy(oracle.spmm_fwd(wo.numpy(), cols.numpy(), vals.float().numpy(),
                                                    dense.detach().float().numpy())).to(dense.dtype)
        core.spmm_raw = cpu_spmm
        n = 333                                        # the last window is partial
        rng = np.random.default_rng(5)
        A = (sps.random(n, n, density=0.03, random_state=7, format="csr", dtype=np.float32) + sps.eye(n, dtype=np.float32, format="csr")).tocsr()
        A.sort_indices()

        def graph_of(m):
            wo, cols, vals = oracle.csr_to_bcsr(n, m.indptr.astype(np.int64), m.indices.astype(np.int32), m.data.astype(np.float32))
            return BCSRGraph(num_nodes=n, num_edges=None, tile_rows=16, tile_cols=8, window_offset=torch.from_numpy(wo),
                             original_col_indices=torch.from_numpy(cols), values_condensed=torch.from_numpy(vals), device=torch.device("cpu"))
        At = A.T.tocsr()
        At.sort_indices()
        g, gt = graph_of(A), graph_of(At)
        g._shared[("T", n, torch.float32)] = (g._versions(), gt)
        torch.manual_seed(3)
        layer = BCSRGraphConv(24, 5)
        params = list(layer.parameters())
        for p in params:
            dist.broadcast(p.data, 0)
        X = torch.from_numpy(rng.standard_normal((n, 24)).astype(np.float32))
        y = torch.from_numpy(rng.integers(0, 5, n))

        def run(graph, h, labels, rows):
            h = h.clone().requires_grad_(True)
            x, w = layer.classifier(graph, h, features_target=h, rows=rows)
            loss = torch.nn.functional.cross_entropy(x @ w, labels[rows], reduction="sum")
            return (loss.detach(), (x @ w).detach()) + torch.autograd.grad(loss, [h] + params)

        keep = torch.arange(0, n, 3)
        full = run(g, X, y, keep)
        dense = torch.from_numpy(A.toarray())
        scores = dense @ X @ layer.weight_neigh.detach() + X @ layer.weight_self.detach()
        assert torch.allclose(full[1], scores[keep], rtol=1e-4, atol=1e-4)
        part = partition_windows_by_tiles(g.window_offset, world, num_rows=n)
        lo, hi = part.rows(rank)

        def shard(graph):
            wo, cols, vals = shard_bcsr(graph.window_offset, graph.original_col_indices, graph.values_condensed, part, rank)
            return BCSRGraph(num_nodes=hi - lo, num_edges=None, tile_rows=16, tile_cols=8, window_offset=wo, original_col_indices=cols,
                             values_condensed=vals, device=torch.device("cpu"), num_rows=hi - lo, num_cols=n)
        sharded = RowShardedGraph(shard(g), part, rank, local_t=RowShardedGraph(shard(gt), part, rank))
        mine = keep[(keep >= lo) & (keep < hi)] - lo
        got = run(sharded, X[lo:hi].contiguous(), y[lo:hi], mine)
        assert torch.allclose(got[1], full[1][(keep >= lo) & (keep < hi)], rtol=1e-4, atol=1e-5)
        assert torch.allclose(got[2], full[2][lo:hi], rtol=1e-3, atol=1e-4)
        for a, b in zip(got[3:], full[3:]):
            total = a.clone()
            dist.all_reduce(total)
            assert torch.allclose(total, b, rtol=1e-3, atol=1e-4)
        out[rank] = 1
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 3])
def test_classifier_of_row_shards_matches_the_single_process(world):
    ctx = mp.get_context("spawn")
    out = ctx.Array("i", world)
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, world, port, out)) for r in range(world)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(timeout=240)
    for p in procs:
        if p.is_alive():
            p.kill()
            p.join()
    assert all(p.exitcode == 0 for p in procs) and list(out) == [1] * world
