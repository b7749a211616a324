"""train_step_full_sharded with ``fused_loss`` on gloo ranks on the CPU: loss and gradients of the single-process step.  The product
kernel and the loss are CUDA-only: the CPU oracle and the loss of the scores take their places; the step, the layer,
its autograd functions, the sharded graph and the collectives are the shipped code."""
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
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        import scipy.sparse as sps
        import oracle
        from graph_rws_b200 import BCSRGraph, core
        from graph_rws_b200.helper import train_step_full_sharded
        from graph_rws_b200.layers import BCSRGraphConv
        from graph_rws_b200.parallel import RowShardedGraph, partition_windows_by_tiles, shard_bcsr

        def cpu_spmm(wo, cols, vals, dense, **kw):
            return torch.from_numpy(oracle.spmm_fwd(wo.numpy(), cols.numpy(), vals.float().numpy(),
                                                    dense.detach().float().numpy())).to(dense.dtype)
        core.spmm_raw = cpu_spmm
        n, classes = 333, 5                            # the last window is partial
        rng = np.random.default_rng(5)
        A = (sps.random(n, n, density=0.03, random_state=7, format="csr", dtype=np.float32) + sps.eye(n, dtype=np.float32, format="csr")).tocsr()
        A.sort_indices()
        At = A.T.tocsr()
        At.sort_indices()

        def graph_of(m):
            wo, cols, vals = oracle.csr_to_bcsr(n, m.indptr.astype(np.int64), m.indices.astype(np.int32), m.data.astype(np.float32))
            return BCSRGraph(num_nodes=n, num_edges=None, tile_rows=16, tile_cols=8, window_offset=torch.from_numpy(wo),
                             original_col_indices=torch.from_numpy(cols), values_condensed=torch.from_numpy(vals), device=torch.device("cpu"))
        g, gt = graph_of(A), graph_of(At)

        class Model(torch.nn.Module):
            def __init__(self):
                super().__init__()
                self.first, self.last = BCSRGraphConv(24, 16), BCSRGraphConv(16, classes)

            def loss(self, graph, features, labels, rows=None, reduction="mean"):
                h = torch.relu(self.first(graph, features, features_target=features))
                x, w = self.last.classifier(graph, h, features_target=h, rows=rows)
                return torch.nn.functional.cross_entropy(x @ w, labels, reduction=reduction)
        torch.manual_seed(3)
        model = Model()
        X = torch.from_numpy(rng.standard_normal((n, 24)).astype(np.float32)).requires_grad_(True)
        y = torch.from_numpy(rng.integers(0, classes, n))
        keep = torch.arange(0, n, 3)
        # the whole graph by dense algebra
        D = torch.from_numpy(A.toarray())
        h = torch.relu(D @ X @ model.first.weight_neigh + X @ model.first.weight_self)
        scores = (D @ h @ model.last.weight_neigh + h @ model.last.weight_self)[keep]
        want = torch.nn.functional.cross_entropy(scores, y[keep])
        grads = torch.autograd.grad(want, list(model.parameters()))
        norm = torch.cat([v.reshape(-1) for v in grads]).norm()
        grads = [v * min(1.0, 1.0 / (float(norm) + 1e-6)) for v in grads]
        part = partition_windows_by_tiles(g.window_offset, world, num_rows=n)
        lo, hi = part.rows(rank)

        def shard(graph):
            wo, cols, vals = shard_bcsr(graph.window_offset, graph.original_col_indices, graph.values_condensed, part, rank)
            return BCSRGraph(num_nodes=hi - lo, num_edges=None, tile_rows=16, tile_cols=8, window_offset=wo, original_col_indices=cols,
                             values_condensed=vals, device=torch.device("cpu"), num_rows=hi - lo, num_cols=n)
        sharded = RowShardedGraph(shard(g), part, rank, local_t=RowShardedGraph(shard(gt), part, rank))
        mine = keep[(keep >= lo) & (keep < hi)] - lo
        loss = train_step_full_sharded(model, sharded, X[lo:hi].detach().contiguous().requires_grad_(True), y[lo:hi], mine, keep.numel(),
                                       torch.optim.SGD(model.parameters(), lr=0.0), fused_loss=True).clone()
        dist.all_reduce(loss)                  # (a step returns its rank's share)
        assert abs(float(loss) - float(want)) <= 1e-4 * float(want)
        for p, v in zip(model.parameters(), grads):
            assert torch.allclose(p.grad, v, rtol=2e-3, atol=1e-4)
        out[rank] = 1
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 3])
def test_fused_step_of_row_shards_matches_the_whole_graph(world):
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
