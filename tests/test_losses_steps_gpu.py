"""What the losses over the class axis share with the rest of a step: the SpMM's recorded times, the pipelined sampled step, and
steps of row-sharded graphs (one rank: the whole graph is its shard)."""
import copy

import pytest
import torch
import torch.nn.functional as F

from test_losses_model_gpu import _close, _graph, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [40, 37])
def test_spmm_times_of_a_fused_loss(width):
    """With timing on every layer's product is timed, the last one's too, at widths that are padded as well."""
    from graph_rws_b200 import core
    from graph_rws_b200.helper import reset_spmm_timings, spmm_timings
    g, graph = _graph()
    model = _model(24, width, 90)
    x = torch.randn(g.num_nodes, 24, device="cuda")
    y = torch.randint(0, 90, (g.num_nodes,), device="cuda")
    want = model.loss(graph, x, y)
    core.set_spmm_timing(True)
    try:
        reset_spmm_timings()
        got = model.loss(graph, x, y)
        times = spmm_timings()
    finally:
        core.set_spmm_timing(False)
        reset_spmm_timings()
    assert len(times) == 2 and all(t > 0.0 for t in times)
    assert abs(float(got.detach()) - float(want.detach())) <= 2e-3 * abs(float(want.detach()))
    model.loss(graph, x, y)
    assert spmm_timings() == [0.0, 0.0]
    reset_spmm_timings()
