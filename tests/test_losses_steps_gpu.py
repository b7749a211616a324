"""What the losses over the class axis share with the rest of a step: the SpMM's recorded times, the pipelined sampled step, and
steps of row-sharded graphs (one rank: the whole graph is its shard)."""
import copy

import pytest
import torch
import torch.nn.functional as F

from test_losses_model_gpu import STEP, _close, _graph, _model

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


@pytest.mark.parametrize("how", ["fused", "distill"])
def test_pipelined_sampled_steps(how):
    """The pipelined step returns the losses of the batches in order, the same as the plain captured step's."""
    from graph_rws_b200.helper import Distillation, graphed_sampled_step
    from graph_rws_b200.sampler import BCSRSampler
    g, graph = _graph(6000, 60000)
    classes = 300
    x = torch.randn(g.num_nodes, 40, device="cuda")
    y = torch.randint(0, classes, (g.num_nodes,), device="cuda")
    batches = [torch.randperm(g.num_nodes, device="cuda")[:256].int() for _ in range(4)]
    teacher = torch.randn(g.num_nodes, classes, device="cuda")
    kw = dict(fused_loss=True) if how == "fused" else dict(distill=Distillation.from_logits(teacher, 6, temperature=3.0, weight=0.25))
    losses = []
    for pipelined in (False, True):
        model = _model(40, 64, classes, layers=3)
        opt = torch.optim.Adam(model.parameters(), lr=0.0, capturable=True)
        step = graphed_sampled_step(model, BCSRSampler([5, 5, 5], verbose=False, seed=4), graph, x, y, opt, 256, pipelined=pipelined, **kw)
        if pipelined:
            step.prime(batches[0], 0)
            got = [float(step(batches[i + 1], i + 1)) for i in range(3)]
        else:
            got = [float(step(batches[i], i)) for i in range(3)]
        losses.append(got)
    assert len(set(losses[0])) == 3
    assert all(abs(a - b) <= 1e-5 * abs(a) for a, b in zip(*losses))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_row_sharded_steps_with_a_fused_loss(dtype):
    """A shard that is the whole graph: the step's loss is the mean over the training rows, and its gradients are the whole graph's."""
    from graph_rws_b200.helper import graphed_full_step, train_step_full, train_step_full_sharded
    from graph_rws_b200.parallel import RowShardedGraph, partition_windows_by_tiles
    g, graph = _graph(dtype=dtype)
    classes = 230
    model = _model(40, 64, classes, layers=3, dtype=dtype)
    ref = copy.deepcopy(model)
    x = torch.randn(g.num_nodes, 40, device="cuda", dtype=dtype)
    y = torch.randint(0, classes, (g.num_nodes,), device="cuda")
    idx = torch.randperm(g.num_nodes, device="cuda")[:1000]
    y[idx[:10]] = -100                     # counted by the caller's number of training rows, not by the sum
    shard = RowShardedGraph.from_full(graph, partition_windows_by_tiles(graph.window_offset, 1, num_rows=g.num_nodes), 0, dtype=dtype)
    want = F.cross_entropy(ref(graph, x)[idx].float(), y[idx], reduction="sum") / 1000
    want.backward()
    torch.nn.utils.clip_grad_norm_(ref.parameters(), max_norm=1.0)
    sgd = torch.optim.SGD(model.parameters(), lr=0.0)
    loss = train_step_full_sharded(model, shard, x, y, idx, 1000, sgd, fused_loss=True)
    assert abs(float(loss) - float(want.detach())) <= 2.0 ** -7 * abs(float(want.detach()))
    # The whole graph takes its first layer's products in the other order, so pre-activations differ by 2 STEP of their size
    # (both operands of a product are rounded), and a ReLU's input that is nearer to 0 than that may change sides: of normalised
    # rows a share of 2 phi(0) 2 STEP <= 1.6 STEP per layer, two layers.  A side changed is an entry of the gradient lost, so norms
    # differ by the root of that share besides the 8 STEP of the roundings themselves.
    for (name, p), q in zip(model.named_parameters(), ref.parameters()):
        err = float((p.grad.double() - q.grad.double()).norm() / q.grad.double().norm())
        assert err <= 8 * STEP[dtype] + (2 * 1.6 * STEP[dtype]) ** 0.5, (name, err)
    # the shard's own scores take all layers but the last one in the same order: the same bits up to there
    ref.zero_grad(set_to_none=True)
    (F.cross_entropy(ref(shard, x)[idx].float(), y[idx], reduction="sum") / 1000).backward()
    torch.nn.utils.clip_grad_norm_(ref.parameters(), max_norm=1.0)
    for (name, p), q in zip(model.named_parameters(), ref.parameters()):
        _close(p.grad, q.grad, dtype, name)
    grads = [p.grad.clone() for p in model.parameters()]
    # Without ignored rows it is the whole graph's step, whose first layer takes its products in the other order: three layers of two
    # rounded operands each move a score by 6 STEP of its size at most, and a row's loss by at most twice what its scores move by.
    kept = idx[10:]
    whole = float(train_step_full(model, graph, x, y, kept, sgd, fused_loss=True))
    assert abs(float(train_step_full_sharded(model, shard, x, y, kept, 990, sgd, fused_loss=True)) - whole) <= 12 * STEP[dtype] * whole
    step = graphed_full_step(model, shard, x, y, idx, torch.optim.Adam(model.parameters(), lr=0.0, capturable=True), num_train=1000, fused_loss=True)
    first, again = float(step()), float(step())
    assert first == again and abs(first - float(loss)) <= 1e-5 * abs(first)
    for p, q in zip(model.parameters(), grads):
        _close(p.grad, q, dtype, "captured")
