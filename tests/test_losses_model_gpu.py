"""GCN_BCSR.loss and the engine's steps on the losses over the class axis: the same value and gradients as
the scores' own loss, in every way a graph comes (whole, sampled blocks), and captured."""
import copy

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def _graph(nodes=3000, edges=24000, seed=5, dtype=torch.float32):
    from graph_rws_b200 import BCSRGraph
    from graph_rws_b200.data import synthetic
    g = synthetic.sym_normalized_csr(nodes, *synthetic.chung_lu_edges(nodes, edges, 2.4, seed))
    return g, BCSRGraph.from_csr(g.num_nodes, g.row_ptr, g.col_idx, g.values, device=torch.device("cuda"), values_dtype=dtype)


def _model(features, hidden, classes, layers=2, dtype=torch.float32, **kw):
    from graph_rws_b200 import GCN_BCSR
    torch.manual_seed(11)
    return GCN_BCSR(features, hidden, classes, num_layers=layers, dropout=0.0, use_checkpoint=False, **kw).cuda().to(dtype)


# The two orders of the last layer's products differ by roundings of the SpMM's operands: TF32 (2^-11) for fp32, the type
# itself otherwise; a gradient passes two such products, and every one of its entries is a sum, so norms are compared.
STEP = {torch.float32: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _close(a, b, dtype, what):
    err = float((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-30))
    assert err <= 8 * STEP[dtype], (what, err)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("classes", [7, 1203])
@pytest.mark.parametrize("residual", [False, True])
def test_loss_is_the_loss_of_the_scores(classes, dtype, residual):
    g, graph = _graph(dtype=dtype)
    model = _model(40, 64, classes, layers=3, dtype=dtype, residual=residual)
    x = torch.randn(g.num_nodes, 40, device="cuda", dtype=dtype)
    y = torch.randint(0, classes, (g.num_nodes,), device="cuda")
    rows = torch.randperm(g.num_nodes, device="cuda")[:700]
    y[rows[:50]] = -100
    for pick in (rows, slice(3, 900), None):
        labels = y if pick is None else y[pick]
        want = F.cross_entropy((model(graph, x) if pick is None else model(graph, x)[pick]).float(), labels)
        want_g = torch.autograd.grad(want, list(model.parameters()))
        got = model.loss(graph, x, labels, rows=pick)
        got_g = torch.autograd.grad(got, list(model.parameters()))
        assert abs(float(got.detach()) - float(want.detach())) <= 8 * STEP[dtype] * abs(float(want))
        for (name, _), a, b in zip(model.named_parameters(), got_g, want_g):
            _close(a, b, dtype, name)
        none = model.loss(graph, x, labels, rows=pick, reduction="none")
        assert none.shape == labels.shape and abs(float(none.detach().sum() / (labels != -100).sum()) - float(got.detach())) <= 1e-4 * abs(float(got.detach()))


def test_loss_gradient_against_dense_algebra():
    """fp64 algebra with the dense adjacency: loss and gradients of a two-layer model without normalisation's
    reordering, within the rounding of the SpMM's operands."""
    from graph_rws_b200 import BCSRGraphConv
    from graph_rws_b200.layers import linear_cross_entropy
    import numpy as np
    g, graph = _graph(500, 3000)
    A = torch.zeros(500, 500, dtype=torch.float64, device="cuda")
    r = np.repeat(np.arange(500), np.diff(g.row_ptr))
    A[torch.from_numpy(r), torch.from_numpy(g.col_idx.astype(np.int64))] = torch.from_numpy(g.values).double().cuda()
    layer = BCSRGraphConv(24, 130).cuda()
    h = torch.randn(500, 24, device="cuda", requires_grad=True)
    y = torch.randint(0, 130, (500,), device="cuda")
    x, w = layer.classifier(graph, h, features_target=h)
    got = torch.autograd.grad(linear_cross_entropy(x, w, y), (h, layer.weight_neigh, layer.weight_self))
    hd, wn, ws = (t.detach().double().requires_grad_(True) for t in (h, layer.weight_neigh, layer.weight_self))
    want = torch.autograd.grad(F.cross_entropy(A @ hd @ wn + hd @ ws, y), (hd, wn, ws))
    for a, b in zip(got, want):
        _close(a, b, torch.float32, "gradient")


def _teacher(g, classes, kept=6):
    from graph_rws_b200.helper import Distillation
    t = torch.randn(g.num_nodes, classes, generator=torch.Generator().manual_seed(3)).cuda()
    return t, Distillation.from_logits(t, kept, temperature=3.0, weight=0.25)


def _expected_distilled(model, graphs, x, rows, nodes, y, teacher, kept=6):
    logits = model(graphs, x)[rows]
    top, ids = teacher.topk(kept, dim=1)
    p = torch.softmax(top[nodes] / 3.0, 1)
    q = torch.log_softmax(logits.float() / 3.0, 1).gather(1, ids[nodes])
    soft = 9.0 * (p * (p.log() - q)).sum(1).mean()
    return 0.75 * F.cross_entropy(logits.float(), y[nodes]) + 0.25 * soft


@pytest.mark.parametrize("how", ["plain", "fused", "distill"])
def test_full_graph_steps(how):
    """train_step_full leaves the gradients of the loss it names (clipped, as all steps do); captured, the same step."""
    from graph_rws_b200.helper import graphed_full_step, train_step_full
    g, graph = _graph()
    classes = 90
    model = _model(40, 64, classes)
    x = torch.randn(g.num_nodes, 40, device="cuda")
    y = torch.randint(0, classes, (g.num_nodes,), device="cuda")
    idx = torch.randperm(g.num_nodes, device="cuda")[:1000]
    teacher, distill = _teacher(g, classes)
    kw = {"plain": {}, "fused": dict(fused_loss=True), "distill": dict(distill=distill)}[how]
    ref = copy.deepcopy(model)
    want = _expected_distilled(ref, graph, x, idx, idx, y, teacher) if how == "distill" else F.cross_entropy(ref(graph, x)[idx], y[idx])
    want.backward()
    torch.nn.utils.clip_grad_norm_(ref.parameters(), max_norm=1.0)
    loss = train_step_full(model, graph, x, y, idx, torch.optim.SGD(model.parameters(), lr=0.0), **kw)
    assert abs(float(loss) - float(want)) <= 2e-3 * abs(float(want))
    for (name, p), q in zip(model.named_parameters(), ref.parameters()):
        _close(p.grad, q.grad, torch.float32, name)
    step = graphed_full_step(model, graph, x, y, idx, torch.optim.Adam(model.parameters(), lr=0.0, capturable=True), **kw)
    first, again = float(step()), float(step())
    assert first == again and abs(first - float(loss)) <= 1e-5 * abs(first)


@pytest.mark.parametrize("how", ["fused", "distill"])
def test_sampled_steps(how):
    from graph_rws_b200.helper import graphed_sampled_step, layer0_inputs, train_epoch_node_sampling, train_step_sampled
    from graph_rws_b200.sampler import BCSRSampler
    g, graph = _graph(6000, 60000)
    classes = 300
    model = _model(40, 64, classes, layers=3)
    x = torch.randn(g.num_nodes, 40, device="cuda")
    y = torch.randint(0, classes, (g.num_nodes,), device="cuda")
    seeds = torch.randperm(g.num_nodes, device="cuda")[:256].int()
    teacher, distill = _teacher(g, classes)
    kw = dict(fused_loss=True) if how == "fused" else dict(distill=distill)
    sampler = BCSRSampler([5, 5, 5], verbose=False, seed=4)
    ref = copy.deepcopy(model)
    blocks, x0 = layer0_inputs(sampler.sample_layers(graph, seeds), x)
    nodes, rows = seeds.long(), slice(0, 256)
    want = _expected_distilled(ref, blocks, x0, rows, nodes, y, teacher) if how == "distill" else F.cross_entropy(ref(blocks, x0)[rows], y[nodes])
    want.backward()
    torch.nn.utils.clip_grad_norm_(ref.parameters(), max_norm=1.0)
    sampler = BCSRSampler([5, 5, 5], verbose=False, seed=4)
    loss = train_step_sampled(model, sampler, graph, x, y, seeds, torch.optim.SGD(model.parameters(), lr=0.0), **kw)
    assert abs(float(loss) - float(want)) <= 2e-3 * abs(float(want))
    for (name, p), q in zip(model.named_parameters(), ref.parameters()):
        _close(p.grad, q.grad, torch.float32, name)
    opt = torch.optim.Adam(model.parameters(), lr=0.0, capturable=True)
    step = graphed_sampled_step(model, BCSRSampler([5, 5, 5], verbose=False, seed=4), graph, x, y, opt, 256, **kw)
    assert abs(float(step(seeds, 0)) - float(loss)) <= 1e-4 * abs(float(loss))
    mean, seen = train_epoch_node_sampling(model, graph, x, y, nodes, opt, BCSRSampler([5, 5, 5], verbose=False, seed=4), batch_size=128, **kw)
    assert seen == 256 and torch.isfinite(mean)


def test_distillation_arguments():
    from graph_rws_b200.helper import Distillation, train_step_full
    g, graph = _graph(500, 3000)
    model = _model(16, 16, 9)
    t, d = _teacher(g, 9, kept=50)
    assert d.scores.shape == (g.num_nodes, 9) and d.ids.dtype == torch.int32      # no more scores than classes
    with pytest.raises(RuntimeError):
        Distillation(t, t[:, :2])
    with pytest.raises(ValueError):
        Distillation(t, t, weight=1.5)
    with pytest.raises(ValueError):
        train_step_full(model, graph, torch.randn(g.num_nodes, 16, device="cuda"), torch.zeros(g.num_nodes, dtype=torch.long, device="cuda"),
                        torch.arange(9, device="cuda"), torch.optim.SGD(model.parameters(), lr=0.0), fused_loss=True, distill=d)
