"""gat_amd.model.GAT with the dense operators: norm="group", skip=True, embedding=(entries, dim)."""
import copy

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from gat_amd.data import Data, convert_to_graph, synthetic_traces

pytestmark = pytest.mark.gpu


def graph_data(n=400, seed=5, columns=2):
    import cases
    ei, n = cases.knn_graph(n=n, f=25, seed=seed)
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(-1, 40, (n, columns), generator=g)
    return Data(torch.rand(n, 25, generator=g), ei, torch.randint(0, 2, (n,), generator=g), ids)


def make(cuda, **kw):
    from gat_amd.model import GAT
    torch.manual_seed(3)
    kw = dict(dict(dropout=0.0, hidden_dim=30, lr=0.05, device=cuda, verbose=False), **kw)
    return GAT(torch.optim.SGD, 25, 2, **kw)


def test_default_network_is_unchanged(cuda):
    m = make(cuda)
    assert sorted({k.split(".")[0] for k in m.state_dict()}) == ["bn1", "bn2", "conv1", "conv2", "conv3"]
    assert isinstance(m.bn1, torch.nn.BatchNorm1d) and m.conv1.in_channels == 25


@pytest.mark.parametrize("kw", [dict(norm="group"), dict(skip=True), dict(embedding=(40, 6, 2)),
                                dict(norm="group", skip=True, embedding=(40, 6, 2))])
def test_fused_operators_match_stock_modules(cuda, kw):
    """loss and every gradient with the fused operators == with the stock modules (fused_glue = False), dropout
    off.  Both are f32 with sums of at most 400 x 240 terms in different orders: within 100 U = 6e-6 of a
    result's largest value each, so 2e-5 between them; the layer biases in front of a BatchNorm have gradients
    whose batch part cancels (2e-4 there, as for the fused BatchNorm)."""
    data = graph_data()
    a = make(cuda, **kw)
    if a.table is not None:      # the stock lookup has no row for "none"
        data.ids.clamp_(min=0)
    b = copy.deepcopy(a)
    b.fused_glue = False
    losses = []
    for m in (a, b):
        m.train()
        out = m(data)
        loss = F.nll_loss(out, data.y.to(cuda))
        loss.backward()
        losses.append(float(loss.detach()))
    assert abs(losses[0] - losses[1]) < 1e-5 * max(abs(losses[1]), 1.0)
    grads = {name: p.grad for name, p in b.named_parameters()}
    for (name, pa), (_, pb) in zip(a.named_parameters(), b.named_parameters()):
        ref = pb.grad
        # att_dst: d att_dst = sum_e dz_e h[dst(e)], d att_src = sum_e dz_e h[src(e)] over the same edges.  The
        # softmax makes dz sum to 0 over a destination's edges (up to LeakyReLU's slopes), where h[dst] is one
        # vector: what is left is a rest of summands |dz_e| |h| whose sum, which the n U bound of an f32 sum
        # refers to, is at least |d att_src|
        size = max(float(ref.abs().max()), 1e-6)
        if name.endswith("att_dst"):
            size = max(size, float(grads[name.replace("att_dst", "att_src")].abs().max()))
        loose = a.norm == "batch" and name in ("conv1.bias", "conv2.bias", "skip1.bias", "skip2.bias")
        atol = (2e-4 if loose else 2e-5) * size
        torch.testing.assert_close(pa.grad, ref, rtol=2e-5, atol=atol, msg=lambda m, name=name: f"{name}: {m}")
    a.eval(), b.eval()
    with torch.no_grad():
        torch.testing.assert_close(a(data), b(data), rtol=2e-5, atol=2e-5)


def test_training_with_everything_on(cuda, tmp_path, monkeypatch):
    """eager and replayed training with dropout run, stay finite and give every parameter a gradient"""
    monkeypatch.chdir(tmp_path)
    X, y = synthetic_traces(1200, 25, seed=5)
    sets = [convert_to_graph(X[:900], y[:900]), convert_to_graph(X[900:], y[900:])]
    for d in sets:
        d.ids = torch.randint(-1, 50, (d.num_nodes,), generator=torch.Generator().manual_seed(1))
    for hipgraph in (False, True):
        m = make(cuda, dropout=0.3, norm="group", skip=True, embedding=(50, 4), epochs=6, lr=0.02, patience=50,
                 hipgraph=hipgraph)
        metrics = m.train_model(*sets)
        assert all(np.isfinite(metrics.train_loss)) and len(set(metrics.train_loss)) == 6
        assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in m.parameters())
        pred = m.test_model(sets[1])
        assert pred.shape == (300,) and pred.dtype == torch.int64


def test_replayed_training_equals_eager(cuda, tmp_path, monkeypatch):
    """without dropout, bit for bit, group norm, skips and the sorted embedding gradient included"""
    monkeypatch.chdir(tmp_path)
    data = graph_data(n=700)
    curves = []
    for hipgraph in (False, True):
        m = make(cuda, norm="group", skip=True, embedding=(40, 6, 2), hipgraph=hipgraph)
        curves.append([m.train_epoch(data)[0] for _ in range(6)])
    assert curves[0] == curves[1]


def test_refusals(cuda):
    with pytest.raises(ValueError, match="norm"):
        make(cuda, norm="layer")
    with pytest.raises(ValueError, match="ids"):
        d = graph_data()
        d.ids = None
        make(cuda, embedding=(40, 6, 2))(d)


def test_codes_of_none_on_stock_modules(cuda):
    """-1 and codes past the table are zero features, without a gradient, on the stock modules too"""
    data = graph_data()
    data.ids[5, 0] = 40
    a = make(cuda, embedding=(40, 6, 2))
    b = copy.deepcopy(a)
    b.fused_glue = False
    dev = a._on_device(data)
    x = [m._features(dev) for m in (a, b)]
    assert torch.equal(x[0], x[1])
    none = (data.ids < 0) | (data.ids >= 40)
    assert not x[1][:, 25:].detach().cpu().view(-1, 2, 6)[none].any()
    up = torch.randn(x[0].shape, generator=torch.Generator().manual_seed(1)).to(cuda)
    grads = [torch.autograd.grad(v, m.table.weight, up)[0] for v, m in zip(x, (a, b))]
    # sums of at most 800 f32 terms in another order: 800 U = 5e-5 of the terms' sizes
    torch.testing.assert_close(grads[0], grads[1], rtol=0, atol=5e-5 * float(up.abs().max()) * 40)
