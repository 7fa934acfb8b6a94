"""The networks' stock path of norm="group": elementary operations, equal to torch's group norm with its gradients, and
never torch's own group norm, whose parameter gradients are wrong on the GPU for [N, C] with N > 128."""
import pytest
import torch
import torch.nn.functional as F


@pytest.mark.parametrize("n", [0, 1, 5, 300])
def test_equals_torch_on_the_cpu(n):
    from gat_amd.dense import stock_group_norm
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, 24, generator=g, dtype=torch.float64, requires_grad=True)
    norm = torch.nn.GroupNorm(8, 24).double()
    with torch.no_grad():
        for p in norm.parameters():
            p.add_(torch.randn(24, generator=g, dtype=torch.float64))
    dy = torch.randn(n, 24, generator=g, dtype=torch.float64)
    leaves = [x, norm.weight, norm.bias]
    a = torch.autograd.grad(stock_group_norm(x, norm), leaves, dy)
    torch.testing.assert_close(stock_group_norm(x.t().contiguous().t(), norm), stock_group_norm(x, norm), rtol=1e-12, atol=1e-12)
    if n == 0:
        assert not a[1].any() and not a[2].any()
        return
    y = norm(x)
    torch.testing.assert_close(stock_group_norm(x, norm), y, rtol=1e-9, atol=1e-9)
    for p, q in zip(a, torch.autograd.grad(y, leaves, dy)):
        torch.testing.assert_close(p, q, rtol=1e-8, atol=1e-8)


def test_the_partitioned_network_does_not_call_torchs(monkeypatch):
    from test_dist_cpu import OracleBackend
    from gat_amd.dist import PartitionedGAT
    model = PartitionedGAT(9, 3, hidden_dim=4, dropout=0.0, backend=OracleBackend(), norm="group").double().train()
    assert not model.fused
    x = torch.randn(200, 32, dtype=torch.float64, generator=torch.Generator().manual_seed(2))
    want = F.elu(model.bn1(x))

    def refuse(*a, **k):
        raise AssertionError("F.group_norm called")
    monkeypatch.setattr(F, "group_norm", refuse)
    torch.testing.assert_close(model._glue(x, model.bn1, 200), want, rtol=1e-9, atol=1e-9)


@pytest.mark.gpu
def test_partitioned_stock_path_gradients_on_the_gpu(cuda):
    """300 rows in f32 on the GPU against 64 bits: sums of at most 300 terms, 300 U = 2e-5 of the terms' sizes"""
    from test_dist_cpu import OracleBackend
    from gat_amd.dist import PartitionedGAT
    torch.manual_seed(1)
    model = PartitionedGAT(9, 3, hidden_dim=4, dropout=0.0, backend=OracleBackend(), norm="group", fused=False).train().to(cuda)
    g = torch.Generator().manual_seed(5)
    x, dy = torch.randn(300, 32, generator=g), torch.randn(300, 32, generator=g)
    got = torch.autograd.grad(model._glue(x.to(cuda), model.bn1, 300), list(model.bn1.parameters()), dy.to(cuda))
    ref = torch.nn.GroupNorm(8, 32).double()
    ref.load_state_dict({k: v.cpu().double() for k, v in model.bn1.state_dict().items()})
    want = torch.autograd.grad(F.elu(ref(x.double())), list(ref.parameters()), dy.double())
    size = float((dy.abs() * 4).sum(0).max())
    for a, b in zip(got, want):
        assert float((a.cpu().double() - b).abs().max()) < 2e-5 * size
