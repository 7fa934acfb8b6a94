"""The dense operators on tensors without elements: nothing in, nothing out, zero gradients of what is shared."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lead", [(0,), (0, 0), (0, 5), (0, 3, 0), (4, 0)])
def test_no_elements(cuda, dtype, lead):
    import gat_amd
    z = lambda *s: torch.ones(*s, dtype=dtype, device=cuda).requires_grad_(True)
    x, w, b, v = z(*lead, 24), z(6, 24), z(6), z(24)
    calls = [(gat_amd.linear_act(x, w, b, "gelu", z(*lead, 6)), (x, w, b)), (gat_amd.dropout(x, 0.5, seed=1), (x,)),
             (gat_amd.embedding(torch.zeros(lead, dtype=torch.long, device=cuda), w), (w,))]
    if lead[0] == 0:
        calls.append((gat_amd.group_norm_act(x, 4, v, v, act="elu"), (x, v)))
    else:
        with pytest.raises(ValueError, match="positions"):
            gat_amd.group_norm_act(x, 4, v, v)
    for y, leaves in calls:
        assert y.shape[:-1] == lead and y.numel() == 0
        for g, t in zip(torch.autograd.grad(y, leaves, torch.zeros_like(y)), leaves):
            assert g.shape == t.shape and not g.any()
    with torch.no_grad():
        assert gat_amd.linear_act(x, w).shape == lead + (6,)
        if lead[0] == 0:
            assert gat_amd.group_norm_act(x, 4, v, v).shape == x.shape
