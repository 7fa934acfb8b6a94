"""The dense operators under torch's transformations: what they cannot take part in is refused, never answered with a
result that lost its tangent or a trace of uninitialised memory."""
import pytest
import torch
import torch.autograd.forward_ad as fwad


def calls(device):
    """(name, function of its operands, the operands)"""
    import gat_amd
    g = torch.Generator().manual_seed(1)
    t = lambda *s: torch.randn(*s, generator=g).to(device)
    ids = torch.tensor([0, 2, 1]).to(device)
    x, w, b, r, v = t(6, 8), t(4, 8), t(4), t(6, 4), t(8)
    return [
        ("linear_act", lambda *a: gat_amd.linear_act(a[0], a[1], a[2], "gelu", a[3]), [x, w, b, r]),
        ("group_norm_act", lambda *a: gat_amd.group_norm_act(a[0], 2, a[1], a[2]), [x, v, v + 1]),
        ("embedding", lambda *a: gat_amd.embedding(ids, a[0]), [w]),
        ("dropout", lambda *a: gat_amd.dropout(a[0], 0.5, seed=3, residual=a[1]), [x, x + 1]),
    ]


def refusals(device):
    for name, f, operands in calls(device):
        for grad in (False, True):
            for i in range(len(operands)):
                with fwad.dual_level():
                    ops = [o.clone().requires_grad_(grad) for o in operands]
                    ops[i] = fwad.make_dual(operands[i].clone(), torch.ones_like(operands[i]))
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        f(*ops)
            with pytest.raises(RuntimeError, match="torch.jit.trace"):
                torch.jit.trace(f, tuple(o.clone().requires_grad_(grad) for o in operands), check_trace=False)


def test_tangents_and_traces_are_refused():
    refusals("cpu")


@pytest.mark.gpu
def test_tangents_and_traces_are_refused_on_the_gpu(cuda):
    refusals(cuda)
    import gat_amd
    x = torch.randn(4, 8, device=cuda)
    with fwad.dual_level():         # dropout that is off hands its operand back, tangent and all
        d = fwad.make_dual(x, torch.ones_like(x))
        for y in (gat_amd.dropout(d, 0.0), gat_amd.dropout(d, 0.5, training=False)):
            assert torch.equal(fwad.unpack_dual(y).tangent, torch.ones_like(x))
    for name, f, operands in calls(cuda):       # nothing is left behind: the same calls without either
        f(*operands)
