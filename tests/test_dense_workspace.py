"""linear_act's backward asks for the workspace that the gradients asked for need, and no more."""
import ctypes as C

import pytest
import torch

from gat_amd import _lib

MB = 1 << 20


def test_sizes():
    lib = _lib.lib()
    of = lambda d, *want: lib.gatmi_linear_bwd_workspace_bytes_of(C.byref(d), *want)
    d = _lib.Linear(100, 8192, 8192, 0, 2)               # one split: dW and db are written by the product itself
    image = 8192 * 8192 * 6
    assert of(d, 0, 1, 1) == 0 and of(d, 0, 1, 0) == 0 and of(d, 0, 0, 0) == 0
    assert image <= of(d, 1, 1, 1) < image + MB
    assert 0 < of(d, 0, 0, 1) < MB
    d = _lib.Linear(1 << 20, 256, 128, 1, 0)             # many splits
    slab = 256 * 128 * 4
    assert of(d, 0, 1, 0) >= 2 * slab and of(d, 0, 1, 0) % slab == 0
    assert 0 < of(d, 0, 0, 1) < MB
    for d in (d, _lib.Linear(300, 64, 2000, 2, 4), _lib.Linear(1, 1, 1, 0, 0), _lib.Linear(0, 5, 7, 0, 1)):
        every = [of(d, x, w, b) for x in (0, 1) for w in (0, 1) for b in (0, 1)]
        assert max(every) <= lib.gatmi_linear_bwd_workspace_bytes(C.byref(d))
        # too small a one is refused before anything is launched
        for x in (0, 1):
            for w in (0, 1):
                for b in (0, 1):
                    need = of(d, x, w, b)
                    if need:
                        args = [256 if v else None for v in (x, w, b)]
                        assert lib.gatmi_linear_bwd(C.byref(d), 256, 256, 256, 256, *args, 256, need - 1, None) == 4
                        assert lib.gatmi_linear_bwd(C.byref(d), 256, 256, 256, 256, *args, None, need, None) == 4
    bad = _lib.Linear(-1, 8, 8, 0, 0)
    assert of(bad, 1, 1, 1) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(100, 300, 200), (5000, 300, 140), (40, 64, 1200), (0, 5, 7), (200, 5, 6)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_choice_of_gradients(cuda, dtype, m, k, n):
    """each subset of the gradients is what all of them together give, bit for bit"""
    import gat_amd
    g = torch.Generator().manual_seed(m)
    x, w, b, r = (torch.randn(*s, generator=g).to(dtype).to(cuda) for s in ((m, k), (n, k), (n,), (m, n)))
    dy = torch.randn(m, n, generator=g).to(dtype).to(cuda)
    every = None
    for which in range(15, 0, -1):
        ts = [t.clone().requires_grad_(bool(which >> i & 1)) for i, t in enumerate((x, w, b, r))]
        y = gat_amd.linear_act(ts[0], ts[1], ts[2], "gelu", ts[3])
        got = torch.autograd.grad(y, [t for t in ts if t.requires_grad], dy)
        if every is None:
            every = got
        at = [i for i in range(4) if which >> i & 1]
        assert all(torch.equal(a, every[i]) for a, i in zip(got, at)), which


@pytest.mark.gpu
def test_memory_of_a_large_weight(cuda):
    """frozen x, 8192 x 8192 weights, one split: the backward holds dW and the slope's product, no second copy of dW"""
    import gat_amd
    x = torch.randn(64, 8192, device=cuda)
    w = (torch.randn(8192, 8192, device=cuda) / 90).requires_grad_(True)
    y = gat_amd.linear_act(x, w, act="elu")
    dy = torch.randn_like(y)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    torch.autograd.grad(y, w, dy)
    assert torch.cuda.max_memory_allocated() - before < 8192 * 8192 * 4 + 64 * MB
    r = torch.randn(64, 8192, device=cuda, requires_grad=True)
    before = torch.cuda.memory_allocated()
    y = gat_amd.linear_act(x * 2, w.detach() * 2, residual=r)       # only the residual: neither factor is kept
    assert torch.cuda.memory_allocated() - before < 16 * MB
