"""PartitionedGAT(norm="group") over gloo on the CPU stand-in backend: the network with group norms between the
layers equals the single-process one, log-probabilities and every gradient, in training and evaluation."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
import torch.nn.functional as F

import cases
from oracle import gat_oracle as O
from test_dist_cpu import OracleBackend


def _worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from gat_amd.dist import PartitionedGAT
        torch.set_num_threads(1)
        ei, n = cases.random_multigraph(n=61, e=400)
        g = torch.Generator().manual_seed(12)
        x = torch.randn(n, 9, generator=g, dtype=torch.float64)
        y = torch.randint(0, 3, (n,), generator=g)
        torch.manual_seed(5)
        ref = O.OracleGAT(9, 3, hidden_dim=4, dropout=0.0).double()
        ref.bn1, ref.bn2 = (torch.nn.GroupNorm(8, 32).double() for _ in range(2))
        with torch.no_grad():
            for p in ref.parameters():
                if p.dim() == 1:
                    p.add_(torch.randn(p.shape, generator=g, dtype=torch.float64) * 0.3)
        model = PartitionedGAT(9, 3, hidden_dim=4, dropout=0.0, backend=OracleBackend(), norm="group").double()
        model.load_state_dict(ref.state_dict())
        part = model.partition_for(ei, n)
        tol = dict(rtol=1e-8, atol=1e-10)
        h = F.elu(ref.bn1(ref.conv1(x, ei)))
        h = F.elu(ref.bn2(ref.conv2(h, ei)))
        ref_logp = F.log_softmax(ref.conv3(h, ei), dim=1)
        F.nll_loss(ref_logp, y).backward()
        model.train()
        logp = model(x[part.lo:part.hi], ei, n)
        model.loss_share(logp, y[part.lo:part.hi], n).backward()
        model.sync_grads()
        torch.testing.assert_close(logp.detach(), ref_logp.detach()[part.lo:part.hi], **tol)
        rp = dict(ref.named_parameters())
        for name, p in model.named_parameters():
            torch.testing.assert_close(p.grad, rp[name].grad, **tol, msg=lambda m, name=name: f"{name}: {m}")
        model.eval()
        with torch.no_grad():
            torch.testing.assert_close(model(x[part.lo:part.hi], ei, n), ref_logp.detach()[part.lo:part.hi], **tol)
        q.put((rank, "ok"))
    except Exception as e:  # noqa: BLE001
        import traceback
        q.put((rank, "".join(traceback.format_exception(type(e), e, e.__traceback__))))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("world,port", [(2, 29671), (3, 29672)])
def test_partitioned_group_norm_network_equals_single_process(world, port):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    res = [q.get(timeout=180) for _ in procs]
    for p in procs:
        p.join(60)
    for rank, msg in res:
        assert msg == "ok", f"rank {rank}: {msg}"


def test_unknown_norm_is_refused():
    from gat_amd.dist import PartitionedGAT
    with pytest.raises(ValueError, match="norm"):
        PartitionedGAT(9, 3, hidden_dim=4, norm="layer")
