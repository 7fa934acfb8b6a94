"""PartitionedGAT(norm="group") with the fused operators on a real MI355X: one rank over RCCL, or several ranks that share
cuda:0 over gloo (the package stages gloo's buffers through the host).  One training step without dropout against the
single-process network in 64 bits, then one with dropout: every rank draws masks of its own, gradients are finite and
the same on all ranks.  Started by tests/test_a3_gpu_group_norm_ranks.py; prints one line a check from rank 0."""
import os, sys
import torch
import torch.distributed as dist
import torch.nn.functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.join(ROOT, "tests"))


def main():
    dev = torch.device("cuda:0")
    torch.cuda.set_device(dev)
    if sys.argv[1] == "nccl":
        dist.init_process_group("nccl", rank=0, world_size=1, device_id=dev)
    else:
        dist.init_process_group("gloo")
    all_ok = True

    def verdict(good, text):
        nonlocal all_ok
        flag = torch.tensor([1 if good else 0], device=dev if sys.argv[1] == "nccl" else "cpu")
        dist.all_reduce(flag, op=dist.ReduceOp.MIN)
        all_ok &= bool(flag.item())
        if dist.get_rank() == 0:
            print(f"{'ok' if flag.item() else 'FAILED'} {text}", flush=True)

    try:
        import cases
        from oracle import gat_oracle as O
        from gat_amd.dist import PartitionedGAT
        ei, n = cases.knn_graph(n=3000, f=25, seed=2)
        g = torch.Generator().manual_seed(3)
        x = torch.rand(n, 25, generator=g)
        y = torch.randint(0, 2, (n,), generator=g)
        torch.manual_seed(7)
        ref = O.OracleGAT(25, 2, hidden_dim=30, dropout=0.0)
        ref.bn1, ref.bn2 = torch.nn.GroupNorm(8, 240), torch.nn.GroupNorm(8, 240)
        model = PartitionedGAT(25, 2, hidden_dim=30, dropout=0.0, norm="group").to(dev)
        model.load_state_dict(ref.state_dict())
        ref = ref.double()
        h = F.elu(ref.bn1(ref.conv1(x.double(), ei)))
        h = F.elu(ref.bn2(ref.conv2(h, ei)))
        ref_logp = F.log_softmax(ref.conv3(h, ei), dim=1)
        ref_loss = F.nll_loss(ref_logp, y)
        ref_loss.backward()
        eid = ei.to(dev)
        part = model.partition_for(eid, n)
        mine = slice(part.lo, part.hi)
        for training in (True, False):
            model.train(training)
            model.zero_grad()
            logp, share = model.forward_loss(x[mine].to(dev), eid, n, y[mine].to(dev))
            share.backward()
            model.sync_grads()
            err = float((logp.detach().cpu().double() - ref_logp.detach()[mine]).abs().max())
            lerr = abs(float(model.global_loss(share)) - float(ref_loss.detach()))
            rp = dict(ref.named_parameters())
            # d att_dst: the softmax makes dz sum to 0 over a destination's edges, where h[dst] is one vector.  What is
            # left in f32 is a rest of summands |dz_e| |h|, whose sum is at least |d att_src|.
            size = {k: float(p.grad.abs().max()) for k, p in rp.items()}
            off = {k: float((p.grad.cpu().double() - rp[k].grad).abs().max())
                   / (max(size[k], size[k.replace("att_dst", "att_src")]) + 1e-12) for k, p in model.named_parameters()}
            worst = max(off, key=off.get)
            gerr = off[worst]
            verdict(model.fused and err < 1e-4 and lerr < 1e-5 and gerr < 1e-3,
                    f"norm=group, training={training}: logp err {err:.2e} loss err {lerr:.2e} worst relative grad err {gerr:.2e} ({worst})")
        torch.manual_seed(7)
        model = PartitionedGAT(25, 2, hidden_dim=30, dropout=0.4, norm="group").to(dev).train()
        seeds = [model._mask_seed() for _ in range(2)]
        logp, share = model.forward_loss(x[mine].to(dev), eid, n, y[mine].to(dev))
        again, _ = model.forward_loss(x[mine].to(dev), eid, n, y[mine].to(dev))
        share.backward()
        model.sync_grads()
        flat = torch.cat([p.grad.flatten() for p in model.parameters()]).cpu()
        every = [None] * dist.get_world_size()
        dist.all_gather_object(every, (seeds, flat.tolist()[:4000]))
        good = bool(torch.isfinite(flat).all()) and not torch.equal(logp, again)
        good &= len({s for q, _ in every for s in q}) == 2 * len(every) and all(q[1] == every[0][1] for q in every)
        verdict(good, "norm=group with dropout: finite, the same gradients on every rank, masks of its own on each")
        torch.cuda.synchronize()
        dist.barrier()
    finally:
        dist.destroy_process_group()
    return 0 if all_ok else 1


if __name__ == "__main__":
    sys.exit(main())
