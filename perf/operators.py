"""The dense operators around a GAT layer, as cases that can be timed and checked.

Four operators of a network's block, each with its gradient:

  linear     y = act(x W^T + b) + residual                          gat_amd.linear_act
  groupnorm  y = act(group_norm(x))  on rows or channels-last data   gat_amd.group_norm_act
  embedding  y[i] = scale * table[ids[i]], zero where there is none  gat_amd.embedding
  dropout    y = keep * x / (1 - p) + residual, keep from a counter  gat_amd.dropout

With `own` false run() computes a case in elementary torch operations in 32 bits; with `own` true it
calls this package.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
WIDTH = {"f32": 4, "bf16": 2, "f16": 2}
NODES = 2449029          # gat_amd.synth "products"


def listed():
    return [
        # one node asked for while serving: latency of a single row through a hidden layer of run.py's width
        dict(name="linear one row", op="linear", rows=1, nin=240, nout=240, act="elu", bias=True, residual=False,
             dtype="f32", train=False),
        # the skip connection beside a hidden layer of run.py's network (8 x 30 channels), 10^5 nodes, training
        dict(name="linear skip 100k", op="linear", rows=100000, nin=240, nout=240, act="elu", bias=True,
             residual=True, dtype="f32", train=True),
        # the same beside a hidden layer of the products-shaped network (4 x 64 channels), bf16 rows, training
        dict(name="linear skip products", op="linear", rows=NODES, nin=256, nout=256, act="gelu", bias=True,
             residual=True, dtype="bf16", train=True),
        # a wide classifier head over one arxiv-shaped batch, odd sizes, inference
        dict(name="linear head odd", op="linear", rows=65537, nin=1024, nout=1001, act="none", bias=True,
             residual=False, dtype="f16", train=False),
        # the Cora-sized graph's hidden rows, inference: launch latency
        dict(name="groupnorm 2708", op="groupnorm", batch=2708, length=1, groups=8, width=30, act="elu",
             dtype="f32", train=False),
        # between two layers of run.py's network: one group per head, 10^5 nodes, training
        dict(name="groupnorm heads 100k", op="groupnorm", batch=100000, length=1, groups=8, width=30, act="elu",
             dtype="f32", train=True),
        # statistics over whole graphs: a batch of three equal graphs of an odd node count, channels last
        dict(name="groupnorm graphs", op="groupnorm", batch=3, length=169343, groups=16, width=16, act="silu",
             dtype="bf16", train=True),
        # a few categorical codes looked up while serving
        dict(name="embedding 169", op="embedding", rows=169, per=1, vocab=1025, dim=30, scale=1.0, missing=0.0,
             dtype="f32", train=False),
        # source and destination port of 10^5 flows, 65536 ports, a few frequent ones, some missing; training
        dict(name="embedding ports", op="embedding", rows=100000, per=2, vocab=65536, dim=30,
             scale=math.sqrt(30.0), missing=0.05, dtype="f32", train=True),
        # learned node features of the products-shaped graph drawn from a large odd table, bf16, training
        dict(name="embedding nodes", op="embedding", rows=NODES, per=1, vocab=1000003, dim=128, scale=1.0,
             missing=0.0, dtype="bf16", train=True),
        # the input dropout of run.py's network, 10^5 nodes, training
        dict(name="dropout 100k", op="dropout", rows=100000, cols=25, p=0.425, residual=False, dtype="f32",
             train=True),
        # dropout in front of a residual sum on the products-shaped graph, bf16, training
        dict(name="dropout residual products", op="dropout", rows=NODES, cols=100, p=0.3, residual=True,
             dtype="bf16", train=True),
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng):
    op = rng.choice(["linear", "groupnorm", "embedding", "dropout"])
    dtype, train = rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.6
    # relu's derivative jumps at 0, where two right results may differ: its gradient is not compared here
    acts = ["none", "elu", "silu", "gelu"] + ([] if train else ["relu"])
    if op == "linear":
        rows, nin, nout = _log(rng, 1, NODES), _log(rng, 1, 1024), _log(rng, 1, 1024)
        while rows * nin * nout > NODES * 256 * 256 or rows * (nin + nout) * WIDTH[dtype] > NODES * 1024:
            rows = max(1, rows // 3)
        return dict(op=op, rows=rows, nin=nin, nout=nout, act=rng.choice(acts), bias=rng.random() < 0.8,
                    residual=rng.random() < 0.5, dtype=dtype, train=train)
    if op == "groupnorm":
        groups, width = _log(rng, 1, 64), _log(rng, 8, 128)
        batch, length = (_log(rng, 1, NODES), 1) if rng.random() < 0.5 else (_log(rng, 1, 64), _log(rng, 2, 300000))
        while batch * length * groups * width * WIDTH[dtype] > NODES * 256:
            batch, length = max(1, batch // 3), max(1, length // 2) if length > 1 else 1
        return dict(op=op, batch=batch, length=length, groups=groups, width=width, act=rng.choice(acts),
                    dtype=dtype, train=train)
    if op == "embedding":
        rows, per, vocab, dim = _log(rng, 1, NODES), rng.choice([1, 1, 2, 5]), _log(rng, 2, 1000003), _log(rng, 1, 512)
        while (rows * per + vocab) * dim * WIDTH[dtype] > NODES * 256:
            rows, vocab = max(1, rows // 2), max(2, vocab // 2)
        return dict(op=op, rows=rows, per=per, vocab=vocab, dim=dim,
                    scale=rng.choice([1.0, math.sqrt(dim), 0.125]), missing=rng.choice([0.0, 0.0, 0.1]),
                    dtype=dtype, train=train)
    rows, cols = _log(rng, 1, NODES), _log(rng, 1, 1024)
    while rows * cols * WIDTH[dtype] > NODES * 200:
        rows = max(1, rows // 3)
    return dict(op=op, rows=rows, cols=cols, p=rng.choice([0.1, 0.3, 0.425, 0.7]), residual=rng.random() < 0.5,
                dtype=dtype, train=train)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)
    dt = DTYPES[case["dtype"]]
    train = case["train"]

    def normal(*shape, scale=1.0, shift=0.0, leaf=False):
        t = (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dt)
        return t.requires_grad_(leaf and train)

    s = {"case": case}
    op = case["op"]
    if op == "linear":
        rows, nin, nout = case["rows"], case["nin"], case["nout"]
        s["x"] = normal(rows, nin, leaf=True)
        s["w"] = normal(nout, nin, scale=1.0 / math.sqrt(nin), leaf=True)
        s["b"] = normal(nout, scale=0.3, leaf=True) if case["bias"] else None
        s["res"] = normal(rows, nout, leaf=True) if case["residual"] else None
        s["dy"] = normal(rows, nout) if train else None
    elif op == "groupnorm":
        c = case["groups"] * case["width"]
        shape = (case["batch"], c) if case["length"] == 1 else (case["batch"], case["length"], c)
        s["x"] = normal(*shape, scale=1.5, shift=0.3, leaf=True)
        s["w"] = normal(c, scale=0.2, shift=1.0, leaf=True)
        s["b"] = normal(c, scale=0.3, leaf=True)
        s["dy"] = normal(*shape) if train else None
    elif op == "embedding":
        shape = (case["rows"], case["per"]) if case["per"] > 1 else (case["rows"],)
        vocab = case["vocab"]
        # a few ids are frequent and most are rare: log-uniform ranks, spread over the table
        rank = (vocab ** torch.rand(*shape, generator=g, device="cuda", dtype=torch.float64)).long() - 1
        ids = rank.clamp_(0, vocab - 1) * 7919 % vocab
        if case["missing"]:
            ids[torch.rand(*shape, generator=g, device="cuda") < case["missing"]] = -1
        s["ids"] = ids
        s["table"] = normal(vocab, case["dim"], leaf=True)
        s["dy"] = normal(*shape, case["dim"]) if train else None
    else:
        s["x"] = normal(case["rows"], case["cols"], leaf=True)
        s["res"] = normal(case["rows"], case["cols"], leaf=True) if case["residual"] else None
        s["seed"] = (int(seed) * 0x9E3779B97F4A7C15 + 0x632BE59BD9B4E019) % (1 << 63)
        s["dy"] = normal(case["rows"], case["cols"]) if train else None
    return s


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {"linear": _plain_linear, "groupnorm": _plain_groupnorm, "embedding": _plain_embedding,
                "dropout": _plain_dropout}[s["case"]["op"]](s)


def _own(s):
    import gat_amd

    case = s["case"]
    op = case["op"]
    if op == "linear":
        leaves = [s["x"], s["w"], s["b"], s["res"]]
        y = gat_amd.linear_act(s["x"], s["w"], s["b"], act=case["act"], residual=s["res"])
    elif op == "groupnorm":
        leaves = [s["x"], s["w"], s["b"]]
        y = gat_amd.group_norm_act(s["x"], case["groups"], s["w"], s["b"], act=case["act"])
    elif op == "embedding":
        leaves = [s["table"]]
        y = gat_amd.embedding(s["ids"], s["table"], scale=case["scale"])
    else:
        leaves = [s["x"], s["res"]]
        y = gat_amd.dropout(s["x"], case["p"], seed=s["seed"], residual=s["res"])
    if not case["train"]:
        return [y]
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], s["dy"])
    return [y.detach(), *grads]


# ---- plain forms, 32 bits throughout, one rounding at the end ---------------------------------
def _act(z, act):
    """(act(z), its derivative)."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.clamp(z, min=0.0), (z > 0).float()
    if act == "elu":
        e = torch.exp(torch.clamp(z, max=0.0))
        return torch.where(z > 0, z, torch.expm1(torch.clamp(z, max=0.0))), torch.where(z > 0, torch.ones_like(z), e)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    phi = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_linear(s):
    case, dt = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    y, d = _act(z, case["act"])
    if s["res"] is not None:
        y = y + s["res"].float()
    out = [y.to(dt)]
    if case["train"]:
        dz = s["dy"].float() * d
        out += [(dz @ w).to(dt), (dz.t() @ x).to(dt)]
        if s["b"] is not None:
            out.append(dz.sum(0).to(dt))
        if s["res"] is not None:
            out.append(s["dy"])
    return out


def _plain_groupnorm(s):
    case, dt = s["case"], s["x"].dtype
    n, length, groups, width = case["batch"], case["length"], case["groups"], case["width"]
    x = s["x"].float().view(n, length, groups, width)
    w, b = s["w"].float().view(groups, width), s["b"].float().view(groups, width)
    mean = x.mean((1, 3), keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean((1, 3), keepdim=True) + 1e-5)
    xh = xc * rstd
    y, d = _act(xh * w + b, case["act"])
    out = [y.to(dt).view(s["x"].shape)]
    if case["train"]:
        du = s["dy"].float().view(x.shape) * d
        dxh = du * w
        dx = rstd * (dxh - dxh.mean((1, 3), keepdim=True) - xh * (dxh * xh).mean((1, 3), keepdim=True))
        out += [dx.to(dt).view(s["x"].shape), (du * xh).sum((0, 1)).to(dt).view(-1), du.sum((0, 1)).to(dt).view(-1)]
    return out


def _plain_embedding(s):
    case, dt, ids = s["case"], s["table"].dtype, s["ids"].view(-1)
    vocab, dim = case["vocab"], case["dim"]
    there = ((ids >= 0) & (ids < vocab)).float().view(-1, 1) * case["scale"]
    at = ids.clamp(0, vocab - 1)
    out = [(s["table"][at].float() * there).to(dt).view(*s["ids"].shape, dim)]
    if case["train"]:
        grad = torch.zeros(vocab, dim, device=ids.device)
        grad.index_add_(0, at, s["dy"].view(-1, dim).float() * there)
        out.append(grad.to(dt))
    return out


def _plain_dropout(s):
    case, dt = s["case"], s["x"].dtype
    rows, cols = case["rows"], case["cols"]
    low = 0xFFFFFFFF
    lo, hi = s["seed"] & low, (s["seed"] >> 32) & low
    r = (torch.arange(rows, device="cuda") * 0x9E3779B1 + lo) & low
    c = (torch.arange(cols, device="cuda") * 0x85EBCA77 + hi) & low
    h = r.view(-1, 1) ^ c.view(1, -1)
    h ^= h >> 15
    h = (h * 0x2C1B3C6D) & low
    h ^= h >> 12
    h = (h * 0x297A2D39) & low
    h ^= h >> 15
    p = float(np.float32(case["p"]))
    factor = ((h >> 8) >= int(p * 16777216.0)).float() * (1.0 / (1.0 - p))
    y = s["x"].float() * factor
    if s["res"] is not None:
        y = y + s["res"].float()
    out = [y.to(dt)]
    if case["train"]:
        out.append((s["dy"].float() * factor).to(dt))
        if s["res"] is not None:
            out.append(s["dy"])
    return out


# ---- the definitions in 64 bits ------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    F = torch.nn.functional
    wide = lambda t: None if t is None else t.detach().double().requires_grad_(case["train"])  # noqa: E731
    apply_act = {"none": lambda v: v, "relu": F.relu, "elu": F.elu, "silu": F.silu, "gelu": F.gelu}
    if case["op"] == "linear":
        x, w, b, res = (wide(s[k]) for k in ("x", "w", "b", "res"))
        y = apply_act[case["act"]](F.linear(x, w, b))
        y = y if res is None else y + res
        leaves = [x, w, b, res]
    elif case["op"] == "groupnorm":
        x, w, b = (wide(s[k]) for k in ("x", "w", "b"))
        # one row per (sample, group), one column per value of it; the gradient is left to autograd
        n, t, k, d = case["batch"], case["length"], case["groups"], case["width"]
        v = x.reshape(n, t, k, d).transpose(1, 2).reshape(n * k, t * d)
        var, mean = torch.var_mean(v, dim=1, unbiased=False, keepdim=True)
        v = ((v - mean) / (var + 1e-5).sqrt()).reshape(n, k, t, d).transpose(1, 2).reshape(n, t, k * d)
        y = apply_act[case["act"]](torch.addcmul(b, v, w)).reshape(x.shape)
        leaves = [x, w, b]
    elif case["op"] == "embedding":
        table = wide(s["table"])
        here = (s["ids"] >= 0) & (s["ids"] < case["vocab"])
        y = F.embedding(torch.where(here, s["ids"], 0), table)
        y = torch.where(here.unsqueeze(-1), y * case["scale"], torch.zeros((), dtype=torch.float64, device="cuda"))
        leaves = [table]
    else:
        x, res = wide(s["x"]), wide(s["res"])
        p = np.float32(case["p"])
        a = np.arange(case["rows"], dtype=np.uint32) * np.uint32(0x9E3779B1) + np.uint32(s["seed"] % (1 << 32))
        b = np.arange(case["cols"], dtype=np.uint32) * np.uint32(0x85EBCA77) + np.uint32(s["seed"] // (1 << 32))
        h = np.bitwise_xor.outer(a, b)
        for shift, factor in ((15, 0x2C1B3C6D), (12, 0x297A2D39), (15, 1)):
            h ^= h >> np.uint32(shift)
            h *= np.uint32(factor)
        keep = torch.from_numpy((h >> np.uint32(8)) >= np.uint32(int(np.float64(p) * 2.0 ** 24))).cuda()
        y = torch.where(keep, x / (1.0 - float(p)), torch.zeros((), dtype=torch.float64, device="cuda"))
        y = y if res is None else y + res
        leaves = [x, res]
    if not case["train"]:
        return [y]
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], s["dy"].double())
    return [y.detach(), *grads]


def work(case):
    """Each input read once, each output written once; a multiply and an add are two operations."""
    width, train = WIDTH[case["dtype"]], case["train"]
    if case["op"] == "linear":
        m, k, n = case["rows"], case["nin"], case["nout"]
        values = m * k + n * k + m * n + (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
        if train:
            values += m * n + m * k + n * k + (n if case["bias"] else 0)
        return {"bytes": values * width, "flops": 2.0 * m * n * k * (3 if train else 1)}
    if case["op"] == "groupnorm":
        c = case["groups"] * case["width"]
        values = case["batch"] * case["length"] * c
        return {"bytes": (values * (4 if train else 2) + c * (4 if train else 2)) * width,
                "flops": values * (30.0 if train else 12.0)}
    if case["op"] == "embedding":
        n, v, d = case["rows"] * case["per"], case["vocab"], case["dim"]
        once = min(n, v)                     # table rows that can be read at all
        return {"bytes": n * 8 + (once * d + n * d) * width + ((n * d + v * d) * width if train else 0),
                "flops": n * d * (2.0 if train else 1.0)}
    values = case["rows"] * case["cols"]
    return {"bytes": values * width * (2 + case["residual"] + (2 if train else 0)), "flops": values * (4.0 if train else 2.0)}
