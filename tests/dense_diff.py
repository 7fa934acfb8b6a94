"""Central differences of the dense operators: the cases, and what the comparison with a gradient can be off
by.  Used by the tests only.

For L(p) = sum_i c_i y_i(p), with parameters p and p +- t v held exactly in the tensors' type:
    | (L(p + t v) - L(p - t v)) / 2t  -  <grad L, v> |
  <=  | the same difference in 64 bits - <its gradient, v> |        (the difference's own error, from the oracle)
    + sum |c| (e_y(p + t v) + e_y(p - t v)) / 2t + sum |v| e_grad   (what y and the gradient may be off by)
v is the gradient itself, so that every part of it counts and nothing cancels."""
import torch

import dense_ref as R

F32 = torch.float32


def oracle(op, p, c, kw):
    """(y, bound), [(gradient, bound)] of sum c y for the parameters p (a list of tensors)"""
    if op == "linear":
        x, w, b, r = p
        ref = R.Linear(x, w, b, r, kw["act"], c, F32)
        return ref.y, [ref.dx, ref.dw, ref.db, (c.double(), 0.0 * c.double())]
    if op == "group_norm":
        x, w, b = p
        ref = R.GroupNorm(x, kw["groups"], w, b, kw["act"], c, F32)
        return ref.y, [ref.dx, ref.dw, ref.db]
    if op == "embedding":
        y, g = R.embedding(kw["ids"], p[0], kw["scale"], c, F32)
        return y, [g]
    x, r = p
    inv = kw["keep"].double() / (1.0 - kw["p"])
    a, g = x.double() * inv, c.double() * inv
    y = a + r.double()
    return (y, 5 * R.U * (a.abs() + y.abs())), [(g, 5 * R.U * g.abs()), (c.double(), 0.0 * c.double())]


def case(op, kw, shapes, seed=3, t=2.0 ** -7):
    """parameters p, p + t v, p - t v, the upstream c, the true steps v and the bound"""
    g = torch.Generator().manual_seed(seed)
    p = [torch.randn(*s, generator=g) for s in shapes]
    y, _ = oracle(op, p, torch.zeros(kw["out"]), kw)
    c = torch.randn(*y[0].shape, generator=g)
    grads = oracle(op, p, c, kw)[1]
    scale = max(float(q.abs().max()) for q, _ in grads)
    hi = [(a.double() + t * q / scale).float() for a, (q, _) in zip(p, grads)]
    lo = [(a.double() - t * q / scale).float() for a, (q, _) in zip(p, grads)]
    v = [(a.double() - b.double()) / (2 * t) for a, b in zip(hi, lo)]
    (yh, eh), (yl, el) = (oracle(op, q, c, kw)[0] for q in (hi, lo))
    diff = float((c.double() * (yh - yl)).sum()) / (2 * t)
    want = sum(float((q * d).sum()) for (q, _), d in zip(grads, v))
    bound = abs(diff - want) + float((c.double().abs() * (eh + el)).sum()) / (2 * t)
    bound += sum(float((e * d.abs()).sum()) for (_, e), d in zip(grads, v))
    return p, hi, lo, c, v, t, want, bound


CASES = [
    ("linear", dict(act="gelu", out=(40, 30)), [(40, 24), (30, 24), (30,), (40, 30)]),
    ("linear", dict(act="elu", out=(3, 17)), [(3, 9), (17, 9), (17,), (3, 17)]),
    ("linear", dict(act="silu", out=(150, 5)), [(150, 33), (5, 33), (5,), (150, 5)]),
    ("group_norm", dict(act="silu", groups=3, out=(20, 24)), [(20, 24), (24,), (24,)]),
    ("group_norm", dict(act="elu", groups=2, out=(3, 17, 10)), [(3, 17, 10), (10,), (10,)]),
    ("embedding", dict(ids=torch.tensor([3, 0, 3, 3, -1, 7, 0, 9]), scale=1.5, out=(8, 12)), [(9, 12)]),
    ("dropout", dict(p=0.4, seed=77, out=(50, 13)), [(50, 13), (50, 13)]),
]
