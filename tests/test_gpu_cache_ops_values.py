"""Values that are hard on the cache operators' arithmetic: rounding beside the output's own,
dominant keys, infinities in visible places."""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _rand(g, *shape, dt, dev):
    return torch.randn(*shape, generator=g).to(dt).to(dev)


def _ref_prefix(q, pk, pv, k, v, lens):
    """decode_prefix from its definition, in 64 bits."""
    B, Hq, T, D = q.shape
    P, grp = pk.shape[1], Hq // pk.shape[0]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, h in itertools.product(range(B), range(pk.shape[0])):
        n = int(lens[b])
        kk, vv = torch.cat([pk[h], k[b, h, :n]]).double(), torch.cat([pv[h], v[b, h, :n]]).double()
        at = torch.arange(P + n, device=q.device)
        for t in range(T):
            x = q[b, h * grp:(h + 1) * grp, t].double() @ kk.t() * D ** -0.5
            o[b, h * grp:(h + 1) * grp, t] = torch.softmax(x.masked_fill(at - P > n - T + t, -math.inf), -1) @ vv
    return o


@pytest.mark.parametrize("dtype,D,B,Hq,Hkv,P,T", [
    # the tensor-memory kernel: one row tile, two, pairs
    ("bf16", 256, 33, 8, 2, 5000, 1), ("f16", 256, 70, 4, 2, 3001, 1), ("bf16", 256, 8, 8, 1, 9000, 1),
    ("bf16", 128, 40, 8, 2, 7001, 1), ("f16", 128, 33, 8, 2, 6000, 2), ("f16", 128, 12, 8, 2, 9000, 1),
    ("bf16", 64, 64, 8, 1, 8000, 1), ("f16", 64, 24, 4, 1, 9000, 1), ("f16", 32, 70, 4, 2, 9000, 1),
])
def test_prefix_rounds_the_output_alone(cuda, dtype, D, B, Hq, Hkv, P, T):
    """Many rows behind one prefix are as exact as a few: P goes into the products to 2^-16 of
    itself, so what is left is the output's rounding.  Over some 10^4 elements the norm of
    that varies by well under 1% (a rounding's square varies by 0.9 of its mean); P to one
    16-bit term would be off by as much as the output, 1.4 together."""
    import _bsa
    g = torch.Generator().manual_seed(P)
    dt = DT[dtype]
    q = _rand(g, B, Hq, T, D, dt=dt, dev=cuda) * 1.5
    pk, pv = (_rand(g, Hkv, P, D, dt=dt, dev=cuda) for _ in range(2))
    k, v = (_rand(g, B, Hkv, 5, D, dt=dt, dev=cuda) for _ in range(2))
    lens = torch.full((B,), 5, dtype=torch.int32, device=cuda)
    o = _bsa.decode_prefix(q, pk, pv, k, v, lens).double()
    ref = _ref_prefix(q, pk, pv, k, v, lens)
    err, once = (x.norm() / ref.norm() for x in (o - ref, ref.to(dt).double() - ref))
    assert err <= 1.05 * once, "%.3g against %.3g of one rounding" % (err, once)


# A sink: one slot that takes nearly all of the weight and holds V = 0, and n slots `gap` nats
# below it, alike in weight, V around 1000, so that the output is theirs alone.  One product of
# a logit is not zero, so it is exact but for fp32 roundings of at most 26 (its size in log2
# units): three of 2^-24 (the product of the scale and log2 e, that with the logit, the
# subtraction of the maximum) and, in fp32, 2^-21 of dropped terms, with 2^-22 of ex2 less than
# 2^-15 together.  A softmax weight goes into the products with two terms: to 2^-16 of itself
# (bf16), and f16 to 2^-25 absolutely with the largest at 2^15, so to 2^-25 2^(26-15) = 2^-14
# at 18 nats.  fp32: three terms, 2^-21 with the dropped products.  Then the output's rounding.
GAPS = (12.1, 14.3, 16.2, 17.9)
TERM = {"bf16": 2 ** -16, "f16": 2 ** -14, "f32": 2 ** -21}


def _sink(dt, D, n, seed, dev):
    """q (4, 1, D) of one head per gap and k, v (1 + n, D), the sink first."""
    g = torch.Generator().manual_seed(seed)
    q = torch.zeros(4, 1, D)
    q[:, 0, 0] = torch.tensor(GAPS) * D ** 0.5 / 8
    k = torch.randn(1 + n, D, generator=g)
    k[:, 0] = 0
    k[0, 0] = 8
    v = 1000 + 250 * torch.randn(1 + n, D, generator=g)
    v[0] = 0
    return (x.to(dt).to(dev) for x in (q, k, v))


def _check_sink(dtype, o, q, k, v, term=None):
    x = q[:, 0].double() @ k.double().t() * q.shape[-1] ** -0.5
    p = torch.softmax(x, -1)
    ref, mean = p @ v.double(), p @ v.double().abs()
    tol = torch.finfo(o.dtype).eps / 2 + 2 ** -15 + (term or TERM[dtype])
    err = (o.double() - ref).norm(dim=-1) / mean.norm(dim=-1)
    assert bool((err <= tol).all()), "%.3g of the norm, %.3g allowed" % (err.max(), tol)
    return p


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,B,Hkv,n", [
    # one launch; splits; so many heads that a warp has thousands of slots to itself
    (64, 1, 1, 1500), (256, 2, 1, 900), (32, 2, 2, 500), (128, 1, 2, 40000), (32, 1, 1, 30000), (64, 40, 8, 20000),
])
def test_weighted_behind_a_sink(cuda, dtype, D, B, Hkv, n):
    import _bsa
    q, k, v = _sink(DT[dtype], D, n, n, cuda)
    w = torch.zeros(B, Hkv, 1 + n, device=cuda)
    o = _bsa.decode_weighted(q.repeat(B, Hkv, 1, 1), k.expand(B, Hkv, -1, -1), v.expand(B, Hkv, -1, -1), w)
    p = _check_sink(dtype, o.view(B, Hkv, 4, D), q, k, v).sum(0)
    assert bool(((w.double() - p).abs() <= 2 ** -14 * p).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,B,Hkv,n,S", [
    # the sink and the others in the prefix: one launch, split kernels; in the own slots
    (64, 2, 1, 1000, 1), (128, 3, 2, 30000, 1), (32, 4, 1, 20000, 1), (256, 1, 2, 9000, 1), (64, 3, 2, 0, 20000),
])
def test_prefix_behind_a_sink(cuda, dtype, D, B, Hkv, n, S):
    import _bsa
    q, k, v = _sink(DT[dtype], D, max(n, S), n, cuda)
    if n:    # no own slots in use
        pk, pv, lens = k.expand(Hkv, -1, -1), v.expand(Hkv, -1, -1), torch.zeros(B, dtype=torch.int32, device=cuda)
        ko = vo = torch.zeros(B, Hkv, S, D, dtype=k.dtype, device=cuda)
    else:
        pk = pv = torch.zeros(Hkv, 0, D, dtype=k.dtype, device=cuda)
        ko, vo = k.expand(B, Hkv, -1, -1), v.expand(B, Hkv, -1, -1)
        lens = torch.full((B,), 1 + S, dtype=torch.int32, device=cuda)
    o = _bsa.decode_prefix(q.repeat(B, Hkv, 1, 1), pk, pv, ko, vo, lens)
    _check_sink(dtype, o.view(B, Hkv, 4, D), q, k, v)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,B,Hkv,n", [
    # many rows: the tensor-memory kernel (one row tile, two, pairs), fp32 rows over the warps;
    # the last three with so many that one split has all of the keys
    (64, 12, 1, 9000), (128, 8, 2, 9000), (128, 70, 1, 12000), (256, 9, 2, 6000),
    (64, 4736, 2, 2900), (128, 4736, 2, 2900), (256, 2368, 2, 2900),
])
def test_prefix_of_many_rows_behind_a_sink(cuda, dtype, D, B, Hkv, n):
    """The tensor-memory kernel's maximum may lag by 2 (log2), f16 terms start at 2^13:
    2^-25 2^(26-13) = 2^-12 of a weight at 18 nats."""
    import _bsa
    q, k, v = _sink(DT[dtype], D, n, n, cuda)
    pk, pv = (x.repeat(Hkv, 1, 1) for x in (k, v))
    pk[1:], pv[1:] = pk[1:].roll(-1, 1), pv[1:].roll(-1, 1)   # the second head's sink comes last
    own = torch.zeros(B, Hkv, 1, D, dtype=k.dtype, device=cuda)
    o = _bsa.decode_prefix(q.repeat(B, Hkv, 1, 1), pk, pv, own, own, torch.zeros(B, dtype=torch.int32, device=cuda))
    _check_sink(dtype, o.view(B, Hkv, 4, D), q, k, v, 2 ** -12 if dtype == "f16" else None)


# Infinities where a row does look.  A V column that holds one is that infinity in the output
# of every row that gives it weight (two of unlike sign: NaN) and the other columns are what
# they are; a K row with -inf (or the type's lowest value) in a column that every query meets
# with a positive number has logit -inf (or far below) and weight 0.
def _infinite(k, v, q, at_v, at_k, low):
    """Puts them into k, v (..., n, D) and returns (columns of v with +inf, -inf, both)."""
    cols = (1, 2, 5)
    for i, j in enumerate(at_v):
        v[..., j, cols[i % 2]] = math.inf if i % 2 == 0 else -math.inf
        v[..., j, cols[2]] = math.inf if i % 2 == 0 else -math.inf
    for j in at_k:
        k[..., j, 7] = low
    q[..., 7] = q[..., 7].abs() + 0.5
    return cols


def _check_infinite(o, ref, tol, cols):
    assert bool((o[..., cols[0]] == math.inf).all()) and bool((o[..., cols[1]] == -math.inf).all())
    assert bool(o[..., cols[2]].isnan().all())
    rest = [d for d in range(o.shape[-1]) if d not in cols]
    err = (o.double() - ref).abs()[..., rest]
    assert bool((err <= tol[..., rest]).all()), "%.3g" % err.max()


def _attend(q, k, v, see, dead):
    """Softmax attention of rows q (R, D) in 64 bits: see (R, n); dead: keys of weight 0."""
    k, v = k.double().clone(), torch.where(v.isfinite(), v.double(), 0.0)
    k[dead] = 0
    x = (q.double() @ k.t() * q.shape[-1] ** -0.5).masked_fill(~see, -math.inf)
    x[:, dead] = -math.inf
    p = torch.softmax(x, -1)
    # the bounds of the other test file: logits, P's terms, the output's rounding
    D = q.shape[-1]
    top = float(q.double().norm(dim=-1).max() * k.norm(dim=-1).max()) * D ** -0.5
    e = 2 * (8 + (3 * D / 8 if q.dtype == torch.float32 else D / 8)) * 2 ** -23 * top + 2 ** -18
    o = p @ v
    return o, p, (2 * e + 2 ** -15) * v.abs().max() + torch.finfo(q.dtype).eps * o.abs()


@pytest.mark.parametrize("low", [-math.inf, "lowest"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,B,Hq,Hkv,L,T,bs", [
    # one launch, splits, several new tokens, selected blocks
    (64, 2, 4, 2, 700, 1, 0), (256, 1, 8, 1, 500, 2, 0), (32, 1, 24, 1, 300, 3, 0), (128, 1, 8, 2, 9000, 1, 0),
    (64, 1, 40, 2, 8000, 4, 0), (256, 1, 4, 2, 7000, 1, 0), (128, 1, 4, 2, 900, 1, 32),
])
def test_weighted_visible_infinities(cuda, dtype, D, B, Hq, Hkv, L, T, bs, low):
    import _bsa
    g = torch.Generator().manual_seed(L)
    dt, grp = DT[dtype], Hq // Hkv
    low = torch.finfo(dt).min if low == "lowest" else low
    q = _rand(g, B, Hq, T, D, dt=dt, dev=cuda)
    k, v = (_rand(g, B, Hkv, L, D, dt=dt, dev=cuda) for _ in range(2))
    w = torch.rand(B, Hkv, L, generator=g).to(cuda)
    at_k = [3, 40, L - T - 1]
    slots, sel, kw = torch.arange(L, device=cuda), None, {}
    if bs:
        ids = [0, 1, (L - 1) // bs]
        slots = torch.cat([torch.arange(i * bs, min(L, (i + 1) * bs), device=cuda) for i in ids])
        sel, kw = torch.tensor(ids, dtype=torch.int32, device=cuda).expand(B, Hkv, 3), dict(bs=bs)
    # the slots of a row's largest and least weight, and one between
    x = q[0, 0, 0].double() @ k[0, 0, slots[:len(slots) - T]].double().t()
    cols = _infinite(k, v, q, [int(slots[x.argmax()]), 33, int(slots[x.argmin()]), 17], at_k, low)
    dead = (slots.unsqueeze(1) == torch.tensor(at_k, device=cuda)).any(1)
    w0 = w.double()
    o = _bsa.decode_weighted(q, k, v, w, sel, L=L, **kw)
    add = torch.zeros_like(w0)
    for b, h, t in itertools.product(range(B), range(Hkv), range(T)):
        see = (slots <= L - T + t).expand(grp, -1)
        rows = slice(h * grp, (h + 1) * grp)
        ref, p, tol = _attend(q[b, rows, t], k[b, h, slots], v[b, h, slots], see, dead)
        _check_infinite(o[b, rows, t], ref, tol, cols)
        add[b, h, slots] += p.sum(0)
    e = 2 ** -9    # of the logits' e above for these sizes (top < 2^6: (8 + 96) 2^-15)
    assert bool(((w.double() - w0 - add).abs() <= e * add + 2 ** -23 * (w0 + add)).all())


@pytest.mark.parametrize("low", [-math.inf, "lowest"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,B,Hq,Hkv,P,S", [
    # one launch, splits; many rows: one row tile, two, pairs, fp32 rows over the warps
    (64, 2, 4, 2, 700, 3), (128, 2, 8, 2, 9000, 5), (64, 12, 4, 1, 9000, 3), (32, 40, 8, 1, 6000, 2),
    (128, 40, 4, 1, 9000, 3), (256, 9, 4, 1, 3000, 3), (256, 40, 4, 1, 5000, 3),
])
def test_prefix_visible_infinities(cuda, dtype, D, B, Hq, Hkv, P, S, low):
    import _bsa
    g = torch.Generator().manual_seed(P)
    dt, grp = DT[dtype], Hq // Hkv
    low = torch.finfo(dt).min if low == "lowest" else low
    q = _rand(g, B, Hq, 1, D, dt=dt, dev=cuda)
    pk, pv = (_rand(g, Hkv, P, D, dt=dt, dev=cuda) for _ in range(2))
    k, v = (_rand(g, B, Hkv, S, D, dt=dt, dev=cuda) for _ in range(2))
    lens = torch.full((B,), S, dtype=torch.int32, device=cuda)
    x = q[0, 0, 0].double() @ pk[0].double().t()
    cols = _infinite(pk, pv, q, [int(x.argmax()), 33, int(x.argmin()), 17], [3, 40, P - 1], low)
    _infinite(k, v, q, [], [0], low)
    v[:, :, 1, cols[0]] = math.inf
    o = _bsa.decode_prefix(q, pk, pv, k, v, lens)
    dead = torch.zeros(P + S, dtype=torch.bool, device=cuda)
    dead[[3, 40, P - 1, P]] = True
    for b, h in itertools.product(range(B), range(Hkv)):
        rows = slice(h * grp, (h + 1) * grp)
        kk, vv = torch.cat([pk[h], k[b, h]]), torch.cat([pv[h], v[b, h]])
        ref, _, tol = _attend(q[b, rows, 0], kk, vv, torch.ones(grp, P + S, dtype=torch.bool, device=cuda), dead)
        _check_infinite(o[b, rows, 0], ref, tol, cols)
