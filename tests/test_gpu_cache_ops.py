"""Weighted decode (bsa_decode_weighted), eviction (bsa_evict) and shared-prefix decode
(bsa_decode_prefix) against their definitions in 64 bits.

Tolerances.  A logit of the kernels is a dot product of D exact products in fp32; at
most n = 8 + D/8 roundings of 2^-23 (the tensor cores truncate) touch a partial sum,
none of which exceeds |q||k| (fp32 operands: six bf16 products for every sixteen dims,
3D/8 roundings, and 2^-23 of |q||k| in dropped terms, n = 8 + 3D/8), so in natural units it is off by at most
d = n 2^-23 |q||k| scale; the offset, the base change and ex2 add at most 2^-18 to the
exponent's effect for logits up to 2^5.  A softmax weight is then off by a factor within
1 +- e, e = 2 d + 2^-18, and with sum p = 1 the output by at most 2 e max|v| plus 2^-15
max|v| for P's second 16-bit term, plus half a step of the output type.  A weight sum
is off by e times its new part and two fp32 roundings of the total.

The tensor-memory kernel for a shared prefix (16-bit types, more than 16 rows per K/V
head, 128 prefix keys or more) rounds each p_j once, to half a step h = eps / 2 of the
type: p_j (1 + d_j) with |d_j| <= h, while l sums the unrounded p_j.  The output moves by
|sum_j p_j d_j v_j| / l <= h sum_j p_j |v_j| / l, the weighted mean of |v|, which the
reference computes beside the output."""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _rand(g, *shape, dt, dev):
    return torch.randn(*shape, generator=g).to(dt).to(dev)


def _rel(q, k, scale):
    """e of the module's docstring for these operands (finite rows only)."""
    D = q.shape[-1]
    kn = k.double().norm(dim=-1)
    top = q.double().norm(dim=-1).max() * kn[torch.isfinite(kn)].max() * scale
    return 2 * (8 + (3 * D / 8 if q.dtype == torch.float32 else D / 8)) * 2 ** -23 * float(top) + 2 ** -18


def _close_o(o, ref, e, vmax, what, once=0.0):
    tol = once + (2 * e + 2 ** -15) * vmax + torch.finfo(o.dtype).eps / 2 * ref.abs() * (1 + 2 ** -8)
    if o.dtype == torch.float32:
        tol = 2 * e * vmax + 2 ** -22 * ref.abs()
    err = (o.double() - ref).abs()
    ok = bool((err <= tol).all()) and bool(torch.isfinite(o.float()).all())
    assert ok, "%s: error %.3g, %.3g over" % (what, err.max().item(), (err - tol).max().item())


def _ref_rows(q, k, v, see, bias, scale):
    """(o, p, p |v|) of rows q (R, D) over keys k, v (n, D): see (R, n) truth values."""
    x = q.double() @ k.double().t() * scale
    if bias is not None:
        x = x + bias.double()
    x = x.masked_fill(~see, -math.inf)
    m = x.max(-1, keepdim=True).values
    p = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m)).masked_fill(~see, 0.0)
    z = p.sum(-1, keepdim=True)
    p = torch.where(z > 0, p / torch.where(z > 0, z, torch.ones_like(z)), torch.zeros_like(p))
    vv = torch.where(torch.isfinite(v.double()), v.double(), torch.zeros_like(v.double()))
    return p @ vv, p, p @ vv.abs()


def _ref_weighted(q, k, v, weight, sel, gate, bs, L, scale):
    B, Hq, T, D = q.shape
    Hkv = k.shape[1]
    grp = Hq // Hkv
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    add = torch.zeros(weight.shape, dtype=torch.float64, device=q.device)
    for b, h in itertools.product(range(B), range(Hkv)):
        slots, bias = torch.arange(L, device=q.device), None
        if sel is not None:
            ids = (sel[b] if sel.dim() == 2 else sel[b, h if sel.shape[1] > 1 else 0]).tolist()
            gr = None if gate is None else (gate[b] if gate.dim() == 2 else gate[b, h if gate.shape[1] > 1 else 0])
            live = [i for i, x in enumerate(ids) if 0 <= x * bs < L and x not in ids[:i]]
            slots = torch.tensor([s for i in live for s in range(ids[i] * bs, min(L, (ids[i] + 1) * bs))],
                                 device=q.device, dtype=torch.long)
            if gate is not None:
                bias = torch.cat([gr[i].expand(min(L, (ids[i] + 1) * bs) - ids[i] * bs) for i in live])
        for t in range(T):
            see = (slots <= L - T + t).unsqueeze(0).expand(grp, -1)
            if bias is not None:
                see = see & (bias > -math.inf).unsqueeze(0)
            if not len(slots):
                continue
            r, p, _ = _ref_rows(q[b, h * grp:(h + 1) * grp, t], k[b, h, slots], v[b, h, slots], see, bias, scale)
            o[b, h * grp:(h + 1) * grp, t] = r
            add[b, h, slots] += p.sum(0)
    return o, add


def _weighted_case(cuda, dtype, D, B, Hq, Hkv, L, T, bs=64, kk=0, gate=False, per_head=True, seed=0, room=5):
    g = torch.Generator().manual_seed(seed)
    dt = DT[dtype]
    q = _rand(g, B, Hq, T, D, dt=dt, dev=cuda)
    k, v = _rand(g, B, Hkv, L + room, D, dt=dt, dev=cuda), _rand(g, B, Hkv, L + room, D, dt=dt, dev=cuda)
    k[:, :, L:], v[:, :, L:] = float("nan"), float("inf")     # unused slots may hold anything
    w = torch.rand(B, Hkv, L + room, generator=g).to(cuda)
    sel = gt = None
    if kk:
        nblk = (L + bs - 1) // bs
        shape = (B, Hkv, kk) if per_head else (B, kk)
        sel = torch.randint(0, nblk, shape, generator=g, dtype=torch.int32).to(cuda)
        gt = torch.randn(shape, generator=g).to(cuda) if gate else None
    return q, k, v, w, sel, gt


def _check_weighted(q, k, v, w, sel, gate, bs, L, scale=None):
    import _bsa
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    ref, add = _ref_weighted(q, k, v, w, sel, gate, bs, L, scale)
    w0 = w.double()
    o = _bsa.decode_weighted(q, k, v, w, sel, gate, bs=bs, L=L, scale=scale)
    e = _rel(q, k[:, :, :L], scale)
    fin = v[:, :, :L][torch.isfinite(v[:, :, :L].float())]
    _close_o(o, ref, e, float(fin.abs().max()), "o")
    err, tol = (w.double() - w0 - add).abs(), e * add + 2 ** -23 * (w0 + add)
    assert bool((err <= tol).all()), "weight: %.3g" % err.max().item()
    assert torch.equal(w[add == 0].double(), w0[add == 0])


@pytest.mark.parametrize("dtype,D,B,Hq,Hkv,L,T", [
    ("bf16", 64, 1, 1, 1, 1, 1), ("bf16", 256, 1, 16, 2, 1000, 1), ("f16", 128, 3, 8, 4, 515, 2),
    ("f32", 64, 2, 4, 2, 129, 1), ("bf16", 32, 2, 6, 2, 333, 3), ("f16", 32, 1, 32, 1, 64, 1),
    ("bf16", 128, 2, 24, 1, 2049, 1), ("f16", 256, 1, 24, 1, 65, 1), ("bf16", 64, 1, 40, 2, 700, 1),
    ("f32", 128, 1, 24, 2, 301, 1), ("f32", 256, 2, 4, 1, 77, 2), ("f32", 32, 1, 40, 1, 1000, 1),
    ("bf16", 128, 1, 8, 1, 20, 20), ("f32", 64, 1, 8, 2, 16, 16), ("bf16", 256, 1, 8, 2, 300, 7),
    ("f16", 64, 1, 2, 2, 17, 2), ("f32", 128, 1, 64, 1, 40, 3), ("bf16", 64, 1, 4, 4, 32, 32),
    ("f16", 128, 1, 8, 8, 9001, 1), ("f32", 256, 1, 1, 1, 1, 1),
    # beyond one cluster: splits and their join
    ("bf16", 64, 1, 40, 2, 5000, 1), ("f32", 128, 1, 24, 2, 2500, 3), ("f32", 32, 1, 40, 1, 3000, 1),
    ("bf16", 256, 1, 24, 1, 2100, 2), ("f16", 32, 2, 6, 2, 4200, 3), ("f32", 256, 1, 2, 1, 2100, 1),
    ("f32", 64, 1, 80, 1, 2200, 1), ("bf16", 128, 40, 8, 8, 2100, 1),
])
def test_weighted_every_slot(cuda, dtype, D, B, Hq, Hkv, L, T):
    q, k, v, w, _, _ = _weighted_case(cuda, dtype, D, B, Hq, Hkv, L, T, seed=D + L)
    _check_weighted(q, k, v, w, None, None, None, L)


@pytest.mark.parametrize("dtype,D,B,Hq,Hkv,L,T,bs,kk,gate,per_head", [
    ("bf16", 64, 2, 8, 4, 1000, 1, 64, 7, True, True), ("f16", 128, 1, 8, 2, 4097, 1, 128, 12, False, True),
    ("f32", 64, 2, 4, 2, 777, 2, 32, 9, True, False), ("bf16", 256, 1, 16, 2, 2000, 3, 96, 6, True, True),
    ("f16", 32, 2, 4, 1, 500, 1, 32, 40, True, False), ("bf16", 128, 1, 4, 2, 31, 1, 64, 3, False, True),
    ("f32", 256, 1, 2, 1, 300, 1, 64, 4, True, True), ("f32", 32, 1, 24, 1, 999, 4, 160, 5, False, True),
    ("f16", 128, 1, 8, 2, 9000, 2, 128, 30, True, True), ("f32", 64, 1, 4, 2, 5000, 1, 64, 40, True, False),
    ("bf16", 64, 2, 12, 1, 20000, 3, 96, 60, False, True),
])
def test_weighted_selected_blocks(cuda, dtype, D, B, Hq, Hkv, L, T, bs, kk, gate, per_head):
    q, k, v, w, sel, gt = _weighted_case(cuda, dtype, D, B, Hq, Hkv, L, T, bs, kk, gate, per_head, seed=L)
    sel[..., 0] = (L - 1) // bs                      # the own block, so that every row sees a key
    sel[..., -1] = sel[..., 0]                       # and a repeated id (its second gate is not used)
    if T > 1:                                        # rows whose own block holds no key yet
        sel[..., 1] = 0
    _check_weighted(q, k, v, w, sel, gt, bs, L)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_weighted_masked_rows_and_values(cuda, dtype):
    """Rows that see nothing, an infinite gate, and infinities / NaN where a row does not look."""
    import _bsa
    L, T, bs = 200, 3, 32
    q, k, v, w, sel, gate = _weighted_case(cuda, dtype, 64, 2, 4, 2, L, T, bs, 4, True, seed=4)
    sel[:] = torch.tensor([6, 2, 4, 0], dtype=torch.int32)
    gate[0] = -math.inf                              # sequence 0: nothing at all
    gate[1, :, 1] = -math.inf
    v[1, :, 64:96] = float("nan")                    # block 2: masked by its gate
    before = w.clone()
    o = _bsa.decode_weighted(q, k, v, w, sel, gate, bs=bs, L=L)
    assert torch.equal(o[0], torch.zeros_like(o[0])) and torch.equal(w[0], before[0])
    _check_weighted(q, k, v, before.clone(), sel, gate, bs, L)
    # the newest tokens' V, hidden from the rows before them
    q, k, v, w, _, _ = _weighted_case(cuda, dtype, 64, 1, 4, 2, L, T, seed=5)
    v[:, :, L - 1] = float("nan")
    k[:, :, L - 1] = 0
    o = _bsa.decode_weighted(q, k, v, w, L=L)
    assert torch.isfinite(o[:, :, :T - 1].float()).all() and torch.isnan(o[:, :, T - 1].float()).all()
    # a NaN query is not mistaken for an empty row
    q[0, 0, 0] = float("nan")
    assert torch.isnan(_bsa.decode_weighted(q, k, v, w, L=L)[0, 0, 0].float()).all()


def test_weighted_bad_block_id_is_reported(cuda):
    import _bsa
    L, bs = 200, 64
    q, k, v, w, sel, _ = _weighted_case(cuda, "bf16", 64, 1, 4, 2, L, 1, bs, 4, seed=6)
    _bsa.check_status(cuda)
    sel[0, 0] = torch.tensor([3, 77, -1, 4], dtype=torch.int32)
    _check_weighted(q, k, v, w, sel, None, bs, L)
    with pytest.raises(_bsa.BsaError) as ei:
        _bsa.check_status(cuda)
    assert ei.value.status == _bsa.ERR_INDEX
    _bsa.check_status(cuda)


def test_weighted_strided_views(cuda):
    """A (B, L, H, D) cache, a padded weight tensor, q cut from a fused projection, given out."""
    import _bsa
    g = torch.Generator().manual_seed(3)
    B, Hq, Hkv, L, T, D = 2, 8, 2, 300, 2, 64
    qkv = _rand(g, B, T, Hq * D * 2, dt=torch.bfloat16, dev=cuda)
    q = qkv[..., Hq * D:].view(B, T, Hq, D).transpose(1, 2)
    k = _rand(g, B, L, Hkv, D, dt=torch.bfloat16, dev=cuda).transpose(1, 2)
    v = _rand(g, B, L, Hkv, 2 * D, dt=torch.bfloat16, dev=cuda)[..., :D].transpose(1, 2)
    w = torch.rand(B, Hkv, 400, generator=g).to(cuda)[:, :, 7:]
    _check_weighted(q, k, v, w, None, None, None, L)
    out = torch.empty(B, T, Hq, D, dtype=q.dtype, device=cuda).transpose(1, 2)
    o = _bsa.decode_weighted(q, k, v, w, L=L, out=out)
    assert o is out and torch.equal(out, _bsa.decode_weighted(q, k, v, w, L=L))
    odd = torch.empty(B * Hq * T * D + 1, dtype=q.dtype, device=cuda)[1:].view(B, Hq, T, D).copy_(q)
    assert torch.equal(out, _bsa.decode_weighted(odd, k, v, w, L=L))   # q and o of any alignment


def test_weighted_far_offsets(cuda):
    """Element offsets past 2^31: the one key that matters sits at the end of the cache."""
    import _bsa
    D, L = 256, (2 ** 31) // 256 + 4097
    k = torch.zeros(1, 1, L, D, dtype=torch.bfloat16, device=cuda)
    v = torch.zeros(1, 1, L, D, dtype=torch.bfloat16, device=cuda)
    q = torch.zeros(1, 2, 1, D, dtype=torch.bfloat16, device=cuda)
    q[..., 0] = 32.0
    k[0, 0, L - 3, 0] = 32.0                          # logit 64 against 0: the rest weigh 9e6 e^-64
    v[0, 0, L - 3] = torch.arange(D, device=cuda).to(torch.bfloat16)
    w = torch.zeros(1, 1, L, device=cuda)
    o = _bsa.decode_weighted(q, k, v, w, L=L)
    assert torch.equal(o[0, 0, 0], v[0, 0, L - 3]) and torch.equal(o[0, 1, 0], v[0, 0, L - 3])
    assert w[0, 0, L - 3].item() == 2.0 and float(w.sum()) == 2.0


# ------------------------------------------------------------------ eviction
def _ref_evict(w, pos, L, budget, seen, recent, sink):
    """Source slot of each kept slot, (B, Hkv, budget)."""
    B, H = w.shape[:2]
    src = torch.arange(budget).repeat(B, H, 1)
    for b, h in itertools.product(range(B), range(H)):
        ws, ps = w[b, h, :L].tolist(), pos[b, h, :L].tolist()
        rank = sorted(range(L), key=lambda i: (not (ps[i] < sink or ps[i] >= seen - recent),
                                               math.inf if ws[i] != ws[i] else -ws[i], i))
        kept = set(rank[:budget])
        holes = [i for i in range(budget) if i not in kept]
        tails = sorted(i for i in kept if i >= budget)
        assert len(holes) == len(tails)
        for i, j in zip(holes, tails):
            src[b, h, i] = j
    return src


def _check_evict(cuda, dtype, D, B, H, L, budget, recent, sink, bs, kind, seed, out=False):
    import _bsa
    g = torch.Generator().manual_seed(seed)
    cap = L + 3
    k, v = _rand(g, B, H, cap, D, dt=DT[dtype], dev=cuda), _rand(g, B, H, cap, D, dt=DT[dtype], dev=cuda)
    w = torch.randn(B, H, cap, generator=g).mul(2).exp()
    if kind == "ties":
        w = torch.randint(0, 3, (B, H, cap), generator=g).float() - 1
        w[w == 0] = -0.0
    elif kind == "special":
        w[:, :, ::3] = float("nan")
        w[:, :, 1::7] = math.inf
        w[:, :, 2::5] = -math.inf
    elif kind == "equal":
        w[:] = 1.0
    pos = torch.stack([torch.randperm(2 * L, generator=g)[:cap].to(torch.int32) if 2 * L >= cap else
                       torch.arange(cap, dtype=torch.int32) for _ in range(B * H)]).view(B, H, cap)
    seen = max(2 * L, cap)
    nb = (cap + bs - 1) // bs
    w, pos = w.to(cuda), pos.to(cuda)
    km = torch.zeros(B, H, nb * bs, D, device=cuda)
    km[:, :, :L] = k[:, :, :L]
    kmin, kmax = (x.contiguous() for x in (km.view(B, H, nb, bs, D).amin(3), km.view(B, H, nb, bs, D).amax(3)))
    src = _ref_evict(w.cpu(), pos.cpu(), L, budget, seen, recent, sink).to(cuda)
    b, h = torch.arange(B, device=cuda).view(-1, 1, 1), torch.arange(H, device=cuda).view(1, -1, 1)
    want = [t[b, h, src] for t in (k, v, w, pos)]
    rest = [t[:, :, budget:].clone() for t in (k, v, w, pos)]
    kw = dict(weight_out=torch.empty(B, H, budget, device=cuda),
              pos_out=torch.empty(B, H, budget, dtype=torch.int32, device=cuda)) if out else {}
    w_in = w.clone()
    _bsa.evict(k, v, w, pos, budget=budget, L=L, seen=seen, recent=recent, sink=sink, kmin=kmin, kmax=kmax,
               bs=bs, **kw)
    got = [k[:, :, :budget], v[:, :, :budget], kw.get("weight_out", w[:, :, :budget]),
           kw.get("pos_out", pos[:, :, :budget])]
    for name, x, y in zip(("k", "v", "weight", "pos"), got, want):
        assert torch.equal(x.nan_to_num(7.0) if x.is_floating_point() else x,
                           y.nan_to_num(7.0) if y.is_floating_point() else y), name
    for name, x, y in zip(("k", "v", "weight", "pos"), (k, v, w, pos), rest):
        assert torch.equal(x[:, :, budget:].nan_to_num(7.0) if x.is_floating_point() else x[:, :, budget:],
                           y.nan_to_num(7.0) if y.is_floating_point() else y), name + " beyond the budget"
    if out:
        assert torch.equal(w.nan_to_num(7.0), w_in.nan_to_num(7.0))
    n = (budget + bs - 1) // bs
    km = torch.zeros(B, H, n * bs, D, device=cuda)
    km[:, :, :budget] = k[:, :, :budget]
    assert torch.equal(kmin[:, :, :n], km.view(B, H, n, bs, D).amin(3))
    assert torch.equal(kmax[:, :, :n], km.view(B, H, n, bs, D).amax(3))


@pytest.mark.parametrize("dtype,D,B,H,L,budget,recent,sink,bs,kind,out", [
    ("bf16", 64, 1, 1, 1, 1, 0, 0, 32, "plain", False), ("bf16", 128, 2, 2, 2, 1, 1, 0, 32, "plain", False),
    ("f16", 64, 2, 3, 1000, 999, 16, 4, 64, "plain", False), ("f32", 32, 1, 2, 777, 100, 10, 1, 32, "ties", True),
    ("bf16", 256, 1, 2, 1025, 512, 0, 0, 128, "ties", False), ("f16", 128, 2, 1, 5000, 2500, 77, 2, 64, "special", False),
    ("f32", 256, 1, 1, 300, 299, 299, 0, 128, "plain", True), ("bf16", 64, 1, 2, 2048, 1024, 100, 9, 64, "equal", False),
    ("f32", 64, 1, 3, 20000, 3333, 500, 4, 128, "special", False), ("bf16", 32, 2, 1, 9000, 8999, 0, 0, 64, "ties", True),
    ("f16", 128, 1, 1, 70000, 1, 0, 1, 64, "plain", False), ("bf16", 64, 1, 1, 70001, 69000, 69000, 0, 1024, "ties", False),
    ("f32", 128, 2, 2, 500, 500, 3, 3, 64, "special", True), ("bf16", 64, 1, 1, 100, 50, 25, 25, 48, "special", False),
])
def test_evict(cuda, dtype, D, B, H, L, budget, recent, sink, bs, kind, out):
    _check_evict(cuda, dtype, D, B, H, L, budget, recent, sink, bs, kind, L + budget, out)


def test_evict_without_summaries_and_with_more_protected_than_budget(cuda):
    """The kernels stay inside the cache when the positions are not what they should be."""
    import _bsa
    g = torch.Generator().manual_seed(1)
    k, v = (_rand(g, 1, 2, 64, 64, dt=torch.bfloat16, dev=cuda) for _ in range(2))
    w, pos = torch.rand(1, 2, 64, generator=g).to(cuda), torch.zeros(1, 2, 64, dtype=torch.int32, device=cuda)
    k0 = k.clone()
    _bsa.evict(k, v, w, pos, budget=10, recent=0, sink=1)      # every slot claims position 0
    assert torch.equal(k, k0)                                  # ties: the first ten stay


def test_evict_strided(cuda):
    import _bsa
    g = torch.Generator().manual_seed(2)
    B, H, L, D, n = 2, 2, 150, 64, 60
    k = _rand(g, B, L, H, D, dt=torch.float16, dev=cuda).transpose(1, 2)
    v = _rand(g, H, B, L, D, dt=torch.float16, dev=cuda).transpose(0, 1)
    w = torch.rand(B, H, 200, generator=g).to(cuda)[:, :, 3:]
    pos = torch.arange(200, dtype=torch.int32, device=cuda).repeat(H, B, 1).transpose(0, 1)
    src = _ref_evict(w.cpu(), pos.cpu(), L, n, L, 5, 5).to(cuda)
    b, h = torch.arange(B, device=cuda).view(-1, 1, 1), torch.arange(H, device=cuda).view(1, -1, 1)
    want = [t[b, h, src] for t in (k, v, w, pos)]
    _bsa.evict(k, v, w, pos, budget=n, L=L, recent=5, sink=5)
    for x, y in zip((k, v, w, pos), want):
        assert torch.equal(x[:, :, :n], y)


# ------------------------------------------------------------------ shared prefix
def _check_prefix(q, pk, pv, k, v, lens, scale=None, out=None):
    import _bsa
    B, Hq, T, D = q.shape
    Hkv, P = pk.shape[:2]
    grp, S = Hq // Hkv, k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    o = _bsa.decode_prefix(q, pk, pv, k, v, lens, scale=scale, out=out)
    ref = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    once, vmax = torch.zeros_like(ref), 1e-30
    for b, h in itertools.product(range(B), range(Hkv)):
        n = min(max(int(lens[b]), 0), S)
        kk, vv = torch.cat([pk[h], k[b, h, :n]]), torch.cat([pv[h], v[b, h, :n]])
        if not len(kk):
            continue
        at = torch.arange(P + n, device=q.device)
        for t in range(T):
            see = (at < P) | (at - P <= n - T + t)
            r, _, mean = _ref_rows(q[b, h * grp:(h + 1) * grp, t], kk, vv, see.expand(grp, -1), None, scale)
            ref[b, h * grp:(h + 1) * grp, t] = r
            if o.dtype != torch.float32 and B * grp * T > 16 and P >= 128:
                once[b, h * grp:(h + 1) * grp, t] = torch.finfo(o.dtype).eps / 2 * mean
        fin = vv[torch.isfinite(vv.float())]
        vmax = max(vmax, float(fin.abs().max()))
    kn = torch.cat([pk.reshape(-1, D), k.reshape(-1, D)])
    kn = kn[torch.isfinite(kn.float()).all(-1)]
    _close_o(o, ref, _rel(q, kn, scale) if len(kn) else 0.0, vmax, "o", once)
    return o


def _prefix_case(cuda, dtype, D, B, Hq, Hkv, P, S, T, seed=0):
    g = torch.Generator().manual_seed(seed)
    dt = DT[dtype]
    q = _rand(g, B, Hq, T, D, dt=dt, dev=cuda)
    pk, pv = _rand(g, Hkv, P, D, dt=dt, dev=cuda), _rand(g, Hkv, P, D, dt=dt, dev=cuda)
    k, v = _rand(g, B, Hkv, S, D, dt=dt, dev=cuda), _rand(g, B, Hkv, S, D, dt=dt, dev=cuda)
    lens = torch.randint(min(T, S), S + 1, (B,), generator=g, dtype=torch.int32)
    for b in range(B):
        k[b, :, int(lens[b]):], v[b, :, int(lens[b]):] = float("nan"), float("-inf")
    return q, pk, pv, k, v, lens.to(cuda)


@pytest.mark.parametrize("dtype,D,B,Hq,Hkv,P,S,T", [
    ("bf16", 64, 1, 1, 1, 1, 1, 1), ("bf16", 64, 2, 8, 2, 1000, 17, 1), ("f16", 128, 5, 8, 2, 777, 33, 2),
    ("f32", 64, 3, 4, 2, 130, 9, 1), ("bf16", 256, 9, 16, 1, 300, 20, 1), ("f16", 64, 40, 8, 1, 2000, 5, 1),
    ("bf16", 32, 3, 6, 3, 500, 70, 3), ("f32", 128, 20, 8, 2, 257, 3, 1), ("f32", 256, 2, 4, 4, 65, 129, 2),
    ("bf16", 128, 17, 32, 2, 4097, 40, 1), ("f16", 256, 3, 24, 3, 129, 2, 2), ("f32", 32, 33, 4, 1, 100, 1, 1),
    ("bf16", 128, 1, 64, 1, 640, 64, 3), ("bf16", 64, 150, 2, 2, 130, 12, 1), ("f16", 128, 2, 2, 2, 8192, 1, 1),
    ("f16", 32, 70, 4, 2, 1111, 30, 1), ("bf16", 256, 66, 8, 4, 1500, 9, 1), ("bf16", 64, 1, 4, 4, 0, 50, 2),
    ("f32", 64, 2, 4, 2, 0, 3, 1), ("f16", 128, 64, 4, 1, 127, 600, 4), ("bf16", 128, 3, 384, 3, 256, 6, 1),
    # more than one launch: two row tiles, one, and the split kernels
    ("bf16", 64, 40, 8, 1, 6000, 5, 1), ("f16", 32, 70, 4, 2, 9000, 30, 1), ("bf16", 64, 150, 2, 2, 5000, 12, 1),
    ("f16", 64, 12, 2, 1, 5001, 9, 3), ("f32", 128, 20, 8, 2, 2600, 3, 1), ("f32", 64, 3, 4, 1, 4000, 600, 2),
    ("bf16", 32, 5, 2, 2, 6000, 70, 1), ("f16", 128, 30, 8, 2, 3000, 700, 2), ("bf16", 256, 3, 8, 2, 4500, 30, 1),
])
def test_prefix(cuda, dtype, D, B, Hq, Hkv, P, S, T):
    _check_prefix(*_prefix_case(cuda, dtype, D, B, Hq, Hkv, P, S, T, seed=P + S))


@pytest.mark.parametrize("dtype,B", [("bf16", 3), ("bf16", 90), ("f32", 3)])
def test_prefix_empty_and_bad_lengths(cuda, dtype, B):
    """Length 0 reads the prefix alone; fewer own slots than new tokens; lengths outside
    [0, S] are clamped and reported; with no prefix either, the row is zero."""
    import _bsa
    q, pk, pv, k, v, lens = _prefix_case(cuda, dtype, 64, B, 4, 2, 200, 10, 2, seed=8)
    k, v = k.nan_to_num(0.5), v.nan_to_num(0.5, neginf=0.5)
    lens[:3] = torch.tensor([0, 1, 10], dtype=torch.int32)
    _bsa.check_status(cuda)
    _check_prefix(q, pk, pv, k, v, lens)
    _bsa.check_status(cuda)
    o = _check_prefix(q, pk[:, :0], pv[:, :0], k, v, lens)
    assert torch.equal(o[0], torch.zeros_like(o[0])) and torch.equal(o[1, :, 0], torch.zeros_like(o[1, :, 0]))
    lens[:2] = torch.tensor([-5, 1000], dtype=torch.int32)
    _check_prefix(q, pk, pv, k, v, lens)
    with pytest.raises(_bsa.BsaError):
        _bsa.check_status(cuda)


@pytest.mark.parametrize("B", [2, 40])
def test_prefix_strided_and_hidden_values(cuda, B):
    g = torch.Generator().manual_seed(9)
    Hq, Hkv, P, S, T, D = 8, 2, 333, 40, 3, 128
    pk = _rand(g, P, Hkv, D, dt=torch.bfloat16, dev=cuda).transpose(0, 1)
    pv = _rand(g, P, Hkv, 2 * D, dt=torch.bfloat16, dev=cuda)[..., D:].transpose(0, 1)
    k = _rand(g, B, S, Hkv, D, dt=torch.bfloat16, dev=cuda).transpose(1, 2)
    v = _rand(g, B, S, Hkv, D, dt=torch.bfloat16, dev=cuda).transpose(1, 2)
    q = _rand(g, B, T, Hq, D, dt=torch.bfloat16, dev=cuda).transpose(1, 2)
    lens = torch.full((B,), 37, dtype=torch.int64, device=cuda)
    out = torch.empty(B, T, Hq, D, dtype=torch.bfloat16, device=cuda).transpose(1, 2)
    assert _check_prefix(q, pk, pv, k, v, lens, scale=0.2, out=out) is out
    import _bsa
    v[:, :, 36] = float("nan")                       # the newest token, seen by the last row alone
    o = _bsa.decode_prefix(q, pk, pv, k, v, lens)
    assert torch.isfinite(o[:, :, :T - 1].float()).all() and torch.isnan(o[:, :, T - 1].float()).all()


# ------------------------------------------------------------------ together
def test_cache_within_a_budget(cuda):
    """Prompt, decode steps, evictions: every step's output and sums against the definition
    on the cache's own contents, every eviction against the rule on the cache's own sums."""
    import decode
    g = torch.Generator().manual_seed(10)
    B, Hq, Hkv, D, bs, budget = 2, 8, 2, 64, 32, 100
    c = decode.DecodeCache(B, Hkv, 300, D, bs=bs, device=cuda, track=True)
    tok = lambda n: (_rand(g, B, Hkv, n, D, dt=torch.bfloat16, dev=cuda) for _ in range(2))  # noqa: E731
    c.append(*tok(250))
    for step in range(6):
        T = 1 + step % 2
        c.append(*tok(T))
        q = _rand(g, B, Hq, T, D, dt=torch.bfloat16, dev=cuda)
        w = c.weight.clone()
        sel = c.select_quest(q, topk=3) if step == 3 else None
        ref, add = _ref_weighted(q, c.k, c.v, w, sel, None, bs, c.L, D ** -0.5)
        o = decode.decode_attention_weighted(q, c, sel)
        e = _rel(q, c.k[:, :, :c.L], D ** -0.5)
        _close_o(o, ref, e, float(c.v.abs().max()), "step %d" % step)
        assert bool(((c.weight.double() - w.double() - add).abs() <= e * add + 2 ** -23 * (w + add)).all())
        src = _ref_evict(c.weight.cpu(), c.pos.cpu(), c.L, budget, c.seen, 20, 4).to(cuda)
        b, h = torch.arange(B, device=cuda).view(-1, 1, 1), torch.arange(Hkv, device=cuda).view(1, -1, 1)
        want = [t[b, h, src] for t in (c.k, c.v, c.weight, c.pos)]
        gone = c.L - budget
        assert c.evict(budget, recent=20, sink=4) == gone and c.L == budget
        for x, y in zip((c.k, c.v, c.weight, c.pos), want):
            assert torch.equal(x[:, :, :budget], y)
        km = torch.zeros(B, Hkv, 128, D, device=cuda)
        km[:, :, :budget] = c.k[:, :, :budget]
        assert torch.equal(c.kmin[:, :, :4], km.view(B, Hkv, 4, bs, D).amin(3))
        assert torch.equal(c.kmax[:, :, :4], km.view(B, Hkv, 4, bs, D).amax(3))
        # the newest token is there, whatever its weight
        assert bool((c.pos[:, :, :budget] == c.seen - 1).any(-1).all())
    assert c.evict(budget) == 0
    # the existing decode reads the same cache
    o = decode.decode_attention(q, c, torch.arange(4, device=cuda, dtype=torch.int32).expand(B, Hkv, 4))
    assert torch.isfinite(o.float()).all()


def test_untracked_cache_refuses(cuda):
    import decode
    c = decode.DecodeCache(1, 1, 64, 64, bs=32, device=cuda)
    c.append(*(torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16, device=cuda) for _ in range(2)))
    with pytest.raises(ValueError):
        c.evict(2)
    with pytest.raises(ValueError):
        decode.decode_attention_weighted(torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device=cuda), c)


def test_prefix_cache(cuda):
    import decode
    g = torch.Generator().manual_seed(11)
    B, Hq, Hkv, P, D = 3, 8, 2, 500, 128
    pk, pv = (_rand(g, Hkv, P, D, dt=torch.bfloat16, dev=cuda) for _ in range(2))
    c = decode.PrefixCache(pk, pv, B, 12)
    own = [[torch.zeros(Hkv, 0, D, dtype=torch.bfloat16, device=cuda) for _ in range(2)] for _ in range(B)]
    for step, (T, active) in enumerate([(1, None), (2, [True, False, True]), (1, [False, True, True]), (3, None)]):
        kn, vn = (_rand(g, B, Hkv, T, D, dt=torch.bfloat16, dev=cuda) for _ in range(2))
        c.append(kn, vn, active)
        if step == 2:
            c.reset(0)
            own[0] = [x[:, :0] for x in own[0]]
        for b in range(B):
            if active is None or active[b]:
                own[b] = [torch.cat([own[b][0], kn[b]], 1), torch.cat([own[b][1], vn[b]], 1)]
        assert c.lens.tolist() == c.used == [x[0].shape[1] for x in own]
        q = _rand(g, B, Hq, T, D, dt=torch.bfloat16, dev=cuda)
        o = decode.prefix_attention(q, c)
        for b in range(B):
            n = own[b][0].shape[1]
            assert torch.equal(c.k[b, :, :n], own[b][0]) and torch.equal(c.v[b, :, :n], own[b][1])
        _check_prefix(q, pk, pv, c.k, c.v, c.lens)
        assert torch.equal(o, decode.prefix_attention(q, c))
    with pytest.raises(ValueError):
        c.append(*(torch.zeros(B, Hkv, 8, D, dtype=torch.bfloat16, device=cuda) for _ in range(2)))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_streams_and_graphs(cuda, dtype):
    """Another stream, and two captured graphs replayed in turn, give the eager results."""
    import _bsa
    L = 1500
    qw = _weighted_case(cuda, dtype, 64, 2, 8, 2, L, 1, seed=12)[:4]
    pf = _prefix_case(cuda, dtype, 64, 30, 8, 2, 700, 9, 1, seed=13)
    g = torch.Generator().manual_seed(14)
    ev = [_rand(g, 1, 2, 256, 64, dt=DT[dtype], dev=cuda) for _ in range(2)] + \
        [torch.rand(1, 2, 256, generator=g).to(cuda), torch.arange(256, dtype=torch.int32, device=cuda).repeat(1, 2, 1)]

    def step(w, e):
        o = _bsa.decode_weighted(qw[0], qw[1], qw[2], w, L=L)
        _bsa.evict(*e, budget=200, recent=10, kmin=None)
        return o, _bsa.decode_prefix(*pf)

    w0, e0 = qw[3].clone(), [t.clone() for t in ev]
    o1, o2 = step(w0, e0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w1, e1 = qw[3].clone(), [t.clone() for t in ev]
        a1, a2 = step(w1, e1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a1, o1) and torch.equal(a2, o2) and torch.equal(w1.nan_to_num(), w0.nan_to_num())
    assert all(torch.equal(x, y) for x, y in zip(e0, e1))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        w, e = qw[3].clone(), [t.clone() for t in ev]
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = step(w, e)
        graphs.append((gr, w, e, outs))
    for n in (1, 2):
        for gr, w, e, outs in graphs:
            w.copy_(qw[3])
            for x, y in zip(e, ev):
                x.copy_(y)
            gr.replay()
        torch.cuda.synchronize()
        for gr, w, e, outs in graphs:
            assert torch.equal(outs[0], o1) and torch.equal(outs[1], o2) and torch.equal(w.nan_to_num(), w0.nan_to_num())
            assert all(torch.equal(x, y) for x, y in zip(e, e0))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_deterministic(cuda, dtype):
    import _bsa
    q, k, v, w, _, _ = _weighted_case(cuda, dtype, 128, 2, 8, 2, 3001, 2, seed=15)
    pf = _prefix_case(cuda, dtype, 128, 33, 8, 2, 2000, 9, 1, seed=16)
    w1, w2 = w.clone(), w.clone()
    assert torch.equal(_bsa.decode_weighted(q, k, v, w1, L=3001), _bsa.decode_weighted(q, k, v, w2, L=3001))
    assert torch.equal(w1, w2)
    assert torch.equal(_bsa.decode_prefix(*pf), _bsa.decode_prefix(*pf))


# ------------------------------------------------------------------ calls off the usual path
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("L", [50, 5000])
def test_weighted_expanded_and_aliased_operands(cuda, dtype, L):
    """K/V read by several batch rows or heads (expanded), V the same tensor as K, a query
    on an odd offset whose rows the output replaces."""
    import _bsa
    B, Hq, Hkv, T, D = 3, 8, 2, 2, 64
    q, k, v, w, _, _ = _weighted_case(cuda, dtype, D, 1, Hq, 1, L, T)
    k, v = k.expand(B, Hkv, -1, -1), v.expand(B, Hkv, -1, -1)
    w = torch.rand(B, Hkv, L, generator=torch.Generator().manual_seed(1)).to(cuda)
    buf = _rand(torch.Generator().manual_seed(2), B, T, Hq, D + 1, dt=DT[dtype], dev=cuda)
    q = buf[..., 1:].transpose(1, 2)
    ref, add = _ref_weighted(q, k, k, w, None, None, 64, L, D ** -0.5)
    e, w0 = _rel(q, k[:, :, :L], D ** -0.5), w.double()
    edge = buf[..., 0].clone()
    o = _bsa.decode_weighted(q, k, k, w, L=L, out=q)
    assert o.data_ptr() == q.data_ptr() and torch.equal(buf[..., 0], edge)
    _close_o(o, ref, e, float(k[:, :, :L].abs().max()), "o")
    assert bool(((w.double() - w0 - add).abs() <= e * add + 2 ** -23 * (w0 + add)).all())


def test_weighted_many_sequences(cuda):
    """More (batch, head) pairs than a grid's second axis holds."""
    import _bsa
    B, L, D = 66000, 9, 32
    g = torch.Generator().manual_seed(3)
    q, k, v = (_rand(g, B, 1, n, D, dt=torch.bfloat16, dev=cuda) for n in (1, L, L))
    w = torch.zeros(B, 1, L, device=cuda)
    o = _bsa.decode_weighted(q, k, v, w)
    p = torch.softmax(q.double() @ k.double().transpose(2, 3) * D ** -0.5, -1)
    e = _rel(q, k, D ** -0.5)
    _close_o(o, p @ v.double(), e, float(v.abs().max()), "o")
    assert bool(((w.double() - p[:, :, 0]).abs() <= e * p[:, :, 0] + 2 ** -23).all())


@pytest.mark.parametrize("dtype,D,B,H,L,budget,recent,sink,bs,kind,out", [
    # slots that do not fit a cluster's registers, ties over several CTAs, one slot left, blocks of one slot
    ("bf16", 32, 1, 2, 300001, 150000, 1000, 4, 128, "plain", False), ("f16", 32, 2, 1, 140000, 139999, 0, 0, 64, "ties", True),
    ("f32", 32, 1, 1, 200000, 77777, 5, 0, 1024, "equal", False), ("bf16", 64, 1, 2, 5000, 1, 1, 0, 64, "plain", False),
    ("bf16", 64, 2, 2, 300, 200, 3, 2, 1, "special", False),
])
def test_evict_long_and_small(cuda, dtype, D, B, H, L, budget, recent, sink, bs, kind, out):
    _check_evict(cuda, dtype, D, B, H, L, budget, recent, sink, bs, kind, L + budget, out)


def test_evict_interleaved_outputs(cuda):
    """Sums and their outputs in one buffer, rows side by side; K and V in one, head by head."""
    import _bsa
    B, H, L, D, n = 2, 3, 700, 64, 300
    g = torch.Generator().manual_seed(5)
    kv = _rand(g, B, L, H, 2, D, dt=torch.bfloat16, dev=cuda)
    k, v = kv[:, :, :, 0].transpose(1, 2), kv[:, :, :, 1].transpose(1, 2)
    wbuf = torch.rand(B, H, 2, L, generator=g).to(cuda)
    pbuf = torch.arange(L, dtype=torch.int32, device=cuda).repeat(B, H, 2, 1)
    src = _ref_evict(wbuf[:, :, 0].cpu(), pbuf[:, :, 0].cpu(), L, n, L, 20, 3).to(cuda)
    b, h = torch.arange(B, device=cuda).view(-1, 1, 1), torch.arange(H, device=cuda).view(1, -1, 1)
    want = [t[b, h, src] for t in (k, v, wbuf[:, :, 0], pbuf[:, :, 0])]
    w0 = wbuf[:, :, 0].clone()
    _bsa.evict(k, v, wbuf[:, :, 0], pbuf[:, :, 0], budget=n, recent=20, sink=3, weight_out=wbuf[:, :, 1],
               pos_out=pbuf[:, :, 1])
    for x, y in zip((k, v, wbuf[:, :, 1], pbuf[:, :, 1]), want):
        assert torch.equal(x[:, :, :n], y)
    assert torch.equal(wbuf[:, :, 0], w0)


@pytest.mark.parametrize("dtype,D,B,Hq,Hkv,P,S,T", [
    # fp32 rows over the warps: several row tiles, a last one of one row, chunks that end inside
    ("f32", 256, 33, 4, 1, 1500, 9, 1), ("f32", 256, 9, 4, 1, 33, 70, 1), ("f32", 128, 43, 6, 2, 2001, 5, 1),
    ("f32", 128, 65, 1, 1, 15, 300, 3), ("f32", 128, 129, 2, 2, 700, 4, 1), ("f32", 64, 300, 4, 1, 1000, 8, 1),
])
def test_prefix_many_rows_fp32(cuda, dtype, D, B, Hq, Hkv, P, S, T):
    _check_prefix(*_prefix_case(cuda, dtype, D, B, Hq, Hkv, P, S, T, seed=P))


@pytest.mark.parametrize("dtype,D,B,Hq,Hkv,P,S,T", [
    # D 256 and more than 128 rows: pairs of CTAs; one key tile, a ragged last one, a second CTA
    # with few rows or none, several row tiles, as many steps as the ring is long and more
    ("bf16", 256, 17, 8, 1, 128, 5, 1), ("f16", 256, 129, 2, 2, 300, 5, 1), ("bf16", 256, 33, 8, 2, 1000, 9, 1),
    ("f16", 256, 70, 8, 2, 20001, 33, 1), ("bf16", 256, 40, 8, 1, 33000, 20, 2), ("f16", 256, 65, 16, 1, 129, 40, 3),
    ("bf16", 256, 64, 4, 2, 70000, 5, 1), ("bf16", 256, 300, 2, 2, 191, 3, 1),
])
def test_prefix_pairs(cuda, dtype, D, B, Hq, Hkv, P, S, T):
    _check_prefix(*_prefix_case(cuda, dtype, D, B, Hq, Hkv, P, S, T, seed=P))


@pytest.mark.parametrize("dtype,B", [("bf16", 2), ("bf16", 40), ("f32", 40)])
def test_prefix_expanded_and_aliased_operands(cuda, dtype, B):
    """A prefix shared by the heads too (expanded), own slots shared by the batch, the
    output in the query's place."""
    import _bsa
    Hq, Hkv, P, S, T, D = 4, 2, 500, 20, 1, 64
    q, pk, pv, k, v, lens = _prefix_case(cuda, dtype, D, B, Hq, Hkv, P, S, T, seed=B)
    k, v = k.nan_to_num(0.0), v.nan_to_num(0.0, 0.0, 0.0)
    pk, pv = pk[:1].expand(Hkv, -1, -1), pv[:1].expand(Hkv, -1, -1)
    k, v = k[:1].expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1)
    want = _check_prefix(q, pk, pv, k, v, lens)
    out = _bsa.decode_prefix(q, pk, pv, k, v, lens, out=q)
    assert out.data_ptr() == q.data_ptr() and torch.equal(out, want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prefix_nan_query_stays_in_its_row(cuda, dtype):
    """A NaN in one head's query stays in its row."""
    import _bsa
    q, pk, pv, k, v, lens = _prefix_case(cuda, dtype, 128, 20, 8, 1, 400, 6, 1)
    k, v = k.nan_to_num(0.0), v.nan_to_num(0.0, 0.0, 0.0)
    want = _bsa.decode_prefix(q, pk, pv, k, v, lens)
    q2 = q.clone()
    q2[3, 5] = float("nan")
    o = _bsa.decode_prefix(q2, pk, pv, k, v, lens)
    assert bool(o[3, 5].isnan().all())
    o[3, 5] = want[3, 5]
    assert torch.equal(o, want)


@pytest.mark.parametrize("B,Hq,Hkv,D,P,T", [(36, 32, 8, 128, 2873, 1), (17, 6, 2, 64, 79856, 4),
                                            (100, 8, 1, 256, 20000, 1), (2, 16, 2, 256, 60000, 1)])
def test_fp32_is_as_exact_as_fp32_arithmetic(cuda, B, Hq, Hkv, D, P, T):
    """The products truncate what they sum, so errors of long sums would all have one sign.
    Summed afresh for every 16 keys, their six products leave at most 6 2^-23 of a part, and
    the D / 16 of a logit about half of 2^-23 each: in the 2-norm that much beside the error
    of the same formula in fp32."""
    import _bsa
    g = torch.Generator().manual_seed(P)
    f32 = torch.float32
    q, pk, pv = (_rand(g, *s, dt=f32, dev=cuda) for s in ((B, Hq, T, D), (Hkv, P, D), (Hkv, P, D)))
    k, v = torch.zeros(2, B, Hkv, 1, D, device=cuda)
    o = _bsa.decode_prefix(q, pk, pv, k, v, torch.zeros(B, dtype=torch.int32, device=cuda)).double()
    ref, plain = torch.empty_like(o), torch.empty_like(o)
    for h in range(Hq):
        for to, dt in ((ref, torch.float64), (plain, f32)):
            kk, vv = pk[h * Hkv // Hq].to(dt), pv[h * Hkv // Hq].to(dt)
            x = torch.softmax(q[:, h].reshape(-1, D).to(dt) @ kk.t() * D ** -0.5, -1) @ vv
            to[:, h] = x.view(B, T, D).double()
    err, of_plain = ((x - ref).norm() / ref.norm() for x in (o, plain))
    assert err <= of_plain + (6 + D / 32) * 2 ** -23
