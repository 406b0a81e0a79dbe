"""Serving operators of the decode cache: their cases, plain forms and exact values.

  weighted  decode attention over a K/V cache that adds every slot's attention weight to a running sum
  evict     reduction of a cache to a budget of slots by that running sum
  prefix    decode attention of a batch whose sequences share one long prefix
"""
import functools
import math
import os
import sys
from types import SimpleNamespace

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@functools.lru_cache(None)
def _fw():
    """The framework's binding (its modules are imported flat from the package folder)."""
    here = os.path.join(os.getcwd(), "fused-block-sparse-attention_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import _bsa
    return _bsa


# ------------------------------------------------------------------ cases
def listed():
    def w(name, B, Hq, Hkv, D, L, T, bs, topk, gate, dtype):
        return dict(name=name, op="weighted", B=B, Hq=Hq, Hkv=Hkv, D=D, L=L, T=T, bs=bs, topk=topk, gate=gate,
                    dtype=dtype)

    def e(name, B, Hkv, D, L, budget, recent, sink, bs, aged, dtype):
        return dict(name=name, op="evict", B=B, Hkv=Hkv, D=D, L=L, budget=budget, recent=recent, sink=sink, bs=bs,
                    aged=aged, dtype=dtype)

    def p(name, B, Hq, Hkv, D, P, S, T, dtype):
        return dict(name=name, op="prefix", B=B, Hq=Hq, Hkv=Hkv, D=D, P=P, S=S, T=T, dtype=dtype)

    return [
        # one sequence early in its answer: the latency of a step
        w("weighted, one short sequence", 1, 16, 2, 256, 1000, 1, 128, 0, False, "bf16"),
        # a small batch of long documents, every slot read
        w("weighted, long caches", 4, 16, 2, 256, 65536, 1, 128, 0, False, "bf16"),
        # block-sparse step over a very long cache: the selected blocks and their gates
        w("weighted, selected blocks", 2, 8, 8, 64, 262144, 1, 64, 16, True, "bf16"),
        # several new tokens at once (drafts to be checked) over an odd length
        w("weighted, four new tokens", 3, 32, 8, 128, 32777, 4, 64, 0, False, "f16"),
        # the type that numerics are checked in
        w("weighted, fp32", 2, 4, 2, 64, 4097, 1, 64, 0, False, "f32"),
        # every step makes room for one new token
        e("evict, one slot a step", 4, 2, 256, 4097, 4096, 64, 4, 128, True, "bf16"),
        # a prompt's cache cut to a quarter once it has been read
        e("evict, a prompt to a quarter", 8, 8, 128, 32768, 8192, 512, 4, 64, False, "f16"),
        # odd sizes, a budget that ends inside a block
        e("evict, odd sizes, fp32", 3, 4, 64, 5000, 777, 33, 1, 32, True, "f32"),
        # two continuations of a short instruction
        p("prefix, short", 2, 8, 2, 64, 1000, 17, 1, "bf16"),
        # a batch of questions about one long document
        p("prefix, long document", 32, 16, 2, 256, 65536, 512, 1, "bf16"),
        # a large batch behind one system prompt
        p("prefix, large batch", 128, 32, 8, 128, 32768, 1024, 1, "f16"),
        # drafts, odd sizes, the type that numerics are checked in
        p("prefix, two new tokens, fp32", 6, 6, 3, 128, 2311, 40, 2, "f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _most(op):
    ws = [work(c) for c in listed() if c["op"] == op]
    return max(w["bytes"] for w in ws), max(w["flops"] for w in ws)


def draw(rng):
    op = rng.choice(["weighted", "weighted", "evict", "prefix", "prefix"])
    most = _most(op)
    while True:
        D, dtype = rng.choice([64, 64, 128, 128, 256, 32]), rng.choice(["bf16", "bf16", "f16", "f32"])
        Hkv, bs = rng.choice([1, 2, 3, 4, 8]), rng.choice([32, 64, 128])
        if op == "weighted":
            grp, T = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 1, 2, 3, 5])
            topk = rng.choice([0, 0, 8, 16, 32])
            c = dict(op=op, B=_log(rng, 1, 16), Hq=Hkv * grp, Hkv=Hkv, D=D, L=_log(rng, 8, 200000), T=T, bs=bs,
                     topk=topk, gate=bool(topk) and rng.random() < 0.5, dtype=dtype)
        elif op == "evict":
            L = _log(rng, 16, 100000)
            budget = L - 1 if rng.random() < 0.3 else max(1, int(L * rng.uniform(0.05, 0.95)))
            c = dict(op=op, B=_log(rng, 1, 16), Hkv=Hkv, D=D, L=L, budget=budget,
                     recent=rng.randint(0, budget // 2), sink=min(budget // 2, rng.randint(0, 4)), bs=bs,
                     aged=rng.random() < 0.5, dtype=dtype)
        else:
            grp, T = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 1, 2, 4])
            c = dict(op=op, B=_log(rng, 1, 160), Hq=Hkv * grp, Hkv=Hkv, D=D, P=_log(rng, 8, 100000),
                     S=_log(rng, T, 1200), T=T, dtype=dtype)
        w = work(c)
        if w["bytes"] <= most[0] and w["flops"] <= most[1]:
            return c


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    c = SimpleNamespace(**case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[c.dtype]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dt)

    s = SimpleNamespace(c=c)
    if c.op == "weighted":
        # a cache with room for more tokens; logits of a few units, as trained heads have them
        cap = (c.L // c.bs + 2) * c.bs
        s.q = normal(c.B, c.Hq, c.T, c.D, scale=1.5)
        s.k, s.v = normal(c.B, c.Hkv, cap, c.D), normal(c.B, c.Hkv, cap, c.D)
        # the sums of some hundred earlier steps; slots not yet written hold zero
        s.weight = torch.randn(c.B, c.Hkv, cap, generator=g, device="cuda").mul_(1.5).exp_()
        s.weight[:, :, c.L:] = 0
        s.sel = s.gate = None
        if c.topk:
            # the layout that the cache's Quest selection gives: picks, own block and sink, ascending, ids may repeat
            own_blk = (c.L - 1) // c.bs
            pick = torch.randint(0, own_blk + 1, (c.B, c.Hkv, c.topk + 2), generator=g, device="cuda",
                                 dtype=torch.int32)
            pick[..., 0], pick[..., 1] = own_blk, 0
            s.sel = pick.sort(-1).values.contiguous()
            if c.gate:
                s.gate = torch.nn.functional.logsigmoid(
                    torch.randn(s.sel.shape, generator=g, device="cuda").mul_(2))
    elif c.op == "evict":
        cap = (c.L // c.bs + 1) * c.bs
        s.k, s.v = normal(c.B, c.Hkv, cap, c.D), normal(c.B, c.Hkv, cap, c.D)
        s.weight = torch.randn(c.B, c.Hkv, cap, generator=g, device="cuda").mul_(1.5).exp_()
        s.pos = torch.arange(cap, device="cuda", dtype=torch.int32).repeat(c.B, c.Hkv, 1)
        s.seen = c.L
        if c.aged:  # earlier evictions: half of the tokens are gone, the others sit in any slot
            s.seen = 2 * c.L
            at = torch.rand(c.B, c.Hkv, c.L, generator=g, device="cuda").argsort(dim=-1)
            s.pos[:, :, :c.L] = (2 * at + torch.randint(0, 2, at.shape, generator=g, device="cuda")).to(torch.int32)
        s.kmin, s.kmax = _pooled(s.k[:, :, :c.L], c.bs)
        s.weight_out = torch.empty(c.B, c.Hkv, c.budget, device="cuda")
        s.pos_out = torch.empty(c.B, c.Hkv, c.budget, device="cuda", dtype=torch.int32)
    else:
        s.q = normal(c.B, c.Hq, c.T, c.D, scale=1.5)
        s.pk, s.pv = normal(c.Hkv, c.P, c.D), normal(c.Hkv, c.P, c.D)
        s.k, s.v = normal(c.B, c.Hkv, c.S, c.D), normal(c.B, c.Hkv, c.S, c.D)
        # ragged continuations: from the new tokens alone to all that there is room for
        s.lens = torch.randint(c.T, c.S + 1, (c.B,), generator=g, device="cuda", dtype=torch.int32)
    return s


# ------------------------------------------------------------------ plain forms
def _softmax(x):
    """Softmax over the last axis; a row of -inf gives zeros."""
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    z = e.sum(-1, keepdim=True)
    return e / torch.where(z > 0, z, torch.ones_like(z))


def _pooled(k, bs):
    """Per-block min and max of the rows, those past the end counted as zeros."""
    B, H, L, D = k.shape
    n = (L + bs - 1) // bs
    x = torch.zeros(B, H, n * bs, D, device=k.device)
    x[:, :, :L] = k
    x = x.view(B, H, n, bs, D)
    return x.amin(3), x.amax(3)


def _weighted(s):
    c = s.c
    grp, dev = c.Hq // c.Hkv, s.q.device
    q = s.q.float().view(c.B, c.Hkv, grp * c.T, c.D)
    row = torch.arange(c.T, device=dev).repeat(grp) + (c.L - c.T)  # position of each query row
    if s.sel is None:
        k, v = s.k[:, :, :c.L].float(), s.v[:, :, :c.L].float()
        key = torch.arange(c.L, device=dev).view(1, 1, 1, -1)
        off = key > row.view(1, 1, -1, 1)
        bias = None
    else:
        kk = s.sel.shape[-1]
        slot = (s.sel.long().unsqueeze(-1) * c.bs + torch.arange(c.bs, device=dev)).view(c.B, c.Hkv, kk * c.bs)
        b, h = torch.arange(c.B, device=dev).view(-1, 1, 1), torch.arange(c.Hkv, device=dev).view(1, -1, 1)
        k, v = s.k[b, h, slot].float(), s.v[b, h, slot].float()
        again = ((s.sel.unsqueeze(-1) == s.sel.unsqueeze(-2)).long().tril(-1).sum(-1) > 0).repeat_interleave(c.bs, -1)
        off = (slot.unsqueeze(2) > row.view(1, 1, -1, 1)) | again.unsqueeze(2)
        bias = None if s.gate is None else s.gate.repeat_interleave(c.bs, -1).unsqueeze(2)
    x = torch.matmul(q, k.transpose(-1, -2)) * c.D ** -0.5
    if bias is not None:
        x = x + bias
    p = _softmax(x.masked_fill(off, float("-inf")))
    o = torch.matmul(p, v).view(c.B, c.Hq, c.T, c.D).to(s.q.dtype)
    if s.sel is None:
        s.weight[:, :, :c.L] += p.sum(2)
    else:
        s.weight.scatter_add_(2, slot, p.sum(2))
    return o, s.weight


def _evict(s):
    c = s.c
    w, pos = s.weight[:, :, :c.L], s.pos[:, :, :c.L]
    kept = (pos < c.sink) | (pos >= s.seen - c.recent)
    order = torch.where(torch.isnan(w), torch.full_like(w, float("-inf")), w).argsort(dim=-1, descending=True, stable=True)
    order = order.gather(-1, kept.gather(-1, order).long().argsort(dim=-1, descending=True, stable=True))
    stays = torch.zeros_like(kept).scatter_(-1, order[..., :c.budget], True)
    hole = ~stays[..., :c.budget]
    tail = stays[..., c.budget:].long().argsort(dim=-1, descending=True, stable=True) + c.budget
    nth = (hole.long().cumsum(-1) - 1).clamp_(0, max(tail.shape[-1] - 1, 0))
    at = torch.arange(c.budget, device=w.device).expand_as(nth)
    src = torch.where(hole, tail.gather(-1, nth), at) if tail.shape[-1] else at
    s.weight_out.copy_(w.gather(-1, src))
    s.pos_out.copy_(pos.gather(-1, src))
    b = torch.arange(c.B, device=w.device).view(-1, 1, 1)
    h = torch.arange(c.Hkv, device=w.device).view(1, -1, 1)
    s.k[:, :, :c.budget], s.v[:, :, :c.budget] = s.k[b, h, src], s.v[b, h, src]
    n = (c.budget + c.bs - 1) // c.bs
    s.kmin[:, :, :n], s.kmax[:, :, :n] = _pooled(s.k[:, :, :c.budget], c.bs)


def _prefix(s):
    c = s.c
    grp, dev = c.Hq // c.Hkv, s.q.device
    rows = s.q.float().view(c.B, c.Hkv, grp * c.T, c.D) * c.D ** -0.5
    shared = rows.transpose(0, 1).reshape(c.Hkv, c.B * grp * c.T, c.D)
    x = torch.matmul(shared, s.pk.float().transpose(-1, -2)).view(c.Hkv, c.B, grp * c.T, c.P)
    y = torch.matmul(rows, s.k.float().transpose(-1, -2))
    last = s.lens.view(-1, 1).long() - c.T + torch.arange(c.T, device=dev).repeat(grp)
    off = torch.arange(c.S, device=dev).view(1, 1, 1, -1) > last.view(c.B, 1, grp * c.T, 1)
    y = y.masked_fill_(off, float("-inf"))
    m = torch.maximum(x.amax(-1).transpose(0, 1), y.amax(-1)).unsqueeze(-1)
    x = x.sub_(m.transpose(0, 1)).exp_()
    y = y.sub_(m).exp_()
    z = x.sum(-1, keepdim=True).transpose(0, 1) + y.sum(-1, keepdim=True)
    o = torch.matmul(x.view(c.Hkv, c.B * grp * c.T, c.P), s.pv.float()).view(c.Hkv, c.B, grp * c.T, c.D)
    o = (o.transpose(0, 1) + torch.matmul(y, s.v.float())) / z
    return o.reshape(c.B, c.Hq, c.T, c.D).to(s.q.dtype)


def run(state):
    s, c = state, state.c
    if c.op == "weighted":
        if own:
            o = _fw().decode_weighted(s.q, s.k, s.v, s.weight, s.sel, s.gate, bs=c.bs, L=c.L)
            return {"o": o, "weight": s.weight}
        o, weight = _weighted(s)
        return {"o": o, "weight": weight}
    if c.op == "evict":
        if own:
            _fw().evict(s.k, s.v, s.weight, s.pos, budget=c.budget, L=c.L, seen=s.seen, recent=c.recent, sink=c.sink,
                        kmin=s.kmin, kmax=s.kmax, bs=c.bs, weight_out=s.weight_out, pos_out=s.pos_out)
        else:
            _evict(s)
        n = (c.budget + c.bs - 1) // c.bs
        return {"k": s.k[:, :, :c.budget], "v": s.v[:, :, :c.budget], "weight": s.weight_out, "pos": s.pos_out,
                "kmin": s.kmin[:, :, :n], "kmax": s.kmax[:, :, :n]}
    if own:
        return {"o": _fw().decode_prefix(s.q, s.pk, s.pv, s.k, s.v, s.lens)}
    return {"o": _prefix(s)}


# ------------------------------------------------------------------ work
def work(case):
    c = SimpleNamespace(**case)
    es = 4 if c.dtype == "f32" else 2
    if c.op == "weighted":
        # with a selection: the expected number of different blocks among random picks
        nblk = (c.L + c.bs - 1) // c.bs
        blocks = min(nblk, 2 + nblk * (1 - (1 - 1 / nblk) ** c.topk)) if c.topk else nblk
        n = min(c.L, blocks * c.bs) if c.topk else c.L
        return {"bytes": c.B * c.Hkv * n * (2 * c.D * es + 8) + 2 * c.B * c.Hq * c.T * c.D * es,
                "flops": 4 * c.B * c.Hq * c.T * n * c.D}
    if c.op == "evict":
        # expected survivors beyond the budget, and the blocks that they change
        m = c.budget * (c.L - c.budget) / c.L
        n = (c.budget + c.bs - 1) // c.bs
        changed = n * (1 - (1 - 1 / n) ** m)
        per = 8 * c.L + 8 * c.budget + 4 * m * c.D * es + max(0.0, changed * c.bs - m) * c.D * es + changed * 8 * c.D
        return {"bytes": c.B * c.Hkv * per, "flops": c.B * c.Hkv * c.L}
    mean = (c.T + c.S) / 2
    return {"bytes": 2 * c.Hkv * (c.P + c.B * mean) * c.D * es + 2 * c.B * c.Hq * c.T * c.D * es + 4 * c.B,
            "flops": 4 * c.B * c.Hq * c.T * c.D * (c.P + mean)}


# ------------------------------------------------------------------ exact values
def exact(case, seed):
    """From the definitions, one sequence and head at a time, in 64 bits."""
    s = prepare(case, seed)
    c = s.c
    if c.op == "evict":
        return _exact_evict(s)
    grp = c.Hq // c.Hkv
    o = torch.zeros(c.B, c.Hq, c.T, c.D, dtype=torch.float64, device="cuda")
    weight = s.weight.double() if c.op == "weighted" else None
    for b in range(c.B):
        for h in range(c.Hkv):
            if c.op == "weighted":
                slots, bias = torch.arange(c.L, device="cuda"), None
                if s.sel is not None:
                    ids = s.sel[b, h].tolist()
                    first = [i for i, blk in enumerate(ids) if blk not in ids[:i]]
                    slots = torch.cat([torch.arange(ids[i] * c.bs, min(c.L, (ids[i] + 1) * c.bs), device="cuda")
                                       for i in first])
                    if s.gate is not None:
                        bias = torch.cat([s.gate[b, h, i].double().expand(min(c.bs, c.L - ids[i] * c.bs))
                                          for i in first])
                k, v, n, end = s.k[b, h, slots].double(), s.v[b, h, slots].double(), None, c.L
            else:
                n, end = c.P, int(s.lens[b])
                k = torch.cat([s.pk[h], s.k[b, h, :end]]).double()
                v = torch.cat([s.pv[h], s.v[b, h, :end]]).double()
                slots, bias = torch.arange(-n, end, device="cuda"), None
            for t in range(c.T):
                x = s.q[b, h * grp:(h + 1) * grp, t].double() @ k.t() / math.sqrt(c.D)
                if bias is not None:
                    x = x + bias
                x[:, slots > end - c.T + t] = float("-inf")
                p = torch.softmax(x, -1).nan_to_num(0.0)
                o[b, h * grp:(h + 1) * grp, t] = p @ v
                if weight is not None:
                    weight[b, h, slots] += p.sum(0)
    return {"o": o, "weight": weight} if c.op == "weighted" else {"o": o}


def _exact_evict(s):
    c = s.c
    n = (c.budget + c.bs - 1) // c.bs
    k, v = s.k[:, :, :c.budget].double().cpu(), s.v[:, :, :c.budget].double().cpu()
    weight = torch.zeros(c.B, c.Hkv, c.budget, dtype=torch.float64)
    for b in range(c.B):
        for h in range(c.Hkv):
            w, pos = s.weight[b, h, :c.L].double().cpu().numpy(), s.pos[b, h, :c.L].cpu().numpy()
            safe = (pos < c.sink) | (pos >= s.seen - c.recent)
            best = np.lexsort((np.arange(c.L), -w, ~safe))[:c.budget]
            src, free = np.arange(c.budget), np.setdiff1d(np.arange(c.budget), best)
            src[free] = np.sort(best[best >= c.budget])
            weight[b, h] = torch.from_numpy(w[src])
            src = torch.from_numpy(src).cuda()
            k[b, h], v[b, h] = s.k[b, h, src].double().cpu(), s.v[b, h, src].double().cpu()
    full = torch.zeros(c.B, c.Hkv, n * c.bs, c.D, dtype=torch.float64)
    full[:, :, :c.budget] = k
    full = full.view(c.B, c.Hkv, n, c.bs, c.D)
    return {"k": k, "v": v, "weight": weight, "pos": None, "kmin": full.min(3).values, "kmax": full.max(3).values}
