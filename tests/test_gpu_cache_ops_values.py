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
