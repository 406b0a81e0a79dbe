"""Calls of the cache operators off the usual path: a first call that is captured, other streams."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_first_call_captured(cuda, monkeypatch):
    """A process whose first call on the device is captured: the status word is no part of the
    graph, so what eager calls report outlives its replays, and is zero before them."""
    import _bsa
    monkeypatch.setattr(_bsa, "_status", {})
    g = torch.Generator().manual_seed(1)
    B, Hq, Hkv, P, S, D = 3, 4, 2, 300, 8, 64
    q, pk, pv, k, v = (torch.randn(*s, generator=g).to(torch.bfloat16).to(cuda) for s in
                       ((B, Hq, 1, D), (Hkv, P, D), (Hkv, P, D), (B, Hkv, S, D), (B, Hkv, S, D)))
    lens = torch.tensor([0, 3, 8], dtype=torch.int32, device=cuda)
    bad = torch.tensor([0, 3, 9], dtype=torch.int32, device=cuda)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = _bsa.decode_prefix(q, pk, pv, k, v, lens)
    _bsa.check_status(cuda)                          # nothing has run yet
    graph.replay()
    assert torch.equal(o, _bsa.decode_prefix(q, pk, pv, k, v, lens))
    _bsa.check_status(cuda)
    _bsa.decode_prefix(q, pk, pv, k, v, bad)
    graph.replay()
    with pytest.raises(_bsa.BsaError) as ei:
        _bsa.check_status(cuda)
    assert ei.value.status == _bsa.ERR_INDEX
    _bsa.check_status(cuda)
    lens.copy_(bad)                                  # and what the graph itself reports
    graph.replay()
    lens.copy_(torch.tensor([1, 2, 3], dtype=torch.int32))
    graph.replay()
    with pytest.raises(_bsa.BsaError):
        _bsa.check_status(cuda)


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_every_instance_of_the_split_kernels(cuda, dtype, D):
    """Row tiles of 8, 16 and 32, in one launch and by splits, all keys and selected ones; the
    last launch also with a second row tile."""
    from test_gpu_cache_ops import _check_weighted, _weighted_case
    for rows, L in ((7, 150), (16, 130), (31, 100), (24, 200), (8, 5000), (15, 4100), (30, 4500), (40, 4001)):
        q, k, v, w, _, _ = _weighted_case(cuda, dtype, D, 1, 2 * rows, 2, L, 1, seed=rows + L)
        _check_weighted(q, k, v, w, None, None, None, L)
        kk = 3 if L < 1000 else 50
        q, k, v, w, sel, gate = _weighted_case(cuda, dtype, D, 1, rows, 1, L, 1, 64, kk, True, seed=L)
        sel[..., 0] = (L - 1) // 64
        _check_weighted(q, k, v, w, sel, gate, 64, L)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_two_streams_at_once(cuda, dtype):
    """The three operators on two streams side by side, each with inputs of its own."""
    import _bsa
    from test_gpu_cache_ops import _prefix_case, _weighted_case
    g = torch.Generator().manual_seed(2)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32

    def inputs(seed):
        ev = [torch.randn(2, 2, 9000, 64, generator=g).to(dt).to(cuda) for _ in range(2)] + \
            [torch.rand(2, 2, 9000, generator=g).to(cuda),
             torch.arange(9000, dtype=torch.int32, device=cuda).repeat(2, 2, 1)]
        return _weighted_case(cuda, dtype, 64, 2, 8, 2, 20000, 2, seed=seed)[:4], ev, \
            _prefix_case(cuda, dtype, 64, 40, 8, 2, 9000, 30, 1, seed=seed)

    def step(w, ev, pf):
        w, ev = [t.clone() for t in w], [t.clone() for t in ev]
        o = _bsa.decode_weighted(*w, L=20000)
        _bsa.evict(*ev, budget=3000, recent=50, sink=2)
        return [o, w[3][:, :, :20000], *ev, _bsa.decode_prefix(*pf)]

    ins = [inputs(s) for s in (1, 2)]
    want = [step(*x) for x in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(step(*ins[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            for x, y in zip(outs, want[i]):
                assert torch.equal(x, y)
