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
