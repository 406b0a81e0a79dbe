"""Calls of the decode caches that must be refused, or be harmless, before anything is launched."""
import pytest
import torch


def _t(*shape, dt=torch.bfloat16):
    return torch.zeros(*shape, dtype=dt)


def _prefix_cache(B=3, Hkv=2, room=6, D=64):
    import decode
    return decode.PrefixCache(_t(Hkv, 9, D), _t(Hkv, 9, D), B, room)


@pytest.mark.parametrize("k,v,active", [
    ((2, 2, 1, 64), (2, 2, 1, 64), None),                # fewer sequences: their rows would lie past the end
    ((1, 2, 1, 64), (1, 2, 1, 64), [True, False, True]),
    ((4, 2, 1, 64), (4, 2, 1, 64), None), ((3, 1, 1, 64), (3, 1, 1, 64), None), ((3, 2, 2, 64), (3, 2, 1, 64), None),
    ((3, 2, 1, 1), (3, 2, 1, 1), None), ((2, 1, 64), (2, 1, 64), None), ((3, 2, 1, 64), (3, 2, 1, 64), [True, True]),
    ((3, 2, 1, 64), (3, 2, 1, 64), [True, False, True, True]),
])
def test_append_of_another_shape_is_refused(k, v, active):
    c = _prefix_cache()
    with pytest.raises(ValueError):
        c.append(torch.ones(k), torch.ones(v), active)
    assert c.used == [0, 0, 0] and c.lens.tolist() == [0, 0, 0] and not c.k.any() and not c.v.any()


@pytest.mark.parametrize("T,active", [(1, [False] * 3), (2, [0, 0, 0]), (0, None)])
def test_append_of_nothing(T, active):
    """No sequence takes part, or no token is new: the cache stays as it is."""
    c = _prefix_cache()
    c.append(torch.ones(3, 2, 2, 64), torch.ones(3, 2, 2, 64), [True, False, True])
    k = c.k.clone()
    c.append(torch.ones(3, 2, T, 64), torch.ones(3, 2, T, 64), active)
    assert c.used == c.lens.tolist() == [2, 0, 2] and torch.equal(c.k, k)


@pytest.fixture
def decode_calls(monkeypatch):
    """decode.py with CPU tensors, its launches recorded."""
    import _bsa
    import decode
    calls = []
    monkeypatch.setattr(_bsa, "pool", lambda x, bs, **kw: [torch.zeros(x.shape[0], x.shape[1], -(-x.shape[2] // bs), x.shape[3])] * 2)
    for name in ("decode_weighted", "decode", "evict"):
        monkeypatch.setattr(_bsa, name, lambda *a, _n=name, **kw: calls.append(_n))
    return decode, calls


def test_rows_of_moved_tokens_are_refused(decode_calls):
    """A row's mask goes by slot.  An eviction may move the newest tokens to freed slots, where
    the rows before them would see them; one row sees every slot and needs no order."""
    decode, calls = decode_calls
    c = decode.DecodeCache(1, 2, 40, 64, bs=8, device="cpu", track=True)
    q = lambda T: _t(1, 4, T, 64)  # noqa: E731
    sel = _t(1, 2, 2, dt=torch.int32)
    c.append(_t(1, 2, 20, 64), _t(1, 2, 20, 64))
    decode.decode_attention_weighted(q(20), c)
    decode.decode_attention(q(3), c, sel)
    assert c.evict(20) == 0                       # nothing went, nothing moved
    decode.decode_attention_weighted(q(3), c)
    assert c.evict(16) == 4
    n = len(calls)
    for s in (None, sel):
        with pytest.raises(ValueError):
            decode.decode_attention_weighted(q(2), c, s)
    assert len(calls) == n
    decode.decode_attention_weighted(q(1), c)
    decode.decode_attention(q(1), c, sel)
    c.append(_t(1, 2, 1, 64), _t(1, 2, 1, 64))
    with pytest.raises(ValueError):
        decode.decode_attention_weighted(q(2), c)
    c.append(_t(1, 2, 2, 64), _t(1, 2, 2, 64))
    decode.decode_attention_weighted(q(3), c)     # appended since: in order again
    with pytest.raises(ValueError):
        decode.decode_attention_weighted(q(4), c)


@pytest.fixture
def ids_of(monkeypatch):
    """_bsa with CPU tensors let through; what the launches would read as ids or lengths."""
    import ctypes

    import _bsa
    got = []
    structs = {"bsa_decode_weighted": (_bsa.DecodeWeightedArgs, "sel", 3), "bsa_decode_prefix": (_bsa.DecodePrefixArgs, "lens", 3)}

    def launch(name, a, like):
        cls, field, n = structs[name]
        at = getattr(cls.from_buffer_copy(a), field)
        got.append(list((ctypes.c_int32 * n).from_address(at)))
    monkeypatch.setattr(_bsa, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(_bsa, "status_tensor", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(_bsa, "_launch", launch)
    return _bsa, got


def test_wide_ids_and_lengths_stay_outside(ids_of):
    """64-bit ids and lengths past 32 bits are outside the cache, not other ids and lengths."""
    bsa, got = ids_of
    for dt, x in ((torch.int64, [2 ** 32 + 1, -2 ** 33, 2]), (torch.int64, [2 ** 31, -2 ** 32 + 1, 0]),
                  (torch.int32, [2 ** 31 - 1, -5, 1]), (torch.int16, [-1, 7, 3])):
        bsa.decode_weighted(_t(1, 2, 1, 64), _t(1, 2, 256, 64), _t(1, 2, 256, 64), _t(1, 2, 256, dt=torch.float32),
                            torch.tensor(x, dtype=dt).view(1, 3), bs=32)
        bsa.decode_prefix(_t(3, 2, 1, 64), _t(2, 8, 64), _t(2, 8, 64), _t(3, 2, 9, 64), _t(3, 2, 9, 64),
                          torch.tensor(x, dtype=dt))
        for ids, end in zip(got[-2:], (8, 9)):
            for a, b in zip(x, ids):
                assert a == b if 0 <= a <= end else not 0 <= b <= end, (a, b)
