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
