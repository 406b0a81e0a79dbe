"""Refusals of the weighted decode, the eviction and the shared-prefix decode, and the
layout of their argument structs: everything that is decided before a launch."""
import ctypes
import os
import subprocess

import pytest
import torch

from conftest import ROOT


def test_struct_layouts(tmp_path):
    import _bsa
    structs = {"bsa_decode_weighted_args": _bsa.DecodeWeightedArgs, "bsa_evict_args": _bsa.EvictArgs,
               "bsa_decode_prefix_args": _bsa.DecodePrefixArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "bsa.h"', "int main(void) {"]
    for cname, cls in structs.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (cname, cname))
        for f, _ in cls._fields_:
            lines.append('printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (cname, f, cname, f))
    lines.append("return 0; }")
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                                  check=True).stdout.splitlines())
    for cname, cls in structs.items():
        assert int(got[cname]) == ctypes.sizeof(cls) == _bsa._PACK[cname[:-5]].size, cname
        for f, _ in cls._fields_:
            assert int(got[cname + "." + f]) == getattr(cls, f).offset, (cname, f)


# Addresses that are never read: every case below is refused before a launch.
P = 4096


def _view(D=64):
    import _bsa
    return _bsa.View(P, 4 * 64 * D, 64 * D, D)


def _weighted():
    import _bsa
    a = _bsa.DecodeWeightedArgs(_bsa.BF16, 1, 4, 2, 60, 64, 32, 1, 3, 0.125)
    a.q = a.k = a.v = a.o = _view()
    a.weight = a.sel = P
    a.weight_sb, a.weight_sh = 2 * 64, 64
    return a


def _evict():
    import _bsa
    a = _bsa.EvictArgs(_bsa.BF16, 1, 2, 60, 64, 32, 30, 5, 1, 60)
    a.k = a.v = _view()
    a.weight = a.pos = a.weight_out = a.pos_out = P
    a.w_sb = a.p_sb = a.wo_sb = a.po_sb = 2 * 64
    a.w_sh = a.p_sh = a.wo_sh = a.po_sh = 64
    return a


def _prefix():
    import _bsa
    a = _bsa.DecodePrefixArgs(_bsa.BF16, 2, 4, 2, 64, 100, 10, 1, 0.125)
    a.q = a.pk = a.pv = a.k = a.v = a.o = _view()
    a.lens = P
    return a


BAD = [
    ("weighted", dict(dtype=3), "DTYPE"), ("weighted", dict(Hq=5), "SHAPE"), ("weighted", dict(T=61), "SHAPE"),
    ("weighted", dict(L=0), "SHAPE"), ("weighted", dict(D=96), "UNSUPPORTED"), ("weighted", dict(D=512), "UNSUPPORTED"),
    ("weighted", dict(bs=48), "UNSUPPORTED"), ("weighted", dict(bs=0), "UNSUPPORTED"), ("weighted", dict(kk=513), "UNSUPPORTED"),
    ("weighted", dict(kk=0), "SHAPE"), ("weighted", dict(scale=0.0), "ARG"), ("weighted", dict(scale=float("nan")), "ARG"),
    ("weighted", dict(scale=float("inf")), "ARG"), ("weighted", dict(weight=None), "ARG"), ("weighted", dict(sel=None, gate=P), "ARG"),
    ("weighted", dict(Hq=2 * 5000), "UNSUPPORTED"), ("weighted", dict(B=0), "SHAPE"), ("weighted", dict(L=1 << 30), "SHAPE"),
    ("evict", dict(dtype=9), "DTYPE"), ("evict", dict(budget=61), "SHAPE"), ("evict", dict(budget=0), "SHAPE"),
    ("evict", dict(recent=30), "SHAPE"), ("evict", dict(recent=-1), "SHAPE"), ("evict", dict(sink=-1), "SHAPE"),
    ("evict", dict(seen=59), "SHAPE"), ("evict", dict(bs=0), "SHAPE"), ("evict", dict(bs=1025), "UNSUPPORTED"),
    ("evict", dict(D=48), "UNSUPPORTED"), ("evict", dict(pos=None), "ARG"), ("evict", dict(weight_out=None), "ARG"),
    ("evict", dict(kmin=P), "ARG"), ("evict", dict(Hkv=0), "SHAPE"),
    ("prefix", dict(dtype=-1), "DTYPE"), ("prefix", dict(Hq=3), "SHAPE"), ("prefix", dict(S=0), "SHAPE"),
    ("prefix", dict(P=-1), "SHAPE"), ("prefix", dict(T=0), "SHAPE"), ("prefix", dict(D=80), "UNSUPPORTED"),
    ("prefix", dict(lens=None), "ARG"), ("prefix", dict(scale=-1.0), "ARG"), ("prefix", dict(P=1 << 30), "SHAPE"),
]


@pytest.mark.parametrize("op,change,code", BAD, ids=lambda x: str(x)[:40])
def test_refused_before_a_launch(op, change, code):
    import _bsa
    L = _bsa.lib()
    name = {"weighted": "bsa_decode_weighted", "evict": "bsa_evict", "prefix": "bsa_decode_prefix"}[op]
    a = {"weighted": _weighted, "evict": _evict, "prefix": _prefix}[op]()
    ws = getattr(L, name + "_workspace")
    assert ws(ctypes.byref(a)) > 0
    assert getattr(L, name)(ctypes.byref(a), None, 0, None) == _bsa.ERR_WORKSPACE
    assert getattr(L, name)(ctypes.byref(a), P, ws(ctypes.byref(a)) - 1, None) == _bsa.ERR_WORKSPACE
    for k, v in change.items():
        setattr(a, k, v)
    assert ws(ctypes.byref(a)) == 0
    assert getattr(L, name)(ctypes.byref(a), P, 1 << 40, None) == getattr(_bsa, "ERR_" + code)
    assert L.bsa_last_error()


@pytest.mark.parametrize("op,view", [("weighted", "k"), ("weighted", "v"), ("evict", "k"), ("evict", "v"),
                                     ("prefix", "k"), ("prefix", "pk"), ("prefix", "pv")])
@pytest.mark.parametrize("field,value,code", [("ptr", None, "ARG"), ("ptr", P + 8, "STRIDE"), ("sl", 68, "STRIDE"),
                                              ("sh", 4097, "STRIDE")])
def test_unaligned_cache_is_refused(op, view, field, value, code):
    import _bsa
    name = {"weighted": "bsa_decode_weighted", "evict": "bsa_evict", "prefix": "bsa_decode_prefix"}[op]
    a = {"weighted": _weighted, "evict": _evict, "prefix": _prefix}[op]()
    setattr(getattr(a, view), field, value)
    assert getattr(_bsa.lib(), name)(ctypes.byref(a), P, 1 << 40, None) == getattr(_bsa, "ERR_" + code)


# Written operands whose rows share memory: two CTAs would write one place.
SHARED = [
    ("weighted", dict(weight_sh=0)), ("weighted", dict(weight_sh=59)), ("weighted", dict(B=2, weight_sb=64)),
    ("weighted", {"o.sh": 0}), ("weighted", {"o.sh": 63}), ("weighted", dict(T=2) | {"o.sl": 0}),
    ("prefix", {"o.sb": 0}), ("prefix", {"o.sh": 32}),
    ("evict", {"k.sl": 0}), ("evict", {"v.sh": 0}), ("evict", {"k.sh": 59 * 64}), ("evict", {"v.sl": 32}),
    ("evict", dict(wo_sh=29, weight_out=P + 65536)), ("evict", dict(po_sh=0, pos_out=P + 65536)),
    ("evict", dict(kmin=P, kmax=P, km_sh=0, km_sn=64)), ("evict", dict(kmin=P, kmax=P, km_sh=64, km_sn=0, budget=60)),
    # an output that meets its source without being it
    ("evict", dict(weight_out=P + 4)), ("evict", dict(weight_out=P - 4)), ("evict", dict(pos_out=P + 59 * 4)),
    ("evict", dict(pos_out=P + 64 * 4)), ("evict", dict(weight_out=P - 29 * 4)), ("evict", dict(wo_sh=128)),
    ("evict", dict(weight_out=P + 63 * 4)),
]
APART = [
    ("weighted", dict(weight_sh=60)), ("weighted", dict(B=2, weight_sb=60, weight_sh=120)), ("weighted", {"o.sh": 64}),
    ("weighted", dict(Hq=2, Hkv=1, weight_sh=0)), ("evict", {"k.sl": 128, "k.sh": 64}),
    ("evict", dict(weight_out=P + 128 * 4)), ("evict", dict(weight_out=P - 30 * 4, w_sh=90, wo_sh=90)),
    ("evict", dict(pos_out=P + 60 * 4, p_sh=90, po_sh=90)), ("evict", dict(Hkv=1, weight_out=P + 60 * 4, wo_sh=0)),
]


def _set(a, change):
    for k, v in change.items():
        view, _, field = k.partition(".")
        setattr(getattr(a, view), field, v) if field else setattr(a, k, v)


@pytest.mark.parametrize("op,change", SHARED, ids=lambda x: str(x)[:40])
def test_shared_rows_are_refused(op, change):
    import _bsa
    a = {"weighted": _weighted, "evict": _evict, "prefix": _prefix}[op]()
    name = {"weighted": "bsa_decode_weighted", "evict": "bsa_evict", "prefix": "bsa_decode_prefix"}[op]
    _set(a, change)
    assert getattr(_bsa.lib(), name)(ctypes.byref(a), P, 1 << 40, None) == _bsa.ERR_STRIDE
    assert b"memory" in _bsa.lib().bsa_last_error() or b"apart" in _bsa.lib().bsa_last_error()


@pytest.mark.parametrize("op,change", APART, ids=lambda x: str(x)[:40])
def test_interleaved_rows_are_accepted(op, change):
    import _bsa
    a = {"weighted": _weighted, "evict": _evict, "prefix": _prefix}[op]()
    name = {"weighted": "bsa_decode_weighted", "evict": "bsa_evict", "prefix": "bsa_decode_prefix"}[op]
    _set(a, change)
    assert getattr(_bsa.lib(), name + "_workspace")(ctypes.byref(a)) > 0


def test_null_args():
    import _bsa
    for name in ("bsa_decode_weighted", "bsa_evict", "bsa_decode_prefix"):
        assert getattr(_bsa.lib(), name)(None, None, 0, None) == _bsa.ERR_ARG
        assert getattr(_bsa.lib(), name + "_workspace")(None) == 0


# ------------------------------------------------------------------ the Python layer
@pytest.fixture
def bsa(monkeypatch):
    """_bsa with CPU tensors let through and the launch recorded instead of made."""
    import _bsa
    calls = []
    monkeypatch.setattr(_bsa, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(_bsa, "status_tensor", lambda device: torch.zeros(1, dtype=torch.int32))
    structs = {"bsa_decode_weighted": _bsa.DecodeWeightedArgs, "bsa_evict": _bsa.EvictArgs,
               "bsa_decode_prefix": _bsa.DecodePrefixArgs}
    monkeypatch.setattr(_bsa, "_launch",
                        lambda name, a, like: calls.append((name, structs[name].from_buffer_copy(a))))
    _bsa.test_calls = calls
    return _bsa


def _t(*shape, dt=torch.bfloat16):
    return torch.zeros(*shape, dtype=dt)


def test_cpu_tensors_are_refused():
    import _bsa
    with pytest.raises(RuntimeError, match="CUDA"):
        _bsa.decode_weighted(_t(1, 2, 1, 64), _t(1, 2, 8, 64), _t(1, 2, 8, 64), _t(1, 2, 8, dt=torch.float32))
    with pytest.raises(RuntimeError, match="CUDA"):
        _bsa.evict(_t(1, 2, 8, 64), _t(1, 2, 8, 64), _t(1, 2, 8, dt=torch.float32), _t(1, 2, 8, dt=torch.int32), budget=4)
    with pytest.raises(RuntimeError, match="CUDA"):
        _bsa.decode_prefix(_t(1, 2, 1, 64), _t(2, 8, 64), _t(2, 8, 64), _t(1, 2, 8, 64), _t(1, 2, 8, 64),
                           _t(1, dt=torch.int32))


def test_weighted_arguments(bsa):
    def call(q=(1, 4, 1, 64), k=(1, 2, 8, 64), v=(1, 2, 8, 64), w=(1, 2, 8), wdt=torch.float32, kdt=torch.bfloat16, **kw):
        return bsa.decode_weighted(_t(*q), _t(*k, dt=kdt), _t(*v), _t(*w, dt=wdt), **kw)
    assert call().shape == (1, 4, 1, 64)
    name, a = bsa.test_calls[-1]
    assert name == "bsa_decode_weighted" and (a.B, a.Hq, a.Hkv, a.L, a.D, a.T, a.kk, a.sel) == (1, 4, 2, 8, 64, 1, 0, None)
    assert abs(a.scale - 0.125) < 1e-7
    sel = _t(1, 2, 3, dt=torch.int32)
    call(sel=sel, gate=_t(1, 2, 3, dt=torch.float64), bs=32, L=5)
    a = bsa.test_calls[-1][1]
    assert (a.L, a.kk, a.bs, a.sel_sb, a.sel_sh, a.gate_sb, a.gate_sh) == (5, 3, 32, 6, 3, 6, 3)
    call(sel=_t(1, 3, dt=torch.int64), bs=32)
    assert bsa.test_calls[-1][1].sel_sh == 0
    n = len(bsa.test_calls)
    for kw in (dict(L=9), dict(k=(1, 2, 8, 32)), dict(v=(2, 2, 8, 64)), dict(w=(1, 2, 7)), dict(w=(1, 1, 8)),
               dict(sel=sel), dict(sel=sel, bs=0), dict(sel=_t(1, 3, 3, dt=torch.int32), bs=32), dict(q=(4, 1, 64)),
               dict(sel=_t(2, 2, 3, dt=torch.int32), bs=32), dict(gate=_t(1, 2, 3)), dict(k=(2, 8, 64)),
               dict(sel=sel, bs=32, gate=_t(1, 2, 4)), dict(wdt=torch.float64), dict(kdt=torch.float16),
               dict(out=_t(1, 4, 2, 64)), dict(out=_t(1, 4, 1, 64, dt=torch.float32))):
        with pytest.raises(bsa.BsaError):
            call(**kw)
    with pytest.raises(bsa.BsaError):   # a cache that would have to be copied
        bsa.decode_weighted(_t(1, 4, 1, 64), _t(1, 2, 64, 8).transpose(2, 3), _t(1, 2, 8, 64), _t(1, 2, 8, dt=torch.float32))
    with pytest.raises(bsa.BsaError):   # the sums are changed in place
        bsa.decode_weighted(_t(1, 4, 1, 64), _t(1, 2, 8, 64), _t(1, 2, 8, 64), _t(1, 2, 16, dt=torch.float32)[..., ::2])
    assert len(bsa.test_calls) == n


def test_evict_arguments(bsa):
    def call(**kw):
        d = dict(k=_t(1, 2, 8, 64), v=_t(1, 2, 8, 64), weight=_t(1, 2, 8, dt=torch.float32), pos=_t(1, 2, 8, dt=torch.int32),
                 budget=4)
        d.update(kw)
        bsa.evict(d.pop("k"), d.pop("v"), d.pop("weight"), d.pop("pos"), **d)
    call()
    a = bsa.test_calls[-1][1]
    assert (a.L, a.budget, a.seen, a.bs, a.kmin) == (8, 4, 8, 64, None) and a.weight_out == a.weight and a.pos_out == a.pos
    km = _t(1, 2, 3, 64, dt=torch.float32)
    call(kmin=km, kmax=km.clone(), bs=2, L=7, seen=100, recent=2, sink=2)
    a = bsa.test_calls[-1][1]
    assert (a.L, a.seen, a.recent, a.sink, a.bs, a.km_sb, a.km_sh, a.km_sn) == (7, 100, 2, 2, 2, 384, 192, 64)
    n = len(bsa.test_calls)
    for kw in (dict(budget=9), dict(budget=0), dict(L=9), dict(recent=5), dict(recent=-1), dict(sink=2 ** 32),
               dict(seen=7), dict(seen=2 ** 31), dict(kmin=km), dict(kmin=km, kmax=km), dict(kmin=km, kmax=km, bs=1),
               dict(kmin=km, kmax=km.to(torch.float16), bs=2), dict(bs=0), dict(bs=2048), dict(v=_t(1, 2, 8, 32)),
               dict(weight=_t(1, 2, 8)), dict(pos=_t(1, 2, 8, dt=torch.int64)), dict(pos=_t(1, 2, 7, dt=torch.int32)),
               dict(weight_out=_t(1, 2, 3, dt=torch.float32)), dict(pos_out=_t(1, 2, 4, dt=torch.int64)),
               dict(k=_t(1, 2, 64, 8).transpose(2, 3)), dict(k=_t(2, 8, 64))):
        with pytest.raises(bsa.BsaError):
            call(**kw)
    assert len(bsa.test_calls) == n


def test_prefix_arguments(bsa):
    def call(q=(2, 4, 1, 64), p=(2, 9, 64), p2=None, k=(2, 2, 5, 64), v=(2, 2, 5, 64), lens=None, pdt=torch.bfloat16, **kw):
        lens = _t(2, dt=torch.int32) if lens is None else lens
        return bsa.decode_prefix(_t(*q), _t(*p, dt=pdt), _t(*(p2 or p), dt=pdt), _t(*k), _t(*v), lens, **kw)
    assert call().shape == (2, 4, 1, 64)
    a = bsa.test_calls[-1][1]
    assert (a.B, a.Hq, a.Hkv, a.D, a.P, a.S, a.T) == (2, 4, 2, 64, 9, 5, 1)
    call(p=(2, 0, 64), lens=_t(2, dt=torch.int64))
    assert bsa.test_calls[-1][1].P == 0
    n = len(bsa.test_calls)
    for kw in (dict(p=(1, 9, 64)), dict(p=(2, 9, 32)), dict(p2=(2, 8, 64)), dict(v=(2, 2, 6, 64)), dict(k=(1, 2, 5, 64)),
               dict(lens=_t(3, dt=torch.int32)), dict(lens=_t(2)), dict(pdt=torch.float16), dict(q=(4, 1, 64)),
               dict(p=(1, 2, 9, 64)), dict(lens=_t(1, 2, dt=torch.int32))):
        with pytest.raises(bsa.BsaError):
            call(**kw)
    assert len(bsa.test_calls) == n


def test_caches_on_the_host(bsa, monkeypatch):
    """The host side of the caches: lengths, capacities, positions."""
    import decode
    monkeypatch.setattr(bsa, "pool", lambda x, bs, **kw: [torch.zeros(x.shape[0], x.shape[1], -(-x.shape[2] // bs), x.shape[3])] * 2)
    c = decode.DecodeCache(1, 2, 10, 64, bs=4, device="cpu", track=True)
    c.append(_t(1, 2, 7, 64), _t(1, 2, 7, 64))
    c.weight[:] = 1
    assert c.evict(7) == 0 and not bsa.test_calls
    assert c.evict(5, recent=2, sink=1) == 2 and (c.L, c.seen) == (5, 7)
    a = bsa.test_calls[-1][1]
    assert (a.L, a.budget, a.seen, a.recent, a.sink, a.bs) == (7, 5, 7, 2, 1, 4)
    c.append(_t(1, 2, 3, 64), _t(1, 2, 3, 64))
    assert c.pos[0, 0, 5:8].tolist() == [7, 8, 9] and c.weight[0, 1, 5:8].tolist() == [0, 0, 0] and c.seen == 10
    with pytest.raises(ValueError):
        c.append(_t(1, 2, 3, 64), _t(1, 2, 3, 64))
    p = decode.PrefixCache(_t(2, 9, 64), _t(2, 9, 64), 2, 3)
    p.append(torch.ones(2, 2, 2, 64), torch.ones(2, 2, 2, 64), [False, True])
    assert p.used == [0, 2] and p.lens.tolist() == [0, 2] and p.k[1, :, :2].eq(1).all() and p.k[0].eq(0).all()
    with pytest.raises(ValueError):
        p.append(_t(2, 2, 2, 64), _t(2, 2, 2, 64))
    assert p.used == [0, 2]
    with pytest.raises(ValueError):
        decode.PrefixCache(_t(2, 9, 64), _t(2, 8, 64), 2, 3)
