"""Refusals of the row-wise operators (layer_norm, pack_rows_e4m3, unpack_rows_e4m3, embedding) that need no
device: of the Python functions, and of the C entry points, which check before they launch."""
import ctypes as C

import pytest
import torch

import llm720_b200 as lib
from llm720_b200 import _lib

F32, BF16, E4M3 = _lib.DTYPE_F32, _lib.DTYPE_BF16, _lib.DTYPE_E4M3


def test_host_tensors_are_refused():
    x = torch.randn(3, 8)
    for call in (lambda: lib.layer_norm(x), lambda: lib.pack_rows_e4m3(x),
                 lambda: lib.unpack_rows_e4m3(x.to(torch.float8_e4m3fn), torch.ones(3)),
                 lambda: lib.embedding(torch.zeros(2, dtype=torch.int64), x)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(ValueError, match="checkpoint"):
        lib.layer_norm(x, checkpoint="int8")


def _norm(native, **kw):
    a = dict(x=16, xs=8, dt=BF16, w=None, b=None, pdt=F32, eps=1e-5, rows=4, dim=8, y=16, mean=None, rstd=None, payload=None,
             scale=None)
    a.update(kw)
    return native.peer_layer_norm(a["x"], a["xs"], a["dt"], a["w"], a["b"], a["pdt"], a["eps"], a["rows"], a["dim"], a["y"],
                                  a["mean"], a["rstd"], a["payload"], a["scale"], None)


def test_layer_norm_entry_refuses_before_any_launch():
    native = _lib.load()
    bad = [dict(x=None), dict(y=None), dict(rows=-1), dict(dim=0), dict(dim=(1 << 20) + 1), dict(xs=-8), dict(dt=E4M3),
           dict(pdt=_lib.DTYPE_F16), dict(eps=-1.0), dict(eps=float("nan")), dict(payload=16), dict(scale=16),
           dict(x=17), dict(y=17), dict(w=18), dict(mean=18)]
    for kw in bad:
        assert _norm(native, **kw) == _lib.ERR_INVALID_ARG, kw
        assert "peer_layer_norm" in _lib.last_error(None)
    assert _norm(native, rows=0, x=None, y=None) == _lib.OK           # nothing to do, nothing launched


def _norm_grad(native, **kw):
    a = dict(dy=16, dys=8, x=16, xs=8, payload=None, scale=None, mean=16, rstd=16, w=None, dt=BF16, pdt=F32, add=None, rows=4,
             dim=8, dx=16, dw=None, db=None, ws=None, wb=0)
    a.update(kw)
    return native.peer_layer_norm_backward(a["dy"], a["dys"], a["x"], a["xs"], a["payload"], a["scale"], a["mean"], a["rstd"],
                                           a["w"], a["dt"], a["pdt"], a["add"], a["rows"], a["dim"], a["dx"], a["dw"], a["db"],
                                           a["ws"], a["wb"], None)


def test_layer_norm_backward_entry_refuses_before_any_launch():
    native = _lib.load()
    need = native.peer_layer_norm_workspace(4, 8)
    assert need > 0
    bad = [dict(dy=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(rows=-1), dict(dim=0), dict(dt=9), dict(xs=-1),
           dict(dys=-1), dict(payload=16), dict(dw=16), dict(dw=16, ws=16, wb=need - 1), dict(db=16, ws=None, wb=need),
           dict(pdt=_lib.DTYPE_F16), dict(dy=17), dict(dx=17), dict(add=17), dict(dw=16, ws=24, wb=need)]
    for kw in bad:
        assert _norm_grad(native, **kw) == _lib.ERR_INVALID_ARG, kw
        assert "peer_layer_norm_backward" in _lib.last_error(None)
    assert _norm_grad(native, rows=0) == _lib.OK


def test_packing_entries_refuse_before_any_launch():
    native = _lib.load()
    pack = lambda x=16, xs=8, dt=BF16, rows=4, dim=8, p=16, s=16: native.peer_pack_rows(x, xs, dt, rows, dim, p, s, None)
    unpack = lambda p=16, s=16, dt=BF16, rows=4, dim=8, o=16: native.peer_unpack_rows(p, s, dt, rows, dim, o, None)
    for kw in (dict(x=None), dict(p=None), dict(s=None), dict(rows=-1), dict(dim=0), dict(dim=1 << 21), dict(dt=E4M3), dict(xs=-1),
               dict(x=17), dict(s=18)):
        assert pack(**kw) == _lib.ERR_INVALID_ARG, kw
    for kw in (dict(o=None), dict(p=None), dict(s=None), dict(rows=-1), dict(dim=0), dict(dim=1 << 21), dict(dt=E4M3), dict(o=17)):
        assert unpack(**kw) == _lib.ERR_INVALID_ARG, kw
    assert pack(rows=0) == _lib.OK and unpack(rows=0) == _lib.OK


def test_embedding_entries_refuse_before_any_launch():
    native = _lib.load()

    def fwd(ids=16, ib=8, n=4, w=16, dt=BF16, V=10, D=8, out=16):
        return native.peer_embedding(ids, ib, n, w, dt, V, D, 1.0, out, None, None)

    for kw in (dict(ids=None), dict(w=None), dict(out=None), dict(ib=2), dict(n=-1), dict(V=0), dict(V=1 << 31), dict(D=0),
               dict(D=1 << 21), dict(dt=E4M3), dict(ids=20), dict(w=17)):
        assert fwd(**kw) == _lib.ERR_INVALID_ARG, kw
        assert "peer_embedding" in _lib.last_error(None)
    assert fwd(n=0) == _lib.OK
    need = native.peer_embedding_workspace(4, 8)
    assert need > 0 and native.peer_embedding_workspace(0, 8) == 0

    def bwd(ids=16, ib=8, n=4, g=16, gs=8, dt=BF16, V=10, D=8, gw=16, ws=16, wb=need):
        return native.peer_embedding_backward(ids, ib, n, g, gs, dt, V, D, 1.0, -1, gw, ws, wb, None)

    for kw in (dict(ids=None), dict(g=None), dict(gw=None), dict(ws=None), dict(wb=need - 1), dict(ib=1), dict(n=-1), dict(V=0),
               dict(D=0), dict(gs=-1), dict(dt=E4M3), dict(n=1 << 31), dict(gw=17), dict(ws=24)):
        assert bwd(**kw) == _lib.ERR_INVALID_ARG, kw
        assert "peer_embedding_backward" in _lib.last_error(None)


def test_workspaces_grow_with_the_sizes():
    native = _lib.load()
    assert native.peer_layer_norm_workspace(16384, 2048) < 64 << 20
    assert native.peer_embedding_workspace(131072, 2048) < 256 << 20
    assert native.peer_layer_norm_workspace(-1, 8) == 0
