"""The dense-head operators' C entries refuse bad arguments on the host, before anything is launched (the pointers here
are never followed), and the wrappers refuse CPU tensors."""
from __future__ import annotations

import ctypes

import pytest
import torch

from tests.conftest import load_pkg

pkg = load_pkg()
L = __import__(pkg.__name__ + "._lib", fromlist=["_lib"])
kernels = __import__(pkg.__name__ + ".kernels", fromlist=["kernels"])
INVALID, WORKSPACE = 1001, 1003
P = ctypes.c_void_p(64)
ODD = ctypes.c_void_p(68)


def refused(name, good: dict, changes: list[tuple[dict, int]]):
    f = getattr(L.lib(), name)
    for change, status in changes:
        assert set(change) <= set(good), change
        args = {**good, **change}
        assert f(*args.values()) == status, (name, change)


def test_layer_norm_entries_refuse():
    fwd = dict(dtype=0, x=P, ldx=8, wt=0, w=None, b=None, y=P, ldy=8, mean=None, rstd=None, n=2, d=8, eps=1e-5, st=None)
    refused("kgat_layer_norm_fwd", fwd, [
        ({"dtype": 3}, INVALID), ({"dtype": -1}, INVALID), ({"x": None}, INVALID), ({"y": None}, INVALID),
        ({"n": -1}, INVALID), ({"d": 0}, INVALID), ({"d": (1 << 20) + 1}, INVALID), ({"ldx": -1}, INVALID),
        ({"ldy": 7}, INVALID), ({"eps": -1.0}, INVALID), ({"eps": float("nan")}, INVALID), ({"mean": P}, INVALID),
        ({"rstd": P}, INVALID), ({"wt": 1}, INVALID), ({"wt": 9}, INVALID), ({"n": 0}, 0), ({"n": 0, "dtype": 5}, INVALID)])
    lib = L.lib()
    need = lib.kgat_layer_norm_bwd_workspace(1, 100, 64)
    assert need >= 128
    assert lib.kgat_layer_norm_bwd_workspace(0, -1, 64) == -1 and lib.kgat_layer_norm_bwd_workspace(0, 1, 0) == -1
    assert lib.kgat_layer_norm_bwd_workspace(3, 1, 64) == -1
    bwd = dict(dtype=1, dy=P, lddy=64, x=P, ldx=64, mean=P, rstd=P, wt=0, w=None, dx=P, lddx=64, dw=P, db=P, n=100, d=64,
               ws=P, wsn=need, st=None)
    refused("kgat_layer_norm_bwd", bwd, [
        ({"dtype": 7}, INVALID), ({"dy": None}, INVALID), ({"x": None}, INVALID), ({"mean": None}, INVALID),
        ({"rstd": None}, INVALID), ({"lddx": 63}, INVALID), ({"lddy": -1}, INVALID), ({"ldx": -1}, INVALID),
        ({"n": -1}, INVALID), ({"d": 0}, INVALID), ({"wt": 2}, INVALID), ({"ws": None}, WORKSPACE),
        ({"wsn": need - 1}, WORKSPACE), ({"db": None, "wsn": 0}, WORKSPACE)])


def test_act8_entries_refuse():
    pack = dict(dtype=0, x=P, ldx=8, n=2, d=8, q=P, e=P, st=None)
    refused("kgat_act8_pack", pack, [
        ({"dtype": 4}, INVALID), ({"x": None}, INVALID), ({"q": None}, INVALID), ({"e": None}, INVALID),
        ({"q": ODD}, INVALID), ({"n": -1}, INVALID), ({"d": 0}, INVALID), ({"d": (1 << 20) + 1}, INVALID),
        ({"ldx": -1}, INVALID), ({"n": 1 << 60}, INVALID), ({"n": 0}, 0)])
    unpack = dict(dtype=0, q=P, e=P, n=2, d=8, x=P, ldx=8, st=None)
    refused("kgat_act8_unpack", unpack, [
        ({"dtype": 4}, INVALID), ({"x": None}, INVALID), ({"q": None}, INVALID), ({"e": None}, INVALID),
        ({"q": ODD}, INVALID), ({"n": -1}, INVALID), ({"d": 0}, INVALID), ({"ldx": 7}, INVALID),
        ({"n": 1 << 60}, INVALID), ({"n": 0}, 0)])
    lib = L.lib()
    need = lib.kgat_act8_wgrad_workspace(2, 2, 1000, 64, 96)
    assert need >= 64
    for n, o, d in ((-1, 4, 4), (1, 0, 4), (1, 4, 0), (1, (1 << 20) + 1, 4)):
        assert lib.kgat_act8_wgrad_workspace(0, 0, n, o, d) == -1
    assert lib.kgat_act8_wgrad_workspace(4, 0, 1, 1, 1) == lib.kgat_act8_wgrad_workspace(0, 3, 1, 1, 1) == -1
    grad = dict(dtype=2, dy=P, lddy=64, xt=2, q=P, e=P, n=1000, o=64, d=96, dW=P, db=P, ws=P, wsn=need, st=None)
    refused("kgat_act8_wgrad", grad, [
        ({"dtype": 4}, INVALID), ({"xt": -1}, INVALID), ({"dy": None}, INVALID), ({"q": None}, INVALID), ({"e": None}, INVALID),
        ({"dW": None}, INVALID), ({"q": ODD}, INVALID), ({"lddy": -1}, INVALID), ({"n": -1}, INVALID), ({"o": 0}, INVALID),
        ({"d": 0}, INVALID), ({"ws": None}, WORKSPACE), ({"wsn": need - 1}, WORKSPACE)])


def test_act8_wgrad_of_one_share_needs_no_workspace():
    """One row's tile is written where it belongs, and so are the zeros of no rows; shares are joined."""
    need = L.lib().kgat_act8_wgrad_workspace
    for dtype in range(3):
        assert need(dtype, dtype, 1, 64, 96) == need(dtype, dtype, 0, 64, 96) == 0
        assert need(dtype, dtype, 64, 4096, 4096) == 0
        assert need(dtype, dtype, 100003, 131, 257) >= 2 * 131 * 258


def test_log_prob_entries_refuse():
    lib = L.lib()
    need = lib.kgat_log_prob_workspace(2, 200000, 20)
    assert need > 0 and lib.kgat_log_prob_workspace(5000, 100, 20) == 0
    for r, c, k in ((-1, 4, 0), (1, 0, 0), (1, 4, -1), (1, 400, 129)):
        assert lib.kgat_log_prob_workspace(r, c, k) == -1
    fwd = dict(dtype=0, s=P, ld=200000, rows=2, cols=200000, scale=1.0, items=P, t=3, k=20, logp=P, stats=P, top=P, tl=P,
               ws=P, wsn=need, st=None)
    refused("kgat_log_prob_fwd", fwd, [
        ({"dtype": 3, "ws": P}, INVALID), ({"s": None}, INVALID), ({"ld": -1}, INVALID), ({"rows": -1}, INVALID),
        ({"cols": 0}, INVALID), ({"scale": 0.0}, INVALID), ({"scale": -1.0}, INVALID), ({"scale": float("nan")}, INVALID),
        ({"scale": float("inf")}, INVALID), ({"items": None}, INVALID), ({"t": -1}, INVALID), ({"t": 1025}, INVALID),
        ({"k": -1}, INVALID), ({"k": 129}, INVALID), ({"cols": 10, "k": 11}, INVALID), ({"logp": None}, INVALID),
        ({"stats": None}, INVALID), ({"top": None}, INVALID), ({"tl": None}, INVALID), ({"ws": None}, WORKSPACE),
        ({"wsn": need - 1}, WORKSPACE), ({"ws": ODD}, WORKSPACE), ({"rows": 0, "ws": None, "wsn": 0}, 0)])
    bwd = dict(dtype=0, s=P, ld=50, rows=2, cols=50, scale=1.0, items=P, t=3, stats=P, dl=P, de=None, ds=P, ldds=50, st=None)
    refused("kgat_log_prob_bwd", bwd, [
        ({"dtype": 3}, INVALID), ({"s": None}, INVALID), ({"ld": -1}, INVALID), ({"rows": -1}, INVALID),
        ({"cols": 0}, INVALID), ({"scale": 0.0}, INVALID), ({"items": None}, INVALID), ({"t": 1025}, INVALID),
        ({"stats": None}, INVALID), ({"dl": None}, INVALID), ({"ds": None}, INVALID), ({"ldds": 49}, INVALID),
        ({"rows": 0}, 0)])


def test_wrappers_refuse_cpu_tensors():
    x, items = torch.zeros(3, 8), torch.zeros(3, 1, dtype=torch.int64)
    one = torch.zeros(3)
    for f in (lambda: kernels.layer_norm_fwd(x), lambda: kernels.layer_norm_bwd(x, x, one, one),
              lambda: kernels.act8_pack(x), lambda: kernels.log_prob_fwd(x, items),
              lambda: kernels.log_prob_bwd(x, items, torch.zeros(4, 3), torch.zeros(3, 1)),
              lambda: kernels.act8_unpack(kernels.Act8(torch.zeros(3, 32, dtype=torch.int8),
                                                       torch.zeros(3, 1, dtype=torch.uint8), (3, 8), torch.float32))):
        with pytest.raises(ValueError):
            f()


def test_row_sharded_model_refuses_checkpoint_sides():
    """The flag would have no effect there."""
    sharded = __import__(pkg.__name__ + ".sharded", fromlist=["sharded"])
    m = sharded.RowShardedKGAT.__new__(sharded.RowShardedKGAT)
    torch.nn.Module.__init__(m)
    m.checkpoint_sides = False
    assert m.checkpoint_sides is False
    with pytest.raises(ValueError, match="checkpoint_sides"):
        m.checkpoint_sides = True
