"""Refusals and workspace sizes of the training entry points: decided on the
host before any HIP call, so these need no GPU.  A pointer that is never
followed stands for each buffer."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(64)
F = ctypes.c_float


@pytest.fixture(scope="module")
def L():
    from q36_amd import moe
    return moe.lib()


def _call(fn, args, **change):
    a = dict(args, **change)
    return fn(*a.values())


LN = dict(x=P, ld_x=64, a=None, ld_a=0, x_fmt=0, w=None, b=None, T=4, d=64, eps=F(1e-6), kind=0, h=None, ld_h=0, y=P,
          ld_y=64, y_fmt=0, stream=None)


@pytest.mark.parametrize("change", [
    {"T": -1}, {"d": 0}, {"d": -5}, {"d": 16385, "ld_x": 20000, "ld_y": 20000}, {"eps": F(-1e-9)}, {"eps": F(float("nan"))},
    {"eps": F(float("inf"))}, {"kind": 2}, {"kind": -1}, {"x_fmt": 2}, {"y_fmt": -1}, {"ld_x": 63}, {"ld_y": 63},
    {"a": P}, {"h": P}, {"a": P, "h": P, "ld_a": 64, "ld_h": 63}, {"a": P, "h": P, "ld_a": 63, "ld_h": 64}, {"x": None},
    {"y": None}, {"ld_x": -64}])
def test_layernorm_refuses(L, change):
    assert _call(L.q36moe_layernorm, LN, **change) == -22


LNB = dict(dy=P, ld_dy=64, y_fmt=0, h=P, ld_h=64, dres=None, ld_dres=0, x_fmt=0, w=None, T=4, d=64, eps=F(1e-6), kind=1,
           dx=P, ld_dx=64, dw=P, db=P, ws=P, ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("change", [
    {"T": -1}, {"d": 0}, {"d": 16385, "ld_dy": 20000, "ld_h": 20000, "ld_dx": 20000}, {"eps": F(float("nan"))}, {"kind": 7},
    {"x_fmt": 3}, {"y_fmt": 2}, {"ld_dy": 63}, {"ld_h": 63}, {"ld_dx": 63}, {"dres": P, "ld_dres": 63},
    {"dres": P, "ld_dres": 64, "dx": None}, {"dx": None, "dw": None, "db": None}, {"dy": None}, {"h": None}, {"ws": None},
    {"ws_bytes": 4 * 2 * 64 * 4 - 1}, {"ws": ctypes.c_void_p(72)}])
def test_layernorm_backward_refuses(L, change):
    assert _call(L.q36moe_layernorm_backward, LNB, **change) == -22


BAL = dict(logits=P, ld=256, idx=P, mask=None, T=4, E=256, k=8, coef=F(1.0), counts=P, psum=P, loss=P, ws=None, n=0,
           stream=None)


@pytest.mark.parametrize("change", [
    {"T": -1}, {"E": 0}, {"E": 257, "ld": 257}, {"ld": 255}, {"k": 0}, {"k": 9}, {"E": 4, "k": 5}, {"logits": None},
    {"idx": None}, {"counts": None}, {"psum": None}, {"loss": None}, {"T": 100000}, {"T": 100000, "ws": P, "n": 64},
    {"T": 100000, "ws": ctypes.c_void_p(72), "n": 1 << 30}, {"T": 1 << 28, "ws": P, "n": 1 << 30}])
def test_balance_loss_refuses(L, change):
    assert _call(L.q36moe_balance_loss, BAL, **change) == -22


TKB = dict(logits=P, ld=256, idx=P, dwt=P, counts=P, mask=None, dloss=None, T=4, E=256, k=8, scale=F(1.0), renorm=1,
           coef=F(1.0), out=P, ld_d=256, stream=None)


@pytest.mark.parametrize("change", [
    {"T": -1}, {"E": 0}, {"E": 257, "ld": 300, "ld_d": 300}, {"ld": 255}, {"ld_d": 255}, {"k": 0}, {"k": 9},
    {"E": 4, "k": 5}, {"dwt": None, "counts": None}, {"logits": None}, {"idx": None}, {"out": None}])
def test_router_topk_backward_refuses(L, change):
    assert _call(L.q36moe_router_topk_backward, TKB, **change) == -22


RLB = dict(w=P, n_rows=257, E=256, x=P, x_fmt=0, T=4, d=2048, dlogits=P, ld=256, dshg=P, ld_shg=1, dw=P, dx=P, ws=P,
           n=1 << 40, stream=None)


@pytest.mark.parametrize("change", [
    {"T": -1}, {"T": (1 << 23) + 1}, {"d": 2000}, {"E": 0}, {"n_rows": 255}, {"n_rows": 258}, {"ld": 255}, {"x_fmt": 2},
    {"dw": None, "dx": None}, {"dlogits": None}, {"x": None}, {"w": None}, {"dshg": None}, {"ld_shg": -1},
    {"T": 100000, "ws": None}, {"T": 100000, "n": 1024},
    {"T": 100000, "ws": ctypes.c_void_p(72)}, {"ld": (1 << 22) + 1}, {"x": ctypes.c_void_p(66), "x_fmt": 1},
    {"dx": ctypes.c_void_p(66), "x_fmt": 1}, {"n_rows": (1 << 20) + 1, "E": 1 << 20, "ld": 1 << 20}])
def test_router_logits_backward_refuses(L, change):
    assert _call(L.q36moe_router_logits_backward, RLB, **change) == -22


def test_no_tokens_is_no_work_where_nothing_is_summed(L):
    assert _call(L.q36moe_layernorm, LN, T=0, x=None, y=None) == 0
    assert _call(L.q36moe_layernorm_backward, LNB, T=0, dy=None, h=None, dw=None, db=None, ws=None) == 0
    assert _call(L.q36moe_router_topk_backward, TKB, T=0, logits=None, out=None) == 0
    assert _call(L.q36moe_router_logits_backward, RLB, T=0, x=None, dw=None) == 0


def test_workspaces_grow_no_further_than_the_chip(L):
    """Partial sums: bounded by the number of workgroups, not by the tokens;
    nothing for a single token."""
    n = L.q36moe_layernorm_backward_workspace
    assert n(1, 2048) == 0 and n(0, 2048) == 0 and n(5, 0) == 0 and n(5, 20000) == 0
    assert 0 < n(2, 7) <= n(100, 7) <= n(1 << 30, 7) == n((1 << 31) - 1, 7) < 1 << 20
    b = L.q36moe_balance_loss_workspace
    assert b(1, 256) == 0 and b(0, 256) == 0 and b(1000, 257) == 0
    assert 0 < b(1 << 15, 256) <= b((1 << 31) - 1, 256) < 1 << 22
    r = L.q36moe_router_logits_backward_workspace
    assert r(0, 257) == 0 and r((1 << 23) + 1, 257) == 0 and r(4, 0) == 0
    assert r(1 << 23, 257) < 1 << 28


def test_python_refuses_host_tensors():
    from q36_amd import moe
    x = torch.zeros(3, 2048)
    idx = torch.zeros(3, 8, dtype=torch.int32)
    for call in (lambda: moe.layernorm(x), lambda: moe.layernorm_backward(x, x), lambda: moe.balance_loss(x, idx),
                 lambda: moe.router_topk_backward(x, idx, x[:, :8]), lambda: moe.router_logits_backward(x, x, 3, x)):
        with pytest.raises(moe.Q36MoEError):
            call()
