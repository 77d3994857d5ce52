"""Refusals of the mixture-of-experts operators (no GPU): every bad argument
is an error before anything touches a device."""
import ctypes

import pytest

import bonsai_b1
from bonsai_b1 import capi

P = 0x10000  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    return bonsai_b1.load()


def routes(**change):
    a = dict(tokens=3, experts=8, top_k=2, expert=P, weight=P, start=P, order=P, place=P)
    a.update(change)
    return capi.RoutesC(*a.values())


BAD_COUNTS = [dict(tokens=-1), dict(experts=0), dict(experts=-8), dict(experts=1025), dict(top_k=0), dict(top_k=-1),
              dict(top_k=9), dict(experts=128, top_k=65), dict(tokens=1 << 23), dict(tokens=1 << 30),
              dict(tokens=(1 << 31) - 1)]


def route(r=None, **change):
    a = dict(logits=P, ld=8, dtype=2, score=0, bias=None, renormalize=1, scale=1.0, routes=r or routes())
    a.update(change)
    return capi.RouteArgs(*a.values())


@pytest.mark.parametrize("change", [
    dict(logits=None), dict(logits=P + 2), dict(logits=P + 1, dtype=0), dict(ld=7), dict(ld=1 << 40), dict(dtype=3),
    dict(dtype=-1), dict(score=2), dict(score=-1), dict(bias=P + 2), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(scale=-float("inf"))])
def test_route(lib, change):
    a = route(**change)
    assert lib.bonsai_b1_route(ctypes.byref(a), None, 0, None) == capi.ERR_ARG
    assert lib.bonsai_b1_route_workspace_bytes(ctypes.byref(a)) == 0


@pytest.mark.parametrize("change", BAD_COUNTS + [dict(expert=None), dict(weight=None), dict(start=None),
                                                 dict(order=None), dict(place=None), dict(expert=P + 2),
                                                 dict(weight=P + 1), dict(start=P + 2), dict(order=P + 3),
                                                 dict(place=P + 2)])
def test_route_arrays(lib, change):
    a = route(routes(**change), ld=1 << 20)
    assert lib.bonsai_b1_route(ctypes.byref(a), None, 0, None) == capi.ERR_ARG


def test_route_workspace(lib):
    few, many = route(), route(routes(tokens=4000))
    assert lib.bonsai_b1_route_workspace_bytes(ctypes.byref(few)) == 0
    assert lib.bonsai_b1_route_workspace_bytes(ctypes.byref(many)) > 0
    most = route(routes(tokens=(1 << 23) - 1, experts=1024), ld=1024)
    assert 0 < lib.bonsai_b1_route_workspace_bytes(ctypes.byref(most)) <= 1 << 20
    assert lib.bonsai_b1_route(ctypes.byref(many), P + 8, 1 << 20, None) == capi.ERR_ARG
    assert lib.bonsai_b1_route(None, None, 0, None) == capi.ERR_ARG


def experts(r=None, **change):
    a = dict(routes=r or routes(), act=P, by_token=1, w=P, in_dim=128, out_dim=128, act_fn=0, packed=None, ldp=0, out=P,
             ldo=128, nonfinite=None, bad=None)
    a.update(change)
    return capi.ExpertsArgs(*a.values())


PACKED = dict(out=None, ldo=0, packed=P, ldp=128)


@pytest.mark.parametrize("change", [
    dict(act=None), dict(act=P + 8), dict(w=None), dict(w=P + 2), dict(in_dim=0), dict(in_dim=96), dict(in_dim=-64),
    dict(out_dim=0), dict(out_dim=-1), dict(act_fn=1), dict(act_fn=2), dict(act_fn=3), dict(out=None),
    dict(out=P + 2), dict(ldo=127), dict(ldo=1 << 40), dict(packed=P, ldp=128), dict(nonfinite=P + 1),
    dict(bad=P + 2), dict(in_dim=65536 + 64), dict(out_dim=(1 << 17) + 1, ldo=1 << 18),
    dict(in_dim=65536, routes=routes(tokens=32768))])
def test_linear_experts(lib, change):
    assert lib.bonsai_b1_linear_experts(ctypes.byref(experts(**change)), None) == capi.ERR_ARG


@pytest.mark.parametrize("change", [
    dict(packed=P + 8), dict(ldp=120), dict(ldp=132), dict(act_fn=3), dict(act_fn=-1), dict(out_dim=120, ldp=128),
    dict(out_dim=96, act_fn=2), dict(out_dim=256, act_fn=2, ldp=120), dict(out=P, ldo=128), dict(ldp=1 << 42)])
def test_linear_experts_packed(lib, change):
    assert lib.bonsai_b1_linear_experts(ctypes.byref(experts(**(PACKED | change))), None) == capi.ERR_ARG


@pytest.mark.parametrize("change", BAD_COUNTS + [dict(start=None), dict(order=None), dict(start=P + 1),
                                                 dict(order=P + 2)])
def test_linear_experts_routes(lib, change):
    assert lib.bonsai_b1_linear_experts(ctypes.byref(experts(routes(**change))), None) == capi.ERR_ARG
    assert lib.bonsai_b1_linear_experts(None, None) == capi.ERR_ARG


@pytest.mark.parametrize("change", [
    dict(y=None), dict(y=P + 8), dict(ldy=60), dict(ldy=66), dict(H=0), dict(H=66), dict(H=-4), dict(residual=P + 4),
    dict(residual=P, ldr=32), dict(residual=P, ldr=65), dict(out=None), dict(out=P + 4), dict(ldo=63), dict(ldo=62),
    dict(residual=P * 2, ldr=128), dict(bad=P + 2), dict(ldy=1 << 40),
    dict(H=(1 << 24) + 4, ldy=1 << 25, ldo=1 << 25)])
def test_combine_experts(lib, change):
    a = dict(routes=ctypes.byref(routes()), y=P, ldy=64, H=64, residual=None, ldr=0, out=P * 2, ldo=64, bad=None)
    a.update(change)
    assert lib.bonsai_b1_combine_experts(*a.values(), None) == capi.ERR_ARG


@pytest.mark.parametrize("change", BAD_COUNTS + [dict(weight=None), dict(place=None), dict(weight=P + 2),
                                                 dict(place=P + 1)])
def test_combine_experts_routes(lib, change):
    r = routes(**change)
    assert lib.bonsai_b1_combine_experts(ctypes.byref(r), P, 64, 64, None, 0, P * 2, 64, None, None) == capi.ERR_ARG
    assert lib.bonsai_b1_combine_experts(None, P, 64, 64, None, 0, P * 2, 64, None, None) == capi.ERR_ARG


def test_python_refusals():
    import torch
    x = torch.zeros(3, 8)
    i = torch.zeros(3, 2, dtype=torch.int32)
    good = bonsai_b1.Routes(i, torch.zeros(3, 2), torch.zeros(9, dtype=torch.int32), i.flatten(), i)
    assert (good.tokens, good.top_k, good.experts) == (3, 2, 8)
    c = capi._routes_c(good)
    assert (c.tokens, c.top_k, c.experts) == (3, 2, 8)
    for bad in (dict(expert=i.long()), dict(weight=torch.zeros(3, 2).double()), dict(weight=torch.zeros(3, 1)),
                dict(place=i.flatten()[:4]), dict(order=i.flatten()[:5]), dict(start=torch.zeros(9)),
                dict(expert=torch.zeros(2, 3, dtype=torch.int32).t()), dict(order=torch.zeros(12, dtype=torch.int32)[::2])):
        a = dict(expert=i, weight=torch.zeros(3, 2), start=good.start, order=good.order, place=i)
        with pytest.raises(ValueError):
            capi._routes_c(bonsai_b1.Routes(**(a | bad)))
    # tensors that are no cuda tensors
    with pytest.raises(ValueError):
        bonsai_b1.route(x, 2)
    with pytest.raises(ValueError):
        bonsai_b1.linear_experts(x, x, good, 64, 64)
    with pytest.raises(ValueError):
        bonsai_b1.combine_experts(x, good)
    for bad in (dict(top_k=0), dict(top_k=9), dict(logits=x[0]), dict(logits=x.double()), dict(logits=x.int())):
        with pytest.raises(ValueError):
            bonsai_b1.route(**({"logits": x, "top_k": 2} | bad))
    with pytest.raises(ValueError):
        bonsai_b1.linear_experts(x, x, good, 64, 64, rows="both")
