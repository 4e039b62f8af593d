"""Refusals of the routing and 4-bit entries (hip_layers.h) that return before
any HIP call, and their sizes: no GPU."""
from __future__ import annotations

import pytest

from turbinator_c_amd import layers

AT = 4096  # an aligned address; never read
ROUTE = dict(logits=AT, row_stride=32, bias=None, valid=None, experts=AT, weights=AT, tokens=5,
             n_experts=8, k=2, groups=1, groups_kept=1, score=0, renormalise=True, scale=1.0,
             dtype=0)
BACK = dict(logits=AT, row_stride=32, experts=AT, dweights=AT, dlogits=AT, tokens=5, n_experts=8,
            k=2, score=0, renormalise=True, scale=1.0, dtype=0)
ORDER = dict(experts=AT, weights=None, offsets=AT, tokens_out=AT, positions=AT, row_weights=None,
             workspace=AT, tokens=5, n_experts=8, k=2)
QUANT = dict(x=AT, row_stride=64, codes=AT, scales=AT, rows=3, k=16, dtype=0)
VALUES = dict(codes=AT, scales=AT, values=AT, rows=3, k=16, dtype=0)
PRODUCT = dict(a_codes=AT, a_scales=AT, a_rows=4, rows=None, w_codes=AT, w_scales=AT,
               offsets=None, bias=None, row_scale=None, out=AT, m=4, n=8, k=16, experts=1, act=0,
               dtype=0)
BIG = 2 ** 31


@pytest.mark.parametrize("change", [
    dict(logits=None), dict(experts=None), dict(weights=None), dict(tokens=0),
    dict(tokens=BIG // 2), dict(n_experts=0), dict(n_experts=1025), dict(k=0), dict(k=9),
    dict(n_experts=64, k=33), dict(groups=0), dict(groups=3), dict(groups=4, groups_kept=5),
    dict(groups=8, groups_kept=1), dict(groups=4, groups_kept=0), dict(score=2), dict(score=-1),
    dict(dtype=3), dict(dtype=-1), dict(logits=AT + 2), dict(row_stride=34),
    dict(dtype=1, row_stride=17), dict(dtype=2, logits=AT + 1)], ids=str)
def test_route(change):
    assert layers.route_device(**{**ROUTE, **change}) == 0


@pytest.mark.parametrize("change", [
    dict(logits=None), dict(experts=None), dict(dweights=None), dict(dlogits=None),
    dict(tokens=0), dict(tokens=BIG // 2), dict(n_experts=0), dict(n_experts=1025), dict(k=0),
    dict(k=9), dict(score=5), dict(dtype=9), dict(logits=AT + 1), dict(dlogits=AT + 2),
    dict(row_stride=30)], ids=str)
def test_route_backward(change):
    assert layers.route_backward_device(**{**BACK, **change}) == 0


@pytest.mark.parametrize("change", [
    dict(experts=None), dict(offsets=None), dict(tokens_out=None), dict(positions=None),
    dict(workspace=None), dict(workspace=AT + 8), dict(weights=AT), dict(row_weights=AT),
    dict(tokens=0), dict(tokens=BIG // 2), dict(n_experts=0), dict(n_experts=1025), dict(k=0),
    dict(k=33)], ids=str)
def test_expert_order(change):
    assert layers.expert_order_device(**{**ORDER, **change}) == 0


@pytest.mark.parametrize("tokens,n,k", [(1, 1, 1), (320, 8, 2), (4097, 1024, 32), (163840, 64, 4),
                                        (2 ** 26, 1024, 31)])
def test_expert_order_workspace(tokens, n, k):
    need = layers.expert_order_workspace_bytes(tokens, n, k)
    # Counts of each expert and of none, for at most 4,096 segments, and totals.
    assert 0 < need <= (n + 1) * 4097 * 4 + 16 and need % 16 == 0


def test_expert_order_workspace_refusals():
    for args in ((0, 8, 2), (5, 0, 2), (5, 1025, 2), (5, 8, 0), (5, 8, 33), (BIG // 2, 8, 2)):
        assert layers.expert_order_workspace_bytes(*args) == 0


@pytest.mark.parametrize("change", [
    dict(x=None), dict(codes=None), dict(scales=None), dict(rows=0), dict(rows=BIG), dict(k=0),
    dict(k=BIG), dict(dtype=3), dict(codes=AT + 8), dict(scales=AT + 2), dict(x=AT + 2),
    dict(row_stride=66), dict(dtype=1, row_stride=33)], ids=str)
def test_quantise(change):
    assert layers.mx4_quantise_device(**{**QUANT, **change}) == 0


@pytest.mark.parametrize("change", [
    dict(codes=None), dict(scales=None), dict(values=None), dict(rows=0), dict(rows=BIG),
    dict(k=0), dict(k=BIG), dict(dtype=-1), dict(codes=AT + 4), dict(scales=AT + 1),
    dict(values=AT + 2)], ids=str)
def test_values(change):
    assert layers.mx4_values_device(**{**VALUES, **change}) == 0


@pytest.mark.parametrize("change", [
    dict(a_codes=None), dict(a_scales=None), dict(w_codes=None), dict(w_scales=None),
    dict(out=None), dict(a_rows=0), dict(a_rows=BIG, m=BIG), dict(m=0), dict(m=5), dict(n=0),
    dict(n=BIG), dict(k=0), dict(k=BIG), dict(experts=0), dict(experts=1025, offsets=AT),
    dict(experts=2), dict(experts=2, offsets=AT, n=2 ** 30), dict(act=3), dict(dtype=3),
    dict(a_codes=AT + 8), dict(w_codes=AT + 8), dict(a_scales=AT + 1), dict(w_scales=AT + 2),
    dict(out=AT + 2), dict(rows=AT, m=BIG)], ids=str)
def test_product(change):
    assert layers.mx4_product_device(**{**PRODUCT, **change}) == 0


def test_padding():
    for k, kp in ((1, 128), (127, 128), (128, 128), (129, 256), (2000, 2048), (2 ** 31 - 1, 2 ** 31)):
        assert layers.mx4_padded(k) == kp
