"""Routing to experts, its gradient and the order of the choices (hip_layers.h)
against plain forms in 64 bits: few and many experts, groups, bias, masked and
empty rows, ties, NaN and infinities, padding tokens, strides.

Tolerances.  A score is off by a few units u = 2^-24 of the exponential, the
sum over the row (at most 1,024 terms, 16 in sequence) and the quotient: 64 u
of itself.  A gradient is a score times a difference of terms that are off by
64 u of their size each.  Without a bias the keys are the logits and the
experts are compared exactly.  Biased keys (below 2) are off by 64 u, so two of
them closer than 128 u may come in either order, and rows whose last kept group
leads by less are not compared.
"""
from __future__ import annotations

import math

import pytest
import torch

from turbinator_c_amd import layers

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def logits_of(seed, t, n, dtype, pitch=None, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    pitch = pitch or n
    wide = torch.full((t, pitch), float("nan"))
    wide[:, pitch - n:] = spread * torch.randn((t, n), generator=g)
    return wide.to(dtype).cuda()[:, pitch - n:]


def bias_of(seed, n):
    g = torch.Generator().manual_seed(seed + 77)
    return (0.1 * torch.randn(n, generator=g)).cuda()


def route(x, k, score="softmax", renorm=True, bias=None, valid=None, groups=1, kept=1,
          scale=1.0, stream=None):
    t, n = x.shape
    experts = torch.full((t, k), -7, dtype=torch.int32, device="cuda")
    weights = torch.full((t, k), 7.0, device="cuda")
    assert layers.route_device(x, x.stride(0) * x.element_size(), bias, valid, experts, weights,
                               t, n, k, groups, kept, layers.SCORES[score], renorm, scale,
                               layers.DTYPES[x.dtype],
                               stream or torch.cuda.current_stream()) == 1
    torch.cuda.synchronize()
    return experts, weights


def oracle(x, k, score, renorm, bias, valid, groups, kept, scale):
    """One row at a time, in 64 bits, by sorting (key, index) pairs.  Returns
    experts, the keys of all experts (NaN as +inf; -inf where never chosen),
    weights of given picks, and the gap between the last kept group and the
    next."""
    x = x.double().cpu()
    t, n = x.shape
    per = n // groups
    s = torch.softmax(x, 1) if score == "softmax" else torch.sigmoid(x)
    key = x if bias is None else s + bias.double().cpu()
    key = torch.where(x == -math.inf, -math.inf, key)
    key = torch.where(torch.isnan(key), math.inf, key)
    experts = torch.full((t, k), -1, dtype=torch.int32)
    gaps = torch.full((t,), math.inf, dtype=torch.float64)
    for r in range(t):
        if valid is not None and not valid[r]:
            key[r] = -math.inf
            continue
        rank = key[r].tolist()
        if kept < groups:
            stands = []
            for g in range(groups):
                two = sorted(rank[g * per:(g + 1) * per], reverse=True)[:2]
                extra = two[1] if bias is not None and len(two) > 1 and two[1] > -math.inf else 0.0
                stands.append(two[0] + extra)
            order = sorted(range(groups), key=lambda g: (-stands[g], g))
            if bias is not None and stands[order[kept - 1]] < math.inf:
                gaps[r] = stands[order[kept - 1]] - stands[order[kept]]
            for g in order[kept:]:
                rank[g * per:(g + 1) * per] = [-math.inf] * per
            key[r] = torch.tensor(rank, dtype=torch.float64)
        order = sorted(range(n), key=lambda e: (-rank[e], e))
        picks = [e for e in order[:k] if rank[e] > -math.inf]
        experts[r, :len(picks)] = torch.tensor(picks, dtype=torch.int32)

    def weights(picks):
        gone, at = picks < 0, picks.long().clamp(min=0)
        if renorm and score == "softmax":
            w = torch.softmax(torch.where(gone, -math.inf, x.gather(1, at)), 1)
        else:
            w = torch.where(gone, 0.0, s.gather(1, at))
            if renorm:
                w = w / w.sum(dim=1, keepdim=True)
        return torch.where(gone, 0.0, w) * scale

    return experts, key, weights, gaps


def check(x, k, score="softmax", renorm=True, bias=None, valid=None, groups=1, kept=1,
          scale=1.0):
    experts, weights = route(x, k, score, renorm, bias, valid, groups, kept, scale)
    want, key, weigh, gaps = oracle(x, k, score, renorm, bias, valid, groups, kept, scale)
    sure = gaps > 128 * U
    assert sure.float().mean() > 0.9 or len(sure) < 20
    got = experts.cpu()
    if bias is None:
        assert torch.equal(got, want)
    else:
        # Keys closer than their error may come in either order: each pick's
        # key must be that of its place.  No expert comes twice.
        assert torch.equal((got < 0)[sure], (want < 0)[sure])
        at, place = (torch.where(e < 0, 0.0, key.gather(1, e.long().clamp(min=0)))
                     for e in (got, want))
        same = (at == place) | ((at - place).abs() <= 128 * U)
        assert same[sure].all()
        low, high = got.sort(dim=1).values[:, :-1], got.sort(dim=1).values[:, 1:]
        assert ((low != high) | (low < 0)).all()
    want_w, got_w = weigh(got), weights.cpu().double()
    nan = torch.isnan(want_w)
    assert torch.equal(torch.isnan(got_w), nan)
    err = torch.where(nan, 0.0, (got_w - want_w).abs() - 64 * U * want_w.abs() - 1e-37)
    assert err.max() <= 0
    return experts, weights


EXPERTS = [(1, 1), (2, 1), (3, 3), (7, 2), (8, 2), (9, 4), (16, 16), (33, 5), (64, 8), (100, 6),
           (128, 32), (256, 8), (500, 3), (513, 7), (1000, 32), (1024, 8)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,k", EXPERTS)
def test_experts_and_weights(torch_cuda, n, k, dtype):
    for i, t in enumerate((1, 37, 261 if n <= 256 else 70)):
        x = logits_of(n + k + t, t, n, dtype)
        print(n, k, dtype, t, flush=True)
        check(x, k, "softmax", True)
        check(x, k, "softmax", False, scale=2.5)
        check(x, k, "sigmoid", True, scale=0.5)
        check(x, k, "sigmoid", False)
        check(x, k, ["softmax", "sigmoid"][i % 2], True, bias=bias_of(n, n))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("n,groups,kept,k", [(8, 4, 2, 3), (8, 8, 3, 2), (64, 8, 4, 4),
                                             (64, 8, 1, 8), (60, 4, 3, 9), (160, 8, 3, 6),
                                             (96, 32, 5, 8), (21, 7, 2, 5), (256, 8, 4, 8),
                                             (1024, 256, 9, 20), (768, 3, 2, 10)])
def test_groups(torch_cuda, n, groups, kept, k, with_bias, score):
    x = logits_of(n + kept, 150, n, torch.float32)
    check(x, k, score, True, bias_of(n, n) if with_bias else None, None, groups, kept)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strided_rows(torch_cuda, dtype):
    for pitch in (25, 32, 40):
        check(logits_of(pitch, 90, 24, dtype, pitch), 4, "softmax", True)


def test_ties_go_to_the_lowest_index(torch_cuda):
    x = torch.zeros((70, 40), device="cuda")
    experts, weights = route(x, 6)
    assert (experts.cpu() == torch.arange(6, dtype=torch.int32)).all()
    x[:, 5] = -0.0
    experts, _ = route(x, 6)
    assert (experts.cpu() == torch.arange(6, dtype=torch.int32)).all()
    x[:, 20:] = 1.0
    experts, _ = route(x, 6, groups=4, kept=2)
    assert (experts.cpu() == torch.arange(20, 26, dtype=torch.int32)).all()
    # Equal groups: the lower ones are kept.
    experts, _ = route(torch.zeros((3, 40), device="cuda"), 20, groups=4, kept=2)
    assert (experts.cpu() == torch.arange(20, dtype=torch.int32)).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("with_bias", [True, False])
def test_masked_experts(torch_cuda, score, renorm, with_bias):
    """-inf logits are never chosen; rows with too few experts left are filled
    with -1, rows without any are empty."""
    x = logits_of(3, 64, 24, torch.float32)
    for r in range(64):
        x[r, torch.randperm(24, generator=torch.Generator().manual_seed(r))[:r % 25]] = -math.inf
    bias = bias_of(4, 24) if with_bias else None
    experts, weights = check(x, 5, score, renorm, bias)
    assert (experts[24] == -1).all() and (weights[24] == 0).all()
    assert (experts[23] >= 0).sum() == 1
    check(x, 5, score, renorm, bias, None, 4, 2)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_lowest_values_as_masks(torch_cuda, dtype, score):
    """Masks of the type's lowest value: chosen last, with weight 0 beside
    others; a row of them alone stays finite."""
    x = logits_of(3, 6, 16, dtype)
    x[:3, 2:] = torch.finfo(dtype).min
    x[3:] = torch.finfo(dtype).min
    experts, weights = route(x, 4, score, True)
    assert torch.isfinite(weights).all()
    assert ((experts >= 0) & (experts < 16)).all()
    assert (weights[:3, 2:] == 0).all()
    assert ((weights[:3].sum(dim=1) - 1).abs() < 8 * U).all()
    assert (experts[3:].cpu() == torch.arange(4, dtype=torch.int32)).all()
    assert (weights[3:] == (0.25 if score == "softmax" else 0.0)).all()


def test_nan_and_inf(torch_cuda):
    x = logits_of(8, 5, 20, torch.float32)
    x[0, 7] = float("nan")
    x[1, 4] = math.inf
    x[2] = float("nan")
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            experts, weights = route(x, 3, score, renorm)
            assert ((experts >= 0) & (experts < 20)).all()
            assert experts[0, 0] == 7 and experts[1, 0] == 4
            assert (experts[2].cpu() == torch.arange(3, dtype=torch.int32)).all()
            assert torch.isnan(weights[0, 0]) and torch.isnan(weights[2]).all()
            assert torch.isfinite(weights[3:]).all()
            if score == "softmax":
                assert torch.isnan(weights[0]).all() and torch.isnan(weights[1, 0])


def test_padding_tokens_are_not_read(torch_cuda):
    x = logits_of(8, 200, 20, torch.bfloat16)
    valid = (torch.arange(200) % 3 != 1).to(torch.uint8).cuda()
    x[valid == 0] = float("nan")
    experts, weights = check(x, 3, "sigmoid", True, bias_of(2, 20), valid, 4, 2)
    assert (experts[valid == 0] == -1).all() and (weights[valid == 0] == 0).all()


def test_other_stream(torch_cuda):
    x = logits_of(8, 5000, 64, torch.bfloat16)
    torch.cuda.synchronize()
    for a, b in zip(route(x, 4), route(x, 4, stream=torch.cuda.Stream())):
        assert torch.equal(a, b)


# --------------------------------------------------------------------------
# Gradient


def weights_of(x, experts, score, renorm, scale):
    """The weights of given experts in 64 bits; -1 has weight 0."""
    gone = experts < 0
    at = experts.long().clamp(min=0)
    if renorm and score == "softmax":
        w = torch.softmax(torch.where(gone, -math.inf, x.gather(1, at)), 1)
    else:
        s = torch.softmax(x, 1) if score == "softmax" else torch.sigmoid(x)
        w = torch.where(gone, 0.0, s.gather(1, at))
        if renorm:
            w = w / w.sum(dim=1, keepdim=True)
    return torch.where(gone, 0.0, w) * scale


def backward(x, experts, dw, score, renorm, scale):
    t, n = x.shape
    dl = torch.full((t, n), 7.0, dtype=x.dtype, device="cuda")
    assert layers.route_backward_device(x, x.stride(0) * x.element_size(), experts, dw, dl, t, n,
                                        experts.shape[1], layers.SCORES[score], renorm, scale,
                                        layers.DTYPES[x.dtype],
                                        torch.cuda.current_stream()) == 1
    torch.cuda.synchronize()
    return dl


def check_backward(x, experts, score, renorm, scale=1.0):
    t, n = x.shape
    g = torch.Generator().manual_seed(t + n)
    dw = torch.randn(experts.shape, generator=g).cuda()
    dl = backward(x, experts, dw, score, renorm, scale)
    xd = x.double().requires_grad_()
    live = (experts >= 0).any(dim=1)
    w = weights_of(xd[live], experts[live], score, renorm, scale)
    (w * dw[live].double()).sum().backward()
    want = xd.grad
    # A score times (its own term - the row's sum of terms).
    size = torch.zeros_like(want)
    wd = w.detach().abs()
    row = (wd * dw[live].double().abs()).sum(dim=1, keepdim=True)
    at = experts[live].long().clamp(min=0)
    part = torch.zeros_like(want[live])
    part.scatter_add_(1, at, wd * (dw[live].double().abs() + row / abs(scale)))
    if score == "softmax" and not renorm:
        part += torch.softmax(x[live].double(), 1) * row
    size[live] = part
    over = (dl.double() - want).abs() - 64 * U * size - HALF_ULP[x.dtype] * want.abs() - \
        LEAST[x.dtype]
    assert over.max() <= 0, over.max()
    return dl


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("n,k", [(1, 1), (2, 2), (7, 2), (8, 2), (33, 5), (64, 8), (100, 32),
                                 (256, 8), (513, 7), (1024, 8)])
def test_gradient(torch_cuda, n, k, score, renorm, dtype):
    for t in (1, 90):
        x = logits_of(n + t, t, n, dtype, n + 3)
        experts, _ = route(x, k, score, renorm)
        print(n, k, score, renorm, dtype, t, flush=True)
        check_backward(x, experts, score, renorm, 2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_a_single_renormalised_choice_has_no_gradient(torch_cuda, score):
    x = logits_of(5, 40, 24, torch.float32)
    experts, weights = route(x, 1, score, True)
    assert (weights == 1).all()
    dw = torch.randn(experts.shape, generator=torch.Generator().manual_seed(3)).cuda()
    assert (backward(x, experts, dw, score, True, 1.0) == 0).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_gradient_of_partial_and_empty_rows(torch_cuda, score, renorm):
    x = logits_of(5, 40, 24, torch.float32)
    experts, _ = route(x, 4, score, renorm)
    experts[::5, 2:] = -1
    experts[3::7] = -1
    x[3::7] = float("nan")  # rows without an expert are not read
    dl = check_backward(torch.where(torch.isnan(x), 0.0, x), experts, score, renorm)
    dw = torch.ones(experts.shape, device="cuda")
    dl = backward(x, experts, dw, score, renorm, 1.0)
    assert (dl[3::7] == 0).all() and torch.isfinite(dl).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_gradient_against_differences(torch_cuda, score, renorm):
    """Central differences of the 64-bit weights, step 1e-6: off by 1e-10."""
    x = logits_of(15, 6, 20, torch.float32)
    experts, _ = route(x, 4, score, renorm)
    g = torch.Generator().manual_seed(1)
    dw = torch.randn(experts.shape, generator=g).cuda()
    dl = backward(x, experts, dw, score, renorm, 1.0)
    for e in range(20):
        step = torch.zeros_like(x, dtype=torch.float64)
        step[:, e] = 1e-6
        up, down = (weights_of(x.double() + s * step, experts, score, renorm, 1.0)
                    for s in (1, -1))
        slope = ((up - down) * dw.double()).sum(dim=1) / 2e-6
        assert ((dl[:, e].double() - slope).abs() <= 1e-6 * (1 + dw.double().abs().sum(dim=1))).all()


# --------------------------------------------------------------------------
# Order


def order(experts, weights, n):
    t, k = experts.shape
    need = layers.expert_order_workspace_bytes(t, n, k)
    ws = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device="cuda")
    offsets = torch.full((n + 1,), -7, dtype=torch.int32, device="cuda")
    tokens, positions = (torch.full((t * k,), -7, dtype=torch.int32, device="cuda")
                         for _ in range(2))
    row_weights = None if weights is None else torch.full((t * k,), 7.0, device="cuda")
    assert layers.expert_order_device(experts, weights, offsets, tokens, positions, row_weights,
                                      ws, t, n, k, torch.cuda.current_stream()) == 1
    torch.cuda.synchronize()
    assert (ws[need:] == 0x5a).all()
    return offsets, tokens, positions, row_weights


def check_order(experts, weights, n):
    t, k = experts.shape
    offsets, tokens, positions, row_weights = order(experts, weights, n)
    flat = experts.reshape(-1).long()
    flat = torch.where((flat < 0) | (flat >= n), n, flat)
    by = flat.sort(stable=True)
    count = torch.bincount(flat, minlength=n + 1)
    want = torch.cat([count.new_zeros(1), count[:n].cumsum(0)])
    assert torch.equal(offsets.long(), want)
    live = by.values < n
    assert torch.equal(tokens.long(), torch.where(live, by.indices // k, -1))
    rows = torch.empty_like(flat)
    rows[by.indices] = torch.where(live, torch.arange(t * k, device="cuda"), -1)
    assert torch.equal(positions.long(), rows)
    if weights is not None:
        assert torch.equal(row_weights, torch.where(live, weights.reshape(-1)[by.indices], 0.0))


@pytest.mark.parametrize("n", [1, 2, 8, 63, 64, 65, 200, 1023, 1024])
def test_order(torch_cuda, n):
    for t, k in ((1, 1), (5, 3), (64, 1), (320, 2), (1023, 2), (2049, 1), (20000, 7)):
        g = torch.Generator().manual_seed(n + t)
        experts = torch.randint(0, n, (t, k), generator=g).to(torch.int32).cuda()
        weights = torch.rand((t, k), generator=g).cuda()
        print(n, t, k, flush=True)
        check_order(experts, weights, n)
        experts[torch.rand((t, k), generator=g).cuda() < 0.2] = -1
        check_order(experts, weights, n)
        check_order(experts, None, n)
        # All to one expert; none at all; numbers outside the experts.
        check_order(torch.full_like(experts, n - 1), weights, n)
        check_order(torch.full_like(experts, -1), weights, n)
        experts[0, 0] = n
        experts[-1, -1] = 2 ** 31 - 1
        check_order(experts, weights, n)


def test_order_of_more_choices_than_segments_hold(torch_cuda):
    """Over 2 million choices: segments longer than the shortest."""
    g = torch.Generator().manual_seed(1)
    check_order(torch.randint(-1, 40, (700_001, 4), generator=g).to(torch.int32).cuda(),
                torch.rand((700_001, 4), generator=g).cuda(), 40)


def test_refusals(torch_cuda):
    x = torch.zeros((4, 8), device="cuda")
    experts = torch.full((4, 2), -7, dtype=torch.int32, device="cuda")
    weights = torch.full((4, 2), 7.0, device="cuda")
    stream = torch.cuda.current_stream()

    def call(x=x, stride=32, experts=experts, weights=weights, t=4, n=8, k=2, groups=1, kept=1,
             score=0, dt=0):
        return layers.route_device(x, stride, None, None, experts, weights, t, n, k, groups,
                                   kept, score, True, 1.0, dt, stream)

    def back(x=x, stride=32, experts=experts, weights=weights, out=x, t=4, n=8, k=2, score=0,
             dt=0):
        return layers.route_backward_device(x, stride, experts, weights, out, t, n, k, score,
                                            True, 1.0, dt, stream)

    for over in (dict(x=None), dict(experts=None), dict(weights=None), dict(t=0), dict(n=0),
                 dict(n=1025, k=2), dict(k=0), dict(k=9), dict(n=64, k=33), dict(t=2 ** 31),
                 dict(t=2 ** 30), dict(score=2), dict(score=-1), dict(dt=3), dict(stride=33),
                 dict(x=x.data_ptr() + 2)):
        assert call(**over) == 0, over
        assert back(**over) == 0, over
    for over in (dict(groups=3), dict(groups=0), dict(groups=4, kept=5), dict(groups=4, kept=0),
                 dict(groups=8, kept=1, k=2)):
        assert call(**over) == 0, over
    assert back(out=None) == 0 and back(out=x.data_ptr() + 2) == 0

    ws = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    ints = [torch.full((64,), -7, dtype=torch.int32, device="cuda") for _ in range(3)]
    good = [experts, None, *ints, None, ws, 4, 8, 2]
    for i, v in ((0, None), (2, None), (3, None), (4, None), (1, weights), (5, weights),
                 (6, None), (6, ws.data_ptr() + 4), (7, 0), (7, 2 ** 31), (8, 0), (8, 1025),
                 (9, 0), (9, 33)):
        args = list(good)
        args[i] = v
        assert layers.expert_order_device(*args, stream) == 0, i
    torch.cuda.synchronize()
    assert (experts == -7).all() and (weights == 7).all() and all((v == -7).all() for v in ints)
    assert layers.expert_order_workspace_bytes(0, 8, 2) == 0
    assert layers.expert_order_workspace_bytes(4, 0, 2) == 0
    assert layers.expert_order_workspace_bytes(2 ** 31, 8, 2) == 0
