"""A balance bias chooses and does not weigh (hip_layers.h), also where it is
NaN: its expert comes first and has the weight of its logit.  A NaN logit makes
its own weight NaN, and the row's where softmax or the sum holds it."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from turbinator_c_amd import layers  # noqa: E402

pytestmark = pytest.mark.gpu


def route(x, bias, k, score, renorm):
    t, n = x.shape
    experts = torch.empty(t, k, dtype=torch.int32, device="cuda")
    weights = torch.empty(t, k, device="cuda")
    assert layers.route_device(x, n * 4, bias, None, experts, weights, t, n, k, 1, 1,
                               layers.SCORES[score], renorm, 1.0, 0,
                               torch.cuda.current_stream()) == 1
    return experts, weights


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("n", [8, 64, 100])
def test_nan_bias_chooses_and_does_not_weigh(torch_cuda, score, renorm, n):
    x = torch.randn(33, n, device="cuda", generator=torch.Generator("cuda").manual_seed(n))
    x[5, 3] = -float("inf")
    bias, far = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    bias[3], far[3] = float("nan"), 100.0
    experts, weights = route(x, bias, 2, score, renorm)
    assert (experts[:5, 0] == 3).all() and (experts[6:, 0] == 3).all() and (experts[5] != 3).all()
    assert torch.isfinite(weights).all()
    # Any bias that puts the expert first gives the same.
    for a, b in zip((experts, weights), route(x, far, 2, score, renorm)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
def test_whose_weights_a_nan_logit_takes(torch_cuda, score, renorm, with_bias):
    x = torch.randn(9, 16, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    x[4, 7] = float("nan")
    bias = torch.linspace(0, 0.1, 16, device="cuda") if with_bias else None
    experts, weights = route(x, bias, 3, score, renorm)
    nan = torch.isnan(weights)
    assert not nan[:4].any() and not nan[5:].any()
    if score == "softmax" or renorm:
        assert nan[4].all()
    else:
        assert torch.equal(nan[4], experts[4] == 7) and experts[4, 0] == 7
