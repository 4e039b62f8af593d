"""Experts' rows whose last ones are cut off (hip_layers.h): offsets[n_experts]
lowered, and the positions from there on set to -1, where each gradient is that
of its entry; and what each of the four entries does with a position that was
left there.

Tolerances as in the entries' own tests; the gradients of the whole chain are
compared in fp32 with automatic differentiation in 64 bits: sums of at most
k + 2 products, dot products as there.
"""
from __future__ import annotations

import pytest
import torch

from turbinator_c_amd import layers

from .test_gpu_expert_rows import (TYPES, check_dots, check_sum, now, out_like, plain_picked,
                                   plain_rows, routing, spread, stride, untouched)

pytestmark = pytest.mark.gpu


def run(x, y, offsets, positions, weights, e):
    """rows, out, dx, the rows' dweights, drows, the sum's dweights."""
    (t, d), k, code, s = x.shape, positions.shape[1], layers.DTYPES[x.dtype], now()
    o, p, w = offsets.cuda(), positions.cuda(), weights.cuda()
    made = [out_like(t * k, d, x.dtype), out_like(t, d, x.dtype), out_like(t, d, x.dtype),
            out_like(t, k, torch.float32), out_like(t * k, d, x.dtype),
            out_like(t, k, torch.float32)]
    rows, out, dx, dw, drows, dv = (view for _, view in made)
    assert layers.expert_rows_device(x, stride(x), o, p, w, rows, t, e, k, d, code, s) == 1
    assert layers.expert_sum_device(y, stride(y), p, w, None, 0, out, t, k, d, code, s) == 1
    assert layers.expert_rows_backward_device(y, stride(y), x, stride(x), p, w, dx, dw, t, k, d,
                                              code, s) == 1
    assert layers.expert_sum_backward_device(x, stride(x), y, stride(y), o, p, w, drows, dv, t, e,
                                             k, d, code, s) == 1
    for buffer, _ in made:
        untouched(buffer)
    return [view.cpu() for _, view in made]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("t,e,k,d,keep", [(1, 4, 2, 9, 1), (40, 8, 3, 130, 57), (40, 8, 3, 130, 0),
                                          (33, 64, 10, 513, 200), (4100, 16, 2, 520, 7000)])
def test_gradients_of_what_is_left(torch_cuda, t, e, k, d, keep, dtype):
    """<out, dout> and <rows, drows> by automatic differentiation: x serves as
    the tokens and as the sum's gradient, y as the rows and as theirs."""
    g = torch.Generator().manual_seed(t + keep)
    offsets, positions = routing(g, t, e, k, 0.1)
    assert keep <= int(offsets[-1])
    offsets = offsets.clamp(max=keep)
    positions = torch.where(positions < keep, positions, -1)
    weights = torch.randn(t, k, generator=g)
    x, y = spread(g, t, d, dtype), spread(g, t * k, d, dtype)
    # Nothing reads the rows that are cut off.
    y[keep:] = float("nan")
    rows, out, dx, dw, drows, dv = run(x, y, offsets, positions, weights, e)

    assert torch.equal(rows, plain_rows(x.cpu(), positions, weights)) and (rows[keep:] == 0).all()
    assert torch.equal(drows, rows)  # the same formula of the same inputs
    v = plain_picked(y.cpu(), positions)
    check_sum(out, v, weights, None, dtype)

    x64, w64 = (a.cpu().double().requires_grad_() for a in (x, weights))
    live = positions >= 0
    token = torch.arange(t)[:, None].expand(-1, k)[live]
    ((w64[live][:, None] * x64[token]) * v[live]).sum().backward()
    want = x64.grad
    size = torch.zeros_like(want).index_add_(0, token, (weights.double()[live][:, None] *
                                                        v[live]).abs())
    assert torch.equal(dx[size.sum(1) == 0], torch.zeros_like(dx[size.sum(1) == 0]))
    check_sum(dx, v, weights, None, dtype)
    # check_sum's and check_dots' formulas are those of the derivatives.
    picked = (v * weights.double()[..., None]).sum(1)
    assert ((picked - want).abs() <= 1e-12 * (size + 1)).all()
    dots = (v * x.cpu().double()[:, None, :]).sum(2)
    assert ((dots - w64.grad).abs() <= 1e-12 * (1 + dots.abs()) * d).all()
    for got in (dw, dv):
        check_dots(got, v, x.cpu(), dtype)
        assert (got[~live] == 0).all()


def test_positions_that_were_left(torch_cuda):
    """Writers of rows take them as none, readers read the row."""
    t, k, d = 3, 2, 40
    g = torch.Generator().manual_seed(1)
    positions = torch.tensor([[0, 5], [4, 1], [2, 3]], dtype=torch.int32)
    offsets = torch.tensor([0, 4], dtype=torch.int32)
    weights = torch.rand(t, k, generator=g) + 0.5
    x, y = spread(g, t, d, torch.float32), spread(g, t * k, d, torch.float32)
    rows, out, dx, dw, drows, dv = run(x, y, offsets, positions, weights, 1)
    known = torch.where(positions < 4, positions, -1)
    assert torch.equal(rows, plain_rows(x.cpu(), known, weights))
    assert torch.equal(drows, rows)
    check_dots(dv, plain_picked(y.cpu(), known), x.cpu(), torch.float32)
    assert dv[0, 1] == 0 and dv[1, 0] == 0
    every = plain_picked(y.cpu(), positions)
    check_sum(out, every, weights, None, torch.float32)
    check_sum(dx, every, weights, None, torch.float32)
    check_dots(dw, every, x.cpu(), torch.float32)


def test_rows_that_no_choice_has(torch_cuda):
    """Below the end they are left as they were, behind it cleared."""
    x = torch.arange(1, 13, device="cuda").float().view(3, 4)
    positions = torch.tensor([2, -1, 0], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    for entry, more in ((layers.expert_rows_device, ()),
                        (layers.expert_sum_backward_device, (None, 0))):
        rows = torch.full((3, 4), 7.0, device="cuda")
        end = (rows,) if not more else (rows, None)
        assert entry(x, 16, *more, offsets, positions, None, *end, 3, 1, 1, 4, 0, now()) == 1
        assert torch.equal(rows, torch.stack([x[2], torch.full_like(x[0], 7), x[0] * 0]))
