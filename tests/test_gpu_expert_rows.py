"""Tokens to their experts' rows and back (hip_layers.h) against 64 bits: odd
widths and elements, choices without a row, rows behind the last expert's,
strides, all types, gradients by formula and by differences, graphs, streams.

Tolerances, u = 2^-24.  A row is one product, rounded to 32 bits and to the
type: compared bit for bit.  A sum of k products by fused additions and one of
the residual is within (k + 2) u of the sum of magnitudes, then rounded to the
type.  A dot product is added up by lanes of n elements of a vector and of every
64th vector after it, and then in pairs: depth n ceil(vectors / 64) + 10.
"""
from __future__ import annotations

import pytest
import torch

from turbinator_c_amd import layers

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def routing(g, t, e, k, missing=0.0):
    """experts [t, k], offsets [e + 1], positions [t, k] on the CPU; -1 for choices without."""
    experts = torch.stack([torch.randperm(max(e, k), generator=g)[:k] for _ in range(t)])
    gone = (torch.rand((t, k), generator=g) < missing) | (experts >= e)
    key = torch.where(gone, e, experts).reshape(-1)
    order = key.sort(stable=True)
    live = order.values < e
    positions = torch.empty(t * k, dtype=torch.int64)
    positions[order.indices] = torch.where(live, torch.arange(t * k), -1)
    count = torch.bincount(key, minlength=e + 1)[:e]
    offsets = torch.cat([count.new_zeros(1), count.cumsum(0)])
    return offsets.int(), positions.view(t, k).int()


def spread(g, m, d, dtype, pitch=None, shift=0):
    """[m, d] on the GPU, rows `pitch` elements apart, NaN between them."""
    pitch = pitch or d
    x = torch.full((m * pitch + shift,), float("nan"))
    view = x[shift:].view(m, pitch)[:, pitch - d:]
    view.copy_(torch.randn((m, d), generator=g) * torch.exp2(torch.randint(-3, 4, (m, 1), generator=g).float()))
    x = x.to(dtype).cuda()
    return x[shift:].view(m, pitch)[:, pitch - d:]


def out_like(m, d, dtype):
    """An output with a margin behind it."""
    buffer = torch.full((m * d + 64,), 7.0, dtype=dtype, device="cuda")
    return buffer, buffer[:m * d].view(m, d)


def untouched(buffer):
    assert (buffer[-64:] == 7).all()


def stride(x):
    return x.stride(0) * x.element_size()


def now():
    return torch.cuda.current_stream()


def depth(d, dtype):
    n = 16 // dtype.itemsize
    n = n if d >= n else 1
    return n * -(-(-(-d // n)) // 64) + 10


def plain_rows(x, positions, weights):
    """64-bit rows as the kernel rounds them, from 32-bit products."""
    t, k = positions.shape
    rows = torch.zeros((t * k, x.shape[1]), dtype=x.dtype)
    v = x[:, None, :].expand(-1, k, -1)
    if weights is not None:
        v = (v.float() * weights[..., None]).to(x.dtype)
    live = positions >= 0
    rows[positions[live].long()] = v[live]
    return rows


def plain_picked(rows, positions):
    v = rows.double()[positions.clamp(min=0).long()]
    return torch.where((positions >= 0)[..., None], v, 0.0)


def check_sum(got, v, weights, residual, dtype):
    """v [t, k, d] in 64 bits."""
    k = v.shape[1]
    terms = v if weights is None else v * weights.double()[..., None]
    want, size = terms.sum(1), terms.abs().sum(1)
    if residual is not None:
        want, size = want + residual.double(), size + residual.double().abs()
    bound = (k + 2) * U * size * 1.001 + HALF[dtype] * want.abs() * 1.01 + LEAST[dtype]
    assert ((got.double() - want).abs() <= bound).all()


def check_dots(got, v, x, dtype):
    terms = v * x.double()[:, None, :]
    bound = depth(x.shape[1], dtype) * U * terms.abs().sum(2) * 1.001 + 1e-37
    assert ((got.double() - terms.sum(2)).abs() <= bound).all()


def run_all(t, e, k, d, dtype, weighted=True, missing=0.1, pitch=None, shift=0, seed=0):
    g = torch.Generator().manual_seed(seed + t + 7 * k + 31 * d)
    code, s = layers.DTYPES[dtype], now()
    offsets, positions = routing(g, t, e, k, missing)
    weights = torch.randn((t, k), generator=g) if weighted else None
    x = spread(g, t, d, dtype, pitch, shift)
    y = spread(g, t * k, d, dtype, pitch and pitch + 3, shift)
    # No row behind the last expert's is read, whatever it holds.
    y[int(offsets[-1]):] = float("nan")
    o, p = offsets.cuda(), positions.cuda()
    w = weights.cuda() if weighted else None

    buffer, rows = out_like(t * k, d, dtype)
    assert layers.expert_rows_device(x, stride(x), o, p, w, rows, t, e, k, d, code, s) == 1
    assert torch.equal(rows.cpu(), plain_rows(x.cpu(), positions, weights))
    untouched(buffer)

    v = plain_picked(y.cpu(), positions)
    for residual in (None, x):
        buffer, out = out_like(t, d, dtype)
        assert layers.expert_sum_device(y, stride(y), p, w, residual, stride(x), out, t, k, d,
                                        code, s) == 1
        check_sum(out.cpu(), v, weights, None if residual is None else x.cpu(), dtype)
        untouched(buffer)
    assert int(offsets[-1]) > 0 or torch.equal(out, x)

    for dots in (True, False):
        buffer, dx = out_like(t, d, dtype)
        dbuffer, dw = out_like(t, k, torch.float32)
        assert layers.expert_rows_backward_device(y, stride(y), x if dots else None, stride(x),
                                                  p, w, dx, dw if dots else None, t, k, d, code,
                                                  s) == 1
        check_sum(dx.cpu(), v, weights, None, dtype)
        if dots:
            check_dots(dw.cpu(), v, x.cpu(), dtype)
        untouched(buffer)
        untouched(dbuffer)
        buffer, drows = out_like(t * k, d, dtype)
        dbuffer, dw = out_like(t, k, torch.float32)
        assert layers.expert_sum_backward_device(x, stride(x), y if dots else None, stride(y), o,
                                                 p, w, drows, dw if dots else None, t, e, k, d,
                                                 code, s) == 1
        assert torch.equal(drows.cpu(), plain_rows(x.cpu(), positions, weights))
        if dots:
            check_dots(dw.cpu(), v, x.cpu(), dtype)
        untouched(buffer)
        untouched(dbuffer)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("t,e,k,d", [
    (1, 1, 1, 1), (1, 8, 2, 3), (3, 4, 2, 7), (5, 8, 3, 8), (2, 8, 1, 9), (64, 8, 2, 33),
    (17, 5, 5, 255), (9, 64, 8, 257), (130, 16, 4, 512), (33, 64, 9, 513), (7, 40, 32, 1001),
    (1, 64, 8, 4096), (5, 16, 17, 2055), (300, 3, 2, 64)])
def test_sizes(torch_cuda, t, e, k, d, dtype):
    run_all(t, e, k, d, dtype)
    run_all(t, e, k, d, dtype, weighted=False, pitch=d + 1, shift=1)


@pytest.mark.parametrize("missing", [0.0, 0.5, 1.0])
def test_missing(torch_cuda, missing):
    run_all(50, 8, 3, 130, torch.bfloat16, missing=missing)
    run_all(50, 8, 10, 5, torch.float32, missing=missing)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_many_tokens(torch_cuda, dtype):
    """Above the bound from which a wave has a token's dot products."""
    run_all(4097, 16, 2, 520, dtype)
    run_all(4200, 16, 9, 530, dtype, pitch=533)


def test_positions_outside(torch_cuda):
    """Positions outside the rows, or behind the last expert's, are no rows."""
    t, k, d = 4, 2, 40
    positions = torch.tensor([[0, 8], [-5, 1], [2, 2 ** 31 - 1], [6, 3]], dtype=torch.int32,
                             device="cuda")
    offsets = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    x = torch.randn(t, d, device="cuda")
    _, rows = out_like(t * k, d, torch.float32)
    assert layers.expert_rows_device(x, d * 4, offsets, positions, None, rows, t, 1, k, d, 0,
                                     now()) == 1
    want = torch.zeros_like(rows)
    want[0], want[1], want[2], want[3] = x[0], x[1], x[2], x[3]
    assert torch.equal(rows, want)
    y = torch.randn(t * k, d, device="cuda")
    out = torch.empty(t, d, device="cuda")
    assert layers.expert_sum_device(y, d * 4, positions, None, None, 0, out, t, k, d, 0, now()) == 1
    assert torch.equal(out, torch.stack([y[0], y[1], y[2], y[6] + y[3]]))
    # Ends past the rows, or below 0, count as all or none of them.
    for end in (-3, 2 ** 31 - 1):
        offsets.fill_(end)
        positions.copy_(torch.arange(t * k).view(t, k))
        assert layers.expert_rows_device(x, d * 4, offsets, positions, None, rows, t, 1, k, d, 0,
                                         now()) == 1
        assert torch.equal(rows, x.repeat_interleave(k, 0) if end > 0 else torch.zeros_like(rows))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_values_pass_as_they_are(torch_cuda, dtype):
    """Inf, NaN, -0 and subnormals: copied without weights, formula with."""
    x = torch.tensor([[float("inf"), float("nan"), -0.0, 1e-40, 6e-8, -float("inf"), 1.0, 2.0]],
                     device="cuda").to(dtype)
    offsets = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    positions = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    rows = torch.empty_like(x)
    raw = torch.int32 if dtype == torch.float32 else torch.int16
    assert layers.expert_rows_device(x, 0, offsets, positions, None, rows, 1, 1, 1, 8,
                                     layers.DTYPES[dtype], now()) == 1
    assert torch.equal(rows.view(raw), x.view(raw))
    w = torch.zeros(1, 1, device="cuda")
    out = torch.empty_like(x)
    assert layers.expert_sum_device(x, 0, positions, w, None, 0, out, 1, 1, 8,
                                    layers.DTYPES[dtype], now()) == 1
    assert torch.isnan(out[0, [0, 1, 5]]).all() and (out[0, [2, 3, 4, 6, 7]] == 0).all()


def test_broadcast_gradient(torch_cuda):
    """One gradient row for all tokens (stride 0), as the mean's."""
    g = torch.Generator().manual_seed(5)
    t, e, k, d = 37, 6, 2, 100
    offsets, positions = routing(g, t, e, k)
    dout = spread(g, 1, d, torch.float32)
    y = spread(g, t * k, d, torch.float32)
    drows, dw = torch.empty(t * k, d, device="cuda"), torch.empty(t, k, device="cuda")
    assert layers.expert_sum_backward_device(dout, 0, y, d * 4, offsets.cuda(), positions.cuda(),
                                             None, drows, dw, t, e, k, d, 0, now()) == 1
    full = dout.cpu().expand(t, d)
    assert torch.equal(drows.cpu(), plain_rows(full.contiguous(), positions, None))
    check_dots(dw.cpu(), plain_picked(y.cpu(), positions), full, torch.float32)


def test_gradients_by_differences(torch_cuda):
    """Everything is linear in each argument: central differences are exact but
    for the roundings of the outputs, divided by the step."""
    g = torch.Generator().manual_seed(9)
    t, e, k, d, h = 6, 5, 3, 20, 0.25
    offsets, positions = routing(g, t, e, k, 0.2)
    o, p = offsets.cuda(), positions.cuda()
    x, dout = (torch.randn(t, d, generator=g) for _ in range(2))
    y, drows = (torch.randn(t * k, d, generator=g) for _ in range(2))
    w = torch.rand(t, k, generator=g)
    y[int(offsets[-1]):] = 0

    def rows_of(x, w):
        rows = torch.empty(t * k, d, device="cuda")
        assert layers.expert_rows_device(x.cuda(), d * 4, o, p, w.cuda(), rows, t, e, k, d, 0,
                                         now()) == 1
        return (rows.cpu().double() * drows.double()).sum()

    def sum_of(y, w):
        out = torch.empty(t, d, device="cuda")
        assert layers.expert_sum_device(y.cuda(), d * 4, p, w.cuda(), None, 0, out, t, k, d, 0,
                                        now()) == 1
        return (out.cpu().double() * dout.double()).sum()

    def slope(f, args, which, i):
        ends = []
        for sign in (1, -1):
            moved = [a.clone() for a in args]
            moved[which].view(-1)[i] += sign * h
            ends.append(f(*moved))
        return float(ends[0] - ends[1]) / (2 * h)

    dx, dw1 = torch.empty(t, d, device="cuda"), torch.empty(t, k, device="cuda")
    assert layers.expert_rows_backward_device(drows.cuda(), d * 4, x.cuda(), d * 4, p, w.cuda(),
                                              dx, dw1, t, k, d, 0, now()) == 1
    dy, dw2 = torch.empty(t * k, d, device="cuda"), torch.empty(t, k, device="cuda")
    assert layers.expert_sum_backward_device(dout.cuda(), d * 4, y.cuda(), d * 4, o, p, w.cuda(),
                                             dy, dw2, t, e, k, d, 0, now()) == 1
    # Each output is off by (k + 2) u of at most 3 * 4.5 * 1, times a gradient
    # of 4.5, over the d columns of the tokens that move (k rows of one).
    bound = 2 * k * d * (k + 2) * U * 13.5 * 4.5 / (2 * h) + 1e-5
    for f, args, grads in ((rows_of, (x, w), (dx, dw1)), (sum_of, (y, w), (dy, dw2))):
        for which, grad in enumerate(grads):
            flat = grad.cpu().view(-1)
            for i in range(0, flat.numel(), 7):
                assert abs(slope(f, args, which, i) - float(flat[i])) <= bound


def test_same_every_time_and_on_another_stream(torch_cuda):
    g = torch.Generator().manual_seed(3)
    t, e, k, d = 700, 12, 4, 515
    offsets, positions = (v.cuda() for v in routing(g, t, e, k, 0.1))
    x, y = spread(g, t, d, torch.bfloat16), spread(g, t * k, d, torch.bfloat16)
    w = torch.rand(t, k, generator=g).cuda()

    def once(stream):
        drows, dx, out = torch.empty_like(y), torch.empty_like(x), torch.empty_like(x)
        dw, dv = torch.empty_like(w), torch.empty_like(w)
        assert layers.expert_sum_backward_device(x, d * 2, y, d * 2, offsets, positions, w, drows,
                                                 dw, t, e, k, d, 1, stream) == 1
        assert layers.expert_rows_backward_device(y, d * 2, x, d * 2, positions, w, dx, dv, t, k,
                                                  d, 1, stream) == 1
        assert layers.expert_sum_device(y, d * 2, positions, w, x, d * 2, out, t, k, d, 1,
                                        stream) == 1
        return drows, dx, out, dw, dv

    first = once(now())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        others = [once(side) for _ in range(3)]
    torch.cuda.synchronize()
    for other in others:
        assert all(torch.equal(a, b) for a, b in zip(first, other))


def test_graph(torch_cuda):
    """Captured once, replayed on other inputs, with eager calls between."""
    g = torch.Generator().manual_seed(4)
    t, e, k, d = 256, 8, 2, 256
    offsets, positions = (v.cuda() for v in routing(g, t, e, k))
    x = spread(g, t, d, torch.bfloat16)
    w = torch.rand(t, k, generator=g).cuda()
    rows = torch.empty(t * k, d, dtype=torch.bfloat16, device="cuda")
    out, dw = torch.empty_like(x), torch.empty_like(w)

    def step():
        s = now()
        assert layers.expert_rows_device(x, d * 2, offsets, positions, None, rows, t, e, k, d, 1,
                                         s) == 1
        assert layers.expert_sum_device(rows, d * 2, positions, w, x, d * 2, out, t, k, d, 1,
                                        s) == 1
        assert layers.expert_rows_backward_device(rows, d * 2, x, d * 2, positions, w, out, dw, t,
                                                  k, d, 1, s) == 1

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        x.copy_(spread(g, t, d, torch.bfloat16))
        o, p = routing(g, t, e, k, 0.1 * i)
        offsets.copy_(o)
        positions.copy_(p)
        step()
        torch.cuda.synchronize()
        want = rows.clone(), out.clone(), dw.clone()
        for b in (rows, out, dw):
            b.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, (rows, out, dw)))


def test_past_four_gib(torch_cuda):
    """Rows past 2^32 bytes: the last tokens' rows at the far end."""
    t, k, d = 140000, 2, 8200
    code = layers.DTYPES[torch.bfloat16]
    x = torch.zeros(1, d, dtype=torch.bfloat16, device="cuda")
    x[0] = torch.arange(d) % 251
    positions = torch.arange(t * k, dtype=torch.int32, device="cuda").view(t, k).flip(0)
    positions = positions.contiguous()
    offsets = torch.tensor([0, t * k], dtype=torch.int32, device="cuda")
    rows = torch.full((t * k, d), 9.0, dtype=torch.bfloat16, device="cuda")
    assert rows.numel() * 2 > 2 ** 32
    assert layers.expert_rows_device(x, 0, offsets, positions, None, rows, t, 1, k, d, code,
                                     now()) == 1
    for i in range(0, t * k, 20000):
        assert (rows[i:i + 20000] == x).all()
    rows[t * k - 1] = 1
    rows[0] = 2
    out = torch.empty(t, d, dtype=torch.bfloat16, device="cuda")
    assert layers.expert_sum_device(rows, d * 2, positions, None, None, 0, out, t, k, d, code,
                                    now()) == 1
    assert torch.equal(out[0], (x[0].float() + 1).bfloat16())
    assert torch.equal(out[-1], (x[0].float() + 2).bfloat16())
    assert torch.equal(out[t // 2], (x[0].float() * 2).bfloat16())
