"""The layer entries together as examples/trained_experts.py uses them: each
entry's result against 64 bits on the very inputs it had, the gradients of the
whole step against automatic differentiation in 64 bits, acting in 8 bits, and
acting captured into a graph.

Tolerances, u = 2^-24.  Per entry as in the entries' own tests.  The whole step
in fp32: a gradient's path has at most nine sums of products, of at most 600
terms each, so each is off by at most 600 u of its sum of magnitudes; of terms
with random signs that sum is about sqrt(600) < 25 times the result's size:
9 * 600 * 25 u < 2^-6 of a gradient's norm.  (A term that is missing, or a wrong
scale, is off by the order of 1.)
"""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def example(torch_cuda):
    path = Path(__file__).resolve().parents[1] / "examples" / "trained_experts.py"
    spec = importlib.util.spec_from_file_location("trained_experts", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def reference(ex, net, planes, dout):
    """Gradients by automatic differentiation in 64 bits, the choice held fixed."""
    leaf = {n: v.detach().cpu().double().requires_grad_()
            for n, v in (("table", net.table), ("router", net.router), ("up", net.up),
                         ("down", net.down), ("planes", planes))}
    ids, experts = net.ids.cpu().long(), net.experts.cpu().long()
    there = (ids >= 0).double()[:, None]
    token = leaf["planes"] + ex.SCALE * leaf["table"][ids.clamp(min=0)] * there
    score = torch.softmax(token @ leaf["router"], 1).gather(1, experts.clamp(min=0))
    weights = score / score.sum(1, keepdim=True) * there
    weights.retain_grad()
    out = token
    for j in range(ex.TOP):
        e = experts[:, j].clamp(min=0)
        y = torch.zeros_like(token)
        for x in range(ex.EXPERTS):
            mine = (e == x).nonzero()[:, 0]
            h = torch.nn.functional.silu(token[mine] @ leaf["up"][x].T)
            y = y.index_add(0, mine, h @ leaf["down"][x].T)
        out = out + weights[:, j, None] * y
    out.backward(dout.cpu().double())
    grads = {n: v.grad for n, v in leaf.items()}
    grads["weights"] = weights.grad * there
    return out.detach(), grads


def near(got, want, share):
    got = got.cpu().double()
    return float((got - want).norm()) <= share * float(want.norm())


@pytest.mark.parametrize("environments", [1, 3])
def test_gradients(example, environments):
    ex = example
    planes, valid = ex.inputs(environments, torch.float32)
    net = ex.TrainedExperts(environments, torch.float32)
    out = net.forward(planes, valid)
    dout = torch.randn(out.shape, generator=torch.Generator().manual_seed(3)).cuda()
    grads = net.learn(dout)
    want_out, want = reference(ex, net, planes, dout)
    assert near(out, want_out, 2.0 ** -6)
    assert torch.equal(out[valid == 0], planes[valid == 0])
    for name, value in want.items():
        assert near(grads[name], value, 2.0 ** -6), name


def test_each_entry(example):
    """bf16, each entry on the inputs that it had."""
    ex = example
    planes, valid = ex.inputs(4)
    net = ex.TrainedExperts(4)
    out = net.forward(planes, valid).clone()
    dout = torch.randn(out.shape, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    grads = net.learn(dout)
    half = 2.0 ** -8
    ids, live = net.ids.cpu().long(), int(net.offsets[-1])
    positions, w = net.positions.cpu().long(), net.weights.cpu().double()
    there = positions >= 0
    assert torch.equal(there[:, 0], valid.cpu() != 0)

    want = planes.cpu().double()
    want[ids >= 0] += ex.SCALE * net.table.cpu().double()[ids[ids >= 0]]
    assert ((net.token.cpu().double() - want).abs() <= (half + U) * 1.01 * want.abs()).all()

    rows = net.rows.cpu()
    assert torch.equal(rows[:live], net.token.cpu()[net.row_token.cpu().long()[:live]])
    assert (rows[live:] == 0).all()

    part = net.part.cpu().double()[positions.clamp(min=0)] * there[..., None]
    terms = part * w[..., None]
    want = net.token.cpu().double() + terms.sum(1)
    size = net.token.cpu().double().abs() + terms.abs().sum(1)
    assert ((out.cpu().double() - want).abs() <= 4.1 * U * size + half * 1.01 * want.abs()).all()

    d = dout.cpu()
    dpart = (d.float()[:, None, :] * net.weights.cpu()[..., None]).bfloat16()
    assert torch.equal(net.dpart.cpu()[positions[there]], dpart[there])
    dots = part * d.double()[:, None, :]
    assert ((net.dweights.cpu().double() - dots.sum(2)).abs() <= 18 * U * dots.abs().sum(2)).all()
    drows = net.drows.cpu().double()[positions.clamp(min=0)] * there[..., None]
    want, size = drows.sum(1), drows.abs().sum(1)
    assert ((net.dtoken.cpu().double() - want).abs() <=
            4.1 * U * size + half * 1.01 * want.abs()).all()

    dplanes = grads["planes"].cpu().double()[ids >= 0] * ex.SCALE
    want, size = (torch.zeros(ex.PLACES, ex.WIDTH, dtype=torch.float64).index_add_(0, ids[ids >= 0], v)
                  for v in (dplanes, dplanes.abs()))
    assert ((net.dtable.cpu().double() - want).abs() <= 90 * U * size).all()


def test_acting_in_eight_bits(example):
    """The first product against the unrounded factors: each is off by at most
    half a step, scale / 2, and the activation's slope is at most 1.1."""
    ex = example
    planes, valid = ex.inputs(2)
    net = ex.TrainedExperts(2)
    trained = net.forward(planes, valid).clone()
    acted = net.act(planes, valid)
    live = int(net.offsets[-1])
    token = net.token.cpu().double()[net.row_token.cpu().long()[:live]]
    step = net.token8.scales.cpu().double()[net.row_token.cpu().long()[:live]][:, None] / 2 * 1.0001
    for e, (lo, hi) in enumerate(zip(net.ends, net.ends[1:])):
        up = net.up[e].cpu().double()
        up_step = net.up8.scales.view(ex.EXPERTS, -1)[e].cpu().double()[:, None] / 2 * 1.0001
        a, da = token[lo:hi], step[lo:hi].expand(-1, ex.WIDTH)
        want = torch.nn.functional.silu(a @ up.T)
        off = a.abs() @ up_step.expand_as(up).T + da @ (up.abs() + up_step).T
        got = net.hidden[lo:hi].cpu().double()
        assert ((got - want).abs() <= 1.1 * off + 2.0 ** -8 * 1.01 * (want.abs() + 1.1 * off) +
                1e-6).all()
    assert (net.hidden[live:] == 0).all()
    assert torch.equal(acted[valid == 0], trained[valid == 0])


def test_acting_in_a_graph(example):
    ex = example
    planes, valid = ex.inputs(2)
    net = ex.TrainedExperts(2)
    net.act(planes, valid)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        net.act(planes, valid)
    for seed in range(3, 6):
        new, mask = ex.inputs(2, seed=seed)
        planes.copy_(new)
        valid.copy_(mask)
        want = net.act(planes, valid).clone()
        torch.cuda.synchronize()
        net.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(net.out, want)
