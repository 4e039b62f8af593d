"""examples/routed_tokens.py: the layer entries together.  Each stage against
64 bits on what the stage before it left, so that a tolerance covers one stage
only; and a captured chain of the entries against eager calls.

Tolerances (u = 2^-24, b = 2^-8 half a unit of bfloat16 relative).  Group norm:
64 * 32 values, sums within 2^-18 of their size, SiLU slope at most 1.1 and
fast exponentials within 8 u: b |y| + 2^-16 (1 + |z|).  Products: 2^-20 sum
|a w|, rounding b.  Gradients: two more sums of the group, the same class, of
the largest term.
"""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

from turbinator_c_amd import layers, synth  # noqa: E402

pytestmark = pytest.mark.gpu
B = 2.0 ** -8


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "routed_tokens.py"
    spec = importlib.util.spec_from_file_location("routed_tokens", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.fixture(scope="module", params=[1, 3, 32])
def acted(example, request):
    batch = synth.make_batch(request.param, seed=11)
    cameras = batch.cameras.copy()
    cameras[0, :4096] = 0  # a black camera: no token of it is routed
    net = example.RoutedTokens(request.param)
    out = net.act(*(torch.from_numpy(a).cuda() for a in (batch.obs, batch.mission, cameras)))
    torch.cuda.synchronize()
    return example, net, out


def within(got, want, room):
    over = (got.double() - want).abs() - room
    assert torch.isfinite(got).all() and (over <= 0).all(), float(over.max())


def normed(example, net, planes):
    x = planes.double().view(net.images, example.PATCHES, example.GROUPS, -1)
    mean = x.mean((1, 3), keepdim=True)
    rstd = (x.var((1, 3), unbiased=False, keepdim=True) + example.EPS).rsqrt()
    h = ((x - mean) * rstd).view(net.images, example.PATCHES, example.WIDTH)
    return h * net.gamma.double() + net.beta.double(), h, rstd


def test_tokens(acted):
    example, net, _ = acted
    z, _, _ = normed(example, net, net.planes)
    y = z * torch.sigmoid(z)
    within(net.token.view_as(y), y, B * y.abs() + 2.0 ** -16 * (1 + z.abs()))


def test_routing(acted):
    example, net, _ = acted
    logits = net.logits.double()
    top = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :example.TOP]
    want = torch.where(net.valid[:, None], top, -1)
    assert torch.equal(net.experts.long(), want)
    assert int((want[:example.PATCHES] >= 0).sum()) == 0
    w = torch.softmax(logits.gather(1, top), 1) * net.valid[:, None]
    within(net.weights, w, 2.0 ** -20)
    # The stable order of the choices, those of no expert behind.
    flat = want.flatten()
    order = torch.sort(torch.where(flat < 0, example.EXPERTS, flat), stable=True).indices
    real = int((flat >= 0).sum())
    assert int(net.offsets[-1]) == real
    assert torch.equal(net.row_token[:real].long(), order[:real] // example.TOP)
    assert torch.equal(net.positions.flatten()[order[:real]].long(),
                       torch.arange(real, device="cuda"))
    assert torch.equal(net.row_weight[:real], net.weights.flatten()[order[:real]])


def expert_rows(example, net, a, w, n):
    """a's rows through their experts' matrices, and the sums of magnitudes."""
    w = w.values().double().view(example.EXPERTS, n, -1)
    out = torch.zeros(len(a), n, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(out)
    for x in range(example.EXPERTS):
        rows = slice(int(net.offsets[x]), int(net.offsets[x + 1]))
        out[rows] = a[rows] @ w[x].t()
        size[rows] = a[rows].abs() @ w[x].abs().t()
    return out, size


def test_experts_and_sum(acted):
    example, net, out = acted
    real = int(net.offsets[-1])
    a = net.token4.values().double()[net.row_token.long().clamp(min=0)]
    z, size = expert_rows(example, net, a, net.up, example.HIDDEN)
    bias = net.up_bias.double().view(example.EXPERTS, -1)
    expert = torch.bucketize(torch.arange(real, device="cuda"), net.offsets[1:].long(),
                             right=True)
    z[:real] += bias[expert]
    h = z * torch.sigmoid(z)
    within(net.hidden[:real], h[:real], B * h[:real].abs() + 2.0 ** -19 * (1 + size[:real]))
    assert not net.hidden[real:].any()
    y, size = expert_rows(example, net, net.hidden4.values().double(), net.down, example.WIDTH)
    w = net.row_weight.double()[:, None]
    within(net.part, y * w, B * (y * w).abs() + 2.0 ** -19 * size)
    there = (net.positions >= 0)[..., None]
    part = net.part.double()[net.positions.clamp(min=0).long()] * there
    total = net.token.double() + part.sum(1)
    # Two roundings to bfloat16: of the sum and of the result.
    within(out, total, 2 * B * (total.abs() + part.abs().sum(1)) + 1e-30)


def test_gradients(acted):
    example, net, out = acted
    torch.manual_seed(4)
    dout = torch.randn_like(out)
    got = net.learn(dout)
    # Router: the softmax of the picks' logits alone.
    logits = net.logits.double().requires_grad_()
    picks = net.experts.long().clamp(min=0)
    w = torch.softmax(logits.gather(1, picks), 1)
    dw = torch.where(net.valid[:, None], got["dweights"].double(), 0.0)
    want, = torch.autograd.grad((w * dw).sum(), logits)
    within(got["dlogits"], want, B * want.abs() + 2.0 ** -18 * (1 + dw.abs().sum(1, keepdim=True)))
    # Stem: group norm and SiLU.
    planes = net.planes.double().requires_grad_()
    gamma, beta = net.gamma.double().requires_grad_(), net.beta.double().requires_grad_()
    x = planes.view(net.images, example.PATCHES, example.GROUPS, -1)
    mean = x.mean((1, 3), keepdim=True)
    rstd = (x.var((1, 3), unbiased=False, keepdim=True) + example.EPS).rsqrt()
    h = ((x - mean) * rstd).view(net.images, example.PATCHES, example.WIDTH)
    z = h * gamma + beta
    dtoken = got["dtoken"].double().view_as(z)
    dx, dg, db = torch.autograd.grad((z * torch.sigmoid(z) * dtoken).sum(), (planes, gamma, beta))
    terms = (dtoken.abs() * 1.1 * gamma.detach().abs()).view(x.shape)
    rough = rstd.detach() * terms.amax((1, 3), keepdim=True) * (2 + h.detach().view(x.shape).abs())
    within(got["planes"], dx, B * dx.abs() + 2.0 ** -16 * rough.reshape(dx.shape))
    within(got["gamma"], dg, 2.0 ** -16 * (1.1 * dtoken.abs() * (1 + h.abs())).sum((0, 1)).detach())
    within(got["beta"], db, 2.0 ** -16 * (1.1 * dtoken.abs()).sum((0, 1)))


def test_captured(example):
    """The entries in a graph, replayed with eager work in between: other
    inputs each time, equal to eager calls bit for bit."""
    t, n, k, width, hidden = 700, 8, 2, 256, 192
    x = torch.randn(t, width, device="cuda").bfloat16()
    logits = torch.randn(t, n, device="cuda")
    w4 = example.FourBit(n * hidden, width).take(torch.randn(n * hidden, width, device="cuda"),
                                                  torch.cuda.current_stream())

    def make():
        def space(*shape, dtype=torch.float32):
            return torch.full(shape, -7, device="cuda").to(dtype)
        i32 = torch.int32
        return {"y": space(t, width, dtype=torch.bfloat16), "mean": space(t, 8), "rstd": space(t, 8),
                "e": space(t, k, dtype=i32), "w": space(t, k), "off": space(n + 1, dtype=i32),
                "tok": space(t * k, dtype=i32), "pos": space(t, k, dtype=i32), "rw": space(t * k),
                "out": space(t * k, hidden, dtype=torch.bfloat16), "dl": space(t, n),
                "x4": example.FourBit(t, width),
                "s1": space(layers.group_norm_workspace_bytes(t, 1, width, 8, 1), dtype=torch.uint8),
                "s2": space(layers.expert_order_workspace_bytes(t, n, k), dtype=torch.uint8)}

    def chain(b, stream):
        done = example.done
        done(layers.group_norm_device(x, 512, 512, None, None, b["y"], b["mean"], b["rstd"], b["s1"],
                                      t, 1, width, 8, 1e-5, 1, 1, stream))
        done(layers.route_device(logits, n * 4, None, None, b["e"], b["w"], t, n, k, 1, 1, 0, True,
                                 1.0, 0, stream))
        done(layers.expert_order_device(b["e"], b["w"], b["off"], b["tok"], b["pos"], b["rw"],
                                        b["s2"], t, n, k, stream))
        b["x4"].take(b["y"], stream)
        done(layers.mx4_product_device(b["x4"].codes, b["x4"].scales, t, b["tok"], w4.codes,
                                       w4.scales, b["off"], None, b["rw"], b["out"], t * k, hidden,
                                       width, n, 1, 1, stream))
        done(layers.route_backward_device(logits, n * 4, b["e"], b["w"], b["dl"], t, n, k, 0, True,
                                          1.0, 0, stream))

    kept, eager = make(), make()
    chain(kept, torch.cuda.current_stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain(kept, torch.cuda.current_stream())
    for turn in range(4):
        x.copy_(torch.randn(t, width, device="cuda"))
        logits.copy_(torch.randn(t, n, device="cuda"))
        graph.replay()
        chain(eager, torch.cuda.current_stream())
        torch.cuda.synchronize()
        for name in ("y", "mean", "rstd", "e", "w", "off", "tok", "pos", "rw", "out", "dl"):
            assert torch.equal(kept[name], eager[name]), (turn, name)
