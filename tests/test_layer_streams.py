"""The layer entries' forms for what is used once, from 64 MB on, that read past
the caches: that the sizes below reach them, without a GPU (csrc/hip_names.c
notes the kernels that are launched), and on the GPU against plain results, with
rows that all differ, odd widths and rows farther apart than they are wide.

Tolerances, u = 2^-24, as in the entries' own tests: a looked-up value is one
fused product and sum; a gradient's sum has depth 64 + count / 512 + 20; a sum
of k products k + 2, a dot product n ceil(vectors / 64) + 10 for n elements in a
vector.
"""
from __future__ import annotations

import pytest
import torch

from turbinator_c_amd import layers

from . import launches
from .test_gpu_expert_rows import depth
from .test_gpu_int8 import plain_quantise, quantise, same

U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
STREAM = 64 << 20
AT = 4096

# dtype, tokens, entries, width
LOOKUPS = [("bf16", 40001, 1000, 1001), ("f32", 20001, 7000, 1003), ("f16", 300001, 50, 130),
           ("bf16", 4300001, 300, 9)]
# dtype, rows, k: a workgroup's rows and a wave's.
QUANTISED = [("bf16", 9001, 4001), ("f32", 2100, 8191), ("f16", 17001, 2049), ("bf16", 20001, 2048),
             ("f32", 50001, 501)]
# dtype, tokens, experts, k, width, whether a wave has a token
CHOICES = [("bf16", 20001, 24, 3, 1001, True), ("f32", 10001, 24, 3, 1001, True),
           ("f16", 30001, 8, 2, 700, True), ("bf16", 10001, 64, 8, 515, True),
           ("bf16", 60001, 64, 9, 131, False), ("f32", 100001, 8, 3, 61, False)]
# dtype, tokens, entries, width, whether a wave has a row
TABLES = [("bf16", 40001, 3000, 1001, True), ("f32", 20003, 50, 999, True),
          ("f16", 200001, 5000, 250, False), ("bf16", 300001, 20000, 130, False),
          ("f32", 1100001, 3, 17, False)]


@pytest.fixture(scope="module")
def noted(tmp_path_factory):
    with launches.noted(launches.load(tmp_path_factory.mktemp("names"))) as run:
        yield run


@pytest.mark.parametrize("dtype,t,entries,d", LOOKUPS)
def test_lookups_stream(dtype, t, entries, d):
    """The lookup's choice is an argument of its kernel: by size alone."""
    assert t * d * SIZE[dtype] > STREAM


@pytest.mark.parametrize("dtype,rows,k", QUANTISED)
def test_quantisation_streams(noted, dtype, rows, k):
    (launch,) = noted("int8_quantise_device", x=AT, row_stride=0, codes=AT, scales=AT, rows=rows,
                      k=k, dtype=layers.DTYPES[dtype])
    assert launch.name == f"quantise_kernel {dtype} {256 if k > 2048 else 64} 1"


# Kinds of experts' rows: the rows' gradient, the sum, its gradient, dots alone.
ROWS_BACK, SUM, SUM_BACK, DOT = 1, 2, 3, 4


@pytest.mark.parametrize("dtype,t,e,k,d,wave", CHOICES)
def test_experts_rows_stream(noted, dtype, t, e, k, d, wave):
    room = 2 if k <= 2 else 4 if k <= 4 else 8
    name = f"token_kernel {dtype} 16 {room} %d {64 if wave else 0} 1"
    common = dict(positions=AT, weights=AT, tokens=t, k=k, width=d, dtype=layers.DTYPES[dtype])
    back = noted("expert_rows_backward_device", drows=AT, drow_stride=0, x=AT, row_stride=0,
                 dx=AT, dweights=AT, **common)
    kinds = [ROWS_BACK] if k <= 8 else [DOT, SUM]
    assert [launch.name for launch in back] == [name % kind for kind in kinds]
    (launch,) = noted("expert_sum_device", rows=AT, row_stride=0, residual=AT, residual_stride=0,
                      out=AT, **common)
    assert launch.name == name % SUM
    (launch,) = noted("expert_sum_backward_device", dout=AT, dout_stride=0, rows=AT, row_stride=0,
                      offsets=AT, drows=AT, dweights=AT, n_experts=e, **common)
    assert launch.name == name % SUM_BACK


@pytest.mark.parametrize("dtype,t,entries,d,wave", TABLES)
def test_table_gradients_stream(noted, dtype, t, entries, d, wave):
    first, join = noted("embed_backward_device", dout=AT, dout_stride=0, ids=AT, order=AT,
                        ranges=AT, scale=1.0, dtable=AT, workspace=AT, tokens=t, entries=entries,
                        width=d, dtype=layers.DTYPES[dtype])
    assert first.name == f"grad_kernel {dtype} 16 {64 if wave else 0} 1"
    assert join.name == "join_kernel"


# --------------------------------------------------------------------------


def now():
    return torch.cuda.current_stream()


def generator(seed):
    return torch.Generator("cuda").manual_seed(seed)


def spread(g, m, d, dtype, extra=0, shift=0):
    """[m, d] on the GPU, rows d + extra elements apart from element `shift`
    on, NaN between them."""
    x = torch.full((m * (d + extra) + shift,), float("nan"), dtype=TYPES[dtype], device="cuda")
    rows = x[shift:].view(m, d + extra)[:, :d]
    rows.copy_(torch.randn((m, d), device="cuda", generator=g))
    return rows


def stride(x):
    return x.stride(0) * x.element_size()


def parts(n, each=20000):
    return [slice(i, min(n, i + each)) for i in range(0, n, each)]


@pytest.mark.gpu
@pytest.mark.parametrize("based", [True, False])
@pytest.mark.parametrize("dtype,t,entries,d", LOOKUPS)
def test_lookup(torch_cuda, dtype, t, entries, d, based):
    g, code, scale = generator(t), layers.DTYPES[dtype], 1.7
    ids = torch.randint(-1, entries + 1, (t,), device="cuda", generator=g).int()
    table = spread(g, entries, d, dtype, 1)
    base = spread(g, t, d, dtype, 3, 1) if based else None
    out = torch.full((t * d + 64,), 7.0, dtype=TYPES[dtype], device="cuda")
    assert layers.embed_device(ids, table, stride(table), base, stride(base) if based else 0,
                               scale, out, t, entries, d, code, now()) == 1
    torch.cuda.synchronize()
    assert (out[-64:] == 7).all()
    out = out[:-64].view(t, d)
    s = float(torch.tensor(scale))
    for part in parts(t, 20000 * 1000 // d):
        known = (ids[part] >= 0) & (ids[part] < entries)
        want = table.double()[torch.where(known, ids[part], 0).long()] * s
        want = torch.where(known[:, None], want, 0.0)
        if based:
            want = want + base[part].double()
        bound = ((U if dtype != "f32" else 0) + HALF[dtype]) * want.abs() * 1.01
        least = 2.0 ** -24 if dtype == "f16" else 1e-37
        assert ((out[part].double() - want).abs() <= bound + least).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,k", QUANTISED)
def test_quantise(torch_cuda, dtype, rows, k):
    g = generator(rows)
    x = spread(g, rows, k, dtype, 5, 1)
    x *= torch.exp2(4 * torch.randn((rows, 1), device="cuda", generator=g)).to(x.dtype)
    x[7, 3], x[rows - 2, k - 1] = float("inf"), float("nan")
    codes, scales = quantise(x)
    # plain_quantise, in parts for the host's memory.
    for part in parts(rows, 5000):
        want_codes, want_scales = plain_quantise(x[part])
        assert same(scales[part].cpu().numpy(), want_scales)
        assert same(codes[part].cpu().numpy(), want_codes)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,t,e,k,d,wave", CHOICES)
def test_experts_rows(torch_cuda, dtype, t, e, k, d, wave):
    g, code, typ = generator(t), layers.DTYPES[dtype], TYPES[dtype]
    experts = torch.rand((t, e), device="cuda", generator=g).argsort(1)[:, :k]
    experts[torch.rand((t, k), device="cuda", generator=g) < 0.1] = e
    order = experts.reshape(-1).sort(stable=True)
    at = torch.arange(t * k, device="cuda")
    positions = torch.empty_like(at).scatter_(0, order.indices,
                                              torch.where(order.values < e, at, -1))
    positions = positions.view(t, k).int()
    ends = torch.searchsorted(order.values, torch.arange(e + 1, device="cuda")).int()
    weights = torch.randn((t, k), device="cuda", generator=g)
    x, y = spread(g, t, d, dtype, 2), spread(g, t * k, d, dtype, 1, 1)
    y[int(ends[-1]):] = float("nan")

    def made(*shape, dtype=typ):
        return torch.full(shape, 7.0, dtype=dtype, device="cuda")

    dx, out, drows = made(t, d), made(t, d), made(t * k, d)
    dw, dv = made(t, k, dtype=torch.float32), made(t, k, dtype=torch.float32)
    assert layers.expert_rows_backward_device(y, stride(y), x, stride(x), positions, weights, dx,
                                              dw, t, k, d, code, now()) == 1
    assert layers.expert_sum_device(y, stride(y), positions, weights, x, stride(x), out, t, k, d,
                                    code, now()) == 1
    assert layers.expert_sum_backward_device(x, stride(x), y, stride(y), ends, positions, weights,
                                             drows, dv, t, e, k, d, code, now()) == 1
    least = 2.0 ** -24 if dtype == "f16" else 1e-37
    assert (drows[int(ends[-1]):] == 0).all()
    for part in parts(t, 2000):
        p, w, token = positions[part], weights[part].double(), x[part].double()
        live = p >= 0
        v = torch.where(live[..., None], y[p.clamp(min=0).long()].double(), 0.0)
        terms = v * w[..., None]
        for got, residual in ((dx, 0 * token), (out, token)):
            want, size = terms.sum(1) + residual, terms.abs().sum(1) + residual.abs()
            bound = (k + 2) * U * size * 1.001 + HALF[dtype] * want.abs() * 1.01 + least
            assert ((got[part].double() - want).abs() <= bound).all()
        dots = v * token[:, None, :]
        bound = depth(d, typ) * U * dots.abs().sum(2) * 1.001 + 1e-37
        for got in (dw, dv):
            assert ((got[part].double() - dots.sum(2)).abs() <= bound).all()
        row = (x[part].float()[:, None, :] * weights[part][..., None]).to(typ)
        assert torch.equal(drows[p[live].long()], row[live])


def sums(at, rows, entries):
    if entries <= 50:
        return torch.stack([rows[at == v].sum(0) for v in range(entries)])
    return rows.new_zeros(entries, rows.shape[1]).index_add_(0, at, rows)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,t,entries,d,wave", TABLES)
def test_table_gradient(torch_cuda, dtype, t, entries, d, wave):
    g, scale = generator(t), 0.6
    # Each entry about in proportion to 1 / its number, some tokens without.
    rank = torch.exp(torch.rand(t, device="cuda", generator=g) *
                     torch.tensor(entries + 1.0).log().item())
    ids = rank.long().clamp(1, entries) - 1
    ids = torch.where(torch.rand(t, device="cuda", generator=g) < 0.02, -1, ids).int()
    dout = spread(g, t, d, dtype, 3, 1)
    dout[ids < 0] = float("nan")
    order = torch.empty(t, dtype=torch.int32, device="cuda")
    ranges = torch.empty(entries, 2, dtype=torch.int32, device="cuda")
    need = max(layers.embed_order_workspace_bytes(t, entries),
               layers.embed_backward_workspace_bytes(t, entries, d))
    space = torch.empty(need, dtype=torch.uint8, device="cuda")
    dtable = torch.full((entries * d + 64,), 7.0, device="cuda")
    assert layers.embed_order_device(ids, order, ranges, space, t, entries, now()) == 1
    assert layers.embed_backward_device(dout, stride(dout), ids, order, ranges, scale, dtable,
                                        space, t, entries, d, layers.DTYPES[dtype], now()) == 1
    torch.cuda.synchronize()
    assert (dtable[-64:] == 7).all()
    live = ids >= 0
    at, rows = ids[live].long(), dout[live].double()
    want, size = (sums(at, v, entries) * float(torch.tensor(scale)) for v in (rows, rows.abs()))
    count = torch.bincount(at, minlength=entries)[:, None]
    bound = (64 + count / 512 + 20) * U * size * 1.001
    assert ((dtable[:-64].view(entries, d).double() - want).abs() <= bound).all()


@pytest.mark.gpu
def test_table_gradient_past_four_gib(torch_cuda):
    """Tokens past 2^32 bytes, each with a row of its own: whole numbers by the
    token's number, whose sums are exact."""
    t, entries, d = 600001, 1001, 4099
    dout = torch.empty((t, d), dtype=torch.bfloat16, device="cuda")
    assert dout.numel() * 2 > 2 ** 32
    columns = torch.arange(d, device="cuda") % 5
    number = torch.arange(t, device="cuda")
    for part in parts(t):
        dout[part] = ((number[part] * 7919 >> 5) % 13 - 6)[:, None] + columns
    ids = ((number * 31) % 1009).clamp(max=entries - 1).int()
    ids[::3] = 5
    order = torch.empty(t, dtype=torch.int32, device="cuda")
    ranges = torch.empty(entries, 2, dtype=torch.int32, device="cuda")
    need = max(layers.embed_order_workspace_bytes(t, entries),
               layers.embed_backward_workspace_bytes(t, entries, d))
    space = torch.empty(need, dtype=torch.uint8, device="cuda")
    dtable = torch.empty(entries, d, device="cuda")
    assert layers.embed_order_device(ids, order, ranges, space, t, entries, now()) == 1
    assert layers.embed_backward_device(dout, d * 2, ids, order, ranges, 1.0, dtable, space, t,
                                        entries, d, 1, now()) == 1
    # Sums of at most 2^21 numbers below 11: below 2^24.
    value = torch.zeros(entries, dtype=torch.int64, device="cuda")
    value.index_add_(0, ids.long(), (number * 7919 >> 5) % 13 - 6)
    count = torch.bincount(ids.long(), minlength=entries)
    want = value[:, None] + count[:, None] * columns
    assert want.abs().max() < 2 ** 24
    assert torch.equal(dtable, want.float())
