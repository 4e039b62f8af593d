"""Refusals of the entries for experts' rows, embeddings and 8-bit rows
(hip_layers.h), their sizes and their launches, without a GPU: the entries'
objects linked against a stand-in for the HIP runtime (csrc/hip_stub.c), which
counts launches and takes them all."""
from __future__ import annotations

import ctypes
import subprocess

import pytest

from turbinator_c_amd import build, layers, native

AT = 4096  # an aligned address; never read
BIG = 2 ** 31
ROWS = dict(x=AT, row_stride=64, offsets=AT, positions=AT, weights=None, rows=AT, tokens=5,
            n_experts=8, k=2, width=16, dtype=0)
ROWS_BACK = dict(drows=AT, drow_stride=64, x=AT, row_stride=64, positions=AT, weights=None,
                 dx=AT, dweights=AT, tokens=5, k=2, width=16, dtype=0)
SUM = dict(rows=AT, row_stride=64, positions=AT, weights=None, residual=None, residual_stride=0,
           out=AT, tokens=5, k=2, width=16, dtype=0)
SUM_BACK = dict(dout=AT, dout_stride=64, rows=AT, row_stride=64, offsets=AT, positions=AT,
                weights=None, drows=AT, dweights=AT, tokens=5, n_experts=8, k=2, width=16,
                dtype=0)
EMBED = dict(ids=AT, table=AT, table_stride=64, base=None, base_stride=0, scale=1.0, out=AT,
             tokens=5, entries=7, width=16, dtype=0)
ORDER = dict(ids=AT, order=AT, ranges=AT, workspace=AT, tokens=5, entries=7)
EMBED_BACK = dict(dout=AT, dout_stride=64, ids=AT, order=AT, ranges=AT, scale=1.0, dtable=AT,
                  workspace=AT, tokens=5, entries=7, width=16, dtype=0)
QUANT = dict(x=AT, row_stride=64, codes=AT, scales=AT, rows=3, k=16, dtype=0)
VALUES = dict(codes=AT, scales=AT, values=AT, rows=3, k=16, dtype=0)
PRODUCT = dict(a_codes=AT, a_scales=AT, a_rows=4, rows=None, w_codes=AT, w_scales=AT,
               offsets=None, bias=None, row_scale=None, out=AT, m=4, n=8, k=16, experts=1, act=0,
               dtype=0)



@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    lib = tmp_path_factory.mktemp("stub") / "entries.so"
    objects = [build.BUILD / f"{name}.hip.o" for name in ("expert_rows", "embed", "int8")]
    source = build.GPU_CHECKS / "hip_stub.c"
    stub_object = lib.with_suffix(".o")
    subprocess.run(["gcc", "-O1", "-fPIC", "-c", str(source), "-o", str(stub_object)], check=True)
    subprocess.run(["g++", "-shared", "-o", str(lib), *map(str, objects), str(stub_object)],
                   check=True)
    names = ("expert_rows", "expert_sum", "embed", "int8")
    return native._load(lib, {n: v for n, v in native.HIP_SIGNATURES.items()
                              if n.startswith(tuple(f"tb_hip_{x}" for x in names))})


@pytest.fixture(autouse=True)
def stubbed(stub, monkeypatch):
    monkeypatch.setattr(layers, "hip_lib", lambda: stub)
    for name in ("stub_launches", "stub_most_threads", "stub_most_shared"):
        ctypes.memset(ctypes.addressof(ctypes.c_char.in_dll(stub, name)), 0,
                      4 if name == "stub_launches" else 8)
    return stub


def launches(stub):
    return ctypes.c_int.in_dll(stub, "stub_launches").value


def refused(entry, args, change):
    status = entry(**{**args, **change})
    return status == 0 and launches(layers.hip_lib()) == 0


TAKEN = [("expert_rows_device", ROWS), ("expert_rows_backward_device", ROWS_BACK),
         ("expert_sum_device", SUM), ("expert_sum_backward_device", SUM_BACK),
         ("embed_device", EMBED), ("embed_order_device", ORDER),
         ("embed_backward_device", EMBED_BACK), ("int8_quantise_device", QUANT),
         ("int8_values_device", VALUES), ("int8_product_device", PRODUCT)]


@pytest.mark.parametrize("name,args", TAKEN, ids=[n for n, _ in TAKEN])
def test_arguments_that_are_taken(stubbed, name, args):
    """What the changes below are made to is taken."""
    assert getattr(layers, name)(**args) == 1 and launches(stubbed) >= 1


@pytest.mark.parametrize("entry,change", [
    ("expert_rows_backward_device", dict(dweights=None, x=None)),
    ("expert_rows_backward_device", dict(k=32, weights=AT)),
    ("expert_sum_backward_device", dict(dweights=None, rows=None)),
    ("expert_sum_backward_device", dict(dout_stride=0)),
    ("embed_device", dict(table_stride=0, base=AT + 4, base_stride=4)),
    ("expert_rows_device", dict(tokens=2 ** 26, k=31, width=4096, n_experts=1024)),
    ("expert_rows_device", dict(tokens=2 ** 31 - 1, k=1, width=3)),
    ("expert_sum_device", dict(tokens=2 ** 31 - 1, k=1, width=70)),
    ("expert_sum_backward_device", dict(tokens=1, k=1, width=2 ** 31 - 1)),
    ("embed_device", dict(tokens=2 ** 31 - 1, entries=2 ** 20, width=1)),
    ("embed_order_device", dict(tokens=2 ** 31 - 1, entries=2 ** 20)),
    ("embed_order_device", dict(tokens=4097, entries=1024)),
    ("embed_backward_device", dict(tokens=2 ** 31 - 1, entries=2 ** 20, width=5000)),
    ("embed_backward_device", dict(tokens=1, entries=2 ** 20, width=2 ** 31 - 1)),
    ("int8_quantise_device", dict(rows=2 ** 31 - 1, k=131072)),
    ("int8_quantise_device", dict(rows=2 ** 31 - 1, k=1)),
    ("int8_values_device", dict(rows=2 ** 31 - 1, k=131072)),
    ("int8_product_device", dict(a_rows=2 ** 31 - 1, m=2 ** 31 - 1, n=128, k=64)),
    ("int8_product_device", dict(a_rows=2 ** 20, m=2 ** 20, n=2 ** 18, k=131072)),
    ("int8_product_device", dict(a_rows=1, m=1, n=2 ** 31 - 1, k=1)),
    ("int8_product_device", dict(a_rows=1, rows=AT, m=2 ** 30, n=2 ** 8, offsets=AT,
                                 experts=1024))], ids=str)
def test_the_largest_launches_fit(stubbed, entry, change):
    """A dimension of a grid holds less than 2^32 threads, a workgroup 64 KB of
    LDS that it asks for when it is launched."""
    assert getattr(layers, entry)(**{**dict(TAKEN)[entry], **change}) == 1
    assert 0 < ctypes.c_double.in_dll(stubbed, "stub_most_threads").value < 2 ** 32
    assert ctypes.c_size_t.in_dll(stubbed, "stub_most_shared").value <= 65536


CHOICES = [dict(tokens=0), dict(tokens=BIG // 2), dict(k=0), dict(k=33), dict(width=0),
           dict(width=BIG), dict(dtype=3), dict(dtype=-1)]
EXPERTS = [dict(n_experts=0), dict(n_experts=1025), dict(offsets=None)]


@pytest.mark.parametrize("change", CHOICES + EXPERTS + [
    dict(x=None), dict(positions=None), dict(rows=None), dict(x=AT + 2), dict(rows=AT + 1),
    dict(row_stride=66), dict(dtype=1, x=AT + 1), dict(dtype=2, row_stride=33)], ids=str)
def test_rows(change):
    assert refused(layers.expert_rows_device, ROWS, change)


@pytest.mark.parametrize("change", CHOICES + [
    dict(drows=None), dict(x=None), dict(positions=None), dict(dx=None), dict(drows=AT + 2),
    dict(x=AT + 2), dict(dx=AT + 3), dict(dweights=AT + 2), dict(drow_stride=30), dict(row_stride=30)], ids=str)
def test_rows_backward(change):
    assert refused(layers.expert_rows_backward_device, ROWS_BACK, change)


@pytest.mark.parametrize("change", CHOICES + [
    dict(rows=None), dict(positions=None), dict(out=None), dict(rows=AT + 2), dict(out=AT + 2),
    dict(row_stride=63), dict(residual=AT + 1), dict(residual=AT, residual_stride=2)], ids=str)
def test_sum(change):
    assert refused(layers.expert_sum_device, SUM, change)


@pytest.mark.parametrize("change", CHOICES + EXPERTS + [
    dict(dout=None), dict(rows=None), dict(positions=None), dict(drows=None), dict(dout=AT + 2),
    dict(rows=AT + 2), dict(drows=AT + 2), dict(dweights=AT + 1), dict(dout_stride=62), dict(row_stride=62)], ids=str)
def test_sum_backward(change):
    assert refused(layers.expert_sum_backward_device, SUM_BACK, change)


SIZES = [dict(tokens=0), dict(tokens=BIG), dict(entries=0), dict(entries=2 ** 20 + 1)]
WIDTHS = [dict(width=0), dict(width=BIG), dict(dtype=3), dict(dtype=-1)]


@pytest.mark.parametrize("change", SIZES + WIDTHS + [
    dict(ids=None), dict(table=None), dict(out=None), dict(table=AT + 2), dict(out=AT + 2),
    dict(base=AT + 2), dict(table_stride=66), dict(base=AT, base_stride=66)], ids=str)
def test_embed(change):
    assert refused(layers.embed_device, EMBED, change)


@pytest.mark.parametrize("change", SIZES + [
    dict(ids=None), dict(order=None), dict(ranges=None), dict(workspace=None),
    dict(ranges=AT + 4), dict(workspace=AT + 8)], ids=str)
def test_embed_order(change):
    assert refused(layers.embed_order_device, ORDER, change)


@pytest.mark.parametrize("change", SIZES + WIDTHS + [
    dict(dout=None), dict(ids=None), dict(order=None), dict(ranges=None), dict(dtable=None),
    dict(workspace=None), dict(workspace=AT + 4), dict(ranges=AT + 4), dict(dout=AT + 2),
    dict(dtable=AT + 2), dict(dout_stride=66), dict(dtype=1, dout_stride=65)], ids=str)
def test_embed_backward(change):
    assert refused(layers.embed_backward_device, EMBED_BACK, change)


@pytest.mark.parametrize("tokens,entries", [(1, 1), (1, 2 ** 20), (4097, 1024), (163840, 32768),
                                            (2 ** 24, 2 ** 20), (2 ** 31 - 1, 2 ** 20)])
def test_embed_workspaces(tokens, entries):
    need = layers.embed_order_workspace_bytes(tokens, entries)
    # The first pass's order, and 256 segments' counts of 1,024 digits and none.
    assert 0 < need <= 4 * tokens + 4 * 256 * 1025 + 48 and need % 16 == 0
    for width in (1, 3, 1024):
        # Two sums for each 32 tokens at the most.
        need = layers.embed_backward_workspace_bytes(tokens, entries, width)
        assert 0 < need <= (tokens // 32 + 1) * 2 * (width + 3) * 4 and need % 16 == 0


def test_embed_workspace_refusals():
    for args in ((0, 5), (BIG, 5), (5, 0), (5, 2 ** 20 + 1)):
        assert layers.embed_order_workspace_bytes(*args) == 0
        assert layers.embed_backward_workspace_bytes(*args, 8) == 0
    assert layers.embed_backward_workspace_bytes(5, 5, 0) == 0
    assert layers.embed_backward_workspace_bytes(5, 5, BIG) == 0


K = [dict(k=0), dict(k=131073), dict(dtype=3), dict(dtype=-1)]


@pytest.mark.parametrize("change", K + [
    dict(x=None), dict(codes=None), dict(scales=None), dict(rows=0), dict(rows=BIG),
    dict(codes=AT + 8), dict(scales=AT + 2), dict(x=AT + 2), dict(row_stride=66),
    dict(dtype=1, row_stride=33)], ids=str)
def test_quantise(change):
    assert refused(layers.int8_quantise_device, QUANT, change)


@pytest.mark.parametrize("change", K + [
    dict(codes=None), dict(scales=None), dict(values=None), dict(rows=0), dict(rows=BIG),
    dict(codes=AT + 4), dict(scales=AT + 1), dict(values=AT + 2)], ids=str)
def test_values(change):
    assert refused(layers.int8_values_device, VALUES, change)


@pytest.mark.parametrize("change", K + [
    dict(a_codes=None), dict(a_scales=None), dict(w_codes=None), dict(w_scales=None),
    dict(out=None), dict(a_rows=0), dict(a_rows=BIG, m=BIG), dict(m=0), dict(m=5), dict(n=0),
    dict(n=BIG), dict(experts=0), dict(experts=1025, offsets=AT), dict(experts=2),
    dict(experts=2, offsets=AT, n=2 ** 30), dict(act=3), dict(act=-1), dict(a_codes=AT + 8),
    dict(w_codes=AT + 8), dict(a_scales=AT + 1), dict(w_scales=AT + 2), dict(out=AT + 2),
    dict(rows=AT, m=BIG), dict(rows=AT, m=2 ** 30, n=2 ** 9)], ids=str)
def test_product(change):
    assert refused(layers.int8_product_device, PRODUCT, change)


def test_padding():
    for k, kp in ((1, 128), (127, 128), (128, 128), (129, 256), (2000, 2048), (131072, 131072)):
        assert layers.int8_padded(k) == kp
