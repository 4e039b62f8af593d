"""Pointers to 32-bit values (ids, positions, offsets, weights, scales) off four
bytes are refused before anything is launched, as hip_layers.h says: uniform
loads would read them from the four bytes before.  Without a GPU."""
from __future__ import annotations

import ctypes

import pytest

from turbinator_c_amd import layers

from . import launches
from .test_expert_embed_int8_refusals import (AT, EMBED, EMBED_BACK, ORDER, PRODUCT, ROWS,
                                              ROWS_BACK, SUM, SUM_BACK)

WORDS = [("expert_rows_device", ROWS, ("offsets", "positions", "weights")),
         ("expert_rows_backward_device", ROWS_BACK, ("positions", "weights", "dweights")),
         ("expert_sum_device", SUM, ("positions", "weights")),
         ("expert_sum_backward_device", SUM_BACK, ("offsets", "positions", "weights", "dweights")),
         ("embed_device", EMBED, ("ids",)),
         ("embed_order_device", ORDER, ("ids", "order")),
         ("embed_backward_device", EMBED_BACK, ("ids", "order", "dtable")),
         ("int8_product_device", PRODUCT, ("a_scales", "rows", "w_scales", "offsets", "bias",
                                           "row_scale")),
         ("mx4_product_device", PRODUCT, ("a_scales", "rows", "w_scales", "offsets", "bias",
                                          "row_scale"))]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    return launches.load(tmp_path_factory.mktemp("names"))


@pytest.mark.parametrize("entry,args,word", [(e, a, w) for e, a, words in WORDS for w in words],
                         ids=lambda v: v if isinstance(v, str) else "")
def test_off_four_bytes(lib, entry, args, word):
    count = ctypes.c_int.in_dll(lib, "names_launches")
    with launches.noted(lib) as run:
        assert run(entry, **{**args, word: AT + 4})
        count.value = 0
        for off in (1, 2, 3):
            assert getattr(layers, entry)(**{**args, word: AT + off}) == 0
        assert count.value == 0
