"""What the embedding gradient's header says of its sums (hip_layers.h): the same
bits on every call with the same arguments, whatever the workspace held; and for
the same tokens among others, within the sums' bound of each other, where the
partial sums are cut at other places or another kernel runs.

Tolerance, u = 2^-24: each of the two is within (64 + count / 512 + 20) u of the
sum of magnitudes (at most 64 rows added in turn, such runs in at least 16
groups, those after one another, the scale).
"""
from __future__ import annotations

import pytest
import torch

from .test_gpu_embed import U, backward, order_of, spread

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("count,before,behind", [(33, 5, 9000), (500, 77, 40), (3000, 4000, 4000)])
def test_an_entry_among_others(torch_cuda, count, before, behind, dtype):
    g = torch.Generator().manual_seed(count)
    mine = spread(g, count, 70, dtype)

    def gradient(before, behind, entries):
        ids = torch.cat([torch.zeros(before), torch.full((count,), 1), torch.full((behind,), 2)])
        ids = ids.int().cuda()
        rows = [spread(g, n, 70, dtype) for n in (before, behind)]
        dout = torch.cat([rows[0], mine, rows[1]])
        order, ranges = order_of(ids, entries)
        first = backward(ids, order, ranges, dout, 0.6, entries)
        again = backward(ids, order, ranges, dout, 0.6, entries)
        assert torch.equal(first, again)
        return first[1].cpu().double()

    want = mine.cpu().double().sum(0) * float(torch.tensor(0.6))
    size = mine.cpu().double().abs().sum(0) * float(torch.tensor(0.6))
    bound = (64 + count / 512 + 20) * U * size * 1.001
    for got in (gradient(0, 0, 2), gradient(before, 0, 3), gradient(before, behind, 3),
                gradient(before, behind, 5000)):
        assert ((got - want).abs() <= bound).all()
