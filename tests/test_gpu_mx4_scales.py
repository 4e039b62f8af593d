"""Every scale byte of the 4-bit form (hip_layers.h), those that quantisation
does not give among them: the values, and products with a factor of one."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from turbinator_c_amd import layers  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
CODES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_values_of_every_scale(torch_cuda, dtype):
    """256 rows, a scale each, of all sixteen codes.  Below 2^128 fp32 and bf16
    hold the values exactly; above, as in fp16 from 65,520 on, they are Inf."""
    k = 32
    codes = torch.zeros(256, 64, dtype=torch.uint8)
    codes[:, :8] = torch.tensor([0x10, 0x32, 0x54, 0x76, 0x98, 0xba, 0xdc, 0xfe])
    scales = torch.full((256, 4), 127, dtype=torch.uint8)
    scales[:, 0] = torch.arange(256)
    out = torch.empty(256, k, dtype=dtype, device="cuda")
    assert layers.mx4_values_device(codes.cuda(), scales.cuda(), out, 256, k,
                                    layers.DTYPES[dtype], torch.cuda.current_stream()) == 1
    unit = torch.exp2(torch.arange(256, dtype=torch.float64) - 127)
    unit[255] = float("nan")
    row = torch.cat([CODES, -CODES, torch.zeros(16, dtype=torch.float64)])
    want = unit[:, None] * row
    got = out.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    if dtype == torch.float16:
        want = want.to(torch.float16).double()
    else:
        want = torch.where(want.abs() < 2.0 ** 128, want, torch.inf * torch.sign(want))
    assert torch.equal(torch.nan_to_num(got, nan=0.0), torch.nan_to_num(want, nan=0.0))
