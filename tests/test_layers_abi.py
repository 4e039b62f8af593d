"""Host side of the layer entries (hip_layers.h), no GPU: workspace sizes over
the whole range of arguments, and refusals that return before any HIP call."""
from __future__ import annotations

import random

from turbinator_c_amd import layers, native


def test_group_norm_workspace_sizes():
    rng = random.Random(5)
    for _ in range(4000):
        per, groups = rng.choice([1, 2, 3, 5, 8, 13, 64, 127, 512, 1000, 1023, 1024]), \
            rng.choice([1, 2, 3, 4, 7, 8, 16, 32, 64])
        images, pixels = rng.choice([1, 3, 1000]), rng.choice([1, 2, 100, 4097, 10 ** 6, 2 ** 31 - 1])
        for dtype in (0, 1, 2):
            for backward in (False, True):
                need = layers.group_norm_workspace_bytes(images, pixels, per * groups, groups,
                                                         dtype, backward)
                assert need > 0 and need % 16 == 0
                # At most 1,024 partial sums of each group or channel of an image.
                columns = per * groups if backward else groups
                assert need <= images * 1024 * columns * 8 + 128 * per * groups * 8 + 16


def test_group_norm_workspace_refusals():
    size = layers.group_norm_workspace_bytes
    assert size(0, 1, 8, 2, 0) == 0
    assert size(1, 0, 8, 2, 0) == 0
    assert size(1, 1, 8, 3, 0) == 0
    assert size(1, 1, 0, 1, 0) == 0
    assert size(1, 1, 8, 0, 0) == 0
    assert size(1, 1, 2050, 2, 0) == 0
    assert size(1, 1, 131072, 1024, 0) == 0
    assert size(1, 1, 8, 2, 3) == 0
    assert size(2 ** 31, 1, 8, 2, 0) == 0


def test_group_norm_refusals_without_gpu():
    lib = native.hip_lib()
    x, odd = 4096, 4098
    assert lib.tb_hip_group_norm_device(None, 32, 32, None, None, x, None, None, x, 1, 1, 8, 2,
                                        1e-5, 0, 0, None) == 0
    assert lib.tb_hip_group_norm_device(odd, 32, 32, None, None, x, None, None, x, 1, 1, 8, 2,
                                        1e-5, 0, 0, None) == 0
    assert lib.tb_hip_group_norm_device(x, 32, 32, None, None, x, None, None, None, 1, 1, 8, 2,
                                        1e-5, 0, 0, None) == 0
    assert lib.tb_hip_group_norm_device(x, 32, 32, None, None, x, None, None, x, 1, 1, 8, 2,
                                        0.0, 0, 0, None) == 0
    assert lib.tb_hip_group_norm_backward_device(x, 32, 32, x, 32, 32, None, None, None, x, x,
                                                 None, None, x, 1, 1, 8, 2, 0, 0, None) == 0
